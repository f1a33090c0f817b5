"""Plain 64-bit forms of the context operators (cache append, decode and
prompt attention, the gated delta rule), in numpy, and the bounds of their
kernels' roundings.

A rounding to a type of p bits is off by at most half a step, HALF[dtype]
relative to the value.
"""
import numpy as np

import nmoe_hip as nh
from oracle import binding as B

HALF = {nh.F32: 2.0 ** -24, nh.BF16: 2.0 ** -8, nh.F16: 2.0 ** -11}
TINY = {nh.F32: 0.0, nh.BF16: 0.0, nh.F16: 2.0 ** -25}  # half the smallest step
NP = {nh.F32: np.float32, nh.BF16: np.uint16, nh.F16: np.float16}


def pack(a, dtype):
    """Values as the device holds them."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == nh.BF16:
        return B.f32_to_bf16(a.ravel()).reshape(a.shape)
    return a.astype(NP[dtype])


def value(a, dtype):
    """What packed values stand for, in 64 bits."""
    if dtype == nh.BF16:
        return B.bf16_to_f32(np.ascontiguousarray(a).ravel()).reshape(a.shape).astype(np.float64)
    return a.astype(np.float64)


def prepared(x, positions, inv_freq, rotary, interleaved, norm, weight, add_one, eps):
    """x [rows, heads, dim] normalised and rotated."""
    x = x.astype(np.float64)
    if norm:
        w = 1.0 if weight is None else weight + (1.0 if add_one else 0.0)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if rotary:
        half = rotary // 2
        a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
        angle = positions.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
        c, s, out = np.cos(angle), np.sin(angle), x.copy()
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        x = out
    return x


def attention(q, k, v, see, scale, dtype):
    """One head: q [nq, D] over k, v [nk, D], query i seeing keys j < see[i].
    Returns out, lse and the bound of out's error, element by element.

    The bound: scores are fp32 sums of D products (at most D half steps of the
    sum of their magnitudes) and times scale; exp2 of them after one more
    product is off by the score's absolute error and 2^-21; the weights round
    once to `dtype` for the products with v (half a step each, against the
    sum of p |v|), those are fp32 sums of at most nk terms, and the result
    rounds to `dtype`."""
    D = q.shape[1]
    out, tol = np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], v.shape[1]))
    lse = np.full(q.shape[0], -np.inf)
    for i in range(q.shape[0]):
        n = int(min(max(see[i], 0), k.shape[0]))
        if n == 0:
            continue
        s = (k[:n] @ q[i]) * scale
        mag = (np.abs(k[:n]) @ np.abs(q[i])).max() * abs(scale)
        top = s.max()
        p = np.exp(s - top)
        lse[i] = top + np.log(p.sum())
        p /= p.sum()
        out[i] = p @ v[:n]
        spread = p @ np.abs(v[:n])
        ds = (D + 8) * 2.0 ** -24 * mag
        rel = 2 * ds + 2.0 ** -20 + n ** 0.5 * 2.0 ** -23
        tol[i] = (HALF[dtype] + rel) * spread + HALF[dtype] * np.abs(out[i]) + 2 * HALF[dtype] ** 2 * spread + TINY[dtype]
    return out, lse, tol


def delta_rule(q, k, v, g, beta, scale, l2, eps, state):
    """One sequence, token by token: q, k [T, Hk, Dk], v [T, Hv, Dv], g, beta
    [T, Hv], state [Hv, Dk, Dv]; out [T, Hv, Dv] and the last state."""
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    if l2:
        q, k = (t / np.sqrt((t * t).sum(-1, keepdims=True) + eps) for t in (q, k))
    G = v.shape[1] // q.shape[1]
    q, k = np.repeat(q, G, 1), np.repeat(k, G, 1)
    S, out = state.astype(np.float64).copy(), np.zeros(v.shape)
    for t in range(v.shape[0]):
        S *= np.exp(g[t].astype(np.float64))[:, None, None]
        u = beta[t].astype(np.float64)[:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
        S += k[t][:, :, None] * u[:, None, :]
        out[t] = scale * np.einsum("hkv,hk->hv", S, q[t])
    return out, S
