"""Plain 64-bit forms of the operators on a cache in 8 bits (a step's pages,
the append), in numpy: codes as their definition has them (a sign, 4 bits of
exponent with bias 7, 3 of fraction; 0x7f and 0xff no number), loops where the
definition speaks of one after the other."""
import math

import numpy as np

LOW, HIGH = -117, 118  # a scale's least and greatest power of two
BLOCK = 16

CODES = np.array([(-1.0 if c & 128 else 1.0) * ((c & 7) * 2.0 ** -9 if (c >> 3 & 15) == 0 else
                                                (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10)) for c in range(256)])
CODES[[0x7F, 0xFF]] = np.nan


def codes_of(y):
    """The codes next to y, ties to the even one, the largest beyond it; NaN for what is no finite number."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.abs(np.where(np.isfinite(y), y, 0.0)), 448.0)
    _, e = np.frexp(a)  # a = m 2^e, 1/2 <= m < 1
    e = np.maximum(e - 1, -6)
    units = np.rint(a * 2.0 ** (3 - e)).astype(np.int64)  # of 2^(e - 3); 16 carries over by itself
    c = np.where(units < 8, units, (e + 6) * 8 + units)
    c = c | np.where(np.signbit(y), 128, 0)
    return np.where(np.isfinite(y), c, 0x7F).astype(np.uint8)


def power_of(x):
    """The power of two of a block of values: the least with which no finite magnitude is above 448."""
    a = np.abs(x[np.isfinite(x)])
    a = float(a.max()) if a.size else 0.0
    if a == 0.0:
        return LOW
    m, e = math.frexp(a)
    return min(max(e - 9 if m <= 0.875 else e - 8, LOW), HIGH)


def append_block(x, lo, codes, power):
    """x [rows, D] new at places lo .. of a block of codes [16, D] whose scale
    is 2^power (of no meaning with lo 0): the block's codes and power after."""
    e = power_of(x)
    codes = codes.copy()
    if lo:
        if e > power:
            with np.errstate(invalid="ignore"):
                codes[:lo] = codes_of(CODES[codes[:lo]] * 2.0 ** (power - e))
        e = max(e, power)
    codes[lo:lo + x.shape[0]] = codes_of(x * 2.0 ** -e)
    return codes, e


def same_codes(a, b):
    """Equal, where any NaN is like any other."""
    return (a == b) | (np.isnan(CODES[a]) & np.isnan(CODES[b]))


def plan(lens, new, free, table, page, num_pages, max_rows):
    """A step's pages, request by request.  lens, new: lists; free: the stack,
    its top last; table [n, max_pages].  Returns everything that is written."""
    n, width = table.shape
    lens, table, stack = [int(v) for v in lens], table.copy(), [int(v) for v in free]
    cap = width * page
    bad = [not 0 <= v <= cap for v in lens]
    up = lambda v: -(-v // page)
    for b in range(n):
        if not bad[b] and new[b] < 0:
            stack += [int(v) for v in table[b, :up(lens[b])]]
    stack = stack[:num_pages]
    full = list(stack)  # what lies in the stack's memory
    asked_pages = asked_rows = 0
    avail = len(stack)
    status, cu, after, positions, slots = [], [0], [], [], []
    for b in range(n):
        if bad[b] or new[b] < 0:
            status.append(2 if bad[b] else 0)
            after.append(lens[b] if bad[b] else 0)
            cu.append(cu[-1])
            continue
        want = int(new[b])
        if lens[b] + want > cap:
            status.append(1)
            after.append(lens[b])
            cu.append(cu[-1])
            continue
        need = up(lens[b] + want) - up(lens[b])
        asked_pages += need
        asked_rows += want
        if (need and asked_pages > avail) or (want and asked_rows > max_rows):
            status.append(1)
            after.append(lens[b])
            cu.append(cu[-1])
            continue
        for i in range(need):
            table[b, up(lens[b]) + i] = stack.pop()
        for j in range(lens[b], lens[b] + want):
            positions.append(j)
            slots.append(int(table[b, j // page]) * page + j % page)
        status.append(0)
        after.append(lens[b] + want)
        cu.append(cu[-1] + want)
    pad = max_rows - len(positions)
    return {"table": table, "stack": np.array(full, np.int32), "free": len(stack), "lens": np.array(after, np.int32),
            "cu": np.array(cu, np.int32), "status": np.array(status, np.int32),
            "positions": np.array(positions + [0] * pad, np.int32), "slots": np.array(slots + [-1] * pad, np.int64)}
