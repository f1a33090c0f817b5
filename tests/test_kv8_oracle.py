"""The 64-bit forms of the cache in 8 bits against themselves: codes and back,
ties, growing blocks."""
import numpy as np

import kv8_oracle as O8


def test_codes_and_back():
    c = np.arange(256, dtype=np.uint8)
    assert O8.same_codes(O8.codes_of(O8.CODES), c).all()
    assert (O8.CODES[0x7E], O8.CODES[0x08], O8.CODES[0x01], O8.CODES[0xFE]) == (448.0, 2.0 ** -6, 2.0 ** -9, -448.0)


def test_nearest_and_ties():
    up = O8.CODES[:0x7F]
    mid = (up[:-1] + up[1:]) / 2
    got = O8.codes_of(mid)
    assert (got % 2 == 0).all() and (np.abs(got.astype(int) - np.arange(126) - 0.5) == 0.5).all()
    rng = np.random.default_rng(0)
    x = np.exp(rng.uniform(-9, 6.1, 5000)) * rng.choice([-1, 1], 5000)
    err = np.abs(O8.CODES[O8.codes_of(x)] - x)
    assert (err <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10)).all()
    assert O8.CODES[O8.codes_of([1e9, -1e9, 449.0])].tolist() == [448.0, -448.0, 448.0]
    assert np.isnan(O8.CODES[O8.codes_of([np.inf, -np.inf, np.nan])]).all()


def test_powers():
    for e in range(O8.LOW, O8.HIGH + 1):
        assert O8.power_of(np.array([448.0 * 2.0 ** e, -1e-40])) == e
        assert O8.power_of(np.array([np.nextafter(448.0 * 2.0 ** e, 1e300)])) == min(e + 1, O8.HIGH)
    assert O8.power_of(np.zeros(3)) == O8.LOW and O8.power_of(np.array([np.inf, np.nan])) == O8.LOW


def test_block_grown_or_at_once():
    """Token by token or at once: the same codes where none is below 2^-6."""
    rng = np.random.default_rng(1)
    x = rng.uniform(1, 400, (16, 64)) * 4.0 ** (np.arange(16)[:, None] % 5)
    codes, power = np.zeros((16, 64), np.uint8), 77
    for p in range(16):
        codes, power = O8.append_block(x[p:p + 1], p, codes, power)
    once, e = O8.append_block(x, 0, codes, 0)
    assert power == e
    normal = np.abs(x) * 2.0 ** -e >= 2.0 ** -6
    assert (codes == once)[normal].all() and normal.mean() > 0.5
