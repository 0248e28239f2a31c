"""The bound that is stated for float32 products on the bfloat16 matrix instructions, shown on the arithmetic itself.

a = hi + mid + lo exactly (8 + 8 + 8 bits, each the rounding to nearest even of what is left).  With a in [1, 2):
|mid| <= 2^-8 (half a step of bfloat16 at 1) and |lo| <= 2^-17 (half a step below 2^-8).  Of the nine partial products of a b the
three that are left out, mid lo', lo mid' and lo lo', are at most 2 2^-25 + 2^-34 = 2^-24 (1 + 2^-10) of 1 <= a b."""
import numpy as np

LEFT_OUT = 2.0 ** -24 * (1 + 2.0 ** -10)
WORST = 1 + 2.0 ** -8 - 2.0 ** -17               # hi 1, mid 2^-8, lo -2^-17


def bfloat16(x):
    """float32 to the nearest bfloat16, ties to even, as float32 (finite values)."""
    bits = x.astype(np.float32).view(np.uint32)
    return ((bits + 0x7fff + ((bits >> 16) & 1)) & np.uint32(0xffff0000)).view(np.float32)


def split(x):
    hi = bfloat16(x)
    mid = bfloat16(x - hi)
    return hi, mid, bfloat16(x - hi - mid)


def left_out(a, b):
    parts = [[p.astype(np.float64) for p in split(x)] for x in (a, b)]
    for x, p in zip((a, b), parts):
        assert np.array_equal(p[0] + p[1] + p[2], x.astype(np.float64))
    (ah, am, al), (bh, bm, bl) = parts
    kept = al * bh + ah * bl + am * bm + am * bh + ah * bm + ah * bh
    exact = a.astype(np.float64) * b.astype(np.float64)
    return np.abs(exact - kept) / np.abs(exact)


def test_left_out_of_random_products():
    rng = np.random.default_rng(0)
    a, b = (rng.standard_normal(1 << 20).astype(np.float32) * 2.0 ** rng.integers(-20, 21, 1 << 20).astype(np.float32)
            for _ in range(2))
    off = left_out(a, b)
    assert off.max() <= LEFT_OUT
    assert off.max() > 2.0 ** -26                  # no quarter of a rounding, as one might hope


def test_left_out_of_the_worst_products():
    one = np.float32(WORST)
    assert [float(p[0]) for p in split(np.array([one]))] == [1.0, 2.0 ** -8, -2.0 ** -17]
    assert 0.99 * 2.0 ** -24 < left_out(np.array([one]), np.array([one]))[0] <= LEFT_OUT
    # every value around the ties of the first and the second part, of either sign and some sizes
    near = np.concatenate([np.float32(1 + 2.0 ** -8) + np.arange(-600, 601, dtype=np.float32) * np.float32(2.0 ** -23),
                           np.float32(1 + 3 * 2.0 ** -9) + np.arange(-600, 601, dtype=np.float32) * np.float32(2.0 ** -23)])
    for other in (near, near[::-1], np.roll(near, 301), -near * np.float32(2.0 ** -30), np.full_like(near, one)):
        assert left_out(near, other).max() <= LEFT_OUT
