"""The factors with which the writer behind the latent projection settles its codes, restated in numpy: for every BF16 value and every block scale
the code of one product (or of two, where the scale has no single factor) is the code of the division, its sign among it."""
import numpy as np
import pytest

f32, wide = np.float32, np.longdouble  # (64 bits of mantissa: a product of 8 and 24 bits and a second term are summed before their one rounding)

BITS = np.concatenate([np.arange(0, 0x7F80, dtype=np.uint32), np.array([0x8000, 0x8001, 0x8100, 0xBF80, 0xC000], dtype=np.uint32)])
VALUES = (BITS << 16).astype(np.uint32).view(f32)  # every finite magnitude, and some negative ones


def e4m3(byte):
    exponent, mantissa = byte >> 3, byte & 7
    return f32(mantissa * 2.0 ** -9) if exponent == 0 else f32((1 + mantissa / 8) * 2.0 ** (exponent - 7))


def e2m1(y):
    a = np.abs(y)
    code = sum(t.astype(np.uint8) for t in (a > 0.25, a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5))
    return code | (np.signbit(y).astype(np.uint8) << 3)


def bits(x):
    return int(x.view(np.uint32))


def from_bits(b):
    return np.uint32(b).view(f32)


def factor(sf8, ckv_scale):
    sf = e4m3(sf8) * ckv_scale
    r = bits(f32(1) / sf)
    border = [f32(1 + 0.25 * i) for i in range(4)]
    near = [(bits(sf * m) + 16) for m in border]
    x = [from_bits(t & 0xFFFF0000) if (t & 0xFFFF) <= 32 else f32(0) for t in near]  # the BF16 number next to border * scale

    def good(products):
        return all((p < m) == (v / sf < m) and (p > m) == (v / sf > m) for p, v, m in zip(products, x, border))

    for step in (0, -1, 1, -2, 2):
        f = from_bits(r + step)
        if good([v * f for v in x]):
            return f, f32(0)
    rest = lambda f: f32(wide(1) - wide(sf) * wide(f))  # noqa: E731
    f = from_bits(r - 1 if rest(from_bits(r)) < 0 else r)
    g = f32(rest(f) * f)
    return (f, g) if sf8 != 0x7E and good([f32(wide(v) * wide(f) + wide(v * g)) for v in x]) else (f32(0), f32(0))


@pytest.mark.filterwarnings("ignore")  # (quotients of the largest values overflow)
@pytest.mark.parametrize("ckv_scale", [1.0, 0.5, 2.0 ** -9, 6.5 / 2688, 0.0031, 3.0])
def test_every_value_at_every_block_scale(ckv_scale):
    ckv_scale, singles, pairs = f32(ckv_scale), 0, 0
    for sf8 in range(1, 127):
        f, g = factor(sf8, ckv_scale)
        if f == 0:
            continue  # (the kernel takes its enclosing products)
        assert g >= 0
        singles, pairs = singles + (g == 0), pairs + (g > 0)
        second = VALUES * g
        y = (VALUES.astype(wide) * wide(f) + second.astype(wide)).astype(f32)
        y = np.where(y == 0, np.where(np.signbit(VALUES * f) & np.signbit(second), f32(-0.0), f32(0.0)), y)  # (only -0 + -0 is -0)
        assert np.array_equal(e2m1(y), e2m1(VALUES / (e4m3(sf8) * ckv_scale)))
    assert singles + pairs >= 124 and (pairs > 40) == (np.frexp(ckv_scale)[0] == 0.5)
