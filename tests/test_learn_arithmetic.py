"""The codes of 8-bit optimizer states, replayed on the host: the quick way (float32, the hardware's e4m3
conversion) against the careful one (float64), and where the quick way may not be taken."""
import numpy as np
import pytest

TINY = 2.0 ** -149


def careful(q, mant, top):
    """The nearest code to q >= 0 in units of the smallest one above zero, a middle to the even code."""
    full = np.arange((16 << mant) - 1)
    lead = 1 << mant
    table = np.where(full >= lead, ((full & (lead - 1)) + lead) * 2.0 ** ((full >> mant) - 1.0), full)
    assert top == full[-1]
    mids = (table[1:] + table[:-1]) / 2
    c = np.searchsorted(mids, q, side="left")
    tie = (c < mids.size) & (mids[np.minimum(c, mids.size - 1)] == q)
    return np.where(tie & (c % 2 == 1), c + 1, c)


def quick_v(q):
    """Code of float32(q) from its bits, and whether it lies in the middle of two; no upper bound."""
    f = q.astype(np.float32)
    f = np.where(q > 0, np.maximum(f, np.float32(1)), np.float32(0))
    small = f < 16
    bits = (f + np.where(small, np.float32(16), np.float32(0))).astype(np.float32).view(np.uint32)
    base = np.where(small, np.uint32(131 << 23), np.uint32(130 << 23))
    code = (bits + np.uint32(0x3ffff) + ((bits >> 19) & 1) - base) >> 19
    return code.astype(np.int64), (bits & 0x7ffff) == 0x40000


def quick_m(q):
    """e4m3 code of float32(q), q >= 0 in units of the scale: nearest, a middle to the even code, above
    464 the code of no number."""
    f = q.astype(np.float32)
    code = careful(f.astype(np.float64) * 512, 3, 126)
    t = f + np.where(f < 2.0 ** -6, np.float32(2.0 ** -6), np.float32(0))
    return np.where(f > 464, 127, code), (t.view(np.uint32) & 0xfffff) == 0x80000


def block(seed, largest, spread):
    rng = np.random.default_rng(seed)
    x = largest * np.concatenate([[1.0], rng.random(254) ** spread, [0.0]])
    return np.concatenate([x, largest * (1 - rng.random(256) * 1e-6)])


@pytest.mark.parametrize("seed", range(60))
def test_the_quick_codes_of_normal_scales_are_the_careful_ones(seed):
    rng = np.random.default_rng(1000 + seed)
    largest = 448 * 2.0 ** -126 * (1 + rng.random()) if seed % 3 == 0 else 10.0 ** rng.uniform(-33, 30)
    for step, unit, quick, mant, top in ((448.0, 512.0, quick_m, 3, 126), (491520.0, 1.0, quick_v, 4, 254)):
        x = block(seed, largest * step / 448.0, 1 + seed % 9)
        scale = float(np.float32(x.max() / step))
        assert scale >= 2.0 ** -126
        q = x / scale
        code, middle = quick(q)
        want = careful(q * unit, mant, top)
        if quick is quick_v:
            want = np.where(q > 0, np.maximum(want, 1), 0)
        assert ((code == want) | middle).all() and code.max() <= top


def test_the_quick_codes_of_subnormal_scales_leave_their_range():
    # why a block whose new scale is a subnormal takes the careful way: rounding the scale moves the largest
    # quotient by up to a half, and past the last code
    past = {"m": 0, "v": 0}
    for units in np.arange(0.5, 64.5, 1.0 / 16)[1:]:
        for name, step, unit, quick, mant, top in (("m", 448.0, 512.0, quick_m, 3, 126),
                                                   ("v", 491520.0, 1.0, quick_v, 4, 254)):
            x = block(3, units * TINY * step, 3)
            scale = float(np.float32(x.max() / step))
            assert 0 < scale < 2.0 ** -126
            q = x / scale
            assert careful(q * unit, mant, top).max() <= top
            past[name] += int(quick(q)[0].max() > top)
    assert past["m"] > 0 and past["v"] > 0


def test_sizes_beyond_the_limits_ask_for_no_scratch():
    # sizes that the calls refuse; some of them are not even representable a step further on
    from image_classification_amd import _lib
    lib = _lib.load()
    big = [1 << 62, (1 << 63) - 1, (1 << 62) + 1]
    for n, groups in [(1000, (1 << 26) + 1), (9000, 1 << 40), ((1 << 31) - 1, 5)] + [(9000, b) for b in big] + \
            [(b, 5) for b in big] + [(-1, 5), (5, 0), (5, -(1 << 63))]:
        assert lib.ic_group_rows_scratch(n, groups) == 0
        assert lib.ic_grouped_matmul_dw_scratch(n, groups, 64, 64, 0) == 0
    for k, out in (((1 << 24) + 1, 8), (8, (1 << 31) - 1), ((1 << 31) - 1, (1 << 31) - 1), (0, 8)):
        assert lib.ic_grouped_matmul_dw_scratch(100_000, 3, k, out, 1) == 0
    for n, v, top in [(b, 70_000, 3) for b in big] + [(4, b, 3) for b in big] + [(4, 70_000, 33), (4, 70_000, -1),
                                                                              (4, 0, 0), (4, (1 << 31) - 255, 3)]:
        assert lib.ic_label_logprobs_scratch(n, v, 0, top) == 0
    # the largest sizes that are taken
    assert lib.ic_group_rows_scratch((1 << 31) - 2, 1 << 26) > 0
    assert lib.ic_grouped_matmul_dw_scratch((1 << 31) - 2, 1, 1 << 24, 1, 0) > 0
    assert lib.ic_label_logprobs_scratch(4, (1 << 31) - 256, 0, 32) > 0
