"""Values at the ends of their ranges: optimizer states whose scales are float32 subnormals."""
import numpy as np
import pytest
import torch

from image_classification_amd import ops
from test_gpu_learn import U, adam_reference, adam_values, check_codes, flat_f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TINY = 2.0 ** -149          # the smallest float32 above zero


# -- 8-bit states that fade ---------------------------------------------------------------------------------
def step8(p, g, m, v, scales, step, betas):
    """One step of 8-bit states, held to its formulas: codes, scales, parameters."""
    hyper = dict(lr=1e-3, betas=betas, eps=1e-8, weight_decay=0.0)
    p0, g0 = flat_f64([p]), flat_f64([g])
    m0, v0 = adam_values(m, v, scales)
    ops.adamw_step([p], [g], m, v, step=step, scales=scales, **hyper)
    rp, rm, rv, upd = adam_reference(p0, g0, m0, v0, step, **hyper)
    check_codes(m, v, scales, rm, np.sqrt(rv))
    # the difference rounds twice, the step's factors about ten times; where m is a float32 subnormal, it and
    # its product with lr round by half of the smallest one each, before the division by at least eps
    tol = 2 * U * (np.abs(p0) + upd) + 12 * U * upd + U * np.abs(rp) + 2 * (TINY / 2) / hyper["eps"]
    assert (np.abs(flat_f64([p]) - rp) <= tol).all()


@pytest.mark.parametrize("betas, steps", [((0.9, 0.999), 1200), ((0.9, 0.95), 3500)])
def test_states_of_zero_gradients_fade(betas, steps):
    # one ordinary step, then none: a block's scale passes through the float32 subnormals, where its
    # rounding is a few per cent.  Scales begin between 1e-8 and 1e-3: m's are below 2^-150, so zero, after
    # ln(1e-3 2^150) / -ln 0.9 = 921 steps; v's, which lose sqrt(b2) a step, are below 2^-126 after
    # ln(1e-5 2^126) / -ln sqrt(0.95) = 2957
    gen = torch.Generator().manual_seed(7)
    p = torch.randn(512, generator=gen).to(DEV)
    g = torch.randn(512, generator=gen).to(DEV)
    g[256:] *= 0.01
    m, v, scales = ops.adamw_states([p], 8)
    step8(p, g, m, v, scales, 1, betas)
    g.zero_()
    for step in range(2, steps + 2):
        small = scales.cpu().numpy()
        if ((small > 0) & (small < 2.0 ** -120)).any():
            step8(p, g, m, v, scales, step, betas)
        else:
            ops.adamw_step([p], [g], m, v, lr=1e-3, step=step, betas=betas, weight_decay=0.0, scales=scales)
    mv, vv = ops.adamw_state_values(m, v, scales)
    assert all(bool(torch.isfinite(q).all()) for q in (p, mv, vv))
    left = scales.cpu().numpy()
    assert (left[0] == 0).all() and ((left[1] < 2.0 ** -126).all() or betas[1] == 0.999)


@pytest.mark.parametrize("largest", [2.9e-37, 5e-38, 1e-41, 3e-43, TINY])
def test_gradients_whose_scales_are_subnormal(largest):
    # a first and a second step; elements of every size below the largest, which has all places in turn
    for at in (0, 3, 100, 255):
        g = torch.from_numpy(np.float32(largest) * np.linspace(-1, 1, 512, dtype=np.float32)).to(DEV)
        g[at], g[256 + at] = largest, -largest
        p = torch.zeros(512, device=DEV)
        m, v, scales = ops.adamw_states([p], 8)
        for step in (1, 2):
            step8(p, g, m, v, scales, step, (0.9, 0.999))


def test_states_that_begin_with_subnormal_scales():
    # every code beside every other, blocks with scales of 1 to 64 units, as a saved state may hold them
    units = np.arange(1, 65, dtype=np.float64)
    m = torch.arange(64 * 256, device=DEV).to(torch.uint8)
    m[(m & 127) == 127] = 126
    v = torch.arange(64 * 256, device=DEV).flip(0).to(torch.uint8).clamp_(max=254)
    scales = torch.from_numpy(np.stack([units * TINY] * 2).astype(np.float32)).to(DEV)
    assert (scales.cpu().numpy() > 0).all()
    p = torch.zeros(64 * 256, device=DEV)
    for step in range(3, 40):
        step8(p, torch.zeros_like(p), m, v, scales, step, (0.9, 0.9))


# -- scores far from zero --------------------------------------------------------------------------------------
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# The exponent (x - M) / T of a term that does not vanish is below 130 and carries 3 roundings; a sum has at most
# 300 in a row and 2 a join; the outer operations round values of at most 150 four times.
ROW_TOL = U * (3 * 130 + 300 + 30 + 4 * 150)


def half_step(t):
    return torch.finfo(t).eps / 2


def far_rows(n, v, t, seed):
    """Rows whose scores lie anywhere in the type's range, a few of each kind, and their labels."""
    gen = torch.Generator().manual_seed(seed)
    most = torch.finfo(t).max
    z = torch.randn(n, v, generator=gen) * 3
    for i in range(n):
        kind = i % 9
        if kind == 0:
            z[i] = max(-1e9, -most)
        elif kind == 1:
            z[i] = -most
        elif kind == 2:
            z[i] += 1e4
        elif kind == 3:
            z[i] -= 1e4
        elif kind == 4:
            z[i] = z[i] * 10 + (1e6 if t != torch.float16 else 3e4)
        elif kind == 5:
            z[i] -= 300
            z[i, torch.rand(v, generator=gen) < 0.5] = -float("inf")
        elif kind == 6:
            z[i] = -most
            z[i, i % v] = 5.0
        elif kind == 7:
            z[i] = -float("inf")
        # (8: ordinary)
    labels = torch.randint(-1, v, (n,), generator=gen)
    return z.to(t), labels


def exact_rows(z, labels, temperature):
    """float64: lse, entropy, label's log probability, log probabilities (of -inf: -inf)."""
    x = z.double()
    top = x.max(1, keepdim=True)[0]
    none = torch.isinf(top)
    d = (x - torch.where(none, torch.zeros_like(top), top)) / temperature
    ln_s = torch.log(torch.exp(d).sum(1, keepdim=True))
    lq = torch.where(none, torch.full_like(d, -float("inf")), d - ln_s)
    p = torch.exp(lq)
    h = -torch.where(p > 0, p * lq, torch.zeros_like(p)).sum(1)
    has = (labels >= 0) & (labels < z.shape[1])
    logp = torch.where(has, lq.gather(1, labels.clamp(min=0).long()[:, None])[:, 0], torch.zeros_like(h))
    return (top / temperature + ln_s)[:, 0], h, logp, lq, p


def check_far_grad(z, labels, a, b, temperature, got):
    _, h, _, lq, p = exact_rows(z, labels, temperature)
    has = (labels >= 0) & (labels < z.shape[1])
    at = torch.nonzero(has)[:, 0]
    g = a.double() * has
    lqf = torch.where(p > 0, lq, torch.zeros_like(lq))
    want = -p * (g[:, None] + b.double()[:, None] * (lqf + h[:, None]))
    factor = g.abs()[:, None] + b.double().abs()[:, None] * (lqf.abs() + h[:, None] + 1)
    size = p * factor
    want[at, labels[at]] += g[at]
    size[at, labels[at]] += g[at].abs()
    none = torch.isinf(z.double().max(1)[0])
    want[none] = 0
    want, size = want / temperature, size / temperature
    # (the hardware's exponential has no subnormals: a p below 2^-126 may be 0)
    tol = (2 * ROW_TOL + 8 * U) * size + 2.0 ** -126 * factor / temperature + half_step(got.dtype) * want.abs() + \
        (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    off = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all())
    bad = (off > tol).any(1)
    assert not bool(bad.any()), (torch.nonzero(bad)[:, 0].tolist(), float((off / tol).max()))


FAR_SHAPES = [(300, 2), (18, 5), (45, 33), (27, 130), (90, 700), (21, 1000), (9, 1030), (18, 2500), (9, 5001),
              (9, 20000), (9, 70001)]


@pytest.mark.parametrize("n, v, t, temperature",
                         [(n, v, t, a) for n, v in FAR_SHAPES for t in TYPES for a in (1.0, 0.7)]
                         + [(2300, 18001, t, 1.0) for t in TYPES[:2]])       # many long rows
def test_gradients_of_scores_far_from_zero(n, v, t, temperature):
    z, labels = far_rows(n, v, t, n + v)
    gen = torch.Generator().manual_seed(9)
    a, b = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    zd, ld, ad, bd = z.to(DEV), labels.to(DEV), a.to(DEV), b.to(DEV)
    _, ent, lse, _, _ = ops.label_logprobs(zd, ld, temperature=temperature)
    got = ops.label_logprobs_grad(zd, ld, lse, ent, ad, bd, temperature)
    check_far_grad(z, labels, a, b, temperature, got)
    # rows that lie apart and begin anywhere, and in place
    wide = torch.full((n, v + 7), 3.0, dtype=t, device=DEV)
    wide[:, 3:3 + v] = zd
    apart = ops.label_logprobs_grad(wide[:, 3:3 + v], ld, lse, ent, ad, bd, temperature)
    check_far_grad(z, labels, a, b, temperature, apart)
    ops.label_logprobs_grad(wide[:, 3:3 + v], ld, lse, ent, ad, bd, temperature, out=wide[:, 3:3 + v])
    assert torch.equal(wide[:, 3:3 + v], apart)
    assert bool((wide[:, :3] == 3).all()) and bool((wide[:, 3 + v:] == 3).all())


def test_gradients_of_scores_far_from_zero_in_a_graph():
    # the same launches whatever the rows hold: ordinary rows when captured, far ones when replayed
    n, v = 18, 40_000
    z, labels = far_rows(n, v, torch.float32, 4)
    ones = torch.ones(n)
    buf, ld, od = torch.zeros(n, v, device=DEV), labels.to(DEV), ones.to(DEV)

    def both():
        _, ent, lse, _, _ = ops.label_logprobs(buf, ld)
        return ops.label_logprobs_grad(buf, ld, lse, ent, od, od)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        rows = z.roll(i, 0)
        buf.copy_(rows)
        ld.copy_(labels.roll(i, 0))
        graph.replay()
        torch.cuda.synchronize()
        check_far_grad(rows, labels.roll(i, 0), ones, ones, 1.0, got)
        assert torch.equal(got, both())


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("v", [37, 1000, 40_000])
@pytest.mark.parametrize("weight", [1e9, 2e30])
def test_large_entropy_weights_beside_masked_scores(v, t, weight):
    # a masked score has p = 0, so its gradient is 0 whatever the weight; the others' is weight times that of 1
    gen = torch.Generator().manual_seed(v)
    z = torch.randn(9, v, generator=gen)
    z[:, 1::3] = -float("inf")
    z[4] -= 3000                                # (a row that is read twice)
    z = z.to(t).to(DEV)
    labels = torch.zeros(9, dtype=torch.int32, device=DEV)
    _, ent, lse, _, _ = ops.label_logprobs(z, labels)
    one = torch.full((9,), 2.0 ** -10, device=DEV)
    # (in float32: a float16 gradient below 2^-25 is 0, and weight times it need not be)
    small = ops.label_logprobs_grad(z.float(), labels, lse, ent, None, one)
    got = ops.label_logprobs_grad(z, labels, lse, ent, None, one * weight)
    assert bool((got[:, 1::3] == 0).all())
    # (float16 ends at 65504)
    want = small.double() * float(torch.tensor(weight, dtype=torch.float32))
    inside = want.abs() < float(torch.finfo(t).max) / 2
    assert bool(inside.any())
    # p lies within ROW_TOL (which both ways of reading a row keep), log p + H within as much of its two terms; the
    # factor rounds twice, the result once
    spread = (z.double() - z.double().max(1, keepdim=True)[0]).clamp(min=-200).abs() + 2 * ent.double()[:, None] + 1
    p = torch.exp(torch.log_softmax(z.double(), 1))
    tol = 2 * (ROW_TOL + 4 * U) * p * spread * weight * 2.0 ** -10 + 4 * U * want.abs() + half_step(t) * want.abs() + \
        (2.0 ** -25 if t == torch.float16 else 0)
    assert bool(((got.double() - want).abs() <= tol)[inside].all())


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("n, v, top", [(27, 2, 2), (40, 5, 5), (18, 64, 7), (18, 130, 32), (18, 700, 3), (18, 2500, 20),
                                       (2060, 2500, 9), (9, 5001, 0), (9, 20000, 32), (9, 70001, 1)])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_log_probabilities_of_rows_anywhere_in_the_range(n, v, top, t, temperature):
    """Each row held to its own size: what one row holds says nothing about another's error."""
    z, labels = far_rows(n, v, t, 3 * n + v)
    logp, ent, lse, tl, ti = ops.label_logprobs(z.to(DEV), labels.to(DEV), top=top, temperature=temperature)
    rl, rh, rp, lq, _ = exact_rows(z, labels, temperature)
    has = (labels >= 0) & (labels < v)
    rp[has & torch.isinf(rl)] = -float("inf")

    def held(got, want, scale, name):
        got = got.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine], want[~fine]), name
        off, tol = (got - want).abs()[fine], (ROW_TOL + scale)[fine]
        assert bool((off <= tol).all()), (name, float((off / tol).max()))

    # lse rounds M / T twice (1 / T and the product) and itself; a log probability the gap to M the same way
    held(lse, rl, 4 * U * rl.abs(), "lse")
    held(ent, rh, 4 * U * rh, "entropy")
    held(logp, rp, 4 * U * rp.abs(), "logp")
    if top:
        order = torch.sort(z.double(), dim=1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(ti.cpu().long(), order)
        want = lq.gather(1, order)
        held(tl, want, 4 * U * want.abs(), "alternatives")


def test_entropies_that_are_known():
    # all equal: ln v; one left: 0; two left: ln 2 -- in every kernel's range of lengths, at any offset
    for v in (2, 3, 64, 65, 1000, 2049, 4097, 30_001):
        for base in (0.0, -1e9, torch.finfo(torch.float32).min, 3e38):
            z = torch.full((3, v), base, device=DEV)
            z[1:, 2:] = -float("inf")
            z[1, 1] = -float("inf")
            _, ent, lse, _, _ = ops.label_logprobs(z)
            want = torch.tensor([np.log(v), 0.0, np.log(2.0)], dtype=torch.float64)
            # s is a whole number, exact up to 2^24: the logarithm's roundings alone
            assert bool(((ent.double().cpu() - want).abs() <= 4 * U * want).all()), (v, base, ent)
            assert bool(((lse.double().cpu() - (z[0, 0].double().cpu() + want)).abs()
                         <= 4 * U * (abs(base) + want)).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_two_hundred_tensors_against_their_formulas(bits):
    # more than one launch's table: every tensor's parameters and states
    gen = torch.Generator().manual_seed(1)
    sizes = [int(q) for q in torch.randint(1, 700, (200,), generator=gen)]
    ps = [torch.randn(n, generator=gen).to(DEV) for n in sizes]
    gs = [torch.randn(n, generator=gen).to(DEV) for n in sizes]
    m, v, scales = ops.adamw_states(ps, bits)
    inside = np.concatenate([np.pad(np.ones(n, bool), (0, -n % 256)) for n in sizes])
    hyper = dict(lr=0.01, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    for step in (1, 2, 3):
        p0, g0 = flat_f64(ps), flat_f64(gs)
        m0, v0 = (m.double().cpu().numpy(), v.double().cpu().numpy()) if bits == 32 else adam_values(m, v, scales)
        ops.adamw_step(ps, gs, m, v, step=step, scales=scales, **hyper)
        rp, rm, rv, upd = adam_reference(p0, g0, m0, v0, step, **hyper)
        # the decay and the difference round twice, the step's factors about ten times
        tol = 2 * U * (np.abs(p0) + upd) + 12 * U * upd + U * np.abs(rp)
        assert (np.abs(flat_f64(ps) - rp) <= tol)[inside].all()
        if bits == 32:
            assert (np.abs(m.double().cpu().numpy() - rm) <= 4 * U * (np.abs(m0) + np.abs(g0)))[inside].all()
            assert (np.abs(v.double().cpu().numpy() - rv) <= 6 * U * rv + 1e-44)[inside].all()
        else:
            check_codes(m, v, scales, rm * inside, np.sqrt(rv) * inside)
        gs = [q * -0.5 for q in gs]


@pytest.mark.parametrize("eps", [0.0, 1e-46, 1e-40, 1e-38])
def test_an_eps_that_no_reciprocal_can_take(eps):
    # in 8 bits an eps below 2^-124 counts as that: what has no state does not move, the rest moves as it should
    gen = torch.Generator().manual_seed(2)
    p = torch.randn(512, generator=gen).to(DEV)
    g = torch.randn(512, generator=gen).to(DEV)
    g[::2] = 0
    p0 = p.clone()
    m, v, scales = ops.adamw_states([p], 8)
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0)
    for step in (1, 2, 3):
        before, m0, v0 = flat_f64([p]), *adam_values(m, v, scales)
        ops.adamw_step([p], [g], m, v, step=step, eps=eps, scales=scales, **hyper)
        rp, rm, rv, upd = adam_reference(before, flat_f64([g]), m0, v0, step, eps=2.0 ** -124, **hyper)
        assert (np.abs(flat_f64([p]) - rp) <= 2 * U * (np.abs(before) + upd) + 12 * U * upd + U * np.abs(rp)).all()
        check_codes(m, v, scales, rm, np.sqrt(rv))
    assert torch.equal(p[::2], p0[::2]) and bool((p[1::2] != p0[1::2]).all())


@pytest.mark.parametrize("largest", [1e37, 8e37, 1e38, 3.4e38])
def test_gradients_near_the_largest_float32(largest):
    # a first step is lr times the sign, whatever the size
    g = torch.from_numpy(np.float32(largest) * np.linspace(-1, 1, 512, dtype=np.float32)).to(DEV)
    p = torch.zeros(512, device=DEV)
    m, v, scales = ops.adamw_states([p], 8)
    for step in (1, 2, 3):
        step8(p, g, m, v, scales, step, (0.9, 0.999))
