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
