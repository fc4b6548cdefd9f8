"""SoftmaxClassifier: the host logic on a float64 stand-in of the operators, and the same on the
device (where the answers are compared with the stand-in's)."""
import numpy as np
import pytest
import torch

from checker_backend import CheckerBackend
from image_classification_amd import SoftmaxClassifier


class LearnChecker(CheckerBackend):
    """The operators in float64 on the CPU, as their documentation states them."""

    def group_rows(self, codes, n_groups):
        c = codes.numpy()
        key = np.where((c >= 0) & (c < n_groups), c, n_groups)
        order = np.argsort(key, kind="stable")
        return (torch.from_numpy(order.astype(np.int32)),
                torch.from_numpy(np.searchsorted(key[order], np.arange(n_groups + 1))))

    @staticmethod
    def _groups(offsets, order):
        for e in range(offsets.shape[0] - 1):
            yield e, order[int(offsets[e]):int(offsets[e + 1])].long()

    def grouped_matmul(self, x, w, offsets, order=None):
        y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
        for e, at in self._groups(offsets, order):
            y[at] = x[at].double() @ w[e].double().t()
        return y.float()

    def grouped_matmul_dx(self, dy, w, offsets, order=None):
        return self.grouped_matmul(dy, w.transpose(1, 2), offsets, order)

    def grouped_matmul_dw(self, dy, x, offsets, order=None):
        dw = torch.zeros(offsets.shape[0] - 1, dy.shape[1], x.shape[1], dtype=torch.float64)
        for e, at in self._groups(offsets, order):
            dw[e] = dy[at].double().t() @ x[at].double()
        return dw.float()

    def label_logprobs(self, logits, labels=None, top=0, temperature=1.0):
        lq = torch.log_softmax(logits.double() / temperature, 1)
        lse = torch.logsumexp(logits.double() / temperature, 1)
        entropy = -(lq.exp() * lq).sum(1)
        logp = None
        if labels is not None:
            ok = (labels >= 0) & (labels < logits.shape[1])
            logp = torch.where(ok, lq.gather(1, labels.long().clamp(0, logits.shape[1] - 1)[:, None])[:, 0],
                               torch.zeros_like(lse)).float()
        idx = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
        return logp, entropy.float(), lse.float(), lq.gather(1, idx).float(), idx.int()

    def label_logprobs_grad(self, logits, labels, lse, entropy, d_logp=None, d_entropy=None,
                            temperature=1.0, out=None):
        z = logits.double().requires_grad_()
        lq = torch.log_softmax(z / temperature, 1)
        loss = (lq.gather(1, labels.long()[:, None])[:, 0] * d_logp.double()).sum()
        if d_entropy is not None:
            loss = loss - ((lq.exp() * lq).sum(1) * d_entropy.double()).sum()
        g = torch.autograd.grad(loss, z)[0].float()
        if out is None:
            return g
        out.copy_(g)
        return out

    def adamw_states(self, params, bits=32):
        self.bits = bits
        return [torch.zeros_like(p).double() for p in params], [torch.zeros_like(p).double() for p in params], None

    def adamw_step(self, params, grads, m, v, lr, step, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                   scales=None):
        for p, g, a, q in zip(params, grads, m, v):
            a.mul_(betas[0]).add_(g.double() * (1 - betas[0]))
            q.mul_(betas[1]).add_(g.double() ** 2 * (1 - betas[1]))
            upd = lr * (a / (1 - betas[0] ** step)) / ((q / (1 - betas[1] ** step)).sqrt() + eps)
            p.copy_((p.double() * (1 - lr * weight_decay) - upd).float())


@pytest.fixture(params=["checker", pytest.param("hip", marks=pytest.mark.gpu)])
def backend(request):
    if request.param == "checker":
        return LearnChecker()
    from image_classification_amd.backend import default_backend
    return default_backend()


def blobs(n, classes, d, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    centres = rng.standard_normal((classes, d)) * 3
    y = rng.integers(0, classes, n)
    return (centres[y] + spread * rng.standard_normal((n, d))).astype(np.float32), y


CASES = [dict(), dict(experts=3), dict(rank=5), dict(experts=4, rank=3, state_bits=8),
         dict(state_bits=8, entropy_weight=0.05), dict(epochs=0)]


@pytest.mark.parametrize("kw", CASES, ids=str)
def test_interface(backend, kw, tmp_path):
    x, y = blobs(700, 6, 21, 0)
    names = np.array(["c%d" % i for i in y])
    kw = dict(dict(epochs=2, batch_size=256, seed=3), **kw)
    c = SoftmaxClassifier(backend=backend, **kw)
    c.train(x, names)
    p = c.predict_proba(x[:50])
    assert p.shape == (50, 6) and p.dtype == np.float64
    assert np.allclose(p.sum(1), 1.0, atol=1e-12)
    best, logp = c.alternatives(x[:50], 3)
    assert best.shape == logp.shape == (50, 3)
    assert (np.diff(logp, axis=1) <= 0).all()
    col = np.searchsorted(c.classes_, best)
    # log p in float32 of values up to 20: 2^-24 * 20 each way
    assert np.abs(np.log(p[np.arange(50)[:, None], col]) - logp).max() < 1e-5
    assert (c.test(x[:50]) == best[:, 0]).all()
    lp, ent = c.log_probabilities(x[:50], list(names[:49]) + ["other"])
    assert lp[49] == 0.0 and (lp[:49] <= 0).all() and (ent >= 0).all()
    assert np.abs(-(p * np.log(p)).sum(1) - ent).max() < 1e-5
    some = c.test_probability(x[:50], 0.2)
    top = np.sort(p, axis=1)
    sure = top[:, -1] - top[:, -2]
    for label, want, gap in zip(some, best[:, 0], sure):
        if abs(gap - 0.2) > 1e-5:
            assert label == (want if gap > 0.2 else -1)
    # a trained classifier ignores further training; one vector is one row; no rows are no answers
    before = [w.clone() for w in c._weights]
    c.train(x, names[::-1])
    assert all(torch.equal(a, b) for a, b in zip(before, c._weights))
    assert c.test(x[0])[0] == best[0, 0]
    assert c.test(x[:0]).shape == (0,) and c.predict_proba(x[:0]).shape == (0, 6)
    # the file holds everything
    c.save_to_file(str(tmp_path / "svm"))
    again = SoftmaxClassifier.load_from_file(str(tmp_path / "svm"), backend=backend)
    assert np.array_equal(again.predict_proba(x[:50]), p)
    # equal seeds, equal weights
    twin = SoftmaxClassifier(backend=backend, **kw)
    twin.train(x, names)
    assert all(torch.equal(a, b) for a, b in zip(twin._weights, c._weights))


@pytest.mark.parametrize("kw", [dict(), dict(rank=4), dict(experts=2, entropy_weight=0.1)], ids=str)
def test_first_steps_follow_the_formulas(backend, kw):
    # one batch, one step: the weights move by lr * g / (|g| + eps), computed here in float64
    x, y = blobs(300, 4, 11, 1)
    c = SoftmaxClassifier(epochs=1, batch_size=300, lr=0.01, weight_decay=0.0, seed=5, backend=backend, **kw)
    c.train(x, y)
    codes = c._route(c._b().f32(x)).cpu().long()
    rows = torch.from_numpy(np.concatenate([x, np.ones((300, 1), np.float32)], 1)).double()
    w = c._weights[-1].double().cpu()
    if "rank" in kw:
        # B was zero, so A has not moved: h = A x with the stored A
        a = c._weights[0].double().cpu()[:, :, :12]
        h = torch.einsum("nrk,nk->nr", a[codes], rows)
    else:
        h = rows
    z = torch.zeros(300, 4, dtype=torch.float64, requires_grad=True)   # all weights began at zero
    lq = torch.log_softmax(z, 1)
    loss = -lq[torch.arange(300), torch.from_numpy(y)].mean()
    loss = loss + kw.get("entropy_weight", 0.0) * (lq.exp() * lq).sum(1).mean()
    assert abs(c.loss_[0] - float(loss.detach())) < 1e-5
    dz = torch.autograd.grad(loss, z)[0]
    g = torch.zeros(w.shape[0], 4, h.shape[1], dtype=torch.float64)
    for e in range(w.shape[0]):
        g[e] = dz[codes == e].t() @ h[codes == e]
    want = -0.01 * g / (g.abs() + 1e-8)
    got = w[:, :4, :h.shape[1]]
    big = g.abs() > 1e-5      # (a sum near zero has no sure sign)
    assert big.double().mean() > 0.8
    assert float((got - want).abs()[big].max()) < 1e-6 + 0.01 * 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(experts=3, rank=6)], ids=str)
def test_device_agrees_with_the_stand_in(kw, tmp_path):
    # the same weights, from a file: a logit is two chains of at most 45 float32 products, and
    # probabilities move by at most twice the largest logit's error
    from image_classification_amd.backend import default_backend
    x, y = blobs(900, 5, 40, 2)
    a = SoftmaxClassifier(epochs=3, batch_size=200, lr=0.02, seed=1, backend=LearnChecker(), **kw)
    a.train(x, y)
    a.save_to_file(str(tmp_path / "c"))
    b = SoftmaxClassifier.load_from_file(str(tmp_path / "c"), backend=default_backend())
    codes = a._route(torch.from_numpy(x))
    size = np.concatenate([np.abs(x), np.ones((900, 1)), np.zeros((900, 3))], 1)
    for w in a._weights:
        size = np.einsum("nck,nk->nc", np.abs(w.numpy())[codes.numpy()], size)
    tol = 2 * 2 * 47 * 2.0 ** -24 * size.max(1, keepdims=True) + 1e-6
    assert (np.abs(a.predict_proba(x) - b.predict_proba(x)) <= tol).all()


def test_refusals():
    b = LearnChecker()
    for kw in (dict(experts=0), dict(rank=0), dict(epochs=-1), dict(batch_size=0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            SoftmaxClassifier(backend=b, **kw)
    x, y = blobs(20, 3, 5, 0)
    c = SoftmaxClassifier(epochs=1, backend=b)
    with pytest.raises(RuntimeError):
        c.test(x)
    with pytest.raises(RuntimeError):
        c.save_to_file("never")
    for bad_x, bad_y in ((x, y[:5]), (x[0], y[:1]), (x[:0], y[:0]), (np.full((3, 2), np.nan), [0, 1, 2]),
                         (x[:, :0], y)):
        with pytest.raises(ValueError):
            SoftmaxClassifier(epochs=1, backend=b).train(bad_x, bad_y)
    with pytest.raises(ValueError):
        SoftmaxClassifier(experts=30, backend=b).train(x, y)
    c.train(x, y)
    for call in (lambda: c.test(x[:, :3]), lambda: c.alternatives(x, 0), lambda: c.alternatives(x, 4),
                 lambda: c.log_probabilities(x, y[:3]), lambda: c.test(np.full((2, 5), np.inf))):
        with pytest.raises(ValueError):
            call()
