"""Distillation loss on the CPU: against the 64-bit formulas and differences, and the refusals."""
import math

import pytest
import torch

from trustworthy_dl import ops


def formula(z, idx, t, labels, V, tau, alpha):
    """(loss, dz [M, W]) row by row from the definition, in 64 bits"""
    M, W = z.shape
    z, t = z.detach().double(), t.double()
    use = (idx >= 0) & (idx < V)
    n_t = max(1, int(use.any(1).sum()))
    ok = ((labels >= 0) & (labels < V)) if labels is not None else torch.zeros(M, dtype=torch.bool, device=z.device)
    n_l = max(1, int(ok.sum()))
    grad = torch.zeros(M, W, dtype=torch.float64, device=z.device)
    loss = 0.0
    for r in range(M):
        e = [(int(i), float(x)) for i, x, u in zip(idx[r], t[r], use[r]) if u and x != -math.inf]
        if e and alpha > 0:
            x = torch.tensor([b for _, b in e], dtype=torch.float64, device=z.device) / tau
            q, lq = torch.softmax(x, 0), torch.log_softmax(x, 0)
            lp = torch.log_softmax(z[r, :V] / tau, 0)
            at = torch.tensor([a for a, _ in e], device=z.device)
            kd = torch.where(q > 0, q * (lq - lp[at]), 0.0).sum()
            loss += alpha * tau * tau * float(kd) / n_t
            grad[r, :V] += alpha * tau / n_t * lp.exp()
            grad[r].index_add_(0, at, -alpha * tau / n_t * q)
        if ok[r] and alpha < 1:
            lp = torch.log_softmax(z[r, :V], 0)
            loss -= (1 - alpha) / n_l * float(lp[labels[r]])
            grad[r, :V] += (1 - alpha) / n_l * lp.exp()
            grad[r, labels[r]] -= (1 - alpha) / n_l
    return loss, grad


def inputs(M, W, V, K, seed=0, dup=True):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(M, W, generator=g) * 2
    idx = torch.randint(0, V, (M, K), generator=g)
    t = torch.randn(M, K, generator=g) * 2 + 3
    if dup and K > 1:
        idx[:, -1] = idx[:, 0]          # the same index twice
    if M > 2:
        idx[1] = -1                     # no entries
        idx[2, K // 2:] = V + 3         # outside the classes: unused
        t[0, 0] = -math.inf
    labels = torch.randint(0, V, (M,), generator=g)
    if M > 3:
        labels[3], labels[0] = -100, V
    return z, idx, t, labels


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.7), (0.5, 0.3), (3.0, 0.0)])
@pytest.mark.parametrize("M,W,V,K", [(5, 13, 13, 4), (4, 16, 11, 1), (1, 7, 7, 7)])
def test_matches_formula(M, W, V, K, tau, alpha):
    z, idx, t, labels = inputs(M, W, V, K)
    z = z.double().requires_grad_(True)
    loss = ops.distillation_loss(z, idx, t, labels, V, temperature=tau, alpha=alpha)
    (g,) = torch.autograd.grad(loss, z)
    want, dz = formula(z, idx, t, labels, V, tau, alpha)
    assert math.isclose(float(loss), want, rel_tol=1e-12, abs_tol=1e-12)
    assert torch.allclose(g, dz, rtol=1e-11, atol=1e-13)


def test_gradient_against_differences():
    z, idx, t, labels = inputs(4, 9, 8, 3)
    f = lambda x: ops.distillation_loss(x, idx, t, labels, 8, temperature=1.7, alpha=0.6)  # noqa: E731
    assert torch.autograd.gradcheck(f, [z.double().requires_grad_(True)])


def test_alpha_zero_is_cross_entropy():
    z, idx, t, labels = inputs(6, 10, 10, 3)
    labels[labels == 10] = 1
    a = ops.distillation_loss(z, idx, t, labels, alpha=0.0)
    assert torch.allclose(a, ops.cross_entropy(z, labels), rtol=1e-6)


def test_no_rows_and_no_entries():
    z, idx, t, labels = inputs(4, 9, 9, 3)
    assert float(ops.distillation_loss(z[:0], idx[:0], t[:0])) == 0.0
    assert float(ops.distillation_loss(z, torch.full_like(idx, -1), t)) == 0.0
    x = z.view(2, 2, 9)
    assert torch.equal(ops.distillation_loss(x, idx.view(2, 2, 3), t.view(2, 2, 3)), ops.distillation_loss(z, idx, t))


def test_refusals():
    z, idx, t, labels = inputs(4, 9, 9, 3)
    f = ops.distillation_loss

    def bad(match, *a, **k):
        with pytest.raises(ValueError, match=match):
            f(*a, **k)
    bad("floating-point logits", z.long(), idx, t)
    bad("num_classes", z, idx, t, labels, 10)
    bad("num_classes", z, idx, t, labels, 0)
    bad("same rows", z, idx[:3], t[:3])
    bad("same rows", z, idx, t[:, :2])
    bad("1 to 1024", z, idx[:, :0], t[:, :0])
    bad("1 to 1024", z, idx[:, :1].expand(4, 1025), t[:, :1].expand(4, 1025))
    bad("teacher_index", z, idx.float(), t)
    bad("teacher_logits", z, idx, t.long())
    bad("no gradient", z, idx, t.requires_grad_(True))
    t = t.detach()
    for x in (0.0, -1.0, math.inf, math.nan):
        bad("temperature", z, idx, t, temperature=x)
    for x in (-0.1, 1.1, math.nan):
        bad("alpha", z, idx, t, labels, alpha=x)
    bad("needs labels", z, idx, t, alpha=0.5)
    bad("labels must be", z, idx, t, labels[:3], alpha=0.5)
    bad("labels must be", z, idx, t, labels.float(), alpha=0.5)


def test_temperatures_out_of_range():
    z, idx, t, labels = inputs(4, 9, 9, 3)
    for x in (1e-50, 1e-30, 1e-7, 1001.0, 1e20, 1e300):     # (1e-50 is 0 in 32 bits, 1e20 squared infinite)
        with pytest.raises(ValueError, match="temperature"):
            ops.distillation_loss(z, idx, t, temperature=x)
    for x in (1e-6, 1000.0):
        want, dz = formula(z, idx, t, None, 9, x, 1.0)
        y = z.double().requires_grad_(True)
        loss = ops.distillation_loss(y, idx, t, temperature=x)
        (g,) = torch.autograd.grad(loss, y)
        assert math.isclose(float(loss.detach()), want, rel_tol=1e-8) and torch.allclose(g, dz, rtol=1e-8, atol=1e-12)


def test_library_refuses_sizes_out_of_range():
    """The C entry point itself, before any launch (it needs no GPU for that)."""
    import ctypes

    from trustworthy_dl.ops import _lib
    from trustworthy_dl.ops.distill import MAX_DIM, _Args
    if not _lib.available():
        pytest.skip("the native library is not built")
    sizes = dict(rows=8, M=4, V=9, W=9, K=3, G=1, dtype=0, tau=1.0, alpha=1.0)

    def refused(**kw):
        a = _Args(**{**sizes, **kw})
        return _lib.lib().tdl_distill(ctypes.addressof(a), None) == 1      # hipErrorInvalidValue
    for kw in (dict(M=0), dict(M=MAX_DIM + 1), dict(W=MAX_DIM + 1), dict(V=10), dict(V=0), dict(K=0), dict(K=1025), dict(G=0), dict(dtype=3),
               dict(tau=0.0), dict(alpha=1.5), dict(alpha=0.5, beta=0.5), dict(rows=0)):
        assert refused(**kw), kw


def test_a_single_row_and_a_single_entry():
    z, idx, t, _ = inputs(1, 9, 9, 3)
    assert torch.equal(ops.distillation_loss(z[0], idx[0], t[0]), ops.distillation_loss(z, idx, t))
    with pytest.raises(ValueError, match="same rows"):
        ops.distillation_loss(z[0], idx[0, 0], t[0, 0])
