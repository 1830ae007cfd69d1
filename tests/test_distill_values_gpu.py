"""Distillation loss on the GPU at logits that are not centred on 0: rows of any shift, far peaks, values of
the type's lowest, gradients replayed from graphs.

Bounds as in test_distill_gpu (a distance d from the row's maximum costs |d| 2^-24 in units of log 2, which
does not grow with the row's shift); a probability below fp32's normal range may be flushed to zero."""
import math

import pytest
import torch

from test_distill import inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -17
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _native():
    from trustworthy_dl.ops import _lib
    _lib.lib()


def definition(z, idx, t, labels, V, tau, alpha):
    """(loss, dz [M, W], sum of the absolute terms of dz [M, W]) in 64 bits"""
    M, W = z.shape
    zd = z.detach()[:, :V].double()
    use = (idx >= 0) & (idx < V) & (t != -math.inf)
    n_t = max(1, int(((idx >= 0) & (idx < V)).any(1).sum()))
    ok = (labels >= 0) & (labels < V)
    n_l = max(1, int(ok.sum()))
    x = torch.where(use, t.double() / tau, -math.inf)
    live = use.any(1)[:, None].double()
    q = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)
    lp = torch.log_softmax(zd / tau, 1)
    at = torch.where(use, idx, 0).long()
    kd = torch.where(q > 0, q * (torch.log(q) - lp.gather(1, at)), 0.0).sum()
    c = alpha * tau / n_t
    target = torch.zeros(M, V, dtype=torch.float64, device=z.device).scatter_add_(1, at, q)
    g = torch.zeros(M, W, dtype=torch.float64, device=z.device)
    size = torch.zeros_like(g)
    g[:, :V] = c * (live * lp.exp() - target)
    size[:, :V] = c * (live * lp.exp() + target)
    loss = alpha * tau * tau * float(kd) / n_t
    if alpha < 1:
        lp = torch.log_softmax(zd, 1)
        hot = torch.zeros(M, V, dtype=torch.float64, device=z.device)
        hot[ok, labels[ok]] = 1.0
        b = (1 - alpha) / n_l
        loss -= b * float(torch.where(hot > 0, hot * lp, 0.0).sum())
        g[:, :V] += b * (ok[:, None].double() * lp.exp() - hot)
        size[:, :V] += b * (ok[:, None].double() * lp.exp() + hot)
    return loss, g, size


def check(z, idx, t, labels, V, tau, alpha, spread=32.0):
    """spread: the largest distance of a teacher's entry or a label from its row's maximum"""
    from trustworthy_dl import ops
    print(f"case {tuple(z.shape)} {z.dtype} V={V} K={idx.shape[1]} tau={tau} alpha={alpha}", flush=True)
    z = z.detach().requires_grad_(True)
    loss = ops.distillation_loss(z, idx, t, labels, V, temperature=tau, alpha=alpha)
    (g,) = torch.autograd.grad(loss, z)
    want, dz, mag = definition(z, idx, t, labels, V, tau, alpha)
    size = alpha * tau * tau * (math.log(idx.shape[1]) + math.log(V) + spread / tau) + (1 - alpha) * (math.log(V) + spread)
    assert abs(float(loss.detach()) - want) <= E * size, (float(loss.detach()), want)
    u = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps + torch.finfo(FP).smallest_normal
    off = (g.double() - dz).abs() - (u * dz.abs() + (1 + u) * E * mag + tiny)
    assert not torch.isnan(g).any(), "NaN"
    assert float(off.max()) <= 0, torch.nonzero(off == off.max())[0].tolist()


def rows(M, V, K, dtype, shift, pad=0, seed=0):
    z, idx, t, labels = inputs(M, V + pad, V, K, seed)
    return (z + shift).to(dtype).to(DEV), idx.to(DEV), t.to(DEV), labels.to(DEV)


FORMS = [(5, 700), (5, 7001), (5, 70001), (600, 9001)]     # a wave a row, in registers, streaming, many rows streaming
MODES = [(1.0, 1.0), (1.0, 0.5), (2.0, 0.7), (4.0, 0.5), (1.5, 0.5)]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("M,V", FORMS)
@pytest.mark.parametrize("tau,alpha", MODES)
def test_shifted_rows(M, V, dtype, tau, alpha):
    """A trained model's logits lie around -30 to -120; the loss does not depend on a row's shift."""
    for shift in (-120.0, -700.0, 90.0):
        check(*rows(M, V, 9, dtype, shift), V, tau, alpha)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V,pad", [(9001, 0), (9001, 6), (8999, 9)])
def test_peaks_in_the_last_pieces_of_negative_rows(dtype, V, pad):
    """Row r has its maximum r columns before the end (or at the row's head): the edge elements and the
    last, partly filled pieces."""
    M = 640
    z, idx, t, labels = rows(M, V, 9, dtype, 0.0, pad)
    z = -200.0 - z.abs()
    r = torch.arange(M, device=DEV)
    z[r[:600], V - 1 - r[:600]] = -100.0
    z[r[600:], r[600:] - 600] = -100.0
    for tau, alpha in ((1.0, 1.0), (2.0, 0.5)):
        check(z.to(dtype), idx, t, labels, V, tau, alpha, spread=110.0)


@pytest.mark.parametrize("dtype,shift", [(BF, -2000.0), (BF, 1e4), (BF, -1e6), (BF, 1e30), (BF, -1e38), (HF, -2000.0), (HF, 3e4), (HF, -6e4),
                                         (FP, -2000.0), (FP, 1e6), (FP, -1e38)])
@pytest.mark.parametrize("M,V", FORMS)
def test_large_logits(M, V, dtype, shift):
    """Shifts at which a product of maximum and 1 / temperature rounds to many units: the type's own steps
    leave some classes at the maximum and others one or more steps below."""
    z, idx, t, labels = inputs(M, V, V, 9)
    step = torch.finfo(dtype).eps * 2.0 ** math.floor(math.log2(abs(shift)))
    z = (shift - torch.round(z.abs()) * min(step, 1e37)).to(dtype).to(DEV) if dtype != FP else (shift + z).to(dtype).to(DEV)
    top = z.max(1, keepdim=True)[0]
    # (entries and labels on classes within reach of the maximum: the loss is a number of ordinary size)
    near = torch.topk(z.float(), 9, dim=1)[1].to(DEV)
    idx = torch.where(idx.to(DEV) >= 0, near, idx.to(DEV))
    labels = torch.where((labels.to(DEV) >= 0) & (labels.to(DEV) < V), near[:, 0], labels.to(DEV))
    assert ((top - z.gather(1, near)).float() <= 32).all()
    for tau, alpha in ((1.0, 1.0), (2.0, 0.7), (1.5, 0.5)):
        check(z, idx, t.to(DEV), labels, V, tau, alpha)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("M,V", FORMS)
def test_rows_of_the_lowest_value(M, V, dtype):
    """Every class of a row at the type's lowest value (all of them masked alike), and all but one."""
    z, idx, t, labels = rows(M, V, 9, dtype, 0.0)
    z[3:] = torch.finfo(dtype).min
    z[4, V - 2] = 1.0
    idx[4], labels[4] = V - 2, V - 2
    for tau, alpha in ((1.0, 1.0), (2.0, 0.7), (0.5, 0.5)):
        check(z, idx, t, labels, V, tau, alpha)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_backward_replayed_by_itself(dtype):
    """Forward and backward as two graphs: each replay of the backward gives the gradient of the upstream
    gradient it is given, whatever the replay before left and whatever happened to its output."""
    from trustworthy_dl import ops
    z, idx, t, labels = rows(37, 3000, 6, dtype, 0.0)
    z.requires_grad_(True)

    def loss(x):
        return ops.distillation_loss(x, idx, t, labels, temperature=2.0, alpha=0.5)

    def eager(x, c):
        y = x.detach().clone().requires_grad_(True)
        return torch.autograd.grad(loss(y), y, torch.tensor(c, device=DEV))[0]
    graphed = torch.cuda.make_graphed_callables(loss, (z,))
    for trial in range(2):
        x = (z.detach() + trial).to(dtype).requires_grad_(True)
        out = graphed(x)
        for c in (3.0, 1.0, 1.0, 0.5, 1.0):
            (g,) = torch.autograd.grad(out, x, torch.tensor(c, device=DEV), retain_graph=True)
            torch.cuda.synchronize()
            assert torch.equal(g, eager(x, c)), c
            g.mul_(0.25)       # (a user's clipping, in place)


@pytest.mark.parametrize("upstream", [1.0, 3.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_hooks_that_change_layouts(dtype, upstream):
    """Saved-tensor hooks that bring every tensor back transposed or with a column stride of 2, or on another
    device, in another type or shape."""
    from trustworthy_dl import ops
    base, idx, t, labels = rows(37, 1003, 9, dtype, 0.0)

    def grad(unpack):
        z = base.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
            loss = ops.distillation_loss(z, idx, t, labels, temperature=2.0, alpha=0.4)
        return torch.autograd.grad(loss, z, torch.tensor(upstream, device=DEV))[0]

    def strided(x):
        store = torch.full((2 * x.numel(),), 7, dtype=x.dtype, device=x.device)
        back = store.view(*x.shape, 2)[..., 0]
        back.copy_(x)
        return back

    def last_first(x):
        return x.transpose(0, -1).contiguous().transpose(0, -1)
    want = grad(lambda x: x)
    for f in (strided, last_first):
        # (rows that start elsewhere are added in another order: two roundings of the value, 2^-20 of the sums)
        assert ((grad(f).double() - want.double()).abs()
                <= torch.finfo(dtype).eps * want.double().abs() + 2.0 ** -20 * want.double().abs().max()).all(), f.__name__
    for f in (lambda x: x.cpu(), lambda x: x[:1], lambda x: x.double()):
        with pytest.raises(RuntimeError, match="came back"):
            grad(f)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("M,V", FORMS)
@pytest.mark.parametrize("tau", [1e-6, 1e-2, 1000.0])
def test_temperatures_at_their_bounds(tau, M, V, dtype):
    z, idx, t, labels = rows(M, V, 9, dtype, -40.0)
    # (at low ones a row has a few classes with all the weight: the distances of its entries, 32 / tau, are known
    # to 2^-24 of themselves, and so are the logarithms of weights no smaller than that)
    from trustworthy_dl import ops
    z = z.detach().requires_grad_(True)
    loss = ops.distillation_loss(z, idx, t, labels, V, temperature=tau, alpha=0.5)
    (g,) = torch.autograd.grad(loss, z)
    want, dz, mag = definition(z, idx, t, labels, V, tau, 0.5)
    size = 0.5 * tau * tau * (math.log(9) + math.log(V) + 32 / tau) + 0.5 * (math.log(V) + 32)
    assert abs(float(loss.detach()) - want) <= E * size
    # a weight of e^(-d / tau): d 2^-24 / tau, for what is not yet zero (d / tau < 104); entries as well
    off = (g.double() - dz).abs() - (torch.finfo(dtype).eps / 2 * dz.abs() + 1.01 * 2 * E * mag + 2.0 ** -126)
    assert float(off.max()) <= 0, torch.nonzero(off == off.max())[0].tolist()


def test_no_grad_makes_no_gradient():
    """Under no_grad, of logits that require a gradient: no buffer of their size."""
    from trustworthy_dl import ops
    z, idx, t, labels = rows(64, 50257, 9, BF, 0.0)
    z.requires_grad_(True)
    want = ops.distillation_loss(z, idx, t, labels, alpha=0.5).detach()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        got = ops.distillation_loss(z, idx, t, labels, alpha=0.5)
    assert torch.cuda.max_memory_allocated() - before < z.numel()
    assert torch.equal(got, want) and not got.requires_grad


def test_sizes_out_of_range_are_refused():
    from trustworthy_dl import ops
    one, idx = torch.zeros(1, 1, dtype=BF, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    n = 1 << 30
    with pytest.raises(ValueError, match="rows and columns"):
        ops.distillation_loss(one.expand(n, 1), idx.expand(n, 1), one.expand(n, 1))
    with pytest.raises(ValueError, match="rows and columns"):
        ops.distillation_loss(one.expand(1, n), idx, one)


def test_more_rows_than_workgroups():
    check(*rows((1 << 21) + 777, 8, 2, FP, 0.0), 8, 2.0, 0.5)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("M,V", FORMS)
def test_forbidden_classes(M, V, dtype):
    """Rows that are -infinity but for a few classes (the first ones, the last one, one in the middle), and one that is
    -infinity throughout: NaN there by the definition, and nowhere else."""
    from trustworthy_dl import ops
    z, idx, t, labels = rows(M, V, 9, dtype, -150.0)
    few = {0: [0, 1, 2], 2: [V - 1], 3: [V // 2, V // 2 + 1]}
    for r, cols in few.items():
        keep = z[r, cols].clone()
        z[r] = -math.inf
        z[r, cols] = keep
        idx[r] = torch.tensor([cols[i % len(cols)] for i in range(9)], device=DEV)
        labels[r] = cols[0]
    for tau, alpha in MODES:
        check(z, idx, t, labels, V, tau, alpha)
    x = z.clone()
    x[4] = -math.inf
    idx[4], labels[4] = 3, 3
    x.requires_grad_(True)
    loss = ops.distillation_loss(x, idx, t, labels, temperature=2.0, alpha=0.5)
    (g,) = torch.autograd.grad(loss, x)
    others = [r for r in range(M) if r != 4]
    assert torch.isnan(loss) and torch.isnan(g[4]).all() and torch.isfinite(g[others]).all()


def test_inference_mode():
    from trustworthy_dl import ops
    z, idx, t, labels = rows(5, 3000, 9, BF, 0.0)
    want = ops.distillation_loss(z, idx, t, labels, temperature=2.0, alpha=0.5)
    with torch.inference_mode():
        assert torch.equal(ops.distillation_loss(z.clone(), idx, t, labels, temperature=2.0, alpha=0.5), want)
