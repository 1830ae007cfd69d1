"""Distillation loss on the GPU against the 64-bit formulas.

Bounds.  In 32 bits every probability carries the error of its exponent's argument, |d| 2^-24 for a
distance d from the row's maximum (inputs here: d < 2^5 in units of log 2), of the sums (a row's tree of
at most 2^5 additions a thread) and a few roundings: 2^-17 relative covers them with a factor to spare.
dz is rounded once to the logits' type, u = eps / 2.  The loss is a mean of such terms: 2^-17 of the mean of
their magnitudes."""
import contextlib
import math

import pytest
import torch

from test_distill import formula, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -17


@pytest.fixture(autouse=True)
def _native():
    from trustworthy_dl.ops import _lib
    _lib.lib()


def magnitudes(z, idx, t, labels, V, tau, alpha):
    """[M, W] sum of the absolute terms of dz"""
    with torch.no_grad():
        neg = formula(z, idx, t, labels, V, tau, alpha)[1]
        use = (idx >= 0) & (idx < V)
        n_t, n_l = max(1, int(use.any(1).sum())), max(1, int(((labels >= 0) & (labels < V)).sum()))
        p = torch.zeros_like(neg)
        zd = z.double()[:, :V]
        p[:, :V] = alpha * tau / n_t * torch.softmax(zd / tau, 1) + (1 - alpha) / n_l * torch.softmax(zd, 1)
        return 2 * p + neg.abs()


def check(z, idx, t, labels, V, tau, alpha, upstream=None):
    from trustworthy_dl import ops
    print(f"case {tuple(z.shape)} {z.dtype} V={V} K={idx.shape[1]} tau={tau} alpha={alpha} up={upstream}", flush=True)
    z = z.detach().requires_grad_(True)
    loss = ops.distillation_loss(z, idx, t, labels, V, temperature=tau, alpha=alpha)
    up = None if upstream is None else torch.tensor(upstream, device=DEV)
    (g,) = torch.autograd.grad(loss, z, up)
    want, dz = formula(z, idx, t, labels, V, tau, alpha)
    c = 1.0 if upstream is None else upstream
    # terms of the loss: q log q and q log p, at most tau^2 (log K + log V + range / tau) a row
    size = alpha * tau * tau * (math.log(idx.shape[1]) + math.log(V) + 32 / tau) + (1 - alpha) * (math.log(V) + 32)
    assert abs(float(loss) - want) <= E * size
    u = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    off = (g.double() - c * dz).abs() - (u * (c * dz).abs() + (1 + u) * E * abs(c) * magnitudes(z, idx, t, labels, V, tau, alpha) + tiny)
    assert float(off.max()) <= 0, torch.nonzero(off == off.max())[0].tolist()
    return loss, g


def on_gpu(M, W, V, K, dtype, seed=0, tdtype=torch.float32, itype=torch.int64):
    z, idx, t, labels = inputs(M, W, V, K, seed)
    return z.to(dtype).to(DEV), idx.to(itype).to(DEV), t.to(tdtype).to(DEV), labels.to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("W,V", [(1, 1), (7, 7), (64, 50), (1000, 1000), (1003, 1003), (4099, 4096), (9001, 9001), (33000, 32999),
                                 (70001, 70001), (140016, 140001)])
def test_lengths_and_types(dtype, W, V):
    check(*on_gpu(5, W, V, min(V, 9), dtype), V, 2.0, 0.7)


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (0.5, 0.3), (4.0, 0.0), (3.0, 0.999)])
@pytest.mark.parametrize("K", [1, 63, 64, 65, 300, 1024])
def test_entries_and_weights(tau, alpha, K):
    check(*on_gpu(6, 2048, 2040, K, torch.bfloat16, tdtype=torch.bfloat16, itype=torch.int32), 2040, tau, alpha)
    check(*on_gpu(3, 9000, 9000, K, torch.float32, tdtype=torch.float16), 9000, tau, alpha)


@pytest.mark.parametrize("upstream", [1.0, 0.25, 3.0, -2.0, 0.0])
def test_upstream_gradients(upstream):
    check(*on_gpu(7, 5003, 5000, 20, torch.bfloat16), 5000, 2.0, 0.6, upstream)
    check(*on_gpu(7, 5003, 5000, 20, torch.float32), 5000, 2.0, 1.0, upstream)


def test_many_rows():
    z, idx, t, labels = on_gpu(2500, 300, 300, 5, torch.float16)
    check(z, idx, t, labels, 300, 2.0, 0.5, 1024.0)     # more rows than the second pass has workgroups


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_and_offsets(dtype):
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(5, 1003, 1003, 6, dtype)
    loss, g = check(z, idx, t, labels, 1003, 1.5, 0.5)
    for pad, skew in ((5, 0), (0, 1), (3, 3), (13, 2)):
        store = torch.full((5 * (1003 + pad) + skew,), 7.0, dtype=dtype, device=DEV)
        view = store[skew:].as_strided((5, 1003), (1003 + pad, 1), skew)
        view.copy_(z)
        view.requires_grad_(True)
        l2 = ops.distillation_loss(view, idx, t, labels, temperature=1.5, alpha=0.5)
        assert abs(float(l2) - float(loss)) <= 2 * E * 100
        (g2,) = torch.autograd.grad(l2, view)
        # (another alignment adds the row in another order: equal to the sums' own error)
        u = torch.finfo(dtype).eps / 2
        assert ((g2.double() - g.double()).abs() <= 2 * u * g.double().abs() + 4 * E / 5 + 1e-12).all()
        assert (store[:skew] == 7).all()
    cols = torch.empty(5, 2 * 1003, dtype=dtype, device=DEV)
    cols[:, ::2] = z
    assert torch.equal(ops.distillation_loss(cols[:, ::2], idx, t, labels, temperature=1.5, alpha=0.5), loss.detach())
    three = ops.distillation_loss(z.view(5, 1, 1003), idx.view(5, 1, 6), t.view(5, 1, 6), labels.view(5, 1), temperature=1.5, alpha=0.5)
    assert torch.equal(three, loss.detach())


def test_no_entries_no_labels():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(4, 500, 500, 3, torch.float32)
    z.requires_grad_(True)
    loss = ops.distillation_loss(z, torch.full_like(idx, -1), t, torch.full_like(labels, -100), alpha=0.5)
    assert float(loss) == 0 and (torch.autograd.grad(loss, z)[0] == 0).all()
    loss = ops.distillation_loss(z[:0], idx[:0], t[:0])
    assert float(loss) == 0 and torch.autograd.grad(loss, z)[0].abs().sum() == 0
    dead = t.clone()
    dead[2] = -math.inf      # a row whose entries teach nothing: counted, no gradient
    loss = ops.distillation_loss(z, idx.clamp(min=0), dead)
    (g,) = torch.autograd.grad(loss, z)
    assert torch.isfinite(loss) and (g[2] == 0).all() and (g[0] != 0).any()


def test_infinities_and_nan_stay_in_their_row():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(6, 3000, 2990, 8, torch.bfloat16)
    idx = idx.clamp(0, 2989)
    t[0] = 1.0
    z[4, 17] = -math.inf                   # a class the student forbids (and the teacher does not name)
    idx[4] = torch.arange(8, device=DEV) + 100
    labels[:] = 5
    z[:, 2990:] = math.nan                 # padding columns are never read
    f = lambda x, y: ops.distillation_loss(x.requires_grad_(True), idx, y, labels, 2990, temperature=2.0, alpha=0.5)  # noqa: E731
    a = z.clone()
    loss = f(a, t)
    (g,) = torch.autograd.grad(loss, a)
    want, dz = formula(torch.where(torch.isnan(z), 0, z), idx, t, labels, 2990, 2.0, 0.5)
    assert abs(float(loss) - want) <= E * 200 and (g[:, 2990:] == 0).all() and g[4, 17] == 0
    for where, bad in (("z", math.nan), ("z", math.inf), ("t", math.nan)):
        b, s = z.clone(), t.clone()
        (b if where == "z" else s)[3, 2] = bad
        loss = f(b, s)
        (gb,) = torch.autograd.grad(loss, b)
        # a teacher's NaN makes its row's weights NaN: by the formula the loss and the columns they stand in
        assert torch.isnan(loss) and torch.isnan(gb[3, :2990] if where == "z" else gb[3, idx[3]]).all()
        keep = [0, 1, 2, 4, 5]
        assert torch.equal(gb[keep], g[keep])


def test_second_backward_and_shared_logits():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(5, 4000, 4000, 6, torch.bfloat16)
    z.requires_grad_(True)
    loss = ops.distillation_loss(z, idx, t, labels, temperature=2.0, alpha=0.5)
    first = torch.autograd.grad(loss, z, retain_graph=True)[0].clone()
    held = torch.autograd.grad(loss, z, retain_graph=True)[0]
    assert torch.equal(first, held)
    torch.autograd.grad(loss, z, torch.tensor(5.0, device=DEV))
    assert torch.equal(first, held)        # an earlier result is not written again
    before = z.detach().clone()
    loss = ops.distillation_loss(z, idx, t, labels, alpha=0.5) * 2 + z.float().mean()
    loss.backward()
    assert torch.equal(z.detach(), before) and torch.isfinite(z.grad).all()
    z2 = z.detach().clone().requires_grad_(True)
    loss = ops.distillation_loss(z2, idx, t, labels, alpha=0.5)
    with torch.no_grad():
        z2.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("upstream", [1.0, 3.0])
def test_tensors_saved_elsewhere(dtype, upstream):
    """Saved-tensor hooks bring the logits back with other strides than the forward saw: the same gradient."""
    from trustworthy_dl import ops
    M, W, K = 37, 1003, 9
    base = torch.randn(M, W + 6, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(dtype)
    index = torch.randint(0, W, (M, K), generator=torch.Generator(device=DEV).manual_seed(6), device=DEV)
    teacher = torch.randn(M, K, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV)
    labels = torch.randint(0, W, (M,), generator=torch.Generator(device=DEV).manual_seed(8), device=DEV)

    def grad(hooks):
        z = base.clone().requires_grad_(True)
        part = z[:, 3:3 + W]
        with hooks:
            loss = ops.distillation_loss(part, index, teacher, labels, temperature=2.0, alpha=0.4)
        return torch.autograd.grad(loss, z, torch.tensor(upstream, device=DEV))[0]
    want = grad(contextlib.nullcontext())
    got = grad(torch.autograd.graph.save_on_cpu())
    # pieces of a row start elsewhere, so sums over a row are taken in another order: both are within the
    # rounding u of one value and 2^-20 of the row's sums (V terms of 2^-24) apart
    u = torch.finfo(dtype).eps / 2
    assert ((want.double() - got.double()).abs() <= 2 * u * want.double().abs() + 2.0 ** -20 * want.double().abs().max()).all()


def test_no_gradient_wanted():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(5, 50304, 50257, 64, torch.bfloat16)
    with torch.no_grad():
        a = ops.distillation_loss(z, idx, t, labels, 50257, temperature=2.0, alpha=0.5)
    b = ops.distillation_loss(z.clone().requires_grad_(True), idx, t, labels, 50257, temperature=2.0, alpha=0.5)
    assert torch.equal(a, b.detach()) and not a.requires_grad


def test_same_bits_streams_and_graphs():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(300, 3000, 3000, 12, torch.bfloat16)
    z.requires_grad_(True)
    up = torch.tensor(1.0, device=DEV)

    def run():
        loss = ops.distillation_loss(z, idx, t, labels, temperature=2.0, alpha=0.5)
        return loss.detach(), torch.autograd.grad(loss, z, up)[0]
    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    streams, res = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            res.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in res for a, b in zip(first, r))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = run()
        graphs.append((g, held))
    for i in range(3):
        with torch.no_grad():
            z.copy_(torch.randn_like(z))
            up.fill_(float(i + 1))
        want = run()
        torch.cuda.synchronize()
        for g, held in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals_on_the_gpu():
    from trustworthy_dl import ops
    z, idx, t, labels = on_gpu(4, 9, 9, 3, torch.float32)
    for a, match in (((z.double(), idx, t), "native distillation_loss"), ((z, idx, t.double()), "teacher logits"),
                     ((z, idx.cpu(), t), "is on"), ((z, idx, t.cpu()), "is on")):
        with pytest.raises(ValueError, match=match):
            ops.distillation_loss(*a)


def test_a_student_step_with_both_operators():
    """Embedding, masked attention over packed documents, tied head, distillation: the gradients of one
    training step against the same chain in 64 bits."""
    from trustworthy_dl import ops
    from trustworthy_dl.ops.layers import linear_t
    B, T, H, D, V, K = 2, 96, 4, 64, 500, 6
    C = H * D
    g = torch.Generator(device=DEV).manual_seed(0)

    def w(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * s).bfloat16().requires_grad_(True)
    x, wq, wo, wte = w(B, T, C), w(C, 3 * C, s=C ** -0.5), w(C, C, s=C ** -0.5), w(512, C, s=0.1)
    ids = torch.tensor([[0] * 40 + [1] * 50 + [-1] * 6, [0] * 96], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, V, (B, T, K), generator=g, device=DEV)
    idx[ids < 0] = -1                       # padding has no teacher ...
    t = torch.randn(B, T, K, generator=g, device=DEV)
    labels = torch.randint(0, V, (B, T), generator=g, device=DEV)
    labels[ids < 0] = -100                  # ... and no label
    mask = ops.attention_mask(B, T, documents=ids)
    qkv = ops.linear(x, wq)
    a = ops.masked_attention_packed(qkv, H, mask, softcap=20.0)
    h = x + ops.linear(a, wo)
    loss = ops.distillation_loss(linear_t(h, wte), idx, t, labels, V, temperature=2.0, alpha=0.5)
    got = torch.autograd.grad(loss, (x, wq, wo, wte))

    xd, wqd, wod, wted = (p.detach().double().requires_grad_(True) for p in (x, wq, wo, wte))
    q, k, v = (xd @ wqd).view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
    s = 20.0 * torch.tanh(q @ k.transpose(-1, -2) / math.sqrt(D) / 20.0)
    s = s.masked_fill(~mask.dense()[:, None], -math.inf)
    p = torch.exp(s - torch.where(torch.isinf(s.amax(-1, keepdim=True)), 0.0, s.amax(-1, keepdim=True)).detach())
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    hd = xd + (p @ v).transpose(1, 2).reshape(B, T, C) @ wod
    z = (hd @ wted.t()).view(B * T, -1)
    want_loss, dz = formula(z, idx.view(-1, K), t.view(-1, K), labels.view(-1), V, 2.0, 0.5)
    want = torch.autograd.grad(z, (xd, wqd, wod, wted), dz)
    # the chain rounds a value to bf16 at most 8 times on the way to any gradient (the products, the
    # probabilities, dS and the gradients between them), each 2^-8 at most of a term's magnitude and
    # independent over sums of many terms: 8 x 2^-8 in the norm bounds them all in phase
    assert abs(float(loss) - want_loss) <= 2.0 ** -5 * want_loss
    for a_, b_, n in zip(got, want, ("x", "wq", "wo", "wte")):
        assert float((a_.double() - b_).norm() / b_.norm()) <= 8 * 2.0 ** -8, n
