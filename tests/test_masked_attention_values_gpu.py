"""Masked attention on the GPU at values and positions away from the ordinary: biases that grow with the
distance, large values under fp16 gradients, long rows, far positions, operands that views, hooks and graphs
bring in other layouts.  Bounds of masked_attention_oracle, others where stated."""
import math

import pytest
import torch

import masked_attention_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _native():
    from trustworthy_dl.ops import _lib
    _lib.lib()


def _rand(seed, *shape, dtype=BF, mul=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * mul).to(dtype)


def _grads(q, k, v, do, mask, **kw):
    from trustworthy_dl import ops
    ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.masked_attention(*ins, mask, **kw)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, ins, do))))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap", [None, 10.0])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [2, 129, 190])
def test_bias_towards_far_keys(T, D, cap, dtype):
    """Negative slopes; the rows behind the last query in its tile would weigh the far keys without bound."""
    from trustworthy_dl import ops
    print(f"case T={T} D={D} cap={cap} {dtype}", flush=True)
    H, Hk = 4, 2
    q, k, v, do = (_rand(i, 2, T, h, D, dtype=dtype) for i, h in enumerate((H, Hk, Hk, H)))
    # (scores below 2^7 in units of log 2, those of rows up to the next multiple of 32 not)
    slopes = torch.tensor([-78.0 / max(T, 129), -0.1, 0.2, -0.3], device=DEV)
    mask = ops.attention_mask(2, T, device=DEV)
    got = _grads(q, k, v, do, mask, softcap=cap, slopes=slopes)
    want = oracle.run(q, k, v, mask.dense(), mask.pos.long(), 1 / math.sqrt(D), cap or 0.0, slopes, do)
    for n, g in got.items():
        assert torch.isfinite(g).all(), n
        oracle.check(g, want[n], n)


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("D", [8, 64, 128])
@pytest.mark.parametrize("size,T", [(16.0, 2), (16.0, 161), (64.0, 70), (1000.0, 300), (1e-3, 161)])
@pytest.mark.parametrize("aligned", [True, False])
def test_fp16_gradients_of_large_values(aligned, size, T, D, cap):
    """|dO . (v - o)| far above |dO|: no gradient overflows that fp16 can hold."""
    from trustworthy_dl import ops
    print(f"case aligned={aligned} size={size} T={T} D={D} cap={cap}", flush=True)
    H, Hk = 4, 2
    q, k = _rand(0, 2, T, H, D, dtype=HF, mul=0.5), _rand(1, 2, T, Hk, D, dtype=HF, mul=1.0 / max(1.0, size / 32))
    if aligned:
        v = (torch.sign(_rand(2, 2, T, Hk, 1, dtype=HF)) * size).expand(2, T, Hk, D).contiguous()
        do = torch.ones(2, T, H, D, dtype=HF, device=DEV)
    else:
        v, do = _rand(2, 2, T, Hk, D, dtype=HF, mul=size), _rand(3, 2, T, H, D, dtype=HF)
    mask = ops.attention_mask(2, T, device=DEV, causal=T > 2)
    got = _grads(q, k, v, do, mask, softcap=cap)
    scale = 1 / math.sqrt(D)
    seen = mask.dense()
    want = oracle.run(q, k, v, seen, mask.pos.long(), scale, cap or 0.0, None, do)
    assert all(float(want[n][0].abs().max()) < 60000 for n in got)      # representable
    # dX is kept times a power of two 2^n with 2^n max|dO_i| max|v_j| / 2 in [2^14, 2^15) (row norms: P (1 - P) times
    # twice them bounds |dX|), so below fp16's normal range it is off by 2^-25 2^-n a visible pair
    step = 2.0 ** -25 * 2.0 ** -14 * 0.5 * float(do.double().norm(dim=-1).max() * v.double().norm(dim=-1).max())
    s = seen.double()[:, None]
    kk, qq = k.double().abs().transpose(1, 2).repeat_interleave(H // Hk, 1), q.double().abs().transpose(1, 2)
    more = {"dq": (s @ kk).transpose(1, 2) * scale * step * (4 if cap else 1),
            "dk": (s.transpose(-1, -2) @ qq).view(2, Hk, H // Hk, T, D).sum(2).transpose(1, 2) * scale * step * (4 if cap else 1)}
    for n, g in got.items():
        assert torch.isfinite(g).all(), n
        oracle.check(g, (want[n][0], want[n][1] + more.get(n, 0.0)), n)


@pytest.mark.parametrize("D", [64, 128])
def test_fp16_weights_of_long_rows(D):
    """166937 keys of equal weight, 2^24 / 100.5 of them: a weight rounded below fp16's normal range would be
    half a step, 0.5 %, off in every term alike."""
    from trustworthy_dl import ops
    Tq, Tk = 40, 166937
    q = torch.zeros(1, Tq, 1, D, dtype=HF, device=DEV)
    k, v = _rand(1, 1, Tk, 1, D, dtype=HF), _rand(2, 1, Tk, 1, D, dtype=HF)
    do = torch.ones(1, Tq, 1, D, dtype=HF, device=DEV)
    mask = ops.attention_mask(1, Tq, Tk, causal=False, device=DEV)
    dv = _grads(q, k, v, do, mask)["dv"].double()
    exact = Tq / Tk
    # P and the result are rounded once each (2^-11), the rest is in 32 bits (2^-13)
    assert ((dv - exact).abs() <= (2.0 ** -10 + 2.0 ** -12) * exact).all()


@pytest.mark.parametrize("Tq", [1, 5, 40, 130])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_small_weights_beside_a_large_one(Tq, D):
    """One key has nearly all the weight, and the others, 2^-25 of it each, half a percent together."""
    from trustworthy_dl import ops
    Tk = 166937
    q, k = torch.zeros(1, Tq, 2, D, dtype=HF, device=DEV), torch.zeros(1, Tk, 1, D, dtype=HF, device=DEV)
    q[..., 0], k[:, 5, :, 0] = 8.0, 17.375 / 8.0 * math.sqrt(D)
    v = torch.ones(1, Tk, 1, D, dtype=HF, device=DEV)
    v[:, 5] = 0
    mask = ops.attention_mask(1, Tq, Tk, causal=False, device=DEV)
    got = ops.masked_attention(q, k, v, mask).double()
    want = oracle.run(q, k, v, mask.dense(), mask.pos.long(), 1 / math.sqrt(D))["out"][0]
    assert ((got - want).abs() <= (2.0 ** -10 + 2.0 ** -12) * want).all()


@pytest.mark.parametrize("Tq", [3, 70])
@pytest.mark.parametrize("cap", [None, 10.0])
def test_distances_at_far_positions(Tq, cap):
    """Positions past 2^24, where neighbours are the same number in 32 bits: the distances are those of the
    same tokens at the start of a row."""
    from trustworthy_dl import ops
    D, far, n = 8, (1 << 24) + 12345, 150
    Tk = far + n
    q, do = _rand(0, 1, Tq, 2, D), _rand(3, 1, Tq, 2, D)
    ks, vs = _rand(1, 1, n, 1, D), _rand(2, 1, n, 1, D)
    k, v = (torch.zeros(1, Tk, 1, D, dtype=BF, device=DEV) for _ in range(2))
    k[:, far:], v[:, far:] = ks, vs
    ids = torch.zeros(1, Tk, dtype=torch.int32, device=DEV)
    ids[:, far:] = 1
    slopes = torch.tensor([0.7, 0.21], device=DEV)
    got = _grads(q, k, v, do, ops.attention_mask(1, Tq, Tk, documents=ids), softcap=cap, slopes=slopes)
    near = ops.attention_mask(1, Tq, n, device=DEV)
    want = oracle.run(q, ks, vs, near.dense(), near.pos.long(), 1 / math.sqrt(D), cap or 0.0, slopes, do)
    for name in ("out", "dq"):
        oracle.check(got[name], want[name], name)
    for name in ("dk", "dv"):
        assert (got[name][:, :far] == 0).all()
        oracle.check(got[name][:, far:], want[name], name)


def test_operands_cut_from_a_flat_buffer():
    """q, k, v and the upstream gradient, dense and at an odd offset, give what aligned copies give."""
    from trustworthy_dl import ops
    B, T, D = 2, 100, 64
    mask = ops.attention_mask(B, T, device=DEV)
    want_in = [_rand(i, B, T, h, D) for i, h in enumerate((4, 2, 2, 4))]
    cut = []
    for t in want_in:
        flat = torch.zeros(t.numel() + 3, dtype=BF, device=DEV)
        flat[3:] = t.flatten()
        cut.append(flat[3:].view(t.shape))
    a, b = _grads(*want_in, mask), _grads(*cut, mask)
    assert all(torch.equal(a[n], b[n]) for n in a)
    x = torch.cat(want_in[:3], 2).reshape(B, T, -1)
    flat = torch.zeros(x.numel() + 1, dtype=BF, device=DEV)
    flat[1:] = x.flatten()
    assert torch.equal(ops.masked_attention_packed(flat[1:].view(x.shape), 4, mask, n_kv_head=2).view(B, T, 4, D), a["out"])


@pytest.mark.parametrize("packed", [True, False])
def test_hooks_that_change_layouts(packed):
    """Saved-tensor hooks that bring every tensor back with other strides and at an odd offset: the same
    gradients.  Ones that bring it back on another device, in another type or shape are refused."""
    from trustworthy_dl import ops
    B, T, H, Hk, D = 2, 150, 4, 2, 64
    x, do = _rand(11, B, T, (H + 2 * Hk) * D), _rand(12, B, T, H * D)
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4], device=DEV)
    mask = ops.attention_mask(B, T, device=DEV)

    def grad(unpack):
        z = x.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            if packed:
                out = ops.masked_attention_packed(z, H, mask, n_kv_head=Hk, slopes=slopes)
            else:
                out = ops.masked_attention(*z.view(B, T, H + 2 * Hk, D).split((H, Hk, Hk), 2), mask, slopes=slopes).reshape(B, T, -1)
        return torch.autograd.grad(out, z, do)[0]

    def strided(t):     # one column in two, from an odd element
        store = torch.full((2 * t.numel() + 1,), 7, dtype=t.dtype, device=t.device)
        back = store[1:].view(*t.shape, 2)[..., 0]
        back.copy_(t)
        return back

    def shifted(t):
        store = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        store[1:] = t.flatten()
        return store[1:].view(t.shape)

    def last_first(t):
        return t.transpose(0, -1).contiguous().transpose(0, -1)
    want = grad(lambda t: t)
    for f in (strided, shifted, last_first):
        assert torch.equal(grad(f), want), f.__name__
    for f in (lambda t: t.cpu(), lambda t: t[:1], lambda t: t.double()):
        with pytest.raises(RuntimeError, match="came back"):
            grad(f)


@pytest.mark.parametrize("what", ["lo", "hi", "pos", "q_table", "k_table"])
def test_a_mask_changed_before_the_backward_pass(what):
    from trustworthy_dl import ops
    mask = ops.attention_mask(1, 40, device=DEV)
    x = _rand(0, 1, 40, 3 * 64).requires_grad_(True)
    outs = [ops.masked_attention_packed(x, 1, mask), ops.masked_attention(*x.view(1, 40, 3, 64).split(1, 2), mask)]
    getattr(mask, what).zero_()
    for out in outs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_a_mask_made_in_inference_mode_serves_training():
    from trustworthy_dl import ops
    x = _rand(0, 1, 40, 3 * 64).requires_grad_(True)
    with torch.inference_mode():
        mask = ops.attention_mask(1, 40, device=DEV)
        seen = ops.masked_attention_packed(x, 1, mask)
    out = ops.masked_attention_packed(x, 1, mask)
    out.sum().backward()
    assert torch.equal(out, seen) and torch.isfinite(x.grad).all()


def test_forward_mode_is_refused():
    """A tangent would be lost where no input wants a gradient."""
    from torch.autograd import forward_ad

    from trustworthy_dl import ops
    mask = ops.attention_mask(1, 40, device=DEV)
    t = [_rand(i, 1, 40, 1, 64) for i in range(3)]
    slopes = torch.tensor([0.1], device=DEV)
    want = ops.masked_attention(*t, mask, slopes=slopes)
    with forward_ad.dual_level():
        assert torch.equal(ops.masked_attention(*t, mask, slopes=slopes), want)
        for i in range(3):
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(t)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.masked_attention(*dual, mask)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.masked_attention(*t, mask, slopes=forward_ad.make_dual(slopes, slopes))
        x = torch.cat(t, 2).reshape(1, 40, -1)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.masked_attention_packed(forward_ad.make_dual(x, x), 1, mask)
        z = _rand(5, 4, 9).float()
        with pytest.raises(NotImplementedError):
            ops.distillation_loss(forward_ad.make_dual(z, z), torch.zeros(4, 2, dtype=torch.long, device=DEV), z[:, :2])


def test_no_grad_keeps_nothing_for_a_backward_pass():
    """Under no_grad, of an input that requires a gradient: the output's memory and no more."""
    from trustworthy_dl import ops
    x = _rand(0, 4, 512, 3 * 8 * 64).requires_grad_(True)
    mask = ops.attention_mask(4, 512, device=DEV)
    want = ops.masked_attention_packed(x, 8, mask)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        got = ops.masked_attention_packed(x, 8, mask)
    assert torch.cuda.max_memory_allocated() - before < 1.25 * want.numel() * 2
    assert torch.equal(got, want.detach()) and not got.requires_grad


def test_sizes_out_of_range_are_refused():
    from trustworthy_dl import ops
    mask = ops.attention_mask(1, 1, device=DEV)
    one = torch.zeros(1, 1, 1, 8, dtype=BF, device=DEV)
    q = one.expand(1, 1, 1 << 21, 8)
    with pytest.raises(ValueError, match="2\\^24 elements"):
        ops.masked_attention(q, q, q, mask)
    n = 1 << 20
    mask = ops.attention_mask(n, 1, device=DEV)
    q, k = one.expand(n, 1, 512, 8), one.expand(n, 1, 32, 8)
    with pytest.raises(ValueError, match="split the batch"):
        ops.masked_attention(q, k, k, mask)


def test_a_mask_dropped_while_another_stream_uses_it():
    """record_stream keeps the mask's memory from its own stream's next tensors until the other is done."""
    from trustworthy_dl import ops
    B, T = 2, 512
    ids = (torch.arange(T, device=DEV) // 100).int().expand(B, T)
    q, k, v = (_rand(i, B, T, 4, 64) for i in range(3))
    want = ops.masked_attention(q, k, v, ops.attention_mask(B, T, documents=ids))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    mask = ops.attention_mask(B, T, documents=ids)
    held = {t.data_ptr() for t in (mask.lo, mask.hi, mask.pos, mask.q_table, mask.k_table)}
    shapes = [(t.shape, t.dtype) for t in (mask.lo, mask.hi, mask.pos, mask.q_table, mask.k_table)]
    side.wait_stream(torch.cuda.current_stream())
    big = _rand(7, 4096, 4096)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(30):      # (work ahead of the call on the side stream)
            big = (big @ big).clamp(-1, 1)
        got = ops.masked_attention(q, k, v, mask)
    mask.record_stream(side)
    del mask
    fresh = [torch.zeros(s, dtype=d, device=DEV) for s, d in shapes]
    assert side.query() or not held & {t.data_ptr() for t in fresh}
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("packed", [True, False])
def test_recomputed_under_checkpointing(packed):
    """Activations that a checkpoint throws away and makes again, attention and loss inside: the same gradients."""
    from torch.utils.checkpoint import checkpoint

    from trustworthy_dl import ops
    B, T, H, D, V = 2, 130, 4, 64, 96
    x = _rand(0, B, T, 3 * H * D)
    w = _rand(1, H * D, V, mul=0.05)
    mask = ops.attention_mask(B, T, documents=(torch.arange(T, device=DEV) // 50).int().expand(B, T))
    g = torch.Generator(device=DEV).manual_seed(2)
    idx, t = torch.randint(0, V, (B, T, 5), generator=g, device=DEV), torch.randn(B, T, 5, generator=g, device=DEV)
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4], device=DEV)

    def loss(z):
        if packed:
            a = ops.masked_attention_packed(z, H, mask, slopes=slopes)
        else:
            a = ops.masked_attention(*(z * 1.0).view(B, T, 3 * H, D).split(H, 2), mask, slopes=slopes).reshape(B, T, -1)
        return ops.distillation_loss(a @ w, idx, t, temperature=2.0)
    grads = []
    for again in (False, True):
        for up in (1.0, 3.0):
            z = x.clone().requires_grad_(True)
            out = checkpoint(loss, z, use_reentrant=False) if again else loss(z)
            grads.append(torch.autograd.grad(out, z, torch.tensor(up, device=DEV))[0])
    assert torch.equal(grads[0], grads[2]) and torch.equal(grads[1], grads[3])
    assert float(grads[0].abs().max()) > 0


@pytest.mark.parametrize("what", ["q", "k", "v"])
def test_forward_by_two_threads_backward_by_both(what):
    """One graph kept for two backward passes, made by two threads at once."""
    import threading

    from trustworthy_dl import ops
    mask = ops.attention_mask(2, 300, device=DEV)
    ins = {n: _rand(i, 2, 300, 4, 64) for i, n in enumerate("qkv")}
    ins[what].requires_grad_(True)
    out = ops.masked_attention(*ins.values(), mask)
    ups = [_rand(7 + i, 2, 300, 4, 64) for i in range(2)]
    want = [torch.autograd.grad(out, ins[what], u, retain_graph=True)[0] for u in ups]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        for _ in range(5):
            got[i] = torch.autograd.grad(out, ins[what], ups[i], retain_graph=True)[0]
        torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T", [1, 20, 200])
def test_rows_that_all_see_nothing(T, dtype):
    """Empty rows alone: zeros everywhere, whatever the operands hold."""
    from trustworthy_dl import ops
    for kw in ({"lengths": torch.zeros(2, dtype=torch.int32, device=DEV)}, {"documents": torch.full((2, T), -1, dtype=torch.int32, device=DEV)}):
        mask = ops.attention_mask(2, T, **kw)
        ins = [torch.full((2, T, h, 64), float("nan"), dtype=dtype, device=DEV) for h in (4, 2, 2, 4)]
        got = _grads(*ins, mask, softcap=5.0)
        assert all((g == 0).all() for g in got.values())
        assert (ops.masked_attention(*ins[:3], mask, return_lse=True)[1] == -math.inf).all()


@pytest.mark.parametrize("T", [20, 200])
def test_inference_mode(T):
    from trustworthy_dl import ops
    t = [_rand(i, 2, T, h, 64) for i, h in enumerate((4, 2, 2))]
    want = ops.masked_attention(*t, ops.attention_mask(2, T, device=DEV))
    with torch.inference_mode():
        u = [x.clone() for x in t]
        mask = ops.attention_mask(2, T, device=DEV)
        assert torch.equal(ops.masked_attention(*u, mask), want)
        assert torch.equal(ops.masked_attention_packed(torch.cat(u, 2).reshape(2, T, -1), 4, mask, n_kv_head=2).view(want.shape), want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap", [20.0, 30.0, 32.0, 33.0, 50.0])
@pytest.mark.parametrize("Tq", [5, 70])
def test_a_capped_row_with_all_weight_on_one_key(Tq, cap, dtype):
    """The result is that key's value: its weight's own rounding cancels against the sum's, whatever the weight is."""
    from trustworthy_dl import ops
    D, Tk = 64, 70
    q, k = torch.zeros(1, Tq, 2, D, dtype=dtype, device=DEV), torch.zeros(1, Tk, 2, D, dtype=dtype, device=DEV)
    # scores of +-x, x = 1.1 cap .. 1.9 cap: weights of e^(2 cap tanh(x / cap)) > e^30 of the others
    q[..., 0] = torch.linspace(1.1, 1.9, Tq, device=DEV).to(dtype)[None, :, None] * cap
    k[..., 0] = -8.0
    k[:, 3, :, 0] = 8.0
    v = _rand(5, 1, Tk, 2, D, dtype=dtype)
    out = ops.masked_attention(q, k, v, ops.attention_mask(1, Tq, Tk, causal=False, device=DEV), softcap=cap)
    assert torch.equal(out, v[:, 3:4].expand(out.shape))


@pytest.mark.parametrize("what", [("documents", "lengths"), ("prefix_rows", "lengths"), ("marks",), ("marks", "lengths"), ("documents", "marks", "lengths"),
                                  ("q_start", "lengths"), ("q_start", "documents"), ("full", "documents", "lengths", "q_start"),
                                  ("full", "lengths"), ("q_start", "prefix_rows")])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (7, 150), (150, 150), (40, 2100)])
def test_masks_put_together(what, Tq, Tk):
    """Combinations of the masks' arguments, 64-bit ones among them: the CPU's intervals, and what they let through."""
    from trustworthy_dl import ops
    B, g = 4, torch.Generator().manual_seed(Tk + len(what))
    kw = {"causal": "full" not in what}
    if "documents" in what:
        ids = torch.cumsum((torch.rand(B, Tk, generator=g) < 0.05).long(), 1) + (1 << 40)
        ids[torch.rand(B, Tk, generator=g) < 0.02] = -1
        kw["documents"] = ids
    if "lengths" in what:
        kw["lengths"] = torch.randint(-2, Tk + 5, (B,), generator=g)
    if "prefix_rows" in what:
        kw["prefix"] = torch.randint(-2, Tk + 5, (B,), generator=g)
    if "marks" in what:
        kw["prefix"] = (torch.rand(B, Tk, generator=g) < 0.8).to(torch.uint8) * 3
    if "q_start" in what:
        kw["q_start"] = torch.randint(-3, Tk, (B,), generator=g)
    cpu = ops.attention_mask(B, Tq, Tk, **kw)
    gpu = ops.attention_mask(B, Tq, Tk, **{n: v.to(DEV) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}, device=DEV)
    for n in ("lo", "hi", "pos"):
        assert torch.equal(getattr(gpu, n).cpu(), getattr(cpu, n)), n
    q, k, v, do = (_rand(i, B, t, h, 64) for i, (t, h) in enumerate(((Tq, 4), (Tk, 2), (Tk, 2), (Tq, 4))))
    got = _grads(q, k, v, do, gpu)
    want = oracle.run(q, k, v, gpu.dense(), gpu.pos.long(), 0.125, 0.0, None, do)
    for n, x in got.items():
        oracle.check(x, want[n], n)
