"""Masked attention on the GPU against the 64-bit definition, with the bounds of masked_attention_oracle."""
import contextlib
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


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(seed, *shape, dtype=BF, mul=1.0):
    return (torch.randn(*shape, generator=_gen(seed), device=DEV) * mul).to(dtype)


def _mask_args(kind, B, Tq, Tk, seed=0):
    g = torch.Generator().manual_seed(seed + 17 * Tk)
    if kind == "causal":
        return {}
    if kind == "full":
        return {"causal": False}
    if kind in ("documents", "documents_prefix"):
        ids = torch.cumsum((torch.rand(B, Tk, generator=g) < 3.0 / max(Tk, 3)).int(), 1).int()
        if Tk > 4:
            ids[:, -(Tk // 9) - 1:] = -1     # padding at the end of every row
            ids[-1] = -1                     # a row of nothing else
        kw = {"documents": ids.to(DEV)}
        if kind == "documents_prefix":
            kw["prefix"] = (torch.rand(B, Tk, generator=g) < 0.9).to(DEV)
        return kw
    if kind == "prefix":
        return {"prefix": torch.randint(-1, Tk + 2, (B,), generator=g).int().to(DEV)}
    lengths = torch.randint(0, Tk + 1, (B,), generator=g).int()
    lengths[0] = Tk
    return {"lengths": lengths.to(DEV)}


@pytest.mark.parametrize("kind", ["causal", "full", "documents", "documents_prefix", "prefix", "lengths"])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 129), (5, 5), (33, 200), (64, 64), (1500, 1500), (77, 3000)])
def test_mask_is_the_cpu_mask(kind, Tq, Tk):
    from trustworthy_dl import ops
    kw = _mask_args(kind, 3, Tq, Tk)
    got = ops.attention_mask(3, Tq, Tk, device=DEV, **kw)
    want = ops.attention_mask(3, Tq, Tk, **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    for n in ("lo", "hi", "pos"):
        assert torch.equal(getattr(got, n).cpu(), getattr(want, n)), n
    # the tables against the intervals
    lo, hi = want.lo.long(), want.hi.long()
    nq = -(-Tq // 32)
    pad = torch.zeros(3, nq * 32 - Tq, dtype=torch.long)
    l32, h32 = (torch.cat([t, pad], 1).view(3, nq, 32) for t in (lo, hi))
    some = h32 > l32
    big = 2 ** 31 - 1
    tab = torch.stack([torch.where(some, l32, big).amin(-1), h32.amax(-1), l32.amax(-1), h32.amin(-1)], -1)
    assert torch.equal(got.q_table.cpu().long(), tab)
    for b in range(3):
        for kb in range(-(-Tk // 128)):
            hit = [t for t in range(nq) if tab[b, t, 0] < (kb + 1) * 128 and tab[b, t, 1] > kb * 128]
            assert got.k_table[b, kb].tolist() == ([hit[0], hit[-1] + 1] if hit else [0, 0])


def _check(B, Tq, Tk, H, Hk, D, dtype, kind, cap=None, alibi=False, train=True, mul=1.0, scale=None, seed=0, mask_args=None):
    from trustworthy_dl import ops
    print(f"case B={B} Tq={Tq} Tk={Tk} H={H} Hk={Hk} D={D} {dtype} {kind} cap={cap} alibi={alibi} train={train}", flush=True)
    q, k, v = _rand(seed, B, Tq, H, D, dtype=dtype, mul=mul), _rand(seed + 1, B, Tk, Hk, D, dtype=dtype), _rand(seed + 2, B, Tk, Hk, D, dtype=dtype)
    do = _rand(seed + 3, B, Tq, H, D, dtype=dtype) if train else None
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device=DEV) if alibi else None
    kw = _mask_args(kind, B, Tq, Tk, seed) if mask_args is None else mask_args
    mask = ops.attention_mask(B, Tq, Tk, device=DEV, **kw)
    if train:
        for t in (q, k, v):
            t.requires_grad_(True)
    out, lse = ops.masked_attention(q, k, v, mask, softcap=cap, slopes=slopes, scale=scale, return_lse=True)
    want = oracle.run(q, k, v, mask.dense(), mask.pos.long(), scale or 1 / math.sqrt(D), cap or 0.0, slopes, do)
    oracle.check(out.detach(), want["out"], "out")
    fin = torch.isfinite(want["lse"])
    assert torch.equal(fin, torch.isfinite(lse)) and (lse[~fin] == -math.inf).all()
    assert ((lse.double() - want["lse"])[fin].abs() <= 2.0 ** -13).all()
    if train:
        for g, n in zip(torch.autograd.grad(out, (q, k, v), do), ("dq", "dk", "dv")):
            oracle.check(g, want[n], n)


@pytest.mark.parametrize("kind", ["causal", "documents", "prefix", "lengths", "full", "documents_prefix"])
@pytest.mark.parametrize("T", [1, 31, 64, 129, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_train_masks_and_lengths(kind, T, D):
    _check(2, T, T, 4, 2, D, BF, kind)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap,alibi", [(None, False), (5.0, False), (None, True), (20.0, True)])
@pytest.mark.parametrize("D,heads", [(64, (3, 3)), (128, (4, 1)), (40, (2, 2)), (96, (6, 2)), (8, (1, 1))])
def test_train_scores_and_heads(dtype, cap, alibi, D, heads):
    _check(2, 161, 161, *heads, D, dtype, "documents", cap=cap, alibi=alibi, mul=3.0 if cap else 1.0)


@pytest.mark.parametrize("Tq,Tk", [(17, 18), (40, 500), (130, 257), (33, 1025)])
def test_queries_at_the_end_of_a_cache(Tq, Tk):
    _check(2, Tq, Tk, 4, 2, 64, BF, "lengths", alibi=True)
    _check(2, Tq, Tk, 2, 1, 128, HF, "causal", cap=10.0)


@pytest.mark.parametrize("Tq", [1, 2, 7, 16])
@pytest.mark.parametrize("Tk", [16, 33, 300, 2050])
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (12, 1)])
def test_few_queries(Tq, Tk, heads):
    for D, dtype, cap, alibi in ((64, BF, None, True), (128, HF, 12.0, False), (128, BF, None, False), (72, BF, 30.0, True)):
        _check(3, Tq, Tk, *heads, D, dtype, "lengths", cap=cap, alibi=alibi, train=False)
    _check(2, Tq, Tk, *heads, 64, BF, "documents", train=True)


def test_more_than_eight_waves_of_queries():
    _check(4, 700, 700, 44, 44, 64, BF, "documents_prefix")     # 8 waves a workgroup
    _check(1, 2300, 2300, 2, 1, 128, BF, "causal", cap=50.0, mul=4.0)


def test_long_positions_keep_their_distance():
    _check(1, 3, 20000, 4, 1, 64, BF, "causal", alibi=True, train=False, mask_args={"q_start": torch.tensor([19997], device=DEV).int()})


def test_strides_views_and_copies():
    from trustworthy_dl import ops
    B, T, H, D = 2, 150, 4, 64
    base = _rand(1, B, T, 3, H, D)
    mask = ops.attention_mask(B, T, device=DEV)
    want = [t.contiguous() for t in base.unbind(2)]
    ref = ops.masked_attention(*want, mask)
    assert torch.equal(ops.masked_attention(*base.unbind(2), mask), ref)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in want]
    assert torch.equal(ops.masked_attention(*heads_first, mask), ref)
    odd = torch.empty(B, T, H, D + 1, dtype=BF, device=DEV)          # rows that are not 16-byte aligned
    odd[..., 1:] = want[0]
    assert torch.equal(ops.masked_attention(odd[..., 1:], want[1], want[2], mask), ref)
    flipped = [t.flip(-1).contiguous() for t in want]
    cols = [torch.empty(B, T, H, 2 * D, dtype=BF, device=DEV) for _ in range(2)]
    for c, f in zip(cols, flipped[:2]):
        c[..., ::2] = f
    got = ops.masked_attention(cols[0][..., ::2], cols[1][..., ::2], want[2], mask)   # column stride 2
    assert torch.equal(got, ops.masked_attention(flipped[0], flipped[1], want[2], mask))
    shared = _rand(5, 1, T, H, D).expand(B, T, H, D)                 # one batch row of keys for all
    assert torch.equal(ops.masked_attention(want[0], shared, shared, mask),
                       ops.masked_attention(want[0], shared.contiguous(), shared.contiguous(), mask))


def test_gradients_of_expanded_and_summed():
    from trustworthy_dl import ops
    B, T, H, D = 3, 70, 2, 64
    mask = ops.attention_mask(B, T, device=DEV)
    q, k1 = _rand(1, B, T, H, D), _rand(2, 1, T, H, D).requires_grad_(True)
    out = ops.masked_attention(q, k1.expand(B, T, H, D), k1.expand(B, T, H, D), mask)
    (g,) = torch.autograd.grad(out.sum(), k1)       # dout is an expanded scalar
    kf = k1.detach().expand(B, T, H, D).contiguous().requires_grad_(True)
    vf = kf.detach().clone().requires_grad_(True)
    dk, dv = torch.autograd.grad(ops.masked_attention(q, kf, vf, mask), (kf, vf), torch.ones_like(out))
    want = (dk.double() + dv.double()).sum(0, keepdim=True)
    # autograd adds the two gradients and the B rows in bf16: at most B + 1 roundings of partial sums
    bound = (B + 1) * 2.0 ** -8 * (dk.double().abs() + dv.double().abs()).sum(0, keepdim=True)
    assert ((g.double() - want).abs() <= bound).all()


def test_packed():
    from trustworthy_dl import ops
    x = _rand(3, 2, 140, (4 + 2 * 2) * 64).requires_grad_(True)
    do = _rand(4, 2, 140, 4 * 64)
    mask = ops.attention_mask(2, 140, device=DEV)
    out = ops.masked_attention_packed(x, 4, mask, n_kv_head=2, softcap=8.0)
    (g,) = torch.autograd.grad(out, x, do)
    y = x.detach().view(2, 140, 8, 64).requires_grad_(True)
    o2 = ops.masked_attention(*y.split((4, 2, 2), 2), mask, softcap=8.0)
    (g2,) = torch.autograd.grad(o2, y, do.view(2, 140, 4, 64))
    assert torch.equal(out, o2.reshape(out.shape)) and torch.equal(g, g2.reshape(g.shape))


def test_same_as_dense_causal_attention():
    from trustworthy_dl import ops
    x = _rand(9, 2, 256, 3 * 4 * 64)
    a, b = ops.causal_attention(x, 4).double(), ops.masked_attention_packed(x, 4, ops.attention_mask(2, 256, device=DEV)).double()
    # both round P and the result once: at most 4 u sum P |v| <= 4 u max |v| apart
    assert (a - b).abs().max() <= 4 * 2.0 ** -8 * x.double().abs().max()


@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("T", [48, 200])
def test_unseen_garbage_has_no_effect(T, D):
    """NaN and infinities in every masked place: padding, another document, behind the cache's length,
    and the future of a causal row."""
    from trustworthy_dl import ops
    B, H, Hk = 2, 4, 2
    cut = T // 3 + 5
    ids = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    ids[:, cut:] = 1
    ids[:, T - 4:] = -1
    mask = ops.attention_mask(B, T, documents=ids)
    q, k, v, do = (_rand(i, B, T, h, D) for i, h in enumerate((H, Hk, Hk, H)))

    def run():
        ins = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out, lse = ops.masked_attention(*ins, mask, return_lse=True)
        return [out.detach(), *torch.autograd.grad(out, ins, do)]
    clean = run()
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in (q, k, v, do):
            t[:, T - 4:] = bad
    with_pad = run()
    for a, b, n in zip(clean, with_pad, ("out", "dq", "dk", "dv")):
        assert torch.equal(a, b), n
    # a key and a value of the second document that are not finite: the first document, and the
    # second's earlier positions, as before; every position that sees them is NaN
    j = cut + 7
    for t, both in ((k, True), (v, False)):
        keep = t[:, j].clone()
        t[:, j, :, 3] = float("nan")
        t[:, j, :, 5] = float("inf")
        got = run()
        for a, b, n in zip(clean, got, ("out", "dq", "dk", "dv")):
            if n in ("out", "dq"):
                assert torch.equal(a[:, :j], b[:, :j]) and torch.equal(a[:, T - 4:], b[:, T - 4:]), n
                hit = b[:, j:T - 4]
                if n == "out" and not both:     # a value: its own columns
                    assert torch.isnan(hit[..., 3]).all() and torch.isposinf(hit[..., 5]).all()
                    rest = [c for c in range(D) if c not in (3, 5)]
                    assert torch.isfinite(hit[..., rest]).all()
                else:
                    assert torch.isnan(hit).all(), n
            else:
                assert torch.equal(a[:, :cut], b[:, :cut]) and torch.equal(a[:, T - 4:], b[:, T - 4:]), n
        t[:, j] = keep
    # an upstream gradient that is not finite reaches the keys its position sees, and no others
    do[:, j, :, 1] = float("inf")
    got = run()
    assert torch.equal(clean[0], got[0])
    assert torch.equal(clean[1][:, :j], got[1][:, :j]) and torch.equal(clean[1][:, j + 1:], got[1][:, j + 1:])
    for a, b in zip(clean[2:], got[2:]):
        assert torch.equal(a[:, :cut], b[:, :cut]) and torch.equal(a[:, j + 1:], b[:, j + 1:])
    assert not torch.isfinite(got[2][:, cut:j + 1]).any()    # inf - inf or inf
    assert torch.isposinf(got[3][:, cut:j + 1, :, 1]).all()
    rest = [c for c in range(D) if c != 1]
    assert torch.equal(got[3][..., rest], clean[3][..., rest])


@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("what", ["dout", "query"])
def test_not_finite_queries_and_gradients_reach_what_they_see(D, what):
    """One row's infinity and NaN: every key that the row sees, in blocks that the row's tile sees whole or
    in part, and nothing else."""
    from trustworthy_dl import ops
    B, T, H, Hk, i = 2, 300, 4, 2, 200
    mask = ops.attention_mask(B, T, device=DEV)
    q, k, v, do = (_rand(n, B, T, h, D) for n, h in enumerate((H, Hk, Hk, H)))

    def run():
        ins = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(ops.masked_attention(*ins, mask), ins, do)
    clean = run()
    t = do if what == "dout" else q
    t[:, i, :, 3] = float("nan")
    t[:, i, :, 5] = float("inf")
    dq, dk, dv = run()
    others = [r for r in range(T) if r != i]
    assert torch.equal(dq[:, others], clean[0][:, others]) and torch.isnan(dq[:, i]).all()
    for g, c in ((dk, clean[1]), (dv, clean[2])):
        assert torch.equal(g[:, i + 1:], c[:, i + 1:])
    assert torch.isnan(dk[:, :i + 1]).all()
    if what == "query":
        assert torch.isnan(dv[:, :i + 1]).all()
    else:      # dV: the gradient's own columns
        assert torch.isnan(dv[:, :i + 1, :, 3]).all() and torch.isposinf(dv[:, :i + 1, :, 5]).all()
        rest = [c for c in range(D) if c not in (3, 5)]
        assert torch.equal(dv[..., rest], clean[2][..., rest])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap", [30.0, 32.0, 33.0, 1000.0])
def test_capped_scores_at_their_bounds(dtype, cap):
    """Scores that saturate the cap on both sides (weights of e^(-2 cap)), and rows all of whose scores do."""
    from trustworthy_dl import ops
    if cap < 2 ** 7 / 1.4427:    # (the oracle's bound is for scores below 2^7)
        _check(2, 161, 161, 3, 3, 64, dtype, "documents", cap=cap, mul=20.0)
    v = _rand(5, 1, 70, 2, 64, dtype=dtype)
    mask = ops.attention_mask(1, 70, causal=False, device=DEV)
    for sign in (1.0, -1.0):
        # every score is the same number near the bound: the mean of the values
        q = torch.full((1, 70, 2, 64), 16.0, dtype=dtype, device=DEV)
        k = torch.full((1, 70, 2, 64), 16.0 * sign, dtype=dtype, device=DEV)
        out, lse = ops.masked_attention(q, k, v, mask, softcap=cap, return_lse=True)
        want = oracle.run(q, k, v, mask.dense(), mask.pos.long(), 0.125, cap)
        oracle.check(out, want["out"], "out")
        # the score less its bound, up to 2 cap: a constant, a sum and a reciprocal of 2^-24, 2^-24 and 2^-23;
        # the bound, its sum and the change of units: 2^-24 of cap each.  Together below cap 2^-20
        assert ((lse.double() - want["lse"]).abs() <= 2.0 ** -13 + cap * 2.0 ** -20).all()


def test_tensors_saved_elsewhere():
    """Saved-tensor hooks bring the operands back contiguous: the same gradients, bit for bit."""
    from trustworthy_dl import ops
    x = _rand(11, 2, 150, (4 + 2 + 2) * 64)
    mask = ops.attention_mask(2, 150, device=DEV)
    do = _rand(12, 2, 150, 4 * 64)

    def grad(packed, hooks):
        z = x.clone().requires_grad_(True)
        with hooks:
            if packed:
                out = ops.masked_attention_packed(z, 4, mask, n_kv_head=2)
            else:
                out = ops.masked_attention(*z.view(2, 150, 8, 64).split((4, 2, 2), 2), mask).reshape(2, 150, -1)
        return torch.autograd.grad(out, z, do)[0]
    for packed in (True, False):
        assert torch.equal(grad(packed, contextlib.nullcontext()), grad(packed, torch.autograd.graph.save_on_cpu()))


@pytest.mark.parametrize("Tk", [100, 1500])
def test_cache_garbage_behind_its_length(Tk):
    from trustworthy_dl import ops
    lengths = torch.tensor([Tk // 2 + 3, 0, Tk], dtype=torch.int32, device=DEV)
    mask = ops.attention_mask(3, 1, Tk, lengths=lengths)
    q, k, v = _rand(0, 3, 1, 8, 128), _rand(1, 3, Tk, 2, 128), _rand(2, 3, Tk, 2, 128)
    clean = ops.masked_attention(q, k, v, mask)
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    assert torch.equal(ops.masked_attention(q, k, v, mask), clean)
    assert (clean[1] == 0).all()
    v[0, 5, 0, 7] = float("nan")      # a visible one
    got = ops.masked_attention(q, k, v, mask)
    assert torch.isnan(got[0, 0, :4, 7]).all()      # its column of the heads that read it, nothing else
    clean[0, 0, :4, 7] = got[0, 0, :4, 7] = 0
    assert torch.equal(got, clean)


def test_huge_scores_and_lowest_values():
    from trustworthy_dl import ops
    low = torch.finfo(BF).min
    q, k, v = _rand(0, 1, 40, 1, 64), _rand(1, 1, 40, 1, 64), _rand(2, 1, 40, 1, 64)
    k[:, 7] = 1e4        # scores of +-1e5: one key takes all or nothing
    m = ops.attention_mask(1, 40, device=DEV)
    want = oracle.run(q, k, v, m.dense(), m.pos.long(), 0.125)["out"][0]
    got = ops.masked_attention(q, k, v, m)
    # the scores' own 32-bit error is 2^-24 x 1e5 x a few here: compare where one key has all the weight
    assert ((got.double() - want).abs() <= 0.05 * v.double().abs().max()).all() and torch.isfinite(got).all()
    q[:, 3:5], k[:, 9] = low, low        # finite inputs whose products overflow: NaN or finite, other rows unharmed
    got2 = ops.masked_attention(q, k, v, m)
    assert torch.equal(got2[:, :3], got[:, :3]) and torch.equal(got2[:, 5:9], got[:, 5:9])


def test_offsets_past_32_bits():
    from trustworthy_dl import ops
    Tk, stride = 4200, 1 << 20          # a cache of 4.4e9 elements, one slice of each token used
    store = torch.empty(Tk * stride, dtype=BF, device=DEV)
    k = store.as_strided((1, Tk, 2, 64), (0, stride, 64, 1))
    v = store.as_strided((1, Tk, 2, 64), (0, stride, 64, 1), 4096)
    kc, vc = _rand(1, 1, Tk, 2, 64), _rand(2, 1, Tk, 2, 64)
    k.copy_(kc)
    v.copy_(vc)
    for Tq in (1, 64):
        q = _rand(3, 1, Tq, 4, 64)
        m = ops.attention_mask(1, Tq, Tk, device=DEV)
        assert torch.equal(ops.masked_attention(q, k, v, m), ops.masked_attention(q, kc, vc, m))


def test_runs_are_the_same_bits_and_streams():
    from trustworthy_dl import ops
    q, k, v, do = (_rand(i, 2, 500, h, 64) for i, h in enumerate((4, 2, 2, 4)))
    mask = ops.attention_mask(2, 500, device=DEV)

    def run():
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.masked_attention(*ins, mask)
        return [out.detach(), *torch.autograd.grad(out, ins, do)]
    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    for s in streams:       # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            res.append(run())
    torch.cuda.synchronize()
    for r in res:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


@pytest.mark.parametrize("Tq,Tk", [(200, 200), (1, 3000)])
def test_captured_and_replayed(Tq, Tk):
    from trustworthy_dl import ops
    q, k, v, do = (_rand(i, 2, t, h, 64) for i, (t, h) in enumerate(((Tq, 4), (Tk, 2), (Tk, 2), (Tq, 4))))
    lengths = torch.tensor([Tk, max(Tq, Tk // 3)], dtype=torch.int32, device=DEV)
    ins = [t.requires_grad_(True) for t in (q, k, v)]

    def run():
        mask = ops.attention_mask(2, Tq, Tk, lengths=lengths)
        out = ops.masked_attention(*ins, mask, softcap=9.0)
        return [out.detach(), *torch.autograd.grad(out, ins, do)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = run()
        graphs.append((g, held))
    for i in range(3):
        with torch.no_grad():
            q.copy_(_rand(50 + i, 2, Tq, 4, 64))
            lengths[1] = max(Tq, Tk // (i + 2))
        want = run()
        torch.cuda.synchronize()
        for g, held in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_only_queries_need_a_gradient():
    from trustworthy_dl import ops
    q, k, v, do = (_rand(i, 1, 90, 2, 64) for i in range(4))
    m = ops.attention_mask(1, 90, device=DEV)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(ops.masked_attention(*full, m), full, do)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.masked_attention(q, k, v, m), q, do)
    assert torch.equal(dq, want[0])


def test_refusals_on_the_gpu():
    from trustworthy_dl import ops
    m = ops.attention_mask(1, 8, device=DEV)

    def bad(match, q, k=None, mask=m, **kw):
        with pytest.raises(ValueError, match=match):
            ops.masked_attention(q, q if k is None else k, q if k is None else k, mask, **kw)
    z = torch.zeros
    bad("bfloat16 and float16", z(1, 8, 2, 64, device=DEV))
    bad("head dims", z(1, 8, 2, 136, device=DEV, dtype=BF))
    bad("head dims", z(1, 8, 2, 20, device=DEV, dtype=BF))
    bad("are on", z(1, 8, 2, 64, dtype=BF))
    bad("are on", z(1, 8, 2, 64, device=DEV, dtype=BF), mask=ops.attention_mask(1, 8))
    bad("slopes must be", z(1, 8, 2, 64, device=DEV, dtype=BF), slopes=z(2))
    with pytest.raises(ValueError, match="is on"):
        ops.attention_mask(1, 8, documents=z(1, 8, dtype=torch.int32), device=DEV)
