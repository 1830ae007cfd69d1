"""Masked attention on the CPU: the mask against its documented meaning, the reference path against the
64-bit definition and differences, and the refusals."""
import math

import pytest
import torch

import masked_attention_oracle as oracle
from trustworthy_dl import ops

G = torch.Generator


def _rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=G().manual_seed(seed), dtype=dtype)


def mask_cases():
    docs = torch.tensor([[0, 0, 0, 5, 5, 2, 2, 2, 2, -1, -1], [3, 3, 1, 3, 3, 3, -1, 4, 4, 4, 4], [7] * 11])
    marks = torch.tensor([[1, 0, 1, 1, 1, 0, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0, 0, 1, 1, 1, 1], [0] * 11], dtype=torch.bool)
    return {
        "causal": dict(),
        "full": dict(causal=False),
        "documents": dict(documents=docs),
        "documents64": dict(documents=docs.long() + (docs > 3).long() * (1 << 40)),
        "documents_full": dict(documents=docs.int(), causal=False),
        "documents_prefix": dict(documents=docs.int(), prefix=marks),
        "prefix_rows": dict(prefix=torch.tensor([0, 4, 30])),
        "prefix_marks": dict(prefix=marks.to(torch.uint8)),
        "lengths": dict(lengths=torch.tensor([11, 4, 0])),
        "lengths_outside": dict(lengths=torch.tensor([-3, 99, 1])),
        "documents_lengths": dict(documents=docs.int(), lengths=torch.tensor([11, 5, 8], dtype=torch.int32)),
        "q_start": dict(q_start=torch.tensor([0, 5, -2])),
    }


@pytest.mark.parametrize("name", list(mask_cases()))
@pytest.mark.parametrize("q_len", [11, 4, 1])
def test_mask_means_what_it_says(name, q_len):
    kw = mask_cases()[name]
    m = ops.attention_mask(3, q_len, 11, **kw)
    seen, first = oracle.dense(3, q_len, 11, **kw)
    assert torch.equal(m.dense(), seen)
    assert torch.equal(m.pos.long(), first)


@pytest.mark.parametrize("heads", [(4, 4), (4, 2), (3, 1)])
@pytest.mark.parametrize("score", [dict(), dict(softcap=2.0), dict(slopes=True), dict(softcap=1.5, slopes=True, scale=0.7)])
@pytest.mark.parametrize("name", ["causal", "documents", "lengths", "documents_prefix", "full"])
def test_reference_matches_definition(heads, score, name):
    H, Hk = heads
    kw = mask_cases()[name]
    q, k, v, do = _rand(3, 11, H, 8), _rand(3, 11, Hk, 8, seed=1), _rand(3, 11, Hk, 8, seed=2), _rand(3, 11, H, 8, seed=3)
    slopes = torch.rand(H, generator=G().manual_seed(4)) if score.get("slopes") else None
    for t in (q, k, v):
        t.requires_grad_(True)
    opt = dict(softcap=score.get("softcap"), scale=score.get("scale"), slopes=slopes)
    out, lse = ops.masked_attention(q, k, v, ops.attention_mask(3, 11, **kw), return_lse=True, **opt)
    grads = torch.autograd.grad(out, (q, k, v), do)
    seen, first = oracle.dense(3, 11, 11, **kw)
    want = oracle.run(q, k, v, seen, first, score.get("scale", 1 / math.sqrt(8)), score.get("softcap", 0.0), slopes, do)
    for got, n in zip((out, *grads), ("out", "dq", "dk", "dv")):
        assert torch.allclose(got, want[n][0], rtol=1e-11, atol=1e-12), n
    assert torch.allclose(lse.double(), want["lse"], rtol=1e-6, atol=1e-6)
    empty = ~seen.any(-1)
    assert (out.transpose(1, 2)[empty[:, None].expand(-1, H, -1)] == 0).all()


def test_gradient_against_differences():
    docs = torch.tensor([[0, 0, 1, 1, 1, -1]])
    m = ops.attention_mask(1, 6, documents=docs)
    slopes = torch.tensor([0.3, 0.1])

    def f(q, k, v):
        return ops.masked_attention(q, k, v, m, softcap=1.2, slopes=slopes)
    ins = [_rand(1, 6, h, 4, seed=i).requires_grad_(True) for i, h in enumerate((2, 1, 1))]
    assert torch.autograd.gradcheck(f, ins)


def test_packed_is_the_same():
    x = _rand(2, 9, 8 * 4).requires_grad_(True)
    m = ops.attention_mask(2, 9)
    got = ops.masked_attention_packed(x, 4, m, n_kv_head=2)
    q, k, v = x.view(2, 9, 8, 4).split((4, 2, 2), 2)
    want = ops.masked_attention(q, k, v, m).reshape(2, 9, 16)
    assert torch.equal(got, want)
    y = _rand(2, 9, 3 * 64, seed=5)
    dense = ops.causal_attention(y, 2)
    assert torch.allclose(ops.masked_attention_packed(y, 2, m, scale=1 / math.sqrt(32)), dense, rtol=1e-5, atol=1e-5)


def test_unseen_keys_have_no_effect():
    q, k, v = _rand(2, 6, 2, 8), _rand(2, 6, 2, 8, seed=1), _rand(2, 6, 2, 8, seed=2)
    m = ops.attention_mask(2, 6, lengths=torch.tensor([4, 6]))
    clean = ops.masked_attention(q, k, v, m)
    k[0, 4:], v[0, 5] = float("nan"), float("inf")
    assert torch.equal(ops.masked_attention(q, k, v, m), clean)


def test_empty_batches():
    for B, T in ((0, 5), (2, 0)):
        q = torch.zeros(B, T, 2, 8, requires_grad=True)
        out = ops.masked_attention(q, q, q, ops.attention_mask(B, T))
        assert out.shape == (B, T, 2, 8)
        out.sum().backward()


def _bad(fn, match):
    with pytest.raises(ValueError, match=match):
        fn()


def test_refusals():
    z = torch.zeros
    _bad(lambda: ops.attention_mask(1, 5, 4), "q_len <= k_len")
    _bad(lambda: ops.attention_mask(1, 1 << 30), "positions")
    _bad(lambda: ops.attention_mask(2, 4, documents=z(2, 5, dtype=torch.int32)), "shape")
    _bad(lambda: ops.attention_mask(2, 4, documents=z(2, 4)), "documents must be")
    _bad(lambda: ops.attention_mask(2, 4, lengths=[1, 2]), "lengths must be")
    _bad(lambda: ops.attention_mask(2, 4, prefix=z(2, 4, dtype=torch.int32)), "prefix must be")
    _bad(lambda: ops.attention_mask(2, 4, prefix=z(2, dtype=torch.int32), causal=False), "causal")
    _bad(lambda: ops.attention_mask(2, 4, prefix=z(2, dtype=torch.int32), documents=z(2, 4, dtype=torch.int32)), "per position")
    m = ops.attention_mask(2, 4)
    q, k = z(2, 4, 4, 8), z(2, 4, 2, 8)
    f = ops.masked_attention
    _bad(lambda: f(q, k, k, None), "made by attention_mask")
    _bad(lambda: f(q, k, k, ops.attention_mask(2, 3)), "the mask is for")
    _bad(lambda: f(q, z(2, 4, 3, 8), z(2, 4, 3, 8), m), "share the KV heads")
    _bad(lambda: f(q, k, z(2, 4, 2, 16), m), "k and v")
    _bad(lambda: f(q, k.half(), k.half(), m), "differ in type")
    _bad(lambda: f(q.long(), k.long(), k.long(), m), "floating-point")
    for s in (0.0, -1.0, math.inf, math.nan):
        _bad(lambda: f(q, k, k, m, scale=s), "scale")
    for c in (0.0, -5.0, 1001.0, math.nan):
        _bad(lambda: f(q, k, k, m, softcap=c), "softcap")
    _bad(lambda: f(q, k, k, m, slopes=z(3)), "slopes must be")
    _bad(lambda: f(q, k, k, m, slopes=z(4).requires_grad_(True)), "constants")
    _bad(lambda: ops.masked_attention_packed(z(2, 4, 100), 3, m), "does not hold")


def test_few_queries_rule():
    from trustworthy_dl.ops.masked_attention import few_queries
    assert few_queries(1, 12, 1, 128, 128) == 0
    for args in ((1, 12, 1, 1, 1), (48, 8, 4, 1, 8191), (1, 1, 8, 16, 1 << 20), (4096, 8, 1, 1, 100)):
        n = few_queries(*args)
        assert 1 <= n <= 64 and (n == 1 or n <= -(-args[4] // 128))


def test_operands_start_at_16_bytes():
    """Dense tensors cut from a flat buffer at an odd offset, which contiguous() returns as they are."""
    from trustworthy_dl.ops.masked_attention import _aligned
    for off in (1, 4, 8):
        flat = torch.randn(3 * 5 * 2 * 64 + off).bfloat16()
        t = flat[off:].view(3, 5, 2, 64)
        a = _aligned(t)
        assert a.data_ptr() % 16 == 0 and torch.equal(a, t) and a.is_contiguous()
        assert (a is t) == (t.data_ptr() % 16 == 0)
    rows = torch.zeros(3, 5, 2, 72).bfloat16()[..., :64]
    assert _aligned(rows) is rows
    assert _aligned(rows.transpose(2, 3)[..., :1].expand(3, 5, 64, 2)).is_contiguous()


def test_largest_launch_and_rows():
    from trustworthy_dl.ops.masked_attention import MAX_GROUPS, few_queries, largest_launch
    for B, Tq, Tk, H, Hk, D in ((2, 8192, 8192, 16, 4, 128), (64, 32768, 32768, 64, 64, 64), (1 << 16, 1, 4096, 32, 8, 128), (1, 1, (1 << 30) - 1, 1, 1, 8)):
        G, n = H // Hk, few_queries(B, Hk, H // Hk, Tq, Tk)
        parts = [B * H * math.ceil(Tq / 128), B * Hk * math.ceil(Tk / 128)]
        if n:
            parts += [B * Hk * n * math.ceil(G * Tq / 32), math.ceil(B * H * Tq / (256 // ((64 if D <= 64 else 128) // 4)))]
        assert largest_launch(B, Tq, Tk, H, Hk, D) == max(parts)
        # (the cheap test in front never hides a launch that is too large)
        assert max(parts) <= B * H * (Tq + Tk)
    assert largest_launch(1 << 22, 512, 512, 1, 1, 64) > MAX_GROUPS or largest_launch(1 << 22, 512, 512, 8, 8, 64) > MAX_GROUPS
    _bad(lambda: ops.attention_mask(1 << 22, 0, 0), "rows")


def test_library_refuses_arguments_out_of_range():
    """The C entry points themselves, before any launch (they need no GPU for that)."""
    import ctypes

    from trustworthy_dl.ops import _lib
    from trustworthy_dl.ops.masked_attention import _Args
    if not _lib.available():
        pytest.skip("the native library is not built")
    good = dict(B=1, Tq=1, Tk=1, H=4, Hk=2, D=64, dtype=1, nsplit=1, scale=1.0, dk=8)
    for kw in (dict(B=0), dict(Tq=0), dict(Tk=0), dict(H=3), dict(D=136), dict(D=12), dict(dtype=0), dict(scale=0.0), dict(cap=-1.0),
               dict(B=1 << 23, nsplit=1), dict(B=1 << 22, nsplit=0), dict(B=1 << 26, nsplit=0)):
        a = _Args(**{**good, **kw})
        fwd = _lib.lib().tdl_masked_attn_fwd(ctypes.addressof(a), None)
        assert fwd == 1, kw      # hipErrorInvalidValue
        if "nsplit" not in kw or kw["B"] > 1 << 23:
            assert _lib.lib().tdl_masked_attn_bwd(ctypes.addressof(a), None) == 1, kw
    assert _lib.lib().tdl_attn_mask(None, 0, None, None, None, None, 1 << 22, 1, 1, 1, None, None, None, None, None, None, None) == 1


def test_scales_out_of_range_and_slopes_that_are_no_tensor():
    m = ops.attention_mask(2, 4)
    q, k = torch.zeros(2, 4, 4, 8), torch.zeros(2, 4, 2, 8)
    for s in (1e-50, 1e-31, 1e31, 1e39, 1e300):      # (1e-50 is 0 in 32 bits, 1e39 infinite)
        _bad(lambda: ops.masked_attention(q, k, k, m, scale=s), "scale")
    for s in (1e-30, 1e30):
        for c in (None, 1e-6, 1000.0):
            assert torch.isfinite(ops.masked_attention(q, k, k, m, scale=s, softcap=c)).all()
    _bad(lambda: ops.masked_attention(q, k, k, m, slopes=[0.1] * 4), "slopes must be")


@pytest.mark.parametrize("cap", [None, 2.0])
def test_padding_has_no_effect_on_gradients(cap):
    """NaN and infinities in the queries, keys, values and upstream gradients of padded positions."""
    ids = torch.tensor([[0, 0, 1, 1, 1, -1, -1], [2, 2, 2, 2, 3, 3, -1]], dtype=torch.int32)
    m = ops.attention_mask(2, 7, documents=ids)
    ins = [_rand(2, 7, h, 8, seed=i) for i, h in enumerate((4, 2, 2, 4))]
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4])

    def run():
        q, k, v = (t.clone().requires_grad_(True) for t in ins[:3])
        out = ops.masked_attention(q, k, v, m, softcap=cap, slopes=slopes)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), ins[3]))
    clean = run()
    for bad in (math.nan, math.inf):
        for t in ins:
            t[ids < 0] = bad
        for a, b in zip(clean, run()):
            assert torch.equal(a, b)
