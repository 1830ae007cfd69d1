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
