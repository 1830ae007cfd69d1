"""Cases that measure the masked attention and distillation operators.

``listed()`` names the fixed cases and ``draw(rng)`` makes more of the same ranges; ``prepare`` makes a
case's inputs on the GPU, ``run`` makes one pass (plain torch operations, or the framework's own calls
where ``own`` is set), ``exact`` computes the same outputs from the definitions in 64 bits and
``work`` counts the bytes and operations that a pass cannot do without.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ cases
def _attn(name, B, Tq, Tk, H, Hk, D, dtype, mask, cap=0.0, alibi=False, train=True, doc=0):
    return {"op": "attention", "name": name, "B": B, "Tq": Tq, "Tk": Tk, "H": H, "Hk": Hk, "D": D, "dtype": dtype,
            "mask": mask, "cap": cap, "alibi": alibi, "train": train, "doc": doc}


def _distill(name, M, V, ld, K, dtype, tau, alpha):
    return {"op": "distill", "name": name, "M": M, "V": V, "ld": ld, "K": K, "dtype": dtype, "tau": tau,
            "alpha": alpha}


def listed():
    return [
        # one layer's training pass of GPT-2-medium on rows packed with several documents each
        _attn("train_packed_medium", 16, 1024, 1024, 16, 16, 64, "bf16", "documents", doc=301),
        # long-context training with shared KV heads and capped scores; the largest case
        _attn("train_long_capped_gqa", 2, 8192, 8192, 16, 4, 128, "bf16", "causal", cap=50.0),
        # prefix-LM fine-tuning (prompt attends both ways) with distance bias at an odd length
        _attn("train_prefix_alibi_odd", 4, 777, 777, 12, 12, 64, "fp16", "prefix", alibi=True),
        # held-out evaluation with GPT-2-xl's 25 heads, capped scores, no gradient
        _attn("eval_xl_capped", 8, 2048, 2048, 25, 25, 64, "bf16", "causal", cap=30.0, train=False),
        # generation for a batch of ragged sequences, one token each, from a shared-head cache
        _attn("decode_batch_ragged", 48, 1, 8191, 32, 8, 128, "bf16", "lengths", alibi=True, train=False),
        # generation for one sequence: latency only
        _attn("decode_single", 1, 1, 1000, 12, 12, 64, "bf16", "lengths", train=False),
        # several new tokens a sequence (checking drafted tokens) against a cache
        _attn("decode_chunk", 4, 7, 5003, 16, 2, 128, "fp16", "lengths", cap=30.0, train=False),
        # loss and gradient over a GPT-2 micro-batch's padded logits, hard and soft targets mixed
        _distill("distill_gpt2_step", 16384, 50257, 50304, 64, "bf16", 2.0, 0.7),
        # a short batch against a few teacher entries: latency
        _distill("distill_small", 24, 50257, 50304, 8, "bf16", 1.0, 1.0),
        # rows of odd length without padding, full precision
        _distill("distill_fp32_odd", 1023, 32003, 32003, 100, "fp32", 1.5, 0.5),
        # a classifier's head: many short rows, soft and hard targets in equal parts
        _distill("distill_short_rows", 8192, 1000, 1000, 16, "fp16", 4.0, 0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "train", "eval", "decode", "decode", "distill", "distill", "distill"])
    if kind in ("train", "eval"):
        Hk = rng.choice([1, 2, 4, 8, 12])
        H = Hk * rng.choice([1, 1, 2, 4])
        mask = rng.choice(["causal", "documents", "prefix", "full"])
        scores = 2 * 16 * 8192 * 8192 // (2 if mask == "full" else 1)   # of the largest listed case
        T = min(_log_int(rng, 1, 8192), int(math.sqrt(0.9 * scores / H)))
        B = max(1, min(_log_int(rng, 1, 32), int(0.9 * scores / (H * T * T))))
        return _attn("", B, T, T, H, Hk, rng.choice([64, 64, 128]), rng.choice(["bf16", "bf16", "fp16"]), mask,
                     cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.choice([False, False, True]),
                     train=kind == "train", doc=max(1, _log_int(rng, max(1, T // 40), T)))
    if kind == "decode":
        Tk = _log_int(rng, 1, 16384)
        Hk = rng.choice([1, 2, 4, 8, 12])
        return _attn("", _log_int(rng, 1, 32), min(Tk, rng.choice([1, 1, 1, 2, 5, 16])), Tk, Hk * rng.choice([1, 3, 4, 8]),
                     Hk, rng.choice([64, 128]), rng.choice(["bf16", "fp16"]), "lengths",
                     cap=rng.choice([0.0, 0.0, 30.0]), alibi=rng.choice([False, True]), train=False)
    V = _log_int(rng, 100, 60000)
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    M = _log_int(rng, 1, min(16384, int(16384 * 50257 / V) // (2 if dt == "fp32" else 1)))
    return _distill("", M, V, rng.choice([V, (V + 63) // 64 * 64]), min(V, _log_int(rng, 1, 256)), dt,
                    rng.choice([1.0, 1.5, 2.0, 4.0]), rng.choice([1.0, 0.9, 0.5, 0.0]))


# ----------------------------------------------------------------------------------------- layouts
def _documents(case):
    """Document lengths of each row (the same in every row, in an order that the seed chooses); the
    last one of a row of 64 or more is padding."""
    T, mean = case["Tk"], case["doc"]
    rng, left, out = random.Random(7 * T + mean), T, []
    pad = T // 50
    left -= pad
    while left > 0:
        n = max(1, min(left, int(mean * rng.uniform(0.2, 1.8))))
        out.append(n)
        left -= n
    return out, pad


def _prefix(case):
    """Prefix length of each row."""
    rng = random.Random(case["Tk"] + case["B"])
    return [rng.randint(0, case["Tk"] // 2) for _ in range(case["B"])]


def _lengths(case):
    """Valid keys of each row of the cache."""
    rng = random.Random(case["Tk"] + 3 * case["B"])
    return [max(case["Tq"], case["Tk"] - rng.randint(0, case["Tk"] * 3 // 4)) if i else case["Tk"]
            for i in range(case["B"])]


def _pairs(case):
    """(visible query-key pairs of one head, keys that some query sees, over all rows)"""
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    if case["mask"] == "full":
        return B * Tq * Tk, B * Tk
    if case["mask"] == "documents":
        docs, pad = _documents(case)
        return B * sum(n * (n + 1) // 2 for n in docs), B * (Tk - pad)
    if case["mask"] == "prefix":
        return sum(Tk * (Tk + 1) // 2 + p * (p - 1) // 2 for p in _prefix(case)), B * Tk
    if case["mask"] == "lengths":
        lens = _lengths(case)
        return sum(Tq * n - Tq * (Tq - 1) // 2 for n in lens), sum(lens)
    return B * Tk * (Tk + 1) // 2, B * Tk


def work(case):
    if case["op"] == "attention":
        e = BYTES[case["dtype"]]
        pairs, keys = _pairs(case)
        pairs *= case["H"]
        q = case["B"] * case["Tq"] * case["H"] * case["D"] * e
        kv = 2 * keys * case["Hk"] * case["D"] * e
        if case["train"]:   # q, k, v, d_out in; out, dq, dk, dv out
            return {"bytes": 4 * q + 2 * kv, "flops": 14 * case["D"] * pairs}
        return {"bytes": 2 * q + kv, "flops": 4 * case["D"] * pairs}
    e = BYTES[case["dtype"]]
    M, V, ld, K = (case[n] for n in ("M", "V", "ld", "K"))
    # logits, teacher entries and labels in, the logits' gradient out; 8 operations an element
    return {"bytes": M * V * e + M * ld * e + M * K * 12 + M * 8, "flops": 8 * M * V}


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_attention(case, seed):
    g, dt, dev = _gen(seed), DTYPES[case["dtype"]], "cuda"
    B, Tq, Tk, H, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    # capped heads are those whose scores grow large: queries four times the usual size
    st = {"case": case, "scale": 1.0 / math.sqrt(D),
          "q": (normal(B, Tq, H, D) * (4.0 if case["cap"] else 1.0)).to(dt),
          "k": normal(B, Tk, Hk, D).to(dt), "v": normal(B, Tk, Hk, D).to(dt),
          "documents": None, "prefix": None, "lengths": None, "slopes": None}
    if case["train"]:
        st["do"] = normal(B, Tq, H, D).to(dt)
        for n in ("q", "k", "v"):
            st[n].requires_grad_(True)
    if case["alibi"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=dev)
    rng = random.Random(seed)
    if case["mask"] == "documents":
        docs, pad = _documents(case)
        rows = []
        for _ in range(B):
            order = list(docs)
            rng.shuffle(order)
            rows.append([i for i, n in enumerate(order) for _ in range(n)] + [-1] * pad)
        st["documents"] = torch.tensor(rows, dtype=torch.int32, device=dev)
    elif case["mask"] == "prefix":
        order = _prefix(case)
        rng.shuffle(order)
        st["prefix"] = torch.tensor(order, dtype=torch.int32, device=dev)
    elif case["mask"] == "lengths":
        order = _lengths(case)
        rng.shuffle(order)
        st["lengths"] = torch.tensor(order, dtype=torch.int32, device=dev)
        for b, n in enumerate(order):   # rows of the cache that hold no token yet
            st["k"][b, n:] = 0
            st["v"][b, n:] = 0
    if own:
        from trustworthy_dl import ops
        st["mask"] = ops.attention_mask(B, Tq, Tk, causal=case["mask"] != "full", documents=st["documents"],
                                        prefix=st["prefix"], lengths=st["lengths"], device=dev)
    return st


def _prepare_logits(case, seed):
    g, dt, dev = _gen(seed), DTYPES[case["dtype"]], "cuda"
    M, V, ld, K = case["M"], case["V"], case["ld"], case["K"]
    z = torch.empty(M, ld, dtype=dt, device=dev)
    z[:, :V] = torch.randn(M, V, generator=g, device=dev) * 2.5
    z[:, V:] = 0
    st = {"case": case, "logits": z.requires_grad_(True), "scale": torch.ones((), device=dev)}
    if case["dtype"] == "fp16":   # a loss scale that keeps half-precision gradients in range
        st["scale"] *= 4.0 * 2 ** int(math.log2(M))
    # a row's teacher entries: distinct classes, largest logit first; some rows have fewer entries
    # (-1 behind them), some none, and some tokens carry no label
    step = max(1, V // K)
    first = torch.randint(0, V, (M, 1), generator=g, device=dev)
    jitter = torch.randint(0, step, (M, K), generator=g, device=dev)
    st["index"] = (first + torch.arange(K, device=dev) * step + jitter) % V
    st["teacher"] = torch.sort(torch.randn(M, K, generator=g, device=dev) * 2.0 + 5.0, dim=1, descending=True)[0]
    used = torch.randint(0, 20 * K, (M, 1), generator=g, device=dev)
    st["index"].masked_fill_(torch.arange(K, device=dev) >= used, -1)
    labels = torch.randint(0, V, (M,), generator=g, device=dev)
    labels[torch.rand(M, generator=g, device=dev) < 0.03] = -100
    st["labels"] = labels
    return st


def prepare(case, seed):
    return _prepare_attention(case, seed) if case["op"] == "attention" else _prepare_logits(case, seed)


# -------------------------------------------------------------------------------- the plain forms
def _visible(st, B, Tq, Tk, dev):
    """[B, Tq, Tk]: which keys each query sees."""
    case = st["case"]
    j = torch.arange(Tk, device=dev).view(1, 1, Tk)
    p = torch.arange(Tq, device=dev).view(1, Tq, 1) + (Tk - Tq)
    if st["lengths"] is not None:
        p = torch.arange(Tq, device=dev).view(1, Tq, 1) + (st["lengths"].view(B, 1, 1) - Tq)
        return (j <= p) & (j < st["lengths"].view(B, 1, 1))
    if case["mask"] == "full":
        return (j >= 0).expand(B, Tq, Tk)
    if st["documents"] is not None:
        d = st["documents"]
        return (j <= p) & (d[:, :, None] == d[:, None, :]) & (d >= 0)[:, None, :]
    if st["prefix"] is not None:
        return (j <= p) | ((j < st["prefix"].view(B, 1, 1)) & (p >= 0))
    return (j <= p).expand(B, Tq, Tk)


def _distance(st, B, Tq, Tk, dev):
    """[B, Tq, Tk]: |query position - key position|"""
    j = torch.arange(Tk, device=dev).view(1, 1, Tk)
    last = st["lengths"].view(B, 1, 1) if st["lengths"] is not None else Tk
    return (torch.arange(Tq, device=dev).view(1, Tq, 1) + (last - Tq) - j).abs()


def _plain_attention(st):
    case = st["case"]
    dt, cap, scale = DTYPES[case["dtype"]], case["cap"], st["scale"]
    q, k, v = (st[n].detach().float().transpose(1, 2) for n in ("q", "k", "v"))   # [B, heads, T, D]
    B, H, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    G = H // Hk
    q = q.reshape(B, Hk, G * Tq, D)      # the queries of a shared head side by side
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, H, Tq, Tk) * scale
    t = None
    if cap:
        t = torch.tanh(s / cap)
        s = cap * t
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, H, 1, 1) * _distance(st, B, Tq, Tk, q.device).float()[:, None]
    vis = _visible(st, B, Tq, Tk, q.device)[:, None]
    s = s.masked_fill(~vis, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del s
    z = p.sum(-1, keepdim=True)
    p = p / torch.where(z == 0, torch.ones_like(z), z)
    o = torch.matmul(p.view(B, Hk, G * Tq, Tk), v).view(B, H, Tq, D)
    out = o.transpose(1, 2).to(dt).contiguous()
    if not case["train"]:
        return out
    do = st["do"].float().transpose(1, 2).reshape(B, Hk, G * Tq, D)
    pg = p.view(B, Hk, G * Tq, Tk)
    dv = torch.matmul(pg.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = pg * (ds - (do * o.reshape(B, Hk, G * Tq, D)).sum(-1, keepdim=True))
    del p, pg
    if cap:
        ds = ds * (1.0 - t * t).view(B, Hk, G * Tq, Tk)
    dq = (torch.matmul(ds, k) * scale).view(B, H, Tq, D)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    return (out, dq.transpose(1, 2).to(dt).contiguous(), dk.transpose(1, 2).to(dt).contiguous(),
            dv.transpose(1, 2).to(dt).contiguous())


def _plain_loss(z, st, V):
    """(loss, gradient of the logits [M, ld]) from 32-bit logits [M, ld]"""
    case = st["case"]
    tau, alpha = case["tau"], case["alpha"]
    idx, lab = st["index"], st["labels"]
    zv = z[:, :V]
    top = zv.amax(1, keepdim=True)
    shifted = zv - top
    use = idx >= 0
    has = use.any(1)
    safe = idx.clamp(min=0)
    t = (st["teacher"].float() / tau).masked_fill(~use, float("-inf"))
    t = t - torch.where(has[:, None], t.amax(1, keepdim=True), torch.zeros_like(t[:, :1]))
    q = torch.where(use, torch.exp(t), torch.zeros_like(t))
    qs = q.sum(1, keepdim=True)
    qs = torch.where(qs == 0, torch.ones_like(qs), qs)
    q = q / qs
    logq = t - torch.log(qs)
    e_tau = torch.exp(shifted / tau)
    s_tau = e_tau.sum(1, keepdim=True)
    logp = shifted.gather(1, safe) / tau - torch.log(s_tau)
    kd = torch.where(q > 0, q * (logq - logp), torch.zeros_like(q)).sum(1) * (tau * tau)
    n_t = has.sum().clamp(min=1).float()
    loss = alpha * kd.sum() / n_t
    d = torch.zeros_like(z)
    dv = e_tau / s_tau * (has[:, None] * (alpha * tau / n_t))
    dv.scatter_add_(1, safe, -q * (alpha * tau / n_t))
    if alpha < 1.0:
        ok = lab >= 0
        n_l = ok.sum().clamp(min=1).float()
        e = torch.exp(shifted)
        s = e.sum(1, keepdim=True)
        pick = shifted.gather(1, lab.clamp(min=0)[:, None])
        loss = loss + (1.0 - alpha) * ((torch.log(s) - pick)[:, 0] * ok).sum() / n_l
        w = ok[:, None] * ((1.0 - alpha) / n_l)
        dv += e / s * w
        dv.scatter_add_(1, lab.clamp(min=0)[:, None], -w)
    d[:, :V] = dv
    return loss, d


def run(state):
    case = state["case"]
    if case["op"] == "attention":
        if not own:
            return _plain_attention(state)
        from trustworthy_dl import ops
        kw = {"softcap": case["cap"] or None, "slopes": state["slopes"]}
        q, k, v = state["q"], state["k"], state["v"]
        out = ops.masked_attention(q, k, v, state["mask"], **kw)
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["do"]))
    kw = {"temperature": case["tau"], "alpha": case["alpha"]}
    if own:
        from trustworthy_dl import ops
        loss = ops.distillation_loss(state["logits"], state["index"], state["teacher"], state["labels"], case["V"], **kw)
        return loss.detach(), torch.autograd.grad(loss, state["logits"], state["scale"])[0]
    loss, d = _plain_loss(state["logits"].detach().float(), state, case["V"])
    return loss, d.mul_(state["scale"]).to(DTYPES[case["dtype"]])


# ------------------------------------------------------------------------ the definitions, 64 bits
def _exact_attention(case, st):
    B, Tq, Tk, H, Hk, D = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
    G, dev, scale = H // Hk, st["q"].device, 1.0 / math.sqrt(D)
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64, device=dev)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Tk, Hk, D, dtype=torch.float64, device=dev) for _ in "kv")
    keys = torch.arange(Tk, device=dev)
    for b in range(B):
        n = Tk if st["lengths"] is None else int(st["lengths"][b])
        pos = torch.arange(Tq, device=dev) + (n - Tq)
        ok = keys[None, :] < n
        if case["mask"] != "full":
            ahead = keys[None, :] > pos[:, None]
            if st["prefix"] is not None:
                ahead = ahead & (keys[None, :] >= int(st["prefix"][b]))
            ok = ok & ~ahead
        if st["documents"] is not None:
            d = st["documents"][b]
            ok = ok & (d[:, None] == d[None, :]) & (d[:, None] >= 0)
        ok = ok.expand(Tq, Tk)
        for h in range(H):
            qh, kh, vh = (x.detach().double() for x in (st["q"][b, :, h], st["k"][b, :, h // G], st["v"][b, :, h // G]))
            x = qh @ kh.T * scale
            y = case["cap"] * torch.tanh(x / case["cap"]) if case["cap"] else x
            if st["slopes"] is not None:
                y = y - float(st["slopes"][h]) * (pos[:, None] - keys[None, :]).abs()
            y = torch.where(ok, y, -math.inf)
            w = torch.nan_to_num(torch.softmax(y, -1), nan=0.0)   # rows that see nothing: zero
            o = w @ vh
            out[b, :, h] = o
            if not case["train"]:
                continue
            g = st["do"][b, :, h].double()
            dv[b, :, h // G] += w.T @ g
            dy = w * (g @ vh.T - (g * o).sum(-1, keepdim=True))
            dx = dy / torch.cosh(x / case["cap"]) ** 2 if case["cap"] else dy
            dq[b, :, h] = dx @ kh * scale
            dk[b, :, h // G] += dx.T @ qh * scale
    return (out, dq, dk, dv) if case["train"] else out


def _exact_rows(case, st, z, r0, n_t, n_l):
    """(loss share, gradient) of the rows whose 64-bit logits over the V classes are ``z``"""
    V, tau, alpha = case["V"], case["tau"], case["alpha"]
    m = z.shape[0]
    rows = slice(r0, r0 + m)
    idx, lab = st["index"][rows], st["labels"][rows]
    entry = idx >= 0
    t = torch.where(entry, st["teacher"][rows].double() / tau, -math.inf)
    q = torch.nan_to_num(torch.softmax(t, 1), nan=0.0)
    some = entry.any(1, keepdim=True).double()
    target = torch.zeros(m, V + 1, dtype=torch.float64, device=z.device)
    target.scatter_add_(1, torch.where(entry, idx, V), q)
    lp = torch.log_softmax(z / tau, 1)
    entropy = torch.where(q > 0, q * torch.log(q), 0.0).sum()
    kd = tau * tau * (entropy - (target[:, :V] * lp).sum())
    d = alpha * tau / n_t * (some * lp.exp() - target[:, :V])
    loss = alpha * kd / n_t
    if alpha < 1:
        keep = (lab >= 0).double()[:, None]
        lp = torch.log_softmax(z, 1)
        hot = torch.zeros(m, V + 1, dtype=torch.float64, device=z.device)
        hot.scatter_(1, torch.where(lab >= 0, lab, V)[:, None], 1.0)
        loss = loss - (1 - alpha) / n_l * (hot[:, :V] * lp).sum()
        d = d + (1 - alpha) / n_l * keep * (lp.exp() - hot[:, :V])
    return loss, d


def _exact_loss(case, st):
    M, V, ld = case["M"], case["V"], case["ld"]
    n_t = max(1, int((st["index"] >= 0).any(1).sum()))
    n_l = max(1, int((st["labels"] >= 0).sum()))
    loss = torch.zeros((), dtype=torch.float64, device=st["index"].device)
    grad = torch.zeros(M, ld, dtype=torch.float64, device=st["index"].device)
    for r0 in range(0, M, 1024):
        z = st["logits"].detach()[r0:r0 + 1024, :V].double()
        part, grad[r0:r0 + 1024, :V] = _exact_rows(case, st, z, r0, n_t, n_l)
        loss += part
    return loss, grad * st["scale"].double()


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        if case["B"] * case["H"] > 4096:   # a product at a time: too many of them
            return None
        return _exact_attention(case, st)
    return _exact_loss(case, st)
