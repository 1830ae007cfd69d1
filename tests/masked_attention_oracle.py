"""64-bit definition of masked attention with the error bound of a 16-bit kernel, for the tests.

Bounds.  u = finfo(dtype).eps / 2 is one rounding to the 16-bit type, d = 2^-13 covers everything that
is done in 32 bits (scores of magnitude < 2^7 in units of log 2: their products, sums over D <= 128 terms,
the exponential, the sums over keys: each a few 2^-24 of the magnitudes, times that magnitude).
  out   P is rounded once (u) before its product, the result once:  (2 u + 2 d) sum_j P |v|
  dV    likewise                                                   (2 u + 2 d) sum_i P |dO|
  delta from out (the bound allows it the error of the rounded one):  e_i = sum_c |dO| (2 u + 2 d) sum_j P |v|
  dS    rounded once: |error| <= (u + d) |dS| + P (e_i + d (sum_c |dO| |v| + |delta|)), so
  dQ    scale sum_j error |k| + (u + d) |dQ|;   dK   scale sum_i error |q| + (u + d) |dK|
fp16 also has a smallest step, 2^-24: a P below 2^-14 is off by up to 2^-25 however small it is (forward: of
a row whose largest is 1 and whose sum is at least 1), which adds 2^-25 sum |v| to out over the visible keys
and 2^-25 sum |dO| to dV.  dS is rounded times 2^n with 2^n max|dO| in [2^6, 2^7), with a cap as a quarter (the derivative r (1 - r) without its 4):
an absolute error of 2^-25 max|dO| / 64 (x 4 with a cap) per visible pair.
With a cap, dS carries the factor 1 - tanh^2 = 4 r (1 - r), exact to a few 2^-24: within d.
"""
import math

import torch


def dense(B, Tq, Tk, causal=True, documents=None, prefix=None, lengths=None, q_start=None):
    """[B, Tq, Tk] booleans and [B] first positions, element by element from the documented meaning."""
    seen = torch.zeros(B, Tq, Tk, dtype=torch.bool)
    first = torch.zeros(B, dtype=torch.long)
    for b in range(B):
        n = Tk if lengths is None else max(0, min(Tk, int(lengths[b])))
        p0 = int(q_start[b]) if q_start is not None else (n - Tq if Tq < Tk else 0)
        first[b] = p0
        start = list(range(Tk))
        for j in range(Tk):
            start[j] = 0 if documents is None else (start[j - 1] if j and int(documents[b, j]) == int(documents[b, j - 1]) else j)
        for i in range(Tq):
            p = p0 + i
            if not 0 <= p < n or (documents is not None and int(documents[b, p]) < 0):
                continue
            lead = 0    # end of the prefix of p's document
            if prefix is not None and prefix.dim() == 1:
                lead = int(prefix[b])
            elif prefix is not None:
                lead = start[p]
                while lead < Tk and bool(prefix[b, lead]):
                    lead += 1
            for j in range(n):
                same = start[j] == start[p]
                seen[b, i, j] = same and (not causal or j <= p or j < lead)
    return seen, first


def run(q, k, v, seen, first, scale, cap=0.0, slopes=None, dout=None):
    """{name: (value, bound)} in 64 bits for out, lse (value only) and, with dout, dq, dk, dv."""
    u = torch.finfo(q.dtype).eps / 2
    d = 2.0 ** -13
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    Q, K, V = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    K, V = (t.repeat_interleave(G, 1) for t in (K, V))
    seen = seen.to(q.device)[:, None]
    x = Q @ K.transpose(-1, -2) * scale
    t = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    s = cap * t if cap else x
    if slopes is not None:
        p = first.to(q.device)[:, None] + torch.arange(Tq, device=q.device)
        dist = (p[:, :, None] - torch.arange(Tk, device=q.device)).abs().double()
        s = s - slopes.double().view(1, H, 1, 1) * dist[:, None]
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    P = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    out = P @ V
    A = P @ V.abs()
    step = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    tiny = step * (seen.double() @ V.abs())
    res = {"out": (out.transpose(1, 2), ((2 * u + 2 * d) * A + tiny).transpose(1, 2)), "lse": lse}
    if dout is None:
        return res
    dO = dout.detach().double().transpose(1, 2)
    delta = (dO * out).sum(-1, keepdim=True)
    dP = dO @ V.transpose(-1, -2)
    dS = P * (dP - delta)
    e = (dO.abs() * ((2 * u + 2 * d) * A + tiny)).sum(-1, keepdim=True)
    err = (u + d) * dS.abs() + P * (e + d * (dO.abs() @ V.abs().transpose(-1, -2) + delta.abs()))
    if cap:
        dS, err = dS * (1 - t * t), err * (1 - t * t) + d * dS.abs() * 2.0 ** -6
    err = err + seen * (step / 64 * (4 if cap else 1) * float(dO.abs().max()))

    def heads(t):   # sum over the query heads of a group
        return t.view(B, Hk, G, Tk, D).sum(2).transpose(1, 2)
    dq, dk, dv = dS @ K * scale, heads(dS.transpose(-1, -2) @ Q * scale), heads(P.transpose(-1, -2) @ dO)
    res["dq"] = (dq.transpose(1, 2), (err @ K.abs() * scale + (u + d) * dq.abs()).transpose(1, 2))
    res["dk"] = (dk, heads(err.transpose(-1, -2) @ Q.abs() * scale) + (u + d) * dk.abs())
    res["dv"] = (dv, heads(((2 * u + 2 * d) * P + step * seen).transpose(-1, -2) @ dO.abs()))
    return res


def check(got, want, name):
    value, bound = want
    # results below the type's normal range are rounded to its smallest step
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - value).abs() - bound - tiny
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{name}: off by {worst:.3e} beyond the bound at {torch.nonzero(off == off.max())[0].tolist()}"
