"""Attention of a prompt and over a paged cache in 64 bits, and how far a kernel's results may be from it.

The bounds count roundings.  With h = finfo(dtype).eps / 2 of the 16-bit rows:
  logits: products of 16-bit values are exact in fp32; 128 of them and their scaling in fp32 are off by at most
  130 * 2^-24 of c sum |q_d k_d|, called e.  exp2 and its argument (one fma, a 1-ulp exponential) add |x| 2^-23.
  probabilities: relative error 2 e + |x| 2^-22, then one rounding to the rows' type (h), for fp16 at least 2^-25
  absolute (half a subnormal step) beside a largest term of one or more;
  out: that error times sum p |v|, and the result's own rounding, h |out|; sums of n terms in fp32 add n 2^-24.
"""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # finfo.eps / 2


def visible(sq, sk, nq, nk, window, sinks, device):
    """[Sq, Sk]: which keys each row of one request sees."""
    i, j = torch.arange(sq, device=device)[:, None], torch.arange(sk, device=device)[None]
    p = nk - nq + i
    ok = (j <= p) & (j < nk) & (i < nq)
    return ok if window is None else ok & ((p - j < window) | (j < sinks))


def attend(q, k, v, seen, dtype, scale=None):
    """One head in 64 bits: q [R, 128], k and v [S, 128], seen [R, S].  Returns (out, lse, p, bound on out, bound on
    lse, relative bound on p)."""
    scale = 128 ** -0.5 if scale is None else scale
    q, k = q.double(), k.double()
    v = torch.where(seen.any(0)[:, None], v.double(), 0.0)  # what no row sees is not used, whatever it holds
    k = torch.where(seen.any(0)[:, None], k, 0.0)
    x = torch.where(seen, (q @ k.t()) * scale, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    out = p @ v
    lse = (torch.where(top == -math.inf, 0.0, top) + torch.log(total))[:, 0]
    h = HALF[dtype]
    err = 130 * 2.0 ** -24 * scale * torch.where(seen, q.abs() @ k.abs().t(), 0.0).amax(-1)
    depth = torch.where(seen, x.abs(), 0.0).amax(-1)
    n = x.shape[1]
    rel = 2 * err + depth * 2.0 ** -22 + n * 2.0 ** -24 + 2.0 ** -21
    size = p @ v.abs()
    bound = (rel + h)[:, None] * size + h * out.abs() + 2.0 ** -126
    if dtype == torch.float16:
        bound = bound + n * 2.0 ** -25 * v.abs().amax() / 1.0 + 2.0 ** -25
    lse_bound = err + depth * 2.0 ** -22 + n * 2.0 ** -24 + 2.0 ** -20
    return out, lse, p, bound, lse_bound, rel


def prompt(q, k, v, window=None, sinks=0, nq=None, nk=None, scale=None):
    """Every head of a padded batch: (out, lse, weights, bound on out, bound on lse, bound on weights)."""
    b, hq, sq, _ = q.shape
    hkv, sk = k.shape[1:3]
    out = torch.zeros(b, hq, sq, 128, dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.zeros(b, hkv, sk, dtype=torch.float64, device=q.device)
    bo, bl, bw = torch.zeros_like(out), torch.zeros(b, hq, sq, dtype=torch.float64, device=q.device), torch.zeros_like(w)
    for i in range(b):
        a, n = (sq if nq is None else nq[i]), (sk if nk is None else nk[i])
        seen = visible(sq, sk, a, n, window, sinks, q.device)
        for h in range(hq):
            kv = h // (hq // hkv)
            o, l, p, tb, tl, rel = attend(q[i, h], k[i, kv], v[i, kv], seen, q.dtype, scale)
            live = seen.any(-1)
            out[i, h], bo[i, h] = torch.where(live[:, None], o, 0.0), torch.where(live[:, None], tb, 0.0)
            lse[i, h], bl[i, h] = torch.where(live, l, -math.inf), torch.where(live, tl, 0.0)
            w[i, kv] += p.sum(0)
            # the kernel's own lse enters exp(x - lse): its bound counts as another relative error
            bw[i, kv] += (p * (rel + tl + l.abs().nan_to_num(posinf=0.0, neginf=0.0) * 2.0 ** -22)[:, None]).sum(0)
    return out, lse, w, bo, bl, bw + w * (hq // hkv * sq) * 2.0 ** -24 + 2.0 ** -126


def close(got, want, bound):
    """Within the bound where the reference is finite, equal (infinities) elsewhere."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine])
    assert torch.isfinite(got[fine]).all()
    over = (got - want).abs()[fine] - bound[fine]
    assert not (over > 0).any(), f"{int((over > 0).sum())} of {over.numel()} values over the bound by up to {over.max().item():.3e}"
