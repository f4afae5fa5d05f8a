"""Attention over shared prefixes and own slots in 64 bits, with the bounds of attention_reference.py."""
import math

import torch

from attention_reference import attend, close


def slots(cache, row, pool):
    """[Hkv, n, 128] of one table row's filled slots, and which have a page."""
    n, page = max(0, min(int(cache.lengths[row]), cache.capacity)), cache.key_pages.shape[2]
    j = torch.arange(n, device=pool.device)
    ids = cache.page_table[row].long()[j // page]
    ok = (ids >= 0) & (ids < pool.shape[0])
    return pool[ids.clamp(0, pool.shape[0] - 1), :, j % page].transpose(0, 1), ok


def shared_by(members, batch):
    """The prefix of each request, -1 for none."""
    of = []
    for g, m in enumerate(members):
        of += [g] * max(0, min(m, batch - len(of)))
    return of + [-1] * (batch - len(of))


def want(q, cache, prefix=None, members=None, query_lengths=None, scale=None):
    """(out, lse, bound on out, bound on lse) of query [B, Hq, S, 128], in 64 bits."""
    b, hq, rows, _ = q.shape
    hkv, dev = cache.key_pages.shape[1], q.device
    group = hq // hkv
    of = [-1] * b if prefix is None else shared_by([b] if members is None else members.tolist(), b)
    out, bound_out = (torch.zeros(b, hq, rows, 128, dtype=torch.float64, device=dev) for _ in range(2))
    lse, bound_lse = torch.full((b, hq, rows), -math.inf, dtype=torch.float64, device=dev), torch.zeros(b, hq, rows, dtype=torch.float64, device=dev)
    for i in range(b):
        k, ok = slots(cache, i, cache.key_pages)
        v, _ = slots(cache, i, cache.value_pages)
        n, before = k.shape[1], 0
        if of[i] >= 0:
            pk, p_ok = slots(prefix, of[i], prefix.key_pages)
            pv, _ = slots(prefix, of[i], prefix.value_pages)
            before = pk.shape[1]
            k, v, ok = torch.cat((pk, k), 1), torch.cat((pv, v), 1), torch.cat((p_ok, ok))
        count = rows if query_lengths is None else max(0, min(int(query_lengths[i]), rows))
        r, j = torch.arange(rows, device=dev)[:, None], torch.arange(before + n, device=dev)
        seen = ok & (r < count) & ((j < before) | (j - before <= n - count + r))
        live = seen.any(-1)
        if not live.any():
            continue
        for h in range(hq):
            kv = h // group
            o, l, _, tb, tl, _ = attend(q[i, h], k[kv], v[kv], seen, q.dtype, scale)
            out[i, h], bound_out[i, h] = torch.where(live[:, None], o, 0.0), torch.where(live[:, None], tb, 0.0)
            lse[i, h], bound_lse[i, h] = torch.where(live, l, -math.inf), torch.where(live, tl, 0.0)
    return out, lse, bound_out, bound_lse


def check(q, cache, prefix=None, members=None, query_lengths=None, scale=None):
    """The call against the definition; its results."""
    import r2omni_amd as ro

    out, lse = ro.paged_prefix_attention(q, cache, prefix, members=members, query_lengths=query_lengths, sm_scale=scale)
    torch.cuda.synchronize()
    q4 = q[:, :, None] if q.ndim == 3 else q
    o, l, bo, bl = want(q4, cache, prefix, members, query_lengths, scale)
    assert out.shape == q.shape and lse.shape == q.shape[:-1] and out.dtype == q.dtype and lse.dtype == torch.float32
    close(out.reshape(q4.shape), o, bo)
    close(lse.reshape(q4.shape[:-1]), l, bl)
    return out, lse
