"""Positions of a request's rows that follow a shared prefix."""
import pytest
import torch

from attention_reference import close
from prefix_reference import check, want
from test_gpu_paged import BF16, FP16, _cache, _cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_behind_a_prefix_stand_where_one_cache_has_them(dtype):
    """A request's rows get positions that go on behind its prefix, and without any their own slots': the same keys and queries, and
    the same attention, as in one cache of all tokens, whose default they are."""
    import r2omni_amd as ro

    dev, n, s = _cuda(), 70, 33
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(1, n + s, 8 + 2 * 2, 128, generator=gen, device=dev).to(dtype).transpose(1, 2)
    rotary = ro.PositionRotary(1e4 ** (-torch.arange(0, 128, 2, device=dev) / 128))
    whole, prefix, own = (_cache(dev, (m,), 2, 16, dtype, m) for m in (n + s, n, s))
    part = lambda a, b: (x[:, :8, a:b], x[:, 8:10, a:b], x[:, 10:, a:b])  # noqa: E731
    q_all = ro.paged_rope_extend(whole, *part(0, n + s), rotary)
    ro.paged_rope_extend(prefix, *part(0, n), rotary)
    q = ro.paged_rope_extend(own, *part(n, n + s), rotary, positions=n + torch.arange(s, device=dev)[None])
    assert torch.equal(q, q_all[:, :, n:])

    def keys(cache, count):
        return torch.cat([cache.key_pages[i] for i in cache.page_table[0].tolist() if i >= 0], 1)[:, :count]

    assert torch.equal(torch.cat((keys(prefix, n), keys(own, s)), 1), keys(whole, n + s))
    out, lse = check(q, own, prefix)
    far, far_lse = check(q, whole)
    _, _, bound, bound_lse = want(q, whole)  # of one rounding and error each
    close(out, far.double(), 2 * bound)
    close(lse, far_lse.double(), 2 * bound_lse)
    from_zero = ro.paged_rope_extend(own, *part(n, n + s), rotary)  # without positions: as if nothing preceded them
    alone = ro.qk_position_rope(*part(n, n + s)[:2], torch.arange(s, device=dev)[None], rotary)
    assert torch.equal(from_zero, alone[0]) and torch.equal(keys(own, s), alone[1][0])
