"""A prompt's attention, the weights of its last rows, the packed cache that they decide, and a decode step on it."""
import pytest
import torch

from attention_reference import close, prompt
from test_gpu_parity import _compare, _cuda

pytestmark = pytest.mark.gpu


def test_prompt_weights_decide_the_packed_cache():
    import r2omni_amd as ro

    dev, hq, hkv, n, window = _cuda(), 28, 4, 1536, 64
    gen = torch.Generator(device=dev).manual_seed(71)
    q, k, v = (torch.randn(1, h, n, 128, generator=gen, device=dev).to(torch.bfloat16) for h in (hq, hkv, hkv))
    # the last rows look for what stands in a few pages
    strong = torch.tensor([3, 17, 18, 40], device=dev)
    q[:, :, -window:] += 0.5 * k.repeat_interleave(hq // hkv, 1)[:, :, strong * 32].mean(2, keepdim=True)
    out, lse = ro.prompt_attention(q, k, v)
    want = prompt(q, k, v)
    close(out, want[0], want[3])
    close(lse, want[1], want[4])
    w = ro.attention_weights(q[:, :, -window:], k, lse[:, :, -window:])

    modality = torch.where(torch.arange(n) < 32, ro.policy.TEXT, ro.policy.VIDEO)
    recent = torch.arange(n) >= n - 64
    table = ro.build_page_table(modality, page_size=32, recent_mask=recent)
    assignment = ro.project_attention_weights_to_pages(table, w[0], fp_tokens=160, int4_tokens=640, int2_tokens=480)
    classes = assignment.page_classes
    assert (classes == ro.PageClass.FP_PAGE).sum() == 5 and (classes == ro.PageClass.INT4_PAGE).sum() == 20
    assert (classes == ro.PageClass.INT2_PAGE).sum() == 15 and (classes == ro.PageClass.EVICTED_PAGE).sum() == 5
    score = w[0].double().sum(0).cpu().view(-1, 32).mean(1)
    ranked = [score[classes == c] for c in (ro.PageClass.FP_PAGE, ro.PageClass.INT4_PAGE, ro.PageClass.INT2_PAGE,
                                            ro.PageClass.EVICTED_PAGE)]
    assert all(a.min() >= b.max() for a, b in zip(ranked, ranked[1:]))
    # a token's rows take part in decoding from the pool that its page went to
    plan = ro.plan_from_pages(table.offsets, table.lengths, classes, recent_fp_capacity=128, device=dev)
    cache = ro.build_three_precision_cache(k[0], v[0], plan)
    assert [p.token_count for p in cache.pools][:3] == [5 * 32 + 32 + 64, 20 * 32, 15 * 32]
    ex = ro.prepare_splitk_executor(cache, ro.allocate_splitk_workspace(cache, num_query_heads=hq))
    step = q[:, :, -1].contiguous()
    _compare(ex(step), ro.triton_mixed_reference(step, cache).float().cpu().numpy(), "decode on the cache")
