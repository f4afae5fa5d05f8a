"""Results lie as their operands do: by the host module and by the Python path, of the rotation, of both calls on the paged cache
and of a prompt's attention, so that a layer's views of one projection come out in the order that its next product takes."""
import pytest
import torch

from test_gpu_paged import BF16, FP16, _cache, _cuda
from test_gpu_position import _rotary
from test_gpu_prefix_calls import _paths

pytestmark = pytest.mark.gpu


def _kept(t):
    """Strides, but for those of axes of one element, which are not used."""
    return [st for st, n in zip(t.stride(), t.shape) if n > 1]


def _dense(t):
    """The strides of a dense tensor whose axes stand in the order of t's."""
    strides, step = [0] * t.ndim, 1
    for axis in sorted((i for i in range(t.ndim) if t.shape[i] > 1), key=lambda i: t.stride(i)):
        strides[axis] = step
        step *= t.shape[axis]
    return [st for st, n in zip(strides, t.shape) if n > 1]


def _operands(how, b, h, rows, dtype, dev):
    """Query rows [b, h, rows, 128] and key rows [b, 2, rows, 128] as a caller may hold them."""
    if how == "projection":  # [b, rows, heads, 128], all heads of one product
        x = torch.randn(b, rows, h + 4, 128, device=dev).to(dtype).transpose(1, 2)
        return x[:, :h], x[:, h : h + 2]
    if how == "own projections":
        return tuple(torch.randn(b, rows, n, 128, device=dev).to(dtype).transpose(1, 2) for n in (h, 2))
    if how == "heads first":  # [h, b, rows, 128]
        return tuple(torch.randn(n, b, rows, 128, device=dev).to(dtype).transpose(0, 1) for n in (h, 2))
    if how == "rows first":  # [rows, b, h, 128], a gap behind each row
        return tuple(torch.randn(rows, b, n, 136, device=dev).to(dtype)[..., :128].permute(1, 2, 0, 3) for n in (h, 2))
    return tuple(torch.randn(b, n, rows, 128, device=dev).to(dtype) for n in (h, 2))


@pytest.mark.parametrize("how", ["projection", "own projections", "heads first", "rows first", "in order"])
@pytest.mark.parametrize("b,rows", [(2, 5), (1, 5), (3, 1), (1, 1), (2, 33)])
def test_results_lie_as_their_operands(how, b, rows):
    import r2omni_amd as ro

    dev, h, dtype = _cuda(), 8, FP16 if rows == 33 else BF16
    q, k = _operands(how, b, h, rows, dtype, dev)
    pos, rotary = torch.arange(rows, device=dev).expand(b, rows), _rotary(dev)
    shared, own = _cache(dev, (50,), 2, 16, dtype, 1), _cache(dev, (40,) * b, 2, 16, dtype, 2)
    prompt, lse = ro.prompt_attention(q, k, k)
    assert _kept(prompt) == _dense(q) and lse.is_contiguous()
    for path in _paths(lambda: (ro.qk_position_rope(q, k, pos, rotary), ro.paged_rope_extend(own, q, k, k, rotary),
                                ro.paged_prefix_attention(q, own, shared))):
        (rq, rk), extended, (out, lse) = path()
        assert _kept(rq) == _kept(extended) == _kept(out) == _dense(q) and _kept(rk) == _dense(k) and lse.is_contiguous()
    if rows == 1:
        token = q[:, :, 0]
        for path in _paths(lambda: ro.paged_prefix_attention(token, own, shared)):
            assert _kept(path()[0]) == _dense(token)


def test_a_fused_projections_heads_join_without_a_copy():
    """Rotation, attention and the view that the output projection takes: one memory."""
    import r2omni_amd as ro

    dev = _cuda()
    x = torch.randn(2, 130, 12, 128, device=dev).to(BF16).transpose(1, 2)
    q, k = ro.qk_position_rope(x[:, :8], x[:, 8:10], torch.arange(130, device=dev).expand(2, 130), _rotary(dev))
    own = _cache(dev, (130, 130), 2, 16, BF16, 3)
    for out in (ro.prompt_attention(q, k, x[:, 10:])[0], ro.paged_prefix_attention(q, own)[0]):
        assert out.transpose(1, 2).reshape(2, 130, 8 * 128).data_ptr() == out.data_ptr()
