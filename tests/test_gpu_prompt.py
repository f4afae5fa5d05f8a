"""prompt_attention and attention_weights on the GPU against the definition in 64 bits."""
import math

import pytest
import torch

from attention_reference import close, prompt

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda:0")


def _rows(dev, b, hq, hkv, sq, sk, dtype, seed, gain=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(b, hq, sq, 128, generator=gen, device=dev) * gain
    k, v = (torch.randn(b, hkv, sk, 128, generator=gen, device=dev) for _ in range(2))
    return q.to(dtype), k.to(dtype), v.to(dtype)


def _check(q, k, v, window=None, sinks=0, nq=None, nk=None, scale=None):
    import r2omni_amd as ro

    dev = q.device
    lengths = {f"{n}_lengths": torch.tensor(x, dtype=torch.int32, device=dev) for n, x in (("query", nq), ("key", nk)) if x is not None}
    want = prompt(q, k, v, window, sinks, nq, nk, scale)
    out, lse = ro.prompt_attention(q, k, v, window=window, sinks=sinks, sm_scale=scale, **lengths)
    w = ro.attention_weights(q, k, lse, window=window, sinks=sinks, sm_scale=scale, **lengths)
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == w.dtype == torch.float32
    close(out, want[0], want[3])
    close(lse, want[1], want[4])
    close(w, want[2], want[5])
    return out, lse, w


# query rows and keys: one token, tile edges (32, 64, 128 and one to either side), odd ones, chunks of a longer prompt
SIZES = [(1, 1), (1, 64), (1, 1000), (2, 2), (31, 33), (32, 32), (63, 64), (65, 65), (64, 129), (127, 127), (128, 128),
         (129, 257), (200, 1031), (333, 333)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sq,sk", SIZES)
def test_sizes(sq, sk, dtype):
    q, k, v = _rows(_cuda(), 1, 4, 2, sq, sk, dtype, seed=sq * 1000 + sk)
    _check(q, k, v)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (16, 2), (28, 4), (32, 8), (5, 1), (20, 1)])
def test_head_layouts(hq, hkv):
    q, k, v = _rows(_cuda(), 2, hq, hkv, 70, 150, BF16, seed=hq)
    _check(q, k, v)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (65, 65), (100, 17), (128, 200), (1000, 4), (1 << 40, 3)])
@pytest.mark.parametrize("sq,sk", [(1, 300), (130, 130), (90, 517)])
def test_windows_and_sinks(window, sinks, sq, sk):
    q, k, v = _rows(_cuda(), 1, 4, 2, sq, sk, BF16, seed=window % 1000 + sinks)
    _check(q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 5)])
def test_ragged_batch_with_garbage_behind_the_lengths(dtype, window, sinks):
    """Empty requests, one row, more rows than keys (its first rows see nothing), a whole one; what lies behind a
    length is infinite or NaN and is not used."""
    nq, nk = [0, 1, 90, 150, 60, 150], [0, 1, 33, 200, 0, 150]
    q, k, v = _rows(_cuda(), 6, 4, 2, 150, 200, dtype, seed=3)
    for i, (a, n) in enumerate(zip(nq, nk)):
        q[i, :, a:] = math.nan
        k[i, :, n:] = math.inf
        v[i, :, n:] = math.nan
    out, lse, w = _check(q, k, v, window, sinks, nq, nk)
    assert not out[2, :, : 90 - 33].any() and (lse[2, :, : 90 - 33] == -math.inf).all()
    assert not w[4].any()


def test_values_that_later_rows_alone_see_may_be_anything():
    """A key's K and V rows do not reach the rows before it, whatever they hold."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 1, 4, 2, 200, 200, BF16, seed=8)
    want, lse = ro.prompt_attention(q, k, v)
    for bad in (math.inf, -math.inf, math.nan):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, 150:] = bad
        v2[:, :, 150] = bad
        v2[:, :, 163:, 5] = bad
        got, got_lse = ro.prompt_attention(q, k2, v2)
        assert torch.equal(got[:, :, :150], want[:, :, :150]) and torch.equal(got_lse[:, :, :150], lse[:, :, :150])
        got, _ = ro.prompt_attention(q, k, v2, window=20, sinks=0)
        clean, _ = ro.prompt_attention(q, k, v, window=20, sinks=0)
        assert torch.equal(got[:, :, :150], clean[:, :, :150])
        assert torch.equal(got[:, :, 183:, :5], clean[:, :, 183:, :5])  # row 150 has left their windows
        assert not torch.isfinite(got[:, :, 165:, 5].float()).any()     # and channel 5 has not
        assert not torch.isfinite(got[:, :, 150:170].float()).any()


def test_large_and_equal_logits():
    dev = _cuda()
    q, k, v = _rows(dev, 1, 4, 2, 130, 300, BF16, seed=5, gain=40.0)
    _check(q, k, v)                     # one key takes everything
    _check(q, k, v, scale=1e-6)         # every key the same
    _check(q * 0, k, v)
    _check(q, k, v, scale=3.0)


@pytest.mark.parametrize("rows_last", [False, True])
def test_strided_views_are_read_in_place(rows_last):
    """Heads as slices of one projection [B, S, (Hq + 2 Hkv) 128], and a cache's longer rows; with rows off 16 bytes
    the operands are copied."""
    import r2omni_amd as ro

    dev = _cuda()
    gen = torch.Generator(device=dev).manual_seed(4)
    qkv = torch.randn(2, 77, 8 * 128 + 8, generator=gen, device=dev).to(BF16)[:, :, 8 if rows_last else 4 :][:, :, : 8 * 128]
    q, k, v = (t.unflatten(2, (-1, 128)).transpose(1, 2) for t in qkv.split((4 * 128, 2 * 128, 2 * 128), dim=2))
    got = _check(q, k, v)
    again = ro.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_outputs_in_place_and_no_write_beside_them():
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 2, 4, 2, 70, 70, BF16, seed=6)
    want, lse = ro.prompt_attention(q, k, v)
    wide = torch.full((2, 70, 6, 128), 7.0, dtype=BF16, device=q.device)
    flat = torch.full((2 * 4 * 70 + 2,), 7.0, device=q.device)
    out, lse2 = wide[:, :, 1:5].transpose(1, 2), flat[1:-1].view(2, 4, 70)
    got = ro.prompt_attention(q, k, v, output=(out, lse2))
    assert got[0] is out and torch.equal(out, want) and torch.equal(lse2, lse)
    assert (wide[:, :, 0] == 7).all() and (wide[:, :, 5] == 7).all() and flat[0] == 7 and flat[-1] == 7
    w = ro.attention_weights(q, k, lse)
    buf = torch.full((2 * 2 * 70 + 2,), 7.0, device=q.device)
    assert ro.attention_weights(q, k, lse, output=buf[1:-1].view(2, 2, 70)).data_ptr() == buf[1:].data_ptr()
    assert torch.equal(buf[1:-1].view(2, 2, 70), w) and buf[0] == 7 and buf[-1] == 7


def test_weights_of_an_observation_window_and_row_sums():
    """The last rows alone count; each row of the prompt gives its weights a sum of one."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 1, 6, 2, 700, 700, BF16, seed=9)
    _, lse = ro.prompt_attention(q, k, v)
    tail = ro.attention_weights(q[:, :, -40:], k, lse[:, :, -40:])
    want = prompt(q[:, :, -40:], k, v)
    close(tail, want[2], want[5])
    whole = ro.attention_weights(q, k, lse)
    # 3 heads x 700 rows, each within 2^-10 of one
    assert (whole.double().sum(-1) - 3 * 700).abs().max() < 3 * 700 * 2.0 ** -10


def test_weights_are_summed_in_one_order_whatever_the_splits():
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 1, 16, 2, 900, 900, BF16, seed=10)
    _, lse = ro.prompt_attention(q, k, v)
    first = ro.attention_weights(q, k, lse)
    for _ in range(3):
        assert torch.equal(ro.attention_weights(q, k, lse), first)


def test_a_captured_call_follows_its_inputs():
    import r2omni_amd as ro

    dev = _cuda()
    q, k, v = _rows(dev, 2, 4, 2, 100, 300, BF16, seed=11)
    nk = torch.tensor([300, 250], dtype=torch.int32, device=dev)
    ro.prompt_attention(q, k, v, key_lengths=nk)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ro.prompt_attention(q, k, v, key_lengths=nk)
        w = ro.attention_weights(q, k, lse, key_lengths=nk)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        nk[1] = 250 - 70 * i
        graph.replay()
        torch.cuda.synchronize()
        o2, l2 = ro.prompt_attention(q, k, v, key_lengths=nk)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        assert torch.equal(w, ro.attention_weights(q, k, l2, key_lengths=nk))


def test_calls_follow_the_current_stream():
    import r2omni_amd as ro

    dev = _cuda()
    q, k, v = _rows(dev, 1, 4, 2, 256, 256, BF16, seed=12)
    want = ro.prompt_attention(q, k, v)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        q2 = q.clone()
        got = ro.prompt_attention(q2, k, v)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(got[0], want[0])
