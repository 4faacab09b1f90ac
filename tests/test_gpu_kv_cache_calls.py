"""The cache calls as programs make them: pools whose memory is replaced, streams that are not the current one."""
from __future__ import annotations

import pytest

from test_gpu_kv_cache import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(attn_lib):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device: there is no fallback path to test")
    from autorust_b200 import ops as _ops
    return _ops


def test_a_pool_whose_memory_is_replaced(ops):
    """Parked on the host, its GPU memory given to others, grown again elsewhere: calls use the memory that the tensors have now."""
    import torch
    s = Setup(ops, 13, [40, 9], Hkv=2, D=64, mean=True)
    s.append([30, 9], [30, 9])
    tensors = (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)
    parked = [x.cpu() for x in tensors]
    for x in tensors:
        x.untyped_storage().resize_(0)
    with pytest.raises(ops._abi.AttnLibraryError, match="null"):
        s.append([40, 9], [10, 0])
    others = [torch.full((p.numel() * p.element_size(),), 77, dtype=torch.uint8, device="cuda") for p in parked for _ in range(3)]
    for x, p in zip(tensors, parked):
        x.untyped_storage().resize_(p.numel() * p.element_size())
        x.copy_(p)
    s.plain = type(s.plain)(*s.cache.k.shape[:4], False, s.k_mean)
    for i, (codes, scales) in enumerate(((parked[0], parked[2]), (parked[1], parked[3]))):
        s.plain.codes[i][:], s.plain.scales[i][:] = codes.numpy(), scales.numpy()
    s.append([40, 9], [10, 0])
    s.check_pool()
    s.check_attention([40, 9], [3, 1], 4)
    s.cache.v.data = s.cache.v.clone()
    s.append([40, 12], [0, 3])
    s.check_pool()
    s.check_attention([40, 12], [3, 1], 4)
    torch.cuda.synchronize()
    assert all((x == 77).all() for x in others)


def _busy_block(torch, nbytes, ms=40):
    """A block of the current stream's pool that was given back while a kernel queued there will still write it; where it lies."""
    x = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(int(ms * 1.9e6))
    x.fill_(0xff)
    return x.data_ptr()


@pytest.mark.parametrize("what", ["attention", "workspace", "read"])
def test_memory_for_another_stream(ops, what):
    """A call on a stream that does not wait for the current one gets no memory that kernels of the current one still write."""
    import torch
    s = Setup(ops, 15, [9000, 300], Hkv=1, D=128, page=32)
    s.append([9000, 300], [9000, 300])
    where = (s.dtable, s.ints([9000, 300]))
    q = s.rows(2, 4)[0].contiguous()
    side = torch.cuda.Stream()
    out = torch.empty_like(q)
    need = ops._abi.load().ar_kv_cache_attention_workspace_bytes(s.cache._pool, ops._kv_batch(s.cache, *where, None, 2), 1, 4, 9024, 1)
    assert need > 0
    starts = s.ints([0, 9000, 9300])
    nbytes, run = {"attention": (q.numel() * 2, lambda **kw: ops.kv_cache_attention(s.cache, q, *where, workspace=torch.empty_like(ws), **kw)),
                   "workspace": (need, lambda **kw: ops.kv_cache_attention(s.cache, q, *where, out=out, **kw)),
                   "read": (2 * 9300 * 128 * 2, lambda **kw: ops.kv_cache_read(s.cache, *where, starts, 9300, **kw)[1])}[what]
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    want = run().clone()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    at = _busy_block(torch, nbytes)
    got = run(stream=side)
    assert what == "workspace" or got.data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # and the result stays while the caller's stream reads it
    if what != "workspace":
        got = run(stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(int(40 * 1.9e6))
        copy = got.clone()
        del got
        with torch.cuda.stream(side):
            torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(0xff)
        torch.cuda.synchronize()
        assert torch.equal(copy, want)
