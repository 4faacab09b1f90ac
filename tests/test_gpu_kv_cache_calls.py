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
