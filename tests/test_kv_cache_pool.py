"""A pool's description follows its tensors' memory (no GPU needed: the tensors only say that they are CUDA tensors)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class OnGpu(torch.Tensor):
    is_cuda = True


def made(fill=0, mean=True, shape=(6, 2, 16, 64)):
    from autorust_b200 import ops
    new = lambda *s, kind=torch.float32: torch.full(s, fill, dtype=kind).as_subclass(OnGpu)
    pages, Hkv, _, D = shape
    return ops.KvCache(new(*shape, kind=torch.int8), new(*shape, kind=torch.int8), new(pages, Hkv), new(pages, Hkv),
                       new(Hkv, D) if mean else None)


def addresses(c):
    p = c._pool
    return [p.k, p.v, p.k_scale, p.v_scale, p.k_mean]


FIELDS = ("k", "v", "k_scale", "v_scale", "k_mean")


@pytest.mark.parametrize("field", FIELDS)
@pytest.mark.parametrize("how", ["set_", "data", "regrown"])
def test_memory_that_is_replaced_is_followed(field, how):
    c = made()
    t, keep = getattr(c, field), []
    if how == "set_":
        t.set_(t.clone())
    elif how == "data":
        t.data = t.clone()
    else:  # parked: freed, something else in its place, grown again
        n = t.untyped_storage().nbytes()
        t.untyped_storage().resize_(0)
        keep = [torch.empty(n, dtype=torch.uint8) for _ in range(4)]
        t.untyped_storage().resize_(n)
    assert addresses(c) == [getattr(c, f).data_ptr() for f in FIELDS]
    del keep


def test_freed_memory_is_no_address():
    c = made()
    c.k.untyped_storage().resize_(0)
    assert c._pool.k is None  # (which the call refuses)


def test_what_is_put_in_place_is_checked():
    c = made(mean=False)
    c.k.data = torch.zeros(5, 2, 16, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="v must be"):  # five pages of keys, six of values
        c._pool
    c = made(mean=False)
    c.k.data = torch.zeros(6, 2, 64, 16, dtype=torch.int8).transpose(2, 3)
    with pytest.raises(ValueError, match="contiguous"):
        c._pool
    c = made(mean=False)
    c.k.resize_(3, 2, 16, 64)  # in place: the same address
    with pytest.raises(ValueError, match="v must be"):
        c._pool


def test_nothing_is_described_twice():
    c = made()
    assert c._pool is c._pool and c._pool.k_mean == c.k_mean.data_ptr()
    assert made(mean=False)._pool.k_mean is None


def test_workspace_of_calls_that_are_refused(attn_lib):
    """As much as the call would, not the size of another type's call or none at all."""
    from autorust_b200 import _abi, ops
    c = made()
    assert ops.kv_cache_attention_workspace(c, 3, 8, 3, 9008) > 0 == ops.kv_cache_attention_workspace(c, 0, 8, 3, 9008)
    with pytest.raises(TypeError, match="float16"):
        ops.kv_cache_attention_workspace(c, 3, 8, 3, 9008, dtype=torch.float16)
    for sizes in ((3, 7, 3, 9008), (3, 8, 3, 0), (3, 8, 0, 9008), (-1, 8, 3, 9008)):
        with pytest.raises(_abi.AttnLibraryError, match="shape"):
            ops.kv_cache_attention_workspace(c, *sizes)
