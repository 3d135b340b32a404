"""Views of the pool's planes keep the pool: a view that outlives the last
reference to its backend still reads the pool, not freed memory."""

import gc
import weakref

import pytest

from pagedkv import B200Backend, CacheConfig

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,size", [("f32", 4), ("bf16", 2), ("f16", 2), ("fp8_e4m3", 1)])
def test_views_keep_the_pool(cuda, dtype, size):
    import torch

    b = B200Backend(CacheConfig(8, 16, 2, 64, 2, size), dtype=dtype)
    ref = weakref.ref(b)
    k, v = b.planes()
    part = v[1, 3]
    part.view(torch.uint8).fill_(56)
    del b, k, v
    gc.collect()
    assert ref() is not None
    torch.cuda.synchronize()
    assert (part.view(torch.uint8) == 56).all()
    del part
    gc.collect()
    assert ref() is None
