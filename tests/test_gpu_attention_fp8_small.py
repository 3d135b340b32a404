"""Decode and multi-query attention over an fp8 pool with bf16 queries below
f16's range: they are brought into it by a power of two, as larger ones are.
Tolerances as in test_gpu_attention_fp8.py."""

import numpy as np
import pytest

from pagedkv.workloads import Stream

from test_gpu_attention import tables_for
from test_gpu_attention_fp8 import TOL, check, run, setup_fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-37, 0.1])
def test_scales_whose_product_underflows(cuda, scale):
    """Scores so small that every key weighs the same."""
    cfg, b, ks, vs = setup_fp8(cuda, num_blocks=100, seed=11)
    ks[:] = 1e-10
    b.set_kv_scales(ks, vs)
    st = Stream(12)
    ctx = np.array([40, 300, 9])
    tables = tables_for(st, cfg, ctx)
    q_np = st.normal(3 * 14 * 128).reshape(3, 14, 128).astype(np.float32)
    q, out, lse = run(cuda, b, "bf16", q_np, tables, ctx, 300, 0, scale=scale)
    assert b.device_error() is None
    check(b, ks, vs, q, out, lse, tables, ctx, 0, scale, TOL["bf16"])
