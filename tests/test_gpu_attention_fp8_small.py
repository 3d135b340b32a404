"""Decode and multi-query attention over an fp8 pool with bf16 queries below
f16's range: they are brought into it by a power of two, as larger ones are.
Tolerances as in test_gpu_attention_fp8.py."""

import numpy as np
import pytest

from pagedkv.workloads import Stream

from test_gpu_attention import tables_for
from test_gpu_attention_fp8 import TOL, check, run, setup_fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-100, -30, -20, -3, 16, 80])
def test_queries_far_from_one(cuda, power):
    cfg, b, ks, vs = setup_fp8(cuda, num_blocks=300, seed=11)
    st = Stream(12)
    ctx = np.array([40, 300, 9, 3000])
    tables = tables_for(st, cfg, ctx)
    q_np = st.normal(4 * 14 * 128).reshape(4, 14, 128).astype(np.float32)
    scale = 0.1 * 2.0 ** -power
    q, out, lse = run(cuda, b, "bf16", q_np * np.float32(2.0 ** power), tables, ctx, 3000, 0, scale=scale)
    assert b.device_error() is None
    check(b, ks, vs, q, out, lse, tables, ctx, 0, scale, TOL["bf16"])


def test_two_query_tokens(cuda):
    """Twice the same query token, the second over one key more: the second's
    result is that of decode over the whole context."""
    import torch

    cfg, b, ks, vs = setup_fp8(cuda, num_blocks=300, seed=11)
    st = Stream(12)
    ctx = np.array([40, 300, 9])
    tables = tables_for(st, cfg, ctx)
    q_np = (st.normal(3 * 14 * 128).reshape(3, 14, 128) * 2.0 ** -25).astype(np.float32)
    scale = 0.1 * 2.0 ** 25
    q = torch.from_numpy(q_np).to(cuda).to(torch.bfloat16)
    two = q.repeat_interleave(2, 0)
    out = torch.full(two.shape, float("nan"), device=cuda, dtype=two.dtype)
    lse = torch.full(two.shape[:2], float("nan"), device=cuda)
    b.paged_attention(two, torch.from_numpy(tables).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda), 300, out,
                      0, softmax_scale=scale, lse=lse, q_len=2)
    torch.cuda.synchronize()
    assert b.device_error() is None
    check(b, ks, vs, q, out[1::2], lse[1::2], tables, ctx, 0, scale, TOL["bf16"])
    check(b, ks, vs, q, out[0::2], lse[0::2], tables, ctx - 1, 0, scale, TOL["bf16"])


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
