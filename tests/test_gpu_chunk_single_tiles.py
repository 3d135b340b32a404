"""Batches of single rows through the tile kernel (max_new_len 2, which bounds
them as well): at the tile borders, and beside the decode kernel. Bounds as in
tests/layer_step.py."""

import numpy as np
import pytest

from tests.layer_step import attention_bounds, ints, make_pool, tables_for, values
from tests.test_gpu_prefill_attention import check_chunk, random_rows, run_chunk
from oracle import layer_step as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool,dtype", [("bf16", "bf16"), ("fp8_e4m3", "bf16")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tile_borders(cuda, d, pool, dtype):
    """A row whose keys end before, at and behind a key tile and a page."""
    new, ctx = [1] * 13, [0, 1, 14, 15, 16, 62, 63, 64, 126, 127, 128, 129, 255]
    for group in (1, 3):
        b = make_pool(cuda, pool, 2, d, num_blocks=140, seed=group)
        tables = tables_for(np.random.default_rng(7), 140, np.add(ctx, new))
        q = random_rows(cuda, (13, 2 * group, d), dtype, seed=3)
        out, lse = run_chunk(cuda, b, q, tables, ctx, new, max_new=2)
        assert b.device_error() is None
        check_chunk(b, q, out, lse, tables, ctx, new, 1, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 7), (256, 2)])
def test_agrees_with_the_decode_kernel(cuda, d, group, dtype):
    """The tiles and decode attention on the same single tokens: each is within
    its bound of the exact values, so they are within the two bounds of each other."""
    import torch

    ctx, new = [99, 1000, 15, 16, 2047], [1] * 5
    b = make_pool(cuda, dtype, 2, d, num_blocks=300)
    tables = tables_for(np.random.default_rng(7), 300, np.add(ctx, 1))
    q = random_rows(cuda, (5, 2 * group, d), dtype, seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new, max_new=2)
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    b.paged_attention(q, ints(cuda, tables), ints(cuda, np.add(ctx, 1)), 2048, out2, 1, lse=lse2)
    torch.cuda.synchronize()
    kp, vp = values(b)
    qs, scale = q.double().cpu().numpy(), d ** -0.5
    want, _ = ref.chunk_attention(kp, vp, 1, qs, tables, ctx, new, scale, d)
    mean_abs, _ = ref.chunk_attention(kp, np.abs(vp), 1, qs, tables, ctx, new, scale, d)
    tol, lse_tol = attention_bounds(qs, kp[1].reshape(-1, d), vp[1], want, mean_abs, dtype, scale, np.add(ctx, 1))
    diff = (out.double() - out2.double()).abs().cpu().numpy()
    assert (diff <= 2 * tol).all()
    assert (lse - lse2).abs().max().item() <= 2 * lse_tol + 2.0 ** -21 * lse.abs().max().item()
