"""paged_attention_chunk with single rows (max_new_len 1: decode's ragged form;
2: the tile kernel) where the queries, the scales or the keys lie far from 1,
and the independence of a row's result from the rows beside it. Bounds as in
tests/layer_step.py."""

import numpy as np
import pytest

from tests.layer_step import make_pool, tables_for
from tests.test_gpu_prefill_attention import check_chunk, random_rows, run_chunk

pytestmark = pytest.mark.gpu

CTX = [100, 300, 0, 2700]
ONES = [1] * 4


def fp8_pool(cuda, d, seed=0):
    b = make_pool(cuda, "fp8_e4m3", 1, d, num_blocks=220, seed=seed)
    return b, tables_for(np.random.default_rng(7), 220, np.add(CTX, 1))


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 7), (256, 16)])
@pytest.mark.parametrize("power", [-60, -30, -20, 16, 60])
def test_fp8_with_queries_far_from_one(cuda, power, d, group, max_new):
    """bf16 queries times 2^power, the softmax scale undoing it: the same scores."""
    b, tables = fp8_pool(cuda, d)
    q = random_rows(cuda, (4, group, d), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q * 2.0 ** power, tables, CTX, ONES, scale=d ** -0.5 * 2.0 ** -power, max_new=max_new)
    assert b.device_error() is None
    # Powers of two are exact throughout: the oracle takes the unscaled form.
    check_chunk(b, q, out, lse, tables, CTX, ONES, 1, "bf16", scale=d ** -0.5)


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("power", [30, 100])
def test_fp8_with_one_head_far_above_the_others(cuda, power, d, max_new):
    """The heads of a group share K and V, not a range: one of them 2^power times
    the others leaves theirs as they are."""
    b, tables = fp8_pool(cuda, d)
    q = random_rows(cuda, (4, 4, d), "bf16", seed=3)
    wide = q * 2.0 ** -20
    wide[:, 2] *= 2.0 ** power
    out, lse = run_chunk(cuda, b, wide, tables, CTX, ONES, scale=d ** -0.5 * 2.0 ** 20, max_new=max_new)
    rest = [0, 1, 3]
    check_chunk(b, q[:, rest], out[:, rest], lse[:, rest], tables, CTX, ONES, 1, "bf16", scale=d ** -0.5)


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("qdtype", ["bf16", "f16"])
@pytest.mark.parametrize("k_scale,scale,zero", [(1e-12, 0.125, True), (1e-30, 0.125, True), (1e-10, 1e-37, False),
                                                (1e-20, 1e-30, True)])
def test_fp8_with_scales_whose_product_underflows(cuda, k_scale, scale, zero, qdtype, max_new):
    """Scores so small that every key weighs the same, masked ones nothing."""
    b, tables = fp8_pool(cuda, 64)
    b.test_scales[0][:] = k_scale
    b.set_kv_scales(*b.test_scales)
    q = random_rows(cuda, (4, 4, 64), qdtype, seed=3)
    if zero:
        q[:, 1] = 0
    out, lse = run_chunk(cuda, b, q, tables, CTX, ONES, scale=scale, max_new=max_new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, CTX, ONES, 1, qdtype, scale=scale)
