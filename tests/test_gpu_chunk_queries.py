"""paged_attention_chunk with single rows (max_new_len 1: decode's ragged form;
2: the tile kernel) where the queries, the scales or the keys lie far from 1,
and the independence of a row's result from the rows beside it. Bounds as in
tests/layer_step.py."""

import numpy as np
import pytest

from tests.layer_step import ints, make_pool, tables_for
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


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_keys_at_minus_infinity_weigh_nothing(cuda, dtype, max_new):
    """Whole pages whose scores are -inf, before and between finite ones."""
    ctx, new = [200, 2700, 70], [1] * 3
    b = make_pool(cuda, dtype, 1, 64, num_blocks=220, layers=1)
    tables = tables_for(np.random.default_rng(7), 220, np.add(ctx, 1))
    k, _ = b.planes()
    for s, pages in enumerate(([0, 1, 2, 3, 4, 9], list(range(64)) + [100], [0, 1, 2, 3])):
        k[0, tables[s, pages], :, 5] = -float("inf")
    q = random_rows(cuda, (3, 4, 64), dtype, seed=3)
    q[..., 5] = q[..., 5].abs() + 0.5
    out, lse = run_chunk(cuda, b, q, tables, ctx, new, layer=0, max_new=max_new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 0, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_keys_at_minus_infinity_in_decode(cuda, dtype):
    """The same through decode attention, with one split and several."""
    import torch

    b = make_pool(cuda, dtype, 1, 64, num_blocks=220, layers=1)
    k, _ = b.planes()
    for count in (2, 200):
        ctx = [200, 70] * (count // 2)
        tables = np.repeat(tables_for(np.random.default_rng(7), 220, [201]), count, 0)  # shared pages
        k[0, tables[0, [0, 1, 2, 9]], :, 5] = -float("inf")
        q = random_rows(cuda, (count, 4, 64), dtype, seed=3)
        q[..., 5] = q[..., 5].abs() + 0.5
        out, lse = torch.full_like(q, float("nan")), torch.full((count, 4), float("nan"), device=cuda)
        b.paged_attention(q, ints(cuda, tables), ints(cuda, np.add(ctx, 1)), 201, out, 0, lse=lse)
        torch.cuda.synchronize()
        assert b.device_error() is None
        check_chunk(b, q, out, lse, tables, ctx, [1] * count, 0, dtype)


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("pool,qdtype", [("bf16", "bf16"), ("f16", "f16"), ("fp8_e4m3", "bf16"), ("fp8_e4m3", "f16")])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 7), (128, 16)])
@pytest.mark.parametrize("factor", [40.0, 0.0, float("nan")])
def test_a_head_does_not_hang_on_the_heads_beside_it(cuda, factor, d, group, pool, qdtype, max_new):
    """One head's queries change, and with them how often its maximum grows along
    the keys: the other heads keep every bit. Few sequences (keys split over
    CTAs) and many (every CTA walks a whole sequence)."""
    import torch

    b = make_pool(cuda, pool, 4, d, num_blocks=220, layers=1)
    hq = 4 * group
    changed = list(range(1, hq, group))
    rest = [h for h in range(hq) if h not in changed]
    for ctx in (CTX, list(range(20, 340, 4))):
        n = len(ctx)
        tables = np.repeat(tables_for(np.random.default_rng(7), 220, [2701]), n, 0)  # shared pages
        q = random_rows(cuda, (n, hq, d), qdtype, seed=3)
        want, want_lse = run_chunk(cuda, b, q, tables, ctx, [1] * n, layer=0, max_new=max_new)
        assert torch.isfinite(want).all()
        q[:, changed] *= factor
        out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * n, layer=0, max_new=max_new)
        assert torch.equal(out[:, rest], want[:, rest]) and torch.equal(lse[:, rest], want_lse[:, rest])
        assert torch.isnan(out[:, changed]).all() == (factor != factor)
