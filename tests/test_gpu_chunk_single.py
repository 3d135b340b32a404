"""paged_attention_chunk where no sequence has more than one row (max_new_len 1):
empty sequences between, padding rows, refused lengths, bad blocks, rows that
are not finite, capture. Bounds as in tests/layer_step.py."""

import numpy as np
import pytest

from pagedkv.errors import InvalidBlock, ShapeMismatch
from tests.layer_step import cu_of, ints, make_pool, tables_for
from tests.test_gpu_prefill_attention import check_chunk, random_rows, run_chunk

pytestmark = pytest.mark.gpu

NEW = [1, 0, 1, 1, 0, 0, 1, 1, 1]
CTX = [0, 5, 15, 16, 0, 40, 700, 3000, 128]


@pytest.mark.parametrize("pool,qdtype", [("bf16", "bf16"), ("f16", "f16"), ("fp8_e4m3", "bf16"), ("fp8_e4m3", "f16")])
@pytest.mark.parametrize("d,hkv,group", [(64, 2, 4), (128, 2, 7), (256, 1, 16), (128, 1, 1), (64, 1, 17)])
def test_matches_oracle(cuda, pool, qdtype, d, hkv, group):
    import torch

    b = make_pool(cuda, pool, hkv, d, num_blocks=300, seed=d + group)
    tables = tables_for(np.random.default_rng(d), 300, np.add(CTX, NEW))
    n = sum(NEW)
    q = random_rows(cuda, (n + 3, hkv * group, d), qdtype, seed=group)
    out, lse = run_chunk(cuda, b, q, tables, CTX, NEW)
    assert b.device_error() is None
    assert torch.isnan(out[n:]).all() and torch.isnan(lse[n:]).all()
    check_chunk(b, q[:n], out, lse, tables, CTX, NEW, 1, qdtype)


def test_many_short_sequences_without_splits(cuda):
    rng = np.random.default_rng(5)
    new = rng.integers(0, 2, 400)
    ctx = rng.integers(0, 60, 400)
    b = make_pool(cuda, "bf16", 2, 64, num_blocks=1700)
    tables = tables_for(rng, 1700, np.add(ctx, new))
    q = random_rows(cuda, (int(new.sum()), 8, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")


@pytest.mark.parametrize("long", [False, True])
def test_refused_lengths(cuda, long):
    """A second row, a negative or too long context: zeros and a record; cu out
    of range: untouched. With and without splits."""
    import torch

    far = 2500 if long else 30
    b = make_pool(cuda, "bf16", 2, 64, num_blocks=700)
    tables = tables_for(np.random.default_rng(7), 700, [far + 1] * 4, extra=2)
    q = random_rows(cuda, (6, 6, 64), "bf16", seed=3)
    for cu, ctx, bad, zero in (([0, 1, 3, 4, 5], [far, 3, 4, 5], 1, [1, 2]), ([0, 1, 2, 3, 4], [far, -1, 4, 5], 1, [1]),
                               ([0, 1, 2, 3, 4], [far, 3, far + 1, 5], 2, [2])):
        out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * 4, cu=cu, max_new=1, max_len=far + 1)
        err = b.device_error()
        assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == bad
        assert (out[zero] == 0).all() and torch.isneginf(lse[zero]).all()
        keep = [s for s in range(4) if s != bad]
        rows = [cu[s] for s in keep]
        check_chunk(b, q[rows], out[rows], lse[rows], tables[keep], [ctx[s] for s in keep], [1] * 3, 1, "bf16")
        assert torch.isnan(out[cu[4]:]).all()
    for cu, bad in (([0, 1, 2, 3, 7], 3), ([-1, 0, 1, 2, 3], 0), ([0, 1, 0, 1, 2], 1)):
        out, lse = run_chunk(cuda, b, q, tables, [far, 3, 4, 5], [1] * 4, cu=cu, max_new=1, max_len=far + 1)
        err = b.device_error()
        assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == bad
        assert torch.isnan(out[4:]).all()


@pytest.mark.parametrize("ctx0", [40, 2700])
def test_rows_and_keys_that_are_not_finite(cuda, ctx0):
    import torch

    b = make_pool(cuda, "bf16", 1, 64, num_blocks=600, layers=1)
    ctx = [ctx0, ctx0 - 5, ctx0 + 1]
    tables = tables_for(np.random.default_rng(7), 600, np.add(ctx, 1))
    k, v = b.planes()
    q = random_rows(cuda, (3, 4, 64), "bf16", seed=3)
    q[1, 2] = float("nan")
    last = tables[0, ctx0 // 16]
    for p in (k, v):
        p[0, last, ctx0 % 16 + 1:] = float("nan")      # behind the sequence
    out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * 3, layer=0)
    bad = torch.zeros((3, 4), dtype=torch.bool, device=cuda)
    bad[1, 2] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.isfinite(out[~bad]).all() and torch.isfinite(lse[~bad]).all()
    k[0, tables[2, 1], 3] = float("nan")               # a key that the third row attends
    out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * 3, layer=0)
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all() and torch.isfinite(out[0]).all()


def test_no_rows_allowed(cuda):
    """max_new_len 0: a sequence with a row is refused, zeros and a record."""
    import torch

    b = make_pool(cuda, "bf16", 2, 64)
    tables = tables_for(np.random.default_rng(7), 128, [9, 9])
    q = random_rows(cuda, (2, 6, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, [8, 8], [0, 1], max_new=0)
    err = b.device_error()
    assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == 1
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and torch.isnan(out[1]).all()
    out, lse = run_chunk(cuda, b, q, tables, [8, 8], [0, 0], max_new=0)
    assert b.device_error() is None and torch.isnan(out).all()


@pytest.mark.parametrize("max_new", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_codes_behind_the_sequence(cuda, d, max_new):
    """An fp8 pool whose slots behind each sequence hold NaN codes, by both kernels."""
    import torch

    ctx = [40, 700, 2703]
    b = make_pool(cuda, "fp8_e4m3", 2, d, num_blocks=600, layers=1)
    tables = tables_for(np.random.default_rng(7), 600, np.add(ctx, 1))
    for p in b.planes():
        codes = p.view(torch.uint8)
        for s, c in enumerate(ctx):
            codes[0, tables[s, c // 16], c % 16 + 1:] = 0x7F
    q = random_rows(cuda, (3, 8, d), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * 3, layer=0, max_new=max_new)
    assert b.device_error() is None
    assert torch.isfinite(out).all()
    check_chunk(b, q, out, lse, tables, ctx, [1] * 3, 0, "bf16")


def test_bad_blocks(cuda):
    import torch

    ctx, new = [100, 10], [1, 1]
    b = make_pool(cuda, "bf16", 2, 64)
    tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
    tables[0, 2] = 1 << 20
    tables[1, 0] = -1
    q = random_rows(cuda, (2, 6, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    err = b.device_error()
    assert err is not None and isinstance(err[0], InvalidBlock) and err[1] in (0, 1)
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()


def test_agrees_with_the_tiles(cuda):
    """The same rows with max_new_len 2 take the tile kernel: within both bounds."""
    b = make_pool(cuda, "f16", 2, 128, num_blocks=300)
    tables = tables_for(np.random.default_rng(3), 300, np.add(CTX, NEW))
    q = random_rows(cuda, (sum(NEW), 8, 128), "f16", seed=4)
    for max_new in (1, 2):
        out, lse = run_chunk(cuda, b, q, tables, CTX, NEW, max_new=max_new)
        check_chunk(b, q, out, lse, tables, CTX, NEW, 1, "f16")


def test_captured_with_changing_lengths(cuda):
    import torch

    b = make_pool(cuda, "bf16", 2, 64, num_blocks=700, layers=1)
    b.attention_reserve()
    tables = tables_for(np.random.default_rng(7), 700, [3000] * 3)
    q = random_rows(cuda, (3, 6, 64), "bf16", seed=3)
    d_t, d_c, d_cu = ints(cuda, tables), ints(cuda, [0, 0, 0]), ints(cuda, [0, 1, 2, 3])
    out, lse = torch.zeros_like(q), torch.zeros((3, 6), device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.paged_attention_chunk(q, d_cu, d_t, d_c, 1, 3000, out, 0, lse=lse)
    for new, ctx in (([1, 1, 1], [100, 2900, 0]), ([0, 1, 1], [9, 2999, 17]), ([1, 0, 0], [63, 4, 5])):
        d_cu.copy_(ints(cuda, cu_of(new)))
        d_c.copy_(ints(cuda, ctx))
        graph.replay()
        torch.cuda.synchronize()
        assert b.device_error() is None
        check_chunk(b, q[:sum(new)], out, lse, tables, ctx, new, 0, "bf16")
