"""Edges of paged_attention_chunk and prompt_attention: very many and very
wide groups and sequences, shared pages, queries that are not finite or far
from 1, outputs at 16-byte alignment, capture without a workspace, two handles
at once, random ragged batches. Bounds as in tests/layer_step.py."""

import numpy as np
import pytest

from oracle import layer_step as ref
from pagedkv.errors import Device
from tests.layer_step import cu_of, ints, make_pool, tables_for, values
from tests.test_gpu_prefill_attention import check, check_chunk, random_rows, run_chunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,group", [(64, 128), (128, 100), (256, 65)])
def test_wide_groups(cuda, d, group):
    """A token's rows nearly or wholly fill a tile: one token per row tile."""
    new, ctx = [3, 1], [140, 0]
    b = make_pool(cuda, "bf16", 1, d, num_blocks=16)
    tables = tables_for(np.random.default_rng(7), 16, np.add(ctx, new))
    q = random_rows(cuda, (4, group, d), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")


@pytest.mark.parametrize("count", [700, 2600])
def test_many_sequences(cuda, count):
    """More sequences than threads that plan, most of them empty or one token."""
    rng = np.random.default_rng(count)
    new = rng.choice([0, 0, 1, 1, 2, 5], count)
    ctx = rng.choice([0, 3, 15, 16, 40], count)
    b = make_pool(cuda, "bf16", 1, 64, num_blocks=4 * count)
    tables = tables_for(rng, 4 * count, np.add(ctx, new))
    q = random_rows(cuda, (int(new.sum()), 2, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")


def test_shared_pages(cuda):
    """Sequences that share their prefix's pages, and one page listed twice."""
    import torch

    new, ctx = [20, 20, 1], [64, 64, 95]
    b = make_pool(cuda, "f16", 2, 64, num_blocks=32)
    tables = tables_for(np.random.default_rng(7), 32, np.add(ctx, new))
    tables[1, :4] = tables[0, :4]
    tables[2, 3] = tables[2, 1]
    q = random_rows(cuda, (41, 4, 64), "f16", seed=3)
    q[20:40] = q[:20]
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "f16")
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("pool,qdtype", [("bf16", "bf16"), ("f16", "f16"), ("fp8_e4m3", "bf16"), ("fp8_e4m3", "f16")])
@pytest.mark.parametrize("group", [4, 7])
def test_rows_that_are_not_finite_stay_alone(cuda, pool, qdtype, group):
    import torch

    new, ctx = [90, 3], [200, 700]
    b = make_pool(cuda, pool, 1, 128, num_blocks=70)
    tables = tables_for(np.random.default_rng(7), 70, np.add(ctx, new))
    q = random_rows(cuda, (93, group, 128), qdtype, seed=3)
    want, want_lse = run_chunk(cuda, b, q, tables, ctx, new)
    bad = [(0, 1), (17, 0), (18, group - 1), (60, 2), (91, 0)]
    for i, h in bad:
        q[i, h, 5] = float("nan")
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    hit = torch.zeros((93, group), dtype=torch.bool, device=cuda)
    for i, h in bad:
        hit[i, h] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


@pytest.mark.parametrize("power", [-60, -20, 16, 60])
def test_fp8_with_queries_far_from_one(cuda, power):
    """bf16 queries times 2^power, the softmax scale undoing it: the same scores,
    so the same outputs within two runs' bounds of one result."""
    new, ctx = [40, 1], [100, 300]
    b = make_pool(cuda, "fp8_e4m3", 1, 64, num_blocks=40)
    tables = tables_for(np.random.default_rng(7), 40, np.add(ctx, new))
    q = random_rows(cuda, (41, 4, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q * 2.0 ** power, tables, ctx, new, scale=0.125 * 2.0 ** -power)
    assert b.device_error() is None
    # Powers of two are exact throughout: the oracle takes the unscaled form.
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16", scale=0.125)


def test_output_at_16_bytes(cuda):
    import torch

    new, ctx = [70, 1, 20], [30, 500, 0]
    b = make_pool(cuda, "bf16", 2, 128, num_blocks=60)
    tables = tables_for(np.random.default_rng(7), 60, np.add(ctx, new))
    q = random_rows(cuda, (91, 6, 128), "bf16", seed=3)
    want, _ = run_chunk(cuda, b, q, tables, ctx, new)
    flat = torch.full((91 * 6 * 128 + 16,), 7.0, device=cuda, dtype=q.dtype)
    out = flat[8:-8].view(91, 6, 128)
    assert out.data_ptr() % 32 == 16
    b.paged_attention_chunk(q, ints(cuda, cu_of(new)), ints(cuda, tables), ints(cuda, ctx), 70, 501, out, 1)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and (flat[:8] == 7).all() and (flat[-8:] == 7).all()


def test_capture_without_a_workspace_is_refused(cuda):
    import torch

    b = make_pool(cuda, "bf16", 1, 64, num_blocks=8)
    q = random_rows(cuda, (4, 2, 64), "bf16", seed=3)
    k = random_rows(cuda, (4, 1, 64), "bf16", seed=4)
    cu, out = ints(cuda, [0, 4]), torch.zeros_like(q)
    one = torch.zeros(1, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(Device, match="reserve"):
            b.prompt_attention(q, k, k, cu, 4, out)
        one.add_(1)
    b.attention_reserve()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.prompt_attention(q, k, k, cu, 4, out)
    graph.replay()
    torch.cuda.synchronize()
    qs, ks = q.double().cpu().numpy(), k.double().cpu().numpy()
    want, want_lse = ref.prompt_attention(qs, ks, ks, [4], 0.125)
    mean_abs, _ = ref.prompt_attention(qs, ks, np.abs(ks), [4], 0.125)
    lse = torch.from_numpy(want_lse).to(cuda)
    check(qs, out, lse, want, want_lse, ks, ks, mean_abs, "bf16", 0.125, [4])


def test_two_handles_at_once(cuda):
    """Calls of two handles on two streams, interleaved: each as if alone."""
    import torch

    new, ctx = [100, 1, 3], [1500, 3000, 2000]
    pools, qs, wants = [], [], []
    for i in range(2):
        b = make_pool(cuda, "bf16", 2, 128, num_blocks=450, layers=1, seed=i)
        tables = tables_for(np.random.default_rng(i), 450, np.add(ctx, new))
        q = random_rows(cuda, (104, 14, 128), "bf16", seed=10 + i)
        wants.append(run_chunk(cuda, b, q, tables, ctx, new, layer=0)[0])
        pools.append((b, ints(cuda, tables)))
        qs.append(q)
    cu, c = ints(cuda, cu_of(new)), ints(cuda, ctx)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(w) for _ in range(10)] for w in wants]
    torch.cuda.synchronize()
    for k in range(10):
        for i, (b, t) in enumerate(pools):
            b.paged_attention_chunk(qs[i], cu, t, c, 100, 3001, outs[i][k], 0, stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, wants[i]) for o in outs[i])


def test_two_graphs_share_the_workspace(cuda):
    """Captured calls of one handle (split items, single rows, a prompt), their
    graphs replayed in turn on one stream: each as if alone."""
    import torch

    b = make_pool(cuda, "bf16", 2, 64, num_blocks=700, layers=1)
    tables = tables_for(np.random.default_rng(7), 700, [5000, 2000])
    t = ints(cuda, tables)
    q = random_rows(cuda, (400, 6, 64), "bf16", seed=3)
    k, v = (random_rows(cuda, (400, 2, 64), "bf16", seed=s) for s in (4, 5))
    few, one, cu = ints(cuda, [0, 30, 47]), ints(cuda, [0, 1, 2]), ints(cuda, [0, 390, 400])
    ctx = ints(cuda, [4900, 1900])
    calls = [lambda o: b.paged_attention_chunk(q, few, t, ctx, 30, 5000, o, 0),
             lambda o: b.paged_attention_chunk(q, one, t, ctx, 1, 5000, o, 0),
             lambda o: b.prompt_attention(q, k, v, cu, 390, o)]
    wants, outs, graphs = [], [], []
    for call in calls:
        wants.append(torch.zeros_like(q))
        call(wants[-1])
    torch.cuda.synchronize()
    for call in calls:
        outs.append(torch.zeros_like(q))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(outs[-1])
    for order in ((0, 1, 2), (2, 0, 1), (1, 1, 0, 0, 2)):
        for o in outs:
            o.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert b.device_error() is None
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))


@pytest.mark.parametrize("seed", range(8))
def test_random_batches(cuda, seed):
    rng = np.random.default_rng(seed)
    d = int(rng.choice([64, 128, 256]))
    hkv, group = int(rng.integers(1, 4)), int(rng.integers(1, 10))
    pool, qd = [("bf16", "bf16"), ("f16", "f16"), ("fp8_e4m3", "bf16"), ("fp8_e4m3", "f16")][seed % 4]
    n = int(rng.integers(1, 9))
    new = rng.integers(0, 90, n)
    new[0] = max(new[0], 1)
    ctx = np.where(rng.random(n) < 0.3, 0, rng.integers(0, 900, n))
    bs = int(rng.choice([16, 32, 48]))
    b = make_pool(cuda, pool, hkv, d, num_blocks=600, block_size=bs, layers=1, seed=seed)
    tables = tables_for(rng, 600, np.add(ctx, new), bs)
    q = random_rows(cuda, (int(new.sum()), hkv * group, d), qd, seed=seed)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new, layer=0)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 0, qd)


def test_values_of_the_pool_are_only_read(cuda):
    b = make_pool(cuda, "bf16", 1, 64, num_blocks=40)
    before = values(b)
    tables = tables_for(np.random.default_rng(7), 40, [500])
    q = random_rows(cuda, (50, 2, 64), "bf16", seed=3)
    run_chunk(cuda, b, q, tables, [450], [50])
    assert all(np.array_equal(x, y) for x, y in zip(values(b), before))
