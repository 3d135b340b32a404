"""paged_attention_chunk and prompt_attention against the float64 oracle
(oracle/layer_step.py), at ragged lengths, odd groups, page and tile borders,
with what they must not read or write; bounds in tests/layer_step.py."""

import numpy as np
import pytest

from oracle import layer_step as ref
from pagedkv.errors import InvalidBlock, ShapeMismatch
from tests.layer_step import attention_bounds, cu_of, ints, make_pool, tables_for, torch_type, values

pytestmark = pytest.mark.gpu


def random_rows(cuda, shape, dtype, seed, std=1.0):
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=cuda) * std).to(torch_type(dtype))


def run_chunk(cuda, b, q, tables, ctx, new, layer=1, scale=None, pad=0, max_new=None, max_len=None, cu=None):
    import torch

    out = torch.full(q.shape, float("nan"), device=cuda, dtype=q.dtype)
    lse = torch.full(q.shape[:2], float("nan"), device=cuda, dtype=torch.float32)
    b.paged_attention_chunk(q, ints(cuda, cu_of(new) if cu is None else cu), ints(cuda, tables), ints(cuda, ctx),
                            max(new) if max_new is None else max_new,
                            int(np.max(np.add(ctx, new))) if max_len is None else max_len, out, layer,
                            softmax_scale=scale, lse=lse)
    torch.cuda.synchronize()
    return out, lse


def check(q, out, lse, want, want_lse, kk, vv, mean_abs, dtype, scale, lengths):
    n = len(want)
    tol, lse_tol = attention_bounds(q, kk, vv, want, mean_abs, dtype, scale, lengths)
    err = np.abs(out[:n].double().cpu().numpy() - want)
    assert (err <= tol).all(), (np.nanmax(err - tol), np.argwhere(~(err <= tol))[:4], np.nanmax(err / tol))
    got = lse[:n].double().cpu().numpy()
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(got), empty)
    diff = np.abs(got[~empty] - want_lse[~empty])
    assert (diff <= lse_tol + 2.0 ** -22 * np.abs(want_lse[~empty])).all(), diff.max()


def check_chunk(b, q, out, lse, tables, ctx, new, layer, dtype, scale=None, pool=None):
    d = q.shape[2]
    scale = scale or d ** -0.5
    kp, vp = pool or values(b)
    qs = q.double().cpu().numpy()
    live = [s for s, n in enumerate(new) if n]
    want, want_lse = ref.chunk_attention(kp, vp, layer, qs, tables, ctx, new, scale, d)
    mean_abs, _ = ref.chunk_attention(kp, np.abs(vp), layer, qs, tables, ctx, new, scale, d)
    per_head = kp[layer].reshape(-1, d)
    per_head = per_head[np.isfinite(per_head).all(1)]
    check(qs, out, lse, want, want_lse, per_head, vp[layer][np.isfinite(vp[layer])], mean_abs, dtype, scale,
          [ctx[s] + new[s] for s in live])


# Rows that fill a tile, miss one, pass one; contexts at page and key-tile borders; empty sequences.
RAGGED = ([1, 0, 5, 130, 17, 64, 1, 33], [0, 40, 300, 0, 128, 127, 511, 16])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,hkv,group", [(64, 2, 4), (128, 2, 7), (256, 1, 2), (128, 3, 1), (64, 1, 5), (128, 1, 16),
                                         (256, 2, 1), (64, 1, 40)])
def test_chunk_matches_oracle(cuda, dtype, d, hkv, group):
    new, ctx = RAGGED
    b = make_pool(cuda, dtype, hkv, d, seed=d + group)
    tables = tables_for(np.random.default_rng(d), 128, np.add(ctx, new))
    q = random_rows(cuda, (sum(new), hkv * group, d), dtype, seed=group)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, dtype)


@pytest.mark.parametrize("qdtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,hkv,group", [(64, 2, 3), (128, 2, 4), (256, 1, 4)])
def test_chunk_over_fp8_matches_oracle(cuda, qdtype, d, hkv, group):
    new, ctx = RAGGED
    b = make_pool(cuda, "fp8_e4m3", hkv, d, seed=d + group, std=3.0)
    tables = tables_for(np.random.default_rng(d), 128, np.add(ctx, new))
    q = random_rows(cuda, (sum(new), hkv * group, d), qdtype, seed=group)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, qdtype)


@pytest.mark.parametrize("dtype,pool", [("bf16", "bf16"), ("f16", "fp8_e4m3")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_few_rows_over_long_contexts(cuda, dtype, pool, d):
    """Contexts long enough to be shared by several CTAs."""
    new, ctx = [1, 3, 0, 20], [5000, 2047, 9000, 7001]
    b = make_pool(cuda, pool, 2, d, num_blocks=1600, layers=1, seed=d)
    tables = tables_for(np.random.default_rng(d), 1600, np.add(ctx, new))
    q = random_rows(cuda, (sum(new), 6, d), dtype, seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new, layer=0)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 0, dtype)


@pytest.mark.parametrize("pool", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("block_size", [32, 48, 128])
def test_other_page_sizes(cuda, block_size, pool):
    new, ctx = RAGGED
    b = make_pool(cuda, pool, 2, 64, num_blocks=64, block_size=block_size, seed=block_size)
    tables = tables_for(np.random.default_rng(7), 64, np.add(ctx, new), block_size)
    q = random_rows(cuda, (sum(new), 6, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")


@pytest.mark.parametrize("lengths", [[1], [2], [127], [128], [129], [255], [256], [257], [0, 0, 3, 0]])
def test_lengths_at_the_tile_borders(cuda, lengths):
    for group in (1, 3):
        b = make_pool(cuda, "bf16", 2, 64, num_blocks=64, seed=sum(lengths))
        for ctx0 in (0, 1, 127, 129):
            ctx = [ctx0] * len(lengths)
            tables = tables_for(np.random.default_rng(7), 64, np.add(ctx, lengths))
            q = random_rows(cuda, (sum(lengths), 2 * group, 64), "bf16", seed=3)
            out, lse = run_chunk(cuda, b, q, tables, ctx, lengths)
            assert b.device_error() is None
            check_chunk(b, q, out, lse, tables, ctx, lengths, 1, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,hkv,group", [(64, 2, 4), (128, 2, 7), (256, 1, 2), (128, 4, 1), (256, 2, 3)])
def test_prompt_matches_oracle(cuda, dtype, d, hkv, group):
    import torch

    new = [1, 130, 0, 17, 300, 64, 2]
    b = make_pool(cuda, "f32", hkv, d, num_blocks=2)
    t = sum(new)
    rows = random_rows(cuda, (t, (group + 2) * hkv * d), dtype, seed=d)
    for fused in (True, False):
        q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split([group * hkv * d, hkv * d, hkv * d], 1))
        if not fused:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        out = torch.full((t, group * hkv, d), float("nan"), device=cuda, dtype=q.dtype)
        lse = torch.full((t, group * hkv), float("nan"), device=cuda)
        b.prompt_attention(q, k, v, ints(cuda, cu_of(new)), max(new), out, lse=lse)
        torch.cuda.synchronize()
        assert b.device_error() is None
        qs, ks, vs = (x.double().cpu().numpy() for x in (q, k, v))
        want, want_lse = ref.prompt_attention(qs, ks, vs, new, d ** -0.5)
        mean_abs, _ = ref.prompt_attention(qs, ks, np.abs(vs), new, d ** -0.5)
        check(qs, out, lse, want, want_lse, ks, vs, mean_abs, dtype, d ** -0.5, new)


def test_large_scores_and_scale(cuda):
    """Maxima that keep growing along the keys, and a scale far from 1 / sqrt(D):
    weights of distant keys underflow, the running maximum moves often."""
    new, ctx = [40, 3], [600, 900]
    b = make_pool(cuda, "bf16", 1, 64, num_blocks=128, layers=1)
    k, _ = b.planes()
    k.mul_(0.25)
    tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
    for s, n in enumerate(np.add(ctx, new)):  # keys grow along the sequence
        for j in range(n):
            k[0, tables[s, j // 16], j % 16] *= 1 + j / 100
    q = random_rows(cuda, (43, 4, 64), "bf16", seed=3)
    for scale in (0.02, 0.5, 3.0):
        out, lse = run_chunk(cuda, b, q, tables, ctx, new, layer=0, scale=scale)
        check_chunk(b, q, out, lse, tables, ctx, new, 0, "bf16", scale=scale)


@pytest.mark.parametrize("pool", ["bf16", "fp8_e4m3"])
def test_what_the_masks_hide_does_not_leak(cuda, pool):
    """NaN and infinities behind each sequence's end, in free blocks, and in the
    keys and values of tokens that a row comes before."""
    import torch

    new, ctx = [33, 1, 130, 7], [20, 50, 0, 300]
    b = make_pool(cuda, pool, 2, 64, seed=1)
    tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
    k, v = b.planes()
    used = set()
    for s, n in enumerate(np.add(ctx, new)):
        used |= set(tables[s, :-(-n // 16)].tolist())
        last = tables[s, (n - 1) // 16]
        for p in (k, v):
            p.view(torch.uint8)[:, last, (n - 1) % 16 + 1:] = 0x7F if pool != "bf16" else 0xFF
    for blk in set(range(128)) - used:
        for p in (k, v):
            p.view(torch.uint8)[:, blk] = 0x7F if pool != "bf16" else 0xFF
    q = random_rows(cuda, (sum(new), 6, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    kp, vp = (np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in values(b))
    check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16", pool=(kp, vp))
    # A later token of the same chunk: rows before it keep every bit.
    row = 34 + 61
    at = 61
    for p in (k, v):
        p.view(torch.uint8)[1, tables[2, at // 16], at % 16] = 0x7F if pool != "bf16" else 0xFF
    out2, lse2 = run_chunk(cuda, b, q, tables, ctx, new)
    first = np.r_[0:row, 34 + 130:sum(new)]
    assert torch.equal(out[first], out2[first]) and torch.equal(lse[first], lse2[first])
    assert torch.isnan(out2[row:34 + 130]).all()


def test_an_infinite_value_reaches_the_rows_that_attend_it(cuda):
    import torch

    new = [90]
    b = make_pool(cuda, "bf16", 1, 64, num_blocks=16)
    tables = tables_for(np.random.default_rng(7), 16, new)
    _, v = b.planes()
    v[1, tables[0, 3], 2, 5] = float("inf")     # token 50, element 5
    v[1, tables[0, 4], 1, 9] = float("-inf")    # token 65, element 9
    q = random_rows(cuda, (90, 2, 64), "bf16", seed=3)
    out, _ = run_chunk(cuda, b, q, tables, [0], new)
    assert (out[50:, :, 5] == float("inf")).all() and (out[65:, :, 9] == float("-inf")).all()
    rest = out.clone()
    rest[50:, :, 5] = 0
    rest[65:, :, 9] = 0
    assert torch.isfinite(rest).all()


def test_packed_neighbours_do_not_leak(cuda):
    """A prompt whose rows are NaN changes no other prompt of the batch."""
    import torch

    new = [60, 40, 50, 200]
    b = make_pool(cuda, "bf16", 1, 64, num_blocks=2)
    q, k, v = (random_rows(cuda, (350, h, 64), "bf16", seed=h) for h in (4, 1, 1))
    outs = []
    for bad in (False, True):
        if bad:
            for x in (q, k, v):
                x[60:100] = float("nan")
        out = torch.zeros((350, 4, 64), device=cuda, dtype=q.dtype)
        b.prompt_attention(q, k, v, ints(cuda, cu_of(new)), 200, out)
        torch.cuda.synchronize()
        outs.append(out)
    keep = np.r_[0:60, 100:350]
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0][keep], outs[1][keep])
    assert torch.isnan(outs[1][60:100]).all()
    # Nor do rows of no sequence, behind the last one.
    out = torch.full((350, 4, 64), 7.0, device=cuda, dtype=q.dtype)
    k[300:], v[300:], q[60:100], k[60:100], v[60:100] = float("nan"), float("nan"), 0, 0, 0
    b.prompt_attention(q, k, v, ints(cuda, cu_of([60, 40, 50, 150])), 200, out)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (out[300:] == 7.0).all()


def test_bad_blocks_are_recorded_and_skipped(cuda):
    import torch

    new, ctx = [20, 1, 5], [100, 40, 0]
    for bad in (-1, 1 << 20):
        b = make_pool(cuda, "bf16", 2, 64)
        tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
        tables[0, 2] = bad
        tables[2, 0] = bad      # a sequence with no key left
        q = random_rows(cuda, (26, 6, 64), "bf16", seed=3)
        out, lse = run_chunk(cuda, b, q, tables, ctx, new)
        err = b.device_error()
        assert err is not None and isinstance(err[0], InvalidBlock) and err[1] in (0, 2)
        check_chunk(b, q, out, lse, tables, ctx, new, 1, "bf16")
        assert (out[21:] == 0).all() and torch.isneginf(lse[21:]).all()


def test_lengths_beyond_the_bounds_are_recorded(cuda):
    import torch

    new, ctx = [4, 9, 2, 3], [10, 5, 70, 8]
    b = make_pool(cuda, "bf16", 1, 64)
    tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
    q = random_rows(cuda, (18, 4, 64), "bf16", seed=3)
    for kw, bad, c in (({"max_new": 8}, 1, ctx), ({"max_len": 40}, 2, ctx), ({}, 3, [10, 5, 70, -1])):
        args = dict(max_new=9, max_len=72)
        args.update(kw)
        out, lse = run_chunk(cuda, b, q, tables, c, new, **args)
        err = b.device_error()
        assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == bad
        lo, hi = cu_of(new)[bad], cu_of(new)[bad + 1]
        assert (out[lo:hi] == 0).all() and torch.isneginf(lse[lo:hi]).all()
        keep = [s for s in range(4) if s != bad]
        rows = np.concatenate([np.arange(cu_of(new)[s], cu_of(new)[s + 1]) for s in keep])
        check_chunk(b, q[rows], out[rows], lse[rows], tables[keep], [c[s] for s in keep], [new[s] for s in keep], 1,
                    "bf16")


def test_rows_of_no_sequence_stay(cuda):
    import torch

    b = make_pool(cuda, "bf16", 1, 64)
    new, ctx = [5, 9], [3, 20]
    tables = tables_for(np.random.default_rng(7), 128, np.add(ctx, new))
    q = random_rows(cuda, (30, 4, 64), "bf16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, new)
    assert b.device_error() is None and torch.isnan(out[14:]).all() and torch.isnan(lse[14:]).all()
    check_chunk(b, q[:14], out, lse, tables, ctx, new, 1, "bf16")
    for cu, index in (([0, 5, 31], 1), ([-2, 5, 14], 0), ([0, 14, 5], 1)):
        out, lse = run_chunk(cuda, b, q, tables, ctx, new, cu=cu, max_new=30, max_len=48)
        err = b.device_error()
        assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == index
        untouched = torch.isnan(out).flatten(1).all(1).cpu().numpy()
        rows = {0: slice(0, 14)}.get(index) or slice(14, 30)
        assert untouched[14:].all()
        assert not untouched[5:14].any() if index == 0 else not untouched[:5].any()


def test_strided_queries_streams_and_repeats_give_the_same_bits(cuda):
    import torch

    new, ctx = [50, 1, 200], [2000, 3000, 100]
    b = make_pool(cuda, "bf16", 2, 128, num_blocks=400, layers=1)
    tables = tables_for(np.random.default_rng(7), 400, np.add(ctx, new))
    wide = random_rows(cuda, (251, 14 * 128 + 64), "bf16", seed=3)
    q = wide[:, 64:].unflatten(1, (14, 128))
    want, want_lse = run_chunk(cuda, b, q.contiguous(), tables, ctx, new, layer=0)
    other = torch.cuda.Stream()
    for stream in (None, other):
        with torch.cuda.stream(stream or torch.cuda.current_stream()):
            out, lse = run_chunk(cuda, b, q, tables, ctx, new, layer=0)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_captured_with_changing_lengths(cuda):
    """Captured once, replayed with other lengths, with a larger eager call in
    between, and beside a second graph on the same handle."""
    import torch

    b = make_pool(cuda, "bf16", 2, 64, num_blocks=700, layers=1)
    b.attention_reserve()
    tables = tables_for(np.random.default_rng(7), 700, [3000, 3000, 3000])
    q = random_rows(cuda, (64, 6, 64), "bf16", seed=3)
    d_t, d_c, d_cu = ints(cuda, tables), ints(cuda, [100, 2900, 0]), ints(cuda, cu_of([30, 1, 33]))
    out = torch.full(q.shape, float("nan"), device=cuda, dtype=q.dtype)
    lse = torch.full(q.shape[:2], float("nan"), device=cuda)
    k = random_rows(cuda, (64, 2, 64), "bf16", seed=9)
    out2 = torch.empty_like(out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=side):
        b.paged_attention_chunk(q, d_cu, d_t, d_c, 64, 3000, out, 0, lse=lse)
    with torch.cuda.graph(g2, stream=side):
        b.prompt_attention(q, k, k, d_cu, 64, out2)
    for new, ctx in (([30, 1, 33], [100, 2900, 0]), ([1, 1, 1], [2999, 17, 2500]), ([0, 64, 0], [0, 2936, 5])):
        d_cu.copy_(ints(cuda, cu_of(new)))
        d_c.copy_(ints(cuda, ctx))
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert b.device_error() is None
        n = sum(new)
        check_chunk(b, q[:n], out, lse, tables, ctx, new, 0, "bf16")
        prompt = out2.clone()
        big = random_rows(cuda, (1500, 6, 64), "bf16", seed=4)
        o, l = run_chunk(cuda, b, big, tables, [1000, 0, 0], [1000, 250, 250], layer=0)
        check_chunk(b, big[:4], o, l, tables, [1000], [4], 0, "bf16")
        eager = torch.empty_like(out2)
        b.prompt_attention(q, k, k, d_cu, 64, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager[:n], prompt[:n])


def test_chunk_of_few_rows_agrees_with_the_decode_kernel(cuda):
    """Both within their bounds of the same values: the framework's own decode
    attention on a uniform batch of single tokens."""
    import torch

    ctx = [99, 1000, 15, 16, 2047]
    b = make_pool(cuda, "f16", 2, 128, num_blocks=300)
    tables = tables_for(np.random.default_rng(7), 300, np.add(ctx, 1))
    q = random_rows(cuda, (5, 14, 128), "f16", seed=3)
    out, lse = run_chunk(cuda, b, q, tables, ctx, [1] * 5)
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    b.paged_attention(q, ints(cuda, tables), ints(cuda, np.add(ctx, 1)), 2048, out2, 1, lse=lse2)
    torch.cuda.synchronize()
    assert (out.float() - out2.float()).abs().max() <= 4 * 2.0 ** -11 * 4  # |v| up to about 4, each side two roundings
    assert (lse - lse2).abs().max() <= 1e-4


def test_a_sequence_in_chunks_is_the_whole_prompt(cuda):
    """The operators together: a prompt's rows rotated, cached and attended at
    once, and the same prompt in ragged chunks through the cache, beside other
    sequences."""
    import torch
    from pagedkv import rope_table

    d, hkv, hq, total = 64, 2, 6, 300
    rows = random_rows(cuda, (total, (hq + 2 * hkv) * d), "bf16", seed=11)
    table = torch.from_numpy(rope_table(512, d)).to(cuda)

    def split(x):
        return [y.unflatten(1, (-1, d)) for y in x.split([hq * d, hkv * d, hkv * d], 1)]

    b = make_pool(cuda, "bf16", hkv, d, num_blocks=64, layers=2)
    tables = ints(cuda, tables_for(np.random.default_rng(7), 64, [total, 200]))
    q, k, v = split(rows.clone())
    cu = torch.zeros(2, device=cuda, dtype=torch.int32)
    b.rope_and_cache(tables[:1], ints(cuda, [0]), ints(cuda, [total]), total, cu, q, k, v, table, 0, k_out=k)
    whole, whole_lse = torch.empty((total, hq, d), device=cuda, dtype=q.dtype), torch.empty((total, hq), device=cuda)
    b.prompt_attention(q, k, v, cu, total, whole, lse=whole_lse)
    parts, lses, at = [], [], 0
    for step, n in enumerate([100, 1, 1, 131, 67]):
        x = torch.cat([rows[at:at + n], rows[:40]])     # beside 40 more tokens of another sequence
        q2, k2, v2 = split(x)
        d_c, d_n = ints(cuda, [at, 40 * step]), ints(cuda, [n, 40])
        cu2 = torch.zeros(3, device=cuda, dtype=torch.int32)
        b.rope_and_cache(tables, d_c, d_n, n + 40, cu2, q2, k2, v2, table, 1)
        out = torch.empty((n + 40, hq, d), device=cuda, dtype=q.dtype)
        lse = torch.empty((n + 40, hq), device=cuda)
        b.paged_attention_chunk(q2, cu2, tables, d_c, max(n, 40), max(at + n, 40 * step + 40), out, 1,
                                lse=lse)
        parts.append(out[:n])
        lses.append(lse[:n])
        at += n
    torch.cuda.synchronize()
    assert b.device_error() is None and at == total
    kp, vp = values(b)
    qs = q.double().cpu().numpy()
    tab = tables.cpu().numpy()
    want, want_lse = ref.chunk_attention(kp, vp, 0, qs, tab[:1], [0], [total], d ** -0.5, d)
    mean_abs, _ = ref.chunk_attention(kp, np.abs(vp), 0, qs, tab[:1], [0], [total], d ** -0.5, d)
    for o, l in ((whole, whole_lse), (torch.cat(parts), torch.cat(lses))):
        check(qs, o, l, want, want_lse, kp[0].reshape(-1, d), vp[0], mean_abs, "bf16", d ** -0.5, [total])


def test_refusals(cuda):
    import torch
    from pagedkv.errors import CacheError, Device, InvalidLayer

    bf, i = torch.bfloat16, torch.zeros(2, device=cuda, dtype=torch.int32)
    t = torch.zeros((1, 4), device=cuda, dtype=torch.int32)

    def rows(h, d=64, n=4, dtype=bf):
        return torch.zeros((n, h, d), device=cuda, dtype=dtype)

    def chunk(b, q, layer=0, max_new=4, max_len=64, scale=None, out=None, tables=t):
        b.paged_attention_chunk(q, i, tables, i[:1], max_new, max_len, rows(*q.shape[1:], n=len(q), dtype=q.dtype)
                                if out is None else out, layer, softmax_scale=scale)

    ok = make_pool(cuda, "bf16", 2, 64, num_blocks=4)
    chunk(ok, rows(4))
    for call, kind in ((lambda: chunk(ok, rows(4), layer=2), InvalidLayer),
                       (lambda: chunk(ok, rows(3)), ShapeMismatch),
                       (lambda: chunk(ok, rows(4), max_len=65), ShapeMismatch),
                       (lambda: chunk(ok, rows(4), max_new=-1), ShapeMismatch),
                       (lambda: chunk(ok, rows(4, dtype=torch.float16)), Device),
                       (lambda: chunk(ok, rows(4, dtype=torch.float32)), Device),
                       (lambda: chunk(ok, rows(4), scale=0.0), Device),
                       (lambda: chunk(ok, rows(4), scale=float("nan")), Device),
                       (lambda: chunk(ok, rows(258)), Device),
                       (lambda: chunk(ok, torch.zeros(2000, device=cuda, dtype=bf)[1:1025].view(4, 4, 64)), Device),
                       (lambda: chunk(ok, torch.zeros((4, 260), device=cuda, dtype=bf)[:, :256].unflatten(1, (4, 64))),
                        ShapeMismatch),
                       (lambda: chunk(make_pool(cuda, "f32", 2, 64, num_blocks=4), rows(4, dtype=torch.float32)), Device),
                       (lambda: chunk(make_pool(cuda, "bf16", 2, 96, num_blocks=4), rows(4, 96)), Device),
                       (lambda: chunk(make_pool(cuda, "bf16", 2, 64, num_blocks=4, block_size=8), rows(4), max_len=8), Device),
                       (lambda: chunk(make_pool(cuda, "bf16", 1, 64, num_blocks=4, shard=(0, 2)), rows(4)), Device),
                       (lambda: ok.prompt_attention(rows(4, dtype=torch.float32), rows(2, dtype=torch.float32),
                                                    rows(2, dtype=torch.float32), i, 4, rows(4, dtype=torch.float32)), Device),
                       (lambda: ok.prompt_attention(rows(4), torch.zeros(2000, device=cuda, dtype=bf)[1:513].view(4, 2, 64),
                                                    torch.zeros(2000, device=cuda, dtype=bf)[1:513].view(4, 2, 64), i, 4,
                                                    rows(4)), Device),
                       (lambda: ok.prompt_attention(rows(4), rows(2), rows(2), i, -1, rows(4)), ShapeMismatch)):
        with pytest.raises(CacheError) as e:
            call()
        assert isinstance(e.value, kind), (e.value, kind)
    torch.cuda.synchronize()
    assert ok.device_error() is None
    # Nothing to do is no error.
    ok.prompt_attention(rows(4, n=0), rows(2, n=0), rows(2, n=0), i[:1], 0, rows(4, n=0))
    ok.paged_attention_chunk(rows(4, n=0), i, t, i[:1], 0, 0, rows(4, n=0), 1)
