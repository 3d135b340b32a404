"""rope_and_cache against the float64 oracle: rotated queries and keys, the
pool's contents, slots and cu_seqlens; what it leaves alone; its device errors.

Tolerances: a' = a c - b n in f32 is two products and a sum, each off by half
a step (2^-24) of at most |a| + |b|: 3 * 2^-24 * (|a| + |b|), with |c|, |n| <= 1
and at most one more step for the fused form; then one rounding to the type
(half a step of the value). An fp8 code is one rounding of the f32 product with
the inverse scale (2^-24 more), half a step of e4m3: 2^-4, or 2^-10 absolute
where the code is subnormal. Values pass through unchanged, bit for bit."""

import numpy as np
import pytest

from oracle import layer_step as ref
from pagedkv import rope_table
from pagedkv.errors import InvalidBlock, ShapeMismatch, SlotOutOfRange
from tests.layer_step import HALF, cu_of, ints, make_pool, tables_for, torch_type, values

pytestmark = pytest.mark.gpu

NEW = [3, 0, 1, 40, 17, 1, 128, 0, 5]
CTX = [0, 9, 15, 16, 1000, 31, 7, 0, 333]


def batch(cuda, b, src, hq, new, ctx, seed, pad=0, fused=True, table_len=1400, rotary=None):
    """Rows (with `pad` rows behind the tokens) and their metadata."""
    import torch

    cfg = b.config()
    d, hkv = cfg.head_dim, b.shard_entry_elems // cfg.head_dim
    t = int(np.sum(new)) + pad
    g = torch.Generator(device=cuda).manual_seed(seed)
    tdt = torch_type(src)
    rows = torch.randn((t, (hq + 2 * hkv) * d), generator=g, device=cuda).to(tdt)
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split([hq * d, hkv * d, hkv * d], 1)) if hq else \
        (None, rows[:, :hkv * d].unflatten(1, (-1, d)), rows[:, hkv * d:].unflatten(1, (-1, d)))
    if not fused:
        q, k, v = (None if x is None else x.contiguous() for x in (q, k, v))
    rng = np.random.default_rng(seed)
    tables = tables_for(rng, cfg.num_blocks, np.add(ctx, new), cfg.block_size)
    cs = rope_table(table_len, rotary or d, base=10000.0)
    return q, k, v, tables, cs


def check_against_oracle(b, before, src, q, q_got, k, k_got, v, cs, tables, ctx, new, layer, interleaved, slots):
    cfg = b.config()
    n = int(np.sum(new))
    seq, pos = ref.positions(ctx, new)
    rot = cs.shape[1]
    f32_err = lambda x: 4 * 2.0 ** -24 * (np.abs(x).max(-1, keepdims=True) * 2)  # noqa: E731
    for x, got in ((q, q_got), (k, k_got)):
        if x is None or got is None:
            continue
        xs = x[:n].double().cpu().numpy()
        want = ref.rotate(xs, cs, pos, rot, interleaved)
        err = np.abs(got[:n].double().cpu().numpy() - want)
        floor = 2.0 ** -25 if src == "f16" else 0.0
        assert (err <= HALF[src] * np.abs(want) * 1.001 + f32_err(xs) + floor).all()
    want_slots = ref.slots(tables, seq, pos, cfg.block_size)
    assert np.array_equal(slots[:n], want_slots)
    after = values(b)
    fp8 = b.elem_bytes == 1
    pool = "fp8_e4m3" if fp8 else src
    h0 = b.elem_offset // cfg.head_dim
    for i, x in enumerate((k, v)):
        xs = x[:n].double().cpu().numpy()
        want = ref.rotate(xs, cs, pos, rot, interleaved) if i == 0 else xs
        blk, off = want_slots // cfg.block_size, want_slots % cfg.block_size
        got = after[i][layer, blk, off].reshape(want.shape)
        err = np.abs(got - want)
        if fp8:
            scale = b.test_scales[i][layer, h0:h0 + want.shape[1]].astype(np.float64)[:, None]
            bound = 448 * scale
            clipped = np.clip(want, -bound, bound)
            tol = HALF[pool] * np.abs(clipped) * 1.001 + 2.0 ** -10 * scale + 2 * f32_err(xs)
            assert (np.abs(got - clipped) <= tol).all()
        else:
            floor = 2.0 ** -25 if src == "f16" else 0.0
            tol = (HALF[src] * np.abs(want) * 1.001 + f32_err(xs) + floor) if i == 0 else 0.0
            assert (err <= tol).all()
        untouched = np.ones(after[i].shape[:3], bool)
        untouched[layer, blk, off] = False
        assert np.array_equal(after[i][untouched], before[i][untouched])


@pytest.mark.parametrize("src,pool", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "fp8_e4m3"),
                                      ("f16", "fp8_e4m3"), ("f32", "fp8_e4m3")])
@pytest.mark.parametrize("hq,hkv,d,rotary,interleaved", [
    (8, 2, 128, 128, False), (7, 1, 64, 64, True), (4, 2, 256, 128, False), (0, 3, 64, 32, True),
    (3, 3, 80, 48, False), (5, 1, 24, 10, False), (2, 2, 4, 4, True), (6, 2, 96, 96, True), (1, 1, 1024, 1024, False)])
def test_matches_oracle(cuda, src, pool, hq, hkv, d, rotary, interleaved):
    import torch

    b = make_pool(cuda, pool, hkv, d, seed=d)
    q, k, v, tables, cs = batch(cuda, b, src, hq, NEW, CTX, seed=hq * 100 + d, rotary=rotary)
    before = values(b)
    n = sum(NEW)
    cu = torch.full((len(NEW) + 1,), -7, device=cuda, dtype=torch.int32)
    slots = torch.full((n,), -9, device=cuda, dtype=torch.int64)
    q_out = None if q is None else torch.full_like(q, 9.0).contiguous()
    k_out = torch.full(k.shape, 9.0, device=cuda, dtype=k.dtype)
    b.rope_and_cache(ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW), n, cu, q, k, v,
                     torch.from_numpy(cs).to(cuda), 1, q_out=q_out, k_out=k_out, interleaved=interleaved,
                     slots_out=slots)
    torch.cuda.synchronize()
    assert b.device_error() is None
    assert np.array_equal(cu.cpu().numpy(), cu_of(NEW))
    check_against_oracle(b, before, src, q, q_out, k, k_out, v, cs, tables, CTX, NEW, 1, interleaved,
                         slots.cpu().numpy())


def test_in_place_gives_the_same_bits(cuda):
    import torch

    outs = []
    for in_place in (False, True):
        b = make_pool(cuda, "bf16", 2, 128, seed=3)
        q, k, v, tables, cs = batch(cuda, b, "bf16", 8, NEW, CTX, seed=5)
        cu = torch.zeros(len(NEW) + 1, device=cuda, dtype=torch.int32)
        q_out = None if in_place else torch.empty(q.shape, device=cuda, dtype=q.dtype)
        k_out = k if in_place else torch.empty(k.shape, device=cuda, dtype=k.dtype)
        b.rope_and_cache(ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW), sum(NEW), cu, q, k, v,
                         torch.from_numpy(cs).to(cuda), 0, q_out=q_out, k_out=k_out)
        torch.cuda.synchronize()
        outs.append([x.clone() for x in (q if in_place else q_out, k_out, *b.planes())])
    assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_any_pitch_and_alignment_gives_the_same_bits(cuda):
    """Rows at an odd offset take the scalar form: same products, same rounding."""
    import torch

    b1, b2 = (make_pool(cuda, "bf16", 2, 64, seed=3) for _ in range(2))
    q, k, v, tables, cs = batch(cuda, b1, "bf16", 4, NEW, CTX, seed=5)
    n = sum(NEW)
    wide = torch.zeros((n, 1 + 8 * 64 + 2), device=cuda, dtype=q.dtype)
    wide[:, 1:1 + 8 * 64] = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    q2, k2, v2 = (x.unflatten(1, (-1, 64)) for x in wide[:, 1:1 + 512].split([256, 128, 128], 1))
    got = []
    for b, (x, y, z) in ((b1, (q, k, v)), (b2, (q2, k2, v2))):
        out = torch.empty((n, 4, 64), device=cuda, dtype=q.dtype)
        cu = torch.zeros(len(NEW) + 1, device=cuda, dtype=torch.int32)
        b.rope_and_cache(ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW), n, cu, x, y, z,
                         torch.from_numpy(cs).to(cuda), 1, q_out=out)
        torch.cuda.synchronize()
        got.append([out, *(p.clone() for p in b.planes())])
    for x, y in zip(*got):
        # Contraction of a c - b n may differ between the two forms by one rounding of the type.
        assert (x.float() - y.float()).abs().max() <= 2 * HALF["bf16"] * x.float().abs().max()


def test_many_sequences_and_decode(cuda):
    import torch

    for new, seed in (([1] * 300, 1), ([2, 0, 1] * 700, 2)):
        b = make_pool(cuda, "bf16", 1, 64, num_blocks=4000, seed=3)
        ctx = [(i * 7) % 29 for i in range(len(new))]
        q, k, v, tables, cs = batch(cuda, b, "bf16", 2, new, ctx, seed=seed, table_len=64)
        before = values(b)
        n = sum(new)
        cu = torch.zeros(len(new) + 1, device=cuda, dtype=torch.int32)
        slots = torch.zeros(n, device=cuda, dtype=torch.int64)
        out = torch.empty(q.shape, device=cuda, dtype=q.dtype)
        b.rope_and_cache(ints(cuda, tables), ints(cuda, ctx), ints(cuda, new), n, cu, q, k, v,
                         torch.from_numpy(cs).to(cuda), 0, q_out=out, slots_out=slots)
        torch.cuda.synchronize()
        assert b.device_error() is None and np.array_equal(cu.cpu().numpy(), cu_of(new))
        check_against_oracle(b, before, "bf16", q, out, k, None, v, cs, tables, ctx, new, 0, False,
                             slots.cpu().numpy())


def test_slots_are_those_of_resolve_and_cache(cuda):
    import torch

    b = make_pool(cuda, "bf16", 2, 64, block_size=24, num_blocks=100)
    q, k, v, tables, cs = batch(cuda, b, "bf16", 2, NEW, CTX, seed=8)
    n = sum(NEW)
    d_t, d_c, d_n = ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW)
    s1, s2 = (torch.zeros(n, device=cuda, dtype=torch.int64) for _ in range(2))
    c1, c2 = (torch.zeros(len(NEW) + 1, device=cuda, dtype=torch.int32) for _ in range(2))
    b.resolve_slots(d_t, d_c, d_n, n, c1, s1)
    b.rope_and_cache(d_t, d_c, d_n, n, c2, q, k, v, torch.from_numpy(cs).to(cuda), 0, slots_out=s2)
    torch.cuda.synchronize()
    assert torch.equal(s1, s2) and torch.equal(c1, c2)


def test_rows_behind_the_tokens_stay(cuda):
    import torch

    b = make_pool(cuda, "f16", 2, 64)
    q, k, v, tables, cs = batch(cuda, b, "f16", 4, NEW, CTX, seed=2, pad=5)
    q0, n = q.clone(), sum(NEW)
    slots = torch.full((n + 5,), -9, device=cuda, dtype=torch.int64)
    cu = torch.zeros(len(NEW) + 1, device=cuda, dtype=torch.int32)
    before = values(b)
    b.rope_and_cache(ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW), n + 5, cu, q, k, v,
                     torch.from_numpy(cs).to(cuda), 1, slots_out=slots)
    torch.cuda.synchronize()
    assert b.device_error() is None
    assert torch.equal(q[n:], q0[n:]) and (slots[n:] == -9).all()
    check_against_oracle(b, before, "f16", q0, q, k, None, v, cs, tables, CTX, NEW, 1, False, slots.cpu().numpy())


def test_refused_lengths_write_nothing(cuda):
    import torch

    for new, ctx, index in (([4, 4], [0, 0], 8), ([2, -1], [0, 0], -1), ([2, 1], [0, -3], -1)):
        b = make_pool(cuda, "bf16", 1, 64)
        q, k, v, tables, cs = batch(cuda, b, "bf16", 2, [3, 3], [0, 0], seed=2)
        before, q0 = values(b), q.clone()
        cu = torch.zeros(3, device=cuda, dtype=torch.int32)
        b.rope_and_cache(ints(cuda, tables), ints(cuda, ctx), ints(cuda, new), 6, cu, q, k, v,
                         torch.from_numpy(cs).to(cuda), 0)
        err = b.device_error()
        assert err is not None and isinstance(err[0], ShapeMismatch) and err[1] == index
        assert torch.equal(q, q0) and all(np.array_equal(x, y) for x, y in zip(values(b), before))


def test_bad_blocks_positions_and_tables_are_recorded(cuda):
    import torch

    new = [2, 2, 2]
    for what in ("block", "table", "angles"):
        ctx = [0, 20, 98]
        b = make_pool(cuda, "bf16", 1, 64)
        q, k, v, tables, cs = batch(cuda, b, "bf16", 2, new, ctx, seed=2, table_len=100 if what != "angles" else 99)
        tables = tables[:, :-1]
        if what == "block":
            tables[1, 1] = 1 << 20
        if what == "table":
            tables = np.ascontiguousarray(tables[:, :1])
            ctx = [0, 20, 8]
        out = torch.full(q.shape, 5.0, device=cuda, dtype=q.dtype)
        slots = torch.zeros(6, device=cuda, dtype=torch.int64)
        cu = torch.zeros(4, device=cuda, dtype=torch.int32)
        before = values(b)
        b.rope_and_cache(ints(cuda, tables), ints(cuda, ctx), ints(cuda, new), 6, cu, q, k, v,
                         torch.from_numpy(cs).to(cuda), 1, q_out=out, slots_out=slots)
        err = b.device_error()
        got = slots.cpu().numpy()
        kind, skipped = {"block": (InvalidBlock, [2, 3]), "table": (SlotOutOfRange, [2, 3]),
                         "angles": (ShapeMismatch, [5])}[what]
        assert err is not None and isinstance(err[0], kind) and err[1] in skipped
        assert (got[skipped] == -1).all() and (np.delete(got, skipped) >= 0).all()
        rotated = (out != 5.0).flatten(1).any(1).cpu().numpy()
        assert rotated.tolist() == [not (what == "angles" and i in skipped) for i in range(6)]
        after = values(b)
        changed = (after[0] != before[0]).any(-1)
        assert changed[1].sum() == 6 - len(skipped) and changed[0].sum() == 0


def test_captured_and_replayed_with_new_lengths(cuda):
    """A padded graph: the lengths change between replays."""
    import torch

    b = make_pool(cuda, "bf16", 2, 64)
    q, k, v, tables, cs = batch(cuda, b, "bf16", 4, [4, 4, 4], [0, 30, 60], seed=2)
    table = torch.from_numpy(cs).to(cuda)
    d_t, d_c, d_n = ints(cuda, tables), ints(cuda, [0, 30, 60]), ints(cuda, [4, 4, 4])
    out = torch.full(q.shape, 5.0, device=cuda, dtype=q.dtype)
    slots = torch.full((12,), -9, device=cuda, dtype=torch.int64)
    cu = torch.zeros(4, device=cuda, dtype=torch.int32)
    call = lambda: b.rope_and_cache(d_t, d_c, d_n, 12, cu, q, k, v, table, 1, q_out=out, slots_out=slots)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for new, ctx in (([4, 4, 4], [0, 30, 60]), ([1, 0, 5], [7, 30, 55]), ([0, 0, 1], [0, 0, 31])):
        d_n.copy_(ints(cuda, new))
        d_c.copy_(ints(cuda, ctx))
        out.fill_(5.0)
        slots.fill_(-9)
        before = values(b)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        assert b.device_error() is None and (out[n:] == 5.0).all() and (slots[n:] == -9).all()
        check_against_oracle(b, before, "bf16", q, out, k, None, v, cs, tables, ctx, new, 1, False,
                             slots.cpu().numpy())


def test_shard_holds_its_heads(cuda):
    import torch

    whole = make_pool(cuda, "fp8_e4m3", 4, 64, seed=1)
    part = make_pool(cuda, "fp8_e4m3", 4, 64, seed=1, shard=(1, 2))
    part.set_kv_scales(*whole.test_scales)
    part.test_scales = whole.test_scales
    q, k, v, tables, cs = batch(cuda, whole, "bf16", 8, NEW, CTX, seed=2, fused=False)
    table = torch.from_numpy(cs).to(cuda)
    args = (ints(cuda, tables), ints(cuda, CTX), ints(cuda, NEW), sum(NEW))
    cu = torch.zeros(len(NEW) + 1, device=cuda, dtype=torch.int32)
    slots = torch.zeros(sum(NEW), device=cuda, dtype=torch.int64)
    whole.rope_and_cache(*args, cu, q.clone(), k, v, table, 1, slots_out=slots)
    part.rope_and_cache(*args, cu, q[:, 4:].clone(), k[:, 2:], v[:, 2:], table, 1)
    torch.cuda.synchronize()
    s = slots.cpu().numpy()
    for x, y in zip(whole.planes(), part.planes()):
        x, y = (p.view(torch.uint8)[1, s // 16, s % 16].cpu().numpy() for p in (x, y))
        assert np.array_equal(x.reshape(len(s), 4, 64)[:, 2:], y.reshape(len(s), 2, 64))


def test_refusals(cuda):
    import torch
    from pagedkv.errors import CacheError, Device, InvalidLayer

    i = torch.zeros(2, device=cuda, dtype=torch.int32)
    t = torch.zeros((1, 4), device=cuda, dtype=torch.int32)

    def call(b, layer=0, dtype=torch.bfloat16, d=64, n=4, rotary=64, positions=9, kv=2):
        q, k = (torch.zeros((4, h, d), device=cuda, dtype=dtype) for h in (4, kv))
        b.rope_and_cache(t, i[:1], i[:1], n, i, q, k, k, torch.zeros((positions, rotary), device=cuda), layer)

    ok = make_pool(cuda, "bf16", 2, 64, num_blocks=4)
    call(ok)
    for make, kind in ((lambda: call(ok, layer=2), InvalidLayer), (lambda: call(ok, layer=-1), InvalidLayer),
                       (lambda: call(ok, dtype=torch.float16), Device), (lambda: call(ok, n=-1), ShapeMismatch),
                       (lambda: call(ok, rotary=66), ShapeMismatch), (lambda: call(ok, rotary=7), ShapeMismatch),
                       (lambda: call(ok, rotary=0), ShapeMismatch), (lambda: call(ok, positions=0), ShapeMismatch),
                       (lambda: call(make_pool(cuda, "bf16", 3, 64, num_blocks=4, shard=(0, 2)), kv=2), (CacheError, ValueError))):
        with pytest.raises((CacheError, ValueError)) as e:
            make()
        assert isinstance(e.value, kind), e.value
    torch.cuda.synchronize()
    assert ok.device_error() is None
    ok.rope_and_cache(t[:0], i[:0], i[:0], 0, i[:1], None, *(torch.zeros((0, 2, 64), device=cuda, dtype=torch.bfloat16),) * 2,
                      torch.zeros((9, 64), device=cuda), 0)
    torch.cuda.synchronize()
    assert ok.device_error() is None
