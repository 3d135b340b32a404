"""rope_and_cache and paged_attention_chunk in a pool whose offsets pass 32 bits
(elements for 16-bit types, bytes for fp8): the same bits as in a small pool
that holds the same blocks at its beginning."""

import numpy as np
import pytest

from pagedkv import B200Backend, CacheConfig, rope_table
from tests.layer_step import cu_of, ints, tables_for, torch_type

pytestmark = pytest.mark.gpu

SMALL = 256


@pytest.mark.parametrize("pool,qdtype,far", [("bf16", "bf16", 280_000), ("f16", "f16", 280_000),
                                             ("fp8_e4m3", "bf16", 540_000)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_far_blocks_give_the_same_bits(cuda, pool, qdtype, far, d):
    import torch

    hkv, group = 256 // d, 3
    new, ctx = [130, 1, 0, 40], [700, 300, 5, 0]
    total = np.add(new, ctx)
    n = int(total.sum())
    tables = tables_for(np.random.default_rng(d), SMALL, total)
    g = torch.Generator(device=cuda).manual_seed(d)
    rows = torch.randn((n, hkv * (group + 2), d), generator=g, device=cuda).to(torch_type(qdtype))
    q, k, v = rows.split([hkv * group, hkv, hkv], 1)
    table = torch.from_numpy(rope_table(1024, d)).to(cuda)
    chunk_q = q[:sum(new)]
    got = []
    for blocks in (far, SMALL):
        first = blocks - SMALL
        b = B200Backend(CacheConfig(blocks, 16, hkv, d, 2, 1 if pool == "fp8_e4m3" else 2), dtype=pool)
        if pool == "fp8_e4m3":
            b.set_kv_scales(np.full((2, hkv), 0.02, np.float32), np.full((2, hkv), 0.03, np.float32))
        t = ints(cuda, np.where(tables < 0, -1, tables + first))
        cu, slots = ints(cuda, cu_of(total)), torch.zeros(n, device=cuda, dtype=torch.int64)
        b.rope_and_cache(t, ints(cuda, [0] * 4), ints(cuda, total), n, cu, q, k, v, table, 1,
                         q_out=torch.empty_like(q).contiguous(), slots_out=slots)
        outs = [slots - first * 16]
        for lens, before in ((new, ctx), ([1, 1, 0, 1], total - 1)):
            m = sum(lens)
            out, lse = torch.zeros_like(chunk_q[:m]).contiguous(), torch.zeros((m, hkv * group), device=cuda)
            b.paged_attention_chunk(chunk_q[:m], ints(cuda, cu_of(lens)), t, ints(cuda, np.maximum(before, 0)),
                                    max(lens), int(total.max()), out, 1, lse=lse)
            outs += [out, lse]
        assert b.device_error() is None
        for p in b.planes():
            assert p.numel() * p.element_size() > 2 ** 32 or blocks == SMALL
            whole = p.view(torch.uint8)
            outs.append(whole[1, first:].clone())
            assert not whole[0].reshape(-1).view(torch.int64).any()
            assert not whole[1, :first].reshape(-1).view(torch.int64).any()
        got.append(outs)
        b.close()
    assert got[0][1].float().abs().max() > 0
    for x, y in zip(*got):
        assert torch.equal(x, y)
