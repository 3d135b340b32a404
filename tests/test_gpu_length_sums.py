"""New-token lengths whose sum passes 32 bits: refused (ShapeMismatch) like any
other sum that does not fit the rows, by every call that scans new_lens."""

import numpy as np
import pytest

from pagedkv.errors import ShapeMismatch
from tests.layer_step import ints, make_pool, tables_for, values
from tests.test_gpu_rope_cache import batch

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1
# Sums modulo 2^32: the rows' count where a 32-bit sum would wrap to it, below
# zero, and the largest that 32 bits hold.
LENGTHS = [[TOP, TOP, 8], [2 ** 30] * 4 + [6], [2 ** 23] * 512 + [6], [6] + [2 ** 31 - 4096] * 2 + [8192],
           [TOP, 1, 0], [TOP] * 3, [TOP, 0, 0], [5, TOP - 5, 0]]


def refused(b):
    err = b.device_error()
    return err is not None and isinstance(err[0], ShapeMismatch)


@pytest.mark.parametrize("new", LENGTHS, ids=lambda x: f"{len(x)}x{x[0]}")
@pytest.mark.parametrize("d", [64, 40])
def test_rope_and_cache(cuda, new, d):
    """Both forms of the kernel (40: heads that are no whole 16s)."""
    import torch

    b = make_pool(cuda, "bf16", 1, d)
    q, k, v, tables, cs = batch(cuda, b, "bf16", 2, [3, 3], [0, 0], seed=2)
    tables = np.repeat(tables[:1], len(new), 0)
    before, q0 = values(b), q.clone()
    cu = torch.zeros(len(new) + 1, device=cuda, dtype=torch.int32)
    slots = torch.full((6,), -9, device=cuda, dtype=torch.int64)
    b.rope_and_cache(ints(cuda, tables), ints(cuda, [0] * len(new)), ints(cuda, new), 6, cu, q, k, v,
                     torch.from_numpy(cs).to(cuda), 0, slots_out=slots)
    torch.cuda.synchronize()
    assert refused(b)
    assert torch.equal(q, q0) and (slots == -9).all()
    assert all(np.array_equal(x, y) for x, y in zip(values(b), before))


@pytest.mark.parametrize("new", LENGTHS, ids=lambda x: f"{len(x)}x{x[0]}")
@pytest.mark.parametrize("pool", ["bf16", "fp8_e4m3"])
def test_resolve(cuda, new, pool):
    import torch

    b = make_pool(cuda, pool, 1, 64)
    tables = ints(cuda, np.repeat(tables_for(np.random.default_rng(7), 128, [64]), len(new), 0))
    ctx, lens = ints(cuda, [0] * len(new)), ints(cuda, new)
    rows = torch.ones((6, 64), device=cuda, dtype=torch.bfloat16)
    before = values(b)
    for fused in (False, True):
        cu = torch.zeros(len(new) + 1, device=cuda, dtype=torch.int32)
        slots = torch.full((6,), -9, device=cuda, dtype=torch.int64)
        if fused:
            b.resolve_and_cache(tables, ctx, lens, 6, cu, rows, rows, layer=1, slots_out=slots)
        else:
            b.resolve_slots(tables, ctx, lens, 6, cu, slots)
        torch.cuda.synchronize()
        assert refused(b)
        assert (slots == -9).all() and all(np.array_equal(x, y) for x, y in zip(values(b), before))


def test_the_largest_lengths_that_fit_are_taken(cuda):
    """Many sequences, empty ones among them, up to the rows that there are."""
    import torch

    rng = np.random.default_rng(5)
    for count in (1, 31, 256, 257, 3000):
        new = rng.choice([0, 1, 2], count)
        new[0] = 2
        t = int(new.sum())
        b = make_pool(cuda, "bf16", 1, 64, num_blocks=count, layers=1)
        tables = np.arange(count, dtype=np.int32)[:, None].copy()
        k = torch.randn((t, 1, 64), device=cuda).to(torch.bfloat16)
        cu = torch.zeros(count + 1, device=cuda, dtype=torch.int32)
        slots = torch.full((t,), -9, device=cuda, dtype=torch.int64)
        b.resolve_and_cache(ints(cuda, tables), ints(cuda, [3] * count), ints(cuda, new), t, cu, k[:, 0], k[:, 0],
                            layer=0, slots_out=slots)
        torch.cuda.synchronize()
        assert b.device_error() is None
        want = np.concatenate([[0], np.cumsum(new)])
        assert np.array_equal(cu.cpu().numpy(), want)
        seq = np.repeat(np.arange(count), new)
        assert np.array_equal(slots.cpu().numpy(), seq * 16 + 3 + np.arange(t) - want[seq])
