"""Refusals of rope_and_cache, paged_attention_chunk and prompt_attention that
the Python binding makes before any library call, the angle table, and the
oracle of the layer step against plain loops. No GPU."""

import numpy as np
import pytest
import torch

from oracle import layer_step as ref
from pagedkv import B200Backend, CacheConfig, rope_table


def hollow(heads=2, d=64):
    b = object.__new__(B200Backend)
    b._cfg = CacheConfig(8, 16, heads, d, 2, 2)
    b.shard_entry_elems = heads * d
    return b


def rows(t, h, d=64, dtype=torch.bfloat16):
    return torch.zeros((t, h, d), dtype=dtype)


@pytest.mark.parametrize("change", [
    dict(k=rows(4, 3)), dict(v=rows(4, 2, dtype=torch.float16)), dict(k=rows(4, 2, 32), v=rows(4, 2, 32)),
    dict(q=rows(4, 4, dtype=torch.float32)), dict(q=rows(3, 4)), dict(q_out=rows(4, 5)), dict(k_out=rows(5, 2)),
    dict(cos_sin=torch.zeros(64)), dict(cos_sin=torch.zeros((9, 64), dtype=torch.float64)),
    dict(cos_sin=torch.zeros((9, 128))[:, ::2]), dict(q=None, q_out=rows(4, 4)), dict(q=rows(4, 64, 4).transpose(1, 2))])
def test_rope_and_cache_refuses(change):
    a = dict(q=rows(4, 4), k=rows(4, 2), v=rows(4, 2), cos_sin=torch.zeros((9, 64)), q_out=None, k_out=None)
    a.update(change)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        hollow().rope_and_cache(i[None], i, i, 4, i, a["q"], a["k"], a["v"], a["cos_sin"], 0, q_out=a["q_out"],
                                k_out=a["k_out"])


@pytest.mark.parametrize("q,out", [
    (rows(4, 4), rows(4, 4, dtype=torch.float32)), (rows(4, 4), rows(4, 3)), (rows(4, 4), rows(8, 4)[::2]),
    (rows(4, 64, 4).transpose(1, 2), rows(4, 4)), (rows(4, 4)[0], rows(4, 4)[0])])
def test_attentions_refuse_rows(q, out):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        hollow().paged_attention_chunk(q, i, i[None], i[:1], 4, 4, out, 0)
    with pytest.raises(ValueError):
        hollow().prompt_attention(q, rows(4, 2), rows(4, 2), i, 4, out)


@pytest.mark.parametrize("k,v", [(rows(3, 2), rows(3, 2)), (rows(4, 1), rows(4, 1)), (rows(4, 2, 32), rows(4, 2, 32)),
                                 (rows(4, 2, dtype=torch.float16),) * 2, (rows(4, 2), rows(4, 3))])
def test_prompt_attention_refuses_keys(k, v):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        hollow().prompt_attention(rows(4, 4), k, v, i, 4, rows(4, 4))


def ints(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("what,bad", [
    ("tables", ints(2, 3, dtype=torch.int64)), ("tables", ints(1, 3)), ("tables", ints(2, 6)[:, ::2]),
    ("tables", ints(2, 6)[:, :3]), ("ctx", ints(2, dtype=torch.int64)), ("ctx", ints(4)[::2]), ("new", ints(1)),
    ("new", ints(2, dtype=torch.int64)), ("cu", ints(2)), ("cu", ints(3, dtype=torch.int64)), ("slots", ints(4)),
    ("slots", ints(3, dtype=torch.int64)), ("lse", torch.zeros(4, 3)), ("lse", torch.zeros(4, 4, dtype=torch.float64)),
    ("lse", torch.zeros(4, 8)[:, ::2])])
def test_lengths_tables_and_side_outputs_are_refused(what, bad):
    """Types, sizes and strides that the kernels would read or write wrongly.
    (With none of them wrong the tensors' device is refused: they are the CPU's.)"""
    a = dict(tables=ints(2, 3), ctx=ints(2), new=ints(2), cu=ints(3), slots=ints(4, dtype=torch.int64),
             lse=torch.zeros(4, 4))
    b = hollow()
    b.device = 0

    def rope(a):
        b.rope_and_cache(a["tables"], a["ctx"], a["new"], 4, a["cu"], rows(4, 4), rows(4, 2), rows(4, 2),
                         torch.zeros((9, 64)), 0, slots_out=a["slots"])

    def chunk(a):
        b.paged_attention_chunk(rows(4, 4), a["cu"], a["tables"], a["ctx"], 4, 4, rows(4, 4), 0, lse=a["lse"])

    def prompt(a):
        b.prompt_attention(rows(4, 4), rows(4, 2), rows(4, 2), a["cu"], 4, rows(4, 4), lse=a["lse"])

    takes = {rope: ("tables", "ctx", "new", "cu", "slots"), chunk: ("tables", "ctx", "cu", "lse"), prompt: ("cu", "lse")}
    for call, names in takes.items():
        with pytest.raises(ValueError, match="device"):
            call(a)
        if what in names and not (call is prompt and bad.dtype is torch.int32):  # its cu gives the count
            with pytest.raises(ValueError, match="dense"):
                call(dict(a, **{what: bad}))


def test_chunk_refuses_another_head_dim():
    """Rows of another head size at a pitch that would cover this backend's."""
    wide = rows(4, 8, 64)[:, :2]
    with pytest.raises(ValueError, match="head_dim"):
        hollow(d=128).paged_attention_chunk(wide, ints(2), ints(1, 1), ints(1), 4, 4, rows(4, 2), 0)


def test_rows_that_lie_over_one_another_are_refused():
    """Expanded rows (pitch 0), or rows at less than their own length."""
    one, i = rows(1, 4), ints(2)
    b = hollow(heads=4)
    for r in (one.expand(4, 4, 64), torch.zeros(600, dtype=torch.bfloat16).as_strided((4, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            b.paged_attention_chunk(r, i, ints(1, 1), ints(1), 4, 4, rows(4, 4), 0)
        with pytest.raises(ValueError, match="overlap"):
            b.prompt_attention(rows(4, 4), r, r, i, 4, rows(4, 4))
        for name in ("q", "k", "q_out", "k_out"):
            a = dict(dict(q=rows(4, 4), k=rows(4, 4), q_out=rows(4, 4), k_out=rows(4, 4)), **{name: r})
            with pytest.raises(ValueError, match="overlap"):
                b.rope_and_cache(ints(1, 1), ints(1), ints(1), 4, i, a["q"], a["k"], r if name == "k" else rows(4, 4),
                                 torch.zeros((9, 64)), 0, q_out=a["q_out"], k_out=a["k_out"])


def test_rope_table():
    t = rope_table(100001, 64, base=1e6)
    assert t.dtype == np.float32 and t.shape == (100001, 64)
    j = np.arange(32)
    angle = 100000 * 1e6 ** (-2 * j / 64)
    assert np.abs(t[100000, :32] - np.cos(angle)).max() < 2 ** -24 + 1e-9
    assert np.abs(t[100000, 32:] - np.sin(angle)).max() < 2 ** -24 + 1e-9
    assert np.array_equal(rope_table(8, 4, inv_freq=[1.0, 0.5])[3], np.float32(
        [np.cos(3.0), np.cos(1.5), np.sin(3.0), np.sin(1.5)]))
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(inv_freq=[1.0]), dict(max_position=0)):
        with pytest.raises(ValueError):
            rope_table(**{"max_position": 4, "rotary_dim": 4, **bad})


def test_oracle_rotation_is_a_complex_product():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(5, 3, 8))
    cs = rope_table(50, 6)
    pos = np.array([0, 1, 7, 49, 3])
    for inter in (False, True):
        y = ref.rotate(x, cs, pos, 6, inter)
        for t in range(5):
            for j in range(3):
                a, b = (2 * j, 2 * j + 1) if inter else (j, j + 3)
                z = (x[t, :, a] + 1j * x[t, :, b]) * complex(cs[pos[t], j], cs[pos[t], 3 + j])
                assert np.allclose(y[t, :, a], z.real) and np.allclose(y[t, :, b], z.imag)
        assert np.array_equal(y[:, :, 6:], x[:, :, 6:])


def test_oracle_chunks_agree_with_the_whole():
    """A prompt's rows in chunks over pages give the prompt's outputs, and the
    framework's decode oracle gives the last row."""
    from oracle.attention import paged_attention

    rng = np.random.default_rng(1)
    q, k, v = rng.normal(size=(50, 4, 8)), rng.normal(size=(50, 2, 8)), rng.normal(size=(50, 2, 8))
    want, lse = ref.prompt_attention(q, k, v, [50], 0.3)
    planes = np.zeros((2, 1, 4, 16, 16))
    table = np.array([[2, 0, 3, 1]], np.int32)
    for j in range(50):
        planes[0, 0, table[0, j // 16], j % 16] = k[j].ravel()
        planes[1, 0, table[0, j // 16], j % 16] = v[j].ravel()
    for c, n in ((0, 20), (20, 1), (21, 29)):
        o, l = ref.chunk_attention(planes[0], planes[1], 0, q[c:c + n], table, [c], [n], 0.3, 8)
        assert np.allclose(o, want[c:c + n]) and np.allclose(l, lse[c:c + n])
    o, l = paged_attention(planes[0], planes[1], 0, q[49:], table, [50], 0.3, 8)
    assert np.allclose(o[0], want[49]) and np.allclose(l[0], lse[49])
