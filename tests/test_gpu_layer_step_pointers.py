"""Addresses that the layer-step entry points refuse before any launch: ones
that are not aligned to their elements, and rows in place at another pitch."""

import pytest

from pagedkv.errors import Device, ShapeMismatch
from tests.layer_step import make_pool

pytestmark = pytest.mark.gpu


def names(text):
    return text.replace(",", " ").split()


ROPE = names("h, tables, table_stride, ctx, new, seqs, tokens, cu, slots, layer, q, q_stride, hq, q_out, qo_stride, "
             "k, v, kv_stride, k_out, ko_stride, src, cos_sin, positions, rotary, interleaved, stream")
CHUNK = names("h, layer, q, src, q_stride, hq, cu, seqs, tokens, max_new, tables, table_stride, ctx, max_len, scale, "
              "out, lse, stream")
PROMPT = names("h, q, k, v, src, q_stride, kv_stride, hq, cu, seqs, tokens, max_len, scale, out, lse, stream")


@pytest.fixture()
def call(cuda):
    """call(what, **changes): the status of one call of the C entry point; a
    change is a value, or a function of the address or number it replaces."""
    import torch
    from pagedkv import _lib

    b = make_pool(cuda, "bf16", 2, 64, num_blocks=4)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, device=cuda, dtype=dtype)  # noqa: E731
    i32 = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    new, cu = i32(1) + 2, i32(2)
    cu[1] = 2
    rows = dict(q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), q_out=z(3, 4, 64), k_out=z(3, 2, 64), out=z(3, 4, 64),
                lse=z(3, 4, dtype=torch.float32), tables=i32(1, 4), ctx=i32(1), new=new, cu=cu,
                slots=z(2, dtype=torch.int64), cos_sin=z(9, 64, dtype=torch.float32))
    base = dict({n: t.data_ptr() for n, t in rows.items()}, h=b._h, table_stride=4, seqs=1, tokens=2, layer=0,
                q_stride=0, hq=4, qo_stride=0, kv_stride=0, ko_stride=0, src=_lib.BF16, positions=9, rotary=64,
                interleaved=0, stream=None, max_new=2, max_len=8, scale=0.125)

    def run(what, **changes):
        a = dict(base)
        for n, c in changes.items():
            a[n] = c(a[n]) if callable(c) else c
        order, f = {"rope": (ROPE, _lib.lib.pkv_rope_and_cache_dev), "chunk": (CHUNK, _lib.lib.pkv_paged_attention_chunk_dev),
                    "prompt": (PROMPT, _lib.lib.pkv_prompt_attention_dev)}[what]
        rc = f(*(a[n] for n in order))
        torch.cuda.synchronize()
        assert b.device_error() is None
        return rc

    run.rows, run.base = rows, base
    return run


def test_addresses_as_given_are_taken(call):
    for what in ("rope", "chunk", "prompt"):
        assert call(what) == 0


@pytest.mark.parametrize("what,name,by", [
    *(("rope", n, 2) for n in names("tables, ctx, new, cu, cos_sin")), ("rope", "slots", 4),
    *(("rope", n, 1) for n in names("q, k, v, q_out, k_out")),
    *(("chunk", n, 2) for n in names("tables, ctx, cu, lse")), *(("chunk", n, 2) for n in names("q, out")),
    *(("prompt", n, 2) for n in names("cu, lse, q, k, v, out"))])
def test_addresses_between_elements_are_refused(call, what, name, by):
    assert call(what, **{name: lambda p: p + by}) == Device.code


def test_rows_in_place_keep_their_pitch(call):
    q, k = call.base["q"], call.base["k"]
    assert call("rope", q_out=q, k_out=k) == 0
    assert call("rope", q_out=q, qo_stride=264) == ShapeMismatch.code
    assert call("rope", k_out=k, ko_stride=136) == ShapeMismatch.code
    assert call("rope", q_out=q, qo_stride=264, tokens=1, new=call.base["ctx"]) == 0  # one row has no pitch
