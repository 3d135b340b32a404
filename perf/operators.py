"""Cases for the step of a model's layer around the paged cache: the new
tokens' queries and keys rotated and appended (rope_and_cache), attention of a
chunk of new tokens over the cache (paged_attention_chunk), and attention over
whole packed prompts before they are cached (prompt_attention).

Every case is one layer's call. Lengths are part of a case (texts of
comma-separated numbers), values come from the seed. The pool holds two
layers and the call works on the second, with block ids in random order.
"""

import math
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LAYERS, LAYER = 2, 1
BLOCK = 16
ROPE_BASE = 1.0e6
# Head layouts (query heads, kv heads, head_dim): 28/4 x 128 is the benchmark's
# model geometry, 32/8 x 64 that of CacheConfig.llama_3_2_1b, 64/8 x 128 the
# large pool of the churn trace; 12/12, 6/2 and 16/1 are one query head per kv
# head, an odd group and a single shared kv head; 256 is the widest head.
LAYOUTS = [(28, 4, 128), (32, 8, 64), (64, 8, 128), (12, 12, 64), (6, 2, 128), (16, 1, 128),
           (8, 4, 256)]


def _text(lens):
    return ",".join(str(int(x)) for x in lens)


def _nums(text):
    return [int(x) for x in text.split(",")]


# ---- cases -----------------------------------------------------------------------


def _append(name, new, ctx, layout, src="bf16", pool="bf16", rotary=None, interleaved=False,
            fused=True):
    hq, hkv, d = layout
    c = {"op": "append", "new": _text(new), "ctx": _text(ctx), "hq": hq, "hkv": hkv, "d": d,
         "src": src, "pool": pool, "rotary": rotary or d, "interleaved": interleaved,
         "fused_rows": fused}
    return dict(c, name=name) if name else c


def _chunk(name, new, ctx, layout, q="bf16", pool="bf16"):
    hq, hkv, d = layout
    c = {"op": "chunk", "new": _text(new), "ctx": _text(ctx), "hq": hq, "hkv": hkv, "d": d,
         "src": q, "pool": pool}
    return dict(c, name=name) if name else c


def _prompt(name, new, layout, dtype="bf16", fused=True):
    hq, hkv, d = layout
    c = {"op": "prompt", "new": _text(new), "hq": hq, "hkv": hkv, "d": d, "src": dtype,
         "fused_rows": fused}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decode step's append: a token of each running sequence.
        _append("append_decode", [1] * 48, [(37 + 611 * i) % 9000 for i in range(48)], (28, 4, 128)),
        # A mixed step: prompt chunks of all lengths, rows taken out of the
        # fused projection's output.
        _append("append_mixed", [1, 130, 977, 1, 0, 2048, 333, 17, 1, 511, 76, 1],
                [4095, 0, 512, 77, 9, 0, 16384, 31, 1000, 3, 0, 123], (28, 4, 128)),
        # A full prefill budget quantised into an fp8 pool, paired channels.
        _append("append_fp8_budget", [8192, 4096, 5001, 3000, 7777, 2702], [0, 8192, 0, 100, 20000, 3],
                (64, 8, 128), pool="fp8", interleaved=True),
        # Speculative drafts and short last chunks over medium contexts.
        _chunk("chunk_drafts", [5, 1, 8, 3, 24, 2, 13, 1, 6, 40, 4, 9],
               [900, 4000, 77, 1333, 0, 2500, 310, 3777, 15, 600, 1800, 3001], (28, 4, 128)),
        # Single tokens over long contexts, each cache page read once.
        _chunk("chunk_single_tokens", [1] * 16, [1023 + 977 * i for i in range(16)], (32, 8, 64), "f16", "f16"),
        # A scheduler step: one prefill chunk beside decoding sequences.
        _chunk("chunk_mixed_step", [512] + [1] * 15 + [200], [6144] + [256 + 401 * i for i in range(15)] + [0],
               (64, 8, 128)),
        # The late chunk of a long document.
        _chunk("chunk_long", [2048], [30720], (28, 4, 128)),
        # Chunks over an fp8 cache.
        _chunk("chunk_fp8", [256, 1024, 77, 300], [8000, 4096, 12001, 0], (32, 8, 128), "bf16", "fp8"),
        # Short prompts, where latency counts.
        _prompt("prompt_short", [17, 64, 101, 5], (32, 8, 64), "f16"),
        # A packed batch of ragged prompts.
        _prompt("prompt_packed", [2048, 333, 1024, 77, 1500, 640, 2000, 129, 1, 440], (28, 4, 128)),
        # The widest head.
        _prompt("prompt_wide_head", [1900, 700, 1200], (8, 4, 256), "bf16", fused=False),
        # One long prompt.
        _prompt("prompt_long", [8192], (28, 4, 128)),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


MOST_SCORES = 28 * 2048 * 32768  # padded scores of the largest listed cases
MOST_FLOPS = 4 * 128 * 28 * (2048 * 30720 + 2048 * 2049 // 2)


def _draw_append(rng):
    seqs = _log_int(rng, 1, 192)
    total = _log_int(rng, seqs, 16384)
    cuts = sorted(rng.randint(0, total) for _ in range(seqs - 1))
    new = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    ctx = [rng.choice([0, rng.randint(1, 40), _log_int(rng, 1, 30000)]) for _ in new]
    layout = rng.choice(LAYOUTS)
    src, pool = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "fp8"), ("f16", "fp8")])
    return _append(None, new, ctx, layout, src, pool, rotary=rng.choice([layout[2], layout[2] // 2]),
                   interleaved=rng.random() < 0.4, fused=rng.random() < 0.7)


def _draw_chunk(rng):
    while True:
        seqs = _log_int(rng, 1, 40)
        top = _log_int(rng, 1, 2048)
        new = [rng.choice([1, rng.randint(0, top), top]) for _ in range(seqs)]
        ctx = [rng.choice([0, rng.randint(1, 300), _log_int(rng, 1, 32000)]) for _ in new]
        layout = rng.choice(LAYOUTS)
        hq, _, d = layout
        n, length = max(new), max(c + m for c, m in zip(ctx, new))
        pairs = sum(m * c + m * (m + 1) // 2 for m, c in zip(new, ctx))
        if (0 < sum(new) and seqs * hq * n * length <= MOST_SCORES and 4 * d * hq * pairs <= MOST_FLOPS
                and seqs * length <= 400_000):
            break
    q, pool = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("f16", "fp8")])
    return _chunk(None, new, ctx, layout, q, pool)


def _draw_prompt(rng):
    while True:
        seqs = _log_int(rng, 1, 24)
        top = _log_int(rng, 1, 8192)
        new = [rng.choice([rng.randint(0, top), _log_int(rng, 1, top), top]) for _ in range(seqs)]
        layout = rng.choice(LAYOUTS)
        hq, _, d = layout
        pairs = sum(m * (m + 1) // 2 for m in new)
        if (0 < sum(new) and seqs * hq * max(new) ** 2 <= MOST_SCORES and 4 * d * hq * pairs <= MOST_FLOPS):
            break
    return _prompt(None, new, layout, rng.choice(["bf16", "f16"]), fused=rng.random() < 0.7)


def draw(rng):
    return rng.choice([_draw_append, _draw_chunk, _draw_prompt])(rng)


# ---- inputs ----------------------------------------------------------------------


def _normal(gen, shape, std=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(std)


def _key_like(gen, rows, heads, d):
    """Keys as projections give them: a few channels with a large constant part."""
    x = _normal(gen, (rows, heads, d))
    bias = _normal(gen, (heads, d), 0.3)
    bias[:, :: max(1, d // 4)] *= 6.0
    return x.add_(bias)


def _rope_table(positions, rotary):
    """[positions][rotary]: cos of each pair's angle, then sin; angles in 64 bits."""
    inv = ROPE_BASE ** (-torch.arange(0, rotary, 2, device=DEV, dtype=torch.float64) / rotary)
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, device=DEV, dtype=dtype)


def _backend(case, planes, scales, num_blocks):
    """The framework's pool with these contents."""
    if "paged-kv-cache_b200" not in sys.path:
        sys.path.insert(0, "paged-kv-cache_b200")
    from pagedkv import B200Backend, CacheConfig

    dtype = {"fp8": "fp8_e4m3"}.get(case["pool"], case["pool"])
    cfg = CacheConfig(num_blocks, BLOCK, case["hkv"], case["d"], LAYERS,
                      {"fp8_e4m3": 1, "f32": 4}.get(dtype, 2))
    b = B200Backend(cfg, dtype=dtype, device=torch.cuda.current_device())
    if case["pool"] == "fp8":
        b.set_kv_scales(scales[0].cpu().numpy(), scales[1].cpu().numpy())
    views = b.planes()
    for to, x in zip(views, planes):
        to.view(torch.uint8).copy_(x.view(torch.uint8))
    b.attention_reserve()
    return b, views


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new = _nums(case["new"])
    ctx = _nums(case["ctx"]) if "ctx" in case else [0] * len(new)
    t, lens = sum(new), [c + n for c, n in zip(ctx, new)]
    src = TYPES[case["src"]]
    st = {"case": case, "tokens": t, "max_new": max(new), "max_len": max(lens),
          "ctx": _ints(ctx), "new": _ints(new),
          "cu": _ints(np.concatenate([[0], np.cumsum(new)]))}
    # The new tokens' rows: columns of the fused projection's output, or dense.
    if case["op"] != "chunk" and case["fused_rows"]:
        rows = torch.empty((t, (hq + 2 * hkv) * d), device=DEV, dtype=src)
        q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split([hq * d, hkv * d, hkv * d], 1))
    else:
        q, k, v = (torch.empty((t, h, d), device=DEV, dtype=src) for h in (hq, hkv, hkv))
    q.copy_(_normal(gen, (t, hq, d), 1.2))
    k.copy_(_key_like(gen, t, hkv, d))
    v.copy_(_normal(gen, (t, hkv, d), 0.8))
    st.update(q=q, k=k, v=v, out=torch.empty((t, hq, d), device=DEV, dtype=src))
    if case["op"] == "prompt":
        if own:
            # The handle that the program keeps: its geometry and workspace serve the call.
            zero = [torch.zeros((LAYERS, 1, BLOCK, hkv * d), device=DEV, dtype=src) for _ in range(2)]
            st["b"], _ = _backend(dict(case, pool=case["src"]), zero, None, 1)
        return st
    # The pool: every sequence's blocks in random order, a few more that stay free.
    need = [-(-n // BLOCK) for n in lens]
    num_blocks = sum(need) + 7
    perm = torch.randperm(num_blocks, generator=gen, device=DEV).int()
    tables = torch.full((len(new), max(need) + 1), -1, device=DEV, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = perm[at:at + n]
        at += n
    slots = num_blocks * BLOCK
    scales = None
    planes = []
    for i in range(2):
        x = _key_like(gen, LAYERS * slots, hkv, d) if i == 0 else _normal(gen, (LAYERS * slots, hkv, d), 0.8)
        if case["pool"] == "fp8":
            scales = scales or (torch.empty((LAYERS, hkv), device=DEV).uniform_(0.02, 0.05, generator=gen),
                                torch.empty((LAYERS, hkv), device=DEV).uniform_(0.01, 0.03, generator=gen))
            x = (x.view(LAYERS, slots, hkv, d) / scales[i][:, None, :, None]).clamp(-448, 448)
            x = x.to(torch.float8_e4m3fn)
        else:
            x = x.to(TYPES[case["pool"]])
        planes.append(x.reshape(LAYERS, num_blocks, BLOCK, hkv * d))
    st.update(tables=tables, scales=scales, k_plane=planes[0], v_plane=planes[1])
    if case["op"] == "append":
        st.update(table=_rope_table(st["max_len"] + 64, case["rotary"]),
                  cu_out=torch.zeros(len(new) + 1, device=DEV, dtype=torch.int32),
                  slots=torch.zeros(t, device=DEV, dtype=torch.int64))
    if own:
        st["b"], (st["k_plane"], st["v_plane"]) = _backend(case, planes, scales, num_blocks)
    return st


# ---- the plain forms ---------------------------------------------------------------


def _rows_of(st):
    """(sequence, index within its new tokens) of every packed row."""
    seqs = torch.repeat_interleave(torch.arange(st["new"].numel(), device=DEV), st["new"].long(),
                                   output_size=st["tokens"])
    return seqs, torch.arange(st["tokens"], device=DEV) - st["cu"].long()[seqs]


def _rotate(x, cs, rotary, interleaved):
    """x [T][H][D] f32 (or f64); cs [T][rotary] cos then sin."""
    c, s = cs[:, None, :rotary // 2], cs[:, None, rotary // 2:]
    r = x[..., :rotary]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., rotary:]], -1)


def _plain_append(st):
    case = st["case"]
    seqs, i = _rows_of(st)
    pos = st["ctx"].long()[seqs] + i
    blk = st["tables"].long()[seqs, pos // BLOCK]
    cs = st["table"][pos]
    q = _rotate(st["q"].float(), cs, case["rotary"], case["interleaved"]).to(st["q"].dtype)
    k = _rotate(st["k"].float(), cs, case["rotary"], case["interleaved"])
    k_rows = k.to(st["k"].dtype)
    for plane, x, j in ((st["k_plane"], k, 0), (st["v_plane"], st["v"].float(), 1)):
        if case["pool"] == "fp8":
            x = (x * (1.0 / st["scales"][j][LAYER])[:, None]).clamp(-448, 448)
        bits = torch.uint8 if case["pool"] == "fp8" else plane.dtype
        plane[LAYER].view(bits)[blk, pos % BLOCK] = x.to(plane.dtype).flatten(1).view(bits)
    return {"q": q, "k": k_rows, "k_plane": st["k_plane"], "v_plane": st["v_plane"],
            "slots": blk * BLOCK + pos % BLOCK, "cu": st["cu"]}


def _attend(q, k, v, limit, rows, scale):
    """q [S][N][Hq][D], k and v [S][L][Hkv][D], limit [S][N]: the keys that a
    query attends. The packed rows' outputs, f32 (f64 for f64 inputs)."""
    s, n, hq, d = q.shape
    length, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    q = q.view(s, n, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(s, hkv, g * n, d)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)).view(s, hkv, g, n, length).mul_(scale)
    masked = torch.arange(length, device=DEV) >= limit[:, :, None]
    sc.masked_fill_(masked[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True).clamp_min(torch.finfo(sc.dtype).min)
    p = sc.sub_(m).exp_()
    total = p.sum(-1)
    o = torch.matmul(p.view(s, hkv, g * n, length), v.permute(0, 2, 1, 3)).view(s, hkv, g, n, d)
    o = o / total.clamp_min(torch.finfo(sc.dtype).tiny)[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(s, n, hq, d)
    return o[rows]


def _padded_queries(st, rows):
    q = torch.zeros((st["new"].numel(), st["max_new"]) + st["q"].shape[1:], device=DEV)
    q[rows] = st["q"].float()
    return q


def _limits(st):
    n = torch.arange(st["max_new"], device=DEV)
    return torch.where(n < st["new"][:, None], st["ctx"][:, None] + n + 1, 0)


def _plain_chunk(st):
    case = st["case"]
    rows = _rows_of(st)
    blocks = -(-st["max_len"] // BLOCK)
    at = st["tables"][:, :blocks].long().clamp_min(0)
    k, v = (p[LAYER][at].float().reshape(at.shape[0], blocks * BLOCK, case["hkv"], case["d"])
            for p in (st["k_plane"], st["v_plane"]))
    if case["pool"] == "fp8":
        k, v = k * st["scales"][0][LAYER][:, None], v * st["scales"][1][LAYER][:, None]
    o = _attend(_padded_queries(st, rows), k, v, _limits(st), rows, case["d"] ** -0.5)
    return o.to(st["q"].dtype)


def _plain_prompt(st):
    case = st["case"]
    rows = _rows_of(st)
    shape = (st["new"].numel(), st["max_new"], case["hkv"], case["d"])
    k, v = torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV)
    k[rows], v[rows] = st["k"].float(), st["v"].float()
    o = _attend(_padded_queries(st, rows), k, v, _limits(st), rows, case["d"] ** -0.5)
    return o.to(st["q"].dtype)


# ---- one pass ----------------------------------------------------------------------


def run(st):
    case = st["case"]
    if not own:
        return {"append": _plain_append, "chunk": _plain_chunk, "prompt": _plain_prompt}[case["op"]](st)
    b = st["b"]
    if case["op"] == "append":
        k_rows = torch.empty(st["k"].shape, device=DEV, dtype=st["k"].dtype)
        b.rope_and_cache(st["tables"], st["ctx"], st["new"], st["tokens"], st["cu_out"], st["q"],
                         st["k"], st["v"], st["table"], LAYER, q_out=st["out"], k_out=k_rows,
                         interleaved=case["interleaved"], slots_out=st["slots"])
        return {"q": st["out"], "k": k_rows, "k_plane": st["k_plane"], "v_plane": st["v_plane"],
                "slots": st["slots"], "cu": st["cu_out"]}
    if case["op"] == "chunk":
        b.paged_attention_chunk(st["q"], st["cu"], st["tables"], st["ctx"], st["max_new"],
                                st["max_len"], st["out"], LAYER)
    else:
        b.prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["max_new"], st["out"])
    return st["out"]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new = _nums(case["new"])
    t = sum(new)
    es = 4 if case["src"] == "f32" else 2
    if case["op"] == "append":
        pool = {"fp8": 1, "f32": 4}.get(case["pool"], 2)
        ctx = _nums(case["ctx"])
        positions = _union([(c, c + n) for c, n in zip(ctx, new) if n])
        pages = sum(-(-(c + n) // BLOCK) - c // BLOCK for c, n in zip(ctx, new) if n)
        # Queries in and out, K in, its rows out and its cache entries, V in and its entries, angles, slots.
        moved = t * (2 * hq * d * es + hkv * d * (3 * es + 2 * pool) + 8) + positions * case["rotary"] * 4
        return {"bytes": moved + 4 * (pages + 3 * len(new) + 1), "flops": t * (hq + hkv) * case["rotary"] * 3}
    if case["op"] == "chunk":
        ctx = _nums(case["ctx"])
        pool = 1 if case["pool"] == "fp8" else 2
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
        read = sum(c + n for n, c in zip(new, ctx) if n)
        return {"bytes": 2 * t * hq * d * es + read * 2 * hkv * d * pool + 4 * (read // BLOCK + 2 * len(new)),
                "flops": 4 * d * hq * pairs}
    pairs = sum(n * (n + 1) // 2 for n in new)
    return {"bytes": 2 * t * (hq + hkv) * d * es + 4 * len(new), "flops": 4 * d * hq * pairs}


def _union(spans):
    total, end = 0, -1
    for a, b in sorted(spans):
        total += max(0, b - max(a, end))
        end = max(end, b)
    return total


# ---- 64 bits, written from the definitions -------------------------------------------


def _as_written(x, pool, scale):
    """What the pool stands for before its rounding: x, or x / scale within fp8's range."""
    return x if pool != "fp8" else (x / scale.double()).clamp(-448.0, 448.0)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    new = _nums(case["new"])
    ctx = _nums(case["ctx"]) if "ctx" in case else [0] * len(new)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g = hq // hkv
    if case["op"] == "append":
        half, tab = case["rotary"] // 2, st["table"].double()
        q, k = st["q"].double().clone(), st["k"].double().clone()
        planes = [st["k_plane"].double(), st["v_plane"].double()]
        slots, row = [], 0
        for s, (n, c) in enumerate(zip(new, ctx)):
            z = torch.complex(tab[c:c + n, :half], tab[c:c + n, half:])[:, None]
            where = slice(row, row + n)
            for x in (q, k):
                lo = x[where, :, 0:2 * half:2] if case["interleaved"] else x[where, :, :half]
                hi = x[where, :, 1:2 * half:2] if case["interleaved"] else x[where, :, half:2 * half]
                y = torch.complex(lo.contiguous(), hi.contiguous()) * z
                lo.copy_(y.real)
                hi.copy_(y.imag)
            p = torch.arange(c, c + n, device=DEV)
            blk = st["tables"][s].long()[p // BLOCK]
            for i, x in enumerate((k, st["v"].double())):
                sc = None if case["pool"] != "fp8" else st["scales"][i][LAYER][:, None]
                planes[i][LAYER, blk, p % BLOCK] = _as_written(x[where], case["pool"], sc).flatten(1)
            slots.append(blk * BLOCK + p % BLOCK)
            row += n
        return {"q": q, "k": k, "k_plane": planes[0], "v_plane": planes[1], "slots": torch.cat(slots),
                "cu": st["cu"]}
    out = torch.zeros((sum(new), hq, d), device=DEV, dtype=torch.float64)
    row = 0
    for s, (n, c) in enumerate(zip(new, ctx)):
        if case["op"] == "chunk":
            p = torch.arange(c + n, device=DEV)
            blk = st["tables"][s].long()[p // BLOCK]
            k, v = (x[LAYER, blk, p % BLOCK].double().view(-1, hkv, d) for x in (st["k_plane"], st["v_plane"]))
            if case["pool"] == "fp8":
                k, v = (x * y[LAYER].double()[:, None] for x, y in zip((k, v), st["scales"]))
        else:
            k, v = st["k"][row:row + n].double(), st["v"][row:row + n].double()
        for h in range(hq):
            for a in range(0, n, 2048):
                b = min(n, a + 2048)
                x = st["q"][row + a:row + b, h].double() @ k[:c + b, h // g].T / math.sqrt(d)
                seen = torch.ones_like(x, dtype=torch.bool).tril(c + a)
                w = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[row + a:row + b, h] = w @ v[:c + b, h // g]
        row += n
    return out
