"""Helpers of the layer-step tests: pools, tables, ragged batches and the error
bounds that the comparisons with the float64 oracle use."""

import numpy as np

from pagedkv import B200Backend, CacheConfig

# Half a step of each type, relative to the value.
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24, "fp8_e4m3": 2.0 ** -4}


def torch_type(name):
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def make_pool(cuda, dtype, kv_heads=2, head_dim=128, layers=2, num_blocks=128, block_size=16, seed=0,
              shard=(0, 1), std=1.0):
    """(backend, K, V as the values they stand for in float64)."""
    import torch

    bytes_ = {"f32": 4, "fp8_e4m3": 1}.get(dtype, 2)
    cfg = CacheConfig(num_blocks, block_size, kv_heads, head_dim, layers, bytes_)
    b = B200Backend(cfg, dtype=dtype, shard_rank=shard[0], num_shards=shard[1])
    g = torch.Generator(device=cuda).manual_seed(seed)
    for p in b.planes():
        p.copy_((torch.randn(p.shape, generator=g, device=cuda) * std).to(p.dtype))
    if dtype == "fp8_e4m3":
        rng = np.random.default_rng(seed)
        scales = [rng.uniform(0.2, 0.5, (layers, kv_heads)).astype(np.float32) for _ in range(2)]
        b.set_kv_scales(*scales)
        b.test_scales = scales
    return b


def values(b):
    """The pool's planes as float64 values (codes times scales for fp8)."""
    d = b.config().head_dim
    out = []
    for i, p in enumerate(b.planes()):
        x = p.float().cpu().numpy().astype(np.float64)
        if p.element_size() == 1:
            sh = x.shape
            h0 = b.elem_offset // d
            s = b.test_scales[i][:, h0:h0 + sh[3] // d].astype(np.float64)
            x = (x.reshape(sh[:3] + (-1, d)) * s[:, None, None, :, None]).reshape(sh)
        out.append(x)
    return out


def tables_for(rng, num_blocks, totals, block_size=16, extra=1):
    need = [-(-int(n) // block_size) for n in totals]
    perm = rng.permutation(num_blocks)
    assert sum(need) <= num_blocks
    t = np.full((len(totals), max(need + [1]) + extra), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = perm[at:at + n]
        at += n
    return t


def ints(cuda, x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(cuda)


def cu_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def attention_bounds(q, kk, vv, want, mean_abs, dtype, scale, lengths):
    """Per-element bound of |out - want| and a bound of |lse - want|.

    q . k over D exact products accumulated in f32, each step off by at most
    2^-22 (a truncating adder) of the partial sums, which sum |q_d k_d| <=
    |q| |k| bounds: a score is off by e_s = scale * D * 2^-22 * max|q| max|k|
    (2-norms). A weight is then off by the factor exp(2 e_s) (its own score and
    the sum's), by 2^-18 for 2^x and the sums, and by half a step where it is
    rounded for the product with V; the output by half a step once more. f16
    weights below 2^-14 are off by 2^-25 of the largest weight each. mean_abs
    is the softmax mean of |v|."""
    u = HALF[dtype]
    d = q.shape[-1]
    qn = np.sqrt((np.asarray(q, np.float64) ** 2).sum(-1)).max(initial=0)
    kn = np.sqrt((np.asarray(kk, np.float64) ** 2).sum(-1)).max(initial=0)
    e_s = scale * d * 2.0 ** -22 * qn * kn
    rel = u + 2 * e_s + 2.0 ** -18
    tol = u * np.abs(want) + rel * (1 + u) * mean_abs
    if dtype == "f16":
        # Weights below 2^-14 of the largest, and outputs below 2^-14.
        tol = tol + max(lengths, default=0) * 2.0 ** -25 * np.abs(vv).max(initial=0) + 2.0 ** -25
    return tol, e_s + 2.0 ** -18 + max(lengths, default=0) * 2.0 ** -24
