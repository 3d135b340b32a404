"""TEST INFRASTRUCTURE ONLY -- float64 restatement of a layer's step over
ragged new tokens: rotation by position, the slots the tokens take, and causal
attention over pool or packed rows. No counterpart in the reference, which
stops at the cache (crates/paged-kv-core/src/backend.rs:18-22)."""

from __future__ import annotations

import numpy as np


def positions(ctx, new):
    """(sequence, position) of every packed row."""
    seq = np.repeat(np.arange(len(new)), new)
    start = np.concatenate([[0], np.cumsum(new)[:-1]]).astype(np.int64)
    pos = np.asarray(ctx, np.int64)[seq] + np.arange(len(seq)) - start[seq]
    return seq, pos


def rotate(x, cos_sin, pos, rotary_dim: int, interleaved: bool):
    """x [T][H][D] rotated by rows `pos` of cos_sin ([P][rotary_dim]: cosines,
    then sines), in 64 bits."""
    y = np.array(x, dtype=np.float64)
    half = rotary_dim // 2
    cs = np.asarray(cos_sin, np.float64)[pos]
    c, s = cs[:, None, :half], cs[:, None, half:]
    ia, ib = ((np.arange(half) * 2, np.arange(half) * 2 + 1) if interleaved
              else (np.arange(half), np.arange(half) + half))
    a, b = y[:, :, ia].copy(), y[:, :, ib].copy()
    y[:, :, ia] = a * c - b * s
    y[:, :, ib] = b * c + a * s
    return y


def slots(tables, seq, pos, block_size: int):
    return np.asarray(tables)[seq, pos // block_size].astype(np.int64) * block_size + pos % block_size


def attend(q, k, v, limits, scale: float):
    """q [N][Hq][D]; k, v [L][Hkv][D]; row i attends keys 0 .. limits[i] - 1.
    (out [N][Hq][D], lse [N][Hq]) in 64 bits; no keys: zeros and -inf. Keys
    that a row does not attend do not enter its sums, whatever they hold."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, lse = np.zeros(q.shape), np.full((n, hq), -np.inf)
    for i in range(n):
        lim = int(limits[i])
        if lim <= 0:
            continue
        for h in range(hq):
            sc = k[:lim, h // group] @ q[i, h] * scale
            m = sc.max()
            p = np.exp(sc - m)
            out[i, h] = p @ v[:lim, h // group] / p.sum()
            lse[i, h] = m + np.log(p.sum())
    return out, lse


def chunk_attention(k_plane, v_plane, layer: int, q, tables, ctx, new, scale: float, head_dim: int,
                    keep=None):
    """Ragged rows q [T][Hq][D] over planes [L][num_blocks][block_size][entry].
    `keep`: bool [blocks] of ids whose keys count (others are skipped)."""
    k_plane, v_plane = np.asarray(k_plane), np.asarray(v_plane)
    bs, kvh = k_plane.shape[2], k_plane.shape[3] // head_dim
    outs, lses, row = [], [], 0
    for s, n in enumerate(new):
        total = int(ctx[s]) + int(n)
        t = np.arange(total)
        blk = np.asarray(tables[s])[t // bs]
        live = (blk >= 0) & (blk < k_plane.shape[1])
        if keep is not None:
            live &= keep[np.clip(blk, 0, len(keep) - 1)]
        t = t[live]
        kk, vv = (p[layer, blk[live], t % bs].reshape(-1, kvh, head_dim) for p in (k_plane, v_plane))
        limits = np.searchsorted(t, int(ctx[s]) + np.arange(n), side="right")
        o, l = attend(np.asarray(q)[row:row + n], kk, vv, limits, scale)
        outs.append(o)
        lses.append(l)
        row += n
    return np.concatenate(outs), np.concatenate(lses)


def prompt_attention(q, k, v, new, scale: float):
    outs, lses, row = [], [], 0
    for n in new:
        at = slice(row, row + n)
        o, l = attend(np.asarray(q)[at], np.asarray(k)[at], np.asarray(v)[at], np.arange(n) + 1, scale)
        outs.append(o)
        lses.append(l)
        row += n
    return np.concatenate(outs), np.concatenate(lses)
