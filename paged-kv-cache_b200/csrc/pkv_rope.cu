// pkv_rope.cu -- rope_and_cache: a layer's new queries and keys rotated by
// position, the keys and values appended to the paged pool. One launch in
// place of a rotation pass over q and k and a cache write.
//
// Token t of the packed rows is token i of sequence s, at position
// p = ctx[s] + i. For each rotated pair (a, b) of a q or k head, with
// c = cos_sin[p][j] and n = cos_sin[p][R / 2 + j]:
//   a' = a c - b n,   b' = b c + a n        (in f32, one rounding at the end)
// where pair j is elements (j, j + R/2) of the head, or (2j, 2j + 1) in the
// interleaved form; elements from R (the rotary dimension) on pass through.
// The slot is table[s][p / block_size] * block_size + p % block_size.
//
// Bounded by HBM: per token q is read and written, k and v are read and
// written to the pool (k also to k_out where asked); a position's angles are
// shared by every head. So a warp takes one token and a run of its heads: the
// angles are loaded once into registers, and the slot is resolved once.
// Within a head, lane item i holds 16 elements, the two 8-element vectors
// that its 8 pairs are made of, so every access is 16 bytes (8 codes for an
// fp8 pool) and a warp covers 32 / (D / 16) heads at a time.
//
// Measured (bf16 rows, heads of 128): 30,768 tokens of 64/8 heads into an fp8
// pool, 1.27 GB, 212 us, 0.92 of a device copy's rate; 4,096 tokens of 28/4
// heads, 81 MB, 15.3 us, 0.81 (the ramp of a launch); 48 single tokens 3.7 us,
// all of it a launch, the prefix scan and one chain of loads (lengths, table,
// angles and rows, stores). f32 rows and pool, 4,096 tokens of 28/4 heads, 161
// MB: 35.7 us, 0.69.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "pkv_device.cuh"
#include "pkv_internal.hpp"

namespace pkv {
namespace {

constexpr int kRopeWarps = kThreads / 32;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// Eight consecutive elements as f32.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(p));
        const float4 b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(p));
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = widen(e[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        __stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
        __stcs(reinterpret_cast<float4 *>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        uint4 w;
        T *e = reinterpret_cast<T *>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = narrow<T>(x[i]);
        __stcs(reinterpret_cast<uint4 *>(p), w);
    }
}

__device__ __forceinline__ void store8_codes(uint8_t *p, const float (&x)[8], float inv) {
    uint2 w;
    w.x = e4m3x2(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv)) |
          (e4m3x2(__fmul_rn(x[2], inv), __fmul_rn(x[3], inv)) << 16);
    w.y = e4m3x2(__fmul_rn(x[4], inv), __fmul_rn(x[5], inv)) |
          (e4m3x2(__fmul_rn(x[6], inv), __fmul_rn(x[7], inv)) << 16);
    __stcs(reinterpret_cast<uint2 *>(p), w);
}

// Where token t goes: its position (-1: the token is skipped) and its pool
// slot (-1: not cached). A sequence index found over a prefix that the
// lengths do not bear out (they changed under the call, or their sum passed
// 32 bits) skips the token too.
struct Place {
    long long pos, slot;
};

__device__ __forceinline__ Place place_of_token(const RopeCacheLaunch &a, const int *s_cu, long long t,
                                                bool report) {
    int lo = 0, hi = (int)a.num_seqs - 1;
    while (lo < hi) {  // last q with s_cu[q] <= t; that sequence has new_lens > 0
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const long long i = t - s_cu[lo];
    const long long ctx = __ldg(a.ctx_lens + lo);
    if (i < 0 || ctx < 0 || t >= s_cu[lo + 1]) return {-1, -1};
    const long long pos = ctx + i;
    if (pos >= a.max_position) {
        if (report) record_error(a.err, kShapeMismatch, t);
        return {-1, -1};
    }
    const long long lb = pos / a.block_size;
    if (lb >= a.table_stride) {
        if (report) record_error(a.err, kSlotOutOfRange, t);
        return {pos, -1};
    }
    const long long blk = __ldg(a.tables + (long long)lo * a.table_stride + lb);
    if (blk < 0 || blk >= a.num_blocks) {
        if (report) record_error(a.err, kInvalidBlock, t);
        return {pos, -1};
    }
    return {pos, blk * a.block_size + (pos - lb * a.block_size)};
}

// The prefix of new_lens in s_cu, published to cu_seqlens by the first CTA.
// The number of rows that hold tokens, or -1 when the lengths are refused: a
// negative one, a sum beyond 31 bits, or more tokens than rows.
__device__ __forceinline__ long long scan_tokens(const RopeCacheLaunch &a, int *s_cu, int *s_warp, int *s_bad) {
    scan_lengths(a.ctx_lens, a.new_lens, (int)a.num_seqs, s_cu, s_warp, s_bad);
    const long long total = s_cu[a.num_seqs];
    const bool refused = *s_bad || total > a.num_tokens;
    if (blockIdx.x == 0) {
        for (int q = threadIdx.x; q <= a.num_seqs; q += kThreads) a.cu_seqlens[q] = s_cu[q];
        if (threadIdx.x == 0 && refused) record_error(a.err, kShapeMismatch, *s_bad ? -1 : total);
    }
    return refused ? -1 : total;
}

// T: source type. FP8: the pool holds E4M3 codes (else it holds T). The
// heads of a token are its q heads, then its k heads, then its v heads.
template <typename T, bool FP8, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) rope_cache_kernel(const RopeCacheLaunch a) {
    using P = std::conditional_t<FP8, uint8_t, T>;
    extern __shared__ int s_cu[];
    __shared__ int s_warp[kThreads / 32];
    __shared__ int s_bad;
    pdl_wait();
    const long long tokens = scan_tokens(a, s_cu, s_warp, &s_bad);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int items = a.head_dim / 16, span = 32 / items;  // lane items per head; heads per step
    const int my_head = lane / items, item = lane - my_head * items;
    const bool in_step = my_head < span;
    const bool rotated = item < a.rotary_dim / 16;
    // First elements of the item's two vectors.
    int e0, e1;
    if (INTERLEAVED || !rotated) e0 = item * 16, e1 = e0 + 8;
    else e0 = item * 8, e1 = a.rotary_dim / 2 + item * 8;
    const int heads = a.num_q_heads + 2 * a.kv_heads;
    const long long units = tokens * a.head_splits;
    for (long long u = (long long)blockIdx.x * kRopeWarps + warp; u < units; u += (long long)gridDim.x * kRopeWarps) {
        const long long t = u / a.head_splits;
        const int part = (int)(u - t * a.head_splits);
        const Place at = place_of_token(a, s_cu, t, part == 0 && lane == 0);
        if (part == 0 && lane == 0 && a.slots_out) a.slots_out[t] = at.slot;
        if (at.pos < 0) continue;
        float c[8], n[8];  // pair j's angle: the item's 8 pairs
        if (rotated) {
            const float *row = a.cos_sin + at.pos * a.rotary_dim + item * 8;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 x = __ldg(reinterpret_cast<const float4 *>(row) + h);
                const float4 y = __ldg(reinterpret_cast<const float4 *>(row + a.rotary_dim / 2) + h);
                c[4 * h] = x.x, c[4 * h + 1] = x.y, c[4 * h + 2] = x.z, c[4 * h + 3] = x.w;
                n[4 * h] = y.x, n[4 * h + 1] = y.y, n[4 * h + 2] = y.z, n[4 * h + 3] = y.w;
            }
        }
        const int h0 = part * a.heads_per_split, h1 = min(heads, h0 + a.heads_per_split);
        for (int h = h0 + my_head; h < h1; h += span) {
            if (!in_step) break;
            const bool is_q = h < a.num_q_heads, is_k = !is_q && h < a.num_q_heads + a.kv_heads;
            const int hh = is_q ? h : (h - a.num_q_heads) % a.kv_heads;
            const T *src = is_q ? static_cast<const T *>(a.q) + t * a.q_stride
                                : static_cast<const T *>(is_k ? a.k : a.v) + t * a.kv_stride;
            src += (long long)hh * a.head_dim;
            // v passes through: its vectors are its item's 16 elements in order.
            const int f0 = is_q || is_k ? e0 : item * 16, f1 = is_q || is_k ? e1 : item * 16 + 8;
            float x[8], y[8];
            load8(src + f0, x);
            load8(src + f1, y);
            if (rotated && (is_q || is_k)) {
                if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = x[2 * j], q = x[2 * j + 1], r = y[2 * j], s = y[2 * j + 1];
                        x[2 * j] = p * c[j] - q * n[j];
                        x[2 * j + 1] = q * c[j] + p * n[j];
                        y[2 * j] = r * c[4 + j] - s * n[4 + j];
                        y[2 * j + 1] = s * c[4 + j] + r * n[4 + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float p = x[j], q = y[j];
                        x[j] = p * c[j] - q * n[j];
                        y[j] = q * c[j] + p * n[j];
                    }
                }
            }
            if (is_q || (is_k && a.k_out)) {
                T *dst = is_q ? static_cast<T *>(a.q_out) + t * a.q_out_stride
                              : static_cast<T *>(a.k_out) + t * a.k_out_stride;
                dst += (long long)hh * a.head_dim;
                store8(dst + f0, x);
                store8(dst + f1, y);
            }
            if (!is_q && at.slot >= 0) {
                P *dst = static_cast<P *>(is_k ? a.k_layer : a.v_layer) +
                         (at.slot * a.kv_heads + hh) * a.head_dim;
                if constexpr (FP8) {
                    const float inv = __ldg((is_k ? a.k_inv : a.v_inv) + hh);
                    store8_codes(dst + f0, x, inv);
                    store8_codes(dst + f1, y, inv);
                } else {
                    store8(dst + f0, x);
                    store8(dst + f1, y);
                }
            }
        }
    }
}

// Any head size, rotary dimension and alignment: a thread takes one pair (or
// one pass-through element) of one head. Bound by instructions: each pair pays
// a 64-bit division and the search for its sequence, which the vector form pays
// once a token, and accesses are of one element. 4,096 tokens of 28/4 heads of
// 80, 20 of them rotated, bf16: 142 us, 0.05 of a device copy's rate.
template <typename T, bool FP8>
__global__ void __launch_bounds__(kThreads) rope_cache_any_kernel(const RopeCacheLaunch a) {
    using P = std::conditional_t<FP8, uint8_t, T>;
    extern __shared__ int s_cu[];
    __shared__ int s_warp[kThreads / 32];
    __shared__ int s_bad;
    pdl_wait();
    const long long tokens = scan_tokens(a, s_cu, s_warp, &s_bad);
    const int half = a.rotary_dim / 2;
    const int items = half + (a.head_dim - a.rotary_dim);  // of a rotated head; v: head_dim elements
    const long long per_token = (long long)(a.num_q_heads + a.kv_heads) * items + (long long)a.kv_heads * a.head_dim;
    const long long total = tokens * per_token, stride = (long long)gridDim.x * kThreads;
    for (long long it = (long long)blockIdx.x * kThreads + threadIdx.x; it < total; it += stride) {
        const long long t = it / per_token;
        long long r = it - t * per_token;
        const bool lead = r == 0;
        const Place at = place_of_token(a, s_cu, t, lead);
        if (lead && a.slots_out) a.slots_out[t] = at.slot;
        if (at.pos < 0) continue;
        int h, i;
        if (r < (long long)(a.num_q_heads + a.kv_heads) * items) {
            h = (int)(r / items);
            i = (int)(r - (long long)h * items);
        } else {
            r -= (long long)(a.num_q_heads + a.kv_heads) * items;
            h = a.num_q_heads + a.kv_heads + (int)(r / a.head_dim);
            i = (int)(r % a.head_dim);
        }
        const bool is_q = h < a.num_q_heads, is_k = !is_q && h < a.num_q_heads + a.kv_heads;
        const int hh = is_q ? h : (h - a.num_q_heads) % a.kv_heads;
        const bool pair = (is_q || is_k) && i < half;
        const int f0 = pair ? (a.interleaved ? 2 * i : i) : (is_q || is_k) ? a.rotary_dim + i - half : i;
        const int f1 = a.interleaved ? f0 + 1 : f0 + half;  // used by pairs alone
        const T *src = is_q ? static_cast<const T *>(a.q) + t * a.q_stride
                            : static_cast<const T *>(is_k ? a.k : a.v) + t * a.kv_stride;
        src += (long long)hh * a.head_dim;
        float x = widen(src[f0]), y = 0.f;
        if (pair) {
            y = widen(src[f1]);
            const float c = __ldg(a.cos_sin + at.pos * a.rotary_dim + i);
            const float n = __ldg(a.cos_sin + at.pos * a.rotary_dim + half + i);
            const float p = x, q = y;
            x = p * c - q * n;
            y = q * c + p * n;
        }
        if (is_q || (is_k && a.k_out)) {
            T *dst = is_q ? static_cast<T *>(a.q_out) + t * a.q_out_stride
                          : static_cast<T *>(a.k_out) + t * a.k_out_stride;
            dst += (long long)hh * a.head_dim;
            dst[f0] = narrow<T>(x);
            if (pair) dst[f1] = narrow<T>(y);
        }
        if (!is_q && at.slot >= 0) {
            P *dst = static_cast<P *>(is_k ? a.k_layer : a.v_layer) + (at.slot * a.kv_heads + hh) * a.head_dim;
            if constexpr (FP8) {
                const float inv = __ldg((is_k ? a.k_inv : a.v_inv) + hh);
                dst[f0] = (uint8_t)(e4m3x2(__fmul_rn(x, inv), 0.f) & 0xffu);
                if (pair) dst[f1] = (uint8_t)(e4m3x2(__fmul_rn(y, inv), 0.f) & 0xffu);
            } else {
                dst[f0] = narrow<T>(x);
                if (pair) dst[f1] = narrow<T>(y);
            }
        }
    }
}

template <typename T, bool FP8>
cudaError_t launch_tp(RopeCacheLaunch a, int sms, cudaStream_t st) {
    const size_t smem = (size_t)(a.num_seqs + 1) * sizeof(int);
    const int heads = a.num_q_heads + 2 * a.kv_heads;
    // Vector form: heads and rotary parts of whole 16-element items, and
    // 16-byte rows (8-byte codes) everywhere.
    const long long es = sizeof(T), pool_es = FP8 ? 1 : sizeof(T);
    bool vec = a.head_dim % 16 == 0 && a.head_dim <= 512 && a.rotary_dim % 16 == 0 &&
               a.kv_stride * es % 16 == 0 && aligned(a.k, 16) && aligned(a.v, 16) &&
               aligned(a.cos_sin, 16) && a.head_dim * pool_es % 8 == 0;
    if (a.num_q_heads)
        vec = vec && a.q_stride * es % 16 == 0 && a.q_out_stride * es % 16 == 0 && aligned(a.q, 16) && aligned(a.q_out, 16);
    if (a.k_out) vec = vec && a.k_out_stride * es % 16 == 0 && aligned(a.k_out, 16);
    auto kern = !vec ? rope_cache_any_kernel<T, FP8>
                : a.interleaved ? rope_cache_kernel<T, FP8, true> : rope_cache_kernel<T, FP8, false>;
    cudaError_t e;
    if (smem > 48 * 1024 &&
        (e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess)
        return e;
    long long blocks;
    if (vec) {
        const int span = 32 / (a.head_dim / 16);
        const int steps = (heads + span - 1) / span;  // of one token
        // Few tokens: split a token's heads over warps until every SM has a CTA's worth.
        const long long want = (long long)sms * kRopeWarps;
        const int splits = (int)std::min<long long>(steps, std::max<long long>(1, want / std::max<long long>(a.num_tokens, 1)));
        const int per = (steps + splits - 1) / splits;
        a.heads_per_split = per * span;
        a.head_splits = (steps + per - 1) / per;
        blocks = (a.num_tokens * a.head_splits + kRopeWarps - 1) / kRopeWarps;
    } else {
        blocks = (a.num_tokens * heads * (long long)a.head_dim + kThreads - 1) / kThreads;
    }
    blocks = std::max<long long>(1, std::min<long long>(blocks, (long long)sms * 4));
    return launch_pdl(kern, dim3((unsigned)blocks), dim3(kThreads), smem, st, a);
}

}  // namespace

cudaError_t launch_rope_cache(const RopeCacheLaunch &a, DType src, DType pool, int sms, cudaStream_t st) {
    const bool fp8 = pool == DType::FP8_E4M3;
    switch (src) {
        case DType::F32: return fp8 ? launch_tp<float, true>(a, sms, st) : launch_tp<float, false>(a, sms, st);
        case DType::BF16:
            return fp8 ? launch_tp<__nv_bfloat16, true>(a, sms, st) : launch_tp<__nv_bfloat16, false>(a, sms, st);
        case DType::F16: return fp8 ? launch_tp<__half, true>(a, sms, st) : launch_tp<__half, false>(a, sms, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace pkv
