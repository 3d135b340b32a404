// pkv_prefill.cu -- causal attention of ragged new tokens: over the paged
// pool (a chunk of new tokens per sequence) or over packed K/V rows (whole
// prompts).
//
// Row i of sequence s, query head qh of kv head h = qh / group, at position
// p = ctx[s] + i:
//   out = sum_{j <= p} softmax_j(scale * q . k_j) v_j
//
// One warp per (row, query head): 32 keys at a time, a lane to a key for the
// scores, a lane to a run of head_dim / 32 elements for the output; the
// running maximum and sum of the softmax in f32.

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

__device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float wide(__half x) { return __half2float(x); }
__device__ __forceinline__ float wide(uint8_t code) {
    unsigned y;
    asm("{\n\t.reg .b16 a;\n\tcvt.u16.u32 a, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(y) : "r"((unsigned)code));
    return __half2float(__ushort_as_half((unsigned short)(y & 0xffffu)));
}
template <typename T>
__device__ __forceinline__ T tight(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 tight<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half tight<__half>(float x) { return __float2half_rn(x); }

// A sequence's rows and keys as the kernel uses them. Lengths that the call
// does not allow are recorded; the rows of one whose lengths alone are wrong
// are written as empty, rows outside the packed ones are not touched.
struct Seq {
    int row0, rows, ctx;  // rows < 0: none
    bool empty;
};
__device__ __forceinline__ Seq sequence(const PrefillLaunch &a, int s, bool report) {
    const int lo = __ldg(a.cu + s), hi = __ldg(a.cu + s + 1);
    const int ctx = a.ctx ? __ldg(a.ctx + s) : 0;
    Seq q{lo, hi - lo, ctx, false};
    if (lo < 0 || hi < lo || hi > a.num_tokens) {
        if (report) record_error(a.err, kShapeMismatch, s);
        q.rows = -1;
    } else if (q.rows > 0 && (ctx < 0 || q.rows > a.max_new || ctx > a.max_len - q.rows)) {
        if (report) record_error(a.err, kShapeMismatch, s);
        q.empty = true;
    }
    return q;
}

template <typename T, typename KV, int D>
__global__ void __launch_bounds__(256) prefill_attention_kernel(const PrefillLaunch a) {
    pdl_wait();
    const int s = blockIdx.x, lane = threadIdx.x & 31;
    const int warp = blockIdx.y * 8 + (threadIdx.x >> 5), warps = gridDim.y * 8;
    const Seq sq = sequence(a, s, warp == 0 && lane == 0);
    const int heads = a.kv_heads * a.group;
    constexpr int E = D / 32;
    for (long long u = warp; u < (long long)max(sq.rows, 0) * heads; u += warps) {
        const int i = (int)(u / heads), qh = (int)(u - (long long)i * heads), h = qh / a.group;
        const T *q = static_cast<const T *>(a.q) + (long long)(sq.row0 + i) * a.q_stride + (long long)qh * D;
        const int keys = sq.empty ? 0 : sq.ctx + i + 1;
        float m = -INFINITY, last = 0.f, l = 0.f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        float ks = 1.f, vs = 1.f;
        if (std::is_same_v<KV, uint8_t>) ks = __ldg(a.k_scale + h), vs = __ldg(a.v_scale + h);
        for (int j0 = 0; j0 < keys; j0 += 32) {
            const int j = j0 + lane;
            long long row = -1;
            if (j < keys) {
                if (a.tables) {
                    const int blk = __ldg(a.tables + (long long)s * a.table_stride + j / a.block_size);
                    if (blk < 0 || blk >= a.num_blocks) record_error(a.err, kInvalidBlock, s);
                    else row = (a.layer_row0 + (long long)blk * a.block_size + j % a.block_size) * a.kv_heads * D;
                } else {
                    row = (long long)(sq.row0 + j) * a.kv_stride;
                }
            }
            float sc = -INFINITY;
            if (row >= 0) {
                const KV *k = static_cast<const KV *>(a.k) + row + (long long)h * D;
                sc = 0.f;
                for (int d = 0; d < D; ++d) sc = fmaf(wide(q[d]), wide(k[d]), sc);
                sc *= a.scale_log2 * ks;
            }
            float mx = sc;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            m = fmaxf(m, mx);
            const float ref = m == -INFINITY ? 0.f : m;  // nothing but -inf so far: weights 0
            const float corr = exp2f(last - ref), p = exp2f(sc - ref);
            last = ref;
            l = l * corr + p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= corr;
            for (int t = 0; t < 32; ++t) {
                const float w = __shfl_sync(0xffffffffu, p, t);
                const long long r = __shfl_sync(0xffffffffu, row, t);
                if (r < 0) continue;
                const KV *v = static_cast<const KV *>(a.v) + r + (long long)h * D + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(w, wide(v[e]), o[e]);
            }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const long long at = (long long)(sq.row0 + i) * heads + qh;
#pragma unroll
        for (int e = 0; e < E; ++e)
            static_cast<T *>(a.out)[at * D + lane * E + e] = tight<T>(l > 0.f ? o[e] / l * vs : l == 0.f ? 0.f : l);
        if (lane == 0 && a.lse) a.lse[at] = l > 0.f ? (m + log2f(l)) * 0.69314718055994531f : l == 0.f ? -INFINITY : l;
    }
}

template <typename T, typename KV>
cudaError_t launch_simple(const PrefillLaunch &a, int sms, cudaStream_t st) {
    const long long warps = (long long)a.max_new * a.kv_heads * a.group;
    const dim3 grid((unsigned)a.num_seqs, (unsigned)std::max<long long>(1, std::min<long long>((warps + 7) / 8, sms * 8)));
    auto kern = a.head_dim == 64 ? prefill_attention_kernel<T, KV, 64>
                : a.head_dim == 128 ? prefill_attention_kernel<T, KV, 128> : prefill_attention_kernel<T, KV, 256>;
    return launch_pdl(kern, grid, dim3(256), 0, st, a);
}

}  // namespace

cudaError_t launch_prefill_attention(const PrefillLaunch &a, DType query, DType kv, int sms, cudaStream_t st) {
    if (a.num_seqs <= 0) return cudaSuccess;
    const bool fp8 = kv == DType::FP8_E4M3;
    if (query == DType::BF16)
        return fp8 ? launch_simple<__nv_bfloat16, uint8_t>(a, sms, st) : launch_simple<__nv_bfloat16, __nv_bfloat16>(a, sms, st);
    if (query == DType::F16)
        return fp8 ? launch_simple<__half, uint8_t>(a, sms, st) : launch_simple<__half, __half>(a, sms, st);
    return cudaErrorInvalidValue;
}

}  // namespace pkv
