// pkv_device.cuh -- device helpers shared by the kernel files: error
// recording, the block-wide scan of per-sequence lengths, the slot rule, and
// the launch-shape helpers of the scatter kernels.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <initializer_list>

#include "pkv_internal.hpp"

namespace pkv {

constexpr int kThreads = 256;

// pkv_status values recorded on the device.
constexpr int kInvalidBlock = 2;
constexpr int kSlotOutOfRange = 5;
constexpr int kShapeMismatch = 6;

__device__ __forceinline__ void record_error(DevError *e, int code, long long index) {
    if (atomicCAS(&e->code, 0, code) == 0) e->index = index;
}

// E4M3 codes of two f32 values, `lo` in the low byte: round to nearest even,
// saturating at +-448 (see pkv_set_kv_scales). The PTX conversion writes its
// first source operand to the upper byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// splitmix64 finaliser (Steele, Lea & Flood, 2014): the per-element hash of
// the plane digests, mix64(((index * 2 + plane) * golden) + f32 bits).
__device__ __forceinline__ unsigned long long mix64(unsigned long long z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

__device__ __forceinline__ unsigned long long elem_hash(long long gidx, int plane, unsigned bits) {
    return mix64(((unsigned long long)gidx * 2 + plane) * 0x9E3779B97F4A7C15ull + bits);
}

// Modulo 2^32: the sums that do not fit are found apart (scan_lengths).
__device__ __forceinline__ unsigned warp_inclusive_scan(unsigned x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// Exclusive prefix of new_lens into s_cu[0..num_seqs] (one contiguous
// segment per thread, then warp shuffles); sets *s_bad when a length or a
// context is negative or the sum does not fit 31 bits (s_cu is then no
// prefix). The scan is modulo 2^32. A step of the prefix adds less than 2^31,
// so the first prefix that passes 31 bits still shows it in bit 31: each is
// checked as it is written. Every thread of the CTA must call it.
__device__ __forceinline__ void scan_lengths(const int *__restrict__ ctx,
                                             const int *__restrict__ nnew, int num_seqs,
                                             int *s_cu, int *s_warp, int *s_bad) {
    const int tid = threadIdx.x;
    if (tid == 0) *s_bad = 0;
    __syncthreads();
    const int seg = (num_seqs + kThreads - 1) / kThreads;
    const int b0 = min(num_seqs, tid * seg);
    const int b1 = min(num_seqs, b0 + seg);
    unsigned local = 0;
    for (int q = b0; q < b1; ++q) {
        const int n = __ldg(nnew + q);
        if (n < 0 || __ldg(ctx + q) < 0) *s_bad = 1;
        local += max(n, 0);
    }
    const unsigned incl = warp_inclusive_scan(local);
    if ((tid & 31) == 31) s_warp[tid >> 5] = (int)incl;
    __syncthreads();
    if (tid < 32) {
        const unsigned w = tid < kThreads / 32 ? (unsigned)s_warp[tid] : 0u;
        const unsigned wi = warp_inclusive_scan(w);
        if (tid < kThreads / 32) s_warp[tid] = (int)(wi - w);
    }
    __syncthreads();
    unsigned run = (unsigned)s_warp[tid >> 5] + incl - local;
    for (int q = b0; q < b1; ++q) {
        s_cu[q] = (int)run;
        run += max(__ldg(nnew + q), 0);
        if ((int)run < 0) *s_bad = 1;
    }
    if (b1 == num_seqs && b0 < b1) s_cu[num_seqs] = (int)run;
    if (num_seqs == 0 && tid == 0) s_cu[0] = 0;
    __syncthreads();
}

// bf16 queries over E4M3 codes are held in f16, each row times `up`, the power
// of two that brings its largest element `top` to [2^13, 2^14) (elements down
// to 2^-28 of it keep their 8 bits); `down`, its inverse, joins the row's
// softmax scale. Rows of zeros, below 2^-100 or with an infinity: as they are
// or nearly.
struct QueryPower {
    float up, down;
};
__device__ __forceinline__ QueryPower query_power(float top) {
    int ex = (int)(__float_as_uint(top) >> 23) - 127;  // top = 2^ex * [1, 2)
    if (ex > 127) ex = 13;
    ex = max(ex, -100);
    return {__uint_as_float((unsigned)(13 - ex + 127) << 23), __uint_as_float((unsigned)(ex - 13 + 127) << 23)};
}

// The least softmax scale (base 2) of scores over E4M3 codes. It is a product
// (softmax scale, K scale, the power of two that the queries were divided by)
// which may underflow, and 0 times the -inf of a masked score would be NaN.
// |q . k| over codes and f16 queries stays below 2^33, so from here down every
// key weighs the same.
constexpr float kLeastFp8Scale = FLT_MIN;

// Programmatic dependent launch. A grid launched with programmatic stream
// serialization may be set up while the previous grid in its stream still
// runs; griddepcontrol.wait then holds it until that grid has completed and
// its writes are visible (a no-op for a grid launched the ordinary way), so
// stream order is kept and only the launch and set-up overlap. Called first,
// by every thread, before any global memory access. Most of the kernels that
// use it release their dependents only by exiting: a release at entry let the
// next step's CTAs take SM slots while this step's still streamed, and the
// decode step got slower (bf16: 5.91 -> 5.98 us, against 5.64 us with the
// release at exit). The attentions that a combine or a join follows release
// it early: it waits for their results in any case, and a tile kernel's CTA
// fills its SM, so that nothing takes a slot beside it.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches kern<<<grid, block, smem, st>>>(args...) with programmatic stream
// serialization (the kernel starts with pdl_wait()).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Combined slot of packed token t: its sequence by binary search over the
// prefix, then BlockTable::slot_for_position. -1 (and an error record when
// `report`) for a logical block past the table or a table entry outside the pool.
__device__ __forceinline__ long long slot_of_token(long long t, const int *s_cu, int num_seqs,
                                                   const int *__restrict__ ctx,
                                                   const int *__restrict__ tables,
                                                   long long table_stride, long long block_size,
                                                   long long num_blocks, DevError *err, bool report) {
    int lo = 0, hi = num_seqs - 1;
    while (lo < hi) {  // last q with s_cu[q] <= t; that sequence has new_lens > 0
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const long long pos = (long long)__ldg(ctx + lo) + (t - s_cu[lo]);
    const long long lb = pos / block_size;
    const long long off = pos - lb * block_size;
    if (lb >= table_stride) {
        if (report) record_error(err, kSlotOutOfRange, t);
        return -1;
    }
    const long long blk = __ldg(tables + (long long)lo * table_stride + lb);
    if (blk < 0 || blk >= num_blocks) {
        if (report) record_error(err, kInvalidBlock, t);
        return -1;
    }
    return blk * block_size + off;
}

inline bool aligned(const void *p, long long a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Layers per grid.y chunk of a scatter launch. Layers are split only when
// the (token, vector) items alone cannot fill one wave of resident CTAs, and
// never below 4 layers per chunk, so every thread keeps 4 layers' K and V
// loads in flight and the per-CTA set-up is paid for over several layers.
inline int layers_per_chunk(long long items, long long num_layers, int sms, long long *chunks) {
    const long long wave = (long long)sms * 4 * kThreads;
    const long long needed = (wave + std::max<long long>(items, 1) - 1) / std::max<long long>(items, 1);
    const long long cap = std::max<long long>(1, (num_layers + 3) / 4);
    const long long c = std::min<long long>(std::max<long long>(needed, 1), cap);
    const int lpc = (int)((num_layers + c - 1) / c);
    *chunks = (num_layers + lpc - 1) / lpc;
    return lpc;
}

// Largest power-of-two vector width (<= 16 bytes) dividing every byte offset.
inline int pick_vector_bytes(long long elem_bytes, std::initializer_list<long long> byte_quantities,
                      std::initializer_list<const void *> ptrs) {
    int vb = 16;
    while (vb > elem_bytes) {
        bool ok = true;
        for (long long q : byte_quantities) ok = ok && (q % vb == 0);
        for (const void *p : ptrs) ok = ok && aligned(p, vb);
        if (ok) break;
        vb /= 2;
    }
    return vb;
}

}  // namespace pkv
