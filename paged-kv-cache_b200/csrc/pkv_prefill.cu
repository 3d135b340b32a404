// pkv_prefill.cu -- causal attention of ragged new tokens: over the paged
// pool (a chunk of new tokens per sequence) or over packed K/V rows (whole
// prompts).
//
// Row i of sequence s, query head qh of kv head h = qh / group, at position
// p = ctx[s] + i:
//   out = sum_{j <= p} softmax_j(scale * q . k_j) v_j
//
// Mapping. An item is up to 2 x 128 query rows of one sequence and kv head
// (a row is a token and a head of the group, so the group shares every K and V
// tile) and walks the key tiles from 0 to its causal end. Both products run on
// the tensor core with f32 accumulators in tensor memory: S = Q K^T from
// shared memory, O += P V with the weights P (rounded to the query type)
// written back over S in tensor memory. The work is the 4 D operations a
// (query, key) pair that the products cost, and one exponential.
// - Row items: two 128-row tiles share each K/V tile; while a warpgroup takes
//   the softmax of one, the tensor core works on the other.
// - Key items (at most 128 rows): both warpgroups hold the same rows and take
//   every other key tile, each with its own O and statistics, merged at the
//   end: few rows are bound by the K/V stream, and this halves the chain of
//   softmaxes that the stream waits for.
// - head_dim 256: O alone takes half of tensor memory, so one row tile, two S
//   buffers, one warpgroup: a tile's products take twice its softmax.
// Schedule. One CTA per SM. The items' costs (keys, plus a constant) are
// summed in order of sequence, head and row; CTA b takes the b-th equal share,
// so lengths need no sorting and few rows over a long context are split along
// the keys. A share that begins or ends inside an item leaves a partial
// (O, max, sum) in a workspace of fixed size, two slots a CTA, and a second
// kernel joins an item's partials in order. Everything is derived from the
// lengths on the device; nothing depends on which CTA finishes first.
// Roles (16 warps): 8 warps softmax and epilogue, one issues the products, one
// brings K and one V by TMA, one plans items and brings Q, four fill the V tiles
// that a mask crosses (and, over an fp8 pool, convert every tile).
//
// Bounds, as measured (kernel and join, 20 calls in a graph, inputs in L2;
// products against 1,630 TFLOP/s, a matrix product's rate in a burst):
// - long rows: a step's chain of products and softmax. 2,048 rows over 32 k keys,
//   28/4 heads of 128: 829 to 866 us, 0.66 to 0.69 of it; a prompt of 8,192: 432
//   us, 0.68. A pair of row tiles takes 3,700 cycles a tile of 128 keys, 2,048 of
//   them products, and no unit is full: a warpgroup's maximum, exponentials and
//   stores of one 64-key step end before it reads the next one's scores. Under a
//   steady load the power limit lowers the clock to 1.68 GHz (922 and 498 us).
// - heads of 64: the same chain, whose products are half and exponentials are as
//   many: 7 of 8 by the special-function unit, 16 a clock and SM. 2,048 rows over
//   8 k keys, 32/8 heads: 197 us, 0.45 of that unit's rate; a prompt of 8,192: 421
//   us, 0.48.
// - prompts of 8,192 rows in ten sequences: 144 us, 0.37: a CTA's start (4 us to
//   its share, 7 us to its first scores, from a cold instruction cache), the
//   queries in and outputs out between items, and the join (5 us).
// - over fp8 (1,657 rows, 32/8 heads of 128): 182 us, 0.43 (195 beside other
//   allocations): the conversion of K and V in four warps takes issue slots from
//   the softmax.
// - head_dim 256: a prompt of 8,192, 8/4 heads, 259 us, 0.65: 1,280 cycles of
//   products a step of 64 keys, of about 1,900. (Two warpgroups with half of a
//   row's keys each took the same time, on long rows and short.) 3,800 rows in
//   three prompts: 48 us, 0.29: start, items' ends and the join.
//
// Roundings to fewer than 32 bits: scores, statistics and outputs are f32. The
// weights are rounded to the type of the products (the queries' type; f16 over
// fp8), which is what the tensor core takes for O += P V; their sum takes them
// unrounded. An output moves by at most half a step of that type times the mean
// |v|; f16 holds a weight below 2^-14 of the largest to 2^-25 of the largest.
//
// Masked keys may hold anything. A masked score is replaced before it is used.
// A masked value still meets a weight of 0 in the product, and 0 * NaN is NaN,
// so V tiles that some row masks are not brought by TMA: rows past the
// sequence and blocks outside the pool become zeros, and elements that are not
// finite become zero and are noted; at the end they are added to the rows
// that do attend them (a weight times an infinity or NaN is that infinity or
// NaN whatever the weight).

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "pkv_device.cuh"
#include "pkv_internal.hpp"
#include "pkv_tcgen05.cuh"

namespace pkv {
namespace {

using namespace tc;

constexpr int kDeviceCode = 9;                            // PKV_ERR_DEVICE
constexpr int kPrefillThreads = 512;
constexpr int kItemRing = 4;
constexpr int kMaskRing = 32;                             // key tiles whose block masks are kept
constexpr int kFlagWords = 12;                            // 3 key tiles of 128 bits
// Registers a thread after the split of the launch's 128 x 512: softmax
// threads hold a row of 128 scores, the others a few addresses.
constexpr int kSoftmaxRegs = 192, kOtherRegs = 64;
static_assert(2 * (kSoftmaxRegs + kOtherRegs) * 128 <= 128 * kPrefillThreads, "register split");
// The reference point of a row's weights moves when a score passes it by more
// than this (base 2): weights stay below 2^8, sums and products keep their
// relative precision, and most tiles skip the rescale of O.
constexpr float kLazy = 8.0f;
// One pair of weights in this many is computed on the FMA units, the others by
// the special-function unit (16 results a clock). More would relieve the unit
// but lengthen a step's chain, since a pair takes more instructions there: with
// every 2nd, 4th and no pair 2,048 rows over 32 k keys took 1.05, 1.03 and 1.01
// times as long as with every 8th, and 1,650 rows over fp8, where four warps
// convert beside them, 1.09, 1.05 and 0.95 times (so none there).
constexpr int kPolyEvery = 8;

enum Source { kPaged = 0, kPagedFp8 = 1, kRows = 2 };

// Tile geometry. Operand tiles are slabs of 64 elements (128 bytes) a row,
// 128-byte swizzled: 16-byte chunk c of row r at c ^ (r % 8).
template <int D, Source SRC>
struct Geom {
    static constexpr int kRowTiles = D == 256 ? 1 : 2;          // 128-row tiles per item
    static constexpr int kKeys = D == 256 ? 64 : 128;           // keys per tile
    static constexpr int kSlabs = D / 64;
    static constexpr int kQTile = 128 * D * 2;
    static constexpr int kTile = kKeys * D * 2;                 // one K or V tile
    // A tile of packed rows is [slab][row][128 B] (one box a slab); a paged one
    // [8 rows][slab][row of 8][128 B], so that one box brings a page's 16 rows.
    static constexpr int kSlab = SRC == kRows ? kKeys * 128 : 1024;      // bytes between slabs
    static constexpr int kGroup8 = SRC == kRows ? 1024 : 1024 * kSlabs;  // and between groups of 8 rows
    static constexpr bool kFp8 = SRC == kPagedFp8;
    static constexpr int kStages = kFp8 ? (D == 64 ? 6 : 3) : (D == 64 ? 10 : 5);
    static constexpr int kRawTile = kKeys * D;                  // fp8: the tile's codes
    static constexpr int kRawStages = kFp8 ? (D == 64 ? 6 : 3) : 0;
    static constexpr int kGranules = kKeys / 16;
    static constexpr int kSteps = kKeys / 64;                   // 64-key steps of a tile
    // head_dim 128: the scores of a tile's two steps by one product of N = 128
    // (N = 64 reads Q from shared memory as often for half the keys: 48 cycles in
    // place of 32 a product, 2,476 in place of 2,048 for a tile's products of two
    // row tiles), although the next scores then wait for both steps' weights:
    // 0.98 of the time on 2,048 rows over 32 k keys. 64: the softmax is
    // longer than the products in any case, and two buffers keep it from waiting.
    static constexpr bool kWide = D == 128;
    static constexpr int kOCol = kRowTiles * 128;               // after two S buffers of 64 columns a row tile
    static constexpr int kStatBytes = 2 * 128 * 8 + (SRC == kPagedFp8 ? 2 * 256 * 4 : 0);  // and the query rows' factors
    static constexpr int kSmem = kRowTiles * kQTile + kStages * kTile + kRawStages * kRawTile + kStatBytes;
    static constexpr int kSlotRows = kRowTiles * 128;           // rows of a partial
    static_assert(kOCol + kRowTiles * D <= 512, "tensor memory");
};

// Costs, as measured at heads of 128 and 256 (a row tile pair and 128 keys of
// 128: 3,700 cycles); heads of 64 share 128's, not measured apart. A key costs a
// row item kRowCost, a key item kKeyCost (one row tile, but its K and V come as
// slowly; over fp8 they are also converted), and an item kItemCost more (queries
// in, outputs out: 10,000 cycles).
template <int ROW_TILES, bool FP8>
struct Rates {
    static constexpr int kRowCost = 8, kKeyCost = ROW_TILES == 1 ? 8 : FP8 ? 7 : 5;
    static constexpr int kItemCost = ROW_TILES == 1 ? 3400 : FP8 ? 4000 : 2600;
};
// Shares do not begin or end closer than this many key tiles to an item's
// ends: the join costs about as much.
constexpr int kSnapRows = 3, kSnapKeys = 2;

struct Header {          // of a partial slot
    int state, pad0;     // 0: none; 1: a piece; 2: the piece reaches the item's last key
    int row0, tokens;    // packed row of the item's first token; its tokens
    int head, two;       // kv head; two row tiles
    int pad[2];
};

struct Params {
    PrefillLaunch a;
    int tile_tokens;     // tokens per 128-row tile: 128 / group
    int wide;            // out takes 32-byte stores
    double share;        // 1 / ctas
    float4 *part_o;      // [2 * ctas][slot rows / 128][D / 4][128]: a column of rows is contiguous
    float2 *part_ml;     // [2 * ctas][slot rows]: reference point (base 2), sum
    Header *headers;     // [2 * ctas]
};

struct Item {
    int seq, head;
    int row0;            // packed row of the first token
    int tokens;
    int key0;            // keys before the first token's own: row i's limit is key0 + i + 1
    int base;            // packed row of key 0 (packed rows only)
    int t0, t1, tiles;   // this piece's key tiles; the item's
    int two;             // row item
    int slot;            // partial slot, or -1: the whole item
    int end;             // no more items
};

// A sequence as every role sees it: rows < 0 are not touched; empty ones are
// written as rows without keys.
struct Seq {
    int row0, rows, ctx;
    bool empty;
};
__device__ __forceinline__ Seq sequence(const PrefillLaunch &a, int s, bool report) {
    const int lo = __ldg(a.cu + s), hi = __ldg(a.cu + s + 1);
    const int ctx = a.ctx ? __ldg(a.ctx + s) : 0;
    Seq q{lo, 0, ctx, false};
    if (lo < 0 || hi < lo || hi > a.num_tokens) {
        if (report) record_error(a.err, kShapeMismatch, s);
        return q;
    }
    q.rows = hi - lo;
    if (q.rows > 0 && (ctx < 0 || q.rows > a.max_new || ctx > a.max_len - q.rows)) {
        if (report) record_error(a.err, kShapeMismatch, s);
        q.empty = true;
        q.ctx = 0;
    }
    return q;
}

// The cost of the items of a sequence. Items 0 .. items - 2 are full; item i
// ends at key ctx + min((i + 1) * per, rows).
// Held in f64: whole numbers far below 2^53, in fewer instructions than 64-bit
// integers take (this code runs once a launch, from a cold instruction cache).
template <int ROW_TILES, bool FP8>
struct Costs {
    using R = Rates<ROW_TILES, FP8>;
    double ctx, per, last;
    int rows, items;
    bool empty;
    __device__ __forceinline__ Costs(const Seq &q, int tile_tokens) {
        const int full = ROW_TILES * tile_tokens;
        ctx = q.ctx;
        per = full;
        rows = q.rows;
        empty = q.empty;
        items = rows > 0 ? (rows - 1) / full + 1 : 0;
        const bool two = ROW_TILES == 2 && rows - (items - 1) * full > tile_tokens;
        last = R::kItemCost + (empty ? 0. : (two ? R::kRowCost : R::kKeyCost) * (ctx + rows));
    }
    // Cost of items 0 .. i - 1, i < items (all full).
    __device__ __forceinline__ double before(int i) const {
        const double n = i;
        if (empty) return n * R::kItemCost;
        return n * (R::kRowCost * ctx + R::kItemCost) + (0.5 * R::kRowCost * per) * (n * (n + 1.));
    }
    __device__ __forceinline__ double head() const { return items ? before(items - 1) + last : 0.; }
    __device__ __forceinline__ double of(int i) const { return i + 1 < items ? before(i + 1) - before(i) : last; }
};

struct Pos {
    int s, h, i, t;  // key tile t of item i of kv head h of sequence s
};

// The place of cost x within sequence s. Rounded to a key tile; within kSnap
// tiles of an item's ends, to that end.
template <int ROW_TILES, int KEYS, bool FP8>
__device__ __forceinline__ Pos locate(const Costs<ROW_TILES, FP8> &c, int s, double x, int tile_tokens) {
    // Quotients and the quadratic by 32-bit floats, then put right.
    const double head = c.head();
    int h = (int)__fdividef((float)x, (float)head);
    while (h > 0 && h * head > x) --h;
    while ((h + 1) * head <= x) ++h;
    double r = x - h * head;
    // The last item lo with before(lo) <= r.
    const float one = (float)(c.empty ? (double)Rates<ROW_TILES, FP8>::kItemCost : c.before(1));
    const float qa = c.empty ? 0.f : 0.5f * Rates<ROW_TILES, FP8>::kRowCost * (float)c.per, qb = one - qa;
    // (sqrt(qb^2 + 4 qa r) - qb) / (2 qa), in the form that holds for qa = 0 too.
    int lo = (int)__fdividef(2.f * (float)r, qb + sqrtf(qb * qb + 4.f * qa * (float)r));
    lo = max(0, min(lo, c.items - 1));
    while (lo > 0 && c.before(lo) > r) --lo;
    while (lo + 1 < c.items && c.before(lo + 1) <= r) ++lo;
    r -= c.before(lo);
    const int end = (int)c.ctx + (int)min((lo + 1) * c.per, (double)c.rows);
    const int tiles = c.empty ? 0 : (end - 1) / KEYS + 1;
    const bool two = ROW_TILES == 2 && (lo + 1 < c.items || c.rows - lo * ROW_TILES * tile_tokens > tile_tokens);
    const int snap = two ? kSnapRows : kSnapKeys;
    int t = (int)(__fdividef((float)r, (float)c.of(lo)) * (float)tiles + 0.5f);
    if (tiles < 2 * snap) t = 2 * t < tiles ? 0 : tiles;
    else if (t < snap) t = 0;
    else if (tiles - t < snap) t = tiles;
    Pos p{s, h, lo, t};
    if (t == tiles && (tiles > 0 || r > 0.)) {  // the item's end is the next one's beginning
        p.t = 0;
        ++p.i;
    }
    return p;
}

template <typename T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {  // a bit 15 / 31 for an element that is not finite
    if constexpr (std::is_same_v<T, __half>) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
    else return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}
__device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float wide(__half x) { return __half2float(x); }

// Two E4M3 codes (the low half of `two`) as f16, exactly.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(h) : "r"(two));
    return h;
}

template <typename T, int D, Source SRC>
__global__ void __launch_bounds__(kPrefillThreads, 1)
prefill_attention_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const __grid_constant__ Params p) {
    using G = Geom<D, SRC>;
    constexpr int NT = G::kRowTiles, KEYS = G::kKeys, ST = G::kStages, RS = G::kRawStages ? G::kRawStages : 1;
    // Type of the products' operands. E4M3 codes become f16, which one conversion
    // gives exactly, and so do bf16 queries over them: each row times the power
    // of two that brings its largest element to [2^13, 2^14), its inverse joining
    // the row's softmax scale.
    using M = std::conditional_t<SRC == kPagedFp8, __half, T>;
    constexpr bool kScaleQ = !std::is_same_v<M, T>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t kv_full[ST], kv_empty[ST], raw_full[RS], raw_empty[RS], by_hand_go[ST];
    __shared__ __align__(8) uint64_t s_full[4], p_full[4], pv_done[2], o_full[2], o_free[2], pair_bar, q_full, q_raw, q_empty, drain;
    __shared__ __align__(8) uint64_t item_full[kItemRing], item_empty[kItemRing];
    __shared__ Item s_item[kItemRing];
    __shared__ unsigned s_flag[kItemRing][kFlagWords + 1];
    __shared__ unsigned char s_mask[kMaskRing];
    __shared__ Pos s_range[2];
    __shared__ Seq s_first;  // the share's first sequence
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_failed;

    const PrefillLaunch &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in the whole warp
    unsigned char *sq = smem, *skv = smem + NT * G::kQTile, *sraw = skv + ST * G::kTile;
    float2 *stat = reinterpret_cast<float2 *>(sraw + G::kRawStages * G::kRawTile);
    float *q_factor = reinterpret_cast<float *>(stat + 2 * 128);
    double *s_scan = reinterpret_cast<double *>(stat);  // while the share is found

    if (smem_u32(smem) & 1023u) {  // the swizzle's atoms would not line up
        if (tid == 0) record_error(a.err, kDeviceCode, blockIdx.x);
        return;
    }
    if (warp == 0) tmem_alloc(&s_tmem, 512);
    if (tid == 32) {
        for (int i = 0; i < ST; ++i) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], 1), mbar_init(&by_hand_go[i], 1);
        for (int i = 0; i < RS; ++i) mbar_init(&raw_full[i], 1), mbar_init(&raw_empty[i], 1);
        for (int i = 0; i < 4; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 128);
        for (int i = 0; i < 2; ++i) mbar_init(&pv_done[i], 1), mbar_init(&o_full[i], 1), mbar_init(&o_free[i], 128);
        mbar_init(&pair_bar, 256), mbar_init(&q_full, 1), mbar_init(&q_raw, 1), mbar_init(&q_empty, 1), mbar_init(&drain, 1);
        for (int i = 0; i < kItemRing; ++i) mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 1 + 2 + 4 + 4 * NT);
        fence_barrier_init();
        s_failed = 0;
    }
    if (tid == 64) prefetch_map(&tq), prefetch_map(&tk), prefetch_map(&tv);
    pdl_wait();
    // The join may be scheduled from here on; it waits for this grid's end.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- this CTA's share ----
    {
        if (tid < 2) p.headers[2 * blockIdx.x + tid].state = 0;
        if (tid == 0) s_range[0] = s_range[1] = Pos{a.num_seqs, 0, 0, 0};  // no work
        const int seg = (a.num_seqs + kPrefillThreads - 1) / kPrefillThreads;
        const int b0 = min(a.num_seqs, tid * seg), b1 = min(a.num_seqs, b0 + seg);
        double local = 0.;
        Seq mine{0, 0, 0, false};  // the first of this thread's sequences: most often the only one
        for (int s = b0; s < b1; ++s) {
            const Seq q = sequence(a, s, blockIdx.x == 0);
            if (s == b0) mine = q;
            const Costs<NT, G::kFp8> c(q, p.tile_tokens);
            local += c.head() * a.kv_heads;
        }
        double incl = local;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        double add = 0., total = 0.;
#pragma unroll
        for (int w = 0; w < kPrefillThreads / 32; ++w) {
            if (w < warp) add += s_scan[w];
            total += s_scan[w];
        }
        const double first = add + incl - local;
#pragma unroll 1  // run once, from a cold instruction cache: the shorter the better
        for (int e = 0; e < 2; ++e) {
            const int b = blockIdx.x + e;
            const double x = floor(total * (b * p.share));
            if (b < (int)gridDim.x && x >= first && x < first + local) {
                double at = first;
                for (int s = b0; s < b1; ++s) {
                    const Seq q = s == b0 ? mine : sequence(a, s, false);
                    const Costs<NT, G::kFp8> c(q, p.tile_tokens);
                    const double w = c.head() * a.kv_heads;
                    if (x < at + w) {
                        if (e == 0) s_first = q;
                        s_range[e] = locate<NT, KEYS, G::kFp8>(c, s, x - at, p.tile_tokens);
                        break;
                    }
                    at += w;
                }
            }
        }
    }
    if (tid == 0) {
        for (int i = 0; i < kItemRing; ++i) s_flag[i][kFlagWords] = 0;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;

    // Waits are bounded: after about 2 s, or once another role has given up,
    // the wait fails, its role leaves, and the CTA drains and ends.
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (s_failed) return false;
            if (clock64() - t0 > kWaitCycles) {
                s_failed = 1;
                record_error(a.err, kDeviceCode, blockIdx.x);
                return false;
            }
        }
        return true;
    };
    // Key tiles that some row masks: from the one that holds the first row's limit.
    auto first_careful = [&](const Item &it) { return (it.key0 + 1) / KEYS; };
    // Places in the K/V ring, relative to the item's first: K runs `ahead`
    // tiles before V.
    auto k_at = [](int i, int ahead) { return i < ahead ? i : 2 * i - ahead + 1; };
    auto v_at = [](int j, int n, int ahead) { return j + min(n, j + ahead); };
    const int ahead_rows = 1, ahead_keys = 2;
    unsigned item_n = 0;  // items taken by this role

    if (warp >= 8 && warp < 12) {
        reg_dealloc<kOtherRegs>();
    } else if (warp >= 12) {
        reg_dealloc<kOtherRegs>();
    } else {
        reg_alloc<kSoftmaxRegs>();
    }

    if (warp < 4 * NT) {
        // ================= softmax and epilogue =================
        const int w = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int group = a.group, tau = row / group, hq = row - tau * group;
        unsigned s_ph = 0, of_ph[2] = {0, 0}, pv_n = 0, pair_n = 0, qn = 0;  // s_ph: a parity bit per S buffer
        unsigned kt = 0;  // key tiles of earlier items
        bool ok = true;
        for (; ok; ++item_n) {
            const unsigned ring = item_n % kItemRing;
            ok = wait(&item_full[ring], (item_n / kItemRing) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            const Item &it = s_item[ring];
            if (it.end) break;
            const int n = it.t1 - it.t0;
            const bool two = NT == 2 && it.two, keys = NT == 2 && !it.two;
            const int my_token = tau + (two && w ? p.tile_tokens : 0);
            const bool live = tau < p.tile_tokens && my_token < it.tokens;
            const int limit = live ? it.key0 + my_token + 1 : 0;
            // Tiles of this warpgroup: a first row tile may end a tile early.
            int mine = n;
            if (two && !w)
                mine = max(0, min(it.t1, (it.key0 + min(p.tile_tokens, it.tokens) + KEYS - 1) / KEYS) - it.t0);
            // The other warpgroup's: its o_full turns too.
            int others = two && w ? max(0, min(it.t1, (it.key0 + min(p.tile_tokens, it.tokens) + KEYS - 1) / KEYS) - it.t0) : n;
            if (keys) mine = (n - w + 1) / 2, others = (n - (w ^ 1) + 1) / 2;
            float scale = a.scale_log2, v_scale = 1.f;
            if constexpr (SRC == kPagedFp8) {
                scale *= __ldg(a.k_scale + it.head), v_scale = __ldg(a.v_scale + it.head);
                if constexpr (!kScaleQ) scale = fmaxf(scale, kLeastFp8Scale);
            }
            float m = -INFINITY, l = 0.f;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int careful = first_careful(it);
            for (int i = 0; i < mine * G::kSteps; ++i) {
                const int j = i / G::kSteps, t = it.t0 + (keys ? 2 * j + w : j);
                const int buf = w * 2 + (i & 1);
                const uint32_t s_addr = tmem + lanes + buf * 64;
                if (!G::kWide || !(i & 1)) {
                    ok = wait(&s_full[buf], (s_ph >> (i & 1)) & 1);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    s_ph ^= 1u << (i & 1);
                    fence_after();
                }
                if (kScaleQ && i == 0)
                    scale = fmaxf(scale * q_factor[(qn & 1) * 256 + (two ? w * 128 : 0) + row], kLeastFp8Scale);
                if (warp_live) {
                    const int first_key = t * KEYS + (i % G::kSteps) * 64;
                    const unsigned blocks =
                        SRC == kRows ? 0xfu : (s_mask[(kt + t - it.t0) % kMaskRing] >> (i % G::kSteps * 4)) & 0xfu;
                    const bool masked = t >= careful || (SRC != kRows && blocks != 0xfu);
                    const int lim = limit - first_key;
                    uint32_t sr[2][32];
                    auto hide = [&](float *x, int c) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (c * 32 + e >= lim) x[e] = -INFINITY;
                        if (SRC != kRows && blocks != 0xfu) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!((blocks >> (c * 2 + e / 16)) & 1u)) x[e] = -INFINITY;
                        }
                    };
                    tmem_ld32(s_addr, sr[0]);
                    tmem_ld32(s_addr + 32, sr[1]);
                    // The row's maximum; NaN among the scores makes it NaN, and with it
                    // the row. (An infinite one gives NaN weights too.)
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        wait_ld32(sr[c]);
                        float *x = reinterpret_cast<float *>(sr[c]);
                        if (masked) hide(x, c);
#pragma unroll
                        for (int k = 0; k < 32; k += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[k + e], x[k + 4 + e]);
                    }
                    const float mt = max3(max_nan(mx[0], mx[1]), mx[2], mx[3]) * scale;
                    // (Rows of no token hold whatever Q's shared memory held: never.)
                    const bool grew = live && !(mt <= m + kLazy);
                    if (__any_sync(0xffffffffu, grew)) {
                        // Only the rows that need it move: a row's result does not hang on
                        // the rows beside it.
                        float mn = grew ? max_nan(m, mt) : m;
                        if (mn == INFINITY) mn = NAN;
                        const float corr = !grew ? 1.f : m == -INFINITY ? 0.f : ex2(m - mn);
                        l *= corr;
                        m = mn;
                        if (i > 0) {
                            // O holds the steps before this one, once the last of
                            // their products is complete (S of this step was issued
                            // after the one before it).
                            ok = wait(&pv_done[w], (pv_n + i - 1) & 1);
                            if (!__all_sync(0xffffffffu, ok)) break;
                            fence_after();
                            const uint32_t o_addr = tmem + lanes + G::kOCol + (NT == 2 ? w * D : 0);
#pragma unroll
                            for (int c = 0; c < D / 16; ++c) {
                                uint32_t o[16];
                                tmem_ld16(o_addr + c * 16, o);
                                wait_ld16(o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st16(o_addr + c * 16, o);
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m;  // nothing yet: weights 2^-inf = 0
                    const uint64_t sc2 = pair(scale, scale), mr2 = pair(-ref, -ref);
                    uint64_t sum[2] = {pair(l, 0.f), pair(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float *s = reinterpret_cast<const float *>(sr[c]);
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x, y;
                            const uint64_t xy = fma2(pair(s[2 * e], s[2 * e + 1]), sc2, mr2);
                            if (!G::kFp8 && e % kPolyEvery == kPolyEvery - 1) {
                                ex2_poly(xy, x, y);
                            } else {
                                unpair(xy, x, y);
                                x = ex2(x);
                                y = ex2(y);
                            }
                            sum[e & 1] = add2(sum[e & 1], pair(x, y));
                            pk[e] = pack2<M>(x, y);
                        }
                        // Over scores that this row has read already.
                        tmem_st16(s_addr + c * 16, pk);
                    }
                    float u, v;
                    unpair(add2(sum[0], sum[1]), u, v);
                    l = u + v;
                    wait_st();
                }
                fence_before();
                mbar_arrive(&p_full[buf]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            pv_n += mine * G::kSteps;
            qn += n > 0;
            kt += n;

            // ---- epilogue: this row's O (key items: the two halves merged) ----
            const long long out_row = (long long)(it.row0 + my_token) * (a.kv_heads * group) + (long long)it.head * group + hq;
            const bool wait_mine = mine > 0;
            if (wait_mine) {
                const int ob = NT == 1 ? 0 : w;
                ok = wait(&o_full[ob], of_ph[ob] & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                ++of_ph[ob];
            }
            int c0 = 0, c1 = D;
            // Factors of the two accumulators; a row item has one.
            float f0 = w == 0 ? 1.f : 0.f, f1 = w == 1 ? 1.f : 0.f;
            bool use0 = w == 0 && mine > 0, use1 = w == 1 && mine > 0;
            if (keys) {
                stat[w * 128 + row] = make_float2(m, l);
                mbar_arrive(&pair_bar);
                ok = wait(&pair_bar, pair_n++ & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                const float2 other = stat[(w ^ 1) * 128 + row];
                const float mm = fmaxf(m, other.x);
                const float mine_f = m == -INFINITY ? 0.f : ex2(m - mm);
                const float other_f = other.x == -INFINITY ? 0.f : ex2(other.x - mm);
                // A NaN sum stays: 0 * NaN.
                l = l * mine_f + other.y * other_f;
                m = mm;
                f0 = w == 0 ? mine_f : other_f;
                f1 = w == 0 ? other_f : mine_f;
                use0 = n > 0;
                use1 = n > 1;
                // Each warpgroup stores half of the elements (of 64, the first all).
                c0 = w * (D == 64 ? 64 : D / 2);
                c1 = D == 64 ? 64 : c0 + D / 2;
                // The wait above covers this warpgroup's half alone.
                if (others > 0) {
                    ok = wait(&o_full[w ^ 1], of_ph[w ^ 1] & 1);
                    if (!__all_sync(0xffffffffu, ok)) break;
                }
            }
            if (NT == 2) of_ph[w ^ 1] += others > 0;
            fence_after();
            const unsigned flagged = s_flag[ring][kFlagWords];
            const float inv = l == 0.f ? 0.f : v_scale / l;
#pragma unroll 1
            for (int c = c0; c < c1 && warp_live; c += 64) {
                float o[64];
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t r[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[k * 32 + i] = 0.f;
                    if (use0) {
                        tmem_ld32(tmem + lanes + G::kOCol + c + k * 32, r);
                        wait_ld32(r);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[k * 32 + i] = __uint_as_float(r[i]) * f0;
                    }
                    if (NT == 2 && use1) {
                        tmem_ld32(tmem + lanes + G::kOCol + D + c + k * 32, r);
                        wait_ld32(r);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[k * 32 + i] = fmaf(__uint_as_float(r[i]), f1, o[k * 32 + i]);
                    }
                }
                if (live && flagged) {
                    // Elements of V that were not finite, for the rows that attend them.
                    for (int b = 0; b < kFlagWords * 32; ++b) {
                        if (!((s_flag[ring][b >> 5] >> (b & 31)) & 1u)) continue;
                        const int key = careful * KEYS + b;
                        if (key >= limit) continue;
                        long long at;
                        if constexpr (SRC == kRows) {
                            at = (long long)(it.base + key) * a.kv_stride;
                        } else {
                            const int blk = __ldg(a.tables + (long long)it.seq * a.table_stride + key / a.block_size);
                            at = (a.layer_row0 + (long long)blk * a.block_size + key % a.block_size) * a.kv_heads * D;
                        }
                        at += (long long)it.head * D + c;
#pragma unroll
                        for (int i = 0; i < 64; ++i) {
                            if constexpr (SRC == kPagedFp8) {
                                if ((__ldg(static_cast<const uint8_t *>(a.v) + at + i) & 0x7fu) == 0x7fu) o[i] = NAN;
                            } else {
                                const float x = wide(static_cast<const T *>(a.v)[at + i]);
                                if (!isfinite(x)) o[i] += x;
                            }
                        }
                    }
                }
                if (it.slot >= 0) {
                    float4 *part = p.part_o + (((long long)it.slot * NT + (two ? w : 0)) * (D / 4) + c / 4) * 128 + row;
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            part[i * 128] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    continue;
                }
                uint32_t x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = pack2<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
                if (!p.wide) {
                    uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + out_row * D + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (live) out[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                    continue;
                }
                // A lane has a row of its own: a store would meet 32 lines. Four lanes
                // exchange 32-byte pieces of their four rows, so that each has one
                // piece of every row and a store covers whole lines. (An item's
                // outputs take 1,000 to 2,000 of its epilogue's 5,000 cycles.)
                const bool hi = lane & 2, lo = lane & 1;
                uint32_t y[2][16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, hi ? x[i] : x[16 + i], 2);
                    const uint32_t own = hi ? x[16 + i] : x[i];
                    y[0][i] = hi ? other : own;
                    y[1][i] = hi ? own : other;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t z[2][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t other = __shfl_xor_sync(0xffffffffu, lo ? y[k][i] : y[k][8 + i], 1);
                        const uint32_t own = lo ? y[k][8 + i] : y[k][i];
                        z[0][i] = lo ? other : own;
                        z[1][i] = lo ? own : other;
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int from = (lane & ~3) | (2 * k + q);
                        const long long r = __shfl_sync(0xffffffffu, live ? out_row : -1, from);
                        if (r >= 0) store32(static_cast<T *>(a.out) + r * D + c + (lane & 3) * 16, z[q]);
                    }
                }
            }
            __syncwarp();
            if (live && (!keys || w == 0)) {
                if (it.slot < 0) {
                    if (a.lse) a.lse[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
                } else {
                    p.part_ml[(long long)it.slot * G::kSlotRows + (two ? w * 128 : 0) + row] = make_float2(m, l);
                }
            }
            if (it.slot >= 0 && tid == 0) {
                Header h{it.t1 == it.tiles ? 2 : 1, 0, it.row0, it.tokens, it.head, two, {0, 0}};
                p.headers[it.slot] = h;
            }
            fence_before();
            if (keys) {  // both halves have read both accumulators, and the statistics
                mbar_arrive(&pair_bar);
                ok = wait(&pair_bar, pair_n++ & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
            }
            if (mine > 0) mbar_arrive(&o_free[NT == 1 ? 0 : w]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[ring]);
        }
    } else if (warp == 8) {
        // ================= the products =================
        // One warp issues them all, the warpgroups' in turn: its order keeps one
        // warpgroup in its softmax while the other's products run (with a warp per
        // warpgroup the two fell into step: 0.99 -> 1.04 ms on 2,048 rows over 32 k
        // keys). The whole warp runs the loops and one lane issues: what is the same
        // in all lanes sits in uniform registers, where tcgen05.mma takes its
        // operands, and need not be moved there for each.
        {
            constexpr uint32_t id_s = instr_desc<M>(128, G::kWide ? 128 : 64, false), id_o = instr_desc<M>(128, D, true);
            constexpr uint32_t hi_q = desc_hi(1024), hi_kv = desc_hi(G::kGroup8);
            constexpr int kScores = G::kWide ? 1 : G::kSteps;  // products a tile's scores take
            const uint32_t lo_q = desc_lo(smem_u32(sq), 16), lo_k = desc_lo(smem_u32(skv), 16),
                           lo_v = desc_lo(smem_u32(skv), G::kSlab);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            unsigned place = 0, turn = 0;  // of the K/V ring, taken in order
            unsigned p_ph = 0, ou[2] = {0, 0}, qn = 0;
            bool ok = true;
            struct Tile {
                unsigned stage, parity;
            };
            auto take = [&]() {
                const Tile x{place, turn};
                if (++place == ST) place = 0, turn ^= 1;
                return x;
            };
            auto all = [&](bool good) { return ok = __all_sync(0xffffffffu, good) != 0; };
            auto full = [&](const Tile &x) { return ok && all(wait(&kv_full[x.stage], x.parity)); };
            auto done_with = [&](uint64_t *bar) {
                if (elect_one()) commit(bar);
                __syncwarp();
            };
            // Step h (64 keys; with kWide, step 0 both) of tile x: its scores for row
            // tile qt into S buffer b of warpgroup w.
            auto scores = [&](int qt, int w, int b, const Tile &x, int h) {
                const uint32_t q = lo_q + qt * (G::kQTile / 16),
                               k = lo_k + x.stage * (G::kTile / 16) + h * (8 * G::kGroup8 / 16);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        mma_ss<hi_q, hi_kv>(tm + (w * 2 + b) * 64, q + (i / 4) * (128 * 128 / 16) + (i % 4) * 2,
                                            k + (i / 4) * (G::kSlab / 16) + (i % 4) * 2, id_s, i > 0);
                    commit(&s_full[w * 2 + b]);
                }
                __syncwarp();
            };
            // O += P V of step h, its weights in S buffer b of warpgroup w.
            auto values = [&](int w, int b, const Tile &x, int h, bool first) {
                if (!ok || !all(wait(&p_full[w * 2 + b], (p_ph >> (w * 2 + b)) & 1))) return;
                p_ph ^= 1u << (w * 2 + b);
                // The first product overwrites the O that the last item's epilogue read.
                if (first && ou[w] > 0 && !all(wait(&o_free[w], (ou[w] - 1) & 1))) return;
                fence_after();
                const uint32_t v = lo_v + x.stage * (G::kTile / 16) + h * (8 * G::kGroup8 / 16);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_ts<hi_kv>(tm + G::kOCol + w * D, tm + (w * 2 + b) * 64 + i * 8, v + i * (2 * G::kGroup8 / 16),
                                      id_o, !first || i > 0);
                    commit(&pv_done[w]);
                }
                __syncwarp();
            };
            for (; ok; ++item_n) {
                const unsigned ring = item_n % kItemRing;
                if (!all(wait(&item_full[ring], (item_n / kItemRing) & 1))) break;
                const Item &item = s_item[ring];
                const int end = __shfl_sync(0xffffffffu, item.end, 0), two = __shfl_sync(0xffffffffu, item.two, 0);
                const int n = __shfl_sync(0xffffffffu, item.t1 - item.t0, 0);
                // Tiles of the first row tile, which may end one early.
                const int n0 = __shfl_sync(
                    0xffffffffu,
                    max(0, min(item.t1, (item.key0 + min(p.tile_tokens, item.tokens) + KEYS - 1) / KEYS) - item.t0), 0);
                if (lane == 0) mbar_arrive(&item_empty[ring]);
                __syncwarp();
                if (end) break;
                if (n == 0) continue;
                if (!all(wait(&q_full, qn & 1))) break;
                ++qn;
                fence_after();
                if (NT == 2 && two) {
                    // Row items: both warpgroups take every tile.
                    Tile k = take();
                    if (!full(k)) break;
                    fence_after();
#pragma unroll
                    for (int h = 0; h < kScores; ++h) {
                        if (n0 > 0) scores(0, 0, h, k, h);
                        scores(1, 1, h, k, h);
                    }
                    done_with(&kv_empty[k.stage]);
                    if (n == 1) done_with(&q_empty);
                    for (int j = 0; j < n; ++j) {
                        const Tile v = take();
                        if (j + 1 < n) k = take();
                        if (!full(v) || (j + 1 < n && !full(k))) break;
                        auto step = [&](int w, int h, int tiles) {
                            if (j >= tiles) return;
                            values(w, h, v, h, j == 0 && h == 0);
                            if (!ok) return;
                            const bool done = h + 1 == G::kSteps;
                            if (done && j + 1 == tiles) done_with(&o_full[w]), ++ou[w];
                            if (j + 1 < tiles && (done || !G::kWide)) scores(w, w, G::kWide ? 0 : h, k, G::kWide ? 0 : h);
                        };
#pragma unroll
                        for (int x = 0; x < 2 * G::kSteps; ++x) {
                            if constexpr (G::kWide) step(x / G::kSteps, x % G::kSteps, x / G::kSteps ? n : n0);
                            else step(x & 1, x >> 1, x & 1 ? n : n0);
                        }
                        if (!ok) break;
                        done_with(&kv_empty[v.stage]);
                        if (j + 1 < n) done_with(&kv_empty[k.stage]);
                        if (j + 2 == n) done_with(&q_empty);
                    }
                } else {
                    // Key items: tiles alternate between the warpgroups. head_dim 256: one
                    // warpgroup, whose S buffers the tiles alternate between.
                    for (int i = 0; i < min(ahead_keys, n); ++i) {
                        const Tile k = take();
                        if (!full(k)) break;
                        fence_after();
#pragma unroll
                        for (int h = 0; h < kScores; ++h) scores(0, NT == 2 ? i : 0, NT == 2 ? h : i, k, h);
                        done_with(&kv_empty[k.stage]);
                    }
                    if (!ok) break;
                    if (n <= ahead_keys) done_with(&q_empty);
                    for (int j = 0; j < n; ++j) {
                        const int w = NT == 2 ? j & 1 : 0;
                        const bool more = j + ahead_keys < n;
                        const Tile v = take();
                        Tile k = v;
                        if (more) k = take();
                        if (!full(v)) break;
#pragma unroll
                        for (int h = 0; h < G::kSteps; ++h) {
                            const int b = NT == 2 ? h : j & 1;
                            values(w, b, v, h, h == 0 && j < NT);
                            if (more && h == 0) full(k);
                            if (ok && more && (!G::kWide || h + 1 == G::kSteps)) scores(0, w, G::kWide ? 0 : b, k, G::kWide ? 0 : h);
                        }
                        if (!ok) break;
                        done_with(&kv_empty[v.stage]);
                        if (more) done_with(&kv_empty[k.stage]);
                        if (j + ahead_keys + 1 == n) done_with(&q_empty);
                        if (j + NT >= n) done_with(&o_full[w]), ++ou[w];
                    }
                }
            }
            // Nothing may be in flight when tensor memory is freed.
            done_with(&drain);
            const long long t0 = clock64();
            while (!mbar_try_wait(&drain, 0) && clock64() - t0 < kWaitCycles) {}
        }
    } else if (warp == 9 || warp == 11) {
        // ================= K (warp 9) and V (warp 11) by TMA =================
        // Each takes its own places of the ring. The products free places in
        // order and each warp skips at most two, fewer than the ring holds, so
        // a stage's parity tells its turns apart.
        const bool is_k = warp == 9;
        const CUtensorMap *map = is_k ? &tk : &tv;
        unsigned pos = 0, kt = 0;
        bool ok = true;
        const uint32_t kv0 = smem_u32(skv), raw0 = smem_u32(sraw);
        for (; ok; ++item_n) {
            const unsigned ring = item_n % kItemRing;
            ok = wait(&item_full[ring], (item_n / kItemRing) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            const Item it = s_item[ring];
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[ring]);
            if (it.end) break;
            const int n = it.t1 - it.t0, ahead = NT == 2 && it.two ? ahead_rows : ahead_keys;
            const int careful = first_careful(it), len = it.key0 + it.tokens;
            // Pages, 32 granules of 16 keys at a time: lane i of `rows` holds the pool
            // row of granule base + i (-1: past the keys or outside the pool); the
            // block ids of the next 32 are on their way meanwhile.
            constexpr int kGroup = 32 / G::kGranules;  // key tiles per 32 granules
            auto block_at = [&](int t) {
                const int key = t * KEYS + lane * 16;
                if (SRC == kRows || t >= it.t1 || key >= len) return -1;
                return __ldg(a.tables + (long long)it.seq * a.table_stride + key / a.block_size);
            };
            int rows = -1, next = block_at(it.t0);
            unsigned usable = 0;  // granules whose keys count, or that a mask hides anyway
            for (int j = 0; j < n; ++j) {
                const int t = it.t0 + j;
                const unsigned at = pos + (is_k ? k_at(j, ahead) : v_at(j, n, ahead));
                if (SRC != kRows && j % kGroup == 0) {
                    const int key = t * KEYS + lane * 16;
                    const bool have = key < len && t + lane / G::kGranules < it.t1;
                    const bool good = have && next >= 0 && next < a.num_blocks;
                    if (is_k && have && !good) record_error(a.err, kInvalidBlock, it.seq);
                    rows = good ? (int)(a.layer_row0 + (long long)next * a.block_size + key % a.block_size) : -1;
                    usable = __ballot_sync(0xffffffffu, good || !have);
                    next = block_at(t + kGroup);
                }
                const bool by_hand = SRC != kPagedFp8 && !is_k && t >= careful;
                uint64_t *full = SRC == kPagedFp8 ? &raw_full[at % RS] : &kv_full[at % ST];
                uint64_t *empty = SRC == kPagedFp8 ? &raw_empty[at % RS] : &kv_empty[at % ST];
                const unsigned turn = SRC == kPagedFp8 ? at / RS : at / ST;
                ok = wait(empty, (turn & 1) ^ 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (by_hand) {
                    if (elect_one()) mbar_arrive(&by_hand_go[at % ST]);
                    __syncwarp();
                    continue;
                }
                if constexpr (SRC == kRows) {
                    if (elect_one()) {
                        mbar_expect_tx(full, G::kTile);
#pragma unroll
                        for (int c = 0; c < G::kSlabs; ++c)
                            tma_load_2d(kv0 + (at % ST) * G::kTile + c * G::kSlab, map, it.head * D + c * 64,
                                        it.base + t * KEYS, full);
                    }
                } else {
                    int y[G::kGranules], loads = 0;
#pragma unroll
                    for (int g = 0; g < G::kGranules; ++g) {
                        y[g] = __shfl_sync(0xffffffffu, rows, j % kGroup * G::kGranules + g);
                        loads += y[g] >= 0;
                    }
                    const unsigned bits = (usable >> (j % kGroup * G::kGranules)) & ((1u << G::kGranules) - 1);
                    if (SRC == kPaged && !is_k && loads < G::kGranules) {
                        // A block outside the pool: its values are zeros.
                        unsigned char *dst = skv + (at % ST) * G::kTile;
#pragma unroll
                        for (int g = 0; g < G::kGranules; ++g)
                            for (int i = lane; y[g] < 0 && i < G::kSlabs * 128; i += 32)
                                *reinterpret_cast<uint4 *>(dst + g * 2 * G::kGroup8 + i * 16) = make_uint4(0, 0, 0, 0);
                        fence_async();
                        __syncwarp();
                    }
                    if (elect_one()) {
                        if (is_k) s_mask[(kt + j) % kMaskRing] = (unsigned char)bits;
                        mbar_expect_tx(full, loads * (SRC == kPagedFp8 ? 16 * D : 16 * D * 2));
#pragma unroll
                        for (int g = 0; g < G::kGranules; ++g) {
                            if (y[g] < 0) continue;
                            if constexpr (SRC == kPagedFp8)
                                tma_load_2d(raw0 + (at % RS) * G::kRawTile + g * 16 * D, map, it.head * D, y[g], full);
                            else
                                tma_load_4d(kv0 + (at % ST) * G::kTile + g * 2 * G::kGroup8, map, 0, 0,
                                            it.head * G::kSlabs, y[g] >> 3, full);
                        }
                    }
                }
                __syncwarp();
            }
            pos += 2 * n;
            kt += n;
        }
        if (!ok && lane == 0) {
            // Copies in flight land before the CTA's memory is given up.
            const long long t0 = clock64();
            while (clock64() - t0 < 20000000ll) {}
        }
    } else if (warp == 10) {
        // ================= items, and Q by TMA =================
        Pos at = s_range[0];
        const Pos end = s_range[1];
        bool fresh = true;
        unsigned qn = 0;
        bool ok = true;
        auto publish = [&](const Item &it) -> bool {
            const unsigned ring = item_n % kItemRing;
            bool good = true;
            if (lane == 0) {
                if (item_n >= kItemRing) good = wait(&item_empty[ring], ((item_n / kItemRing) & 1) ^ 1);
                if (good) {
                    s_item[ring] = it;
                    for (int i = 0; i <= kFlagWords; ++i) s_flag[ring][i] = 0;
                    mbar_arrive(&item_full[ring]);
                }
            }
            ++item_n;
            return __shfl_sync(0xffffffffu, good, 0);
        };
        while (ok && at.s < a.num_seqs && at.s <= end.s) {
            // The next sequence with rows, from at.s on: 32 at a time.
            const int s = at.s + lane;
            Seq q{0, 0, 0, false};
            if (fresh) {
                if (lane == 0) q = s_first;
                fresh = false;
            } else if (s < a.num_seqs) {
                q = sequence(a, s, false);
            }
            const unsigned some = __ballot_sync(0xffffffffu, q.rows > 0);
            if (!some) {
                at = Pos{at.s + 32, 0, 0, 0};
                continue;
            }
            const int src = __ffs(some) - 1;
            if (src > 0) at = Pos{at.s + src, 0, 0, 0};
            q.row0 = __shfl_sync(0xffffffffu, q.row0, src);
            q.rows = __shfl_sync(0xffffffffu, q.rows, src);
            q.ctx = __shfl_sync(0xffffffffu, q.ctx, src);
            q.empty = __shfl_sync(0xffffffffu, q.empty, src);
            const int per = NT * p.tile_tokens, items = (q.rows - 1) / per + 1;
            for (; ok && at.h < a.kv_heads; ++at.h, at.i = 0) {
                for (; ok && at.i < items; ++at.i, at.t = 0) {
                    const bool last = at.s == end.s && at.h == end.h && at.i == end.i;
                    const bool past = at.s > end.s || (at.s == end.s && (at.h > end.h || (at.h == end.h && at.i > end.i)));
                    if (past || (last && end.t <= at.t)) goto planned;
                    Item it{};
                    it.seq = at.s;
                    it.head = at.h;
                    const int tok0 = at.i * per;
                    it.row0 = q.row0 + tok0;
                    it.tokens = min(per, q.rows - tok0);
                    it.key0 = q.ctx + tok0;
                    it.base = q.row0;
                    it.tiles = q.empty ? 0 : (it.key0 + it.tokens - 1) / KEYS + 1;
                    it.t0 = at.t;
                    it.t1 = last ? end.t : it.tiles;
                    it.two = NT == 2 && it.tokens > p.tile_tokens;
                    it.slot = it.t0 > 0 ? 2 * (int)blockIdx.x : it.t1 < it.tiles ? 2 * (int)blockIdx.x + 1 : -1;
                    if (!(ok = publish(it))) break;
                    if (it.t1 > it.t0) {
                        if (elect_one()) {
                            if (qn > 0) ok = wait(&q_empty, (qn - 1) & 1);
                            if (ok) {
                                const int tiles = it.two ? 2 : 1;
                                const uint32_t bytes = (uint32_t)p.tile_tokens * a.group * 128;
                                uint64_t *bar = kScaleQ ? &q_raw : &q_full;
                                mbar_expect_tx(bar, tiles * G::kSlabs * bytes);
                                for (int x = 0; x < tiles; ++x)
                                    for (int c = 0; c < G::kSlabs; ++c)
                                        tma_load_3d(smem_u32(sq) + x * G::kQTile + c * (128 * 128), &tq, c * 64,
                                                    it.head * a.group, it.row0 + x * p.tile_tokens, bar);
                            }
                        }
                        ++qn;
                        ok = __all_sync(0xffffffffu, ok);
                    }
                }
            }
            at = Pos{at.s + 1, 0, 0, 0};
        }
    planned:
        if (ok) {
            Item it{};
            it.end = 1;
            publish(it);
        }
        if (!ok && lane == 0) {
            const long long t0 = clock64();
            while (clock64() - t0 < 20000000ll) {}
        }
    } else if (warp >= 12) {
        // ================= V tiles by hand; fp8 conversion =================
        constexpr int kT = 128;
        const int t128 = tid & 127;
        unsigned pos = 0, kt = 0, go_ph = 0, qn = 0;
        bool ok = true;
        auto together = [&](bool good) -> bool {  // all of these warps, and whether all are well
            int r;
            __syncwarp();
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
                "barrier.cta.red.and.aligned.pred q, 2, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                : "=r"(r) : "r"((int)good), "n"(kT) : "memory");
            return r != 0;
        };
        for (; ok; ++item_n) {
            const unsigned ring = item_n % kItemRing;
            ok = together(wait(&item_full[ring], (item_n / kItemRing) & 1));
            if (!ok) break;
            const Item it = s_item[ring];
            if (it.end) break;
            const int n = it.t1 - it.t0, ahead = NT == 2 && it.two ? ahead_rows : ahead_keys;
            const int careful = first_careful(it), len = it.key0 + it.tokens;
            auto note = [&](int key) {
                const int b = key - careful * KEYS;
                if (b >= 0 && b < kFlagWords * 32) {
                    atomicOr(&s_flag[ring][b >> 5], 1u << (b & 31));
                    s_flag[ring][kFlagWords] = 1;
                }
            };
            if constexpr (SRC != kPagedFp8) {
                for (int t = max(it.t0, careful); t < it.t1; ++t) {
                    const unsigned at = pos + v_at(t - it.t0, n, ahead);
                    // The K/V warp has seen the stage empty; one turn of this
                    // barrier per tile filled here.
                    ok = together(wait(&by_hand_go[at % ST], (go_ph >> (at % ST)) & 1));
                    if (!ok) break;
                    go_ph ^= 1u << (at % ST);
                    unsigned char *dst = skv + (at % ST) * G::kTile;
                    constexpr int kUnits = D / 8;                       // 16-byte units of a row
                    constexpr int kBatch = 8;
#pragma unroll 1
                    for (int b = t128; b < KEYS * kUnits; b += kBatch * kT) {
                        uint4 x[kBatch];
#pragma unroll
                        for (int e = 0; e < kBatch; ++e) {
                            const int i = b + e * kT, r = i / kUnits, u = i % kUnits, key = t * KEYS + r;
                            x[e] = make_uint4(0, 0, 0, 0);
                            if (key >= len || r >= KEYS) continue;
                            const T *src = static_cast<const T *>(a.v) + (long long)it.head * D + u * 8;
                            if constexpr (SRC == kPaged) {
                                const int blk = __ldg(a.tables + (long long)it.seq * a.table_stride + key / a.block_size);
                                if (blk < 0 || blk >= a.num_blocks) continue;
                                src += (a.layer_row0 + (long long)blk * a.block_size + key % a.block_size) * a.kv_heads * D;
                            } else {
                                src += (long long)(it.base + key) * a.kv_stride;
                            }
                            x[e] = *reinterpret_cast<const uint4 *>(src);
                        }
#pragma unroll
                        for (int e = 0; e < kBatch; ++e) {
                            const int i = b + e * kT, r = i / kUnits, u = i % kUnits;
                            if (r >= KEYS) break;
                            uint32_t wds[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
                            uint32_t bad = 0;
#pragma unroll
                            for (int k = 0; k < 4; ++k) bad |= nonfinite_mask<T>(wds[k]);
                            if (bad) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t m = nonfinite_mask<T>(wds[k]);
                                    if (m & 0x8000u) wds[k] &= 0xffff0000u;
                                    if (m & 0x80000000u) wds[k] &= 0x0000ffffu;
                                }
                                note(t * KEYS + r);
                            }
                            *reinterpret_cast<uint4 *>(dst + (u / 8) * G::kSlab + (r >> 3) * G::kGroup8 + (r & 7) * 128 + (((u % 8) ^ (r & 7)) << 4)) =
                                make_uint4(wds[0], wds[1], wds[2], wds[3]);
                        }
                    }
                    fence_async();
                    together(true);
                    if (t128 == 0) mbar_arrive(&kv_full[at % ST]);
                }
            } else {
                if (kScaleQ && n > 0) {
                    // A row's factor is kept per item (the softmax of the last item may
                    // still read the other).
                    ok = together(wait(&q_raw, qn & 1));
                    if (!ok) break;
                    // 8 lanes to a row, a 16-byte chunk of each slab to a lane.
                    for (int r0 = t128 >> 3; r0 < (it.two ? 256 : 128); r0 += 2 * (kT / 8)) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int r = r0 + k * (kT / 8);
                            uint4 *q = reinterpret_cast<uint4 *>(sq + (r >> 7) * G::kQTile + (r & 127) * 128 + (lane & 7) * 16);
                            uint4 x[G::kSlabs];
                            __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
                            for (int c = 0; c < G::kSlabs; ++c) {
                                x[c] = q[c * (128 * 128 / 16)];
                                const __nv_bfloat162 *e = reinterpret_cast<const __nv_bfloat162 *>(&x[c]);
                                most = __hmax2(most, __hmax2(__hmax2(__habs2(e[0]), __habs2(e[1])), __hmax2(__habs2(e[2]), __habs2(e[3]))));
                            }
                            float top = fmaxf(__low2float(most), __high2float(most));
#pragma unroll
                            for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            const QueryPower pw = query_power(top);
                            if ((lane & 7) == 0) q_factor[(qn & 1) * 256 + r] = pw.down;
#pragma unroll
                            for (int c = 0; c < G::kSlabs; ++c) {
                                const __nv_bfloat162 *e = reinterpret_cast<const __nv_bfloat162 *>(&x[c]);
                                uint32_t y[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) y[i] = pack2<__half>(__low2float(e[i]) * pw.up, __high2float(e[i]) * pw.up);
                                q[c * (128 * 128 / 16)] = make_uint4(y[0], y[1], y[2], y[3]);
                            }
                        }
                    }
                    ++qn;
                    fence_async();
                    together(true);
                    if (t128 == 0) mbar_arrive(&q_full);
                }
                for (int f = 0; f < 2 * n && ok; ++f) {
                    bool is_k;
                    int j;
                    const int lead = min(ahead, n), both = n - lead;
                    if (f < lead) is_k = true, j = f;
                    else if (f - lead < 2 * both) is_k = (f - lead) & 1, j = ((f - lead) >> 1) + (is_k ? ahead : 0);
                    else is_k = false, j = both + (f - lead - 2 * both);
                    const int t = it.t0 + j;
                    const unsigned at = pos + f;
                    bool good = wait(&raw_full[at % RS], (at / RS) & 1);
                    good = good && wait(&kv_empty[at % ST], ((at / ST) & 1) ^ 1);
                    ok = together(good);
                    if (!ok) break;
                    unsigned char *dst = skv + (at % ST) * G::kTile;
                    const unsigned char *src = sraw + (at % RS) * G::kRawTile;
                    const unsigned bits = s_mask[(kt + j) % kMaskRing];
                    constexpr int kUnits = D / 16;  // of 16 codes a row
                    // Value tiles with rows that some or all queries must not meet: those
                    // past the sequence or in blocks outside the pool are zeros, and NaN
                    // codes are zeros and noted.
                    const bool edge = !is_k && (t >= careful || bits != (1u << G::kGranules) - 1);
                    auto convert = [&](auto with_edge) {
#pragma unroll 4
                        for (int i = t128; i < KEYS * kUnits; i += kT) {
                            const int r = i / kUnits, u = i % kUnits;
                            uint4 x = *reinterpret_cast<const uint4 *>(src + i * 16);
                            uint32_t *w4 = reinterpret_cast<uint32_t *>(&x);
                            if constexpr (decltype(with_edge)::value) {
                                if (t * KEYS + r >= len || !((bits >> (r / 16)) & 1u)) x = make_uint4(0, 0, 0, 0);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t hit = ((w4[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                                    if (hit && t >= careful) {
                                        w4[k] &= ~((hit >> 7) * 0xffu);
                                        note(t * KEYS + r);
                                    }
                                }
                            }
                            unsigned char *row = dst + (u / 4) * G::kSlab + (r >> 3) * G::kGroup8 + (r & 7) * 128;
                            const int c = 2 * (u % 4);
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                *reinterpret_cast<uint4 *>(row + (((c + k) ^ (r & 7)) << 4)) =
                                    make_uint4(codes_to_f16(w4[2 * k]), codes_to_f16(w4[2 * k] >> 16),
                                               codes_to_f16(w4[2 * k + 1]), codes_to_f16(w4[2 * k + 1] >> 16));
                        }
                    };
                    if (edge) convert(std::true_type{});
                    else convert(std::false_type{});
                    fence_async();
                    together(true);
                    if (t128 == 0) {
                        mbar_arrive(&kv_full[at % ST]);
                        mbar_arrive(&raw_empty[at % RS]);
                    }
                }
            }
            if (!ok) break;
            pos += 2 * n;
            kt += n;
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[ring]);
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        tmem_free(tmem, 512);
    }
}

// Joins the partials of one split item, from the CTA whose share the item
// begins in on: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in the
// order of the keys. A thread takes a row and 16 of its elements; a warp's
// loads are contiguous. Bound by latency: a launch, the search for the item's
// pieces, two dependent loads: about 5 us behind the tile kernel whether few or
// many items are split. (A block of 1,024 threads for a whole row tile, 8 times
// fewer blocks: the same within 2 us on every shape tried.)
constexpr int kJoinElems = 16;
template <typename T, int D, int ROW_TILES>
__global__ void __launch_bounds__(128) prefill_join_kernel(const __grid_constant__ Params p, int ctas) {
    __shared__ int s_slot[512];
    __shared__ int s_count;
    pdl_wait();
    const PrefillLaunch &a = p.a;
    const int b = blockIdx.x, w = blockIdx.y / (D / kJoinElems), c = blockIdx.y % (D / kJoinElems) * kJoinElems;
    const Header h = p.headers[2 * b + 1];
    if (!h.state || (w && !h.two)) return;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {  // the later pieces: up to the one that ends the item
        int n = 0;
        for (int i0 = b + 1; i0 < ctas; i0 += 32) {
            const int i = i0 + lane;
            const int state = i < ctas ? p.headers[2 * i].state : 0;
            unsigned some = __ballot_sync(0xffffffffu, state);
            const unsigned end = __ballot_sync(0xffffffffu, state == 2);
            if (end) some &= (2u << (__ffs(end) - 1)) - 1;
            if ((some >> lane) & 1u) s_slot[n + __popc(some & ((1u << lane) - 1))] = 2 * i;
            n += __popc(some);
            if (end) break;
        }
        if (lane == 0) s_count = n;
    }
    __syncthreads();
    const int group = a.group, row = threadIdx.x, tau = row / group, token = tau + w * p.tile_tokens;
    if (tau >= p.tile_tokens || token >= h.tokens) return;
    const int count = s_count + 1;
    auto slot = [&](int i) { return (long long)(i == 0 ? 2 * b + 1 : s_slot[i - 1]) * ROW_TILES + w; };
    float M = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < count; ++i) M = fmaxf(M, p.part_ml[slot(i) * 128 + row].x);
    float L = 0.f, acc[kJoinElems];
#pragma unroll
    for (int e = 0; e < kJoinElems; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
        const long long at = slot(i);
        const float2 ml = p.part_ml[at * 128 + row];
        const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
        L = fmaf(ml.y, f, L);
        const float4 *o = p.part_o + (at * (D / 4) + c / 4) * 128 + row;
#pragma unroll
        for (int e = 0; e < kJoinElems / 4; ++e) {
            const float4 x = __ldcs(o + e * 128);
            acc[4 * e] = fmaf(x.x, f, acc[4 * e]);
            acc[4 * e + 1] = fmaf(x.y, f, acc[4 * e + 1]);
            acc[4 * e + 2] = fmaf(x.z, f, acc[4 * e + 2]);
            acc[4 * e + 3] = fmaf(x.w, f, acc[4 * e + 3]);
        }
    }
    const float v_scale = a.v_scale ? __ldg(a.v_scale + h.head) : 1.f;
    const float inv = L == 0.f ? 0.f : v_scale / L;
    const long long out_row = (long long)(h.row0 + token) * (a.kv_heads * group) + (long long)h.head * group + (row - tau * group);
    T *out = static_cast<T *>(a.out) + out_row * D + c;
#pragma unroll
    for (int e = 0; e < kJoinElems; e += 8)
        *reinterpret_cast<uint4 *>(out + e) =
            make_uint4(pack2<T>(acc[e] * inv, acc[e + 1] * inv), pack2<T>(acc[e + 2] * inv, acc[e + 3] * inv),
                       pack2<T>(acc[e + 4] * inv, acc[e + 5] * inv), pack2<T>(acc[e + 6] * inv, acc[e + 7] * inv));
    if (c == 0 && a.lse) a.lse[out_row] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 f = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    return f;
}

// [rows][cols] elements, row pitch `stride`, boxes of box_rows x box_cols.
bool map_2d(CUtensorMap *m, CUtensorMapDataType t, int es, const void *base, long long cols, long long rows,
            long long stride, int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(stride * es)};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    return encoder()(m, t, 2, const_cast<void *>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A pool plane as [rows / 8][slabs of 64][8 rows][64]: a box is 16 rows of a
// head, groups of 8 rows outermost, as the paged tile has them.
bool map_pages(CUtensorMap *m, CUtensorMapDataType t, const void *base, long long entry, long long rows, int slabs) {
    const cuuint64_t dims[4] = {64, 8, (cuuint64_t)(entry / 64), (cuuint64_t)(rows / 8)};
    const cuuint64_t strides[3] = {(cuuint64_t)(entry * 2), 128, (cuuint64_t)(entry * 16)};
    const cuuint32_t box[4] = {64, 8, (cuuint32_t)slabs, 2}, ones[4] = {1, 1, 1, 1};
    return encoder()(m, t, 4, const_cast<void *>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, Source SRC>
cudaError_t launch_tiles(const PrefillLaunch &a, const PrefillWorkspace &ws, int sms, cudaStream_t st) {
    using G = Geom<D, SRC>;
    if (!encoder()) return cudaErrorNotSupported;
    const CUtensorMapDataType t = std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int heads = a.kv_heads * a.group, tile_tokens = 128 / a.group;
    alignas(64) CUtensorMap tq, tk, tv;
    {
        // [tokens][heads][D]; a box is 64 elements of a tile's tokens and the group's heads: its rows in order.
        const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)a.num_tokens};
        const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.q_stride * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)tile_tokens}, ones[3] = {1, 1, 1};
        if (encoder()(&tq, t, 3, const_cast<void *>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    const long long entry = (long long)a.kv_heads * D;
    bool ok;
    if constexpr (SRC == kRows) {
        ok = map_2d(&tk, t, 2, a.k, entry, a.num_tokens, a.kv_stride, 64, G::kKeys, CU_TENSOR_MAP_SWIZZLE_128B) &&
             map_2d(&tv, t, 2, a.v, entry, a.num_tokens, a.kv_stride, 64, G::kKeys, CU_TENSOR_MAP_SWIZZLE_128B);
    } else if constexpr (SRC == kPagedFp8) {
        ok = map_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, entry, a.pool_rows, entry, D, 16, CU_TENSOR_MAP_SWIZZLE_NONE) &&
             map_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.v, entry, a.pool_rows, entry, D, 16, CU_TENSOR_MAP_SWIZZLE_NONE);
    } else {
        ok = map_pages(&tk, t, a.k, entry, a.pool_rows, D / 64) && map_pages(&tv, t, a.v, entry, a.pool_rows, D / 64);
    }
    if (!ok) return cudaErrorInvalidValue;
    const int ctas = std::min(sms, ws.ctas);
    Params p{a, tile_tokens, aligned(a.out, 32), 1.0 / ctas, nullptr, nullptr, nullptr};
    unsigned char *at = static_cast<unsigned char *>(ws.base);
    p.part_o = reinterpret_cast<float4 *>(at);
    at += (size_t)2 * ws.ctas * G::kSlotRows * D * sizeof(float);
    p.part_ml = reinterpret_cast<float2 *>(at);
    at += (size_t)2 * ws.ctas * G::kSlotRows * sizeof(float2);
    p.headers = reinterpret_cast<Header *>(at);
    auto kern = prefill_attention_kernel<T, D, SRC>;
    // Once per kernel and device.
    static std::atomic<unsigned long long> prepared{0};
    cudaError_t e;
    if (a.device >= 64 || !((prepared.load() >> a.device) & 1)) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem)) != cudaSuccess) return e;
        if (a.device < 64) prepared |= 1ull << a.device;
    }
    if ((e = launch_pdl(kern, dim3((unsigned)ctas), dim3(kPrefillThreads), G::kSmem, st, tq, tk, tv, p)) != cudaSuccess) return e;
    // Items of fewer tiles than two snaps are never split.
    if (a.max_len <= (2 * std::min(kSnapRows, kSnapKeys) - 1) * G::kKeys) return cudaSuccess;
    return launch_pdl(prefill_join_kernel<T, D, G::kRowTiles>, dim3((unsigned)ctas, G::kRowTiles * (D / kJoinElems)), dim3(128), 0, st, p, ctas);
}

template <typename T, Source SRC>
cudaError_t launch_source(const PrefillLaunch &a, const PrefillWorkspace &ws, int sms, cudaStream_t st) {
    switch (a.head_dim) {
        case 64: return launch_tiles<T, 64, SRC>(a, ws, sms, st);
        case 128: return launch_tiles<T, 128, SRC>(a, ws, sms, st);
        case 256: return launch_tiles<T, 256, SRC>(a, ws, sms, st);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_type(const PrefillLaunch &a, DType kv, const PrefillWorkspace &ws, int sms, cudaStream_t st) {
    if (!a.tables) return launch_source<T, kRows>(a, ws, sms, st);
    return kv == DType::FP8_E4M3 ? launch_source<T, kPagedFp8>(a, ws, sms, st) : launch_source<T, kPaged>(a, ws, sms, st);
}

}  // namespace

size_t prefill_workspace_bytes(int head_dim, int ctas) {
    const size_t rows = head_dim == 256 ? 128 : 256;
    return (size_t)2 * ctas * (rows * (head_dim * sizeof(float) + sizeof(float2)) + sizeof(Header));
}

cudaError_t launch_prefill_attention(const PrefillLaunch &a, DType query, DType kv, const PrefillWorkspace &ws, int sms,
                                     cudaStream_t st) {
    if (a.num_seqs <= 0 || a.num_tokens <= 0) return cudaSuccess;
    if (ws.ctas > 512) return cudaErrorInvalidValue;
    if (query == DType::BF16) return launch_type<__nv_bfloat16>(a, kv, ws, sms, st);
    if (query == DType::F16) return launch_type<__half>(a, kv, ws, sms, st);
    return cudaErrorInvalidValue;
}

}  // namespace pkv
