// Attention on the fp16 tensor cores at fp32 accuracy (adb_tc16.hpp says how an fp32 product is made of fp16 ones).
//
// The keys and values are first turned into images of 128 rows (adb_attention_images: one read and one write of them, 4 bytes
// per element each way), so that the kernel proper fetches ready operands by bulk copies however the caller's tensors
// are strided.
//
// Rows of an image are held in units of their own where they differ much in size; every loop over tiles exists a second time
// for that (BY_ROWS), so that a result is as exact as what it is made of, whatever stands beside it.
//
// Measured on 2 x 4096 tokens, 16 heads of 128, causal: images 49 us (5.5 TB/s), forward 397 us, images of the gradient's
// four operands 118 us, dq 679 us, dk and dv 973 + 15 us; at the tensor cores' own rate the products take 190, 285 and 380 us.
// With rows that differ by up to 2^40 forward and gradient take 2.55 ms instead of 2.18.  Error against 64 bits 8e-7 of a
// result's norm; fp32 products in cuBLAS: 1.7e-6.
#include <cuda_runtime.h>

#include <type_traits>

#include "adb_attention.hpp"
#include "adb_tc16.hpp"

namespace adb {
namespace {

using namespace tc16;

constexpr int KT = 128;                 // keys of a tile
// Warps that do the arithmetic between the products: PARTS threads a row, each with a share of its columns.
// (8 warps instead of 16: dk and dv 1204 us instead of 988, its code too long for the instruction cache.)
constexpr int PARTS = 4;
constexpr int SOFTMAX_WARPS = 4 * PARTS, MMA_WARP = SOFTMAX_WARPS, LOAD_WARP = SOFTMAX_WARPS + 1;
constexpr int THREADS = 32 * (SOFTMAX_WARPS + 2);
// Weights of a tile are kept in units that make the row's largest 2^15: half of fp16's smallest step, 2^-25, is 2^-40 of it,
// and a weight of 2^-18 of the row's largest still has both halves' 22 bits.
constexpr float P_SHIFT = 15.f;

// ------------------------------------------------------------------------------------------ images
struct ImageJob {
    Strided4 src;
    uint8_t* image;
    // Units of the image: one for a tile whose rows are of similar size, [batch * heads][tiles], negative where every row
    // has its own; and, in any case, row by row in whole tiles, [batch * heads][tiles * 128].
    float *scale, *rows;
    float4* docs;     // [batch][tiles]: smallest and largest document number of a tile, and whether all of its tokens are used; or null
    // for queries, in rows padded to whole tiles: the logarithm lse (+inf where a query sees nothing, so that its weights
    // vanish), and the gradient of the output times the output
    float *lse, *delta;
    int heads, tokens, tiles, of_keys, vec;
};
struct ImageArgs {
    AttentionArgs a;
    ImageJob job[4];
};

constexpr int IMAGE_WARPS = 16;
// Rows share a unit when none but rows of zeros has its largest magnitude below 2^-10 of the tile's: half of fp16's
// smallest step is then at most 2^-29 of any row's largest, 1/32 of half an fp32 step of it.
constexpr float SIMILAR = 1.f / 1024.f;

template <int P>
__global__ void __launch_bounds__(32 * IMAGE_WARPS, 2) adb_attention_images(const ImageArgs args) {
    constexpr int LPR = 16 * P, RPW = 32 / LPR, RUN = ROWS / IMAGE_WARPS, N = RUN / RPW;   // lanes of a row, rows a warp reads at a time, rows of a warp, times
    __shared__ float most[IMAGE_WARPS], least[IMAGE_WARPS];
    __shared__ int doc_lo, doc_hi, doc_gaps;
    const ImageJob& job = args.job[blockIdx.z];
    const int tile = blockIdx.x, bh = blockIdx.y;
    if (tile >= job.tiles || bh >= args.a.s.batch * job.heads) return;
    const int b = bh / job.heads, h = bh % job.heads;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = 4 * (lane % LPR), dim = int(args.a.s.dim);
    const Sight sight(args.a, b);
    const float* src = job.src.p + b * job.src.bs + h * job.src.hs;
    float4 v[N];
    float top = 0.f, low = INFINITY;   // of the rows' largest magnitudes
    auto quad = [&](const float* p, bool vec) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (vec) {
            if (c < dim) x = __ldg(reinterpret_cast<const float4*>(p));
        } else {
            if (c < dim) x.x = __ldg(p);
            if (c + 1 < dim) x.y = __ldg(p + 1);
            if (c + 2 < dim) x.z = __ldg(p + 2);
            if (c + 3 < dim) x.w = __ldg(p + 3);
        }
        return x;
    };
    auto token = [&](int i) { return tile * ROWS + warp * RUN + i * RPW + lane / LPR; };
    auto used = [&](int t) { return t < job.tokens && (job.of_keys ? sight.key_used(t) : sight.query_used(t + sight.shift)); };
    const int64_t padded0 = int64_t(bh) * job.tiles * ROWS;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = used(token(i)) ? quad(src + int64_t(token(i)) * job.src.ts + c, job.vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (job.delta) {
        const float* out = args.a.out.p + b * args.a.out.bs + h * args.a.out.hs + c;
        float4 o[N];
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = used(token(i)) ? quad(out + int64_t(token(i)) * args.a.out.ts, args.a.out_vec) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = fmaf(v[i].x, o[i].x, fmaf(v[i].y, o[i].y, fmaf(v[i].z, o[i].z, v[i].w * o[i].w)));
#pragma unroll
            for (int m = LPR / 2; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
            if (lane % LPR == 0) job.delta[padded0 + token(i)] = s;
        }
    }
    if (job.lse)
        for (int r = threadIdx.x; r < ROWS; r += 32 * IMAGE_WARPS) {
            const int t = tile * ROWS + r;
            const float x = used(t) ? __ldg(args.a.lse_in + int64_t(bh) * job.tokens + t) : -INFINITY;
            job.lse[padded0 + t] = x == -INFINITY ? INFINITY : x;
        }
    auto row_top = [&](const float4& x) {
        float m = fmaxf(fmaxf(finite_magnitude(x.x), finite_magnitude(x.y)), fmaxf(finite_magnitude(x.z), finite_magnitude(x.w)));
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    };
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float m = row_top(v[i]);
        top = fmaxf(top, m);
        low = fminf(low, m == 0.f ? INFINITY : m);
    }
    if (RPW > 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 16));
    }
    if (lane == 0) { most[warp] = top; least[warp] = low; }
    if (threadIdx.x == 0) { doc_lo = 0x7fffffff; doc_hi = -1; doc_gaps = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < IMAGE_WARPS; w++) { top = fmaxf(top, most[w]); low = fminf(low, least[w]); }
    const bool similar = low >= top * SIMILAR;
    const float scale = tile_scale(top);
    uint8_t* image = job.image + (int64_t(bh) * job.tiles + tile) * image_bytes(P);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int row = warp * RUN + i * RPW + lane / LPR;
        const float own = similar ? scale : tile_scale(row_top(v[i])), inv = 1.f / own;
        if (lane % LPR == 0) job.rows[padded0 + token(i)] = own;
        uint2 hi, lo;
        const float4 x = make_float4(v[i].x * inv, v[i].y * inv, v[i].z * inv, v[i].w * inv);
        halves(x.x, x.y, hi.x, lo.x);
        halves(x.z, x.w, hi.y, lo.y);
        const int at = (c / 64) * PANEL_BYTES + row * 128 + ((((c % 64) / 8) ^ (row & 7)) * 16) + (c % 8) * 2;
        *reinterpret_cast<uint2*>(image + at) = hi;
        *reinterpret_cast<uint2*>(image + P * PANEL_BYTES + at) = lo;
    }
    if (threadIdx.x == 0) job.scale[int64_t(bh) * job.tiles + tile] = similar ? scale : -scale;
    const bool ranges = job.docs && h == 0;
    if (ranges && threadIdx.x < ROWS) {
        const int t = tile * ROWS + threadIdx.x, at = job.of_keys ? t : t + sight.shift;
        if (t < job.tokens && (job.of_keys ? sight.key_used(t) : sight.query_used(at))) {
            const int d = __float_as_int(sight.docs[at] + 0.f);   // numbers that are not negative order like their bits
            atomicMin(&doc_lo, d);
            atomicMax(&doc_hi, d);
        } else
            doc_gaps = 1;
    }
    if (!ranges) return;
    __syncthreads();
    if (threadIdx.x == 0)
        job.docs[int64_t(b) * job.tiles + tile] =
            doc_hi < 0 ? make_float4(INFINITY, -1.f, 0.f, 0.f) : make_float4(__int_as_float(doc_lo), __int_as_float(doc_hi), doc_gaps ? 0.f : 1.f, 0.f);
}

// ------------------------------------------------------------------------------------------ which tiles of the other side count
struct Walk {
    int begin, end;              // tiles
    const float4* range;         // document numbers of runs of 128 tokens, or null
    float lo, hi;                // this block's
    int halves;                  // 1: tiles are 64 tokens, half a run
    __device__ __forceinline__ int from(int t) const {
        for (; t < end; t++) {
            if (!range) return t;
            const float4 r = __ldg(range + (t >> halves));
            if (r.x <= hi && r.y >= lo) return t;
        }
        return -1;
    }
    __device__ __forceinline__ int first() const { return from(begin); }
    // documents hide nothing between this block and tile t: all of both lie in one
    __device__ __forceinline__ bool one_document(int t) const {
        if (!range) return true;
        const float4 r = __ldg(range + (t >> halves));
        return r.z != 0.f && r.x == r.y && lo == hi && r.x == lo;
    }
    // what block blockIdx.y of gridDim.y takes of the walk
    __device__ __forceinline__ void share() {
        const int n = max(end - begin, 0), at = begin;
        begin = at + int(int64_t(n) * blockIdx.y / gridDim.y);
        end = at + int(int64_t(n) * (blockIdx.y + 1) / gridDim.y);
    }
};

// Blocks that own queries: heads go in rounds whose keys and values fit into L2 together; within a round the longest tiles of
// all heads start first, so that the SMs finish together.
__device__ __forceinline__ void own_tile(int heads, int round, int tiles, int& bh, int& tile) {
    const int first = int(blockIdx.x / unsigned(round * tiles)) * round, in = int(blockIdx.x) - first * tiles, n = min(round, heads - first);
    bh = first + in % n;
    tile = tiles - 1 - in / n;
}
int heads_in_round(const AttentionShape& s, int P) {
    const int64_t bytes = 2 * ((s.tk + ROWS - 1) / ROWS) * image_bytes(P), most = s.batch * s.heads;   // of one key head
    const int64_t n = (int64_t(48) << 20) / bytes * (s.heads / s.kv_heads);
    return int(std::max<int64_t>(1, std::min(n, most)));
}

enum : int { GAVE_UP_Q = ATTENTION_GAVE_UP, GAVE_UP_SLOT, GAVE_UP_DATA, GAVE_UP_S, GAVE_UP_P, GAVE_UP_O_FULL, GAVE_UP_O_EMPTY, GAVE_UP_MEET };

// a thread's share of a row as fp32, zero outside
template <int N>
__device__ __forceinline__ void load_row_part(const float* p, int c0, int dim, bool on, bool vec, float (&x)[N]) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) {
            if (vec) {
                if (c0 + c < dim) v = __ldg(reinterpret_cast<const float4*>(p + c0 + c));
            } else {
                if (c0 + c < dim) v.x = __ldg(p + c0 + c);
                if (c0 + c + 1 < dim) v.y = __ldg(p + c0 + c + 1);
                if (c0 + c + 2 < dim) v.z = __ldg(p + c0 + c + 2);
                if (c0 + c + 3 < dim) v.w = __ldg(p + c0 + c + 3);
            }
        }
        x[c] = v.x; x[c + 1] = v.y; x[c + 2] = v.z; x[c + 3] = v.w;
    }
}
template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < N; c++) m = fmaxf(m, finite_magnitude(x[c]));
    return m;
}
// N values of a row into tensor memory as an operand
template <int N>
__device__ __forceinline__ void store_halves(uint32_t column, const float (&x)[N], float f) {
#pragma unroll
    for (int c = 0; c < N; c += 16) tmem_store_halves(column + c, x + c, f);
}
template <int N>
__device__ __forceinline__ void store_row_part(float* p, int c0, int dim, bool vec, const float (&x)[N], float f) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        const float4 v = make_float4(x[c] * f, x[c + 1] * f, x[c + 2] * f, x[c + 3] * f);
        if (vec) {
            if (c0 + c < dim) *reinterpret_cast<float4*>(p + c0 + c) = v;
        } else {
            if (c0 + c < dim) p[c0 + c] = v.x;
            if (c0 + c + 1 < dim) p[c0 + c + 1] = v.y;
            if (c0 + c + 2 < dim) p[c0 + c + 2] = v.z;
            if (c0 + c + 3 < dim) p[c0 + c + 3] = v.w;
        }
    }
}
// Whether some of n tiles of either operand have units by row (each of `threads` threads looks at some of them).  A block
// then takes the units of all its tiles row by row, in code of its own, so that the usual case does not pay for it.
__device__ __forceinline__ bool units_by_row(const float* one, const float* other, int n, int thread, int threads) {
    bool any = false;
    for (int i = thread; i < n; i += threads) any |= fminf(__ldg(one + i), __ldg(other + i)) < 0.f;   // (both loads at once)
    return any;
}
// What a row's unit is multiplied with to give its largest magnitude, within a factor of two.
constexpr float ROW_TOP = 16384.f;
// a factor that is finite, so that zeros stay zeros
__device__ __forceinline__ float in_range(float f) { return fmaxf(fminf(f, 3.4e38f), -3.4e38f); }
// A product of units that may lie at opposite ends of the range: x * a row's factor * a column's, the factor below one first.
// Only a product that is out of range itself, or whose factors are 2^186 apart, leaves it.
struct RowFactor {
    float before, after;
    __device__ __forceinline__ explicit RowFactor(float f) : before(fabsf(f) < 1.f ? f * (1.f / ROW_TOP) : 1.f / ROW_TOP), after(fabsf(f) < 1.f ? ROW_TOP : in_range(f * ROW_TOP)) {}
    __device__ __forceinline__ float operator()(float x, float column) const { return x * before * column * after; }
};
// a tile's columns times the units of the rows they stand for (16-byte boundary) and the row's own factor
template <int N>
__device__ __forceinline__ void times_rows(uint32_t (&r)[N], const float* units, const RowFactor& own) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(units + c));
        const float f[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) r[c + e] = __float_as_uint(own(__uint_as_float(r[c + e]), f[e]));
    }
}
template <int N>
__device__ __forceinline__ void times_rows(float (&x)[N], const float* units, float factor = 1.f) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(units + c));
        const float f[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) x[c + e] *= f[e] * factor;
    }
}
// the warps that share a quadrant's rows
__device__ __forceinline__ void row_sync(int quad) { asm volatile("bar.sync %0, %1;" ::"r"(1 + quad), "n"(32 * PARTS) : "memory"); }
// largest, or sum, of what the row's threads put down
__device__ __forceinline__ float row_max(const float* cell, int row) {
    float x = cell[row];
#pragma unroll
    for (int p = 1; p < PARTS; p++) x = fmaxf(x, cell[p * ROWS + row]);
    return x;
}
__device__ __forceinline__ float row_sum(const float* cell, int row) {
    float x = cell[row];
#pragma unroll
    for (int p = 1; p < PARTS; p++) x += cell[p * ROWS + row];
    return x;
}

// A product as three: the small ones first, so that the truncating additions meet a small sum.
// First operand in tensor memory, second an image contracted over its columns.
template <int P, int PANEL>
__device__ __forceinline__ void scores_mma(uint32_t e, uint32_t d, uint32_t a, uint32_t image, uint32_t id) {
    const uint32_t b = desc_low(image, 0);
    constexpr auto at = [](int half, int j) { return uint32_t(half * P * PANEL + (j / 4) * PANEL + (j % 4) * 32) >> 4; };
#pragma unroll
    for (int j = 0; j < 4 * P; j++) {   // 16 columns each
        mma_ts(e, d, a + 16 * j + 8, b + at(0, j), id, j != 0);
        mma_ts(e, d, a + 16 * j, b + at(1, j), id, 1);
    }
#pragma unroll
    for (int j = 0; j < 4 * P; j++) mma_ts(e, d, a + 16 * j, b + at(0, j), id, 1);
}
// the same with the first operand an image of 128 rows in shared memory
template <int P, int PANEL>
__device__ __forceinline__ void scores_mma_ss(uint32_t e, uint32_t d, uint32_t own, uint32_t image, uint32_t id) {
    const uint32_t a = desc_low(own, 0), b = desc_low(image, 0);
    constexpr auto at = [](int panel, int half, int j) { return uint32_t(half * P * panel + (j / 4) * panel + (j % 4) * 32) >> 4; };
#pragma unroll
    for (int j = 0; j < 4 * P; j++) {
        mma_ss(e, d, a + at(PANEL_BYTES, 1, j), b + at(PANEL, 0, j), id, j != 0);
        mma_ss(e, d, a + at(PANEL_BYTES, 0, j), b + at(PANEL, 1, j), id, 1);
    }
#pragma unroll
    for (int j = 0; j < 4 * P; j++) mma_ss(e, d, a + at(PANEL_BYTES, 0, j), b + at(PANEL, 0, j), id, 1);
}
// first operand in tensor memory, second an image contracted over its rows, 16 at a time
template <int P, int PANEL, int STEPS>
__device__ __forceinline__ void rows_mma(uint32_t e, uint32_t d, uint32_t a, uint32_t image, uint32_t id) {
    const uint32_t b = desc_low(image, PANEL);
    constexpr auto at = [](int half, int j) { return uint32_t(half * P * PANEL + j * 2048) >> 4; };
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        mma_ts(e, d, a + 16 * j + 8, b + at(0, j), id, j != 0);
        mma_ts(e, d, a + 16 * j, b + at(1, j), id, 1);
    }
#pragma unroll
    for (int j = 0; j < STEPS; j++) mma_ts(e, d, a + 16 * j, b + at(0, j), id, 1);
}

// ------------------------------------------------------------------------------------------ forward
// A block owns 128 queries of one head; keys and values pass by in tiles of 128.  Roles:
//   loading warp, one thread    bulk copies of key and value images into a ring of three slots
//   issuing warp, one thread    S = Q K^T (into one of two buffers) and O = P V, in the order S0 S1 O0 S2 O1 ... so that the
//                               tensor cores work on S(i+1) while the weights of tile i are computed
//   16 warps                    four threads a row, a quarter of the columns each: scores out of tensor memory, the running
//                               maximum (shared between the four through shared memory), weights back as fp16 halves over
//                               the scores they came from, then O of the tile before added to the result in registers
// Q lives in tensor memory (read there, the products fetch only the other operand from shared memory, which would
// otherwise be the bound), O is drained after every tile: the tensor core truncates as it accumulates, so a sum over a
// long sequence is kept by rounded adds in registers.  Tensor memory: Q 128 columns, S 2 x 128, O 128.
struct ForwardArgs {
    AttentionArgs a;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale, *k_rows, *v_rows;
    const float4* doc_range;
    int* status;
    int q_vec, o_vec, round;
    float* partial;   // of blocks that share a tile
};

template <int P>
struct ForwardShared {
    static constexpr int SLOTS = P == 2 ? 3 : 6;
    static constexpr int SLOT_BYTES = image_bytes(P);
    static constexpr int BARS = 2 * SLOTS + 7;
    static constexpr int BYTES = 1024 + SLOTS * SLOT_BYTES + 3 * PARTS * ROWS * 4 + BARS * 8 + 16 + 2 * SOFTMAX_WARPS * 4 + 16;
};

template <int P, bool CAP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1) adb_attention_tc(const ForwardArgs f) {
    using Shared = ForwardShared<P>;
    constexpr int SLOTS = Shared::SLOTS, DP = 64 * P, SHARE = DP / PARTS, KEYS = KT / PARTS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    float* exchange = reinterpret_cast<float*>(gen + SLOTS * Shared::SLOT_BYTES);   // [3][PARTS][128]
    const uint32_t bars = base + SLOTS * Shared::SLOT_BYTES + 3 * PARTS * ROWS * 4;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (SLOTS + s); };
    auto s_full = [&](int i) { return bars + 8u * (2 * SLOTS + i); };
    auto p_ready = [&](int i) { return bars + 8u * (2 * SLOTS + 2 + i); };
    const uint32_t o_full = bars + 8u * (2 * SLOTS + 4), o_empty = o_full + 8, q_ready = o_full + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + (bars - base) + Shared::BARS * 8);
    volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* doc_span = const_cast<int*>(reinterpret_cast<volatile int*>(tmem_slot + 2));   // [2]
    volatile int* agreed = reinterpret_cast<volatile int*>(tmem_slot + 4);              // [2][SOFTMAX_WARPS]: tile parity, warp
    volatile int* by_row = agreed + 2 * SOFTMAX_WARPS;                                  // [4]: what each quadrant found

    const AttentionArgs& a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tq = int(a.s.tq), dim = int(a.s.dim), heads = int(a.s.heads), kv_heads = int(a.s.kv_heads);
    const int q_tiles = (tq + ROWS - 1) / ROWS, k_tiles = (int(a.s.tk) + KT - 1) / KT;
    int bh, tile;
    own_tile(int(a.s.batch) * heads, f.round, q_tiles, bh, tile);
    const int b = bh / heads, h = bh % heads, g = h / (heads / kv_heads), q0 = tile * ROWS;
    const Sight sight(a, b);

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { bar_init(full(s), 1); bar_init(empty(s), 1); }
        for (int i = 0; i < 2; i++) { bar_init(s_full(i), 1); bar_init(p_ready(i), SOFTMAX_WARPS); }
        bar_init(o_full, 1);
        bar_init(o_empty, SOFTMAX_WARPS);
        bar_init(q_ready, SOFTMAX_WARPS);
        *stop = by_row[0] = by_row[1] = by_row[2] = by_row[3] = 0;
        doc_span[0] = 0x7fffffff;
        doc_span[1] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(smem_u32((const void*)tmem_slot), 512);
    __syncthreads();
    if (sight.docs && threadIdx.x < ROWS && q0 + int(threadIdx.x) < tq) {
        const int pos = q0 + int(threadIdx.x) + sight.shift;
        if (sight.query_used(pos)) {
            const int d = __float_as_int(sight.docs[pos] + 0.f);
            atomicMin(&doc_span[0], d);
            atomicMax(&doc_span[1], d);
        }
    }
    const int64_t image0 = (int64_t(b) * kv_heads + g) * k_tiles;
    const int tiles_end = (max(sight.keys_end(min(q0 + ROWS, tq) - 1 + sight.shift), 0) + KT - 1) / KT;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk walk;
    walk.begin = walk.halves = 0;
    walk.end = tiles_end;
    walk.range = sight.docs ? f.doc_range + int64_t(b) * k_tiles : nullptr;
    walk.lo = sight.docs && doc_span[1] < 0 ? INFINITY : __int_as_float(doc_span[0]);
    walk.hi = doc_span[1] < 0 ? -1.f : __int_as_float(doc_span[1]);
    walk.share();

    if (warp == LOAD_WARP) {
        if (lane == 0) {
            uint32_t n = 0;
            auto fetch = [&](const uint8_t* images, int tile) {
                const int s = n % SLOTS;
                if (!bar_wait(empty(s), ((n / SLOTS) & 1) ^ 1, stop, f.status, GAVE_UP_SLOT)) return false;
                bar_expect(full(s), Shared::SLOT_BYTES);
                bulk_load(base + s * Shared::SLOT_BYTES, images + (image0 + tile) * Shared::SLOT_BYTES, Shared::SLOT_BYTES, full(s));
                n++;
                return true;
            };
            int t = walk.first();
            bool ok = t < 0 || fetch(f.k, t);
            while (ok && t >= 0) {
                const int next = walk.from(t + 1);
                ok = (next < 0 || fetch(f.k, next)) && fetch(f.v, t);
                t = next;
            }
            // copies in flight must land before the block ends (only after a wait ran out is anything left here)
            if (!ok)
                for (uint32_t k = n > SLOTS ? n - SLOTS : 0; k < n; k++)
                    for (uint32_t it = 0; it < SPIN_LIMIT && !bar_test(full(k % SLOTS), (k / SLOTS) & 1); it++) __nanosleep(64);
        }
    } else if (warp == MMA_WARP) {
        constexpr uint32_t id_s = idesc(KT, false), id_o = idesc(DP, true);
        const uint32_t e = elect(), tm = uniform(tmem), from = uniform(base);
        uint32_t n = 0;
        auto slot = [&](uint32_t k) { return from + (k % SLOTS) * Shared::SLOT_BYTES; };
        auto landed = [&](uint32_t k) { return bar_wait_warp(full(k % SLOTS), (k / SLOTS) & 1, stop, f.status, GAVE_UP_DATA); };
        int t = uniform(walk.first());
        bool ok = t < 0 || bar_wait_warp(q_ready, 0, stop, f.status, GAVE_UP_Q);
        fence_after();
        auto scores = [&](int i) {
            if (!landed(n)) return false;
            scores_mma<P, PANEL_BYTES>(e, tm + 128 + 128 * (i & 1), tm, slot(n), id_s);
            mma_commit(e, empty(n % SLOTS));
            mma_commit(e, s_full(i & 1));
            n++;
            return true;
        };
        if (ok && t >= 0) ok = scores(0);
        for (int i = 0; ok && t >= 0; i++) {
            const int next = uniform(walk.from(t + 1));
            if (next >= 0 && !scores(i + 1)) break;
            // (waits for O's drain are satisfied at once for the first tile: the barrier's phase before the first)
            if (!bar_wait_warp(p_ready(i & 1), (i >> 1) & 1, stop, f.status, GAVE_UP_P) || !bar_wait_warp(o_empty, (i & 1) ^ 1, stop, f.status, GAVE_UP_O_EMPTY) || !landed(n)) break;
            fence_after();
            rows_mma<P, PANEL_BYTES, 8>(e, tm + 384, tm + 128 + 128 * (i & 1), slot(n), id_o);
            mma_commit(e, empty(n % SLOTS));
            mma_commit(e, o_full);
            n++;
            t = next;
        }
    } else {
        const int quad = warp & 3, part = warp >> 2, row = 32 * quad + lane, q = q0 + row, pos = q + sight.shift;
        const uint32_t lanes = tmem + (uint32_t(32 * quad) << 16);
        const bool on = q < tq && sight.query_used(pos);
        const float doc = on && sight.docs ? sight.docs[pos] : 0.f;
        float q_scale;
        {
            float x[SHARE];
            load_row_part<SHARE>(a.q.p + b * a.q.bs + int64_t(on ? q : 0) * a.q.ts + h * a.q.hs, part * SHARE, dim, on, f.q_vec, x);
            if (units_by_row(f.k_scale + image0, f.v_scale + image0, tiles_end, 32 * part + lane, 32 * PARTS)) by_row[quad] = 1;
            exchange[part * ROWS + row] = largest(x);
            row_sync(quad);
            q_scale = tile_scale(row_max(exchange, row));
            store_halves<SHARE>(lanes + part * SHARE, x, 1.f / q_scale);
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(q_ready);
            row_sync(quad);
        }
        auto arithmetic = [&](auto units) {
            constexpr bool BY_ROWS = decltype(units)::value;
            const ScoreOf score(a, h);
            [[maybe_unused]] const float cap2 = score.cap2, slope2 = score.slope2;
            float acc[SHARE], m = -INFINITY, l = 0.f, keep = 0.f, v_first = 1.f, v_before = 0.f;
#pragma unroll
            for (int c = 0; c < SHARE; c++) acc[c] = 0.f;
            bool ok = true;
            auto drain = [&](int i) {   // O of tile i
                if (!bar_wait_warp(o_full, i & 1, stop, f.status, GAVE_UP_O_FULL)) return false;
                fence_after();
                uint32_t r[SHARE];
                tmem_load(lanes + 384 + part * SHARE, r);
                tmem_wait_load();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(o_empty);
                if (v_first != 1.f)
#pragma unroll
                    for (int c = 0; c < SHARE; c++) r[c] = __float_as_uint(__uint_as_float(r[c]) * v_first);
#pragma unroll
                for (int c = 0; c < SHARE; c++) acc[c] = fmaf(__uint_as_float(r[c]), v_before, acc[c] * keep);
                return true;
            };
            int i = 0;
            const int pos_first = q0 + sight.shift;
            int t = walk.first();
            bool docs_next = t >= 0 && !walk.one_document(t);
            float k_next = t >= 0 ? __ldg(f.k_scale + image0 + t) : 0.f, v_next = t >= 0 ? __ldg(f.v_scale + image0 + t) : 0.f;
            for (int next; t >= 0; t = next, i++) {
                const int k0 = t * KT + KEYS * part;
                const float mul = BY_ROWS ? 1.f : in_range(q_scale * k_next * score.mul);
                float v_scale = v_next;
                const int64_t row0 = (image0 + t) * ROWS + KEYS * part;
                const bool by_docs = docs_next;
                next = walk.from(t + 1);
                if (next >= 0) {   // a tile ahead: a load takes longer than the waits below should
                    docs_next = !walk.one_document(next);
                    k_next = __ldg(f.k_scale + image0 + next);
                    v_next = __ldg(f.v_scale + image0 + next);
                }
                // a warp that gives up still meets the others once, so that none waits for it for good
                ok = ok && bar_wait_warp(s_full(i & 1), (i >> 1) & 1, stop, f.status, GAVE_UP_S);
                fence_after();
                const uint32_t at = lanes + 128 + 128 * (i & 1) + KEYS * part;
                float s[KEYS];
                {
                    uint32_t r[KEYS];
                    tmem_load(at, r);
                    tmem_wait_load();
                    if constexpr (BY_ROWS) times_rows(r, f.k_rows + row0, RowFactor(q_scale * score.mul));
#pragma unroll
                    for (int c = 0; c < KEYS; c++) s[c] = __uint_as_float(r[c]) * mul;
                }
                if constexpr (CAP) {
#pragma unroll
                    for (int c = 0; c < KEYS; c++) s[c] = cap2 * tanh_exact(s[c]);
                }
                if constexpr (BIAS) {
                    const float away = float(pos - k0);
#pragma unroll
                    for (int c = 0; c < KEYS; c++) s[c] = fmaf(-slope2, fabsf(away - float(c)), s[c]);
                }
                const int k_last = k0 + KEYS - 1;
                if (k_last >= sight.n || by_docs || (sight.causal && k_last > pos_first && k_last >= sight.prefix)) {
                    // keys from `ahead` on are hidden by the length or the order
                    const int ahead = (sight.causal ? min(sight.n, max(pos + 1, sight.prefix)) : sight.n) - k0;
#pragma unroll
                    for (int c = 0; c < KEYS; c++)
                        if (c >= ahead || (by_docs && __ldg(sight.docs + k0 + c) != doc)) s[c] = -INFINITY;
                }
                float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < KEYS; c++) tops[c & 3] = fmaxf(tops[c & 3], s[c]);
                float* cell = exchange + (i & 1) * PARTS * ROWS;
                cell[part * ROWS + row] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                if (lane == 0) agreed[SOFTMAX_WARPS * (i & 1) + warp] = ok;
                row_sync(quad);
#pragma unroll
                for (int p = 0; p < PARTS; p++) ok = ok && agreed[SOFTMAX_WARPS * (i & 1) + 4 * p + quad];
                if (!ok) break;
                // weights in units of the tile's own largest, sums and results in units of the largest so far
                const float tile_top = row_max(cell, row), top = fmaxf(m, tile_top), base = top == -INFINITY ? 0.f : top;
                const float from = (tile_top == -INFINITY ? 0.f : tile_top) - P_SHIFT;
                const float fade = ex2(m - base), unit = ex2(tile_top - base - P_SHIFT);
                m = top;
                float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < KEYS; c++) {
                    s[c] = ex2(s[c] - from);
                    sums[c & 3] += s[c];
                }
                if constexpr (BY_ROWS) {   // the largest weight times unit of a row sets the unit of its weights
                    times_rows(s, f.v_rows + row0, 0.5f);   // (in range whatever the values are)
                    float* units = exchange + 2 * PARTS * ROWS;
                    units[part * ROWS + row] = largest(s);
                    row_sync(quad);
                    const float own = tile_scale(row_max(units, row));
                    v_scale = own * 2.f;
#pragma unroll
                    for (int c = 0; c < KEYS; c++) s[c] *= 1.f / own;
                }
                store_halves<KEYS>(at, s, 1.f);
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(p_ready(i & 1));
                l = fmaf(l, fade, ((sums[0] + sums[1]) + (sums[2] + sums[3])) * unit);
                if (i > 0) ok = drain(i - 1);
                keep = fade;
                // (two steps where the product would be a subnormal number and lose bits of its own)
                const bool tiny = v_scale < 0x1p-100f;
                v_first = tiny ? unit : 1.f;
                v_before = tiny ? v_scale : v_scale * unit;
            }
            if (ok && i > 0) ok = drain(i - 1);
            float* cell = exchange + (i & 1) * PARTS * ROWS;   // (the last tile's may still be being read)
            cell[part * ROWS + row] = l;
            row_sync(quad);
            if (ok) {
                l = row_sum(cell, row);
                if (q < tq) {
                    const bool any = on && l != 0.f;
                    if (gridDim.y > 1) {   // a share of the keys: joined with the others later
                        float* p = f.partial + ((((int64_t(b) * tq + q) * heads + h) * gridDim.y) + blockIdx.y) * (dim + 2);
                        if (!any)
#pragma unroll
                            for (int c = 0; c < SHARE; c++) acc[c] = 0.f;
                        store_row_part<SHARE>(p, part * SHARE, dim, false, acc, 1.f);
                        if (part == 0) {
                            p[dim] = any ? m : -INFINITY;
                            p[dim + 1] = any ? l : 0.f;
                        }
                    } else if (a.o) {
                        if (!any)
#pragma unroll
                            for (int c = 0; c < SHARE; c++) acc[c] = 0.f;
                        store_row_part<SHARE>(a.o + ((int64_t(b) * tq + q) * heads + h) * dim, part * SHARE, dim, f.o_vec, acc, any ? 1.f / l : 0.f);
                    }
                    if (gridDim.y == 1 && a.lse && part == 0) a.lse[int64_t(bh) * tq + q] = any ? m + log2f(l) : -INFINITY;
                }
            }
        };
        if (__builtin_expect(by_row[quad] == 0, 1)) arithmetic(std::false_type{});
        else arithmetic(std::true_type{});
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == MMA_WARP) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------------------------------ gradient
// Seven products where five would do: the scores and the weights' gradients are formed once in a kernel that owns queries
// (dq) and once in one that owns keys (dk, dv), so that every sum has one owner, nothing is added by atomics of several
// blocks and a gradient has the same bits in every run.  The other side passes by in tiles of 64 tokens, two roles fetch and
// multiply and 16 warps do the arithmetic between the products, as in the forward kernel.
//
// What goes back into tensor memory as an operand (weights and the scores' gradients) is divided by a power of two that the
// row's four threads agree on for every tile, from the largest magnitude among the 64 that they hold; the factor comes back
// when the accumulator is emptied into registers, as does the scale of the passing tile's image.  So the error of a
// gradient is a fraction of what it is made of, whatever the size of rows that it does not see.
// Accumulators are emptied into registers after every tile: each addition in tensor memory truncates, by 2^-24 of the sum
// so far on average and always towards zero, and the first keys of a causal sequence get their largest terms first
// (emptied every 8 tiles, dk and dv of 1500 tokens were off by 2.5e-6, against 1e-6 for fp32 sums).
constexpr int GT = 64;      // tokens of a passing tile
constexpr int SUB_BYTES = GT * 128;

struct GradArgs {
    AttentionArgs a;
    ImageJob k, v, q, dout;
    int* status;
    int out_vec, round;
    float *dq, *dk, *dv;   // the results, or the parts of blocks that share a tile, one behind the other
};

// half an image (64 rows): a piece for each half and panel
template <int P>
__device__ __forceinline__ void fetch_half_image(uint32_t dst, const uint8_t* images, int64_t image0, int t, uint32_t bar) {
    const uint8_t* src = images + (image0 + (t >> 1)) * image_bytes(P) + (t & 1) * SUB_BYTES;
#pragma unroll
    for (int i = 0; i < 2 * P; i++) bulk_load(dst + i * SUB_BYTES, src + i * PANEL_BYTES, SUB_BYTES, bar);
}
// The largest of what a row's four threads hold, exchanged through shared memory: meeting `count` of the quadrant's warps.
// (A barrier with a bounded wait: a warp that gave up does not come.  Two meetings in turn use different cells: a cell is
// written again only after the meeting between, to which everybody came after reading it.)
__device__ __forceinline__ bool row_largest(float& most, float* exchange, uint32_t meet, uint32_t count, int part, int row, volatile int* stop, int* status) {
    float* cell = exchange + (count & 1) * PARTS * ROWS;
    cell[part * ROWS + row] = most;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(meet);
    if (!bar_wait_warp(meet, count & 1, stop, status, GAVE_UP_MEET)) return false;
    most = row_max(cell, row);
    return true;
}

// dq.  Tensor memory (P panels): Q and dO 64 P columns each, dq 64 P, S 64, dP 64 (over which ds is written).
// Order of the products: S0 dP0 | S1 dq0 dP1 | S2 dq1 dP2 ...: the weights of tile i + 1 are computed beside dq(i) and
// dP(i+1), ds(i) beside S(i+1).
template <int P>
struct QueryGradShared {
    static constexpr int SLOTS = 3;   // of keys and of values
    static constexpr int SLOT_BYTES = 2 * P * SUB_BYTES;
    static constexpr int BARS = 4 * SLOTS + 11;
    static constexpr int BYTES = 1024 + 2 * SLOTS * SLOT_BYTES + 2 * PARTS * ROWS * 4 + BARS * 8 + 32;
};

template <int P, bool CAP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1) adb_attention_tc_dq(const GradArgs f) {
    using Shared = QueryGradShared<P>;
    constexpr int SLOTS = Shared::SLOTS, SLOT = Shared::SLOT_BYTES, DP = 64 * P, SHARE = DP / PARTS, KEYS = GT / PARTS;
    constexpr uint32_t C_Q = 0, C_DO = DP, C_DQ = 2 * DP, C_S = 3 * DP, C_DP = 3 * DP + 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    float* exchange = reinterpret_cast<float*>(gen + 2 * SLOTS * SLOT);   // [2][PARTS][128]
    const uint32_t bars = base + 2 * SLOTS * SLOT + 2 * PARTS * ROWS * 4;
    auto k_slot = [&](uint32_t n) { return base + (n % SLOTS) * SLOT; };
    auto v_slot = [&](uint32_t n) { return base + (SLOTS + n % SLOTS) * SLOT; };
    auto k_full = [&](uint32_t n) { return bars + 8u * (n % SLOTS); };
    auto k_empty = [&](uint32_t n) { return bars + 8u * (SLOTS + n % SLOTS); };
    auto v_full = [&](uint32_t n) { return bars + 8u * (2 * SLOTS + n % SLOTS); };
    auto v_empty = [&](uint32_t n) { return bars + 8u * (3 * SLOTS + n % SLOTS); };
    const uint32_t own_ready = bars + 8u * (4 * SLOTS), s_full = own_ready + 8, s_taken = own_ready + 16, dp_full = own_ready + 24,
                   ds_ready = own_ready + 32, acc_full = own_ready + 40, acc_taken = own_ready + 48, meet = own_ready + 56;   // meet: one for each quadrant
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + (bars - base) + Shared::BARS * 8);
    volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* by_row = stop + 1;   // [4]: what each quadrant found

    const AttentionArgs& a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tq = int(a.s.tq), dim = int(a.s.dim), heads = int(a.s.heads), kv_heads = int(a.s.kv_heads);
    const int q_tiles = f.q.tiles, k_tiles = f.k.tiles;
    int bh, tile;
    own_tile(int(a.s.batch) * heads, f.round, q_tiles, bh, tile);
    const int b = bh / heads, h = bh % heads, g = h / (heads / kv_heads), q0 = tile * ROWS;
    const Sight sight(a, b);
    const int64_t image0 = (int64_t(b) * kv_heads + g) * k_tiles;
    const int keys_end = max(sight.keys_end(min(q0 + ROWS, tq) - 1 + sight.shift), 0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { bar_init(k_full(s), 1); bar_init(k_empty(s), 1); bar_init(v_full(s), 1); bar_init(v_empty(s), 1); }
        bar_init(own_ready, SOFTMAX_WARPS);
        bar_init(s_full, 1);
        bar_init(s_taken, SOFTMAX_WARPS);
        bar_init(dp_full, 1);
        bar_init(ds_ready, SOFTMAX_WARPS);
        bar_init(acc_full, 1);
        bar_init(acc_taken, SOFTMAX_WARPS);
        for (int i = 0; i < 4; i++) {
            bar_init(meet + 8 * i, PARTS);
            by_row[i] = 0;
        }
        *stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(smem_u32((const void*)tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk walk;
    walk.begin = 0;
    walk.halves = 1;
    walk.end = (keys_end + GT - 1) / GT;
    walk.share();
    walk.range = sight.docs ? f.k.docs + int64_t(b) * k_tiles : nullptr;
    if (sight.docs) {
        const float4 own = __ldg(f.q.docs + int64_t(b) * q_tiles + q0 / ROWS);
        walk.lo = own.x;
        walk.hi = own.y;
    }

    if (warp == LOAD_WARP) {
        if (lane == 0) {
            uint32_t n = 0;
            bool ok = true;
            for (int t = walk.first(); t >= 0; t = walk.from(t + 1), n++) {
                const uint32_t phase = ((n / SLOTS) & 1) ^ 1;
                ok = bar_wait(k_empty(n), phase, stop, f.status, GAVE_UP_SLOT);
                if (!ok) break;
                bar_expect(k_full(n), SLOT);
                fetch_half_image<P>(k_slot(n), f.k.image, image0, t, k_full(n));
                // (a values' slot is free before its tile's keys' slot)
                ok = bar_wait(v_empty(n), phase, stop, f.status, GAVE_UP_SLOT);
                if (!ok) { n++; break; }
                bar_expect(v_full(n), SLOT);
                fetch_half_image<P>(v_slot(n), f.v.image, image0, t, v_full(n));
            }
            if (!ok)   // copies in flight must land before the block ends
                for (uint32_t k = n > SLOTS ? n - SLOTS : 0; k < n; k++)
                    for (uint32_t it = 0; it < SPIN_LIMIT && !(bar_test(k_full(k), (k / SLOTS) & 1) && bar_test(v_full(k), (k / SLOTS) & 1)); it++) __nanosleep(64);
        }
    } else if (warp == MMA_WARP) {
        constexpr uint32_t id_s = idesc(GT, false), id_acc = idesc(DP, true);
        const uint32_t e = elect(), tm = uniform(tmem), from = uniform(base);
        auto landed = [&](uint32_t bar, uint32_t n) { return bar_wait_warp(bar, (n / SLOTS) & 1, stop, f.status, GAVE_UP_DATA); };
        auto keys = [&](uint32_t n) { return from + (n % SLOTS) * SLOT; };
        auto values = [&](uint32_t n) { return from + (SLOTS + n % SLOTS) * SLOT; };
        auto s_product = [&](uint32_t n) {
            if (!landed(k_full(n), n)) return false;
            scores_mma<P, SUB_BYTES>(e, tm + C_S, tm + C_Q, keys(n), id_s);
            mma_commit(e, s_full);
            return true;
        };
        auto dp_product = [&](uint32_t n) {
            if (!landed(v_full(n), n)) return false;
            scores_mma<P, SUB_BYTES>(e, tm + C_DP, tm + C_DO, values(n), id_s);
            mma_commit(e, v_empty(n));
            mma_commit(e, dp_full);
            return true;
        };
        int t = uniform(walk.first());
        bool ok = t >= 0 && bar_wait_warp(own_ready, 0, stop, f.status, GAVE_UP_Q);
        fence_after();
        ok = ok && s_product(0) && dp_product(0);
        for (uint32_t n = 0; ok; n++) {
            const int next = uniform(walk.from(t + 1));
            if (next >= 0) {
                if (!bar_wait_warp(s_taken, n & 1, stop, f.status, GAVE_UP_S)) break;
                fence_after();
                if (!s_product(n + 1)) break;
            }
            // (for the first tile the wait for an emptied accumulator is over at once: the phase before the first)
            if (!bar_wait_warp(ds_ready, n & 1, stop, f.status, GAVE_UP_P) || !bar_wait_warp(acc_taken, (n & 1) ^ 1, stop, f.status, GAVE_UP_O_EMPTY)) break;
            fence_after();
            rows_mma<P, SUB_BYTES, 4>(e, tm + C_DQ, tm + C_DP, keys(n), id_acc);
            mma_commit(e, k_empty(n));
            mma_commit(e, acc_full);
            if (next < 0 || !dp_product(n + 1)) break;
            t = next;
        }
    } else {
        const int quad = warp & 3, part = warp >> 2, row = 32 * quad + lane, q = q0 + row, pos = q + sight.shift;
        const uint32_t lanes = tmem + (uint32_t(32 * quad) << 16);
        const bool on = q < tq && sight.query_used(pos);
        const float doc = on && sight.docs ? sight.docs[pos] : 0.f;
        const float lse = f.q.lse[int64_t(bh) * q_tiles * ROWS + q], delta = f.dout.delta[int64_t(bh) * q_tiles * ROWS + q];
        float own_scale[2];
#pragma unroll
        for (int which = 0; which < 2; which++) {
            const Strided4& src = which ? a.dout : a.q;
            float x[SHARE];
            load_row_part<SHARE>(src.p + b * src.bs + int64_t(on ? q : 0) * src.ts + h * src.hs, part * SHARE, dim, on, which ? f.dout.vec : f.q.vec, x);
            if (!which && units_by_row(f.k.scale + image0, f.v.scale + image0, (keys_end + ROWS - 1) / ROWS, 32 * part + lane, 32 * PARTS)) by_row[quad] = 1;
            exchange[part * ROWS + row] = largest(x);
            row_sync(quad);
            own_scale[which] = tile_scale(row_max(exchange, row));
            const uint32_t column = which ? C_DO : C_Q;
            store_halves<SHARE>(lanes + column + part * SHARE, x, 1.f / own_scale[which]);
            row_sync(quad);
        }
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(own_ready);
        auto arithmetic = [&](auto units) {
            constexpr bool BY_ROWS = decltype(units)::value;
            const ScoreOf score(a, h);
            float acc[SHARE], factor = 0.f;   // of the accumulator that has not been emptied yet
#pragma unroll
            for (int c = 0; c < SHARE; c++) acc[c] = 0.f;
            bool ok = true;
            uint32_t n = 0;
            auto drain = [&](uint32_t tile) {
                if (!bar_wait_warp(acc_full, tile & 1, stop, f.status, GAVE_UP_O_FULL)) return false;
                fence_after();
                uint32_t r[SHARE];
                tmem_load(lanes + C_DQ + part * SHARE, r);
                tmem_wait_load();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(acc_taken);
#pragma unroll
                for (int c = 0; c < SHARE; c++) acc[c] = fmaf(__uint_as_float(r[c]), factor, acc[c]);
                return true;
            };
            const int pos_first = q0 + sight.shift;
            int t = walk.first();
            bool docs_next = t >= 0 && !walk.one_document(t);
            float k_next = t >= 0 ? __ldg(f.k.scale + image0 + (t >> 1)) : 0.f, v_next = t >= 0 ? __ldg(f.v.scale + image0 + (t >> 1)) : 0.f;
            for (int next; t >= 0; t = next, n++) {
                const int k0 = t * GT + KEYS * part;
                const bool by_docs = docs_next;
                const float k_scale = BY_ROWS ? 1.f / ROW_TOP : k_next;
                const float mul = BY_ROWS ? 1.f : in_range(own_scale[0] * k_next * score.mul), dp_mul = BY_ROWS ? 1.f : in_range(own_scale[1] * v_next);
                const int64_t row0 = image0 * ROWS + t * GT + KEYS * part;
                next = walk.from(t + 1);
                if (next >= 0) {   // a tile ahead
                    docs_next = !walk.one_document(next);
                    k_next = __ldg(f.k.scale + image0 + (next >> 1));
                    v_next = __ldg(f.v.scale + image0 + (next >> 1));
                }
                float p[KEYS];   // weights, times the scores' bend
                uint32_t r[KEYS];
                if (!bar_wait_warp(s_full, n & 1, stop, f.status, GAVE_UP_S)) { ok = false; break; }
                fence_after();
                tmem_load(lanes + C_S + KEYS * part, r);
                tmem_wait_load();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(s_taken);
                if constexpr (BY_ROWS) times_rows(r, f.k.rows + row0, RowFactor(own_scale[0] * score.mul));
#pragma unroll
                for (int c = 0; c < KEYS; c++) {
                    float s = __uint_as_float(r[c]) * mul, bend = 1.f;
                    if constexpr (CAP) {
                        const float w = tanh_exact(s);
                        bend = fmaf(-w, w, 1.f);
                        s = score.cap2 * w;
                    }
                    if constexpr (BIAS) s = fmaf(-score.slope2, fabsf(float(pos - k0 - c)), s);
                    p[c] = CAP ? ex2(s - lse) * bend : ex2(s - lse);
                }
                const int k_last = k0 + KEYS - 1;
                if (k_last >= sight.n || by_docs || (sight.causal && k_last > pos_first && k_last >= sight.prefix)) {
                    const int ahead = (sight.causal ? min(sight.n, max(pos + 1, sight.prefix)) : sight.n) - k0;
#pragma unroll
                    for (int c = 0; c < KEYS; c++)
                        if (c >= ahead || (by_docs && __ldg(sight.docs + k0 + c) != doc)) p[c] = 0.f;
                }
                if (n > 0) ok = drain(n - 1);     // beside the product dP
                if (!ok || !bar_wait_warp(dp_full, n & 1, stop, f.status, GAVE_UP_S)) { ok = false; break; }
                fence_after();
                tmem_load(lanes + C_DP + KEYS * part, r);
                tmem_wait_load();
                if constexpr (BY_ROWS) times_rows(r, f.v.rows + row0, RowFactor(own_scale[1]));
#pragma unroll
                for (int c = 0; c < KEYS; c++) {
                    p[c] = p[c] == 0.f ? 0.f : p[c] * fmaf(__uint_as_float(r[c]), dp_mul, -delta);
                }
                if constexpr (BY_ROWS) times_rows(p, f.k.rows + row0, ROW_TOP);
                float most = 0.f;   // (an infinity may set the unit: it reaches every element of the row's sum anyway)
#pragma unroll
                for (int c = 0; c < KEYS; c++) most = fmaxf(most, fabsf(p[c]));
                if (!row_largest(most, exchange, meet + 8 * quad, n, part, row, stop, f.status)) { ok = false; break; }
                const float unit = tile_scale(most);
                factor = unit * k_scale;   // (powers of two: exact down to 2^-149)
                store_halves<KEYS>(lanes + C_DP + KEYS * part, p, 1.f / unit);
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(ds_ready);
            }
            if (ok && n > 0) ok = drain(n - 1);
            if (ok && q < tq) {
                if (!on)
#pragma unroll
                    for (int c = 0; c < SHARE; c++) acc[c] = 0.f;
                store_row_part<SHARE>(f.dq + ((int64_t(blockIdx.y) * a.s.batch + b) * tq + q) * heads * dim + h * dim, part * SHARE, dim, f.out_vec, acc, a.scale);
            }
        };
        if (__builtin_expect(by_row[quad] == 0, 1)) arithmetic(std::false_type{});
        else arithmetic(std::true_type{});
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == MMA_WARP) tmem_free(tmem, 512);
}

// dk and dv of 128 keys, over the queries of every head that shares them.  Everything is transposed: a thread's row is a key,
// its columns are queries, whose logarithms and deltas come in with the queries' images.
// Tensor memory: K 64 P columns, dk and dv 64 P each, S^T 64 (over which the weights are written), dP^T 64 (over which ds is);
// V is an operand in shared memory (two panels) or in tensor memory (one).
// Order of the products: S0 dP0 | dv0 S1 dk0 dP1 | dv1 S2 dk1 dP2 ...
template <int P>
struct KeyGradShared {
    static constexpr int SLOTS = P == 2 ? 2 : 4;   // of queries and of the outputs' gradients
    static constexpr int DATA_BYTES = 2 * P * SUB_BYTES;
    static constexpr int STATS_BYTES = 4 * GT * 4;   // of the tile's queries: logarithms, deltas, units of q and of do
    static constexpr int OWN_BYTES = P == 2 ? image_bytes(P) : 0;
    static constexpr int BARS = 4 * SLOTS + 14;
    static constexpr int BYTES = 1024 + OWN_BYTES + 2 * SLOTS * DATA_BYTES + SLOTS * STATS_BYTES + 2 * PARTS * ROWS * 4 + BARS * 8 + 16;
};

// the tiles of queries of one head after another
struct HeadWalk {
    Walk walk;
    int head, last, t;
    __device__ __forceinline__ bool start(const Walk& w, int first_head, int heads) {
        walk = w;
        head = first_head;
        last = first_head + heads - 1;
        t = walk.first();
        return t >= 0;
    }
    __device__ __forceinline__ bool next() {
        t = walk.from(t + 1);
        if (t < 0) {
            if (head == last) return false;
            head++;
            t = walk.first();
        }
        return true;
    }
};

// The arithmetic's warps hold 64 accumulators a thread; some of the registers for that come from a warpgroup that hardly
// needs any.
constexpr int KEY_THREADS = 32 * (SOFTMAX_WARPS + 4), KEY_REGS = 96, KEY_REGS_MANY = 112, KEY_REGS_FEW = 32;
static_assert(32 * SOFTMAX_WARPS * KEY_REGS_MANY + 128 * KEY_REGS_FEW <= KEY_THREADS * KEY_REGS, "the split must fit what the block was launched with");

// Two kernels: the second takes the blocks whose queries have units by row (a block of the other kernel returns at once).
// In one kernel the two loops took registers from one another: 1083 us instead of 980 for the usual one (2 x 4096 tokens, 16
// heads of 128); blocks that return take 15 of them (4 with one block an SM).
template <int P, bool CAP, bool BIAS, bool BY_ROWS>
__global__ void __launch_bounds__(KEY_THREADS, 1) adb_attention_tc_dkv(const GradArgs f) {
    using Shared = KeyGradShared<P>;
    constexpr int SLOTS = Shared::SLOTS, DATA = Shared::DATA_BYTES, STATS = Shared::STATS_BYTES, DP = 64 * P, SHARE = DP / PARTS, QUERIES = GT / PARTS;
    constexpr uint32_t C_K = 0, C_DK = DP, C_DV = 2 * DP, C_S = 3 * DP, C_DP = 3 * DP + 64, C_V = 3 * DP + 128;   // C_V: one panel only
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    constexpr int AT_DATA = Shared::OWN_BYTES, AT_STATS = AT_DATA + 2 * SLOTS * DATA, AT_EXCHANGE = AT_STATS + SLOTS * STATS,
                  AT_BARS = AT_EXCHANGE + 2 * PARTS * ROWS * 4;
    const uint32_t bars = base + AT_BARS;
    float* exchange = reinterpret_cast<float*>(gen + AT_EXCHANGE);   // [2][PARTS][128]
    auto q_slot = [&](uint32_t n) { return base + AT_DATA + (n % SLOTS) * DATA; };
    auto o_slot = [&](uint32_t n) { return base + AT_DATA + (SLOTS + n % SLOTS) * DATA; };
    auto stats = [&](uint32_t n) { return AT_STATS + int(n % SLOTS) * STATS; };
    auto q_full = [&](uint32_t n) { return bars + 8u * (n % SLOTS); };
    auto q_empty = [&](uint32_t n) { return bars + 8u * (SLOTS + n % SLOTS); };
    auto o_full = [&](uint32_t n) { return bars + 8u * (2 * SLOTS + n % SLOTS); };
    auto o_empty = [&](uint32_t n) { return bars + 8u * (3 * SLOTS + n % SLOTS); };
    const uint32_t own_ready = bars + 8u * (4 * SLOTS), own_landed = own_ready + 8, s_full = own_ready + 16, p_ready = own_ready + 24,
                   dp_full = own_ready + 32, ds_ready = own_ready + 40, dv_full = own_ready + 48, dv_taken = own_ready + 56, dk_full = own_ready + 64,
                   dk_taken = own_ready + 72, meet = own_ready + 80;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + AT_BARS + Shared::BARS * 8);
    volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const AttentionArgs& a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tq = int(a.s.tq), tk = int(a.s.tk), dim = int(a.s.dim), heads = int(a.s.heads), kv_heads = int(a.s.kv_heads), group = heads / kv_heads;
    const int q_tiles = f.q.tiles, k_tiles = f.k.tiles;
    // under a causal mask the first keys have the most queries: they start first, over all heads
    const int bg = int(blockIdx.x % unsigned(int(a.s.batch) * kv_heads)), tile = int(blockIdx.x / unsigned(int(a.s.batch) * kv_heads));
    const int b = bg / kv_heads, g = bg % kv_heads, k0 = tile * ROWS;
    const Sight sight(a, b);
    const int64_t own_image = int64_t(bg) * k_tiles + tile;
    const int64_t head0 = int64_t(b) * heads + int64_t(g) * group;   // first of the heads that share these keys

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { bar_init(q_full(s), 1); bar_init(q_empty(s), 1); bar_init(o_full(s), 1); bar_init(o_empty(s), 1); }
        bar_init(own_ready, SOFTMAX_WARPS);
        bar_init(own_landed, 1);
        bar_init(s_full, 1);
        bar_init(p_ready, SOFTMAX_WARPS);
        bar_init(dp_full, 1);
        bar_init(ds_ready, SOFTMAX_WARPS);
        bar_init(dv_full, 1);
        bar_init(dv_taken, SOFTMAX_WARPS);
        bar_init(dk_full, 1);
        bar_init(dk_taken, SOFTMAX_WARPS);
        for (int i = 0; i < 4; i++) bar_init(meet + 8 * i, PARTS);
        *stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const bool by_rows = units_by_row(f.q.scale + head0 * q_tiles, f.dout.scale + head0 * q_tiles, group * q_tiles, int(threadIdx.x), KEY_THREADS);
    if (bool(__syncthreads_or(by_rows)) != BY_ROWS) return;
    if (warp == MMA_WARP) tmem_alloc(smem_u32((const void*)tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk walk;
    walk.halves = 1;
    walk.begin = sight.causal && k0 >= sight.prefix ? max(0, k0 - sight.shift) / GT : 0;
    walk.end = k0 < sight.n ? (tq + GT - 1) / GT : 0;
    walk.share();
    walk.range = sight.docs ? f.q.docs + int64_t(b) * q_tiles : nullptr;
    if (sight.docs) {
        const float4 own = __ldg(f.k.docs + int64_t(b) * k_tiles + tile);
        walk.lo = own.x;
        walk.hi = own.y;
    }
    HeadWalk at;
    const bool any = at.start(walk, 0, group);

    if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KEY_REGS_FEW));
        if (warp == LOAD_WARP) {
            if (lane == 0 && any) {
                if constexpr (P == 2) {
                    bar_expect(own_landed, image_bytes(P));
                    bulk_load(base, f.v.image + own_image * image_bytes(P), image_bytes(P), own_landed);
                }
                uint32_t n = 0;
                bool ok = true, more = true;
                for (; more; more = at.next(), n++) {
                    const uint32_t phase = ((n / SLOTS) & 1) ^ 1;
                    const int64_t image0 = (head0 + at.head) * q_tiles, row0 = (head0 + at.head) * q_tiles * ROWS + int64_t(at.t) * GT;
                    ok = bar_wait(q_empty(n), phase, stop, f.status, GAVE_UP_SLOT);
                    if (!ok) break;
                    bar_expect(q_full(n), DATA + (BY_ROWS ? 4 : 2) * GT * 4);
                    fetch_half_image<P>(q_slot(n), f.q.image, image0, at.t, q_full(n));
                    bulk_load(base + stats(n), f.q.lse + row0, GT * 4, q_full(n));
                    bulk_load(base + stats(n) + GT * 4, f.dout.delta + row0, GT * 4, q_full(n));
                    if constexpr (BY_ROWS) {
                        bulk_load(base + stats(n) + 2 * GT * 4, f.q.rows + row0, GT * 4, q_full(n));
                        bulk_load(base + stats(n) + 3 * GT * 4, f.dout.rows + row0, GT * 4, q_full(n));
                    }
                    ok = bar_wait(o_empty(n), phase, stop, f.status, GAVE_UP_SLOT);
                    if (!ok) { n++; break; }
                    bar_expect(o_full(n), DATA);
                    fetch_half_image<P>(o_slot(n), f.dout.image, image0, at.t, o_full(n));
                }
                if (!ok) {   // copies in flight must land before the block ends
                    for (uint32_t k = n > SLOTS ? n - SLOTS : 0; k < n; k++)
                        for (uint32_t it = 0; it < SPIN_LIMIT && !(bar_test(q_full(k), (k / SLOTS) & 1) && bar_test(o_full(k), (k / SLOTS) & 1)); it++) __nanosleep(64);
                    if constexpr (P == 2)
                        for (uint32_t it = 0; it < SPIN_LIMIT && !bar_test(own_landed, 0); it++) __nanosleep(64);
                }
            }
        } else if (warp == MMA_WARP) {
            constexpr uint32_t id_s = idesc(GT, false), id_acc = idesc(DP, true);
            const uint32_t e = elect(), tm = uniform(tmem), from = uniform(base);
            auto landed = [&](uint32_t bar, uint32_t n) { return bar_wait_warp(bar, (n / SLOTS) & 1, stop, f.status, GAVE_UP_DATA); };
            auto queries = [&](uint32_t n) { return from + AT_DATA + (n % SLOTS) * DATA; };
            auto gradients = [&](uint32_t n) { return from + AT_DATA + (SLOTS + n % SLOTS) * DATA; };
            auto s_product = [&](uint32_t n) {
                if (!landed(q_full(n), n)) return false;
                scores_mma<P, SUB_BYTES>(e, tm + C_S, tm + C_K, queries(n), id_s);
                mma_commit(e, s_full);
                return true;
            };
            auto dp_product = [&](uint32_t n) {
                if (!landed(o_full(n), n)) return false;
                if constexpr (P == 1) scores_mma<P, SUB_BYTES>(e, tm + C_DP, tm + C_V, gradients(n), id_s);
                else scores_mma_ss<P, SUB_BYTES>(e, tm + C_DP, from, gradients(n), id_s);
                mma_commit(e, dp_full);
                return true;
            };
            bool ok = any && bar_wait_warp(own_ready, 0, stop, f.status, GAVE_UP_Q);
            if constexpr (P == 2) ok = ok && bar_wait_warp(own_landed, 0, stop, f.status, GAVE_UP_DATA);
            fence_after();
            ok = ok && s_product(0) && dp_product(0);
            for (uint32_t n = 0; ok; n++) {
                const bool more = uniform(int(at.next()));
                const uint32_t before = (n & 1) ^ 1;   // phase of the accumulators' emptying after the tile before
                if (!bar_wait_warp(p_ready, n & 1, stop, f.status, GAVE_UP_P) || !bar_wait_warp(dv_taken, before, stop, f.status, GAVE_UP_O_EMPTY)) break;
                fence_after();
                rows_mma<P, SUB_BYTES, 4>(e, tm + C_DV, tm + C_S, gradients(n), id_acc);
                mma_commit(e, o_empty(n));
                mma_commit(e, dv_full);
                if (more && !s_product(n + 1)) break;
                if (!bar_wait_warp(ds_ready, n & 1, stop, f.status, GAVE_UP_P) || !bar_wait_warp(dk_taken, before, stop, f.status, GAVE_UP_O_EMPTY)) break;
                fence_after();
                rows_mma<P, SUB_BYTES, 4>(e, tm + C_DK, tm + C_DP, queries(n), id_acc);
                mma_commit(e, q_empty(n));
                mma_commit(e, dk_full);
                if (!more || !dp_product(n + 1)) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KEY_REGS_MANY));
        const int quad = warp & 3, part = warp >> 2, row = 32 * quad + lane, j = k0 + row;
        const uint32_t lanes = tmem + (uint32_t(32 * quad) << 16);
        const bool on = j < tk && sight.key_used(j);
        const float doc = on && sight.docs ? sight.docs[j] : 0.f;
        const float k_scale = __ldg(f.k.rows + own_image * ROWS + row), v_scale = __ldg(f.v.rows + own_image * ROWS + row);
#pragma unroll
        for (int which = 0; which < (P == 1 ? 2 : 1); which++) {   // the block's own operands, in their images' units
            const Strided4& src = which ? a.v : a.k;
            float x[SHARE];
            load_row_part<SHARE>(src.p + b * src.bs + int64_t(on ? j : 0) * src.ts + g * src.hs, part * SHARE, dim, on, which ? f.v.vec : f.k.vec, x);
            const uint32_t column = which ? C_V : C_K;
            store_halves<SHARE>(lanes + column + part * SHARE, x, 1.f / (which ? v_scale : k_scale));
        }
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(own_ready);
        const int64_t out_row = (((int64_t(blockIdx.y) * a.s.batch + b) * tk + j) * kv_heads + g) * dim;
        bool ok = true;
        uint32_t n = 0;
        float dk[SHARE], dv[SHARE], dk_factor = 0.f, dv_factor = 0.f;   // factors: of the accumulators that have not been emptied yet
#pragma unroll
        for (int c = 0; c < SHARE; c++) dk[c] = dv[c] = 0.f;
        auto drain = [&](uint32_t full, uint32_t taken, uint32_t column, uint32_t tile, float (&acc)[SHARE], float factor) {
            if (!bar_wait_warp(full, tile & 1, stop, f.status, GAVE_UP_O_FULL)) return false;
            fence_after();
#pragma unroll
            for (int c = 0; c < SHARE; c += 16) {   // (16 at a time: registers)
                uint32_t r[16];
                tmem_load(lanes + column + part * SHARE + c, r);
                tmem_wait_load();
#pragma unroll
                for (int k = 0; k < 16; k++) acc[c + k] = fmaf(__uint_as_float(r[k]), factor, acc[c + k]);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(taken);
            return true;
        };
        float q_next = 0.f, o_next = 0.f, slope_next = 0.f;
        bool docs_next = false;
        auto look = [&]() {   // what belongs to the tile of queries that `at` stands on
            if constexpr (!BY_ROWS) {
                const int64_t image = (head0 + at.head) * q_tiles + (at.t >> 1);
                q_next = __ldg(f.q.scale + image);
                o_next = __ldg(f.dout.scale + image);
            }
            docs_next = !walk.one_document(at.t);
            if constexpr (BIAS) slope_next = __ldg(a.slopes + g * group + at.head) * LOG2E;
        };
        if (any) look();
        const ScoreOf score(a, g * group);   // (but for the slope the same for every head)
        [[maybe_unused]] const RowFactor own_q(k_scale * score.mul), own_o(v_scale);
        for (bool more = any; more; n++) {
            const int q0 = at.t * GT + QUERIES * part;   // the thread's first query
            const bool by_docs = docs_next;
            [[maybe_unused]] const float slope2 = slope_next;
            const float q_scale = BY_ROWS ? 1.f / ROW_TOP : q_next, o_scale = BY_ROWS ? 1.f / ROW_TOP : o_next;
            const float mul = BY_ROWS ? 1.f : in_range(q_next * k_scale * score.mul), dp_mul = BY_ROWS ? 1.f : in_range(o_next * v_scale);
            more = at.next();
            if (more) look();   // a tile ahead
            if (!ok || !bar_wait_warp(q_full(n), (n / SLOTS) & 1, stop, f.status, GAVE_UP_DATA) || !bar_wait_warp(s_full, n & 1, stop, f.status, GAVE_UP_S)) { ok = false; break; }
            fence_after();
            const float4* lse = reinterpret_cast<const float4*>(gen + stats(n)) + QUERIES / 4 * part;
            const float4* delta = lse + GT / 4;
            [[maybe_unused]] const float4 *q_unit = lse + 2 * GT / 4, *o_unit = lse + 3 * GT / 4;
            const bool partly = by_docs || (sight.causal && q0 + sight.shift < k0 + ROWS - 1 && k0 + ROWS - 1 >= sight.prefix);
            const int behind = sight.causal && j >= sight.prefix ? j - sight.shift - q0 : 0;   // queries in front of the key
            static_assert(QUERIES == 16, "a thread's columns of a tile");
            float p[QUERIES], most = 0.f;   // weights
            [[maybe_unused]] float bends[CAP ? QUERIES : 1];
            uint32_t r[QUERIES];
            {
                tmem_load(lanes + C_S + QUERIES * part, r);
                tmem_wait_load();
#pragma unroll
                for (int c = 0; c < QUERIES; c += 4) {
                    const float4 ls = lse[c / 4], one = make_float4(1.f, 1.f, 1.f, 1.f), qu = BY_ROWS ? q_unit[c / 4] : one, ou = BY_ROWS ? o_unit[c / 4] : one;
                    const float l4[4] = {ls.x, ls.y, ls.z, ls.w}, q4[4] = {qu.x, qu.y, qu.z, qu.w}, o4[4] = {ou.x, ou.y, ou.z, ou.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float s = BY_ROWS ? own_q(__uint_as_float(r[c + e]), q4[e]) : __uint_as_float(r[c + e]) * mul;
                        if constexpr (CAP) {
                            const float w = tanh_exact(s);
                            bends[c + e] = fmaf(-w, w, 1.f);
                            s = score.cap2 * w;
                        }
                        if constexpr (BIAS) s = fmaf(-slope2, fabsf(float(q0 + c + e + sight.shift - j)), s);
                        float w = ex2(s - l4[e]);
                        if (partly) {
                            const int q = q0 + c + e;
                            if (c + e < behind || (by_docs && (q >= tq || q + sight.shift < 0 || __ldg(sight.docs + q + sight.shift) != doc))) w = 0.f;
                        }
                        p[c + e] = w;
                        most = fmaxf(most, BY_ROWS ? w * (o4[e] * ROW_TOP) : w);
                    }
                }
                if (!row_largest(most, exchange, meet + 8 * quad, 2 * n, part, row, stop, f.status)) { ok = false; break; }
                const float unit = tile_scale(most);
                dv_factor = unit * o_scale;
                if constexpr (BY_ROWS) {
                    float x[QUERIES];
#pragma unroll
                    for (int c = 0; c < QUERIES; c += 4) {
                        const float4 ou = o_unit[c / 4];
                        const float o4[4] = {ou.x, ou.y, ou.z, ou.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) x[c + e] = p[c + e] * (o4[e] * ROW_TOP);
                    }
                    store_halves<QUERIES>(lanes + C_S + QUERIES * part, x, 1.f / unit);
                } else
                    store_halves<QUERIES>(lanes + C_S + QUERIES * part, p, 1.f / unit);
            }
            if constexpr (CAP)
#pragma unroll
                for (int c = 0; c < QUERIES; c++) p[c] *= bends[c];
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_ready);
            if (n > 0) ok = drain(dk_full, dk_taken, C_DK, n - 1, dk, dk_factor);   // beside the product dP
            if (!ok || !bar_wait_warp(dp_full, n & 1, stop, f.status, GAVE_UP_S)) { ok = false; break; }
            fence_after();
            tmem_load(lanes + C_DP + QUERIES * part, r);
            tmem_wait_load();
            most = 0.f;
#pragma unroll
            for (int c = 0; c < QUERIES; c += 4) {
                const float4 de = delta[c / 4], one = make_float4(1.f, 1.f, 1.f, 1.f), qu = BY_ROWS ? q_unit[c / 4] : one, ou = BY_ROWS ? o_unit[c / 4] : one;
                const float d4[4] = {de.x, de.y, de.z, de.w}, q4[4] = {qu.x, qu.y, qu.z, qu.w}, o4[4] = {ou.x, ou.y, ou.z, ou.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float w = BY_ROWS ? own_o(__uint_as_float(r[c + e]), o4[e]) - d4[e] : fmaf(__uint_as_float(r[c + e]), dp_mul, -d4[e]);
                    p[c + e] = p[c + e] == 0.f ? 0.f : p[c + e] * w;
                    if constexpr (BY_ROWS) p[c + e] *= q4[e] * ROW_TOP;
                    most = fmaxf(most, fabsf(p[c + e]));
                }
            }
            if (!row_largest(most, exchange, meet + 8 * quad, 2 * n + 1, part, row, stop, f.status)) { ok = false; break; }
            const float unit = tile_scale(most);
            dk_factor = unit * q_scale;   // (powers of two: exact down to 2^-149)
            store_halves<QUERIES>(lanes + C_DP + QUERIES * part, p, 1.f / unit);
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(ds_ready);
            ok = drain(dv_full, dv_taken, C_DV, n, dv, dv_factor);                  // beside the product S
        }
        if (ok && n > 0) ok = drain(dk_full, dk_taken, C_DK, n - 1, dk, dk_factor);
        if (ok && j < tk) {
            if (!on)   // no query sees the key, whatever its row was compared with
#pragma unroll
                for (int c = 0; c < SHARE; c++) dk[c] = dv[c] = 0.f;
            if (f.dk) store_row_part<SHARE>(f.dk + out_row, part * SHARE, dim, f.out_vec, dk, a.scale);
            if (f.dv) store_row_part<SHARE>(f.dv + out_row, part * SHARE, dim, f.out_vec, dv, 1.f);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == MMA_WARP) tmem_free(tmem, 512);
}

// out[i] = sum of `parts` numbers n apart, in order
__global__ void __launch_bounds__(256) adb_attention_add(const float* part, float* out, int64_t n, int parts) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        float s = part[i];
        for (int p = 1; p < parts; p++) s += part[p * n + i];
        out[i] = s;
    }
}
cudaError_t add_parts(const float* part, float* out, int64_t n, int64_t parts, int sm_count, CUstream_st* stream) {
    adb_attention_add<<<unsigned(std::min<int64_t>((n + 255) / 256, int64_t(sm_count) * 8)), 256, 0, stream>>>(part, out, n, int(parts));
    return cudaGetLastError();
}

template <class K, class A>
cudaError_t launch(K kernel, dim3 grid, int threads, int smem, CUstream_st* stream, const A& args) {
    cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<grid, threads, smem, stream>>>(args);
    return cudaGetLastError();
}

template <int P>
cudaError_t forward(const ForwardArgs& f, dim3 grid, CUstream_st* stream) {
    constexpr int smem = ForwardShared<P>::BYTES;
    const bool cap = f.a.cap > 0.f, bias = f.a.slopes != nullptr;
    if (cap) return bias ? launch(adb_attention_tc<P, true, true>, grid, THREADS, smem, stream, f) : launch(adb_attention_tc<P, true, false>, grid, THREADS, smem, stream, f);
    return bias ? launch(adb_attention_tc<P, false, true>, grid, THREADS, smem, stream, f) : launch(adb_attention_tc<P, false, false>, grid, THREADS, smem, stream, f);
}

bool aligned_rows(const float* p, int64_t dim) { return aligned16(p) && dim % 4 == 0; }

// the workspace, cut up
struct Cut {
    uint8_t* at;
    template <class T> T* take(int64_t n) {
        T* p = reinterpret_cast<T*>(at);
        at += (n * int64_t(sizeof(T)) + 255) / 256 * 256;
        return p;
    }
};
ImageJob image_job(Cut& cut, const Strided4& src, const AttentionShape& s, bool of_keys, int P) {
    ImageJob j{};
    j.src = src;
    j.of_keys = of_keys;
    j.heads = int(of_keys ? s.kv_heads : s.heads);
    j.tokens = int(of_keys ? s.tk : s.tq);
    j.tiles = (j.tokens + ROWS - 1) / ROWS;
    j.vec = fits16(src, s.dim);
    const int64_t n = s.batch * j.heads * j.tiles;
    j.image = cut.take<uint8_t>(n * image_bytes(P));
    j.scale = cut.take<float>(n);
    j.rows = cut.take<float>(n * ROWS);
    return j;
}
cudaError_t images(const ImageArgs& im, int jobs, int P, CUstream_st* stream) {
    unsigned x = 0, y = 0;
    for (int i = 0; i < jobs; i++) {
        x = std::max(x, unsigned(im.job[i].tiles));
        y = std::max(y, unsigned(im.a.s.batch * im.job[i].heads));
    }
    if (P == 1) adb_attention_images<1><<<dim3(x, y, unsigned(jobs)), 32 * IMAGE_WARPS, 0, stream>>>(im);
    else adb_attention_images<2><<<dim3(x, y, unsigned(jobs)), 32 * IMAGE_WARPS, 0, stream>>>(im);
    return cudaGetLastError();
}
template <int P, bool KEYS>
cudaError_t grad_kernel(const GradArgs& f, dim3 grid, CUstream_st* stream) {
    const bool cap = f.a.cap > 0.f, bias = f.a.slopes != nullptr;
    auto go = [&](auto c, auto s) {
        constexpr bool CAP = decltype(c)::value, BIAS = decltype(s)::value;
        if constexpr (KEYS) {
            // its warps share out the registers it is launched with: fewer than that sum would leave them waiting (the build
            // checks the compiler's count; a library built another way is refused here)
            auto one = [&](auto kernel) {
                cudaFuncAttributes attr;
                cudaError_t e = cudaFuncGetAttributes(&attr, (const void*)kernel);
                if (e != cudaSuccess) return e;
                if (attr.numRegs < KEY_REGS) return cudaErrorInvalidKernelImage;
                return launch(kernel, grid, KEY_THREADS, KeyGradShared<P>::BYTES, stream, f);
            };
            const cudaError_t e = one(adb_attention_tc_dkv<P, CAP, BIAS, false>);
            return e == cudaSuccess ? one(adb_attention_tc_dkv<P, CAP, BIAS, true>) : e;
        }
        else return launch(adb_attention_tc_dq<P, CAP, BIAS>, grid, THREADS, QueryGradShared<P>::BYTES, stream, f);
    };
    if (cap) return bias ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    return bias ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
}

}  // namespace

int attention_tc_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    const AttentionShape& s = a.s;
    const int P = attention_panels(s.dim), tiles = int((s.tk + KT - 1) / KT);
    Cut cut{reinterpret_cast<uint8_t*>(a.work)};
    ImageArgs im{};
    im.a = a;
    im.job[0] = image_job(cut, a.k, s, true, P);
    im.job[1] = image_job(cut, a.v, s, true, P);
    if (a.docs) im.job[0].docs = cut.take<float4>(s.batch * tiles);
    cudaError_t e = images(im, 2, P, stream);
    int n = 2;
    if (e == cudaSuccess) {
        ForwardArgs f{};
        f.a = a;
        f.k = im.job[0].image; f.v = im.job[1].image;
        f.k_scale = im.job[0].scale; f.v_scale = im.job[1].scale;
        f.k_rows = im.job[0].rows; f.v_rows = im.job[1].rows;
        f.doc_range = im.job[0].docs;
        f.status = a.status;
        f.q_vec = fits16(a.q, s.dim);
        f.o_vec = aligned_rows(a.o, s.dim);
        f.round = heads_in_round(s, P);
        const int64_t shares = attention_forward_shares(s, a.sm_count);
        if (shares > 1) f.partial = cut.take<float>(s.batch * s.tq * s.heads * shares * (s.dim + 2));
        const dim3 blocks(unsigned(s.batch * s.heads * attention_tc_tiles(s.tq)), unsigned(shares));
        e = P == 1 ? forward<1>(f, blocks, stream) : forward<2>(f, blocks, stream);
        if (e == cudaSuccess && shares > 1) {
            attention_join(a, int(shares), f.partial, stream);
            e = cudaGetLastError();
            n++;
        }
    }
    if (e == cudaSuccess) return n;
    err = cudaGetErrorString(e);
    return -1;
}

int attention_tc_grad_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    const AttentionShape& s = a.s;
    const int P = attention_panels(s.dim);
    Cut cut{reinterpret_cast<uint8_t*>(a.work)};
    ImageArgs im{};
    im.a = a;
    im.a.out_vec = fits16(a.out, s.dim);
    const Strided4* const src[4] = {&a.k, &a.v, &a.q, &a.dout};
    for (int i = 0; i < 4; i++) im.job[i] = image_job(cut, *src[i], s, i < 2, P);
    const int k_tiles = im.job[0].tiles, q_tiles = im.job[2].tiles;
    im.job[2].lse = cut.take<float>(s.batch * s.heads * q_tiles * ROWS);
    im.job[3].delta = cut.take<float>(s.batch * s.heads * q_tiles * ROWS);
    if (a.docs) {
        im.job[0].docs = cut.take<float4>(s.batch * k_tiles);
        im.job[2].docs = cut.take<float4>(s.batch * q_tiles);
    }
    cudaError_t e = images(im, 4, P, stream);
    int n = 1;
    GradArgs f{};
    f.a = a;
    f.k = im.job[0]; f.v = im.job[1]; f.q = im.job[2]; f.dout = im.job[3];
    f.status = a.status;
    f.round = heads_in_round(s, P);
    if (e == cudaSuccess && a.dq) {
        const int64_t shares = attention_dq_shares(s, a.sm_count), size = s.batch * s.tq * s.heads * s.dim;
        f.dq = shares > 1 ? cut.take<float>(shares * size) : a.dq;
        f.out_vec = aligned_rows(f.dq, s.dim);
        const dim3 blocks(unsigned(s.batch * s.heads * q_tiles), unsigned(shares));
        e = P == 1 ? grad_kernel<1, false>(f, blocks, stream) : grad_kernel<2, false>(f, blocks, stream);
        n++;
        if (e == cudaSuccess && shares > 1) {
            e = add_parts(f.dq, a.dq, size, shares, a.sm_count, stream);
            n++;
        }
    }
    if (e == cudaSuccess && (a.dk || a.dv)) {
        const int64_t shares = attention_dkv_shares(s, a.sm_count), size = s.batch * s.tk * s.kv_heads * s.dim;
        auto place = [&](float* out) { return out && shares > 1 ? cut.take<float>(shares * size) : out; };
        f.dk = place(a.dk);
        f.dv = place(a.dv);
        f.out_vec = aligned_rows(f.dk, s.dim) && aligned_rows(f.dv, s.dim);
        const dim3 blocks(unsigned(s.batch * s.kv_heads * k_tiles), unsigned(shares));
        e = P == 1 ? grad_kernel<1, true>(f, blocks, stream) : grad_kernel<2, true>(f, blocks, stream);
        n += 2;
        for (int i = 0; i < 2; i++) {
            float *part = i ? f.dv : f.dk, *out = i ? a.dv : a.dk;
            if (e == cudaSuccess && shares > 1 && out) {
                e = add_parts(part, out, size, shares, a.sm_count, stream);
                n++;
            }
        }
    }
    if (e == cudaSuccess) return n;
    err = cudaGetErrorString(e);
    return -1;
}

}  // namespace adb
