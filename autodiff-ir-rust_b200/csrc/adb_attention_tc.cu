// Attention on the fp16 tensor cores at fp32 accuracy (adb_tc16.hpp says how an fp32 product is made of fp16 ones).
//
// The keys and values are first turned into images of 128 rows (adb_attention_images: one read and one write of them, 4 bytes
// per element each way), so that the kernel proper fetches ready operands by bulk copies however the caller's tensors
// are strided.
#include <cuda_runtime.h>

#include "adb_attention.hpp"
#include "adb_tc16.hpp"

namespace adb {
namespace {

using namespace tc16;

constexpr int KT = 128;                 // keys of a tile
constexpr int SOFTMAX_WARPS = 8;
constexpr int THREADS = 32 * (SOFTMAX_WARPS + 2);
constexpr float P_SHIFT = 10.f;         // weights are kept 2^10 times as large: a weight of 2^-24 still has 20 bits

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ------------------------------------------------------------------------------------------ images
struct ImageJob {
    Strided4 src;
    uint8_t* image;
    float* scale;     // [batch * heads][tiles]
    float* norm;      // largest Euclidean norm of a tile's rows, or null
    int heads, tokens, tiles, of_keys, vec;
};
struct ImageArgs {
    AttentionArgs a;
    ImageJob job[4];
    float2* doc_range;   // [batch][key tiles]: smallest and largest document number, or null
};

template <int P>
__global__ void __launch_bounds__(256) adb_attention_images(const ImageArgs args) {
    constexpr int LPR = 16 * P, RPW = 32 / LPR, N = ROWS / 8 / RPW;   // lanes of a row, rows a warp reads at a time, times
    __shared__ float most[8], longest[8];
    __shared__ int doc_lo, doc_hi;
    const ImageJob& job = args.job[blockIdx.z];
    const int tile = blockIdx.x, bh = blockIdx.y;
    if (tile >= job.tiles || bh >= args.a.s.batch * job.heads) return;
    const int b = bh / job.heads, h = bh % job.heads;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = 4 * (lane % LPR), dim = int(args.a.s.dim);
    const Sight sight(args.a, b);
    const float* src = job.src.p + b * job.src.bs + h * job.src.hs;
    float4 v[N];
    float top = 0.f, len = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int t = tile * ROWS + warp * (ROWS / 8) + i * RPW + lane / LPR;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (t < job.tokens && (job.of_keys ? sight.key_used(t) : sight.query_used(t + sight.shift))) {
            const float* p = src + int64_t(t) * job.src.ts + c;
            if (job.vec) {
                if (c < dim) v[i] = __ldg(reinterpret_cast<const float4*>(p));
            } else {
                if (c < dim) v[i].x = __ldg(p);
                if (c + 1 < dim) v[i].y = __ldg(p + 1);
                if (c + 2 < dim) v[i].z = __ldg(p + 2);
                if (c + 3 < dim) v[i].w = __ldg(p + 3);
            }
        }
        top = fmaxf(fmaxf(fmaxf(top, finite_magnitude(v[i].x)), finite_magnitude(v[i].y)), fmaxf(finite_magnitude(v[i].z), finite_magnitude(v[i].w)));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) most[warp] = top;
    if (threadIdx.x == 0) { doc_lo = 0x7fffffff; doc_hi = -1; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = fmaxf(top, most[w]);
    const float scale = tile_scale(top), inv = 1.f / scale;
    uint8_t* image = job.image + (int64_t(bh) * job.tiles + tile) * image_bytes(P);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int row = warp * (ROWS / 8) + i * RPW + lane / LPR;
        uint2 hi, lo;
        const float4 x = make_float4(v[i].x * inv, v[i].y * inv, v[i].z * inv, v[i].w * inv);
        halves(x.x, x.y, hi.x, lo.x);
        halves(x.z, x.w, hi.y, lo.y);
        const int at = (c / 64) * PANEL_BYTES + row * 128 + ((((c % 64) / 8) ^ (row & 7)) * 16) + (c % 8) * 2;
        *reinterpret_cast<uint2*>(image + at) = hi;
        *reinterpret_cast<uint2*>(image + P * PANEL_BYTES + at) = lo;
        if (job.norm) {
            float s = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            len = fmaxf(len, s);
        }
    }
    if (threadIdx.x == 0) job.scale[int64_t(bh) * job.tiles + tile] = scale;
    if (job.norm) {
        if (RPW > 1) len = fmaxf(len, __shfl_xor_sync(0xffffffffu, len, 16));
        if (lane == 0) longest[warp] = len;
    }
    const bool ranges = args.doc_range && job.of_keys && blockIdx.z == 0 && h == 0;
    if (ranges && threadIdx.x < ROWS) {
        const int j = tile * ROWS + threadIdx.x;
        if (j < job.tokens && sight.key_used(j)) {
            const int d = __float_as_int(sight.docs[j] + 0.f);   // numbers that are not negative order like their bits
            atomicMin(&doc_lo, d);
            atomicMax(&doc_hi, d);
        }
    }
    if (!job.norm && !ranges) return;
    __syncthreads();
    if (threadIdx.x) return;
    if (job.norm) {
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) l = fmaxf(l, longest[w]);
        job.norm[int64_t(bh) * job.tiles + tile] = sqrtf(l) * scale;
    }
    if (ranges) args.doc_range[int64_t(b) * job.tiles + tile] = doc_hi < 0 ? make_float2(INFINITY, -1.f) : make_float2(__int_as_float(doc_lo), __int_as_float(doc_hi));
}

// ------------------------------------------------------------------------------------------ which tiles of the other side count
struct Walk {
    int begin, end;              // tiles
    const float2* range;         // document numbers of the tiles, or null
    float lo, hi;                // this block's
    __device__ __forceinline__ int from(int t) const {
        for (; t < end; t++) {
            if (!range) return t;
            const float2 r = __ldg(range + t);
            if (r.x <= hi && r.y >= lo) return t;
        }
        return -1;
    }
    __device__ __forceinline__ int first() const { return from(begin); }
};

enum : int { GAVE_UP_Q = ATTENTION_GAVE_UP, GAVE_UP_SLOT, GAVE_UP_DATA, GAVE_UP_S, GAVE_UP_P, GAVE_UP_O_FULL, GAVE_UP_O_EMPTY };

// a thread's half row of a tensor as fp32, zero outside
template <int N>
__device__ __forceinline__ void load_half_row(const float* p, int c0, int dim, bool on, bool vec, float (&x)[N]) {
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
// N values of a row into tensor memory: high halves from column `hi` on, what they leave from column `lo` on
template <int N>
__device__ __forceinline__ void store_halves(uint32_t hi, uint32_t lo, const float (&x)[N], float f) {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
        uint32_t h[16], l[16];
#pragma unroll
        for (int k = 0; k < 16; k++) halves(x[c + 2 * k] * f, x[c + 2 * k + 1] * f, h[k], l[k]);
        tmem_store16(hi + c / 2, h);
        tmem_store16(lo + c / 2, l);
    }
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
__device__ __forceinline__ void pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); }

// products with the first operand (hi, lo: `half_cols` columns apart) in tensor memory and the second an image contracted over its columns
template <int P>
__device__ __forceinline__ void scores_mma(uint32_t d, uint32_t a, uint32_t image, uint32_t panel, uint32_t half_bytes, uint32_t id) {
    constexpr int STEPS = 4 * P;   // 16 columns each
    auto b = [&](int half, int j) { return desc(image + half * half_bytes + (j / 4) * panel + (j % 4) * 32, 0, 1024); };
#pragma unroll
    for (int j = 0; j < STEPS; j++) {   // the small terms first, then the dominant one
        mma_ts(d, a + 32 * P + 8 * j, b(0, j), id, j != 0);
        mma_ts(d, a + 8 * j, b(1, j), id, 1);
    }
#pragma unroll
    for (int j = 0; j < STEPS; j++) mma_ts(d, a + 8 * j, b(0, j), id, 1);
}
// the second operand an image contracted over its rows, 16 at a time
template <int STEPS>
__device__ __forceinline__ void rows_mma(uint32_t d, uint32_t a, uint32_t image, uint32_t panel, uint32_t half_bytes, uint32_t id, bool accumulate) {
    auto b = [&](int half, int j) { return desc(image + half * half_bytes + j * 2048, panel, 1024); };
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        mma_ts(d, a + 8 * STEPS + 8 * j, b(0, j), id, accumulate || j != 0);
        mma_ts(d, a + 8 * j, b(1, j), id, 1);
    }
#pragma unroll
    for (int j = 0; j < STEPS; j++) mma_ts(d, a + 8 * j, b(0, j), id, 1);
}

// ------------------------------------------------------------------------------------------ forward
// A block owns 128 queries of one head; keys and values pass by in tiles of 128.  Roles:
//   warp 9, one thread   bulk copies of key and value images into a ring of three slots
//   warp 8, one thread   S = Q K^T (into one of two buffers) and O = P V, in the order S0 S1 O0 S2 O1 ... so that the
//                        tensor cores work on S(i+1) while the weights of tile i are computed
//   warps 0-7            two threads a row, half of the columns each: scores out of tensor memory, the running maximum
//                        (shared between the two through shared memory), weights back as fp16 halves over the scores
//                        they came from, then O of the tile before added to the result in registers
// Q lives in tensor memory (read there, the products fetch only the other operand from shared memory, which would
// otherwise be the bound), O is drained after every tile: the tensor core truncates as it accumulates, so a sum over a
// long sequence is kept by rounded adds in registers.  Tensor memory: Q 128 columns, S 2 x 128, O 128.
struct ForwardArgs {
    AttentionArgs a;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const float2* doc_range;
    int* status;
    int q_vec, o_vec;
};

template <int P>
struct ForwardShared {
    static constexpr int SLOTS = P == 2 ? 3 : 6;
    static constexpr int SLOT_BYTES = image_bytes(P);
    static constexpr int BARS = 2 * SLOTS + 7;
    static constexpr int BYTES = 1024 + SLOTS * SLOT_BYTES + 2 * 2 * ROWS * 4 + BARS * 8 + 16 + 16 * 4;
};

template <int P, bool CAP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1) adb_attention_tc(const ForwardArgs f) {
    using Shared = ForwardShared<P>;
    constexpr int SLOTS = Shared::SLOTS, DP = 64 * P, HALF = DP / 2, N_ACC = HALF;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    float* exchange = reinterpret_cast<float*>(gen + SLOTS * Shared::SLOT_BYTES);   // [2][2][128]
    const uint32_t bars = base + SLOTS * Shared::SLOT_BYTES + 2 * 2 * ROWS * 4;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (SLOTS + s); };
    auto s_full = [&](int i) { return bars + 8u * (2 * SLOTS + i); };
    auto p_ready = [&](int i) { return bars + 8u * (2 * SLOTS + 2 + i); };
    const uint32_t o_full = bars + 8u * (2 * SLOTS + 4), o_empty = o_full + 8, q_ready = o_full + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + (bars - base) + Shared::BARS * 8);
    volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* doc_span = const_cast<int*>(reinterpret_cast<volatile int*>(tmem_slot + 2));   // [2]
    volatile int* agreed = reinterpret_cast<volatile int*>(tmem_slot + 4);              // [2][2][4]: tile parity, half, quadrant

    const AttentionArgs& a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tq = int(a.s.tq), dim = int(a.s.dim), heads = int(a.s.heads), kv_heads = int(a.s.kv_heads);
    const int q_tiles = (tq + ROWS - 1) / ROWS, k_tiles = (int(a.s.tk) + KT - 1) / KT;
    const int bh = int(blockIdx.x / q_tiles), b = bh / heads, h = bh % heads, g = h / (heads / kv_heads);
    const int q0 = (q_tiles - 1 - int(blockIdx.x % q_tiles)) * ROWS;   // the longest tiles of a head start first
    const Sight sight(a, b);

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { bar_init(full(s), 1); bar_init(empty(s), 1); }
        for (int i = 0; i < 2; i++) { bar_init(s_full(i), 1); bar_init(p_ready(i), SOFTMAX_WARPS); }
        bar_init(o_full, 1);
        bar_init(o_empty, SOFTMAX_WARPS);
        bar_init(q_ready, SOFTMAX_WARPS);
        *stop = 0;
        doc_span[0] = 0x7fffffff;
        doc_span[1] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) tmem_alloc(smem_u32((const void*)tmem_slot), 512);
    __syncthreads();
    if (sight.docs && threadIdx.x < ROWS && q0 + int(threadIdx.x) < tq) {
        const int pos = q0 + int(threadIdx.x) + sight.shift;
        if (sight.query_used(pos)) {
            const int d = __float_as_int(sight.docs[pos] + 0.f);
            atomicMin(&doc_span[0], d);
            atomicMax(&doc_span[1], d);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk walk;
    walk.begin = 0;
    walk.end = (max(sight.keys_end(min(q0 + ROWS, tq) - 1 + sight.shift), 0) + KT - 1) / KT;
    walk.range = sight.docs ? f.doc_range + int64_t(b) * k_tiles : nullptr;
    walk.lo = sight.docs && doc_span[1] < 0 ? INFINITY : __int_as_float(doc_span[0]);
    walk.hi = doc_span[1] < 0 ? -1.f : __int_as_float(doc_span[1]);
    const int64_t image0 = (int64_t(b) * kv_heads + g) * k_tiles;

    if (warp == 9) {
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
    } else if (warp == 8) {
        if (lane == 0) {
            constexpr uint32_t id_s = idesc(KT, false), id_o = idesc(DP, true), half_bytes = P * PANEL_BYTES;
            uint32_t n = 0;
            auto slot = [&](uint32_t k) { return base + (k % SLOTS) * Shared::SLOT_BYTES; };
            auto landed = [&](uint32_t k) { return bar_wait(full(k % SLOTS), (k / SLOTS) & 1, stop, f.status, GAVE_UP_DATA); };
            int t = walk.first();
            bool ok = t < 0 || bar_wait(q_ready, 0, stop, f.status, GAVE_UP_Q);
            fence_after();
            auto scores = [&](int i) {
                if (!landed(n)) return false;
                scores_mma<P>(tmem + 128 + 128 * (i & 1), tmem, slot(n), PANEL_BYTES, half_bytes, id_s);
                mma_commit(empty(n % SLOTS));
                mma_commit(s_full(i & 1));
                n++;
                return true;
            };
            if (ok && t >= 0) ok = scores(0);
            for (int i = 0; ok && t >= 0; i++) {
                const int next = walk.from(t + 1);
                if (next >= 0 && !scores(i + 1)) break;
                // (waits for O's drain are satisfied at once for the first tile: the barrier's phase before the first)
                if (!bar_wait(p_ready(i & 1), (i >> 1) & 1, stop, f.status, GAVE_UP_P) || !bar_wait(o_empty, (i & 1) ^ 1, stop, f.status, GAVE_UP_O_EMPTY) || !landed(n)) break;
                fence_after();
                rows_mma<8>(tmem + 384, tmem + 128 + 128 * (i & 1), slot(n), PANEL_BYTES, half_bytes, id_o, false);
                mma_commit(empty(n % SLOTS));
                mma_commit(o_full);
                n++;
                t = next;
            }
        }
    } else {
        const int quad = warp & 3, half = warp >> 2, row = 32 * quad + lane, q = q0 + row, pos = q + sight.shift;
        const uint32_t lanes = tmem + (uint32_t(32 * quad) << 16);
        const bool on = q < tq && sight.query_used(pos);
        const float doc = on && sight.docs ? sight.docs[pos] : 0.f;
        float q_scale;
        {
            float x[HALF];
            load_half_row<HALF>(a.q.p + b * a.q.bs + int64_t(on ? q : 0) * a.q.ts + h * a.q.hs, half * HALF, dim, on, f.q_vec, x);
            exchange[half * ROWS + row] = largest(x);
            pair_sync(quad);
            q_scale = tile_scale(fmaxf(exchange[row], exchange[ROWS + row]));
            store_halves<HALF>(lanes + half * (HALF / 2), lanes + DP / 2 + half * (HALF / 2), x, 1.f / q_scale);
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(q_ready);
            pair_sync(quad);
        }
        const ScoreOf score(a, h);
        const float cap2 = score.cap2, slope2 = score.slope2;
        float acc[N_ACC], m = -INFINITY, l = 0.f, keep = 0.f, v_before = 0.f;
#pragma unroll
        for (int c = 0; c < N_ACC; c++) acc[c] = 0.f;
        bool ok = true;
        auto drain = [&](int i) {   // O of tile i
            if (!bar_wait_warp(o_full, i & 1, stop, f.status, GAVE_UP_O_FULL)) return false;
            fence_after();
#pragma unroll
            for (int c = 0; c < N_ACC; c += 32) {
                uint32_t r[32];
                tmem_load32(lanes + 384 + half * HALF + c, r);
                tmem_wait_load();
#pragma unroll
                for (int k = 0; k < 32; k++) acc[c + k] = fmaf(__uint_as_float(r[k]), v_before, acc[c + k] * keep);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(o_empty);
            return true;
        };
        int i = 0;
        const int pos_first = q0 + sight.shift;
        for (int t = walk.first(); t >= 0; t = walk.from(t + 1), i++) {
            const int k0 = t * KT + 64 * half;
            const float mul = q_scale * __ldg(f.k_scale + image0 + t) * score.mul, v_scale = __ldg(f.v_scale + image0 + t);
            // a warp that gives up still meets its partner once, so that neither waits for the other for good
            ok = ok && bar_wait_warp(s_full(i & 1), (i >> 1) & 1, stop, f.status, GAVE_UP_S);
            fence_after();
            const uint32_t at = lanes + 128 + 128 * (i & 1);
            float s[64];
            {
                uint32_t r[32];
                tmem_load32(at + 64 * half, r);
                tmem_wait_load();
#pragma unroll
                for (int c = 0; c < 32; c++) s[c] = __uint_as_float(r[c]) * mul;
                tmem_load32(at + 64 * half + 32, r);
                tmem_wait_load();
#pragma unroll
                for (int c = 0; c < 32; c++) s[32 + c] = __uint_as_float(r[c]) * mul;
            }
            if constexpr (CAP) {
#pragma unroll
                for (int c = 0; c < 64; c++) s[c] = cap2 * tanh_exact(s[c]);
            }
            if constexpr (BIAS) {
                const float away = float(pos - k0);
#pragma unroll
                for (int c = 0; c < 64; c++) s[c] = fmaf(-slope2, fabsf(away - float(c)), s[c]);
            }
            const bool partly = k0 + 63 >= sight.n || sight.docs || (sight.causal && k0 + 63 > pos_first && k0 + 63 >= sight.prefix);
            if (partly) {
                // keys from `ahead` on are hidden by the length or the order
                const int ahead = (sight.causal ? min(sight.n, max(pos + 1, sight.prefix)) : sight.n) - k0;
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (c >= ahead || (sight.docs && __ldg(sight.docs + k0 + c) != doc)) s[c] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int c = 1; c < 64; c++) top = fmaxf(top, s[c]);
            float* cell = exchange + (i & 1) * 2 * ROWS;
            cell[half * ROWS + row] = top;
            if (lane == 0) agreed[8 * (i & 1) + 4 * half + quad] = ok;
            fence_before();
            pair_sync(quad);     // both halves hold their scores: they may be overwritten
            fence_after();
            ok = agreed[8 * (i & 1) + quad] && agreed[8 * (i & 1) + 4 + quad];
            if (!ok) break;
            top = fmaxf(m, fmaxf(cell[row], cell[ROWS + row]));
            const float from = (top == -INFINITY ? 0.f : top) - P_SHIFT;
            const float fade = ex2(m - from - P_SHIFT);
            m = top;
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
                s[c] = ex2(s[c] - from);
                s[c + 1] = ex2(s[c + 1] - from);
                sum0 += s[c];
                sum1 += s[c + 1];
            }
            store_halves<64>(at + 32 * half, at + 64 + 32 * half, s, 1.f);
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_ready(i & 1));
            l = fmaf(l, fade, sum0 + sum1);
            if (i > 0) ok = drain(i - 1);
            keep = fade;
            v_before = v_scale;
        }
        if (ok && i > 0) ok = drain(i - 1);
        float* cell = exchange + (i & 1) * 2 * ROWS;   // (the last tile's may still be being read)
        cell[half * ROWS + row] = l;
        pair_sync(quad);
        if (ok) {
            l = cell[row] + cell[ROWS + row];
            if (q < tq) {
                const bool any = on && l != 0.f;
                if (a.o) {
                    if (!any)
#pragma unroll
                        for (int c = 0; c < N_ACC; c++) acc[c] = 0.f;
                    store_row_part<N_ACC>(a.o + ((int64_t(b) * tq + q) * heads + h) * dim, half * HALF, dim, f.o_vec, acc, any ? 1.f / l : 0.f);
                }
                if (a.lse && half == 0) a.lse[int64_t(bh) * tq + q] = any ? m + (log2f(l) - P_SHIFT) : -INFINITY;
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 8) tmem_free(tmem, 512);
}

bool fits16(const Strided4& t, int64_t dim) {
    return (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && dim % 4 == 0 && t.bs % 4 == 0 && t.ts % 4 == 0 && t.hs % 4 == 0;
}

template <class K, class A>
cudaError_t launch(K kernel, unsigned grid, int threads, int smem, CUstream_st* stream, const A& args) {
    cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<grid, threads, smem, stream>>>(args);
    return cudaGetLastError();
}

template <int P>
cudaError_t forward(const ForwardArgs& f, unsigned grid, CUstream_st* stream) {
    constexpr int smem = ForwardShared<P>::BYTES;
    const bool cap = f.a.cap > 0.f, bias = f.a.slopes != nullptr;
    if (cap) return bias ? launch(adb_attention_tc<P, true, true>, grid, THREADS, smem, stream, f) : launch(adb_attention_tc<P, true, false>, grid, THREADS, smem, stream, f);
    return bias ? launch(adb_attention_tc<P, false, true>, grid, THREADS, smem, stream, f) : launch(adb_attention_tc<P, false, false>, grid, THREADS, smem, stream, f);
}

// the workspace, cut up
struct Cut {
    uint8_t* at;
    template <class T> T* take(int64_t n) {
        T* p = reinterpret_cast<T*>(at);
        at += (n * int64_t(sizeof(T)) + 255) / 256 * 256;
        return p;
    }
};

}  // namespace

int attention_tc_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    const AttentionShape& s = a.s;
    const int P = attention_panels(s.dim), tiles = int((s.tk + KT - 1) / KT);
    const int64_t n = s.batch * s.kv_heads * tiles;
    Cut cut{reinterpret_cast<uint8_t*>(a.work)};
    ImageArgs im{};
    im.a = a;
    im.job[0] = {a.k, cut.take<uint8_t>(n * image_bytes(P)), cut.take<float>(n), nullptr, int(s.kv_heads), int(s.tk), tiles, 1, fits16(a.k, s.dim)};
    im.job[1] = {a.v, cut.take<uint8_t>(n * image_bytes(P)), cut.take<float>(n), nullptr, int(s.kv_heads), int(s.tk), tiles, 1, fits16(a.v, s.dim)};
    im.doc_range = a.docs ? cut.take<float2>(s.batch * tiles) : nullptr;
    const dim3 grid(unsigned(tiles), unsigned(s.batch * s.kv_heads), 2);
    if (P == 1) adb_attention_images<1><<<grid, 256, 0, stream>>>(im);
    else adb_attention_images<2><<<grid, 256, 0, stream>>>(im);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) {
        ForwardArgs f{};
        f.a = a;
        f.k = im.job[0].image; f.v = im.job[1].image;
        f.k_scale = im.job[0].scale; f.v_scale = im.job[1].scale;
        f.doc_range = im.doc_range;
        f.status = a.status;
        f.q_vec = fits16(a.q, s.dim);
        f.o_vec = (reinterpret_cast<uintptr_t>(a.o) & 15) == 0 && s.dim % 4 == 0;
        const unsigned blocks = unsigned(s.batch * s.heads * ((s.tq + ROWS - 1) / ROWS));
        e = P == 1 ? forward<1>(f, blocks, stream) : forward<2>(f, blocks, stream);
    }
    if (e == cudaSuccess) return 2;
    err = cudaGetErrorString(e);
    return -1;
}

}  // namespace adb
