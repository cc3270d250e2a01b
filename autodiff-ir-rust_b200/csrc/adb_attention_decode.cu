// Attention of a few queries against a long cache: the work is reading the keys and values once.
//
// The cache is cut into ranges of keys; a block takes one range of one key head with up to 8 of the query rows (tokens and
// heads) that share it, and a second kernel joins the ranges' maxima, sums and results in the order of the ranges.  Bound
// by HBM: 8 bytes per key and element; R query rows cost 4 R flops on the 8 bytes, within what the CUDA cores do beside it
// up to 8 rows.  Eight lanes read a key together (a lane holds every eighth quad of elements), a warp four keys at once;
// each group of eight lanes has a running maximum and sum of its own, and groups, warps and ranges meet only at the end.
// Loads go to shared memory asynchronously, three steps deep, each thread fetching what it will read itself: no barrier,
// and up to 128 KiB in flight on every SM.
//
// Measured, 32 sequences of 8192 to 16384 keys, 32 heads over 8 of 128, 3.2 GB: 475 us, the copy rate.  With loads into
// registers 960 us; through shared memory, every lane working out every row's scores, 790 us (issue 57 % busy, most of it
// that); each lane the scores of one row, 475.  One sequence of 1025 keys: 13 us with the joining kernel.
#include <cuda_runtime.h>

#include "adb_attention.hpp"

namespace adb {
namespace {

constexpr int THREADS = 256, GROUPS = THREADS / 8, STAGES = 3;
// keys a group takes at a time: a step of the block is 32 KiB (64 for the largest heads)
__host__ __device__ constexpr int step_keys(int nv) { return nv == 1 ? 4 : nv == 2 ? 2 : 1; }
__host__ __device__ constexpr int stage_quads(int nv) { return 2 * step_keys(nv) * nv * THREADS; }
static_assert(ATTENTION_SPLIT_STEP == GROUPS * 4, "keys a block takes at a time, at most");

// Sums of R numbers over eight lanes, each lane left with the one whose row it owns (8 / R lanes own a row together): a lane
// that gives half of its numbers away at each exchange needs R - 1 + log2(8 / R) of them instead of 3 R, and what follows
// from a sum (the score, its exponential) is worked out once instead of eight times.
template <int R> __device__ __forceinline__ int own_row(int l8) { return l8 * R / 8; }
template <int R>
__device__ __forceinline__ float own_sum(float (&x)[R], int l8) {
    int held = R;
#pragma unroll
    for (int m = 4; m; m >>= 1) {
        if (held > 1) {
            held /= 2;
#pragma unroll
            for (int k = 0; k < held; k++) {
                const bool upper = l8 & m;
                const float give = upper ? x[k] : x[held + k], keep = upper ? x[held + k] : x[k];
                x[k] = keep + __shfl_xor_sync(0xffffffffu, give, m);
            }
        } else
            x[0] += __shfl_xor_sync(0xffffffffu, x[0], m);
    }
    return x[0];
}

// 16 bytes, or zeros
__device__ __forceinline__ void fetch(float4* dst, const float* src, bool use) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(use ? 16 : 0) : "memory");
}

// R rows, heads of up to 32 NV elements.  partial: [rows of the whole problem][ranges][dim + 2]
template <int R, int NV>
__global__ void __launch_bounds__(THREADS, R * NV <= 16 && NV <= 4 ? 2 : 1) adb_attention_split(const AttentionArgs a, const int ranges, const int range_keys, float* partial) {
    constexpr int WARPS = THREADS / 32, STEP = step_keys(NV), QUADS = stage_quads(NV);
    extern __shared__ float4 ring[];                                    // [STAGES][keys, values][STEP][NV][THREADS]
    float4(*so)[R][NV * 8] = reinterpret_cast<float4(*)[R][NV * 8]>(ring);   // [WARPS], once the loop is over
    static_assert(WARPS * R * NV * 8 <= STAGES * QUADS, "the warps' results fit into the ring");
    __shared__ float4 sq[R][NV * 8];
    __shared__ float sm[WARPS][R], sl[WARPS][R];
    const int dim = int(a.s.dim), heads = int(a.s.heads), kv_heads = int(a.s.kv_heads), group = heads / kv_heads, tq = int(a.s.tq);
    const int rows = group * tq, chunks = (rows + R - 1) / R;
    // the key heads of the same tokens one after another: their rows lie side by side in memory
    int at = int(blockIdx.x);
    const int chunk = at % chunks;
    at /= chunks;
    const int g = at % kv_heads;
    at /= kv_heads;
    const int range = at % ranges, b = at / ranges;
    const Sight sight(a, b);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l8 = lane % 8, sub = lane / 8;

    for (int e = threadIdx.x; e < R * NV * 32; e += THREADS) {
        const int r = e / (NV * 32), c = e % (NV * 32), row = chunk * R + r, i = row / group, h = g * group + row % group;
        const bool used = row < rows && c < dim && sight.query_used(i + sight.shift);
        reinterpret_cast<float*>(sq[r])[c] = used ? __ldg(a.q.p + b * a.q.bs + int64_t(i) * a.q.ts + h * a.q.hs + c) : 0.f;
    }
    __syncthreads();
    // the row this lane owns of the R
    const int row = chunk * R + own_row<R>(l8), pos = row / group + sight.shift;
    const bool on = row < rows && sight.query_used(pos);
    const float doc = on && sight.docs ? sight.docs[pos] : 0.f;
    const ScoreOf score(a, g * group + (row < rows ? row % group : 0));
    float m = -INFINITY, l = 0.f;
    float4 acc[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int v = 0; v < NV; v++) acc[r][v] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float *kp = a.k.p + b * a.k.bs + g * a.k.hs + 4 * l8, *vp = a.v.p + b * a.v.bs + g * a.v.hs + 4 * l8;
    const int last_pos = tq - 1 + sight.shift;
    const int end = min(sight.keys_end(last_pos), (range + 1) * range_keys);
    const int first = range * range_keys + warp * 4 + sub, steps = max(0, (end - range * range_keys + GROUPS * STEP - 1) / (GROUPS * STEP));
    auto request = [&](int step) {
        if (step < steps) {
            float4* to = ring + (step % STAGES) * QUADS + threadIdx.x;
#pragma unroll
            for (int u = 0; u < STEP; u++) {
                const int j = first + (step * STEP + u) * GROUPS;
                const bool use = j < end && sight.key_used(j);
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    const bool here = use && 4 * l8 + 32 * v < dim;
                    fetch(to + (u * NV + v) * THREADS, kp + (here ? int64_t(j) * a.k.ts + 32 * v : 0), here);
                    fetch(to + ((STEP + u) * NV + v) * THREADS, vp + (here ? int64_t(j) * a.v.ts + 32 * v : 0), here);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    request(0);
    request(1);
    for (int step = 0; step < steps; step++) {
        request(step + 2);
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        const float4* from = ring + (step % STAGES) * QUADS + threadIdx.x;
        const int j0 = first + step * STEP * GROUPS;
        float dots[STEP][R];
#pragma unroll
        for (int u = 0; u < STEP; u++)
#pragma unroll
            for (int r = 0; r < R; r++) dots[u][r] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float4 x[STEP];
#pragma unroll
            for (int u = 0; u < STEP; u++) x[u] = from[(u * NV + v) * THREADS];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float4 q = sq[r][8 * v + l8];
#pragma unroll
                for (int u = 0; u < STEP; u++) dots[u][r] = fmaf(q.w, x[u].w, fmaf(q.z, x[u].z, fmaf(q.y, x[u].y, fmaf(q.x, x[u].x, dots[u][r]))));
            }
        }
        float s[STEP], top = m;
#pragma unroll
        for (int u = 0; u < STEP; u++) {
            const int j = j0 + u * GROUPS;
            float bend;
            const float dot = own_sum<R>(dots[u], l8);
            s[u] = on && j < end && sight.key_used(j) && sight.sees(pos, j, doc) ? score(dot, pos, j, bend) : -INFINITY;
            top = fmaxf(top, s[u]);
        }
        const float base = top == -INFINITY ? 0.f : top, keep = ex2(m - base);
        // (a maximum that stays needs no rescaling: every factor is one.  Maxima rise rarely after the first steps.)
        if (__any_sync(0xffffffffu, top > m)) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float f = __shfl_sync(0xffffffffu, keep, sub * 8 + r * (8 / R));
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    acc[r][v].x *= f; acc[r][v].y *= f; acc[r][v].z *= f; acc[r][v].w *= f;
                }
            }
        }
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < STEP; u++) {
            s[u] = ex2(s[u] - base);
            sum += s[u];
        }
        l = fmaf(l, keep, sum);
#pragma unroll
        for (int u = 0; u < STEP; u++) {
            float p[R];
#pragma unroll
            for (int r = 0; r < R; r++) p[r] = __shfl_sync(0xffffffffu, s[u], sub * 8 + r * (8 / R));
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const float4 x = from[((STEP + u) * NV + v) * THREADS];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    acc[r][v].x = fmaf(p[r], x.x, acc[r][v].x);
                    acc[r][v].y = fmaf(p[r], x.y, acc[r][v].y);
                    acc[r][v].z = fmaf(p[r], x.z, acc[r][v].z);
                    acc[r][v].w = fmaf(p[r], x.w, acc[r][v].w);
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // the warp's four groups, then the block's warps
#pragma unroll
    for (int r = 0; r < R; r++) {
        const float mr = __shfl_sync(0xffffffffu, m, sub * 8 + r * (8 / R)), lr = __shfl_sync(0xffffffffu, l, sub * 8 + r * (8 / R));
        float top = fmaxf(mr, __shfl_xor_sync(0xffffffffu, mr, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float keep = ex2(mr - (top == -INFINITY ? 0.f : top));
        float sum = lr * keep;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane == 0) { sm[warp][r] = top; sl[warp][r] = sum; }
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float o[4] = {acc[r][v].x * keep, acc[r][v].y * keep, acc[r][v].z * keep, acc[r][v].w * keep};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                o[e] += __shfl_xor_sync(0xffffffffu, o[e], 8);
                o[e] += __shfl_xor_sync(0xffffffffu, o[e], 16);
            }
            if (sub == 0) so[warp][r][8 * v + l8] = make_float4(o[0], o[1], o[2], o[3]);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < R * NV * 32; e += THREADS) {
        const int r = e / (NV * 32), c = e % (NV * 32), row = chunk * R + r;
        if (row >= rows || c >= dim) continue;
        float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, sm[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = ex2(sm[w][r] - base);
            sum = fmaf(sl[w][r], f, sum);
            o = fmaf(reinterpret_cast<const float*>(so[w][r])[c], f, o);
        }
        const int i = row / group, h = g * group + row % group;
        const int64_t out = (int64_t(b) * tq + i) * heads + h;
        if (ranges > 1) {
            float* p = partial + (out * ranges + range) * (dim + 2);
            p[c] = o;
            if (c == 0) { p[dim] = top; p[dim + 1] = sum; }
        } else {
            if (a.o) a.o[out * dim + c] = sum == 0.f ? 0.f : o / sum;
            if (a.lse && c == 0) a.lse[(int64_t(b) * heads + h) * tq + i] = sum == 0.f ? -INFINITY : top + log2f(sum);
        }
    }
}

// one row of the result a block
__global__ void __launch_bounds__(128) adb_attention_join(const AttentionArgs a, const int ranges, const float* partial) {
    const int dim = int(a.s.dim);
    const int64_t row = blockIdx.x;
    const float* p = partial + row * ranges * (dim + 2);
    float top = -INFINITY;
    for (int s = threadIdx.x % 32; s < ranges; s += 32) top = fmaxf(top, p[int64_t(s) * (dim + 2) + dim]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    for (int c = threadIdx.x; c < dim; c += 128) {
        float sum = 0.f, o = 0.f;
        for (int s = 0; s < ranges; s++) {
            const float* x = p + int64_t(s) * (dim + 2);
            const float f = ex2(x[dim] - base);
            sum = fmaf(x[dim + 1], f, sum);
            o = fmaf(x[c], f, o);
        }
        if (a.o) a.o[row * dim + c] = sum == 0.f ? 0.f : o / sum;
        if (a.lse && c == 0) {
            const int64_t h = row % a.s.heads, bt = row / a.s.heads, b = bt / a.s.tq, t = bt - b * a.s.tq;
            a.lse[(b * a.s.heads + h) * a.s.tq + t] = sum == 0.f ? -INFINITY : top + log2f(sum);
        }
    }
}

template <int R, int NV>
cudaError_t one(const AttentionArgs& a, unsigned grid, int ranges, int keys, CUstream_st* stream) {
    constexpr int smem = STAGES * stage_quads(NV) * int(sizeof(float4));
    const cudaError_t e = cudaFuncSetAttribute((const void*)adb_attention_split<R, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    adb_attention_split<R, NV><<<grid, THREADS, smem, stream>>>(a, ranges, keys, a.work);
    return cudaGetLastError();
}
template <int NV>
cudaError_t split(const AttentionArgs& a, int rows, int64_t blocks_of_one, int ranges, int keys, CUstream_st* stream) {
    // the fewest rows that hold them all, at most what registers take
    constexpr int MOST = NV <= 4 ? 8 : 4;
    const int R = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : MOST;
    const unsigned grid = unsigned(blocks_of_one * ((rows + R - 1) / R) * ranges);
    return R == 1   ? one<1, NV>(a, grid, ranges, keys, stream)
           : R == 2 ? one<2, NV>(a, grid, ranges, keys, stream)
           : R == 4 ? one<4, NV>(a, grid, ranges, keys, stream)
                    : one<MOST, NV>(a, grid, ranges, keys, stream);
}

}  // namespace

void attention_join(const AttentionArgs& a, int ranges, const float* partial, CUstream_st* stream) {
    adb_attention_join<<<unsigned(a.s.batch * a.s.tq * a.s.heads), 128, 0, stream>>>(a, ranges, partial);
}

int attention_split_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    const AttentionShape& s = a.s;
    const int rows = int(s.heads / s.kv_heads * s.tq), ranges = int(attention_ranges(s, a.sm_count)), keys = int(attention_range_keys(s, a.sm_count));
    const int64_t blocks = s.batch * s.kv_heads;
    cudaError_t e = s.dim <= 32    ? split<1>(a, rows, blocks, ranges, keys, stream)
                    : s.dim <= 64  ? split<2>(a, rows, blocks, ranges, keys, stream)
                    : s.dim <= 96  ? split<3>(a, rows, blocks, ranges, keys, stream)
                    : s.dim <= 128 ? split<4>(a, rows, blocks, ranges, keys, stream)
                                   : split<8>(a, rows, blocks, ranges, keys, stream);
    if (e == cudaSuccess && ranges > 1) {
        attention_join(a, ranges, a.work, stream);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) return ranges > 1 ? 2 : 1;
    err = cudaGetErrorString(e);
    return -1;
}

}  // namespace adb
