// Attention and its gradient on the CUDA cores: the general kernels, for every head size, stride and mask.  They serve heads
// of more than 128 elements, short sequences (fewer than 64 keys), few queries over keys off the 16-byte grid, batches of
// more than 65535 heads, and devices made with ADB_FLAG_SIMT_DOT.
//
//   forward   o = sum_j p_j v_j,  p = softmax of the scores; one pass over the keys with the running maximum and sum
//   gradient  p_ij = exp2(s_ij - lse_i),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i) bend_ij scale
//             dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// One block per tile of T queries (forward, dq) or T keys (dk, dv; all query heads of a key head one after another, so
// that nothing is added by atomics and a gradient has the same bits in every run).  Tiles of the other side pass through
// shared memory; a thread owns 4 x 4 scores and 4 rows of the result.  Scores, sums and results are fp32.
// Bound by fp32 FMAs fed from shared memory: 2 x 4096 tokens, 16 heads of 128, causal, forward and gradient took 34.7 ms,
// against 2.2 ms on the tensor cores.
#include <cuda_runtime.h>

#include "adb_attention.hpp"

namespace adb {
namespace {

// rows [first, first + T) of one head, zero where `used` says no; columns padded to a multiple of 4 with zeros
template <int T, class Used>
__device__ __forceinline__ void load_tile(float* dst, int ld, const float* src, int64_t ts, int first, int dim, bool vec, Used used) {
    const int quads = (dim + 3) / 4;
    for (int e = threadIdx.x; e < T * quads; e += blockDim.x) {
        const int r = e / quads, c = 4 * (e - r * quads);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (used(first + r)) {
            const float* p = src + int64_t(first + r) * ts + c;
            if (vec) v = __ldg(reinterpret_cast<const float4*>(p));
            else {
                v.x = __ldg(p);
                if (c + 1 < dim) v.y = __ldg(p + 1);
                if (c + 2 < dim) v.z = __ldg(p + 2);
                if (c + 3 < dim) v.w = __ldg(p + 3);
            }
        }
        *reinterpret_cast<float4*>(dst + r * ld + c) = v;
    }
}

__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
    return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}

// acc[i][j] = a[4 ty + i] . b[tx + (T/4) j]
template <int T>
__device__ __forceinline__ void tile_dots(const float* a, const float* b, int ld, int dim, int ty, int tx, float (&acc)[4][4]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
    for (int c = 0; c < dim; c += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * ld + c);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = *reinterpret_cast<const float4*>(b + (tx + T / 4 * j) * ld + c);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = dot4(x[i], y[j], acc[i][j]);
    }
}

// acc[i][c] += sum_k w(k, 4 ty + i) * b[k][column c of the thread].  ROWS: w is held [row][k], else [k][row].
template <int T, int NC, bool ROWS>
__device__ __forceinline__ void tile_accumulate(const float* w, const float* b, int ld, int dim, int ty, int tx, float4 (&acc)[4][NC]) {
    constexpr int LW = T + 4;
    for (int k = 0; k < T; k++) {
        float x[4];
        if constexpr (ROWS) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = w[(4 * ty + i) * LW + k];
        } else {
            const float4 t = *reinterpret_cast<const float4*>(w + k * LW + 4 * ty);
            x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
        }
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int col = 4 * tx + T * c;
            if (col >= dim) break;
            const float4 y = *reinterpret_cast<const float4*>(b + k * ld + col);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                acc[i][c].x = fmaf(x[i], y.x, acc[i][c].x);
                acc[i][c].y = fmaf(x[i], y.y, acc[i][c].y);
                acc[i][c].z = fmaf(x[i], y.z, acc[i][c].z);
                acc[i][c].w = fmaf(x[i], y.w, acc[i][c].w);
            }
        }
    }
}

// columns of row `dst` that the thread owns, multiplied by f (f = 0: zeros, whatever the sum met on its way)
template <int T, int NC>
__device__ __forceinline__ void store_columns(float* dst, const float4 (&v)[NC], float f, int dim, int tx) {
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = 4 * tx + T * c;
        if (col < dim) dst[col] = f == 0.f ? 0.f : v[c].x * f;
        if (col + 1 < dim) dst[col + 1] = f == 0.f ? 0.f : v[c].y * f;
        if (col + 2 < dim) dst[col + 2] = f == 0.f ? 0.f : v[c].z * f;
        if (col + 3 < dim) dst[col + 3] = f == 0.f ? 0.f : v[c].w * f;
    }
}

template <int W> __device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int o = W / 2; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
template <int W> __device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int o = W / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

struct Vec { bool q, k, v, out, dout; };

__host__ __device__ constexpr int padded(int dim) { return (dim + 3) / 4 * 4 + 4; }

// T x T tiles, (T / 4)^2 threads; NC: groups of T columns of the result (NC * T >= dim)
template <int T, int NC>
__global__ void __launch_bounds__((T / 4) * (T / 4)) adb_attention_simt(const AttentionArgs a, const Vec vec) {
    extern __shared__ float4 raw[];
    const int dim = int(a.s.dim), ld = padded(dim), tq = int(a.s.tq);
    float* sq = reinterpret_cast<float*>(raw);
    float *sk = sq + T * ld, *sv = sk + T * ld, *sp = sv + T * ld;
    const int tx = threadIdx.x % (T / 4), ty = threadIdx.x / (T / 4);
    const int tiles = (tq + T - 1) / T;
    const int64_t bh = blockIdx.x / tiles;
    const int heads = int(a.s.heads), b = int(bh / heads), h = int(bh % heads), g = h / (heads / int(a.s.kv_heads));
    const int q0 = (tiles - 1 - int(blockIdx.x % tiles)) * T;   // under a causal mask the longest tiles of a head start first
    const Sight sight(a, b);
    const ScoreOf score(a, h);
    auto query_used = [&](int i) { return i < tq && sight.query_used(i + sight.shift); };
    auto key_used = [&](int j) { return sight.key_used(j); };
    load_tile<T>(sq, ld, a.q.p + b * a.q.bs + h * a.q.hs, a.q.ts, q0, dim, vec.q, query_used);
    float m[4], l[4], doc[4];
    bool on[4];
    float4 acc[4][NC];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        m[i] = -INFINITY;
        l[i] = 0.f;
        on[i] = query_used(q0 + 4 * ty + i);
        doc[i] = on[i] && sight.docs ? sight.docs[q0 + 4 * ty + i + sight.shift] : 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int end = sight.keys_end(min(q0 + T, tq) - 1 + sight.shift);
    for (int k0 = 0; k0 < end; k0 += T) {
        __syncthreads();
        load_tile<T>(sk, ld, a.k.p + b * a.k.bs + g * a.k.hs, a.k.ts, k0, dim, vec.k, key_used);
        load_tile<T>(sv, ld, a.v.p + b * a.v.bs + g * a.v.hs, a.v.ts, k0, dim, vec.v, key_used);
        __syncthreads();
        float s[4][4];
        tile_dots<T>(sq, sk, ld, dim, ty, tx, s);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int pos = q0 + 4 * ty + i + sight.shift;
            float top = -INFINITY, bend;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int key = k0 + tx + T / 4 * j;
                s[i][j] = on[i] && key_used(key) && sight.sees(pos, key, doc[i]) ? score(s[i][j], pos, key, bend) : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
            const float next = fmaxf(m[i], lanes_max<T / 4>(top));
            const float base = next == -INFINITY ? 0.f : next;
            const float keep = exp2f(m[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = exp2f(s[i][j] - base);
                sum += s[i][j];
                sp[(4 * ty + i) * (T + 4) + tx + T / 4 * j] = s[i][j];
            }
            l[i] = l[i] * keep + lanes_sum<T / 4>(sum);
            m[i] = next;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                acc[i][c].x *= keep; acc[i][c].y *= keep; acc[i][c].z *= keep; acc[i][c].w *= keep;
            }
        }
        __syncwarp();   // a row's scores are written and read by the T / 4 lanes that share it
        tile_accumulate<T, NC, true>(sp, sv, ld, dim, ty, tx, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int q = q0 + 4 * ty + i;
        if (q >= tq) break;
        if (a.o) store_columns<T, NC>(a.o + ((int64_t(b) * tq + q) * heads + h) * dim, acc[i], l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]), dim, tx);
        if (a.lse && tx == 0) a.lse[bh * tq + q] = l[i] > 0.f ? m[i] + log2f(l[i]) : (l[i] == 0.f ? -INFINITY : l[i]);
    }
}

// delta[b, h, i] = do . o, a warp for each
__global__ void __launch_bounds__(256) adb_attention_delta(const AttentionArgs a) {
    const int64_t at = int64_t(blockIdx.x) * 8 + threadIdx.x / 32, n = a.s.batch * a.s.heads * a.s.tq;
    if (at >= n) return;
    // tokens outermost, so that neighbouring warps read neighbouring heads
    const int64_t h = at % a.s.heads, bt = at / a.s.heads, b = bt / a.s.tq, t = bt - b * a.s.tq;
    const Sight sight(a, b);
    float s = 0.f;
    if (sight.query_used(int(t) + sight.shift)) {
        const float *x = a.out.p + b * a.out.bs + t * a.out.ts + h * a.out.hs, *y = a.dout.p + b * a.dout.bs + t * a.dout.ts + h * a.dout.hs;
        for (int c = threadIdx.x % 32; c < a.s.dim; c += 32) s = fmaf(x[c], y[c], s);
        s = lanes_sum<32>(s);
    }
    if (threadIdx.x % 32 == 0) a.work[(b * a.s.heads + h) * a.s.tq + t] = s;
}

// the probabilities and the scores' gradients of a tile pair, both times what the sums need; rows are queries
template <int T>
__device__ __forceinline__ void grad_tile(const AttentionArgs& a, const Sight& sight, const ScoreOf& score, const float* sq, const float* sk,
                                          const float* sdo, const float* sv, int ld, int dim, int q0, int k0, int ty, int tx,
                                          const float* lse, const float* delta, float* sp, float* sds) {
    constexpr int LW = T + 4;
    float s[4][4], dp[4][4];
    tile_dots<T>(sq, sk, ld, dim, ty, tx, s);
    tile_dots<T>(sdo, sv, ld, dim, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int q = q0 + 4 * ty + i, pos = q + sight.shift;
        const bool on = q < a.s.tq && sight.query_used(pos);
        const float doc = on && sight.docs ? sight.docs[pos] : 0.f;
        const float ls = on ? lse[q] : 0.f, de = on ? delta[q] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int key = k0 + tx + T / 4 * j;
            float p = 0.f, ds = 0.f, bend;
            if (on && sight.key_used(key) && sight.sees(pos, key, doc)) {
                p = exp2f(score(s[i][j], pos, key, bend) - ls);
                ds = p * (dp[i][j] - de) * bend * a.scale;
            }
            if (sp) sp[(4 * ty + i) * LW + tx + T / 4 * j] = p;
            sds[(4 * ty + i) * LW + tx + T / 4 * j] = ds;
        }
    }
}

template <int T, int NC>
__global__ void __launch_bounds__((T / 4) * (T / 4)) adb_attention_simt_dq(const AttentionArgs a, const Vec vec) {
    extern __shared__ float4 raw[];
    const int dim = int(a.s.dim), ld = padded(dim), tq = int(a.s.tq);
    float* sq = reinterpret_cast<float*>(raw);
    float *sdo = sq + T * ld, *sk = sdo + T * ld, *sv = sk + T * ld, *sds = sv + T * ld;
    const int tx = threadIdx.x % (T / 4), ty = threadIdx.x / (T / 4);
    const int tiles = (tq + T - 1) / T;
    const int64_t bh = blockIdx.x / tiles;
    const int heads = int(a.s.heads), b = int(bh / heads), h = int(bh % heads), g = h / (heads / int(a.s.kv_heads));
    const int q0 = (tiles - 1 - int(blockIdx.x % tiles)) * T;
    const Sight sight(a, b);
    const ScoreOf score(a, h);
    auto query_used = [&](int i) { return i < tq && sight.query_used(i + sight.shift); };
    auto key_used = [&](int j) { return sight.key_used(j); };
    load_tile<T>(sq, ld, a.q.p + b * a.q.bs + h * a.q.hs, a.q.ts, q0, dim, vec.q, query_used);
    load_tile<T>(sdo, ld, a.dout.p + b * a.dout.bs + h * a.dout.hs, a.dout.ts, q0, dim, vec.dout, query_used);
    float4 acc[4][NC];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int c = 0; c < NC; c++) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int end = sight.keys_end(min(q0 + T, tq) - 1 + sight.shift);
    for (int k0 = 0; k0 < end; k0 += T) {
        __syncthreads();
        load_tile<T>(sk, ld, a.k.p + b * a.k.bs + g * a.k.hs, a.k.ts, k0, dim, vec.k, key_used);
        load_tile<T>(sv, ld, a.v.p + b * a.v.bs + g * a.v.hs, a.v.ts, k0, dim, vec.v, key_used);
        __syncthreads();
        grad_tile<T>(a, sight, score, sq, sk, sdo, sv, ld, dim, q0, k0, ty, tx, a.lse_in + bh * tq, a.work + bh * tq, nullptr, sds);
        __syncwarp();
        tile_accumulate<T, NC, true>(sds, sk, ld, dim, ty, tx, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int q = q0 + 4 * ty + i;
        if (q >= tq) break;
        store_columns<T, NC>(a.dq + ((int64_t(b) * tq + q) * heads + h) * dim, acc[i], query_used(q) ? 1.f : 0.f, dim, tx);
    }
}

template <int T, int NC>
__global__ void __launch_bounds__((T / 4) * (T / 4)) adb_attention_simt_dkv(const AttentionArgs a, const Vec vec) {
    extern __shared__ float4 raw[];
    const int dim = int(a.s.dim), ld = padded(dim), tq = int(a.s.tq);
    float* sq = reinterpret_cast<float*>(raw);
    float *sdo = sq + T * ld, *sk = sdo + T * ld, *sv = sk + T * ld, *sp = sv + T * ld, *sds = sp + T * (T + 4);
    const int tx = threadIdx.x % (T / 4), ty = threadIdx.x / (T / 4);
    const int kv_heads = int(a.s.kv_heads), group = int(a.s.heads) / kv_heads;
    const int tiles = (int(a.s.tk) + T - 1) / T, bg = int(blockIdx.x) / tiles;
    const int b = bg / kv_heads, g = bg % kv_heads;
    const int k0 = (int(blockIdx.x) % tiles) * T;
    const Sight sight(a, b);
    auto query_used = [&](int i) { return i < tq && sight.query_used(i + sight.shift); };
    auto key_used = [&](int j) { return sight.key_used(j); };
    load_tile<T>(sk, ld, a.k.p + b * a.k.bs + g * a.k.hs, a.k.ts, k0, dim, vec.k, key_used);
    load_tile<T>(sv, ld, a.v.p + b * a.v.bs + g * a.v.hs, a.v.ts, k0, dim, vec.v, key_used);
    float4 dk[4][NC], dv[4][NC];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int c = 0; c < NC; c++) dk[i][c] = dv[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    // queries in front of the tile's first key see nothing of it (unless it lies in the prefix)
    const int start = sight.causal && k0 >= sight.prefix ? max(0, k0 - sight.shift) / T * T : 0;
    for (int h = g * group; h < (g + 1) * group; h++) {
        const ScoreOf score(a, h);
        const int64_t bh = int64_t(b) * a.s.heads + h;
        for (int q0 = start; q0 < tq; q0 += T) {
            __syncthreads();
            load_tile<T>(sq, ld, a.q.p + b * a.q.bs + h * a.q.hs, a.q.ts, q0, dim, vec.q, query_used);
            load_tile<T>(sdo, ld, a.dout.p + b * a.dout.bs + h * a.dout.hs, a.dout.ts, q0, dim, vec.dout, query_used);
            __syncthreads();
            grad_tile<T>(a, sight, score, sq, sk, sdo, sv, ld, dim, q0, k0, ty, tx, a.lse_in + bh * tq, a.work + bh * tq, sp, sds);
            __syncthreads();
            tile_accumulate<T, NC, false>(sp, sdo, ld, dim, ty, tx, dv);
            tile_accumulate<T, NC, false>(sds, sq, ld, dim, ty, tx, dk);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int j = k0 + 4 * ty + i;
        if (j >= a.s.tk) break;
        const int64_t at = ((int64_t(b) * a.s.tk + j) * kv_heads + g) * dim;
        if (a.dk) store_columns<T, NC>(a.dk + at, dk[i], 1.f, dim, tx);
        if (a.dv) store_columns<T, NC>(a.dv + at, dv[i], 1.f, dim, tx);
    }
}

template <class K>
bool launch_tiles(K kernel, const AttentionArgs& a, const Vec& vec, int T, int64_t tokens, int64_t heads, size_t smem, CUstream_st* stream, std::string& err) {
    cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e == cudaSuccess) {
        kernel<<<unsigned((tokens + T - 1) / T * a.s.batch * heads), (T / 4) * (T / 4), smem, stream>>>(a, vec);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) return true;
    err = cudaGetErrorString(e);
    return false;
}

}  // namespace

int attention_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    const bool few = a.s.tq < 64 && fits16(a.k, a.s.dim) && fits16(a.v, a.s.dim);
    if (attention_uses_tc(a.s) && !(few && attention_prefers_rows(a.s))) return attention_tc_launch(a, stream, err);
    if (few) return attention_split_launch(a, stream, err);
    const int dim = int(a.s.dim), ld = padded(dim);
    const Vec vec{fits16(a.q, dim), fits16(a.k, dim), fits16(a.v, dim), false, false};
    const size_t smem = (size_t(3) * 64 * ld + 64 * 68) * 4;
    const bool ok = dim <= 64    ? launch_tiles(adb_attention_simt<64, 1>, a, vec, 64, a.s.tq, a.s.heads, smem, stream, err)
                    : dim <= 128 ? launch_tiles(adb_attention_simt<64, 2>, a, vec, 64, a.s.tq, a.s.heads, smem, stream, err)
                                 : launch_tiles(adb_attention_simt<64, 4>, a, vec, 64, a.s.tq, a.s.heads, smem, stream, err);
    return ok ? 1 : -1;
}

int attention_grad_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err) {
    if (attention_grad_uses_tc(a.s)) return attention_tc_grad_launch(a, stream, err);
    const int dim = int(a.s.dim), ld = padded(dim);
    const Vec vec{fits16(a.q, dim), fits16(a.k, dim), fits16(a.v, dim), false, fits16(a.dout, dim)};
    const int T = dim <= 128 ? 64 : 32;
    const size_t tiles = size_t(4) * T * ld * 4, square = size_t(T) * (T + 4) * 4;
    adb_attention_delta<<<unsigned((a.s.batch * a.s.heads * a.s.tq + 7) / 8), 256, 0, stream>>>(a);
    if (cudaError_t e = cudaGetLastError()) { err = cudaGetErrorString(e); return -1; }
    int n = 1;
    if (a.dq) {
        const bool ok = dim <= 64    ? launch_tiles(adb_attention_simt_dq<64, 1>, a, vec, T, a.s.tq, a.s.heads, tiles + square, stream, err)
                        : dim <= 128 ? launch_tiles(adb_attention_simt_dq<64, 2>, a, vec, T, a.s.tq, a.s.heads, tiles + square, stream, err)
                                     : launch_tiles(adb_attention_simt_dq<32, 8>, a, vec, T, a.s.tq, a.s.heads, tiles + square, stream, err);
        if (!ok) return -1;
        n++;
    }
    if (a.dk || a.dv) {
        const bool ok = dim <= 64    ? launch_tiles(adb_attention_simt_dkv<64, 1>, a, vec, T, a.s.tk, a.s.kv_heads, tiles + 2 * square, stream, err)
                        : dim <= 128 ? launch_tiles(adb_attention_simt_dkv<64, 2>, a, vec, T, a.s.tk, a.s.kv_heads, tiles + 2 * square, stream, err)
                                     : launch_tiles(adb_attention_simt_dkv<32, 8>, a, vec, T, a.s.tk, a.s.kv_heads, tiles + 2 * square, stream, err);
        if (!ok) return -1;
        n++;
    }
    return n;
}

}  // namespace adb
