// Root-mean-square norm with the residual's addition, and its gradient.
//
//   h = x + r,   n = h / sqrt(mean(h^2) + eps),   y = n * g
//   dn = dy * g,   dx = dr = dh + (dn - n * mean(dn * n)) / sqrt(mean(h^2) + eps),   dg = sum over rows of dy * n
//
// Both are bound by HBM: 16 bytes per element forward (x, r in; y, h out), 16 backward (h, dy, dh in; dx out).  A row is
// read once: a warp (rows of up to 1024 elements) or a block holds its share of the row in registers while the sums run
// through shuffles and, across warps, shared memory in a fixed order.  Sums are fp32: a thread adds at most 32 products
// one after another (a 1024th of the row where rows are wider than registers hold), the rest is a tree; dg adds a block's
// rows one after another, then the blocks.
//
// Measured: 65536 rows of 1024, forward and gradient, 2.15 GB in 340 us = 6.3 TB/s, 0.97 of the copy rate.  2001 rows of 5003
// (no 16-byte access fits, a block a row): forward 31 us = 5.2 TB/s, gradient about 50 us = 3.2 TB/s, bound by the two
// barriers of a row with 16 warps an SM (1024 threads of half the share: 49 us; the next row's loads ahead: 53 us, spills).
#include <cuda_runtime.h>

#include "adb_oper.hpp"

namespace adb {
namespace {

template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* shared) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = threadIdx.x / 32, first = threadIdx.x / TPR * W;
        __syncthreads();   // the previous row's sums have been read
        if (threadIdx.x % 32 == 0)
#pragma unroll
            for (int i = 0; i < N; i++) shared[warp * N + i] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) t += shared[(first + w) * N + i];
            s[i] = t;
        }
    }
}

// A thread's share of a row: 4V elements.  VEC: four neighbours at 4 * (lane + i * TPR); otherwise single ones at
// lane + j * TPR (rows whose length or stride does not allow 16-byte accesses).
template <int TPR, int V, bool VEC>
__device__ __forceinline__ void load_row(const float* p, int lane, int width, float (&v)[4 * V]) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = 4 * (lane + i * TPR);
            const float4 t = c < width ? __ldg(reinterpret_cast<const float4*>(p + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
            const int c = lane + j * TPR;
            v[j] = c < width ? __ldg(p + c) : 0.f;
        }
    }
}
template <int TPR, int V, bool VEC>
__device__ __forceinline__ void store_row(float* p, int lane, int width, const float (&v)[4 * V]) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = 4 * (lane + i * TPR);
            if (c < width) *reinterpret_cast<float4*>(p + c) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
            const int c = lane + j * TPR;
            if (c < width) p[c] = v[j];
        }
    }
}

template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) adb_rms_norm(const NormArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ float shared[THREADS / 32];
    const int lane = threadIdx.x % TPR, width = int(a.width);
    const int64_t row = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
    const bool on = row < a.rows;
    float h[4 * V], g[4 * V];
    load_row<TPR, V, VEC>(a.x + (on ? row : 0) * a.x_rs, lane, width, h);
    if (a.residual) {
        float r[4 * V];
        load_row<TPR, V, VEC>(a.residual + (on ? row : 0) * a.r_rs, lane, width, r);
#pragma unroll
        for (int j = 0; j < 4 * V; j++) h[j] += r[j];
    }
    if (a.y) load_row<TPR, V, VEC>(a.scale, lane, width, g);
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < 4 * V; j++) s[0] = fmaf(h[j], h[j], s[0]);
    row_sums<TPR>(s, shared);
    if (!on) return;
    if (a.h) store_row<TPR, V, VEC>(a.h + row * a.width, lane, width, h);
    if (!a.y) return;
    const float inv = 1.f / sqrtf(s[0] / float(width) + a.eps);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) h[j] = h[j] * inv * g[j];
    store_row<TPR, V, VEC>(a.y + row * a.width, lane, width, h);
}

// rows too wide for registers: a block walks the row twice (the second time through the caches)
__global__ void __launch_bounds__(1024) adb_rms_norm_long(const NormArgs a) {
    __shared__ float shared[32];
    const int64_t row = blockIdx.x;
    const float* x = a.x + row * a.x_rs;
    const float* r = a.residual ? a.residual + row * a.r_rs : nullptr;
    float s[1] = {0.f};
    for (int64_t c = threadIdx.x; c < a.width; c += 1024) {
        const float h = r ? x[c] + r[c] : x[c];
        s[0] = fmaf(h, h, s[0]);
        if (a.h) a.h[row * a.width + c] = h;
    }
    row_sums<1024>(s, shared);
    if (!a.y) return;
    const float inv = 1.f / sqrtf(s[0] / float(a.width) + a.eps);
    for (int64_t c = threadIdx.x; c < a.width; c += 1024) {
        const float h = r ? x[c] + r[c] : x[c];
        a.y[row * a.width + c] = h * inv * a.scale[c];
    }
}

// Every block walks rows blockIdx, blockIdx + grid, ... and keeps its part of dg in registers; the blocks' parts are added
// by adb_column_sums in the order of the blocks, so that a gradient has the same bits in every run.
template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) adb_rms_norm_grad(const NormGradArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ float shared[THREADS / 32 * 2];
    __shared__ float parts[RPB > 1 ? RPB * TPR * 4 * V : 1];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR, width = int(a.width);
    float acc[4 * V];
#pragma unroll
    for (int j = 0; j < 4 * V; j++) acc[j] = 0.f;
    for (int64_t base = int64_t(blockIdx.x) * RPB; base < a.rows; base += int64_t(gridDim.x) * RPB) {
        const int64_t row = base + sub;
        const bool on = row < a.rows;
        float h[4 * V], d[4 * V];
        load_row<TPR, V, VEC>(a.h + (on ? row : 0) * a.h_rs, lane, width, h);
        load_row<TPR, V, VEC>(a.dy + (on ? row : 0) * a.dy_rs, lane, width, d);
        float g[4 * V];
        load_row<TPR, V, VEC>(a.scale, lane, width, g);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
            s[0] = fmaf(h[j], h[j], s[0]);
            s[1] = fmaf(d[j] * g[j], h[j], s[1]);
        }
        row_sums<TPR>(s, shared);
        const float inv = 1.f / sqrtf(s[0] / float(width) + a.eps);
        const float along = s[1] / float(width) * inv * inv;
        if (!on) continue;
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
            acc[j] = fmaf(d[j], h[j] * inv, acc[j]);
            d[j] = inv * (d[j] * g[j] - h[j] * along);
        }
        if (!a.dx) continue;
        if (a.dh) {
            load_row<TPR, V, VEC>(a.dh + row * a.dh_rs, lane, width, h);
#pragma unroll
            for (int j = 0; j < 4 * V; j++) d[j] += h[j];
        }
        store_row<TPR, V, VEC>(a.dx + row * a.width, lane, width, d);
    }
    if (!a.dscale) return;
    if constexpr (RPB > 1) {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) parts[(sub * 4 * V + j) * TPR + lane] = acc[j];
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int j = 0; j < 4 * V; j++)
            for (int q = 1; q < RPB; q++) acc[j] += parts[(q * 4 * V + j) * TPR + lane];
    }
    store_row<TPR, V, VEC>(a.work + int64_t(blockIdx.x) * a.width, lane, width, acc);
}

__global__ void __launch_bounds__(1024) adb_rms_norm_grad_long(const NormGradArgs a) {
    __shared__ float shared[64];
    const int64_t row = blockIdx.x;
    const float *h = a.h + row * a.h_rs, *dy = a.dy + row * a.dy_rs;
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < a.width; c += 1024) {
        s[0] = fmaf(h[c], h[c], s[0]);
        s[1] = fmaf(dy[c] * a.scale[c], h[c], s[1]);
    }
    row_sums<1024>(s, shared);
    const float inv = 1.f / sqrtf(s[0] / float(a.width) + a.eps);
    const float along = s[1] / float(a.width) * inv * inv;
    if (threadIdx.x == 0) a.work[row] = inv;
    if (!a.dx) return;
    for (int64_t c = threadIdx.x; c < a.width; c += 1024) {
        const float d = inv * (dy[c] * a.scale[c] - h[c] * along);
        a.dx[row * a.width + c] = a.dh ? d + a.dh[row * a.dh_rs + c] : d;
    }
}
// dg of wide rows: each thread owns a column of one of gridDim.y ranges of rows
__global__ void __launch_bounds__(256) adb_rms_norm_grad_columns(const NormGradArgs a) {
    const int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (c >= a.width) return;
    const int64_t lo = a.rows * blockIdx.y / gridDim.y, hi = a.rows * (blockIdx.y + 1) / gridDim.y;
    float s = 0.f;
    for (int64_t r = lo; r < hi; r++) s = fmaf(a.dy[r * a.dy_rs + c], a.h[r * a.h_rs + c] * a.work[r], s);
    a.work[a.rows + int64_t(blockIdx.y) * a.width + c] = s;
}

// out[c] = sum over rows of part[rows][width]; 32 columns by 32 row lanes a block, added in a fixed order
__global__ void __launch_bounds__(1024) adb_column_sums(const float* part, float* out, int rows, int64_t width) {
    __shared__ float t[32][33];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    const int64_t c = int64_t(blockIdx.x) * 32 + x;
    float s = 0.f;
    if (c < width) {
#pragma unroll 4
        for (int r = y; r < rows; r += 32) s += part[int64_t(r) * width + c];
    }
    t[y][x] = s;
    __syncthreads();
    s = t[x][y];   // a warp for each column
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int64_t own = int64_t(blockIdx.x) * 32 + y;
    if (x == 0 && own < width) out[own] = s;
}

int launched(int n, std::string& err) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return n;
    err = cudaGetErrorString(e);
    return -1;
}

}  // namespace

int rms_norm_launch(const NormArgs& a, CUstream_st* stream, std::string& err) {
    const bool vec = a.width % 4 == 0 && a.x_rs % 4 == 0 && a.r_rs % 4 == 0 && aligned16(a.x) && aligned16(a.residual) &&
                     aligned16(a.scale) && aligned16(a.y) && aligned16(a.h);
    if (a.rows > int64_t(0x7fffffff)) { err = "norm over more than 2^31 rows"; return -1; }
#define ADB_NORM(TPR, V)                                                                             \
    do {                                                                                             \
        constexpr int T = TPR > 256 ? TPR : 256;                                                     \
        const unsigned grid = unsigned((a.rows + T / TPR - 1) / (T / TPR));                          \
        if (vec) adb_rms_norm<TPR, V, true><<<grid, T, 0, stream>>>(a);                              \
        else adb_rms_norm<TPR, V, false><<<grid, T, 0, stream>>>(a);                                 \
    } while (0)
    if (a.width <= 128) ADB_NORM(32, 1);
    else if (a.width <= 256) ADB_NORM(32, 2);
    else if (a.width <= 512) ADB_NORM(32, 4);
    else if (a.width <= 1024) ADB_NORM(32, 8);
    else if (a.width <= 2048) ADB_NORM(128, 4);
    else if (a.width <= 4096) ADB_NORM(256, 4);
    else if (a.width <= 8192) ADB_NORM(512, 4);
    else if (a.width <= 16384) ADB_NORM(1024, 4);
    else adb_rms_norm_long<<<unsigned(a.rows), 1024, 0, stream>>>(a);
#undef ADB_NORM
    return launched(1, err);
}

int rms_norm_grad_launch(const NormGradArgs& a, CUstream_st* stream, std::string& err) {
    if (a.rows > int64_t(0x7fffffff)) { err = "norm over more than 2^31 rows"; return -1; }
    const unsigned column_blocks = unsigned((a.width + 31) / 32);
    if (a.width > NORM_GRAD_ONE_PASS) {
        adb_rms_norm_grad_long<<<unsigned(a.rows), 1024, 0, stream>>>(a);
        if (!a.dscale) return launched(1, err);
        const unsigned ranges = unsigned(std::min<int64_t>(a.rows, 64));
        adb_rms_norm_grad_columns<<<dim3(unsigned((a.width + 255) / 256), ranges), 256, 0, stream>>>(a);
        adb_column_sums<<<column_blocks, 1024, 0, stream>>>(a.work + a.rows, a.dscale, int(ranges), a.width);
        return launched(3, err);
    }
    const bool vec = a.width % 4 == 0 && a.h_rs % 4 == 0 && a.dy_rs % 4 == 0 && a.dh_rs % 4 == 0 && aligned16(a.h) &&
                     aligned16(a.dy) && aligned16(a.dh) && aligned16(a.scale) && aligned16(a.dx) && aligned16(a.work);
    const unsigned grid = unsigned(norm_grad_blocks(a.rows, a.width, a.sm_count));
#define ADB_NORM_GRAD(TPR, V)                                                                        \
    do {                                                                                             \
        constexpr int T = TPR > 256 ? TPR : 256;                                                     \
        if (vec) adb_rms_norm_grad<TPR, V, true><<<grid, T, 0, stream>>>(a);                         \
        else adb_rms_norm_grad<TPR, V, false><<<grid, T, 0, stream>>>(a);                            \
    } while (0)
    if (a.width <= 128) ADB_NORM_GRAD(32, 1);
    else if (a.width <= 256) ADB_NORM_GRAD(32, 2);
    else if (a.width <= 512) ADB_NORM_GRAD(32, 4);
    else if (a.width <= 1024) ADB_NORM_GRAD(32, 8);
    else if (a.width <= 2048) ADB_NORM_GRAD(256, 2);
    else if (a.width <= 4096) ADB_NORM_GRAD(512, 2);
    else if (a.width <= 8192) ADB_NORM_GRAD(512, 4);
    else ADB_NORM_GRAD(1024, 4);
#undef ADB_NORM_GRAD
    if (!a.dscale) return launched(1, err);
    adb_column_sums<<<column_blocks, 1024, 0, stream>>>(a.work, a.dscale, int(grid), a.width);
    return launched(2, err);
}

}  // namespace adb
