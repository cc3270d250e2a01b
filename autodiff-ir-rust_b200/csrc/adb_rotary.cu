// Rotary positions: pairs of a head's elements turned by an angle that grows with the token's position.
//
//   (a, b) -> gain * (a cos t - b sin t, b cos t + a sin t),   t = position * frequency of the pair
//
// Pairs are neighbours (interleaved) or element i of the first half with element i of the second half of the turned
// part; elements behind the turned part pass through.  The gradient is the turn by -t.
//
// The angle of a far position does not fit fp32: at position 10^6 an fp32 product is off by 0.03 of a radian.  The table
// holds each frequency in turns as the sum of two floats, the product is formed exactly (fma gives its rounding error)
// and only its distance from a whole number of turns is kept, so that sine and cosine are good to about 2e-7 up to
// positions of 2^24.
//
// Bound by HBM: 8 bytes per element; 4 x 4096 tokens of 32 heads of 128, 537 MB, take 94 us = 5.7 TB/s, 0.87 of the copy rate.
// A block takes a few tokens: their sines and cosines go into shared memory once and
// serve every head.
#include <cuda_runtime.h>

#include "adb_oper.hpp"

namespace adb {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_PAIRS_SHARED = int(ROTARY_MAX_PAIRS);   // sines and cosines held by a block (32 KiB)

__device__ __forceinline__ float2 turn_of(const float* table, int64_t pairs, int p, float pos, float gain, int inverse) {
    const float hi = __ldg(table + p), lo = __ldg(table + pairs + p);
    const float whole = pos * hi;
    const float rest = fmaf(pos, hi, -whole) + pos * lo;        // what the rounded product lost
    const float part = (whole - rintf(whole)) + rest;           // the first difference is exact
    float s, c;
    sincospif(2.f * part, &s, &c);
    return make_float2(c * gain, (inverse ? -s : s) * gain);
}

// VEC: 16-byte accesses (turned part a multiple of 8 elements, strides and bases to match).
template <bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(THREADS) adb_rotary(const RotaryArgs a, const int tokens_per_block) {
    __shared__ float2 cs[MAX_PAIRS_SHARED];
    const int pairs = int(a.pairs), dim = int(a.dim), heads = int(a.heads);
    const int64_t all = a.batch * a.tokens;
    const int64_t first = int64_t(blockIdx.x) * tokens_per_block;
    const int n = int(min(int64_t(tokens_per_block), all - first));
    for (int e = threadIdx.x; e < n * pairs; e += THREADS) {
        const int64_t bt = first + e / pairs, b = bt / a.tokens, t = bt - b * a.tokens;
        const float pos = a.positions ? a.positions[b * a.p_bs + t * a.p_ts] : float(a.offset + t);
        cs[e] = turn_of(a.table, a.pairs, e % pairs, pos, a.gain, a.inverse);
    }
    __syncthreads();
    constexpr int W = VEC ? 4 : 1;
    // work items of one head: the turned pairs (W of them, or 2 pairs of neighbours), then the rest, W elements each
    const int turned = VEC ? (INTERLEAVED ? pairs / 2 : pairs / 4) : pairs;
    const int items = turned + (dim - 2 * pairs) / W;
    const int per_token = items * heads;
    for (int e = threadIdx.x; e < n * per_token; e += THREADS) {
        const int k = e / per_token, r = e - k * per_token, head = r / items, i = r - head * items;
        const int64_t bt = first + k, b = bt / a.tokens, t = bt - b * a.tokens;
        const float* src = a.x + b * a.x_bs + t * a.x_ts + head * a.x_hs;
        float* dst = a.y + (bt * heads + head) * dim;
        const float2* w = cs + k * pairs;
        if (i >= turned) {
            const int c = 2 * pairs + (i - turned) * W;
            if constexpr (VEC) *reinterpret_cast<float4*>(dst + c) = __ldg(reinterpret_cast<const float4*>(src + c));
            else dst[c] = __ldg(src + c);
        } else if constexpr (VEC && INTERLEAVED) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(src + 4 * i));
            const float2 p = w[2 * i], q = w[2 * i + 1];
            *reinterpret_cast<float4*>(dst + 4 * i) =
                make_float4(v.x * p.x - v.y * p.y, v.y * p.x + v.x * p.y, v.z * q.x - v.w * q.y, v.w * q.x + v.z * q.y);
        } else if constexpr (VEC) {
            const float4 u = __ldg(reinterpret_cast<const float4*>(src + 4 * i));
            const float4 v = __ldg(reinterpret_cast<const float4*>(src + pairs + 4 * i));
            const float2 p0 = w[4 * i], p1 = w[4 * i + 1], p2 = w[4 * i + 2], p3 = w[4 * i + 3];
            *reinterpret_cast<float4*>(dst + 4 * i) =
                make_float4(u.x * p0.x - v.x * p0.y, u.y * p1.x - v.y * p1.y, u.z * p2.x - v.z * p2.y, u.w * p3.x - v.w * p3.y);
            *reinterpret_cast<float4*>(dst + pairs + 4 * i) =
                make_float4(v.x * p0.x + u.x * p0.y, v.y * p1.x + u.y * p1.y, v.z * p2.x + u.z * p2.y, v.w * p3.x + u.w * p3.y);
        } else {
            const int ca = INTERLEAVED ? 2 * i : i, cb = INTERLEAVED ? 2 * i + 1 : pairs + i;
            const float u = __ldg(src + ca), v = __ldg(src + cb);
            const float2 p = w[i];
            dst[ca] = u * p.x - v * p.y;
            dst[cb] = v * p.x + u * p.y;
        }
    }
}

}  // namespace

int rotary_launch(const RotaryArgs& a, CUstream_st* stream, std::string& err) {
    const bool vec = a.pairs % (a.interleaved ? 2 : 4) == 0 && a.dim % 4 == 0 && a.x_bs % 4 == 0 && a.x_ts % 4 == 0 &&
                     a.x_hs % 4 == 0 && aligned16(a.x) && aligned16(a.y);
    // enough tokens for a block to have 4096 elements, as long as every SM still gets two blocks
    const int64_t all = a.batch * a.tokens;
    int64_t tpb = std::max<int64_t>(1, 4096 / (a.heads * a.dim));
    tpb = std::min(tpb, std::max<int64_t>(1, all / (2 * a.sm_count)));
    tpb = std::min<int64_t>(tpb, MAX_PAIRS_SHARED / a.pairs);
    const int64_t grid = (all + tpb - 1) / tpb;
    if (grid > int64_t(0x7fffffff)) { err = "rotary over more than 2^31 tokens"; return -1; }
    if (a.interleaved) {
        if (vec) adb_rotary<true, true><<<unsigned(grid), THREADS, 0, stream>>>(a, int(tpb));
        else adb_rotary<true, false><<<unsigned(grid), THREADS, 0, stream>>>(a, int(tpb));
    } else {
        if (vec) adb_rotary<false, true><<<unsigned(grid), THREADS, 0, stream>>>(a, int(tpb));
        else adb_rotary<false, false><<<unsigned(grid), THREADS, 0, stream>>>(a, int(tpb));
    }
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 1;
    err = cudaGetErrorString(e);
    return -1;
}

}  // namespace adb
