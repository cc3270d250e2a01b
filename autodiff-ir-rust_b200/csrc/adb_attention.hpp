// What the attention kernels share: which keys a query sees, and how a product of query and key becomes a score.
//
// Query i of Tq stands at position i + n - Tq of its sequence, n being the sequence's length (the count of keys unless
// `lengths` says otherwise): the queries are the last ones.  It sees key j when j < n and, as far as these are given,
//   causal    j <= position, or j < prefix of the sequence (a prefix sees itself whole)
//   docs      both positions carry the same document number, which is not negative (negative: padding)
// Under the causal mask or with lengths, a query that would stand before the first key sees nothing.  A query that sees
// nothing has an output of zeros, a logarithm of -inf and no gradient.
//
// Scores are kept in base 2 (multiplied by log2 e), so that every exponential is one ex2:
//   s = scale * q.k;   s = cap * tanh(s / cap);   s -= slope * |position - j|
#pragma once
#include <cuda_runtime.h>

#include "adb_oper.hpp"

namespace adb {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// whole number of tokens out of a float that a caller filled (NaN and negative numbers: none)
__device__ __forceinline__ int token_count(const float* p, int64_t b, int most) {
    return p ? int(fminf(fmaxf(__ldg(p + b), 0.f), float(most))) : most;
}

// one sequence's masks
struct Sight {
    int n, shift, prefix, causal, hide_before;
    const float* docs;   // this sequence's, or null
    __device__ __forceinline__ Sight(const AttentionArgs& a, int64_t b) {
        n = token_count(a.lengths, b, int(a.s.tk));
        shift = n - int(a.s.tq);
        prefix = a.prefix ? token_count(a.prefix, b, int(a.s.tk)) : 0;
        causal = a.causal;
        hide_before = a.causal || a.lengths;
        docs = a.docs ? a.docs + b * a.s.tk : nullptr;
    }
    // rows of the operands that no pair can reach: their contents (padding, unused cache) never enter a product
    __device__ __forceinline__ bool key_used(int j) const { return j < n && !(docs && !(docs[j] >= 0.f)); }
    __device__ __forceinline__ bool query_used(int pos) const {
        return !(hide_before && pos < 0) && pos < n && !(docs && !(docs[pos] >= 0.f));
    }
    // the first key that no query up to `last_pos` sees
    __device__ __forceinline__ int keys_end(int last_pos) const {
        return causal ? min(n, max(last_pos + 1, prefix)) : n;
    }
    // key j is used and the query is; `doc` is the query's document
    __device__ __forceinline__ bool sees(int pos, int j, float doc) const {
        return (!causal || j <= pos || j < prefix) && (!docs || docs[j] == doc);
    }
};

// tanh to fp32 accuracy from one ex2 and one reciprocal; near zero, where 1 - 2 / (e + 1) cancels, its odd series (the
// first omitted term, 1382/155925 x^10 of x, is 5.2e-8 at 0.3: less than an fp32 rounding)
__device__ __forceinline__ float tanh_exact(float x) {
    const float e = exp2f(2.f * LOG2E * fabsf(x));
    const float far = copysignf(1.f - __fdividef(2.f, e + 1.f), x);
    const float y = x * x;
    float t = fmaf(y, 62.f / 2835.f, -17.f / 315.f);
    t = fmaf(y, t, 2.f / 15.f);
    t = fmaf(y, t, -1.f / 3.f);
    const float near = fmaf(x * y, t, x);
    return fabsf(x) < 0.3f ? near : far;
}

struct ScoreOf {
    float mul, cap2, slope2;   // plain: scale * log2 e;  capped: scale / cap, then cap * log2 e
    int capped;
    __device__ __forceinline__ ScoreOf(const AttentionArgs& a, int head) {
        capped = a.cap > 0.f;
        mul = capped ? a.scale / a.cap : a.scale * LOG2E;
        cap2 = a.cap * LOG2E;
        slope2 = a.slopes ? __ldg(a.slopes + head) * LOG2E : 0.f;
    }
    // the score in base 2; `bend` is its derivative by scale * q.k (without the log2 e)
    __device__ __forceinline__ float operator()(float dot, int pos, int j, float& bend) const {
        float s = dot * mul;
        bend = 1.f;
        if (capped) {
            const float t = tanh_exact(s);
            bend = fmaf(-t, t, 1.f);
            s = t * cap2;
        }
        return slope2 != 0.f ? fmaf(-slope2, fabsf(float(pos - j)), s) : s;
    }
};

}  // namespace adb
