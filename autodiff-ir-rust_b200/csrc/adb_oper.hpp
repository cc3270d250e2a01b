// Operators of transformer layers: what the lowering has to know about them (shapes, workspaces) and how the runtime
// launches them.  Host-only declarations; the kernels are in adb_norm.cu, adb_rotary.cu and adb_attention*.cu.
#pragma once
#include <algorithm>
#include <cstdint>
#include <string>

struct CUstream_st;

namespace adb {

// ------------------------------------------------------------------------------------------ root-mean-square norm
struct NormArgs {
    const float *x = nullptr, *residual = nullptr, *scale = nullptr;   // residual may be null
    float *y = nullptr, *h = nullptr;                                  // either may be null; contiguous rows
    int64_t rows = 0, width = 0, x_rs = 0, r_rs = 0;                   // row strides in elements
    float eps = 0.f;
};
struct NormGradArgs {
    const float *h = nullptr, *scale = nullptr, *dy = nullptr, *dh = nullptr;   // dh may be null
    float *dx = nullptr, *dscale = nullptr, *work = nullptr;                    // dx or dscale may be null
    int64_t rows = 0, width = 0, h_rs = 0, dy_rs = 0, dh_rs = 0;
    float eps = 0.f;
    int sm_count = 148;
};
constexpr int64_t NORM_GRAD_ONE_PASS = 16384;   // widest row whose share stays in a thread's registers
// blocks of the gradient kernel: each adds its rows' part of dscale in registers and writes one row of partial sums
inline int64_t norm_grad_blocks(int64_t rows, int64_t width, int sm_count) {
    const int64_t rows_per_block = width <= 1024 ? 8 : 1;
    const int64_t blocks = (rows + rows_per_block - 1) / rows_per_block;
    return std::min<int64_t>(blocks, int64_t(sm_count) * (width <= 1024 ? 2 : width <= 2048 ? 4 : width <= 4096 ? 2 : 1));
}
inline int64_t norm_grad_workspace(int64_t rows, int64_t width, int sm_count) {
    if (width > NORM_GRAD_ONE_PASS) return rows + width * std::min<int64_t>(rows, 64);
    return norm_grad_blocks(rows, width, sm_count) * width;
}

// ------------------------------------------------------------------------------------------ rotary positions
constexpr int64_t ROTARY_MAX_PAIRS = 4096;   // a block keeps a token's sines and cosines in shared memory
struct RotaryArgs {
    const float *x = nullptr, *table = nullptr, *positions = nullptr;   // positions may be null: offset + token
    float* y = nullptr;                                                 // contiguous
    int64_t batch = 0, tokens = 0, heads = 0, dim = 0, pairs = 0;
    int64_t x_bs = 0, x_ts = 0, x_hs = 0, p_bs = 0, p_ts = 0;
    int64_t offset = 0;
    int interleaved = 0, inverse = 0;
    float gain = 1.f;
    int sm_count = 148;
};

// ------------------------------------------------------------------------------------------ attention
constexpr int64_t ATTENTION_MAX_DIM = 256;
struct AttentionShape {
    int64_t batch = 0, tq = 0, tk = 0, heads = 0, kv_heads = 0, dim = 0;
    bool cuda_cores = false;   // fp32 products only (ADB_FLAG_SIMT_DOT)
};
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
struct Strided4 {   // [batch, tokens, heads, dim], dim contiguous
    const float* p = nullptr;
    int64_t bs = 0, ts = 0, hs = 0;
};
// rows that 16-byte accesses fit
inline bool fits16(const Strided4& t, int64_t dim) {
    return t.p && aligned16(t.p) && dim % 4 == 0 && t.bs % 4 == 0 && t.ts % 4 == 0 && t.hs % 4 == 0;
}
struct AttentionArgs {
    AttentionShape s;
    Strided4 q, k, v, out, dout;            // out (as an operand) and dout: gradient only
    int out_vec = 0;                        // out can be read 16 bytes at a time
    const float *slopes = nullptr, *docs = nullptr, *prefix = nullptr, *lengths = nullptr;   // each may be null
    float *o = nullptr, *lse = nullptr;     // forward results (contiguous; lse in base 2; either may be null)
    const float* lse_in = nullptr;
    float *dq = nullptr, *dk = nullptr, *dv = nullptr;   // gradient results (contiguous; each may be null)
    float* work = nullptr;
    int* status = nullptr;   // device word in which a kernel records that a bounded wait ran out
    int causal = 0;
    float scale = 1.f, cap = 0.f;
    int sm_count = 148;
};
// The tensor-core kernels (adb_attention_tc.cu) take heads of up to 128 elements, padded to panels of 64, and tiles of
// 128 tokens.
constexpr int64_t ATTENTION_TC_MAX_DIM = 128, ATTENTION_TC_TILE = 128;
constexpr int ATTENTION_GAVE_UP = 33;   // first code of a bounded wait of theirs that ran out
inline int attention_panels(int64_t dim) { return dim <= 64 ? 1 : 2; }
// With few queries a tile of 128 is mostly padding and the keys are worth reading once only: adb_attention_decode.cu.  From
// 8 queries on the tile can be the faster one all the same, and it takes what that kernel's 16-byte accesses do not fit: one query of
// 32 x 16384 keys, 32 heads over 8 of 126, 3.6 ms against 39 in the general kernel; 1025 keys, 8 over 2 of 62: 32 us / 188.
inline bool attention_uses_tc(const AttentionShape& s) {
    return !s.cuda_cores && s.dim <= ATTENTION_TC_MAX_DIM && (s.tq >= 8 || s.dim % 4) && s.tk >= 64 && s.batch * s.heads <= 65535;
}
// The tile costs making images of the cache (12 bytes moved for 4) and a tile for each head, the kernel for few queries as much
// again for every 8 rows (queries of the heads that share a key head): it is the better one up to 8 rows of 128 elements.
// Tile against the other, us: 8 rows of 128, 8 x 16384 keys of 32 heads 2107 / 1176, 2000 keys 61 / 55 (4 x 2000: 156 / 169);
// 8 rows of 64, 128 x 512 of 16 heads 427 / 149, 300 of 8 heads 22 / 16; 12 rows of 64, 256 x 200 of 16 heads 502 / 333; 16
// rows of 32, 16 x 4000 of 16 heads 353 / 160.  More rows: 15 of 128, 2000 of 32 heads 62 / 88, 8 x 2000 291 / 375; 32 of 128,
// 8000 of 4 key heads 51 / 92, 32 x 16384 of 8 key heads 3539 / 4371; 24 of 64, 8 x 4000 of 32 heads 365 / 356.
inline bool attention_prefers_rows(const AttentionShape& s) { return s.tq < 64 && s.heads / s.kv_heads * s.tq * s.dim <= 1024; }
// How many blocks share one tile's walk over the other side when there are fewer tiles than SMs: as many as fill the SMs,
// each with at least `least` steps.  Their results are added (or joined) in order by a kernel of their own.
inline int64_t attention_shares(int64_t tiles, int64_t steps, int64_t least, int sm_count) {
    return std::max<int64_t>(1, std::min(int64_t(sm_count) / tiles, steps / least));
}
inline int64_t attention_tc_tiles(int64_t tokens) { return (tokens + ATTENTION_TC_TILE - 1) / ATTENTION_TC_TILE; }
inline int64_t attention_forward_shares(const AttentionShape& s, int sm_count) {
    return attention_shares(s.batch * s.heads * attention_tc_tiles(s.tq), attention_tc_tiles(s.tk), 4, sm_count);
}
inline int64_t attention_dq_shares(const AttentionShape& s, int sm_count) {
    return attention_shares(s.batch * s.heads * attention_tc_tiles(s.tq), 2 * attention_tc_tiles(s.tk), 4, sm_count);
}
inline int64_t attention_dkv_shares(const AttentionShape& s, int sm_count) {
    return attention_shares(s.batch * s.kv_heads * attention_tc_tiles(s.tk), 2 * attention_tc_tiles(s.tq), 4, sm_count);
}
// Few queries (adb_attention_decode.cu): the keys are cut into ranges, so that about eight rounds of two blocks per SM
// have work and a range keeps a block busy for at least one step.
constexpr int64_t ATTENTION_SPLIT_STEP = 128;
inline int64_t attention_range_keys(const AttentionShape& s, int sm_count) {
    const int64_t rows = s.heads / s.kv_heads * s.tq, blocks = s.batch * s.kv_heads * ((rows + 7) / 8);
    const int64_t keys = (s.tk * blocks + int64_t(sm_count) * 16 - 1) / (int64_t(sm_count) * 16);
    return (std::max(keys, ATTENTION_SPLIT_STEP) + ATTENTION_SPLIT_STEP - 1) / ATTENTION_SPLIT_STEP * ATTENTION_SPLIT_STEP;
}
inline int64_t attention_ranges(const AttentionShape& s, int sm_count) {
    const int64_t keys = attention_range_keys(s, sm_count);
    return (s.tk + keys - 1) / keys;
}
inline int64_t attention_workspace(const AttentionShape& s, int sm_count) {
    const int64_t parts = s.batch * s.tq * s.heads * attention_ranges(s, sm_count) * (s.dim + 2);   // of ranges of keys
    if (!attention_uses_tc(s)) return parts;
    // images of keys and values, their scales by tile and by row, document numbers; each part begins on a 256-byte boundary
    const int64_t tiles = attention_tc_tiles(s.tk), n = s.batch * s.kv_heads * tiles, shares = attention_forward_shares(s, sm_count);
    const int64_t images = 2 * (n * (attention_panels(s.dim) * 8192 + 1 + ATTENTION_TC_TILE) + 128) + 4 * s.batch * tiles + 64 +
                           (shares > 1 ? s.batch * s.tq * s.heads * shares * (s.dim + 2) : 0);
    return attention_prefers_rows(s) ? std::max(images, parts) : images;   // (which of the two also depends on the operands' strides)
}
// The gradient takes them whatever the count of queries: the CUDA-core kernels' tiles of 64 are just as empty.
inline bool attention_grad_uses_tc(const AttentionShape& s) {
    return !s.cuda_cores && s.dim <= ATTENTION_TC_MAX_DIM && s.tk >= 64 && s.batch * s.heads <= 65535;
}
inline int64_t attention_grad_workspace(const AttentionShape& s, int sm_count) {
    if (!attention_grad_uses_tc(s)) return s.batch * s.heads * s.tq;   // one number per query: the gradient of the output times the output
    const int64_t kt = attention_tc_tiles(s.tk), qt = attention_tc_tiles(s.tq);
    const int64_t nk = s.batch * s.kv_heads * kt, nq = s.batch * s.heads * qt;
    const int64_t q_shares = attention_dq_shares(s, sm_count), k_shares = attention_dkv_shares(s, sm_count);
    // images of four operands with their scales, logarithms and deltas in whole tiles, document numbers
    return 2 * ((nk + nq) * (attention_panels(s.dim) * 8192 + 1 + ATTENTION_TC_TILE) + 256) + 2 * (nq * ATTENTION_TC_TILE + 64) +
           4 * s.batch * (kt + qt) + 128 + (q_shares > 1 ? q_shares * s.batch * s.tq * s.heads * s.dim + 64 : 0) +
           (k_shares > 1 ? 2 * (k_shares * s.batch * s.tk * s.kv_heads * s.dim + 64) : 0);
}

// Each enqueues its kernels on `stream` and returns how many, or -1 with `err` set.
int rms_norm_launch(const NormArgs& a, CUstream_st* stream, std::string& err);
int rms_norm_grad_launch(const NormGradArgs& a, CUstream_st* stream, std::string& err);
int rotary_launch(const RotaryArgs& a, CUstream_st* stream, std::string& err);
int attention_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err);
int attention_grad_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err);
// joins partial[rows][ranges][dim + 2] (unscaled result, maximum, sum) into the output and the logarithms
void attention_join(const AttentionArgs& a, int ranges, const float* partial, CUstream_st* stream);
// few queries (with many, over fewer than 64 keys, the general kernel: 4096 queries of 16 heads over 60 keys 160 us against
// 469); 16-byte accesses to keys and values
int attention_split_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err);
// where attention_uses_tc
int attention_tc_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err);
int attention_tc_grad_launch(const AttentionArgs& a, CUstream_st* stream, std::string& err);

}  // namespace adb
