// fp32 products on the fp16 tensor cores of sm_100a: operands as sums of two halves, and the tcgen05 instructions for them.
//
// An fp32 value x is held as s (hi + lo) with s a power of two and hi, lo fp16: hi is x / s rounded to 11 bits, lo the rest
// rounded to 11 more.  s is a row's own, or shared by the rows of a tile when they are of similar size: it puts the largest
// magnitude into [2^14, 2^15), so that a value 2^-17 of it still has all 22 bits and the error of any value is below 2^-39
// of the largest.  A product is
// lo.hi + hi.lo + hi.hi in fp32 accumulators (lo.lo is below 2^-22 of it): three fp16 instructions at twice the rate of the
// tf32 ones that the dot kernels use, and half their bytes in shared memory.
//
// Tiles are kept as images of 128 rows: [hi | lo][panels of 64 columns][128 rows][128 bytes], 16-byte chunks of a row
// permuted by the row's number modulo 8 (the 128-byte swizzle).  The same image serves as an operand contracted over
// its columns (K-major descriptor) and as one contracted over its rows (MN-major descriptor), and it is one run of memory,
// so a plain bulk copy brings it in.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace adb {
namespace tc16 {

constexpr int ROWS = 128;
constexpr int PANEL_BYTES = ROWS * 128;                     // 64 columns of 128 rows
__host__ __device__ constexpr int image_bytes(int panels) { return 2 * panels * PANEL_BYTES; }
constexpr uint32_t SPIN_LIMIT = 1u << 22;                   // bounded waits: about half a second, then the kernel gives up

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false when the block was told to stop or the limit ran out (the block is then told, and `code` goes to the status word)
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* stop, int* status, int code) {
    for (uint32_t it = 0; it < SPIN_LIMIT; it++) {
        if (bar_test(bar, parity)) return true;
        if (*stop) return false;
        if (it > 64) __nanosleep(64);
    }
    *stop = 1;
    atomicCAS(status, 0, code);
    return false;
}
// the warp's lanes wait together and agree on the outcome
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* stop, int* status, int code) {
    const bool ok = bar_wait(bar, parity, stop, status, code);
    return __all_sync(0xffffffffu, ok);
}
// bytes from memory, both addresses on 16-byte boundaries
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
// Products are issued by a whole warp that runs in step, one lane of which (`elected`) takes the instruction: the tensor
// instructions want their operands in uniform registers, and a value that the compiler knows to be the same in all lanes is
// there already.  Issued from a branch that only one lane enters, every operand of every instruction is moved over first:
// the gradient kernels, whose instructions should take 32 and 64 cycles, then spent 140 to 165 on each.
__device__ __forceinline__ uint32_t elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// the barrier arrives once every instruction issued so far by this lane has finished
__device__ __forceinline__ void mma_commit(uint32_t elected, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected) : "memory");
}

// Shared-memory descriptor, 128-byte swizzle, strides in bytes.  Its low word (address and leading stride) may be moved by
// a distance / 16; the high word depends on the layout alone.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFF) >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t DESC_HIGH = (1024u >> 4) | 1u << 14 | 2u << 29;   // groups of 8 rows 1024 bytes apart
// fp16 operands, fp32 accumulator, M = 128; the second operand contracted over its rows (MN-major) or its columns
__host__ __device__ constexpr uint32_t idesc(int n, bool b_rows, int m = 128) {
    return (1u << 4) | (b_rows ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}
// First operand in tensor memory (lane = row, a column holds two neighbouring fp16 values), second in shared memory.
// An operand made of halves has 16 columns for 16 elements: 8 with the high halves, then 8 with the low ones, so that it can
// take the place of the 16 fp32 values it was made from.
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 y;\n\t"
        "setp.ne.b32 e, %6, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(accumulate), "r"(DESC_HIGH), "r"(elected) : "memory");
}
// both operands in shared memory
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\t"
        "setp.ne.b32 e, %6, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 x, {%1, %5};\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(accumulate), "r"(DESC_HIGH), "r"(elected) : "memory");
}

// 32 columns of the warp's 32 lanes; the values may be used after tmem_wait_load
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { tmem_load32(taddr, r); }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) { tmem_load16(taddr, r); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two values as a pair of fp16 and the pair of what that rounding left
__device__ __forceinline__ void halves(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - back.x, y - back.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// 16 elements of a row as an operand, in 16 columns
__device__ __forceinline__ void tmem_store_halves(uint32_t taddr, const float* x, float f) {
    uint32_t r[16];
#pragma unroll
    for (int k = 0; k < 8; k++) halves(x[2 * k] * f, x[2 * k + 1] * f, r[k], r[8 + k]);
    tmem_store16(taddr, r);
}
// The power of two that divides a magnitude into [2^14, 2^15), whatever finite number it is: 2^113 for the largest.  It and
// its inverse are normal numbers: from 2^-112 downwards it is 2^-126, of which half of fp16's smallest step is still less
// than an fp32 subnormal.  Zero gets that too.
__device__ __forceinline__ float tile_scale(float largest) {
    const int e = min(max(int(__float_as_uint(fmaxf(largest, 0.f)) >> 23) - 127 - 14, -126), 113);
    return __uint_as_float(uint32_t(e + 127) << 23);
}
__device__ __forceinline__ float finite_magnitude(float x) {
    const float m = fabsf(x);
    return m < INFINITY ? m : 0.f;
}

}  // namespace tc16
}  // namespace adb
