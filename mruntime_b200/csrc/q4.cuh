// q4.cuh -- 4-bit codes as tensor-core operands, shared by the 4-bit weight
// product (gemv_q4.cu) and the attention over 4-bit keys and values
// (kv_q4_attn.cu).
//
// A code c in 0..15 placed in the low mantissa bits of an otherwise zero FP16
// is the subnormal c * 2^-24, and in the next four bits c * 2^-20; the tensor
// cores multiply FP16 subnormals exactly, so a 32-bit word of eight codes
// becomes four operand registers with four ANDs and one shift, without a
// conversion or a subtraction.  The powers of two and the zero points are
// taken out of the FP32 sums afterwards.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace mrt {

constexpr uint32_t kNib0 = 0x000F000Fu;  // codes at bits 0-3 of each half: value c * 2^-24
constexpr uint32_t kNib1 = 0x00F000F0u;  // codes at bits 4-7 of each half: value c * 2^-20

// Nibble position, within the 32-bit word of eight consecutive columns, of
// column j: (0,1) -> nibbles 0 and 4, (2,3) -> 2 and 6, (4,5) -> 1 and 5,
// (6,7) -> 3 and 7.  One mask yields two neighbouring columns as the halves of
// an operand register, the word and the word shifted by eight with the first
// mask columns 0-3, with the second 4-7: the other operand's registers are
// neighbours of one 16-byte load.
__host__ __device__ __forceinline__ int pair_nibble(int j) {
    return ((j & 1) << 2) | (j & 2) | (j >> 2);
}

// D += A(16 x 16, row) * B(16 x 8, col), FP16 operands, FP32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A * B.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// The 8 x 8 matrix of 16-bit values that a warp holds one row pair a lane, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

// The hardware's own forms, off by some 2^-22: far below the roundings to 16 bits
// that follow wherever they are used.  (They take a denormal for zero.)
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float fast_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Asynchronous 16-byte copy global -> shared (zeros when !valid; src must be readable all the same).
__device__ __forceinline__ void copy_async_16(uint32_t smem_dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(smem_dst), "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}

__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A kernel's attributes, set once a device: its dynamic shared memory, and all of
// a multiprocessor's memory as shared memory.  (These kernels run beside the last
// CTAs of the one before and the first of the next: where one asks for another
// share, it keeps the next one's CTAs off the multiprocessors that it is on.)
template <auto KERNEL>
cudaError_t prepare_kernel(int smem) {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
    return e;
}

// Two FP32 values in one 64-bit register pair.  (A product of pairs that only a
// sum uses is fused with it: use them where one rounding is as good as two.)
__device__ __forceinline__ uint64_t pair2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}

__device__ __forceinline__ uint64_t pair2(float lo, float hi) { return pair2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float low2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

}  // namespace mrt
