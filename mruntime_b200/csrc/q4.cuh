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

namespace mrt {

constexpr uint32_t kNib0 = 0x000F000Fu;  // codes at bits 0-3 of each half: value c * 2^-24
constexpr uint32_t kNib1 = 0x00F000F0u;  // codes at bits 4-7 of each half: value c * 2^-20

// Nibble position, within the 32-bit word of eight consecutive columns, of
// column j: (0,1) -> nibbles 0 and 4, (2,3) -> 1 and 5, (4,5) -> 2 and 6,
// (6,7) -> 3 and 7, so that one mask yields two neighbouring columns as the
// halves of one operand register.
__host__ __device__ __forceinline__ int pair_nibble(int j) { return (j >> 1) + ((j & 1) << 2); }

// D += A(16 x 16, row) * B(16 x 8, col), FP16 operands, FP32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace mrt
