// gemv_q4.cu -- y = x * W^T for a few tokens with W held as 4-bit codes and a
// scale and a zero point for every `group` columns of a row, and the weight
// handle that holds them (mrt_weight_q4_*).  The 4-bit form of the decode
// products of gemv.cu (the reference's Backend::gemm at few rows,
// src/core/cpu_backend.cpp:72-169).
//
//   y[m][n] = sum_g s[n][g] * ( sum_{k in g} c[n][k] x[m][k]  -  z[n][g] sum_{k in g} x[m][k] )
//
// so the codes go to the tensor cores as they are and the zero points meet
// only the group sums of x, once per (row, group).
//
// Layout.  Rows in tiles of 16, columns in blocks of 128; a (tile, block) is
// 1 KB in the order of the MMA's A fragments: [row half][lane][16 bytes], lane
// (r, c) = (lane / 4, lane % 4) holding for row r (+ 8 in the second half)
// four words, word i = the codes of columns 32 i + 8 c .. + 7, so that each
// 32-column stretch of the sum is one word deep in every lane (groups of 32
// end between words) and a warp's load is 512 contiguous bytes.  Scales:
// [tile][group][r] pairs (row r, row r + 8); zero points the same, one byte
// with row r in the low half.  Columns past K have scale 0.
#include <algorithm>
#include <string>
#include <vector>

#include "common.cuh"
#include "ctx.h"
#include "kernels.h"
#include "q4.cuh"

// Opaque handle of the public header.
struct mrt_weight_q4_s {
    int device = -1;
    int64_t n = 0, k = 0, group = 0;
    int64_t tiles = 0;   // ceil(n / 16)
    int64_t blocks = 0;  // ceil(k / 128)
    uint4* codes = nullptr;      // [tiles][blocks][64]
    uint32_t* scales = nullptr;  // [tiles][blocks * 128 / group][8] FP16 pairs
    uint8_t* zeros = nullptr;    // [tiles][blocks * 128 / group][8], or null: every zero point is 8
    uint16_t* bias = nullptr;    // FP16 [n] or null
};

namespace mrt {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
    if (dt == MRT_FP32) return static_cast<const float*>(p)[i];
    const uint16_t v = static_cast<const uint16_t*>(p)[i];
    return dt == MRT_BF16 ? bf16_bits_to_f32(v) : f16_bits_to_f32(v);
}

// ------------------------------------------------------------------ upload

struct Q4Store {
    uint4* codes;
    uint32_t* scales;
    uint8_t* zeros;
    int64_t n, k, group, blocks;
};

__device__ __forceinline__ void store_code(const Q4Store& w, int64_t n, int64_t k, uint32_t code) {
    const int64_t tile = n >> 4, block = k >> 7;
    const int row = static_cast<int>(n & 15), kk = static_cast<int>(k & 127);
    const int lane = (row & 7) * 4 + ((kk >> 3) & 3);
    uint32_t* word = reinterpret_cast<uint32_t*>(w.codes + (tile * w.blocks + block) * 64 + (row >> 3) * 32 + lane) +
                     (kk >> 5);
    atomicOr(word, code << (4 * pair_nibble(kk & 7)));
}

__device__ __forceinline__ void store_scale(const Q4Store& w, int64_t n, int64_t g, uint16_t scale, uint32_t zero) {
    const int64_t i = ((n >> 4) * (w.blocks * 128 / w.group) + g) * 8 + (n & 7);
    reinterpret_cast<uint16_t*>(w.scales + i)[(n >> 3) & 1] = scale;
    if (w.zeros != nullptr)
        atomicOr(reinterpret_cast<uint32_t*>(w.zeros) + (i >> 2), zero << (8 * (i & 3) + 4 * ((n >> 3) & 1)));
}

// One warp per (row, group).  Codes given ([n][k / 2] bytes, the even column
// in the low half): laid out as they are.
__global__ void q4_import_kernel(const uint8_t* codes, const void* scales, int sdt, const uint8_t* zeros, Q4Store w) {
    const int64_t groups = w.k / w.group;
    const int64_t id = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (id >= w.n * groups) return;
    const int64_t n = id / groups, g = id - n * groups;
    for (int j = lane; j < w.group; j += 32) {
        const int64_t k = g * w.group + j;
        const uint8_t b = codes[n * (w.k / 2) + (k >> 1)];
        store_code(w, n, k, (k & 1) ? b >> 4 : b & 15u);
    }
    if (lane == 0)
        store_scale(w, n, g, f32_to_f16_bits(ld_any(scales, sdt, n * groups + g)),
                    zeros != nullptr ? zeros[n * groups + g] & 15u : 8u);
}

// Codes from a full-precision weight: round to nearest on the group's range,
// widened to hold zero (asymmetric) or centred on code 8 (symmetric).
__global__ void q4_quantise_kernel(const void* src, int dt, Q4Store w) {
    const int64_t groups = w.k / w.group;
    const int64_t id = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (id >= w.n * groups) return;
    const int64_t n = id / groups, g = id - n * groups;
    float lo = 0.0f, hi = 0.0f;
    for (int j = lane; j < w.group; j += 32) {
        const float v = ld_any(src, dt, n * w.k + g * w.group + j);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    const float step = w.zeros != nullptr ? __fmul_rn(hi - lo, 1.0f / 15.0f) : __fmul_rn(fmaxf(-lo, hi), 1.0f / 7.0f);
    const uint16_t sb = f32_to_f16_bits(fminf(fmaxf(step, 5.9604644775390625e-8f), 65504.0f));
    const float inv = __fdiv_rn(1.0f, f16_bits_to_f32(sb));
    const float z = w.zeros != nullptr ? fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f) : 8.0f;
    for (int j = lane; j < w.group; j += 32) {
        const int64_t k = g * w.group + j;
        const float c = rintf(__fmul_rn(ld_any(src, dt, n * w.k + k), inv)) + z;
        store_code(w, n, k, static_cast<uint32_t>(fminf(fmaxf(c, 0.0f), 15.0f)));  // NaN becomes code 0
    }
    if (lane == 0) store_scale(w, n, g, sb, static_cast<uint32_t>(z));
}

__global__ void q4_read_kernel(Q4Store w, uint16_t* dst, int64_t ld) {
    const int64_t total = w.n * w.k;
    for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < total;
         e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t n = e / w.k, k = e - n * w.k;
        const int row = static_cast<int>(n & 15), kk = static_cast<int>(k & 127);
        const int lane = (row & 7) * 4 + ((kk >> 3) & 3);
        const uint32_t word = reinterpret_cast<const uint32_t*>(w.codes + ((n >> 4) * w.blocks + (k >> 7)) * 64 +
                                                                (row >> 3) * 32 + lane)[kk >> 5];
        const int c = (word >> (4 * pair_nibble(kk & 7))) & 15;
        const int64_t i = ((n >> 4) * (w.blocks * 128 / w.group) + k / w.group) * 8 + (n & 7);
        const float s = f16_bits_to_f32(reinterpret_cast<const uint16_t*>(w.scales + i)[(n >> 3) & 1]);
        const int z = w.zeros != nullptr ? (w.zeros[i] >> (4 * ((n >> 3) & 1))) & 15 : 8;
        dst[n * ld + k] = f32_to_f16_bits(__fmul_rn(s, static_cast<float>(c - z)));
    }
}

// ------------------------------------------------------------------ product

struct GemvQ4Args {
    const uint4* codes;
    const uint32_t* scales;
    const uint8_t* zeros;  // or null: 8
    int n, k, blocks, group;
    const uint16_t* x;
    int64_t ldx;
    int x_vec;  // x rows can be read 16 bytes at a time
    void* y;
    int64_t ldy;
    int out_f32;
    const uint16_t* bias;
    const uint16_t* res;
    int64_t ldr;
    int M;
    int chunk;  // column blocks of x in shared memory at a time
};

// Two token tiles of eight at most in one launch.
constexpr int kMaxTokens = 16;

// Bytes of dynamic shared memory: x rows (padded so that eight rows land in
// different banks) and their group sums.
__host__ __device__ __forceinline__ int x_stride(int chunk) { return chunk * 256 + 64; }

// One CTA per 16 rows, its eight warps taking the column blocks in turn.  x is
// staged in shared memory chunk by chunk together with its group sums.
template <int NT>
__global__ void __launch_bounds__(kThreads) gemv_q4_kernel(const GemvQ4Args a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float red[kWarps][16][NT * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int tile = blockIdx.x;
    const int per_block = 128 / a.group;  // groups in a column block
    const int stride = x_stride(a.chunk);
    float* xs = reinterpret_cast<float*>(smem + a.M * stride);  // [group of the chunk][NT * 8]

    griddep_wait();
    griddep_launch_dependents();
    float tot[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) tot[t][j] = 0.0f;

    for (int b0 = 0; b0 < a.blocks; b0 += a.chunk) {
        const int nb = min(a.chunk, a.blocks - b0);
        __syncthreads();
        // Stage x: 8 columns per thread and step, their sum to the group's.
        for (int i = threadIdx.x; i < (a.M * nb * 16 + 31) / 32 * 32; i += kThreads) {
            const int m = i / (nb * 16), p = i - m * nb * 16;
            const int k = b0 * 128 + p * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (m < a.M && k < a.k) {  // K is a multiple of 32
                const uint16_t* src = a.x + m * a.ldx + k;
                if (a.x_vec) {
                    v = *reinterpret_cast<const uint4*>(src);
                } else {
                    v.x = src[0] | static_cast<uint32_t>(src[1]) << 16;
                    v.y = src[2] | static_cast<uint32_t>(src[3]) << 16;
                    v.z = src[4] | static_cast<uint32_t>(src[5]) << 16;
                    v.w = src[6] | static_cast<uint32_t>(src[7]) << 16;
                }
            }
            const uint32_t h[4] = {v.x, v.y, v.z, v.w};
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
                s += f.x + f.y;
            }
            for (int o = 1; o < a.group / 8; o <<= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (m < a.M) {
                *reinterpret_cast<uint4*>(smem + m * stride + p * 16) = v;
                if ((p & (a.group / 8 - 1)) == 0) xs[(p / (a.group / 8)) * NT * 8 + m] = s * 5.9604644775390625e-8f;
            }
        }
        __syncthreads();
        for (int b = warp; b < nb; b += kWarps) {
            const uint4* src = a.codes + (static_cast<int64_t>(tile) * a.blocks + b0 + b) * 64 + lane;
            const uint4 lo = ld_stream_16B(src), hi = ld_stream_16B(src + 32);
            const uint32_t w0[4] = {lo.x, lo.y, lo.z, lo.w}, w1[4] = {hi.x, hi.y, hi.z, hi.w};
            float ev[NT][4], od[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i % (a.group / 32) == 0) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) ev[t][j] = od[t][j] = 0.0f;
                }
                const uint32_t u0 = w0[i] >> 8, u1 = w1[i] >> 8;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (t * 8 + r < a.M)
                        x = *reinterpret_cast<const uint4*>(smem + (t * 8 + r) * stride + b * 256 + i * 64 + c * 16);
                    mma_f16(ev[t], w0[i] & kNib0, w1[i] & kNib0, u0 & kNib0, u1 & kNib0, x.x, x.z);
                    mma_f16(od[t], w0[i] & kNib1, w1[i] & kNib1, u0 & kNib1, u1 & kNib1, x.y, x.w);
                }
                if ((i + 1) % (a.group / 32) == 0) {  // the group ends here
                    const int g = b * per_block + i / (a.group / 32);
                    const int64_t gi = (static_cast<int64_t>(tile) * a.blocks * per_block + b0 * per_block + g) * 8 + r;
                    const uint32_t sp = __ldg(a.scales + gi);
                    const uint32_t zp = a.zeros != nullptr ? __ldg(a.zeros + gi) : 0x88u;
                    const float s0 = f16_bits_to_f32(static_cast<uint16_t>(sp)), s1 = f16_bits_to_f32(static_cast<uint16_t>(sp >> 16));
                    const float z0 = static_cast<float>(zp & 15u), z1 = static_cast<float>(zp >> 4);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float2 sx = *reinterpret_cast<const float2*>(xs + g * NT * 8 + t * 8 + c * 2);
                        const float x0 = t * 8 + c * 2 < a.M ? sx.x : 0.0f, x1 = t * 8 + c * 2 + 1 < a.M ? sx.y : 0.0f;
                        tot[t][0] = fmaf(s0, fmaf(-z0, x0, fmaf(od[t][0], 0.0625f, ev[t][0])), tot[t][0]);
                        tot[t][1] = fmaf(s0, fmaf(-z0, x1, fmaf(od[t][1], 0.0625f, ev[t][1])), tot[t][1]);
                        tot[t][2] = fmaf(s1, fmaf(-z1, x0, fmaf(od[t][2], 0.0625f, ev[t][2])), tot[t][2]);
                        tot[t][3] = fmaf(s1, fmaf(-z1, x1, fmaf(od[t][3], 0.0625f, ev[t][3])), tot[t][3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        red[warp][r][t * 8 + c * 2] = tot[t][0];
        red[warp][r][t * 8 + c * 2 + 1] = tot[t][1];
        red[warp][r + 8][t * 8 + c * 2] = tot[t][2];
        red[warp][r + 8][t * 8 + c * 2 + 1] = tot[t][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * 8; i += kThreads) {
        const int row = i & 15, m = i >> 4;
        const int64_t n = tile * 16LL + row;
        if (m >= a.M || n >= a.n) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += red[w][row][m];
        s *= 16777216.0f;
        if (a.out_f32) {
            static_cast<float*>(a.y)[m * a.ldy + n] = s;
        } else {
            const uint16_t h = round_out(s, a.bias, n);
            static_cast<uint16_t*>(a.y)[m * a.ldy + n] = add_residual(h, a.res, m * a.ldr + n);
        }
    }
}

template <int NT>
cudaError_t launch(const GemvQ4Args& a, cudaStream_t s) {
    const int smem = a.M * x_stride(a.chunk) + a.chunk * (128 / a.group) * NT * 8 * 4;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.n + 15) / 16));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemv_q4_kernel<NT>, a);
    if (e == cudaSuccess) note_launches(1);
    return e;
}

cudaError_t launch_gemv_q4(GemvQ4Args a, cudaStream_t s) {
    // The chunk of x that fits 32 KB (48 KB is what a launch has without asking).
    a.chunk = std::max(1, std::min(a.blocks, 32768 / (a.M * 256 + (128 / a.group) * 64)));
    return a.M <= 8 ? launch<1>(a, s) : launch<2>(a, s);
}

// ------------------------------------------------------------------ handles

void free_handle(mrt_weight_q4_s* w) {
    if (w == nullptr) return;
    if (w->codes) cudaFree(w->codes);
    if (w->scales) cudaFree(w->scales);
    if (w->zeros) cudaFree(w->zeros);
    if (w->bias) cudaFree(w->bias);
    delete w;
}

Q4Store store_of(const mrt_weight_q4_s* w) {
    return Q4Store{w->codes, w->scales, w->zeros, w->n, w->k, w->group, w->blocks};
}

int check_shape(int64_t N, int64_t K, int64_t group) {
    if (group != 32 && group != 64 && group != 128) return set_error(MRT_ERR_SHAPE, "group must be 32, 64 or 128");
    if (N <= 0 || K <= 0 || N > (1LL << 31) - 16 || K > (1LL << 31) - 128)
        return set_error(MRT_ERR_SHAPE, "N and K must be positive and fit in 31 bits");
    if (K % group != 0) return set_error(MRT_ERR_SHAPE, "K must be a multiple of the group");
    return MRT_OK;
}

bool any_dtype(int dt) { return dt == MRT_FP16 || dt == MRT_BF16 || dt == MRT_FP32; }
size_t dtype_size(int dt) { return dt == MRT_FP32 ? 4 : 2; }

// Handle with zeroed storage (codes and zero points are OR-ed in).
int new_handle(int64_t N, int64_t K, int64_t group, bool zeros, cudaStream_t s, mrt_weight_q4_s** out) {
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    mrt_weight_q4_s* w = new mrt_weight_q4_s();
    w->device = c->device;
    w->n = N;
    w->k = K;
    w->group = group;
    w->tiles = (N + 15) / 16;
    w->blocks = (K + 127) / 128;
    const size_t cb = static_cast<size_t>(w->tiles) * w->blocks * 1024;
    const size_t gs = static_cast<size_t>(w->tiles) * (w->blocks * 128 / group) * 8;
    cudaError_t e = cudaMalloc(&w->codes, cb);
    if (e == cudaSuccess) e = cudaMalloc(&w->scales, gs * 4);
    if (e == cudaSuccess && zeros) e = cudaMalloc(&w->zeros, gs);
    if (e == cudaSuccess) e = cudaMemsetAsync(w->codes, 0, cb, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(w->scales, 0, gs * 4, s);
    if (e == cudaSuccess && zeros) e = cudaMemsetAsync(w->zeros, 0, gs, s);
    if (e != cudaSuccess) {
        free_handle(w);
        return cuda_error(e, "allocating 4-bit weight storage");
    }
    *out = w;
    return MRT_OK;
}

// `src` itself when it is on the device, else a staged copy (freed by the caller).
cudaError_t on_device(const void* src, size_t bytes, int src_on_device, cudaStream_t s, const void** out, void** stage) {
    *stage = nullptr;
    *out = src;
    if (src == nullptr || src_on_device) return cudaSuccess;
    cudaError_t e = cudaMalloc(stage, bytes);
    if (e == cudaSuccess) e = cudaMemcpyAsync(*stage, src, bytes, cudaMemcpyHostToDevice, s);
    *out = *stage;
    return e;
}

unsigned warp_blocks(int64_t warps) { return static_cast<unsigned>((warps * 32 + kThreads - 1) / kThreads); }

int finish(mrt_weight_q4_s* w, cudaError_t e, cudaStream_t s, mrt_weight_q4* out) {
    const cudaError_t e2 = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = e2;
    if (e != cudaSuccess) {
        free_handle(w);
        return cuda_error(e, "uploading the 4-bit weight");
    }
    *out = w;
    return MRT_OK;
}

}  // namespace
}  // namespace mrt

using namespace mrt;

extern "C" int mrt_weight_q4_upload(const void* src, int src_dtype, int src_on_device, int64_t N, int64_t K,
                                    int64_t group, int symmetric, void* stream, mrt_weight_q4* out) {
    clear_error();
    if (out == nullptr) return set_error(MRT_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (src == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL weight");
    if (!any_dtype(src_dtype)) return set_error(MRT_ERR_DTYPE, "weight dtype must be FP16, BF16 or FP32");
    int rc = check_shape(N, K, group);
    if (rc != MRT_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    mrt_weight_q4_s* w = nullptr;
    if ((rc = new_handle(N, K, group, !symmetric, s, &w)) != MRT_OK) return rc;
    const void* d = nullptr;
    void* stage = nullptr;
    cudaError_t e = on_device(src, static_cast<size_t>(N) * K * dtype_size(src_dtype), src_on_device, s, &d, &stage);
    if (e == cudaSuccess) {
        q4_quantise_kernel<<<warp_blocks(N * (K / group)), kThreads, 0, s>>>(d, src_dtype, store_of(w));
        note_launches(1);
        e = cudaGetLastError();
    }
    rc = finish(w, e, s, out);
    if (stage) cudaFree(stage);
    return rc;
}

extern "C" int mrt_weight_q4_import(const void* codes, const void* scales, int scale_dtype, const void* zeros,
                                    int src_on_device, int64_t N, int64_t K, int64_t group, void* stream,
                                    mrt_weight_q4* out) {
    clear_error();
    if (out == nullptr) return set_error(MRT_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (codes == nullptr || scales == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL codes or scales");
    if (!any_dtype(scale_dtype)) return set_error(MRT_ERR_DTYPE, "scale dtype must be FP16, BF16 or FP32");
    int rc = check_shape(N, K, group);
    if (rc != MRT_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    mrt_weight_q4_s* w = nullptr;
    if ((rc = new_handle(N, K, group, zeros != nullptr, s, &w)) != MRT_OK) return rc;
    const size_t ng = static_cast<size_t>(N) * (K / group);
    const void *dc = nullptr, *ds = nullptr, *dz = nullptr;
    void *sc = nullptr, *ss = nullptr, *sz = nullptr;
    cudaError_t e = on_device(codes, static_cast<size_t>(N) * (K / 2), src_on_device, s, &dc, &sc);
    if (e == cudaSuccess) e = on_device(scales, ng * dtype_size(scale_dtype), src_on_device, s, &ds, &ss);
    if (e == cudaSuccess) e = on_device(zeros, ng, src_on_device, s, &dz, &sz);
    if (e == cudaSuccess) {
        q4_import_kernel<<<warp_blocks(static_cast<int64_t>(ng)), kThreads, 0, s>>>(
            static_cast<const uint8_t*>(dc), ds, scale_dtype, static_cast<const uint8_t*>(dz), store_of(w));
        note_launches(1);
        e = cudaGetLastError();
    }
    rc = finish(w, e, s, out);
    if (sc) cudaFree(sc);
    if (ss) cudaFree(ss);
    if (sz) cudaFree(sz);
    return rc;
}

extern "C" int mrt_weight_q4_attach_bias(mrt_weight_q4 w, const void* src, int src_dtype, int src_on_device,
                                         void* stream) {
    clear_error();
    if (w == nullptr || src == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL weight or bias");
    if (!any_dtype(src_dtype)) return set_error(MRT_ERR_DTYPE, "bias dtype must be FP16, BF16 or FP32");
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    if (c->device != w->device) return set_error(MRT_ERR_INVALID_ARG, "weight lives on another device");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (w->bias == nullptr) e = cudaMalloc(&w->bias, static_cast<size_t>(w->n) * 2);
    if (e != cudaSuccess) {
        w->bias = nullptr;
        return cuda_error(e, "allocating bias storage");
    }
    const void* d = nullptr;
    void* stage = nullptr;
    e = on_device(src, static_cast<size_t>(w->n) * dtype_size(src_dtype), src_on_device, s, &d, &stage);
    if (e == cudaSuccess) e = launch_convert(d, src_dtype, w->bias, MRT_FP16, w->n, s);
    const cudaError_t e2 = cudaStreamSynchronize(s);
    if (stage) cudaFree(stage);
    if (e == cudaSuccess) e = e2;
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "uploading the bias");
}

extern "C" int mrt_weight_q4_shape(mrt_weight_q4 w, int64_t* n, int64_t* k, int64_t* group) {
    if (w == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL weight");
    if (n) *n = w->n;
    if (k) *k = w->k;
    if (group) *group = w->group;
    return MRT_OK;
}

extern "C" int mrt_weight_q4_read(mrt_weight_q4 w, void* dst_dev, int64_t ld, void* stream) {
    clear_error();
    if (w == nullptr || dst_dev == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL argument");
    if (ld < w->k) return set_error(MRT_ERR_SHAPE, "ld must be >= K");
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    if (c->device != w->device) return set_error(MRT_ERR_INVALID_ARG, "weight lives on another device");
    const int64_t blocks = std::min<int64_t>((w->n * w->k + kThreads - 1) / kThreads, c->sms * 32LL);
    q4_read_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        store_of(w), static_cast<uint16_t*>(dst_dev), ld);
    note_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "reading the 4-bit weight");
}

extern "C" int mrt_weight_q4_free(mrt_weight_q4 w) {
    free_handle(w);
    return MRT_OK;
}

extern "C" int mrt_gemv_q4(mrt_weight_q4 w, const void* x_dev, int64_t ldx, const void* res_dev, int64_t ldr,
                           void* y_dev, int y_dtype, int64_t ldy, int64_t M, unsigned flags, void* stream) {
    clear_error();
    if (w == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL weight");
    if (y_dtype != MRT_FP16 && y_dtype != MRT_FP32) return set_error(MRT_ERR_DTYPE, "y must be FP16 or FP32");
    if (M < 0) return set_error(MRT_ERR_SHAPE, "M must be >= 0");
    if ((flags & ~MRT_GEMM_BIAS) != 0) return set_error(MRT_ERR_INVALID_ARG, "unknown flag");
    const bool use_bias = (flags & MRT_GEMM_BIAS) != 0;
    if (use_bias && w->bias == nullptr) return set_error(MRT_ERR_INVALID_ARG, "MRT_GEMM_BIAS without an attached bias");
    if (y_dtype == MRT_FP32 && (use_bias || res_dev != nullptr))
        return set_error(MRT_ERR_UNSUPPORTED, "bias and residual need an FP16 output");
    if (M == 0) return MRT_OK;
    if (x_dev == nullptr || y_dev == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL x or y");
    if (ldx < w->k || ldy < w->n || (res_dev != nullptr && ldr < w->n))
        return set_error(MRT_ERR_SHAPE, "ldx must be >= K, ldy and ldr >= N");
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    if (c->device != w->device) return set_error(MRT_ERR_INVALID_ARG, "weight lives on another device");
    GemvQ4Args a{};
    a.codes = w->codes;
    a.scales = w->scales;
    a.zeros = w->zeros;
    a.n = static_cast<int>(w->n);
    a.k = static_cast<int>(w->k);
    a.blocks = static_cast<int>(w->blocks);
    a.group = static_cast<int>(w->group);
    a.ldx = ldx;
    a.x_vec = (reinterpret_cast<uintptr_t>(x_dev) & 15) == 0 && (ldx & 7) == 0;
    a.ldy = ldy;
    a.out_f32 = y_dtype == MRT_FP32;
    a.bias = use_bias ? w->bias : nullptr;
    a.ldr = ldr;
    for (int64_t m = 0; m < M; m += kMaxTokens) {
        a.M = static_cast<int>(std::min<int64_t>(kMaxTokens, M - m));
        a.x = static_cast<const uint16_t*>(x_dev) + m * ldx;
        a.y = static_cast<uint8_t*>(y_dev) + m * ldy * (a.out_f32 ? 4 : 2);
        a.res = res_dev != nullptr ? static_cast<const uint16_t*>(res_dev) + m * ldr : nullptr;
        const cudaError_t e = launch_gemv_q4(a, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) return cuda_error(e, "4-bit gemv launch");
    }
    return MRT_OK;
}
