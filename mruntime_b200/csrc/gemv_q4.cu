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
// Layout.  Rows in tiles of 16, columns in blocks of 128; a (tile, block) is one
// contiguous piece, brought in by one bulk copy:
//
//   codes   1 KB in the order of the MMA's A fragments: [row half][lane][16
//           bytes], lane (r, c) = (lane / 4, lane % 4) holding for row r (+ 8 in
//           the second half) four words, word i = the codes of columns 32 i + 8 c
//           .. + 7, so that each 32-column stretch of the sum is one word deep in
//           every lane (groups of 32 end between words)
//   scales  [r][group of the block] FP16 pairs (row r, row r + 8)
//   zeros   [r][group of the block] bytes, row r in the low half, padded to 16
//           bytes; absent when every zero point is 8
//
// Columns past K have scale 0.
#include <algorithm>
#include <string>
#include <vector>

#include "common.cuh"
#include "ctx.h"
#include "kernels.h"
#include "q4.cuh"

namespace mrt {

// How a launch runs (plan_gemv()).
struct GemvPlan {
    int warps = 0, tiles = 0, ks = 0;  // warps and tiles of a CTA; slices of K.  0: no such launch
    int per_sm = 0;                    // CTAs a multiprocessor
    int share = 0;                     // block pairs of a warp
    bool joins = false;                // warps share tiles
    int at_once = 0;                   // row tiles of a launch
    double us = 0.0;                   // of all launches, as told
};
constexpr int kMaxTokens = 16;  // of a launch: two token tiles of eight

}  // namespace mrt

// Opaque handle of the public header.
struct mrt_weight_q4_s {
    int device = -1;
    int64_t n = 0, k = 0, group = 0;
    int64_t tiles = 0;   // ceil(n / 16)
    int64_t blocks = 0;  // ceil(k / 128)
    bool zeros = false;  // zero points of its own (else all are 8)
    int piece = 0;       // bytes of a (tile, block)
    uint8_t* data = nullptr;
    uint16_t* bias = nullptr;    // FP16 [n] or null
    mrt::GemvPlan plans[mrt::kMaxTokens + 1];  // by tokens
};

namespace mrt {
namespace {

// Warps that a multiprocessor's registers have room for, by token tiles.
__host__ __device__ constexpr int most_warps(int nt) { return nt == 1 ? 24 : 16; }

// Barrier of the CTAs of a cluster (every thread).
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A shared-memory address as CTA `rank` of the cluster has it.
__device__ __forceinline__ uint32_t cluster_address(uint32_t smem_addr, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr), "r"(rank));
    return a;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
    if (dt == MRT_FP32) return static_cast<const float*>(p)[i];
    const uint16_t v = static_cast<const uint16_t*>(p)[i];
    return dt == MRT_BF16 ? bf16_bits_to_f32(v) : f16_bits_to_f32(v);
}

// ------------------------------------------------------------------ upload

struct Q4Store {
    uint8_t* data;
    int piece, zeros;
    int64_t n, k, group, blocks;
    __device__ __forceinline__ uint8_t* at(int64_t tile, int64_t block) const { return data + (tile * blocks + block) * piece; }
};

constexpr int kCodeBytes = 1024;
__host__ __device__ __forceinline__ int zeros_at(int per) { return kCodeBytes + per * 32; }
__host__ __device__ __forceinline__ int piece_bytes(int per, bool zeros) {
    return zeros_at(per) + (zeros ? (per * 8 + 15) / 16 * 16 : 0);
}

// The word of columns k .. k + 7 (k a multiple of 8) of row n.
__device__ __forceinline__ uint32_t* word_of(const Q4Store& w, int64_t n, int64_t k) {
    const int row = static_cast<int>(n & 15), kk = static_cast<int>(k & 127);
    return reinterpret_cast<uint32_t*>(w.at(n >> 4, k >> 7)) + ((row >> 3) * 32 + (row & 7) * 4 + ((kk >> 3) & 3)) * 4 + (kk >> 5);
}

// Scale and zero point of group g of row n.
__device__ __forceinline__ uint16_t* scale_of(const Q4Store& w, int64_t n, int64_t g) {
    const int per = static_cast<int>(128 / w.group);
    const int i = static_cast<int>(n & 7) * per + static_cast<int>(g % per);
    return reinterpret_cast<uint16_t*>(w.at(n >> 4, g / per) + kCodeBytes) + i * 2 + ((n >> 3) & 1);
}

__device__ __forceinline__ uint8_t* zero_of(const Q4Store& w, int64_t n, int64_t g) {
    const int per = static_cast<int>(128 / w.group);
    return w.at(n >> 4, g / per) + zeros_at(per) + static_cast<int>(n & 7) * per + static_cast<int>(g % per);
}

// Codes given: [n][k / 2] bytes, the even column in the low half.
__global__ void q4_import_kernel(const uint8_t* codes, const void* scales, int sdt, const uint8_t* zeros, Q4Store w) {
    const int64_t tile = blockIdx.x / w.blocks, block = blockIdx.x - tile * w.blocks;
    const int per = static_cast<int>(128 / w.group);
    const int64_t groups = w.k / w.group;
    uint8_t* piece = w.at(tile, block);
    const int t = threadIdx.x;  // one thread a word
    const int64_t n = tile * 16 + (t >> 7) * 8 + ((t >> 4) & 7), k = block * 128 + (t & 3) * 32 + ((t >> 2) & 3) * 8;
    uint32_t word = 0;
    if (n < w.n && k < w.k) {
        const uint8_t* src = codes + n * (w.k / 2) + k / 2;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t b = src[j];
            word |= (b & 15u) << (4 * pair_nibble(2 * j)) | (b >> 4) << (4 * pair_nibble(2 * j + 1));
        }
    }
    reinterpret_cast<uint32_t*>(piece)[t] = word;
    if (t < 8 * per) {  // one thread a pair of rows of a group
        const int64_t g = block * per + t % per;
        uint32_t pair = 0, zero = 0;
        for (int h = 0; h < 2; ++h) {
            const int64_t row = tile * 16 + t / per + h * 8;
            if (row >= w.n || g >= groups) continue;
            pair |= static_cast<uint32_t>(f32_to_f16_bits(ld_any(scales, sdt, row * groups + g))) << (16 * h);
            if (zeros != nullptr) zero |= (zeros[row * groups + g] & 15u) << (4 * h);
        }
        reinterpret_cast<uint32_t*>(piece + kCodeBytes)[t] = pair;
        if (w.zeros) piece[zeros_at(per) + t] = static_cast<uint8_t>(zero);
    }
}

// Codes from a full-precision weight: round to nearest on the group's range,
// widened to hold zero (asymmetric) or centred on code 8 (symmetric).  One warp
// per (row, group); storage is zeroed before.
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
    const float step = w.zeros ? __fmul_rn(hi - lo, 1.0f / 15.0f) : __fmul_rn(fmaxf(-lo, hi), 1.0f / 7.0f);
    const uint16_t sb = f32_to_f16_bits(fminf(fmaxf(step, 5.9604644775390625e-8f), 65504.0f));
    const float inv = __fdiv_rn(1.0f, f16_bits_to_f32(sb));
    const float z = w.zeros ? fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f) : 8.0f;
    for (int j = lane; j < w.group; j += 32) {
        const int64_t k = g * w.group + j;
        const float c = rintf(__fmul_rn(ld_any(src, dt, n * w.k + k), inv)) + z;
        const uint32_t code = static_cast<uint32_t>(fminf(fmaxf(c, 0.0f), 15.0f));  // NaN becomes code 0
        atomicOr(word_of(w, n, k), code << (4 * pair_nibble(static_cast<int>(k & 7))));
    }
    if (lane == 0) {
        *scale_of(w, n, g) = sb;
        if (w.zeros) {
            uint8_t* p = zero_of(w, n, g);
            const uintptr_t a = reinterpret_cast<uintptr_t>(p);
            atomicOr(reinterpret_cast<uint32_t*>(a & ~uintptr_t(3)),
                     static_cast<uint32_t>(z) << (8 * (a & 3) + 4 * ((n >> 3) & 1)));
        }
    }
}

__global__ void q4_read_kernel(Q4Store w, uint16_t* dst, int64_t ld) {
    const int64_t total = w.n * w.k;
    for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < total;
         e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t n = e / w.k, k = e - n * w.k;
        const int c = (*word_of(w, n, k) >> (4 * pair_nibble(static_cast<int>(k & 7)))) & 15;
        const int z = w.zeros ? (*zero_of(w, n, k / w.group) >> (4 * ((n >> 3) & 1))) & 15 : 8;
        dst[n * ld + k] = f32_to_f16_bits(__fmul_rn(f16_bits_to_f32(*scale_of(w, n, k / w.group)), static_cast<float>(c - z)));
    }
}

// ------------------------------------------------------------------ product

struct GemvQ4Args {
    const uint8_t* data;
    int piece, zeros;
    int n, k, blocks, tiles;
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
    int tiles_cta;  // row tiles of a CTA
    int share;      // block pairs of a warp
    int slice;      // column blocks of a CTA
    int stages;     // pieces that a warp has under way
    int* err_flag;
};

constexpr int kMaxStages = 4, kMinStages = 2;
constexpr int kPair = 2;  // neighbouring pieces that a stage holds
constexpr int kSmemMost = 218 * 1024;  // of a multiprocessor's CTAs together

// Shared memory: the warps' rings; x rows of the CTA's columns, 64 bytes apart
// from a multiple of 128 so that eight rows' reads fall into different banks;
// their group sums; two sums a warp of tiles that it shares.
__host__ __device__ __forceinline__ int x_stride(int slice) { return slice * 256 + 64; }
__host__ __device__ __forceinline__ int gemv_smem(int M, int slice, int per, int nt, int warps, bool sums, int stages, int piece) {
    return warps * stages * kPair * piece + M * x_stride(slice) + slice * per * nt * 32 + (sums ? 2 * warps * 16 * nt * 32 : 0);
}

// Wait for a bulk copy, bounded like every wait of the library; once one has
// given up (`late`) the warp's others hardly wait.
__device__ __forceinline__ void wait_piece(uint64_t* bar, uint32_t parity, int* flag, bool& late) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t it = 1; !mbar_try_wait(bar, parity); ++it) {
        if ((it & 255u) != 0) continue;
        if (t0 == 0) t0 = globaltimer_ns();
        if (globaltimer_ns() - t0 > (late ? kWaitLimitNs >> 10 : kWaitLimitNs)) {
            late = true;
            raise_error(flag, kErrTmaWait);
            return;
        }
    }
}

__device__ __forceinline__ void store_y(const GemvQ4Args& a, int64_t n, int m, float sum) {
    const float v = sum * 16777216.0f;
    if (a.out_f32) {
        static_cast<float*>(a.y)[m * a.ldy + n] = v;
    } else {
        const uint16_t h = round_out(v, a.bias, n);
        static_cast<uint16_t*>(a.y)[m * a.ldy + n] = add_residual(h, a.res, m * a.ldr + n);
    }
}

// What bounds it: for few tokens the weights' bytes, so every warp keeps up to
// eight pieces of them under way (two a copy), the first before it waits for the
// kernel that makes x (with loads into registers, four deep, a warp waited for
// more than it asked for: 21.5 us for 37888 x 3584 at one token); and the chain of
// instructions that make operands of a piece (about 140 a KB): 15.4 us for 37888 x
// 3584 at one token (70.6 MB, 4.6 TB/s), 70 for 152064 x 3584 at 16 (286 MB, 4.1
// TB/s: beside them x from shared memory, eight KB a KB of codes).  No unit is full
// there: at one token issue slots are at 50%, the ALU at 48, four warps a scheduler
// that issue every 7.5 cycles, 1.9 of them the instructions' own latency, 1.2 pieces
// and 1.0 the ALU.  Small
// weights are bound by a launch and x's way into the CTAs: 896 x 896 3.2 us;
// long sums of several tokens by x in every CTA: 3584 x 18944 at 7, groups of
// 32, 18 us (40 MB).  x is brought in once a CTA, with its group sums, and CTAs
// stay for all the row tiles they take.
//
// Split.  A CTA has row tiles next to one another (grid x) and a slice of the
// columns (grid y); its tiles' block pairs, in order, are dealt to its warps in
// equal stretches, so that all warps work to the end whatever the shape (with a
// warp a tile, or a fixed number of warps a tile, 152064 x 3584 took 80 us at 16
// tokens, 57 at one; now 70 and 50; a small weight's end is 0.2 us longer).  A warp
// that has a whole tile stores it; the others leave their sums in shared memory
// (at most two a warp: of the tile it begins in and of the one it ends in),
// and they are added in order.  Slices' sums the CTAs of a cluster (1, KS) add
// through each other's shared memory, each a part of the rows.
template <int PER, int NT, bool ZEROS>
__global__ void __launch_bounds__(most_warps(NT) * 32, 1) gemv_q4_kernel(const GemvQ4Args a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t s_full[most_warps(NT)][kMaxStages];
    __shared__ int2 s_first[32];  // the shared tile that a warp is the first of (-1: none), its pairs of it
    const int warps = blockDim.x >> 5, threads = blockDim.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int stage_bytes = kPair * a.piece;
    uint8_t* ring = smem + warp * a.stages * stage_bytes;
    uint8_t* xb = smem + warps * a.stages * stage_bytes;
    const int stride = x_stride(a.slice);
    float* xs = reinterpret_cast<float*>(xb + a.M * stride);  // [group of the slice][NT * 8]
    float* red = xs + a.slice * PER * NT * 8;                 // [warp][2][16][NT * 8]
    const int b0 = blockIdx.y * a.slice, nb = min(a.slice, a.blocks - b0);
    // The warp's stretch.  (A last slice that is short counts its tiles' pairs like
    // the others, so that shares are alike in all CTAs of a cluster.)
    const int tile_lo = blockIdx.x * a.tiles_cta, here = min(a.tiles_cta, a.tiles - tile_lo);
    const int pairs = (a.slice + kPair - 1) / kPair, real = (nb + kPair - 1) / kPair;
    const int total = here * pairs, per = a.share;
    const int p0 = min(warp * per, total), p1 = min(p0 + per, total);
    // The next pair to fetch (lane 0's), and its place in its tile.
    const int t0 = p0 / pairs;
    int f_p = p0, f_in = p0 - t0 * pairs;
    const uint8_t* f_src = a.data + (static_cast<int64_t>(tile_lo + t0) * a.blocks + b0) * a.piece;
    auto fetch = [&](int stage) {
        if (lane != 0) return;
        if (f_in >= real) {
            f_p += pairs - f_in;
            f_in = 0;
            f_src += static_cast<int64_t>(a.blocks) * a.piece;
        }
        if (f_p >= p1) return;
        const uint32_t bytes = nb - f_in * kPair >= kPair ? stage_bytes : a.piece;
        mbar_arrive_expect_tx(&s_full[warp][stage], bytes);
        bulk_load(ring + stage * stage_bytes, f_src + f_in * stage_bytes, bytes, &s_full[warp][stage]);
        ++f_p;
        ++f_in;
    };
    if (lane == 0) {
        for (int i = 0; i < a.stages; ++i) mbar_init(&s_full[warp][i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    for (int i = 0; i < a.stages; ++i) fetch(i);

    griddep_wait();
    griddep_launch_dependents();
    // x, 8 columns a thread and step, and the groups' sums: four loads under way a
    // thread, whole warps, so that a group's lanes are there for its sum.
    const int row_chunks = nb * 16, chunks = a.M * row_chunks;
    for (int i0 = threadIdx.x; i0 < (chunks + 31) / 32 * 32; i0 += threads * 4) {
        uint4 v[4];
        int at[4];  // token and chunk of its row
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = i0 + q * threads, m = i / row_chunks, p = i - m * row_chunks, k = b0 * 128 + p * 8;
            at[q] = m << 16 | p;
            v[q] = make_uint4(0, 0, 0, 0);
            if (m < a.M && k < a.k) {  // K is a multiple of 32
                const uint16_t* src = a.x + m * a.ldx + k;
                if (a.x_vec) {
                    v[q] = *reinterpret_cast<const uint4*>(src);
                } else {
                    v[q].x = src[0] | static_cast<uint32_t>(src[1]) << 16;
                    v[q].y = src[2] | static_cast<uint32_t>(src[3]) << 16;
                    v[q].z = src[4] | static_cast<uint32_t>(src[5]) << 16;
                    v[q].w = src[6] | static_cast<uint32_t>(src[7]) << 16;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int m = at[q] >> 16, p = at[q] & 0xFFFF;
            const uint32_t h[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
                s += f.x + f.y;
            }
            constexpr int kLanes = 16 / PER;  // lanes of a group
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (m < a.M) {
                *reinterpret_cast<uint4*>(xb + m * stride + p * 16) = v[q];
                if ((p & (kLanes - 1)) == 0) xs[(p / kLanes) * NT * 8 + m] = s * 5.9604644775390625e-8f;
            }
        }
    }
    __syncthreads();

    int stage = 0;
    uint32_t phase = 0;
    bool late = false;
    // Columns past M of a token tile repeat its last token: never stored.
    const uint8_t* x_row[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) x_row[t] = xb + min(t * 8 + r, a.M - 1) * stride + c * 16;
    int in = p0 - t0 * pairs, tile = tile_lo + t0;
    int2 first = make_int2(-1, 0);
    for (int p = p0; p < p1; in = 0, ++tile) {
        const int count = min(p1 - p, pairs - in);  // of this tile
        uint64_t tot[NT][2];  // rows r and r + 8: tokens 2c, 2c + 1 of a token tile
#pragma unroll
        for (int t = 0; t < NT; ++t) tot[t][0] = tot[t][1] = 0;
#pragma unroll 1
        for (int b = in * kPair, b1 = min((in + count) * kPair, nb); b < b1; b += kPair) {
            wait_piece(&s_full[warp][stage], phase, a.err_flag, late);
            const uint8_t* piece = ring + stage * stage_bytes;
            uint4 lo[kPair], hi[kPair];
            uint32_t sp[kPair][PER], zp[kPair];
#pragma unroll
            for (int u = 0; u < kPair; ++u, piece += a.piece) {  // (of a lone block the second is an old one: not used)
                lo[u] = *reinterpret_cast<const uint4*>(piece + lane * 16);
                hi[u] = *reinterpret_cast<const uint4*>(piece + 512 + lane * 16);
                if constexpr (PER == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(piece + kCodeBytes + r * 16);
                    sp[u][0] = v.x; sp[u][1] = v.y; sp[u][2] = v.z; sp[u][3] = v.w;
                    zp[u] = ZEROS ? *reinterpret_cast<const uint32_t*>(piece + zeros_at(PER) + r * 4) : 0u;
                } else if constexpr (PER == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(piece + kCodeBytes + r * 8);
                    sp[u][0] = v.x; sp[u][1] = v.y;
                    zp[u] = ZEROS ? *reinterpret_cast<const uint16_t*>(piece + zeros_at(PER) + r * 2) : 0u;
                } else {
                    sp[u][0] = *reinterpret_cast<const uint32_t*>(piece + kCodeBytes + r * 4);
                    zp[u] = ZEROS ? piece[zeros_at(PER) + r] : 0u;
                }
            }
            __syncwarp();
            fetch(stage);
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1;
            }
#pragma unroll
            for (int u = 0; u < kPair; ++u) {
                if (b + u >= nb) break;
                const uint32_t w0[4] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w}, w1[4] = {hi[u].x, hi[u].y, hi[u].z, hi[u].w};
                float ev[NT][4], od[NT][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    constexpr int kWords = 4 / PER;  // of a group
                    const uint32_t u0 = w0[i] >> 8, u1 = w1[i] >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint4 x = *reinterpret_cast<const uint4*>(x_row[t] + (b + u) * 256 + i * 64);
                        if (i % kWords == 0) {
                            mma_f16_first(ev[t], w0[i] & kNib0, w1[i] & kNib0, u0 & kNib0, u1 & kNib0, x.x, x.y);
                            mma_f16_first(od[t], w0[i] & kNib1, w1[i] & kNib1, u0 & kNib1, u1 & kNib1, x.z, x.w);
                        } else {
                            mma_f16(ev[t], w0[i] & kNib0, w1[i] & kNib0, u0 & kNib0, u1 & kNib0, x.x, x.y);
                            mma_f16(od[t], w0[i] & kNib1, w1[i] & kNib1, u0 & kNib1, u1 & kNib1, x.z, x.w);
                        }
                    }
                    if ((i + 1) % kWords == 0) {  // the group ends here
                        const int g = i / kWords;
                        const float s0 = f16_bits_to_f32(static_cast<uint16_t>(sp[u][g])), s1 = f16_bits_to_f32(static_cast<uint16_t>(sp[u][g] >> 16));
                        // (2^23 + z in FP32 is 0x4B000000 | z)
                        const float z0 = ZEROS ? __uint_as_float(0x4B000000u | ((zp[u] >> (8 * g)) & 15u)) - 8388608.0f : 8.0f;
                        const float z1 = ZEROS ? __uint_as_float(0x4B000000u | ((zp[u] >> (8 * g + 4)) & 15u)) - 8388608.0f : 8.0f;
                        const float* xg = xs + ((b + u) * PER + g) * NT * 8 + c * 2;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const uint64_t sx = *reinterpret_cast<const uint64_t*>(xg + t * 8);
                            const uint64_t sixteenth = pair2(0.0625f, 0.0625f);
                            const uint64_t e0 = fma2(pair2(od[t][0], od[t][1]), sixteenth, pair2(ev[t][0], ev[t][1]));
                            const uint64_t e1 = fma2(pair2(od[t][2], od[t][3]), sixteenth, pair2(ev[t][2], ev[t][3]));
                            tot[t][0] = fma2(pair2(s0, s0), fma2(pair2(-z0, -z0), sx, e0), tot[t][0]);
                            tot[t][1] = fma2(pair2(s1, s1), fma2(pair2(-z1, -z1), sx, e1), tot[t][1]);
                        }
                    }
                }
            }
        }
        if (count == pairs && gridDim.y == 1) {  // the warp has whole sums
            const int64_t n = tile * 16LL + r;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int m = t * 8 + c * 2 + (j & 1);
                    const int64_t row = n + (j >> 1) * 8;
                    if (m < a.M && row < a.n) store_y(a, row, m, (j & 1) ? high2(tot[t][j >> 1]) : low2(tot[t][j >> 1]));
                }
        } else {
            const int place = p == p0 ? 0 : 1;
            if (in == 0) first = make_int2(tile * 2 + place, count);
            float* part = red + (warp * 2 + place) * 16 * NT * 8;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                *reinterpret_cast<uint64_t*>(part + r * NT * 8 + t * 8 + c * 2) = tot[t][0];
                *reinterpret_cast<uint64_t*>(part + (r + 8) * NT * 8 + t * 8 + c * 2) = tot[t][1];
            }
        }
        p += count;
    }
    if (gridDim.y == 1 && a.share % pairs == 0) return;  // no tile is shared
    if (lane == 0) s_first[warp] = first;
    const int ranks = gridDim.y, rank = blockIdx.y, halves = threads >> 4, row = threadIdx.x & 15;
    if (ranks == 1) __syncthreads();
    else cluster_barrier();
    // Half a warp a (tile, token): the first warp's part, then those of the warps
    // that begin inside the tile.
    const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, lane < warps && s_first[lane].x >= 0);
    constexpr int kPart = 16 * NT * 8;
    for (int q = rank * halves + (threadIdx.x >> 4);; q += ranks * halves) {
        uint32_t rest = firsts;
        int m = q;
        for (; rest != 0 && m >= a.M; m -= a.M) rest &= rest - 1;
        if (rest == 0) break;
        const int w = __ffs(rest) - 1;
        const int2 f = s_first[w];
        const int64_t n = (f.x >> 1) * 16LL + row;
        if (n >= a.n) continue;
        const float* part = red + (w * 2 + (f.x & 1)) * kPart + row * NT * 8 + m;
        float s = 0.0f;
        if (ranks == 1) {
            s = *part;
            part = red + (w * 2 + 2) * kPart + row * NT * 8 + m;
            for (int have = f.y; have < pairs; part += 8 * kPart) {  // four asked for, then added
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k, have += a.share) x[k] = have < pairs ? part[k * 2 * kPart] : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) s += x[k];
            }
        } else {
            for (int v = w, have = f.y;; have += a.share) {
                const uint32_t at = smem_u32(part);
                float x[8];  // all asked for, then added
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = k < ranks ? ld_cluster_f32(cluster_address(at, k)) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) s += x[k];
                if (have >= pairs) break;
                part = red + ++v * 2 * kPart + row * NT * 8 + m;
            }
        }
        store_y(a, n, m, s);
    }
    if (ranks > 1) cluster_barrier();  // the others have read this CTA's sums
}

// Candidates by time, in microseconds.  A multiprocessor with all its warps
// works off a piece in 0.041 us (with four groups in 0.046), a warp alone in
// 0.445; x comes into every CTA from L2; larger CTAs start later, and joining
// sums costs.  The numbers are a fit to every candidate's time for twenty
// weights, 896 x 896 to 152064 x 3584 at 1 to 16 tokens: times are told within
// 12% on average, and the choice costs 2% over the best.
constexpr int kWarps[] = {1, 2, 3, 4, 6, 8, 10, 12, 14, 16, 20, 24};

// `parts`: also launches over a part of the row tiles after one another.  (A
// warp of a CTA with a slice of K keeps two sums, so such a CTA takes no more
// tiles than it has warps.)
GemvPlan plan_gemv(int M, int tiles, int blocks, int per, int piece, int sms, bool parts) {
    GemvPlan best;
    const int nt = M <= 8 ? 1 : 2;
    for (int per_sm = nt == 1 ? 3 : 2; per_sm > 0; --per_sm)
        for (int ks = 1; ks <= 8; ks *= 2)
            for (int warps : kWarps) {
                const int slice = (blocks + ks - 1) / ks, pairs = (slice + kPair - 1) / kPair;
                if (warps * per_sm > most_warps(nt) || (ks > 1 && (ks - 1) * slice >= blocks)) continue;
                // (Clusters of four and eight leave some multiprocessors idle: of 148
                // they reach 132 and 120.)
                const int room = std::max(1, sms * per_sm * (ks < 4 ? 16 : (ks == 4 ? 14 : 13)) / (16 * ks));
                int64_t tiles_cta = (tiles + room - 1) / room;
                int launches = 1, at_once = tiles;
                if (ks > 1 && tiles_cta > warps) {
                    if (!parts) continue;
                    launches = static_cast<int>((tiles_cta + warps - 1) / warps);
                    tiles_cta = (tiles_cta + launches - 1) / launches;
                    at_once = static_cast<int>(room * tiles_cta);
                }
                const int64_t share = (tiles_cta * pairs + warps - 1) / warps;
                if (tiles_cta * pairs < warps) continue;
                const bool joins = ks > 1 || share % pairs != 0;
                if (gemv_smem(M, slice, per, nt, warps, joins, kMinStages, piece) > kSmemMost / per_sm) continue;
                const int64_t ctas = (std::min(at_once, tiles) + tiles_cta - 1) / tiles_cta * ks;
                // of the busiest multiprocessor, of all of them
                const double busiest = static_cast<double>((ctas + sms - 1) / sms) * tiles_cta * slice;
                const double mean = static_cast<double>(std::min(at_once, tiles)) * blocks / sms;
                const double a_piece = (per == 4 ? 0.0463 : 0.0407) * (nt == 1 ? 1.0 : 1.73) * (0.942 + 0.058 * most_warps(nt) / (warps * per_sm));
                const double work = std::max((0.797 * busiest + 0.203 * mean) * a_piece, share * kPair * 0.445);
                const double x = ctas * 256.0 / 11.8e6 * M * slice + M * slice * 16.0 / (warps * 32) * 0.0843;
                const double shares = share < pairs ? std::min<double>(warps, static_cast<double>(pairs) / share) : 1.0;  // of a tile
                const double us = work + x + 0.0574 * warps + (joins ? 0.3 + 0.04 * shares : 0.0) + (ks > 1 ? 2.05 + 0.029 * ks : 0.0);
                if (best.warps == 0 || us * launches < best.us)
                    best = GemvPlan{warps, static_cast<int>(tiles_cta), ks, per_sm, static_cast<int>(share), joins, at_once, us * launches};
            }
    return best;
}

template <int PER, int NT, bool ZEROS>
cudaError_t launch(GemvQ4Args a, const GemvPlan& p, cudaStream_t s) {
    a.stages = kMaxStages;
    auto bytes = [&] { return gemv_smem(a.M, a.slice, PER, NT, p.warps, p.joins, a.stages, a.piece); };
    while (bytes() > kSmemMost / p.per_sm) --a.stages;
    if (a.stages < kMinStages) return cudaErrorInvalidValue;  // (the plan says that they fit)
    cudaError_t e = prepare_kernel<gemv_q4_kernel<PER, NT, ZEROS>>(kSmemMost);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.tiles + p.tiles - 1) / p.tiles), static_cast<unsigned>(p.ks));
    cfg.blockDim = dim3(static_cast<unsigned>(p.warps) * 32);
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes());
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = static_cast<unsigned>(p.ks);
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ks > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, gemv_q4_kernel<PER, NT, ZEROS>, a);
    if (e == cudaSuccess) note_launches(1);
    return e;
}

// Tokens of the next launch: sixteen, or as many as leave x room in shared
// memory (0: not even one does).
int tokens_at_once(const GemvPlan* plans, int64_t M) {
    int m = static_cast<int>(std::min<int64_t>(M, kMaxTokens));
    while (m > 0 && plans[m].warps == 0) m = m > 8 ? 8 : m / 2;
    return m;
}

// Plans of a weight by tokens.  Where no launch can take all of it, launches over
// parts of its rows, unless fewer tokens at a time are quicker (16 tokens on 28768
// x 18944, groups of 32: eight launches, against four over the whole weight).
void plan_weight(GemvPlan* plans, int tiles, int blocks, int per, int piece, int sms) {
    for (int m = 1; m <= kMaxTokens; ++m) {
        plans[m] = plan_gemv(m, tiles, blocks, per, piece, sms, false);
        if (plans[m].warps > 0) continue;
        double us = 0.0;  // of fewer at a time
        for (int left = m, t; left > 0; left -= t) {
            t = tokens_at_once(plans, left);
            if (t == 0) break;
            us += plans[t].us;
        }
        const GemvPlan p = plan_gemv(m, tiles, blocks, per, piece, sms, true);
        if (p.warps > 0 && (us == 0.0 || p.us < us)) plans[m] = p;
    }
}

cudaError_t launch_gemv_q4(GemvQ4Args a, const GemvPlan& p, int per, cudaStream_t s) {
    a.tiles_cta = p.tiles;
    a.share = p.share;
    a.slice = (a.blocks + p.ks - 1) / p.ks;
    const bool z = a.zeros != 0;
    switch (per * 2 + (a.M > 8)) {
        case 2: return z ? launch<1, 1, true>(a, p, s) : launch<1, 1, false>(a, p, s);
        case 3: return z ? launch<1, 2, true>(a, p, s) : launch<1, 2, false>(a, p, s);
        case 4: return z ? launch<2, 1, true>(a, p, s) : launch<2, 1, false>(a, p, s);
        case 5: return z ? launch<2, 2, true>(a, p, s) : launch<2, 2, false>(a, p, s);
        case 8: return z ? launch<4, 1, true>(a, p, s) : launch<4, 1, false>(a, p, s);
        default: return z ? launch<4, 2, true>(a, p, s) : launch<4, 2, false>(a, p, s);
    }
}


// ------------------------------------------------------------------ handles

void free_handle(mrt_weight_q4_s* w) {
    if (w == nullptr) return;
    if (w->data) cudaFree(w->data);
    if (w->bias) cudaFree(w->bias);
    delete w;
}

Q4Store store_of(const mrt_weight_q4_s* w) {
    return Q4Store{w->data, w->piece, w->zeros ? 1 : 0, w->n, w->k, w->group, w->blocks};
}

int check_shape(int64_t N, int64_t K, int64_t group) {
    if (group != 32 && group != 64 && group != 128) return set_error(MRT_ERR_SHAPE, "group must be 32, 64 or 128");
    if (N <= 0 || K <= 0 || N > (1LL << 31) - 16 || K > (1LL << 31) - 128)
        return set_error(MRT_ERR_SHAPE, "N and K must be positive and fit in 31 bits");
    if (K % group != 0) return set_error(MRT_ERR_SHAPE, "K must be a multiple of the group");
    if ((N + 15) / 16 * ((K + 127) / 128) > (1LL << 31) - 1) return set_error(MRT_ERR_SHAPE, "the weight is too large");
    return MRT_OK;
}

bool any_dtype(int dt) { return dt == MRT_FP16 || dt == MRT_BF16 || dt == MRT_FP32; }
size_t dtype_size(int dt) { return dt == MRT_FP32 ? 4 : 2; }

// Handle with its storage, zeroed.
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
    w->zeros = zeros;
    w->piece = piece_bytes(static_cast<int>(128 / group), zeros);
    plan_weight(w->plans, static_cast<int>(w->tiles), static_cast<int>(w->blocks), static_cast<int>(128 / group), w->piece, c->sms);
    const size_t bytes = static_cast<size_t>(w->tiles) * w->blocks * w->piece;
    cudaError_t e = cudaMalloc(&w->data, bytes);
    if (e == cudaSuccess) e = cudaMemsetAsync(w->data, 0, bytes, s);
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

constexpr int kThreads = 256;  // of the upload kernels
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
        q4_import_kernel<<<static_cast<unsigned>(w->tiles * w->blocks), 256, 0, s>>>(
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
    a.piece = w->piece;
    a.zeros = w->zeros ? 1 : 0;
    a.err_flag = c->d_err;
    a.k = static_cast<int>(w->k);
    a.blocks = static_cast<int>(w->blocks);
    a.ldx = ldx;
    a.x_vec = (reinterpret_cast<uintptr_t>(x_dev) & 15) == 0 && (ldx & 7) == 0;
    a.ldy = ldy;
    a.out_f32 = y_dtype == MRT_FP32;
    a.ldr = ldr;
    const int per = static_cast<int>(128 / w->group);
    for (int64_t m = 0; m < M; m += a.M) {
        a.M = tokens_at_once(w->plans, M - m);
        if (a.M == 0) return set_error(MRT_ERR_SHAPE, "K is too large for a token in shared memory");
        const GemvPlan& plan = w->plans[a.M];
        a.x = static_cast<const uint16_t*>(x_dev) + m * ldx;
        for (int64_t t = 0; t < w->tiles; t += plan.at_once) {
            const int64_t row = t * 16;
            a.tiles = static_cast<int>(std::min<int64_t>(w->tiles - t, plan.at_once));
            a.n = static_cast<int>(w->n - row);
            a.data = w->data + t * w->blocks * w->piece;
            a.y = static_cast<uint8_t*>(y_dev) + (m * ldy + row) * (a.out_f32 ? 4 : 2);
            a.bias = use_bias ? w->bias + row : nullptr;
            a.res = res_dev != nullptr ? static_cast<const uint16_t*>(res_dev) + m * ldr + row : nullptr;
            const cudaError_t e = launch_gemv_q4(a, plan, per, static_cast<cudaStream_t>(stream));
            if (e != cudaSuccess) return cuda_error(e, "4-bit gemv launch");
        }
    }
    return MRT_OK;
}
