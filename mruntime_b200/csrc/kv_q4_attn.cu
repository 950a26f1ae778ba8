// kv_q4_attn.cu -- softmax attention of new tokens' queries over a paged cache
// held in 4 bits (kv_q4.h): the reference's attention op
// (src/core/cpu_backend.cpp:171-290) over such a cache.
#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "ctx.h"
#include "kernels.h"
#include "kv_q4.h"
#include "q4.cuh"

namespace mrt {
namespace {

constexpr int kThreads = 256;

struct AttnQ4Args {
    KvView v;
    int dtype, heads, causal;
    float scale;
    const uint16_t* q;
    int64_t ldq;
    uint16_t* out;
    int64_t ldo;
};

__device__ __forceinline__ float widen(uint16_t h, int dtype) {
    return dtype == MRT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

__device__ __forceinline__ uint16_t narrow(float f, int dtype) {
    if (dtype == MRT_FP16) return f32_to_f16_bits(f);
    return f != f ? static_cast<uint16_t>(0x7FC0) : f32_to_bf16_bits(f);
}

// One CTA per token, one warp per query head at a time, one key at a time with
// the running maximum and sum of the softmax.
template <int PER>
__global__ void __launch_bounds__(kThreads) attn_q4_rows_kernel(const AttnQ4Args a) {
    constexpr int D = PER * 32;
    __shared__ int s_seq;
    griddep_wait();
    griddep_launch_dependents();
    const KvView& v = a.v;
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) s_seq = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < v.seqs; b += blockDim.x)
        if (v.q_start[b] <= t && t < v.q_start[b + 1]) s_seq = b;
    __syncthreads();
    const int b = s_seq;
    if (b < 0) return;
    int first, n, kv;
    if (!kv_seq(v, b, &first, &n, &kv)) {
        if (threadIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
        return;
    }
    const int keys = a.causal ? kv - n + (t - first) + 1 : kv;  // may be 0 or less: no key
    for (int h = warp; h < a.heads; h += kThreads / 32) {
        const int kh = h / (a.heads / v.kv_heads);
        float q[PER], o[PER];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            q[j] = widen(a.q[t * a.ldq + h * D + lane * PER + j], a.dtype) * a.scale;
            o[j] = 0.0f;
        }
        const uint8_t* block = nullptr;
        for (int p = 0; p < keys; ++p) {
            const int token = p & (kKvBlock - 1);
            if (token == 0) {
                block = kv_block_at(v, v.table + static_cast<int64_t>(b) * v.ld_table, kh, p);
                if (block == nullptr) {
                    if (lane == 0) raise_error(v.err_flag, kErrBadPage);
                    break;
                }
            }
            const uint32_t ks = reinterpret_cast<const uint32_t*>(block + kv_k_scales(D))[token];
            const uint32_t vs = reinterpret_cast<const uint32_t*>(block + kv_v_scales(D))[token];
            const int w = lane * PER / 8;
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(block + kv_k_word(D, token, w));
            const uint32_t vw = *reinterpret_cast<const uint32_t*>(block + kv_v_word(D, token, w));
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int c = (kw >> (4 * pair_nibble((lane * PER + j) & 7))) & 15;
                s = fmaf(q[j], static_cast<float>(c - static_cast<int>(ks >> 16)), s);
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
            s *= f16_bits_to_f32(static_cast<uint16_t>(ks));
            const float m2 = fmaxf(m, s), fix = expf(m - m2), e = expf(s - m2);
            const float ev = e * f16_bits_to_f32(static_cast<uint16_t>(vs));
            l = l * fix + e;
            m = m2;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int c = (vw >> (4 * ((lane * PER + j) & 7))) & 15;
                o[j] = fmaf(ev, static_cast<float>(c - static_cast<int>(vs >> 16)), o[j] * fix);
            }
        }
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
        for (int j = 0; j < PER; ++j) a.out[t * a.ldo + h * D + lane * PER + j] = narrow(o[j] * inv, a.dtype);
    }
}

// Four neighbouring channels of an output row (any alignment of the row).
__device__ __forceinline__ void store_out4(uint16_t* dst, const AttnQ4Args& a, float4 x, float inv) {
    dst[0] = narrow(x.x * inv, a.dtype);
    dst[1] = narrow(x.y * inv, a.dtype);
    dst[2] = narrow(x.z * inv, a.dtype);
    dst[3] = narrow(x.w * inv, a.dtype);
}

// ------------------------------------------------------------------ few rows

// Rows of one (sequence, kv head) are its new tokens times the query heads that
// share it; up to 32 of them ride as the MMA's N while keys are its M: scores
// S^T[16 keys x 8 rows] = K Q^T, transposed in registers into the second
// product's operand, O^T[16 channels x 8 rows] += V^T P^T.  K and V codes are
// the M operands straight from their bytes (q4.cuh).
//
// Softmax.  In powers of two, with a value's scale taken into the exponent:
// y = scale log2(e) q.k + log2 s_v, p' = 2^(y - m), m the running maximum of y.
// So p' is the probability times its value's scale, relative to the largest
// such product: FP16 operands keep eleven bits of whatever matters, however
// unlike the scales are.  The sum is of p' / s_v, and the zero points' part of
// the output, sum p' z (of the same rounded p'), is one number a row.
//
// Split.  The 32-token tiles of all (sequence, kv head) units, in order, are
// dealt to the CTAs in equal contiguous stretches, whatever the lengths: no
// CTA waits for a long sequence, and no plan from the host is needed (lengths
// are read here).  A CTA's warps take a stretch's tiles in turn, each with its
// own ring of asynchronous copies, and join at the end of the unit.  A unit
// that spans CTAs leaves its parts in scratch (two places a CTA: a unit that
// began earlier, and one that goes on) and attn_q4_join_kernel adds them in
// order.
constexpr int kTile = 32;
constexpr int kTileBlocks = kTile / kKvBlock;

struct RowsArgs {
    AttnQ4Args a;
    int group;          // query heads of a kv head
    int split;          // 0: every unit is one CTA's
    float* part_o;      // [2 * grid][8 NT][D]
    float2* part_ml;    // [2 * grid][8 NT]
    int grid;
};

// Tiles of sequence b (0: none of its rows is computed).
__device__ __forceinline__ int seq_tiles(const KvView& v, int b) {
    int first, n, kv;
    if (!kv_seq(v, b, &first, &n, &kv) || n == 0) return 0;
    return max(1, (kv + kTile - 1) / kTile);
}

// Sum over the block of one 64-bit number a thread (every thread gets it).
template <int W>
__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
    __syncthreads();
    int64_t t = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) t += s[w];
    return t;
}

__device__ __forceinline__ int64_t tiles_a_cta(int64_t total, int grid, int warps) {
    const int64_t per = (total + grid - 1) / grid;
    return per < warps ? warps : per;
}

template <int D, int NT, int W>
struct RowsShape {
    static constexpr int kRows = NT * 8;
    static constexpr int kBlock = kKvBlock * (D + 8);
    static constexpr int kStage = kTileBlocks * kBlock;
    static constexpr int kStages = W > 8 ? 2 : 4;
    static constexpr int kRing = W * kStages * kStage;
    static constexpr int kMerge = W * kRows * D * 4;
    static constexpr int kQ = NT * (D / 32) * 32 * 16;
    static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge) + kQ;
};

// The codes of one word as the halves of two operand registers each.
template <int D, int NT, int W>
__global__ void __launch_bounds__(W * 32) attn_q4_few_kernel(const RowsArgs args) {
    using S = RowsShape<D, NT, W>;
    constexpr int kWords = D / 32;  // words of a lane: K row part, and V channel stretch of two tokens
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_sum[W];
    __shared__ int s_seq;
    __shared__ int64_t s_at;
    __shared__ float s_fac[S::kRows], s_sumq[S::kRows];
    __shared__ int s_limit[S::kRows];
    __shared__ float s_m[W][S::kRows], s_l[W][S::kRows];
    uint8_t* ring = smem;
    float* merge = reinterpret_cast<float*>(smem);  // once the ring has run dry
    uint4* qf = reinterpret_cast<uint4*>(smem + S::kBytes - S::kQ);
    const AttnQ4Args& a = args.a;
    const KvView& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;

    griddep_wait();
    griddep_launch_dependents();

    // This CTA's stretch of the tiles, and the sequence it begins in.
    int64_t mine = 0;
    for (int b = threadIdx.x; b < v.seqs; b += W * 32) {
        mine += seq_tiles(v, b);
        int f, n, kv;
        if (!kv_seq(v, b, &f, &n, &kv) && blockIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
    }
    const int64_t total = block_sum<W>(mine, s_sum) * v.kv_heads;
    int64_t at, end;
    int seq;
    int64_t seq_at;  // tile number at which the sequence begins
    if (args.split) {
        const int64_t per = tiles_a_cta(total, args.grid, W);
        at = blockIdx.x * per;
        end = min(total, at + per);
        if (at >= end) return;
        int64_t before = 0;
        seq = -1;
        seq_at = 0;
        for (int b0 = 0; seq < 0; b0 += W * 32) {  // ends: at < total
            const int b = b0 + threadIdx.x;
            const int64_t t = b < v.seqs ? static_cast<int64_t>(seq_tiles(v, b)) * v.kv_heads : 0;
            int64_t incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t u = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += u;
            }
            __syncthreads();
            if (threadIdx.x == 0) s_seq = -1;
            if (lane == 31) s_sum[warp] = incl;
            __syncthreads();
            int64_t base = before;
            for (int w = 0; w < warp; ++w) base += s_sum[w];
            if (at >= base + incl - t && at < base + incl) {
                s_seq = b;
                s_at = base + incl - t;
            }
            for (int w = 0; w < W; ++w) before += s_sum[w];
            __syncthreads();
            seq = s_seq;
            seq_at = s_at;
        }
    } else {
        seq = blockIdx.x / v.kv_heads;
        const int t = seq_tiles(v, seq);
        if (t == 0) return;
        seq_at = 0;
        at = static_cast<int64_t>(blockIdx.x % v.kv_heads) * t;
        end = at + t;
    }
    const int64_t range_begin = at;

    while (at < end) {
        // The next unit of the stretch: tiles [t0, t1) of (seq, head).
        int tiles = seq_tiles(v, seq);
        while (at >= seq_at + static_cast<int64_t>(tiles) * v.kv_heads) {
            seq_at += static_cast<int64_t>(tiles) * v.kv_heads;
            ++seq;
            tiles = seq_tiles(v, seq);
        }
        const int head = static_cast<int>((at - seq_at) / tiles);
        const int64_t unit_at = seq_at + static_cast<int64_t>(head) * tiles;
        const int t0 = static_cast<int>(at - unit_at);
        const int t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - at)));
        int first, n, kv;
        kv_seq(v, seq, &first, &n, &kv);
        const int rows = n * args.group;  // <= 8 NT

        // q: each row to FP16 by a power of two (its largest channel to
        // 2^13..2^14: FP16 and BF16 rows keep all their bits down to 2^-23 of
        // it), in the order of the MMA's B fragments.
        for (int row = warp; row < S::kRows; row += W) {
            constexpr int PER = D / 32;
            float x[PER], big = 0.0f;
            const int i = row / args.group, g = row - i * args.group;
            const bool live = row < rows;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                x[j] = live ? widen(a.q[(first + i) * a.ldq + (head * args.group + g) * D + lane * PER + j], a.dtype) : 0.0f;
                big = fmaxf(big, fabsf(x[j]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            int e = big > 0.0f && big <= 3.402823466e38f ? ilogbf(big) - 13 : 0;
            e = max(e, -100);
            const float down = scalbnf(1.0f, -e);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int ch = lane * PER + j, word = (ch % (D / 4)) >> 3, jj = ch & 7;
                const float y = x[j] * down;
                const __half h = __float2half_rn((jj & 2) ? y * 0.0625f : y);
                sum += __half2float(h) * ((jj & 2) ? 16.0f : 1.0f);
                const int slot = ((row >> 3) * kWords + word) * 32 + (row & 7) * 4 + ch / (D / 4);
                // registers x, y: columns (0,1), (4,5); z, w: (2,3), (6,7)
                reinterpret_cast<__half*>(qf + slot)[((jj & 2) ? 4 : 0) + ((jj & 4) ? 2 : 0) + (jj & 1)] = h;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (lane == 0) {
                s_fac[row] = scalbnf(a.scale * 1.4426950408889634f, 24 + e);
                s_sumq[row] = sum * 5.9604644775390625e-8f;
                s_limit[row] = !live ? 0 : (a.causal ? kv - n + i + 1 : kv);
            }
        }
        __syncthreads();
        float fac[NT][2], sq[NT][2];
        int limit[NT][2], limit_min = 0x7FFFFFFF;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = t * 8 + c * 2 + j;
                fac[t][j] = s_fac[row];
                sq[t][j] = s_sumq[row];
                limit[t][j] = s_limit[row];
                if (row < rows) limit_min = min(limit_min, limit[t][j]);
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) limit_min = min(limit_min, __shfl_xor_sync(0xFFFFFFFFu, limit_min, o));
        uint4 qr[NT <= 2 ? NT : 1][kWords];
        if constexpr (NT <= 2) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < kWords; ++i) qr[t][i] = qf[(t * kWords + i) * 32 + lane];
        }

        float m[NT][2], l[NT][2], zs[NT][2], o[D / 16][NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[t][j] = -INFINITY;
                l[t][j] = zs[t][j] = 0.0f;
            }
#pragma unroll
            for (int ct = 0; ct < D / 16; ++ct)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[ct][t][j] = 0.0f;
        }

        // This warp's tiles: t0 + warp, + W, ...; lane l holds the page of the
        // l-th of the next 32 blocks.
        const int32_t* row_table = v.table + static_cast<int64_t>(seq) * v.ld_table;
        uint8_t* my_ring = ring + warp * S::kStages * S::kStage;
        const uint32_t my_ring_u32 = smem_u32(my_ring);
        const int count = t1 - t0 > warp ? (t1 - t0 - warp + W - 1) / W : 0;
        const uint8_t* blk = nullptr;  // lane's block address, or null
        auto fill = [&](int i) {       // addresses of blocks of tiles i .. i + 15
            const int tile = t0 + warp + (i + (lane >> 1)) * W;
            const int pos = tile * kTile + (lane & 1) * kKvBlock;
            blk = nullptr;
            if (i + (lane >> 1) < count && pos < kv) {
                blk = kv_block_at(v, row_table, head, pos);
                if (blk == nullptr) raise_error(v.err_flag, kErrBadPage);
            }
        };
        auto issue = [&](int i) {
            if (i < count) {
                if ((i & 15) == 0) fill(i);
                const uint32_t dst = my_ring_u32 + (i % S::kStages) * S::kStage;
#pragma unroll
                for (int h = 0; h < kTileBlocks; ++h) {
                    const uint64_t src = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(blk), (i & 15) * 2 + h);
                    const uint8_t* p = src != 0 ? reinterpret_cast<const uint8_t*>(src) : v.data;
#pragma unroll
                    for (int x = 0; x < (S::kBlock + 511) / 512; ++x) {
                        const int off = x * 512 + lane * 16;
                        if (off < S::kBlock) copy_async_16(dst + h * S::kBlock + off, p + off, src != 0);
                    }
                }
            }
            copy_async_commit();
        };
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) issue(i);

        for (int i = 0; i < count; ++i) {
            copy_async_wait<S::kStages - 2>();
            __syncwarp();
            issue(i + S::kStages - 1);
            const uint8_t* stage = my_ring + (i % S::kStages) * S::kStage;
            const int pos0 = (t0 + warp + i * W) * kTile;
            const bool inner = pos0 + kTile <= limit_min;  // every row sees every token

            float y[kTileBlocks][NT][4];
            float rs[kTileBlocks][2], zv[kTileBlocks][2];
#pragma unroll
            for (int h = 0; h < kTileBlocks; ++h) {
                const uint8_t* b = stage + h * S::kBlock;
                uint32_t k0[kWords], k1[kWords];
                const uint8_t* kp = b + r * (D / 2) + c * (D / 8);
                if constexpr (D == 128) {
                    const uint4 u0 = *reinterpret_cast<const uint4*>(kp), u1 = *reinterpret_cast<const uint4*>(kp + 4 * D);
                    k0[0] = u0.x; k0[1] = u0.y; k0[2] = u0.z; k0[3] = u0.w;
                    k1[0] = u1.x; k1[1] = u1.y; k1[2] = u1.z; k1[3] = u1.w;
                } else {
                    const uint2 u0 = *reinterpret_cast<const uint2*>(kp), u1 = *reinterpret_cast<const uint2*>(kp + 4 * D);
                    k0[0] = u0.x; k0[1] = u0.y;
                    k1[0] = u1.x; k1[1] = u1.y;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[h][t][j] = 0.0f;
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    const uint32_t s0 = k0[w] >> 8, s1 = k1[w] >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        uint4 q;
                        if constexpr (NT <= 2) q = qr[t][w];
                        else q = qf[(t * kWords + w) * 32 + lane];
                        mma_f16(y[h][t], k0[w] & kNib0, k1[w] & kNib0, s0 & kNib0, s1 & kNib0, q.x, q.y);
                        mma_f16(y[h][t], k0[w] & kNib1, k1[w] & kNib1, s0 & kNib1, s1 & kNib1, q.z, q.w);
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int token = half * 8 + r;
                    uint32_t ks = reinterpret_cast<const uint32_t*>(b + kv_k_scales(D))[token];
                    uint32_t vs = reinterpret_cast<const uint32_t*>(b + kv_v_scales(D))[token];
                    if (pos0 + h * kKvBlock + token >= kv) ks = vs = 0x3C00u;  // nobody's: scale 1, zero point 0
                    if ((vs & 0xFFFFu) == 0) vs |= 1u;  // never stored: holds zeros whatever its scale
                    const float sk = f16_bits_to_f32(static_cast<uint16_t>(ks)), sv = f16_bits_to_f32(static_cast<uint16_t>(vs));
                    const float zk = static_cast<float>(ks >> 16), lv = fast_log2(sv);
                    rs[h][half] = fast_rcp(sv);
                    zv[h][half] = static_cast<float>(vs >> 16);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float& e = y[h][t][half * 2 + j];
                            e = fmaf(fmaf(-zk, sq[t][j], e) * sk, fac[t][j], lv);
                            if (!inner && pos0 + h * kKvBlock + token >= limit[t][j]) e = -INFINITY;
                        }
                }
            }
            uint32_t pb[kTileBlocks][NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float base[2], fix[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float big = fmaxf(fmaxf(y[0][t][j], y[0][t][2 + j]), fmaxf(y[1][t][j], y[1][t][2 + j]));
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, off));
                    big = fmaxf(big, m[t][j]);
                    base[j] = big == -INFINITY ? 0.0f : big;  // no key seen yet
                    fix[j] = fast_exp2(m[t][j] - base[j]);
                    m[t][j] = big;
                }
                if (__any_sync(0xFFFFFFFFu, fix[0] != 1.0f || fix[1] != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        l[t][j] *= fix[j];
                        zs[t][j] *= fix[j];
#pragma unroll
                        for (int ct = 0; ct < D / 16; ++ct) {
                            o[ct][t][j] *= fix[j];
                            o[ct][t][2 + j] *= fix[j];
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < kTileBlocks; ++h)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float p[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float e = y[h][t][half * 2 + j];
                            p[j] = fast_exp2(e - base[j]);
                            // a masked token's scale may be NaN: it must not enter the sum
                            const float add = p[j] * rs[h][half];
                            l[t][j] += !inner && e == -INFINITY ? 0.0f : add;
                        }
                        const __half2 hp = __floats2half2_rn(p[0], p[1]);
                        const float2 back = __half22float2(hp);
                        zs[t][0] = fmaf(back.x, zv[h][half], zs[t][0]);
                        zs[t][1] = fmaf(back.y, zv[h][half], zs[t][1]);
                        pb[h][t][half] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&hp));
                    }
            }
#pragma unroll
            for (int h = 0; h < kTileBlocks; ++h) {
                const uint8_t* vp = stage + h * S::kBlock + kv_v_codes(D) + lane * (D / 8);
                // [token half][token of the pair][word]
                uint32_t vw[2][2][D / 64];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if constexpr (D == 128) {
                        const uint4 u = *reinterpret_cast<const uint4*>(vp + half * 4 * D);
                        vw[half][0][0] = u.x; vw[half][0][1] = u.y;
                        vw[half][1][0] = u.z; vw[half][1][1] = u.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(vp + half * 4 * D);
                        vw[half][0][0] = u.x;
                        vw[half][1][0] = u.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < D / 64; ++w)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {  // nibbles 0-3, then 4-7
                        const uint32_t x0 = __byte_perm(vw[0][0][w], vw[0][1][w], hi ? 0x7632 : 0x5410);
                        const uint32_t x1 = __byte_perm(vw[1][0][w], vw[1][1][w], hi ? 0x7632 : 0x5410);
                        const uint32_t u0 = x0 >> 8, u1 = x1 >> 8;
                        const int ct = w * 4 + hi * 2;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            mma_f16(o[ct][t], x0 & kNib0, x0 & kNib1, x1 & kNib0, x1 & kNib1, pb[h][t][0], pb[h][t][1]);
                            mma_f16(o[ct + 1][t], u0 & kNib0, u0 & kNib1, u1 & kNib0, u1 & kNib1, pb[h][t][0], pb[h][t][1]);
                        }
                    }
            }
            __syncwarp();
        }
        copy_async_wait<0>();

        // Join the warps: channel r D/8 + 2 ct in o[ct][.][0..1] (times 2^-24),
        // the next one in [2..3] (times 2^-20).
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], off);
                    zs[t][j] += __shfl_xor_sync(0xFFFFFFFFu, zs[t][j], off);
                }
        __syncthreads();  // every warp is done with the ring
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = t * 8 + c * 2 + j;
                if (r == 0) {
                    s_m[warp][row] = m[t][j];
                    s_l[warp][row] = l[t][j];
                }
                float* dst = merge + (warp * S::kRows + row) * D + r * (D / 8);
#pragma unroll
                for (int ct = 0; ct < D / 16; ++ct)
                    *reinterpret_cast<float2*>(dst + 2 * ct) =
                        make_float2(fmaf(o[ct][t][j], 16777216.0f, -zs[t][j]), fmaf(o[ct][t][2 + j], 1048576.0f, -zs[t][j]));
            }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == tiles;
        const int64_t slot = blockIdx.x * 2LL + (unit_at > range_begin ? 1 : 0);
        for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
            const int row = i / (D / 4), ch = (i - row * (D / 4)) * 4;
            float big = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) big = fmaxf(big, s_m[w][row]);
            const float base = big == -INFINITY ? 0.0f : big;
            float sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = fast_exp2(s_m[w][row] - base);
                const float4 x = *reinterpret_cast<const float4*>(merge + (w * S::kRows + row) * D + ch);
                sum = fmaf(s_l[w][row], f, sum);
                acc.x = fmaf(x.x, f, acc.x);
                acc.y = fmaf(x.y, f, acc.y);
                acc.z = fmaf(x.z, f, acc.z);
                acc.w = fmaf(x.w, f, acc.w);
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
                const int qi = row / args.group, g = row - qi * args.group;
                store_out4(a.out + (first + qi) * a.ldo + (head * args.group + g) * D + ch, a, acc, inv);
            } else {
                *reinterpret_cast<float4*>(args.part_o + (slot * S::kRows + row) * D + ch) = acc;
                if (ch == 0) args.part_ml[slot * S::kRows + row] = make_float2(big, sum);
            }
        }
        __syncthreads();
        at += t1 - t0;
    }
}

// Adds the parts of the units that span CTAs.  One CTA per (unit, row); its
// eight warps take the parts in turn.
template <int D, int NT, int W>
__global__ void __launch_bounds__(kThreads) attn_q4_join_kernel(const RowsArgs args) {
    constexpr int kRows = NT * 8, PER = D / 32;
    __shared__ int64_t s_sum[kThreads / 32];
    __shared__ float s_m[kThreads / 32], s_l[kThreads / 32];
    __shared__ float s_o[kThreads / 32][D];
    griddep_wait();
    griddep_launch_dependents();
    const AttnQ4Args& a = args.a;
    const KvView& v = a.v;
    const int seq = blockIdx.x / v.kv_heads, head = blockIdx.x - seq * v.kv_heads, row = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = seq_tiles(v, seq);
    int first, n, kv;
    if (tiles == 0 || !kv_seq(v, seq, &first, &n, &kv) || row >= n * args.group) return;
    int64_t all = 0, before = 0;
    for (int b = threadIdx.x; b < v.seqs; b += kThreads) {
        const int t = seq_tiles(v, b);
        all += t;
        if (b < seq) before += t;
    }
    const int64_t total = block_sum<kThreads / 32>(all, s_sum) * v.kv_heads;
    const int64_t unit_at = block_sum<kThreads / 32>(before, s_sum) * v.kv_heads + static_cast<int64_t>(head) * tiles;
    const int64_t per = tiles_a_cta(total, args.grid, W);
    const int64_t c0 = unit_at / per, c1 = (unit_at + tiles - 1) / per;
    if (c0 == c1) return;  // that CTA stored the output
    float m = -INFINITY, l = 0.0f, o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = 0.0f;
    for (int64_t p = c0 + warp; p <= c1; p += kThreads / 32) {
        const int64_t at = (p * 2 + (unit_at > p * per ? 1 : 0)) * kRows + row;
        const float2 ml = args.part_ml[at];
        float x[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = args.part_o[at * D + lane * PER + j];
        const float big = fmaxf(m, ml.x), base = big == -INFINITY ? 0.0f : big;
        const float f0 = fast_exp2(m - base), f1 = fast_exp2(ml.x - base);
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] = o[j] * f0 + x[j] * f1;
        m = big;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) s_o[warp][lane * PER + j] = o[j];
    __syncthreads();
    if (threadIdx.x < D) {
        float big = -INFINITY;
        for (int w = 0; w < kThreads / 32; ++w) big = fmaxf(big, s_m[w]);
        const float base = big == -INFINITY ? 0.0f : big;
        float sum = 0.0f, acc = 0.0f;
        for (int w = 0; w < kThreads / 32; ++w) {
            const float f = fast_exp2(s_m[w] - base);
            sum = fmaf(s_l[w], f, sum);
            acc = fmaf(s_o[w][threadIdx.x], f, acc);
        }
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
        const int qi = row / args.group, g = row - qi * args.group;
        a.out[(first + qi) * a.ldo + (head * args.group + g) * D + threadIdx.x] = narrow(acc * inv, a.dtype);
    }
}

}  // namespace
}  // namespace mrt

using namespace mrt;

static int check_attention(mrt_kv_q4 kv, const mrt_kv_batch* batch, int64_t heads, KvView* v) {
    const int rc = kv_view(kv, batch, v);
    if (rc != MRT_OK) return rc;
    if (heads <= 0 || heads > 65535 || heads % kv->kv_heads != 0)
        return set_error(MRT_ERR_SHAPE, "heads must be a positive multiple of kv_heads");
    if (batch->seqs * kv->kv_heads > (1LL << 31) - 1) return set_error(MRT_ERR_SHAPE, "too many sequences and heads");
    return MRT_OK;
}

namespace mrt {
namespace {

// How a call runs, by its sizes alone.
struct Plan {
    int few;     // 8-row tiles of the few-rows kernel, 0: more rows than it takes
    int split;   // its units may span CTAs
    int grid;
    size_t o_bytes, ml_bytes;
};

constexpr int kSplitWarps = 4, kWholeWarps = 16;

Plan make_plan(const KvView& v, int64_t heads, int sms) {
    Plan p{};
    const int64_t rows = heads / v.kv_heads * std::max(v.max_q_len, 1);
    if (rows > 32) return p;
    p.few = static_cast<int>((rows + 7) / 8);
    // Few short units: one CTA of sixteen warps each and no join.
    const int64_t units = static_cast<int64_t>(v.seqs) * v.kv_heads;
    p.split = !(v.max_kv_len <= kWholeWarps * 2 * kTile && units <= sms && p.few <= 2);
    p.grid = p.split ? sms * (p.few <= 2 ? 3 : 2) : static_cast<int>(units);
    if (p.split) {
        p.o_bytes = static_cast<size_t>(p.grid) * 2 * p.few * 8 * v.head_dim * 4;
        p.ml_bytes = static_cast<size_t>(p.grid) * 2 * p.few * 8 * 8;
    }
    return p;
}

template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) note_launches(1);
    return e;
}

template <int D, int NT, int W>
cudaError_t launch_few_w(const RowsArgs& r, int rows, cudaStream_t s) {
    constexpr int smem = RowsShape<D, NT, W>::kBytes;
    // Set at every call: it costs little and holds for whichever device is current.
    cudaError_t e = cudaFuncSetAttribute(attn_q4_few_kernel<D, NT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_pdl(attn_q4_few_kernel<D, NT, W>, dim3(r.grid), W * 32, smem, s, r);
    if (e == cudaSuccess && r.split)
        e = launch_pdl(attn_q4_join_kernel<D, NT, W>, dim3(r.a.v.seqs * r.a.v.kv_heads, rows), kThreads, 0, s, r);
    return e;
}

template <int D>
cudaError_t launch_few(const RowsArgs& r, int few, int rows, cudaStream_t s) {
    if (!r.split) return few == 1 ? launch_few_w<D, 1, kWholeWarps>(r, rows, s) : launch_few_w<D, 2, kWholeWarps>(r, rows, s);
    switch (few) {
        case 1: return launch_few_w<D, 1, kSplitWarps>(r, rows, s);
        case 2: return launch_few_w<D, 2, kSplitWarps>(r, rows, s);
        case 3: return launch_few_w<D, 3, kSplitWarps>(r, rows, s);
        default: return launch_few_w<D, 4, kSplitWarps>(r, rows, s);
    }
}

}  // namespace
}  // namespace mrt

extern "C" int mrt_kv_q4_attention_workspace(mrt_kv_q4 kv, const mrt_kv_batch* batch, int64_t heads, size_t* bytes) {
    clear_error();
    if (bytes == nullptr) return set_error(MRT_ERR_INVALID_ARG, "bytes is NULL");
    *bytes = 0;
    KvView v{};
    int rc = check_attention(kv, batch, heads, &v);
    if (rc != MRT_OK) return rc;
    int sms = 0;
    if ((rc = kv_bind(kv, &v, &sms)) != MRT_OK) return rc;
    const Plan p = make_plan(v, heads, sms);
    *bytes = p.o_bytes + p.ml_bytes;
    return MRT_OK;
}

extern "C" int mrt_kv_q4_attention(mrt_kv_q4 kv, const mrt_kv_batch* batch, int dtype, const void* q_dev, int64_t ldq,
                                   int64_t heads, void* out_dev, int64_t ldo, float scale, int causal, void* ws_dev,
                                   size_t ws_bytes, void* stream) {
    clear_error();
    AttnQ4Args a{};
    int rc = check_attention(kv, batch, heads, &a.v);
    if (rc != MRT_OK) return rc;
    if (dtype != MRT_FP16 && dtype != MRT_BF16) return set_error(MRT_ERR_DTYPE, "dtype must be FP16 or BF16");
    if (a.v.seqs == 0 || a.v.tokens == 0) return MRT_OK;
    if (q_dev == nullptr || out_dev == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL q or out");
    const int64_t D = kv->head_dim;
    if (ldq < heads * D || ldo < heads * D) return set_error(MRT_ERR_SHAPE, "a token's stride must cover its heads");
    int sms = 0;
    if ((rc = kv_bind(kv, &a.v, &sms)) != MRT_OK) return rc;
    const Plan plan = make_plan(a.v, heads, sms);
    if (plan.o_bytes > 0) {
        if (ws_dev == nullptr || ws_bytes < plan.o_bytes + plan.ml_bytes)
            return set_error(MRT_ERR_INVALID_ARG, "scratch is NULL or smaller than mrt_kv_q4_attention_workspace says");
        if ((reinterpret_cast<uintptr_t>(ws_dev) & 255) != 0)
            return set_error(MRT_ERR_INVALID_ARG, "scratch must be 256-byte aligned");
    }
    a.dtype = dtype;
    a.heads = static_cast<int>(heads);
    a.causal = causal != 0;
    a.scale = scale;
    a.q = static_cast<const uint16_t*>(q_dev);
    a.ldq = ldq;
    a.out = static_cast<uint16_t*>(out_dev);
    a.ldo = ldo;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (plan.few > 0) {
        RowsArgs r{};
        r.a = a;
        r.group = static_cast<int>(heads / kv->kv_heads);
        r.split = plan.split;
        r.grid = plan.grid;
        r.part_o = static_cast<float*>(ws_dev);
        r.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws_dev) + plan.o_bytes);
        const int rows = r.group * std::max(a.v.max_q_len, 1);
        e = D == 128 ? launch_few<128>(r, plan.few, rows, s) : launch_few<64>(r, plan.few, rows, s);
    } else {
        e = D == 128 ? launch_pdl(attn_q4_rows_kernel<4>, dim3(a.v.tokens), kThreads, 0, s, a)
                     : launch_pdl(attn_q4_rows_kernel<2>, dim3(a.v.tokens), kThreads, 0, s, a);
    }
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "4-bit attention launch");
}
