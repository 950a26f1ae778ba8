// kv_q4_attn.cu -- softmax attention of new tokens' queries over a paged cache
// held in 4 bits (kv_q4.h): the reference's attention op
// (src/core/cpu_backend.cpp:171-290) over such a cache.
#include <cuda_bf16.h>

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
    int dtype, causal;
    float scale;
    const uint16_t* q;
    int64_t ldq;
    uint16_t* out;
    int64_t ldo;
};

__device__ __forceinline__ float widen(uint16_t h, int dtype) {
    return dtype == MRT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

// Two neighbouring outputs, rounded to nearest.
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, int dtype) {
    if (dtype == MRT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store2(uint16_t* dst, uint32_t v) {
    if ((reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
        *reinterpret_cast<uint32_t*>(dst) = v;
    } else {
        dst[0] = static_cast<uint16_t>(v);
        dst[1] = static_cast<uint16_t>(v >> 16);
    }
}

// Own writes to shared memory come before later asynchronous ones.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------------ few rows

// Rows of one (sequence, kv head) are its new tokens times the query heads that
// share it; up to 32 of them ride as the MMA's N while keys are its M: scores
// S^T[16 keys x 8 rows] = K Q^T, transposed in registers into the second
// product's operand, O^T[16 channels x 8 rows] += V^T P^T.  K and V codes are
// the M operands straight from their bytes (q4.cuh).
//
// Softmax.  In powers of two, with a value's scale taken into the exponent:
// y = scale log2(e) q.k + log2 s_v, p' = 2^(y - m), m seven to fifteen below the
// running maximum of y (so it seldom has to be moved).  So p' is the probability
// times its value's scale, relative to the largest such product: FP16 operands keep
// eleven bits of whatever matters, down to 2^-21 of the largest, however unlike the
// scales are.
// The sum is of p' / s_v, and the zero points' part of the output, sum p' z (of
// the same rounded p'), is one more row of the second product.
//
// What bounds it: latency.  64 sequences of up to 8192 tokens (175 MB, 7 of 8 rows
// used) take 41 us where the bytes would take 27 at the copy's rate and the 406
// instructions a warp and tile, half of them the masks that make operands of codes,
// 17; beginning, joining and the CTAs' uneven ends are 9.  168 registers leave a
// scheduler three warps, each of which issues every six cycles (1.6 of them the
// instructions' own latency, 0.6 each pages, shared memory, the ALU): issue slots
// 46%, ALU 44.  One of 131071 tokens (70 MB) takes 20 us for 11 (of 22, with
// four CTAs a multiprocessor, 4 passed until the first tile was there, 13 with the
// tiles, 5 with the parts).
//
// More rows cost registers first: from nine on there are two CTAs a multiprocessor,
// and with 24 rows 16 bytes a thread are spilled, with 32 rows 624, of 16 rows of
// a lone unit's sixteen warps 280 (9 x 3 x 6000 tokens, 21 rows: 19 us for 3, four
// tiles a warp and eight warps a multiprocessor, issue slots 31%).
//
// Split.  The 32-token tiles of all (sequence, kv head) units, in order, are
// dealt to the CTAs in equal contiguous stretches, whatever the lengths: no
// CTA waits for a long sequence, and no plan from the host is needed (lengths
// are read here).  (Each unit counts unit_cost() tiles more than it has, for the
// time it takes to begin and to end one.)  A CTA's warps take a stretch's tiles in turn, each with its
// own ring of bulk copies, and join at the end of the unit, the next unit's
// first tiles already under way.  A unit that spans CTAs leaves its parts in
// scratch (two places a CTA: a unit that began earlier, and one that goes on)
// and attn_q4_join_kernel adds them in order.
constexpr int kTile = 32;
constexpr int kTileBlocks = kTile / kKvBlock;
constexpr float kLowest = -3.402823466e38f;  // m before any key: 2^(m - anything seen) is 0
// Exponents of a row's probabilities as FP16 operands: the largest's when m is set,
// and what is not passed before m is moved (2^16 is infinity there).
constexpr float kTop = 7.0f, kFar = 15.0f;

struct RowsArgs {
    AttnQ4Args a;
    int group;          // query heads of a kv head
    uint32_t group_magic;  // row * it >> 16 = row / group for row < 32
    int vec;            // q's rows can be read 16 bytes at a time
    int split;          // 0: every unit is one CTA's
    float* part_o;      // [2 * grid][8 NT][D]
    float2* part_ml;    // [2 * grid][8 NT]
    int grid;
    int warps;          // of a CTA
};

// Tiles of sequence b (0: none of its rows is computed), and the places that
// each of its units has among those that are dealt.
__device__ __forceinline__ int seq_tiles(const KvView& v, int b) {
    int first, n, kv;
    if (!kv_seq(v, b, &first, &n, &kv) || n == 0) return 0;
    return max(1, (kv + kTile - 1) / kTile);
}

// (64 x 8192 tokens 42.1 us, without 43.3; 9 x 3 x 6000 18.9 and 22.8.)
__host__ __device__ constexpr int unit_cost(int rows) { return rows <= 16 ? 8 : 16; }
__device__ __forceinline__ int unit_places(int tiles, int cost) { return tiles > 0 ? tiles + cost : 0; }

__device__ __forceinline__ int tiles_a_cta(int total, int grid, int warps) {
    const int per = (total + grid - 1) / grid;
    return per < warps ? warps : per;
}

template <int D, int NT, int W>
struct RowsShape {
    static constexpr bool kWhole = W > 8;  // a CTA has one unit, all of it
    static constexpr int kRows = NT * 8;
    static constexpr int kBlock = kKvBlock * (D + 8);
    static constexpr int kStage = kTileBlocks * kBlock;
    static constexpr int kStages = kWhole ? 2 : 3;
    static constexpr int kRing = W * kStages * kStage;
    // A warp's part of a unit: eight rows in the last slot of its ring, the others
    // behind the rings; of a lone unit, all in its ring.
    static constexpr int kOthers = kWhole ? 0 : W * (kRows - 8) * D * 4;
    static constexpr int kQ = NT * (D / 32) * 32 * 16;
    static constexpr int kScales = W * kTile * 16;  // of a tile's tokens, a warp's own
    static constexpr int kBytes = kRing + kOthers + kScales + kQ;
    static_assert((kWhole ? kRows : 8) * D * 4 <= (kWhole ? kStages : 1) * kStage, "parts fit");
    static __device__ __forceinline__ float* part(uint8_t* smem, int w, int row) {
        if (kWhole) return reinterpret_cast<float*>(smem + w * kStages * kStage) + row * D;
        if (row < 8) return reinterpret_cast<float*>(smem + (w * kStages + kStages - 1) * kStage) + row * D;
        return reinterpret_cast<float*>(smem + kRing) + (w * (kRows - 8) + row - 8) * D;
    }
};

// A part of a (sequence, kv head) as a CTA works on it.
struct RowsUnit {
    int seq, head, tiles, at;  // `at`: number of its first tile among all places
    int t0, t1;                // tiles of this CTA
    int first, n, kv;
};

// Wait for a warp's bulk copies, bounded; once one wait has given up (`late`)
// the warp's others hardly wait.
__device__ __forceinline__ void wait_tile(uint64_t* bar, uint32_t parity, int* flag, bool& late) {
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

// Eight 16-bit values at any alignment of two bytes.
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool vec) {
    if (vec) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = p[2 * j] | static_cast<uint32_t>(p[2 * j + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// True on one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

template <int D, int NT, int W>
__global__ void __launch_bounds__(W * 32, W > 8 ? 1 : (NT == 1 ? 3 : 2)) attn_q4_few_kernel(const RowsArgs args) {
    using S = RowsShape<D, NT, W>;
    constexpr int kWords = D / 32;               // words of a lane: K row part, and V channel stretch of two tokens
    // q is laid out eight channels a lane: lanes of a row, rows of a pass, passes.
    constexpr int kRowLanes = D / 8, kPass = W * 32 / kRowLanes, kPasses = (S::kRows + kPass - 1) / kPass;
    constexpr int kCost = unit_cost(S::kRows);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[W][S::kStages];
    __shared__ int s_sum[W];
    __shared__ int s_seq, s_at;
    __shared__ float s_fac[S::kRows];
    __shared__ int s_limit[S::kRows];
    __shared__ float s_m[W][S::kRows], s_l[W][S::kRows];
    uint4* qf = reinterpret_cast<uint4*>(smem + S::kBytes - S::kQ);
    const AttnQ4Args& a = args.a;
    const KvView& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    uint8_t* ring = smem + warp * S::kStages * S::kStage;
    float4* scales = reinterpret_cast<float4*>(smem + S::kRing + S::kOthers) + warp * kTile;

    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < S::kStages; ++i) mbar_init(&s_full[warp][i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();

    // This CTA's stretch of the tiles, and the unit it begins in.
    RowsUnit u;
    int at, end, seq_at;  // seq_at: tile number at which the unit's sequence begins
    if constexpr (!S::kWhole) {
        int incl, t, base, chunk;
        auto scan = [&](int b0) {  // places of W * 32 sequences from b0 on
            const int b = b0 + threadIdx.x;
            t = b < v.seqs ? unit_places(seq_tiles(v, b), kCost) * v.kv_heads : 0;
            incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += x;
            }
            if (lane == 31) s_sum[warp] = incl;
            __syncthreads();
            base = chunk = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w < warp) base += s_sum[w];
                chunk += s_sum[w];
            }
            __syncthreads();
        };
        int total = 0;
        for (int b0 = (v.seqs - 1) / (W * 32) * (W * 32); b0 >= 0; b0 -= W * 32) {  // the first ones last
            scan(b0);
            total += chunk;
        }
        if (blockIdx.x == 0)
            for (int b = threadIdx.x; b < v.seqs; b += W * 32) {
                int f, n, kv;
                if (!kv_seq(v, b, &f, &n, &kv)) raise_error(v.err_flag, kErrBadPage);
            }
        const int per = tiles_a_cta(total, args.grid, W);
        at = static_cast<int>(min(static_cast<int64_t>(total), static_cast<int64_t>(blockIdx.x) * per));
        end = min(total - at, per) + at;
        if (at >= end) return;
        if (threadIdx.x == 0) s_seq = -1;
        __syncthreads();
        for (int b0 = 0, before = 0;;) {
            const int lo = before + base + incl - t;
            if (at >= lo && at < lo + t) {
                s_seq = b0 + threadIdx.x;
                s_at = lo;
            }
            before += chunk;
            b0 += W * 32;
            if (at < before || b0 >= v.seqs) break;
            scan(b0);
        }
        __syncthreads();
        u.seq = s_seq;
        seq_at = s_at;
        if (u.seq < 0) return;  // (never, unless the lengths are written meanwhile)
        u.tiles = seq_tiles(v, u.seq);
    } else {
        u.seq = blockIdx.x / v.kv_heads;
        u.tiles = seq_tiles(v, u.seq);
        int f, n, kv;
        if (!kv_seq(v, u.seq, &f, &n, &kv) && threadIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
        if (u.tiles == 0) return;
        at = seq_at = 0;
        end = u.tiles;
    }
    const int range_begin = at;

    // The unit that place `at` lies in; false: none with a tile before `end`.
    auto find = [&]() {
        if (at >= end) return false;
        if constexpr (S::kWhole) {
            u.head = blockIdx.x % v.kv_heads;
            u.at = 0;
        } else {
            int places;
            while (at >= seq_at + (places = unit_places(u.tiles, kCost)) * v.kv_heads) {
                seq_at += places * v.kv_heads;
                if (++u.seq >= v.seqs) return false;
                u.tiles = seq_tiles(v, u.seq);
            }
            u.head = (at - seq_at) / places;
            u.at = seq_at + u.head * places + kCost;
        }
        u.t0 = max(at - u.at, 0);
        u.t1 = min(u.tiles, end - u.at);
        at = u.at + u.tiles;  // the next unit's first place
        kv_seq(v, u.seq, &u.first, &u.n, &u.kv);
        return u.t0 < u.t1;
    };

    // This warp's tiles of the unit: t0 + warp, + W, ....  Lane l sees to block l of
    // sixteen of them: its page's number (asked for sixteen tiles early), its own.
    int count, page_next, blk = -2;
    const int32_t* row_table;
    auto block_pos = [&](int i) { return (u.t0 + warp + (i + (lane >> 1)) * W) * kTile + (lane & 1) * kKvBlock; };
    auto ask = [&](int i) {  // -2: no such block
        const int pos = block_pos(i);
        page_next = -2;
        if (i + (lane >> 1) < count && pos < u.kv) {
            const int slot = kv_slot(v, pos);
            page_next = slot < v.ld_table ? row_table[slot] : -1;
        }
    };
    auto issue = [&](int i, int slot) {
        if (i >= count) return;
        if ((i & 15) == 0) {
            const int pos = block_pos(i);
            blk = -2;
            if (page_next != -2) {
                blk = kv_block_in(v, page_next, kv_slot(v, pos), u.head, pos);
                if (blk < 0) {
                    raise_error(v.err_flag, kErrBadPage);
                    blk = -2;
                }
            }
            ask(i + 16);
        }
        // A tile's two blocks are neighbours where a page holds both.
        const int n0 = __shfl_sync(0xFFFFFFFFu, blk, (i & 15) * 2), n1 = __shfl_sync(0xFFFFFFFFu, blk, (i & 15) * 2 + 1);
        if (elect_one()) {
            uint64_t* bar = &s_full[warp][slot];
            uint8_t* dst = ring + slot * S::kStage;
            mbar_arrive_expect_tx(bar, (n0 >= 0 ? S::kBlock : 0) + (n1 >= 0 ? S::kBlock : 0));
            const bool both = n1 == n0 + 1;
            if (n0 >= 0) bulk_load(dst, v.data + static_cast<int64_t>(n0) * S::kBlock, both ? S::kStage : S::kBlock, bar);
            if (n1 >= 0 && !both) bulk_load(dst + S::kBlock, v.data + static_cast<int64_t>(n1) * S::kBlock, S::kBlock, bar);
        }
        __syncwarp();
    };
    // q of the rows that this thread lays out.
    uint4 qw[kPasses];
    const int q_row = threadIdx.x / kRowLanes, q_lane = threadIdx.x & (kRowLanes - 1);
    auto start = [&]() {
        row_table = v.table + static_cast<int64_t>(u.seq) * v.ld_table;
        count = u.t1 - u.t0 > warp ? (u.t1 - u.t0 - warp + W - 1) / W : 0;
        ask(0);
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
            const int row = q_row + k * kPass, i = row * args.group_magic >> 16, g = row - i * args.group;
            qw[k] = make_uint4(0, 0, 0, 0);
            if (row < u.n * args.group)
                qw[k] = load8(a.q + (u.first + i) * a.ldq + (u.head * args.group + g) * D + q_lane * 8, args.vec);
        }
#pragma unroll
        for (int i = 0; i < (S::kWhole ? S::kStages : S::kStages - 1); ++i) issue(i, i);
    };
    if (!find()) return;
    start();
    uint32_t phases = 0;  // of the ring's slots
    bool late = false;

    for (;;) {
        // q: each row to FP16 by a power of two (its largest channel to
        // 2^13..2^14: FP16 and BF16 rows keep all their bits down to 2^-23 of
        // it), in the order of the MMA's B fragments.
        const int rows = u.n * args.group;  // <= 8 NT
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
            const int row = q_row + k * kPass;
            const uint32_t w[4] = {qw[k].x, qw[k].y, qw[k].z, qw[k].w};
            float x[8], big = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = widen(static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1))), a.dtype);
                big = fmaxf(big, fabsf(x[j]));
            }
#pragma unroll
            for (int o = kRowLanes / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            const int e = big < INFINITY ? max((__float_as_int(big) >> 23) - 140, -100) : 0;
            // Channels 0-3 of a word meet codes times 2^-24, 4-7 codes times 2^-20.
            const float down = pow2(-e), down16 = down * 0.0625f;
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float f = j < 2 ? down : down16;
                const __half2 h = __floats2half2_rn(x[2 * j] * f, x[2 * j + 1] * f);
                y[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (S::kRows % kPass != 0 && row >= S::kRows) break;
            qf[((row >> 3) * kWords + q_lane % kWords) * 32 + (row & 7) * 4 + q_lane / kWords] = make_uint4(y[0], y[1], y[2], y[3]);
            if (q_lane == 0) {
                s_fac[row] = a.scale * (1.4426950408889634f * 4096.0f) * pow2(12 + e);
                s_limit[row] = row >= rows ? 0 : (a.causal ? u.kv - u.n + static_cast<int>(row * args.group_magic >> 16) + 1 : u.kv);
            }
        }
        __syncthreads();
        if constexpr (!S::kWhole) issue(S::kStages - 1, S::kStages - 1);  // its slot held the last unit's part
        float fac[NT][2], sq[NT][2];  // sq: sum of q over the channels, as a code of one meets it
        int limit_min = 0x7FFFFFFF;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float ones[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const uint4 q = qf[(t * kWords + w) * 32 + lane];
                mma_f16(ones, 0x00010001u, 0x00010001u, 0x00010001u, 0x00010001u, q.x, q.y);
                mma_f16(ones, 0x00100010u, 0x00100010u, 0x00100010u, 0x00100010u, q.z, q.w);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = t * 8 + c * 2 + j;
                fac[t][j] = s_fac[row];
                sq[t][j] = ones[j];
                if (row < rows) limit_min = min(limit_min, s_limit[row]);
            }
        }
        limit_min = __reduce_min_sync(0xFFFFFFFFu, limit_min);
        uint4 qr[NT == 1 ? NT : 1][kWords];
        if constexpr (NT == 1) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) qr[0][i] = qf[i * 32 + lane];
        }

        float m[NT][2], l[NT][2], zs[NT][4], o[D / 16][NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[t][j] = kLowest;
                l[t][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                zs[t][j] = 0.0f;
#pragma unroll
                for (int ct = 0; ct < D / 16; ++ct) o[ct][t][j] = 0.0f;
            }
        }

#pragma unroll 1
        for (int i = 0, slot = 0; i < count; ++i) {
            wait_tile(&s_full[warp][slot], (phases >> slot) & 1, v.err_flag, late);
            phases ^= 1u << slot;
            const uint8_t* stage = ring + slot * S::kStage;
            const int pos0 = (u.t0 + warp + i * W) * kTile;

            {  // a token a lane: its scales as the sums need them
                const uint8_t* b = stage + (lane >> 4) * S::kBlock + (lane & 15) * 4;
                const uint32_t ks = *reinterpret_cast<const uint32_t*>(b + kv_k_scales(D));
                const float sk = f16_bits_to_f32(static_cast<uint16_t>(ks)), zk = f16_bits_to_f32(static_cast<uint16_t>(ks >> 16));
                // (never stored: scale 0; it holds zeros whatever its scale)
                const float sv = max_nan(f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(b + kv_v_scales(D))), 5.9604644775390625e-8f);
                // A row that sees a NaN scale has a NaN p; the others' sums must not.
                scales[lane] = make_float4(sk, -zk, fast_log2(sv), fminf(fast_rcp(sv), 16777216.0f));
                __syncwarp();
            }
            float y[kTileBlocks][NT][4];
            float rs[kTileBlocks][2];
            uint32_t z[kTileBlocks][2];  // zero points of V: tokens 2c, 2c + 1 and 2c + 8, 2c + 9
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
                for (int w = 0; w < kWords; ++w) {
                    const uint32_t s0 = k0[w] >> 8, s1 = k1[w] >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        uint4 q;
                        if constexpr (NT == 1) q = qr[t][w];
                        else q = qf[(t * kWords + w) * 32 + lane];
                        if (w == 0) mma_f16_first(y[h][t], k0[w] & kNib0, k1[w] & kNib0, s0 & kNib0, s1 & kNib0, q.x, q.y);
                        else mma_f16(y[h][t], k0[w] & kNib0, k1[w] & kNib0, s0 & kNib0, s1 & kNib0, q.x, q.y);
                        mma_f16(y[h][t], k0[w] & kNib1, k1[w] & kNib1, s0 & kNib1, s1 & kNib1, q.z, q.w);
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float4 sc = scales[h * kKvBlock + half * 8 + r];
                    rs[h][half] = sc.w;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float& e = y[h][t][half * 2 + j];
                            e = fmaf(fmaf(sc.y, sq[t][j], e) * sc.x, fac[t][j], sc.z);
                        }
                    const uint2 zw = *reinterpret_cast<const uint2*>(b + kv_v_scales(D) + half * 32 + c * 8);
                    z[h][half] = __byte_perm(zw.x, zw.y, 0x7632);
                }
            }
            if (pos0 + kTile > limit_min) {  // some row does not see every token
#pragma unroll
                for (int h = 0; h < kTileBlocks; ++h)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int pos = pos0 + h * kKvBlock + half * 8;
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                if (pos + r >= s_limit[t * 8 + c * 2 + j]) y[h][t][half * 2 + j] = -INFINITY;
                        // (of tokens and pages that are nobody's: bytes of any kind)
                        const __half2 zz = __hmin2(__hmax2(*reinterpret_cast<const __half2*>(&z[h][half]), __float2half2_rn(0.0f)),
                                                   __float2half2_rn(15.0f));
                        z[h][half] = *reinterpret_cast<const uint32_t*>(&zz);
                    }
            }
            bool far = false;
            float big[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    big[t][j] = fmaxf(fmaxf(y[0][t][j], y[0][t][2 + j]), fmaxf(y[1][t][j], y[1][t][2 + j]));
                    far |= big[t][j] > m[t][j] + kFar;
                }
            if (__any_sync(0xFFFFFFFFu, far)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = fmaxf(big[t][j] - kTop, m[t][j]);
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, off));
                        const float fix = fast_exp2(m[t][j] - x);
                        m[t][j] = x;
                        l[t][j] *= fix;
                        zs[t][j] *= fix;
#pragma unroll
                        for (int ct = 0; ct < D / 16; ++ct) {
                            o[ct][t][j] *= fix;
                            o[ct][t][2 + j] *= fix;
                        }
                    }
            }
#pragma unroll
            for (int h = 0; h < kTileBlocks; ++h) {
                uint32_t pb[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float p[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            p[j] = fast_exp2(y[h][t][half * 2 + j] - m[t][j]);
                            l[t][j] = fmaf(p[j], rs[h][half], l[t][j]);
                        }
                        const __half2 hp = __floats2half2_rn(p[0], p[1]);
                        pb[t][half] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&hp));
                    }
                    mma_f16(zs[t], z[h][0], 0u, z[h][1], 0u, pb[t][0], pb[t][1]);
                }
                const uint8_t* vp = stage + h * S::kBlock + kv_v_codes(D) + lane * (D / 8);
                uint32_t v0[kWords], v1[kWords];  // tokens 0-7, 8-15
                if constexpr (D == 128) {
                    const uint4 u0 = *reinterpret_cast<const uint4*>(vp), u1 = *reinterpret_cast<const uint4*>(vp + 4 * D);
                    v0[0] = u0.x; v0[1] = u0.y; v0[2] = u0.z; v0[3] = u0.w;
                    v1[0] = u1.x; v1[1] = u1.y; v1[2] = u1.z; v1[3] = u1.w;
                } else {
                    const uint2 u0 = *reinterpret_cast<const uint2*>(vp), u1 = *reinterpret_cast<const uint2*>(vp + 4 * D);
                    v0[0] = u0.x; v0[1] = u0.y;
                    v1[0] = u1.x; v1[1] = u1.y;
                }
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    const uint32_t s0 = v0[w] >> 8, s1 = v1[w] >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_f16(o[2 * w][t], v0[w] & kNib0, v0[w] & kNib1, v1[w] & kNib0, v1[w] & kNib1, pb[t][0], pb[t][1]);
                        mma_f16(o[2 * w + 1][t], s0 & kNib0, s0 & kNib1, s1 & kNib0, s1 & kNib1, pb[t][0], pb[t][1]);
                    }
                }
            }
            __syncwarp();  // the slot is read
            issue(i + S::kStages, slot);
            slot = slot == S::kStages - 1 ? 0 : slot + 1;
        }

        // Join the warps, with the next unit's copies under way.
        const RowsUnit done = u;
        const bool more = !S::kWhole && find();
        if (more) start();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], off);
                const int row = t * 8 + c * 2 + j;
                if (r == 0) {
                    s_m[warp][row] = m[t][j];
                    s_l[warp][row] = l[t][j];
                }
                // channel r D/8 + 2 ct in o[ct][.][0..1] (times 2^-24), the next one in [2..3] (times 2^-20)
                float* dst = S::part(smem, warp, row) + r * (D / 8);
#pragma unroll
                for (int ct = 0; ct < D / 16; ++ct)
                    *reinterpret_cast<float2*>(dst + 2 * ct) =
                        make_float2(fmaf(o[ct][t][j], 16777216.0f, -zs[t][j]), fmaf(o[ct][t][2 + j], 1048576.0f, -zs[t][j]));
            }
        fence_async_smem();  // the slot's next copy comes after these
        __syncthreads();
        const bool whole = done.t0 == 0 && done.t1 == done.tiles;
        const int64_t place = blockIdx.x * 2LL + (done.at > range_begin ? 1 : 0);
        for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
            const int row = i / (D / 4), ch = (i - row * (D / 4)) * 4;
            float big = kLowest;
#pragma unroll
            for (int w = 0; w < W; ++w) big = fmaxf(big, s_m[w][row]);
            float sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = fast_exp2(s_m[w][row] - big);
                const float4 x = *reinterpret_cast<const float4*>(S::part(smem, w, row) + ch);
                sum = fmaf(s_l[w][row], f, sum);
                acc.x = fmaf(x.x, f, acc.x);
                acc.y = fmaf(x.y, f, acc.y);
                acc.z = fmaf(x.z, f, acc.z);
                acc.w = fmaf(x.w, f, acc.w);
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : fast_rcp(sum);
                const int qi = row * args.group_magic >> 16, g = row - qi * args.group;
                uint16_t* dst = a.out + (done.first + qi) * a.ldo + (done.head * args.group + g) * D + ch;
                store2(dst, narrow2(acc.x * inv, acc.y * inv, a.dtype));
                store2(dst + 2, narrow2(acc.z * inv, acc.w * inv, a.dtype));
            } else {
                *reinterpret_cast<float4*>(args.part_o + (place * S::kRows + row) * D + ch) = acc;
                if (ch == 0) args.part_ml[place * S::kRows + row] = make_float2(big, sum);
            }
        }
        if (!more) break;
    }
}

// Adds the parts of the units that span CTAs, in order.  One CTA per (unit,
// row), a warp (half a warp) a part, kJoinParts of each asked for at a time.
// Of THREADS threads: many parts of few rows, or few of many.
template <int D, int THREADS>
__global__ void __launch_bounds__(THREADS) attn_q4_join_kernel(const RowsArgs args, int kRows) {
    const int kCost = unit_cost(kRows);
    constexpr int kJoinParts = THREADS > 64 ? 10 : 4;
    constexpr int LANES = D / 4;  // of a part: four channels each
    static_assert(kJoinParts <= LANES, "a thread a part");
    constexpr int threads = THREADS, warps = THREADS / 32;
    __shared__ int s_a[warps], s_b[warps];
    __shared__ float s_w[threads];
    __shared__ float s_big[warps], s_sum[warps];
    __shared__ float4 s_o[threads];
    const AttnQ4Args& a = args.a;
    const KvView& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = blockIdx.x / v.kv_heads, head = blockIdx.x - seq * v.kv_heads, row = blockIdx.y;
    // The call's lengths are older than the kernel whose parts this one waits for
    // (that kernel lets this one start once it has waited for all before it).
    int all = 0, before = 0;
    for (int b = threadIdx.x; b < v.seqs; b += threads) {
        const int t = unit_places(seq_tiles(v, b), kCost);
        all += t;
        if (b < seq) before += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    }
    if (lane == 0) {
        s_a[warp] = all;
        s_b[warp] = before;
    }
    __syncthreads();
    all = before = 0;
#pragma unroll 1
    for (int w = 0; w < warps; ++w) {
        all += s_a[w];
        before += s_b[w];
    }
    const int tiles = seq_tiles(v, seq);
    int first, n, kv;
    const bool live = kv_seq(v, seq, &first, &n, &kv) && tiles != 0 && row < n * args.group;
    const int unit_at = before * v.kv_heads + head * unit_places(tiles, kCost) + kCost;
    const int per = tiles_a_cta(all * v.kv_heads, args.grid, args.warps);
    const int c0 = unit_at / per, c1 = (unit_at + tiles - 1) / per;
    griddep_wait();
    griddep_launch_dependents();
    if (!live || c0 == c1) return;  // (the one CTA stored the output)
    auto place = [&](int p) { return (p * 2LL + (unit_at > p * per ? 1 : 0)) * kRows + row; };
    float m = kLowest, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int ch = (threadIdx.x % LANES) * 4, mine = threadIdx.x / LANES, step = threads / LANES;
    for (int p0 = c0; p0 <= c1; p0 += kJoinParts * step) {
        const int parts = min(kJoinParts * step, c1 - p0 + 1);
        float4 x[kJoinParts];
#pragma unroll
        for (int k = 0; k < kJoinParts; ++k)
            x[k] = mine + k * step < parts ? *reinterpret_cast<const float4*>(args.part_o + place(p0 + mine + k * step) * D + ch)
                                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float2 ml = make_float2(kLowest, 0.0f);
        if (threadIdx.x < parts) ml = args.part_ml[place(p0 + threadIdx.x)];
        float big = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
        if (lane == 0) s_big[warp] = big;
        __syncthreads();
        big = m;
#pragma unroll
        for (int w = 0; w < warps; ++w) big = fmaxf(big, s_big[w]);
        const float f = fast_exp2(ml.x - big), fix = fast_exp2(m - big);
        s_w[threadIdx.x] = f;
        l = fmaf(l, fix, threadIdx.x < parts ? ml.y * f : 0.0f);
        acc = make_float4(acc.x * fix, acc.y * fix, acc.z * fix, acc.w * fix);
        m = big;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kJoinParts; ++k) {
            if (mine + k * step >= parts) break;
            const float g = s_w[mine + k * step];
            acc.x = fmaf(x[k].x, g, acc.x);
            acc.y = fmaf(x[k].y, g, acc.y);
            acc.z = fmaf(x[k].z, g, acc.z);
            acc.w = fmaf(x[k].w, g, acc.w);
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    if (lane == 0) s_sum[warp] = l;
    s_o[threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.x < LANES) {
        float sum = 0.0f;
        for (int w = 0; w < warps; ++w) sum += s_sum[w];
        for (int k = 1; k < step; ++k) {
            const float4 x = s_o[k * LANES + threadIdx.x];
            acc = make_float4(acc.x + x.x, acc.y + x.y, acc.z + x.z, acc.w + x.w);
        }
        const float inv = sum == 0.0f ? 0.0f : fast_rcp(sum);
        const int qi = row * args.group_magic >> 16, g = row - qi * args.group;
        uint16_t* dst = a.out + (first + qi) * a.ldo + (head * args.group + g) * D + ch;
        store2(dst, narrow2(acc.x * inv, acc.y * inv, a.dtype));
        store2(dst + 2, narrow2(acc.z * inv, acc.w * inv, a.dtype));
    }
}

// ------------------------------------------------------------------ many rows

// TMEM accesses in MMA-fragment order, 16 lanes (rows) at a time: lane (r, c)
// of the warp gets, of every eight 32-bit columns, columns 2c and 2c + 1 of
// rows r and r + 8.  (A thread then meets a quarter of the columns instead of
// all of them, so what belongs to a column is loaded a quarter as often.)
__device__ __forceinline__ void tmem_ld_frag64(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
        "}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld_frag32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15"
        "}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_st_frag32(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16"
        "};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// 32 columns of 32 bits, one register a column and row: lane (r, c) holds, of
// every four columns, column c of rows r and r + 8.
__device__ __forceinline__ void tmem_st_pairs32(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16"
        "};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The products take descriptors by their low words (address, leading offset);
// the high word is the same for every panel here, so a step along K is one
// 32-bit addition and nothing is worth keeping in registers.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;  // stride, version, swizzle (smem_desc_k128)

__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr) { return (smem_addr & 0x3FFFFu) >> 4 | 1u << 16; }

// D[tmem] (+)= A[smem] * B[smem]^T.
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}

// mbar_try_wait that may sleep up to 0.1 ms before it answers: a warp that waits
// leaves its scheduler to the others instead of asking again and again.
__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
        : "memory");
    return ok != 0;
}

// Wait for a phase, bounded: after kWaitLimitNs, or once another thread of the
// CTA has given up, the wait ends.  The unit under way is then run through
// without waiting (every access stays in bounds whatever was computed), and each
// role leaves where it would begin the next one: a unit that was not waited for
// may be anything.  Unlike mbar_wait it does not look at the device's error flag:
// a bad page of one sequence must not end another's waits.
__device__ __forceinline__ void wait_phase(uint64_t* bar, uint32_t parity, volatile int* gave_up, int* flag, int code) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t it = 1; !try_wait_long(bar, parity); ++it) {
        if ((it & 63u) != 0) continue;  // the clock is far away: not read in a wait that ends soon
        if (*gave_up) return;
        if (t0 == 0) t0 = globaltimer_ns();
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            *gave_up = 1;
            raise_error(flag, code);
            return;
        }
    }
}

__device__ __forceinline__ bool gave_up(const volatile int* flag) { return *flag != 0; }
// The same answer for all lanes.
__device__ __forceinline__ bool warp_gave_up(const volatile int* flag) { return __any_sync(0xFFFFFFFFu, *flag != 0); }

// Many rows (prompts, chunks of prompts): tcgen05 flash attention.  A CTA
// takes 256 rows of a (sequence, kv head) -- new tokens times the query heads
// that share it -- as two tiles of 128, and keys 64 at a time:
//
//   warps 0-7, 8-15  softmax of tile 0, 1, sixteen rows a warp: S from TMEM,
//                    P back into its place
//   warps 16-23      codes from the pages into the tensor cores' swizzled
//                    layout, K as the integers c - z (exact), V as values
//                    s (c - z) rounded to FP16 (finite: append sees to it); four
//                    warps the even key tiles, four the odd ones
//   warps 24, 25     S_i = Q_i K^T
//   warps 26, 27     O_i += P_i V (P from TMEM)
//   warps 28-30      Q into its panels
//   warp 31          the walk over the CTA's units, published a few ahead
//
// Roles meet only at mbarriers, and units follow one another without a stop.
// TMEM: two S (P in its first half) for each row tile, O_0, O_1: the scores of
// the next keys are there while the softmax works on these, so neither waits
// for the other's whole chain (with 128 keys and one S a tile, softmax 4000 and
// products 2600 cycles alternated).
//
// A key's scale multiplies its column of S, so scores are as exact as FP32; a
// value's goes into the operand, at the price of one more rounding (2^-11 of
// each value, independent from token to token like that of P, and averaged
// with it), because every number that a column needs in the softmax is a
// shared-memory read for every pair of rows; with the value's scale in the
// exponent, as in the few-rows kernel, a column needed three.  (With V as c - z
// times a power of two, exact, and the rest of its scale multiplied into the
// probability, a call's error against 64 bits is 2.9e-4 of its norm instead of
// 3.5e-4, 2.1e-4 being the FP16 output's, but the 2048 tokens below take 523 to 531
// us instead of 471.)  Scores come out
// of one fused operation relative to m, which lies 2^7 below the largest
// probability when it is set and moves only when a row exceeds it by 2^15 (P then
// still fits FP16): rows' maxima are joined, scores moved and O in TMEM rescaled in
// that case alone.  (From the upper end of FP16's range down, P keeps its bits to
// 2^-21 of the row's largest: where one key without a value takes most of a row, as
// a first token often does, the output is made of probabilities that small.  With m
// at the largest, to 2^-14, 300 tokens behind 5700 whose first key was e^14 ahead, with
// 2^-12 of the others' value, were off by 2.0e-3 of their norm, now by 2.9e-4.)
// All loops are short: with the softmax unrolled over its rows the kernel had
// 148 KB of code and every step of every role waited for its instructions.
//
// What bounds it: 2048 tokens behind 14000 (28 heads on 4 of 128 channels) take
// 471 us in a short run, 441 GFLOP at 56% of the rate of a large bf16 product, and
// 520 to 530 at the clocks of a long one (50%).  Issue slots
// (62% used) and shared memory (two thirds: Q and K for S, V for O, the codes'
// stores, the columns' scales) come first, the exponentials' unit has 38%, the
// tensor cores' 38.  Two prompts of 1800 and 966 tokens behind 100 and 54 (14
// heads on 2 of 64) take 40 us, 9 of them until the first scores are there and 4
// for the parts.
//
// Units' key tiles are dealt to the CTAs in equal contiguous stretches, as in
// the few-rows kernel (each unit at kManyCost tiles more than it has: without,
// the two prompts took 70 us), parts of units that span CTAs joined from
// scratch.
constexpr int kManyRows = 256, kManyKeys = 64;
constexpr int kSoftmaxWarps = 16, kCodesWarps = 8, kManyWarps = kSoftmaxWarps + kCodesWarps + 8;
constexpr int kManyThreads = kManyWarps * 32;
constexpr int kLoaders = 96;  // threads that bring Q
constexpr int kManyCost = 4;  // of a unit's begin and end, in key tiles

struct ManyPart {  // a unit that begins in a CTA's stretch and goes on
    int seq, head, row0;
    int place;     // 0 or 1: which of the CTA's two places holds its part
    int last_cta;  // < 0: none
};

struct ManyArgs {
    AttnQ4Args a;
    int group, grid;
    uint32_t group_magic;  // high word of x * it = x / group for x < 2^16 (group 1: 0)
    float* part_o;     // [2 * grid][256][D]
    float2* part_ml;   // [2 * grid][256]
    ManyPart* parts;   // [grid]
};

// Key tiles of a sequence's row tiles.  Row tile x < count - 1 ends with token
// (256 x + 255) / group, and causal rows see keys up to themselves.  (The host
// has checked that rows and tile numbers fit in 31 bits.)
struct ManySeq {
    int first, n, kv, group, causal;
    int count;  // row tiles, 0: nothing to do
    __device__ __forceinline__ int past() const { return max(kv - n, 0); }
    __device__ __forceinline__ int tiles(int x) const {
        if (!causal) return max(1, (kv + kManyKeys - 1) / kManyKeys);
        const int last = min(n - 1, (kManyRows * x + kManyRows - 1) / group);
        return (past() + last) / kManyKeys + 1;
    }
};

// sum_{i < n} floor((a i + b) / m), the lattice points under a line, by the known
// Euclid-like method (reciprocity of sums of floors; Graham, Knuth and Patashnik,
// Concrete Mathematics, 3.5): the axes are exchanged until the line is flat.  a n + b fits in 32 bits (checked
// on the host); so does the sum, whose parts may wrap.
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint32_t sum = 0;
#pragma unroll 1
    while (n > 0) {
        const uint32_t qa = a / m, qb = b / m;
        sum += static_cast<uint32_t>(static_cast<uint64_t>(n) * (n - 1) / 2) * qa + n * qb;
        a -= qa * m;
        b -= qb * m;
        const uint32_t top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// Places of row tiles 0 .. x - 1: their key tiles, and what the units cost.
__device__ __forceinline__ int many_before(const ManySeq& s, int x) {
    if (x == 0) return 0;
    if (!s.causal) return x * (s.tiles(0) + kManyCost);
    const int y = min(x, s.count - 1);
    int t = y + x * kManyCost + static_cast<int>(floor_sum(y, kManyKeys * s.group, kManyRows, kManyRows - 1 + s.past() * s.group));
    if (x == s.count) t += s.tiles(s.count - 1);
    return t;
}

__device__ __forceinline__ bool many_seq(const ManyArgs& g, int b, ManySeq* s) {
    const bool ok = kv_seq(g.a.v, b, &s->first, &s->n, &s->kv);
    s->group = g.group;
    s->causal = g.a.causal;
    s->count = ok ? (s->n * g.group + kManyRows - 1) / kManyRows : 0;
    return ok;
}

template <int D>
struct ManyShape {
    static constexpr int kPanel = 128 * 128;                // Q: 128 rows of 64 16-bit columns
    static constexpr int kQ = 2 * (D / 64) * kPanel;
    static constexpr int kKPanel = kManyKeys * 128;         // K: 64 rows of 64 channels
    static constexpr int kK = (D / 64) * kKPanel;           // a stage
    static constexpr int kV = D * 128;                      // V^T: D rows of 64 keys
    static constexpr int kColsRow = 80, kCols = 4 * kColsRow;  // [c][k]: scales of columns 8k + 2c, + 1; rows in different banks
    static constexpr int kStages = 4;
    static constexpr int kBytes = 1024 + kQ + kStages * (kK + kV + kCols);
};

// 16 bytes (eight 16-bit columns) of row `row` in a swizzled panel of 128-byte rows.
__device__ __forceinline__ uint32_t panel_at(uint32_t base, int row, int chunk) {
    return base + row * 128 + ((chunk ^ (row & 7)) << 4);
}

__device__ __forceinline__ void st_shared_16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// (A NaN is passed over.)
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

constexpr uint32_t kSixteenth = 0x2C002C00u;  // FP16 1/16 twice

// Codes at bits 0-3 / 4-7 of each half less the zero points, as FP16: z1024 =
// the halves 1024 + z, z64 = -(64 + z).  1024 + c and (1024 + 16 c) / 16 are exact.
__device__ __forceinline__ uint32_t nib0_f16(uint32_t w, uint32_t z1024) { return h2_sub((w & kNib0) | 0x64006400u, z1024); }
__device__ __forceinline__ uint32_t nib1_f16(uint32_t w, uint32_t z64) {
    return h2_fma((w & kNib1) | 0x64006400u, kSixteenth, z64);
}

// A unit as one CTA works on it.
struct ManyUnit {
    int seq, head, first, n, kv;  // sequence and kv head, the sequence's first row, new and held tokens
    int row0, rows;               // of the unit's rows
    int tok0, head0;              // row0's token and query head of the group
    int t0, count;                // its key tiles that are this CTA's; count = 0: no more units
    int whole, place;             // all of them are; where its part goes else
    __device__ __forceinline__ int row_tiles() const { return rows > 128 ? 2 : 1; }
};
constexpr int kUnits = 4;  // published ahead

// A CTA's stretch of the key tiles, unit by unit.
struct ManyWalk {
    int at, end, begin;  // places: next, end and begin of the stretch
    int unit_at, tiles;  // where the unit begins, its key tiles (kManyCost places on)
    ManySeq sq;
    int seq, head, x;    // the unit: sequence, kv head, row tile

    __device__ __forceinline__ bool next(const ManyArgs& g, ManyUnit* u) {
        u->count = 0;
        if (at >= end) return false;
        tiles = sq.tiles(x);
        if (at >= unit_at + tiles + kManyCost) {
            unit_at += tiles + kManyCost;
            if (++x == sq.count) {
                x = 0;
                if (++head == g.a.v.kv_heads) {
                    head = 0;
                    do {
                        if (++seq >= g.a.v.seqs) return false;
                        many_seq(g, seq, &sq);
                    } while (sq.count == 0);
                }
            }
            tiles = sq.tiles(x);
        }
        u->seq = seq;
        u->head = head;
        u->first = sq.first;
        u->n = sq.n;
        u->kv = sq.kv;
        u->row0 = x * kManyRows;
        u->rows = min(kManyRows, sq.n * g.group - u->row0);
        const int first_at = unit_at + kManyCost;
        u->t0 = max(at - first_at, 0);
        u->count = max(min(tiles, end - first_at) - u->t0, 0);
        u->whole = u->count == tiles;
        u->place = first_at > begin ? 1 : 0;
        const int x = u->row0 / g.group;
        u->tok0 = x;
        u->head0 = u->row0 - x * g.group;
        at = first_at + tiles;
        return u->count > 0;
    }
};

template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Registers a thread: at launch, and as the roles share them out (in groups of
// four warps: four of softmax, two of codes, products, Q).  (4 to 12 bytes a thread
// are spilled.)
constexpr int kManyRegs = 64, kSoftmaxRegs = 72, kCodesRegs = 72, kOtherRegs = 40;
static_assert(kManyWarps == 32, "a lane a warp in the scan");
static_assert(4 * kSoftmaxRegs + 2 * kCodesRegs + 2 * kOtherRegs == 8 * kManyRegs, "the roles share what the launch has");

template <int D, bool BF16>
__global__ void __launch_bounds__(kManyThreads, 1) attn_q4_many_kernel(const ManyArgs args) {
    using S = ManyShape<D>;
    constexpr int kPanels = D / 64, dtype = BF16 ? MRT_BF16 : MRT_FP16;
    extern __shared__ uint8_t smem_raw[];
    // s_full, s_empty: a stage of K, V and column scales.  Per row tile and S:
    // s_scores: S; s_probs: P; s_done: the product that used it.  s_free: O has
    // been read.  s_q, s_q_free: Q.
    __shared__ uint64_t s_full[S::kStages], s_empty[S::kStages], s_scores[2][2], s_probs[2][2], s_done[2][2], s_free[2], s_q, s_q_free;
    __shared__ uint64_t s_unit_full[kUnits], s_unit_empty[kUnits], s_drain[4];
    __shared__ ManyUnit s_unit[kUnits];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up, s_seq, s_at, s_tiles, s_sum[kManyWarps];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t q_u32 = smem_u32(smem), k_u32 = q_u32 + S::kQ, v_u32 = k_u32 + S::kStages * S::kK;
    uint8_t* cols = smem + S::kQ + S::kStages * (S::kK + S::kV);
    const AttnQ4Args& a = args.a;
    const KvView& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(&s_full[i], 128);
            mbar_init(&s_empty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&s_scores[i][b], 1);
                mbar_init(&s_probs[i][b], 8);
                mbar_init(&s_done[i][b], 1);
            }
            mbar_init(&s_free[i], 8);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&s_drain[i], 1);
        for (int i = 0; i < kUnits; ++i) {
            mbar_init(&s_unit_full[i], 1);
            mbar_init(&s_unit_empty[i], kManyWarps - 1);  // each warp but the walker's
        }
        mbar_init(&s_q, kLoaders);
        mbar_init(&s_q_free, 2);
        s_gave_up = 0;
        fence_barrier_init();
    }
    if (warp == kSoftmaxWarps + kCodesWarps) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    griddep_launch_dependents();  // after the allocation: whoever follows may want TMEM of its own
    griddep_wait();

    // This CTA's stretch, and the unit it begins in.
    int t, lo, chunk;  // places of the thread's sequence; of those before it and of all in a scan
    auto scan = [&](int b0) {
        const int b = b0 + threadIdx.x;
        t = 0;
        if (b < v.seqs) {
            ManySeq q;
            if (!many_seq(args, b, &q) && blockIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
            t = many_before(q, q.count) * v.kv_heads;
        }
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= o) incl += up;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int warps = s_sum[lane];  // (as many warps as lanes)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, warps, o);
            if (lane >= o) warps += up;
        }
        chunk = __shfl_sync(0xFFFFFFFFu, warps, 31);
        const int before = __shfl_sync(0xFFFFFFFFu, warps, (warp + 31) & 31);
        lo = (warp > 0 ? before : 0) + incl - t;
    };
    int total = 0;
#pragma unroll 1
    for (int b0 = (v.seqs - 1) / kManyThreads * kManyThreads; b0 >= 0; b0 -= kManyThreads) {  // the first ones last
        scan(b0);
        total += chunk;
    }
    const int per = (total + args.grid - 1) / args.grid;
    ManyWalk walk;
    walk.at = walk.begin = static_cast<int>(min(static_cast<int64_t>(total), static_cast<int64_t>(blockIdx.x) * per));
    walk.end = walk.at + min(total - walk.at, per);
    walk.head = walk.x = walk.unit_at = 0;
    if (walk.at < walk.end) {
        if (threadIdx.x == 0) s_seq = 0;
        __syncthreads();
#pragma unroll 1
        for (int b0 = 0, before = 0;;) {
            if (walk.at >= before + lo && walk.at < before + lo + t) {
                s_seq = b0 + threadIdx.x;
                s_at = before + lo;
                s_tiles = t / v.kv_heads;
            }
            before += chunk;
            b0 += kManyThreads;
            if (walk.at < before || b0 >= v.seqs) break;
            scan(b0);
        }
        __syncthreads();
        walk.seq = s_seq;
        walk.unit_at = s_at;
        many_seq(args, walk.seq, &walk.sq);
        const int a_head = s_tiles;
        walk.head = (walk.at - walk.unit_at) / a_head;
        walk.unit_at += walk.head * a_head;
        const int off = walk.at - walk.unit_at;
        int span = walk.sq.count;  // the row tile lies in [x, x + span)
        int skip = 0;           // key tiles before row tile x
#pragma unroll 1
        while (span > 1) {
            const int step = (span + kManyThreads - 1) / kManyThreads;
            const int mid = walk.x + threadIdx.x * step;
            const bool in = mid < walk.x + span;
            const int t = in ? many_before(walk.sq, mid) : 0;
            const int n = __syncthreads_count(in && t <= off);
            if (static_cast<int>(threadIdx.x) == n - 1) s_at = t;
            __syncthreads();
            skip = s_at;
            const int next = walk.x + (n - 1) * step;
            span = min(step, walk.x + span - next);
            walk.x = next;
        }
        walk.unit_at += skip;
    }
    // Key tiles so far: of the CTA, of the role's row tile.
    uint32_t stage_it = 0, tile_it = 0;

    if (warp < kSoftmaxWarps) {
        // -------------------------------------------------------------- softmax
        registers_up<kSoftmaxRegs>();
        const int i = warp >> 3, r = lane >> 2, c = lane & 3;
        const int row_in = (warp & 3) * 32 + ((warp >> 2) & 1) * 16 + r;  // this lane's rows of the tile: it and + 8
        const uint32_t lanes = static_cast<uint32_t>(row_in - r) << 16;
        const uint32_t t_rows = tmem + i * 128 + lanes, t_o = tmem + 256 + i * D + lanes;
        for (uint32_t n = 0;; ++n) {
            const ManyUnit& u = s_unit[n % kUnits];
            wait_phase(&s_unit_full[n % kUnits], (n / kUnits) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
            if (warp_gave_up(&s_gave_up)) break;
            const int count = u.count;
            if (count == 0) break;
            if (i < u.row_tiles()) {
                // Scores are kept relative to m, once a row has seen a key: `far` is what may
                // not be passed (-inf before: any key).
                float m[2], far[2];
                uint64_t l[2];  // sums over even and over odd columns
                int limit[2], limit_min = 0x7FFFFFFF;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = i * 128 + row_in + b * 8;
                    m[b] = 0.0f;
                    far[b] = -INFINITY;
                    l[b] = 0;
                    limit[b] = 0;
                    if (row < u.rows) {
                        limit[b] = a.causal ? u.kv - u.n + (u.row0 + row) / args.group + 1 : u.kv;
                        limit_min = min(limit_min, limit[b]);
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) limit_min = min(limit_min, __shfl_xor_sync(0xFFFFFFFFu, limit_min, o));
#pragma unroll 1
                for (int j = 0; j < count; ++j) {
                    const uint32_t it = stage_it + j, st = it % S::kStages, t = tile_it + j, buf = t & 1;
                    const uint32_t t_s = t_rows + buf * kManyKeys;
                    const int pos0 = (u.t0 + j) * kManyKeys;
                    wait_phase(&s_full[st], (it / S::kStages) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
                    wait_phase(&s_scores[i][buf], (t >> 1) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
                    __syncwarp();
                    tc_fence_after();
                    // e = scale log2(e) s_k S - m: [row][column]
                    float e[2][16];
                    {
                        const uint64_t less[2] = {pair2(-m[0], -m[0]), pair2(-m[1], -m[1])};
                        uint32_t s[32];
                        tmem_ld_frag64(t_s, s);
                        const uint8_t* kl = cols + st * S::kCols + c * S::kColsRow;
#pragma unroll
                        for (int k = 0; k < 8; k += 2) {
                            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(kl + k * 8);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint64_t x = fma2(pair2(s[k * 4 + i * 2], s[k * 4 + i * 2 + 1]), i < 2 ? w.x : w.y, less[i & 1]);
                                e[i & 1][(k + (i >> 1)) * 2] = low2(x);
                                e[i & 1][(k + (i >> 1)) * 2 + 1] = high2(x);
                            }
                        }
                    }
                    if (pos0 + kManyKeys > limit_min) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int left = limit[b] - pos0 - c * 2;
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if ((k >> 1) * 8 + (k & 1) >= left) e[b][k] = -INFINITY;
                        }
                    }
                    float big[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 16; ++k) big[k & 1] = max3(big[k & 1], e[k & 1][k & ~1], e[k & 1][k | 1]);
                    if (__any_sync(0xFFFFFFFFu, big[0] > far[0] || big[1] > far[1])) {
                        float fix[2];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            float x = fmaxf(big[b], __shfl_xor_sync(0xFFFFFFFFu, big[b], 1));
                            x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 2));
                            const bool seen = far[b] > 0.0f;
                            const float up = x > (seen ? kTop : -INFINITY) ? x - kTop : 0.0f;
                            fix[b] = seen ? fast_exp2(-up) : 1.0f;
                            if (x > -INFINITY) far[b] = kFar;
                            m[b] += up;
                            l[b] = mul2(l[b], pair2(fix[b], fix[b]));
#pragma unroll
                            for (int k = 0; k < 16; ++k) e[b][k] -= up;
                        }
                        if (j > 0) {  // O, once the last product into it has ended
                            wait_phase(&s_done[i][buf ^ 1], ((t - 1) >> 1) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
                            __syncwarp();
                            tc_fence_after();
#pragma unroll 1
                            for (int ch = 0; ch < D; ch += 32) {
                                uint32_t o[16];
                                tmem_ld_frag32(t_o + ch, o);
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fix[(k >> 1) & 1]);
                                tmem_st_frag32(t_o + ch, o);
                            }
                        }
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float p0 = fast_exp2(e[k & 1][k & ~1]), p1 = fast_exp2(e[k & 1][k | 1]);
                        l[k & 1] = add2(l[k & 1], pair2(p0, p1));
                        const __half2 hp = __floats2half2_rn(p0, p1);
                        p[k] = *reinterpret_cast<const uint32_t*>(&hp);
                    }
                    tmem_st_pairs32(t_s, p);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_probs[i][buf]);
                }
                // The output, or the unit's part of it.
                const uint32_t last = tile_it + count - 1;
                wait_phase(&s_done[i][last & 1], (last >> 1) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
                __syncwarp();
                tc_fence_after();
                const bool whole = u.whole;
                const int64_t slot = blockIdx.x * 2LL + u.place;
                float sums[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    sums[b] = low2(l[b]) + high2(l[b]);
                    sums[b] += __shfl_xor_sync(0xFFFFFFFFu, sums[b], 1);
                    sums[b] += __shfl_xor_sync(0xFFFFFFFFu, sums[b], 2);
                }
#pragma unroll 1
                for (int ch = 0; ch < D; ch += 32) {
                    uint32_t o[16];
                    __syncwarp();
                    tmem_ld_frag32(t_o + ch, o);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int row = i * 128 + row_in + b * 8;
                        if (row >= u.rows) continue;
                        if (whole) {
                            const float inv = sums[b] == 0.0f ? 0.0f : fast_rcp(sums[b]);
                            const int tok = (u.row0 + row) / args.group, gh = u.row0 + row - tok * args.group;
                            uint16_t* dst = a.out + (u.first + tok) * a.ldo + (u.head * args.group + gh) * D + ch + c * 2;
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                store2(dst + k * 8, narrow2(__uint_as_float(o[k * 4 + b * 2]) * inv,
                                                            __uint_as_float(o[k * 4 + b * 2 + 1]) * inv, dtype));
                        } else {
                            float* dst = args.part_o + (slot * kManyRows + row) * D + ch + c * 2;
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *reinterpret_cast<float2*>(dst + k * 8) =
                                    make_float2(__uint_as_float(o[k * 4 + b * 2]), __uint_as_float(o[k * 4 + b * 2 + 1]));
                            if (ch == 0 && c == 0) args.part_ml[slot * kManyRows + row] = make_float2(far[b] > 0.0f ? m[b] : -INFINITY, sums[b]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[i]);
                tile_it += count;
            }
            stage_it += count;
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_unit_empty[n % kUnits]);
        }
    } else if (warp < kSoftmaxWarps + kCodesWarps) {
        // -------------------------------------------------------------- codes to operands
        registers_up<kCodesRegs>();
        // A group's first two warps take K, a token a lane; the others V, a lane eight
        // tokens (a half block) of a stretch of D / 8 channels: eight neighbouring lanes
        // write eight different 16-byte columns of V^T.
        const int group = (warp >> 2) & 1;
        const bool is_k = (warp & 2) == 0;
        const int token = (warp & 1) * 32 + lane;
        const int v_half = lane & 7, v_r = (warp & 1) * 4 + (lane >> 3);
        const int block_in = is_k ? token >> 4 : v_half >> 1;
        const int offset = is_k ? (token & 15) * (D / 2) : kv_v_codes(D) + (v_half & 1) * 4 * D + v_r * (D / 2);
        const float fac = a.scale * 1.4426950408889634f;
        for (uint32_t n = 0;; ++n) {
            const ManyUnit& u = s_unit[n % kUnits];
            wait_phase(&s_unit_full[n % kUnits], (n / kUnits) & 1, &s_gave_up, v.err_flag, kErrEpiWait);
            if (warp_gave_up(&s_gave_up)) break;
            const int count = u.count;
            if (count == 0) break;
            const int32_t* row_table = v.table + static_cast<int64_t>(u.seq) * v.ld_table;
            // Lane l holds the number of block l of eight tiles (-1: none): of those under
            // way and, fetched early, of the next eight.
            auto locate = [&](int j) {
                const int pos = (u.t0 + j) * kManyKeys + lane * kKvBlock;
                return j + (lane >> 2) < count && pos < u.kv ? kv_block_number(v, row_table, u.head, pos) : -2;
            };
            int blocks = locate(0), blocks_next = locate(8);
            uint4 w[D / 32], z[2];  // the codes; K: scales of the token, V: of the eight tokens
            auto fetch = [&](int j) {
                if ((j & 7) < 2 && j >= 8) {  // the group's first tile of eight
                    blocks = blocks_next;
                    blocks_next = locate((j & ~7) + 8);
                }
                const int at = __shfl_sync(0xFFFFFFFFu, blocks, (j & 7) * 4 + block_in);
                if (at == -1) raise_error(v.err_flag, kErrBadPage);
#pragma unroll
                for (int k = 0; k < D / 32; ++k) w[k] = make_uint4(0, 0, 0, 0);
                z[0] = z[1] = make_uint4(0, 0, 0, 0);
                if (at >= 0) {
                    const uint8_t* b = v.data + static_cast<int64_t>(at) * kv_block_bytes(D);
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) w[k] = *reinterpret_cast<const uint4*>(b + offset + k * 16);
                    if (is_k) {
                        z[0].x = reinterpret_cast<const uint32_t*>(b + kv_k_scales(D))[token & 15];
                        z[0].y = reinterpret_cast<const uint32_t*>(b + kv_v_scales(D))[token & 15];
                    } else {
                        z[0] = *reinterpret_cast<const uint4*>(b + kv_v_scales(D) + (v_half & 1) * 32);
                        z[1] = *reinterpret_cast<const uint4*>(b + kv_v_scales(D) + (v_half & 1) * 32 + 16);
                    }
                }
            };
            const int j0 = (group ^ stage_it) & 1;
            if (j0 < count) fetch(j0);
#pragma unroll 1
            for (int j = j0; j < count; j += 2) {
                const uint32_t it = stage_it + j, st = it % S::kStages;
                if (it >= S::kStages)
                    wait_phase(&s_empty[st], (it / S::kStages - 1) & 1, &s_gave_up, v.err_flag, kErrTmaWait);
                __syncwarp();
                if (is_k) {
                    // The column's scale; NaN when K or V of the token is, which so reaches the
                    // rows that see it and no other (its codes are zeros).
                    float sk = f16_bits_to_f32(static_cast<uint16_t>(z[0].x)) * fac;
                    if ((z[0].y & 0x7C00u) == 0x7C00u) sk = __int_as_float(0x7FFFFFFF);
                    *reinterpret_cast<float*>(cols + st * S::kCols + ((token >> 1) & 3) * S::kColsRow + (token >> 3) * 8 +
                                              (token & 1) * 4) = sk;
                    const uint32_t z1024 = h2_add(__byte_perm(z[0].x, 0, 0x3232), 0x64006400u), zz = z1024 & kNib0;
                    const uint32_t z64 = 0xD400D400u | zz << 4, z128 = 0x43004300u | zz;
                    const uint32_t kst = k_u32 + st * S::kK;
#pragma unroll
                    for (int k = 0; k < D / 8; ++k) {
                        const uint4 q4 = w[k >> 2];
                        const uint32_t x = (k & 3) == 0 ? q4.x : (k & 3) == 1 ? q4.y : (k & 3) == 2 ? q4.z : q4.w;
                        uint32_t e0, e1, e2, e3;
                        if constexpr (BF16) {
                            e0 = bf2_sub((x & kNib0) | 0x43004300u, z128);
                            e1 = bf2_sub(((x >> 8) & kNib0) | 0x43004300u, z128);
                            e2 = bf2_sub(((x >> 4) & kNib0) | 0x43004300u, z128);
                            e3 = bf2_sub(((x >> 12) & kNib0) | 0x43004300u, z128);
                        } else {
                            e0 = nib0_f16(x, z1024);
                            e1 = nib0_f16(x >> 8, z1024);
                            e2 = nib1_f16(x, z64);
                            e3 = nib1_f16(x >> 8, z64);
                        }
                        st_shared_16(panel_at(kst + (k >> 3) * S::kKPanel, token, k & 7), e0, e1, e2, e3);
                    }
                } else {
                    // Token pairs' zero points and scales; then, for each word of a token, its
                    // eight channels as rows of V^T.
                    uint32_t z1024[4], z64[4], sv[4];
                    const uint32_t zw[8] = {z[0].x, z[0].y, z[0].z, z[0].w, z[1].x, z[1].y, z[1].z, z[1].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        z1024[k] = h2_add(__byte_perm(zw[2 * k], zw[2 * k + 1], 0x7632), 0x64006400u);
                        z64[k] = 0xD400D400u | (z1024[k] & kNib0) << 4;
                        sv[k] = __byte_perm(zw[2 * k], zw[2 * k + 1], 0x5410);
                        if ((sv[k] & 0x7C00u) == 0x7C00u) sv[k] &= 0xFFFF0000u;  // NaN: see above
                        if ((sv[k] & 0x7C000000u) == 0x7C000000u) sv[k] &= 0xFFFFu;
                    }
                    const uint32_t vst = v_u32 + st * S::kV;
#pragma unroll 2
                    for (int hw = 0; hw < D / 32; ++hw) {  // word of a pair
                        uint32_t x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if constexpr (D == 128) {  // 16 bytes a pair
                                x[k] = w[k].x;
                                w[k].x = w[k].y;
                                w[k].y = w[k].z;
                                w[k].z = w[k].w;
                            } else {  // 8 bytes a pair
                                x[k] = (k & 1) ? w[k >> 1].z : w[k >> 1].x;
                                if (k & 1) w[k >> 1].z = w[k >> 1].w;
                                else w[k >> 1].x = w[k >> 1].y;
                            }
                        }
                        const int ch = v_r * (D / 8) + hw * 4;
                        auto store = [&](int row, auto&& value) {
                            st_shared_16(panel_at(vst, row, v_half), h2_mul(value(0), sv[0]), h2_mul(value(1), sv[1]),
                                         h2_mul(value(2), sv[2]), h2_mul(value(3), sv[3]));
                        };
                        store(ch, [&](int k) { return nib0_f16(x[k], z1024[k]); });
                        store(ch + 1, [&](int k) { return nib1_f16(x[k], z64[k]); });
                        store(ch + 2, [&](int k) { return nib0_f16(x[k] >> 8, z1024[k]); });
                        store(ch + 3, [&](int k) { return nib1_f16(x[k] >> 8, z64[k]); });
                    }
                }
                fence_async_smem();
                mbar_arrive(&s_full[st]);
                __syncwarp();
                if (j + 2 < count) fetch(j + 2);
            }
            stage_it += count;
            __syncwarp();  // (no tile of the unit may be this group's: every lane has read it all the same)
            if (lane == 0) mbar_arrive(&s_unit_empty[n % kUnits]);
        }
    } else if (warp < kSoftmaxWarps + kCodesWarps + 4) {
        // -------------------------------------------------------------- products
        registers_down<kOtherRegs>();
        const int i = warp & 1;
        const uint32_t t_rows = tmem + i * 128;
        if (lane == 0 && (warp & 2) == 0) {  // scores
            const uint32_t idesc = idesc_f16_f32(128, kManyKeys) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
            for (uint32_t n = 0;; ++n) {
                const ManyUnit& u = s_unit[n % kUnits];
                wait_phase(&s_unit_full[n % kUnits], (n / kUnits) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                if (gave_up(&s_gave_up)) break;
                const int count = u.count, row_tiles = u.row_tiles();
                mbar_arrive(&s_unit_empty[n % kUnits]);
                if (count == 0) break;
                wait_phase(&s_q, n & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                if (i >= row_tiles) {
                    mbar_arrive(&s_q_free);
                    stage_it += count;
                    continue;
                }
#pragma unroll 1
                for (int j = 0; j < count; ++j) {
                    const uint32_t it = stage_it + j, t = tile_it + j, buf = t & 1, st = it % S::kStages;
                    wait_phase(&s_full[st], (it / S::kStages) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                    // P in their place has been used
                    if (t >= 2) wait_phase(&s_done[i][buf], ((t >> 1) - 1) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                    tc_fence_after();
                    uint32_t qd = desc_low(q_u32 + i * kPanels * S::kPanel), kd = desc_low(k_u32 + st * S::kK);
#pragma unroll 1
                    for (int p = 0; p < kPanels; ++p, qd += S::kPanel >> 4, kd += S::kKPanel >> 4)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc_mma_ss(t_rows + buf * kManyKeys, qd + k * 2, kd + k * 2, idesc, p + k > 0);
                    tc_commit(&s_scores[i][buf]);
                }
                tc_commit(&s_q_free);
                tile_it += count;
                stage_it += count;
            }
        } else if (lane == 0) {  // output
            const uint32_t idesc = idesc_f16_f32(128, D), t_o = tmem + 256 + i * D;
            uint32_t units = 0;  // with this row tile
            for (uint32_t n = 0;; ++n) {
                const ManyUnit& u = s_unit[n % kUnits];
                wait_phase(&s_unit_full[n % kUnits], (n / kUnits) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                if (gave_up(&s_gave_up)) break;
                const int count = u.count, row_tiles = u.row_tiles();
                mbar_arrive(&s_unit_empty[n % kUnits]);
                if (count == 0) break;
                if (i >= row_tiles) {  // the other tile's alone: only give back what it uses
                    for (int j = 0; j < count; ++j) {
                        const uint32_t it = stage_it + j;
                        wait_phase(&s_full[it % S::kStages], (it / S::kStages) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                        mbar_arrive(&s_empty[it % S::kStages]);
                    }
                    stage_it += count;
                    continue;
                }
#pragma unroll 1
                for (int j = 0; j < count; ++j) {
                    const uint32_t it = stage_it + j, t = tile_it + j, buf = t & 1, st = it % S::kStages;
                    if (j == 0) {
                        if (units > 0) wait_phase(&s_free[i], (units - 1) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                        ++units;
                    }
                    wait_phase(&s_full[st], (it / S::kStages) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                    wait_phase(&s_probs[i][buf], (t >> 1) & 1, &s_gave_up, v.err_flag, kErrMmaWait);
                    tc_fence_after();
                    const uint32_t vd = desc_low(v_u32 + st * S::kV), pt = t_rows + buf * kManyKeys;
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_ts(t_o, pt + k * 8, vd + k * 2, idesc, j + k > 0);
                    tc_commit(&s_done[i][buf]);
                    tc_commit(&s_empty[st]);
                }
                tile_it += count;
                stage_it += count;
            }
        }
        if (lane == 0) {  // TMEM is freed and shared memory given up once all that this thread asked for has ended
            tc_commit(&s_drain[warp & 3]);
            mbar_wait(&s_drain[warp & 3], 0, nullptr, kErrDrainWait);
        }
        __syncwarp();
    } else {
        // (Before the roles part: the four warps of a group give up registers with one instruction.)
        registers_down<kOtherRegs>();
        if (warp < kManyWarps - 1) {
            // ---------------------------------------------------------- Q, as it is
            const bool vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.ldq & 7) == 0;
            const int tid = threadIdx.x - (kManyThreads - 128), ch = tid & (D / 8 - 1);
            for (uint32_t n = 0;; ++n) {
                const ManyUnit& u = s_unit[n % kUnits];
                wait_phase(&s_unit_full[n % kUnits], (n / kUnits) & 1, &s_gave_up, v.err_flag, kErrTmaWait);
                if (warp_gave_up(&s_gave_up) || u.count == 0) break;
                if (n > 0) wait_phase(&s_q_free, (n - 1) & 1, &s_gave_up, v.err_flag, kErrTmaWait);
                const uint16_t* q0 = a.q + (u.first + u.tok0) * a.ldq + u.head * args.group * D + ch * 8;
#pragma unroll 2
                for (int row = tid / (D / 8); row < u.row_tiles() * 128; row += kLoaders / (D / 8)) {
                    const uint32_t dst = panel_at(q_u32 + ((row >> 7) * kPanels + (ch >> 3)) * S::kPanel, row & 127, ch & 7);
                    const bool live = row < u.rows;
                    const int x = live ? u.head0 + row : 0, dt = args.group_magic != 0 ? __umulhi(x, args.group_magic) : x;
                    const uint16_t* src = q0 + dt * a.ldq + (x - dt * args.group) * D;
                    if (vec) {
                        copy_async_16(dst, src, live);
                    } else {
                        const uint4 w = live ? load8(src, false) : make_uint4(0, 0, 0, 0);
                        st_shared_16(dst, w.x, w.y, w.z, w.w);
                    }
                }
                copy_async_commit();
                copy_async_wait<0>();
                fence_async_smem();
                mbar_arrive(&s_q);
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_unit_empty[n % kUnits]);
            }
        } else {
            // ---------------------------------------------------------- the walk
            if (lane == 0) {
                ManyPart part{0, 0, 0, 0, -1};
                bool more = true;
                for (uint32_t n = 0; more; ++n) {
                    if (n >= kUnits)
                        wait_phase(&s_unit_empty[n % kUnits], (n / kUnits - 1) & 1, &s_gave_up, v.err_flag, kErrTmaWait);
                    if (gave_up(&s_gave_up)) break;
                    ManyUnit& u = s_unit[n % kUnits];
                    more = walk.next(args, &u);
                    if (more && u.t0 == 0 && !u.whole)
                        part = ManyPart{u.seq, u.head, u.row0, u.place, (walk.unit_at + kManyCost + walk.tiles - 1) / per};
                    mbar_arrive(&s_unit_full[n % kUnits]);
                }
                args.parts[blockIdx.x] = part;
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + kCodesWarps) tmem_dealloc(tmem, 512);
}

// Adds the parts of a unit that spans CTAs: CTAs of 32 rows per CTA it begins
// in, a quarter of a warp a row.
constexpr int kJoinRows = kThreads / 8;

template <int D>
__global__ void __launch_bounds__(kThreads) attn_q4_many_join_kernel(const ManyArgs args) {
    constexpr int PER = D / 32;  // float4 of a lane
    griddep_wait();
    griddep_launch_dependents();
    const ManyPart part = args.parts[blockIdx.x];
    if (part.last_cta < 0) return;
    const AttnQ4Args& a = args.a;
    int first, n, kv;
    kv_seq(a.v, part.seq, &first, &n, &kv);
    const int row = blockIdx.y * kJoinRows + threadIdx.x / 8, lane = threadIdx.x & 7;
    if (part.row0 + row >= n * args.group) return;
    float m = -INFINITY, l = 0.0f;
    float4 o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = blockIdx.x; p <= part.last_cta; ++p) {
        const int64_t at = (p * 2LL + (p == static_cast<int>(blockIdx.x) ? part.place : 0)) * kManyRows + row;
        const float2 ml = args.part_ml[at];
        float4 x[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = *reinterpret_cast<const float4*>(args.part_o + at * D + j * 32 + lane * 4);
        const float big = fmaxf(m, ml.x), base = big == -INFINITY ? 0.0f : big;
        const float f0 = fast_exp2(m - base), f1 = fast_exp2(ml.x - base);
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            o[j].x = o[j].x * f0 + x[j].x * f1;
            o[j].y = o[j].y * f0 + x[j].y * f1;
            o[j].z = o[j].z * f0 + x[j].z * f1;
            o[j].w = o[j].w * f0 + x[j].w * f1;
        }
        m = big;
    }
    const float inv = l == 0.0f ? 0.0f : fast_rcp(l);
    const int tok = (part.row0 + row) / args.group, gh = part.row0 + row - tok * args.group;
    uint16_t* dst = a.out + (first + tok) * a.ldo + (part.head * args.group + gh) * D + lane * 4;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        store2(dst + j * 32, narrow2(o[j].x * inv, o[j].y * inv, a.dtype));
        store2(dst + j * 32 + 2, narrow2(o[j].z * inv, o[j].w * inv, a.dtype));
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
    // Rows and tiles are numbered in 31 bits.
    const double group = static_cast<double>(heads / kv->kv_heads), keys = static_cast<double>(batch->max_kv_len) + 128;
    const double rows = static_cast<double>(batch->tokens) * group;
    if (rows + 512.0 * batch->seqs + keys * group > 2147483647.0 || static_cast<double>(batch->seqs) * kv->kv_heads * (keys / kTile + unit_cost(32)) > 2147483647.0 ||
        (rows / kManyRows + batch->seqs) * kv->kv_heads * (keys / kManyKeys + kManyCost) > 2147483647.0)
        return set_error(MRT_ERR_SHAPE, "too many rows and keys for one call");
    return MRT_OK;
}

namespace mrt {
namespace {

// How a call runs, by its sizes alone.
struct Plan {
    int few;     // 8-row tiles of the few-rows kernel, 0: the many-rows kernel
    int split;   // units may span CTAs
    int grid;
    size_t o_bytes, ml_bytes, part_bytes;  // scratch, in this order
    size_t bytes() const { return o_bytes + ml_bytes + part_bytes; }
};

constexpr int kSplitWarps = 4, kWholeWarps = 16;

Plan make_plan(const KvView& v, int64_t heads, int sms) {
    Plan p{};
    const int64_t rows = heads / v.kv_heads * std::max(v.max_q_len, 1);
    // Rows beside the keys' 16 of an MMA while they fill four of its tiles: 9 x 6000
    // tokens, 28 rows, 24.8 us against 33.0 of the many-rows kernel, 64 x 8192 110
    // against 164, 1 x 131071 47 against 92.
    if (rows > 32) {
        p.split = 1;
        p.grid = sms;
        p.o_bytes = static_cast<size_t>(p.grid) * 2 * kManyRows * v.head_dim * 4;
        p.ml_bytes = static_cast<size_t>(p.grid) * 2 * kManyRows * 8;
        p.part_bytes = static_cast<size_t>(p.grid) * sizeof(ManyPart);
        return p;
    }
    p.few = static_cast<int>((rows + 7) / 8);
    // Few short units: one CTA of sixteen warps each and no join (1 x 517 tokens 5.4 us
    // against 6.7 split, 8 x 1000 7.6 against 12.6; but 1 x 2000 10.2 against 7.5).
    const int64_t units = static_cast<int64_t>(v.seqs) * v.kv_heads;
    p.split = !(v.max_kv_len <= kWholeWarps * 2 * kTile && units <= sms && p.few <= 2);
    // Three CTAs of four warps a multiprocessor (64 x 8192 tokens 41.0 us, 1 x 131071
    // 21.6; four, 41.3 and 22.9; two of eight warps 43.9 and 22.4), two where rows take
    // the registers (14 rows, 64 x 8192 58.6 us and 9 x 6000 15.6; three, which spill,
    // 61.9 and 19.1).
    p.grid = p.split ? sms * (p.few == 1 ? 3 : 2) : static_cast<int>(units);
    if (p.split) {
        p.o_bytes = static_cast<size_t>(p.grid) * 2 * p.few * 8 * v.head_dim * 4;
        p.ml_bytes = static_cast<size_t>(p.grid) * 2 * p.few * 8 * 8;
    }
    return p;
}

template <auto KERNEL, typename... A>
cudaError_t launch_pdl(dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
    cudaError_t e = prepare_kernel<KERNEL>(smem);
    if (e != cudaSuccess) return e;
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
    e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
    if (e == cudaSuccess) note_launches(1);
    return e;
}

template <int D, int NT, int W>
cudaError_t launch_few_w(const RowsArgs& r, int rows, cudaStream_t s) {
    cudaError_t e = launch_pdl<attn_q4_few_kernel<D, NT, W>>(dim3(r.grid), W * 32, RowsShape<D, NT, W>::kBytes, s, r);
    if (e != cudaSuccess || !r.split) return e;
    const dim3 grid(r.a.v.seqs * r.a.v.kv_heads, rows);  // a CTA a (unit, row)
    // Units of 20 parts and more are worth a large CTA.  7 rows (444 parts in all): 1 x 131071 tokens (111 parts) 20.5 us
    // against 27.7, 4 x 30000 (28) 16.2 against 20.0, 5 x 30000 (22) 17.8 against 21.6, 6 x 30000 (18) 23.1 against 23.5;
    // 8 x 30000 (14) 26.8 against 26.4, 16 x 4000 (7) 20.9 against 13.7.  14 rows (296): 1 x 131071 (74) 26.7 against 31.1,
    // 3 x 30000 (25) 21.5 both ways, 4 x 30000 (18) 24.0 against 22.2.
    return static_cast<int64_t>(grid.x) * 20 <= r.grid ? launch_pdl<attn_q4_join_kernel<D, 512>>(grid, 512, 0, s, r, NT * 8)
                                                       : launch_pdl<attn_q4_join_kernel<D, 64>>(grid, 64, 0, s, r, NT * 8);
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

template <int D, bool BF16>
cudaError_t launch_many(const ManyArgs& m, cudaStream_t s) {
    const cudaError_t e = launch_pdl<attn_q4_many_kernel<D, BF16>>(dim3(m.grid), kManyThreads, ManyShape<D>::kBytes, s, m);
    if (e != cudaSuccess) return e;
    return launch_pdl<attn_q4_many_join_kernel<D>>(dim3(m.grid, kManyRows / kJoinRows), kThreads, 0, s, m);
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
    *bytes = p.bytes();
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
        if (ws_dev == nullptr || ws_bytes < plan.bytes())
            return set_error(MRT_ERR_INVALID_ARG, "scratch is NULL or smaller than mrt_kv_q4_attention_workspace says");
        if ((reinterpret_cast<uintptr_t>(ws_dev) & 255) != 0)
            return set_error(MRT_ERR_INVALID_ARG, "scratch must be 256-byte aligned");
    }
    a.dtype = dtype;
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
        r.group_magic = (65536 + r.group - 1) / r.group;
        r.vec = (reinterpret_cast<uintptr_t>(q_dev) & 15) == 0 && (ldq & 7) == 0;
        r.split = plan.split;
        r.grid = plan.grid;
        r.warps = kSplitWarps;
        r.part_o = static_cast<float*>(ws_dev);
        r.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws_dev) + plan.o_bytes);
        const int rows = r.group * std::max(a.v.max_q_len, 1);
        e = D == 128 ? launch_few<128>(r, plan.few, rows, s) : launch_few<64>(r, plan.few, rows, s);
    } else {
        ManyArgs m{};
        m.a = a;
        m.group = static_cast<int>(heads / kv->kv_heads);
        m.group_magic = m.group > 1 ? static_cast<uint32_t>(((1ull << 32) + m.group - 1) / m.group) : 0;
        m.grid = plan.grid;
        m.part_o = static_cast<float*>(ws_dev);
        m.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws_dev) + plan.o_bytes);
        m.parts = reinterpret_cast<ManyPart*>(static_cast<uint8_t*>(ws_dev) + plan.o_bytes + plan.ml_bytes);
        if (D == 128)
            e = dtype == MRT_BF16 ? launch_many<128, true>(m, s) : launch_many<128, false>(m, s);
        else
            e = dtype == MRT_BF16 ? launch_many<64, true>(m, s) : launch_many<64, false>(m, s);
    }
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "4-bit attention launch");
}
