// kv_q4.cu -- a paged key/value cache held in 4 bits: its handle, the append of
// new tokens with the position rotation on the way (the rotation of the
// reference's RoPE op, src/core/cpu_backend.cpp:332-379), and reading rows back.
//
// Every (token, head) row of D channels has one scale and one zero point:
//   lo = min(0, min x), hi = max(0, max x)
//   s  = max(fp16((hi - lo) / 15), 2^-24),  z = rint(-lo / s),  c = rint(x / s) + z
// (both clamped to 0..15), and holds the values s (c - z).  Where codes could so
// mean more than FP16 holds (s max(z, 15 - z) > 65504: a row that reaches beyond
// 60000), s is then lowered until they do not: all held values are finite as
// FP16 operands, and a token that a row does not see adds 0 times a number.  One scale a row
// rather than one for every 32 channels: the attention kernel then multiplies
// a key's scale into one score and a value's into one probability, and the
// codes go to the tensor cores untouched.
//
// The rotation angle p theta^(-2i/D) is exact for any position: a pair's turns
// per position are held as a fraction of 2^64, so p times it, wrapping, is the
// phase, and only the remainder goes through sincospi (in 64 bits; a token's
// pairs are shared by all its heads).
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

int kv_view(mrt_kv_q4 kv, const mrt_kv_batch* b, KvView* out) {
    if (kv == nullptr || b == nullptr) return set_error(MRT_ERR_INVALID_ARG, "NULL cache or batch");
    if (b->seqs < 0 || b->tokens < 0 || b->max_q_len < 0 || b->max_kv_len < 0)
        return set_error(MRT_ERR_SHAPE, "batch sizes must be >= 0");
    const int64_t lim = (1LL << 31) - 256;
    if (b->seqs > 65535 || b->tokens > lim || b->max_q_len > lim || b->max_kv_len > lim || b->ld_table > lim)
        return set_error(MRT_ERR_SHAPE, "batch sizes must fit in 31 bits, sequences in 16");
    if (b->seqs > 0 && b->tokens > 0) {
        if (b->q_start_dev == nullptr || b->kv_len_dev == nullptr || b->table_dev == nullptr)
            return set_error(MRT_ERR_INVALID_ARG, "NULL q_start, kv_len or table");
        if (b->max_kv_len > b->ld_table * kv->page_tokens)
            return set_error(MRT_ERR_SHAPE, "max_kv_len is more than ld_table pages hold");
    }
    KvView v{};
    v.data = kv->data;
    v.pages = static_cast<int>(kv->pages);
    v.page_tokens = static_cast<int>(kv->page_tokens);
    const int blocks = v.page_tokens / kKvBlock;
    v.page_shift = (blocks & (blocks - 1)) == 0 ? __builtin_ctz(blocks) : -1;
    v.kv_heads = static_cast<int>(kv->kv_heads);
    v.head_dim = static_cast<int>(kv->head_dim);
    v.seqs = static_cast<int>(b->seqs);
    v.tokens = static_cast<int>(b->tokens);
    v.max_q_len = static_cast<int>(b->max_q_len);
    v.max_kv_len = static_cast<int>(b->max_kv_len);
    v.ld_table = static_cast<int>(b->ld_table);
    v.q_start = b->q_start_dev;
    v.kv_len = b->kv_len_dev;
    v.table = b->table_dev;
    *out = v;
    return MRT_OK;
}

int kv_bind(mrt_kv_q4 kv, KvView* v, int* sms) {
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    if (c->device != kv->device) return set_error(MRT_ERR_INVALID_ARG, "cache lives on another device");
    v->err_flag = c->d_err;
    if (sms) *sms = c->sms;
    return MRT_OK;
}

namespace {

constexpr int kThreads = 256;

struct Freqs {
    uint64_t turn[64];
};

struct AppendArgs {
    KvView v;
    int dtype, heads, rotate;
    int tokens;  // of a CTA
    int rows;    // of a token that a CTA takes (grid y covers the others)
    const uint16_t* q;
    int64_t ldq;
    uint16_t* q_out;
    int64_t ldqo;
    const uint16_t* k;
    int64_t ldk;
    const uint16_t* val;
    int64_t ldv;
    int vec;  // rows can be read and written 16 bytes at a time
    uint64_t row_magic;  // 2^40 / rows, rounded up: i * it >> 40 = i / rows for i rows < 2^40
};

constexpr int kMaxTokens = 8;  // of a CTA

__device__ __forceinline__ float widen(uint32_t h, int dtype) {
    return dtype == MRT_BF16 ? bf16_bits_to_f32(static_cast<uint16_t>(h)) : __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
}

// Two neighbouring values, rounded to nearest.
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, int dtype) {
    if (dtype == MRT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight neighbouring 16-bit values at any alignment of two bytes.
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool vec) {
    if (vec) return *reinterpret_cast<const uint4*>(p);
    uint4 v;
    v.x = p[0] | static_cast<uint32_t>(p[1]) << 16;
    v.y = p[2] | static_cast<uint32_t>(p[3]) << 16;
    v.z = p[4] | static_cast<uint32_t>(p[5]) << 16;
    v.w = p[6] | static_cast<uint32_t>(p[7]) << 16;
    return v;
}

__device__ __forceinline__ void store8(uint16_t* p, uint4 v, bool vec) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[2 * j] = static_cast<uint16_t>(w[j]);
        p[2 * j + 1] = static_cast<uint16_t>(w[j] >> 16);
    }
}

// Sequence and position of `count` rows from t0 on (block-wide): seq[i] < 0 for
// a row that is nobody's or breaks the call's bounds.  The first block looks at
// every sequence, so that one whose rows no block has is reported too.
__device__ __forceinline__ void find_rows(const KvView& v, int t0, int count, int* seq, int* pos) {
    if (threadIdx.x < count) seq[threadIdx.x] = -1;
    __syncthreads();
    const bool every = blockIdx.x == 0 && blockIdx.y == 0;
    for (int b = threadIdx.x; b < v.seqs; b += blockDim.x) {
        const int f = v.q_start[b], e = v.q_start[b + 1];
        if (!every && (e <= t0 || f >= t0 + count || e <= f)) continue;
        int first, n, kv;
        if (!kv_seq(v, b, &first, &n, &kv)) {
            raise_error(v.err_flag, kErrBadPage);
            continue;
        }
        for (int i = max(f - t0, 0); i < min(e - t0, count); ++i) {
            const int p = kv - n + (t0 + i - f);
            if (p < 0) continue;
            seq[i] = b;
            pos[i] = p;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ void widen8(uint4 w, int dtype, float (&x)[8]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = widen(v[j >> 1] >> (16 * (j & 1)) & 0xFFFFu, dtype);
}

__device__ __forceinline__ uint4 narrow8(const float (&x)[8], int dtype) {
    return make_uint4(narrow2(x[0], x[1], dtype), narrow2(x[2], x[3], dtype), narrow2(x[4], x[5], dtype),
                      narrow2(x[6], x[7], dtype));
}

// The codes of eight values: rint(x inv) + z, kept in 0..15 (adding 1.5 * 2^23
// rounds to the nearest whole number, ties to even, and leaves it in the low
// bits).  The product has its own rounding: scalar operations, because a product
// and a sum of register pairs become one fused operation.
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], float inv, int z, bool value) {
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = __float_as_int(__fadd_rn(__fmul_rn(x[j], inv), 12582912.0f)) - 0x4B400000 + z;
        word |= static_cast<uint32_t>(min(max(c, 0), 15)) << (4 * (value ? j : pair_nibble(j)));
    }
    return word;
}

// A row of D channels is D / 16 lanes, each with eight channels and the eight
// that the rotation pairs them with, so a warp has four or eight rows, no value
// changes lanes and every lane packs whole words.  CTAs take tokens (prompts:
// eight, so that the angles' sines, in 64 bits, and the search for the sequence
// are shared by many rows) and all their rows, or, when tokens are few, a stretch
// of them.  Five prompts of up to 2900 tokens (9758 tokens, 36 rows of 128) take
// 38.5 us where their bytes (165 MB) would take 25, and 9.6 to be read back (25
// MB, 3.8).  No unit is full there (issue slots 42%, ALU 28%): of the ten cycles
// between a warp's instructions 3.6 wait for global loads, as no row is under way
// before the token's place and sines are known, and 1.6 for shared memory and the
// sines.  33 tokens take 3.7 us, a launch and four loads that wait for one another.
template <int D>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs a, const Freqs f) {
    constexpr int LANES = D / 16, HALF = D / 2;
    __shared__ __align__(16) float cs[kMaxTokens * HALF], sn[kMaxTokens * HALF];
    __shared__ int s_seq[kMaxTokens], s_pos[kMaxTokens];
    griddep_wait();
    griddep_launch_dependents();
    const KvView& v = a.v;
    const int t0 = blockIdx.x * a.tokens, count = min(a.tokens, v.tokens - t0);
    find_rows(v, t0, count, s_seq, s_pos);
    if (a.rotate) {
        for (int i = threadIdx.x; i < count * HALF; i += kThreads) {
            const int t = i / HALF, j = i - t * HALF;
            if (s_seq[t] < 0) continue;
            const double half_turns = static_cast<double>(static_cast<int64_t>(static_cast<uint64_t>(s_pos[t]) * f.turn[j])) * 0x1p-63;
            double sv, cv;
            sincospi(half_turns, &sv, &cv);
            cs[i] = static_cast<float>(cv);
            sn[i] = static_cast<float>(sv);
        }
        __syncthreads();
    }
    const int lane = threadIdx.x & (LANES - 1);
    const int rows = a.heads + 2 * v.kv_heads, row0 = blockIdx.y * a.rows, here = min(a.rows, rows - row0);
    const int items = count * here;
    // Whole warps go round, so that a row's lanes are there for its shuffles.
#pragma unroll 1
    for (int i0 = 0; i0 < items; i0 += kThreads / LANES) {
        const int i = i0 + threadIdx.x / LANES;
        const int t = static_cast<int>(static_cast<uint64_t>(i) * a.row_magic >> 40);  // i / here for a whole token's rows
        const int ti = a.tokens > 1 ? t : 0, row = row0 + i - ti * here;
        const bool live = i < items && s_seq[ti] >= 0;
        const bool is_q = row < a.heads, is_v = row >= a.heads + v.kv_heads;
        const int h = is_q ? row : (is_v ? row - a.heads - v.kv_heads : row - a.heads);
        const int64_t tok = t0 + ti;
        const int ch = h * D + lane * 8;
        float x0[8] = {}, x1[8] = {};
        if (live) {
            const uint16_t* src = (is_q ? a.q + tok * a.ldq : (is_v ? a.val + tok * a.ldv : a.k + tok * a.ldk)) + ch;
            const uint4 w0 = load8(src, a.vec), w1 = load8(src + HALF, a.vec);
            widen8(w0, a.dtype, x0);
            widen8(w1, a.dtype, x1);
            if (a.rotate && !is_v) {
                const float4* c4 = reinterpret_cast<const float4*>(cs + ti * HALF + lane * 8);
                const float4* s4 = reinterpret_cast<const float4*>(sn + ti * HALF + lane * 8);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float c[4] = {c4[j].x, c4[j].y, c4[j].z, c4[j].w}, s[4] = {s4[j].x, s4[j].y, s4[j].z, s4[j].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {  // products and sums each rounded
                        float &p = x0[j * 4 + k], &q = x1[j * 4 + k];
                        const float y = __fsub_rn(__fmul_rn(p, c[k]), __fmul_rn(q, s[k]));
                        q = __fadd_rn(__fmul_rn(p, s[k]), __fmul_rn(q, c[k]));
                        p = y;
                    }
                }
            }
            if (is_q) {
                uint16_t* dst = a.q_out + tok * a.ldqo + ch;
                store8(dst, narrow8(x0, a.dtype), a.vec);
                store8(dst + HALF, narrow8(x1, a.dtype), a.vec);
            }
        }
        const bool held = live && !is_q;
        if (!__any_sync(0xFFFFFFFFu, held)) continue;
        float lo = 0.0f, hi = 0.0f;
        bool odd = false;  // NaN, infinity, or beyond FP16
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo = fminf(lo, fminf(x0[j], x1[j]));
            hi = fmaxf(hi, fmaxf(x0[j], x1[j]));
            const float sum = fabsf(x0[j]) + fabsf(x1[j]);
            odd |= sum != sum;  // a NaN (a sum of magnitudes is none else)
        }
        odd |= !(fmaxf(-lo, hi) <= 65504.0f);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        const uint32_t group = __ballot_sync(0xFFFFFFFFu, odd) >> (threadIdx.x & 31 & ~(LANES - 1));
        odd = (group & ((1u << LANES) - 1)) != 0;
        if (!held) continue;
        const int pos = s_pos[ti], token = pos & (kKvBlock - 1);
        uint8_t* block = kv_block_at(v, v.table + static_cast<int64_t>(s_seq[ti]) * v.ld_table, h, pos);
        if (block == nullptr) {
            if (lane == 0) raise_error(v.err_flag, kErrBadPage);
            continue;
        }
        uint16_t sb = __half_as_ushort(__float2half_rn(fmaxf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 5.9604644775390625e-8f)));
        float inv = __frcp_rn(__half2float(__ushort_as_half(sb)));
        float zero = fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f);
        const float most = fmaxf(zero, 15.0f - zero);  // a code's distance from the zero point
        if (__half2float(__ushort_as_half(sb)) * most > 65504.0f) {
            sb = __half_as_ushort(__float2half_rd(__fdiv_rd(65504.0f, most)));
            inv = __frcp_rn(__half2float(__ushort_as_half(sb)));
        }
        uint32_t w0 = codes8(x0, inv, static_cast<int>(zero), is_v), w1 = codes8(x1, inv, static_cast<int>(zero), is_v);
        if (odd) {  // no scale says what the row holds: it reads back as NaN
            w0 = w1 = 0;
            sb = 0x7FFFu;
            zero = 0.0f;
        }
        if (is_v) {
            uint16_t* d0 = reinterpret_cast<uint16_t*>(block + kv_v_half(D, token, lane));
            uint16_t* d1 = reinterpret_cast<uint16_t*>(block + kv_v_half(D, token, lane + LANES));
            d0[0] = static_cast<uint16_t>(w0);
            d0[2] = static_cast<uint16_t>(w0 >> 16);
            d1[0] = static_cast<uint16_t>(w1);
            d1[2] = static_cast<uint16_t>(w1 >> 16);
        } else {
            *reinterpret_cast<uint32_t*>(block + kv_k_word(D, token, lane)) = w0;
            *reinterpret_cast<uint32_t*>(block + kv_k_word(D, token, lane + LANES)) = w1;
        }
        if (lane == 0)
            reinterpret_cast<uint32_t*>(block + (is_v ? kv_v_scales(D) : kv_k_scales(D)))[token] =
                sb | static_cast<uint32_t>(__half_as_ushort(__float2half_rn(zero))) << 16;
    }
}

struct ReadArgs {
    KvView v;
    int dtype, tokens;
    uint16_t* k;
    int64_t ldk;
    uint16_t* val;
    int64_t ldv;
    int vec;
    uint64_t row_magic;
};

template <int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadArgs a) {
    constexpr int LANES = D / 16, HALF = D / 2;
    __shared__ int s_seq[kMaxTokens], s_pos[kMaxTokens];
    griddep_wait();
    griddep_launch_dependents();
    const KvView& v = a.v;
    const int t0 = blockIdx.x * a.tokens, count = min(a.tokens, v.tokens - t0);
    find_rows(v, t0, count, s_seq, s_pos);
    const int lane = threadIdx.x & (LANES - 1), rows = 2 * v.kv_heads;
#pragma unroll 1
    for (int i = threadIdx.x / LANES; i < count * rows; i += kThreads / LANES) {
        const int t = static_cast<int>(static_cast<uint64_t>(i) * a.row_magic >> 40), row = i - t * rows;
        const bool value = row >= v.kv_heads;
        const int h = value ? row - v.kv_heads : row;
        uint16_t* dst = value ? a.val : a.k;
        if (dst == nullptr || s_seq[t] < 0) continue;
        const int pos = s_pos[t], token = pos & (kKvBlock - 1);
        const uint8_t* block = kv_block_at(v, v.table + static_cast<int64_t>(s_seq[t]) * v.ld_table, h, pos);
        if (block == nullptr) {
            if (lane == 0) raise_error(v.err_flag, kErrBadPage);
            continue;
        }
        const uint32_t sz = reinterpret_cast<const uint32_t*>(block + (value ? kv_v_scales(D) : kv_k_scales(D)))[token];
        const float s = __half2float(__ushort_as_half(static_cast<uint16_t>(sz)));
        const uint64_t s2 = pair2(s, s);
        const float less = -8388608.0f - __half2float(__ushort_as_half(static_cast<uint16_t>(sz >> 16)));  // -(2^23 + z): exact
        const uint64_t less2 = pair2(less, less);
        dst += (t0 + t) * (value ? a.ldv : a.ldk) + h * D + lane * 8;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int wi = lane + part * LANES;
            uint32_t w;
            if (value) {
                const uint16_t* p = reinterpret_cast<const uint16_t*>(block + kv_v_half(D, token, wi));
                w = p[0] | static_cast<uint32_t>(p[2]) << 16;
            } else {
                w = *reinterpret_cast<const uint32_t*>(block + kv_k_word(D, token, wi));
            }
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // 2^23 + c in FP32 is 0x4B000000 | c
                const uint32_t c0 = (w >> (4 * (value ? 2 * j : pair_nibble(2 * j)))) & 15u;
                const uint32_t c1 = (w >> (4 * (value ? 2 * j + 1 : pair_nibble(2 * j + 1)))) & 15u;
                const uint64_t v = mul2(s2, add2(pair2(0x4B000000u | c0, 0x4B000000u | c1), less2));
                x[2 * j] = low2(v);
                x[2 * j + 1] = high2(v);
            }
            store8(dst + part * HALF, narrow8(x, a.dtype), a.vec);
        }
    }
}

uint64_t magic_of(int rows) { return ((1ull << 40) + rows - 1) / rows; }

// Tokens of a CTA: as many as leave every multiprocessor two CTAs (append and
// read of 9758 tokens 50 us, with one token a CTA 114; of 33 6.6 us, with eight a
// CTA 13.3; of 700 9.1, against 12.6 and 13.5).
int tokens_of(int tokens, int sms) { return std::max(1, std::min(kMaxTokens, tokens / (2 * sms))); }

bool aligned16(const void* p, int64_t ld) { return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0); }

template <auto KERNEL, typename... A>
cudaError_t launch_pdl(dim3 grid, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
    if (e == cudaSuccess) note_launches(1);
    return e;
}

}  // namespace
}  // namespace mrt

using namespace mrt;

extern "C" int mrt_kv_q4_create(int64_t pages, int64_t page_tokens, int64_t kv_heads, int64_t head_dim,
                                float rope_theta, mrt_kv_q4* out) {
    clear_error();
    if (out == nullptr) return set_error(MRT_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (pages <= 0 || pages > (1LL << 31) - 1 || kv_heads <= 0 || kv_heads > 65535)
        return set_error(MRT_ERR_SHAPE, "pages and kv_heads must be positive");
    if (page_tokens <= 0 || page_tokens % kKvBlock != 0 || page_tokens > (1 << 20))
        return set_error(MRT_ERR_SHAPE, "page_tokens must be a multiple of 16");
    if (static_cast<double>(pages) * kv_heads * (page_tokens / kKvBlock) > 2147483647.0)
        return set_error(MRT_ERR_SHAPE, "pages, heads and page_tokens are too large together");
    if (head_dim != 64 && head_dim != 128) return set_error(MRT_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (!(rope_theta == 0.0f || (rope_theta >= 1.0f && rope_theta <= 3.4e38f)))
        return set_error(MRT_ERR_INVALID_ARG, "rope_theta must be 0 (no rotation) or >= 1");
    DevCtx* c = current_ctx();
    if (!c) return MRT_ERR_CUDA;
    mrt_kv_q4_s* kv = new mrt_kv_q4_s();
    kv->device = c->device;
    kv->pages = pages;
    kv->page_tokens = page_tokens;
    kv->kv_heads = kv_heads;
    kv->head_dim = head_dim;
    kv->rotate = rope_theta != 0.0f;
    for (int64_t i = 0; i < 64; ++i) {
        // theta^(-2i/D) / (2 pi) turns, times 2^64 (below 2^62)
        const long double turns = i < head_dim / 2 && kv->rotate
                                      ? powl(static_cast<long double>(rope_theta), -2.0L * i / head_dim) / 6.283185307179586476925286766559L
                                      : 0.0L;
        kv->freq[i] = static_cast<uint64_t>(roundl(turns * 18446744073709551616.0L));
    }
    const size_t bytes = static_cast<size_t>(pages) * kv_heads * (page_tokens / kKvBlock) * kv_block_bytes(static_cast<int>(head_dim));
    cudaError_t e = cudaMalloc(&kv->data, bytes);
    if (e == cudaSuccess) {
        e = cudaMemset(kv->data, 0, bytes);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();  // done before any stream uses it
        if (e != cudaSuccess) cudaFree(kv->data);
    }
    if (e != cudaSuccess) {
        delete kv;
        return cuda_error(e, "allocating the 4-bit cache");
    }
    *out = kv;
    return MRT_OK;
}

extern "C" int mrt_kv_q4_free(mrt_kv_q4 kv) {
    if (kv == nullptr) return MRT_OK;
    cudaFree(kv->data);
    delete kv;
    return MRT_OK;
}

static int check_dtype(int dtype) {
    return dtype == MRT_FP16 || dtype == MRT_BF16 ? MRT_OK : set_error(MRT_ERR_DTYPE, "dtype must be FP16 or BF16");
}

extern "C" int mrt_kv_q4_append(mrt_kv_q4 kv, const mrt_kv_batch* batch, int dtype, const void* q_dev, int64_t ldq,
                                int64_t heads, void* q_out_dev, int64_t ldqo, const void* k_dev, int64_t ldk,
                                const void* v_dev, int64_t ldv, void* stream) {
    clear_error();
    AppendArgs a{};
    int rc = kv_view(kv, batch, &a.v);
    if (rc != MRT_OK || (rc = check_dtype(dtype)) != MRT_OK) return rc;
    if (heads < 0 || heads > 65535) return set_error(MRT_ERR_SHAPE, "heads must be in [0, 65535]");
    if (a.v.seqs == 0 || a.v.tokens == 0) return MRT_OK;
    if (k_dev == nullptr || v_dev == nullptr || (heads > 0 && (q_dev == nullptr || q_out_dev == nullptr)))
        return set_error(MRT_ERR_INVALID_ARG, "NULL q, q_out, k or v");
    const int64_t D = kv->head_dim;
    if (ldk < kv->kv_heads * D || ldv < kv->kv_heads * D || (heads > 0 && (ldq < heads * D || ldqo < heads * D)))
        return set_error(MRT_ERR_SHAPE, "a token's stride must cover its heads");
    int sms = 0;
    if ((rc = kv_bind(kv, &a.v, &sms)) != MRT_OK) return rc;
    a.dtype = dtype;
    a.heads = static_cast<int>(heads);
    a.rotate = kv->rotate ? 1 : 0;
    a.q = static_cast<const uint16_t*>(q_dev);
    a.ldq = ldq;
    a.q_out = static_cast<uint16_t*>(q_out_dev);
    a.ldqo = ldqo;
    a.k = static_cast<const uint16_t*>(k_dev);
    a.ldk = ldk;
    a.val = static_cast<const uint16_t*>(v_dev);
    a.ldv = ldv;
    a.vec = aligned16(a.q, ldq) && aligned16(a.q_out, ldqo) && aligned16(a.k, ldk) && aligned16(a.val, ldv);
    a.tokens = tokens_of(a.v.tokens, sms);
    const int rows = a.heads + 2 * a.v.kv_heads, pass = kThreads / static_cast<int>(D / 16);
    // Few tokens: no more than a pass a CTA (33 of 36 rows: 6.6 us, whole tokens 6.9).
    a.rows = a.tokens > 1 ? rows : std::min(pass, 16);
    a.row_magic = magic_of(rows);
    Freqs f;
    for (int i = 0; i < 64; ++i) f.turn[i] = kv->freq[i];
    const dim3 grid(static_cast<unsigned>((a.v.tokens + a.tokens - 1) / a.tokens), static_cast<unsigned>((rows + a.rows - 1) / a.rows));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = D == 128 ? launch_pdl<kv_append_kernel<128>>(grid, s, a, f) : launch_pdl<kv_append_kernel<64>>(grid, s, a, f);
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "4-bit cache append launch");
}

extern "C" int mrt_kv_q4_read(mrt_kv_q4 kv, const mrt_kv_batch* batch, int dtype, void* k_dev, int64_t ldk, void* v_dev,
                              int64_t ldv, void* stream) {
    clear_error();
    ReadArgs a{};
    int rc = kv_view(kv, batch, &a.v);
    if (rc != MRT_OK || (rc = check_dtype(dtype)) != MRT_OK) return rc;
    if (a.v.seqs == 0 || a.v.tokens == 0 || (k_dev == nullptr && v_dev == nullptr)) return MRT_OK;
    const int64_t D = kv->head_dim;
    if ((k_dev != nullptr && ldk < kv->kv_heads * D) || (v_dev != nullptr && ldv < kv->kv_heads * D))
        return set_error(MRT_ERR_SHAPE, "a token's stride must cover its heads");
    int sms = 0;
    if ((rc = kv_bind(kv, &a.v, &sms)) != MRT_OK) return rc;
    a.dtype = dtype;
    a.k = static_cast<uint16_t*>(k_dev);
    a.ldk = ldk;
    a.val = static_cast<uint16_t*>(v_dev);
    a.ldv = ldv;
    a.vec = aligned16(k_dev, ldk) && aligned16(v_dev, ldv);
    a.row_magic = magic_of(2 * a.v.kv_heads);
    a.tokens = tokens_of(a.v.tokens, sms);
    const dim3 grid(static_cast<unsigned>((a.v.tokens + a.tokens - 1) / a.tokens));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = D == 128 ? launch_pdl<kv_read_kernel<128>>(grid, s, a) : launch_pdl<kv_read_kernel<64>>(grid, s, a);
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "4-bit cache read launch");
}
