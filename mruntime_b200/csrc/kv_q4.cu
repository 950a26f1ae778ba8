// kv_q4.cu -- a paged key/value cache held in 4 bits: its handle, the append of
// new tokens with the position rotation on the way (the rotation of the
// reference's RoPE op, src/core/cpu_backend.cpp:332-379), and reading rows back.
//
// Every (token, head) row of D channels has one scale and one zero point:
//   lo = min(0, min x), hi = max(0, max x)
//   s  = max(fp16((hi - lo) / 15), 2^-24),  z = rint(-lo / s),  c = rint(x / s) + z
// (both clamped to 0..15), and holds the values s (c - z).  One scale a row
// rather than one for every 32 channels: the attention kernel then multiplies
// a key's scale into one score and a value's into one probability, and the
// codes go to the tensor cores untouched.
//
// The rotation angle p theta^(-2i/D) is exact for any position: a pair's turns
// per position are held as a fraction of 2^64, so p times it, wrapping, is the
// phase, and only the remainder goes through sincospi (in 64 bits; a token's
// pairs are shared by all its heads).
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
constexpr int kWarps = kThreads / 32;

struct Freqs {
    uint64_t turn[64];
};

struct AppendArgs {
    KvView v;
    int dtype, heads, rotate, per_cta;
    const uint16_t* q;
    int64_t ldq;
    uint16_t* q_out;
    int64_t ldqo;
    const uint16_t* k;
    int64_t ldk;
    const uint16_t* val;
    int64_t ldv;
};

__device__ __forceinline__ float widen(uint16_t h, int dtype) {
    return dtype == MRT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

__device__ __forceinline__ uint16_t narrow(float f, int dtype) {
    if (dtype == MRT_FP16) return f32_to_f16_bits(f);
    return f != f ? static_cast<uint16_t>(0x7FC0) : f32_to_bf16_bits(f);
}

// The sequence of row t (block-wide; -1: none, or a sequence outside its bounds).
__device__ __forceinline__ int find_seq(const KvView& v, int t, int* s_seq) {
    if (threadIdx.x == 0) *s_seq = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < v.seqs; b += blockDim.x)
        if (v.q_start[b] <= t && t < v.q_start[b + 1]) *s_seq = b;
    __syncthreads();
    return *s_seq;
}

// Lane l's D / 32 neighbouring channels of a row.
template <int PER>
__device__ __forceinline__ void load_row(const uint16_t* p, int lane, int dtype, float (&x)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = widen(p[lane * PER + j], dtype);
}

// Row quantised into its block's words and scale.
template <int PER>
__device__ __forceinline__ void store_row(uint8_t* block, int token, int lane, bool value, const float (&x)[PER]) {
    constexpr int D = PER * 32;
    float lo = 0.0f, hi = 0.0f;
    bool odd = false;  // NaN, infinity, or beyond FP16
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        odd |= !(fabsf(x[j]) <= 65504.0f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    odd = __any_sync(0xFFFFFFFFu, odd);
    uint16_t sb = f32_to_f16_bits(fmaxf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 5.9604644775390625e-8f));
    const float inv = __fdiv_rn(1.0f, f16_bits_to_f32(sb));
    const float z = fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f);
    uint32_t zero = static_cast<uint32_t>(z);
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t c = static_cast<uint32_t>(fminf(fmaxf(__fadd_rn(rintf(__fmul_rn(x[j], inv)), z), 0.0f), 15.0f));
        const int in_word = (lane * PER + j) & 7;
        word |= c << (4 * (value ? in_word : pair_nibble(in_word)));
    }
#pragma unroll
    for (int o = 1; o < 8 / PER; o <<= 1) word |= __shfl_xor_sync(0xFFFFFFFFu, word, o);
    if (odd) {  // no scale says what the row holds: it reads back as NaN
        word = 0;
        sb = 0x7FFFu;
        zero = 0;
    }
    const int w = lane * PER / 8;
    if (lane % (8 / PER) == 0)
        *reinterpret_cast<uint32_t*>(block + (value ? kv_v_word(D, token, w) : kv_k_word(D, token, w))) = word;
    if (lane == 0)
        reinterpret_cast<uint32_t*>(block + (value ? kv_v_scales(D) : kv_k_scales(D)))[token] = sb | zero << 16;
}

// One CTA per token (and stretch of heads), one warp per head at a time.
template <int PER>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs a, const Freqs f) {
    constexpr int D = PER * 32, HALF = D / 2;
    __shared__ float cs[HALF], sn[HALF];
    __shared__ int s_seq;
    griddep_wait();
    griddep_launch_dependents();
    const KvView& v = a.v;
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = find_seq(v, t, &s_seq);
    if (b < 0) return;
    int first, n, kv;
    if (!kv_seq(v, b, &first, &n, &kv)) {
        if (threadIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
        return;
    }
    const int pos = kv - n + (t - first);
    if (pos < 0) return;
    if (a.rotate && threadIdx.x < HALF) {
        const double half_turns =
            static_cast<double>(static_cast<int64_t>(static_cast<uint64_t>(pos) * f.turn[threadIdx.x])) * 0x1p-63;
        double sv, cv;
        sincospi(half_turns, &sv, &cv);
        cs[threadIdx.x] = static_cast<float>(cv);
        sn[threadIdx.x] = static_cast<float>(sv);
    }
    __syncthreads();
    const int tasks = a.heads + 2 * v.kv_heads;
    const int last = min(tasks, static_cast<int>(blockIdx.y + 1) * a.per_cta);
    for (int task = blockIdx.y * a.per_cta + warp; task < last; task += kWarps) {
        const bool is_q = task < a.heads, is_v = task >= a.heads + v.kv_heads;
        const int h = is_q ? task : (is_v ? task - a.heads - v.kv_heads : task - a.heads);
        const uint16_t* src = is_q ? a.q + t * a.ldq : (is_v ? a.val + t * a.ldv : a.k + t * a.ldk);
        float x[PER];
        load_row<PER>(src + h * D, lane, a.dtype, x);
        if (!is_v && a.rotate) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float other = __shfl_xor_sync(0xFFFFFFFFu, x[j], 16);
                const int i = (lane & 15) * PER + j;
                const float c = cs[i], s = sn[i];
                x[j] = lane < 16 ? __fsub_rn(__fmul_rn(x[j], c), __fmul_rn(other, s))
                                 : __fadd_rn(__fmul_rn(other, s), __fmul_rn(x[j], c));
            }
        }
        if (is_q) {
#pragma unroll
            for (int j = 0; j < PER; ++j) a.q_out[t * a.ldqo + h * D + lane * PER + j] = narrow(x[j], a.dtype);
            continue;
        }
        uint8_t* block = kv_block_at(v, v.table + static_cast<int64_t>(b) * v.ld_table, h, pos);
        if (block == nullptr) {
            if (lane == 0) raise_error(v.err_flag, kErrBadPage);
            continue;
        }
        store_row<PER>(block, pos & (kKvBlock - 1), lane, is_v, x);
    }
}

struct ReadArgs {
    KvView v;
    int dtype;
    uint16_t* k;
    int64_t ldk;
    uint16_t* val;
    int64_t ldv;
};

template <int PER>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadArgs a) {
    constexpr int D = PER * 32;
    __shared__ int s_seq;
    griddep_wait();
    griddep_launch_dependents();
    const KvView& v = a.v;
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = find_seq(v, t, &s_seq);
    if (b < 0) return;
    int first, n, kv;
    if (!kv_seq(v, b, &first, &n, &kv)) {
        if (threadIdx.x == 0) raise_error(v.err_flag, kErrBadPage);
        return;
    }
    const int pos = kv - n + (t - first);
    if (pos < 0) return;
    for (int task = warp; task < 2 * v.kv_heads; task += kWarps) {
        const bool value = task >= v.kv_heads;
        const int h = value ? task - v.kv_heads : task;
        uint16_t* dst = value ? a.val : a.k;
        if (dst == nullptr) continue;
        dst += t * (value ? a.ldv : a.ldk) + h * D;
        const uint8_t* block = kv_block_at(v, v.table + static_cast<int64_t>(b) * v.ld_table, h, pos);
        if (block == nullptr) {
            if (lane == 0) raise_error(v.err_flag, kErrBadPage);
            continue;
        }
        const int token = pos & (kKvBlock - 1);
        const uint32_t sz = reinterpret_cast<const uint32_t*>(block + (value ? kv_v_scales(D) : kv_k_scales(D)))[token];
        const float s = f16_bits_to_f32(static_cast<uint16_t>(sz));
        const int z = static_cast<int>(sz >> 16);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int ch = lane * PER + j;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(
                block + (value ? kv_v_word(D, token, ch >> 3) : kv_k_word(D, token, ch >> 3)));
            const int nib = value ? ch & 7 : pair_nibble(ch & 7);
            const int c = (w >> (4 * nib)) & 15;
            dst[ch] = narrow(__fmul_rn(s, static_cast<float>(c - z)), a.dtype);
        }
    }
}

template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
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
    const int tasks = a.heads + 2 * a.v.kv_heads;
    a.per_cta = tasks;
    Freqs f;
    for (int i = 0; i < 64; ++i) f.turn[i] = kv->freq[i];
    const dim3 grid(static_cast<unsigned>(a.v.tokens), static_cast<unsigned>((tasks + a.per_cta - 1) / a.per_cta));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = D == 128 ? launch_pdl(kv_append_kernel<4>, grid, kThreads, s, a, f)
                                   : launch_pdl(kv_append_kernel<2>, grid, kThreads, s, a, f);
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
    if ((rc = kv_bind(kv, &a.v, nullptr)) != MRT_OK) return rc;
    a.dtype = dtype;
    a.k = static_cast<uint16_t*>(k_dev);
    a.ldk = ldk;
    a.val = static_cast<uint16_t*>(v_dev);
    a.ldv = ldv;
    const dim3 grid(static_cast<unsigned>(a.v.tokens));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = D == 128 ? launch_pdl(kv_read_kernel<4>, grid, kThreads, s, a)
                                   : launch_pdl(kv_read_kernel<2>, grid, kThreads, s, a);
    return e == cudaSuccess ? MRT_OK : cuda_error(e, "4-bit cache read launch");
}
