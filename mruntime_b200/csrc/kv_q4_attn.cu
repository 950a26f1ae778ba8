// kv_q4_attn.cu -- softmax attention of new tokens' queries over a paged cache
// held in 4 bits (kv_q4.h): the reference's attention op
// (src/core/cpu_backend.cpp:171-290) over such a cache.
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

}  // namespace
}  // namespace mrt

using namespace mrt;

static int check_attention(mrt_kv_q4 kv, const mrt_kv_batch* batch, int64_t heads, KvView* v) {
    const int rc = kv_view(kv, batch, v);
    if (rc != MRT_OK) return rc;
    if (heads <= 0 || heads > 65535 || heads % kv->kv_heads != 0)
        return set_error(MRT_ERR_SHAPE, "heads must be a positive multiple of kv_heads");
    return MRT_OK;
}

extern "C" int mrt_kv_q4_attention_workspace(mrt_kv_q4 kv, const mrt_kv_batch* batch, int64_t heads, size_t* bytes) {
    clear_error();
    if (bytes == nullptr) return set_error(MRT_ERR_INVALID_ARG, "bytes is NULL");
    KvView v{};
    const int rc = check_attention(kv, batch, heads, &v);
    if (rc != MRT_OK) return rc;
    *bytes = 0;
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
    (void)ws_dev;
    (void)ws_bytes;
    a.dtype = dtype;
    a.heads = static_cast<int>(heads);
    a.causal = causal != 0;
    a.scale = scale;
    a.q = static_cast<const uint16_t*>(q_dev);
    a.ldq = ldq;
    a.out = static_cast<uint16_t*>(out_dev);
    a.ldo = ldo;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.v.tokens));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = D == 128 ? cudaLaunchKernelEx(&cfg, attn_q4_rows_kernel<4>, a)
                                   : cudaLaunchKernelEx(&cfg, attn_q4_rows_kernel<2>, a);
    if (e != cudaSuccess) return cuda_error(e, "4-bit attention launch");
    note_launches(1);
    return MRT_OK;
}
