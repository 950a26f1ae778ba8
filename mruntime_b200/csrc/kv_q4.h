// kv_q4.h -- the paged 4-bit cache: its handle, the device view that kernels
// take, and the layout of a 16-token block (kv_q4.cu, kv_q4_attn.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "mrt_b200.h"

// Opaque handle of the public header.
struct mrt_kv_q4_s {
    int device = -1;
    int64_t pages = 0, page_tokens = 0, kv_heads = 0, head_dim = 0;
    uint8_t* data = nullptr;
    bool rotate = false;
    uint64_t freq[64];  // turns per position, as a fraction of 2^64, of each channel pair
};

namespace mrt {

// Layout.  [page][kv head][block of 16 tokens][block bytes].  A block of 16
// tokens of one head is one contiguous run of 16 (D + 8) bytes:
//
//   K codes   16 rows of D / 2 bytes, a token each: eight channels a word, in
//             the nibble order of pair_nibble().
//   V codes   2 halves (tokens 0-7, 8-15) of 32 lanes (r, c) = (channel
//             stretch, token pair): channels [r D/8, (r + 1) D/8) of tokens
//             2c and 2c + 1, four channels a word, token 2c's in the low half.
//   K scales  16 words: FP16 scale | FP16 zero point << 16.
//   V scales  16 words.
//
// Both orders are those in which the attention kernel's lanes read their MMA
// fragments, so that every shared-memory read is a full conflict-free vector,
// and every row is whole bytes of its own: tokens can be written one at a time.
constexpr int kKvBlock = 16;

__host__ __device__ __forceinline__ int kv_block_bytes(int D) { return kKvBlock * (D + 8); }
__host__ __device__ __forceinline__ int kv_v_codes(int D) { return kKvBlock * D / 2; }
__host__ __device__ __forceinline__ int kv_k_scales(int D) { return kKvBlock * D; }
__host__ __device__ __forceinline__ int kv_v_scales(int D) { return kKvBlock * D + 64; }

// Byte offset in a block of the K word `w` (channels 8w..8w+7) of token t.
__host__ __device__ __forceinline__ int kv_k_word(int D, int t, int w) { return t * (D / 2) + w * 4; }
// The same for V channels 8w..8w+3; those of the next four channels lie four bytes on.
__host__ __device__ __forceinline__ int kv_v_half(int D, int t, int w) {
    const int per = D / 64;  // eights of a stretch
    const int r = w / per, j = w - r * per;
    return kv_v_codes(D) + (t >> 3) * 4 * D + (r * 4 + ((t & 7) >> 1)) * (D / 8) + j * 8 + (t & 1) * 2;
}

// A cache and the sequences of one call, as kernels see them.
struct KvView {
    uint8_t* data;
    int pages, page_tokens, kv_heads, head_dim;
    int seqs, tokens, max_q_len, max_kv_len, ld_table;
    int page_shift;  // log2 of a page's blocks, or -1
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    int* err_flag;
};

// Place, in a sequence's table row, of the page that holds position `pos`.
__device__ __forceinline__ int kv_slot(const KvView& v, int pos) {
    const int block = pos / kKvBlock;
    return v.page_shift >= 0 ? block >> v.page_shift : block / (v.page_tokens / kKvBlock);
}

// Number in the pool of the block of that page that holds it, or -1 when it is
// no page of the cache.
__device__ __forceinline__ int kv_block_in(const KvView& v, int page, int slot, int head, int pos) {
    const int blocks = v.page_tokens / kKvBlock;
    return page < 0 || page >= v.pages ? -1 : (page * v.kv_heads + head) * blocks + (pos / kKvBlock - slot * blocks);
}

// Both for a sequence whose table row is given.
__device__ __forceinline__ int kv_block_number(const KvView& v, const int32_t* row, int head, int pos) {
    const int slot = kv_slot(v, pos);
    return kv_block_in(v, slot < v.ld_table ? row[slot] : -1, slot, head, pos);
}

// The block itself, or null.
__device__ __forceinline__ uint8_t* kv_block_at(const KvView& v, const int32_t* row, int head, int pos) {
    const int n = kv_block_number(v, row, head, pos);
    return n < 0 ? nullptr : v.data + static_cast<int64_t>(n) * kv_block_bytes(v.head_dim);
}

// New tokens and held tokens of sequence b; false (raising the error) when
// they break the call's own bounds.
__device__ __forceinline__ bool kv_seq(const KvView& v, int b, int* first, int* n_new, int* n_held) {
    const int f = v.q_start[b], n = v.q_start[b + 1] - f, kv = v.kv_len[b];
    *first = f;
    *n_new = n;
    *n_held = kv;
    return f >= 0 && n >= 0 && n <= v.max_q_len && f <= v.tokens - n && kv >= 0 && kv <= v.max_kv_len;
}

// Host side: checks of a handle and batch, and the view (no device work).
int kv_view(mrt_kv_q4 kv, const mrt_kv_batch* b, KvView* out);
// The current device's context when it is the handle's; sets view.err_flag.
int kv_bind(mrt_kv_q4 kv, KvView* v, int* sms);

}  // namespace mrt
