// The paged quantised KV cache: layout and kernel interfaces shared by the
// cache kernels (kv_cache.cu) and the attention that reads it
// (kv_attention.cu).
//
// pages: uint8 [num_pages, kv_heads, page_size / 16, block bytes].  A block is
// 16 tokens of one head, contiguous, so one bulk copy brings it to shared
// memory:
//     16 rows of K | 16 rows of V | 16 fp16 scales of K | 16 fp16 scales of V
// A row is head_dim * bits / 8 bytes (two's complement; int4: low nibble =
// even element); block bytes = 32 * row + 64.
//
// Rows are permuted inside their 16-row part so that the attention kernel's
// shared-memory reads touch every bank once.  It reads K with lane (g, t) =
// (lane / 4, lane % 4) on token g and a quarter of the row chosen by t, and V
// on tokens 2t + {0, 1, 8, 9} and an eighth of the row chosen by g:
//   row >= 128 bytes: 16-byte chunk c of token j lies at chunk c ^ (j & 7);
//   row == 64: tokens 2, 3 (and 6, 7, ...) swap rows, chunk c lies at
//              c ^ 2 for tokens with bit 2 set;
//   row == 32: tokens 4..7 (12..15) swap rows pairwise.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace clb {

constexpr int kKvBlock = 16;  // tokens of a block

__host__ __device__ constexpr int kv_row_bytes(int head_dim, int bits) {
    return head_dim * bits / 8;
}
__host__ __device__ constexpr int kv_block_bytes(int row) { return 2 * kKvBlock * row + 64; }

// Byte offset of byte b of token j's row inside its 16-row part.
template <int kRow>
__host__ __device__ constexpr int kv_offset(int j, int b) {
    static_assert(kRow == 32 || kRow == 64 || kRow == 128 || kRow == 256, "row bytes");
    int row = j, chunk = b >> 4;
    if (kRow >= 128) {
        chunk ^= j & 7;
    } else if (kRow == 64) {
        row = j ^ ((j >> 1) & 1);
        chunk ^= (j >> 1) & 2;
    } else {
        row = j ^ ((j >> 2) & 1);
    }
    return row * kRow + chunk * 16 + (b & 15);
}

// Codes written to the status word of the cache and attention kernels
// (continuing the codes of gemv_common.cuh and gemv_tc.cuh).
constexpr int kStatusKvIndex = 7;      // a page, slot or position lies outside its range
constexpr int kStatusTimeoutKv = 8;    // the attention gave up waiting for a block of the cache

// Element types of q / k / v and of the outputs.
constexpr int kTypeF16 = 0, kTypeBf16 = 1;

struct KvCacheArgs {
    uint8_t* pages;
    const int64_t* slots;  // token -> page * page_size + offset; < 0: skipped
    void* k;               // [tokens, kv_heads, head_dim], written by the read kernel
    void* v;
    int64_t k_token, k_head, v_token, v_head;  // strides in elements
    int64_t tokens, num_pages;
    int kv_heads, head_dim, bits, page_size, type;
};
cudaError_t launch_kv_write(const KvCacheArgs& a, cudaStream_t stream);
cudaError_t launch_kv_read(const KvCacheArgs& a, cudaStream_t stream);

struct QkRopeArgs {
    const void* x[2];   // q, k: [tokens, heads, head_dim]
    void* y[2];
    const void* w[2];   // norm weights [head_dim], both or neither
    int64_t x_token[2], x_head[2], y_token[2], y_head[2];  // strides in elements
    int heads[2];
    const float* table;  // [table_rows, rotary]: rotary / 2 cosines, then the sines
    int64_t table_rows;
    const void* positions;  // int32 or int64 [tokens]
    int positions64;
    int64_t tokens;
    int head_dim, rotary, interleaved, type;
    float eps;
};
cudaError_t launch_qknorm_rope(const QkRopeArgs& a, cudaStream_t stream);

struct KvAttentionArgs {
    const void* q;  // [batch, new, kv_heads * group, head_dim], strides in elements
    int64_t q_batch, q_new, q_head;
    const uint8_t* pages;
    int64_t num_pages;
    const int32_t* table;  // [batch, table_stride]; max_pages entries of each row are readable
    int64_t table_stride;
    int max_pages;
    const int32_t* lengths;  // [batch] tokens in the cache, the new ones included
    int fixed_length;        // >= 0: the length of every sequence (lengths unused)
    int batch, new_tokens, kv_heads, group, head_dim, bits, page_size, type;
    int causal;  // row i of a sequence sees tokens up to length - new + i
    int window;  // > 0: the last `window` of those; below max_pages * page_size
    float scale;
    void* out;        // [batch, new, heads, head_dim] contiguous (type), or null
    float* out_f32;   // the same in fp32 instead (partial results), or null
    float* lse;       // [batch, new, heads] natural log, or null (required with out_f32)
    const float* front;      // fp32 results over tokens in front of these, or null:
    const float* front_lse;  // [front_parts] of them and their lse
    int front_parts;
    int front_by_tensor_cores;  // written by the launch just before (launch_kv_prefix)
    void* workspace;
};
// Workspace bytes of a call (zero-filled before its first use).
size_t kv_attention_workspace();
// Whether the kernel's 32-bit count of blocks holds every length that the page
// table allows.
bool kv_attention_fits(const KvAttentionArgs& a);
// Whether its division by estimates holds the row tiles of a sequence's heads.
bool kv_attention_tiles_fit(const KvAttentionArgs& a);
cudaError_t launch_kv_attention(const KvAttentionArgs& a, cudaStream_t stream);

// Attention of all rows (new_tokens of one sequence) over fixed_length tokens that
// every row sees, on the tensor cores (kv_prefix.cu): whether it is the faster
// kernel for these arguments, the partial results it writes (out_f32 and lse
// hold that many, one after the other), the launch.
bool kv_prefix_takes(const KvAttentionArgs& a);
int kv_prefix_parts(const KvAttentionArgs& a);
cudaError_t launch_kv_prefix(const KvAttentionArgs& a, cudaStream_t stream);
cudaError_t read_kv_prefix_status(int clear, int* status);

// Reads (optionally clears) the status word of the cache kernels.
cudaError_t read_kv_status(int clear, int* status);
cudaError_t read_kv_attention_status(int clear, int* status);
cudaError_t read_qknorm_rope_status(int clear, int* status);

}  // namespace clb
