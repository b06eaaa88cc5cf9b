// Host side of the language model's serving operators (serve.cu): argument checks and launches.  A failed check
// throws Fail, which the C entries turn into their status and message.
#pragma once

#include <cuda_runtime.h>

#include "../../include/b200diff.h"

namespace b2d {

struct ServeDevice {
    int num_sms;
    int* status;  // the context's device-side status words (StatusWord)
};

void kv_check(const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads);
void kv_append(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int src_type, const void* k,
               const void* v, int64_t row_stride, cudaStream_t st);
void kv_gather(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int dst_type, void* k,
               void* v, int64_t row_stride, cudaStream_t st);
size_t paged_attention_workspace(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads);
void paged_attention(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, bool bf16,
                     const void* q, int64_t q_row, void* o, int64_t o_row, int heads, float scale, int window,
                     void* workspace, size_t workspace_bytes, cudaStream_t st);
// NEOX rotation of the batch's projected rows qkv [rows, (heads + 2 kv_heads) head_dim] (fp32) at their positions, tables
// cos / sin [positions][head_dim / 2]: q rounded to fp16 into q16 [rows, heads x head_dim], k in place.
void rope_rows(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, float* qkv, int heads,
               const float* cos, const float* sin, void* q16, cudaStream_t st);
// Row of each sequence's last new token of x [rows, width] (fp32) -> out [seqs, width]; zeros without new tokens.
void last_rows(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, const float* x, int width,
               float* out, cudaStream_t st);
void sample_tokens(const ServeDevice& dev, const b2d_sample_request* request, cudaStream_t st);

}  // namespace b2d
