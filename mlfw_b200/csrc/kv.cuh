// The key/value cache as the kernels and launchers see it (kv_cache.cu, kv_attention.cu).
#pragma once
#include "common.cuh"
#include "kv_layout.h"

// Behind the opaque handle of the C ABI: geometry and the caller's buffers.  Holds no device memory of its own.
struct b200q_kv_cache {
  b200q_ctx* ctx = nullptr;
  int64_t pages = 0;
  int page_shift = 0, heads = 0, head_dim = 0;
  int8_t *k = nullptr, *v = nullptr;
  float *ks = nullptr, *vs = nullptr;
};

namespace b200q {

// What every call on the cache says about its sequences.
struct KvBatch {
  int B, T;
  const int32_t* page_table;
  int64_t max_pages;
  const int32_t *start, *count;
};

// Workspace of the attention: a counter and an item per block of the largest grid, then two slots per block for pieces of
// items (128 rows of 128 with their sums: 39 MB on 148 SMs).  Its size depends on the GPU only, so a recording never finds it moved.
constexpr int KV_BLOCKS_PER_SM = 2, KV_SLOT_FLOATS = 128 * (128 + 2);
inline size_t kv_item_bytes(const b200q_ctx* ctx) { return (size_t)ctx->sm_count * KV_BLOCKS_PER_SM * 16; }
inline size_t kv_counter_bytes(const b200q_ctx* ctx) { return ((size_t)ctx->sm_count * KV_BLOCKS_PER_SM * sizeof(uint32_t) + 255) & ~size_t(255); }
int kv_workspace(b200q_ctx* ctx);

int launch_kv_append(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* k, const float* v, int64_t ld_k, int64_t ld_v);
int launch_kv_read(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, float* k_out, float* v_out, int64_t ld_k, int64_t ld_v);
int launch_kv_keep(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const int32_t* keep);
int launch_kv_attention(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* q, int64_t ld_q, int H, const uint64_t* tree,
                        float scale, float* out, int64_t ld_o);

}  // namespace b200q
