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

// Workspace of the attention: a counter and an item per block (one block per SM), then two slots per block for pieces of items
// (128 rows of 128 and three numbers more in the room of four: 20 MB on 148 SMs).  Its size depends on the GPU only, so a recording never finds it moved.
constexpr int KV_SLOT_FLOATS = 128 * (128 + 4);
inline size_t kv_item_bytes(const b200q_ctx* ctx) { return (size_t)ctx->sm_count * 16; }
inline size_t kv_counter_bytes(const b200q_ctx* ctx) { return ((size_t)ctx->sm_count * sizeof(uint32_t) + 255) & ~size_t(255); }
int kv_workspace(b200q_ctx* ctx);

// The calls on a cache follow one another within microseconds (append, attention, keep), so each kernel is launched as a
// programmatic dependent of the one before it: its blocks come while that one drains, and kv_after_previous holds back
// everything until it has completed.  With profiling on, an event sits between the two and the overlap is off.
// A block may thus be resident while kernels two or three back still write what it is going to read (codes, scales, queries,
// page tables, rows to keep): none of that is read-only for the lifetime of the kernel, so it is loaded with coherent loads
// (plain or __ldcg; L2 is where the writers' stores are) and never through __ldg or a const __restrict__ pointer.
#ifdef __CUDACC__
__device__ __forceinline__ void kv_after_previous() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
int kv_launch(b200q_ctx* ctx, void (*kernel)(P...), dim3 grid, int threads, size_t smem, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->profiling ? 0 : 1;
  B200Q_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
  ctx->launches++;
  return 0;
}
#endif

int launch_kv_append(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* k, const float* v, int64_t ld_k, int64_t ld_v);
int launch_kv_read(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, float* k_out, float* v_out, int64_t ld_k, int64_t ld_v);
int launch_kv_keep(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const int32_t* keep);
int launch_kv_attention(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* q, int64_t ld_q, int H, const uint64_t* tree,
                        float scale, float* out, int64_t ld_o);

}  // namespace b200q
