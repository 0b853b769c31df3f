// Shared by the kernels of the token-paged 8-bit cache.
#pragma once
#include "common.cuh"

namespace magi {

constexpr int kPgMaxEntries = 1024;  // entries of one call
constexpr int kPgMaxPages = (1 << 21) - 2;  // kPgMaxEntries * (kPgMaxPages + 1) fits 32 bits
constexpr int kPgMaxSeqs = 65536;    // rows of a page table

// Device-side view of a magi_token_cache.
struct PagedView {
  int n_layers, n_pages, page_tokens, n_kv_heads, max_seqs, per_row;
  uint8_t* k8;
  uint8_t* v8;
  float* k_scale;
  float* v_scale;
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  int32_t* ws;  // see paged_cache.cu
  int32_t* uses;        // [n_pages]  use * 4 + continued * 2 + written, see paged_cache.cu
  int32_t* k_use;       // [n_layers][n_pages][n_kv_heads]
  int32_t* v_use;
};

// Checks a cache description and fills the view; MAGI_OK or the error that was set on ctx.
int paged_view(magi_ctx* ctx, const magi_token_cache* c, PagedView* v);

inline int* status_word(magi_ctx* ctx) {
  return reinterpret_cast<int*>(reinterpret_cast<char*>(ctx->workspace) + offsetof(PlanHeader, status));
}

// Makes the context's device current for a launch and puts the caller's back.
struct DeviceScope {
  int prev = 0;
  bool moved;
  explicit DeviceScope(const magi_ctx* ctx) {
    cudaGetDevice(&prev);
    moved = prev != ctx->device;
    if (moved) cudaSetDevice(ctx->device);
  }
  ~DeviceScope() {
    if (moved) cudaSetDevice(prev);
  }
};

}  // namespace magi
