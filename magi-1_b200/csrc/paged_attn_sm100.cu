// Attention over the token-paged 8-bit cache.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "paged.cuh"
#include "ptx_sm100.cuh"

namespace magi {
using namespace ptx;

struct PagedAttnKernelParams {
  PagedView c;
  int layer;
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  float* lse;
  const int32_t* seqs;
  const int32_t* cu_q;
  int n, total_q, hq, group, max_q;
  float scale_log2;
  int causal, window;
  int* status;
};

// Plain form: one warp per (query row, head), a lane holds four channels, online softmax in fp32.
__global__ void __launch_bounds__(128) paged_attn_plain_kernel(const PagedAttnKernelParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + warp;
  const int t = (int)(unit / p.hq), head = (int)(unit % p.hq);
  if (t >= p.total_q) return;
  int b = t, row = 0, n_q = 1;
  if (p.cu_q) {
    int lo = 0, hi = p.n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_q[mid] <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
    row = t - p.cu_q[b];
    n_q = p.cu_q[b + 1] - p.cu_q[b];
    if (row < 0 || row >= n_q) return;
  }
  const int seq = p.seqs[b];
  const int P = p.c.page_tokens;
  int len = 0;
  if (seq >= 0 && seq < p.c.max_seqs) len = min(p.c.lens[seq], p.c.per_row * P);
  else if (lane == 0) *p.status = MAGI_E_RANGE;
  const int pos = len - n_q + row;
  const int end = p.causal ? pos + 1 : len, begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int kvh = head / p.group;
  float qv[4];
  const __nv_bfloat16* q = p.q + (int64_t)t * p.q_st + (int64_t)head * p.q_sh + lane * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = __bfloat162float(q[i]);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = begin; k < end; ++k) {
    const int page = p.c.table[(int64_t)seq * p.c.per_row + k / P];
    if (page < 0 || page >= p.c.n_pages) {
      if (lane == 0) *p.status = MAGI_E_RANGE;
      continue;
    }
    const int64_t blk = ((int64_t)p.layer * p.c.n_pages + page) * p.c.n_kv_heads + kvh;
    const int64_t off = (blk * P + k % P) * kHeadDim + lane * 4;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(p.c.k8 + off), vw = *reinterpret_cast<const uint32_t*>(p.c.v8 + off);
    float s = 0.f, vv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half_raw a = __nv_cvt_fp8_to_halfraw((kw >> (8 * i)) & 0xff, __NV_E4M3), c = __nv_cvt_fp8_to_halfraw((vw >> (8 * i)) & 0xff, __NV_E4M3);
      s = fmaf(qv[i], __half2float(*reinterpret_cast<const __half*>(&a)), s);
      vv[i] = __half2float(*reinterpret_cast<const __half*>(&c)) * p.c.v_scale[blk];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.c.k_scale[blk] * p.scale_log2;
    const float m_new = fmaxf(m, s);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref), w = exp2f(s - ref);
    l = l * alpha + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * alpha + w * vv[i];
    m = m_new;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  __nv_bfloat16* o = p.out + (int64_t)t * p.o_st + (int64_t)head * p.o_sh + lane * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __float2bfloat16_rn(acc[i] * inv);
  if (p.lse && lane == 0) p.lse[(int64_t)t * p.hq + head] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace magi

extern "C" int64_t magi_paged_attn_workspace_bytes(magi_ctx* ctx, int32_t max_q, int32_t n_q_heads, int32_t n_kv_heads) { return 16; }

extern "C" int magi_paged_attn_fwd(magi_ctx* ctx, const magi_token_cache* cache, const magi_paged_attn_params* p, void* stream) {
  using namespace magi;
  if (!ctx) return MAGI_E_BADARG;
  PagedAttnKernelParams k = {};
  if (int rc = paged_view(ctx, cache, &k.c)) return rc;
  if (!p || p->struct_size != sizeof(magi_paged_attn_params)) return set_err(ctx, MAGI_E_BADARG, "paged attn: bad struct_size");
  if (p->layer < 0 || p->layer >= k.c.n_layers) return set_err(ctx, MAGI_E_BADARG, "paged attn: no layer %d", p->layer);
  if (p->n < 0 || p->total_q < 0 || p->max_q < 0 || p->n_q_heads <= 0 || p->window < 0)
    return set_err(ctx, MAGI_E_BADARG, "paged attn: negative size");
  if (p->n_q_heads % k.c.n_kv_heads) return set_err(ctx, MAGI_E_BADARG, "paged attn: n_q_heads must be a multiple of the cache's kv heads");
  if (p->n > kPgMaxEntries) return set_err(ctx, MAGI_E_NOMEM, "paged attn: more than %d entries", kPgMaxEntries);
  if (!p->cu_q && (p->max_q != 1 || p->total_q != p->n))
    return set_err(ctx, MAGI_E_BADARG, "paged attn: without cu_q every entry has one query row");
  if (p->n == 0 || p->total_q == 0 || p->max_q == 0) return MAGI_OK;
  if (!p->q || !p->out || !p->seqs || !p->workspace) return set_err(ctx, MAGI_E_BADARG, "paged attn: null tensor");
  if (((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out) | reinterpret_cast<uintptr_t>(p->workspace)) & 15) ||
      ((p->q_stride_t | p->q_stride_h | p->o_stride_t | p->o_stride_h) & 7))
    return set_err(ctx, MAGI_E_ALIGN, "paged attn: q, out and workspace must be 16-byte aligned with strides multiples of 8 elements");
  k.layer = p->layer;
  k.q = static_cast<const __nv_bfloat16*>(p->q);
  k.q_st = p->q_stride_t;
  k.q_sh = p->q_stride_h;
  k.out = static_cast<__nv_bfloat16*>(p->out);
  k.o_st = p->o_stride_t;
  k.o_sh = p->o_stride_h;
  k.lse = p->lse;
  k.seqs = p->seqs;
  k.cu_q = p->cu_q;
  k.n = p->n;
  k.total_q = p->total_q;
  k.max_q = p->max_q;
  k.hq = p->n_q_heads;
  k.group = p->n_q_heads / k.c.n_kv_heads;
  k.scale_log2 = (p->softmax_scale > 0.f ? p->softmax_scale : 1.0f / sqrtf((float)kHeadDim)) * 1.4426950408889634f;
  k.causal = p->causal;
  k.window = p->window;
  k.status = status_word(ctx);
  DeviceScope dev(ctx);
  const int64_t units = (int64_t)p->total_q * p->n_q_heads;
  paged_attn_plain_kernel<<<(unsigned)((units + 3) / 4), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(k);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_err(ctx, MAGI_E_CUDA, "paged attn launch failed: %s", cudaGetErrorString(e));
  return MAGI_OK;
}
