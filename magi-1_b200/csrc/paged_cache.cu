// Token-paged 8-bit cache: quantised append and page book-keeping, all of it on the device.
//
// A page of one layer holds page_tokens tokens as [kv head][token][128] e4m3 codes of K and of V, with one power-of-two
// scale per head.  A power of two costs an 8-bit float no precision, divides without rounding, and lets a page whose range
// grows be re-quantised without a second rounding error except at the subnormal end of e4m3.
//
// Book-keeping: a call first runs one block that checks every entry and picks the pages (reserve, branch, compact), so that
// it can be refused as a whole, and then, where pages have to be moved, a grid that copies them.  Free pages are those with
// a reference count of zero, lowest number first, so the same calls give the same tables every time.  They are looked for from page
// 0 on by that one block: a page for one sequence takes 5 us in a pool of 1000, 34 us behind 10^5 pages in use, 300 us behind 10^6.
//
// A page that changes hands keeps its old scale until something is written to it.  Each time reserve takes a page it counts a use
// of it (page_uses), and the scale of a (layer, page, head), K and V apart, carries the use that it was set in (scale_uses): where
// the two differ the page is still empty in that layer, and append takes the scale that the new tokens need.  So a reservation can
// be appended in parts, and reserve writes one number per page instead of a scale per layer and head.  Tokens in front of a later
// reservation count as there in every layer, once the page has been written to in one: hence two bits beside the count.
//
// workspace (int32): [0] number of moves, [1] 1 = the call was accepted, [4 .. 4 + n_pages) source of each move,
// [4 + n_pages .. 4 + 2 n_pages) its destination, [4 + 2 n_pages .. 4 + 3 n_pages) new number of a moved page.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "paged.cuh"

namespace magi {

constexpr int kPlanThreads = 1024;
constexpr int kStrip = 16;  // reference counts a planning thread looks at per step
constexpr int kMinExp = -60, kMaxExp = 60;

__device__ __forceinline__ int pages_of(int64_t tokens, int page_tokens) { return (int)((tokens + page_tokens - 1) / page_tokens); }

// Exclusive prefix sum over the block (1024 threads); *total gets the sum.  Ends with a barrier.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += y;
  }
  const int before = warp == 0 ? 0 : __shfl_sync(0xffffffffu, w, warp - 1);
  *total = __shfl_sync(0xffffffffu, w, 31);
  __syncthreads();
  return before + x - v;
}

// The 16 counts [i, i + 16) as a bit mask of those that are > 0 (beyond n: neither).
__device__ __forceinline__ uint32_t live_mask(const int32_t* refs, int64_t i, int n, uint32_t* valid) {
  uint32_t m = 0, ok = 0;
#pragma unroll
  for (int k = 0; k < kStrip; ++k)
    if (i + k < n) {
      ok |= 1u << k;
      if (refs[i + k] > 0) m |= 1u << k;
    }
  *valid = ok;
  return m;
}

// Writes the numbers of the first `need` free pages to ids; returns how many there are (<= need).  Whole block.
__device__ int find_free(const int32_t* refs, int n_pages, int need, int32_t* ids, int* warp_sums) {
  int found = 0;
  for (int64_t base = 0; base < n_pages && found < need; base += (int64_t)kPlanThreads * kStrip) {
    const int64_t i = base + (int64_t)threadIdx.x * kStrip;
    uint32_t valid;
    const uint32_t live = live_mask(refs, i, n_pages, &valid);
    uint32_t free_bits = valid & ~live;
    int total;
    int at = found + block_scan(__popc(free_bits), warp_sums, &total);
    while (free_bits && at < need) {
      ids[at++] = (int32_t)(i + __ffs(free_bits) - 1);
      free_bits &= free_bits - 1;
    }
    found += total;
  }
  __syncthreads();
  return found < need ? found : need;
}

constexpr int kWritten = 1, kContinued = 2;  // page_uses: use * 4 and these
__device__ __forceinline__ int next_use(int uses) { return (int)(((uint32_t)uses & ~3u) + 4u); }  // may wrap: it is only compared

// ------------------------------------------------------------------------------------------------ reserve
__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(const PagedView c, const int32_t* __restrict__ seqs,
                                                               const int32_t* __restrict__ n_new, int n, int32_t* __restrict__ starts,
                                                               int* status) {
  __shared__ uint32_t named[kPgMaxSeqs / 32];
  __shared__ int prefix[kPlanThreads + 1];
  __shared__ int warp_sums[32];
  const int i = threadIdx.x;
  for (int w = i; w < (c.max_seqs + 31) / 32; w += kPlanThreads) named[w] = 0;
  __syncthreads();
  int seq = 0, len = 0, add = 0, need = 0, tail = -1;
  bool bad = false;
  if (i < n) {
    seq = seqs[i];
    add = n_new[i];
    bad = seq < 0 || seq >= c.max_seqs || add < 0;
    if (!bad) {
      bad = atomicOr(&named[seq >> 5], 1u << (seq & 31)) >> (seq & 31) & 1u;
      len = c.lens[seq];
      bad = bad || len < 0 || (int64_t)len + add > (int64_t)c.per_row * c.page_tokens || (int64_t)len + add > INT32_MAX;
    }
    if (!bad) {
      // more than there are is as good as one more than there are (and keeps the sum over the entries within 32 bits)
      need = min(pages_of((int64_t)len + add, c.page_tokens) - pages_of(len, c.page_tokens), c.n_pages + 1);
      if (add > 0 && len % c.page_tokens) {  // the page that is continued must be this sequence's alone
        tail = c.table[(int64_t)seq * c.per_row + len / c.page_tokens];
        bad = tail < 0 || tail >= c.n_pages || c.refs[tail] != 1;
      }
    }
  }
  int refuse = __syncthreads_or(bad) ? MAGI_E_RANGE : 0;
  int total = 0;
  const int before = block_scan(need, warp_sums, &total);
  prefix[i] = before;
  if (i == 0) prefix[kPlanThreads] = total;
  __syncthreads();
  int32_t* ids = c.ws + 4;
  if (!refuse && total > 0) {
    if (total > c.n_pages || find_free(c.refs, c.n_pages, total, ids, warp_sums) < total) refuse = MAGI_E_NOMEM;
  }
  if (refuse) {
    if (i == 0) *status = refuse;
    if (i < n) starts[i] = -1;
    return;
  }
  if (i < n) {
    starts[i] = len;
    c.lens[seq] = len + add;
    if (tail >= 0 && c.uses[tail] & kWritten) c.uses[tail] |= kContinued;
    // few pages each (one at most for a token): the entry's own thread places them
    if (need <= 4)
      for (int k = 0; k < need; ++k) {
        const int id = ids[before + k];
        c.table[(int64_t)seq * c.per_row + pages_of(len, c.page_tokens) + k] = id;
        c.refs[id] = 1;
        c.uses[id] = next_use(c.uses[id]);
      }
  }
  if (!__syncthreads_or(need > 4)) return;
  // prompts: the block walks over all pages, each finds its entry
  for (int k = i; k < total; k += kPlanThreads) {
    int lo = 0, hi = n;  // prefix[lo] <= k < prefix[hi] (entries without pages have equal prefixes)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= k) lo = mid;
      else hi = mid;
    }
    const int s = seqs[lo];
    const int new_len = starts[lo] + n_new[lo];
    const int last = pages_of(new_len, c.page_tokens);              // pages of the sequence from now on
    const int taken = (lo + 1 < kPlanThreads ? prefix[lo + 1] : total) - prefix[lo];
    if (taken <= 4) continue;                                        // placed above
    const int id = ids[k];
    c.table[(int64_t)s * c.per_row + last - taken + k - prefix[lo]] = id;
    c.refs[id] = 1;
    c.uses[id] = next_use(c.uses[id]);
  }
}

// ------------------------------------------------------------------------------------------------ fork / copy
// Checks, picks the new pages and lists the page copies.
__global__ void __launch_bounds__(kPlanThreads) branch_plan_kernel(const PagedView c, const int32_t* __restrict__ src,
                                                                   const int32_t* __restrict__ dst, int n, int share, int* status) {
  __shared__ uint32_t named[kPgMaxSeqs / 32];
  __shared__ int prefix[kPlanThreads + 1];
  __shared__ int first[kPlanThreads];  // first own page of the entry
  __shared__ int warp_sums[32];
  const int i = threadIdx.x;
  for (int w = i; w < (c.max_seqs + 31) / 32; w += kPlanThreads) named[w] = 0;
  __syncthreads();
  int s = 0, d = 0, len = 0, need = 0;
  bool bad = false;
  if (i < n) {
    s = src[i];
    d = dst[i];
    bad = s < 0 || s >= c.max_seqs || d < 0 || d >= c.max_seqs;
    if (!bad) {
      bad = atomicOr(&named[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u;
      len = c.lens[s];
      bad = bad || c.lens[d] != 0 || len < 0 || len > (int64_t)c.per_row * c.page_tokens;
    }
  }
  __syncthreads();
  if (i < n && !bad) bad = named[s >> 5] >> (s & 31) & 1u;  // a source that this call fills
  if (i < n && !bad) {
    const int used = pages_of(len, c.page_tokens);
    first[i] = share ? len / c.page_tokens : 0;
    need = min(used - first[i], c.n_pages + 1);
  }
  int refuse = __syncthreads_or(bad) ? MAGI_E_RANGE : 0;
  // the pages that are about to be shared or copied have to exist
  if (!refuse) {
    bool broken = false;
    for (int e = i >> 5; e < n; e += kPlanThreads / 32) {
      const int se = src[e], used = pages_of(c.lens[se], c.page_tokens);
      for (int p = i & 31; p < used; p += 32) {
        const int id = c.table[(int64_t)se * c.per_row + p];
        broken = broken || id < 0 || id >= c.n_pages;
      }
    }
    if (__syncthreads_or(broken)) refuse = MAGI_E_RANGE;
  }
  int total = 0;
  const int before = block_scan(need, warp_sums, &total);
  prefix[i] = before;
  __syncthreads();
  int32_t* from = c.ws + 4;
  int32_t* to = from + c.n_pages;
  if (!refuse && total > 0) {
    if (total > c.n_pages || find_free(c.refs, c.n_pages, total, to, warp_sums) < total) refuse = MAGI_E_NOMEM;
  }
  if (i == 0) {
    if (refuse) *status = refuse;
    c.ws[0] = refuse ? 0 : total;
    c.ws[1] = refuse ? 0 : 1;
  }
  if (refuse) return;
  for (int k = i; k < total; k += kPlanThreads) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= k) lo = mid;
      else hi = mid;
    }
    const int slot = first[lo] + k - prefix[lo];
    from[k] = c.table[(int64_t)src[lo] * c.per_row + slot];
    c.table[(int64_t)dst[lo] * c.per_row + slot] = to[k];
    c.refs[to[k]] = 1;
  }
}

// ------------------------------------------------------------------------------------------------ compact
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagedView c) {
  __shared__ int warp_sums[32];
  int32_t* from = c.ws + 4;
  int32_t* to = from + c.n_pages;
  int32_t* renamed = to + c.n_pages;
  constexpr int64_t kStep = (int64_t)kPlanThreads * kStrip;
  int live_pages = 0;
  {
    int mine = 0, total;
    for (int64_t base = 0; base < c.n_pages; base += kStep) {
      uint32_t valid;
      mine += __popc(live_mask(c.refs, base + (int64_t)threadIdx.x * kStrip, c.n_pages, &valid));
    }
    block_scan(mine, warp_sums, &total);
    live_pages = total;
  }
  int holes = 0, movers = 0;
  for (int64_t base = 0; base < c.n_pages; base += kStep) {
    const int64_t i = base + (int64_t)threadIdx.x * kStrip;
    uint32_t valid;
    const uint32_t live = live_mask(c.refs, i, c.n_pages, &valid);
    const int64_t below = live_pages - i;
    const uint32_t low = below <= 0 ? 0u : below >= kStrip ? 0xffffu : (1u << below) - 1u;
    uint32_t hole = valid & ~live & low, mover = live & ~low;
    // both counts in one scan: a strip holds at most 2^14 of each
    int total;
    const int both = block_scan(__popc(hole) | (__popc(mover) << 16), warp_sums, &total);
    int ah = holes + (both & 0xffff), am = movers + (both >> 16);
    while (hole) {
      to[ah++] = (int32_t)(i + __ffs(hole) - 1);
      hole &= hole - 1;
    }
    while (mover) {
      from[am++] = (int32_t)(i + __ffs(mover) - 1);
      mover &= mover - 1;
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __syncthreads();  // holes == movers
  for (int k = threadIdx.x; k < movers; k += kPlanThreads) {
    renamed[from[k]] = to[k];
    c.refs[to[k]] = c.refs[from[k]];
    c.refs[from[k]] = 0;
  }
  if (threadIdx.x == 0) {
    c.ws[0] = movers;
    c.ws[1] = live_pages;
  }
}

// ------------------------------------------------------------------------------------------------ page copies
constexpr int kMoveThreads = 256;
constexpr int kMoveBytes = kMoveThreads * 16 * 4;  // 16 KB per step: four 16-byte loads in flight per thread

// Copies the listed pages, codes and scales, in every layer: a step of the grid-strided loop is up to 16 KB of one page of
// one layer of K or V.  The moves come from the workspace, so the host need not know how many there are.  297 MB: 97 us,
// 6.1 TB/s read and written.
__device__ void move_pages(const PagedView& c) {
  const int n_moves = c.ws[0];
  const int32_t* from = c.ws + 4;
  const int32_t* to = from + c.n_pages;
  const int64_t page_bytes = (int64_t)c.n_kv_heads * c.page_tokens * kHeadDim;
  const int steps = (int)((page_bytes + kMoveBytes - 1) / kMoveBytes);
  // scales, and whether they count: a page is as written, or as empty, as the one it comes from
  const int64_t scales = (int64_t)n_moves * 2 * c.n_layers * c.n_kv_heads;
  for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < scales; i += (int64_t)gridDim.x * kMoveThreads) {
    const int h = (int)(i % c.n_kv_heads);
    int64_t r = i / c.n_kv_heads;
    const bool kv = r & 1;
    r >>= 1;
    const int layer = (int)(r % c.n_layers), k = (int)(r / c.n_layers);
    const int64_t s = ((int64_t)layer * c.n_pages + from[k]) * c.n_kv_heads + h, d = ((int64_t)layer * c.n_pages + to[k]) * c.n_kv_heads + h;
    float* scale = kv ? c.v_scale : c.k_scale;
    int32_t* use = kv ? c.v_use : c.k_use;
    const int uses_s = c.uses[from[k]], use_d = c.uses[to[k]] >> 2;
    scale[d] = scale[s];
    use[d] = use[s] == uses_s >> 2 ? use_d : use_d - 1;
    if (layer == 0 && !kv && h == 0) c.uses[to[k]] = use_d << 2 | (uses_s & 3);  // the use itself stays, which others read
  }
  const int64_t total = (int64_t)n_moves * c.n_layers * 2 * steps;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int step = (int)(u % steps);
    int64_t r = u / steps;
    const int kv = (int)(r & 1);
    r >>= 1;
    const int layer = (int)(r % c.n_layers);
    const int k = (int)(r / c.n_layers);
    const int64_t ps = (int64_t)layer * c.n_pages + from[k], pd = (int64_t)layer * c.n_pages + to[k];
    uint8_t* pool = kv ? c.v8 : c.k8;
    const uint4* s = reinterpret_cast<const uint4*>(pool + ps * page_bytes) + (int64_t)step * (kMoveBytes / 16);
    uint4* d = reinterpret_cast<uint4*>(pool + pd * page_bytes) + (int64_t)step * (kMoveBytes / 16);
    const int left = (int)(page_bytes / 16 - (int64_t)step * (kMoveBytes / 16));
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((int)threadIdx.x + j * kMoveThreads < left) v[j] = s[threadIdx.x + j * kMoveThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((int)threadIdx.x + j * kMoveThreads < left) d[threadIdx.x + j * kMoveThreads] = v[j];
  }
}

__global__ void __launch_bounds__(kMoveThreads) branch_apply_kernel(const PagedView c, const int32_t* __restrict__ src,
                                                                    const int32_t* __restrict__ dst, int n, int share) {
  if (!c.ws[1]) return;
  for (int e = blockIdx.x; e < n; e += gridDim.x) {
    const int s = src[e], d = dst[e], len = c.lens[s];
    if (share)
      for (int p = threadIdx.x; p < len / c.page_tokens; p += kMoveThreads) {
        const int id = c.table[(int64_t)s * c.per_row + p];
        c.table[(int64_t)d * c.per_row + p] = id;
        atomicAdd(&c.refs[id], 1);
      }
    if (threadIdx.x == 0) c.lens[d] = len;
  }
  move_pages(c);
}

__global__ void __launch_bounds__(kMoveThreads) compact_apply_kernel(const PagedView c) {
  const int live_pages = c.ws[1];
  if (c.ws[0] == 0) return;
  const int32_t* renamed = c.ws + 4 + 2 * (int64_t)c.n_pages;
  const int64_t cells = (int64_t)c.max_seqs * c.per_row;
  for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < cells; i += (int64_t)gridDim.x * kMoveThreads) {
    const int id = c.table[i];
    if (id >= live_pages && id < c.n_pages) c.table[i] = renamed[id];
  }
  move_pages(c);
}

// ------------------------------------------------------------------------------------------------ free
// One block per entry; every block checks the whole list, so that the call is refused by all of them or by none.
__global__ void __launch_bounds__(256) free_kernel(const PagedView c, const int32_t* __restrict__ seqs, int n, int* status) {
  __shared__ uint32_t named[kPgMaxSeqs / 32];
  for (int w = threadIdx.x; w < (c.max_seqs + 31) / 32; w += blockDim.x) named[w] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = seqs[i];
    if (s < 0 || s >= c.max_seqs) bad = true;
    else bad = bad || (atomicOr(&named[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u);
  }
  if (__syncthreads_or(bad)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *status = MAGI_E_RANGE;
    return;
  }
  const int seq = seqs[blockIdx.x];
  int32_t* row = c.table + (int64_t)seq * c.per_row;
  for (int p = threadIdx.x; p < c.per_row; p += blockDim.x) {
    const int id = row[p];
    if (id >= 0 && id < c.n_pages) atomicSub(&c.refs[id], 1);
    row[p] = -1;
  }
  if (threadIdx.x == 0) c.lens[seq] = 0;
}

// ------------------------------------------------------------------------------------------------ append
struct AppendParams {
  const __nv_bfloat16* x[2];  // K, V
  int64_t st[2], sh[2];
  const int32_t* seqs;
  const int32_t* starts;
  const int32_t* cu;
  int n, max_new, total, layer;
};

// Exponent of the smallest power of two that keeps `amax` within e4m3's 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return amax > 0.f ? min(max(e, kMinExp), kMaxExp) : kMinExp;
}

__device__ __forceinline__ uint2 pack8_e4m3(const float* f) {
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * k], f[4 * k + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * k + 2], f[4 * k + 3]), __NV_SATFINITE, __NV_E4M3);
    w[k] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// One block per (page that an entry touches, kv head, entry, K or V), heads next to each other, as their rows lie in memory:
// 256 threads, thread = (row group, 8 channels); the page's new tokens stay in registers between the search for the largest
// value and the conversion, so HBM sees one read and one half-size write.  Tokens that the page holds already are read only
// when its scale grows.  What a block has to look up is asked for as early as its address is known - entry; length, page and
// new tokens; references and scale - because for one token these three trips to memory are the whole time (64 sequences:
// 6.2 us; 12.3 one after the other).  Prompts are bound by HBM and issue slots: 2001 to 21600 tokens 63.5 us, 5.2 TB/s (74 us
// with the maximum taken one value at a time, 88 with pages instead of heads next to each other in the grid).
// kSlots: new tokens of a page that a thread takes, 16 apart (1 when a call has at most 16 per entry: fewer registers, so
// that more blocks of a batch are resident at once).
template <int kSlots>
__global__ void __launch_bounds__(256, 5) paged_append_kernel(const PagedView c, const AppendParams p, int page_shift, int* status) {
  const int entry = blockIdx.y >> 1;
  const bool kv = blockIdx.y & 1;
  const int nth = blockIdx.x / c.n_kv_heads, head = blockIdx.x - nth * c.n_kv_heads;
  const int start = p.starts[entry], seq = p.seqs[entry];
  const int row0 = p.cu ? p.cu[entry] : entry;
  const int count = p.cu ? p.cu[entry + 1] - row0 : 1;
  if (start < 0 || count == 0) return;
  const int P = c.page_tokens, slot = (start >> page_shift) + nth;
  if (nth > 0 && slot > (start + (int64_t)count - 1) >> page_shift) return;
  bool bad = count < 0 || count > p.max_new || row0 < 0 || (int64_t)row0 + count > p.total || seq < 0 || seq >= c.max_seqs ||
             slot >= c.per_row;
  const int len = bad ? -1 : c.lens[seq];
  const int page = bad ? -1 : c.table[(int64_t)seq * c.per_row + slot];
  const int base = slot << page_shift;                // position of the page's first token
  const int lo = max(start, base) - base;             // new tokens: rows [lo, hi) of the page
  const int hi = bad ? lo : (int)min((int64_t)start + count - base, (int64_t)P);
  const int64_t st = kv ? p.st[1] : p.st[0];
  // row r of the page: x + r * st
  const __nv_bfloat16* x = (kv ? p.x[1] : p.x[0]) + ((int64_t)row0 + base - start) * st + (int64_t)head * (kv ? p.sh[1] : p.sh[0]);
  const int col = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4;
  const int first = kSlots == 1 ? lo : 0;
  uint4 v[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int r = first + r0 + i * 16;
    v[i] = make_uint4(0, 0, 0, 0);
    if (r >= lo && r < hi) v[i] = __ldg(reinterpret_cast<const uint4*>(x + (int64_t)r * st + col));
  }
  bad = bad || (int64_t)start + count > len || len > (int64_t)c.per_row << page_shift || page < 0 || page >= c.n_pages;
  const int64_t block = ((int64_t)p.layer * c.n_pages + (bad ? 0 : page)) * c.n_kv_heads + head;
  float* scale = (kv ? c.v_scale : c.k_scale) + block;
  int32_t* scale_use = (kv ? c.v_use : c.k_use) + block;
  uint8_t* codes = (kv ? c.v8 : c.k8) + block * P * kHeadDim;
  const int refs = bad ? 0 : c.refs[page];
  const int uses = bad ? 0 : c.uses[page], use = uses >> 2, set_in = *scale_use;
  const float stored = *scale;
  // largest finite magnitude, as bits: two at a time, and one by one only where some are not finite
  uint32_t tops = 0;
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    tops = __vmaxu2(__vmaxu2(__vmaxu2(tops, v[i].x & 0x7fff7fffu), v[i].y & 0x7fff7fffu),
                    __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
  uint32_t top = max(tops & 0xffffu, tops >> 16);
  if (top >= 0x7f80u) {
    top = 0;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a = w[k] & 0x7fffu, b = w[k] >> 16 & 0x7fffu;
        if (a < 0x7f80u) top = max(top, a);
        if (b < 0x7f80u) top = max(top, b);
      }
    }
  }
  __syncwarp();
  __shared__ uint32_t s_top[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  if (refs != 1) {  // none, or others that share it
    if (threadIdx.x == 0) *status = MAGI_E_RANGE;
    return;
  }
  const int held = min(len - base, P);                // tokens of the sequence in the page, new ones included
  // Tokens beside the new ones.  An empty page has none, reserved or not, but for those that an earlier reservation covers.
  const bool others = set_in == use ? lo > 0 || hi < held : lo > 0 && uses & kContinued;
  const float before = others ? stored : 0.f;
  __syncthreads();  // every thread has read the scale and its use before one of them replaces them
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, s_top[i]);
  const int e = scale_exponent(__uint_as_float(top << 16));
  const float needed = __uint_as_float((uint32_t)(e + 127) << 23);
  const float after = fmaxf(before, needed);
  // both are powers of two, unless the caller's memory says otherwise: then the quotient is rounded once
  const float inv = __frcp_rn(after);
  if (threadIdx.x == 0) {
    if (after != before) *scale = after;
    if (set_in != use) *scale_use = use;
    if (!(uses & kWritten) && head == 0 && !kv) atomicOr(&c.uses[page], kWritten);
  }
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int r = first + r0 + i * 16;
    if (r < lo || r >= hi) continue;
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16) * inv;
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u) * inv;
    }
    *reinterpret_cast<uint2*>(codes + r * kHeadDim + col) = pack8_e4m3(f);
  }
  if (others && after != before) {
    const float ratio = before * inv;
#pragma unroll 1
    for (int rb = r0; rb < held; rb += 64) {
      uint2 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = rb + i * 16;
        if (r < held && (r < lo || r >= hi)) raw[i] = *reinterpret_cast<const uint2*>(codes + r * kHeadDim + col);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = rb + i * 16;
        if (r >= held || (r >= lo && r < hi)) continue;
        const uint8_t* b = reinterpret_cast<const uint8_t*>(&raw[i]);
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const __half_raw hr = __nv_cvt_fp8_to_halfraw(b[k], __NV_E4M3);
          f[k] = __half2float(*reinterpret_cast<const __half*>(&hr)) * ratio;
        }
        *reinterpret_cast<uint2*>(codes + r * kHeadDim + col) = pack8_e4m3(f);
      }
    }
  }
}

int paged_view(magi_ctx* ctx, const magi_token_cache* c, PagedView* v) {
  if (!c || c->struct_size != sizeof(magi_token_cache)) return set_err(ctx, MAGI_E_BADARG, "token cache: bad struct_size");
  if (c->n_layers <= 0 || c->n_pages <= 0 || c->n_kv_heads <= 0 || c->max_seqs <= 0 || c->max_pages_per_seq <= 0)
    return set_err(ctx, MAGI_E_BADARG, "token cache: sizes must be positive");
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return set_err(ctx, MAGI_E_BADARG, "token cache: page_tokens must be 16, 32, 64 or 128, got %d", c->page_tokens);
  if (c->max_seqs > kPgMaxSeqs) return set_err(ctx, MAGI_E_NOMEM, "token cache: more than %d sequences", kPgMaxSeqs);
  if (c->n_pages > kPgMaxPages) return set_err(ctx, MAGI_E_NOMEM, "token cache: more than %d pages", kPgMaxPages);
  if (c->n_kv_heads > 65535) return set_err(ctx, MAGI_E_BADARG, "token cache: too many heads");
  if ((int64_t)c->max_pages_per_seq * c->page_tokens > INT32_MAX)
    return set_err(ctx, MAGI_E_NOMEM, "token cache: a sequence of max_pages_per_seq pages exceeds 2^31 tokens");
  if ((int64_t)c->n_layers * c->n_pages * c->n_kv_heads * c->page_tokens > INT32_MAX)
    return set_err(ctx, MAGI_E_NOMEM, "token cache: more than 2^31 rows of 128 bytes");
  if (!c->k8 || !c->v8 || !c->k_scale || !c->v_scale || !c->page_table || !c->seq_lens || !c->page_refs || !c->workspace)
    return set_err(ctx, MAGI_E_BADARG, "token cache: null tensor");
  if ((reinterpret_cast<uintptr_t>(c->k8) | reinterpret_cast<uintptr_t>(c->v8) | reinterpret_cast<uintptr_t>(c->workspace)) & 15)
    return set_err(ctx, MAGI_E_ALIGN, "token cache: k8, v8 and workspace must be 16-byte aligned");
  *v = {c->n_layers, c->n_pages, c->page_tokens, c->n_kv_heads, c->max_seqs, c->max_pages_per_seq,
        static_cast<uint8_t*>(c->k8), static_cast<uint8_t*>(c->v8), c->k_scale, c->v_scale,
        c->page_table, c->seq_lens, c->page_refs, static_cast<int32_t*>(c->workspace), c->page_uses, c->scale_uses,
        c->scale_uses ? c->scale_uses + (int64_t)c->n_layers * c->n_pages * c->n_kv_heads : nullptr};
  return MAGI_OK;
}

static int check_uses(magi_ctx* ctx, const PagedView& v) {
  return v.uses && v.k_use ? MAGI_OK : set_err(ctx, MAGI_E_BADARG, "token cache: null page_uses or scale_uses");
}

static int check_entries(magi_ctx* ctx, const void* a, const void* b, int n, const char* what) {
  if (n < 0 || (n > 0 && (!a || !b))) return set_err(ctx, MAGI_E_BADARG, "%s: null index array or negative count", what);
  if (n > kPgMaxEntries) return set_err(ctx, MAGI_E_NOMEM, "%s: more than %d entries", what, kPgMaxEntries);
  return MAGI_OK;
}

static int launched(magi_ctx* ctx, const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_err(ctx, MAGI_E_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return MAGI_OK;
}

}  // namespace magi

using namespace magi;

extern "C" int64_t magi_token_cache_workspace_bytes(int32_t n_pages) { return n_pages > 0 ? 16 + 12 * (int64_t)n_pages : 0; }

extern "C" int magi_token_cache_reserve(magi_ctx* ctx, const magi_token_cache* cache, const int32_t* seqs, const int32_t* n_new,
                                        int n, int32_t* starts, void* stream) {
  if (!ctx) return MAGI_E_BADARG;
  PagedView v;
  if (int rc = paged_view(ctx, cache, &v)) return rc;
  if (int rc = check_entries(ctx, seqs, n_new, n, "token cache reserve")) return rc;
  if (n == 0) return MAGI_OK;
  if (!starts) return set_err(ctx, MAGI_E_BADARG, "token cache reserve: null starts");
  if (int rc = check_uses(ctx, v)) return rc;
  DeviceScope dev(ctx);
  reserve_kernel<<<1, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(v, seqs, n_new, n, starts, status_word(ctx));
  return launched(ctx, "token cache reserve");
}

extern "C" int magi_token_cache_append(magi_ctx* ctx, const magi_token_cache* cache, int layer, const int32_t* seqs,
                                       const int32_t* starts, const int32_t* cu_new, int n, int max_new, int total_new,
                                       const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                       int64_t v_stride_h, void* stream) {
  if (!ctx) return MAGI_E_BADARG;
  PagedView view;
  if (int rc = paged_view(ctx, cache, &view)) return rc;
  if (int rc = check_entries(ctx, seqs, starts, n, "token cache append")) return rc;
  if (layer < 0 || layer >= view.n_layers) return set_err(ctx, MAGI_E_BADARG, "token cache append: no layer %d", layer);
  if (max_new < 0 || total_new < 0) return set_err(ctx, MAGI_E_BADARG, "token cache append: negative size");
  if (!cu_new && (max_new != 1 || total_new != n))
    return set_err(ctx, MAGI_E_BADARG, "token cache append: without cu_new every entry has one token");
  if (n == 0 || max_new == 0 || total_new == 0) return MAGI_OK;
  if (!k || !v) return set_err(ctx, MAGI_E_BADARG, "token cache append: null k or v");
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) || ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7))
    return set_err(ctx, MAGI_E_ALIGN, "token cache append: k and v must be 16-byte aligned with strides multiples of 8 elements");
  if (int rc = check_uses(ctx, view)) return rc;
  AppendParams p = {{static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v)}, {k_stride_t, v_stride_t},
                    {k_stride_h, v_stride_h}, seqs, starts, cu_new, n, max_new, total_new, layer};
  // pages that max_new tokens can touch, no more than a sequence can hold
  int64_t slots = ((int64_t)max_new + view.page_tokens - 2) / view.page_tokens + 1;
  slots = std::min<int64_t>(slots, std::min(view.per_row, view.n_pages));
  const int shift = __builtin_ctz(view.page_tokens);
  const dim3 grid((unsigned)(slots * view.n_kv_heads), 2 * n);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  DeviceScope dev(ctx);
  if (max_new <= 16) paged_append_kernel<1><<<grid, 256, 0, st>>>(view, p, shift, status_word(ctx));
  else paged_append_kernel<8><<<grid, 256, 0, st>>>(view, p, shift, status_word(ctx));
  return launched(ctx, "token cache append");
}

extern "C" int magi_token_cache_branch(magi_ctx* ctx, const magi_token_cache* cache, const int32_t* src, const int32_t* dst, int n,
                                       int share, void* stream) {
  if (!ctx) return MAGI_E_BADARG;
  PagedView v;
  if (int rc = paged_view(ctx, cache, &v)) return rc;
  if (int rc = check_entries(ctx, src, dst, n, "token cache branch")) return rc;
  if (n == 0) return MAGI_OK;
  if (int rc = check_uses(ctx, v)) return rc;
  DeviceScope dev(ctx);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  branch_plan_kernel<<<1, kPlanThreads, 0, st>>>(v, src, dst, n, share, status_word(ctx));
  branch_apply_kernel<<<ctx->sm_count * 8, kMoveThreads, 0, st>>>(v, src, dst, n, share);
  return launched(ctx, "token cache branch");
}

extern "C" int magi_token_cache_free(magi_ctx* ctx, const magi_token_cache* cache, const int32_t* seqs, int n, void* stream) {
  if (!ctx) return MAGI_E_BADARG;
  PagedView v;
  if (int rc = paged_view(ctx, cache, &v)) return rc;
  if (int rc = check_entries(ctx, seqs, seqs, n, "token cache free")) return rc;
  if (n == 0) return MAGI_OK;
  DeviceScope dev(ctx);
  free_kernel<<<n, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(v, seqs, n, status_word(ctx));
  return launched(ctx, "token cache free");
}

extern "C" int magi_token_cache_compact(magi_ctx* ctx, const magi_token_cache* cache, void* stream) {
  if (!ctx) return MAGI_E_BADARG;
  PagedView v;
  if (int rc = paged_view(ctx, cache, &v)) return rc;
  if (int rc = check_uses(ctx, v)) return rc;
  DeviceScope dev(ctx);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(v);
  compact_apply_kernel<<<ctx->sm_count * 8, kMoveThreads, 0, st>>>(v);
  return launched(ctx, "token cache compact");
}
