// Shared by the attention kernels over the token-paged cache: how a call is seen on the device, how its 128-key tiles are
// dealt out to the blocks, the walk over a block's part, the loading warp, and warp-level helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "paged.cuh"
#include "ptx_sm100.cuh"

namespace magi {
using namespace ptx;

constexpr int kPaTile = 128;                   // keys of a tile
constexpr int kPaTileBytes = kPaTile * kHeadDim;
constexpr int kPromptRows = 256;               // query rows of a block in the prompt form
constexpr int kPaNear = 128;                   // entries with rows that a block's part can reach, kept in shared memory
constexpr int kPaSpread = 48;                  // see plan_tiles
// P = 2^(w - reference + 12).  The reference of a row is the exact maximum when it is set and stays while no weight exceeds
// e5m2's 57344 = 2^15.8, that is until the maximum has grown 14-fold: in nearly every tile the tensor core goes on summing in
// TMEM, and the few-row form needs one vote of the group in place of the maxima.  A weight is carried as three e5m2 terms (see
// split_weights): 2^-9 of it, and e5m2's smallest step, 2^-16, leaves 2^-17, which is 2^-29 of the reference.  So a long tail of
// small weights behind one large one keeps its mass: at 2^-20 of the largest each is still within 2^-9 of its value.
constexpr float kPaShift = 12.0f, kPaLimit = 15.8f;

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
  int n, total_q, max_q, hq, group;
  uint32_t group_mul;  // see by_group()
  int group_shift;
  float scale_log2;
  int causal, window;
  int* status;
  int page_shift;      // log2(page_tokens)
  int rows_total;      // rows of the tensor maps
  struct PaHeader* headers;  // [blocks]
  float* parts;        // [blocks][2][rows][128] accumulators of units that lie in several blocks
  float2* stats;       // [blocks][2][rows] their maximum and sum
};

// n / group for 0 <= n < 2^31, by a product with floor(2^(31 + l) / group) + 1, l = ceil(log2 group) (Granlund and Montgomery's
// division by an invariant): the walk from unit to unit divides often, and every warp does it.
__device__ __forceinline__ int by_group(const PagedAttnKernelParams& p, int n) {
  return p.group_shift < 0 ? n : (int)(__umulhi((uint32_t)n, p.group_mul) >> p.group_shift);
}
inline void set_group(PagedAttnKernelParams* p, int group) {
  int l = 0;
  while ((1ll << l) < group) ++l;
  p->group = group;
  p->group_shift = l - 1;
  p->group_mul = l > 0 ? (uint32_t)((1ull << (31 + l)) / (unsigned)group + 1) : 0u;
}

// What a block leaves behind about its last unit, when others continue it.
struct PaHeader {
  int open;         // 1: the unit starts in this block and ends in block `last`
  int last;
  int row0, h;      // of its entry, its kv head
  int first, rows;  // its flattened rows
  int pad[2];
};

// One entry of the call as the kernels see it; rows and lengths that make no sense count as none.
struct PaEntry {
  int seq, len, row0, n_q;
};

__device__ __forceinline__ PaEntry load_entry(const PagedAttnKernelParams& p, int b, bool* bad) {
  PaEntry e;
  e.seq = p.seqs[b];
  e.row0 = p.cu_q ? p.cu_q[b] : b;
  e.n_q = p.cu_q ? p.cu_q[b + 1] - e.row0 : 1;
  e.len = 0;
  bool wrong = false;
  if (e.n_q < 0 || e.n_q > p.max_q || e.row0 < 0 || (int64_t)e.row0 + e.n_q > p.total_q) {
    wrong = true;
    e.n_q = 0;
  }
  if (e.seq >= 0 && e.seq < p.c.max_seqs) {
    e.len = p.c.lens[e.seq];
    const int64_t room = (int64_t)p.c.per_row << p.page_shift;
    if (e.len < 0 || e.len > room) {
      wrong = true;
      e.len = 0;
    }
  } else {
    wrong = true;
    e.seq = 0;
  }
  *bad = wrong;
  return e;
}

// First position that a row at `pos` sees.  Rows in front of a sequence have negative positions, and a window may be as large as
// 32 bits hold: nothing is subtracted that could wrap.
__device__ __forceinline__ int window_begin(const PagedAttnKernelParams& p, int pos) {
  return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
}

// Row tile j of an entry: query rows (token, head of the group) flattened, kRows at a time.
struct PaUnit {
  int first, rows;      // flattened rows [first, first + rows)
  int pos_a, pos_z;     // positions of its first and last token
  int tile0, tiles;     // 128-key tiles that some row may see; at least one, so that rows that see nothing are written
};

template <int kRows>
__device__ __forceinline__ int unit_tiles(const PagedAttnKernelParams& p, const PaEntry& e, int j, PaUnit* u) {
  const int first = j * kRows;
  const int rows = min(kRows, e.n_q * p.group - first);
  const int pos_a = e.len - e.n_q + by_group(p, first);
  const int pos_z = e.len - e.n_q + by_group(p, first + rows - 1);
  const int end = p.causal ? pos_z + 1 : e.len;
  const int begin = window_begin(p, pos_a);
  int tile0 = 0, tiles = 1;
  if (end > begin) {
    tile0 = begin / kPaTile;
    tiles = (end + kPaTile - 1) / kPaTile - tile0;
  }
  if (u) *u = {first, rows, pos_a, pos_z, tile0, tiles};
  return tiles;
}

template <int kRows>
__device__ __forceinline__ int row_tiles(const PagedAttnKernelParams& p, const PaEntry& e) {
  return (e.n_q * p.group + kRows - 1) / kRows;
}

// Where a block's part of the tiles starts; every role walks from there by itself.
struct PaStart {
  int64_t t0, t1;       // tiles [t0, t1)
  int64_t per_block;
  int h, j, off;        // unit of the first entry in `near`, and where in its weight
  int extra;            // weight of an entry beside its units'
};

__device__ __forceinline__ void tma_load_2d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem_dst)), "l"(src) : "memory");
}
// One arrival on the barrier once this thread's earlier cp.async have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Largest value over the warp, NaN left out.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));  // volatile: not to be moved under a branch
  return r;
}

// A whole warp waits, its lanes staying together (the warp-wide instructions that follow need all lanes at once, and a branch
// on the lane left lane 0 behind on its own): all ask, the warp votes.  Bounded; gives up at once where another warp did.  A warp
// that sits out other warps' work is given the word that this work counts in: its time starts again when that moves.
__device__ __forceinline__ bool warp_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const volatile int* progress) {
  long long t0 = clock64();
  int seen = 0;
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    if (progress && *progress != seen) {
      seen = *progress;
      t0 = clock64();
    }
    if (__any_sync(0xffffffffu, clock64() - t0 > 1000000000LL)) *abort_flag = 1;
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  return true;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const volatile int* progress = nullptr) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return warp_wait_long(bar, parity, abort_flag, progress);
}
// One arrival for the warp, after what all its lanes did before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred l;\n\t"
      "setp.eq.u32 l, %1, 0;\n\t"
      "@l mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(threadIdx.x & 31)
      : "memory");
}

// Which tiles are this block's: the tiles of all units in a row, dealt out in contiguous parts of equal weight.  A unit weighs
// its tiles and kCost more for what it takes to begin and end one, as if it had so many empty tiles in front.  An entry weighs
// 1 / kPaSpread of a block's part more (nothing in small calls): with at most 1024 entries on B blocks a part then reaches no
// more than kPaSpread + 1024 / B + 2 entries that have rows, which fit in shared memory from 14 blocks on.  So every warp of the
// block walks over one and the same list, read once: lengths that change while the call runs spoil the result, no more.
// Whole block; scratch needs kPlanScratch bytes.  The caller puts a barrier behind it.
constexpr int kPlanScratch = (8 + 4 + (int)sizeof(PaEntry)) * kPgMaxEntries;
template <int R, int kThreads, int kCost>
__device__ __forceinline__ void plan_tiles(const PagedAttnKernelParams& p, uint8_t* scratch, PaStart* start, PaEntry* near) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hkv = p.c.n_kv_heads;
  int64_t* sums = reinterpret_cast<int64_t*>(scratch);  // [n] tiles of an entry, then their prefix sums
  PaEntry* entries = reinterpret_cast<PaEntry*>(scratch + 8 * kPgMaxEntries);
  int* counts = reinterpret_cast<int*>(entries + kPgMaxEntries);  // [n] entries with rows up to here
  const bool single = (int64_t)p.max_q * p.group <= R;                   // one row tile per entry
  bool any_bad = false;
  for (int b = threadIdx.x; b < p.n; b += kThreads) {
    bool bad;
    const PaEntry e = load_entry(p, b, &bad);
    any_bad |= bad;
    entries[b] = e;
    if (single) sums[b] = e.n_q > 0 ? (int64_t)(unit_tiles<R>(p, e, 0, nullptr) + kCost) * hkv : 0;
  }
  if (any_bad && blockIdx.x == 0) *p.status = MAGI_E_RANGE;
  __syncthreads();
  if (!single) {
    for (int b = warp; b < p.n; b += kThreads / 32) {
      const PaEntry e = entries[b];
      const int n_j = row_tiles<R>(p, e);
      int64_t w = 0;
      for (int j = lane; j < n_j; j += 32) w += unit_tiles<R>(p, e, j, nullptr) + kCost;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
      if (lane == 0) sums[b] = w * hkv;
    }
    __syncthreads();
  }
  if (warp == 0) {
    int64_t carry = 0;
    int count = 0;
    for (int b0 = 0; b0 < p.n; b0 += 32) {
      int64_t x = b0 + lane < p.n ? sums[b0 + lane] : 0;
      const uint32_t rows = __ballot_sync(0xffffffffu, x > 0);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (b0 + lane < p.n) {
        sums[b0 + lane] = carry + x;
        counts[b0 + lane] = count + __popc(rows & (0xffffffffu >> (31 - lane)));
      }
      carry += __shfl_sync(0xffffffffu, x, 31);
      count += __popc(rows);
    }
    __syncwarp();
    const int64_t extra = min(carry / ((int64_t)gridDim.x * kPaSpread), (int64_t)1 << 30);
    auto weight_to = [&](int b) { return sums[b] + extra * counts[b]; };  // of entries 0 .. b
    const int64_t total = carry + extra * count;
    const int64_t per_block = (total + gridDim.x - 1) / gridDim.x;
    const int64_t t0 = min((int64_t)blockIdx.x * per_block, total), t1 = min(t0 + per_block, total);
    if (t0 < t1) {
      int b = 0;  // first entry whose sum exceeds t0
      for (int b0 = 0; b0 < p.n; b0 += 32) {
        const bool over = b0 + lane < p.n && weight_to(b0 + lane) > t0;
        const uint32_t m = __ballot_sync(0xffffffffu, over);
        if (m) {
          b = b0 + __ffs(m) - 1;
          break;
        }
      }
      const int64_t per_head = (sums[b] - (b > 0 ? sums[b - 1] : 0)) / hkv;
      int64_t rem = t0 - (b > 0 ? weight_to(b - 1) : 0);
      int h = 0, j = 0;
      if (rem >= extra) {  // else in front of the entry's first unit
        rem -= extra;
        h = (int)(rem / per_head);
        rem -= h * per_head;
        if (!single) {
          const PaEntry e = entries[b];
          const int n_j = row_tiles<R>(p, e);
          for (int j0 = 0; j0 < n_j; j0 += 32) {
            const int64_t mine = j0 + lane < n_j ? unit_tiles<R>(p, e, j0 + lane, nullptr) + kCost : 0;
            int64_t x = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
              if (lane >= d) x += y;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, x > rem);
            if (m) {
              const int f = __ffs(m) - 1;
              rem -= __shfl_sync(0xffffffffu, x - mine, f);
              j = j0 + f;
              break;
            }
            rem -= __shfl_sync(0xffffffffu, x, 31);
          }
        }
        if (h == 0 && j == 0) rem += extra;
      }
      for (int b0 = b, found = 0; b0 < p.n && found < kPaNear; b0 += 32) {
        const bool has = b0 + lane < p.n && entries[b0 + lane].n_q > 0;
        const uint32_t m = __ballot_sync(0xffffffffu, has);
        const int at = found + __popc(m & ((1u << lane) - 1));
        if (has && at < kPaNear) near[at] = entries[b0 + lane];
        found += __popc(m);
      }
      if (lane == 0) *start = {t0, t1, per_block, h, j, (int)rem, (int)extra};
    } else if (lane == 0) {
      *start = {t0, t0, per_block, 0, 0, 0, 0};
    }
    if (lane == 0) p.headers[blockIdx.x].open = 0;
  }
}

// The walk over a block's segments (a segment = the tiles of one unit that are its own), the same in every role.
template <int R, int kCost>
struct PaWalk {
  const PagedAttnKernelParams& p;
  const PaEntry* near;
  int64_t t, t1;        // weight: the segment's start, the block's end
  int e, h, j, at;      // unit (its entry as a place in `near`), and where in its weight the segment starts
  int extra, n_j, cost, weight;  // of the unit: weight in front of its tiles; weight of the segment
  int first, n_seg;     // its tiles [first, first + n_seg) of the unit's
  PaEntry ent;
  PaUnit unit;

  __device__ __forceinline__ PaWalk(const PagedAttnKernelParams& params, const PaStart& st, const PaEntry* entries)
      : p(params), near(entries), t(st.t0), t1(st.t1), e(0), h(st.h), j(st.j), at(st.off), extra(st.extra) {
    if (t < t1) fetch();
  }
  __device__ __forceinline__ void fetch() {
    ent = near[e];
    n_j = row_tiles<R>(p, ent);
  }
  // The current segment; false behind the last one.
  __device__ __forceinline__ bool segment() {
    while (t < t1) {
      unit_tiles<R>(p, ent, j, &unit);
      cost = (h | j) == 0 ? kCost + extra : kCost;
      weight = (int)min((int64_t)(unit.tiles + cost - at), t1 - t);
      first = max(at - cost, 0);
      n_seg = max(at + weight - cost, 0) - first;
      if (n_seg > 0) return true;
      advance();  // none of the unit's tiles are in this block
    }
    return false;
  }
  __device__ __forceinline__ bool whole() const { return first == 0 && n_seg == unit.tiles; }
  // The block that the unit's last tile is in.
  __device__ __forceinline__ int last_block(int64_t per_block) const { return (int)((t - at + unit.tiles + cost - 1) / per_block); }
  __device__ __forceinline__ void advance() {
    t += weight;
    if (t >= t1) return;
    at = 0;
    if (++j < n_j) return;
    j = 0;
    if (++h < p.c.n_kv_heads) return;
    h = 0;
    if (++e < kPaNear) fetch();
    else t = t1;  // not reached: see plan_tiles
  }
};

// The loading warp: the pages of K and V of every tile into a ring of 16 KB stages (K of tile i is fill 2i, V 2i + 1), the
// scales of its pages by cp.async into slot i % kSlots.
template <int R, int kCost, int kStages, int kSlots>
__device__ __forceinline__ void load_tiles(const PagedAttnKernelParams& p, PaWalk<R, kCost>& w, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                                           uint8_t* ring, float* scales, uint64_t* kv_full, uint64_t* kv_empty, uint64_t* sc_full,
                                           volatile int* abort_flag) {
  const int lane = threadIdx.x & 31;
  const int P = p.c.page_tokens, per_tile = kPaTile >> p.page_shift;
  int fill = 0;
  bool ok = true;
  for (; w.segment() && ok; w.advance()) {
    const int32_t* row = p.c.table + (int64_t)w.ent.seq * p.c.per_row;
    const int first_page = (w.unit.tile0 + w.first) * per_tile;
    const int pages = (int)(((int64_t)w.ent.len + P - 1) >> p.page_shift);  // pages that hold tokens
    int ahead = lane < per_tile && first_page + lane < pages ? row[first_page + lane] : -1;
    for (int i = 0; i < w.n_seg && ok; ++i) {
      const int page0 = first_page + i * per_tile;
      const bool mine = lane < per_tile && page0 + lane < pages;
      const int id = ahead;
      const int next = page0 + per_tile + lane;
      ahead = i + 1 < w.n_seg && lane < per_tile && next < pages ? row[next] : -1;  // in flight while this tile is loaded
      const bool lost = mine && (id < 0 || id >= p.c.n_pages);
      if (lost) *p.status = MAGI_E_RANGE;
      const int n_load = min(per_tile, max(0, pages - page0));
      // a page that does not exist is read behind the last row, which fills zeros
      const int64_t block = lost ? 0 : ((int64_t)p.layer * p.c.n_pages + max(id, 0)) * p.c.n_kv_heads + w.h;
      const int y = lost ? p.rows_total : (int)(block << p.page_shift);
      const int slot = (fill >> 1) % kSlots;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++fill) {
        const int stage = fill % kStages, use = fill / kStages;
        if (use > 0) ok = warp_wait(&kv_empty[stage], (use & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&kv_full[stage], n_load << (p.page_shift + 7));
        __syncwarp();
        if (mine) tma_load_2d(ring + stage * kPaTileBytes + (lane << (p.page_shift + 7)), kv ? tm_v : tm_k, &kv_full[stage], 0, y);
        if (kv == 0) {
          if (mine) {
            cp_async_4(scales + slot * 16 + lane, p.c.k_scale + block);
            cp_async_4(scales + slot * 16 + 8 + lane, p.c.v_scale + block);
          }
          cp_async_arrive(&sc_full[slot]);
        }
        __syncwarp();
      }
    }
  }
  if (!ok) {  // given up: let the copies in flight land before the block leaves
    int late = 0;
    for (int f = max(0, fill - kStages); f < fill; ++f) mbar_wait(&kv_full[f % kStages], (f / kStages) & 1, &late, 100000000LL);
  }
  __syncwarp();
}

// Four bf16 of a query row (a lane's share of its 128 channels) as two e4m3 terms, the row scaled by the power of two that
// brings its largest entry into (224, 448].  Returns that power's inverse; whole warp, one row.
__device__ __forceinline__ float split_query(uint2 raw, uint32_t* hi, uint32_t* lo) {
  // magnitudes of bf16 compare as whole numbers; NaN and infinity are the largest
  const uint32_t a = raw.x & 0x7fff7fffu, b = raw.y & 0x7fff7fffu;
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(a & 0xffffu, a >> 16), max(b & 0xffffu, b >> 16)));
  // below 2^-92 the entries keep fewer bits: their scores are then below 2^-16 whatever the keys are
  const int e = max((int)(top >> 7) - 127 - ((top & 0x7fu) <= 0x60u ? 8 : 7), -100);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  const float f0 = __uint_as_float(raw.x << 16) * inv, f1 = __uint_as_float(raw.x & 0xffff0000u) * inv;
  const float f2 = __uint_as_float(raw.y << 16) * inv, f3 = __uint_as_float(raw.y & 0xffff0000u) * inv;
  const uint32_t h = pack4_e4m3(f0, f1, f2, f3);
  // what the first term leaves: at most eight significant bits, exact in fp16 (and zero below its 2^-25)
  const float2 d01 = __half22float2(__hsub2(__floats2half2_rn(f0, f1), __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3))));
  const float2 d23 = __half22float2(__hsub2(__floats2half2_rn(f2, f3), __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(h >> 16), __NV_E4M3))));
  const bool odd = top >= 0x7f80u;  // a row with NaN or infinity has no softmax: NaN throughout
  *hi = odd ? 0x7f7f7f7fu : h;
  *lo = odd ? 0u : pack4_e4m3(d01.x, d01.y, d23.x, d23.y);
  return __uint_as_float((uint32_t)(127 + e) << 23);
}

// P of four keys (or rows) as three e5m2 terms, each taken from what those before it left.  An e5m2 is the upper byte of an fp16:
// the first term is cut off, which keeps NaN, the other two are rounded.  The first leaves the lower 8 of fp16's 11 bits; the
// second rounds these at 3 bits, the third what remains, 5 bits and a sign, at 3 again: at most 2^-10 of the weight beside the
// 2^-11 of its rounding to fp16, 2^-9.4 in all, and 2^-17 where the last step is e5m2's smallest.  Remainders are exact in fp16.
__device__ __forceinline__ void split_weights(float p0, float p1, float p2, float p3, uint32_t* t0, uint32_t* t1, uint32_t* t2) {
  auto half2_of = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
  auto bits_of = [](__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); };
  const uint32_t h01 = bits_of(__floats2half2_rn(p0, p1)), h23 = bits_of(__floats2half2_rn(p2, p3));
  const uint32_t r01 = bits_of(__hsub2(half2_of(h01), half2_of(h01 & 0xff00ff00u)));
  const uint32_t r23 = bits_of(__hsub2(half2_of(h23), half2_of(h23 & 0xff00ff00u)));
  const uint32_t u01 = r01 + 0x00800080u, u23 = r23 + 0x00800080u;
  const uint32_t v01 = bits_of(__hsub2(half2_of(r01), half2_of(u01 & 0xff00ff00u))) + 0x00800080u;
  const uint32_t v23 = bits_of(__hsub2(half2_of(r23), half2_of(u23 & 0xff00ff00u))) + 0x00800080u;
  *t0 = __byte_perm(h01, h23, 0x7531);
  *t1 = __byte_perm(u01, u23, 0x7531);
  *t2 = __byte_perm(v01, v23, 0x7531);
}

// Row `key` of a V tile in shared memory: its NaN codes become zero, their places go to bits (channel c: word c / 32).
__device__ __forceinline__ void take_nan(uint4* vrow, int key, uint32_t (&bits)[4]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint4 q = vrow[c ^ (key & 7)];
    const uint32_t wd[4] = {q.x, q.y, q.z, q.w};
    uint32_t kept[4], any = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t is = __vcmpeq4(wd[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
      kept[k] = wd[k] & ~is;
      any |= is;
      bits[c >> 1] |= ((is & 1u) | (is >> 7 & 2u) | (is >> 14 & 4u) | (is >> 21 & 8u)) << ((c & 1) * 16 + k * 4);
    }
    if (any) vrow[c ^ (key & 7)] = make_uint4(kept[0], kept[1], kept[2], kept[3]);
  }
}

}  // namespace magi
