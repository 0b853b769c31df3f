// Attention over the token-paged 8-bit cache, for sm_100a: one kernel from a single new token to whole prompts.
//
//   s = scale * q . (k8 sk),  o = sum_k softmax(s)_k (v8 sv),  sk, sv powers of two per (page, kv head)
//
// The scores are formed TRANSPOSED, S^T [128 keys x R rows] = K8 Q^T and O^T [128 channels x R rows] = V8^T P^T, so that
// the long side of every product is the cache: the e4m3 tiles go from HBM through TMA and shared memory to tcgen05.mma
// (kind::f8f6f4, M = 128) exactly as they are stored, nothing is ever converted to a wider type, and a tile costs the same
// few instructions whether a sequence has one new token (R = 16 covers 16 query heads of a kv head) or many.  K8 is the
// K-major A operand of the first product, V8 - stored [key][channel] - the MN-major A operand of the second.
//
// Precision: Q and P are carried as two e4m3 terms each (value + rounding residual; two instructions that accumulate into
// the same columns).  bf16 has 8 significant bits and two e4m3 terms hold 8, so Q loses nothing except what lies 2^-17
// below its row's largest entry; P is rounded to 2^-8 of each weight, like the bf16 result.  Sums, maxima and the output
// accumulator are fp32 in registers.  The V scale is folded into the exponent, w = s log2e + log2(sv), and the running
// maximum is taken over w: then every P is at most 1 however different the pages' scales are, O needs no scale per page
// and the denominator adds P / sv.
//
// Work: the 128-key tiles of all (sequence, kv head, row tile) units in a row are dealt out to the blocks in equal
// contiguous parts, so a long sequence is split over many blocks and ragged batches balance; the lengths are read on the
// device.  A block finishes the units that lie inside its part; for the (at most two) that do not it leaves maximum, sum
// and accumulator in the workspace, and a second kernel joins them in the order of the keys (no atomics: the same bits
// every time).
//
//   warp 0     TMA: pages of K and V into a ring of 16 KB tiles, their scales by cp.async beside them
//   warp 1     UMMA issuer (one thread)
//   warps 2+   G groups of four: thread = key of S^T, then channel of O^T; a group takes RG of the R rows
// Every wait is bounded (MAGI_E_TIMEOUT).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "paged.cuh"
#include "ptx_sm100.cuh"

namespace magi {
using namespace ptx;

int make_rows_map(magi_ctx* ctx, CUtensorMap* m, const void* base, int rows, int box_rows, const char* what);

constexpr int kPaTile = 128;                   // keys of a tile
constexpr int kPaTileBytes = kPaTile * kHeadDim;
constexpr int kPaNear = 64;                    // entries whose lengths a block keeps in shared memory
// P = 2^(w - reference + 5).  The reference of a row is the exact maximum when it is set and stays while no weight exceeds
// e4m3's 448 = 2^8.8, that is until the maximum has grown 14-fold: nearly every tile then needs one vote of the group in
// place of its maxima, and the tensor core goes on summing in TMEM.  The residual term is e5m2, whose smallest step is 2^-16:
// a weight is dropped only below 2^-22 of the reference, so a long tail of small weights behind one large one keeps its mass.
constexpr float kPaShift = 5.0f, kPaLimit = 8.8f;

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
  float scale_log2;
  int causal, window;
  int* status;
  int page_shift;      // log2(page_tokens)
  int rows_total;      // rows of the tensor maps
  struct PaHeader* headers;  // [blocks]
  float* parts;        // [blocks][2][R][128] accumulators of units that lie in several blocks
  float2* stats;       // [blocks][2][R] their maximum and sum
};

// What a block leaves behind about its last unit, when others continue it.
struct PaHeader {
  int open;        // 1: the unit starts in this block and ends in block `last`
  int b, h, j;     // entry, kv head, row tile
  int last;
  int pad[3];
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
  const int pos_a = e.len - e.n_q + first / p.group;
  const int pos_z = e.len - e.n_q + (first + rows - 1) / p.group;
  const int end = p.causal ? pos_z + 1 : e.len;
  const int begin = p.window > 0 ? max(0, pos_a - p.window + 1) : 0;
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
  int b, h, j, off;     // unit and tile within it
};

template <int RG, int G>
struct PaShared {
  static constexpr int kRows = RG * G;
  static constexpr int kStages = kRows == 16 ? 5 : kRows == 32 ? 4 : 6;
  static constexpr int kWarps = 4 * G;                         // softmax warps
  static constexpr int kFirst = 2;                             // the first of them
  static constexpr int kThreads = 32 * (kFirst + kWarps);
  static constexpr int kRing = 0;
  // Two buffers of P, a byte per (key, row) and term.  Up to 32 rows: all four share the 128-byte rows [key] of one tile
  // (term 0 of buffer 0 and 1, then term 1 of both, 32 bytes each); else each is a tile of its own.
  static constexpr int kPBuf = kRows <= 32 ? 32 : 2 * kPaTileBytes;
  static constexpr int kPTerm = kRows <= 32 ? 64 : kPaTileBytes;
  static constexpr int kP = kRing + kStages * kPaTileBytes;
  static constexpr int kQ = kP + (kRows <= 32 ? 1 : 4) * kPaTileBytes;  // [2 terms][kRows][128 bytes]
  static constexpr int kScales = kQ + 2 * kRows * 128;         // [kStages][2][8] page scales of the last kStages tiles
  static constexpr int kMax = kScales + kStages * 64;          // [G][4][RG] warp maxima, and sums at a unit's end
  static constexpr int kNegM = kMax + G * 4 * RG * 4;          // [kRows]
  static constexpr int kFactor = kNegM + kRows * 4;            // [kRows]
  static constexpr int kRowS = kFactor + kRows * 4;            // [2][kRows] scale of a query row
  static constexpr int kRowPos = kRowS + 2 * kRows * 4;        // [2][kRows] its position
  static constexpr int kInv = kRowPos + 2 * kRows * 4;         // [kWarps][RG]
  static constexpr int kAt = kInv + kWarps * RG * 4;           // [kWarps][RG] where a row of the result starts
  static constexpr int kNan = kAt + kWarps * RG * 8;             // [2][128][4] channels whose V is NaN (boundary tiles)
  static constexpr int kNanAny = kNan + 2 * kPaTile * 16;      // [2][4] whether a warp's keys have any
  static constexpr int kNear = kNanAny + 32;                   // [kPaNear] entries
  static constexpr int kStart = kNear + kPaNear * 16;
  static constexpr int kBar = kStart + 64;
  static constexpr int kNumBars = 3 * kStages + 8;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kTotal = kMisc + 16;
  static constexpr int kDynamic = kTotal + 1024;
  static constexpr uint32_t kTmemCols = kRows <= 32 ? 4 * kRows : 512;             // S twice, O (the allocation is a power of two)
};
static_assert(PaShared<16, 1>::kDynamic * 2 + 2048 <= 233472, "two blocks of the small form per SM");
static_assert(PaShared<32, 1>::kDynamic * 2 + 2048 <= 233472, "two blocks of the middle form per SM");
static_assert(PaShared<32, 3>::kDynamic <= 232448, "shared memory per block");

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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld32(taddr, r);
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

// A whole warp waits, its lanes staying together: lane 0 asks, by predicate and not by branch, and the warp votes.  (32 lanes
// asking for one barrier are served one after the other, about 200 cycles a question; a branch on the lane leaves lane 0
// behind on its own, and the warp-wide instructions that follow need all lanes at once.)
__device__ __forceinline__ bool warp_wait(bool ok, uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (!ok) return false;
  const uint32_t addr = smem_u32(bar), lane = threadIdx.x & 31;
  long long t0 = 0;
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred l, p;\n\t"
        "setp.eq.u32 l, %3, 0;\n\t"
        "setp.ne.u32 p, %3, %3;\n\t"
        "@l mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity), "r"(lane), "r"((uint32_t)MAGI_WAIT_HINT_NS)
        : "memory");
    if (__any_sync(0xffffffffu, done)) break;
    const long long now = clock64();
    if (t0 == 0) t0 = now;
    const bool late = now - t0 > 1000000000LL;
    if (__any_sync(0xffffffffu, late)) *abort_flag = 1;
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  __syncwarp();  // what lane 0 has seen is there for the others
  return true;
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

// Barriers of a softmax group (128 threads) and of all softmax warps.  A warp counts once only if its lanes arrive together.
__device__ __forceinline__ bool group_any(int id, bool v) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.u32 a, %1, 0;\n\t"
      "bar.red.or.pred b, %2, 128, a;\n\t"
      "selp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}
template <int N>
__device__ __forceinline__ void all_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

template <int RG, int G>
__global__ void __launch_bounds__(PaShared<RG, G>::kThreads, G == 1 ? 2 : 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ PagedAttnKernelParams p) {
  using L = PaShared<RG, G>;
  constexpr int R = L::kRows;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* sc_full = kv_empty + kStages;  // page scales of a tile: by tile, not by stage, since the softmax reads them after K has left
  uint64_t* s_full = sc_full + kStages;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* q_full = o_full + 2;
  uint64_t* drain_bar = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  PaStart* start = reinterpret_cast<PaStart*>(smem + L::kStart);
  PaEntry* near = reinterpret_cast<PaEntry*>(smem + L::kNear);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = p.c.n_kv_heads;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&sc_full[s], 32);  // each lane of the loading warp
      mbar_init(&kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], L::kWarps);
      mbar_init(&o_full[x], 1);
    }
    mbar_init(q_full, L::kWarps);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  // ---- which tiles are this block's: sums over the entries in the (still unused) ring
  {
    int64_t* sums = reinterpret_cast<int64_t*>(smem + L::kRing);           // [n] tiles of an entry, then their prefix sums
    PaEntry* entries = reinterpret_cast<PaEntry*>(smem + L::kRing + 8 * kPgMaxEntries);
    const bool single = (int64_t)p.max_q * p.group <= R;                   // one row tile per entry
    bool any_bad = false;
    for (int b = threadIdx.x; b < p.n; b += L::kThreads) {
      bool bad;
      const PaEntry e = load_entry(p, b, &bad);
      any_bad |= bad;
      entries[b] = e;
      if (single) sums[b] = e.n_q > 0 ? (int64_t)unit_tiles<R>(p, e, 0, nullptr) * hkv : 0;
    }
    if (any_bad && blockIdx.x == 0) *p.status = MAGI_E_RANGE;
    __syncthreads();
    if (!single) {
      for (int b = warp; b < p.n; b += L::kThreads / 32) {
        const PaEntry e = entries[b];
        const int n_j = row_tiles<R>(p, e);
        int64_t w = 0;
        for (int j = lane; j < n_j; j += 32) w += unit_tiles<R>(p, e, j, nullptr);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
        if (lane == 0) sums[b] = w * hkv;
      }
      __syncthreads();
    }
    if (warp == 0) {
      int64_t carry = 0;
      for (int b0 = 0; b0 < p.n; b0 += 32) {
        int64_t x = b0 + lane < p.n ? sums[b0 + lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += y;
        }
        if (b0 + lane < p.n) sums[b0 + lane] = carry + x;
        carry += __shfl_sync(0xffffffffu, x, 31);
      }
      __syncwarp();
      const int64_t total = carry;
      const int64_t per_block = (total + gridDim.x - 1) / gridDim.x;
      const int64_t t0 = min((int64_t)blockIdx.x * per_block, total), t1 = min(t0 + per_block, total);
      if (t0 < t1) {
        int b = 0;  // first entry whose sum exceeds t0
        for (int b0 = 0; b0 < p.n; b0 += 32) {
          const bool over = b0 + lane < p.n && sums[b0 + lane] > t0;
          const uint32_t m = __ballot_sync(0xffffffffu, over);
          if (m) {
            b = b0 + __ffs(m) - 1;
            break;
          }
        }
        const int64_t before = b > 0 ? sums[b - 1] : 0;
        const int64_t per_head = (sums[b] - before) / hkv;
        const int h = (int)((t0 - before) / per_head);
        int64_t rem = (t0 - before) - h * per_head;
        int j = 0;
        if (!single) {
          const PaEntry e = entries[b];
          const int n_j = row_tiles<R>(p, e);
          for (int j0 = 0; j0 < n_j; j0 += 32) {
            const int64_t mine = j0 + lane < n_j ? unit_tiles<R>(p, e, j0 + lane, nullptr) : 0;
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
        for (int i = lane; i < kPaNear; i += 32)
          if (b + i < p.n) near[i] = entries[b + i];
        if (lane == 0) *start = {t0, t1, per_block, b, h, j, (int)rem};
      } else if (lane == 0) {
        *start = {t0, t0, per_block, 0, 0, 0, 0};
      }
      if (lane == 0) p.headers[blockIdx.x].open = 0;
    }
  }
  fence_proxy_async_smem();  // the ring goes over to TMA
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PaStart st = *start;

  // The walk over this block's segments (a segment = the tiles of one unit that are its own), the same in every role.
  int64_t t = st.t0;
  int b = st.b, h = st.h, j = st.j, off = st.off;
  PaEntry ent;
  PaUnit unit;
  int n_j = 0;
  auto fetch_entry = [&]() {
    if (b - st.b < kPaNear) ent = near[b - st.b];
    else {
      bool bad;
      ent = load_entry(p, b, &bad);
    }
    n_j = row_tiles<R>(p, ent);
  };
  auto next_unit = [&]() {
    off = 0;
    if (++j < n_j) return;
    j = 0;
    if (++h < hkv) return;
    h = 0;
    do {
      if (++b >= p.n) return;
      fetch_entry();
    } while (n_j == 0);
  };
  if (t < st.t1) fetch_entry();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const int P = p.c.page_tokens, per_tile = kPaTile >> p.page_shift;
    float* scales = reinterpret_cast<float*>(smem + L::kScales);
    int fill = 0;  // tiles of the ring: K of tile i is fill 2i, V 2i + 1
    bool ok = true;
    while (t < st.t1 && ok) {
      unit_tiles<R>(p, ent, j, &unit);
      const int n_seg = (int)min((int64_t)(unit.tiles - off), st.t1 - t);
      const int32_t* row = p.c.table + (int64_t)ent.seq * p.c.per_row;
      const int first_page = (unit.tile0 + off) * per_tile;
      const int pages = (int)(((int64_t)ent.len + P - 1) >> p.page_shift);  // pages that hold tokens
      int ahead = lane < per_tile && first_page + lane < pages ? row[first_page + lane] : -1;
      for (int i = 0; i < n_seg && ok; ++i) {
        const int page0 = first_page + i * per_tile;
        const bool mine = lane < per_tile && page0 + lane < pages;
        int id = ahead;
        const int next = page0 + per_tile + lane;
        ahead = i + 1 < n_seg && lane < per_tile && next < pages ? row[next] : -1;  // in flight while this tile is loaded
        const bool lost = mine && (id < 0 || id >= p.c.n_pages);
        if (lost) *p.status = MAGI_E_RANGE;
        const int n_load = min(per_tile, max(0, pages - page0));
        // a page that does not exist is read behind the last row, which fills zeros
        const int64_t block = lost ? 0 : ((int64_t)p.layer * p.c.n_pages + max(id, 0)) * hkv + h;
        const int y = lost ? p.rows_total : (int)(block << p.page_shift);
        const int slot = (fill >> 1) % kStages;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++fill) {
          const int stage = fill % kStages, use = fill / kStages;
          if (use > 0) ok = warp_wait(ok, &kv_empty[stage], (use & 1) ^ 1, abort_flag);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&kv_full[stage], n_load << (p.page_shift + 7));
          __syncwarp();
          if (mine) tma_load_2d(smem + L::kRing + stage * kPaTileBytes + (lane << (p.page_shift + 7)), kv ? &tm_v : &tm_k, &kv_full[stage], 0, y);
          if (kv == 0 && mine) {
            cp_async_4(scales + slot * 16 + lane, p.c.k_scale + block);
            cp_async_4(scales + slot * 16 + 8 + lane, p.c.v_scale + block);
          }
          if (kv == 0) cp_async_arrive(&sc_full[slot]);
        }
      }
      t += n_seg;
      if (t < st.t1) next_unit();
    }
    if (!ok) {  // given up: let the copies in flight land before the block leaves
      int late = 0;
      for (int f = max(0, fill - kStages); f < fill; ++f) mbar_wait(&kv_full[f % kStages], (f / kStages) & 1, &late, 100000000LL);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ UMMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc(kPaTile, R, 0, 0, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc(kHeadDim, R, 0, 0, 1, 1), idesc_r = umma_idesc(kHeadDim, R, 0, 1, 1, 1);  // B e4m3, e5m2
      constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);  // 1024 bytes between groups of 8 rows, 128-byte swizzle
      const uint32_t ring = (smem_u32(smem + L::kRing) >> 4) | (1u << 16);
      const uint32_t q_lo = (smem_u32(smem + L::kQ) >> 4) | (1u << 16);
      const uint32_t p_lo = (smem_u32(smem + L::kP) >> 4) | (1u << 16);
      bool ok = true;
      int i = 0;       // tiles so far
      int units = 0;
      bool pending = false;  // the second product of tile i - 1 is still to be issued
      bool opens = true;     // that tile is its segment's first: O starts from zero
      auto second = [&](int k) {
        const int fill = 2 * k + 1, stage = fill % kStages;
        ok = mbar_wait(&kv_full[stage], (uint32_t)(fill / kStages) & 1, abort_flag);
        ok = ok && mbar_wait(&p_full[k & 1], (uint32_t)(k >> 1) & 1, abort_flag);
        if (!ok) return;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + 2 * R;
        const uint32_t a = ring + stage * (kPaTileBytes >> 4), bb = p_lo + (k & 1) * (L::kPBuf >> 4);
        if (opens) umma_ss_f8_lh<0>(d, a, bb, desc_hi, idesc_o);
        else umma_ss_f8_lh<1>(d, a, bb, desc_hi, idesc_o);
#pragma unroll
        for (int s = 1; s < 8; ++s)  // 32 keys per instruction; then the residual term
          umma_ss_f8_lh<1>(d, a + (s & 3) * 256, bb + (s & 3) * 256 + (s >> 2) * (L::kPTerm >> 4), desc_hi, s < 4 ? idesc_o : idesc_r);
        umma_commit(&o_full[k & 1]);
        umma_commit(&kv_empty[stage]);
      };
      while (t < st.t1 && ok) {
        unit_tiles<R>(p, ent, j, &unit);
        const int n_seg = (int)min((int64_t)(unit.tiles - off), st.t1 - t);
        if (pending) second(i - 1);  // the next unit's rows are written only after the last tile of this one is through
        pending = false;
        if (ok) ok = mbar_wait(q_full, units & 1, abort_flag);
        for (int x = 0; x < n_seg && ok; ++x, ++i) {
          const int fill = 2 * i, stage = fill % kStages;
          ok = mbar_wait(&kv_full[stage], (uint32_t)(fill / kStages) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after_sync();
          // S buffer i & 1 is free: the second product of tile i - 2 waited for the warps that had read it
          const uint32_t d = tmem_base + (i & 1) * R;
          const uint32_t a = ring + stage * (kPaTileBytes >> 4);
          umma_ss_f8_lh<0>(d, a, q_lo, desc_hi, idesc_s);
#pragma unroll
          for (int s = 1; s < 8; ++s)  // 32 channels per instruction; then the residual term
            umma_ss_f8_lh<1>(d, a + (s & 3) * 2, q_lo + (s & 3) * 2 + (s >> 2) * (R * 8), desc_hi, idesc_s);
          umma_commit(&s_full[i & 1]);
          umma_commit(&kv_empty[stage]);
          if (pending) second(i - 1);
          pending = true;
          opens = x == 0;
        }
        ++units;
        t += n_seg;
        if (t < st.t1) next_unit();
      }
      if (ok && pending) second(i - 1);
      if (!ok) {  // given up: the instructions issued so far still read shared memory and write TMEM
        int late = 0;
        umma_commit(drain_bar);
        mbar_wait(drain_bar, 0, &late, 100000000LL);
      }
    }
    __syncwarp();
  } else if (warp >= L::kFirst) {
    // ------------------------------------------------------------------ softmax and output
    // No early exits in here: a warp whose wait gave up goes on without waiting, so that the named barriers always meet.
    const int sw = warp - L::kFirst, g = sw >> 2;  // softmax warp, its group
    const int quarter = warp & 3;             // TMEM lanes of this warp
    const int key = quarter * 32 + lane;      // key of the tile; channel of the output
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_o = tmem_base + lane_base + 2 * R + g * RG;
    const float* scales = reinterpret_cast<const float*>(smem + L::kScales);
    float* max_sh = reinterpret_cast<float*>(smem + L::kMax) + g * 4 * RG;
    float* neg_m = reinterpret_cast<float*>(smem + L::kNegM) + g * RG;     // kPaShift - reference maximum of a row
    float* factor = reinterpret_cast<float*>(smem + L::kFactor) + g * RG;
    float* inv_sh = reinterpret_cast<float*>(smem + L::kInv) + sw * RG;
    int64_t* at_sh = reinterpret_cast<int64_t*>(smem + L::kAt) + sw * RG;
    uint32_t* nan_sh = reinterpret_cast<uint32_t*>(smem + L::kNan);
    uint32_t* nan_any = reinterpret_cast<uint32_t*>(smem + L::kNanAny);
    bool ok = true;
    int i = 0, units = 0;
    int fixes = 0;                            // boundary tiles so far
    while (t < st.t1) {
      unit_tiles<R>(p, ent, j, &unit);
      const int n_seg = (int)min((int64_t)(unit.tiles - off), st.t1 - t);
      float* row_s = reinterpret_cast<float*>(smem + L::kRowS) + (units & 1) * R;
      int* row_pos = reinterpret_cast<int*>(smem + L::kRowPos) + (units & 1) * R;
      // ---- query rows of the unit as two e4m3 terms, each row scaled by a power of two so that its largest entry is in (224, 448]
      {
        constexpr int kMine = R / L::kWarps;
        uint2 raw[kMine];
        int toks[kMine];
#pragma unroll
        for (int x = 0; x < kMine; ++x) {
          const int r = sw + x * L::kWarps, flat = unit.first + r, tok = flat / p.group;
          toks[x] = tok;
          raw[x] = make_uint2(0, 0);
          if (r < unit.rows)
            raw[x] = *reinterpret_cast<const uint2*>(p.q + (int64_t)(ent.row0 + tok) * p.q_st + (int64_t)(h * p.group + flat - tok * p.group) * p.q_sh + lane * 4);
        }
#pragma unroll
        for (int x = 0; x < kMine; ++x) {
          const int r = sw + x * L::kWarps;
          float f[4] = {__uint_as_float(raw[x].x << 16), __uint_as_float(raw[x].x & 0xffff0000u), __uint_as_float(raw[x].y << 16), __uint_as_float(raw[x].y & 0xffff0000u)};
          const float top = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
          const bool odd = !(fabsf(f[0]) < INFINITY && fabsf(f[1]) < INFINITY && fabsf(f[2]) < INFINITY && fabsf(f[3]) < INFINITY);
          const uint32_t bits = __float_as_uint(warp_max(top));
          // below 2^-92 the entries keep fewer bits: their scores are then below 2^-16 whatever the keys are
          const int e = max((int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7), -100);
          const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
          uint32_t hi = 0x7f7f7f7fu, lo = 0;  // a row with NaN or infinity has no softmax: NaN throughout
          if (!__any_sync(0xffffffffu, odd)) {
            float res[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] *= inv;
            hi = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3) |
                 (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3) << 16;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(hi >> (8 * k)), __NV_E4M3);
              res[k] = f[k] - __half2float(*reinterpret_cast<const __half*>(&hr));
            }
            lo = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(res[0], res[1]), __NV_SATFINITE, __NV_E4M3) |
                 (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(res[2], res[3]), __NV_SATFINITE, __NV_E4M3) << 16;
          }
          const int at = r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(smem + L::kQ + at) = hi;
          *reinterpret_cast<uint32_t*>(smem + L::kQ + R * 128 + at) = lo;
          if (lane == 0) {
            row_s[r] = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
            row_pos[r] = ent.len - ent.n_q + toks[x];
          }
        }
        if ((sw & 3) == 0 && lane < RG) neg_m[lane] = INFINITY;
      }
      fence_proxy_async_smem();
      warp_arrive(q_full);
      ok = warp_wait(ok, q_full, units & 1, abort_flag);  // the other warps' row scales and positions
      const bool idle = g * RG >= unit.rows;  // a group without rows only keeps step
      float m = -INFINITY;    // lane r < RG: reference maximum of row r, at most kPaLimit - kPaShift below the running one
      uint32_t nan_rows = 0;  // rows whose result in this thread's channel is NaN (boundary tiles)
      uint64_t l2[RG / 2];    // sums over this thread's keys, rows in pairs
#pragma unroll
      for (int k = 0; k < RG / 2; ++k) l2[k] = 0;
      const float4* s4 = reinterpret_cast<const float4*>(row_s + g * RG);
      const float4* n4 = reinterpret_cast<const float4*>(neg_m);
#pragma unroll 1
      for (int x = 0; x < n_seg; ++x, ++i) {
        const int k0 = (unit.tile0 + off + x) * kPaTile, pos = k0 + key;
        ok = warp_wait(ok, &sc_full[i % kStages], (uint32_t)(i / kStages) & 1, abort_flag);
        ok = warp_wait(ok, &s_full[i & 1], (uint32_t)(i >> 1) & 1, abort_flag);
        const bool tail = k0 + kPaTile > ent.len;                                             // keys behind the sequence's end
        // keys before it that not every row sees
        const bool edge = (p.causal && min(k0 + kPaTile, ent.len) - 1 > unit.pos_a) || (p.window > 0 && k0 <= unit.pos_z - p.window);
        if (G > 1 && idle) {
          if (edge) {
            all_sync<32 * L::kWarps>(1 + G);
            ++fixes;
          }
          warp_arrive(&p_full[i & 1]);
          continue;
        }
        tc_fence_after_sync();
        const uint32_t t_s = tmem_base + lane_base + (i & 1) * R + g * RG;
        float w[RG];  // exponents of the weights: s log2e + log2(sv) - reference + kPaShift
        tmem_ld<RG>(t_s, reinterpret_cast<uint32_t*>(w));
        const float ks = scales[(i % kStages) * 16 + (key >> p.page_shift)];
        const uint32_t vs = __float_as_uint(scales[(i % kStages) * 16 + 8 + (key >> p.page_shift)]);
        const float bias = (float)((int)(vs >> 23) - 127);                                    // log2 of a power of two
        const float inv_vs = pos < ent.len ? __uint_as_float(0x7f000000u - vs) : 0.f;         // behind the end there is no page
        const uint64_t ks2 = f2_pack(ks, ks), bias2 = f2_pack(bias, bias);
        auto hide = [&]() {
          const int* rp = row_pos + g * RG;
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            const int at = rp[r];
            const bool seen = pos < ent.len && (!p.causal || pos <= at) && (p.window <= 0 || pos > at - p.window);
            if (!seen) w[r] = -INFINITY;
          }
        };
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < RG; r += 4) {
          const float4 s = s4[r / 4], n = n4[r / 4];
          f2_unpack(f2_fma(f2_mul(f2_pack(w[r], w[r + 1]), ks2), f2_pack(s.x, s.y), f2_add(bias2, f2_pack(n.x, n.y))), w[r], w[r + 1]);
          f2_unpack(f2_fma(f2_mul(f2_pack(w[r + 2], w[r + 3]), ks2), f2_pack(s.z, s.w), f2_add(bias2, f2_pack(n.z, n.w))), w[r + 2], w[r + 3]);
        }
        if (tail || edge) hide();
        float top = fmaxf(w[0], w[1]);
#pragma unroll
        for (int r = 2; r < RG; r += 2) top = max3(top, w[r], w[r + 1]);
        if (group_any(1 + g, top > kPaLimit)) {
          // ---- some row's reference is too low (always so in a unit's first tile): the exact maxima, from the scores again
          tmem_ld<RG>(t_s, reinterpret_cast<uint32_t*>(w));
          tmem_wait_ld();
#pragma unroll
          for (int r = 0; r < RG; r += 4) {
            const float4 s = s4[r / 4];
            w[r] = fmaf(w[r] * ks, s.x, bias);
            w[r + 1] = fmaf(w[r + 1] * ks, s.y, bias);
            w[r + 2] = fmaf(w[r + 2] * ks, s.z, bias);
            w[r + 3] = fmaf(w[r + 3] * ks, s.w, bias);
          }
          if (tail || edge) hide();
          float mine = -INFINITY;
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            const float mx = warp_max(w[r]);
            if (lane == r) mine = mx;
          }
          if (lane < RG) max_sh[(sw & 3) * RG + lane] = mine;
          group_sync(1 + g);
          if (lane < RG) {
            const float m_new = fmaxf(fmaxf(fmaxf(m, max_sh[lane]), max_sh[RG + lane]), fmaxf(max_sh[2 * RG + lane], max_sh[3 * RG + lane]));
            if ((sw & 3) == 0) {
              neg_m[lane] = kPaShift - m_new;
              factor[lane] = m_new == -INFINITY ? 1.0f : ex2(m - m_new);
            }
            m = m_new;
          }
          group_sync(1 + g);
          const float4* f4 = reinterpret_cast<const float4*>(factor);
#pragma unroll
          for (int r = 0; r < RG; r += 4) {
            const float4 n = n4[r / 4], f = f4[r / 4];
            w[r] = w[r] == -INFINITY ? w[r] : w[r] + n.x;
            w[r + 1] = w[r + 1] == -INFINITY ? w[r + 1] : w[r + 1] + n.y;
            w[r + 2] = w[r + 2] == -INFINITY ? w[r + 2] : w[r + 2] + n.z;
            w[r + 3] = w[r + 3] == -INFINITY ? w[r + 3] : w[r + 3] + n.w;
            l2[r / 2] = f2_mul(l2[r / 2], f2_pack(f.x, f.y));
            l2[r / 2 + 1] = f2_mul(l2[r / 2 + 1], f2_pack(f.z, f.w));
          }
          if (x > 0) {  // what the tensor core has summed so far
            ok = warp_wait(ok, &o_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1, abort_flag);
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < RG; c += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int r = 0; r < 16; r += 4) {
                const float4 f = f4[(c + r) / 4];
                o[r] = __float_as_uint(__uint_as_float(o[r]) * f.x);
                o[r + 1] = __float_as_uint(__uint_as_float(o[r + 1]) * f.y);
                o[r + 2] = __float_as_uint(__uint_as_float(o[r + 2]) * f.z);
                o[r + 3] = __float_as_uint(__uint_as_float(o[r + 3]) * f.w);
              }
              tmem_st16(t_o + c, o);
            }
            tmem_wait_st();
          }
        }
        // ---- weights, their sum, and P as two e4m3 terms
        uint32_t hi[RG / 4], lo[RG / 4];
        const uint64_t inv2 = f2_pack(inv_vs, inv_vs);
#pragma unroll
        for (int r = 0; r < RG; r += 4) {
          const float p0 = ex2(w[r]), p1 = ex2(w[r + 1]), p2 = ex2(w[r + 2]), p3 = ex2(w[r + 3]);
          l2[r / 2] = f2_fma(f2_pack(p0, p1), inv2, l2[r / 2]);
          l2[r / 2 + 1] = f2_fma(f2_pack(p2, p3), inv2, l2[r / 2 + 1]);
          // first term e4m3; what it leaves, exact in fp16, as e5m2: the upper byte of an fp16, rounded
          const uint32_t h = pack4_e4m3(p0, p1, p2, p3);
          const __half2 d01 = __hsub2(__floats2half2_rn(p0, p1), __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3)));
          const __half2 d23 = __hsub2(__floats2half2_rn(p2, p3), __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(h >> 16), __NV_E4M3)));
          hi[r / 4] = h;
          lo[r / 4] = __byte_perm(*reinterpret_cast<const uint32_t*>(&d01) + 0x00800080u, *reinterpret_cast<const uint32_t*>(&d23) + 0x00800080u, 0x7531);
        }
        // the buffer of tile i - 2
        if (i >= 2) ok = warp_wait(ok, &o_full[i & 1], (uint32_t)((i - 2) >> 1) & 1, abort_flag);
        uint8_t* pb = smem + L::kP + key * 128 + (R <= 32 ? 0 : (i & 1) * L::kPBuf);
#pragma unroll
        for (int c = 0; c < RG / 16; ++c) {
          const int chunk = R <= 32 ? (i & 1) * 2 + c : g * (RG / 16) + c;  // 16 rows of the R
          const int at0 = (chunk ^ (key & 7)) << 4, at1 = R <= 32 ? ((chunk + 4) ^ (key & 7)) << 4 : L::kPTerm + at0;
          *reinterpret_cast<uint4*>(pb + at0) = make_uint4(hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
          *reinterpret_cast<uint4*>(pb + at1) = make_uint4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
        }
        if (tail || edge) {
          // A weight of zero does not silence a NaN: V of keys behind the end becomes zero, and NaN codes of keys that only
          // some rows see are taken out of the product and come back through the sums of the rows that do see them.
          const int v_fill = 2 * i + 1, v_stage = v_fill % kStages;
          ok = warp_wait(ok, &kv_full[v_stage], (uint32_t)(v_fill / kStages) & 1, abort_flag);
          __syncwarp();
          uint4* vrow = reinterpret_cast<uint4*>(smem + L::kRing + v_stage * kPaTileBytes + key * 128);
          if (g == 0) {
            if (pos >= ent.len) {
#pragma unroll
              for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0, 0, 0, 0);
            }
            if (edge) {
              uint32_t nan_bits[4] = {0, 0, 0, 0};
              if (pos < ent.len) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                  const uint4 q = vrow[c ^ (key & 7)];
                  const uint32_t wd[4] = {q.x, q.y, q.z, q.w};
                  uint32_t kept[4];
                  uint32_t any = 0;
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const uint32_t is = __vcmpeq4(wd[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    kept[k] = wd[k] & ~is;
                    any |= is;
                    nan_bits[c >> 1] |= ((is & 1u) | (is >> 7 & 2u) | (is >> 14 & 4u) | (is >> 21 & 8u)) << ((c & 1) * 16 + k * 4);
                  }
                  if (any) vrow[c ^ (key & 7)] = make_uint4(kept[0], kept[1], kept[2], kept[3]);
                }
              }
              *reinterpret_cast<uint4*>(nan_sh + ((fixes & 1) * kPaTile + key) * 4) = make_uint4(nan_bits[0], nan_bits[1], nan_bits[2], nan_bits[3]);
              const uint32_t some = __ballot_sync(0xffffffffu, (nan_bits[0] | nan_bits[1] | nan_bits[2] | nan_bits[3]) != 0);
              if (lane == 0) nan_any[(fixes & 1) * 4 + (sw & 3)] = some;
            }
          }
          if (edge) {
            all_sync<32 * L::kWarps>(1 + G);
            const uint32_t* any = nan_any + (fixes & 1) * 4;
            if (any[0] | any[1] | any[2] | any[3]) {
              // this thread's channel: the rows that see a key whose V is NaN there
              const uint32_t* words = nan_sh + (fixes & 1) * kPaTile * 4 + quarter;
#pragma unroll 1
              for (int kk = 0; kk < kPaTile; ++kk) {
                if (!(words[kk * 4] >> lane & 1u)) continue;
                const int at_key = k0 + kk;
#pragma unroll 1
                for (int r = 0; r < RG; ++r) {
                  const int at = row_pos[g * RG + r];
                  if ((!p.causal || at_key <= at) && (p.window <= 0 || at_key > at - p.window)) nan_rows |= 1u << r;
                }
              }
            }
            ++fixes;
          }
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        warp_arrive(&p_full[i & 1]);
      }
      // ---- the accumulator, the sum over the keys, then the result or what another block needs to go on
      ok = warp_wait(ok, &o_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1, abort_flag);
      tc_fence_after_sync();
      float o[RG];
      tmem_ld<RG>(t_o, reinterpret_cast<uint32_t*>(o));
      {
        float v[RG];
#pragma unroll
        for (int k = 0; k < RG / 2; ++k) f2_unpack(l2[k], v[2 * k], v[2 * k + 1]);
        // halves of the rows change lanes while the sums are formed: lane x ends with row x (RG = 32) or x / 2 (RG = 16)
        int width = RG;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          if (width > 1) {
            width >>= 1;
#pragma unroll
            for (int k = 0; k < RG / 2; ++k)
              if (k < width) {
                const float send = lane & d ? v[k] : v[k + width], keep = lane & d ? v[k + width] : v[k];
                v[k] = keep + __shfl_xor_sync(0xffffffffu, send, d);
              }
          } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
          }
        }
        if (RG == 32 || (lane & 1) == 0) max_sh[(sw & 3) * RG + (RG == 32 ? lane : lane >> 1)] = v[0];
      }
      group_sync(1 + g);
      const int row = g * RG + lane;  // of lanes < RG
      const float total = lane < RG ? (max_sh[lane] + max_sh[RG + lane]) + (max_sh[2 * RG + lane] + max_sh[3 * RG + lane]) : 0.f;
      tmem_wait_ld();
      if (nan_rows) {
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (nan_rows >> r & 1u) o[r] = __uint_as_float(0x7fffffffu);
      }
      if (off == 0 && n_seg == unit.tiles) {
        const bool owned = lane < RG && row < unit.rows;
        const int flat = unit.first + (owned ? row : 0), tok = flat / p.group, head = h * p.group + flat - tok * p.group;
        if (owned && ok) {
          if (p.lse && (sw & 3) == 0)
            p.lse[(int64_t)(ent.row0 + tok) * p.hq + head] = total != 0.f ? (m - kPaShift + log2f(total)) * 0.6931471805599453f : -INFINITY;
        }
        if (lane < RG) {
          inv_sh[lane] = total != 0.f ? 1.0f / total : 0.f;  // nothing seen: zero
          at_sh[lane] = (int64_t)(ent.row0 + tok) * p.o_st + (int64_t)head * p.o_sh;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (ok && g * RG + r < unit.rows) p.out[at_sh[r] + key] = __float2bfloat16_rn(o[r] * inv_sh[r]);
        __syncwarp();
      } else {
        const int64_t slot = 2 * (int64_t)blockIdx.x + (off == 0 ? 1 : 0);
        float* part = p.parts + slot * R * kHeadDim + (int64_t)g * RG * kHeadDim;
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (g * RG + r < unit.rows) part[r * kHeadDim + key] = o[r];
        if ((sw & 3) == 0 && lane < RG) p.stats[slot * R + row] = make_float2(m, total);
        if (off == 0 && sw == 0 && lane == 0)
          p.headers[blockIdx.x] = {1, b, h, j, (int)((t + unit.tiles - 1) / st.per_block), {0, 0, 0}};
      }
      ++units;
      t += n_seg;
      if (t < st.t1) next_unit();
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) *p.status = MAGI_E_TIMEOUT;
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// Joins the parts of a unit that several blocks worked on: block (i, r) takes row r of the unit that main block i left open,
// its eight warps take every eighth part, in the order of the keys.
template <int R>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedAttnKernelParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PaHeader hd = p.headers[blockIdx.x];
  if (!hd.open) return;
  bool bad;
  const PaEntry e = load_entry(p, hd.b, &bad);
  PaUnit u;
  unit_tiles<R>(p, e, hd.j, &u);
  const int r = blockIdx.y;
  if (r >= u.rows) return;
  __shared__ float s_max[8], s_sum[8];
  __shared__ float4 s_acc[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_parts = hd.last - blockIdx.x + 1;
  auto slot = [&](int k) { return k == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * (int64_t)(blockIdx.x + k); };
  float top = -INFINITY;
  for (int k = threadIdx.x; k < n_parts; k += 256) top = fmaxf(top, p.stats[slot(k) * R + r].x);
  top = warp_max(top);
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, s_max[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = warp; k < n_parts; k += 8) {
    const int64_t s = slot(k) * R + r;
    const float2 ml = p.stats[s];
    const float4 o = *reinterpret_cast<const float4*>(p.parts + s * kHeadDim + lane * 4);
    const float f = ex2(ml.x - ref);
    sum = fmaf(ml.y, f, sum);
    acc.x = fmaf(o.x, f, acc.x);
    acc.y = fmaf(o.y, f, acc.y);
    acc.z = fmaf(o.z, f, acc.z);
    acc.w = fmaf(o.w, f, acc.w);
  }
  s_acc[warp][lane] = acc;
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  float total = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    total += s_sum[w];
    o += reinterpret_cast<const float*>(s_acc[w])[threadIdx.x];
  }
  const int flat = u.first + r, tok = flat / p.group, head = hd.h * p.group + flat - tok * p.group;
  p.out[(int64_t)(e.row0 + tok) * p.o_st + (int64_t)head * p.o_sh + threadIdx.x] = __float2bfloat16_rn(total != 0.f ? o / total : 0.f);
  if (p.lse && threadIdx.x == 0)
    p.lse[(int64_t)(e.row0 + tok) * p.hq + head] = total != 0.f ? (top - kPaShift + log2f(total)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------------------------- host side
// Rows of a block's unit: up to 16 or 32 (query tokens times heads of a group) fit a form of which an SM holds two blocks;
// more go 96 at a time through the large one.
static int form_rows(int64_t max_q, int group) { return max_q * group <= 16 ? 16 : max_q * group <= 32 ? 32 : 96; }
static int form_blocks(const magi_ctx* ctx, int rows) { return ctx->sm_count * (rows == 96 ? 1 : 2); }

static int64_t workspace_bytes(const magi_ctx* ctx, int rows) {
  const int64_t blocks = form_blocks(ctx, rows);
  return blocks * (int64_t)sizeof(PaHeader) + 2 * blocks * rows * (kHeadDim * 4 + 8);
}

template <int RG, int G>
static int launch_paged(magi_ctx* ctx, const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnKernelParams& k, cudaStream_t st) {
  using L = PaShared<RG, G>;
  static bool configured[64] = {};  // per device: opt in to > 48 KB of dynamic shared memory once
  if (ctx->device >= 64 || !configured[ctx->device]) {
    MAGI_CUDA_OK(ctx, cudaFuncSetAttribute(paged_attn_kernel<RG, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamic));
    if (ctx->device < 64) configured[ctx->device] = true;
  }
  const int blocks = form_blocks(ctx, L::kRows);
  paged_attn_kernel<RG, G><<<blocks, L::kThreads, L::kDynamic, st>>>(tk, tv, k);
  MAGI_CUDA_OK(ctx, cudaGetLastError());
  const int64_t rows = (int64_t)k.max_q * k.group;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, (unsigned)(rows < L::kRows ? rows : L::kRows), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MAGI_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, paged_join_kernel<L::kRows>, k));
  return MAGI_OK;
}

}  // namespace magi

extern "C" int64_t magi_paged_attn_workspace_bytes(magi_ctx* ctx, int32_t max_q, int32_t n_q_heads, int32_t n_kv_heads) {
  if (!ctx || max_q < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads) return 0;
  return magi::workspace_bytes(ctx, magi::form_rows(max_q, n_q_heads / n_kv_heads));
}

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
  while ((1 << k.page_shift) < k.c.page_tokens) ++k.page_shift;
  k.rows_total = k.c.n_layers * k.c.n_pages * k.c.n_kv_heads * k.c.page_tokens;
  const int rows = form_rows(p->max_q, k.group);
  const int64_t blocks = form_blocks(ctx, rows);
  k.headers = static_cast<PaHeader*>(p->workspace);
  k.parts = reinterpret_cast<float*>(k.headers + blocks);
  k.stats = reinterpret_cast<float2*>(k.parts + 2 * blocks * rows * kHeadDim);
  CUtensorMap tk, tv;
  if (int rc = make_rows_map(ctx, &tk, cache->k8, k.rows_total, k.c.page_tokens, "paged attn k8")) return rc;
  if (int rc = make_rows_map(ctx, &tv, cache->v8, k.rows_total, k.c.page_tokens, "paged attn v8")) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 16) return launch_paged<16, 1>(ctx, tk, tv, k, st);
  if (rows == 32) return launch_paged<32, 1>(ctx, tk, tv, k, st);
  return launch_paged<32, 3>(ctx, tk, tv, k, st);
}
