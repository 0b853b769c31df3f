// Attention over the token-paged 8-bit cache, prompt form: more than 32 query rows per kv head, for sm_100a.
//
// Same products, precision and work split as the few-row form (paged_attn_sm100.cu), with the rows across: S [128 rows x 128
// keys] = Q K8^T and O [128 rows x 128 channels] = P V8, a thread owning a row.  Maximum, reference and sum of a row then live
// in its thread, and the fixed cost of a tile (barriers, tensor memory latency) is spread over 64 elements of each thread.
//
// A block works on 256 rows (query tokens times the heads of a kv head, flattened), two tiles of 128 that take turns on the
// tensor core.  K and V tiles are read once for all 256 rows.  Two warpgroups share a row tile, 64 keys each (and 64 channels of
// the result): with one, the latencies of its conversions lay open, 7000 cycles a tile.  They exchange the row maxima through
// shared memory, one barrier a tile.  P goes back over S in TMEM (32 keys: 8 columns for each of its three terms) and is the A
// operand of the second product from there.
//
// What bounds it: issue slots (56 % busy, about 14 instructions per weight) and the latency of tensor memory between them; the
// tensor pipe is busy 41 %, a fifth of that for the third term of P.  428 GFLOP over ragged prompts: 700 us; 996 GFLOP over one
// prompt of 9001 tokens: 1393 us, 715 TFLOP/s.  Steps on the way, on the ragged prompts: with two terms of P, which lost the
// weights of a long tail, 616 us, 629 with products and sums one at a time instead of in pairs; the third term with P stored 24
// words at a time (spills) 741, four at a time 684.  A tile's weights against the reference as it stands, checked afterwards, would
// save the pass for the maximum, but one of 128 rows asks for a new reference in most tiles: 926 us against 669 then.  A unit
// costs about five tiles to begin and end (739 us counted as 3 tiles and with the queries split 16 rows at a time, 674 at 4, 669
// at 5, 677 at 6).
//
//   warp 0 TMA, warp 1 UMMA issuer, warps 2, 3 idle, warps 4-19 softmax (warpgroup 2 x + half: row tile x, keys 64 half ..)
//   TMEM columns: S of row tile 0, 1 at 0, 128; O at 256, 384
#include <type_traits>

#include "paged_attn.cuh"

namespace magi {

int launch_prompt_join(magi_ctx* ctx, const PagedAttnKernelParams& k, cudaStream_t st);

struct PromptShared {
  static constexpr int kStages = 8;
  static constexpr int kSlots = 8;                             // tiles whose page scales are kept
  static constexpr int kCost = 5;                              // beginning and ending a unit, in tiles (see above)
  static constexpr int kThreads = 640;
  static constexpr int kRing = 0;
  static constexpr int kQ = kRing + kStages * kPaTileBytes;    // [2 terms][2 warpgroups][128 rows][128 bytes]
  static constexpr int kScales = kQ + 4 * kPaTileBytes;        // [kSlots][2][8]
  static constexpr int kNan = kScales + kSlots * 64;           // [2][128][4] channels whose V is NaN (boundary tiles)
  static constexpr int kNanAny = kNan + 2 * kPaTile * 16;      // [2][4] whether a warp's keys have any
  static constexpr int kTop = kNanAny + 32;                    // [2 buffers][2 row tiles][2 halves][128] row maxima, and sums at the end
  static constexpr int kRowS = kTop + 2 * 4 * 128 * 4;         // [2 row tiles][128] scale of a query row
  static constexpr int kNear = kRowS + 2 * 128 * 4;
  static constexpr int kStart = kNear + kPaNear * 16;
  static constexpr int kBar = kStart + 64;
  static constexpr int kNumBars = 2 * kStages + kSlots + 9;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kDynamic = kMisc + 16 + 1024;
};
static_assert(PromptShared::kDynamic <= 232448, "shared memory per block");
static_assert(PromptShared::kStages * kPaTileBytes >= kPlanScratch, "the plan's scratch is in the ring");

// The two warpgroups of row tile x.
__device__ __forceinline__ void pair_sync(int x) {
  __syncwarp();
  asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");
}
// kGroup: consecutive keys that share a page, and so scales, for sure (page_tokens, at most 32).
template <int kGroup>
__global__ void __launch_bounds__(PromptShared::kThreads, 1)
paged_prompt_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedAttnKernelParams p) {
  using L = PromptShared;
  constexpr int R = kPromptRows, kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* sc_full = kv_empty + kStages;
  uint64_t* q_full = sc_full + L::kSlots;  // [2] by row tile, as the next three
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* drain_bar = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  volatile int* progress = reinterpret_cast<volatile int*>(smem + L::kMisc + 8);  // tiles whose weights are through
  PaStart* start = reinterpret_cast<PaStart*>(smem + L::kStart);
  PaEntry* near = reinterpret_cast<PaEntry*>(smem + L::kNear);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < L::kSlots; ++s) mbar_init(&sc_full[s], 32);  // each lane of the loading warp
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 8);
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 8);
      mbar_init(&o_full[x], 1);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *progress = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  plan_tiles<R, L::kThreads, L::kCost>(p, smem + L::kRing, start, near);
  fence_proxy_async_smem();  // the ring goes over to TMA
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PaStart st = *start;
  PaWalk<R, L::kCost> walk(p, st, near);

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    __syncwarp();
    load_tiles<R, L::kCost, kStages, L::kSlots>(p, walk, &tm_k, &tm_v, smem + L::kRing, reinterpret_cast<float*>(smem + L::kScales), kv_full, kv_empty, sc_full, abort_flag);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ UMMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc(128, kPaTile, 0, 0, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc(128, kHeadDim, 1, 0, 0, 1);  // P is e5m2, V e4m3
      constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);  // 1024 bytes between groups of 8 rows, 128-byte swizzle
      const uint32_t ring = (smem_u32(smem + L::kRing) >> 4) | (1u << 16);
      const uint32_t q_lo = (smem_u32(smem + L::kQ) >> 4) | (1u << 16);
      constexpr uint32_t kTile16 = kPaTileBytes >> 4;
      bool ok = true;
      int i = 0;                       // tiles so far
      int seen[2] = {0, 0}, units[2] = {0, 0};  // key tiles and units of each row tile
      auto scores = [&](int x, int fill) {  // S of row tile x
        const uint32_t a = q_lo + x * kTile16, b = ring + (fill % kStages) * kTile16, d = tmem_base + x * 128;
        umma_ss_f8_lh<0>(d, a, b, desc_hi, idesc_s);
#pragma unroll
        for (int s = 1; s < 8; ++s)  // 32 channels per instruction; then the residual term
          umma_ss_f8_lh<1>(d, a + (s & 3) * 2 + (s >> 2) * 2 * kTile16, b + (s & 3) * 2, desc_hi, idesc_s);
        umma_commit(&s_full[x]);
      };
      for (; ok && walk.segment(); walk.advance()) {
        const int nx = walk.unit.rows > 128 ? 2 : 1;
        ok = mbar_wait(&kv_full[(2 * i) % kStages], (uint32_t)(2 * i / kStages) & 1, abort_flag);
        for (int x = 0; x < nx && ok; ++x) {
          ok = mbar_wait(&q_full[x], units[x]++ & 1, abort_flag);
          if (!ok) break;
          tc_fence_after_sync();
          scores(x, 2 * i);
        }
        if (ok) umma_commit(&kv_empty[(2 * i) % kStages]);
        for (int k = 0; k < walk.n_seg && ok; ++k, ++i) {
          *progress = i;
          const bool more = k + 1 < walk.n_seg;
          const int v_fill = 2 * i + 1, k_fill = 2 * i + 2;
          ok = mbar_wait(&kv_full[v_fill % kStages], (uint32_t)(v_fill / kStages) & 1, abort_flag);
          if (ok && more) ok = mbar_wait(&kv_full[k_fill % kStages], (uint32_t)(k_fill / kStages) & 1, abort_flag);
          for (int x = 0; x < nx && ok; ++x) {
            ok = mbar_wait(&p_full[x], seen[x]++ & 1, abort_flag);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t b = ring + (v_fill % kStages) * kTile16, d = tmem_base + 256 + x * 128, a = tmem_base + x * 128;
            if (k == 0) umma_ts_f8_lh<0>(d, a, b, desc_hi, idesc_o);
            else umma_ts_f8_lh<1>(d, a, b, desc_hi, idesc_o);
#pragma unroll
            for (int s = 1; s < 12; ++s)  // 32 keys per instruction: 8 columns of P, 32 rows of V; then the other two terms
              umma_ts_f8_lh<1>(d, a + (s & 3) * 32 + (s >> 2) * 8, b + (s & 3) * 256, desc_hi, idesc_o);
            if (!more) umma_commit(&o_full[x]);
            if (x == nx - 1) umma_commit(&kv_empty[v_fill % kStages]);
            if (more) {
              scores(x, k_fill);
              if (x == nx - 1) umma_commit(&kv_empty[k_fill % kStages]);
            }
          }
        }
      }
      if (!ok) {  // given up: the instructions issued so far still read shared memory and write TMEM
        int late = 0;
        umma_commit(drain_bar);
        mbar_wait(drain_bar, 0, &late, 100000000LL);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax and output
    // No early exits in here: a warp whose wait gave up goes on, so that the named barriers always meet.
    const int x = (warp - 4) >> 3, half = (warp - 4) >> 2 & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;  // of the tile's 128; also the key whose V row this thread looks after (x = half = 0)
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem_base + lane_base + x * 128, t_o = t_s + 256;
    const float* scales = reinterpret_cast<const float*>(smem + L::kScales);
    uint4* nan_sh = reinterpret_cast<uint4*>(smem + L::kNan);
    volatile uint32_t* nan_any = reinterpret_cast<uint32_t*>(smem + L::kNanAny);
    float* top_mine = reinterpret_cast<float*>(smem + L::kTop) + (x * 2 + half) * 128 + row;
    const float* top_other = reinterpret_cast<const float*>(smem + L::kTop) + (x * 2 + (half ^ 1)) * 128 + row;
    float* row_s = reinterpret_cast<float*>(smem + L::kRowS) + x * 128;
    int i = 0;                 // tiles of the block so far
    int seen = 0, units = 0;   // key tiles and units of this row tile
    for (; walk.segment(); walk.advance()) {
      const PaUnit& unit = walk.unit;
      const PaEntry& ent = walk.ent;
      const int n_seg = walk.n_seg, first = walk.first;
      const int nx = unit.rows > 128 ? 2 : 1;
      if (x >= nx) {  // a short unit leaves the second row tile out
        i += n_seg;
        continue;
      }
      // ---- 16 query rows per warp as two e4m3 terms
      const int flat = unit.first + x * 128 + row;
      const int tok = by_group(p, flat), head = walk.h * p.group + flat - tok * p.group;
      const bool owned = x * 128 + row < unit.rows;
      const long long q_at = (int64_t)(ent.row0 + tok) * p.q_st + (int64_t)head * p.q_sh;
      {
        uint2 raw[8];
        auto fetch = [&](int r0) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const long long at = __shfl_sync(0xffffffffu, q_at, r0 + r);
            raw[r] = make_uint2(0, 0);
            if (x * 128 + quarter * 32 + r0 + r < unit.rows) raw[r] = *reinterpret_cast<const uint2*>(p.q + at + lane * 4);
          }
        };
        fetch(half * 16);
#pragma unroll 1
        for (int r0 = half * 16; r0 < half * 16 + 16; r0 += 8) {
          uint2 now[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) now[r] = raw[r];
          if (r0 == half * 16) fetch(r0 + 8);  // in flight while the first eight are split
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            uint32_t hi, lo;
            const float scale = split_query(now[r], &hi, &lo);
            const int tr = quarter * 32 + r0 + r;
            uint8_t* at = smem + L::kQ + x * kPaTileBytes + tr * 128 + (((lane >> 2) ^ (tr & 7)) << 4) + (lane & 3) * 4;
            *reinterpret_cast<uint32_t*>(at) = hi;
            *reinterpret_cast<uint32_t*>(at + 2 * kPaTileBytes) = lo;
            row_s[tr] = scale;  // every lane the same
          }
        }
      }
      fence_proxy_async_smem();
      warp_arrive(&q_full[x]);
      warp_wait(&q_full[x], units & 1, abort_flag);  // the other half's row scales
      const float c1 = row_s[row] * p.scale_log2;
      const int at_pos = ent.len - ent.n_q + tok, from = window_begin(p, at_pos);
      float m = -INFINITY;                  // reference maximum, at most kPaLimit - kPaShift below the running one
      float l = 0.f;                        // sum of the weights
      uint32_t nan_ch[4] = {0, 0, 0, 0};    // channels of this row that are NaN (boundary tiles)
#pragma unroll 1
      for (int k = 0; k < n_seg; ++k, ++i, ++seen) {
        const int k0 = (unit.tile0 + first + k) * kPaTile;
        // The scores first: row tile 1 leaves short units out without waiting for their tiles, so that its slot of the scales may be
        // more than one fill behind, which the parity does not show.  Scores of tile i are issued behind row tile 0's weights of the
        // tile before, and row tile 0 waits for the scales of every tile: the slot is then in tile i's phase or has completed it.
        warp_wait(&s_full[x], seen & 1, abort_flag, progress);  // row tile 1 sits out any number of short units
        warp_wait(&sc_full[i % L::kSlots], (uint32_t)(i / L::kSlots) & 1, abort_flag);
        tc_fence_after_sync();
        const float* sc = scales + (i % L::kSlots) * 16;
        const bool tail = k0 + kPaTile > ent.len;  // keys behind the sequence's end
        // keys before it that not every row sees
        const bool edge = (p.causal && min(k0 + kPaTile, ent.len) - 1 > unit.pos_a) || k0 < window_begin(p, unit.pos_z);
        const bool border = __any_sync(0xffffffffu, tail || edge);  // the vote lets the branches on it be uniform ones
        const int last = min(p.causal ? at_pos : ent.len - 1, ent.len - 1) - k0;               // columns [begin, last] are seen
        const int begin = max(from - k0, 0);
        // 32 keys at a time, twice over: the scores stay in TMEM in between, so that a thread holds 32 of them and not all.
        // w = s log2e + log2(sv) = raw * kc + bias; the sum adds P / sv.
        constexpr int kPer = 32 / kGroup;
        auto factors = [&](int at, float (&kc)[kPer], float (&bias)[kPer], float (&inv)[kPer]) {
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
            const int pg = (at + g * kGroup) >> p.page_shift;
            const uint32_t vs = __float_as_uint(sc[8 + pg]);
            kc[g] = fminf(sc[pg] * c1, 3.0e38f);  // finite: a raw score of zero stays zero
            bias[g] = __uint_as_float(0x4b000000u | vs >> 23) - 8388735.0f;  // its exponent: 2^23 + (e + 127) - (2^23 + 127)
            inv[g] = at + g * kGroup <= last ? __uint_as_float(0x7f000000u - vs) : 0.f;  // behind the end there may be no page
          }
        };
        // At the borders: columns that no row of this warp sees are left out, those that all rows see are like any other.
        int all_last = 0, all_begin = 0, any_last = 0, any_begin = 0;
        if (border) {
          all_last = __reduce_min_sync(0xffffffffu, last), all_begin = __reduce_max_sync(0xffffffffu, begin);
          any_last = __reduce_max_sync(0xffffffffu, last), any_begin = __reduce_min_sync(0xffffffffu, begin);
        }
        auto hidden = [&](int at) { return at > any_last || at + 31 < any_begin; };
        auto mixed = [&](int at) { return at + 31 > all_last || at < all_begin; };
        float top = -INFINITY;
        // The largest exponent of 32 keys.  It belongs to the largest score of a page, as kc is not negative.
        auto find_top = [&](int at, float (&s)[32]) {
          if (border && mixed(at)) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = at + c <= last && at + c >= begin ? s[c] : -INFINITY;
          }
          float kc[kPer], bias[kPer], inv[kPer];
          factors(at, kc, bias, inv);
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
            float t0 = fmaxf(s[g * kGroup], s[g * kGroup + 1]), t1 = fmaxf(s[g * kGroup + 2], s[g * kGroup + 3]);
#pragma unroll
            for (int c = g * kGroup + 4; c < (g + 1) * kGroup; c += 4) {
              t0 = max3(t0, s[c], s[c + 1]);
              t1 = max3(t1, s[c + 2], s[c + 3]);
            }
            t0 = fmaxf(t0, t1);
            top = fmaxf(top, t0 == -INFINITY ? t0 : fmaf(t0, kc[g], bias[g]));
          }
        };
        if (!border) {
          float s0[32], s1[32];
          tmem_ld32(t_s + half * 64, reinterpret_cast<uint32_t*>(s0));
          tmem_ld32(t_s + half * 64 + 32, reinterpret_cast<uint32_t*>(s1));
          tmem_wait_ld();
          find_top(half * 64, s0);
          find_top(half * 64 + 32, s1);
        } else {
#pragma unroll 1
          for (int at = half * 64; at < half * 64 + 64; at += 32)
            if (!hidden(at)) {
              float s[32];
              tmem_ld32(t_s + at, reinterpret_cast<uint32_t*>(s));
              tmem_wait_ld();
              find_top(at, s);
            }
        }
        top_mine[(seen & 1) * 512] = top;
        pair_sync(x);
        top = fmaxf(top, top_other[(seen & 1) * 512]);
        const bool need = top > m + (kPaLimit - kPaShift);
        if (__any_sync(0xffffffffu, need)) {
          // some row's reference is too low (always so in a unit's first tile): it becomes the maximum
          const float m_new = need ? top : m;
          const float f = need ? ex2(m - m_new) : 1.0f;
          m = m_new;
          l *= f;
          if (k > 0) {  // what the tensor core has summed so far: this tile's scores were issued behind it
#pragma unroll 1
            for (int c = half * 2; c < half * 2 + 2; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
              tmem_st32(t_o + c * 32, o);
            }
          }
        }
        // ---- weights, their sum, and P as three terms: 32 keys at the first 24 of their scores' columns
        const float plus = m == -INFINITY ? 0.f : kPaShift - m;
        auto weigh_keys = [&](int at) {
          float s[32], kc[kPer], bias[kPer], inv[kPer];
          uint64_t sum[kPer], kc2[kPer], bias2[kPer];
          tmem_ld32(t_s + at, reinterpret_cast<uint32_t*>(s));
          factors(at, kc, bias, inv);
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
            bias[g] += plus;
            sum[g] = 0;
            kc2[g] = f2_pack(kc[g], kc[g]);
            bias2[g] = f2_pack(bias[g], bias[g]);
          }
          tmem_wait_ld();
          uint32_t w[12];
          auto weigh = [&](auto masked) {  // exponentials and conversions run in different pipes: four keys of each in turn
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const int g = c / kGroup, k4 = c / 4 & 3;
              float p[4];
              f2_unpack(f2_fma(f2_pack(s[c], s[c + 1]), kc2[g], bias2[g]), p[0], p[1]);
              f2_unpack(f2_fma(f2_pack(s[c + 2], s[c + 3]), kc2[g], bias2[g]), p[2], p[3]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                p[e] = ex2(p[e]);
                if constexpr (decltype(masked)::value) p[e] = at + c + e <= last && at + c + e >= begin ? p[e] : 0.f;
              }
              sum[g] = f2_add(sum[g], f2_add(f2_pack(p[0], p[1]), f2_pack(p[2], p[3])));
              split_weights(p[0], p[1], p[2], p[3], &w[k4], &w[4 + k4], &w[8 + k4]);
              if (k4 == 3) {
                tmem_st4(t_s + at + c / 16 * 4, w);
                tmem_st4(t_s + at + 8 + c / 16 * 4, w + 4);
                tmem_st4(t_s + at + 16 + c / 16 * 4, w + 8);
              }
            }
          };
          if (border && mixed(at)) weigh(std::true_type());
          else weigh(std::false_type());
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
            float a, b;
            f2_unpack(sum[g], a, b);
            l = fmaf(a + b, inv[g], l);
          }
        };
        if (!border) {
          weigh_keys(half * 64);
          weigh_keys(half * 64 + 32);
        } else {
#pragma unroll 1
          for (int at = half * 64; at < half * 64 + 64; at += 32) {
            if (hidden(at)) {
              uint32_t w[16];
#pragma unroll
              for (int c = 0; c < 16; ++c) w[c] = 0;
              tmem_st16(t_s + at, w);
              tmem_st8(t_s + at + 16, w);
            } else {
              weigh_keys(at);
            }
          }
        }
        if (border) {
          // A weight of zero does not silence a NaN: V of keys behind the end becomes zero, and NaN codes of keys that only
          // some rows see are taken out of the product and come back in the rows that do see them.
          const int v_fill = 2 * i + 1, buf = i & 1;
          if (x == 0 && half == 0) {
            warp_wait(&kv_full[v_fill % kStages], (uint32_t)(v_fill / kStages) & 1, abort_flag);
            uint4* vrow = reinterpret_cast<uint4*>(smem + L::kRing + (v_fill % kStages) * kPaTileBytes + row * 128);
            if (k0 + row >= ent.len) {
#pragma unroll
              for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0, 0, 0, 0);
            }
            if (edge) {
              uint32_t bits[4] = {0, 0, 0, 0};
              if (k0 + row < ent.len) take_nan(vrow, row, bits);
              nan_sh[buf * kPaTile + row] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
              nan_any[buf * 4 + quarter] = __any_sync(0xffffffffu, (bits[0] | bits[1] | bits[2] | bits[3]) != 0);  // every lane the same
            }
            fence_proxy_async_smem();
          }
          if (edge) {
            // Row tile 0 goes on when its two halves are through; row tile 1, which runs behind it, waits for its list.  Row tile 0
            // can be a tile ahead (its next scores are issued before row tile 1's weights are waited for), so the barrier and
            // the list go by the tile's parity.
            if (x == 0) {
              pair_sync(0);
              if (nx == 2 && half == 0) asm volatile("bar.arrive %0, 384;" ::"r"(3 + buf) : "memory");
            } else {
              __syncwarp();
              asm volatile("bar.sync %0, 384;" ::"r"(3 + buf) : "memory");
            }
            const volatile uint32_t* any = nan_any + buf * 4;
            if (any[0] | any[1] | any[2] | any[3]) {
#pragma unroll 1
              for (int kk = max(begin, 0); kk <= min(last, kPaTile - 1); ++kk) {
                const uint4 w = nan_sh[buf * kPaTile + kk];
                nan_ch[0] |= w.x;
                nan_ch[1] |= w.y;
                nan_ch[2] |= w.z;
                nan_ch[3] |= w.w;
              }
              __syncwarp();
            }
          }
        }
        tmem_wait_st();
        tc_fence_before_sync();
        warp_arrive(&p_full[x]);
      }
      // ---- the result, or what another block needs to go on
      warp_wait(&o_full[x], units & 1, abort_flag);
      const bool ok = *abort_flag == 0;
      ++units;
      tc_fence_after_sync();
      top_mine[0] = l;  // the maxima of the last tile have been read by both halves before its scores were consumed ...
      pair_sync(x);
      const float total = l + top_other[0];
      pair_sync(x);     // ... and the sums before the next tile's maxima
      const bool whole = walk.whole();
      const float inv = whole ? (total != 0.f ? 1.0f / total : 0.f) : 1.0f;  // nothing seen: zero
      const int64_t slot = (2 * (int64_t)blockIdx.x + (first == 0 ? 1 : 0)) * R + x * 128 + row;
      __nv_bfloat16* out = p.out + (int64_t)(ent.row0 + (owned ? tok : 0)) * p.o_st + (int64_t)head * p.o_sh;
      float* part = p.parts + (slot - x * 128 - row) * kHeadDim + (x * 128 + row) * 4;  // [channel / 4][row][4]
#pragma unroll 1
      for (int c = half * 2; c < half * 2 + 2; ++c) {
        float o[32];
        tmem_ld32(t_o + c * 32, reinterpret_cast<uint32_t*>(o));
        tmem_wait_ld();
        const uint32_t nan_bits = c == 0 ? nan_ch[0] : c == 1 ? nan_ch[1] : c == 2 ? nan_ch[2] : nan_ch[3];
#pragma unroll
        for (int q = 0; q < 32; ++q) o[q] = nan_bits >> q & 1u ? __uint_as_float(0x7fffffffu) : o[q] * inv;
        if (owned && ok) {
          if (whole) {
#pragma unroll
            for (int q = 0; q < 32; q += 8)
              *reinterpret_cast<uint4*>(out + c * 32 + q) = make_uint4(pack_bf16x2(o[q], o[q + 1]), pack_bf16x2(o[q + 2], o[q + 3]), pack_bf16x2(o[q + 4], o[q + 5]), pack_bf16x2(o[q + 6], o[q + 7]));
          } else {
#pragma unroll
            for (int q = 0; q < 32; q += 4) *reinterpret_cast<float4*>(part + (c * 32 + q) * R) = make_float4(o[q], o[q + 1], o[q + 2], o[q + 3]);
          }
        }
        __syncwarp();
      }
      if (owned && half == 0) {
        if (!whole) p.stats[slot] = make_float2(m, total);
        else if (p.lse && ok)
          p.lse[(int64_t)(ent.row0 + tok) * p.hq + head] = total != 0.f ? (m - kPaShift + log2f(total)) * 0.6931471805599453f : -INFINITY;
      }
      if (!whole && first == 0 && threadIdx.x == 128)
        p.headers[blockIdx.x] = {1, walk.last_block(st.per_block), ent.row0, walk.h, unit.first, unit.rows, {0, 0}};
      __syncwarp();
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) *p.status = MAGI_E_TIMEOUT;
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

int launch_paged_prompt(magi_ctx* ctx, const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnKernelParams& k, cudaStream_t st) {
  static bool configured[64] = {};  // per device: opt in to > 48 KB of dynamic shared memory once
  if (ctx->device >= 64 || !configured[ctx->device]) {
    MAGI_CUDA_OK(ctx, cudaFuncSetAttribute(paged_prompt_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShared::kDynamic));
    MAGI_CUDA_OK(ctx, cudaFuncSetAttribute(paged_prompt_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShared::kDynamic));
    if (ctx->device < 64) configured[ctx->device] = true;
  }
  const auto kernel = k.c.page_tokens == 16 ? paged_prompt_kernel<16> : paged_prompt_kernel<32>;
  kernel<<<ctx->sm_count, PromptShared::kThreads, PromptShared::kDynamic, st>>>(tk, tv, k);
  MAGI_CUDA_OK(ctx, cudaGetLastError());
  return launch_prompt_join(ctx, k, st);
}

}  // namespace magi
