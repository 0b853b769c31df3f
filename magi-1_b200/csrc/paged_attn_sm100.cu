// Attention over the token-paged 8-bit cache, for sm_100a: few query rows per kv head (new tokens), and the entry point.
//
//   s = scale * q . (k8 sk),  o = sum_k softmax(s)_k (v8 sv),  sk, sv powers of two per (page, kv head)
//
// The scores are formed TRANSPOSED, S^T [128 keys x R rows] = K8 Q^T and O^T [128 channels x R rows] = V8^T P^T, so that
// the long side of every product is the cache: the e4m3 tiles go from HBM through TMA and shared memory to tcgen05.mma
// (kind::f8f6f4, M = 128) exactly as they are stored, nothing is ever converted to a wider type, and a tile costs the same
// few instructions whether a sequence has one new token (R = 16 covers 16 query heads of a kv head) or several (R = 32).  K8
// is the K-major A operand of the first product, V8 - stored [key][channel] - the MN-major A operand of the second.
//
// Precision: Q is carried as two e4m3 terms, P as three e5m2 ones (value, then what is left of it, added up by the tensor core).
// bf16 has 8 significant bits and two e4m3 terms hold 8, so Q loses nothing except what lies 2^-17 below its row's largest entry;
// P is off by 2^-9 of a weight and 2^-29 of the reference at most, V's scale included (two terms, e4m3 and e5m2, kept 2^-7 of a
// weight down to 2^-11 of the reference and 2^-3 below 2^-16: a result that many small weights bring, behind one key that holds
// most of the mass, was off by several per cent).  Sums and maxima are fp32 in registers, the output accumulator fp32 in TMEM.
// The V scale is folded into the exponent, w = s log2e + log2(sv), and a row's reference is taken over w: then P stays within
// e5m2 however different the pages' scales are, O needs no scale per page and the denominator adds P / sv.
//
// Work: the 128-key tiles of all (sequence, kv head, row tile) units in a row are dealt out to the blocks in equal
// contiguous parts, so a long sequence is split over many blocks and ragged batches balance; the lengths are read on the
// device.  A block finishes the units that lie inside its part; for the (at most two) that do not it leaves maximum, sum
// and accumulator in the workspace, and a second kernel joins them in the order of the keys (no atomics: the same bits
// every time).
//
// What bounds it: HBM, once the batch fills the machine (8 sequences of 10^5 tokens, 1.9 GB: 303 us, 97 % of the copy rate;
// 64 of 300 to 8191: 104 us, of which 7 pass until the first tile is in and 3 in the join), else the latencies of one tile: plan 2 us,
// first tile 2, softmax and output 2, join 2.  Two blocks per SM with five stages of 16 KB: one's softmax hides behind the
// other's loads (three with three stages: 121 us for the batch, against 108 then).
//
//   warp 0     TMA: pages of K and V into a ring of 16 KB tiles, their scales by cp.async beside them
//   warp 1     UMMA issuer (one thread)
//   warps 2+   R / 16 groups of four: thread = key of S^T, then channel of O^T; a group takes 16 of the R rows (32 rows in one
//              group: 21 us against 16.5 for 16 sequences of 2 to 5 tokens with a window of 4099)
// Every wait is bounded (MAGI_E_TIMEOUT).
#include "paged_attn.cuh"

namespace magi {

int make_rows_map(magi_ctx* ctx, CUtensorMap* m, const void* base, int rows, int box_rows, const char* what);
int launch_paged_prompt(magi_ctx* ctx, const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnKernelParams& k, cudaStream_t st);

template <int R>
struct PaShared {
  static constexpr int kStages = R == 16 ? 5 : 4;
  static constexpr int kBlocksPerSm = 2;
  static constexpr int kSlots = 8;                             // tiles whose page scales are kept
  // beginning and ending a unit, in tiles (64 sequences of 300 to 8191: 121 us at 1, 112 at 2, 108 at 4, 110 at 6)
  static constexpr int kCost = 4;
  static constexpr int kGroups = R / 16;                       // of four softmax warps, 16 rows each
  static constexpr int kThreads = 64 + 128 * kGroups;
  static constexpr int kRing = 0;
  // P, a byte per (key, row) and term, two buffers, in tiles of 128-byte rows [key], eight pieces of 16 bytes each; the lists of
  // channels whose V is NaN (boundary tiles) are in pieces that P leaves free.
  //   R = 16: one tile, term t of buffer b in piece 4 b + t, the list in piece 3
  //   R = 32: terms 0 and 1 of buffer b in pieces 4 b and 4 b + 2 of the first tile (two pieces each), term 2 in 2 b of the second,
  //           where lists 0 and 1 are in pieces 4 and 5
  // Terms 0 and 1 side by side are one operand of 2 R rows: with an instruction for each term (12 instead of 8 a tile) 8 sequences
  // of 10^5 tokens took 312 us instead of 290.
  static constexpr int kP = kRing + kStages * kPaTileBytes;
  static constexpr int kPTiles = R / 16;
  static constexpr int kQ = kP + kPTiles * kPaTileBytes;       // [2 terms][R][128 bytes]
  __host__ __device__ static constexpr int piece(int term, int buffer) {  // of 16 bytes, its tile's 1024 included
    return R == 16 ? buffer * 4 + term : term == 2 ? kPaTileBytes / 16 + buffer * 2 : buffer * 4 + term * 2;
  }
  static constexpr int kScales = kQ + 2 * R * 128;             // [kSlots][2][8]
  static constexpr int kMax = kScales + kSlots * 64;           // [4][R] warp maxima, and sums at a unit's end
  static constexpr int kNegM = kMax + 4 * R * 4;               // [R]
  static constexpr int kFactor = kNegM + R * 4;                // [R]
  static constexpr int kRowS = kFactor + R * 4;                // [2][R] scale of a query row
  static constexpr int kRowKeys = kRowS + 2 * R * 4;           // [2][R] the keys it sees: first one, how many
  static constexpr int kInv = kRowKeys + 2 * R * 8;            // [4][R]
  static constexpr int kAt = kInv + 4 * R * 4;                 // [4][R] where a row of the result starts
  static constexpr int kNan = kP + (kPTiles - 1) * kPaTileBytes;  // tile of the lists
  static constexpr int kNanPiece = R == 16 ? 3 : 4;            // the first one's piece
  static constexpr int kNanAny = kAt + 4 * R * 8;              // [kGroups][4] whether a warp's keys have any
  static constexpr int kNear = kNanAny + kGroups * 16;         // [kPaNear] entries
  static constexpr int kStart = kNear + kPaNear * 16;
  static constexpr int kBar = kStart + 64;
  static constexpr int kNumBars = 2 * kStages + kSlots + 8;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kTotal = kMisc + 16;
  static constexpr int kDynamic = kTotal + 1024;
  static constexpr uint32_t kTmemCols = 4 * R;                 // S twice; O of the terms 0 and 2, O of term 1
  static_assert(kDynamic * kBlocksPerSm + 1024 * kBlocksPerSm <= 233472, "blocks of an SM share its memory");
  static_assert(kStages * kPaTileBytes >= kPlanScratch, "the plan's scratch is in the ring");
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Barriers of the four softmax warps of group g.  A warp counts once only if its lanes arrive together.
__device__ __forceinline__ bool group_any(int g, bool v) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.u32 a, %1, 0;\n\t"
      "bar.red.or.pred b, %2, 128, a;\n\t"
      "selp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(1 + g)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int g) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
}
template <int R>
__global__ void __launch_bounds__(PaShared<R>::kThreads, PaShared<R>::kBlocksPerSm)
paged_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ PagedAttnKernelParams p) {
  using L = PaShared<R>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* sc_full = kv_empty + kStages;  // page scales of a tile
  uint64_t* s_full = sc_full + L::kSlots;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* q_full = o_full + 2;
  uint64_t* drain_bar = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
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
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4 * L::kGroups);
      mbar_init(&o_full[x], 1);
    }
    mbar_init(q_full, 4 * L::kGroups);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
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
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    load_tiles<R, L::kCost, kStages, L::kSlots>(p, walk, &tm_k, &tm_v, smem + L::kRing, reinterpret_cast<float*>(smem + L::kScales), kv_full, kv_empty, sc_full, abort_flag);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ UMMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc(kPaTile, R, 0, 0, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc(kHeadDim, 2 * R, 0, 1, 1, 1), idesc_r = umma_idesc(kHeadDim, R, 0, 1, 1, 1);  // V is e4m3, P e5m2
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
        const uint32_t a = ring + stage * (kPaTileBytes >> 4), bb = p_lo + L::piece(0, k & 1), br = p_lo + L::piece(2, k & 1);
        if (opens) umma_ss_f8_lh<0>(d, a, bb, desc_hi, idesc_o);
        else umma_ss_f8_lh<1>(d, a, bb, desc_hi, idesc_o);
#pragma unroll
        for (int s = 1; s < 4; ++s) umma_ss_f8_lh<1>(d, a + s * 256, bb + s * 256, desc_hi, idesc_o);  // 32 keys per instruction
#pragma unroll
        for (int s = 0; s < 4; ++s) umma_ss_f8_lh<1>(d, a + s * 256, br + s * 256, desc_hi, idesc_r);
        umma_commit(&o_full[k & 1]);
        umma_commit(&kv_empty[stage]);
      };
      for (; ok && walk.segment(); walk.advance()) {
        if (pending) second(i - 1);  // the next unit's rows are written only after the last tile of this one is through
        pending = false;
        if (ok) ok = mbar_wait(q_full, units & 1, abort_flag);
        for (int x = 0; x < walk.n_seg && ok; ++x, ++i) {
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
      }
      if (ok && pending) second(i - 1);
      if (!ok) {  // given up: the instructions issued so far still read shared memory and write TMEM
        int late = 0;
        umma_commit(drain_bar);
        mbar_wait(drain_bar, 0, &late, 100000000LL);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output
    // No early exits in here: a warp whose wait gave up goes on, so that the named barriers always meet.
    constexpr int RG = 16;                    // rows of a group
    const int sw = warp - 2, g = sw >> 2, wq = sw & 3;
    const int quarter = warp & 3;             // TMEM lanes of this warp
    const int key = quarter * 32 + lane;      // key of the tile; channel of the output
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_o = tmem_base + lane_base + 2 * R + g * RG;
    const float* scales = reinterpret_cast<const float*>(smem + L::kScales);
    float* max_sh = reinterpret_cast<float*>(smem + L::kMax) + g * 4 * RG;
    float* neg_m = reinterpret_cast<float*>(smem + L::kNegM) + g * RG;  // kPaShift - reference maximum of a row
    float* factor = reinterpret_cast<float*>(smem + L::kFactor) + g * RG;
    float* inv_sh = reinterpret_cast<float*>(smem + L::kInv) + sw * RG;
    int64_t* at_sh = reinterpret_cast<int64_t*>(smem + L::kAt) + sw * RG;
    int i = 0, units = 0;
    for (; walk.segment(); walk.advance()) {
      const PaUnit& unit = walk.unit;
      const PaEntry& ent = walk.ent;
      const int n_seg = walk.n_seg, first = walk.first, h = walk.h;
      float* row_s = reinterpret_cast<float*>(smem + L::kRowS) + (units & 1) * R;
      int2* row_keys = reinterpret_cast<int2*>(smem + L::kRowKeys) + (units & 1) * R;
      // ---- query rows of the unit as two e4m3 terms, each row scaled by a power of two so that its largest entry is in (224, 448]
      {
        constexpr int kMine = 4, kWarps = 4 * L::kGroups;
        uint2 raw[kMine];
        int toks[kMine];
#pragma unroll
        for (int x = 0; x < kMine; ++x) {
          const int r = sw + x * kWarps, flat = unit.first + r;
          toks[x] = by_group(p, flat);
          raw[x] = make_uint2(0, 0);
          if (r < unit.rows)
            raw[x] = *reinterpret_cast<const uint2*>(p.q + (int64_t)(ent.row0 + toks[x]) * p.q_st + (int64_t)(h * p.group + flat - toks[x] * p.group) * p.q_sh + lane * 4);
        }
#pragma unroll
        for (int x = 0; x < kMine; ++x) {
          const int r = sw + x * kWarps;
          uint32_t hi, lo;
          const float scale = split_query(raw[x], &hi, &lo);
          uint8_t* to = smem + L::kQ + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(to) = hi;
          *reinterpret_cast<uint32_t*>(to + R * 128) = lo;
          row_s[r] = scale * p.scale_log2;  // every lane the same
          const int at = ent.len - ent.n_q + toks[x], from = window_begin(p, at);
          row_keys[r] = make_int2(from, max((p.causal ? min(at + 1, ent.len) : ent.len) - from, 0));
        }
      }
      fence_proxy_async_smem();
      warp_arrive(q_full);
      warp_wait(q_full, units & 1, abort_flag);  // the other warps' row scales and positions
      float m = -INFINITY;    // lane r < RG: reference maximum of row r of the group, at most kPaLimit - kPaShift below the running one
      uint32_t nan_rows = 0;  // rows whose result in this thread's channel is NaN (boundary tiles)
      uint64_t l2[RG / 2];    // sums over this thread's keys, rows in pairs
#pragma unroll
      for (int k = 0; k < RG / 2; ++k) l2[k] = 0;
      const float4* s4 = reinterpret_cast<const float4*>(row_s + g * RG);
      const float4* n4 = reinterpret_cast<const float4*>(neg_m);
#pragma unroll 1
      for (int x = 0; x < n_seg; ++x, ++i) {
        const int k0 = (unit.tile0 + first + x) * kPaTile, pos = k0 + key;
        warp_wait(&sc_full[i % L::kSlots], (uint32_t)(i / L::kSlots) & 1, abort_flag);
        warp_wait(&s_full[i & 1], (uint32_t)(i >> 1) & 1, abort_flag);
        const bool tail = k0 + kPaTile > ent.len;                                             // keys behind the sequence's end
        // keys before it that not every row sees
        const bool edge = (p.causal && min(k0 + kPaTile, ent.len) - 1 > unit.pos_a) || k0 < window_begin(p, unit.pos_z);
        tc_fence_after_sync();
        const uint32_t t_s = tmem_base + lane_base + (i & 1) * R + g * RG;
        float w[RG];  // exponents of the weights: s log2e + log2(sv) - reference + kPaShift
        tmem_ld16(t_s, reinterpret_cast<uint32_t*>(w));
        const float ks = scales[(i % L::kSlots) * 16 + (key >> p.page_shift)];
        const uint32_t vs = __float_as_uint(scales[(i % L::kSlots) * 16 + 8 + (key >> p.page_shift)]);
        const float bias = (float)((int)(vs >> 23) - 127);                                    // log2 of a power of two
        const float inv_vs = pos < ent.len ? __uint_as_float(0x7f000000u - vs) : 0.f;         // behind the end there is no page
        const uint64_t ks2 = f2_pack(ks, ks), bias2 = f2_pack(bias, bias);
        auto hide = [&]() {
          const int4* keys = reinterpret_cast<const int4*>(row_keys + g * RG);
#pragma unroll
          for (int r = 0; r < RG; r += 2) {
            const int4 k = keys[r / 2];
            if ((uint32_t)(pos - k.x) >= (uint32_t)k.y) w[r] = -INFINITY;
            if ((uint32_t)(pos - k.z) >= (uint32_t)k.w) w[r + 1] = -INFINITY;
          }
        };
        tmem_wait_ld();
        bool low = x == 0;  // some row's reference is too low (there is none in a unit's first tile)
        if (!low) {
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
          low = group_any(g, top > kPaLimit);
        }
        if (low) {
          // ---- the exact maxima, from the scores again
          if (x > 0) {
            tmem_ld16(t_s, reinterpret_cast<uint32_t*>(w));
            tmem_wait_ld();
          }
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
          if (lane < RG) max_sh[wq * RG + lane] = mine;
          group_sync(g);
          if (lane < RG) {
            const float m_new = fmaxf(fmaxf(fmaxf(m, max_sh[lane]), max_sh[RG + lane]), fmaxf(max_sh[2 * RG + lane], max_sh[3 * RG + lane]));
            if (wq == 0) {
              neg_m[lane] = kPaShift - m_new;
              factor[lane] = m_new == -INFINITY ? 1.0f : ex2(m - m_new);
            }
            m = m_new;
          }
          group_sync(g);
          const float4* f4 = reinterpret_cast<const float4*>(factor);
#pragma unroll
          for (int r = 0; r < RG; r += 4) {
            const float4 n = n4[r / 4];
            w[r] = w[r] == -INFINITY ? w[r] : w[r] + n.x;
            w[r + 1] = w[r + 1] == -INFINITY ? w[r + 1] : w[r + 1] + n.y;
            w[r + 2] = w[r + 2] == -INFINITY ? w[r + 2] : w[r + 2] + n.z;
            w[r + 3] = w[r + 3] == -INFINITY ? w[r + 3] : w[r + 3] + n.w;
          }
          if (x > 0) {  // what has been summed so far, here and by the tensor core
            warp_wait(&o_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1, abort_flag);
            tc_fence_after_sync();
#pragma unroll
            for (int r = 0; r < RG; r += 4) {
              const float4 f = f4[r / 4];
              l2[r / 2] = f2_mul(l2[r / 2], f2_pack(f.x, f.y));
              l2[r / 2 + 1] = f2_mul(l2[r / 2 + 1], f2_pack(f.z, f.w));
            }
#pragma unroll 1
            for (uint32_t t = t_o; t <= t_o + R; t += R) {
              uint32_t o[RG];
              tmem_ld16(t, o);
              tmem_wait_ld();
#pragma unroll
              for (int r = 0; r < RG; r += 4) {
                const float4 f = f4[r / 4];
                o[r] = __float_as_uint(__uint_as_float(o[r]) * f.x);
                o[r + 1] = __float_as_uint(__uint_as_float(o[r + 1]) * f.y);
                o[r + 2] = __float_as_uint(__uint_as_float(o[r + 2]) * f.z);
                o[r + 3] = __float_as_uint(__uint_as_float(o[r + 3]) * f.w);
              }
              tmem_st16(t, o);
            }
            tmem_wait_st();
          }
        }
        // ---- weights, their sum, and P as three terms
        uint32_t t0[RG / 4], t1[RG / 4], t2[RG / 4];
        const uint64_t inv2 = f2_pack(inv_vs, inv_vs);
#pragma unroll
        for (int r = 0; r < RG; r += 4) {
          const float p0 = ex2(w[r]), p1 = ex2(w[r + 1]), p2 = ex2(w[r + 2]), p3 = ex2(w[r + 3]);
          l2[r / 2] = f2_fma(f2_pack(p0, p1), inv2, l2[r / 2]);
          l2[r / 2 + 1] = f2_fma(f2_pack(p2, p3), inv2, l2[r / 2 + 1]);
          split_weights(p0, p1, p2, p3, &t0[r / 4], &t1[r / 4], &t2[r / 4]);
        }
        // the buffer of tile i - 2
        if (i >= 2) warp_wait(&o_full[i & 1], (uint32_t)((i - 2) >> 1) & 1, abort_flag);
        uint8_t* pb = smem + L::kP + key * 128;
        auto place = [&](int term) {  // 128-byte swizzle: a row's pieces change places by the key
          const int at = L::piece(term, i & 1) + g;
          return reinterpret_cast<uint4*>(pb + (at >> 10) * kPaTileBytes + (((at & 7) ^ (key & 7)) << 4));
        };
        *place(0) = make_uint4(t0[0], t0[1], t0[2], t0[3]);
        *place(1) = make_uint4(t1[0], t1[1], t1[2], t1[3]);
        *place(2) = make_uint4(t2[0], t2[1], t2[2], t2[3]);
        if (tail || edge) {
          // A weight of zero does not silence a NaN: V of keys behind the end becomes zero, and NaN codes of keys that only
          // some rows see are taken out of the product and come back through the sums of the rows that do see them.  The first
          // group does that; the second can be a tile behind it, not two, so the lists go by the tile's parity.
          const int v_fill = 2 * i + 1, v_stage = v_fill % kStages, buf = i & (L::kGroups - 1);
          auto nan_of = [&](int k) { return reinterpret_cast<uint4*>(smem + L::kNan + k * 128 + (((L::kNanPiece + buf) ^ (k & 7)) << 4)); };
          volatile uint32_t* nan_any = reinterpret_cast<uint32_t*>(smem + L::kNanAny) + buf * 4;
          if (g == 0) {
            warp_wait(&kv_full[v_stage], (uint32_t)(v_fill / kStages) & 1, abort_flag);
            __syncwarp();
            uint4* vrow = reinterpret_cast<uint4*>(smem + L::kRing + v_stage * kPaTileBytes + key * 128);
            if (pos >= ent.len) {
#pragma unroll
              for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0, 0, 0, 0);
            }
            if (edge) {
              uint32_t bits[4] = {0, 0, 0, 0};
              if (pos < ent.len) take_nan(vrow, key, bits);
              *nan_of(key) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
              nan_any[wq] = __any_sync(0xffffffffu, (bits[0] | bits[1] | bits[2] | bits[3]) != 0);  // every lane the same
            }
          }
          if (edge) {
            __syncwarp();
            asm volatile("bar.sync 3, %0;" ::"n"(128 * L::kGroups) : "memory");
            if (nan_any[0] | nan_any[1] | nan_any[2] | nan_any[3]) {
              // this thread's channel: the rows that see a key whose V is NaN there
#pragma unroll 1
              for (int kk = 0; kk < kPaTile; ++kk) {
                if (!(reinterpret_cast<const uint32_t*>(nan_of(kk))[quarter] >> lane & 1u)) continue;
#pragma unroll 1
                for (int r = 0; r < RG; ++r) {
                  const int2 k = row_keys[g * RG + r];
                  if ((uint32_t)(k0 + kk - k.x) < (uint32_t)k.y) nan_rows |= 1u << r;
                }
              }
              __syncwarp();
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        warp_arrive(&p_full[i & 1]);
      }
      // ---- the accumulator, the sum over the keys, then the result or what another block needs to go on
      warp_wait(&o_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1, abort_flag);
      const bool ok = *abort_flag == 0;
      tc_fence_after_sync();
      float o[RG], o1[RG];
      tmem_ld16(t_o, reinterpret_cast<uint32_t*>(o));
      tmem_ld16(t_o + R, reinterpret_cast<uint32_t*>(o1));
      {
        float v[RG];
#pragma unroll
        for (int k = 0; k < RG / 2; ++k) f2_unpack(l2[k], v[2 * k], v[2 * k + 1]);
        // halves of the rows change lanes while the sums are formed: lanes 2 x and 2 x + 1 end with row x
        int width = RG;
#pragma unroll
        for (int d = 16; d > 1; d >>= 1) {
          width >>= 1;
#pragma unroll
          for (int k = 0; k < RG / 2; ++k)
            if (k < width) {
              const float send = lane & d ? v[k] : v[k + width], keep = lane & d ? v[k + width] : v[k];
              v[k] = keep + __shfl_xor_sync(0xffffffffu, send, d);
            }
        }
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
        if ((lane & 1) == 0) max_sh[wq * RG + (lane >> 1)] = v[0];
      }
      group_sync(g);
      const int row = g * RG + lane;  // of lanes < RG
      const float total = lane < RG ? (max_sh[lane] + max_sh[RG + lane]) + (max_sh[2 * RG + lane] + max_sh[3 * RG + lane]) : 0.f;
      tmem_wait_ld();
#pragma unroll
      for (int r = 0; r < RG; ++r) o[r] += o1[r];
      if (nan_rows) {
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (nan_rows >> r & 1u) o[r] = __uint_as_float(0x7fffffffu);
      }
      const int rows = unit.rows - g * RG;  // of this group, when positive
      if (walk.whole()) {
        const bool owned = lane < RG && lane < rows;
        const int flat = unit.first + (owned ? row : 0), tok = by_group(p, flat), head = h * p.group + flat - tok * p.group;
        if (owned && ok) {
          if (p.lse && wq == 0)
            p.lse[(int64_t)(ent.row0 + tok) * p.hq + head] = total != 0.f ? (m - kPaShift + log2f(total)) * 0.6931471805599453f : -INFINITY;
        }
        if (lane < RG) {
          inv_sh[lane] = total != 0.f ? 1.0f / total : 0.f;  // nothing seen: zero
          at_sh[lane] = (int64_t)(ent.row0 + tok) * p.o_st + (int64_t)head * p.o_sh;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (ok && r < rows) p.out[at_sh[r] + key] = __float2bfloat16_rn(o[r] * inv_sh[r]);
        __syncwarp();
      } else {
        const int64_t slot = 2 * (int64_t)blockIdx.x + (first == 0 ? 1 : 0);
        float* part = p.parts + (slot * R + g * RG) * kHeadDim;
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (r < rows) part[r * kHeadDim + key] = o[r];
        if (wq == 0 && lane < RG) p.stats[slot * R + row] = make_float2(m, total);
        if (first == 0 && sw == 0 && lane == 0) p.headers[blockIdx.x] = {1, walk.last_block(st.per_block), ent.row0, h, unit.first, unit.rows, {0, 0}};
      }
      ++units;
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

// Joins the parts of a unit that several blocks worked on, in the order of the keys: block (i, y) works on the unit that
// main block i left open.  kWide: its eight warps share one row (few rows in many parts), else each has a row of its own (and
// the parts lie [channel / 4][row][4], as the prompt form's threads, a row each, store them side by side).
template <int R, bool kWide>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedAttnKernelParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PaHeader hd = p.headers[blockIdx.x];
  if (!hd.open) return;
  __shared__ float s_sum[8];
  __shared__ float4 s_acc[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = kWide ? blockIdx.y : blockIdx.y * 8 + warp;
  if (r >= hd.rows) return;
  const int n_parts = hd.last - blockIdx.x + 1;
  auto slot = [&](int k) { return (k == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * (int64_t)(blockIdx.x + k)) * R + r; };
  float top = -INFINITY;  // every warp looks at all maxima of its row
  for (int k = lane; k < n_parts; k += 32) top = fmaxf(top, p.stats[slot(k)].x);
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = kWide ? warp : 0; k < n_parts; k += kWide ? 8 : 1) {
    const int64_t s = slot(k);
    const float2 ml = p.stats[s];
    const float4 o = *reinterpret_cast<const float4*>(p.parts + (kWide ? s * kHeadDim + lane * 4 : (s - r) * kHeadDim + (lane * R + r) * 4));
    const float f = ex2(ml.x - ref);
    sum = fmaf(ml.y, f, sum);
    acc.x = fmaf(o.x, f, acc.x);
    acc.y = fmaf(o.y, f, acc.y);
    acc.z = fmaf(o.z, f, acc.z);
    acc.w = fmaf(o.w, f, acc.w);
  }
  if (kWide) {
    s_acc[warp][lane] = acc;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp > 0) return;
    sum = s_sum[0];
    acc = s_acc[0][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      const float4 o = s_acc[w][lane];
      sum += s_sum[w];
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
    }
  }
  const float inv = sum != 0.f ? 1.0f / sum : 0.f;
  const int flat = hd.first + r, tok = by_group(p, flat), head = hd.h * p.group + flat - tok * p.group;
  *reinterpret_cast<uint2*>(p.out + (int64_t)(hd.row0 + tok) * p.o_st + (int64_t)head * p.o_sh + lane * 4) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0)
    p.lse[(int64_t)(hd.row0 + tok) * p.hq + head] = sum != 0.f ? (top - kPaShift + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------------------------- host side
// The join follows its main kernel without a gap: its blocks are placed early and wait for the main grid's memory.
template <int R, bool kWide>
static int launch_join(magi_ctx* ctx, const PagedAttnKernelParams& k, int blocks, cudaStream_t st) {
  const int64_t rows = (int64_t)k.max_q * k.group < R ? (int64_t)k.max_q * k.group : R;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, (unsigned)(kWide ? rows : (rows + 7) / 8), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MAGI_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, paged_join_kernel<R, kWide>, k));
  return MAGI_OK;
}

// Rows of a block's unit: up to 16 or 32 (query tokens times heads of a group) fit the forms with the keys across, of which an
// SM holds two blocks; more go 256 at a time through the form with the rows across.
static int form_rows(int64_t max_q, int group) { return max_q * group <= 16 ? 16 : max_q * group <= 32 ? 32 : kPromptRows; }
static int form_blocks(const magi_ctx* ctx, int rows) {
  return ctx->sm_count * (rows == 16 ? PaShared<16>::kBlocksPerSm : rows == 32 ? PaShared<32>::kBlocksPerSm : 1);
}

static int64_t workspace_bytes(const magi_ctx* ctx, int rows) {
  const int64_t blocks = form_blocks(ctx, rows);
  return blocks * (int64_t)sizeof(PaHeader) + 2 * blocks * rows * (kHeadDim * 4 + 8);
}

template <int R>
static int launch_paged(magi_ctx* ctx, const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnKernelParams& k, cudaStream_t st) {
  using L = PaShared<R>;
  static bool configured[64] = {};  // per device: opt in to > 48 KB of dynamic shared memory once
  if (ctx->device >= 64 || !configured[ctx->device]) {
    MAGI_CUDA_OK(ctx, cudaFuncSetAttribute(paged_attn_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamic));
    if (ctx->device < 64) configured[ctx->device] = true;
  }
  const int blocks = form_blocks(ctx, R);
  paged_attn_kernel<R><<<blocks, L::kThreads, L::kDynamic, st>>>(tk, tv, k);
  MAGI_CUDA_OK(ctx, cudaGetLastError());
  return launch_join<R, true>(ctx, k, blocks, st);
}

int launch_prompt_join(magi_ctx* ctx, const PagedAttnKernelParams& k, cudaStream_t st) {
  return launch_join<kPromptRows, false>(ctx, k, form_blocks(ctx, kPromptRows), st);
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
  if (!(p->softmax_scale <= 2e38f))  // times log2 e it has to be finite
    return set_err(ctx, MAGI_E_BADARG, "paged attn: softmax_scale must be a number up to 2e38");
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
  set_group(&k, p->n_q_heads / k.c.n_kv_heads);
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
  if (rows == 16) return launch_paged<16>(ctx, tk, tv, k, st);
  if (rows == 32) return launch_paged<32>(ctx, tk, tv, k, st);
  return launch_paged_prompt(ctx, tk, tv, k, st);
}
