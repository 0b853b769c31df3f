// Rotary embedding by position, both channel layouts, on the first rot_dim channels of a head, forward and transposed:
//     (a, b) -> mscale * (a cos - b sin, b cos + a sin),  angle = positions[t] * inv_freq[i]
// Memory-bound: each element is read once and written once in 16-byte pieces.  A block takes a group of tokens, forms the
// group's cosines and sines once in shared memory while its first channels are on their way (64-bit product, reduced to a
// fraction of a turn before it becomes fp32: at position 10^6 a 32-bit product alone would be 0.03 radians off) and applies
// them to every head.  What takes time beside the memory is instructions: threads walk over their pieces by adding steps,
// without a division, and 16-bit results are rounded two at a time.  21600 x 24 x 128: bf16 49 us (5.4 TB/s), fp32 86 us
// (6.2 TB/s).  Off the 16-byte grid elements move one at a time: the same sizes from an odd start 139 and 143 us, 21600 x 24 x 96
// with 50 channels turned 130 and 134 us.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace magi {

constexpr int kRotThreads = 256;
constexpr int kRotAngles = 2048;  // angles a block holds: 16 KB
constexpr int kRotBatch = 4;      // 16-byte pieces that a thread has in flight

struct RotaryKernelParams {
  const void* x;
  void* out;
  int64_t x_st, x_sh, o_st, o_sh;
  const void* positions;
  int pos64;
  int T, H, dim, half;
  int group;            // tokens of a block
  int heads_per_block;
  int inverse;
  float mscale;
  const double* inv_freq;
};

template <class E>
__device__ __forceinline__ float to_f(E v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class E>
__device__ __forceinline__ E from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

template <class E, int V>
struct alignas(sizeof(E) * V) Piece {
  E v[V];
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f(v[i]);
  }
  __device__ __forceinline__ void pack(const float* f) {  // two at a time where the type has that conversion
    if constexpr (sizeof(E) == 2 && V > 1) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        uint32_t w;
        if constexpr (std::is_same<E, __half>::value) w = pack2(__floats2half2_rn(f[i], f[i + 1]));
        else w = pack2(__floats2bfloat162_rn(f[i], f[i + 1]));
        *reinterpret_cast<uint32_t*>(v + i) = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = from_f<E>(f[i]);
    }
  }
  template <class T>
  static __device__ __forceinline__ uint32_t pack2(T w) {
    return *reinterpret_cast<const uint32_t*>(&w);
  }
};

// A unit is V channels of "half"'s first part with their V partners, or V consecutive channels of the interleaved layout,
// or V channels behind rot_dim that are copied.  V = 1 is the form for odd sizes and unaligned views (interleaved: one pair).
template <class E, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads, 4) rotary_kernel(const RotaryKernelParams p) {
  __shared__ float2 cs[kRotAngles];
  const int t0 = blockIdx.x * p.group;
  const int nt = min(p.group, p.T - t0);
  constexpr int kStep = kInterleaved && V == 1 ? 2 : V;  // channels that a rotated unit covers in its first part
  constexpr bool kPair = V == 1 || !kInterleaved;        // a rotated unit has two pieces
  constexpr int kBatch = kPair ? kRotBatch / 2 : kRotBatch;
  // angles of a unit; the i-th angles of all units lie side by side, so that the lanes of a warp read neighbours
  constexpr int kAngles = kPair ? V : V / 2;
  const int side = p.half / kAngles;
  const int rot_units = kInterleaved ? 2 * p.half / kStep : p.half / kStep;
  const int units = rot_units + (p.dim - 2 * p.half) / V;
  const int h0 = blockIdx.y * p.heads_per_block, nh = min(p.heads_per_block, p.H - h0);
  // this thread's unit (token t, head h, piece k), and the way to its next one, as the digits of kRotThreads
  int h = threadIdx.x / units, k = threadIdx.x - h * units, t = h / nh;
  h -= t * nh;
  int dh = kRotThreads / units;
  const int dk = kRotThreads - dh * units, dt = dh / nh;
  dh -= dt * nh;
  // where its head starts, and the steps
  const E* x = static_cast<const E*>(p.x) + (int64_t)(t0 + t) * p.x_st + (int64_t)(h0 + h) * p.x_sh;
  E* o = static_cast<E*>(p.out) + (int64_t)(t0 + t) * p.o_st + (int64_t)(h0 + h) * p.o_sh;
  const int64_t x_step = dt * p.x_st + dh * p.x_sh, x_turn = p.x_st - nh * p.x_sh;
  const int64_t o_step = dt * p.o_st + dh * p.o_sh, o_turn = p.o_st - nh * p.o_sh;
  auto channel = [&](int u) {  // first channel of a unit
    return kStep == V ? u * V + (kPair && u >= rot_units ? p.half : 0) : u < rot_units ? u * kStep : u + p.half;
  };
  Piece<E, V> lo[kBatch], hi[kBatch];
  int at_t[kBatch], at_k[kBatch];
  E* at[kBatch];
  auto load = [&]() {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      at_t[b] = t, at_k[b] = k;
      const int c = channel(k);
      at[b] = o + c;
      if (t < nt) {
        lo[b] = *reinterpret_cast<const Piece<E, V>*>(x + c);
        if (kPair && k < rot_units) hi[b] = *reinterpret_cast<const Piece<E, V>*>(x + c + (kInterleaved ? 1 : p.half));
      }
      k += dk, h += dh, t += dt, x += x_step, o += o_step;
      if (k >= units) k -= units, ++h, x += p.x_sh, o += p.o_sh;
      if (h >= nh) h -= nh, ++t, x += x_turn, o += o_turn;
    }
  };
  load();  // in flight while the angles are formed
  for (int i = threadIdx.x; i < nt * p.half; i += kRotThreads) {
    const int a = i / p.half, c = i - a * p.half;
    const double pos = p.pos64 ? (double)__ldg(reinterpret_cast<const long long*>(p.positions) + t0 + a)
                               : (double)__ldg(reinterpret_cast<const int*>(p.positions) + t0 + a);
    const double turns = pos * (__ldg(p.inv_freq + c) * 0.15915494309189535);  // 1 / (2 pi)
    float s, co;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
    cs[a * p.half + c % kAngles * side + c / kAngles] = make_float2(co * p.mscale, (p.inverse ? -s : s) * p.mscale);
  }
  __syncthreads();
  while (true) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (at_t[b] >= nt) continue;
      const int u = at_k[b];
      if (u < rot_units) {
        const float2* a = cs + at_t[b] * p.half + u;
        float f[V], g[V];
        lo[b].unpack(f);
        if constexpr (kPair) {
          hi[b].unpack(g);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 r = a[i * side];
            const float l = f[i];
            f[i] = l * r.x - g[i] * r.y;
            g[i] = g[i] * r.x + l * r.y;
          }
          hi[b].pack(g);
          *reinterpret_cast<Piece<E, V>*>(at[b] + (kInterleaved ? 1 : p.half)) = hi[b];
        } else {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 r = a[i / 2 * side];
            const float l = f[i];
            f[i] = l * r.x - f[i + 1] * r.y;
            f[i + 1] = f[i + 1] * r.x + l * r.y;
          }
        }
        lo[b].pack(f);
      }
      *reinterpret_cast<Piece<E, V>*>(at[b]) = lo[b];
    }
    if (t >= nt) return;
    load();
  }
}

template <class E>
static void launch_rotary(const RotaryKernelParams& k, bool vec, bool inter, dim3 grid, cudaStream_t st) {
  constexpr int V = 16 / sizeof(E);
  if (vec) {
    if (inter) rotary_kernel<E, V, true><<<grid, kRotThreads, 0, st>>>(k);
    else rotary_kernel<E, V, false><<<grid, kRotThreads, 0, st>>>(k);
  } else {
    if (inter) rotary_kernel<E, 1, true><<<grid, kRotThreads, 0, st>>>(k);
    else rotary_kernel<E, 1, false><<<grid, kRotThreads, 0, st>>>(k);
  }
}

}  // namespace magi

extern "C" int magi_rotary_fwd(magi_ctx* ctx, const magi_rotary_params* p, void* stream) {
  using namespace magi;
  if (!ctx) return MAGI_E_BADARG;
  if (!p || p->struct_size != sizeof(magi_rotary_params)) return set_err(ctx, MAGI_E_BADARG, "rotary: bad struct_size");
  if (p->dtype != MAGI_DTYPE_BF16 && p->dtype != MAGI_DTYPE_F16 && p->dtype != MAGI_DTYPE_F32)
    return set_err(ctx, MAGI_E_BADARG, "rotary: dtype is bf16, fp16 or fp32");
  if (p->T < 0 || p->H <= 0 || p->head_dim <= 0 || p->rot_dim < 0 || p->rot_dim > p->head_dim || p->rot_dim % 2)
    return set_err(ctx, MAGI_E_BADARG, "rotary: bad shape (rot_dim must be even and at most head_dim)");
  if (p->rot_dim / 2 > kRotAngles) return set_err(ctx, MAGI_E_BADARG, "rotary: rot_dim above %d", 2 * kRotAngles);
  if (p->T == 0) return MAGI_OK;
  if (!p->x || !p->out || !p->positions || (p->rot_dim > 0 && !p->inv_freq)) return set_err(ctx, MAGI_E_BADARG, "rotary: null tensor");
  const int esz = p->dtype == MAGI_DTYPE_F32 ? 4 : 2;
  const int V = 16 / esz;
  if ((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->out)) % esz)
    return set_err(ctx, MAGI_E_ALIGN, "rotary: x and out must be aligned to their type");
  // 16-byte pieces wherever every row, both parts of a head and the tail start on one; single channels otherwise
  const bool vec = !((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->out)) & 15) && p->x_stride_t % V == 0 &&
                   p->x_stride_h % V == 0 && p->out_stride_t % V == 0 && p->out_stride_h % V == 0 && p->head_dim % V == 0 &&
                   p->rot_dim % (p->interleaved ? V : 2 * V) == 0;
  RotaryKernelParams k = {p->x, p->out, p->x_stride_t, p->x_stride_h, p->out_stride_t, p->out_stride_h, p->positions,
                          p->positions_are_int64, p->T, p->H, p->head_dim, p->rot_dim / 2, 1, p->H, p->inverse, p->mscale, p->inv_freq};
  // tokens of a block: three batches for its threads (21600 x 24 x 128 bf16, interleaved: 49 us; two 54 us, six 54 us), no
  // more angles than it holds
  const int64_t per_token = (int64_t)p->H * p->head_dim / (vec ? V : 1);
  int64_t group = (3 * kRotBatch * kRotThreads + per_token - 1) / per_token;
  if (k.half > 0 && group > kRotAngles / k.half) group = kRotAngles / k.half;
  if (group > p->T) group = p->T;
  k.group = (int)group;
  const int64_t bx = ((int64_t)p->T + group - 1) / group;
  // few tokens: the heads are split over blocks, each of which forms the angles again
  int by = 1;
  while (bx * by < ctx->sm_count && by * 2 <= p->H && group * per_token / (by * 2) >= kRotThreads) by *= 2;
  k.heads_per_block = (p->H + by - 1) / by;
  const dim3 grid((unsigned)bx, (unsigned)((p->H + k.heads_per_block - 1) / k.heads_per_block));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int prev = 0;
  cudaGetDevice(&prev);
  if (prev != ctx->device) cudaSetDevice(ctx->device);
  if (p->dtype == MAGI_DTYPE_F32) launch_rotary<float>(k, vec, p->interleaved, grid, st);
  else if (p->dtype == MAGI_DTYPE_F16) launch_rotary<__half>(k, vec, p->interleaved, grid, st);
  else launch_rotary<__nv_bfloat16>(k, vec, p->interleaved, grid, st);
  const cudaError_t e = cudaGetLastError();
  if (prev != ctx->device) cudaSetDevice(prev);
  if (e != cudaSuccess) return set_err(ctx, MAGI_E_CUDA, "rotary launch failed: %s", cudaGetErrorString(e));
  return MAGI_OK;
}
