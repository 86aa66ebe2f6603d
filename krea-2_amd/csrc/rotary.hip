// Rotary positions of queries and keys: every pair (a, b) of a head's rotated part turns by the token's angle,
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = 2 pi pos[axis(i)] turns[i],
// i the pair's index, pos the token's position along the pair's axis, m a factor on the rotated part; the rest of the
// head is copied.  The transpose (inverse != 0: t -> -t) is the backward pass.  Pairs lie side by side (interleaved:
// 2 i, 2 i + 1) or half the rotated part apart (half: i, i + rotary_dim / 2).
//
// Angles are products in float64 less their whole turns, cos and sin of the rest in float32, and every product and sum of
// the rotation in float32, rounded once to the tensor's type.  The product keeps 2^-53 of |pos turns| (a position of 2^24
// still has its angle to 3e-10 turns; in float32 it would have no digit left), the rest 2^-26 turns.
//
// Bound: reading and writing the heads once.  A workgroup takes a run of (token, head) rows, q's heads before k's in
// every token; its threads first compute the cos / sin of the run's tokens into LDS, once for all heads, then a thread
// turns vectors of one head position, stepping through the run's rows.  4608 x 60 heads of 128 bf16: 31 us (4.6 TB/s), 16896
// of them 99 us (5.2).
#include <hip/hip_fp16.h>

#include "k2q_common.h"

namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_MAX_DIM = 4096;       // head size
constexpr int RT_MAX_ROTARY = 1024;
constexpr int RT_LDS = 32768;          // bytes of cos / sin at most

struct RotArgs {
  const void* x[2];
  void* o[2];
  int64_t xb[2], xl[2], xh[2], ob[2], ol[2], oh[2];   // strides in elements: batch, token, head
  int h0, h;               // q's heads, all heads
  int L;
  uint32_t rows;           // B * L * h
  int D, rd;
  const void* pos;
  int pos_type;
  int64_t pb, pl, pa;
  const double* turns;
  const int* axis;         // null: one axis
  float m, sign;
  int turned, items;       // a row's turned vectors, all its vectors
  int width, slots;        // threads side by side on a row, rows side by side
  uint32_t run;            // rows per workgroup
  int dt, dh;              // slots / h, slots % h
};

__device__ __forceinline__ double position(const RotArgs& a, int64_t i) {
  switch (a.pos_type) {
    case K2Q_POS_I64: return (double)static_cast<const int64_t*>(a.pos)[i];
    case K2Q_POS_I32: return (double)static_cast<const int*>(a.pos)[i];
    case K2Q_POS_F32: return (double)static_cast<const float*>(a.pos)[i];
    default: return static_cast<const double*>(a.pos)[i];
  }
}

template <typename T>
struct Cvt;
template <>
struct Cvt<float> {
  static __device__ __forceinline__ float in(float v) { return v; }
  static __device__ __forceinline__ float out(float v) { return v; }
};
template <>
struct Cvt<__bf16> {
  static __device__ __forceinline__ float in(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 out(float v) { return (__bf16)v; }
};
template <>
struct Cvt<_Float16> {
  static __device__ __forceinline__ float in(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 out(float v) { return (_Float16)v; }
};

// V elements as one aligned load and store (two of 16 bytes for eight f32).
template <typename T, int V>
struct Vec {
  typedef T Raw __attribute__((ext_vector_type(V)));
  Raw v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = v; }
  __device__ __forceinline__ float get(int i) const { return Cvt<T>::in(v[i]); }
  __device__ __forceinline__ void put(int i, float f) { v[i] = Cvt<T>::out(f); }
};
template <typename T>
struct Vec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ float get(int) const { return Cvt<T>::in(v); }
  __device__ __forceinline__ void put(int, float f) { v = Cvt<T>::out(f); }
};

__device__ __forceinline__ void turn(float& a, float& b, const float2& cs) {
  const float x = a, y = b;
  a = x * cs.x - y * cs.y;
  b = x * cs.y + y * cs.x;
}

template <typename T, bool kHalf, int V>
__global__ __launch_bounds__(RT_THREADS) void rotary_kernel(RotArgs a) {
  extern __shared__ float2 cs[];
  const uint32_t r0 = blockIdx.x * a.run;
  const uint32_t r1 = a.rows - r0 < a.run ? a.rows : r0 + a.run;
  const uint32_t t0 = r0 / a.h;
  const int nf = a.rd / 2;
  const int n = (int)((r1 - 1) / a.h - t0 + 1) * nf;
  for (int i = threadIdx.x; i < n; i += RT_THREADS) {
    const uint32_t tok = t0 + i / nf;
    const int f = i % nf;
    const double p = position(a, (int64_t)(tok / a.L) * a.pb + (int64_t)(tok % a.L) * a.pl +
                                     (a.axis ? a.axis[f] * a.pa : 0));
    double t = p * a.turns[f];
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    cs[i] = make_float2(c * a.m, s * a.m * a.sign);
  }
  __syncthreads();

  const int slot = threadIdx.x / a.width, j0 = threadIdx.x % a.width;
  if (slot >= a.slots) return;
  uint32_t r = r0 + slot;
  if (r >= r1) return;
  uint32_t tok = r / a.h;
  int head = (int)(r % a.h);
  int b = (int)(tok / a.L), l = (int)(tok % a.L);
  for (; r < r1; r += a.slots) {
    const int w = head >= a.h0;
    const int hh = w ? head - a.h0 : head;
    const T* x = static_cast<const T*>(a.x[w]) + (b * a.xb[w] + l * a.xl[w] + hh * a.xh[w]);
    T* o = static_cast<T*>(a.o[w]) + (b * a.ob[w] + l * a.ol[w] + hh * a.oh[w]);
    const float2* c = cs + (tok - t0) * nf;
    for (int j = j0; j < a.items; j += a.width) {
      if (j >= a.turned) {                    // V copied elements
        Vec<T, V> u;
        const int e = a.rd + V * (j - a.turned);
        u.load(x + e);
        u.store(o + e);
      } else if constexpr (kHalf || V == 1) { // V pairs from two vectors
        constexpr bool kBeside = !kHalf;
        const int ia = kBeside ? 2 * j : V * j, ib = kBeside ? 2 * j + 1 : nf + V * j;
        Vec<T, V> u, v;
        u.load(x + ia);
        v.load(x + ib);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float f = u.get(i), g = v.get(i);
          turn(f, g, c[V * j + i]);
          u.put(i, f);
          v.put(i, g);
        }
        u.store(o + ia);
        v.store(o + ib);
      } else {                                // V / 2 pairs from one
        Vec<T, V> u;
        u.load(x + V * j);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          float f = u.get(2 * i), g = u.get(2 * i + 1);
          turn(f, g, c[V / 2 * j + i]);
          u.put(2 * i, f);
          u.put(2 * i + 1, g);
        }
        u.store(o + V * j);
      }
    }
    tok += a.dt;
    l += a.dt;
    head += a.dh;
    if (head >= a.h) {
      head -= a.h;
      ++tok;
      ++l;
    }
    while (l >= a.L) {
      l -= a.L;
      ++b;
    }
  }
}

template <typename T, bool kHalf>
void launch(const RotArgs& a, int vec, unsigned grid, int lds, hipStream_t st) {
  switch (vec) {
    case 8: hipLaunchKernelGGL((rotary_kernel<T, kHalf, 8>), dim3(grid), dim3(RT_THREADS), lds, st, a); break;
    case 4: hipLaunchKernelGGL((rotary_kernel<T, kHalf, 4>), dim3(grid), dim3(RT_THREADS), lds, st, a); break;
    case 2: hipLaunchKernelGGL((rotary_kernel<T, kHalf, 2>), dim3(grid), dim3(RT_THREADS), lds, st, a); break;
    default: hipLaunchKernelGGL((rotary_kernel<T, kHalf, 1>), dim3(grid), dim3(RT_THREADS), lds, st, a); break;
  }
}

template <typename T>
void launch_t(const RotArgs& a, bool half, int vec, unsigned grid, int lds, hipStream_t st) {
  if (half) launch<T, true>(a, vec, grid, lds, st);
  else launch<T, false>(a, vec, grid, lds, st);
}

}  // namespace

extern "C" int k2q_rotary(const k2q_rotary_heads* t, int64_t n, int dtype, int64_t B, int64_t L, int64_t D,
                          int64_t rotary_dim, int layout, const void* positions, int pos_type, int64_t pos_b,
                          int64_t pos_l, int64_t pos_a, const double* turns, const int32_t* axis, float factor,
                          int inverse, void* stream) {
  if (!t || n < 1 || n > 2 || B < 1 || L < 1 || D < 2 || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > D || !positions ||
      !turns || !k2q_aligned(turns, 8) || !k2q_aligned(axis, 4) || layout < 0 || layout > K2Q_ROTARY_HALF ||
      dtype < K2Q_DTYPE_BF16 || dtype > K2Q_DTYPE_F16 || pos_type < K2Q_POS_I64 || pos_type > K2Q_POS_F64 ||
      !k2q_aligned(positions, pos_type == K2Q_POS_I64 || pos_type == K2Q_POS_F64 ? 8 : 4))
    return K2Q_EINVAL;
  if (D > RT_MAX_DIM || rotary_dim > RT_MAX_ROTARY) return K2Q_EUNSUPPORTED;
  const int size = dtype == K2Q_DTYPE_F32 ? 4 : 2;
  const bool half = layout == K2Q_ROTARY_HALF;
  RotArgs a{};
  // The widest vector that cuts the rotated part (each half of it), the rest and every row's start into whole ones
  const int rest = (int)(D - rotary_dim);
  int vec = 8;
  auto narrow = [&](int64_t elements) {
    while (elements % vec) vec >>= 1;
  };
  narrow(half ? rotary_dim / 2 : rotary_dim);
  narrow(rest);
  int64_t heads = 0;
  for (int i = 0; i < 2; ++i) {
    const k2q_rotary_heads& s = t[i < n ? i : 0];
    const int64_t strides[6] = {s.x_b, s.x_l, s.x_h, s.o_b, s.o_l, s.o_h};
    if (!s.x || !s.o || s.heads < 1 || !k2q_aligned(s.x, size) || !k2q_aligned(s.o, size)) return K2Q_EINVAL;
    const int64_t extent[3] = {B, L, s.heads};
    for (int d = 0; d < 6; ++d)
      if (extent[d % 3] > 1) narrow(strides[d]);
    narrow((int64_t)(reinterpret_cast<uintptr_t>(s.x) / size));
    narrow((int64_t)(reinterpret_cast<uintptr_t>(s.o) / size));
    a.x[i] = s.x;
    a.o[i] = s.o;
    a.xb[i] = s.x_b; a.xl[i] = s.x_l; a.xh[i] = s.x_h;
    a.ob[i] = s.o_b; a.ol[i] = s.o_l; a.oh[i] = s.o_h;
    if (i < n) {
      if (s.heads > 0x7fffffff) return K2Q_EUNSUPPORTED;
      heads += s.heads;
    }
  }
  // row indexes and their steps stay below 2^32 (2^31 per factor: signed token and batch indexes)
  if (L > 0x3fffffff || B > 0x3fffffff || heads > 0x3fffffff || B * L > 0x3fffffff || B * L * heads > 0x7fffffff)
    return K2Q_EUNSUPPORTED;
  a.h0 = (int)t[0].heads;
  a.h = (int)heads;
  a.L = (int)L;
  a.rows = (uint32_t)(B * L * heads);
  a.D = (int)D;
  a.rd = (int)rotary_dim;
  a.pos = positions;
  a.pos_type = pos_type;
  a.pb = pos_b;
  a.pl = pos_l;
  a.pa = pos_a;
  a.turns = turns;
  a.axis = axis;
  a.m = factor;
  a.sign = inverse ? -1.f : 1.f;
  const int nf = a.rd / 2;
  a.turned = half || vec == 1 ? nf / vec : a.rd / vec;
  a.items = a.turned + rest / vec;
  a.width = a.items < RT_THREADS ? a.items : RT_THREADS;
  a.slots = RT_THREADS / a.width;
  // Rows per workgroup: 16 KB of heads, fewer where the rows would not give every CU four workgroups, no more tokens than
  // fit LDS.  4608 x 60 heads of 128 bf16, us at 16 / 32 / 64 / 128 rows (interleaved) 41 / 33 / 30 / 32, at 32 / 64 / 128 /
  // 256 (half) 32 / 32 / 34 / 38; below 16 KB the cos / sin of a token are made too often, above it the last ones wait.
  int64_t steps = 16384 / ((int64_t)a.slots * a.D * size);
  const int64_t fill = (int64_t)a.rows / ((int64_t)a.slots * 4 * k2q_cu_count());
  steps = steps > fill ? fill : steps;
  steps = steps < 1 ? 1 : steps;
  const int64_t most = RT_LDS / (8 * nf);                    // tokens whose cos / sin fit
  while (steps > 1 && (steps * a.slots - 1) / a.h + 2 > most) --steps;
  if ((a.slots - 1) / a.h + 2 > most) a.slots = (int)((most - 2) * a.h + 1);
  a.dt = a.slots / a.h;
  a.dh = a.slots % a.h;
  a.run = (uint32_t)(steps * a.slots);
  const int64_t tokens = (a.run - 1) / a.h + 2 < B * L ? (a.run - 1) / a.h + 2 : B * L;
  const unsigned grid = (unsigned)((a.rows + (int64_t)a.run - 1) / a.run);
  const int lds = (int)(tokens * nf * 8);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case K2Q_DTYPE_BF16: launch_t<__bf16>(a, half, vec, grid, lds, st); break;
    case K2Q_DTYPE_F32: launch_t<float>(a, half, vec, grid, lds, st); break;
    default: launch_t<_Float16>(a, half, vec, grid, lds, st); break;
  }
  return k2q_launch_status();
}
