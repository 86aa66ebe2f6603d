// Low-rank adapters of many requests beside one projection: row t of a batch has adapter a = ids[t / per] of a bank of factors
// A (count x R x K) and B (count x N x R), or none, and
//   out[t] = y[t] + u[t] B_a^T,  u[t] = s_a x[t] A_a^T              (LoRALinear.forward, reference lora.py:43-48, by row)
// with the gradients g = s_a dy B_a, dx = g A_a (+ the base's), dA_a = sum_t g[t]^T x[t], dB_a = sum_t dy[t]^T u[t].
//
// Two forms of product make all of it.  "Down" reduces wide rows to an adapter's rank (u from x and A, g from dy and B),
// "up" widens them again and adds (out from u and B, dx from g and A); each takes its factor with the wide index contiguous
// (A) or the rank contiguous (B).  The third form, "sums", reduces over an adapter's rows (dA from g and x, dB from u and
// dy).  All run on 16x16x32 bf16 MFMAs with f32 sums: what is in f32 (factors, u, g) goes in as two bf16 parts, or three on the
// way to a gradient in f32; y, x, dy are bf16 as they are.
//
// Rows may come in any order.  A tile of 64 rows goes over the adapters that it finds in it, one after another: rows of one
// request lie together, so that is one adapter, or two, in all but the smallest batches.
#include <type_traits>

#include "k2q_common.h"
#include "rotation.h"

namespace {

constexpr int ROWS = 64;              // rows of a tile
constexpr int THREADS = 256;          // 4 waves
constexpr int RANKS = 128;            // most ranks that an "up" workgroup holds at once
constexpr int LS = 72;                // a wave's 64 columns of a row in LDS, 16 bytes off the banks' turn

struct Rows {
  const void* ids;
  const int32_t* ranks;     // nullable
  const float* scales;      // nullable
  float mul;
  int32_t wide;             // ids are 64-bit
  int32_t per;              // rows of an id
  int32_t T;
  int32_t count;
  int32_t R;                // rank of the bank's storage
};

// The adapter of an id: -1 for none, and for numbers that are no adapter's.
__device__ __forceinline__ int adapter_at(const Rows& a, int i) {
  const int64_t id = a.wide ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
  return id < 0 || id >= a.count ? -1 : (int)id;
}

__device__ __forceinline__ int adapter_of(const Rows& a, int row) { return row >= a.T ? -2 : adapter_at(a, row / a.per); }

// Ranks of an adapter that count.
__device__ __forceinline__ int rank_of(const Rows& a, int id) {
  if (id < 0) return 0;
  if (!a.ranks) return a.R;
  return max(0, min(a.ranks[id], a.R));
}

// The same in whole MFMA tiles: what u and g hold, zeros behind the adapter's own ranks.  Storage between the two may hold
// anything (zeros would not do: 0 x NaN is NaN), so the sums there are dropped and a factor's values taken out.
__device__ __forceinline__ int whole(int rank) { return (rank + 15) & ~15; }

// A vector of ranks j .. j + 3, of which those below r count.
__device__ __forceinline__ v4f counted(v4f v, int j, int r) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = j + e < r ? v[e] : 0.f;
  return v;
}

// 8 bf16 values, of which the first n count.
__device__ __forceinline__ v8bf counted(v8bf v, int n) {
  v4u w = __builtin_bit_cast(v4u, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] &= (2 * i < n ? 0xffffu : 0u) | (2 * i + 1 < n ? 0xffff0000u : 0u);
  return __builtin_bit_cast(v8bf, w);
}

__device__ __forceinline__ float scale_of(const Rows& a, int id) { return a.scales ? a.mul * a.scales[id] : a.mul; }

// 8 values in f32 as N bf16 parts: their rounding, that of the rest, that of the rest's rest.  Two are 2^-17 of a value off at
// most, for products that end in bf16; three hold all 24 bits, for gradients that end in f32.
template <int N>
struct Parts {
  v8bf p[N];
};

template <int N>
__device__ __forceinline__ Parts<N> split(const float (&v)[8]) {
  Parts<N> s;
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v4u h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      r[2 * i] -= __uint_as_float(h[i] << 16);
      r[2 * i + 1] -= __uint_as_float(h[i] & 0xffff0000u);
    }
    s.p[n] = __builtin_bit_cast(v8bf, h);
  }
  return s;
}

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <typename F>
constexpr bool kF32 = sizeof(F) == 4;

// Fragments of a factor for one MFMA step of 32: Q tiles, a lane's 8 values of the reduction each, in N parts (1: bf16).
template <typename F, int Q, int N>
struct Frag {
  v8bf p[N][Q];
};

// Reduction contiguous: value e of tile q is p[q * tile + e].
template <typename F, int Q, int N>
__device__ __forceinline__ void load_contiguous(const F* p, int64_t tile, const bool (&ok)[Q], Frag<F, Q, N>& f) {
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if constexpr (kF32<F>) {
      v4f a = {0.f, 0.f, 0.f, 0.f}, b = a;
      if (ok[q]) {
        a = *reinterpret_cast<const v4f*>(p + q * tile);
        b = *reinterpret_cast<const v4f*>(p + q * tile + 4);
      }
      const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      const Parts<N> s = split<N>(v);
#pragma unroll
      for (int n = 0; n < N; ++n) f.p[n][q] = s.p[n];
    } else {
      v4u a = {0, 0, 0, 0};
      if (ok[q]) a = *reinterpret_cast<const v4u*>(p + q * tile);
      f.p[0][q] = __builtin_bit_cast(v8bf, a);
    }
  }
}

// Reduction strided: value e of tile q is p[e * step + q], so that Q tiles come with one vector load a value.
template <typename F, int Q, int N>
__device__ __forceinline__ void load_strided(const F* p, int64_t step, bool ok, Frag<F, Q, N>& f) {
  typedef F VecT __attribute__((ext_vector_type(Q > 1 ? Q : 2)));
  if constexpr (kF32<F>) {
    float v[Q][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (Q == 1) {
        v[0][e] = ok ? p[e * step] : 0.f;
      } else {
        VecT t = {};
        if (ok) t = *reinterpret_cast<const VecT*>(p + e * step);
#pragma unroll
        for (int q = 0; q < Q; ++q) v[q][e] = t[q];
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Parts<N> s = split<N>(v[q]);
#pragma unroll
      for (int n = 0; n < N; ++n) f.p[n][q] = s.p[n];
    }
  } else {
    typedef uint16_t VecU __attribute__((ext_vector_type(Q > 1 ? Q : 2)));
    uint32_t v[Q][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (Q == 1) {
        v[0][e] = ok ? reinterpret_cast<const uint16_t*>(p)[e * step] : 0;
      } else {
        VecU t = {};
        if (ok) t = *reinterpret_cast<const VecU*>(reinterpret_cast<const uint16_t*>(p) + e * step);
#pragma unroll
        for (int q = 0; q < Q; ++q) v[q][e] = t[q];
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      v4u w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[q][2 * i] | v[q][2 * i + 1] << 16;
      f.p[0][q] = __builtin_bit_cast(v8bf, w);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Down: part[slice][t][j] = sum over the slice's columns c of x[t][c] F_a[j][c], scaled where one slice is all
// ---------------------------------------------------------------------------------------------------------------
// A workgroup: 64 rows, a slice of columns, Q tiles of 16 ranks.  Its waves take 64 columns in turn (a row's 128 bytes of x),
// all 64 rows and all ranks, so that a factor's fragment serves four MFMAs; their sums meet in LDS.  (A slice's row
// tiles on one die, so that its part of the factors comes into one cache: 171 -> 166 us at 4 x 4608 rows x 6144 with the "up",
// but 156 -> 160 where a quarter of the rows has no adapter, and with the tiles spread over them 245 -> 278 at 16896 x 16384.)
template <typename F, bool kWide, int Q>
__global__ __launch_bounds__(THREADS) void down_kernel(Rows rows, const uint16_t* x, int C, const F* factor, int64_t one,
                                                       int slice_cols, float* part) {
  constexpr int RS = 16 * Q + 4;        // a row of sums in LDS
  constexpr int N = kF32<F> ? 3 : 1;    // u and g go into gradients in f32, and a served row has a trained one's bits
  extern __shared__ float sums[];       // 4 waves x 64 rows x RS
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, m = lane % 16, g = lane / 16;
  const int row0 = blockIdx.x * ROWS, j0 = blockIdx.z * 16 * Q;
  const int begin = blockIdx.y * slice_cols, end = min(C, begin + slice_cols);
  const int id = adapter_of(rows, row0 + lane);
  const uint16_t* xr[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) xr[t] = x + (int64_t)min(row0 + 16 * t + m, rows.T - 1) * C + 8 * g;
  uint64_t left = __ballot(id >= 0);
  while (left) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mask = __ballot(id == a);
    left &= ~mask;
    const int r = rank_of(rows, a);
    if (j0 >= r) continue;
    const float scale = scale_of(rows, a);
    v4f acc[4][Q] = {};
    bool ok[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) ok[q] = j0 + 16 * q + m < r;
    const bool some = j0 + Q * m < r;
    const F* f = factor + a * one;
    for (int c0 = begin + 64 * wave; c0 < end; c0 += 64 * 4) {
      v8bf xv[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t) xv[h][t] = *reinterpret_cast<const v8bf*>(xr[t] + c0 + 32 * h);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 32 * h + 8 * g;
        Frag<F, Q, N> fr;
        if constexpr (kWide) load_contiguous<F, Q, N>(f + (int64_t)(j0 + m) * C + c, 16 * (int64_t)C, ok, fr);
        else load_strided<F, Q, N>(f + (int64_t)c * rows.R + j0 + Q * m, rows.R, some, fr);
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) acc[t][q] = mfma(fr.p[n][q], xv[h][t], acc[t][q]);
      }
    }
    // a lane's sums: token 16 t + m, ranks 16 q + 4 g + i, or (strided) Q (4 g + i) + q
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float* s = sums + (wave * ROWS + 16 * t + m) * RS;
      if constexpr (kWide) {
#pragma unroll
        for (int q = 0; q < Q; ++q) *reinterpret_cast<v4f*>(s + 16 * q + 4 * g) = acc[t][q];
      } else {
#pragma unroll
        for (int k = 0; k < Q; ++k) {       // a lane's 4 Q ranks follow each other
          v4f v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[t][(4 * k + e) % Q][(4 * k + e) / Q];
          *reinterpret_cast<v4f*>(s + 4 * Q * g + 4 * k) = v;
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * 4 * Q; i += THREADS) {
      const int row = i / (4 * Q), j = 4 * (i % (4 * Q));
      if (!(mask >> row & 1) || j0 + j >= whole(r)) continue;
      v4f v = *reinterpret_cast<const v4f*>(sums + row * RS + j);
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const v4f*>(sums + (w * ROWS + row) * RS + j);
      if (gridDim.y == 1) v *= scale;
      if constexpr (!kWide) v = counted(v, j0 + j, r);      // else nothing was loaded there
      *reinterpret_cast<v4f*>(part + ((int64_t)blockIdx.y * rows.T + row0 + row) * rows.R + j0 + j) = v;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Up: out[t][c] = y[t][c] + sum_j u[t][j] F_a[j][c]
// ---------------------------------------------------------------------------------------------------------------
// A workgroup: 64 rows, 256 columns at a time.  It holds u in LDS in two bf16 halves; a wave takes 64 columns of all rows, so
// that a factor's fragment (in f32 split on its way) serves four tiles, and y's vectors are on their way while it computes.  The
// order of a tile's columns among MFMA rows is chosen so that a lane ends with 16 columns of a row in two pieces of 8.  y comes
// and out goes in whole lines of 128 bytes, 8 rows an instruction, past the cache, and changes places with the lanes' pieces in
// LDS.  In pieces (4 lanes to 64 bytes of a row) and through the cache the forward took 172 us for 153 at 4 x 4608 rows x 6144 (226
// MB of y and of out: 86 us, 5.4 TB/s), 246 for 222 at 16896 x 16384 -> 6144 with 389 for 346 in the backward, 93 for 83 at
// 4 x 768 x 6144 -> 16384 with rank 64 in f32; a call between the base's product and a reader of out gains as much (57 MB 91.5 ->
// 83, 12 MB 30.3 -> 29.6 with both).
template <typename F, bool kWide>
__global__ __launch_bounds__(THREADS) void up_kernel(Rows rows, const float* u, const uint16_t* y, int C, const F* factor,
                                                     int64_t one, int held, int passes, int groups, int slices, float* sum,
                                                     uint16_t* out) {
  constexpr int TR = 4;                 // tiles of 16 rows
  extern __shared__ uint16_t halves[];  // u in two halves of ROWS x RS, then a place of ROWS x LS for each wave
  const int RS = held + 8;              // 16 bytes off the banks' turn
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, m = lane % 16, g = lane / 16;
  uint16_t *hi = halves, *lo = halves + ROWS * RS, *mine = halves + 2 * ROWS * RS + wave * ROWS * LS;
  const int at = lane / 8 * LS + 8 * (lane % 8);      // a lane's 16 bytes of a line
  // a row's columns on neighbouring workgroups
  const int row0 = blockIdx.x / groups * ROWS, first = blockIdx.x % groups * passes;
  const int id = adapter_of(rows, row0 + lane);
  uint64_t left = __ballot(id >= -1);
  while (left) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mask = __ballot(id == a);
    left &= ~mask;
    const int own = rank_of(rows, a), r = whole(own);
    const F* f = factor + (int64_t)max(a, 0) * one;
    const float scale = slices > 1 && a >= 0 ? scale_of(rows, a) : 1.f;
    uint32_t live = 0;      // a lane's rows of lines, 8 k + lane / 8
#pragma unroll
    for (int k = 0; k < 8; ++k) live |= (uint32_t)(mask >> (8 * k + lane / 8) & 1) << k;
    for (int p = 0; p < passes; ++p) {
      const int c0 = (first + p) * 256 + 64 * wave;
      const bool in = c0 < C;
      const int64_t line = (int64_t)(row0 + lane / 8) * C + c0 + 8 * (lane % 8);
      v4u old[8] = {};
      asm volatile("" : "+v"(live));      // tested where it is wanted: eight masks held through the loop spill scalars
      if (y && in) {
        const uint16_t* from = y + line;
#pragma unroll
        for (int k = 0; k < 8; ++k, from += 8 * (int64_t)C)
          if (live >> k & 1) old[k] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(from));
      }
      v4f acc[TR][4] = {};
      for (int j0 = 0; j0 < r; j0 += held) {
        const int n = min(held, r - j0), n32 = (n + 31) & ~31;
        if (p == 0 || r > held) {
          __syncthreads();
          for (int i = threadIdx.x; i < ROWS * (n32 / 8); i += THREADS) {
            const int row = i / (n32 / 8), j = 8 * (i % (n32 / 8));
            float v[8] = {};
            if ((mask >> row & 1) && j < n) {
              const float* q = u + (int64_t)(row0 + row) * rows.R + j0 + j;
              v4f b = *reinterpret_cast<const v4f*>(q), c = *reinterpret_cast<const v4f*>(q + 4);
              if (slices > 1) {       // as join_kernel does it
                const int64_t next = (int64_t)rows.T * rows.R;
#pragma unroll 4
                for (int s = 1; s < slices; ++s) {
                  b += *reinterpret_cast<const v4f*>(q + s * next);
                  c += *reinterpret_cast<const v4f*>(q + s * next + 4);
                }
                b *= scale;
                c *= scale;
                if (sum && first + p == 0) {
                  float* to = sum + (int64_t)(row0 + row) * rows.R + j0 + j;
                  *reinterpret_cast<v4f*>(to) = b;
                  *reinterpret_cast<v4f*>(to + 4) = c;
                }
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] = b[e];
                v[e + 4] = c[e];
              }
            }
            const Parts<2> s = split<2>(v);
            *reinterpret_cast<v8bf*>(hi + row * RS + j) = s.p[0];
            *reinterpret_cast<v8bf*>(lo + row * RS + j) = s.p[1];
          }
          __syncthreads();
        }
        if (in) {
          constexpr int N = kF32<F> ? 2 : 1;
          // 32 ranks of the reduction, or the last 16, of which lanes g and g + 2 then have the same ones: those below 2 the
          // factor's (f32) or u's (bf16 factors) upper parts, the others the lower, and a product fewer does (dx of 16896 x 16384,
          // rank 16 in f32, with its "down": 127 -> 120 us)
          auto step = [&](int j, auto last) {
            const int of = j + 8 * (last ? g % 2 : g);
            const bool upper = g < 2;
            Frag<F, 4, N> fr;
            if constexpr (kWide) {
              // MFMA row m of tile q: column 32 (m / 2 % 2) + 8 (m / 4) + 4 (m % 2) + q, four tiles with one load
              const int col = 32 * (m % 4 / 2) + 8 * (m / 4) + 4 * (m % 2);
              load_strided<F, 4, N>(f + (int64_t)(j0 + of) * C + c0 + col, C, true, fr);
            } else {
              // row m of tile q: column 32 (q / 2) + 8 (m / 4) + 4 (q % 2) + m % 4
              const bool ok[2] = {of < n, of < n};      // always: a step later than without it, 83 us for 87 at rank 64 in f32
              const F* b = f + (int64_t)(c0 + 8 * (m / 4) + m % 4) * rows.R + j0 + of;
              Frag<F, 2, N> half[2];
              load_contiguous<F, 2, N>(b, 4 * (int64_t)rows.R, ok, half[0]);
              load_contiguous<F, 2, N>(b + 32 * (int64_t)rows.R, 4 * (int64_t)rows.R, ok, half[1]);
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < N; ++k) fr.p[k][q] = half[q / 2].p[k][q % 2];
            }
            if (j0 + j + (last ? 16 : 32) > own) {      // the adapter's last ranks
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < N; ++k) fr.p[k][q] = counted(fr.p[k][q], own - j0 - of);
            }
            if constexpr (last && N > 1) {
#pragma unroll
              for (int q = 0; q < 4; ++q) fr.p[0][q] = upper ? fr.p[0][q] : fr.p[1][q];
            }
#pragma unroll
            for (int t = 0; t < TR; ++t) {
              const int e = (16 * t + m) * RS + of;
              if constexpr (last && N == 1) {
                const v8bf u = *reinterpret_cast<const v8bf*>((upper ? hi : lo) + e);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[t][q] = mfma(fr.p[0][q], u, acc[t][q]);
                continue;
              }
              const v8bf uh = *reinterpret_cast<const v8bf*>(hi + e), ul = *reinterpret_cast<const v8bf*>(lo + e);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                acc[t][q] = mfma(fr.p[0][q], uh, acc[t][q]);
                acc[t][q] = mfma(fr.p[0][q], ul, acc[t][q]);
                if constexpr (!last && N > 1) acc[t][q] = mfma(fr.p[1][q], uh, acc[t][q]);
              }
            }
          };
          for (int j = 0; j + 32 <= n; j += 32) step(j, std::false_type{});
          if (n % 32) step(n / 32 * 32, std::true_type{});
        }
      }
      if (!in) continue;
      // a lane: row 16 t + m, columns 32 h + 8 g + e.  The wave's own place: its LDS operations stay in order
      v4u pieces[TR][2] = {};
      uint16_t* place = mine + m * LS + 8 * g;
      if (y) {
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<v4u*>(mine + at + 8 * k * LS) = old[k];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < TR; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) pieces[t][h] = *reinterpret_cast<const v4u*>(place + 16 * t * LS + 32 * h);
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int t = 0; t < TR; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const v4u b = pieces[t][h];
          v4u o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int e = 2 * i + k;      // of 8
              // strided: tile e % 4 holds column 4 (e / 4) + e % 4 of the piece in its MFMA row 2 h + e / 4
              const float d = kWide ? acc[t][e % 4][2 * h + e / 4] : acc[t][2 * h + e / 4][e % 4];
              v[k] = d + (k ? __uint_as_float(b[i] & 0xffff0000u) : __uint_as_float(b[i] << 16));
            }
            o[i] = pack_bf16x2(v[0], v[1]);
          }
          *reinterpret_cast<v4u*>(place + 16 * t * LS + 32 * h) = o;
        }
      }
      __builtin_amdgcn_wave_barrier();
      uint16_t* to = out + line;
#pragma unroll
      for (int k = 0; k < 8; ++k, to += 8 * (int64_t)C) {
        const v4u o = *reinterpret_cast<const v4u*>(mine + at + 8 * k * LS);
        if (live >> k & 1) __builtin_nontemporal_store(o, reinterpret_cast<v4u*>(to));
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------------------------------------------
// One row a workgroup: its adapter's factors are read as they lie, once, by vectors, on the vector unit; a row of another
// request on another workgroup.  Rows that share an adapter read it again from L2.
template <typename F>
__device__ __forceinline__ void load8(const F* p, float (&v)[8]) {
  if constexpr (kF32<F>) {
    const v4f a = *reinterpret_cast<const v4f*>(p), b = *reinterpret_cast<const v4f*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    const v4u w = *reinterpret_cast<const v4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// Workgroups in the order that the hardware deals to its 8 dies, one each in turn: the same part of the columns for all rows
// goes to one die, row after row, so that rows of one adapter find its factors in that die's L2 (64 rows of 32 adapters: up
// 23 -> 15 us).  With fewer than 8 parts a row's parts follow each other.
struct RowPart {
  int row, part;
};

__device__ __forceinline__ RowPart row_part(int T, int parts) {
  const int id = blockIdx.x;
  if (parts < 8) return {id / parts, id % parts};
  return {id / 8 % T, id / 8 / T * 8 + id % 8};
}

int64_t row_parts(int64_t T, int64_t parts) { return T * (parts < 8 ? parts : (parts + 7) / 8 * 8); }

// A wave's sums of four ranks over columns begin .. end of a row; f: the first of them.
template <typename F>
__device__ __forceinline__ v4f four_ranks(const uint16_t* x, const F* f, int C, int begin, int end) {
  float acc[4] = {};
#pragma unroll 2
  for (int c = begin + 8 * (int)(threadIdx.x % 64); c < end; c += 512) {
    float xv[8], fv[4][8];
    load8(x + c, xv);
#pragma unroll
    for (int q = 0; q < 4; ++q) load8(f + (int64_t)q * C + c, fv[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[q] = __builtin_fmaf(xv[e], fv[q][e], acc[q]);
  }
  v4f sum;
#pragma unroll
  for (int q = 0; q < 4; ++q) sum[q] = k2q_rot::wave_sum(acc[q]);
  return sum;
}

// Down: a wave takes 4 ranks over the slice's columns, a workgroup 16.
template <typename F>
__global__ __launch_bounds__(THREADS) void down_row_kernel(Rows rows, const uint16_t* x, int C, const F* factor, int64_t one,
                                                           int slice_cols, int slices, float* part) {
  const RowPart at = row_part(rows.T, slices * (rows.R / 16));
  const int row = at.row, slice = at.part % slices, lane = threadIdx.x % 64;
  const int j = at.part / slices * 16 + threadIdx.x / 64 * 4;
  const int a = __builtin_amdgcn_readfirstlane(adapter_of(rows, row));
  const int r = rank_of(rows, a);
  if (j >= whole(r)) return;
  const int begin = slice * slice_cols, end = min(C, begin + slice_cols);
  const v4f sum = four_ranks(x + (int64_t)row * C, factor + a * one + (int64_t)j * C, C, begin, end);
  if (lane == 0) *reinterpret_cast<v4f*>(part + ((int64_t)slice * rows.T + row) * rows.R + j) = counted(sum, j, r);
}

// Up, from B: L lanes share a column's ranks, 16 bytes each, and a wave's 64 columns come in L steps; then every lane has one
// column's sum.  kBoth: the workgroup makes the row's u itself, as the "down" does it in one slice.
template <typename F, int L, bool kBoth>
__global__ __launch_bounds__(THREADS) void up_row_kernel(Rows rows, const float* part, int slices, float* sum, const uint16_t* y,
                                                         int C, const F* factor, int64_t one, const uint16_t* x, int K,
                                                         const F* A, uint16_t* out) {
  constexpr int E = 16 / sizeof(F);
  extern __shared__ float u[];          // R
  const RowPart of = row_part(rows.T, (C + THREADS - 1) / THREADS);
  const int row = of.row, lane = threadIdx.x % 64, sub = E * (lane % L);
  const int a = __builtin_amdgcn_readfirstlane(adapter_of(rows, row));
  const int r = rank_of(rows, a);
  const int c0 = of.part * THREADS + threadIdx.x / 64 * 64, mine = c0 + lane % L * (64 / L) + lane / L;
  const bool in = c0 < C;
  // the columns' factors are on their way before u is added up
  const F* f = factor + max(a, 0) * one + (int64_t)(c0 + lane / L) * rows.R + sub;
  v4u w[L] = {};
  auto fetch = [&](int j) {
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (in && j + sub < r) w[i] = *reinterpret_cast<const v4u*>(f + (int64_t)i * (64 / L) * rows.R + j);
  };
  fetch(0);
  const float base = y && in ? bf16_bits_to_f32(y[(int64_t)row * C + mine]) : 0.f;
  if (r) {
    const float scale = scale_of(rows, a);
    if constexpr (kBoth) {
      const F* from = A + (int64_t)a * rows.R * K;
      for (int j = threadIdx.x / 64 * 4; j < whole(r); j += 16) {
        const v4f v = counted(four_ranks(x + (int64_t)row * K, from + (int64_t)j * K, K, 0, K) * scale, j, r);
        if (lane) continue;
        *reinterpret_cast<v4f*>(u + j) = v;
        if (sum && of.part == 0) *reinterpret_cast<v4f*>(sum + (int64_t)row * rows.R + j) = v;
      }
    } else {
      for (int j = threadIdx.x; j < whole(r); j += THREADS) {
        const float* p = part + (int64_t)row * rows.R + j;
        float v = *p;
#pragma unroll 4
        for (int s = 1; s < slices; ++s) v += p[(int64_t)s * rows.T * rows.R];
        v *= scale;
        u[j] = v;
        if (sum && of.part == 0) sum[(int64_t)row * rows.R + j] = v;
      }
    }
    __syncthreads();
  }
  if (!in) return;
  float d[L] = {};
  for (int j = 0; j < r; j += L * E) {
    if (j) fetch(j);
    if (j + sub < r) {
      if (r % E) {      // of the adapter's last vector
        const int n = r - j - sub;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t keep = kF32<F> ? k < n ? ~0u : 0u : (2 * k < n ? 0xffffu : 0u) | (2 * k + 1 < n ? 0xffff0000u : 0u);
#pragma unroll
          for (int i = 0; i < L; ++i) w[i][k] &= keep;
        }
      }
      float uv[E];
#pragma unroll
      for (int e = 0; e < E; ++e) uv[e] = u[j + sub + e];
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float v = kF32<F> ? __uint_as_float(w[i][e % 4])
                                  : e % 2 ? __uint_as_float(w[i][e / 2 % 4] & 0xffff0000u) : __uint_as_float(w[i][e / 2 % 4] << 16);
          d[i] = __builtin_fmaf(v, uv[e], d[i]);
        }
    }
  }
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float t = d[i];
    t += k2q_rot::dpp_f<0xB1>(t);
    if constexpr (L > 2) t += k2q_rot::dpp_f<0x4E>(t);
    if constexpr (L > 4) t += k2q_rot::dpp_f<0x141>(t);
    if constexpr (L > 8) t += k2q_rot::dpp_f<0x140>(t);
    v = lane % L == i ? t : v;
  }
  out[(int64_t)row * C + mine] = (uint16_t)f32_to_bf16_bits(base + v);
}

// The slices' sums, scaled: once, ahead of an "up" whose workgroups would each add them up (4 x 768 rows, 22 slices of 64
// ranks, 24 workgroups a row: 57 us; added up once, both take 24), or where the sums over rows want them.
__global__ __launch_bounds__(THREADS) void join_kernel(Rows rows, const float* part, int slices, float* sum) {
  const int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 4;
  const int row = (int)(i / rows.R), j = (int)(i % rows.R);
  const int a = adapter_of(rows, row);
  if (a < 0 || j >= whole(rank_of(rows, a))) return;
  v4f v = *reinterpret_cast<const v4f*>(part + i);
#pragma unroll 4
  for (int s = 1; s < slices; ++s) v += *reinterpret_cast<const v4f*>(part + (int64_t)s * rows.T * rows.R + i);
  *reinterpret_cast<v4f*>(sum + i) = v * scale_of(rows, a);
}

// ---------------------------------------------------------------------------------------------------------------
// Sums over an adapter's rows
// ---------------------------------------------------------------------------------------------------------------
// Rows by adapter: the batch's ids sorted (stably), and the pieces of at most `chunk` rows that workgroups take.
struct Item {
  int32_t a, begin, end;      // rows begin .. end of the adapter's, in the order of the batch
  int32_t slot;               // where its partial sums go: -1, the adapter has no other piece
};

struct Plan {
  int32_t* head;      // pieces
  int32_t* start;     // count + 1: an adapter's first place in order
  int32_t* first;     // count + 1: its first piece
  int32_t* order;     // ids in the order of their adapters
  Item* items;
};

constexpr int PLAN = 1024;            // threads: one an adapter
constexpr int HELD = 32768;           // ids in LDS, for both passes: 16896 ids 26 -> 14 us

// Inclusive sums of three values over the workgroup's threads; waves: 3 x 16 in LDS.
__device__ __forceinline__ void scan(int (&v)[3], int32_t* waves) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    for (int d = 1; d < 64; d *= 2) {
      const int t = __shfl_up(v[k], d);
      if (lane >= d) v[k] += t;
    }
  if (lane == 63)
    for (int k = 0; k < 3; ++k) waves[16 * k + wave] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int t = lane < wave ? waves[16 * k + lane] : 0;      // the waves before this one
#pragma unroll
    for (int d = 8; d; d /= 2) t += __shfl_xor(t, d);
    v[k] += __shfl(t, 0);
  }
}

// One workgroup: every wave counts a run of ids, then places it; no atomics, so the order is the batch's.
__global__ __launch_bounds__(PLAN) void plan_kernel(Rows rows, int ids, int chunk, Plan plan) {
  extern __shared__ int32_t lds[];      // 16 waves x count, then 48, then as many ids as fit
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = rows.count;
  int32_t* mine = lds + wave * n;
  int16_t* held = reinterpret_cast<int16_t*>(lds + 16 * n + 48);
  const int most = min(ids, HELD);
  for (int i = threadIdx.x; i < 16 * n; i += PLAN) lds[i] = 0;
  auto hold = [&](auto* p) {        // a branch on the type inside would wait for each load by itself: 20 us at 16896 ids
    for (int i0 = threadIdx.x; i0 < most; i0 += 8 * PLAN) {
      int64_t id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) id[k] = p[min(i0 + k * PLAN, most - 1)];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k * PLAN < most) held[i0 + k * PLAN] = (int16_t)(id[k] < 0 || id[k] >= n ? -1 : id[k]);
    }
  };
  if (rows.wide) hold(static_cast<const int64_t*>(rows.ids));
  else hold(static_cast<const int32_t*>(rows.ids));
  __syncthreads();
  const int run = (ids + 15) / 16, begin = min(ids, wave * run), end = min(ids, begin + run);
  for (int pass = 0; pass < 2; ++pass) {
    for (int i0 = begin; i0 < end; i0 += 64) {
      const int i = i0 + lane, id = i >= end ? -1 : i < most ? held[i] : adapter_at(rows, i);
      uint64_t left = __ballot(id >= 0);
      while (left) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t mask = __ballot(id == a);
        left &= ~mask;
        const int at = mine[a];
        if (pass && id == a) plan.order[at + __popcll(mask & ((uint64_t(1) << lane) - 1))] = i;
        if (lane == 0) mine[a] = at + __popcll(mask);
      }
    }
    __syncthreads();
    if (pass) break;
    const int a = threadIdx.x;
    int total = 0;
    if (a < n)
      for (int w = 0; w < 16; ++w) total += lds[w * n + a];
    // one at least, without rows: its sums are zeros
    const int of = total * rows.per, pieces = a < n ? max(of / chunk + (of % chunk != 0), 1) : 0;
    const int shared = pieces > 1 ? pieces : 0;
    int sums[3] = {total, pieces, shared};
    scan(sums, lds + 16 * n);
    const int first = sums[1] - pieces, slot = sums[2] - shared;
    int at = sums[0] - total;
    if (a < n) {
      plan.start[a] = at;
      for (int w = 0; w < 16; ++w) {
        const int c = lds[w * n + a];
        lds[w * n + a] = at;
        at += c;
      }
    }
    if (a < n) {
      plan.first[a] = first;
      for (int p = 0; p < pieces; ++p)
        plan.items[first + p] = Item{a, p * chunk, p + 1 < pieces ? (p + 1) * chunk : of, pieces > 1 ? slot + p : -1};
    }
    if (a == n - 1) {
      plan.start[n] = sums[0];
      plan.head[0] = plan.first[n] = sums[1];
    }
    __syncthreads();
  }
}

struct Job {
  const uint16_t* x;      // T x C
  const float* p;         // T x R, scaled
  int C;
  int blocks;             // of 128 columns
  int swapped;            // the result is C x R (dB), else R x C (dA)
  int64_t one;            // R C
  void* out;
  float* part;            // slots of R C
};

constexpr int COLS = 128;
constexpr int JOBS = 2;

struct Jobs {
  Job j[JOBS];
  int32_t blocks;         // of all
};

// A workgroup: 128 columns of a piece's rows, Q tiles of 16 ranks.  Its waves take 32 rows in turn; both operands come with
// the wide index contiguous and the rows strided, so a lane loads 8 rows of 8 columns (and of Q ranks) and turns them in
// registers: each 16-byte load of x serves 8 MFMA tiles.  The waves' sums are added in LDS in their order.
template <typename F, int Q>
__global__ __launch_bounds__(THREADS, 2) void sums_kernel(Rows rows, Plan plan, Jobs jobs) {
  constexpr int RR = 16 * Q;
  constexpr int HALF = COLS / 2, PART = RR * HALF + 4 * (RR > HALF ? RR : HALF);
  extern __shared__ float sums[];       // 4 waves x PART
  if ((int)blockIdx.y >= plan.head[0]) return;
  const Item it = plan.items[blockIdx.y];
  const int second = (int)blockIdx.x >= jobs.j[0].blocks;
  const Job job = jobs.j[second];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, m = lane % 16, g = lane / 16;
  const int c0 = ((int)blockIdx.x - (second ? jobs.j[0].blocks : 0)) * COLS, j0 = blockIdx.z * RR;
  const int r = rank_of(rows, it.a), C = job.C;
  const bool some = j0 + Q * m < whole(r), in = c0 + 8 * m < C;
  const int32_t* order = plan.order + plan.start[it.a];
  const uint16_t* x = job.x + c0 + (in ? 8 * m : 0);
  const float* p = job.p + j0 + (some ? Q * m : 0);
  typedef float VecT __attribute__((ext_vector_type(Q > 1 ? Q : 2)));
  v4f acc[8][Q] = {};
  if (j0 < r)
    for (int b = it.begin + 32 * wave; b < it.end; b += 32 * 4) {
      // lane l finds row b + l; past the piece's end the last one, whose factor is zero
      const int at = min(b + lane % 32, it.end - 1), q = at / rows.per;
      const int row = order[q] * rows.per + (at - q * rows.per);
      v4u xv[8];
      float pv[Q][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t of = __shfl(row, 8 * g + e);
        xv[e] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(x + of * C));      // read no more
        const bool live = some && b + 8 * g + e < it.end;
        if constexpr (Q == 1) {
          pv[0][e] = live ? p[of * rows.R] : 0.f;
        } else {
          VecT t = {};
          if (live) t = *reinterpret_cast<const VecT*>(p + of * rows.R);
#pragma unroll
          for (int k = 0; k < Q; ++k) pv[k][e] = t[k];
        }
      }
      constexpr int N = kF32<F> ? 3 : 2;
      Parts<N> ps[Q];
#pragma unroll
      for (int k = 0; k < Q; ++k) ps[k] = split<N>(pv[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(xv[2 * i + 1][k / 2], xv[2 * i][k / 2], k % 2 ? 0x07060302u : 0x05040100u);
        const v8bf xf = __builtin_bit_cast(v8bf, w);
#pragma unroll
        for (int t = 0; t < Q; ++t)
#pragma unroll
          for (int n = 0; n < N; ++n) acc[k][t] = mfma(xf, ps[t].p[n], acc[k][t]);
      }
    }
  // a lane: columns 8 (4 g + i) + k, ranks Q m + t.  Half of the columns (k below 4, then the rest) of all waves meet in LDS,
  // with the index that the result has inside inside; the sums leave in vectors of 4.
  const int inner = job.swapped ? RR : HALF, ld = inner + 4;
  for (int h = 0; h < 2; ++h) {
    float* s = sums + wave * PART;
    if (job.swapped) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          VecT v;
#pragma unroll
          for (int t = 0; t < Q; ++t) v[t] = h ? acc[4 + k][t][i] : acc[k][t][i];
          float* to = s + (4 * (4 * g + i) + k) * ld + Q * m;
          if constexpr (Q == 1) *to = v[0];
          else *reinterpret_cast<VecT*>(to) = v;
        }
    } else {
#pragma unroll
      for (int t = 0; t < Q; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4f v;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = h ? acc[4 + k][t][i] : acc[k][t][i];
          *reinterpret_cast<v4f*>(s + (Q * m + t) * ld + 4 * (4 * g + i)) = v;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < RR * HALF / 4; i += THREADS) {
      const int o = i / (inner / 4), e = 4 * (i % (inner / 4));
      const int lc = job.swapped ? o : e;
      const int c = c0 + lc / 4 * 8 + 4 * h + lc % 4, j = j0 + (job.swapped ? e : o);
      if (c >= C || j >= rows.R) continue;
      v4f v = *reinterpret_cast<const v4f*>(sums + o * ld + e);
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const v4f*>(sums + w * PART + o * ld + e);
      // zeros behind the adapter's ranks: products with what is not finite in x are none
      v = job.swapped ? counted(v, j, r) : j < r ? v : v4f{0.f, 0.f, 0.f, 0.f};
      const int64_t at = job.swapped ? (int64_t)c * rows.R + j : (int64_t)j * C + c;
      if (it.slot >= 0) {
        *reinterpret_cast<v4f*>(job.part + it.slot * job.one + at) = v;
      } else if constexpr (kF32<F>) {
        *reinterpret_cast<v4f*>(static_cast<float*>(job.out) + it.a * job.one + at) = v;
      } else {
        *reinterpret_cast<v2u*>(static_cast<uint16_t*>(job.out) + it.a * job.one + at) =
            v2u{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    }
    __syncthreads();
  }
}

// What pieces left: the sum of an adapter's in their order.
template <typename F>
__global__ __launch_bounds__(THREADS) void pieces_kernel(Plan plan, Jobs jobs) {
  const int a = blockIdx.y, second = (int)blockIdx.x >= jobs.j[0].blocks;
  const Job job = jobs.j[second];
  const int first = plan.first[a], n = plan.first[a + 1] - first;
  const int64_t i = ((int64_t)((int)blockIdx.x - (second ? jobs.j[0].blocks : 0)) * THREADS + threadIdx.x) * 4;
  if (n == 1 || i >= job.one) return;
  const float* p = job.part + plan.items[first].slot * job.one + i;
  v4f v = *reinterpret_cast<const v4f*>(p);
  for (int s = 1; s < n; ++s) v += *reinterpret_cast<const v4f*>(p + s * job.one);
  if constexpr (kF32<F>)
    *reinterpret_cast<v4f*>(static_cast<float*>(job.out) + a * job.one + i) = v;
  else
    *reinterpret_cast<v2u*>(static_cast<uint16_t*>(job.out) + a * job.one + i) =
        v2u{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// ---------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------
int64_t up16(int64_t n) { return (n + 15) & ~int64_t(15); }

int check(const k2q_bank* b, int64_t T, int64_t per) {
  if (!b || !b->A || !b->B || !k2q_aligned(b->A, 16) || !k2q_aligned(b->B, 16) || b->count < 1 || b->R < 16 || b->R % 16 ||
      b->K < 64 || b->K % 64 || b->N < 64 || b->N % 64 || (b->dtype != K2Q_DTYPE_BF16 && b->dtype != K2Q_DTYPE_F32) ||
      !b->ids || !k2q_aligned(b->ids, b->ids64 ? 8 : 4) || !k2q_aligned(b->ranks, 4) || !k2q_aligned(b->scales, 4) || T < 1 ||
      per < 1 || T % per)
    return K2Q_EINVAL;
  // The row numbers of a piece, up to T + its length, fit 32 bits; and so do the threads of a launch: T C / 64 of "up",
  // T R / 4 of the join, R (K + N) / 4 of the gradients' join.
  const int64_t most = b->K > b->N ? b->K : b->N;
  if (b->count > K2Q_MAX_ADAPTERS || b->R > K2Q_MAX_RANK || T > 1 << 30 || most > 1 << 24 || T * most > (int64_t)1 << 37 ||
      T * b->R > (int64_t)1 << 33 || b->R * most > (int64_t)1 << 31)
    return K2Q_EUNSUPPORTED;
  return K2Q_OK;
}

Rows rows_of(const k2q_bank* b, int64_t T, int64_t per) {
  return {b->ids, b->ranks, b->scales, b->scale, b->ids64, (int32_t)per, (int32_t)T, b->count, b->R};
}

int tiles_of(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : 4; }

// Slices of a "down" over C columns: up to 16 workgroups a CU, so that the last ones end together, of 1024 columns or more (a
// workgroup's sums in LDS cost as much as 500 columns); where that leaves fewer than two a CU, slices down to 256 columns.
// 16896 x 16384, rank 16, us at 1 / 3 / 5 / 10 / 16 slices (with the "up") 337 / 265 / 258 / 248 / 244; 18432 x 6144, rank 32
// 191 / 177 / 170 / 172 / 177; 1000 x 2560 at 1 / 3 / 5 / 10 58 / 37 / 30 / 26.
int down_slices(int64_t T, int64_t C, int64_t R) {
  const int64_t groups = ((T + ROWS - 1) / ROWS) * ((R + 16 * tiles_of(R) - 1) / (16 * tiles_of(R)));
  const int64_t cus = k2q_cu_count(), large = C / 1024, most = (C + 255) / 256;
  int64_t s = 16 * cus / groups;
  s = s > large ? large : s;
  if (groups * s < 2 * cus) s = (2 * cus + groups - 1) / groups;
  s = s > most ? most : s < 1 ? 1 : s;
  const int64_t cols = ((C + s - 1) / s + 255) / 256 * 256;
  return (int)((C + cols - 1) / cols);
}

template <typename F, bool kWide>
void launch_down(const Rows& rows, const uint16_t* x, int64_t C, const void* f, int slices, float* part, hipStream_t st) {
  const int64_t cols = ((C + slices - 1) / slices + 255) / 256 * 256, one = (int64_t)rows.R * C;
  const int q = tiles_of(rows.R);
  const dim3 grid((unsigned)((rows.T + ROWS - 1) / ROWS), (unsigned)slices, (unsigned)((rows.R + 16 * q - 1) / (16 * q)));
  const int lds = 4 * ROWS * (16 * q + 4) * 4;
  const F* factor = static_cast<const F*>(f);
  auto go = [&](auto kernel, std::atomic<uint64_t>& once) {
    (void)k2q_lds_limit_once(kernel, lds, once);
    hipLaunchKernelGGL(kernel, grid, dim3(THREADS), lds, st, rows, x, (int)C, factor, one, (int)cols, part);
  };
  static std::atomic<uint64_t> once[3];
  if (q == 1) go(down_kernel<F, kWide, 1>, once[0]);
  else if (q == 2) go(down_kernel<F, kWide, 2>, once[1]);
  else go(down_kernel<F, kWide, 4>, once[2]);
}

void launch_join(const Rows& rows, const float* part, int slices, float* sum, hipStream_t st) {
  if (slices == 1) return;      // scaled already
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)(((int64_t)rows.T * rows.R / 4 + THREADS - 1) / THREADS)), dim3(THREADS), 0,
                     st, rows, part, slices, sum);
}

// Slices that the "up" adds up itself, in the order of the join: where all of its workgroups together read 32 MB or less of
// them, which costs less than a launch.  us of the forward with and without the join, by what they read: 685 x 640 -> 448, rank
// 16 (0.3 MB) 12.6 / 10.2; 1000 x 2560 -> 6144, rank 16 (15 MB) 26.0 / 25.3; 546 x 1600 -> 8384, rank 64 (32 MB) 20.8 / 19.6;
// 4000 x 6144 -> 16384, rank 16 (66 MB) 81.8 / 84.9; 4 x 768 x 6144 -> 16384, rank 64 (201 MB) 92.8 / 99.6.
constexpr int64_t JOIN = 32 << 20;

// Passes over 256 columns with one staging of u: two (four where the factor's rows are long and its loads wider), fewer
// where a CU would not get six workgroups.  4 x 4608 rows x 6144 at 1 / 2 / 4 passes 163 / 154 / 154 us, 16896 x 16384 (dx, with
// the factors' sums) 388 / 365 / 355.
template <typename F, bool kWide>
void launch_up(const Rows& rows, const float* part, int slices, float* sum, const uint16_t* y, int64_t C, const void* f,
               uint16_t* out, hipStream_t st) {
  const int64_t tiles = (rows.T + ROWS - 1) / ROWS, blocks = (C + 255) / 256, most = kWide ? 4 : 2;
  int64_t passes = tiles * blocks / (6 * (int64_t)k2q_cu_count());
  passes = passes < 1 ? 1 : passes > most ? most : passes;
  const int64_t groups = (blocks + passes - 1) / passes;
  const int held = rows.R < RANKS ? (rows.R + 31) & ~31 : RANKS;
  if (slices > 1 && (int64_t)slices * rows.T * rows.R * 4 * groups > JOIN) {
    float* to = sum ? sum : const_cast<float*>(part);       // or the first slice's place
    launch_join(rows, part, slices, to, st);
    part = to;
    slices = 1;
  }
  static std::atomic<uint64_t> once;
  (void)k2q_lds_limit_once(up_kernel<F, kWide>, (2 * ROWS * (RANKS + 8) + 4 * ROWS * LS) * 2, once);
  const int lds = (2 * ROWS * (held + 8) + 4 * ROWS * LS) * 2;
  hipLaunchKernelGGL((up_kernel<F, kWide>), dim3((unsigned)(tiles * groups)), dim3(THREADS), lds, st, rows,
                     part, y, (int)C, static_cast<const F*>(f), (int64_t)rows.R * C, held, (int)passes, (int)groups, slices, sum,
                     out);
}

// Few rows: the form of single rows, whose time grows with the rows, where that of tiles grows with the adapters that a tile
// meets, e at most.  us of rows / tiles, 6144 -> 16384 in f32 with rank 64; 6144 -> 6144 in f32 with rank 16:
//   one adapter       64 rows   23 / 20;  8.4 / 15      128 rows  37 / 20;  11 / 14     256 rows  71 / 22;  17 / 15
//   4 in any order    96 rows   38 / 51;  9.9 / 30      192 rows  59 / 53;  15 / 30     512 rows  137 / 60;  29 / 30
//   16 in any order   256 rows  80 / 170;  18 / 91      512 rows  152 / 193;  31 / 90   1024 rows  292 / 318;  59 / 110
//   16 that lie together                                 256 rows  77 / 69;  18 / 37    512 rows  140 / 48;  31 / 29
//   64 in any order   384 rows  174 / 486;  37 / 215    768 rows  321 / 768;  56 / 258  1024 rows  422 / 827;  77 / 268
//   64 that lie together                                 384 rows  156 / 161;  38 / 73  768 rows  267 / 151;  46 / 50
// Only the device knows which it is: the bound lies between the two orders' own.
bool few_rows(const k2q_bank* b, int64_t T, int64_t per) {
  const int64_t of_tile = (ROWS + per - 1) / per, e = of_tile < b->count ? of_tile : b->count;
  return T <= 768 && T <= 64 + 16 * e;
}

// Few rows: slices that give every CU four workgroups, of 512 columns or more.
int row_slices(int64_t T, int64_t C, int64_t R) {
  const int64_t groups = T * (R / 16), most = (C + 511) / 512;
  int64_t s = (4 * (int64_t)k2q_cu_count() + groups - 1) / groups;
  s = s > most ? most : s;
  const int64_t cols = ((C + s - 1) / s + 511) / 512 * 512;
  return (int)((C + cols - 1) / cols);
}

// One launch, whose workgroups each make their row's u: where an adapter's A has 192 KB at most, and all workgroups together
// read 32 MB at most.  us in a graph, two launches / one, bf16: 512 -> 1024 (f32), 1 and 64 rows 4.7 / 3.1, 5.3 / 3.5; 2560 ->
// 2560, 1, 32 (26 MB) and 64 rows (52 MB) 4.9 / 3.9, 5.3 / 4.8, 6.1 / 6.9; 6144 -> 1536, rank 16 (192 KB) 5.6 / 5.6, and the host
// makes one launch less; 1024 -> 4096, rank 64 in f32 (256 KB) 5.9 / 7.3; 6144 -> 16384, 8 rows (101 MB) 6.1 / 7.1.
constexpr int64_t ONE = 192 << 10, ALL = 32 << 20;

template <typename F>
void launch_rows(const Rows& rows, const uint16_t* x, int64_t K, const void* A, float* part, float* sum, const uint16_t* y,
                 int64_t N, const void* B, uint16_t* out, hipStream_t st) {
  const int64_t parts = (N + THREADS - 1) / THREADS;
  const int64_t read = rows.R * K * (int64_t)sizeof(F);
  const bool both = read <= ONE && rows.T * parts * read <= ALL;
  const int slices = row_slices(rows.T, K, rows.R);
  const int64_t cols = ((K + slices - 1) / slices + 511) / 512 * 512;
  if (!both)
    hipLaunchKernelGGL(down_row_kernel<F>, dim3((unsigned)row_parts(rows.T, slices * (rows.R / 16))), dim3(THREADS), 0, st,
                       rows, x, (int)K, static_cast<const F*>(A), (int64_t)rows.R * K, (int)cols, slices, part);
  const dim3 grid((unsigned)row_parts(rows.T, parts));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(THREADS), (size_t)rows.R * 4, st, rows, part, slices, sum, y, (int)N,
                       static_cast<const F*>(B), (int64_t)rows.R * N, x, (int)K, static_cast<const F*>(A), out);
  };
  auto of = [&](auto b) {
    const int lanes = (int)(rows.R * sizeof(F) / 16);
    if (lanes <= 2) go(up_row_kernel<F, 2, b.value>);
    else if (lanes <= 4) go(up_row_kernel<F, 4, b.value>);
    else if (lanes <= 8) go(up_row_kernel<F, 8, b.value>);
    else go(up_row_kernel<F, 16, b.value>);
  };
  if (both) of(std::true_type{});
  else of(std::false_type{});
}

struct Sums {
  int64_t chunk, items, slots;
  int64_t plan_bytes;
};

// Rows of a piece: all pieces together give every CU two workgroups, and a piece 256 rows or more.
Sums sums_plan(const k2q_bank* b, int64_t T, int64_t per) {
  const int ranks = 16 * tiles_of(b->R);
  const int64_t blocks = ((b->K + COLS - 1) / COLS + (b->N + COLS - 1) / COLS) * ((b->R + ranks - 1) / ranks);
  const int64_t want = (2 * (int64_t)k2q_cu_count() + blocks - 1) / blocks;
  int64_t chunk = ((T + want - 1) / want + 127) / 128 * 128;
  chunk = chunk < 256 ? 256 : chunk;
  const int64_t whole = T / chunk;
  return {chunk, whole + b->count, 2 * whole, 4 * up16(1 + 2 * (b->count + 1)) + 16 * (whole + b->count) + 4 * up16(T / per)};
}

}  // namespace

extern "C" int64_t k2q_bank_fwd_ws_bytes(const k2q_bank* b, int64_t T, int64_t per) {
  if (check(b, T, per) != K2Q_OK) return 0;
  return (int64_t)(few_rows(b, T, per) ? row_slices(T, b->K, b->R) : down_slices(T, b->K, b->R)) * T * b->R * 4;
}

extern "C" int k2q_bank_fwd(const k2q_bank* b, int64_t T, int64_t per, const uint16_t* x, const uint16_t* y, uint16_t* out,
                            float* u, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = check(b, T, per);
  if (rc != K2Q_OK) return rc;
  if (!x || !out || !ws || !k2q_aligned(x, 16) || !k2q_aligned(y, 16) || !k2q_aligned(out, 16) || !k2q_aligned(u, 16) ||
      !k2q_aligned(ws, 16) || ws_bytes < k2q_bank_fwd_ws_bytes(b, T, per))
    return K2Q_EINVAL;
  const Rows rows = rows_of(b, T, per);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(ws);
  if (few_rows(b, T, per)) {
    if (b->dtype == K2Q_DTYPE_F32) launch_rows<float>(rows, x, b->K, b->A, part, u, y, b->N, b->B, out, st);
    else launch_rows<uint16_t>(rows, x, b->K, b->A, part, u, y, b->N, b->B, out, st);
    return k2q_launch_status();
  }
  const int slices = down_slices(T, b->K, b->R);
  if (slices == 1 && u) part = u;
  if (b->dtype == K2Q_DTYPE_F32) {
    launch_down<float, true>(rows, x, b->K, b->A, slices, part, st);
    launch_up<float, false>(rows, part, slices, u, y, b->N, b->B, out, st);
  } else {
    launch_down<uint16_t, true>(rows, x, b->K, b->A, slices, part, st);
    launch_up<uint16_t, false>(rows, part, slices, u, y, b->N, b->B, out, st);
  }
  return k2q_launch_status();
}

extern "C" int64_t k2q_bank_bwd_ws_bytes(const k2q_bank* b, int64_t T, int64_t per, int need_factors) {
  if (check(b, T, per) != K2Q_OK) return 0;
  const int64_t down = (int64_t)down_slices(T, b->N, b->R) * T * b->R * 4;
  if (!need_factors) return down;
  const Sums s = sums_plan(b, T, per);
  return down + T * b->R * 4 + s.plan_bytes + s.slots * b->R * (b->K + b->N) * 4;
}

extern "C" int k2q_bank_bwd(const k2q_bank* b, int64_t T, int64_t per, const uint16_t* dy, const uint16_t* x, const float* u,
                            const uint16_t* base, uint16_t* dx, void* dA, void* dB, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = check(b, T, per);
  if (rc != K2Q_OK) return rc;
  if (!dy || (!dx && !dA && !dB) || (dA && !x) || (dB && !u) || !k2q_aligned(dy, 16) || !k2q_aligned(x, 16) ||
      !k2q_aligned(u, 16) || !k2q_aligned(base, 16) || !k2q_aligned(dx, 16) || !k2q_aligned(dA, 16) || !k2q_aligned(dB, 16) ||
      !ws || !k2q_aligned(ws, 16) || ws_bytes < k2q_bank_bwd_ws_bytes(b, T, per, dA || dB))
    return K2Q_EINVAL;
  const Rows rows = rows_of(b, T, per);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int slices = down_slices(T, b->N, b->R);
  const bool f32 = b->dtype == K2Q_DTYPE_F32;
  float* part = static_cast<float*>(ws);
  float* g = dA || dB ? part + slices * T * b->R : part;
  int left = slices;        // of g, for the "up"
  if (dx || dA) {
    if (f32) launch_down<float, false>(rows, dy, b->N, b->B, slices, slices == 1 ? g : part, st);
    else launch_down<uint16_t, false>(rows, dy, b->N, b->B, slices, slices == 1 ? g : part, st);
    if (dA || slices == 1) {
      launch_join(rows, part, slices, g, st);
      left = 1;
    }
  }
  // dx last: dy is still in the last-level cache for dB, and what dx would push out of it is read no more
  auto input = [&] {
    if (!dx) return k2q_launch_status();
    if (f32) launch_up<float, true>(rows, left > 1 ? part : g, left, nullptr, base, b->K, b->A, dx, st);
    else launch_up<uint16_t, true>(rows, left > 1 ? part : g, left, nullptr, base, b->K, b->A, dx, st);
    return k2q_launch_status();
  };
  if (!dA && !dB) return input();
  const Sums s = sums_plan(b, T, per);
  const int ids = (int)(T / per), n = b->count;
  Plan plan;
  plan.items = reinterpret_cast<Item*>(g + T * b->R);
  plan.head = reinterpret_cast<int32_t*>(plan.items + s.items);
  plan.start = plan.head + 1;
  plan.first = plan.start + n + 1;
  plan.order = plan.head + up16(1 + 2 * (n + 1));
  float* pieces = reinterpret_cast<float*>(plan.order + up16(ids));
  const int lds = (16 * n + 48) * 4 + 2 * (int)(ids < HELD ? up16(ids) : HELD);
  static std::atomic<uint64_t> once;
  int rl = k2q_lds_limit_once(plan_kernel, (16 * K2Q_MAX_ADAPTERS + 48) * 4 + 2 * HELD, once);
  if (rl != K2Q_OK) return rl;
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(PLAN), lds, st, rows, ids, (int)s.chunk, plan);
  Jobs jobs{};
  int k = 0;
  auto job = [&](const uint16_t* t, const float* p, int64_t C, int swapped, void* out) {
    jobs.j[k] = {t, p, (int)C, (int)((C + COLS - 1) / COLS), swapped, (int64_t)b->R * C, out, pieces};
    jobs.blocks += jobs.j[k++].blocks;
    pieces += s.slots * b->R * C;
  };
  if (dB) job(dy, u, b->N, 1, dB);
  if (dA) job(x, g, b->K, 0, dA);
  const int q = tiles_of(b->R);
  const dim3 grid((unsigned)jobs.blocks, (unsigned)s.items, (unsigned)((b->R + 16 * q - 1) / (16 * q)));
  const int sums_lds = 4 * (16 * q * (COLS / 2) + 4 * (16 * q > COLS / 2 ? 16 * q : COLS / 2)) * 4;
  static std::atomic<uint64_t> sums_once[6];
  int sl = K2Q_OK;
  auto go = [&](auto kernel, int i) {
    sl = k2q_lds_limit_once(kernel, sums_lds, sums_once[i]);
    if (sl == K2Q_OK) hipLaunchKernelGGL(kernel, grid, dim3(THREADS), sums_lds, st, rows, plan, jobs);
  };
  if (q == 1) f32 ? go(sums_kernel<float, 1>, 0) : go(sums_kernel<uint16_t, 1>, 1);
  else if (q == 2) f32 ? go(sums_kernel<float, 2>, 2) : go(sums_kernel<uint16_t, 2>, 3);
  else f32 ? go(sums_kernel<float, 4>, 4) : go(sums_kernel<uint16_t, 4>, 5);
  if (sl != K2Q_OK) return sl;
  if (!s.slots) return input();
  for (int i = 0; i < k; ++i) jobs.j[i].blocks = (int)((jobs.j[i].one / 4 + THREADS - 1) / THREADS);
  jobs.blocks = jobs.j[0].blocks + (k > 1 ? jobs.j[1].blocks : 0);
  const dim3 rest((unsigned)jobs.blocks, (unsigned)n);
  if (f32) hipLaunchKernelGGL(pieces_kernel<float>, rest, dim3(THREADS), 0, st, plan, jobs);
  else hipLaunchKernelGGL(pieces_kernel<uint16_t>, rest, dim3(THREADS), 0, st, plan, jobs);
  return input();
}
