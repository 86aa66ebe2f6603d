// Producer-fused rotate/quant: the elementwise or row-normalising operation that makes a quantized
// linear's input, fused into the same register pass that rotates and quantizes it.
//
//   * SwiGLU (reference mmdit.py:177-178, `self.down(F.silu(self.gate(x)) * self.up(x))`):
//       h = bf16(bf16(silu(g)) * u),  silu(g) = g / (1 + exp(-g)) in float32,
//     the rounding order of the reference's eager bf16 ops (F.silu returns bf16, the product rounds again).
//   * Modulated RMSNorm (reference mmdit.py:314-317 with RMSNorm.forward at mmdit.py:156-161):
//       n = bf16((x * rsqrt(mean(x^2) + eps)) * (w + 1))   [float32, the whole row]
//       h = bf16(bf16(bf16(1 + p) * n) + b)               [p, b: the bf16 modulation scale / shift of the
//                                                          row's batch entry]
//   * RMSNorm with the residual's addition (mmdit.py:317-318: `x = x + pregate * attn`, then the norm of x):
//       t = bf16(gate * y)  (t = y without a gate),  r = bf16(x + t),
//     and the norm above of r, modulated or not.  r is written too: it is the residual stream.  The roundings are those
//     of the eager bf16 ops: r equals theirs, h and the codes those of the norm above on r, bit for bit (the eager norm's
//     mean square is summed in another order: one value of h in about 1e5 is a bf16 step from its).
//     9 bytes an element: 2 x 4608 x 6144 in 110 us (4.6 TB/s; a copy of 4 GB runs at 4.9).
// All write h (bf16, the tensor the next linear receives: its LoRA down-projection and the saved input of
// the backward read it) and the int8 codes + scales of rotate/quant applied to h, computed from the same
// registers, so the codes equal those of a separate rotate/quant call on h bit for bit.
//
// The backward of the SwiGLU product (dg, du from dh) is the elementwise swiglu_bwd_kernel:
//   s = bf16(silu(g)), du = bf16(dh * s), ds = bf16(dh * u),
//   dg = bf16((ds * sig) * (1 + g * (1 - sig))) with sig = 1 / (1 + exp(-g)),
// the derivative d/dg [g sig(g)] = sig(g) (1 + g (1 - sig(g))) applied with the reference autograd's
// bf16 roundings (each eager op rounds its result to bf16).
#include "rotation.h"

namespace {

using namespace k2q_rot;

enum { PROD_SWIGLU = 0, PROD_RMSMOD = 1, PROD_RESNORM = 2 };

struct ProdArgs {
  const __bf16* x0;          // SwiGLU: gate output g;  RMSNorm: x
  const __bf16* x1;          // SwiGLU: up output u;  residual norm: y
  int64_t ld0, ld1;          // row strides of x0 / x1 (elements)
  const float* nw;           // RMSNorm scale parameter (K,), the norm weight is nw + nwadd
  float nwadd;
  const uint16_t* mscale;    // bf16 modulation scale, entry b = row / rpb at mscale + b * ldm (residual norm: nullable)
  const uint16_t* mshift;    // bf16 modulation shift, same indexing with ldb
  const uint16_t* gate;      // residual norm: bf16 gate, same indexing with ldg, or null
  int64_t ldm, ldb, ldg, rpb;
  float eps;
  int64_t M;
  int K;
  uint16_t* r;               // residual norm: M x K bf16, the new residual stream
  bool stream;               // residual norm: r and h are stored past the caches
  uint16_t* h;               // M x K bf16 (row stride K)
  int8_t* q;                 // M x K int8 codes of h R
  float* s;                  // M per-row scales
};

__device__ __forceinline__ float bf16r(float f) { return bf16_bits_to_f32(f32_to_bf16_bits(f)); }

// 16 bf16 values, past the caches where `stream`.
__device__ __forceinline__ void put16_bf16(uint16_t* p, const float (&v)[16], bool stream) {
  if (!stream) {
    store16_bf16(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v4u h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = pack_bf16x2(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
    __builtin_nontemporal_store(h, reinterpret_cast<v4u*>(p) + i);
  }
}

// Element i of eight bf16 values.
__device__ __forceinline__ float bf16_of(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  return i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : __uint_as_float(w[i >> 1] << 16);
}

// v where keep, else zeros: by component (a select between two uint4 objects puts them in scratch memory).
__device__ __forceinline__ uint4 keep_if(bool keep, uint4 v) {
  return make_uint4(keep ? v.x : 0u, keep ? v.y : 0u, keep ? v.z : 0u, keep ? v.w : 0u);
}

// Two values rounded to bf16 by one v_cvt_pk_bf16_f32 (round to nearest even), unpacked in place.
__device__ __forceinline__ void bf16r2(float& a, float& b) {
  const uint32_t u = pack_bf16x2(a, b);
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xffff0000u);
}

// sigmoid(g) = 1 / (1 + exp(-g)) with exp(-g) = 2^(-g log2 e) on v_exp_f32 and the reciprocal on v_rcp_f32:
// a few float32 ulp from the correctly rounded quotient, which the bf16 rounding of the result hides except
// in rare near-ties (the reference's own exp differs from the oracle's by as much).
__device__ __forceinline__ float sigmoid_f32(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f));
}

__device__ __forceinline__ float silu_f32(float g) { return g * sigmoid_f32(g); }

template <int PROD, int WPR, int kNCH, bool kTail>
__global__ __launch_bounds__(256) void prodquant_kernel(ProdArgs a) {
  constexpr int T = 64 * WPR;
  constexpr int CW = T * 16;
  constexpr int ROWS = 4 / WPR;
  __shared__ float sred[2][4];

  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR;
  const int t = (wave % WPR) * 64 + lane;
  const int l = t & 15;
  const int off = lane_offset(t);
  const bool row_ok = row < a.M;
  const int K = a.K;
  const int64_t rr = row_ok ? row : 0;

  // Loads are unconditional from clamped (always valid) addresses, which keeps the kernel free of branches
  // and lets each chunk's operands die before the next chunk's arrive; lanes past K hold zeros (their
  // Hadamard blocks enter the row absmax).
  float v[kNCH][16];
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = c * CW + off;
    const bool ok = !kTail || col < K;
    load16<__bf16>(a.x0 + rr * a.ld0 + (ok ? col : 0), true, v[c]);
    if (kTail) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[c][i] = ok ? v[c][i] : 0.f;
    }
  }

  if (PROD == PROD_SWIGLU) {
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const int col = c * CW + off;
      float u[16];
      load16<__bf16>(a.x1 + rr * a.ld1 + (!kTail || col < K ? col : 0), true, u);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {   // silu(0) * u = 0 past K
        float s0 = silu_f32(v[c][i]), s1 = silu_f32(v[c][i + 1]);
        bf16r2(s0, s1);
        float h0 = s0 * u[i], h1 = s1 * u[i + 1];
        bf16r2(h0, h1);
        v[c][i] = h0;
        v[c][i + 1] = h1;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    const int64_t b = rr / a.rpb;
    if (PROD == PROD_RESNORM) {
      const uint16_t* mg = a.gate ? a.gate + b * a.ldg : nullptr;
      uint4 yv[kNCH][2];      // loaded whole: a load behind a store of r would wait for its turn
#pragma unroll
      for (int c = 0; c < kNCH; ++c) {
        const int col = c * CW + off;
        const uint4* yp = reinterpret_cast<const uint4*>(a.x1 + rr * a.ld1 + (!kTail || col < K ? col : 0));
        yv[c][0] = yp[0];
        yv[c][1] = yp[1];
      }
#pragma unroll
      for (int c = 0; c < kNCH; ++c) {
        const int col = c * CW + off;
        const bool ok = !kTail || col < K;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = bf16_of(yv[c][i >> 3], i & 7);
        if (mg) {
          float g[16];
          load16<__bf16>(reinterpret_cast<const __bf16*>(mg) + (ok ? col : 0), true, g);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            y[i] *= g[i];
            y[i + 1] *= g[i + 1];
            bf16r2(y[i], y[i + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float r0 = v[c][i] + y[i], r1 = v[c][i + 1] + y[i + 1];
          bf16r2(r0, r1);
          v[c][i] = ok ? r0 : 0.f;
          v[c][i + 1] = ok ? r1 : 0.f;
        }
        if (row_ok && ok) put16_bf16(a.r + row * (int64_t)K + col, v[c], a.stream);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < kNCH; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += v[c][i] * v[c][i];   // squares rounded, then summed (x.pow(2).mean())
    ss = wave_sum(ss);
    if (WPR > 1) {
      if (lane == 0) sred[0][wave] = ss;
      __syncthreads();
      const int w0 = (wave / WPR) * WPR;
      ss = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) ss += sred[0][w0 + w];
    }
    const float rinv = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)K) + a.eps));
    const bool mod = PROD == PROD_RMSMOD || a.mscale;
    const uint16_t* ms = mod ? a.mscale + b * a.ldm : nullptr;
    const uint16_t* mb = mod ? a.mshift + b * a.ldb : nullptr;
    // Per chunk: the norm weight (f32) and the two modulation vectors (bf16, kept packed) are loaded and
    // consumed before the next chunk's, so at most one chunk of them is live (occupancy).
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const int col = c * CW + off;
      const bool ok = !kTail || col < K;
      const int cc = ok ? col : 0;
      // unconditional loads from a clamped (always valid) address; lanes past K are zeroed below
      float w[16];
      load16<float>(a.nw + cc, true, w);
      if (!mod) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float n0 = (v[c][i] * rinv) * (w[i] + a.nwadd), n1 = (v[c][i + 1] * rinv) * (w[i + 1] + a.nwadd);
          bf16r2(n0, n1);
          v[c][i] = !kTail || ok ? n0 : 0.f;
          v[c][i + 1] = !kTail || ok ? n1 : 0.f;
        }
        continue;
      }
      const uint4 pv0 = reinterpret_cast<const uint4*>(ms + cc)[0], pv1 = reinterpret_cast<const uint4*>(ms + cc)[1];
      const uint4 bv0 = reinterpret_cast<const uint4*>(mb + cc)[0], bv1 = reinterpret_cast<const uint4*>(mb + cc)[1];
      const uint32_t pw[8] = {pv0.x, pv0.y, pv0.z, pv0.w, pv1.x, pv1.y, pv1.z, pv1.w};
      const uint32_t bw[8] = {bv0.x, bv0.y, bv0.z, bv0.w, bv1.x, bv1.y, bv1.z, bv1.w};
#pragma unroll
      for (int i = 0; i < 16; i += 2) {   // element pairs share each bf16 conversion
        float n0 = (v[c][i] * rinv) * (w[i] + a.nwadd), n1 = (v[c][i + 1] * rinv) * (w[i + 1] + a.nwadd);
        bf16r2(n0, n1);
        float p0 = 1.f + __uint_as_float(pw[i >> 1] << 16), p1 = 1.f + __uint_as_float(pw[i >> 1] & 0xffff0000u);
        bf16r2(p0, p1);
        float m0 = p0 * n0, m1 = p1 * n1;
        bf16r2(m0, m1);
        float h0 = m0 + __uint_as_float(bw[i >> 1] << 16), h1 = m1 + __uint_as_float(bw[i >> 1] & 0xffff0000u);
        bf16r2(h0, h1);
        v[c][i] = !kTail || ok ? h0 : 0.f;   // blocks past K must stay zero: they enter the row absmax
        v[c][i + 1] = !kTail || ok ? h1 : 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if (row_ok) {
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const int col = c * CW + off;
      if (col < K) {
        if (PROD == PROD_RESNORM) put16_bf16(a.h + row * (int64_t)K + col, v[c], a.stream);
        else store16_bf16(a.h + row * (int64_t)K + col, v[c]);
      }
    }
  }

  const float c1 = (l & 1) ? -1.f : 1.f;
  const float c2 = (l & 2) ? -1.f : 1.f;
  const float c8 = (l & 8) ? -1.f : 1.f;
  const float sigma = c1 * c2 * c8;
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    rotate16(v[c], c1, c2, c8);
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[c][i]));
  }
  amax = wave_max(amax);
  if (WPR > 1) {
    if (lane == 0) sred[1][wave] = amax;
    __syncthreads();
    const int w0 = (wave / WPR) * WPR;
#pragma unroll
    for (int w = 0; w < WPR; ++w) amax = fmaxf(amax, sred[1][w0 + w]);
  }
  amax = fmaxf(amax, 1e-8f);
  const float inv = __fdiv_rn(127.f, amax);
  if (!row_ok) return;
  if (t == 0) a.s[row] = __fdiv_rn(amax, 127.f);
  const float mul = inv * sigma;
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = c * CW + off;
    if (col < K) store_codes16(a.q + row * (int64_t)K + col, v[c], mul);
  }
}

template <int PROD, int WPR, bool kTail>
void launch_prod_nch(const ProdArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.M + (4 / WPR) - 1) / (4 / WPR)));
  const int nch = (a.K + 1024 * WPR - 1) / (1024 * WPR);
  switch (nch) {
    case 1: hipLaunchKernelGGL((prodquant_kernel<PROD, WPR, 1, kTail>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((prodquant_kernel<PROD, WPR, 2, kTail>), grid, dim3(256), 0, st, a); break;
    case 3: hipLaunchKernelGGL((prodquant_kernel<PROD, WPR, 3, kTail>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((prodquant_kernel<PROD, WPR, 4, kTail>), grid, dim3(256), 0, st, a); break;
  }
}

// kTail: K is not a whole number of chunks, so some lanes' columns lie past K.
template <int PROD, int WPR>
void launch_prod_wpr(const ProdArgs& a, hipStream_t st) {
  if (a.K % (1024 * WPR)) launch_prod_nch<PROD, WPR, true>(a, st);
  else launch_prod_nch<PROD, WPR, false>(a, st);
}

template <int PROD>
int launch_prod(const ProdArgs& a, hipStream_t st) {
  if (a.K <= 4096) launch_prod_wpr<PROD, 1>(a, st);
  else if (a.K <= 8192) launch_prod_wpr<PROD, 2>(a, st);
  else launch_prod_wpr<PROD, 4>(a, st);
  return k2q_launch_status();
}

int check_prod_common(int64_t M, int64_t K, const uint16_t* h, const int8_t* q, const float* s) {
  if (M < 1 || K < K2Q_HADAMARD || K % K2Q_HADAMARD) return K2Q_EINVAL;
  if (K > 16384) return K2Q_EUNSUPPORTED;
  if (!h || !q || !s || !k2q_aligned(h, 16) || !k2q_aligned(q, 16) || !k2q_aligned(s, 4)) return K2Q_EINVAL;
  return K2Q_OK;
}

// 8 elements per lane per step: dh, g, u in; dg, du out (all bf16, contiguous, n elements, n % 8 == 0).
__global__ __launch_bounds__(256) void swiglu_bwd_kernel(const uint4* __restrict__ dh, const uint4* __restrict__ g,
                                                         const uint4* __restrict__ u, int64_t n8,
                                                         uint4* __restrict__ dg, uint4* __restrict__ du) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t)gridDim.x * blockDim.x) {
    const uint4 a = dh[i], b = g[i], c = u[i];
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w}, cw[4] = {c.x, c.y, c.z, c.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float rg[2], ru[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float d = bf16_bits_to_f32((aw[j] >> (16 * e)) & 0xffffu);
        const float x = bf16_bits_to_f32((bw[j] >> (16 * e)) & 0xffffu);
        const float up = bf16_bits_to_f32((cw[j] >> (16 * e)) & 0xffffu);
        const float sig = sigmoid_f32(x);
        const float sl = bf16r(x * sig);   // the forward's silu_f32, bit for bit
        ru[e] = d * sl;
        const float ds = bf16r(d * up);
        rg[e] = (ds * sig) * (1.f + x * (1.f - sig));
      }
      og[j] = pack_bf16x2(rg[0], rg[1]);
      ou[j] = pack_bf16x2(ru[0], ru[1]);
    }
    dg[i] = make_uint4(og[0], og[1], og[2], og[3]);
    du[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

struct NormBwdArgs {
  const uint16_t* dh;        // M x K bf16: gradient of h
  const uint16_t* x;         // M x K: the norm's input (the residual norm's r)
  int64_t M;
  int K;
  const float* nw;           // norm weight = nw + nwadd
  float nwadd, eps;
  const uint16_t* mscale;    // B x K bf16 modulation scale (residual norm: nullable)
  int64_t ldm, rpb;
  uint16_t* dx;
  // the residual norm's
  const uint16_t* dr;        // gradient of r from its other readers, or null
  const uint16_t* gate;      // B x K bf16 or null
  int64_t ldg;
  uint16_t* dy;              // gradient of y, written where there is a gate (without one it is dx)
  float* stats;              // M pairs (rsqrt, the subtracted term's factor c) for the column sums, or null
};

// Input gradient of the modulated RMSNorm (the autograd of the forward's eager ops for x alone):
//   dn = bf16(dh * bf16(1 + p)),  g = dn * (w + 1),  r = rsqrt(mean x^2 + eps),
//   dx = bf16(g r - x (r^3 / K) sum_k(g x)).
// With a residual (kRes) x is the new stream, whose other readers' gradient joins it, and the gate scales it on the way to
// y, all in f32 with one rounding of each result; eager: dn and dx above rounded as they are there, the sum before the gate:
//   dR = dr + dx,  dx = bf16(dR),  dy = bf16(gate * dR).
// A team of 64 * WPR lanes owns a row; lane t handles the 8-element chunks at 8 t + 8 T c, c < kNCH, held
// packed (bf16 pairs) between the two row reductions.  Bound by its reads and writes.  The form that rounds once keeps
// dr in registers from the start and spreads a row over more lanes (fewer registers each, more rows in flight): 4608 x
// 6144 with a gate in 51.8 us alone (5.5 TB/s) and 57 in a training pass (4.9), with the eager roundings 60.4; the other
// two keep the order of the row sums that their results have.
enum { BWD_NORM = 0, BWD_EAGER = 1, BWD_ONCE = 2 };    // without a residual; with it, rounded as the eager ops; once

template <int MODE, int WPR, int kNCH>
__global__ __launch_bounds__(256) void rmsmod_bwd_kernel(NormBwdArgs a) {
  constexpr bool kRes = MODE != BWD_NORM, steps = MODE != BWD_ONCE;
  constexpr int T = 64 * WPR;
  constexpr int ROWS = 4 / WPR;
  __shared__ float sred[2][4];
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR;
  const int t = (wave % WPR) * 64 + lane;
  const bool row_ok = row < a.M;
  const int64_t rr = row_ok ? row : 0;
  const int K = a.K;
  const bool mod = !kRes || a.mscale;
  const uint16_t* ms = mod ? a.mscale + (rr / a.rpb) * a.ldm : nullptr;

  uint4 xv[kNCH], dv[kNCH], rv[kNCH];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = 8 * t + 8 * T * c;
    const bool ok = col < K;
    const int cc = ok ? col : 0;
    xv[c] = *reinterpret_cast<const uint4*>(a.x + rr * K + cc);
    dv[c] = *reinterpret_cast<const uint4*>(a.dh + rr * K + cc);
    if (MODE == BWD_ONCE) rv[c] = *reinterpret_cast<const uint4*>((a.dr ? a.dr : a.x) + rr * K + cc);
    if (!ok) xv[c] = dv[c] = make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {xv[c].x, xv[c].y, xv[c].z, xv[c].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e0 = __uint_as_float(w[j] << 16), e1 = __uint_as_float(w[j] & 0xffff0000u);
      ss += e0 * e0;
      ss += e1 * e1;
    }
  }
  ss = wave_sum(ss);
  if (WPR > 1) {
    if (lane == 0) sred[0][wave] = ss;
    __syncthreads();
    const int w0 = (wave / WPR) * WPR;
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) ss += sred[0][w0 + w];
  }
  const float r = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)K) + a.eps));
  // g = bf16(dh * p1) * (w + 1), kept in f32 (8 per chunk) for the final pass
  float gv[kNCH][8];
  float dot = 0.f;
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = 8 * t + 8 * T * c;
    const int cc = col < K ? col : 0;
    float w[8];
    const float4 w0 = *reinterpret_cast<const float4*>(a.nw + cc), w1 = *reinterpret_cast<const float4*>(a.nw + cc + 4);
    w[0] = w0.x; w[1] = w0.y; w[2] = w0.z; w[3] = w0.w; w[4] = w1.x; w[5] = w1.y; w[6] = w1.z; w[7] = w1.w;
    const uint4 pv = mod ? *reinterpret_cast<const uint4*>(ms + cc) : make_uint4(0, 0, 0, 0);
    const uint32_t pw[4] = {pv.x, pv.y, pv.z, pv.w};
    const uint32_t dw[4] = {dv[c].x, dv[c].y, dv[c].z, dv[c].w};
    const uint32_t xw[4] = {xv[c].x, xv[c].y, xv[c].z, xv[c].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // without a modulation p = 0: dh times one, exact
      float p0 = 1.f + __uint_as_float(pw[j] << 16), p1 = 1.f + __uint_as_float(pw[j] & 0xffff0000u);
      bf16r2(p0, p1);
      float n0 = __uint_as_float(dw[j] << 16) * p0, n1 = __uint_as_float(dw[j] & 0xffff0000u) * p1;
      if (steps) bf16r2(n0, n1);
      const float g0 = n0 * (w[2 * j] + a.nwadd), g1 = n1 * (w[2 * j + 1] + a.nwadd);
      gv[c][2 * j] = g0;
      gv[c][2 * j + 1] = g1;
      dot += g0 * __uint_as_float(xw[j] << 16);
      dot += g1 * __uint_as_float(xw[j] & 0xffff0000u);
    }
  }
  dot = wave_sum(dot);
  if (WPR > 1) {
    if (lane == 0) sred[1][wave] = dot;
    __syncthreads();
    const int w0 = (wave / WPR) * WPR;
    dot = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) dot += sred[1][w0 + w];
  }
  if (!row_ok) return;
  const float c3 = __fdiv_rn(r * r * r * dot, (float)K);
  if (kRes && a.stats && t == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(r, c3);
  const uint16_t* mg = kRes && a.gate ? a.gate + (row / a.rpb) * a.ldg : nullptr;
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = 8 * t + 8 * T * c;
    if (col >= K) continue;
    const uint32_t xw[4] = {xv[c].x, xv[c].y, xv[c].z, xv[c].w};
    float d[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      d[2 * j] = gv[c][2 * j] * r - __uint_as_float(xw[j] << 16) * c3;
      d[2 * j + 1] = gv[c][2 * j + 1] * r - __uint_as_float(xw[j] & 0xffff0000u) * c3;
    }
    if (kRes && a.dr) {
      const uint4 rc = MODE == BWD_ONCE ? rv[c] : *reinterpret_cast<const uint4*>(a.dr + row * K + col);
      const uint32_t rw[4] = {rc.x, rc.y, rc.z, rc.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (steps) bf16r2(d[2 * j], d[2 * j + 1]);
        d[2 * j] = __uint_as_float(rw[j] << 16) + d[2 * j];
        d[2 * j + 1] = __uint_as_float(rw[j] & 0xffff0000u) + d[2 * j + 1];
      }
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(d[2 * j], d[2 * j + 1]);
    *reinterpret_cast<uint4*>(a.dx + row * K + col) = make_uint4(o[0], o[1], o[2], o[3]);
    if (mg) {
      const uint4 gg = *reinterpret_cast<const uint4*>(mg + col);
      const uint32_t gw[4] = {gg.x, gg.y, gg.z, gg.w};
      uint32_t e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (steps) bf16r2(d[2 * j], d[2 * j + 1]);
        e[j] = pack_bf16x2(__uint_as_float(gw[j] << 16) * d[2 * j], __uint_as_float(gw[j] & 0xffff0000u) * d[2 * j + 1]);
      }
      *reinterpret_cast<uint4*>(a.dy + row * K + col) = make_uint4(e[0], e[1], e[2], e[3]);
    }
  }
}

template <int MODE, int WPR>
void launch_rmsmod_bwd(const NormBwdArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.M + (4 / WPR) - 1) / (4 / WPR)));
  const int nch = (a.K + 512 * WPR - 1) / (512 * WPR);
#define K2Q_RMB(N)                                                                             \
  case N:                                                                                      \
    hipLaunchKernelGGL((rmsmod_bwd_kernel<MODE, WPR, N>), grid, dim3(256), 0, st, a);          \
    break;
  switch (nch) {
    K2Q_RMB(1) K2Q_RMB(2) K2Q_RMB(3) K2Q_RMB(4) K2Q_RMB(5) K2Q_RMB(6) K2Q_RMB(7)
    default: hipLaunchKernelGGL((rmsmod_bwd_kernel<MODE, WPR, 8>), grid, dim3(256), 0, st, a); break;
  }
#undef K2Q_RMB
}

// Columns up to which a wave has a row of its own; twice as many take two waves, more four.
constexpr int bwd_narrow(int mode) { return mode == BWD_ONCE ? 1024 : 4096; }

template <int MODE>
void launch_norm_bwd(const NormBwdArgs& a, hipStream_t st) {
  constexpr int NARROW = bwd_narrow(MODE);
  if (a.K <= NARROW) launch_rmsmod_bwd<MODE, 1>(a, st);
  else if (a.K <= 2 * NARROW) launch_rmsmod_bwd<MODE, 2>(a, st);
  else launch_rmsmod_bwd<MODE, 4>(a, st);
}

// Whether a launch of the row pass holds M rows: HIP counts its threads in 32 bits.
bool norm_bwd_fits(int64_t M, int64_t K, int mode) {
  const int waves = K <= bwd_narrow(mode) ? 1 : K <= 2 * bwd_narrow(mode) ? 2 : 4;
  return (M * waves + 3) / 4 * 256 <= 0xffffffffll;
}

// Column sums of the residual norm's backward: the gradients of what is broadcast over the rows of a batch entry,
//   dscale = sum_m dh n,  dshift = sum_m dh,  dgate = sum_m dR y,  and over every row  dw = sum_m dn x r,
// with n as in the forward and dn, dR unrounded in f32 (from the row statistics that the pass above left).  Rows are cut
// into strips of one batch entry each; a workgroup sums one strip of 512 columns (lane: 8 columns, its four waves: every
// fourth row).  Where an entry is one strip its sums are the gradients and are written here; else they and the sums over
// every row leave as f32 partials, which a second launch adds in order: no atomics, the same result every time.  Only the
// sums asked for have partials, one after another in the order below.
// Entries of a few rows (kFew) are a wave's own, several of them one after another: a strip is then the rows of four waves
// and spans entries, so the partials of the sums over every row stay few (one strip an entry would leave 4 bytes a sum for
// every 2 of a row), and no wave is without a row.
// Where nothing read h (kStream) dR = dr: the same pass makes dy = bf16(gate dr) and the gate's gradient, and is all there
// is.
// Bound by reading dh, r, y and dr once more: 2304 x 16384 in 58.5 us (5.2 TB/s), kFew with a gate and a modulation a row
// 9216 x 6144 in 201 (4.5 TB/s with the modulation and the gradients of the vectors), kStream 9216 x 6144 in 81 (4.2); the join 4 to 5.
constexpr int CS_COLS = 512;

struct ColSumArgs {
  const uint16_t *dh, *dr, *x, *y;   // M x K bf16 (dr: null for none; y: row stride ldy, null: no gate's gradient)
  const float* stats;                // M pairs
  int64_t M, ldy, rpb;
  int K, strips, strip_rows;         // strips per batch entry, rows per strip; kFew: rows per wave
  const float* nw;
  float nwadd;
  const uint16_t* mscale;            // or null
  int64_t ldm;
  const uint16_t* gate;              // kStream
  int64_t ldg;
  uint16_t* dy;
  int parts, direct;                 // bits of the sums that leave as partials, and of those that are written whole
  float* part;                       // strip x (the sums of `parts`) x K
  uint16_t *dscale, *dshift, *dgate; // entries x K
};

enum { CS_W = 0, CS_SCALE = 1, CS_SHIFT = 2, CS_GATE = 3 };

// Where sum k lies among those of `bits`.
__device__ __forceinline__ int cs_slot(int bits, int k) { return __popc(bits & ((1 << k) - 1)); }

__device__ __forceinline__ void put8_bf16(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                            pack_bf16x2(v[6], v[7]));
}

__device__ __forceinline__ void put_direct(const ColSumArgs& a, int64_t entry, int col, const float (&acc)[4][8]) {
  const int64_t o = entry * a.K + col;
  if (a.direct & 1 << CS_SCALE) put8_bf16(a.dscale + o, acc[CS_SCALE]);
  if (a.direct & 1 << CS_SHIFT) put8_bf16(a.dshift + o, acc[CS_SHIFT]);
  if (a.direct & 1 << CS_GATE) put8_bf16(a.dgate + o, acc[CS_GATE]);
}

template <bool kStream, bool kFew>
__global__ __launch_bounds__(256) void resnorm_colsum_kernel(ColSumArgs a) {
  __shared__ float red[3][64][33];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int K = a.K;
  const uint32_t tiles = (uint32_t)(K + CS_COLS - 1) / CS_COLS, piece = blockIdx.x / tiles;
  const int col = (int)(blockIdx.x % tiles) * CS_COLS + 8 * lane;
  const bool ok = col < K;
  const int cc = ok ? col : 0;
  int64_t entry, m0, m1;
  if (kFew) {
    m0 = ((int64_t)piece * 4 + wave) * a.strip_rows;      // a whole number of entries
    m1 = m0 + a.strip_rows < a.M ? m0 + a.strip_rows : a.M;
    entry = m0 / a.rpb;
  } else {
    entry = piece / a.strips;
    m0 = entry * a.rpb + (int64_t)(piece % a.strips) * a.strip_rows;
    const int64_t mend = (entry + 1) * a.rpb;
    m1 = m0 + a.strip_rows < mend ? m0 + a.strip_rows : mend;
    m0 += wave;
  }
  float w[8], p1[8], acc[4][8] = {}, tot[4][8] = {};
  const uint16_t* vec = kStream ? a.gate : a.mscale;      // the entries' vector
  const int64_t ldv = kStream ? a.ldg : a.ldm;
  if (!kStream)
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = a.nw[cc + i] + a.nwadd;
  auto set_entry = [&](const uint4& v) {      // p1: bf16(1 + the modulation), or the gate
#pragma unroll
    for (int i = 0; i < 8; ++i) p1[i] = kStream ? bf16_of(v, i) : vec ? bf16r(1.f + bf16_of(v, i)) : 1.f;
  };
  // what is absent is read as x (dr): no branch between a row's loads (with: 5 % of both passes, 1536 x 6144)
  const uint16_t* x = kStream ? a.dr : a.x;
  const uint16_t *yp = a.y ? a.y : x, *rp = !kStream && a.y && a.dr ? a.dr : x;
  const int64_t ly = a.y ? a.ldy : K;
  struct Row {
    uint4 d, x, y, r, v;
    float2 st;
  };
  auto load = [&](int64_t m, int64_t e) {
    Row t;
    t.x = *reinterpret_cast<const uint4*>(x + m * K + cc);
    t.y = *reinterpret_cast<const uint4*>(yp + m * ly + cc);
    if (!kStream) {
      t.st = *reinterpret_cast<const float2*>(a.stats + 2 * m);
      t.d = *reinterpret_cast<const uint4*>(a.dh + m * K + cc);
      t.r = *reinterpret_cast<const uint4*>(rp + m * K + cc);
    }
    if (kFew && vec) t.v = *reinterpret_cast<const uint4*>(vec + e * ldv + cc);
    return t;
  };
  auto add = [&](int64_t m, Row t) {
    t.y = keep_if(a.y, t.y);
    if (kStream) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dR = bf16_of(t.x, i);
        e[i] = p1[i] * dR;
        acc[CS_GATE][i] = __builtin_fmaf(dR, bf16_of(t.y, i), acc[CS_GATE][i]);
      }
      if (a.dy && ok) put8_bf16(a.dy + m * K + col, e);
      return;
    }
    t.r = keep_if(a.y && a.dr, t.r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = bf16_of(t.d, i), xv = bf16_of(t.x, i);
      const float dn = d * p1[i], xr = xv * t.st.x;
      acc[CS_W][i] = __builtin_fmaf(dn, xr, acc[CS_W][i]);
      acc[CS_SCALE][i] = __builtin_fmaf(d, bf16r(xr * w[i]), acc[CS_SCALE][i]);
      acc[CS_SHIFT][i] += d;
      const float dR = bf16_of(t.r, i) + (dn * w[i] * t.st.x - xv * t.st.y);
      acc[CS_GATE][i] = __builtin_fmaf(dR, bf16_of(t.y, i), acc[CS_GATE][i]);
    }
  };
  if (kFew) {
    if (m0 < m1) {
      Row next = load(m0, entry);
      int64_t left = a.rpb;
      for (int64_t m = m0; m < m1; ++m) {
        const Row t = next;
        const bool last = --left == 0;
        if (m + 1 < m1) next = load(m + 1, last ? entry + 1 : entry);
        set_entry(t.v);
        add(m, t);
        if (!last) continue;
        if (ok) put_direct(a, entry, col, acc);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            tot[k][i] += acc[k][i];
            acc[k][i] = 0.f;
          }
        left = a.rpb;
        ++entry;
      }
    }
    if (!a.parts) return;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k][i] = tot[k][i];
  } else {
    set_entry(vec ? *reinterpret_cast<const uint4*>(vec + entry * ldv + cc) : make_uint4(0, 0, 0, 0));
    for (int64_t m = m0; m < m1; m += 4) add(m, load(m, entry));
    if (!(a.parts | a.direct)) return;
  }
  if (wave)
#pragma unroll
    for (int i = 0; i < 32; ++i) red[wave - 1][lane][i] = acc[i >> 3][i & 7];
  __syncthreads();
  if (wave || !ok) return;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc[k][i] = ((acc[k][i] + red[0][lane][8 * k + i]) + red[1][lane][8 * k + i]) + red[2][lane][8 * k + i];
  if (!kFew) put_direct(a, entry, col, acc);
  float* out = a.part + (int64_t)piece * __popc(a.parts) * K + col;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (a.parts & 1 << k) {
      float4* o = reinterpret_cast<float4*>(out + (int64_t)cs_slot(a.parts, k) * K);
      o[0] = make_float4(acc[k][0], acc[k][1], acc[k][2], acc[k][3]);
      o[1] = make_float4(acc[k][4], acc[k][5], acc[k][6], acc[k][7]);
    }
}

// Many partials of the sums over every row: 64 of them folded into one, 64 columns of one sum a workgroup, its four waves
// every fourth partial, then the waves in order.  With the join behind it a value passes 16 + 4 and then a sixteenth of
// the folded ones' additions, however many entries there are.
constexpr int CS_FOLD = 64;

__global__ __launch_bounds__(256) void resnorm_colsum_fold_kernel(const float* part, int K, int64_t pieces, int sums,
                                                                  float* out) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t tiles = (uint32_t)(K + 63) / 64, per = tiles * sums;
  const uint32_t group = blockIdx.x / per;
  const int sum = (int)(blockIdx.x % per / tiles), col = (int)(blockIdx.x % tiles) * 64 + lane;
  const int64_t i0 = (int64_t)group * CS_FOLD, i1 = i0 + CS_FOLD < pieces ? i0 + CS_FOLD : pieces;
  float f = 0.f;
  if (col < K) {
#pragma unroll 8
    for (int64_t i = i0 + wave; i < i1; i += 4) f += part[(i * sums + sum) * K + col];
  }
  red[wave][lane] = f;
  __syncthreads();
  if (wave || col >= K) return;
  out[((int64_t)group * sums + sum) * K + col] = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
}

// The strips' partials joined: 64 columns a workgroup, its NW waves every NW-th strip, then the waves in order.  Column
// tiles of the batch entries (the bits of `per_entry`: scale, shift and gate gradients, bf16), then those of the sums over
// every entry (`whole`: the norm weight's, f32, and those of a vector that every entry shares), which are sums over
// `pieces` partials.  `parts`: the sums that have partials.
struct JoinArgs {
  const float* part;
  int K, strips, parts, per_entry, whole;
  int64_t entries, pieces;            // entries: 0 where only `whole` is joined
  float* dnw;
  uint16_t *dscale, *dshift, *dgate;
};

// NS sums (at `off` of a strip's partials) of the strips from i in steps of NW: the loads of eight strips are issued
// together (four of several sums by four waves, which have no more of an entry), those past the end repeat the first and
// add nothing; a last one goes alone (64 x 32 x 6144, a strip a wave: 44.6 us, with the repeats 47.6).
template <int NS, int NW>
__device__ __forceinline__ void join_strips(const float* p, int64_t i, int64_t end, int64_t stride, const int (&off)[4],
                                            float (&f)[4]) {
  constexpr int U = NW < 16 && NS > 1 ? 4 : 8, step = NW;
  for (; i + step < end; i += U * step) {
    float v[U][NS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* q = p + (i + u * step < end ? i + u * step : i) * stride;
#pragma unroll
      for (int s = 0; s < NS; ++s) v[u][s] = q[off[s]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < NS; ++s) f[s] += i + u * step < end ? v[u][s] : 0.f;
  }
  if (i < end)
#pragma unroll
    for (int s = 0; s < NS; ++s) f[s] += p[i * stride + off[s]];
}

template <int NW>
__global__ __launch_bounds__(64 * NW) void resnorm_colsum_join_kernel(JoinArgs a) {
  __shared__ float red[4][NW][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = a.K;
  const uint32_t tiles = (uint32_t)(K + 63) / 64;
  const int col = (int)(blockIdx.x % tiles) * 64 + lane;
  const int64_t entry = blockIdx.x / tiles;
  const bool all = entry == a.entries;
  const int want = all ? a.whole : a.per_entry;
  if (!want) return;
  const int64_t i0 = (all ? 0 : entry * a.strips) + wave, i1 = all ? a.pieces : (entry + 1) * a.strips;
  const int64_t stride = (int64_t)__popc(a.parts) * K;
  const float* p = a.part + (col < K ? col : 0);
  int off[4] = {};
  float f[4] = {};
#pragma unroll
  for (int s = 0, rest = want; s < 4; ++s, rest &= rest - 1)
    if (rest) off[s] = cs_slot(a.parts, __ffs(rest) - 1) * K;
  switch (__popc(want)) {
    case 1: join_strips<1, NW>(p, i0, i1, stride, off, f); break;
    case 2: join_strips<2, NW>(p, i0, i1, stride, off, f); break;
    case 3: join_strips<3, NW>(p, i0, i1, stride, off, f); break;
    default: join_strips<4, NW>(p, i0, i1, stride, off, f);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) red[s][wave][lane] = f[s];
  __syncthreads();
  if (wave || col >= K) return;
  const int64_t o = all ? col : entry * K + col;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!(want & 1 << k)) continue;
    const int s = cs_slot(want, k);
    float t = red[s][0][lane];
#pragma unroll
    for (int v = 1; v < NW; ++v) t += red[s][v][lane];
    if (k == CS_W) a.dnw[o] = t;
    else (k == CS_SCALE ? a.dscale : k == CS_SHIFT ? a.dshift : a.dgate)[o] = (uint16_t)f32_to_bf16_bits(t);
  }
}

// The gradients that are sums over rows: which are asked for, where they go, and the partials' memory.
struct ColOut {
  int asked, whole;                  // bits asked for; of those, the sums over every entry
  float* dnw;
  uint16_t *dscale, *dshift, *dgate;
  float* part;
};

int64_t fold_groups(int64_t pieces) { return (pieces + CS_FOLD - 1) / CS_FOLD; }
constexpr int64_t CS_MANY = 1024;    // partials that one join adds

// 16 waves where an entry has as many strips (the whole backward, us, four waves / 16: 9216 x 6144 156 / 150, 4608 x 2048
// 41.3 / 38.8), or where the strips' entries are written already (`direct`) and only the sums over every entry are left.
// Which of the gradients are asked for changes no order.
void launch_join(const ColOut& c, int parts, bool direct, int64_t K, int64_t entries, int strips, int64_t pieces,
                 hipStream_t st) {
  const int per_entry = direct ? 0 : c.asked & ~c.whole;
  JoinArgs a{c.part, (int)K, strips, parts, per_entry, c.asked & c.whole, per_entry ? entries : 0, pieces, c.dnw, c.dscale,
             c.dshift, c.dgate};
  const int64_t tiles = (K + 63) / 64;
  if (direct && pieces > CS_MANY) {
    const int sums = __builtin_popcount(parts);
    const int64_t groups = fold_groups(pieces);
    float* folded = c.part + pieces * sums * K;
    hipLaunchKernelGGL(resnorm_colsum_fold_kernel, dim3((unsigned)(tiles * sums * groups)), dim3(256), 0, st, c.part, (int)K,
                       pieces, sums, folded);
    a.part = folded;
    a.pieces = groups;
  }
  const dim3 grid((unsigned)(tiles * (a.entries + 1)));
  if (strips >= 16 || direct) hipLaunchKernelGGL(resnorm_colsum_join_kernel<16>, grid, dim3(1024), 0, st, a);
  else hipLaunchKernelGGL(resnorm_colsum_join_kernel<4>, grid, dim3(256), 0, st, a);
}

struct ColPlan {
  bool few;
  int strips, rows;                  // per entry; rows per strip, or per wave where `few`
  int64_t pieces;
};

// Strips per batch entry: about two workgroups a CU over the column tiles, at least 8 rows each (all three passes, us, at
// 8 / 16 / 32 rows: 333 x 2560 14.9 / 15.1 / 17.0, 4 x 64 x 1024 10.6 / 12.0 / 14.6, 2 x 1000 x 512 14.5 / 15.3 / 17.5).
// Entries of fewer than 16 rows, where every wave of a workgroup has one: as many workgroups, a wave's entries at least four
// rows (one strip an entry / this, all three passes, us: 4099 x 1 x 640 129 / 24, 1000 x 13 x 2048 142 / 96, 9216 x 1 x 6144
// 1568 / 343).
ColPlan colsum_plan(int64_t rpb, int64_t K, int64_t entries, int cus) {
  const int64_t tiles = (K + CS_COLS - 1) / CS_COLS;
  if (rpb < 16 && entries >= 4) {
    const int64_t wgs = (2 * cus + tiles - 1) / tiles, least = (3 + rpb) / rpb;
    int64_t own = (entries + 4 * wgs - 1) / (4 * wgs);      // entries per wave
    own = own < least ? least : own;
    return {true, 1, (int)(own * rpb), (entries + 4 * own - 1) / (4 * own)};
  }
  int64_t s = (2 * cus + tiles * entries - 1) / (tiles * entries);
  const int64_t most = (rpb + 7) / 8;
  s = s < 1 ? 1 : s > most ? most : s;
  int64_t rows = (rpb + s - 1) / s;
  s = (rpb + rows - 1) / rows;
  rows = (rpb + s - 1) / s;
  return {false, (int)s, (int)rows, entries * s};
}

// Floats of partials, at most: every sum, folded ones behind them.
int64_t colsum_floats(const ColPlan& p, int64_t K) {
  return (p.pieces + (p.pieces > CS_MANY ? fold_groups(p.pieces) : 0)) * 4 * K;
}

// The column pass and its join.  `a` holds the operands.
template <bool kStream>
void launch_colsum(ColSumArgs a, const ColOut& c, const ColPlan& p, int64_t entries, hipStream_t st) {
  const int per_entry = c.asked & ~c.whole, direct = p.strips == 1 ? per_entry : 0;
  a.strips = p.strips;
  a.strip_rows = p.rows;
  a.direct = direct;
  a.parts = c.asked & ~direct;
  a.part = c.part;
  a.dscale = c.dscale;
  a.dshift = c.dshift;
  a.dgate = c.dgate;
  const dim3 grid((unsigned)((a.K + CS_COLS - 1) / CS_COLS * p.pieces));
  if (p.few) hipLaunchKernelGGL((resnorm_colsum_kernel<kStream, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((resnorm_colsum_kernel<kStream, false>), grid, dim3(256), 0, st, a);
  if (a.parts) launch_join(c, a.parts, p.strips == 1, a.K, entries, p.strips, p.pieces, st);
}

// The row pass that rounds once and its column sums in one, which reads dh, r, y and dr once: a workgroup a CU owns a strip
// of one entry's rows, a lane the same columns of every row (those of the row pass with four waves, whose row sums and
// results it repeats bit for bit), so its column sums stay in registers (one wave per SIMD has 512) and no wave meets
// another over them.  Both row sums cross the waves behind one barrier (neither needs the other's result) while the next
// row is loaded (without: 47.6 us for 42.0).  Two passes / this one, with the join, us: 9216 x 6144 201 / 152, 4608 x 6144
// 100 / 84, 2 x 768 x 6144 41.6 / 35.8, 1024 x 6144 30.1 / 28.6, 768 x 6144 25.7 / 25.6, 4096 x 8192 121 / 100, 768 x 8192
// 30.1 / 31.0, 768 x 2560 18.1 / 18.1, 16 x 128 x 6144 50.9 / 46.3, 64 x 32 x 6144 49.5 / 44.6, 200 x 64 x 2560 118 / 108;
// for the norm weight's gradient alone 2 x 768 x 6144 36.7 / 26.7, 768 x 6144 21.9 / 19.0.
template <int kNCH>
__global__ __launch_bounds__(256, 1) void resnorm_bwd_cols_kernel(NormBwdArgs a, const uint16_t* y, int64_t ldy, int strips,
                                                                  int strip_rows, int asked, float* part) {
  __shared__ float2 sred[2][4];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, K = a.K;
  const int64_t entry = blockIdx.x / strips;
  const int64_t m0 = entry * a.rpb + (int64_t)(blockIdx.x % strips) * strip_rows, mend = (entry + 1) * a.rpb;
  const int64_t m1 = m0 + strip_rows < mend ? m0 + strip_rows : mend;
  const uint16_t* mg = a.gate ? a.gate + entry * a.ldg : nullptr;
  // what is absent is read as x
  const uint16_t *yp = y ? y : a.x, *rp = a.dr ? a.dr : a.x;
  const int64_t ly = y ? ldy : K;
  float w[kNCH][8], acc[kNCH][4][8] = {};
  uint4 pv[kNCH], gg[kNCH];
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = 8 * t + 2048 * c, cc = col < K ? col : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[c][i] = a.nw[cc + i] + a.nwadd;
    pv[c] = a.mscale ? *reinterpret_cast<const uint4*>(a.mscale + entry * a.ldm + cc) : make_uint4(0, 0, 0, 0);
    gg[c] = mg ? *reinterpret_cast<const uint4*>(mg + cc) : make_uint4(0, 0, 0, 0);
  }
  uint4 xn[kNCH], dn[kNCH], rn[kNCH], yn[kNCH];
  auto load = [&](int64_t m) {
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const int col = 8 * t + 2048 * c, cc = col < K ? col : 0;
      xn[c] = *reinterpret_cast<const uint4*>(a.x + m * K + cc);
      dn[c] = *reinterpret_cast<const uint4*>(a.dh + m * K + cc);
      rn[c] = *reinterpret_cast<const uint4*>(rp + m * K + cc);
      yn[c] = *reinterpret_cast<const uint4*>(yp + m * ly + cc);
    }
  };
  load(m0);
  for (int64_t m = m0; m < m1; ++m) {
    uint4 xv[kNCH], dv[kNCH], rv[kNCH], yv[kNCH];
    float gv[kNCH][8], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const bool ok = 8 * t + 2048 * c < K;
      xv[c] = keep_if(ok, xn[c]);
      dv[c] = keep_if(ok, dn[c]);
      rv[c] = keep_if(a.dr, rn[c]);
      yv[c] = keep_if(y, yn[c]);
    }
    load(m + 1 < m1 ? m + 1 : m);
#pragma unroll
    for (int c = 0; c < kNCH; ++c)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float x0 = bf16_of(xv[c], i), x1 = bf16_of(xv[c], i + 1);
        ss += x0 * x0;
        ss += x1 * x1;
        float p0 = 1.f + bf16_of(pv[c], i), p1 = 1.f + bf16_of(pv[c], i + 1);
        bf16r2(p0, p1);
        gv[c][i] = bf16_of(dv[c], i) * p0 * w[c][i];
        gv[c][i + 1] = bf16_of(dv[c], i + 1) * p1 * w[c][i + 1];
        dot += gv[c][i] * x0;
        dot += gv[c][i + 1] * x1;
      }
    ss = wave_sum(ss);
    dot = wave_sum(dot);
    float2* red = sred[(m - m0) & 1];       // written again two rows later, behind the next row's barrier
    if (lane == 0) red[wave] = make_float2(ss, dot);
    __syncthreads();
    ss = dot = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      ss += red[v].x;
      dot += red[v].y;
    }
    const float r = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)K) + a.eps));
    const float c3 = __fdiv_rn(r * r * r * dot, (float)K);
#pragma unroll
    for (int c = 0; c < kNCH; ++c) {
      const int col = 8 * t + 2048 * c;
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = bf16_of(xv[c], i), dh = bf16_of(dv[c], i), xr = x * r;
        d[i] = gv[c][i] * r - x * c3;
        if (a.dr) d[i] = bf16_of(rv[c], i) + d[i];
        const float dnv = dh * bf16r(1.f + bf16_of(pv[c], i));
        acc[c][CS_W][i] = __builtin_fmaf(dnv, xr, acc[c][CS_W][i]);
        acc[c][CS_SCALE][i] = __builtin_fmaf(dh, bf16r(xr * w[c][i]), acc[c][CS_SCALE][i]);
        acc[c][CS_SHIFT][i] += dh;
        acc[c][CS_GATE][i] = __builtin_fmaf(d[i], bf16_of(yv[c], i), acc[c][CS_GATE][i]);
      }
      if (col >= K) continue;
      uint32_t o[4], e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = pack_bf16x2(d[2 * j], d[2 * j + 1]);
        e[j] = pack_bf16x2(bf16_of(gg[c], 2 * j) * d[2 * j], bf16_of(gg[c], 2 * j + 1) * d[2 * j + 1]);
      }
      *reinterpret_cast<uint4*>(a.dx + m * K + col) = make_uint4(o[0], o[1], o[2], o[3]);
      if (mg) *reinterpret_cast<uint4*>(a.dy + m * K + col) = make_uint4(e[0], e[1], e[2], e[3]);
    }
  }
#pragma unroll
  for (int c = 0; c < kNCH; ++c) {
    const int col = 8 * t + 2048 * c;
    if (col >= K) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (asked & 1 << k) {
        float4* out = reinterpret_cast<float4*>(part + ((int64_t)blockIdx.x * __popc(asked) + cs_slot(asked, k)) * K + col);
        out[0] = make_float4(acc[c][k][0], acc[c][k][1], acc[c][k][2], acc[c][k][3]);
        out[1] = make_float4(acc[c][k][4], acc[c][k][5], acc[c][k][6], acc[c][k][7]);
      }
  }
}

// The workspace: row statistics, then the partials, 16-byte aligned.
int64_t stats_floats(int64_t M) { return (2 * M + 3) / 4 * 4; }

// Strips per entry of that pass, one workgroup a CU of at least four rows each, eight where there are more than eight entries
// (their partials are joined one by one, where the two passes write a short entry's sums at once: 64 x 16 x 6144 29.2 / 31.9
// us, 128 x 8 x 6144 30.1 / 37.5, 200 x 8 x 6144 46.3 / 47.5); 0 (the two passes) where they would leave a quarter of the CUs
// idle, or the columns are not the four-wave row pass's or too many for the registers.
int fused_strips(int64_t rpb, int64_t K, int64_t entries, int cus) {
  if (K <= 2048 || K > 8192) return 0;
  int64_t s = cus / entries;
  const int64_t most = rpb / (entries > 8 ? 8 : 4);
  s = s > most ? most : s;
  if (s < 1 || 4 * entries * s < 3 * cus) return 0;
  const int64_t rows = (rpb + s - 1) / s;
  return (int)((rpb + rows - 1) / rows);
}

}  // namespace

extern "C" int k2q_rmsmod_bwd(const uint16_t* dh, const uint16_t* x, int64_t M, int64_t K, const float* norm_scale,
                              float eps, const uint16_t* mod_scale, int64_t ld_mod, int64_t rows_per_batch,
                              uint16_t* dx, void* stream) {
  if (M < 1 || K < 8 || K % 8) return K2Q_EINVAL;
  if (K > 16384) return K2Q_EUNSUPPORTED;
  if (!dh || !x || !norm_scale || !mod_scale || !dx || !k2q_aligned(dh, 16) || !k2q_aligned(x, 16) ||
      !k2q_aligned(norm_scale, 16) || !k2q_aligned(mod_scale, 16) || !k2q_aligned(dx, 16) || ld_mod < 0 ||
      ld_mod % 8 || rows_per_batch < 1 || !(eps >= 0.f))
    return K2Q_EINVAL;
  NormBwdArgs a{};
  a.dh = dh;
  a.x = x;
  a.M = M;
  a.K = (int)K;
  a.nw = norm_scale;
  a.nwadd = 1.f;
  a.eps = eps;
  a.mscale = mod_scale;
  a.ldm = ld_mod;
  a.rpb = rows_per_batch;
  a.dx = dx;
  launch_norm_bwd<BWD_NORM>(a, static_cast<hipStream_t>(stream));
  return k2q_launch_status();
}

extern "C" int k2q_swiglu_rotquant(const uint16_t* gate, int64_t ldg, const uint16_t* up, int64_t ldu, int64_t M,
                                   int64_t K, uint16_t* h, int8_t* q, float* s, void* stream) {
  int rc = check_prod_common(M, K, h, q, s);
  if (rc) return rc;
  if (!gate || !up || !k2q_aligned(gate, 16) || !k2q_aligned(up, 16) || ldg < K || ldu < K || ldg % 8 || ldu % 8)
    return K2Q_EINVAL;
  ProdArgs a{};
  a.x0 = reinterpret_cast<const __bf16*>(gate);
  a.x1 = reinterpret_cast<const __bf16*>(up);
  a.ld0 = ldg;
  a.ld1 = ldu;
  a.M = M;
  a.K = (int)K;
  a.h = h;
  a.q = q;
  a.s = s;
  return launch_prod<PROD_SWIGLU>(a, static_cast<hipStream_t>(stream));
}

extern "C" int k2q_rmsmod_rotquant(const uint16_t* x, int64_t ldx, int64_t M, int64_t K, const float* norm_scale,
                                   float eps, const uint16_t* mod_scale, const uint16_t* mod_shift, int64_t ld_mod,
                                   int64_t rows_per_batch, uint16_t* h, int8_t* q, float* s, void* stream) {
  int rc = check_prod_common(M, K, h, q, s);
  if (rc) return rc;
  if (!x || !norm_scale || !mod_scale || !mod_shift || !k2q_aligned(x, 16) || !k2q_aligned(norm_scale, 16) ||
      !k2q_aligned(mod_scale, 16) || !k2q_aligned(mod_shift, 16) || ldx < K || ldx % 8 || ld_mod < 0 ||
      ld_mod % 8 || rows_per_batch < 1 || !(eps >= 0.f))
    return K2Q_EINVAL;
  ProdArgs a{};
  a.x0 = reinterpret_cast<const __bf16*>(x);
  a.ld0 = ldx;
  a.nw = norm_scale;
  a.nwadd = 1.f;
  a.mscale = mod_scale;
  a.mshift = mod_shift;
  a.ldm = a.ldb = ld_mod;
  a.rpb = rows_per_batch;
  a.eps = eps;
  a.M = M;
  a.K = (int)K;
  a.h = h;
  a.q = q;
  a.s = s;
  return launch_prod<PROD_RMSMOD>(a, static_cast<hipStream_t>(stream));
}

namespace {

// A per-entry row vector (gate, modulation scale or shift): 16-byte aligned rows, row stride ld (0: one entry).
bool rowvec_ok(const uint16_t* p, int64_t ld) { return k2q_aligned(p, 16) && ld >= 0 && ld % 8 == 0; }

}  // namespace

extern "C" int k2q_resnorm_rotquant(const uint16_t* x, int64_t ldx, const uint16_t* y, int64_t ldy,
                                    const uint16_t* gate, int64_t ld_gate, int64_t M, int64_t K,
                                    const float* norm_scale, float scale_add, float eps, const uint16_t* mod_scale,
                                    int64_t ld_scale, const uint16_t* mod_shift, int64_t ld_shift,
                                    int64_t rows_per_batch, uint16_t* r, uint16_t* h, int8_t* q, float* s,
                                    void* stream) {
  int rc = check_prod_common(M, K, h, q, s);
  if (rc) return rc;
  if (M > 0x7fffffff) return K2Q_EUNSUPPORTED;
  if (!x || !y || !norm_scale || !r || !k2q_aligned(x, 16) || !k2q_aligned(y, 16) || !k2q_aligned(norm_scale, 16) ||
      !k2q_aligned(r, 16) || ldx < K || ldx % 8 || ldy < K || ldy % 8 || rows_per_batch < 1 || !(eps >= 0.f) ||
      !rowvec_ok(gate, ld_gate) || !rowvec_ok(mod_scale, ld_scale) || !rowvec_ok(mod_shift, ld_shift) ||
      !mod_scale != !mod_shift)
    return K2Q_EINVAL;
  ProdArgs a{};
  a.x0 = reinterpret_cast<const __bf16*>(x);
  a.x1 = reinterpret_cast<const __bf16*>(y);
  a.ld0 = ldx;
  a.ld1 = ldy;
  a.nw = norm_scale;
  a.nwadd = scale_add;
  a.mscale = mod_scale;
  a.mshift = mod_shift;
  a.gate = gate;
  a.ldm = ld_scale;
  a.ldb = ld_shift;
  a.ldg = ld_gate;
  a.rpb = rows_per_batch;
  a.eps = eps;
  a.M = M;
  a.K = (int)K;
  a.r = r;
  // r and h of a pass that does not fit the 256 MB last-level cache leave it to the reads (same box, us, cached / streamed:
  // 4608 x 6144, 255 MB, 59.3 / 61.4; 4608 x 8192 84.6 / 79.5; 9216 x 6144 118.1 / 112.8; 2304 x 16384 87.1 / 81.9)
  a.stream = M * K * 9 > (int64_t)256 << 20;
  a.h = h;
  a.q = q;
  a.s = s;
  return launch_prod<PROD_RESNORM>(a, static_cast<hipStream_t>(stream));
}

extern "C" int k2q_swiglu_bwd(const uint16_t* dh, const uint16_t* gate, const uint16_t* up, int64_t n,
                              uint16_t* dgate, uint16_t* dup, void* stream) {
  if (n < 1 || n % 8 || !dh || !gate || !up || !dgate || !dup) return K2Q_EINVAL;
  if (!k2q_aligned(dh, 16) || !k2q_aligned(gate, 16) || !k2q_aligned(up, 16) || !k2q_aligned(dgate, 16) ||
      !k2q_aligned(dup, 16))
    return K2Q_EINVAL;
  const int64_t n8 = n / 8;
  const int64_t blocks = (n8 + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 8192 ? blocks : 8192);
  hipLaunchKernelGGL(swiglu_bwd_kernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream),
                     reinterpret_cast<const uint4*>(dh), reinterpret_cast<const uint4*>(gate),
                     reinterpret_cast<const uint4*>(up), n8, reinterpret_cast<uint4*>(dgate),
                     reinterpret_cast<uint4*>(dup));
  return k2q_launch_status();
}

extern "C" int64_t k2q_resnorm_bwd_ws_bytes(int64_t M, int64_t K, int64_t rows_per_batch) {
  if (M < 1 || K < 8 || K % 8 || K > 16384 || rows_per_batch < 1 || M % rows_per_batch) return 0;
  const int64_t entries = M / rows_per_batch;
  const int cus = k2q_cu_count();
  const int64_t two = colsum_floats(colsum_plan(rows_per_batch, K, entries, cus), K),
                one = entries * fused_strips(rows_per_batch, K, entries, cus) * 4 * K;
  return (stats_floats(M) + (two > one ? two : one)) * 4;
}

namespace {

// The sums asked for; those of `shared` vectors (and the norm weight's always) are over every entry.
ColOut col_out(float* dnorm, uint16_t* dscale, uint16_t* dshift, uint16_t* dgate, int shared, int64_t entries, float* part) {
  const int asked = (dnorm ? 1 << CS_W : 0) | (dscale ? 1 << CS_SCALE : 0) | (dshift ? 1 << CS_SHIFT : 0) |
                    (dgate ? 1 << CS_GATE : 0);
  const int whole = 1 << CS_W | (entries == 1 ? 0 : (shared & K2Q_SHARED_SCALE ? 1 << CS_SCALE : 0) |
                                                        (shared & K2Q_SHARED_SHIFT ? 1 << CS_SHIFT : 0) |
                                                        (shared & K2Q_SHARED_GATE ? 1 << CS_GATE : 0));
  return {asked, whole, dnorm, dscale, dshift, dgate, part};
}

bool shared_ok(int shared) { return shared >= 0 && shared <= (K2Q_SHARED_SCALE | K2Q_SHARED_SHIFT | K2Q_SHARED_GATE); }

}  // namespace

extern "C" int k2q_resnorm_bwd(const uint16_t* dh, const uint16_t* dr, const uint16_t* r, int64_t M, int64_t K,
                               const float* norm_scale, float scale_add, float eps, const uint16_t* mod_scale,
                               int64_t ld_scale, const uint16_t* gate, int64_t ld_gate, int64_t rows_per_batch,
                               int eager, uint16_t* dx, uint16_t* dy, const uint16_t* y, int64_t ldy, float* dnorm,
                               uint16_t* dscale, uint16_t* dshift, uint16_t* dgate, int shared, void* ws,
                               int64_t ws_bytes, void* stream) {
  if (M < 1 || K < 8 || K % 8) return K2Q_EINVAL;
  if (K > 16384 || M > 0x7fffffff) return K2Q_EUNSUPPORTED;
  if (!dh || !r || !norm_scale || !dx || !k2q_aligned(dh, 16) || !k2q_aligned(dr, 16) || !k2q_aligned(r, 16) ||
      !k2q_aligned(norm_scale, 16) || !k2q_aligned(dx, 16) || !k2q_aligned(dy, 16) || !rowvec_ok(mod_scale, ld_scale) ||
      !rowvec_ok(gate, ld_gate) || rows_per_batch < 1 || !(eps >= 0.f) || !gate != !dy || !shared_ok(shared))
    return K2Q_EINVAL;
  const bool cols = dnorm || dscale || dshift || dgate;
  const int64_t entries = M / rows_per_batch;
  if (cols) {
    if (M % rows_per_batch || !ws || !k2q_aligned(ws, 16) || ws_bytes < k2q_resnorm_bwd_ws_bytes(M, K, rows_per_batch) ||
        ((dscale || dshift) && !mod_scale) || !k2q_aligned(dscale, 16) || !k2q_aligned(dshift, 16) ||
        !k2q_aligned(dgate, 16) || (dgate && (!gate || !y || !k2q_aligned(y, 16) || ldy < K || ldy % 8)))
      return K2Q_EINVAL;
  }
  if (!norm_bwd_fits(M, K, eager ? BWD_EAGER : BWD_ONCE)) return K2Q_EUNSUPPORTED;
  NormBwdArgs a{};
  a.dh = dh;
  a.x = r;
  a.M = M;
  a.K = (int)K;
  a.nw = norm_scale;
  a.nwadd = scale_add;
  a.eps = eps;
  a.mscale = mod_scale;
  a.ldm = ld_scale;
  a.rpb = rows_per_batch;
  a.dx = dx;
  a.dr = dr;
  a.gate = gate;
  a.ldg = ld_gate;
  a.dy = dy;
  a.stats = cols ? static_cast<float*>(ws) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const ColOut out = col_out(dnorm, dscale, dshift, dgate, shared, entries, cols ? a.stats + stats_floats(M) : nullptr);
  const int fs = cols && !eager ? fused_strips(rows_per_batch, K, entries, k2q_cu_count()) : 0;
  if (fs) {
    const int rows = (int)((rows_per_batch + fs - 1) / fs);
#define K2Q_RBC(N)                                                                                                        \
  hipLaunchKernelGGL(resnorm_bwd_cols_kernel<N>, dim3((unsigned)(entries * fs)), dim3(256), 0, st, a, dgate ? y : nullptr, \
                     ldy, fs, rows, out.asked, out.part)
    if (K <= 4096) K2Q_RBC(2);
    else if (K <= 6144) K2Q_RBC(3);
    else K2Q_RBC(4);
#undef K2Q_RBC
    launch_join(out, out.asked, false, K, entries, fs, entries * fs, st);
    return k2q_launch_status();
  }
  if (eager) launch_norm_bwd<BWD_EAGER>(a, st);
  else launch_norm_bwd<BWD_ONCE>(a, st);
  if (!cols) return k2q_launch_status();
  ColSumArgs c{};
  c.dh = dh;
  c.x = r;
  c.y = dgate ? y : nullptr;
  c.dr = dr;
  c.stats = a.stats;
  c.M = M;
  c.ldy = ldy;
  c.rpb = rows_per_batch;
  c.K = (int)K;
  c.nw = norm_scale;
  c.nwadd = scale_add;
  c.mscale = mod_scale;
  c.ldm = ld_scale;
  launch_colsum<false>(c, out, colsum_plan(rows_per_batch, K, entries, k2q_cu_count()), entries, st);
  return k2q_launch_status();
}

extern "C" int k2q_resnorm_stream_bwd(const uint16_t* dr, int64_t M, int64_t K, const uint16_t* gate, int64_t ld_gate,
                                      int64_t rows_per_batch, uint16_t* dy, const uint16_t* y, int64_t ldy,
                                      uint16_t* dgate, int shared, void* ws, int64_t ws_bytes, void* stream) {
  if (M < 1 || K < 8 || K % 8) return K2Q_EINVAL;
  if (K > 16384 || M > 0x7fffffff) return K2Q_EUNSUPPORTED;
  if (!dr || !gate || (!dy && !dgate) || !k2q_aligned(dr, 16) || !k2q_aligned(dy, 16) || !rowvec_ok(gate, ld_gate) ||
      rows_per_batch < 1 || M % rows_per_batch || !shared_ok(shared))
    return K2Q_EINVAL;
  if (dgate && (!y || !k2q_aligned(y, 16) || ldy < K || ldy % 8 || !k2q_aligned(dgate, 16) || !ws || !k2q_aligned(ws, 16) ||
                ws_bytes < k2q_resnorm_bwd_ws_bytes(M, K, rows_per_batch)))
    return K2Q_EINVAL;
  const int64_t entries = M / rows_per_batch;
  hipStream_t st = static_cast<hipStream_t>(stream);
  ColSumArgs c{};
  c.dr = dr;
  c.y = dgate ? y : nullptr;
  c.M = M;
  c.ldy = ldy;
  c.rpb = rows_per_batch;
  c.K = (int)K;
  c.gate = gate;
  c.ldg = ld_gate;
  c.dy = dy;
  launch_colsum<true>(c, col_out(nullptr, nullptr, nullptr, dgate, shared, entries, static_cast<float*>(ws)),
                      colsum_plan(rows_per_batch, K, entries, k2q_cu_count()), entries, st);
  return k2q_launch_status();
}
