// The step behind a backward pass, over many tensors in few launches: the gradients' norm and their scaling to a largest
// one (the trainer's clip_grad_norm_, reference train_t2i_lora_cached.py:329), and AdamW (the line after it) with moments in
// 32 bits or in 8.
//
// A launch takes up to TENSORS tensors by value, in its argument block: pointers move from step to step (autograd allocates
// gradients anew), and nothing has to be copied to the device or kept there.  A workgroup finds its tensor by bisecting the
// workgroups' prefix sums, on the scalar unit.  A list of a few tensors goes in a block of FEW, which the host writes faster.
#include <math.h>

#include <type_traits>

#include "k2q_common.h"
#include "rotation.h"

namespace {

constexpr int TENSORS = 64;           // 40 bytes each and 4: 2.8 KB of arguments
constexpr int FEW = 8;
constexpr int THREADS = 256;
constexpr int BLOCK = K2Q_MOMENT_BLOCK;

// Elements of a workgroup.  A step streams: nothing that it reads or writes is wanted again before a whole training step has
// gone by, so all of it passes by the last-level cache.  214.7M parameters in f32, us at 2048 / 4096 / 8192 / 32768 elements
// 1136 / 1160 / 1177 / 1249 through that cache, 1029 at 2048 past it (5.8 TB/s, as much as torch.add of large operands).
constexpr int64_t CHUNK = 2048;

struct Item {
  void* p;
  void* g;
  int64_t n;
  int64_t at;         // the tensor's place in the moments' buffers
  int32_t slot;       // its scalars
  int32_t vec;        // p and g take vector loads
};

template <int N>
struct Table {
  Item t[N];
  uint32_t first[N];          // a tensor's first workgroup
  int32_t count;
  uint32_t blocks;
};

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& a, uint32_t wg) {
  int lo = 0;
#pragma unroll
  for (int s = N / 2; s; s >>= 1)
    if (lo + s < a.count && a.first[lo + s] <= wg) lo += s;
  return lo;
}

// 4 values of a tensor from element e on.  kWhole: all of them are the tensor's, and vectors are aligned, so that the loads of
// several turns of a loop leave together; else what lies past its end reads as zero and is not written.
template <bool kWhole, bool kPast, typename T>
__device__ __forceinline__ v4f load(const T* p, int64_t e, int64_t n) {
  typedef T VecT __attribute__((ext_vector_type(4)));
  VecT q;
  if constexpr (kWhole) {
    const VecT* at = reinterpret_cast<const VecT*>(p + e);
    q = kPast ? __builtin_nontemporal_load(at) : *at;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = e + j < n ? p[e + j] : (T)0.f;
  }
  return v4f{(float)q[0], (float)q[1], (float)q[2], (float)q[3]};
}

template <bool kWhole, typename T>
__device__ __forceinline__ void store(T* p, int64_t e, int64_t n, const T (&v)[4]) {
  typedef T VecT __attribute__((ext_vector_type(4)));
  if constexpr (kWhole) {
    __builtin_nontemporal_store((VecT{v[0], v[1], v[2], v[3]}), reinterpret_cast<VecT*>(p + e));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e + j < n) p[e + j] = v[j];
  }
}

// f(first element of a turn, whole) for a workgroup's turns of THREADS x V elements; whole: a bool constant, as above.
template <int V, class F>
__device__ __forceinline__ void each_turn(const Item& it, int64_t begin, int64_t end, F&& f) {
  const int turns = (int)((end - begin + THREADS * V - 1) / (THREADS * V));
  if (it.vec && end <= it.n && (end - begin) % (THREADS * V) == 0) {
#pragma unroll 4
    for (int i = 0; i < turns; ++i) f(begin + i * (THREADS * V), std::true_type{});
  } else {
    for (int i = 0; i < turns; ++i) f(begin + i * (THREADS * V), std::false_type{});
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Norm and scaling
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  return v;
}

// Sums of squares of runs of `chunk` elements, one a workgroup.  The sums are in 64 bits: squares of 32-bit values neither
// overflow nor vanish there, and the card adds them at half the 32-bit rate, ten times what the reads need.
template <typename T, int N>
__global__ __launch_bounds__(THREADS) void sumsq_kernel(Table<N> a, int64_t chunk, double* part) {
  __shared__ double sums[THREADS / 64];
  const int i = tensor_of(a, blockIdx.x);
  const Item& it = a.t[i];
  const T* g = static_cast<const T*>(it.g);
  const int64_t begin = (int64_t)(blockIdx.x - a.first[i]) * chunk;
  const int64_t n = it.n, end = begin + chunk < n ? begin + chunk : n;
  double s = 0;
  each_turn<4>(it, begin, end, [&](int64_t e, auto whole) {
    e += threadIdx.x * 4;
    if (!whole && e >= end) return;
    const v4f v = load<whole, false>(g, e, n);      // kept: the step reads it next
#pragma unroll
    for (int j = 0; j < 4; ++j) s = __builtin_fma((double)v[j], (double)v[j], s);
  });
  s = wave_add(s);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The norm and the factor that brings it to max_norm, from the partial sums in a fixed order; for every thread of a workgroup
// of N.
struct Norm {
  float norm, by;
};

template <int N>
__device__ __forceinline__ Norm norm_of(const double* part, int64_t n, double max_norm) {
  __shared__ double sums[N / 64];
  double s = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += N) s += part[i];
  s = wave_add(s);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < N / 64; ++i) s += sums[i];
  const double norm = sqrt(s), by = max_norm / (norm + 1e-6);
  return {(float)norm, by > 1.0 ? 1.f : (float)by};      // a norm that is no number gives a factor that is none
}

__global__ __launch_bounds__(1024) void norm_kernel(const double* part, int64_t n, double max_norm, float* out) {
  const Norm v = norm_of<1024>(part, n, max_norm);
  if (threadIdx.x) return;
  out[0] = v.norm;
  out[1] = v.by;
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// Gradients times norm[1]; with few partial sums (parts) every workgroup adds them up itself and the first writes the norm,
// which saves a launch.
template <typename T, int N>
__global__ __launch_bounds__(THREADS) void scale_kernel(Table<N> a, int64_t chunk, const double* part, int64_t parts,
                                                        double max_norm, float* norm) {
  const int i = tensor_of(a, blockIdx.x);
  const Item& it = a.t[i];
  T* g = static_cast<T*>(it.g);
  float f;
  if (part) {
    const Norm v = norm_of<THREADS>(part, parts, max_norm);
    f = v.by;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      norm[0] = v.norm;
      norm[1] = v.by;
    }
  } else {
    f = norm[1];
  }
  const int64_t begin = (int64_t)(blockIdx.x - a.first[i]) * chunk;
  const int64_t n = it.n, end = begin + chunk < n ? begin + chunk : n;
  each_turn<4>(it, begin, end, [&](int64_t e, auto whole) {
    e += threadIdx.x * 4;
    if (!whole && e >= end) return;
    const v4f v = load<whole, true>(g, e, n);
    T o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (T)(v[j] * f);
    store<whole>(g, e, n, o);
  });
}

// ---------------------------------------------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------------------------------------------
// 32 random bits: two rounds of a shift and a product modulo 2^32, with constants of low bias found by C. Wellons (public
// domain).  Every element of a step has its own: its place, mixed with the seed's and the step's.
__device__ __forceinline__ uint32_t mix(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  return h ^ (h >> 16);
}

struct Scalars {
  float decay;      // 1 - lr weight_decay
  float size;       // lr / (1 - beta1^t)
  float root;       // 1 / sqrt(1 - beta2^t)
  uint32_t key;
};

// The tensors' places among the counts: neighbours, or, where tensors without a gradient lie between them, each one's (448
// small tensors, every second without one, a step with its norm: 896 us with a launch for each run, 65 with one launch).
struct Run {
  int32_t first;
  __device__ int32_t of(int i) const { return first + i; }
};

struct Places {
  static constexpr int MOST = 512;
  int32_t at[MOST];
  __device__ int32_t of(int i) const { return at[i]; }
};

// A step's scalars for every tensor, in 64 bits (1 - beta^t loses digits in 32), the count of steps one further, and the norm.
// One that is not finite stops the step: nothing of the tensors changes.
template <class P>
__global__ __launch_bounds__(1024) void begin_kernel(P places, float* steps, int n, double lr, const float* lr_of, double beta1,
                                                     double beta2, double decay, const double* squares, int64_t count,
                                                     double max_norm, float* norm, uint32_t seed, Scalars* out) {
  const int i = blockIdx.x * 1024 + threadIdx.x;
  if (squares) {
    const Norm v = norm_of<1024>(squares, count, max_norm);
    if (i == 0) {
      norm[0] = v.norm;
      norm[1] = v.by;
    }
    if (!finite(v.norm)) return;
  }
  if (i >= n) return;
  const int at = places.of(i);
  const float t = steps[at] + 1.f;
  steps[at] = t;
  if (lr_of) lr = (double)lr_of[0];
  Scalars s;
  s.decay = (float)(1.0 - lr * decay);
  s.size = (float)(lr / (1.0 - pow(beta1, (double)t)));
  s.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
  s.key = mix(mix(seed) ^ (uint32_t)t);
  out[i] = s;
}

// Numbers in 8 bits.  The first moment: sign, 4 bits of exponent and 3 of fraction (OCP e4m3, so a state is a
// float8_e4m3fn tensor), scaled so that the block's largest magnitude is 448.  The root of the second: 4 bits of each, no
// sign, scaled so that the largest is 31744 (code 255).  The step between neighbours is 2^-3 and 2^-4 of a value at most, over
// 17 and 19 binary orders below the largest, and evenly spaced below those.  A moment moves by a tenth (a thousandth) of its
// distance to the gradient, less than half a code, so that rounding to the nearest would leave it where it is: the code is
// chosen at random between the two neighbours, with the chances that make its mean the value.  No root above zero becomes
// zero: the parameter would move by m / eps.
constexpr float M_TOP = 448.f, V_TOP = 31744.f;
constexpr float SMALLEST = 0x1p-100f;     // a block whose largest value is under this holds zeros: 448 / it stays finite

constexpr uint32_t INFINITE = 0x7F800000u;

// A value a of 0 to the format's top.  Where numbers are evenly spaced, below 2^-6 (1 for roots), x = (a + 2^-6) / 2 lies in
// the binary order below and has a's steps there; from 2^-6 on a is the larger of the two.  The code is then the exponent and
// the kept bits of x, less those of x at a = 0.
__device__ __forceinline__ uint32_t code_m(float m, float by, uint32_t random) {
  const float a = fminf(fabsf(m) * by, M_TOP), x = fmaxf(a, __builtin_fmaf(a, 0.5f, 0x1p-7f));
  const uint32_t code = (__float_as_uint(x) + (random & 0xFFFFu) * 16u - (120u << 23)) >> 20;
  return code | (__float_as_uint(m) >> 24 & 0x80u);
}

__device__ __forceinline__ uint32_t code_v(float r, float by, uint32_t random) {
  const float a = fminf(r * by, V_TOP), x = fmaxf(a, __builtin_fmaf(a, 0.5f, 0.5f));
  const uint32_t code = (__float_as_uint(x) + (random >> 16) * 8u - (126u << 23)) >> 19;
  return max(code, min(__float_as_uint(a), 1u));
}

// A value's bits without the sign, 0 for one that is not finite.
__device__ __forceinline__ uint32_t below_infinite(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < INFINITE ? b : 0;
}

__device__ __forceinline__ float value_v(uint32_t c) {
  const float x = __uint_as_float((c << 19) + (126u << 23));
  return fminf(x, __builtin_fmaf(x, 2.f, -1.f));
}

template <int I>
__device__ __forceinline__ float value_m(uint32_t w) {
  return __builtin_amdgcn_cvt_f32_fp8((int)w, I);
}

__device__ __forceinline__ float decode_m(uint32_t w, int i) {
  switch (i) {
    case 0: return value_m<0>(w);
    case 1: return value_m<1>(w);
    case 2: return value_m<2>(w);
    default: return value_m<3>(w);
  }
}

// The largest of a value's 32 neighbours (half a wave), of the bits of values of 0 and more: what is not finite is largest.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}

__device__ __forceinline__ uint32_t half_max(uint32_t v) {
  v = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(v))));
  return max(v, (uint32_t)__shfl_xor((int)v, 16));
}

struct Step {
  void* m;            // 32 bits: floats; 8 bits: codes
  void* v;
  float* m_scale;
  float* v_scale;
  const Scalars* scalars;
  const float* norm;  // {norm, factor}, or null
  float beta1, alpha1, beta2, alpha2, eps;
  int stochastic;
};

// Parameters in 16 bits that are rounded at random: 16 random bits below the kept ones, then the rest is cut off.
template <typename T>
__device__ __forceinline__ T rounded(float p, int stochastic, uint32_t random) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16)) {
    if (stochastic) {     // infinite bits end with zeros and stay; those of a NaN could carry past its sign
      const uint32_t bits = __float_as_uint(p) + (random & 0xFFFFu);
      return __builtin_bit_cast(T, (uint16_t)((p != p ? 0x7FC00000u : bits) >> 16));
    }
  }
  return (T)p;
}


// One element's moments and parameter, in 32 bits:
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,  p = decay p - size m / (root sqrt(v) + eps)
// Moments in 32 bits are bound by memory, and their root and quotient are rounded correctly.  With codes (kCodes) every
// operation that leads to a code rounds on its own and correctly, so that a code is what the formula's 32-bit operations
// give: fused or off by an ulp, one in 2^18 fell to the other side of its border, and the element's next update moved by up to an
// eighth.  The parameter's quotient alone is the hardware's there, 1 ulp off: the vector unit is as busy as memory (about 65
// operations an element, 85 with random rounding of the parameter).
template <bool kCodes>
__device__ __forceinline__ void moments_of(const Step& a, float g, float& m, float& v) {
  if constexpr (kCodes) {
    m = m * a.beta1 + g * a.alpha1;
    v = v * a.beta2 + g * g * a.alpha2;
  } else {
    m = __builtin_fmaf(m, a.beta1, g * a.alpha1);
    v = __builtin_fmaf(v, a.beta2, g * g * a.alpha2);
  }
}

template <bool kCodes>
__device__ __forceinline__ float updated(const Step& a, const Scalars& s, float m, float r, float p) {
  const float d = __builtin_fmaf(r, s.root, a.eps), u = kCodes ? m * __builtin_amdgcn_rcpf(d) : m / d;
  return __builtin_fmaf(p, s.decay, -s.size * u);
}

// The root of a value from LEAST to below infinity: a Newton step from the hardware's reciprocal root, whose residual is exact
// there.  Rounded correctly but where the root lies within 2^-21 of a step from the middle of two.  bf16 parameters with random
// rounding, with the hardware's roots and reciprocals / this and divisions / sqrtf: 396M with codes at random 785 / 808 / 895 us,
// 434M of a training's 858 / 900.
constexpr uint32_t LEAST = 0x0D800000u;      // 2^-100

__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(v), r = v * y;
  return __builtin_fmaf(__builtin_fmaf(-r, r, v), 0.5f * y, r);
}

template <typename T, bool kCodes, int N>
__global__ __launch_bounds__(THREADS) void adamw_kernel(Table<N> a, int64_t chunk, Step st) {
  float by = 1.f;
  if (st.norm) {
    if (!finite(st.norm[0])) return;
    by = st.norm[1];
  }
  const int i = tensor_of(a, blockIdx.x);
  const Item& it = a.t[i];
  const Scalars s = st.scalars[it.slot];
  T* P = static_cast<T*>(it.p);
  const T* G = static_cast<const T*>(it.g);
  const int64_t n = it.n, at = it.at, begin = (int64_t)(blockIdx.x - a.first[i]) * chunk;
  // moments reach to the end of the last block
  const int64_t end = begin + chunk < n ? begin + chunk : (n + BLOCK - 1) / BLOCK * BLOCK;
  // A thread has one quad of neighbours, or, with codes, two, and 32 threads a block.  Two quads of 4-byte values lie 128 apart,
  // so that each vector instruction takes whole lines; of 2-byte values side by side, 16 bytes.
  constexpr int QUADS = kCodes ? 2 : 1, V = 4 * QUADS;
  constexpr int GAP = sizeof(T) == 4 ? 128 : 4, NEXT = !kCodes || sizeof(T) == 4 ? 4 : 8;
  each_turn<V>(it, begin, end, [&](int64_t e, auto whole) {
    const int t = threadIdx.x;
    e += kCodes ? t / 32 * BLOCK + t % 32 * NEXT : t * NEXT;
    if (!whole && e >= end) return;
    const uint64_t place = (uint64_t)(at + e);
    v4f p[QUADS], g[QUADS], m[QUADS], v[QUADS], r[QUADS];
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
      p[q] = load<whole, true>(P, e + q * GAP, n);
      g[q] = load<whole, true>(G, e + q * GAP, n);
    }
    uint32_t random[V];
    if (kCodes || st.stochastic) {
      const uint32_t key = s.key ^ (uint32_t)(place >> 32) * 0x9E3779B9u;     // a block does not straddle 2^32
#pragma unroll
      for (int j = 0; j < V; ++j) random[j] = mix((uint32_t)(place + j / 4 * GAP + j % 4) ^ key);
    }
    if constexpr (kCodes) {
      uint8_t *cm = static_cast<uint8_t*>(st.m) + place, *cv = static_cast<uint8_t*>(st.v) + place;
      uint32_t wm[2], wv[2];
      if constexpr (GAP == 4) {
        const v2u a = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(cm));
        const v2u b = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(cv));
        wm[0] = a[0], wm[1] = a[1], wv[0] = b[0], wv[1] = b[1];
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          wm[q] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(cm + q * GAP));
          wv[q] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(cv + q * GAP));
        }
      }
      const float sm = st.m_scale[place / BLOCK], sv = st.v_scale[place / BLOCK];
      uint32_t bm = 0, bv = 0, far = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int q = j / 4, i = j % 4;
        const float root = value_v(wv[q] >> (8 * i) & 0xFFu) * sv;
        float mj = decode_m(wm[q], i) * sm, vj = root * root;
        moments_of<true>(st, g[q][i] * by, mj, vj);
        m[q][i] = mj;
        r[q][i] = vj;
        bm = max(bm, __float_as_uint(mj) & 0x7FFFFFFFu);
        far = max(far, __float_as_uint(vj) - LEAST);
      }
      if (__ballot(far >= INFINITE - LEAST)) {      // zeros too
#pragma unroll
        for (int j = 0; j < V; ++j) r[j / 4][j % 4] = sqrtf(r[j / 4][j % 4]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j / 4][j % 4] = root_of(r[j / 4][j % 4]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int q = j / 4, i = j % 4;
        p[q][i] = updated<true>(st, s, m[q][i], r[q][i], p[q][i]);
        bv = max(bv, __float_as_uint(r[q][i]) & 0x7FFFFFFFu);
      }
      bm = half_max(bm);
      bv = half_max(bv);
      // A block with a value that is not finite, on a branch that no other takes: the scales are those of the rest
      const bool spoilt = __ballot(bm >= INFINITE || bv >= INFINITE);
      if (spoilt) {
        bm = bv = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          bm = max(bm, below_infinite(m[j / 4][j % 4]));
          bv = max(bv, below_infinite(r[j / 4][j % 4]));
        }
        bm = half_max(bm);
        bv = half_max(bv);
      }
      float am = __uint_as_float(bm), av = __uint_as_float(bv);
      am = am < SMALLEST ? 0.f : am;
      av = av < SMALLEST ? 0.f : av;
      const float fm = am > 0.f ? M_TOP * (1.f / am) : 0.f;
      const float fv = av > 0.f ? V_TOP * (1.f / av) : 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        wm[q] = wv[q] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          wm[q] |= code_m(m[q][i], fm, random[4 * q + i]) << (8 * i);
          wv[q] |= code_v(r[q][i], fv, random[4 * q + i]) << (8 * i);
        }
      }
      if (spoilt) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int q = j / 4, i = j % 4;
          if (__float_as_uint(m[q][i]) * 2 >= INFINITE * 2) wm[q] = (wm[q] & ~(0xFFu << (8 * i))) | 0x7Fu << (8 * i);
          if (__float_as_uint(r[q][i]) * 2 >= INFINITE * 2) wv[q] |= 0xFFu << (8 * i);
        }
      }
      if constexpr (GAP == 4) {
        __builtin_nontemporal_store((v2u{wm[0], wm[1]}), reinterpret_cast<v2u*>(cm));
        __builtin_nontemporal_store((v2u{wv[0], wv[1]}), reinterpret_cast<v2u*>(cv));
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          __builtin_nontemporal_store(wm[q], reinterpret_cast<uint32_t*>(cm + q * GAP));
          __builtin_nontemporal_store(wv[q], reinterpret_cast<uint32_t*>(cv + q * GAP));
        }
      }
      if (t % 32 == 0) {
        st.m_scale[place / BLOCK] = am * (1.f / M_TOP);
        st.v_scale[place / BLOCK] = av * (1.f / V_TOP);
      }
    } else {
      v4f* fm = reinterpret_cast<v4f*>(static_cast<float*>(st.m) + place);
      v4f* fv = reinterpret_cast<v4f*>(static_cast<float*>(st.v) + place);
      v4f wm = __builtin_nontemporal_load(fm), wv = __builtin_nontemporal_load(fv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mj = wm[i], vj = wv[i];
        moments_of<false>(st, g[0][i] * by, mj, vj);
        wm[i] = mj;
        wv[i] = vj;
        p[0][i] = updated<false>(st, s, mj, sqrtf(vj), p[0][i]);
      }
      __builtin_nontemporal_store(wm, fm);
      __builtin_nontemporal_store(wv, fv);
    }
    T o[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      o[j] = rounded<T>(p[j / 4][j % 4], st.stochastic, st.stochastic ? mix(random[j] ^ 0x9E3779B9u) : 0u);
    if constexpr (whole && QUADS == 2 && GAP == 4) {      // one store: half ones past the cache write lines twice
      typedef T Vec8 __attribute__((ext_vector_type(8)));
      __builtin_nontemporal_store((Vec8{o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]}), reinterpret_cast<Vec8*>(P + e));
    } else {
#pragma unroll
      for (int q = 0; q < QUADS; ++q) store<whole>(P, e + q * GAP, n, {o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]});
    }
  });
}

// What codes stand for: m and v, in 32 bits or bf16.
template <typename T>
__global__ __launch_bounds__(THREADS) void moments_kernel(const uint8_t* cm, const float* m_scale, const uint8_t* cv,
                                                          const float* v_scale, int64_t n, T* m, T* v) {
  const int64_t e = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 8;
  if (e >= n) return;
  const v2u wm = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(cm + e));
  const v2u wv = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(cv + e));
  const float sm = m_scale[e / BLOCK], sv = v_scale[e / BLOCK];
  typedef T Vec8 __attribute__((ext_vector_type(8)));
  Vec8 om, ov;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    om[j] = (T)(decode_m(wm[j / 4], j % 4) * sm);
    const float root = value_v(wv[j / 4] >> (8 * (j % 4)) & 0xFFu) * sv;
    ov[j] = (T)(root * root);
  }
  *reinterpret_cast<Vec8*>(m + e) = om;
  *reinterpret_cast<Vec8*>(v + e) = ov;
}

// ---------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------
constexpr int64_t MOST = (int64_t)1 << 34;      // elements of a tensor: 2^23 workgroups, for a launch's threads fit 32 bits

int size_of(int dtype) { return dtype == K2Q_DTYPE_F32 ? 4 : 2; }

int check(const k2q_step_tensor* t, int64_t count, bool params) {
  if (!t || count < 1) return K2Q_EINVAL;
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].dtype < K2Q_DTYPE_BF16 || t[i].dtype > K2Q_DTYPE_F16 || t[i].n < 1 || !t[i].g ||
        !k2q_aligned(t[i].g, size_of(t[i].dtype)) ||
        (params && (!t[i].p || !k2q_aligned(t[i].p, size_of(t[i].dtype)) || t[i].at < 0 || t[i].at % BLOCK || t[i].index < 0)))
      return K2Q_EINVAL;
    if (t[i].n > MOST || t[i].at > (int64_t)1 << 46) return K2Q_EUNSUPPORTED;
  }
  return K2Q_OK;
}

// Elements of a workgroup: CHUNK, or less, down to one turn of its threads, where a CU would not get four workgroups.
int64_t step_chunk(const k2q_step_tensor* t, int64_t count, int64_t least) {
  int64_t total = 0, chunk = CHUNK;
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  while (chunk > least && total / chunk < 4 * (int64_t)k2q_cu_count()) chunk /= 2;
  return chunk;
}

// The same for the norm, which has at most about 16384 partial sums.
int64_t norm_chunk(const k2q_step_tensor* t, int64_t count) {
  int64_t total = 0, chunk = step_chunk(t, count, 4 * THREADS);
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  while (total / chunk > 16384) chunk *= 2;
  return chunk;
}

int64_t norm_parts(const k2q_step_tensor* t, int64_t count) {
  const int64_t chunk = norm_chunk(t, count);
  int64_t parts = 0;
  for (int64_t i = 0; i < count; ++i) parts += (t[i].n + chunk - 1) / chunk;
  return parts;
}

// f(table) over the tensors of one type, N and fewer than 2^24 workgroups at a time.  Behind a pass over the gradients they go
// backwards: what that pass read last is still in the last-level cache.
template <int N, class F>
void tables(const k2q_step_tensor* t, int64_t count, int dtype, int64_t chunk, bool backwards, F&& f) {
  Table<N> a{};
  for (int64_t k = 0; k < count; ++k) {
    const int64_t i = backwards ? count - 1 - k : k;
    if (t[i].dtype != dtype) continue;
    const uint32_t blocks = (uint32_t)((t[i].n + chunk - 1) / chunk);
    if (a.count == N || (a.count && a.blocks + blocks >= 1u << 24)) {
      f(a);
      a.count = 0;
      a.blocks = 0;
    }
    const uintptr_t both = (uintptr_t)t[i].p | (uintptr_t)t[i].g;
    a.t[a.count] = {t[i].p, t[i].g, t[i].n, t[i].at, (int32_t)i, both % 16 == 0};
    a.first[a.count++] = a.blocks;
    a.blocks += blocks;
  }
  if (a.count) f(a);
}

template <class F>
void each_table(const k2q_step_tensor* t, int64_t count, int dtype, int64_t chunk, bool backwards, F&& f) {
  if (count <= FEW) tables<FEW>(t, count, dtype, chunk, backwards, f);
  else tables<TENSORS>(t, count, dtype, chunk, backwards, f);
}

template <class F>
void by_type(F&& f) {
  f(K2Q_DTYPE_BF16, __bf16{});
  f(K2Q_DTYPE_F32, float{});
  f(K2Q_DTYPE_F16, _Float16{});
}

}  // namespace

extern "C" int64_t k2q_grad_norm_ws_bytes(const k2q_step_tensor* t, int64_t count) {
  return check(t, count, false) != K2Q_OK ? 0 : 8 * norm_parts(t, count);
}

extern "C" int k2q_grad_norm(const k2q_step_tensor* t, int64_t count, double max_norm, void* ws, int64_t ws_bytes, float* out,
                             int scale, void* stream) {
  int rc = check(t, count, false);
  if (rc != K2Q_OK) return rc;
  const int64_t parts = norm_parts(t, count);
  int64_t chunk = norm_chunk(t, count);
  if (!(max_norm >= 0) || !ws || ws_bytes < 8 * parts || !k2q_aligned(ws, 16) || !k2q_aligned(out, 8) || (scale && !out))
    return K2Q_EINVAL;
  double* part = static_cast<double*>(ws);
  const double* sums = part;
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type([&](int dtype, auto T) {
    each_table(t, count, dtype, chunk, false, [&](const auto& a) {
      hipLaunchKernelGGL((sumsq_kernel<decltype(T), std::extent_v<decltype(a.first)>>), dim3(a.blocks), dim3(THREADS), 0, st,
                         a, chunk, part);
      part += a.blocks;
    });
  });
  const bool itself = scale && parts <= 2 * THREADS;
  if (out && !itself) hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, st, sums, parts, max_norm, out);
  if (!scale) return k2q_launch_status();
  chunk = step_chunk(t, count, 4 * THREADS);
  by_type([&](int dtype, auto T) {
    each_table(t, count, dtype, chunk, true, [&](const auto& a) {
      hipLaunchKernelGGL((scale_kernel<decltype(T), std::extent_v<decltype(a.first)>>), dim3(a.blocks), dim3(THREADS), 0, st,
                         a, chunk, itself ? sums : nullptr, parts, max_norm, out);
    });
  });
  return k2q_launch_status();
}

extern "C" int64_t k2q_adamw_ws_bytes(int64_t count) { return count < 1 ? 0 : count * (int64_t)sizeof(Scalars); }

extern "C" int k2q_adamw(const k2q_step_tensor* t, int64_t count, int state_bits, void* exp_avg, void* exp_avg_sq,
                         float* avg_scale, float* sq_scale, float* steps, double lr, const float* lr_of, double beta1,
                         double beta2, double eps, double weight_decay, const double* squares, int64_t n_squares,
                         double max_norm, float* norm, int stochastic, uint32_t seed, void* ws, int64_t ws_bytes,
                         void* stream) {
  int rc = check(t, count, true);
  if (rc != K2Q_OK) return rc;
  if ((state_bits != 32 && state_bits != 8) || !exp_avg || !exp_avg_sq || !k2q_aligned(exp_avg, 16) ||
      !k2q_aligned(exp_avg_sq, 16) || (state_bits == 8 && (!avg_scale || !sq_scale)) || !k2q_aligned(avg_scale, 4) ||
      !k2q_aligned(sq_scale, 4) || !steps || !k2q_aligned(steps, 4) || !(beta1 >= 0 && beta1 < 1) ||
      !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(lr == lr) || !(weight_decay >= 0) || !k2q_aligned(lr_of, 4) ||
      (squares && (n_squares < 1 || !k2q_aligned(squares, 8) || !(max_norm >= 0) || !norm || !k2q_aligned(norm, 8))) ||
      !ws || !k2q_aligned(ws, 16) || ws_bytes < k2q_adamw_ws_bytes(count) || count > 0x7fffffff)
    return K2Q_EINVAL;
  for (int64_t i = 0; i < count; ++i)
    if ((stochastic && t[i].dtype == K2Q_DTYPE_F16) || (i && t[i].index <= t[i - 1].index)) return K2Q_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Scalars* scalars = static_cast<Scalars*>(ws);
  auto begin = [&](const auto& places, int64_t first, int64_t n) {
    hipLaunchKernelGGL(begin_kernel<std::decay_t<decltype(places)>>, dim3((unsigned)((n + 1023) / 1024)), dim3(1024), 0, st,
                       places, steps, (int)n, lr, lr_of, beta1, beta2, weight_decay, squares, n_squares, max_norm, norm, seed,
                       scalars + first);
  };
  if (t[count - 1].index - t[0].index == count - 1) {
    begin(Run{t[0].index}, 0, count);
  } else {
    Places p;
    for (int64_t i = 0; i < count; i += Places::MOST) {
      const int64_t n = count - i < Places::MOST ? count - i : Places::MOST;
      for (int64_t j = 0; j < n; ++j) p.at[j] = t[i + j].index;
      begin(p, i, n);
    }
  }
  const int64_t chunk = step_chunk(t, count, (state_bits == 8 ? 8 : 4) * THREADS);
  const Step s{exp_avg, exp_avg_sq, avg_scale, sq_scale, scalars, squares ? norm : nullptr, (float)beta1, (float)(1 - beta1),
               (float)beta2, (float)(1 - beta2), (float)eps, stochastic};
  by_type([&](int dtype, auto T) {
    each_table(t, count, dtype, chunk, squares != nullptr, [&](const auto& a) {
      constexpr int N = std::extent_v<decltype(a.first)>;
      if (state_bits == 8)
        hipLaunchKernelGGL((adamw_kernel<decltype(T), true, N>), dim3(a.blocks), dim3(THREADS), 0, st, a, chunk, s);
      else
        hipLaunchKernelGGL((adamw_kernel<decltype(T), false, N>), dim3(a.blocks), dim3(THREADS), 0, st, a, chunk, s);
    });
  });
  return k2q_launch_status();
}

extern "C" int k2q_moments(const uint8_t* avg, const float* avg_scale, const uint8_t* sq, const float* sq_scale, int64_t n,
                           int dtype, void* m, void* v, void* stream) {
  if (!avg || !avg_scale || !sq || !sq_scale || !m || !v || n < BLOCK || n % BLOCK || !k2q_aligned(avg, 8) ||
      !k2q_aligned(sq, 8) || !k2q_aligned(avg_scale, 4) || !k2q_aligned(sq_scale, 4) || !k2q_aligned(m, 16) ||
      !k2q_aligned(v, 16) || (dtype != K2Q_DTYPE_BF16 && dtype != K2Q_DTYPE_F32))
    return K2Q_EINVAL;
  if (n > MOST) return K2Q_EUNSUPPORTED;
  const dim3 grid((unsigned)((n / 8 + THREADS - 1) / THREADS));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2Q_DTYPE_BF16)
    hipLaunchKernelGGL(moments_kernel<__bf16>, grid, dim3(THREADS), 0, st, avg, avg_scale, sq, sq_scale, n,
                       static_cast<__bf16*>(m), static_cast<__bf16*>(v));
  else
    hipLaunchKernelGGL(moments_kernel<float>, grid, dim3(THREADS), 0, st, avg, avg_scale, sq, sq_scale, n,
                       static_cast<float*>(m), static_cast<float*>(v));
  return k2q_launch_status();
}
