// Skinny-M W8A8 forward (M <= 8 tokens): the adaLN modulation linears of the DiT run at M = batch
// (mmdit.py:314-317 modulate with one vector per sample), where the 256 x 256 MFMA tiles would hold 2
// valid rows out of 256 and a few dozen workgroups would have to stream the whole weight.  This path is
// HBM-bound on the weight read (N x K bytes, once): every wave streams GV_ROWS weight rows with 16-byte
// loads (a lane owns bytes 16 l + 1024 c of a row), dots them against the M token rows with
// v_dot4_i32_i8 (exact int32, the same sums as the MFMA path), and reduces across the wave with
// shuffles (integer adds: exact, order-free).
//
// The epilogue is the MFMA kernel's, term for term: f = fma(float(acc), (s_x 2^-7) s_w, bias); with LoRA,
// L = sum_j bf16(B[n,j]) bf16(s u[m,j]) in f32 is added to f; the result is rounded to bf16 once.  Without
// LoRA both paths give identical bits; with LoRA only L's summation order differs (the MFMA's internal
// order vs sequential here).
//
// The W4A8 form (k2q_launch_gemv_w4a8) streams packed int4 rows the same way: N x K / 2 bytes of codes and N x K / 32 of
// bf16 group scales, once.  A 16-byte load holds 32 weights, half of a 64-wide scale group, so a lane's exact int32 dot
// with the activation codes is scaled by its own group's scale and added in f32:
//   y[m][n] = bf16((s_x[m] 2^-7) sum_g s4[g][n] (sum_{k in g} q_x q_w) + bias + LoRA).
// In a packed chunk of 8 bytes byte j holds code j in its low and code j + 8 in its high nibble: a 32-bit word shifted
// left by 4 and masked, or masked alone, is four weights of consecutive k times 16, dotted as they are with four
// consecutive activation codes; the factor 16 leaves in the epilogue (a power of two: exact).
#include "k2q_common.h"

namespace {

constexpr int GV_ROWS = 4;    // weight rows per wave
constexpr int GV_WAVES = 4;   // waves per workgroup
constexpr int GV_CHUNK = 4;   // 1 KB row chunks per lane in flight (4 KB of every row per pass)

struct GemvArgs {
  const int8_t* qx;      // M x K
  const float* sx;       // M
  const int8_t* qw;      // N x K
  const float* sw;       // N
  const float* bias;     // N or null
  const float* u;        // M x r or null
  const float* lora_b;   // N x r
  int r;
  float lora_scale;
  int64_t M, N, K;
  uint16_t* y;           // M x N bf16
};

// The LoRA term of one output: sum_j bf16(B[n, j]) bf16(scale u[m, j]) in f32, j ascending (r % 4 == 0).
__device__ __forceinline__ float lora_dot(const float* ub, const float* bb, int r, float scale) {
  float l = 0.f;
  for (int j = 0; j < r; j += 4) {
    const v4f uv = *reinterpret_cast<const v4f*>(ub + j);
    const v4f bv = *reinterpret_cast<const v4f*>(bb + j);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      l = __builtin_fmaf(bf16_bits_to_f32(f32_to_bf16_bits(bv[e])),
                         bf16_bits_to_f32(f32_to_bf16_bits(uv[e] * scale)), l);
  }
  return l;
}

template <int MT>
__global__ __launch_bounds__(64 * GV_WAVES) void gemv_w8_kernel(GemvArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t n0 = ((int64_t)blockIdx.x * GV_WAVES + (threadIdx.x >> 6)) * GV_ROWS;
  if (n0 >= p.N) return;   // the kernel has no barriers: a wave past the end simply leaves

  const int8_t* wrow[GV_ROWS];
#pragma unroll
  for (int i = 0; i < GV_ROWS; ++i) {
    const int64_t n = n0 + i < p.N ? n0 + i : p.N - 1;
    wrow[i] = p.qw + n * p.K;
  }
  int acc[GV_ROWS][MT];
#pragma unroll
  for (int i = 0; i < GV_ROWS; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = 0;

  for (int64_t kb = 0; kb < p.K; kb += 1024 * GV_CHUNK) {
    v4i w[GV_CHUNK][GV_ROWS];
#pragma unroll
    for (int c = 0; c < GV_CHUNK; ++c) {
      const int64_t k = kb + 1024 * c + 16 * lane;
#pragma unroll
      for (int i = 0; i < GV_ROWS; ++i)
        w[c][i] = k < p.K ? __builtin_nontemporal_load(reinterpret_cast<const v4i*>(wrow[i] + k)) : v4i{0};
    }
#pragma unroll
    for (int c = 0; c < GV_CHUNK; ++c) {
      const int64_t k = kb + 1024 * c + 16 * lane;
      if (k >= p.K) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const v4i xv = *reinterpret_cast<const v4i*>(p.qx + m * p.K + k);
#pragma unroll
        for (int i = 0; i < GV_ROWS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][m] = __builtin_amdgcn_sdot4(w[c][i][e], xv[e], acc[i][m], false);
      }
    }
  }

  // Wave reduction: afterwards every lane holds every (row, token) sum.
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < GV_ROWS; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[i][m] += __shfl_xor(acc[i][m], off, 64);

  // Lane i + GV_ROWS m writes y[m][n0 + i].
  if (lane >= GV_ROWS * MT) return;
  const int i = lane % GV_ROWS, m = lane / GV_ROWS;
  const int64_t n = n0 + i;
  if (n >= p.N) return;
  int a = 0;
#pragma unroll
  for (int ii = 0; ii < GV_ROWS; ++ii)
#pragma unroll
    for (int mm = 0; mm < MT; ++mm) a = (ii == i && mm == m) ? acc[ii][mm] : a;

  const float sxm = p.sx[m] * 0.0078125f;   // 2^-7: the two unnormalised rotations
  const float bi = p.bias ? p.bias[n] : 0.f;
  float f = __builtin_fmaf((float)a, sxm * p.sw[n], bi);
  if (p.u) f += lora_dot(p.u + (int64_t)m * p.r, p.lora_b + n * p.r, p.r, p.lora_scale);
  p.y[(int64_t)m * p.N + n] = (uint16_t)f32_to_bf16_bits(f);
}

struct Gemv4Args {
  const int8_t* qx;      // M x K
  const float* sx;       // M
  const uint8_t* qw;     // N x K / 2 packed
  const uint16_t* s4;    // K / 64 x N bf16
  const float* bias;     // N or null
  const float* u;        // M x r or null
  const float* lora_b;   // N x r
  int r;
  float lora_scale;
  int64_t N;
  int K;
  uint16_t* y;           // M x N bf16
  int waves, teams;      // waves on one team's rows, teams per workgroup
};

// 32 weights of one row against 32 activation codes (x[0..7]: four codes a word, k ascending); 16 times the dot.
__device__ __forceinline__ int dot32_i4(const v4u& w, const v4i& x0, const v4i& x1) {
  int d = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {      // a 16-wide chunk: words 2 j (k 0-3, 8-11) and 2 j + 1 (k 4-7, 12-15)
    const v4i& x = j ? x1 : x0;
    d = __builtin_amdgcn_sdot4((int)((w[2 * j] << 4) & 0xf0f0f0f0u), x[0], d, false);
    d = __builtin_amdgcn_sdot4((int)((w[2 * j + 1] << 4) & 0xf0f0f0f0u), x[1], d, false);
    d = __builtin_amdgcn_sdot4((int)(w[2 * j] & 0xf0f0f0f0u), x[2], d, false);
    d = __builtin_amdgcn_sdot4((int)(w[2 * j + 1] & 0xf0f0f0f0u), x[3], d, false);
  }
  return d;
}

// v + its neighbour's v under a DPP permutation of 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// Sums over the wave of NV values (NV even or 1): afterwards lane l holds in v[0..] the sums of the values that its
// 32-lane half, then 16-lane row, took.  Each swap folds two values into one register (32 lanes apart, then 16), so a
// value costs one add per stage for every two; the four stages inside a row are DPP adds.  The tree of one value is the
// same for every NV.
template <int NV>
__device__ __forceinline__ void wave_sums(float (&v)[NV], float (&out)[(NV + 3) / 4]) {
  constexpr int H = (NV + 1) / 2, Q = (H + 1) / 2;
  float h[H];
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(i + H < NV ? v[i + H] : v[i]),
                                                    false, false);
    h[i] = __uint_as_float(p[0]) + __uint_as_float(p[1]);      // lanes 0-31: value i, 32-63: value i + H
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[i]), __float_as_uint(i + Q < H ? h[i + Q] : h[i]),
                                                    false, false);
    float f = __uint_as_float(p[0]) + __uint_as_float(p[1]);   // odd 16-lane rows: h[i + Q]
    f = dpp_add<0xB1>(f);      // quad_perm xor 1
    f = dpp_add<0x4E>(f);      // quad_perm xor 2
    f = dpp_add<0x141>(f);     // row_half_mirror
    out[i] = dpp_add<0x140>(f);   // row_mirror
  }
}

// A team of `waves` waves owns GV_ROWS rows; a wave takes every `waves`-th 2048-wide step of K (16 bytes a lane), at most
// G4_STEPS of them, all loads issued before the first is used.  The team's sums meet in LDS.
constexpr int G4_STEPS = 2;         // K <= 16384: four waves of two steps
constexpr int G4_K = 2048;

template <int MT>
__global__ __launch_bounds__(256) void gemv_w4_kernel(Gemv4Args p) {
  constexpr int NV = GV_ROWS * MT, NS = (NV + 3) / 4;
  __shared__ float red[4][4 * NS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int team = wave / p.waves, part = wave % p.waves;
  // workgroups of one XCD (dispatched round-robin over eight) take neighbouring rows: the 128-byte lines of the scales,
  // 64 rows wide, are then read by one XCD's L2 instead of all eight
  const uint32_t per = gridDim.x >> 3, rest = gridDim.x & 7, x = blockIdx.x & 7, i = blockIdx.x >> 3;
  const int64_t block = x * per + (x < rest ? x : rest) + i;
  const int64_t n0 = (block * p.teams + team) * GV_ROWS;
  const bool live = n0 < p.N;       // N % 4 == 0: a team's four rows are all there or none is
  const int kb = p.K / 2;           // bytes per row
  const uint8_t* w0 = p.qw + (live ? n0 : 0) * kb;
  v4u w[G4_STEPS][GV_ROWS];
  v2u sv[G4_STEPS];
#pragma unroll
  for (int s = 0; s < G4_STEPS; ++s) {
    const int k = G4_K * (part + s * p.waves) + 32 * lane;
    const bool ok = live && k < p.K;
    sv[s] = v2u{0, 0};
    if (ok) sv[s] = *reinterpret_cast<const v2u*>(p.s4 + (int64_t)(k >> 6) * p.N + n0);
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r) {
      w[s][r] = v4u{0, 0, 0, 0};
      if (ok) w[s][r] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(w0 + (int64_t)r * kb + (k >> 1)));
    }
  }
  float acc[NV] = {};
#pragma unroll
  for (int s = 0; s < G4_STEPS; ++s) {
    const int k = G4_K * (part + s * p.waves) + 32 * lane;
    if (k >= p.K) break;
    const float sc[GV_ROWS] = {__uint_as_float(sv[s][0] << 16), __uint_as_float(sv[s][0] & 0xffff0000u),
                               __uint_as_float(sv[s][1] << 16), __uint_as_float(sv[s][1] & 0xffff0000u)};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const v4i x0 = *reinterpret_cast<const v4i*>(p.qx + (int64_t)m * p.K + k);
      const v4i x1 = *reinterpret_cast<const v4i*>(p.qx + (int64_t)m * p.K + k + 16);
#pragma unroll
      for (int r = 0; r < GV_ROWS; ++r)
        acc[GV_ROWS * m + r] = __builtin_fmaf((float)dot32_i4(w[s][r], x0, x1), sc[r], acc[GV_ROWS * m + r]);
    }
  }
  float sum[NS];
  wave_sums<NV>(acc, sum);
  if ((lane & 15) == 0) {
#pragma unroll
    for (int j = 0; j < NS; ++j) red[wave][(lane >> 4) * NS + j] = sum[j];
  }
  __syncthreads();
  if (part || !live || lane >= NV) return;
  // value `lane` = GV_ROWS m + r: row 2 (upper half of the values) + (second half of those) of red, in order
  const int m = lane / GV_ROWS, r = lane % GV_ROWS;
  constexpr int H = (NV + 1) / 2;
  const int up = lane >= H, in = lane - up * H, odd = in >= NS;
  const int at = (2 * up + odd) * NS + in - odd * NS;
  float a = 0.f;
  for (int v = 0; v < p.waves; ++v) a += red[wave + v][at];
  const int64_t n = n0 + r;
  float f = __builtin_fmaf(a, p.sx[m] * (0.0078125f * 0.0625f), p.bias ? p.bias[n] : 0.f);
  if (p.u) f += lora_dot(p.u + (int64_t)m * p.r, p.lora_b + n * p.r, p.r, p.lora_scale);
  p.y[(int64_t)m * p.N + n] = (uint16_t)f32_to_bf16_bits(f);
}

template <int MT>
int launch4_mt(Gemv4Args p, hipStream_t st) {
  const int steps = (p.K + G4_K - 1) / G4_K;
  p.waves = steps < 4 ? steps : 4;
  p.teams = 4 / p.waves;
  const int64_t rows_per_wg = (int64_t)GV_ROWS * p.teams;
  const int64_t grid = (p.N + rows_per_wg - 1) / rows_per_wg;
  if (grid > 0x7fffffff) return K2Q_EUNSUPPORTED;
  hipLaunchKernelGGL(gemv_w4_kernel<MT>, dim3((unsigned)grid), dim3(64 * p.waves * p.teams), 0, st, p);
  return k2q_launch_status();
}

template <int MT>
int launch_mt(const GemvArgs& p, hipStream_t st) {
  const int64_t rows_per_wg = (int64_t)GV_ROWS * GV_WAVES;
  const int64_t grid = (p.N + rows_per_wg - 1) / rows_per_wg;
  if (grid > 0x7fffffff) return K2Q_EUNSUPPORTED;
  hipLaunchKernelGGL(gemv_w8_kernel<MT>, dim3((unsigned)grid), dim3(64 * GV_WAVES), 0, st, p);
  return k2q_launch_status();
}

}  // namespace

// Called by k2q_gemm_w8a8 after its argument checks, for 1 <= M <= K2Q_GEMV_MAX_M.
int k2q_launch_gemv_w8a8(const int8_t* qx, const float* sx, const int8_t* qw, const float* sw, const float* bias,
                         const float* u, const float* lora_b, int r, float lora_scale, int64_t M, int64_t N,
                         int64_t K, uint16_t* y, hipStream_t st) {
  GemvArgs p{qx, sx, qw, sw, bias, u, lora_b, u ? r : 0, lora_scale, M, N, K, y};
  switch (M) {
    case 1: return launch_mt<1>(p, st);
    case 2: return launch_mt<2>(p, st);
    case 3: return launch_mt<3>(p, st);
    case 4: return launch_mt<4>(p, st);
    case 5: return launch_mt<5>(p, st);
    case 6: return launch_mt<6>(p, st);
    case 7: return launch_mt<7>(p, st);
    case 8: return launch_mt<8>(p, st);
    default: return K2Q_EINVAL;
  }
}

// Called by k2q_gemm_w4a8 after its argument checks (N % 4 == 0, K % 128 == 0), for 1 <= M <= K2Q_GEMV_MAX_M.
int k2q_launch_gemv_w4a8(const int8_t* qx, const float* sx, const uint8_t* qw4, const uint16_t* sw4, const float* bias,
                         const float* u, const float* lora_b, int r, float lora_scale, int64_t M, int64_t N,
                         int64_t K, uint16_t* y, hipStream_t st) {
  if (K > 4 * G4_STEPS * G4_K) return K2Q_EUNSUPPORTED;
  Gemv4Args p{qx, sx, qw4, sw4, bias, u, lora_b, u ? r : 0, lora_scale, N, (int)K, y, 1, 1};
  switch (M) {
    case 1: return launch4_mt<1>(p, st);
    case 2: return launch4_mt<2>(p, st);
    case 3: return launch4_mt<3>(p, st);
    case 4: return launch4_mt<4>(p, st);
    case 5: return launch4_mt<5>(p, st);
    case 6: return launch4_mt<6>(p, st);
    case 7: return launch4_mt<7>(p, st);
    case 8: return launch4_mt<8>(p, st);
    default: return K2Q_EINVAL;
  }
}
