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
#include "rotation.h"

namespace {

using namespace k2q_rot;

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

// The LoRA term of one output: sum_j bf16(B[n, j]) bf16(scale u[m, j]) in f32, j ascending (r % 16 == 0).  The loads of 16
// ranks are issued together: their latency is all that a workgroup waits for at its end.
__device__ __forceinline__ float lora_dot(const float* ub, const float* bb, int r, float scale) {
  float l = 0.f;
  for (int j = 0; j < r; j += 16) {
    v4f uv[4], bv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bv[i] = *reinterpret_cast<const v4f*>(bb + j + 4 * i);
      uv[i] = *reinterpret_cast<const v4f*>(ub + j + 4 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        l = __builtin_fmaf(bf16_bits_to_f32(f32_to_bf16_bits(bv[i][e])),
                           bf16_bits_to_f32(f32_to_bf16_bits(uv[i][e] * scale)), l);
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
  const __bf16* x;       // kQuant: the token's row, whose codes and scale go to q and s
  int8_t* q;
  float* s;
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

// Orders a wave's LDS writes before its lanes' reads of one another's.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The epilogue: a is 16 times the scaled sum of row n and token m.
__device__ __forceinline__ void gemv4_store(const Gemv4Args& p, int m, int64_t n, float a, float sx) {
  float f = __builtin_fmaf(a, sx * (0.0078125f * 0.0625f), p.bias ? p.bias[n] : 0.f);
  if (p.u) f += lora_dot(p.u + (int64_t)m * p.r, p.lora_b + n * p.r, p.r, p.lora_scale);
  p.y[(int64_t)m * p.N + n] = (uint16_t)f32_to_bf16_bits(f);
}

// This workgroup's place when those of one XCD (dispatched round-robin over eight) take neighbouring rows: the 128-byte
// lines of the scales, 64 rows wide, are then read by one XCD's L2 instead of all eight.
__device__ __forceinline__ int64_t xcd_block() {
  const uint32_t per = gridDim.x >> 3, rest = gridDim.x & 7, x = blockIdx.x & 7, i = blockIdx.x >> 3;
  return x * per + (x < rest ? x : rest) + i;
}

// v + its neighbour's v under a DPP permutation of 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// Sums over the wave of NV values (NV % 4 == 0): afterwards every lane of 16-lane row 2 u + o holds in out[i] the sum of
// value i + u NV / 2 + o NV / 4.  Each swap folds two values into one register (32 lanes apart, then 16), so a stage costs
// one add for two values; the four stages inside a row are DPP adds.  The tree of one value is the same for every NV.
template <int NV>
__device__ __forceinline__ void wave_sums(float (&v)[NV], float (&out)[NV / 4]) {
  static_assert(NV % 4 == 0, "values fold in fours");
  constexpr int H = NV / 2, Q = NV / 4;
  float h[H];
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + H]), false, false);
    h[i] = __uint_as_float(p[0]) + __uint_as_float(p[1]);      // lanes 0-31: value i, 32-63: value i + H
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[i]), __float_as_uint(h[i + Q]), false, false);
    float f = __uint_as_float(p[0]) + __uint_as_float(p[1]);   // odd 16-lane rows: h[i + Q]
    f = dpp_add<0xB1>(f);      // quad_perm xor 1
    f = dpp_add<0x4E>(f);      // quad_perm xor 2
    f = dpp_add<0x141>(f);     // row_half_mirror
    out[i] = dpp_add<0x140>(f);   // row_mirror
  }
}

// The same product on the matrix cores: a workgroup owns 16 or 32 rows, its waves split K into 1024-wide segments (512
// bytes of a row, 16 scale groups).  One 16 x 16 x 64 MFMA is 16 weight rows against up to 16 token rows over a scale group:
// lane (c = lane % 16, b = lane / 16) holds the 8 bytes of row c and the 16 codes of token c at k = 64 g + 16 b, and gets
// the dots of row c with the token operand's rows 4 b .. 4 b + 3.  Loaded in that layout a row's bytes come 32 at a time
// (2.9 TB/s); so a wave loads whole row segments, 16 bytes a lane, and turns them through its own piece of LDS: row c,
// 16-byte unit q at unit q ^ 2 (c % 8), which spreads the eight rows of a read over all banks.  With at most 8 tokens half
// of a token operand would be idle: its rows 8-15 hold the same tokens' codes of the next group, so one register serves two
// MFMAs, whose results for tokens 0-7 are rows 0-7 (even groups) and rows 8-15 (odd groups): eight tokens over 36864 x 6144
// in 29.7 us, 36.8 with a register each (112 of them instead of 78).
constexpr int GM_ROWS = 16;
constexpr int GM_SEG = 1024;
constexpr int GM_GROUPS = GM_SEG / 64;
constexpr int GM_WAVES = 8;         // K <= 16 segments: two a wave, or 16 waves
constexpr int GM_LDS = GM_ROWS * GM_SEG / 2 + GM_GROUPS * GM_ROWS * 2;   // a wave's piece: codes, then scales

// A workgroup has RT tiles of 16 rows and up to 8 RT waves; a wave takes STEPS segments, its tiles in turn through its LDS.
template <int STEPS, int RT>
__global__ __launch_bounds__(64 * GM_WAVES * RT) void gemv_w4_mfma_kernel(Gemv4Args p, int M) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, b = lane >> 4;
  const int64_t n0 = xcd_block() * (GM_ROWS * RT);
  const int kb = p.K >> 1;
  // loads: lane's row 2 i + lane / 32 (clamped to the last), its 16 bytes at 16 (lane % 32) of the segment; its scales'
  // group lane / 4 and four rows
  int64_t s0[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) s0[t] = n0 + 16 * t + 4 * (lane & 3) < p.N ? n0 + 16 * t + 4 * (lane & 3) : p.N - 4;
  const int tok = c & 7;
  const int8_t* xp = p.qx + (int64_t)(tok < M ? tok : 0) * p.K + 64 * (c >> 3) + 16 * b;
  v4u w[STEPS][RT][GM_ROWS / 2];
  v2u sc[STEPS][RT];
  v4i x[GM_GROUPS / 2];
  auto load_x = [&](int k0) {      // K % 128 == 0: groups come in pairs
#pragma unroll
    for (int g = 0; g < GM_GROUPS / 2; ++g)
      x[g] = *reinterpret_cast<const v4i*>(xp + (k0 + 128 * g < p.K ? k0 + 128 * g : 0));
  };
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k0 = GM_SEG * (wave + s * p.waves);
    if (k0 >= p.K) break;
    const int k = k0 + 32 * (lane & 31), g = (k0 >> 6) + (lane >> 2);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int i = 0; i < GM_ROWS / 2; ++i) {
        const int64_t at = n0 + 16 * t + 2 * i + (lane >> 5), row = at < p.N ? at : p.N - 1;
        w[s][t][i] = v4u{0, 0, 0, 0};
        if (k < p.K) w[s][t][i] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p.qw + row * kb + (k >> 1)));
      }
      sc[s][t] = v2u{0, 0};
      if (64 * g < p.K) sc[s][t] = *reinterpret_cast<const v2u*>(p.s4 + (int64_t)g * p.N + s0[t]);
    }
    if (s == 0) load_x(k0);
  }
  float acc[RT][4] = {};
  uint8_t* wt = lds + GM_LDS * wave;
  uint16_t* st = reinterpret_cast<uint16_t*>(wt + GM_ROWS * GM_SEG / 2);
  const int sw = 2 * (c & 7);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k0 = GM_SEG * (wave + s * p.waves);
    if (k0 >= p.K) break;
    if (s) load_x(k0);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      wave_fence();
#pragma unroll
      for (int i = 0; i < GM_ROWS / 2; ++i) {
        const int r = 2 * i + (lane >> 5);
        *reinterpret_cast<v4u*>(wt + r * (GM_SEG / 2) + 16 * ((lane & 31) ^ (2 * (r & 7)))) = w[s][t][i];
      }
      *reinterpret_cast<v2u*>(st + 4 * lane) = sc[s][t];
      wave_fence();
      // groups past K: codes and scales are zeros
#pragma unroll
      for (int g = 0; g < GM_GROUPS; g += 2) {
        v4i d[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int unit = (2 * (g + h) + (b >> 1)) ^ sw;
          const v2u q = *reinterpret_cast<const v2u*>(wt + c * (GM_SEG / 2) + 16 * unit + 8 * (b & 1));
          const v4i a = {(int)((q[0] << 4) & 0xf0f0f0f0u), (int)((q[1] << 4) & 0xf0f0f0f0u), (int)(q[0] & 0xf0f0f0f0u),
                         (int)(q[1] & 0xf0f0f0f0u)};
          d[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[g / 2], a, v4i{0, 0, 0, 0}, 0, 0, 0);
        }
        const float f = bf16_bits_to_f32(st[GM_ROWS * (g + (b >> 1)) + c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf((float)(b < 2 ? d[0][i] : d[1][i]), f, acc[t][i]);
      }
    }
  }
  wave_fence();
  float* red = reinterpret_cast<float*>(wt);      // 8 tokens x the rows, over the wave's own codes
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] += __shfl_xor(acc[t][i], 32, 64);      // even groups' sum plus odd groups'
    if (b < 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[GM_ROWS * RT * (4 * b + i) + 16 * t + c] = acc[t][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GM_ROWS * RT * M; i += 64 * p.waves) {
    const int m = i / (GM_ROWS * RT), r = i % (GM_ROWS * RT);
    const int64_t n = n0 + r;
    if (n >= p.N) continue;
    float a = 0.f;
    for (int v = 0; v < p.waves; ++v) a += reinterpret_cast<const float*>(lds + GM_LDS * v)[i];
    gemv4_store(p, m, n, a, p.sx[m]);
  }
}

template <int STEPS, int RT>
int launch4_mfma(const Gemv4Args& p, int M, hipStream_t st) {
  static std::atomic<uint64_t> lds_set{0};
  const int rc = k2q_lds_limit_once(gemv_w4_mfma_kernel<STEPS, RT>, GM_LDS * GM_WAVES * RT, lds_set);
  if (rc) return rc;
  const int64_t grid = (p.N + GM_ROWS * RT - 1) / (GM_ROWS * RT);
  if (grid > 0x7fffffff) return K2Q_EUNSUPPORTED;
  hipLaunchKernelGGL((gemv_w4_mfma_kernel<STEPS, RT>), dim3((unsigned)grid), dim3(64 * p.waves), GM_LDS * p.waves, st, p, M);
  return k2q_launch_status();
}

// 16 rows a workgroup, or 32 and a wave a segment where that is one workgroup a CU or less and 16 rows would be more than
// one: the CUs with two then end last, and every workgroup reads all tokens' codes.  It takes a CU's LDS and registers
// for itself, so it loses in more than one round and, with few segments, where it has little more in flight.  us, 16 rows /
// 32 rows, M = 3, then M = 8:
//   4096 x 16384   10.3 / 12.3   11.3 / 13.7       6144 x 12288   11.8 / 11.5   14.0 / 12.5
//   4352 x 16384   13.8 / 12.3   16.9 / 13.8      12288 x 12288   18.4 / 23.2   20.4 / 23.4
//   6144 x 16384   14.4 / 13.7   17.4 / 15.0       4352 x 9344     9.8 / 10.0   11.5 / 10.7
//   8192 x 16384   15.7 / 15.7   18.5 / 16.6       8192 x 8320    10.2 / 10.8   11.3 / 11.5
int launch4_mfma(Gemv4Args p, int M, hipStream_t st) {
  const int segs = (p.K + GM_SEG - 1) / GM_SEG, cus = k2q_cu_count();
  if (segs > GM_WAVES + 1 && p.N > GM_ROWS * cus && p.N <= 2 * GM_ROWS * cus) {
    p.waves = segs;
    return launch4_mfma<1, 2>(p, M, st);
  }
  p.waves = segs < GM_WAVES ? segs : GM_WAVES;
  return segs <= GM_WAVES ? launch4_mfma<1, 1>(p, M, st) : launch4_mfma<2, 1>(p, M, st);
}

constexpr int G4_K = 2048;

// A team of `waves` waves owns R rows; a wave takes every `waves`-th 2048-wide step of K (16 bytes a lane), STEPS of
// them, all weight loads issued before the first is used.  The team's sums meet in LDS.
//
// kQuant: the codes are made here from x, by every workgroup for itself (rotated in registers, one row maximum over the
// team, the arithmetic of rotquant_kernel bit for bit) while its weight loads are in flight; the first writes them out.
template <int MT, int R, int STEPS, bool kQuant>
__global__ __launch_bounds__(256) void gemv_w4_kernel(Gemv4Args p) {
  constexpr int NV = R * MT, NS = NV / 4, H = NV / 2;
  __shared__ float red[4][4 * NS];
  static_assert(!kQuant || (MT == 1 && STEPS == 1), "codes are made for one token and one step");
  __shared__ __attribute__((aligned(16))) int8_t codes[kQuant ? 4 : 1][kQuant ? G4_K : 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int team = wave / p.waves, part = wave % p.waves;
  const int64_t n0 = (xcd_block() * p.teams + team) * R;
  const bool live = n0 < p.N;
  const int kb = p.K / 2;           // bytes per row
  // N % 4 == 0: rows come in fours, the last team's second four may be missing (its loads repeat the first)
  const int64_t base = live ? n0 : 0, half = R > 4 && n0 + 4 < p.N ? 4 : 0;
  v4u w[STEPS][R];
  v2u sv[STEPS][R / 4];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k = G4_K * (part + s * p.waves) + 32 * lane;
    const bool ok = live && k < p.K;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      w[s][r] = v4u{0, 0, 0, 0};
      const int64_t row = base + (r & 3) + (r >> 2) * half;
      if (ok) w[s][r] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p.qw + row * kb + (k >> 1)));
    }
#pragma unroll
    for (int q = 0; q < R / 4; ++q) {
      sv[s][q] = v2u{0, 0};
      if (ok) sv[s][q] = *reinterpret_cast<const v2u*>(p.s4 + (int64_t)(k >> 6) * p.N + base + q * half);
    }
  }
  float sx = 0.f;
  if constexpr (kQuant) {
    const int off = G4_K * part + lane_offset(lane), l = lane & 15;
    const float c1 = (l & 1) ? -1.f : 1.f, c2 = (l & 2) ? -1.f : 1.f, c8 = (l & 8) ? -1.f : 1.f;
    float v[2][16], amax = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) load16<__bf16>(p.x + off + 1024 * h, off + 1024 * h < p.K, v[h]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      rotate16(v[h], c1, c2, c8);
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[h][i]));
    }
    amax = wave_max(amax);
    if (lane == 0) red[wave][0] = amax;
    __syncthreads();
    for (int i = 0; i < p.waves; ++i) amax = fmaxf(amax, red[team * p.waves + i][0]);
    __syncthreads();                                    // red is written again below
    amax = fmaxf(amax, 1e-8f);
    const float mul = __fdiv_rn(127.f, amax) * (c1 * c2 * c8);
    sx = __fdiv_rn(amax, 127.f);
    const bool write = blockIdx.x == 0 && team == 0;
    if (write && part == 0 && lane == 0) p.s[0] = sx;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 c = pack_codes16(v[h], mul);
      *reinterpret_cast<uint4*>(codes[wave] + lane_offset(lane) + 1024 * h) = c;
      if (write && off + 1024 * h < p.K) *reinterpret_cast<uint4*>(p.q + off + 1024 * h) = c;
    }
    wave_fence();
  }
  float acc[NV] = {};
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k = G4_K * (part + s * p.waves) + 32 * lane;
    if (k >= p.K) break;
    v4i x[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int8_t* xp = kQuant ? codes[wave] + 32 * lane : p.qx + (int64_t)m * p.K + k;
      x[m][0] = *reinterpret_cast<const v4i*>(xp);
      x[m][1] = *reinterpret_cast<const v4i*>(xp + 16);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t sw = sv[s][r >> 2][(r >> 1) & 1];
      const float sc = __uint_as_float(r & 1 ? sw & 0xffff0000u : sw << 16);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[R * m + r] = __builtin_fmaf((float)dot32_i4(w[s][r], x[m][0], x[m][1]), sc, acc[R * m + r]);
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
  // value `lane` = R m + r: row 2 (upper half of the values) + (second half of those) of red, in order
  const int m = lane / R, r = lane % R;
  const int up = lane >= H, in = lane - up * H, odd = in >= NS;
  const int at = (2 * up + odd) * NS + in - odd * NS;
  if (n0 + r >= p.N) return;
  float a = 0.f;
  for (int v = 0; v < p.waves; ++v) a += red[wave + v][at];
  gemv4_store(p, m, n0 + r, a, kQuant ? sx : p.sx[m]);
}

template <int MT, int R, int STEPS, bool kQuant>
int launch4_mrs(const Gemv4Args& p, hipStream_t st) {
  const int64_t rows_per_wg = (int64_t)R * p.teams;
  const int64_t grid = (p.N + rows_per_wg - 1) / rows_per_wg;
  if (grid > 0x7fffffff) return K2Q_EUNSUPPORTED;
  hipLaunchKernelGGL((gemv_w4_kernel<MT, R, STEPS, kQuant>), dim3((unsigned)grid), dim3(64 * p.waves * p.teams), 0, st, p);
  return k2q_launch_status();
}

template <int MT, int R, bool kQuant = false>
int launch4_mr(Gemv4Args p, hipStream_t st) {
  const int steps = (p.K + G4_K - 1) / G4_K;
  p.waves = steps < 4 ? steps : 4;
  p.teams = 4 / p.waves;
  if constexpr (kQuant) return launch4_mrs<MT, R, 1, true>(p, st);
  else return steps <= 4 ? launch4_mrs<MT, R, 1, false>(p, st) : launch4_mrs<MT, R, 2, false>(p, st);
}

// Which kernel.  A 16-row workgroup a CU needs N >= 4096; below that teams of four rows fill more of the chip.  From
// there on one or two tokens are bound by the weight stream and take eight rows a team (the activation codes are read
// from L1 once for twice the rows), more tokens would be bound by those reads (64 bytes a clock: 3 us a token at 36864 x
// 6144) and take the matrix cores, which read them into one register for 16 rows.  Kernel times, us, on codes that no
// cache holds (teams of 4 / teams of 8 / matrix cores):
//   N x K          M = 1                M = 2                M = 3                M = 8
//   1536 x 6144    3.6 / 3.7 / 5.3      4.0 / 4.1 / 5.5      4.3 / 4.4 / 5.5      5.4 / 5.4 / 5.8
//   6144 x 6144    6.2 / 6.2 / 7.5      6.9 / 7.4 / 7.6      7.6 / 7.6 / 7.8      11.2 / 11.1 / 8.7
//   36864 x 6144   24.3 / 22.4 / 25.6   26.9 / 25.3 / 25.1   29.9 / 25.4 / 25.7   47.5 / 43.4 / 29.7
//   6144 x 16384   13.6 / 12.3 / 14.0   15.1 / 13.3 / 14.2   16.5 / 14.6 / 13.7   24.8 / 20.8 / 15.0
// Below 4096 the first row alone is measured on both; just below it a deep K would be faster on the matrix cores too (eight
// tokens: 4032 x 16384 on teams of four 17.4, 4096 x 16384 on the matrix cores 11.6).
constexpr int64_t G4_WIDE = 4096;

template <int MT>
int launch4_mt(const Gemv4Args& p, hipStream_t st) {
  if (p.N < G4_WIDE) return launch4_mr<MT, 4>(p, st);
  if constexpr (MT <= 2) return launch4_mr<MT, 8>(p, st);
  else return launch4_mfma(p, MT, st);
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
  if (K > 4 * 2 * G4_K) return K2Q_EUNSUPPORTED;
  Gemv4Args p{qx, sx, qw4, sw4, bias, u, lora_b, u ? r : 0, lora_scale, N, (int)K, y, 1, 1, nullptr, nullptr, nullptr};
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

// One token through a linear, its codes not given: one launch instead of two where every workgroup's own rotation hides
// behind its weight loads.  Both launches against one, us: 512 x 512 4.7 / 3.3, 1536 x 6144 6.1 / 5.5, 4096 x 6144
// 7.8 / 7.1, 6144 x 6144 8.7 / 8.7; no gain beyond, at two tokens (1536 x 6144 6.5 / 7.6) or two steps of K (2048 x 16384
// 9.7 / 9.6).
bool k2q_gemv_w4a8_quantizes(int64_t M, int64_t N, int64_t K) { return M == 1 && N < 2 * G4_WIDE && K <= 4 * G4_K; }

// Called by k2q_linear_fwd for such shapes, after the checks of k2q_gemm_w4a8: the codes of x are written to qx, sx.
int k2q_launch_gemv_w4a8_quant(const uint16_t* x, int8_t* qx, float* sx, const uint8_t* qw4, const uint16_t* sw4,
                               const float* bias, int64_t N, int64_t K, uint16_t* y, hipStream_t st) {
  const Gemv4Args p{qx, sx, qw4, sw4, bias, nullptr, nullptr, 0, 0.f, N, (int)K, y, 1, 1,
                    reinterpret_cast<const __bf16*>(x), qx, sx};
  return N < G4_WIDE ? launch4_mr<1, 4, true>(p, st) : launch4_mr<1, 8, true>(p, st);
}
