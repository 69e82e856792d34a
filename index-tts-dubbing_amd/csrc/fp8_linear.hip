// Linear layers in block-scaled e4m3: y = act(Q(x) Q(w)^T + bias) + residual, Q = one power-of-two scale per 128
// consecutive k of a row (fp8.h), both operands.
//
// bf16 outputs: the product of two scaled blocks is 2^(ex + ew) * sum of 128 code products, exactly one
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes both exponents as operands: the scales cost no vector instruction.  Its
// sums are f32, but within one instruction it aligns the 128 products to the largest and cuts what lies more than some
// 13 bits below it (measured on normal data: 1.5e-5 of the result's rms; the bf16 result rounds by 1.7e-3).
// f32 outputs: codes times scale are exact in bf16, and v_mfma_f32_16x16x32_bf16 adds exact products to f32 (measured
// 1.2e-8 of the rms), at half the rate and one conversion per two codes.
#include "fp8.h"

namespace {

using itts::e4m3_inv_scale;
using itts::e4m3_pack4;
using itts::e4m3_prescale;
using itts::e4m3_scale_byte;
using itts::finite_f;

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

constexpr int kMaxK = 1 << 20;
constexpr int kMaxN = 1 << 24;

// ---- quantiser ----------------------------------------------------------------------------------
// 16 lanes per block of 128, 8 values each: one 16-B (bf16) or two 16-B (f32) loads per lane, the block's maximum by
// four DPP steps, 8 bytes out.  VEC: rows are 16-B aligned and the lane's 8 values lie within K; otherwise value by value.
template <typename T>
__device__ __forceinline__ void load_vals(const T* row, int k, int K, bool vec, float (&v)[8]);
template <>
__device__ __forceinline__ void load_vals<float>(const float* row, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(row + k), b = *reinterpret_cast<const f32x4_t*>(row + k + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : 0.f;
  }
}
template <>
__device__ __forceinline__ void load_vals<uint16_t>(const uint16_t* row, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(row + k);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? bf2f(row[k + i]) : 0.f;
  }
}

// codes of this lane's 8 values and the scale byte of its 16-lane block
__device__ __forceinline__ int quant8(const float (&v)[8], u32x2_t& codes) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_f(v[i]) ? fabsf(v[i]) : 0.f);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
  const int byte = e4m3_scale_byte(a);
  const float inv = e4m3_inv_scale(byte);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = e4m3_prescale(v[i], inv);
  codes[0] = e4m3_pack4(q[0], q[1], q[2], q[3]);
  codes[1] = e4m3_pack4(q[4], q[5], q[6], q[7]);
  return byte;
}

template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int K, int kb4,
                                                         bool vec, uint8_t* __restrict__ q, int64_t ldq,
                                                         uint8_t* __restrict__ s, int64_t lds) {
  // one 16-lane group per (row, block); kb4 = blocks rounded up to 4 (scale bytes behind the last block: 127)
  const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  const int l = threadIdx.x & 15;
  const int64_t m = id / kb4;
  const int kb = (int)(id - m * kb4);
  if (m >= M) return;  // whole 16-lane groups leave together; the shuffles stay within a group
  float v[8];
  load_vals(x + m * ldx, kb * 128 + 8 * l, K, vec, v);
  u32x2_t c;
  const int byte = quant8(v, c);
  if (kb * 128 < K) *reinterpret_cast<u32x2_t*>(q + m * ldq + kb * 128 + 8 * l) = c;
  if (l == 0) s[m * lds + kb] = (uint8_t)byte;
}

// ---- product ------------------------------------------------------------------------------------
__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == 1) {
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return 0.5f * v * (1.0f + tanhf(u));
  }
  if (act == 2) return v / (1.0f + expf(-v));
  return v;
}

struct LinearArgs {
  const uint8_t *xq, *xs, *wq, *ws;
  int64_t ldxq, ldxs, ldw, ldws;
  int64_t M;
  int N, KB;
  const float* bias;
  const float* residual;
  int64_t ldr;
  void* y;
  int64_t ldy;
  int act;
  bool out_bf16, vec_out;
};

// 16 consecutive outputs n .. n + 15 of row m: bias, activation, residual, store
__device__ __forceinline__ void store16(const LinearArgs& p, int64_t m, int n, const float (&acc)[16]) {
  if (m >= p.M) return;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = min(n + i, p.N - 1);
    v[i] = apply_act(acc[i] + (p.bias ? p.bias[c] : 0.f), p.act);
    if (p.residual) v[i] += p.residual[m * p.ldr + c];
  }
  if (p.vec_out && n + 16 <= p.N) {
    if (p.out_bf16) {
      u32x4_t* d = reinterpret_cast<u32x4_t*>((uint16_t*)p.y + m * p.ldy + n);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        d[h] = u32x4_t{pack2bf(v[8 * h], v[8 * h + 1]), pack2bf(v[8 * h + 2], v[8 * h + 3]),
                       pack2bf(v[8 * h + 4], v[8 * h + 5]), pack2bf(v[8 * h + 6], v[8 * h + 7])};
    } else {
      f32x4_t* d = reinterpret_cast<f32x4_t*>((float*)p.y + m * p.ldy + n);
#pragma unroll
      for (int h = 0; h < 4; ++h) d[h] = f32x4_t{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    }
  } else {
    for (int i = 0; i < 16; ++i) {
      if (n + i >= p.N) break;
      if (p.out_bf16) ((uint16_t*)p.y)[m * p.ldy + n + i] = f2bf(v[i]);
      else ((float*)p.y)[m * p.ldy + n + i] = v[i];
    }
  }
}

__device__ __forceinline__ i32x8_t frag(const uint8_t* p) {  // bytes p .. +15 and p + 64 .. +79
  const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p), b = *reinterpret_cast<const u32x4_t*>(p + 64);
  return i32x8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// eight codes (two dwords) times their block's scale as bf16: exact but for bf16 denormals
__device__ __forceinline__ bf16x8_t dequant8(int lo, int hi, float scale) {
  u32x4_t w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return __builtin_bit_cast(bf16x8_t, w);
}

// One wave per 16 rows of x and 64 of w, operands straight from global memory.  W is the A operand, so a lane's four
// results are four of W's rows at one row of x; W's rows are dealt to the four A fragments as 16 (r / 4) + 4 j + r % 4
// (fragment j, row r), which makes a lane's 16 results 16 consecutive columns of y, and the four lane groups' 64.
template <bool EXACT>
__global__ __launch_bounds__(256) void fp8_linear_direct_kernel(LinearArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, c = lane >> 4;
  const int n0 = blockIdx.x * 64;
  const int64_t m = ((int64_t)blockIdx.y * 4 + wave) * 16 + r;
  const uint8_t* xr = p.xq + min(m, p.M - 1) * p.ldxq + 16 * c;
  const uint8_t* xsr = p.xs + min(m, p.M - 1) * p.ldxs;
  const uint8_t *wr[4], *wsr[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = min(n0 + 16 * (r >> 2) + 4 * j + (r & 3), p.N - 1);
    wr[j] = p.wq + (int64_t)n * p.ldw + 16 * c;
    wsr[j] = p.ws + (int64_t)n * p.ldws;
  }
  f32x4_t acc[4] = {};
  for (int kb = 0; kb < p.KB; ++kb) {
    const i32x8_t xf = frag(xr + kb * 128);
    const int sx = xsr[kb];
    bf16x8_t xb[4];
    if constexpr (EXACT) {
#pragma unroll
      for (int e = 0; e < 4; ++e) xb[e] = dequant8(xf[2 * e], xf[2 * e + 1], itts::e4m3_scale(sx));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x8_t wf = frag(wr[j] + kb * 128);
      const int sw = wsr[j][kb];
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dequant8(wf[2 * e], wf[2 * e + 1], itts::e4m3_scale(sw)), xb[e],
                                                           acc[j], 0, 0, 0);
      } else {
        acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[j], 0, 0, 0, sw, 0, sx);
      }
    }
  }
  float v[16];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * j + i] = acc[j][i];
  store16(p, m, n0 + 16 * c, v);
}

int launch_quant(const char* fn, const void* x, int64_t ldx, int dtype, int64_t M, int K, uint8_t* q, int64_t ldq,
                 uint8_t* s, int64_t lds, hipStream_t st) {
  const int kb4 = ((K + 127) / 128 + 3) / 4 * 4;
  const int64_t blocks = (M * kb4 + 15) / 16;
  ITTS_REQUIRE(blocks <= 0x7FFFFFFF, fn, "too many rows for one launch");
  const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (dtype == ITTS_F32 ? 4 : 8) == 0;
  if (dtype == ITTS_F32)
    hipLaunchKernelGGL(quant_rows_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, (const float*)x, ldx, M, K, kb4,
                       vec, q, ldq, s, lds);
  else
    hipLaunchKernelGGL(quant_rows_kernel<uint16_t>, dim3((unsigned)blocks), dim3(256), 0, st, (const uint16_t*)x, ldx, M,
                       K, kb4, vec, q, ldq, s, lds);
  return itts::check_launch(fn);
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t code_pitch(int K) { return round_up(K, 128); }
int64_t scale_pitch(int K) { return round_up(round_up(K, 128) / 128, 4); }

}  // namespace

extern "C" int itts_fp8_quant_rows(const void* x, int64_t ldx, int x_dtype, int64_t M, int K, uint8_t* q, int64_t ldq,
                                   uint8_t* s, int64_t lds, void* stream) {
  const char* fn = "itts_fp8_quant_rows";
  ITTS_REQUIRE(x_dtype == ITTS_F32 || x_dtype == ITTS_BF16, fn, "x must be f32 or bf16");
  ITTS_REQUIRE(M >= 0 && K >= 1 && K <= kMaxK && ldx >= K, fn, "bad sizes");
  ITTS_REQUIRE(ldq >= code_pitch(K) && ldq % 16 == 0 && lds >= scale_pitch(K) && lds % 4 == 0, fn,
               "code rows need K rounded up to 128 bytes, scale rows ceil(K / 128) rounded up to 4");
  if (M == 0) return 0;
  ITTS_REQUIRE(x && q && s && ((uintptr_t)q & 15) == 0 && ((uintptr_t)s & 3) == 0, fn, "null or misaligned pointer");
  return launch_quant(fn, x, ldx, x_dtype, M, K, q, ldq, s, lds, itts::as_stream(stream));
}

extern "C" int64_t itts_fp8_linear_workspace_bytes(int64_t M, int N, int K) {
  if (M < 0 || N < 1 || N > kMaxN || K < 1 || K > kMaxK || M > ((int64_t)1 << 40) / code_pitch(K)) return -1;
  return round_up(M * (code_pitch(K) + scale_pitch(K)), 256);
}

extern "C" int itts_fp8_linear(const void* x, int64_t ldx, int x_dtype, int64_t M, int K, const uint8_t* wq, int64_t ldw,
                               const uint8_t* ws, int64_t ldws, int N, const float* bias, int act, const float* residual,
                               int64_t ldr, void* y, int64_t ldy, int out_dtype, void* workspace, void* stream) {
  const char* fn = "itts_fp8_linear";
  ITTS_REQUIRE(x_dtype == ITTS_F32 || x_dtype == ITTS_BF16, fn, "x must be f32 or bf16");
  ITTS_REQUIRE(out_dtype == ITTS_F32 || out_dtype == ITTS_BF16, fn, "y must be f32 or bf16");
  ITTS_REQUIRE(act >= 0 && act <= 2, fn, "act must be 0 (none), 1 (gelu_tanh) or 2 (SiLU)");
  ITTS_REQUIRE(itts_fp8_linear_workspace_bytes(M, N, K) >= 0 && ldx >= K && ldy >= N && (!residual || ldr >= N), fn,
               "bad sizes");
  ITTS_REQUIRE(ldw >= code_pitch(K) && ldw % 16 == 0 && ldws >= scale_pitch(K) && ldws % 4 == 0, fn,
               "weight rows need K rounded up to 128 bytes, scale rows ceil(K / 128) rounded up to 4");
  if (M == 0) return 0;
  ITTS_REQUIRE(x && wq && ws && y && workspace, fn, "null pointer");
  ITTS_REQUIRE((((uintptr_t)wq | (uintptr_t)workspace) & 15) == 0 && ((uintptr_t)ws & 3) == 0, fn, "misaligned pointer");
  ITTS_REQUIRE((M + 63) / 64 <= 65535, fn, "too many rows for one launch");
  uint8_t* xq = (uint8_t*)workspace;
  uint8_t* xs = xq + M * code_pitch(K);
  hipStream_t st = itts::as_stream(stream);
  if (int rc = launch_quant(fn, x, ldx, x_dtype, M, K, xq, code_pitch(K), xs, scale_pitch(K), st)) return rc;
  const int es = out_dtype == ITTS_F32 ? 4 : 2;
  LinearArgs p{xq, xs, wq, ws, code_pitch(K), scale_pitch(K), ldw, ldws, M, N, (K + 127) / 128, bias, residual, ldr, y, ldy,
               act, out_dtype == ITTS_BF16, ((uintptr_t)y & 15) == 0 && (ldy * es) % 16 == 0};
  const dim3 g((N + 63) / 64, (unsigned)((M + 63) / 64));
  if (p.out_bf16) hipLaunchKernelGGL(fp8_linear_direct_kernel<false>, g, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(fp8_linear_direct_kernel<true>, g, dim3(256), 0, st, p);
  return itts::check_launch(fn);
}
