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
// gelu_tanh(v) = v / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3); SiLU(v) = v / (1 + exp(-v)): one exp2 and one
// reciprocal each (both within about an ulp) instead of tanhf's branches, which cost more than the product did
__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == 0) return v;
  constexpr float kLog2e = 1.4426950408889634f, kA = -2.f * 0.7978845608028654f * kLog2e;
  const float e = act == 1 ? v * fmaf(kA * 0.044715f, v * v, kA) : -kLog2e * v;
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e));
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

// 16 consecutive outputs n .. n + 15 of row m (bias added): activation, residual, store
__device__ __forceinline__ void store16(const LinearArgs& p, int64_t m, int n, float (&v)[16]) {
  if (m >= p.M) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] = apply_act(v[i], p.act);
    if (p.residual) v[i] += p.residual[m * p.ldr + min(n + i, p.N - 1)];
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

// ---- tiles ----
// BM x BN outputs per workgroup in waves of WM x WN, k in steps of one block.  A step's rows (128 bytes each) go from
// global memory to LDS by DMA, 1 KB per wave instruction (8 whole rows), two steps in turn: step i + 1 is requested before
// step i's products and waited for after them.  16-B slot s of LDS row i holds chunk s ^ (i / 2) % 8, so the 16 rows of a
// fragment read lie on distinct banks; the DMA writes lane by lane, so each lane fetches the chunk that belongs where it
// writes.  W is the A operand: a lane's results are W rows at one row of x.  The 64 W rows of a wave's four fragments are
// dealt as 16 (r / 4) + 4 j + r % 4 (fragment j, row r), which makes a lane's 16 results 16 consecutive columns of y and
// the four lane groups' 64: whole lines are written without going through LDS.
typedef __attribute__((address_space(3))) void lds_void;

template <bool EXACT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void fp8_linear_tile_kernel(LinearArgs p) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN;
  constexpr int FM = WM / 16, FN = WN / 16;
  constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;  // DMA instructions per wave and step
  static_assert(WN % 64 == 0 && XI * 8 * NW == BM && WI * 8 * NW == BN, "whole instructions, whole groups of 64 columns");
  // separate arrays: the compiler then sees that reads of one step do not wait for the DMA into the other
  __shared__ __attribute__((aligned(1024))) uint8_t sx0[BM * 128], sx1[BM * 128], sw0[BN * 128], sw1[BN * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4;
  const int wm = (wave / NWN) * WM, wn = (wave % NWN) * WN;
  // consecutive tiles (columns fastest) on one XCD: they share rows of x and all of w in its L2
  const int ntn = (p.N + BN - 1) / BN;
  const int nblk = gridDim.x, q8 = nblk / 8, r8 = nblk % 8;
  const int xcd = blockIdx.x % 8, lid = xcd * q8 + min(xcd, r8) + blockIdx.x / 8;
  const int64_t m0 = (int64_t)(lid / ntn) * BM;
  const int n0 = (lid % ntn) * BN;

  const int dr = lane >> 3, ds = lane & 7;
  uint32_t xoff[XI], woff[WI];
  const uint8_t* xbase = p.xq + m0 * p.ldxq;
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = 8 * (wave * XI + i) + dr;
    const int64_t left = p.M - 1 - m0;
    xoff[i] = (uint32_t)(row < left ? row : left) * (uint32_t)p.ldxq + 16 * (ds ^ (row >> 1 & 7));
  }
  const uint8_t* wbase = p.wq + (int64_t)n0 * p.ldw;
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    const int row = 8 * (wave * WI + i) + dr;
    const int n = (row & ~63) + 16 * (row >> 2 & 3) + 4 * (row >> 4 & 3) + (row & 3);
    woff[i] = (uint32_t)min(n, p.N - 1 - n0) * (uint32_t)p.ldw + 16 * (ds ^ (row >> 1 & 7));
  }
  auto issue = [&](int kb, uint8_t* X, uint8_t* W) {
#pragma unroll
    for (int i = 0; i < XI; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(xbase + (int64_t)kb * 128 + xoff[i]),
                                       (lds_void*)(X + 1024 * (wave * XI + i)), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < WI; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(wbase + (int64_t)kb * 128 + woff[i]),
                                       (lds_void*)(W + 1024 * (wave * WI + i)), 16, 0, 0);
  };
  // scale bytes of the lane's rows, four blocks to a dword
  const uint8_t *xsr[FM], *wsr[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + wm + 16 * i + r;
    xsr[i] = p.xs + (m < p.M ? m : p.M - 1) * p.ldxs;
  }
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int n = n0 + wn + 64 * (j >> 2) + 16 * (r >> 2) + 4 * (j & 3) + (r & 3);
    wsr[j] = p.ws + (int64_t)min(n, p.N - 1) * p.ldws;
  }
  uint32_t xsc[FM], wsc[FN];
  auto scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < FM; ++i) xsc[i] = *reinterpret_cast<const uint32_t*>(xsr[i] + kb);
#pragma unroll
    for (int j = 0; j < FN; ++j) wsc[j] = *reinterpret_cast<const uint32_t*>(wsr[j] + kb);
  };

  f32x4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int a0 = r * 128 + ((c ^ (r >> 1 & 7)) << 4), a1 = r * 128 + (((4 + c) ^ (r >> 1 & 7)) << 4);
  auto read = [&](const uint8_t* s, int row) -> i32x8_t {
    const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(s + row * 128 + a0), hi = *reinterpret_cast<const u32x4_t*>(s + row * 128 + a1);
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  auto compute = [&](const uint8_t* X, const uint8_t* W) {
    if constexpr (EXACT) {
      bf16x8_t wb[FN][4];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const i32x8_t f = read(W, wn + 16 * j);
        const float s = __uint_as_float((wsc[j] & 0xFF) << 23);
#pragma unroll
        for (int e = 0; e < 4; ++e) wb[j][e] = dequant8(f[2 * e], f[2 * e + 1], s);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const i32x8_t f = read(X, wm + 16 * i);
        const float s = __uint_as_float((xsc[i] & 0xFF) << 23);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bf16x8_t xb = dequant8(f[2 * e], f[2 * e + 1], s);
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j][e], xb, acc[i][j], 0, 0, 0);
        }
      }
    } else {
      i32x8_t wf[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) wf[j] = read(W, wn + 16 * j);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const i32x8_t xf = read(X, wm + 16 * i);
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf, acc[i][j], 0, 0, 0, wsc[j], 0, xsc[i]);
      }
    }
  };
  auto step = [&](int kb, uint8_t* X, uint8_t* W, uint8_t* nextX, uint8_t* nextW) {
    // this wave's part of the step has landed and its reads of the other slot are done; after the barrier everyone's
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kb + 1 < p.KB) issue(kb + 1, nextX, nextW);
    compute(X, W);
    if (((kb + 1) & 3) == 0 && kb + 1 < p.KB) {
      scales(kb + 1);
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) xsc[i] >>= 8;
#pragma unroll
      for (int j = 0; j < FN; ++j) wsc[j] >>= 8;
    }
  };
  issue(0, sx0, sw0);
  scales(0);
  for (int kb = 0; kb < p.KB; kb += 2) {
    step(kb, sx0, sw0, sx1, sw1);
    if (kb + 1 < p.KB) step(kb + 1, sx1, sw1, sx0, sw0);
  }
#pragma unroll
  for (int g = 0; g < FN / 4; ++g) {
    const int n = n0 + wn + 64 * g + 16 * c;
    float bias[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) bias[i] = p.bias ? p.bias[min(n + i, p.N - 1)] : 0.f;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = acc[i][4 * g + j][e] + bias[4 * j + e];
      store16(p, m0 + wm + 16 * i + r, n, v);
    }
  }
}

// ---- few rows ----
// 16 columns of y and MT x 16 rows per workgroup; its eight waves take the blocks of k in turn and add their parts in LDS.
// x is quantised on the way (a lane holds 32 of a row's 128 values; four lanes share the block), so there is one launch
// and no workspace; w's fragments come straight from global memory: with few rows the bytes of w are the cost.
constexpr int kFewWaves = 8;

template <typename T>
__device__ __forceinline__ void load16(const T* row, int k, int K, bool vec, float (&v)[16]) {
  float h[8];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    load_vals(row, k + 8 * g, K, vec, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * g + i] = h[i];
  }
}

template <bool EXACT, typename T, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void fp8_linear_few_kernel(LinearArgs p, const T* __restrict__ x, int64_t ldx, int K, bool vec) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const uint8_t* wr = p.wq + (int64_t)min(n0 + r, p.N - 1) * p.ldw + 16 * c;
  const uint8_t* wsr = p.ws + (int64_t)min(n0 + r, p.N - 1) * p.ldws;
  const T* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r;
    xr[t] = x + (m < p.M ? m : p.M - 1) * ldx;
  }
  f32x4_t acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < p.KB; kb += kFewWaves) {
    const i32x8_t wf = frag(wr + kb * 128);
    const int sw = wsr[kb];
    float v[MT][2][16];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int g = 0; g < 2; ++g) load16(xr[t], 128 * kb + 64 * g + 16 * c, K, vec, v[t][g]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float a = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 16; ++i) a = fmaxf(a, finite_f(v[t][g][i]) ? fabsf(v[t][g][i]) : 0.f);
      a = fmaxf(a, __shfl_xor(a, 16, 64));
      a = fmaxf(a, __shfl_xor(a, 32, 64));
      const int sx = e4m3_scale_byte(a);
      const float inv = e4m3_inv_scale(sx);
      i32x8_t xf;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          xf[4 * g + i] = (int)e4m3_pack4(e4m3_prescale(v[t][g][4 * i], inv), e4m3_prescale(v[t][g][4 * i + 1], inv),
                                          e4m3_prescale(v[t][g][4 * i + 2], inv), e4m3_prescale(v[t][g][4 * i + 3], inv));
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dequant8(wf[2 * e], wf[2 * e + 1], itts::e4m3_scale(sw)),
                                                           dequant8(xf[2 * e], xf[2 * e + 1], itts::e4m3_scale(sx)), acc[t], 0, 0, 0);
      } else {
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[t], 0, 0, 0, sw, 0, sx);
      }
    }
  }
  __shared__ f32x4_t part[kFewWaves][MT][64];
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // 16 MT rows x 16 columns over the threads, columns fastest
  for (int i = threadIdx.x; i < MT * 256; i += 64 * kFewWaves) {
    const int row = i >> 4, col = i & 15;
    const int t = row >> 4, src = (col >> 2) * 16 + (row & 15);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v += part[w][t][src][col & 3];
    const int64_t m = m0 + row;
    const int n = n0 + col;
    if (m < p.M && n < p.N) {
      v = apply_act(v + (p.bias ? p.bias[n] : 0.f), p.act);
      if (p.residual) v += p.residual[m * p.ldr + n];
      if (p.out_bf16) ((uint16_t*)p.y)[m * p.ldy + n] = f2bf(v);
      else ((float*)p.y)[m * p.ldy + n] = v;
    }
  }
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

#ifndef FEWM
#define FEWM 256
#endif
bool few_rows(int64_t M, int N) { return M <= FEWM; }

template <bool EXACT, int BM, int BN, int WM, int WN>
void launch_tile(const LinearArgs& p, hipStream_t st) {
  const int64_t g = ((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  hipLaunchKernelGGL((fp8_linear_tile_kernel<EXACT, BM, BN, WM, WN>), dim3((unsigned)g), dim3(64 * (BM / WM) * (BN / WN)), 0, st, p);
}
#ifndef VAR
#define VAR 0
#endif
template <bool EXACT>
void launch_tiles(const LinearArgs& p, hipStream_t st) {
  if (VAR == 0) launch_tile<EXACT, 256, 256, 128, 64>(p, st);
  else if (VAR == 1) launch_tile<EXACT, 128, 128, 64, 64>(p, st);
  else if (VAR == 2) launch_tile<EXACT, 128, 256, 64, 64>(p, st);
  else if (VAR == 3) launch_tile<EXACT, 256, 128, 128, 64>(p, st);
  else if (VAR == 4) launch_tile<EXACT, 64, 128, 32, 64>(p, st);
}
template <typename T>
void launch_few(const T* x, int64_t ldx, int K, bool vec, const LinearArgs& p, hipStream_t st) {
  const int mt = p.M <= 16 ? 1 : 2;
  const dim3 g((p.N + 15) / 16, (unsigned)((p.M + 16 * mt - 1) / (16 * mt))), b(64 * kFewWaves);
  if (p.out_bf16) {
    if (mt == 1) hipLaunchKernelGGL((fp8_linear_few_kernel<false, T, 1>), g, b, 0, st, p, x, ldx, K, vec);
    else hipLaunchKernelGGL((fp8_linear_few_kernel<false, T, 2>), g, b, 0, st, p, x, ldx, K, vec);
  } else {
    if (mt == 1) hipLaunchKernelGGL((fp8_linear_few_kernel<true, T, 1>), g, b, 0, st, p, x, ldx, K, vec);
    else hipLaunchKernelGGL((fp8_linear_few_kernel<true, T, 2>), g, b, 0, st, p, x, ldx, K, vec);
  }
}

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
  const int es = out_dtype == ITTS_F32 ? 4 : 2;
  LinearArgs p{xq, xs, wq, ws, code_pitch(K), scale_pitch(K), ldw, ldws, M, N, (K + 127) / 128, bias, residual, ldr, y, ldy,
               act, out_dtype == ITTS_BF16, ((uintptr_t)y & 15) == 0 && (ldy * es) % 16 == 0};
  if (few_rows(M, N)) {
    const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (x_dtype == ITTS_F32 ? 4 : 8) == 0;
    if (x_dtype == ITTS_F32) launch_few((const float*)x, ldx, K, vec, p, st);
    else launch_few((const uint16_t*)x, ldx, K, vec, p, st);
    return itts::check_launch(fn);
  }
  if (int rc = launch_quant(fn, x, ldx, x_dtype, M, K, xq, code_pitch(K), xs, scale_pitch(K), st)) return rc;
  if (p.out_bf16) launch_tiles<false>(p, st);
  else launch_tiles<true>(p, st);
  return itts::check_launch(fn);
}
