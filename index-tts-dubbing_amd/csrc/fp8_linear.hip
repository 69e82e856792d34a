// Linear layers in block-scaled e4m3: y = act(Q(x) Q(w)^T + bias) + residual, Q = one power-of-two scale per 128
// consecutive k of a row (fp8.h), both operands.
//
// bf16 outputs: the product of two scaled blocks is 2^(ex + ew) * sum of 128 code products, exactly one
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes both exponents as operands: the scales cost no vector instruction.  Its
// sums are f32, but within one instruction it aligns the 128 products to the largest and cuts what lies more than some
// 13 bits below it (measured on normal data: 1.5e-5 of the result's rms; the bf16 result rounds by 1.7e-3).
// f32 outputs: codes times scale are exact in bf16, and v_mfma_f32_16x16x32_bf16 adds exact products to f32 (measured
// 1.2e-8 of the rms), at half the rate and one conversion per two codes.
//
// Times in this file are of whole calls in a replayed graph, the quantising pass included, bf16 results without an activation unless
// said.  What bounds it: few rows the launch and the trip to memory (1 x 1024 x 4096: 3.4 us for 4.3 MB, 96 x 4096 x 1024: 8.3);
// large sizes the matrix unit (8192 x 8192 x 8192: 443 us = 2.48 PFLOP/s) less the tiles' first fetch and last store (14400 x 1024 x
// 4096: 91 us, with GELU 107 = 1.13 PFLOP/s: four turns of 256 tiles of eight steps each).
#include <type_traits>

#include "fp8.h"
#include "fp8_rows.h"

namespace {

using itts::e4m3_pack4;

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;

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
__device__ __forceinline__ int quant8(float (&v)[8], u32x2_t& codes) {
  auto reduce = [](uint32_t m) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    return m;
  };
  const int byte = itts::e4m3_scaled(v, reduce(itts::max_bits(v)), reduce);
  codes[0] = e4m3_pack4(v[0], v[1], v[2], v[3]);
  codes[1] = e4m3_pack4(v[4], v[5], v[6], v[7]);
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
template <int ACT>
__device__ __forceinline__ float apply_act(float v) {
  if constexpr (ACT == 0) return v;
  constexpr float kLog2e = 1.4426950408889634f, kA = -2.f * 0.7978845608028654f * kLog2e;
  const float e = ACT == 1 ? v * fmaf(kA * 0.044715f, v * v, kA) : -kLog2e * v;
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

// ---- epilogue of the tile kernels ----
// Activation and residual are compile-time: with a test per value (and the wait for an optional load beside each store) the
// epilogue of a 256 x 256 tile took 22 us, more than its products over k = 1024.
template <int WN>
constexpr int kPitch = WN + 4;  // floats: rows r and r + 1 four banks apart
template <int WN>
constexpr int kBand = 2 * (WN / 64) * 16 * (64 * 4 + 16);  // bytes of a wave's part of the LDS; 16 rows of kPitch floats fit too

// A sum as a vector register.  AGPR: it stays in its accumulator register until here (left to itself the compiler copies a
// wave's 256 sums at once, and spills).
template <bool AGPR>
__device__ __forceinline__ float sum_of(float a) {
  if constexpr (!AGPR) return a;
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}
template <bool AGPR>
__device__ __forceinline__ f32x4_t sums_of(f32x4_t a) {
  return f32x4_t{sum_of<AGPR>(a[0]), sum_of<AGPR>(a[1]), sum_of<AGPR>(a[2]), sum_of<AGPR>(a[3])};
}

// N a multiple of 16 and aligned rows: a lane has 16 neighbouring results of a row.  They go through the wave's own part of
// the LDS in their final type, so that neighbouring lanes store neighbouring 16 bytes (stored from where they are, neighbouring
// lanes on neighbouring rows, f32 results of 3500 x 512 x 3600 took 36 us instead of 30).  A row's residual is
// requested before the stores of the row before (a load waits for the stores before it).
template <bool BF16, bool AGPR, int ACT, bool RES, int FM, int FN>
__device__ __forceinline__ void store_direct(const LinearArgs& p, f32x4_t (&acc)[FM][FN], uint8_t* band, int64_t m0, int n0) {
  constexpr int G = FN / 4, ES = BF16 ? 2 : 4;
  constexpr int PITCH = 64 * ES + 16, CHUNKS = 4 * ES;  // a row's 64 results in the LDS; 16-B pieces of them
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int left = (int)(p.M - m0 < 16 * FM ? p.M - m0 : 16 * FM);  // rows of the wave's tile
  f32x4_t bias[G][4], res[RES ? G : 1][4];
  bool in[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int n = n0 + 64 * g + 16 * c;
    in[g] = n < p.N;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      bias[g][i] = p.bias && in[g] ? *reinterpret_cast<const f32x4_t*>(p.bias + n + 4 * i) : f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto load_res = [&](int i) {
    if constexpr (RES) {
      const int row = 16 * i + r;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (in[g] && row < left) {
          const float* src = p.residual + (m0 + row) * p.ldr + n0 + 64 * g + 16 * c;
#pragma unroll
          for (int j = 0; j < 4; ++j) res[g][j] = *reinterpret_cast<const f32x4_t*>(src + 4 * j);
        }
    }
  };
  load_res(0);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    __builtin_amdgcn_sched_barrier(0);  // row by row: the sums leave the accumulator registers as they are needed
    const int row = 16 * i + r;
    f32x4_t v[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[g][j][e] = apply_act<ACT>(sum_of<AGPR>(acc[i][4 * g + j][e]) + bias[g][j][e]);
        if constexpr (RES) v[g][j] = v[g][j] + res[g][j];
      }
    if (i + 1 < FM) load_res(i + 1);
    uint8_t* const buf = band + (i & 1) * (G * 16 * PITCH);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int k = 0; k < ES; ++k) {
        u32x4_t w;
        if constexpr (BF16)
          w = u32x4_t{pack2bf(v[g][2 * k][0], v[g][2 * k][1]), pack2bf(v[g][2 * k][2], v[g][2 * k][3]),
                      pack2bf(v[g][2 * k + 1][0], v[g][2 * k + 1][1]), pack2bf(v[g][2 * k + 1][2], v[g][2 * k + 1][3])};
        else
          w = __builtin_bit_cast(u32x4_t, v[g][k]);
        *reinterpret_cast<u32x4_t*>(buf + (16 * g + r) * PITCH + 16 * ES * c + 16 * k) = w;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the band is this wave's own: no barrier
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int k = 0; k < ES; ++k) {
        const int at = 64 / CHUNKS * k + lane / CHUNKS, chunk = lane % CHUNKS;
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(buf + (16 * g + at) * PITCH + 16 * chunk);
        const int col = n0 + 64 * g + chunk * (16 / ES);
        if (16 * i + at < left && col < p.N)
          *reinterpret_cast<u32x4_t*>((uint8_t*)p.y + ((m0 + 16 * i + at) * p.ldy + col) * ES) = w;
      }
  }
}

// Any N and pitch: bands of 16 rows go through the wave's own part of the LDS, then lanes walk the rows with neighbouring
// columns, so that whole lines are written all the same (stored from the registers, 1337 x 1000 x 8194 took 44 us more).
template <bool BF16, bool AGPR, int ACT, bool RES, int FM, int FN>
__device__ __forceinline__ void store_banded(const LinearArgs& p, f32x4_t (&acc)[FM][FN], float* band, int64_t m0, int n0) {
  constexpr int WN = 16 * FN, CI = WN / 64;
  const int lane = threadIdx.x & 63, fr = lane & 15, fc = lane >> 4;
  const int left = (int)(p.M - m0 < 16 * FM ? p.M - m0 : 16 * FM);
  float bias[CI];
#pragma unroll
  for (int k = 0; k < CI; ++k) bias[k] = p.bias ? p.bias[min(n0 + lane + 64 * k, p.N - 1)] : 0.f;
#pragma unroll
  for (int b = 0; b < FM; ++b) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<f32x4_t*>(&band[fr * kPitch<WN> + 64 * (j >> 2) + 16 * fc + 4 * (j & 3)]) = sums_of<AGPR>(acc[b][j]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the band is this wave's own: no barrier
#pragma unroll 1
    for (int t = 0; t < min(16, left - 16 * b); t += 4) {  // four rows a turn; the band's last rows may be none of M's
      float v[4][CI];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < CI; ++k) {
          v[u][k] = apply_act<ACT>(band[(t + u) * kPitch<WN> + lane + 64 * k] + bias[k]);
          if constexpr (RES) {
            const int row = min(16 * b + t + u, left - 1), col = min(n0 + lane + 64 * k, p.N - 1);
            v[u][k] += p.residual[(m0 + row) * p.ldr + col];
          }
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < CI; ++k) {
          const int row = 16 * b + t + u, col = n0 + lane + 64 * k;
          if (row < left && col < p.N) {
            if constexpr (BF16) ((uint16_t*)p.y)[(m0 + row) * p.ldy + col] = f2bf(v[u][k]);
            else ((float*)p.y)[(m0 + row) * p.ldy + col] = v[u][k];
          }
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}
template <bool BF16, bool AGPR, int ACT, int FM, int FN>
__device__ __forceinline__ void store_tile(const LinearArgs& p, f32x4_t (&acc)[FM][FN], float* band, int64_t m0, int n0) {
  if (m0 >= p.M) return;
  if (p.vec_out) {
    if (p.residual) store_direct<BF16, AGPR, ACT, true>(p, acc, (uint8_t*)band, m0, n0);
    else store_direct<BF16, AGPR, ACT, false>(p, acc, (uint8_t*)band, m0, n0);
  } else {
    if (p.residual) store_banded<BF16, AGPR, ACT, true>(p, acc, band, m0, n0);
    else store_banded<BF16, AGPR, ACT, false>(p, acc, band, m0, n0);
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
// the four lane groups' 64.
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kScaleBlocks = 64;  // blocks of k whose scales the LDS holds at once

template <bool EXACT, int ACT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void fp8_linear_tile_kernel(LinearArgs p) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN;
  constexpr int FM = WM / 16, FN = WN / 16;
  constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;  // DMA instructions per wave and step
  static_assert(WN % 64 == 0 && XI * 8 * NW == BM && WI * 8 * NW == BN, "whole instructions, whole groups of 64 columns");
  // separate arrays: the compiler then sees that reads of one step do not wait for the DMA into the other
  __shared__ __attribute__((aligned(1024))) uint8_t sx0[BM * 128], sx1[BM * 128], sw0[BN * 128], sw1[BN * 128];
  __shared__ __attribute__((aligned(16))) uint8_t ss[(BM + BN) * kScaleBlocks];
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
    woff[i] = (uint32_t)itts::fetched_row(row, p.N - 1 - n0) * (uint32_t)p.ldw + 16 * (ds ^ (row >> 1 & 7));
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
  // The scale bytes of kScaleBlocks blocks, x's rows then w's in the order of the LDS rows; dword d of row i at
  // d ^ (i / 4) % 16, so that a fragment's 16 rows lie on distinct banks.  (Fetched from memory as they are needed, 16 rows
  // far apart at a time, they cost as much as the products.)
  auto stage_scales = [&](int kb) {
    for (int row = threadIdx.x; row < BM + BN; row += 64 * NW) {
      const uint8_t* src;
      if (row < BM) {
        const int64_t left = p.M - 1 - m0;
        src = p.xs + (m0 + (row < left ? row : left)) * p.ldxs;
      } else {
        src = p.ws + (int64_t)(n0 + itts::fetched_row(row - BM, p.N - 1 - n0)) * p.ldws;
      }
      for (int d = 0; d < min(kScaleBlocks, p.KB - kb + 3) >> 2; ++d)
        ((uint32_t*)ss)[row * (kScaleBlocks / 4) + (d ^ (row >> 2 & 15))] = ((const uint32_t*)(src + kb))[d];
    }
  };
  uint32_t xsc[FM], wsc[FN];
  auto scales = [&](int kb) {  // four blocks' bytes of the lane's rows
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = wm + 16 * i + r;
      xsc[i] = ((const uint32_t*)ss)[row * (kScaleBlocks / 4) + ((kb >> 2 & 15) ^ (row >> 2 & 15))];
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int row = BM + wn + 16 * j + r;
      wsc[j] = ((const uint32_t*)ss)[row * (kScaleBlocks / 4) + ((kb >> 2 & 15) ^ (row >> 2 & 15))];
    }
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
    if ((kb & (kScaleBlocks - 1)) == 0 && kb) {  // everyone has read the scales before
      stage_scales(kb);
      __syncthreads();
    }
    if (kb + 1 < p.KB) issue(kb + 1, nextX, nextW);
    if ((kb & 3) == 0) {
      scales(kb);
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) xsc[i] >>= 8;
#pragma unroll
      for (int j = 0; j < FN; ++j) wsc[j] >>= 8;
    }
    compute(X, W);
  };
  issue(0, sx0, sw0);
  stage_scales(0);
  for (int kb = 0; kb < p.KB; kb += 2) {
    step(kb, sx0, sw0, sx1, sw1);
    if (kb + 1 < p.KB) step(kb + 1, sx1, sw1, sx0, sw0);
  }
  __syncthreads();  // the steps' LDS becomes the waves' bands
  static_assert((NW + 3) / 4 * kBand<WN> <= (BM < BN ? BM : BN) * 128, "the bands fit");
  uint8_t* const part = (wave & 2) ? (wave & 1 ? sw1 : sw0) : (wave & 1 ? sx1 : sx0);
  store_tile<!EXACT, false, ACT>(p, acc, (float*)(part + (wave >> 2) * kBand<WN>), m0 + wm, n0 + wn);
}

// ---- large tiles ----
// 256 x 256 outputs in four waves of 128 x 128, one per SIMD: a wave's 16 fragments feed 64 products, so a step costs the
// LDS 1536 clocks (128 KB read, 64 KB written by the DMA, 128 B a clock) against the matrix unit's 2048; with waves of
// 128 x 64 both take 2048.  One wave per SIMD has to overlap by itself, so a step is straight-line code in rows of eight
// products with the fragments of later rows requested between them.  The step's one barrier stands before its last three
// rows, when all of the step's fragments are in registers: behind it the step's LDS is free for the DMA of the step after
// next, which has a whole step to land, and the next step's fragments are read under the last rows' products.
// Rows of x behind M are read from the workspace's padding, for rows of w behind N the last row again (their results are not
// stored): every address lies within its buffer, none is left to the buffer resource's bounds.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const T* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, (uint32_t)(bytes < 0xFFFFFFFFll ? bytes : 0xFFFFFFFFll), 0x00020000);
}

// The 256 accumulator registers of a wave are all sums.  As a builtin the compiler moves a third of them on every turn of the
// loop and spills; as assembly they stay.  A sum is next touched 64 products later, operands come from the LDS (the
// compiler waits for those), and what the vector unit writes or reads next to a product is kept apart by s_nop.  That the compiler
// adds no vector instruction of its own there -- it knows of no wait that these products need -- is checked in the assembly when this
// file is built.  (An s_nop before every product would do as well: 8192 x 8192 x 8192 443 -> 451 us.)
template <int S>  // which byte of the scale registers
__device__ __forceinline__ void product_agpr(f32x4_t& acc, const i32x8_t& w, const i32x8_t& x, uint32_t ws, uint32_t xs) {
  if constexpr (S == 0)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
  else
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
}
// the matrix unit has finished and the vector unit's writes have landed, for every sum
template <int F>
__device__ __forceinline__ void settle(f32x4_t (&acc)[F][F]) {
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) asm volatile("" : "+a"(acc[i][j]));
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) asm volatile("" : "+a"(acc[i][j]));
}

template <int ACT>
__global__ __launch_bounds__(256, 1) void fp8_linear_large_kernel(LinearArgs p) {
  constexpr int F = 8;
  __shared__ __attribute__((aligned(1024))) uint8_t sx0[256 * 128], sx1[256 * 128], sw0[256 * 128], sw1[256 * 128];
  __shared__ __attribute__((aligned(16))) uint8_t ss[512 * kScaleBlocks];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4;
  const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;
  const int ntn = (p.N + 255) / 256;
  const int nblk = gridDim.x, q8 = nblk / 8, r8 = nblk % 8;
  const int xcd = blockIdx.x % 8, lid = xcd * q8 + min(xcd, r8) + blockIdx.x / 8;
  const int64_t m0 = (int64_t)(lid / ntn) * 256;
  const int n0 = (lid % ntn) * 256;

  // DMA instruction i of a wave fills LDS rows 64 wave + 8 i + dr; the swizzle of its lanes' chunks depends on i's parity alone
  const int dr = lane >> 3, ds = lane & 7;
  const int ldx = (int)p.ldxq, ldw = (int)p.ldw;
  const auto xrs = buffer_of(p.xq + m0 * ldx, (int64_t)256 * ldx);
  const auto wrs = buffer_of(p.wq + (int64_t)n0 * ldw, (int64_t)(p.N - n0) * ldw);
  uint32_t xoff[2], woff[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int chunk = 16 * (ds ^ (4 * (i & 1) + (dr >> 1)));
    if (i < 2) xoff[i] = dr * ldx + chunk;
    woff[i] = itts::fetched_row(64 * wave + 8 * i + dr, p.N - 1 - n0) * ldw + chunk;
  }
  // x's and w's rows of a step: eight instructions each
  auto issue_x = [&](int i, int kb, uint8_t* X) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xrs, (lds_void*)(X + 1024 * (wave * F + i)), 16, xoff[i & 1],
                                             (64 * wave + 8 * i) * ldx + 128 * kb, 0, 0);
  };
  auto issue_w = [&](int i, int kb, uint8_t* W) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs, (lds_void*)(W + 1024 * (wave * F + i)), 16, woff[i], 128 * kb, 0, 0);
  };
  // All of the tile's scale bytes, x's rows then w's in the order of its LDS rows; dword d of row i at d ^ (i / 4) % 16, so
  // that a fragment's 16 rows lie on distinct banks.  (Fetched from memory as they are needed, 16 rows far apart at a time,
  // they cost as much as the products.)
  {
    const int row = threadIdx.x, swz = row >> 2 & 15;
    const int64_t left = p.M - 1 - m0;
    const uint32_t* xs = (const uint32_t*)(p.xs + (m0 + (row < left ? row : left)) * p.ldxs);
    const uint32_t* ws = (const uint32_t*)(p.ws + (int64_t)(n0 + itts::fetched_row(row, p.N - 1 - n0)) * p.ldws);
    for (int d = 0; d < (p.KB + 3) >> 2; ++d) {
      ((uint32_t*)ss)[row * (kScaleBlocks / 4) + (d ^ swz)] = xs[d];
      ((uint32_t*)ss)[(256 + row) * (kScaleBlocks / 4) + (d ^ swz)] = ws[d];
    }
  }
  uint32_t xsc[F], wsc[F];  // two blocks' bytes of the lane's rows
  auto scales = [&](int kb, uint32_t (&x)[F], uint32_t (&w)[F]) {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      // rows wm + 16 i + r and wn + 16 i + r: row / 4 % 16 = (4 i + r / 4) % 16
      const int at = 4 * ((kb >> 2) ^ ((4 * i + (r >> 2)) & 15)) + (kb & 2);
      x[i] = *reinterpret_cast<const uint16_t*>(ss + (wm + 16 * i + r) * kScaleBlocks + at);
      w[i] = *reinterpret_cast<const uint16_t*>(ss + (256 + wn + 16 * i + r) * kScaleBlocks + at);
    }
  };
  f32x4_t acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int a0 = r * 128 + ((c ^ (r >> 1 & 7)) << 4), a1 = r * 128 + (((4 + c) ^ (r >> 1 & 7)) << 4);
  auto read = [&](const uint8_t* s, int row) -> i32x8_t {
    const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(s + row * 128 + a0), hi = *reinterpret_cast<const u32x4_t*>(s + row * 128 + a1);
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  i32x8_t w[F], xf[4];
  // one step (S: byte of the scales): W's fragments in w, row 0's in xf[0]; leaves the next step's there
  auto step = [&](auto tag, int kb, uint8_t* X, uint8_t* W, uint8_t* nextX, uint8_t* nextW) {
    constexpr int S = decltype(tag)::value;
    auto product = [&](int i, int j) { product_agpr<S>(acc[i][j], w[j], xf[i & 3], wsc[j], xsc[i]); };
    const int next = min(kb + 1, p.KB - 1), after = min(kb + 2, p.KB - 1);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      if (i == 0) xf[1] = read(X, wm + 16);
      if (i < 4) xf[(i + 2) & 3] = read(X, wm + 16 * (i + 2));
      if (i == 4) {
        xf[2] = read(X, wm + 16 * 6);
        xf[3] = read(X, wm + 16 * 7);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < F; ++j) {
        product(i, j);
        if (i < 2 && (j & 1)) {  // the rest of the next step's DMA, a few products apart: a burst holds up the products
          issue_w(4 * i + (j >> 1), next, nextW);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // this step's fragments are here, this wave's part of the next has landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    xf[0] = read(nextX, wm);
#pragma unroll
    for (int j = 0; j < F; ++j) {
      product(5, j);
      product(6, j);
      product(7, j);
      w[j] = read(nextW, wn + 16 * j);
      issue_x(j, after, X);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int i = 0; i < F; ++i) {
    issue_x(i, 0, sx0);
    issue_w(i, 0, sw0);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  scales(0, xsc, wsc);
#pragma unroll
  for (int j = 0; j < F; ++j) w[j] = read(sw0, wn + 16 * j);
  xf[0] = read(sx0, wm);
#pragma unroll
  for (int i = 0; i < F; ++i) issue_x(i, min(1, p.KB - 1), sx1);
  settle(acc);
  using std::integral_constant;
  int kb = 0;
  for (; kb + 2 <= p.KB; kb += 2) {
    uint32_t xn[F], wnx[F];
    scales(min(kb + 2, (p.KB - 1) & ~1), xn, wnx);
    step(integral_constant<int, 0>{}, kb, sx0, sw0, sx1, sw1);
    step(integral_constant<int, 1>{}, kb + 1, sx1, sw1, sx0, sw0);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      xsc[i] = xn[i];
      wsc[i] = wnx[i];
    }
#pragma unroll
    for (int i = 0; i < F; ++i) asm volatile("" : "+v"(xsc[i]), "+v"(wsc[i]));
    asm volatile("s_nop 7" ::: "memory");
  }
  if (kb < p.KB) step(integral_constant<int, 0>{}, kb, sx0, sw0, sx1, sw1);
  __builtin_amdgcn_s_waitcnt(0x0070);  // the last steps' DMA repeats the last block into LDS that nothing reads
  settle(acc);
  __syncthreads();  // the steps' LDS becomes the waves' bands
  static_assert(kBand<128> <= 256 * 128 && 16 * kPitch<128> * 4 <= kBand<128>, "the bands fit");
  uint8_t* const part = (wave & 2) ? (wave & 1 ? sw1 : sw0) : (wave & 1 ? sx1 : sx0);
  store_tile<true, true, ACT>(p, acc, (float*)part, m0 + wm, n0 + wn);
}

// ---- few rows ----
// 16 columns of y and MT x 16 rows per workgroup; its eight waves take the blocks of k in turn and add their parts in LDS, in
// wave order.  With few rows the bytes of w and the latency of fetching them are the cost.  x comes as codes, or as values
// that are quantised on the way (a lane holds 32 of a row's 128 values; four lanes share the block): one launch and no
// workspace.
constexpr int kFewWaves = 8;

// 32 values of a row as they come from memory: chunks k .. +15 and k + 64 .. +79
template <typename T>
struct Raw32 {
  static constexpr int N = sizeof(T);  // 16-B pieces of 16 values: 2 (bf16) or 4 (f32)
  u32x4_t w[2][N];
  __device__ __forceinline__ void load(const T* row, int k, int K, bool vec) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int kk = k + 64 * g;
      if (vec && kk + 16 <= K) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[g][i] = *reinterpret_cast<const u32x4_t*>(row + kk + i * (16 / N));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = kk + (16 / N) * i + (4 / N) * e;
            if constexpr (N == 4) w[g][i][e] = at < K ? __float_as_uint(row[at]) : 0u;
            else w[g][i][e] = (at < K ? (uint32_t)row[at] : 0u) | (at + 1 < K ? (uint32_t)row[at + 1] << 16 : 0u);
          }
      }
    }
  }
  __device__ __forceinline__ uint32_t max_bits() const {  // f32 bits of the largest magnitude
    if constexpr (N == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) m = max(m, w[g][i][e] & 0x7FFFFFFFu);
      return m;
    } else {  // two at a time
      u16x2_t m = {0, 0};
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w[g][i][e] & 0x7FFF7FFFu));
      return (uint32_t)max(m[0], m[1]) << 16;
    }
  }
  __device__ __forceinline__ float value(int g, int i) const {  // i: 0 .. 15
    if constexpr (N == 4) return __uint_as_float(w[g][i >> 2][i & 3]);
    else return __uint_as_float(i & 1 ? w[g][i >> 3][(i & 7) >> 1] & 0xFFFF0000u : w[g][i >> 3][(i & 7) >> 1] << 16);
  }
};

// the lane's 32 values as codes, and their block's scale
template <typename T>
__device__ __forceinline__ i32x8_t codes(const Raw32<T>& raw, int& scale) {
  float v[32];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[16 * g + i] = raw.value(g, i);
  auto reduce = [](uint32_t m) {  // the four lanes of the row
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    return max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  };
  scale = itts::e4m3_scaled(v, reduce(raw.max_bits()), reduce);
  i32x8_t f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (int)e4m3_pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  return f;
}

// T: bf16 or f32 values, or codes (with their scales in p).  A wave's blocks of w (and of codes) go to its own part of the
// LDS by DMA, two slots in turn, in the layout of the tile kernels: the matrix unit wants neighbouring lanes on neighbouring
// rows, and the load path handles such lanes one by one (59 accesses per load instruction; fetched to registers that way,
// 96 x 4096 x 1024 took 13.2 us instead of 8.2).
template <bool EXACT, typename T, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void fp8_linear_few_kernel(LinearArgs p, const T* __restrict__ x, int64_t ldx, int K, bool vec) {
  constexpr bool CODES = std::is_same_v<T, uint8_t>;
  constexpr int DMA = 2 + (CODES ? 2 * MT : 0);  // instructions of 8 rows: w's 16, then x's
  constexpr int SLOT = 1024 * DMA;
  __shared__ __attribute__((aligned(1024))) uint8_t s0[kFewWaves * SLOT], s1[kFewWaves * SLOT];
  __shared__ f32x4_t part[kFewWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const uint8_t* src[DMA];
#pragma unroll
  for (int i = 0; i < DMA; ++i) {
    const int row = 8 * i + (lane >> 3), chunk = 16 * ((lane & 7) ^ (row >> 1 & 7));
    src[i] = (i < 2 ? p.wq + (int64_t)min(n0 + row, p.N - 1) * p.ldw : p.xq + min(m0 + row - 16, p.M - 1) * p.ldxq) + chunk;
  }
  auto issue = [&](int kb, uint8_t* slot) {
#pragma unroll
    for (int i = 0; i < DMA; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(src[i] + 128 * kb), (lds_void*)(slot + SLOT * wave + 1024 * i), 16, 0, 0);
  };
  const int nb = (p.KB - wave + kFewWaves - 1) / kFewWaves;  // this wave's blocks: wave + 8 i
  if (nb > 0) issue(wave, s0);
  // scale bytes of four of the wave's blocks at a time, lane group c those of block i + c
  const uint8_t* wsr = p.ws + (int64_t)min(n0 + r, p.N - 1) * p.ldws;
  const uint8_t* xsr[MT];
  const T* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = min(m0 + 16 * t + r, p.M - 1);
    xr[t] = x + m * ldx;
    xsr[t] = p.xs + m * p.ldxs;
  }
  int ws4 = 0, xs4[MT];
  auto load_scales = [&](int i) {
    const int kb = min(wave + kFewWaves * (i + c), p.KB - 1);
    ws4 = wsr[kb];
#pragma unroll
    for (int t = 0; t < MT; ++t) xs4[t] = CODES ? xsr[t][kb] : 0;
  };
  load_scales(0);
  Raw32<T> raw[CODES ? 1 : MT];
  auto load_raw = [&](int kb) {
    if constexpr (!CODES) {
#pragma unroll
      for (int t = 0; t < MT; ++t) raw[t].load(xr[t], 128 * kb + 16 * c, K, vec);
    }
  };
  if (nb > 0) load_raw(wave);
  // bias and residual of the one result that this thread adds up
  static_assert(MT <= 2, "one result per thread");
  const int row = threadIdx.x >> 4, col = threadIdx.x & 15;
  const bool mine = row < 16 * MT && m0 + row < p.M && n0 + col < p.N;
  const float bias = p.bias && mine ? p.bias[n0 + col] : 0.f;
  const float residual = p.residual && mine ? p.residual[(m0 + row) * p.ldr + n0 + col] : 0.f;

  f32x4_t acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int a0 = r * 128 + ((c ^ (r >> 1 & 7)) << 4), a1 = r * 128 + (((4 + c) ^ (r >> 1 & 7)) << 4);
  auto read = [&](const uint8_t* s) -> i32x8_t {
    const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(s + a0), hi = *reinterpret_cast<const u32x4_t*>(s + a1);
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  auto step = [&](int i, uint8_t* slot, uint8_t* other) {
    const uint8_t* s = slot + SLOT * wave;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): the block has landed, this wave's reads of the other slot are done
    asm volatile("" ::: "memory");
    Raw32<T> now[CODES ? 1 : MT];
    if constexpr (!CODES) {
#pragma unroll
      for (int t = 0; t < MT; ++t) now[t] = raw[t];
    }
    const int at = r + 16 * (i & 3);
    const int sw = __shfl(ws4, at, 64);
    int sx[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) sx[t] = CODES ? __shfl(xs4[t], at, 64) : 0;
    if (i + 1 < nb) {
      issue(wave + kFewWaves * (i + 1), other);
      load_raw(wave + kFewWaves * (i + 1));
      if (((i + 1) & 3) == 0) load_scales(i + 1);
    }
    const i32x8_t wf = read(s);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      i32x8_t xf;
      if constexpr (CODES) xf = read(s + 2048 * (1 + t));
      else xf = codes(now[t], sx[t]);
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dequant8(wf[2 * e], wf[2 * e + 1], itts::e4m3_scale(sw)),
                                                           dequant8(xf[2 * e], xf[2 * e + 1], itts::e4m3_scale(sx[t])), acc[t], 0, 0, 0);
      } else {
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[t], 0, 0, 0, sw, 0, sx[t]);
      }
    }
  };
  for (int i = 0; i < nb; i += 2) {
    step(i, s0, s1);
    if (i + 1 < nb) step(i + 1, s1, s0);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  if (!mine) return;
  float v = bias;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) v += part[w][row >> 4][(col >> 2) * 16 + (row & 15)][col & 3];
  v = p.act == 0 ? v : p.act == 1 ? apply_act<1>(v) : apply_act<2>(v);
  v += residual;
  const int64_t at = (m0 + row) * p.ldy + n0 + col;
  if (p.out_bf16) ((uint16_t*)p.y)[at] = f2bf(v);
  else ((float*)p.y)[at] = v;
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

// x quantised within the product (one launch, no workspace) while that is done by few: with more rows or a long k the
// same values are quantised once per 16 columns of y.  Measured, us (this / quantised first): 1 x 1024 x 4096 3.4 / 5.0,
// 16 x 4096 x 1024 6.7 / 7.3, 32 x 1024 x 4096 5.6 / 5.9, 32 x 2048 x 1024 7.0 / 6.3, 32 x 4096 x 1024 11.0 / 7.9.
bool few_rows(int64_t M, int K) { return M <= 16 || (M <= 32 && K <= 1024); }
// 32 x 16 outputs per workgroup with k split among its waves, while that is at most three turns of the 256 CUs: a 128 x 128
// tile takes 0.8 us per block of k, one after the other.  Measured, us (this / such tiles, both with the quantising pass of
// 2.5): 96 x 4096 x 1024 8.3 / 29, 96 x 1024 x 4096 10.0 / 12.3, 300 x 1024 x 1024 10.2 / 12.4, 800 x 256 x 2048 25 / 8.5.
bool some_rows(int64_t M, int N) { return ((M + 31) / 32) * ((N + 15) / 16) <= 768; }
// 256 x 256 tiles once they keep most of the 256 CUs busy (and the scales of all of k fit the LDS beside them).  Measured,
// us with the quantising pass (these / 128 x 128): 14400 x 1024 x 4096 91 / 102, with GELU 107 / 115, 14400 x 4096 x 1024 82 / 101,
// 8192 x 8192 x 8192 443 / 646, 3000 x 1024 x 4096 (192 tiles) 26 / 30, 2000 x 1024 x 4096 (128 tiles) 24 / 20.
bool large_tiles(int64_t M, int N, int K) {
  return M > 128 && N > 128 && ((M + 255) / 256) * ((N + 255) / 256) >= 160 && K <= 128 * kScaleBlocks;
}

template <bool EXACT, int BM, int BN, int WM, int WN>
void launch_tile(const LinearArgs& p, hipStream_t st) {
  const dim3 g((unsigned)(((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN))), b(64 * (BM / WM) * (BN / WN));
  if (p.act == 0) hipLaunchKernelGGL((fp8_linear_tile_kernel<EXACT, 0, BM, BN, WM, WN>), g, b, 0, st, p);
  else if (p.act == 1) hipLaunchKernelGGL((fp8_linear_tile_kernel<EXACT, 1, BM, BN, WM, WN>), g, b, 0, st, p);
  else hipLaunchKernelGGL((fp8_linear_tile_kernel<EXACT, 2, BM, BN, WM, WN>), g, b, 0, st, p);
}
void launch_large(const LinearArgs& p, hipStream_t st) {
  const dim3 g((unsigned)(((p.M + 255) / 256) * ((p.N + 255) / 256))), b(256);
  if (p.act == 0) hipLaunchKernelGGL(fp8_linear_large_kernel<0>, g, b, 0, st, p);
  else if (p.act == 1) hipLaunchKernelGGL(fp8_linear_large_kernel<1>, g, b, 0, st, p);
  else hipLaunchKernelGGL(fp8_linear_large_kernel<2>, g, b, 0, st, p);
}
template <typename T, int MT>
void launch_few(const T* x, int64_t ldx, int K, bool vec, const LinearArgs& p, hipStream_t st) {
  const dim3 g((p.N + 15) / 16, (unsigned)((p.M + 16 * MT - 1) / (16 * MT))), b(64 * kFewWaves);
  if (p.out_bf16) hipLaunchKernelGGL((fp8_linear_few_kernel<false, T, MT>), g, b, 0, st, p, x, ldx, K, vec);
  else hipLaunchKernelGGL((fp8_linear_few_kernel<true, T, MT>), g, b, 0, st, p, x, ldx, K, vec);
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
  return few_rows(M, K) ? 0 : round_up(M, 256) * (code_pitch(K) + scale_pitch(K));  // whole tiles of rows
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
  ITTS_REQUIRE(ldw >= code_pitch(K) && ldw % 16 == 0 && ldws >= scale_pitch(K) && ldws % 4 == 0 && ldw <= 4 * kMaxK &&
                   ldws <= kMaxK,
               fn, "weight rows need K rounded up to 128 bytes, scale rows ceil(K / 128) rounded up to 4");
  if (M == 0) return 0;
  const bool few = few_rows(M, K);
  ITTS_REQUIRE(x && wq && ws && y && (few || workspace), fn, "null pointer");
  ITTS_REQUIRE((((uintptr_t)wq | (uintptr_t)workspace) & 15) == 0 && ((uintptr_t)ws & 3) == 0, fn, "misaligned pointer");
  ITTS_REQUIRE(((M + 127) / 128) * ((N + 127) / 128) <= 0x7FFFFFFF, fn, "too many tiles for one launch");
  uint8_t* xq = (uint8_t*)workspace;
  uint8_t* xs = xq + round_up(M, 256) * code_pitch(K);
  hipStream_t st = itts::as_stream(stream);
  const int es = out_dtype == ITTS_F32 ? 4 : 2;
  LinearArgs p{xq, xs, wq, ws, code_pitch(K), scale_pitch(K), ldw, ldws, M, N, (K + 127) / 128, bias, residual, ldr, y, ldy,
               act, out_dtype == ITTS_BF16, ((uintptr_t)y & 15) == 0 && (ldy * es) % 16 == 0 && N % 16 == 0 &&
                   ((uintptr_t)bias & 15) == 0 && ((uintptr_t)residual & 15) == 0 && (!residual || ldr % 4 == 0)};
  if (few) {
    const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (x_dtype == ITTS_F32 ? 4 : 8) == 0;
    if (x_dtype == ITTS_F32 && M <= 16) launch_few<float, 1>((const float*)x, ldx, K, vec, p, st);
    else if (x_dtype == ITTS_F32) launch_few<float, 2>((const float*)x, ldx, K, vec, p, st);
    else if (M <= 16) launch_few<uint16_t, 1>((const uint16_t*)x, ldx, K, vec, p, st);
    else launch_few<uint16_t, 2>((const uint16_t*)x, ldx, K, vec, p, st);
    return itts::check_launch(fn);
  }
  if (int rc = launch_quant(fn, x, ldx, x_dtype, M, K, xq, code_pitch(K), xs, scale_pitch(K), st)) return rc;
  if (some_rows(M, N)) launch_few<uint8_t, 2>(xq, p.ldxq, K, true, p, st);
  else if (!p.out_bf16) launch_tile<true, 128, 128, 64, 64>(p, st);
  else if (large_tiles(M, N, K)) launch_large(p, st);
  else launch_tile<false, 128, 128, 64, 64>(p, st);
  return itts::check_launch(fn);
}
