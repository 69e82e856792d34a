// Attention of one new token (itts_attn_decode_kv8) or of a tree of drafted tokens (itts_attn_tree) per row over a KV
// cache in block-scaled e4m3 (fp8.h) or bf16.
//
// One wave walks its share of a row and K/V head's keys in tiles of 32, with NQ x 16 query columns (column = drafted
// token * group + query head of the group), everything in registers:
//   S^T [32 keys][columns] = K Q^T     (A = K, B = Q^T; v_mfma_f32_16x16x32_bf16, two per 32 dims)
//   running maximum and sum per column (a column's keys lie in the lanes l, l ^ 16, l ^ 32, l ^ 48)
//   O^T [dims][columns] += V^T P^T     (A = V^T, B = P^T; v_mfma_f32_16x16x32_f16 / _bf16)
// S^T leaves a lane with keys 4 c + i and 16 + 4 c + i (c = lane / 16) of its column, which is a B operand of the second
// product when V's keys are taken in the same order, so P never moves between lanes.  V's lane loads hd / 16 dims of
// its eight keys and pairs them by v_perm: no LDS.  The order of dims within the first product is free, so K's lane
// takes 16 consecutive bytes.
//
// Types: e4m3 K times its scale is exact in bf16 (any exponent), so q enters as bf16 and is exact when it is bf16; an f32
// q enters as three bf16 parts (24 bits).  While the scales of a wave's V keep within a factor 2^12 of each other, e4m3 V is
// exact in f16 relative to the largest, and P enters as f16 in [0, 2^15] (half step 2^-12 of a weight, below the bf16 output's
// 2^-9) or, for f32 outputs, as two f16 parts (2^-23); of weights below 2^-27 (two parts: 2^-16) of the largest fewer bits are left,
// down to 2^-38.  Where the scales lie further apart -- in a drafted token that other columns do not see, or in keys without
// weight -- the wave takes its tiles once more with V as bf16, which is exact with any scale, and P as two bf16 parts (2^-17) or three
// for f32 outputs: every finite V counts where it is seen and nowhere else.  That costs the second walk: 1.3 to 2 times the time
// (131 keys 5.3 -> 7.0 us; 64 tokens x 4 heads over 16301 keys 116 -> 220).  bf16 V: P as two bf16 parts.
// Maxima, sums and both products accumulate in f32.
//
// What bounds it, and what it takes (whole calls in a replayed graph): few tokens over long rows run at the memory's rate (8 rows x
// 4 heads, up to 32749 keys of 128 dims: 216 MB in 45 us = 4.8 TB/s, the join of the splits among them); with lineage tables (96
// rows x 16 heads, up to 483 keys of 64 dims) it is the tables' and addresses' arithmetic, 29 us for 78 MB; short rows cost a
// launch and one trip to memory (131 keys: 5.3 us); many columns (64 tokens x 4 heads, 16301 keys: 116 us for 27 GFLOP, 112 MB)
// the vector instructions around the products, some 250 per 32 keys and 32 columns, half of them for K's and V's conversion.
#pragma once
#include <type_traits>

#include "fp8.h"

namespace itts {
namespace attn {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;

struct AttnArgs {
  ItTsKvCache c;
  const void* q;
  int64_t q_sb, q_st, q_sh;
  bool q_f32, tree, out_f32;
  int T, G;
  const int32_t *kv_len, *pad, *n_tokens, *kv_rows;
  int64_t ld_rows;
  const uint64_t* mask;
  int64_t mask_sb;
  float qk_scale;  // scale * log2(e)
  void* out;
  int64_t o_sb, o_st, o_sh;
  // set by attend()
  bool negate, q_vec, o_vec;
  int units, qblocks, nsplit;
  float *part, *part_ml;  // [unit][split][column][hd], [unit][split][column][maximum, sum of weights relative to it]
};

// The column's reference follows the running maximum once that is more than a factor 2^kLag (bf16: 2^kWideLag) ahead.  In f16 P is
// held times 2^kPUp relative to it, so within 2^15, and V's codes times 2^7 relative to the largest scale: both within f16.  A shorter
// lag holds smaller weights and rescales O more often (lags of 2^8 / 2^4 / 2^2 / 2^1, us: 64 tokens x 4 heads over 16301 keys 112 / 114
// / 116 / 119; few columns alike).
constexpr int kLag = 2;
constexpr int kPUp = 15 - kLag;
constexpr int kVUp = 7;
// In bf16 P has f32's exponents and stays within 1: a sum of P V overflows no sooner than a sum of V.
constexpr int kWideLag = 8;
constexpr int kWideUp = -kWideLag;
// Scales of V within a factor 2^kSpread of each other go through f16: V is exact there up to 2^22, and what f16 loses of a
// weight (below 2^-38 of the largest) counts for little whatever its V.
constexpr int kSpread = 12;

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
// low / high halves of two dwords
__device__ __forceinline__ uint32_t lo16(uint32_t a, uint32_t b) { return perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t hi16(uint32_t a, uint32_t b) { return perm(b, a, 0x07060302u); }

__device__ __forceinline__ void store4(const AttnArgs& a, int64_t at, f32x4_t y) {
  if (a.o_vec) {
    if (a.out_f32) *reinterpret_cast<f32x4_t*>((float*)a.out + at) = y;
    else *reinterpret_cast<u32x2_t*>((uint16_t*)a.out + at) = u32x2_t{pack2bf(y[0], y[1]), pack2bf(y[2], y[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (a.out_f32) ((float*)a.out)[at + i] = y[i];
      else ((uint16_t*)a.out)[at + i] = f2bf(y[i]);
    }
  }
}

// larger of two scores as the median with the largest float (an infinite score makes its column NaN all the same): fmaxf
// first brings both into canonical form, two more instructions each (with V's scales as f32 bits 4 us of 120
// for 64 tokens x 4 heads over 16301 keys)
__device__ __forceinline__ float max2(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, 3.4028234663852886e38f); }
// 1 / the sum of a token's weights, for an output: a row that sees nothing gives 0; where every score that it sees is -inf there
// is no weight to divide by, and the result is NaN
__device__ __forceinline__ float inverse_sum(const AttnArgs& a, float sum, int b, int t, int len, int n) {
  if (sum != 0.f) return 1.f / sum;
  bool sees = (a.pad ? max(a.pad[b], 0) : 0) < len;
  if (a.tree) sees |= (a.mask[(int64_t)b * a.mask_sb + t] & (n < 64 ? (1ull << n) - 1 : ~0ull)) != 0;
  return sees ? __builtin_nanf("") : 0.f;
}

// max over the four lanes that hold a column: lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(max2(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ int max_rows(int v) {
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  const int w = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)w, (uint32_t)w, false, false);
  return max((int)b[0], (int)b[1]);
}

constexpr int kWaves = 4;  // waves of a workgroup take its tiles in turn

// waves per SIMD that the registers are held to: the most that leave the loop without spills (32 x 16 heads, 64 tokens with an
// f32 q over 600 keys of a bf16 cache: 36 us at two, 56 at one)
template <bool E4M3, bool LINEAGE, int HD, int QN, int NQ>
constexpr int waves_per_simd() {
  if (E4M3 && HD == 64) return NQ == 1 || (QN == 1 && !LINEAGE) ? 3 : 2;
  if (HD == 64) return 2;
  if (E4M3) return NQ == 1 || (QN == 1 && !LINEAGE) ? 2 : 1;
  return 1;
}

template <bool E4M3, bool LINEAGE, int HD, int QN, int PN, int NQ>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<E4M3, LINEAGE, HD, QN, NQ>())) void attn_cached_kernel(AttnArgs a) {
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int KW = HD * ES / 64;  // 16-B pieces of K per lane and 16 keys; dwords of V per lane and key
  constexpr int KS = HD / 32;       // MFMA steps of the first product
  constexpr int DT = HD / 16;       // 16-dim tiles of the second
  constexpr int COLS = 16 * NQ;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
  // workgroup -> (unit = (row, K/V head), query block, split).  The query blocks of one (unit, split) read the same keys:
  // they get ids 8 apart, so they land on one XCD one after the other and share its L2
  const int per = 8 * a.qblocks;
  const int grp = blockIdx.x / per, in = blockIdx.x - grp * per;
  const int us = grp * 8 + (in & 7), qb = in >> 3;
  const int unit = us / a.nsplit, split = us - unit * a.nsplit;
  if (unit >= a.units) return;
  const int b = unit / a.c.heads, h = unit - b * a.c.heads;
  const int G = a.G, C = a.T * G;

  int len = a.kv_len[b];
  int n = a.tree ? (a.n_tokens ? a.n_tokens[b] : a.T) : 0;
  const bool refuse = len < 0 || n < 0 || n > a.T || len > a.c.max_kv - n;
  if (refuse) len = n = 0;  // no position is derived from what is refused
  const int first = a.pad ? max(a.pad[b], 0) : 0;
  const int hi = len + n;
  const int nt = a.tree ? n : 1;  // tokens that have an output

  // the split's tiles: base = begin + 32 (wave + kWaves i) < end
  int begin = min(first, len) & ~31, end = hi;
  if (a.nsplit > 1) {
    const int tiles = max((hi - begin + 31) >> 5, 0);
    const int each = (tiles + a.nsplit - 1) / a.nsplit;
    begin += 32 * each * split;
    end = min(hi, begin + 32 * each);
  }

  const int last = a.c.max_kv - 1;
  auto key = [&](int tile, int u) { return tile + 4 * c + (u & 3) + 16 * (u >> 2); };  // the lane's eight keys
  const char* kbase = (const char*)a.c.k + (int64_t)h * a.c.hs * ES;
  const char* vbase = (const char*)a.c.v + (int64_t)h * a.c.hs * ES;
  constexpr uint32_t ROW = HD * ES;  // bytes from key to key
  const uint32_t klane = ROW * r + 16 * c, vlane = ROW * 4 * c + 4 * KW * r;
  const uint8_t* ksbase = E4M3 ? a.c.k_scale + (int64_t)h * a.c.shs : nullptr;
  const uint8_t* vsbase = E4M3 ? a.c.v_scale + (int64_t)h * a.c.shs : nullptr;
  const int32_t* rows = LINEAGE ? a.kv_rows + (int64_t)b * a.ld_rows : nullptr;
  if constexpr (!LINEAGE) {
    kbase += (int64_t)b * a.c.bs * ES;
    vbase += (int64_t)b * a.c.bs * ES;
    if constexpr (E4M3) {
      ksbase += (int64_t)b * a.c.sbs;
      vsbase += (int64_t)b * a.c.sbs;
    }
  }

  // A tile of 32 keys as it comes from memory.  Loads stay within the cache by its capacity alone (positions at or behind
  // the row's end are masked later), so the first tile is requested without waiting for kv_len.
  u32x4_t tk[2][KW];   // K rows of keys r and 16 + r: 16-B pieces
  int tks[2];          // their scale bytes
  uint32_t tv[8][KW];  // hd / 16 values of the lane's eight keys 4 c + i, 16 + 4 c + i
  uint32_t tvs[2];     // their scale bytes
  uint32_t tbad = 0;   // LINEAGE: bit u: key u's cache row is none
  int rk[2], rv[8];    // LINEAGE: cache rows of the next tile's keys
  auto load_rows = [&](int base) {
    if constexpr (LINEAGE) {
#pragma unroll
      for (int f = 0; f < 2; ++f) rk[f] = rows[min(base + 16 * f + r, last)];
      if (base + 31 <= last) {
#pragma unroll
        for (int g = 0; g < 2; ++g) __builtin_memcpy(&rv[4 * g], rows + base + 16 * g + 4 * c, 16);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) rv[u] = rows[min(key(base, u), last)];
      }
    }
  };
  auto load = [&](int base) {
    if constexpr (LINEAGE) {
      tbad = 0;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int p = min(base + 16 * f + r, last);
        const int64_t at = (unsigned)rk[f] < (unsigned)a.c.rows ? rk[f] : 0;
        const char* src = kbase + (at * a.c.bs * ES + p * ROW + 16 * c);
#pragma unroll
        for (int i = 0; i < KW; ++i) tk[f][i] = *reinterpret_cast<const u32x4_t*>(src + 64 * i);
        if constexpr (E4M3) tks[f] = ksbase[at * a.c.sbs + p];
      }
      uint32_t sb[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = min(key(base, u), last);
        const bool ok = (unsigned)rv[u] < (unsigned)a.c.rows;
        tbad |= ok ? 0u : 1u << u;
        const int64_t at = ok ? rv[u] : 0;
        __builtin_memcpy(tv[u], vbase + (at * a.c.bs * ES + p * ROW + 4 * KW * r), 4 * KW);
        if constexpr (E4M3) sb[u] = vsbase[at * a.c.sbs + p];
      }
      if constexpr (E4M3) {
#pragma unroll
        for (int g = 0; g < 2; ++g) tvs[g] = sb[4 * g] | sb[4 * g + 1] << 8 | sb[4 * g + 2] << 16 | sb[4 * g + 3] << 24;
      }
    } else if (base + 31 <= last) {
      // uniform base, one lane offset each for K and V: the keys are immediates
      const char* kt = kbase + (int64_t)base * ROW;
      const char* vt = vbase + (int64_t)base * ROW;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
#pragma unroll
        for (int i = 0; i < KW; ++i) tk[f][i] = *reinterpret_cast<const u32x4_t*>(kt + (klane + 16 * ROW * f + 64 * i));
        if constexpr (E4M3) tks[f] = ksbase[base + (uint32_t)(r + 16 * f)];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) __builtin_memcpy(tv[u], vt + (vlane + ROW * ((u & 3) + 16 * (u >> 2))), 4 * KW);
      if constexpr (E4M3) {  // four neighbouring bytes at a time
#pragma unroll
        for (int g = 0; g < 2; ++g) __builtin_memcpy(&tvs[g], vsbase + base + (uint32_t)(16 * g + 4 * c), 4);
      }
    } else {
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int p = min(base + 16 * f + r, last);
#pragma unroll
        for (int i = 0; i < KW; ++i) tk[f][i] = *reinterpret_cast<const u32x4_t*>(kbase + (p * ROW + 16 * c + 64 * i));
        if constexpr (E4M3) tks[f] = ksbase[p];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) __builtin_memcpy(tv[u], vbase + (min(key(base, u), last) * ROW + 4 * KW * r), 4 * KW);
      if constexpr (E4M3) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          tvs[g] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) tvs[g] |= (uint32_t)vsbase[min(key(base, 4 * g + i), last)] << (8 * i);
        }
      }
    }
  };
  int base;
  auto load_first = [&] {
    base = begin + 32 * wave;
    if (base <= last) {
      load_rows(base);
      load(base);
      if (base + 32 * kWaves <= last) load_rows(base + 32 * kWaves);
    }
  };
  load_first();

  // this lane's columns, their masks and Q.  No other workgroup takes these columns, and all four waves have read them before the
  // first barrier: the result may lie where Q is.
  int col[NQ], tok[NQ];
  uint64_t msk[NQ];
  u32x4_t qf[NQ][KS][QN];
  float m[NQ];    // reference of the column's exponentials, in scaled scores; -inf: nothing seen yet
  f32x4_t l[NQ];  // the sum of P: every element the same (a product of P with ones)
  f32x4_t o[NQ][DT];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    col[j] = (qb * NQ + j) * 16 + r;
    const int cc = min(col[j], C - 1);
    tok[j] = cc / G;
    msk[j] = 0;
    if (a.tree) {
      msk[j] = a.mask[(int64_t)b * a.mask_sb + tok[j]];
      if (n < 64) msk[j] &= (1ull << n) - 1;
    }
    const int64_t off = (int64_t)b * a.q_sb + tok[j] * a.q_st + (int64_t)(h * G + cc - tok[j] * G) * a.q_sh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // the eight dims that K's lane holds at this step
      const int d0 = E4M3 ? 64 * (s >> 1) + 16 * c + 8 * (s & 1) : 32 * s + 8 * c;
      float x[8];
      if (a.q_f32) {
        const float* src = (const float*)a.q + off + d0;
        if (a.q_vec) {
          const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(src), up = *reinterpret_cast<const f32x4_t*>(src + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = up[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = src[e];
        }
      } else {
        const uint16_t* src = (const uint16_t*)a.q + off + d0;
        if (a.q_vec) {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = bf2f(src[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // a negative scale is taken into q, so that the largest score is the largest product
        float x0 = a.negate ? -x[2 * e] : x[2 * e], x1 = a.negate ? -x[2 * e + 1] : x[2 * e + 1];
#pragma unroll
        for (int t = 0; t < QN; ++t) {
          const uint32_t w = pack2bf(x0, x1);
          qf[j][s][t][e] = w;
          x0 -= __uint_as_float(w << 16);
          x1 -= __uint_as_float(w & 0xFFFF0000u);
        }
      }
    }
    m[j] = -__builtin_inff();
    l[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) o[j][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  int vref = 0;          // e4m3: V is held relative to 2^(vref - 127)
  uint32_t low = ~0u;    // smallest scale that this lane has met, as f32 bits (less one at most)
  uint32_t odd = 0;      // non-zero: V held a NaN or infinity at a drafted token

  // V^T operands [16-dim tile][8 keys]; dim tile d holds the lane's dims (hd / 16) r + d.  f16: e4m3 V as f16, otherwise bf16
  auto v_frags = [&](auto f16, const uint32_t (&v)[8][KW], const float (&sc)[8], u32x4_t (&vf)[DT]) {
    auto two = [&](uint32_t w, float s, auto up) {
      if constexpr (decltype(f16)::value)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, decltype(up)::value));
      else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, decltype(up)::value));
    };
    constexpr std::false_type lower{};
    constexpr std::true_type upper{};
#pragma unroll
    for (int i = 0; i < KW; ++i) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) {
        if constexpr (E4M3) {
          const uint32_t a0 = two(v[u][i], sc[u], lower), a1 = two(v[u][i], sc[u], upper);
          const uint32_t b0 = two(v[u + 1][i], sc[u + 1], lower), b1 = two(v[u + 1][i], sc[u + 1], upper);
          vf[4 * i][u / 2] = lo16(a0, b0);
          vf[4 * i + 1][u / 2] = hi16(a0, b0);
          vf[4 * i + 2][u / 2] = lo16(a1, b1);
          vf[4 * i + 3][u / 2] = hi16(a1, b1);
        } else {
          vf[2 * i][u / 2] = lo16(v[u][i], v[u + 1][i]);
          vf[2 * i + 1][u / 2] = hi16(v[u][i], v[u + 1][i]);
        }
      }
    }
  };
  auto pv = [&](auto f16, u32x4_t vf, u32x4_t pf, f32x4_t acc) -> f32x4_t {
    if constexpr (decltype(f16)::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, vf), __builtin_bit_cast(f16x8_t, pf), acc, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, pf), acc, 0, 0, 0);
  };

  // Which of a tile's 32 keys are seen, as bits: all columns' prefix, and a column's drafted tokens
  auto below = [](int i) -> uint32_t { return i <= 0 ? 0u : i >= 32 ? ~0u : (1u << i) - 1; };  // bits 0 .. i - 1
  auto prefix_bits = [&](int tile) { return below(len - tile) & ~below(first - tile); };
  auto drafted_bits = [&](int tile, uint64_t mask) -> uint32_t {
    const int d = tile - len;
    return d >= 64 ? 0u : d >= 0 ? (uint32_t)(mask >> d) : d > -32 ? (uint32_t)(mask << -d) : 0u;
  };
  auto mine = [&](uint32_t bits) { return (bits >> (4 * c) & 0xFu) | (bits >> (16 + 4 * c) & 0xFu) << 4; };

  // A drafted token's V that is not finite reaches only the columns that see it.  Such values enter the products as 0;
  // here a product of (1 where V is the special value) and (1 where the column sees the key) counts them.
  auto not_finite = [&](int tile) {
    constexpr std::bool_constant<E4M3> f16{};
    constexpr uint32_t kOne = E4M3 ? 0x3C00u : 0x3F80u;
    const uint32_t drafted = mine(below(hi - tile) & ~below(len - tile));
    uint32_t w8[8][KW];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = min(key(tile, u), last);
      int64_t at = 0;
      if constexpr (LINEAGE) {
        const int row = rows[p];
        at = ((unsigned)row < (unsigned)a.c.rows ? row : 0) * a.c.bs * ES;
      }
      __builtin_memcpy(w8[u], vbase + (at + p * ROW + 4 * KW * r), 4 * KW);
    }
#pragma unroll 1
    for (int kind = 0; kind < (E4M3 ? 1 : 3); ++kind) {
      float one[8];
      uint32_t ind[8][KW];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        one[u] = 1.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t w = drafted >> u & 1 ? w8[u][i] : 0u;
          uint32_t v = 0;
          if constexpr (E4M3) {
            v = ((((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0x38u;  // e4m3 1.0
          } else {
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
              const uint32_t x16 = w >> (16 * s2) & 0xFFFFu;
              const int is = (x16 & 0x7F80u) != 0x7F80u ? -1 : (x16 & 0x7Fu) ? 0 : x16 >> 15 ? 2 : 1;
              if (is == kind) v |= kOne << (16 * s2);
            }
          }
          ind[u][i] = v;
        }
      }
      u32x4_t nf[DT];
      v_frags(f16, ind, one, nf);
      const float what = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const uint32_t vis = mine(drafted_bits(tile, msk[j]));
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[e] = (vis >> (2 * e) & 1) * kOne | (vis >> (2 * e + 1) & 1) * (kOne << 16);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f32x4_t count = pv(f16, nf[d], pf, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (count[i] > 0.f) o[j][d][i] += what;
        }
      }
    }
  };

  // The loop over the tiles.  wide: V as bf16, exact with any scale, and P in one more part of 8 bits each instead of 11.
  auto walk = [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value, F16 = E4M3 && !WIDE;
    constexpr std::bool_constant<F16> f16{};
    constexpr int PP = PN + (WIDE ? 1 : 0);
    constexpr uint32_t kOnes = (F16 ? 0x3C00u : 0x3F80u) * 0x10001u;
    const u32x4_t ones = u32x4_t{kOnes, kOnes, kOnes, kOnes};
    for (; base < end; base += 32 * kWaves) {
      const int tile = base;
      // an edge tile holds keys that some column may not see (before the padding's end, drafted, behind the row's end)
      const bool edge = tile < first || tile + 32 > len;
      uint32_t some = 0xFF;  // which of the lane's eight keys some column may see
      if (edge) {
        const uint32_t drafted = mine(below(hi - tile) & ~below(len - tile));
        some = mine(prefix_bits(tile)) | drafted;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            const uint32_t w = some >> u & 1 ? tv[u][i] : 0u;
            uint32_t bits;  // a drafted token's values that are not finite
            if constexpr (E4M3) bits = (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
            else bits = (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 15;
            bits *= (drafted >> u & 1) * (E4M3 ? 0xFFu : 0xFFFFu);
            odd |= bits;
            tv[u][i] = w & ~bits;
          }
        }
      }
      float sv[8];
      float rescale = 1.f;
      if constexpr (E4M3) {
        int vs[8];  // the scales as f32 bits, which order like them
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const uint32_t w = tvs[u >> 2];
          vs[u] = ((u & 3) == 3 ? w >> 1 : w << (23 - 8 * (u & 3))) & 0x7F800000u;
        }
        if (edge) {  // what nothing is seen of has no part in the reference; its V is 0
#pragma unroll
          for (int u = 0; u < 8; ++u) vs[u] = some >> u & 1 ? vs[u] : 0;
#pragma unroll
          for (int u = 0; u < 8; ++u) low = min(low, (uint32_t)vs[u] - 1);  // 0, an unseen key's, becomes the largest
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u) low = min(low, (uint32_t)vs[u]);
        }
        if constexpr (WIDE) {
#pragma unroll
          for (int u = 0; u < 8; ++u) sv[u] = __uint_as_float(vs[u]);
        } else {
          int top = max(max(max(vs[0], vs[1]), max(vs[2], vs[3])), max(max(vs[4], vs[5]), max(vs[6], vs[7])));
          top = __builtin_amdgcn_readfirstlane(max_rows(top)) >> 23;  // 16 lanes each hold the same eight bytes
          if (top > vref) {
            rescale = vref == 0 ? 0.f : __builtin_amdgcn_exp2f((float)(vref - top));
            vref = top;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) sv[u] = __builtin_ldexpf(__uint_as_float(vs[u]), 127 + kVUp - vref);
        }
      }
      u32x4_t vf[DT], kf[2][KS];
      v_frags(f16, tv, sv, vf);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if constexpr (E4M3) {
          const float sc = itts::e4m3_scale(tks[f]);
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              kf[f][2 * i + (w >> 1)][2 * (w & 1)] =
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(tk[f][i][w], sc, false));
              kf[f][2 * i + (w >> 1)][2 * (w & 1) + 1] =
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(tk[f][i][w], sc, true));
            }
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) kf[f][s] = tk[f][s];
        }
      }
      const uint32_t bad = tbad;
      const bool any_bad = LINEAGE && __any(bad != 0);
      // the tile is in its operands: the next one is requested into the same registers
      if (tile + 32 * kWaves < end) {
        load(tile + 32 * kWaves);
        if (LINEAGE && tile + 64 * kWaves < end) load_rows(tile + 64 * kWaves);
      }
      // the columns' scores and their maxima (a.qk_scale > 0); all columns go through each stage together, so that
      // one's products cover another's latencies
      float x[NQ][8], top[NQ];
      bool grow = rescale != 1.f;
      auto scores = [&](const u32x4_t (&low)[2][KS]) {  // low: what the lower parts of q meet
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          f32x4_t s[2];
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            s[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < KS; ++e)
#pragma unroll
              for (int q = QN - 1; q >= 0; --q)
                s[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, q ? low[f][e] : kf[f][e]),
                                                               __builtin_bit_cast(bf16x8_t, qf[j][e][q]), s[f], 0, 0, 0);
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) x[j][u] = s[u >> 2][u & 3];
        }
      };
      scores(kf);
      if constexpr (!E4M3 && QN > 1) {  // an infinite K times a lower part of 0 is NaN: once more without such products
        bool nan = false;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int u = 0; u < 8; ++u) nan |= x[j][u] != x[j][u];
        if (__any(nan)) {
          u32x4_t low[2][KS];
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int e = 0; e < KS; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t w = kf[f][e][i];
                low[f][e][i] = w & ~(((((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xFFFFu);
              }
          scores(low);
        }
      }
      if (any_bad) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int u = 0; u < 8; ++u) x[j][u] = bad >> u & 1 ? __builtin_nanf("") : x[j][u];
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          const uint32_t vis = mine(prefix_bits(tile) | drafted_bits(tile, msk[j]));
#pragma unroll
          for (int u = 0; u < 8; ++u) x[j][u] = vis >> u & 1 ? x[j][u] : -__builtin_inff();
        }
      }
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        top[j] = max_rows(max2(max2(max2(x[j][0], x[j][1]), max2(x[j][2], x[j][3])),
                               max2(max2(x[j][4], x[j][5]), max2(x[j][6], x[j][7]))) * a.qk_scale);
        grow |= top[j] > m[j] + (F16 ? kLag : kWideLag);
      }
      if (__any(grow)) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          const float next = fmaxf(m[j], top[j]);
          const float f = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[j] - next);
          m[j] = next;
          l[j] = l[j] * f;
          const float fo = f * rescale;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[j][d] = o[j][d] * fo;
        }
      }
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float p[8];
        const float shift = (float)(F16 ? kPUp : kWideUp) - (m[j] == -__builtin_inff() ? 0.f : m[j]);
#pragma unroll
        for (int u = 0; u < 8; ++u) p[u] = __builtin_amdgcn_exp2f(fmaf(x[j][u], a.qk_scale, shift));
#pragma unroll
        for (int q = 0; q < PP; ++q) {
          u32x4_t pf;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (F16) {
              const f16x2_t w = {(_Float16)p[2 * e], (_Float16)p[2 * e + 1]};
              pf[e] = __builtin_bit_cast(uint32_t, w);
              if (q + 1 < PP) p[2 * e] -= (float)w[0], p[2 * e + 1] -= (float)w[1];
            } else {
              const uint32_t w = pack2bf(p[2 * e], p[2 * e + 1]);
              pf[e] = w;
              if (q + 1 < PP) p[2 * e] -= __uint_as_float(w << 16), p[2 * e + 1] -= __uint_as_float(w & 0xFFFF0000u);
            }
          }
          l[j] = pv(f16, ones, pf, l[j]);
#pragma unroll
          for (int d = 0; d < DT; ++d) o[j][d] = pv(f16, vf[d], pf, o[j][d]);
        }
      }
    }  };
  bool absolute = !E4M3;  // o holds sums of P V as they are
  walk(std::false_type{});
  if constexpr (E4M3) {
    if (__builtin_expect(__any((int)min(low, kInfBits) < (vref - kSpread) * (1 << 23) - 1), 0)) {  // V's scales turned out too far apart: all tiles once more
      absolute = true;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        m[j] = -__builtin_inff();
        l[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[j][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      load_first();
      walk(std::true_type{});
    }
  }
  if (__builtin_expect(__any(odd != 0), 0)) {  // the drafted tokens' tiles of this wave once more
    for (int tile = begin + 32 * wave; tile < end; tile += 32 * kWaves)
      if (tile + 32 > len) not_finite(tile);
  }

  // ---- the waves' parts: common maximum and V reference, then O and the sums added in wave order ----
  // The common V reference is the largest.  Where a wave has none, or the waves' lie so far apart that f32 would lose the least
  // beside it, O is brought to the sums of P V that it stands for, with P in bf16's scale.
  constexpr int LDC = HD + 4;
  __shared__ float so[kWaves][COLS][LDC];
  __shared__ float sm[kWaves][COLS], sl[kWaves][COLS];
  __shared__ int sr[kWaves];
  if (lane == 0) sr[wave] = absolute ? -1 : vref;
  if (c == 0) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) sm[wave][16 * j + r] = m[j];
  }
  __syncthreads();
  int up = 0, p_up = kWideUp;  // O holds its values times 2^-up, and P's scale is 2^p_up
  float rel = 1.f;             // what this wave's O is brought to the common reference by
  if constexpr (E4M3) {
    int top_ref = 0, low_ref = 255;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      top_ref = max(top_ref, sr[w]);
      low_ref = min(low_ref, sr[w] == 0 ? 255 : sr[w]);
    }
    if (__builtin_expect(low_ref < top_ref - 64 || low_ref < 0, 0)) {
      if (!absolute) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          l[j][0] = __builtin_ldexpf(l[j][0], kWideUp - kPUp);
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][d][i] = __builtin_ldexpf(o[j][d][i], vref - 127 - kVUp + kWideUp - kPUp);
        }
      }
    } else {
      up = top_ref - 127 - kVUp;
      p_up = kPUp;
      rel = __builtin_amdgcn_exp2f((float)(vref - top_ref));  // 0 for a wave without keys
    }
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    if (col[j] >= C) continue;
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm[w][16 * j + r]);
    const float fl = top == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[j] - top);
    const float fo = fl * rel;
    if (c == 0) sl[wave][16 * j + r] = l[j][0] * fl;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < DT; d += 4)
        *reinterpret_cast<f32x4_t*>(&so[wave][16 * j + r][(4 * c + i) * DT + d]) =
            f32x4_t{o[j][d][i] * fo, o[j][d + 1][i] * fo, o[j][d + 2][i] * fo, o[j][d + 3][i] * fo};
  }
  __syncthreads();
  auto times = [](f32x4_t v, int e) -> f32x4_t {
    return f32x4_t{__builtin_ldexpf(v[0], e), __builtin_ldexpf(v[1], e), __builtin_ldexpf(v[2], e), __builtin_ldexpf(v[3], e)};
  };
  const int cols = min(COLS, C - qb * COLS);
  for (int i = threadIdx.x; i < cols * (HD / 4); i += 64 * kWaves) {
    const int cl = i / (HD / 4), d = 4 * (i - cl * (HD / 4));
    float sum = 0.f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      sum += sl[w][cl];
      acc = acc + *reinterpret_cast<const f32x4_t*>(&so[w][cl][d]);
    }
    const int cg = qb * COLS + cl;
    if (a.nsplit > 1) {
      // the split's own result, which is no larger than V, and its weight among the splits
      const int64_t at = ((int64_t)unit * a.nsplit + split) * C + cg;
      *reinterpret_cast<f32x4_t*>(a.part + at * HD + d) = times(acc * (sum == 0.f ? 1.f : 1.f / sum), up);
      if (d == 0) {
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm[w][cl]);
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = __builtin_ldexpf(sum, -p_up);
      }
    } else {
      const int t = cg / G;
      if (!refuse && t >= nt) continue;
      const float inv = refuse ? __builtin_nanf("") : inverse_sum(a, sum, b, t, len, n);
      store4(a, (int64_t)b * a.o_sb + t * a.o_st + (int64_t)(h * G + cg - t * G) * a.o_sh + d, times(acc * inv, up));
    }
  }
}

// ---- launches, by the types and the query tiles (attn_cached_*.hip hold the instances) ----
// Columns of 16 that a wave takes at once.  Two share a tile's loads and conversions; four (64 dims) spill or run at one wave
// per SIMD, and so do two of 128 dims with an f32 q.  Measured, us (one / two / four): 32 x 16 heads, 64 tokens over 600 keys
// of 64 dims 27 / 24 / 24, f32 q 33 / 30 / 45, bf16 cache 39 / 29 / 40; 4 x 8 heads x 4, 64 tokens over 16000 keys of 128 dims
// 189 / 120 / -, f32 q 191 / 197 / -; 8 x 8 heads x 4, 8 tokens over 4000 keys of 128 dims 23.5 / 25.4 / -, f32 q 25 / 36 / -.
inline int query_tiles(bool e4m3, int cols, bool q_f32, int hd) {
  if (cols <= 16) return 1;
  return e4m3 && hd == 128 && (q_f32 || cols <= 32) ? 1 : 2;
}

template <bool E4M3, bool LINEAGE, int HD, int QN, int PN, int NQ>
void launch_one(const AttnArgs& a, hipStream_t s) {
  const int64_t us = ((int64_t)a.units * a.nsplit + 7) / 8 * 8;
  hipLaunchKernelGGL((attn_cached_kernel<E4M3, LINEAGE, HD, QN, PN, NQ>), dim3((unsigned)(us * a.qblocks)),
                     dim3(64 * kWaves), 0, s, a);
}
template <bool E4M3, bool LINEAGE, int HD, int QN, int PN>
void launch_nq(const AttnArgs& a, hipStream_t s) {
  constexpr bool ONE = E4M3 && HD == 128 && QN == 3;
  if (ONE || query_tiles(E4M3, a.T * a.G, a.q_f32, HD) == 1) launch_one<E4M3, LINEAGE, HD, QN, PN, 1>(a, s);
  else if constexpr (!ONE) launch_one<E4M3, LINEAGE, HD, QN, PN, 2>(a, s);
}
// bf16 V takes P as two parts, e4m3 V for f32 outputs alone
template <bool E4M3, bool LINEAGE, int HD>
void launch_types(const AttnArgs& a, hipStream_t s) {
  if (a.q_f32) {
    if (!E4M3 || a.out_f32) launch_nq<E4M3, LINEAGE, HD, 3, 2>(a, s);
    else if constexpr (E4M3) launch_nq<E4M3, LINEAGE, HD, 3, 1>(a, s);
  } else {
    if (!E4M3 || a.out_f32) launch_nq<E4M3, LINEAGE, HD, 1, 2>(a, s);
    else if constexpr (E4M3) launch_nq<E4M3, LINEAGE, HD, 1, 1>(a, s);
  }
}
template <bool E4M3, int HD>
void launch_attn(const AttnArgs& a, hipStream_t s);

}  // namespace attn
}  // namespace itts

#define ITTS_ATTN_CACHED_INSTANCES(E4M3, HD)                                   \
  template <>                                                                  \
  void itts::attn::launch_attn<E4M3, HD>(const AttnArgs& a, hipStream_t s) {   \
    if (a.kv_rows) launch_types<E4M3, true, HD>(a, s);                         \
    else launch_types<E4M3, false, HD>(a, s);                                  \
  }
