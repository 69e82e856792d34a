// Attention of one new token (itts_attn_decode_kv8) or of a tree of drafted tokens (itts_attn_tree) per row over a KV
// cache in block-scaled e4m3 (fp8.h) or bf16.
//
// One wave walks its share of a row and K/V head's keys in tiles of 32, with up to NQ x 16 query columns (column = drafted
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
// q enters as three bf16 parts (24 bits).  e4m3 V is exact in f16 relative to the largest scale of the keys seen so far
// (2^-31 of it at the least: smaller ones round), P enters as f16 in [0, 2^15] (half step 2^-12 of a weight, below the
// bf16 output's 2^-9) or, for f32 outputs, as two f16 parts (2^-23).  bf16 V: P as two bf16 parts (2^-17).
// Maxima, sums and both products accumulate in f32.
#include <type_traits>

#include "fp8.h"

namespace {

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
  float *part, *part_ml;  // [unit][split][column][hd], [unit][split][column][maximum, sum]
};

constexpr int kPUp = 15;  // P is held times 2^15, V's codes times 2^7 relative to the largest scale: both within f16
constexpr int kVUp = 7;

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

// one tile of 32 keys as it comes from memory
template <bool E4M3, int HD>
struct Tile {
  static constexpr int KW = HD * (E4M3 ? 1 : 2) / 64;
  u32x4_t k[2][KW];   // K rows of keys r and 16 + r: 16-B pieces
  int ks[2];          // their scale bytes
  uint32_t v[8][KW];  // hd / 16 values of the lane's eight keys
  int vs[8];          // their scale bytes
  uint32_t bad;       // bit u: the lane's key u has a lineage entry outside the cache
};

// max over the four lanes that hold a column: lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ int max_rows(int v) {
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  const int w = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)w, (uint32_t)w, false, false);
  return max((int)b[0], (int)b[1]);
}

constexpr int kWaves = 4;  // waves of a workgroup take its tiles in turn

template <bool E4M3, int HD, int QN, int PN, int NQ>
__global__ __launch_bounds__(64 * kWaves) void attn_cached_kernel(AttnArgs a) {
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int KW = HD * ES / 64;  // 16-B pieces of K per lane and 16 keys; dwords of V per lane and key
  constexpr int KS = HD / 32;       // MFMA steps of the first product
  constexpr int DT = HD / 16;       // 16-dim tiles of the second
  constexpr int COLS = 16 * NQ;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c = lane >> 4;
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

  // this lane's columns, their masks and Q
  int col[NQ], tok[NQ];
  uint64_t msk[NQ];
  u32x4_t qf[NQ][KS][QN];
  float m[NQ];
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
      if (n < 64) msk[j] &= (1ull << max(n, 0)) - 1;
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
  int vref = 0;  // e4m3: V is held relative to 2^(vref - 127)

  const char* kbase = (const char*)a.c.k + (int64_t)h * a.c.hs * ES;
  const char* vbase = (const char*)a.c.v + (int64_t)h * a.c.hs * ES;
  const uint8_t* ksbase = E4M3 ? a.c.k_scale + (int64_t)h * a.c.shs : nullptr;
  const uint8_t* vsbase = E4M3 ? a.c.v_scale + (int64_t)h * a.c.shs : nullptr;
  const int last = a.c.max_kv - 1;
  // Loads stay within the cache by its capacity alone (positions at or behind the row's end are masked later), so the
  // first tile is requested without waiting for kv_len.
  auto load = [&](Tile<E4M3, HD>& t, int base) {
    t.bad = 0;
    if (a.kv_rows) {
      const int32_t* rows = a.kv_rows + (int64_t)b * a.ld_rows;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int p = min(base + 16 * f + r, last);
        const int row = rows[p];
        const int64_t at = (unsigned)row < (unsigned)a.c.rows ? row : 0;
        const char* src = kbase + (at * a.c.bs + (int64_t)p * HD) * ES + 16 * c;
#pragma unroll
        for (int i = 0; i < KW; ++i) t.k[f][i] = *reinterpret_cast<const u32x4_t*>(src + 64 * i);
        if constexpr (E4M3) t.ks[f] = ksbase[at * a.c.sbs + p];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = min(base + 4 * c + (u & 3) + 16 * (u >> 2), last);
        const int row = rows[p];
        const bool ok = (unsigned)row < (unsigned)a.c.rows;
        t.bad |= ok ? 0u : 1u << u;
        const int64_t at = ok ? row : 0;
        __builtin_memcpy(t.v[u], vbase + (at * a.c.bs + (int64_t)p * HD) * ES + 4 * KW * r, 4 * KW);
        if constexpr (E4M3) t.vs[u] = vsbase[at * a.c.sbs + p];
      }
      return;
    }
    const char* kr = kbase + (int64_t)b * a.c.bs * ES + 16 * c;
    const char* vr = vbase + (int64_t)b * a.c.bs * ES + 4 * KW * r;
    const uint8_t* ksr = ksbase + (int64_t)b * a.c.sbs;
    const uint8_t* vsr = vsbase + (int64_t)b * a.c.sbs;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int p = min(base + 16 * f + r, last);
#pragma unroll
      for (int i = 0; i < KW; ++i) t.k[f][i] = *reinterpret_cast<const u32x4_t*>(kr + p * (HD * ES) + 64 * i);
      if constexpr (E4M3) t.ks[f] = ksr[p];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = min(base + 4 * c + (u & 3) + 16 * (u >> 2), last);
      __builtin_memcpy(t.v[u], vr + p * (HD * ES), 4 * KW);
    }
    if constexpr (E4M3) {
      if (base + 31 <= last) {  // four neighbouring bytes at a time
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t w;
          __builtin_memcpy(&w, vsr + base + 16 * g + 4 * c, 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) t.vs[4 * g + i] = w >> (8 * i) & 0xFF;
        }
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) t.vs[u] = vsr[min(base + 4 * c + (u & 3) + 16 * (u >> 2), last)];
      }
    }
  };
  // V^T operands [16-dim tile][8 keys]; dim tile d holds the lane's dims (hd / 16) r + d
  auto v_frags = [&](const uint32_t (&v)[8][KW], const float (&sc)[8], u32x4_t (&vf)[DT]) {
#pragma unroll
    for (int i = 0; i < KW; ++i) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) {
        if constexpr (E4M3) {
          const uint32_t a0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u][i], sc[u], false));
          const uint32_t a1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u][i], sc[u], true));
          const uint32_t b0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u + 1][i], sc[u + 1], false));
          const uint32_t b1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u + 1][i], sc[u + 1], true));
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
  auto pv = [&](u32x4_t vf, u32x4_t pf, f32x4_t acc) -> f32x4_t {
    if constexpr (E4M3)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, vf), __builtin_bit_cast(f16x8_t, pf), acc, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, pf), acc, 0, 0, 0);
  };
  constexpr uint32_t kOne = E4M3 ? 0x3C00u : 0x3F80u;
  const u32x4_t ones = u32x4_t{kOne * 0x10001u, kOne * 0x10001u, kOne * 0x10001u, kOne * 0x10001u};

  // A drafted token's V that is not finite reaches only the columns that see it.  Such values enter the products as 0;
  // here a product of (1 where V is the special value) and (1 where the column sees the key) counts them.
  auto not_finite = [&](int base) {
    Tile<E4M3, HD> t;
    load(t, base);
#pragma unroll 1
    for (int kind = 0; kind < (E4M3 ? 1 : 3); ++kind) {
      float one[8];
      uint32_t ind[8][KW];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        one[u] = 1.f;
        const int p = base + 4 * c + (u & 3) + 16 * (u >> 2);
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t w = p >= len && p < hi ? t.v[u][i] : 0u;
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
      v_frags(ind, one, nf);
      const float what = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pf[e] = 0;
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            const int u = 2 * e + s2, p = base + 4 * c + (u & 3) + 16 * (u >> 2);
            if (p >= len && p < hi && (msk[j] >> ((p - len) & 63) & 1)) pf[e] |= kOne << (16 * s2);
          }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f32x4_t count = pv(nf[d], pf, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (count[i] > 0.f) o[j][d][i] += what;
        }
      }
    }
  };

  // EDGE: the tile holds keys that some column may not see (before the padding's end, drafted, behind the row's end)
  auto process = [&](Tile<E4M3, HD>& t, int base, auto edge_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    uint32_t some = 0xFF;  // which of the lane's eight keys some column may see
    uint32_t odd = 0;      // non-zero: V holds a NaN or infinity at a drafted token
    if constexpr (EDGE) {
      some = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = base + 4 * c + (u & 3) + 16 * (u >> 2);
        if (p < len ? p >= first : p < hi) some |= 1u << u;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t w = some >> u & 1 ? t.v[u][i] : 0u;
          uint32_t bits;  // a drafted token's values that are not finite
          if constexpr (E4M3) bits = (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
          else bits = (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 15;
          if (p < len) bits = 0;
          bits *= E4M3 ? 0xFFu : 0xFFFFu;
          odd |= bits;
          t.v[u][i] = w & ~bits;
        }
      }
    }
    float sv[8];
    float rescale = 1.f;
    if constexpr (E4M3) {
      int top = vref;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = max(top, !EDGE || some >> u & 1 ? t.vs[u] : 0);
      top = __builtin_amdgcn_readfirstlane(max_rows(top));  // 16 lanes each hold the same eight bytes
      if (top != vref) {
        rescale = vref == 0 ? 0.f : __builtin_amdgcn_exp2f((float)(vref - top));
        vref = top;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        sv[u] = !EDGE || some >> u & 1 ? __uint_as_float((uint32_t)max(t.vs[u] - vref + 127 + kVUp, 0) << 23) : 1.f;
    }
    u32x4_t vf[DT];
    v_frags(t.v, sv, vf);
    u32x4_t kf[2][KS];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if constexpr (E4M3) {
        const float sc = itts::e4m3_scale(t.ks[f]);
#pragma unroll
        for (int i = 0; i < KW; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            kf[f][2 * i + (w >> 1)][2 * (w & 1)] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t.k[f][i][w], sc, false));
            kf[f][2 * i + (w >> 1)][2 * (w & 1) + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t.k[f][i][w], sc, true));
          }
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[f][s] = t.k[f][s];
      }
    }
    const bool any_bad = __any(t.bad != 0);
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
            s[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[f][e]),
                                                           __builtin_bit_cast(bf16x8_t, qf[j][e][q]), s[f], 0, 0, 0);
      }
      float x[8];
      uint32_t vis = 0xFF;
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = s[u >> 2][u & 3];
      if constexpr (EDGE) {
        vis = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = base + 4 * c + (u & 3) + 16 * (u >> 2);
          const bool see = p < len ? p >= first : p < hi && (msk[j] >> ((p - len) & 63) & 1);
          vis |= (uint32_t)see << u;
        }
      }
      if (EDGE || any_bad) {
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = vis >> u & 1 ? (t.bad >> u & 1 ? __builtin_nanf("") : x[u]) : -__builtin_inff();
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      // m: of the scaled scores (a.qk_scale >= 0); -inf as long as the column has seen nothing
      top = fmaxf(m[j], EDGE && vis == 0 ? -__builtin_inff() : top * a.qk_scale);
      top = max_rows(top);
      const float ref = top == -__builtin_inff() ? 0.f : top;
      const float ra = __builtin_amdgcn_exp2f(m[j] - ref) * rescale;
      // the factors of O and of the sum differ where V's reference has changed
      if (__any(top > m[j]) || rescale != 1.f) {
        const float rl = __builtin_amdgcn_exp2f(m[j] - ref);
        l[j] = l[j] * rl;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[j][d] = o[j][d] * ra;
      }
      m[j] = top;
      float p[8];
      const float shift = (float)kPUp - ref;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float z = EDGE ? (vis >> u & 1 ? fmaf(x[u], a.qk_scale, shift) : -__builtin_inff()) : fmaf(x[u], a.qk_scale, shift);
        p[u] = __builtin_amdgcn_exp2f(z);
      }
#pragma unroll
      for (int q = 0; q < PN; ++q) {
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (E4M3) {
            const f16x2_t w = {(_Float16)p[2 * e], (_Float16)p[2 * e + 1]};
            pf[e] = __builtin_bit_cast(uint32_t, w);
            if (q + 1 < PN) p[2 * e] -= (float)w[0], p[2 * e + 1] -= (float)w[1];
          } else {
            const uint32_t w = pack2bf(p[2 * e], p[2 * e + 1]);
            pf[e] = w;
            if (q + 1 < PN) p[2 * e] -= __uint_as_float(w << 16), p[2 * e + 1] -= __uint_as_float(w & 0xFFFF0000u);
          }
        }
        l[j] = pv(ones, pf, l[j]);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[j][d] = pv(vf[d], pf, o[j][d]);
      }
    }
    if constexpr (EDGE) {
      if (__any(odd != 0)) not_finite(base);
    }
  };

  {
    Tile<E4M3, HD> cur, nxt;
    int base = begin + 32 * wave;
    if (base <= last) load(cur, base);
    while (base < end) {
      const int next = base + 32 * kWaves;
      if (next < end) load(nxt, next);
      if (base < first || base + 32 > len) process(cur, base, std::true_type{});
      else process(cur, base, std::false_type{});
      cur = nxt;
      base = next;
    }
  }

  // ---- the waves' parts: common maximum and V reference, then O and the sums added in wave order ----
  constexpr int LDC = HD + 4;
  __shared__ float so[kWaves][COLS][LDC];
  __shared__ float sm[kWaves][COLS], sl[kWaves][COLS];
  __shared__ int sr[kWaves];
  if (lane == 0) sr[wave] = vref;
  if (c == 0) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) sm[wave][16 * j + r] = m[j];
  }
  __syncthreads();
  int top_ref = 0;
  if constexpr (E4M3) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top_ref = max(top_ref, sr[w]);
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    if (col[j] >= C) continue;
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm[w][16 * j + r]);
    const float fl = top == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[j] - top);
    const float fo = E4M3 ? fl * __builtin_amdgcn_exp2f((float)(vref - top_ref)) : fl;
    if (c == 0) sl[wave][16 * j + r] = l[j][0] * fl;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < DT; d += 4)
        *reinterpret_cast<f32x4_t*>(&so[wave][16 * j + r][(4 * c + i) * DT + d]) =
            f32x4_t{o[j][d][i] * fo, o[j][d + 1][i] * fo, o[j][d + 2][i] * fo, o[j][d + 3][i] * fo};
  }
  __syncthreads();
  const float vscale = E4M3 ? __builtin_amdgcn_exp2f((float)(top_ref - 127 - kVUp)) : 1.f;
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
      const int64_t at = ((int64_t)unit * a.nsplit + split) * C + cg;
      *reinterpret_cast<f32x4_t*>(a.part + at * HD + d) = acc * vscale;
      if (d == 0) {
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm[w][cl]);
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = sum;
      }
    } else {
      const int t = cg / G;
      if (!refuse && t >= nt) continue;
      const float inv = refuse ? __builtin_nanf("") : sum == 0.f ? 0.f : vscale / sum;
      store4(a, (int64_t)b * a.o_sb + t * a.o_st + (int64_t)(h * G + cg - t * G) * a.o_sh + d, acc * inv);
    }
  }
}

// the splits' parts of one column: common maximum, O and the sums added in split order; one wave per column
template <int HD>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  const int C = a.T * a.G;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int unit = (int)(id / C), cg = (int)(id - (int64_t)unit * C);
  if (unit >= a.units) return;
  const int b = unit / a.c.heads, h = unit - b * a.c.heads;
  const int t = cg / a.G;
  const int len = a.kv_len[b];
  const int n = a.tree ? (a.n_tokens ? a.n_tokens[b] : a.T) : 0;
  const bool refuse = len < 0 || n < 0 || n > a.T || len > a.c.max_kv - n;
  if (!refuse && t >= (a.tree ? n : 1)) return;
  // lane = (quarter or half of the splits, 4 dims)
  constexpr int L = HD / 4, P = 64 / L;
  const int d = 4 * (lane % L), g = lane / L;
  float top = -__builtin_inff();
  for (int s = lane; s < a.nsplit; s += 64) top = fmaxf(top, a.part_ml[2 * (((int64_t)unit * a.nsplit + s) * C + cg)]);
  top = wave_max(top);
  const float ref = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < a.nsplit; s += P) {
    const int64_t at = ((int64_t)unit * a.nsplit + s) * C + cg;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
    sum += f * a.part_ml[2 * at + 1];
    acc = acc + *reinterpret_cast<const f32x4_t*>(a.part + at * HD + d) * f;
  }
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
    sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
  }
  if (g != 0) return;
  const float inv = refuse ? __builtin_nanf("") : sum == 0.f ? 0.f : 1.f / sum;
  store4(a, (int64_t)b * a.o_sb + t * a.o_st + (int64_t)(h * a.G + cg - t * a.G) * a.o_sh + d, acc * inv);
}

// columns of 16 that one wave takes at once, by their number and what fits the registers (three parts of an f32 q in 128
// dims: two)
int query_tiles(int cols, bool q_f32, int hd) { return cols <= 16 ? 1 : cols <= 32 || (q_f32 && hd == 128) ? 2 : 4; }
int query_blocks(int cols, bool q_f32, int hd) {
  const int per = 16 * query_tiles(cols, q_f32, hd);
  return (cols + per - 1) / per;
}
// Splits over the keys: enough workgroups for two on each of the 256 CUs, none with fewer than 512 keys of the expected
// longest row (each wave then has four tiles to keep the next one's loads in flight).
int splits(int64_t workgroups, int max_len) {
  const int64_t want = (512 + workgroups - 1) / (workgroups > 0 ? workgroups : 1);
  const int64_t most = (max_len + 511) / 512;
  return (int)(want < most ? (want > 1 ? want : 1) : (most > 1 ? most : 1));
}

template <bool E4M3, int HD, int QN, int PN, int NQ>
void launch(const AttnArgs& a, hipStream_t s) {
  const int64_t us = ((int64_t)a.units * a.nsplit + 7) / 8 * 8;
  hipLaunchKernelGGL((attn_cached_kernel<E4M3, HD, QN, PN, NQ>), dim3((unsigned)(us * a.qblocks)), dim3(64 * kWaves), 0, s, a);
}
template <bool E4M3, int HD, int QN, int PN>
void launch_nq(const AttnArgs& a, int nq, hipStream_t s) {
  if (nq == 1) launch<E4M3, HD, QN, PN, 1>(a, s);
  else if (nq == 2) launch<E4M3, HD, QN, PN, 2>(a, s);
  else if constexpr (!(QN == 3 && HD == 128)) launch<E4M3, HD, QN, PN, 4>(a, s);
}
template <int HD>
void launch_types(const AttnArgs& a, int nq, hipStream_t s) {
  if (a.c.dtype == ITTS_E4M3) {
    if (a.q_f32) {
      if (a.out_f32) launch_nq<true, HD, 3, 2>(a, nq, s);
      else launch_nq<true, HD, 3, 1>(a, nq, s);
    } else {
      if (a.out_f32) launch_nq<true, HD, 1, 2>(a, nq, s);
      else launch_nq<true, HD, 1, 1>(a, nq, s);
    }
  } else {
    if (a.q_f32) launch_nq<false, HD, 3, 2>(a, nq, s);
    else launch_nq<false, HD, 1, 2>(a, nq, s);
  }
  if (a.nsplit > 1) {
    const int64_t cols = (int64_t)a.units * a.T * a.G;
    hipLaunchKernelGGL((attn_join_kernel<HD>), dim3((unsigned)((cols + 3) / 4)), dim3(256), 0, s, a);
  }
}

int attend(const char* fn, AttnArgs& a, int B, int q_dtype, int out_dtype, int max_len, void* workspace, void* stream) {
  ITTS_REQUIRE(q_dtype == ITTS_F32 || q_dtype == ITTS_BF16, fn, "q must be f32 or bf16");
  ITTS_REQUIRE(out_dtype == ITTS_BF16 || (out_dtype == ITTS_F32 && a.c.dtype == ITTS_E4M3), fn,
               "out must be bf16, or f32 over an e4m3 cache");
  const int64_t need = itts_attn_cached_workspace_bytes(&a.c, B, a.T, a.G, max_len, q_dtype);
  ITTS_REQUIRE(need >= 0, fn, "bad sizes (1 <= T <= 64, 1 <= group <= 4096, rows x heads x query blocks of one launch)");
  ITTS_REQUIRE(a.kv_rows ? a.ld_rows >= a.c.max_kv || B <= 1 : B <= a.c.rows, fn,
               "more rows than the cache holds, or a short lineage table");
  ITTS_REQUIRE(a.qk_scale == a.qk_scale && a.qk_scale - a.qk_scale == 0.f, fn, "the scale must be finite");
  if (B == 0) return 0;
  ITTS_REQUIRE(a.q && a.kv_len && a.out, fn, "null pointer");
  ITTS_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0), fn, "null or misaligned workspace");
  const int cols = a.T * a.G, hd = a.c.head_dim;
  const int qs = a.q_f32 ? 4 : 2, os = a.out_f32 ? 4 : 2;
  a.negate = a.qk_scale < 0.f;
  a.qk_scale = a.negate ? -a.qk_scale : a.qk_scale;
  a.q_vec = ((uintptr_t)a.q & 15) == 0 && ((a.q_sb | a.q_st | a.q_sh) * qs) % 16 == 0;
  a.o_vec = ((uintptr_t)a.out & 15) == 0 && ((a.o_sb | a.o_st | a.o_sh) * os) % 16 == 0;
  a.units = B * a.c.heads;
  a.qblocks = query_blocks(cols, a.q_f32, hd);
  a.nsplit = splits((int64_t)a.units * a.qblocks, max_len);
  a.part = (float*)workspace;
  a.part_ml = a.part + (int64_t)a.units * a.nsplit * cols * hd;
  const int nq = query_tiles(cols, a.q_f32, hd);
  if (hd == 64) launch_types<64>(a, nq, itts::as_stream(stream));
  else launch_types<128>(a, nq, itts::as_stream(stream));
  return itts::check_launch(fn);
}

}  // namespace

extern "C" int64_t itts_attn_cached_workspace_bytes(const ItTsKvCache* c, int B, int T, int group, int max_len, int q_dtype) {
  if (itts::check_kv_cache("itts_attn_cached_workspace_bytes", c) || B < 0 || T < 1 || T > 64 || group < 1 ||
      group > 4096 || max_len < 0 || (q_dtype != ITTS_F32 && q_dtype != ITTS_BF16))
    return -1;
  const int64_t units = (int64_t)B * c->heads, cols = (int64_t)T * group;
  const int qblocks = query_blocks((int)cols, q_dtype == ITTS_F32, c->head_dim);
  const int nsplit = splits(units * qblocks, max_len);
  if ((units * nsplit + 7) * qblocks > 0x7FFFFF00 || units * cols > 0x7FFFFF00) return -1;
  return nsplit > 1 ? units * nsplit * cols * (c->head_dim + 2) * 4 : 0;
}

extern "C" int itts_attn_decode_kv8(const ItTsKvCache* c, const void* q, int64_t q_sb, int64_t q_sh, int q_dtype, int B,
                                    int group, const int32_t* kv_len, const int32_t* pad, const int32_t* kv_rows,
                                    int64_t ld_rows, float scale, int max_len, void* out, int64_t o_sb, int64_t o_sh,
                                    int out_dtype, void* workspace, void* stream) {
  const char* fn = "itts_attn_decode_kv8";
  if (int rc = itts::check_kv_cache(fn, c)) return rc;
  ITTS_REQUIRE(c->dtype == ITTS_E4M3, fn, "the cache must hold e4m3 codes");
  AttnArgs a{*c, q, q_sb, 0, q_sh, q_dtype == ITTS_F32, false, out_dtype == ITTS_F32, 1, group, kv_len, pad, nullptr,
             kv_rows, ld_rows, nullptr, 0, scale * 1.4426950408889634f, out, o_sb, 0, o_sh};
  return attend(fn, a, B, q_dtype, out_dtype, max_len, workspace, stream);
}

extern "C" int itts_attn_tree(const ItTsKvCache* c, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int q_dtype,
                              int B, int T, int group, const int32_t* kv_len, const int32_t* pad, const int32_t* n_tokens,
                              const uint64_t* mask, int64_t mask_sb, const int32_t* kv_rows, int64_t ld_rows, float scale,
                              int max_len, void* out, int64_t o_sb, int64_t o_st, int64_t o_sh, int out_dtype,
                              void* workspace, void* stream) {
  const char* fn = "itts_attn_tree";
  if (int rc = itts::check_kv_cache(fn, c)) return rc;
  ITTS_REQUIRE(mask || B == 0, fn, "null mask");
  AttnArgs a{*c, q, q_sb, q_st, q_sh, q_dtype == ITTS_F32, true, out_dtype == ITTS_F32, T, group, kv_len, pad, n_tokens,
             kv_rows, ld_rows, mask, mask_sb, scale * 1.4426950408889634f, out, o_sb, o_st, o_sh};
  return attend(fn, a, B, q_dtype, out_dtype, max_len, workspace, stream);
}
