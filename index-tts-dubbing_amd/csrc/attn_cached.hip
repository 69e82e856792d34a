// Attention of one new token (itts_attn_decode_kv8) or of a tree of drafted tokens (itts_attn_tree) per row over a KV
// cache in block-scaled e4m3 (fp8.h) or bf16.
//
// One wave walks a row and K/V head's keys in tiles of 32, with up to NQ x 16 query columns (column = drafted token *
// group + query head of the group), everything in registers:
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
  int T, G, qblocks;
  const int32_t *kv_len, *pad, *n_tokens, *kv_rows;
  int64_t ld_rows;
  const uint64_t* mask;
  int64_t mask_sb;
  float qk_scale;  // scale * log2(e)
  void* out;
  int64_t o_sb, o_st, o_sh;
};

constexpr int kPUp = 15;  // P is held times 2^15, V's codes times 2^7 relative to the largest scale: both within f16
constexpr int kVUp = 7;

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
// low / high halves of two dwords
__device__ __forceinline__ uint32_t lo16(uint32_t a, uint32_t b) { return perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t hi16(uint32_t a, uint32_t b) { return perm(b, a, 0x07060302u); }

template <typename V8>
__device__ __forceinline__ V8 as8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(V8, u32x4_t{a, b, c, d});
}

// one tile of 32 keys as it comes from memory
template <bool E4M3, int HD>
struct Tile {
  static constexpr int ES = E4M3 ? 1 : 2;
  u32x4_t k[2][HD * ES / 64];      // K rows of keys r and 16 + r: 16-B pieces
  int ks[2];                       // their scale bytes
  uint32_t v[8][HD * ES / 64];     // hd / 16 values of the lane's eight keys
  int vs[8];
  uint32_t bad;                    // bit u: the lane's key u has a lineage entry outside the cache
};

template <bool E4M3, int HD, int QN, int PN, int NQ>
__global__ __launch_bounds__(64) void attn_cached_kernel(AttnArgs a) {
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int KW = HD * ES / 64;  // 16-B pieces of K per lane and 16 keys; dwords of V per lane and key
  constexpr int KS = HD / 32;       // MFMA steps of the first product
  constexpr int DT = HD / 16;       // 16-dim tiles of the second
  const int lane = threadIdx.x, r = lane & 15, c = lane >> 4;
  const int h = blockIdx.y;
  const int b = blockIdx.z / a.qblocks, qb = blockIdx.z - b * a.qblocks;
  const int G = a.G, C = a.T * G;

  const int len = a.kv_len[b];
  const int n = a.tree ? (a.n_tokens ? a.n_tokens[b] : a.T) : 0;
  const bool refuse = len < 0 || n < 0 || n > a.T || len > a.c.max_kv - n;
  const int first = a.pad ? max(a.pad[b], 0) : 0;
  const int hi = len + n;
  const int nt = a.tree ? n : 1;  // tokens that have an output

  // this lane's columns, their masks and Q
  int col[NQ], tok[NQ];
  uint64_t msk[NQ];
  u32x4_t qf[NQ][KS][QN];
  float m[NQ], l[NQ];
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
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x0, x1;
        if (a.q_f32) {
          x0 = ((const float*)a.q)[off + d0 + 2 * e];
          x1 = ((const float*)a.q)[off + d0 + 2 * e + 1];
        } else {
          x0 = bf2f(((const uint16_t*)a.q)[off + d0 + 2 * e]);
          x1 = bf2f(((const uint16_t*)a.q)[off + d0 + 2 * e + 1]);
        }
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
    l[j] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[j][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  int vref = 0;  // e4m3: V is held relative to 2^(vref - 127)

  const char* kbase = (const char*)a.c.k + (int64_t)h * a.c.hs * ES;
  const char* vbase = (const char*)a.c.v + (int64_t)h * a.c.hs * ES;
  auto cache_row = [&](int p, bool& bad) -> int64_t {
    int row = b;
    if (a.kv_rows) {
      row = a.kv_rows[(int64_t)b * a.ld_rows + p];
      bad = (unsigned)row >= (unsigned)a.c.rows;
      if (bad) row = 0;
    }
    return row;
  };
  auto load = [&](Tile<E4M3, HD>& t, int base) {
    bool bad = false;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int p = min(base + 16 * f + r, hi - 1);
      const int64_t row = cache_row(p, bad);
      const char* src = kbase + (row * a.c.bs + (int64_t)p * HD) * ES + 16 * c;
#pragma unroll
      for (int i = 0; i < KW; ++i) t.k[f][i] = *reinterpret_cast<const u32x4_t*>(src + 64 * i);
      if constexpr (E4M3) t.ks[f] = a.c.k_scale[row * a.c.sbs + h * a.c.shs + p];
    }
    t.bad = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = min(base + 4 * c + (u & 3) + 16 * (u >> 2), hi - 1);
      bad = false;
      const int64_t row = cache_row(p, bad);
      t.bad |= (uint32_t)bad << u;
      const char* src = vbase + (row * a.c.bs + (int64_t)p * HD) * ES + 4 * KW * r;
      if constexpr (KW == 1) t.v[u][0] = *reinterpret_cast<const uint32_t*>(src);
      else if constexpr (KW == 2) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(src);
        t.v[u][0] = w[0], t.v[u][1] = w[1];
      } else {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.v[u][i] = w[i];
      }
      if constexpr (E4M3) t.vs[u] = a.c.v_scale[row * a.c.sbs + h * a.c.shs + p];
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

  auto process = [&](Tile<E4M3, HD>& t, int base) {
    const bool edge = base < first || base + 32 > len;
    // which of the lane's eight keys some column may see, and what is not finite among the drafted tokens' V
    uint32_t some = 0xFF;
    uint32_t odd = 0;  // non-zero: V holds a NaN or infinity at a drafted token
    uint32_t ov[8][KW];
    if (edge) {
      some = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = base + 4 * c + (u & 3) + 16 * (u >> 2);
        if (p < len ? p >= first : p < hi) some |= 1u << u;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          uint32_t w = some >> u & 1 ? t.v[u][i] : 0u;
          uint32_t bits;  // a drafted token's values that are not finite
          if constexpr (E4M3) bits = (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
          else bits = (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 15;
          if (p < len) bits = 0;
          bits *= E4M3 ? 0xFFu : 0xFFFFu;
          ov[u][i] = w & bits;
          odd |= bits;
          t.v[u][i] = w & ~bits;
        }
      }
    }
    // K's operands, and S^T
    float sv[8];
    float rescale = 1.f;
    if constexpr (E4M3) {
      int top = vref;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = max(top, some >> u & 1 ? t.vs[u] : 0);
      top = max(top, __shfl_xor(top, 16, 64));
      top = max(top, __shfl_xor(top, 32, 64));
      rescale = vref == 0 ? 0.f : exp2f((float)(vref - top));
      vref = top;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        sv[u] = some >> u & 1 ? __uint_as_float((uint32_t)max(t.vs[u] - vref + 127 + kVUp, 0) << 23) : 1.f;
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
      for (int u = 0; u < 8; ++u) x[u] = s[u >> 2][u & 3] * a.qk_scale;
      if (edge) {
        vis = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = base + 4 * c + (u & 3) + 16 * (u >> 2);
          const bool see = p < len ? p >= first : p < hi && (msk[j] >> ((p - len) & 63) & 1);
          vis |= (uint32_t)see << u;
        }
      }
      if (edge || t.bad) {
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = vis >> u & 1 ? (t.bad >> u & 1 ? __builtin_nanf("") : x[u]) : -__builtin_inff();
      }
      float top = m[j];
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, x[u]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float ref = top == -__builtin_inff() ? 0.f : top;
      const float alpha = exp2f(m[j] - ref);
      m[j] = top;
      float p[8];
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        p[u] = exp2f(x[u] - ref + (float)kPUp);
        sum += p[u];
      }
      l[j] = l[j] * alpha + sum;
      const float ra = alpha * rescale;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[j][d] = o[j][d] * ra;
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
#pragma unroll
        for (int d = 0; d < DT; ++d) o[j][d] = pv(vf[d], pf, o[j][d]);
      }
      // a drafted token's V that is not finite reaches only the columns that see it: count them by a third product,
      // 1 where V is the special value times 1 where the column sees the key
      if (__any(odd != 0)) {
        constexpr uint32_t kOne = E4M3 ? 0x3C00u : 0x3F80u;
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[e] = (vis >> (2 * e) & 1 ? kOne : 0u) | (vis >> (2 * e + 1) & 1 ? kOne << 16 : 0u);
        for (int kind = 0; kind < (E4M3 ? 1 : 3); ++kind) {
          uint32_t ind[8][KW];
          float one[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            one[u] = 1.f;
#pragma unroll
            for (int i = 0; i < KW; ++i) {
              const uint32_t w = ov[u][i];
              if constexpr (E4M3) {
                ind[u][i] = ((((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0x38u;  // e4m3 1.0
              } else {
                uint32_t v = 0;
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                  const uint32_t x16 = w >> (16 * s2) & 0xFFFFu;
                  const int is = (x16 & 0x7F80u) != 0x7F80u ? -1 : (x16 & 0x7Fu) ? 0 : x16 >> 15 ? 2 : 1;
                  if (is == kind) v |= kOne << (16 * s2);
                }
                ind[u][i] = v;
              }
            }
          }
          u32x4_t nf[DT];
          v_frags(ind, one, nf);
          const float what = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const f32x4_t count = pv(nf[d], pf, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (count[i] > 0.f) o[j][d][i] += what;
          }
        }
      }
    }
  };

  if (!refuse) {
    Tile<E4M3, HD> t;
    // the prefix from pad on, then the drafted tokens; an empty prefix starts at the tile of kv_len
    for (int base = min(first, len) & ~31; base < hi; base += 32) {
      load(t, base);
      process(t, base);
    }
  }

  const float vscale = E4M3 ? exp2f((float)(vref - 127 - kVUp)) : 1.f;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    float sum = l[j];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (col[j] >= C || (!refuse && tok[j] >= nt)) continue;
    const float inv = sum == 0.f ? 0.f : vscale / sum;
    const int64_t off = (int64_t)b * a.o_sb + tok[j] * a.o_st + (int64_t)(h * G + col[j] - tok[j] * G) * a.o_sh;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const float y = refuse ? __builtin_nanf("") : o[j][d][i] * inv;
        const int64_t at = off + (4 * c + i) * DT + d;
        if (a.out_f32) ((float*)a.out)[at] = y;
        else ((uint16_t*)a.out)[at] = f2bf(y);
      }
  }
}

template <bool E4M3, int HD, int QN, int PN, int NQ>
void launch(const AttnArgs& a, int B, hipStream_t s) {
  AttnArgs p = a;
  p.qblocks = (a.T * a.G + 16 * NQ - 1) / (16 * NQ);
  hipLaunchKernelGGL((attn_cached_kernel<E4M3, HD, QN, PN, NQ>), dim3(1, a.c.heads, B * p.qblocks), dim3(64), 0, s, p);
}
template <bool E4M3, int HD, int QN, int PN>
void launch_nq(const AttnArgs& a, int B, hipStream_t s) {
  const int cols = a.T * a.G;
  if (cols <= 16) launch<E4M3, HD, QN, PN, 1>(a, B, s);
  else if (cols <= 32 || (QN == 3 && HD == 128)) launch<E4M3, HD, QN, PN, 2>(a, B, s);
  else if constexpr (!(QN == 3 && HD == 128)) launch<E4M3, HD, QN, PN, 4>(a, B, s);
}
template <int HD>
void launch_types(const AttnArgs& a, int B, hipStream_t s) {
  if (a.c.dtype == ITTS_E4M3) {
    if (a.out_f32) launch_nq<true, HD, 3, 2>(a, B, s);
    else if (a.q_f32) launch_nq<true, HD, 3, 1>(a, B, s);
    else launch_nq<true, HD, 1, 1>(a, B, s);
  } else {
    if (a.q_f32) launch_nq<false, HD, 3, 2>(a, B, s);
    else launch_nq<false, HD, 1, 2>(a, B, s);
  }
}

int attend(const char* fn, const AttnArgs& a, int B, int q_dtype, int out_dtype, int max_len, void* workspace,
           void* stream) {
  ITTS_REQUIRE(q_dtype == ITTS_F32 || q_dtype == ITTS_BF16, fn, "q must be f32 or bf16");
  ITTS_REQUIRE(out_dtype == ITTS_BF16 || (out_dtype == ITTS_F32 && a.c.dtype == ITTS_E4M3), fn,
               "out must be bf16, or f32 over an e4m3 cache");
  ITTS_REQUIRE(B >= 0 && a.T >= 1 && a.T <= 64 && a.G >= 1 && a.G <= 4096 && max_len >= 0, fn, "bad sizes");
  ITTS_REQUIRE(a.kv_rows ? a.ld_rows >= a.c.max_kv || B <= 1 : B <= a.c.rows, fn,
               "more rows than the cache holds, or a short lineage table");
  ITTS_REQUIRE((int64_t)B * ((a.T * a.G + 15) / 16) <= 65535, fn, "too many rows for one launch");
  if (B == 0) return 0;
  ITTS_REQUIRE(a.q && a.kv_len && a.out, fn, "null pointer");
  if (a.c.head_dim == 64) launch_types<64>(a, B, itts::as_stream(stream));
  else launch_types<128>(a, B, itts::as_stream(stream));
  return itts::check_launch(fn);
}

}  // namespace

extern "C" int64_t itts_attn_cached_workspace_bytes(const ItTsKvCache* c, int B, int T, int group, int max_len, int q_dtype) {
  if (itts::check_kv_cache("itts_attn_cached_workspace_bytes", c) || B < 0 || T < 1 || T > 64 || group < 1 ||
      group > 4096 || max_len < 0 || (q_dtype != ITTS_F32 && q_dtype != ITTS_BF16))
    return -1;
  return 0;
}

extern "C" int itts_attn_decode_kv8(const ItTsKvCache* c, const void* q, int64_t q_sb, int64_t q_sh, int q_dtype, int B,
                                    int group, const int32_t* kv_len, const int32_t* pad, const int32_t* kv_rows,
                                    int64_t ld_rows, float scale, int max_len, void* out, int64_t o_sb, int64_t o_sh,
                                    int out_dtype, void* workspace, void* stream) {
  const char* fn = "itts_attn_decode_kv8";
  if (int rc = itts::check_kv_cache(fn, c)) return rc;
  ITTS_REQUIRE(c->dtype == ITTS_E4M3, fn, "the cache must hold e4m3 codes");
  AttnArgs a{*c, q, q_sb, 0, q_sh, q_dtype == ITTS_F32, false, out_dtype == ITTS_F32, 1, group, 1, kv_len, pad, nullptr,
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
  AttnArgs a{*c, q, q_sb, q_st, q_sh, q_dtype == ITTS_F32, true, out_dtype == ITTS_F32, T, group, 1, kv_len, pad, n_tokens,
             kv_rows, ld_rows, mask, mask_sb, scale * 1.4426950408889634f, out, o_sb, o_st, o_sh};
  return attend(fn, a, B, q_dtype, out_dtype, max_len, workspace, stream);
}
