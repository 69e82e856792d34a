// The C entries of attention over a cache (kernels: attn_cached.h): argument checks, the split over keys, the join of
// the splits' parts.
#include <cfloat>
#include <cmath>

#include "attn_cached.h"

namespace {

using namespace itts::attn;

// the splits' results of one column, each times its share of the weights, added in split order; one wave per column
template <int HD>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  const int C = a.T * a.G;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int unit = (int)(id / C), cg = (int)(id - (int64_t)unit * C);
  if (unit >= a.units) return;
  const int b = unit / a.c.heads, h = unit - b * a.c.heads;
  // lane = (quarter or half of the splits, 4 dims); the first splits' parts are requested before anything else is known
  constexpr int L = HD / 4, P = 64 / L, EARLY = 4;
  const int d = 4 * (lane % L), g = lane / L;
  const int64_t base = (int64_t)unit * a.nsplit * C + cg;
  auto at = [&](int s) { return base + (int64_t)s * C; };
  f32x4_t early[EARLY];
  float em[EARLY], el[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) {
    const int64_t e = at(min(g + P * i, a.nsplit - 1));
    early[i] = *reinterpret_cast<const f32x4_t*>(a.part + e * HD + d);
    em[i] = a.part_ml[2 * e];
    el[i] = a.part_ml[2 * e + 1];
  }
  const int t = cg / a.G;
  const int len = a.kv_len[b];
  const int n = a.tree ? (a.n_tokens ? a.n_tokens[b] : a.T) : 0;
  const bool refuse = len < 0 || n < 0 || n > a.T || len > a.c.max_kv - n;
  if (!refuse && t >= (a.tree ? n : 1)) return;
  float top = -__builtin_inff();
  for (int s = lane; s < a.nsplit; s += 64) top = fmaxf(top, a.part_ml[2 * at(s)]);
  top = wave_max(top);
  const float ref = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  for (int s = lane; s < a.nsplit; s += 64)
    sum += __builtin_amdgcn_exp2f(a.part_ml[2 * at(s)] - ref) * a.part_ml[2 * at(s) + 1];
  sum = wave_sum(sum);
  const float inv = refuse ? __builtin_nanf("") : inverse_sum(a, sum, b, t, len, n);
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (g + P * i < a.nsplit) acc = acc + early[i] * (__builtin_amdgcn_exp2f(em[i] - ref) * el[i] * inv);
  for (int s = g + P * EARLY; s < a.nsplit; s += P)
    acc = acc + *reinterpret_cast<const f32x4_t*>(a.part + at(s) * HD + d) *
                    (__builtin_amdgcn_exp2f(a.part_ml[2 * at(s)] - ref) * a.part_ml[2 * at(s) + 1] * inv);
#pragma unroll
  for (int o = L; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
  if (g != 0) return;
  store4(a, (int64_t)b * a.o_sb + t * a.o_st + (int64_t)(h * a.G + cg - t * a.G) * a.o_sh + d, acc);
}

int query_blocks(bool e4m3, int cols, bool q_f32, int hd) {
  const int per = 16 * query_tiles(e4m3, cols, q_f32, hd);
  return (cols + per - 1) / per;
}
// Splits over the keys: enough workgroups for two on each of the 256 CUs, none with fewer than 512 keys of the expected
// longest row (each wave then has four tiles to keep the next one's loads in flight).  Measured, us (kernel + join, with 512
// / 1024 / 2048 workgroups wanted): 8 x 4 heads over 32749 keys 46 + 5 / 46 + 7 / 52 + 11, 64 tokens of 4 x 8 heads over
// 16301 keys 125 + 6 / 124 + 7 / 139 + 9; 32 x 16 heads over 565 keys unsplit 14, in two 17 + 6.
int splits(int64_t workgroups, int max_len) {
  const int64_t want = (512 + workgroups - 1) / (workgroups > 0 ? workgroups : 1);
  const int64_t most = (max_len + 511) / 512;
  return (int)(want < most ? (want > 1 ? want : 1) : (most > 1 ? most : 1));
}

int attend(const char* fn, AttnArgs& a, int B, int q_dtype, int out_dtype, int max_len, void* workspace, void* stream) {
  ITTS_REQUIRE(q_dtype == ITTS_F32 || q_dtype == ITTS_BF16, fn, "q must be f32 or bf16");
  ITTS_REQUIRE(out_dtype == ITTS_BF16 || (out_dtype == ITTS_F32 && a.c.dtype == ITTS_E4M3), fn,
               "out must be bf16, or f32 over an e4m3 cache");
  const int64_t need = itts_attn_cached_workspace_bytes(&a.c, B, a.T, a.G, max_len, q_dtype);
  ITTS_REQUIRE(need >= 0, fn, "bad sizes (1 <= T <= 64, 1 <= group <= 4096, rows x heads x query blocks of one launch)");
  ITTS_REQUIRE(a.kv_rows ? a.ld_rows >= a.c.max_kv || a.ld_rows == 0 : B <= a.c.rows, fn,
               "more rows than the cache holds, or a short lineage table");
  ITTS_REQUIRE(a.qk_scale == a.qk_scale && a.qk_scale - a.qk_scale == 0.f, fn, "the scale must be finite");
  if (B == 0) return 0;
  ITTS_REQUIRE(a.q && a.kv_len && a.out, fn, "null pointer");
  ITTS_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0), fn, "null or misaligned workspace");
  const int cols = a.T * a.G, hd = a.c.head_dim;
  const int qs = a.q_f32 ? 4 : 2, os = a.out_f32 ? 4 : 2;
  a.negate = a.qk_scale < 0.f;
  a.qk_scale = fmaxf(fabsf(a.qk_scale), FLT_MIN);  // 0: every score is 0 but for what underflows, and -inf stays -inf
  a.q_vec = ((uintptr_t)a.q & 15) == 0 && ((a.q_sb | a.q_st | a.q_sh) * qs) % 16 == 0;
  a.o_vec = ((uintptr_t)a.out & 15) == 0 && ((a.o_sb | a.o_st | a.o_sh) * os) % 16 == 0;
  a.units = B * a.c.heads;
  a.qblocks = query_blocks(a.c.dtype == ITTS_E4M3, cols, a.q_f32, hd);
  a.nsplit = splits((int64_t)a.units * a.qblocks, max_len);
  a.part = (float*)workspace;
  a.part_ml = a.part + (int64_t)a.units * a.nsplit * cols * hd;
  hipStream_t s = itts::as_stream(stream);
  if (a.c.dtype == ITTS_E4M3) {
    if (hd == 64) launch_attn<true, 64>(a, s);
    else launch_attn<true, 128>(a, s);
  } else {
    if (hd == 64) launch_attn<false, 64>(a, s);
    else launch_attn<false, 128>(a, s);
  }
  if (a.nsplit > 1) {
    const unsigned g = (unsigned)(((int64_t)a.units * cols + 3) / 4);
    if (hd == 64) hipLaunchKernelGGL(attn_join_kernel<64>, dim3(g), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(attn_join_kernel<128>, dim3(g), dim3(256), 0, s, a);
  }
  return itts::check_launch(fn);
}

}  // namespace

extern "C" int64_t itts_attn_cached_workspace_bytes(const ItTsKvCache* c, int B, int T, int group, int max_len, int q_dtype) {
  if (itts::check_kv_cache("itts_attn_cached_workspace_bytes", c) || B < 0 || T < 1 || T > 64 || group < 1 ||
      group > 4096 || max_len < 0 || (q_dtype != ITTS_F32 && q_dtype != ITTS_BF16))
    return -1;
  const int64_t units = (int64_t)B * c->heads, cols = (int64_t)T * group;
  const int qblocks = query_blocks(c->dtype == ITTS_E4M3, (int)cols, q_dtype == ITTS_F32, c->head_dim);
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
