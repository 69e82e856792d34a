// The 8-bit KV cache: K and V of a token quantised as they are written (one power-of-two scale per token, head and
// K or V over the head's hd values, fp8.h), and read back.  Layout beside the bf16 cache's: codes [row][head][pos][hd],
// scale bytes [row][head][pos].
//
// Pure traffic: a token and head reads hd values and writes hd + 1 bytes for each of K and V.  hd / 8 lanes per vector,
// eight values per lane, so a lane's 16-B (bf16) or 32-B (f32) load becomes one 8-B store.
#include "fp8.h"

namespace {

using itts::e4m3_inv_scale;
using itts::e4m3_pack4;
using itts::e4m3_prescale;
using itts::e4m3_scale;
using itts::e4m3_scale_byte;
using itts::finite_f;

struct Kv8Args {
  ItTsKvCache c;
  const void *k, *v;  // write: sources; read: destinations
  int64_t k_st, k_sh, v_st, v_sh;
  const int32_t *row, *pos;
  int64_t units;  // tokens * heads * 2
  bool vec;
};

template <typename T>
__device__ __forceinline__ void ld8(const T* p, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    } else {
      const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(a[i] << 16);
        v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = St<T>::ld(p + i);
  }
}
template <typename T>
__device__ __forceinline__ void st8(T* p, bool vec, const float (&v)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
      *reinterpret_cast<u32x4_t*>(p) =
          u32x4_t{pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) St<T>::st(p + i, v[i]);
  }
}

// unit u = (token * heads + head) * 2 + (0: K, 1: V); lanes 0 .. HD / 8 - 1 of the unit hold 8 values each
template <typename T, int HD, bool WRITE>
__global__ __launch_bounds__(256) void kv8_kernel(Kv8Args a) {
  constexpr int L = HD / 8;
  const int64_t u = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const int l = threadIdx.x % L;
  if (u >= a.units) return;  // whole groups of L lanes leave together
  const bool isv = u & 1;
  const int64_t th = u >> 1;
  const int64_t t = th / a.c.heads;
  const int h = (int)(th - t * a.c.heads);
  const int row = a.row[t], pos = a.pos[t];
  const bool ok = (unsigned)row < (unsigned)a.c.rows && (unsigned)pos < (unsigned)a.c.max_kv;
  const int64_t slot = (int64_t)row * a.c.bs + (int64_t)h * a.c.hs + (int64_t)pos * HD + 8 * l;
  const int64_t sslot = (int64_t)row * a.c.sbs + (int64_t)h * a.c.shs + pos;
  uint8_t* codes = (uint8_t*)(isv ? a.c.v : a.c.k);
  uint8_t* scale = isv ? a.c.v_scale : a.c.k_scale;
  const int64_t off = t * (isv ? a.v_st : a.k_st) + h * (isv ? a.v_sh : a.k_sh) + 8 * l;
  float v[8];
  if constexpr (WRITE) {
    if (!ok) return;
    ld8((const T*)(isv ? a.v : a.k) + off, a.vec, v);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_f(v[i]) ? fabsf(v[i]) : 0.f);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const int byte = e4m3_scale_byte(m);
    const float inv = e4m3_inv_scale(byte);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = e4m3_prescale(v[i], inv);
    *reinterpret_cast<u32x2_t*>(codes + slot) =
        u32x2_t{e4m3_pack4(q[0], q[1], q[2], q[3]), e4m3_pack4(q[4], q[5], q[6], q[7])};
    if (l == 0) scale[sslot] = (uint8_t)byte;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (ok) {
      const u32x2_t c = *reinterpret_cast<const u32x2_t*>(codes + slot);
      const float s = e4m3_scale(scale[sslot]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
        v[4 * i] = lo[0] * s;
        v[4 * i + 1] = lo[1] * s;
        v[4 * i + 2] = hi[0] * s;
        v[4 * i + 3] = hi[1] * s;
      }
    }
    st8((T*)(isv ? const_cast<void*>(a.v) : const_cast<void*>(a.k)) + off, a.vec, v);
  }
}

template <bool WRITE>
int launch(const char* fn, const ItTsKvCache* c, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
           int64_t v_sh, int dtype, const int32_t* row, const int32_t* pos, int M, void* stream) {
  if (int rc = itts::check_kv_cache(fn, c)) return rc;
  ITTS_REQUIRE(c->dtype == ITTS_E4M3, fn, "the cache must hold e4m3 codes");
  ITTS_REQUIRE(dtype == ITTS_F32 || dtype == ITTS_BF16, fn, "k and v must be f32 or bf16");
  ITTS_REQUIRE(M >= 0, fn, "negative token count");
  if (M == 0) return 0;
  ITTS_REQUIRE(k && v && row && pos, fn, "null pointer");
  const int es = dtype == ITTS_F32 ? 4 : 2;
  const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((k_st | k_sh | v_st | v_sh) * es) % 16 == 0;
  Kv8Args a{*c, k, v, k_st, k_sh, v_st, v_sh, row, pos, (int64_t)M * c->heads * 2, vec};
  const int64_t blocks = (a.units * (c->head_dim / 8) + 255) / 256;
  ITTS_REQUIRE(blocks <= 0x7FFFFFFF, fn, "too many tokens for one launch");
  hipStream_t s = itts::as_stream(stream);
  const dim3 g((unsigned)blocks), b(256);
  if (dtype == ITTS_F32) {
    if (c->head_dim == 64) hipLaunchKernelGGL((kv8_kernel<float, 64, WRITE>), g, b, 0, s, a);
    else hipLaunchKernelGGL((kv8_kernel<float, 128, WRITE>), g, b, 0, s, a);
  } else {
    if (c->head_dim == 64) hipLaunchKernelGGL((kv8_kernel<uint16_t, 64, WRITE>), g, b, 0, s, a);
    else hipLaunchKernelGGL((kv8_kernel<uint16_t, 128, WRITE>), g, b, 0, s, a);
  }
  return itts::check_launch(fn);
}

}  // namespace

namespace itts {
int check_kv_cache(const char* fn, const ItTsKvCache* c) {
  ITTS_REQUIRE(c, fn, "null cache");
  ITTS_REQUIRE(c->dtype == ITTS_E4M3 || c->dtype == ITTS_BF16, fn, "a cache holds e4m3 codes or bf16");
  ITTS_REQUIRE(c->head_dim == 64 || c->head_dim == 128, fn, "head_dim must be 64 or 128");
  ITTS_REQUIRE(c->rows >= 1 && c->heads >= 1 && c->max_kv >= 1 && c->max_kv <= (1 << 20) && c->heads <= 65535, fn,
               "bad cache sizes");
  ITTS_REQUIRE(c->k && c->v && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, fn, "null or misaligned cache");
  const int64_t head = (int64_t)c->max_kv * c->head_dim;
  const int unit = c->dtype == ITTS_E4M3 ? 16 : 8;  // 16-B loads
  ITTS_REQUIRE((c->hs >= head || c->heads == 1) && (c->bs >= head || c->rows == 1) && c->hs % unit == 0 &&
                   c->bs % unit == 0,
               fn, "cache strides: whole positions and 16 bytes");
  if (c->dtype == ITTS_E4M3)
    ITTS_REQUIRE(c->k_scale && c->v_scale && (c->shs >= c->max_kv || c->heads == 1) && (c->sbs >= c->max_kv || c->rows == 1),
                 fn, "bad scale bytes or strides");
  return 0;
}
}  // namespace itts

extern "C" int itts_kv8_write(const ItTsKvCache* c, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                              int64_t v_sh, int dtype, const int32_t* row, const int32_t* pos, int M, void* stream) {
  return launch<true>("itts_kv8_write", c, k, k_st, k_sh, v, v_st, v_sh, dtype, row, pos, M, stream);
}

extern "C" int itts_kv8_read(const ItTsKvCache* c, const int32_t* row, const int32_t* pos, int M, void* k, int64_t k_st,
                             int64_t k_sh, void* v, int64_t v_st, int64_t v_sh, int dtype, void* stream) {
  return launch<false>("itts_kv8_read", c, k, k_st, k_sh, v, v_st, v_sh, dtype, row, pos, M, stream);
}
