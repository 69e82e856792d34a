// The 8-bit KV cache: K and V of a token quantised as they are written (one power-of-two scale per token, head and
// K or V over the head's hd values, fp8.h), and read back.  Layout beside the bf16 cache's: codes [row][head][pos][hd],
// scale bytes [row][head][pos].
//
// Pure traffic: a token and head reads hd values and writes hd + 1 bytes for each of K and V.  hd / 8 lanes per vector,
// eight values per lane, so a lane's 16-B (bf16) or 32-B (f32) load becomes one 8-B store.  A head's values of one token are a
// piece of hd bytes somewhere in the cache, so what bounds it is the latency of scattered pieces, not arithmetic: 24000 tokens
// of 16 heads x 64 in bf16 take 42 us to write and 45 to read (147 MB each, 3.4 TB/s; a large copy reaches 5); 32 tokens 3.
#include "fp8.h"

namespace {

using itts::e4m3_pack4;
using itts::e4m3_scale;

struct Kv8Args {
  ItTsKvCache c;
  const void *k, *v;  // write: sources; read: destinations
  int64_t k_st, k_sh, v_st, v_sh;
  const int32_t *row, *pos;
  int M, heads, lanes, per_block;  // tokens; heads of a group, their lanes (heads x 2 x hd / 8); tokens side by side
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

// The heads are dealt to the eight XCDs (workgroup id % 8), so that a line of the cache -- 128 / hd positions of a head,
// or 128 positions' scale bytes -- is written or read through one L2 whatever the order of the slots: tokens in random
// order otherwise cost a partial line in several L2s for each byte.  A token takes (heads of the group) x 2 x HD / 8 lanes
// (K or V, then head, then eight values), whole workgroups of 256 along grid y where that is more; a lane keeps its place
// and goes through TURNS tokens whose loads are all in flight together.
template <typename T, int HD, bool WRITE, int TURNS>
__global__ __launch_bounds__(256) void kv8_kernel(Kv8Args a) {
  constexpr int L = HD / 8;
  const int slot = a.per_block > 1 ? (int)threadIdx.x / a.lanes : 0;
  const int u = blockIdx.y * 256 + threadIdx.x - slot * a.lanes;
  if (u >= a.lanes || slot >= a.per_block) return;  // whole groups of L lanes leave together
  const int l = u % L, h = (int)(blockIdx.x & 7) * a.heads + ((u / L) >> 1);
  if (h >= a.c.heads) return;
  const bool isv = (u / L) & 1;
  uint8_t* codes = (uint8_t*)(isv ? a.c.v : a.c.k) + (int64_t)h * a.c.hs + 8 * l;
  uint8_t* scale = (isv ? a.c.v_scale : a.c.k_scale) + (int64_t)h * a.c.shs;
  T* side = (T*)const_cast<void*>(isv ? a.v : a.k) + h * (isv ? a.v_sh : a.k_sh) + 8 * l;
  const int64_t st = isv ? a.v_st : a.k_st;
  const int64_t t0 = ((int64_t)(blockIdx.x >> 3) * a.per_block + slot) * TURNS;
  if (t0 >= a.M) return;
  bool ok[TURNS];
  int64_t cs[TURNS], ss[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int64_t t = t0 + i < a.M ? t0 + i : a.M - 1;
    const int row = a.row[t], pos = a.pos[t];
    ok[i] = (unsigned)row < (unsigned)a.c.rows && (unsigned)pos < (unsigned)a.c.max_kv;
    cs[i] = ok[i] ? (int64_t)row * a.c.bs + (int64_t)pos * HD : 0;
    ss[i] = ok[i] ? (int64_t)row * a.c.sbs + pos : 0;
  }
  if constexpr (WRITE) {
    float v[TURNS][8];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) ld8(side + (t0 + i < a.M ? t0 + i : a.M - 1) * st, a.vec, v[i]);
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      auto reduce = [](uint32_t m) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        return m;
      };
      const int byte = itts::e4m3_scaled(v[i], reduce(itts::max_bits(v[i])), reduce);
      const float(&q)[8] = v[i];
      if (ok[i] && t0 + i < a.M) {
        *reinterpret_cast<u32x2_t*>(codes + cs[i]) =
            u32x2_t{e4m3_pack4(q[0], q[1], q[2], q[3]), e4m3_pack4(q[4], q[5], q[6], q[7])};
        if (l == 0) scale[ss[i]] = (uint8_t)byte;
      }
    }
  } else {
    u32x2_t c[TURNS];
    int byte[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      c[i] = *reinterpret_cast<const u32x2_t*>(codes + cs[i]);
      byte[i] = scale[ss[i]];
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      if (t0 + i >= a.M) break;
      const float s = e4m3_scale(byte[i]);
      float v[8];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[i][g], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[i][g], true);
        v[4 * g] = ok[i] ? lo[0] * s : 0.f;
        v[4 * g + 1] = ok[i] ? lo[1] * s : 0.f;
        v[4 * g + 2] = ok[i] ? hi[0] * s : 0.f;
        v[4 * g + 3] = ok[i] ? hi[1] * s : 0.f;
      }
      st8(side + (t0 + i) * st, a.vec, v);
    }
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
  // Four tokens a lane where that leaves workgroups enough, one where latency counts.  Measured, us (one / four): 32 tokens
  // written 3.1 / 4.7, 4096 read 7.9 / 7.5, 24000 written 29.1 / 27.3 and read 29.2 / 27.9 (slots in order).
  const int turns = M >= 4096 ? 4 : 1;
  const int group = (c->heads + 7) / 8;
  const int64_t lanes = (int64_t)group * 2 * (c->head_dim / 8);
  const int per = lanes < 256 ? (int)(256 / lanes) : 1;
  Kv8Args a{*c, k, v, k_st, k_sh, v_st, v_sh, row, pos, M, group, (int)lanes, per, vec};
  const int64_t blocks = 8 * ((M + (int64_t)per * turns - 1) / ((int64_t)per * turns)), deep = (lanes + 255) / 256;
  ITTS_REQUIRE(deep <= 65535 && blocks <= 0x7FFFFFFF, fn, "too many tokens or heads for one launch");
  hipStream_t s = itts::as_stream(stream);
  const dim3 g((unsigned)blocks, (unsigned)deep), b(256);
  auto go = [&](auto kernel4, auto kernel1) {
    if (turns == 4) hipLaunchKernelGGL(kernel4, g, b, 0, s, a);
    else hipLaunchKernelGGL(kernel1, g, b, 0, s, a);
  };
  if (dtype == ITTS_F32) {
    if (c->head_dim == 64) go(kv8_kernel<float, 64, WRITE, 4>, kv8_kernel<float, 64, WRITE, 1>);
    else go(kv8_kernel<float, 128, WRITE, 4>, kv8_kernel<float, 128, WRITE, 1>);
  } else {
    if (c->head_dim == 64) go(kv8_kernel<uint16_t, 64, WRITE, 4>, kv8_kernel<uint16_t, 64, WRITE, 1>);
    else go(kv8_kernel<uint16_t, 128, WRITE, 4>, kv8_kernel<uint16_t, 128, WRITE, 1>);
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
