// Attention over an e4m3 cache, head size 64 (attn_cached.h).
#include "attn_cached.h"

namespace itts {
namespace attn {
namespace {

template <int HD, bool LINEAGE, int QN, int PN, int NQ>
void launch(const AttnArgs& a, hipStream_t s) {
  const int64_t us = ((int64_t)a.units * a.nsplit + 7) / 8 * 8;
  hipLaunchKernelGGL((attn_cached_kernel<true, LINEAGE, HD, QN, PN, NQ>), dim3((unsigned)(us * a.qblocks)),
                     dim3(64 * kWaves), 0, s, a);
}
template <int HD, bool LINEAGE, int QN, int PN>
void launch_nq(const AttnArgs& a, int nq, hipStream_t s) {
  if (nq == 1) launch<HD, LINEAGE, QN, PN, 1>(a, s);
  else if (HD == 128 || nq == 2) launch<HD, LINEAGE, QN, PN, 2>(a, s);
  else if constexpr (HD == 64) launch<HD, LINEAGE, QN, PN, 4>(a, s);
}
template <int HD, bool LINEAGE>
void launch_types(const AttnArgs& a, int nq, hipStream_t s) {
  if (a.q_f32) {
    if (a.out_f32) launch_nq<HD, LINEAGE, 3, 2>(a, nq, s);
    else launch_nq<HD, LINEAGE, 3, 1>(a, nq, s);
  } else {
    if (a.out_f32) launch_nq<HD, LINEAGE, 1, 2>(a, nq, s);
    else launch_nq<HD, LINEAGE, 1, 1>(a, nq, s);
  }
}

}  // namespace

template <>
void launch_attn<true, 64>(const AttnArgs& a, int nq, hipStream_t s) {
  if (a.kv_rows) launch_types<64, true>(a, nq, s);
  else launch_types<64, false>(a, nq, s);
}

}  // namespace attn
}  // namespace itts
