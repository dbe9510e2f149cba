// Shared by the two kernels of the attention over the paged cache.
#pragma once

#include "paged.cuh"
#include "paged_plan.h"

namespace d2sd {
namespace paged {

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  int64_t q_st, q_sh, o_st, o_sh, lse_st;  // element strides
  const uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
  const int32_t* page_table;
  int64_t page_table_len;
  int64_t first_entry;  // page_table null: entry first_entry is page 0, and so on
  const int32_t* plan;
  float* slots;  // partial states (paged_plan.h)
  const float* sinks;
  int32_t* status;
  PageGeom g;
  float scale_log2;
  int32_t sink_mode;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) { return pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 1 / sum and log-sum-exp (base 2) of a row with weights relative to m and their sum l:
// 0 and -inf for a row that saw no key, NaN for one with a NaN. m and log2 l are both
// large where they nearly cancel (8-bit values' exponents and f16's headroom are in m),
// so l's exponent, whole, goes to m before its mantissa's logarithm is added.
__device__ __forceinline__ float row_factor(float m, float l, float& lse2) {
  const uint32_t bits = __float_as_uint(l), x = bits >> 23;
  if (x - 1u < 254u) {  // positive and normal
    lse2 = m + (static_cast<int>(x) - 127) + log2f(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u));
    return 1.f / l;
  }
  lse2 = l > 0.f ? m + log2f(l) : (l == 0.f ? -INFINITY : l);
  return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
}
// Factor of the attention sink: o *= sigmoid(lse - sink) (include/d2sd.h). A row
// without a key keeps its 0, with a sink of -inf too.
__device__ __forceinline__ float sink_factor(float lse2, float sink, int mode) {
  if (lse2 == -INFINITY) return 0.f;
  const float x = (mode == D2SD_SINK_EXACT ? lse2 * kLn2 : lse2) - sink;
  return 1.f / (1.f + expf(-x));
}

// Tensor maps of K and V pools of row pages: boxes of 16 rows by 64 values, 128-byte
// swizzled, at (value, slot, head, page) (paged_tiles.cu).
int encode_pages(CUtensorMap* tk, CUtensorMap* tv, const AttnArgs& a, int32_t dtype, int32_t head_dim,
                 int32_t num_kv_heads);

// Units of more than 16 query rows (paged_tiles.cu); num_tokens of q for its copies;
// split: no unit of the plan has more rows than one q tile.
int launch_tiles(const AttnArgs& a, int32_t dtype, int32_t head_dim, bool scaled, int64_t num_tokens,
                 int32_t num_qo_heads, int32_t num_kv_heads, bool split, int ctas, void* stream);

}  // namespace paged
}  // namespace d2sd
