// attention_internal.cuh — the moe_attn handle, the kernels' parameter blocks and the helpers that the
// paged-attention kernels share.
#pragma once
#include <cuda.h>

#include <exception>

#include "moe_internal.cuh"
#include "tensor_map.cuh"

struct moe_attn {
  moe_attn_desc d;
  int group;            // query heads per key/value head
  int sms;
  int64_t page_stride;  // elements
  float scale;
  void* workspace = nullptr;    // one allocation; the counters and the error word come first
  size_t zeroed_bytes = 0;
  int64_t bytes = 0;
  int32_t *counters = nullptr, *group_counters = nullptr;  // decode: arrivals per (sequence, head) and per group of parts
  float* partial = nullptr;                                // parts of split (sequence, head)s: weighted values,
  float2 *partial_ml = nullptr, *group_ml = nullptr;       // maxima and sums
  int32_t* pf_counters = nullptr;  // prefill: arrivals per (item, tile, warp), then the two work words
  float4* pf_partial = nullptr;    // pieces of cut items
  float2* pf_ml = nullptr;
  int32_t* err = nullptr;
  uint32_t wait_limit;  // SM clocks
  CUtensorMap k_map, v_map;  // prefill's page boxes
};

namespace moe {
namespace attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Pools {
  void* k;
  void* v;
  int64_t page_stride;  // elements
  int num_pages, page_shift;
};

struct DecodeParams {
  const void* q;
  int64_t q_token_stride, q_head_stride;
  const int32_t* seq_lens;
  const int32_t* page_table;
  int max_pages, B, heads, kv_heads, group;
  int row_blocks;  // blocks of query heads per key/value head
  Pools pools;
  float scale, softcap;
  int window;
  void* y;
  float* lse;
  float* partial;
  float2 *partial_ml, *group_ml;
  int32_t *counters, *group_counters;
  int32_t* err;
};

struct PrefillParams {
  const void* q;
  int64_t q_token_stride, q_head_stride;
  const int32_t* cu_q;
  const int32_t* seq_lens;
  const int32_t* page_table;
  int max_pages, B, T, heads, kv_heads, group;
  int num_pages, page_shift;
  float scale, softcap;
  int window;
  void* y;
  float* lse;
  float4* partial;     // pieces of items that are cut along the keys
  float2* partial_ml;
  int32_t* counters;   // arrivals per (item, tile, warp)
  int32_t* work;       // [0] pieces taken, [1] CTAs that have left
  int32_t* err;
  uint32_t wait_limit;  // SM clocks
};

// Rows of query heads that one decode work unit holds, and the sizes that follow from them.
inline int decode_rows(int group) { return group <= 8 ? 8 : 16; }
inline int decode_row_blocks(int group) { return ceil_div(group, decode_rows(group)); }
int decode_max_ctas(int sms);

// Per-device kernel attributes of the handle's variant; called with its device current.
moe_status prepare_decode(const moe_attn& a);
moe_status prepare_prefill(const moe_attn& a);
size_t prefill_partial_bytes(const moe_attn& a);
size_t prefill_ml_bytes(const moe_attn& a);
size_t prefill_counters(const moe_attn& a);
moe_status launch_decode(const moe_attn& a, const DecodeParams& p, cudaStream_t st);
moe_status launch_prefill(const moe_attn& a, const PrefillParams& p, cudaStream_t st);
// 4-D map over a pool: box of 64 values x min(page_size, 128) tokens of one head of one page, SWIZZLE_128B.
moe_status make_page_tmap(CUtensorMap* map, int dtype, const void* pool, int head_dim, int page_size, int kv_heads,
                          int64_t num_pages, int64_t page_stride);

// ---- element types ------------------------------------------------------------------------------

template <class T>
struct Elem;
// The weights of the second product are rounded to the values' type. kWeightBits: powers of two that they may be scaled up by
// and stay finite when the largest is 1. In f16 an unscaled weight below 2^-25 would be lost from the values but not from the
// f32 sum (all of the output where a first key with no value scores 17.5 above the rest); bf16 has f32's exponents.
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kWeightBits = 0;
  static constexpr float kLeast = 1.17549435e-38f;  // smallest normal value
  static __device__ __forceinline__ uint32_t pack_down(float lo, float hi) {  // towards zero
    uint32_t v;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a, b0, b1);
  }
};
template <>
struct Elem<__half> {
  static constexpr int kWeightBits = 15;
  static constexpr float kLeast = 5.9604645e-08f;  // smallest value
  static __device__ __forceinline__ uint32_t pack_down(float lo, float hi) {
    uint32_t v;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(d, a, b0, b1);
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same, kept in program order with its like.
__device__ __forceinline__ float ex2_ordered(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// softcap * tanh(x / softcap) in units of log2, of scores v before their scale. softcap * (1 - 2 / (e^2t + 1)), t = x / softcap,
// is off by about 2^-23 of the cap, however small the score is; caps above WIDE_CAP, of which that would be
// more than a weight can take, use tanh's series t - t^3 / 3 + 2 t^5 / 15 - 17 t^7 / 315 + 62 t^9 / 2835 (2^-26 relative) for |t| < 1/4.
struct Cap {
  float in, out, slope, gain;  // 2 / ln 2 * scale / softcap, softcap / ln 2, scale / softcap, scale / ln 2
  bool wide;
};
constexpr float WIDE_CAP = 64.0f;

__device__ __forceinline__ Cap make_cap(float scale, float softcap) {
  return {fminf(2.0f * LOG2E * scale / softcap, 3.0e38f), softcap * LOG2E, scale / softcap, scale * LOG2E, softcap > WIDE_CAP};
}

__device__ __forceinline__ float capped_score(const Cap& c, float v) {
  return c.out - __fdividef(2.0f * c.out, ex2(v * c.in) + 1.0f);
}

__device__ __forceinline__ float wide_capped_score(const Cap& c, float v) {
  const float t = v * c.slope, t2 = t * t;
  const float r = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  return fabsf(t) < 0.25f ? v * c.gain * r : capped_score(c, v);
}

__device__ __forceinline__ void latch(int32_t* err, moe_status st) { atomicCAS(err, 0, (int32_t)st); }

}  // namespace attn
}  // namespace moe
