// attention.cu — the moe_attn handle, its C ABI, and the append kernel of the paged key/value cache.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>

#include "attention_internal.cuh"

namespace moe {
namespace attn {

// ---- append ----------------------------------------------------------------------------------------
//
// Per token and head: u = x / sqrt(mean(x^2) + eps) * w (optional), then pair i of the first rope_dim
// values (a, b) -> (a c - b s, b c + a s) with (c, s) = rope_table[position of the pair's axis][i].
// Floor: (heads + 2 kv_heads) * head_dim * 2 bytes read and as many written per token; with a few arithmetic instructions
// per byte the kernel is bound by its instruction count as much as by its bytes, so the layout is chosen to need no
// exchange between lanes but the norm's sum: a row (one head of one token) is held by head_dim / 8 lanes, lane l with
// two chunks of 4 values that contain both members of its 4 pairs 4 l .. 4 l + 3 (halves: at 4 l and rope_dim / 2 + 4 l; adjacent
// pairs and values past rope_dim: at 8 l and 8 l + 4). A lane group takes up to ROWS rows of one token and one kind (q, k or
// v): their loads are in flight together, and weight and angle of a value are multiplied once for all of them,
//   out_a = inv (a (w_a c) - b (w_b s)),  out_b = inv (b (w_b c) + a (w_a s)),  inv = 1 / sqrt(mean(x^2) + eps).
// Blocks are (lanes of a row, lane groups, tokens), so a thread finds its work without a division.
constexpr int APPEND_THREADS = 256;
// A window above this (2,080,374,784 positions) is none: position arithmetic beside it would leave 32 bits.
constexpr int MAX_WINDOW = 0x7c000000;
// Rows per lane group, measured at 4096 tokens of 32 + 2 x 4 heads of 128: 2 rows 33.8 us, 4: 20.2, 8: 21.2 (4 in a whole call:
// 21.6, 4.0 TB/s).
constexpr int ROWS = 4;

struct AppendParams {
  const void *q, *k, *v;
  void* q_out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  const int32_t* positions;
  const int64_t* slots;
  int T, heads, kv_heads;
  Pools pools;
  const float* rope_table;
  int rope_positions, rope_dim, rope_axes, adjacent;
  int axis1, axis2;  // first pair of axis 1 and of axis 2
  const void *q_norm, *k_norm;
  float eps;
  int32_t* err;
};

template <class T, int D>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(AppendParams p) {
  constexpr int LPR = D / 8;  // lanes of a row
  pdl_wait();
  pdl_trigger();
  const int l = threadIdx.x;
  const int64_t t64 = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
  const bool live = t64 < p.T;
  const int64_t t = live ? t64 : 0;
  // this lane group's rows: `count` of them, row_stride apart
  const int q_groups = (p.heads + ROWS - 1) / ROWS, kv_groups = (p.kv_heads + ROWS - 1) / ROWS;
  int group = blockIdx.y * blockDim.y + threadIdx.y;
  const bool is_q = group < q_groups, is_v = group >= q_groups + kv_groups;
  group -= is_q ? 0 : is_v ? q_groups + kv_groups : q_groups;
  const int head = group * ROWS;
  const int count = live ? min(ROWS, (is_q ? p.heads : p.kv_heads) - head) : 0;  // <= 0: nothing here
  const int64_t row_stride = is_q ? p.q_hs : is_v ? p.v_hs : p.k_hs;
  const T* src = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) + t * (is_q ? p.q_ts : is_v ? p.v_ts : p.k_ts) +
                 head * row_stride;
  const int half = p.rope_dim / 2;
  const bool turns = 8 * l < p.rope_dim;
  const bool split = turns && !p.adjacent;  // the chunks lie half a rotation apart
  const int off0 = split ? 4 * l : 8 * l, off1 = split ? half + 4 * l : 8 * l + 4;

  uint2 x[ROWS][2];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    x[i][0] = x[i][1] = make_uint2(0, 0);
    if (i < count) {
      x[i][0] = *reinterpret_cast<const uint2*>(src + i * row_stride + off0);
      x[i][1] = *reinterpret_cast<const uint2*>(src + i * row_stride + off1);
    }
  }
  // weights of this lane's values
  const T* nw = static_cast<const T*>(is_v ? nullptr : is_q ? p.q_norm : p.k_norm);
  float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
  if (nw) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(nw + (e ? off1 : off0)));
      const float2 lo = Elem<T>::unpack(v.x), hi = Elem<T>::unpack(v.y);
      w[4 * e] = lo.x, w[4 * e + 1] = lo.y, w[4 * e + 2] = hi.x, w[4 * e + 3] = hi.y;
    }
  }
  // slot and positions: a token that fails a check is stored nowhere
  bool ok = live;
  const int64_t slot = live ? p.slots[t] : -1;
  int pos[3] = {0, 0, 0};
  if (live && p.rope_dim > 0) {
#pragma unroll
    for (int a = 0; a < 3; ++a)
      if (a < p.rope_axes) pos[a] = p.positions[(int64_t)a * p.T + t];
  }
  if (live && (slot < 0 || slot >= ((int64_t)p.pools.num_pages << p.pools.page_shift))) {
    ok = false;
    if (slot != -1) latch(p.err, MOE_ERR_BAD_IDS);
  }
  float c[4] = {1, 1, 1, 1}, s[4] = {0, 0, 0, 0};
  if (ok && p.rope_dim > 0) {
#pragma unroll
    for (int a = 0; a < 3; ++a)
      if (pos[a] < 0 || pos[a] >= p.rope_positions) ok = false;
    if (!ok) latch(p.err, MOE_ERR_BAD_IDS);
    if (ok && turns && !is_v) {
      if (p.rope_axes == 1) {  // one table row: two pairs per 16-byte load
        const float4* row = reinterpret_cast<const float4*>(p.rope_table + ((int64_t)pos[0] * half + 4 * l) * 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 cs = __ldg(row + i);
          c[2 * i] = cs.x, s[2 * i] = cs.y, c[2 * i + 1] = cs.z, s[2 * i + 1] = cs.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * l + i;
          const int at = j >= p.axis2 ? pos[2] : j >= p.axis1 ? pos[1] : pos[0];
          const float2 cs = __ldg(reinterpret_cast<const float2*>(p.rope_table) + (int64_t)at * half + j);
          c[i] = cs.x;
          s[i] = cs.y;
        }
      }
    }
  }
  if (count <= 0) return;  // whole lane groups: the sums below are each within one
  T* dst;
  int64_t dst_stride;
  if (is_q) {
    dst = static_cast<T*>(p.q_out) + t * p.o_ts + head * p.o_hs;
    dst_stride = p.o_hs;
  } else {
    if (!ok) return;
    const int64_t page = slot >> p.pools.page_shift;
    const int at = (int)(slot & ((1 << p.pools.page_shift) - 1));
    dst_stride = (int64_t)D << p.pools.page_shift;
    dst = static_cast<T*>(is_v ? p.pools.v : p.pools.k) + page * p.pools.page_stride + head * dst_stride + at * D;
  }
  if (is_v || (is_q && !ok)) {  // values as they are; zeros for a token that is stored nowhere
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (i >= count) break;
      *reinterpret_cast<uint2*>(dst + i * dst_stride + off0) = ok ? x[i][0] : make_uint2(0, 0);
      *reinterpret_cast<uint2*>(dst + i * dst_stride + off1) = ok ? x[i][1] : make_uint2(0, 0);
    }
    return;
  }
  const int lane = (threadIdx.x + blockDim.x * (threadIdx.y + blockDim.y * threadIdx.z)) & 31;
  const unsigned group_mask = ((1u << LPR) - 1u) << (lane & ~(LPR - 1));
  // values a_i, b_i of pair i: chunk 0 and chunk 1 (halves), or neighbours
  const bool adj = p.adjacent;
  float wac[4], wbs[4], wbc[4], was[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float wa = adj ? w[2 * i] : w[i], wb = adj ? w[2 * i + 1] : w[4 + i];
    wac[i] = wa * c[i], wbs[i] = wb * s[i], wbc[i] = wb * c[i], was[i] = wa * s[i];
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (i >= count) break;
    float f[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 lo = Elem<T>::unpack(x[i][e].x), hi = Elem<T>::unpack(x[i][e].y);
      f[4 * e] = lo.x, f[4 * e + 1] = lo.y, f[4 * e + 2] = hi.x, f[4 * e + 3] = hi.y;
    }
    float inv = 1.0f;
    if (nw) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
#pragma unroll
      for (int o = LPR / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(group_mask, ss, o);
      inv = rsqrtf(ss * (1.0f / D) + p.eps);
    }
    float g[8];
    if (!turns) {  // past rope_dim: no partner's value may reach these
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = inv * (f[j] * w[j]);
    } else if (adj) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[2 * j] = inv * (f[2 * j] * wac[j] - f[2 * j + 1] * wbs[j]);
        g[2 * j + 1] = inv * (f[2 * j + 1] * wbc[j] + f[2 * j] * was[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[j] = inv * (f[j] * wac[j] - f[4 + j] * wbs[j]);
        g[4 + j] = inv * (f[4 + j] * wbc[j] + f[j] * was[j]);
      }
    }
    *reinterpret_cast<uint2*>(dst + i * dst_stride + off0) = make_uint2(Elem<T>::pack(g[0], g[1]), Elem<T>::pack(g[2], g[3]));
    *reinterpret_cast<uint2*>(dst + i * dst_stride + off1) = make_uint2(Elem<T>::pack(g[4], g[5]), Elem<T>::pack(g[6], g[7]));
  }
}

template <class T>
static cudaError_t launch_append(const AppendParams& p, int D, cudaStream_t st) {
  const int lanes = D / 8, groups = ceil_div(p.heads, ROWS) + 2 * ceil_div(p.kv_heads, ROWS);
  const int by = std::min(groups, APPEND_THREADS / lanes);
  const int bz = std::max(1, std::min(p.T, APPEND_THREADS / (lanes * by)));
  const dim3 block(lanes, by, bz), grid((unsigned)ceil_div(p.T, bz), (unsigned)ceil_div(groups, by));
  return D == 64 ? launch_pdl(append_kernel<T, 64>, grid, block, 0, st, p)
                 : launch_pdl(append_kernel<T, 128>, grid, block, 0, st, p);
}

// No C++ exception crosses the C ABI.
template <class F>
static moe_status guarded(F&& f) noexcept {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return MOE_ERR_OOM;
  } catch (...) {
    return MOE_ERR_INVALID;
  }
}

static moe_status bad(const char* call, const char* what) {
  return fail(MOE_ERR_INVALID, std::string(call) + ": " + what);
}

static bool rows_ok(const void* p, int64_t ts, int64_t hs) { return !((uintptr_t)p & 15) && ts % 8 == 0 && hs % 8 == 0; }

static Pools pools_of(const moe_attn& a) {
  int shift = 0;
  while ((1 << shift) < a.d.page_size) ++shift;
  return Pools{a.d.k_pool, a.d.v_pool, a.page_stride, (int)a.d.num_pages, shift};
}

static moe_status validate(const moe_attn_desc& d) {
  const char* me = "moe_attn_create";
  if (d.dtype != MOE_ATTN_BF16 && d.dtype != MOE_ATTN_F16)
    return fail(MOE_ERR_UNSUPPORTED, "moe_attn_create: dtype must be bf16 or f16");
  if (d.head_dim != 64 && d.head_dim != 128)
    return fail(MOE_ERR_UNSUPPORTED, "moe_attn_create: head_dim must be 64 or 128");
  if (d.num_kv_heads <= 0 || d.num_heads <= 0 || d.num_heads % d.num_kv_heads || d.num_heads / d.num_kv_heads > 128 ||
      d.num_heads > 65536)
    return bad(me, "num_heads must be a multiple of num_kv_heads, at most 128 times it");
  if (d.page_size != 16 && d.page_size != 32 && d.page_size != 64 && d.page_size != 128)
    return bad(me, "page_size must be 16, 32, 64 or 128");
  if (d.num_pages <= 0 || d.num_pages * d.page_size > 0x7fffffffll || d.num_pages > 0x7fffffffll)
    return bad(me, "num_pages * page_size must be in 1 .. 2^31 - 1");
  const int64_t packed = (int64_t)d.num_kv_heads * d.page_size * d.head_dim;
  if (d.page_stride && (d.page_stride < packed || d.page_stride % 8))
    return bad(me, "page_stride must be a multiple of 8 that holds a page");
  if (!d.k_pool || !d.v_pool || ((uintptr_t)d.k_pool & 15) || ((uintptr_t)d.v_pool & 15))
    return bad(me, "the pools must be 16-byte aligned device memory");
  if (!(d.scale >= 0.0f) || !std::isfinite(d.scale) || !(d.softcap >= 0.0f) || !std::isfinite(d.softcap) || d.window < 0)
    return bad(me, "scale, softcap and window must be finite and not negative");
  if (d.rope_dim < 0 || d.rope_dim % 16 || d.rope_dim > d.head_dim)
    return bad(me, "rope_dim must be a multiple of 16 up to head_dim");
  if (d.rope_dim) {
    if (!d.rope_table || ((uintptr_t)d.rope_table & 15) || d.rope_positions <= 0)
      return bad(me, "rope_dim needs a 16-byte aligned rope_table with rope_positions rows");
    if (d.rope_pairs != MOE_ROPE_HALVES && d.rope_pairs != MOE_ROPE_ADJACENT) return bad(me, "unknown rope_pairs");
    if (d.rope_axes != 1 && d.rope_axes != 3) return bad(me, "rope_axes must be 1 or 3");
    if (d.rope_axes == 3) {
      int64_t sum = 0;
      for (int a = 0; a < 3; ++a) {
        if (d.rope_sections[a] < 0) return bad(me, "negative rope section");
        sum += d.rope_sections[a];
      }
      if (sum != d.rope_dim / 2) return bad(me, "rope_sections must sum to rope_dim / 2");
    }
  }
  if (((uintptr_t)d.q_norm & 15) || ((uintptr_t)d.k_norm & 15)) return bad(me, "norm weights must be 16-byte aligned");
  if ((d.q_norm || d.k_norm) && !(d.norm_eps >= 0.0f)) return bad(me, "norm_eps must not be negative");
  if (d.max_seqs <= 0 || (int64_t)d.max_seqs * d.num_heads > (1 << 28)) return bad(me, "max_seqs out of range");
  return MOE_OK;
}

}  // namespace attn
}  // namespace moe

using namespace moe;
using namespace moe::attn;

extern "C" moe_status moe_attn_create(const moe_attn_desc* desc, moe_attn** out) {
  return guarded([&]() -> moe_status {
    if (!desc || !out) return bad("moe_attn_create", "null desc or out");
    *out = nullptr;
    MOE_TRY(validate(*desc));
    DeviceGuard guard(desc->device);
    if (!guard.ok) return bad("moe_attn_create", "no such device");
    moe_attn* a = new (std::nothrow) moe_attn();
    if (!a) return fail(MOE_ERR_OOM, "moe_attn_create: host allocation failed");
    a->d = *desc;
    if (a->d.window > MAX_WINDOW) a->d.window = 0;
    a->group = desc->num_heads / desc->num_kv_heads;
    a->wait_limit = (uint32_t)WAIT_CYCLES;
    a->scale = desc->scale > 0.0f ? desc->scale : 1.0f / std::sqrt((float)desc->head_dim);
    a->page_stride =
        desc->page_stride ? desc->page_stride : (int64_t)desc->num_kv_heads * desc->page_size * desc->head_dim;
    const moe_status st = [&]() -> moe_status {
      MOE_CUDA_TRY(cudaDeviceGetAttribute(&a->sms, cudaDevAttrMultiProcessorCount, desc->device));
      // the workspace, one allocation (a handle is made per layer): each part at a multiple of 256 bytes
      const int rows = decode_rows(a->group);
      const size_t slots = (size_t)decode_max_ctas(a->sms) * 2;  // a decode CTA leaves at most two partial results
      const size_t units = (size_t)desc->max_seqs * desc->num_kv_heads * decode_row_blocks(a->group);
      size_t end = 0;
      auto part = [&](size_t bytes) {
        const size_t at = end;
        end += (bytes + 255) / 256 * 256;
        return at;
      };
      const size_t o_cnt = part((units + slots) * sizeof(int32_t));
      const size_t o_pf_cnt = part((prefill_counters(*a) + 2) * sizeof(int32_t));
      const size_t o_err = part(sizeof(int32_t));
      a->zeroed_bytes = end;  // the words above start at zero
      const size_t o_acc = part(slots * rows * desc->head_dim * sizeof(float));
      const size_t o_ml = part(2 * slots * rows * sizeof(float2));
      const size_t o_pf_acc = part(prefill_partial_bytes(*a)), o_pf_ml = part(prefill_ml_bytes(*a));
      MOE_CUDA_TRY(cudaMalloc(&a->workspace, end));
      a->bytes = (int64_t)end;
      unsigned char* w = static_cast<unsigned char*>(a->workspace);
      a->counters = reinterpret_cast<int32_t*>(w + o_cnt);
      a->group_counters = a->counters + units;
      a->pf_counters = reinterpret_cast<int32_t*>(w + o_pf_cnt);
      a->err = reinterpret_cast<int32_t*>(w + o_err);
      a->partial = reinterpret_cast<float*>(w + o_acc);
      a->partial_ml = reinterpret_cast<float2*>(w + o_ml);
      a->group_ml = a->partial_ml + slots * rows;
      a->pf_partial = reinterpret_cast<float4*>(w + o_pf_acc);
      a->pf_ml = reinterpret_cast<float2*>(w + o_pf_ml);
      MOE_CUDA_TRY(cudaMemset(w, 0, a->zeroed_bytes));
      MOE_CUDA_TRY(cudaStreamSynchronize(cudaStreamLegacy));  // in place for a first call on any stream
      MOE_TRY(prepare_decode(*a));
      MOE_TRY(prepare_prefill(*a));
      for (int i = 0; i < 2; ++i)
        MOE_TRY(make_page_tmap(i ? &a->v_map : &a->k_map, desc->dtype, i ? desc->v_pool : desc->k_pool, desc->head_dim,
                               desc->page_size, desc->num_kv_heads, desc->num_pages, a->page_stride));
      return MOE_OK;
    }();
    if (st != MOE_OK) {
      const std::string msg = last_error_message();
      moe_attn_destroy(a);
      return fail(st, msg);
    }
    *out = a;
    return MOE_OK;
  });
}

extern "C" void moe_attn_destroy(moe_attn* a) {
  if (!a) return;
  DeviceGuard guard(a->d.device);
  cudaFree(a->workspace);
  delete a;
}

extern "C" int64_t moe_attn_device_bytes(const moe_attn* a) { return a ? a->bytes : 0; }

extern "C" moe_status moe_attn_append(moe_attn* a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                      const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                      int64_t v_token_stride, int64_t v_head_stride, int T, const int32_t* positions,
                                      const int64_t* slots, void* q_out, int64_t out_token_stride,
                                      int64_t out_head_stride, void* stream) {
  return guarded([&]() -> moe_status {
    const char* me = "moe_attn_append";
    if (!a) return bad(me, "null handle");
    if (T < 0) return bad(me, "T must not be negative");
    if (T == 0) return MOE_OK;
    if (!q || !k || !v || !slots || !q_out || (a->d.rope_dim && !positions)) return bad(me, "null pointer");
    if (!rows_ok(q, q_token_stride, q_head_stride) || !rows_ok(k, k_token_stride, k_head_stride) ||
        !rows_ok(v, v_token_stride, v_head_stride) || !rows_ok(q_out, out_token_stride, out_head_stride))
      return bad(me, "rows must be 16-byte aligned with strides that are multiples of 8");
    AppendParams p{};
    p.q = q, p.k = k, p.v = v, p.q_out = q_out;
    p.q_ts = q_token_stride, p.q_hs = q_head_stride, p.k_ts = k_token_stride, p.k_hs = k_head_stride;
    p.v_ts = v_token_stride, p.v_hs = v_head_stride, p.o_ts = out_token_stride, p.o_hs = out_head_stride;
    p.positions = positions, p.slots = slots, p.T = T;
    p.heads = a->d.num_heads, p.kv_heads = a->d.num_kv_heads;
    p.pools = pools_of(*a);
    p.rope_table = a->d.rope_table, p.rope_positions = a->d.rope_positions, p.rope_dim = a->d.rope_dim;
    p.rope_axes = a->d.rope_axes, p.adjacent = a->d.rope_pairs == MOE_ROPE_ADJACENT;
    const bool axes = a->d.rope_axes == 3;
    p.axis1 = axes ? a->d.rope_sections[0] : a->d.rope_dim;
    p.axis2 = axes ? a->d.rope_sections[0] + a->d.rope_sections[1] : a->d.rope_dim;
    p.q_norm = a->d.q_norm, p.k_norm = a->d.k_norm, p.eps = a->d.norm_eps;
    p.err = a->err;
    DeviceGuard guard(a->d.device);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    MOE_CUDA_TRY(a->d.dtype == MOE_ATTN_BF16 ? launch_append<__nv_bfloat16>(p, a->d.head_dim, st)
                                             : launch_append<__half>(p, a->d.head_dim, st));
    return MOE_OK;
  });
}

extern "C" moe_status moe_attn_decode(moe_attn* a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                      const int32_t* seq_lens, const int32_t* page_table, int max_pages, int B,
                                      void* y, float* lse, void* stream) {
  return guarded([&]() -> moe_status {
    const char* me = "moe_attn_decode";
    if (!a) return bad(me, "null handle");
    if (B < 0 || B > a->d.max_seqs) return bad(me, "B must be in 0 .. max_seqs");
    if (B == 0) return MOE_OK;
    if (!q || !seq_lens || !y || max_pages < 0 || (max_pages && !page_table)) return bad(me, "null pointer or no pages");
    if (!rows_ok(q, q_token_stride, q_head_stride) || ((uintptr_t)y & 15))
      return bad(me, "rows must be 16-byte aligned with strides that are multiples of 8");
    if ((int64_t)max_pages * a->d.page_size > 0x7fffffffll) return bad(me, "max_pages * page_size above 2^31 - 1");
    DecodeParams p{};
    p.q = q, p.q_token_stride = q_token_stride, p.q_head_stride = q_head_stride;
    p.seq_lens = seq_lens, p.page_table = page_table, p.max_pages = max_pages, p.B = B;
    p.heads = a->d.num_heads, p.kv_heads = a->d.num_kv_heads, p.group = a->group;
    p.row_blocks = decode_row_blocks(a->group);
    p.pools = pools_of(*a);
    p.scale = a->scale, p.softcap = a->d.softcap, p.window = a->d.window;
    p.y = y, p.lse = lse;
    p.partial = a->partial, p.partial_ml = a->partial_ml, p.group_ml = a->group_ml;
    p.counters = a->counters, p.group_counters = a->group_counters, p.err = a->err;
    DeviceGuard guard(a->d.device);
    return launch_decode(*a, p, static_cast<cudaStream_t>(stream));
  });
}

extern "C" moe_status moe_attn_prefill(moe_attn* a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                       const int32_t* cu_q, const int32_t* seq_lens, const int32_t* page_table,
                                       int max_pages, int B, int T, void* y, float* lse, void* stream) {
  return guarded([&]() -> moe_status {
    const char* me = "moe_attn_prefill";
    if (!a) return bad(me, "null handle");
    if (B < 0 || T < 0) return bad(me, "B and T must not be negative");
    if (T == 0) return MOE_OK;
    if (!q || !y || max_pages < 0 || (B > 0 && (!cu_q || !seq_lens || (max_pages && !page_table))))
      return bad(me, "null pointer or no pages");
    if (!rows_ok(q, q_token_stride, q_head_stride) || ((uintptr_t)y & 15))
      return bad(me, "rows must be 16-byte aligned with strides that are multiples of 8");
    if ((int64_t)max_pages * a->d.page_size > 0x7fffffffll) return bad(me, "max_pages * page_size above 2^31 - 1");
    PrefillParams p{};
    p.q = q, p.q_token_stride = q_token_stride, p.q_head_stride = q_head_stride;
    p.cu_q = cu_q, p.seq_lens = seq_lens, p.page_table = page_table, p.max_pages = max_pages, p.B = B, p.T = T;
    p.heads = a->d.num_heads, p.kv_heads = a->d.num_kv_heads, p.group = a->group;
    const Pools pools = pools_of(*a);
    p.num_pages = pools.num_pages, p.page_shift = pools.page_shift;
    p.scale = a->scale, p.softcap = a->d.softcap, p.window = a->d.window;
    p.y = y, p.lse = lse, p.err = a->err;
    p.partial = a->pf_partial, p.partial_ml = a->pf_ml, p.counters = a->pf_counters;
    p.work = a->pf_counters + prefill_counters(*a);
    p.wait_limit = a->wait_limit;
    DeviceGuard guard(a->d.device);
    return launch_prefill(*a, p, static_cast<cudaStream_t>(stream));
  });
}

extern "C" moe_status moe_attn_set_wait_limit(moe_attn* a, int64_t sm_clocks) {
  return guarded([&]() -> moe_status {
    const char* me = "moe_attn_set_wait_limit";
    if (!a) return bad(me, "null handle");
    if (sm_clocks < 1 || sm_clocks > WAIT_CYCLES) return bad(me, "the limit must be in 1 .. 400000000 SM clocks");
    a->wait_limit = (uint32_t)sm_clocks;
    return MOE_OK;
  });
}

extern "C" moe_status moe_attn_check(moe_attn* a, void* stream) {
  return guarded([&]() -> moe_status {
    if (!a) return bad("moe_attn_check", "null handle");
    DeviceGuard guard(a->d.device);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int32_t word = 0;
    MOE_CUDA_TRY(cudaMemcpyAsync(&word, a->err, sizeof(word), cudaMemcpyDeviceToHost, st));
    MOE_CUDA_TRY(cudaStreamSynchronize(st));
    if (!word) return MOE_OK;
    // a call that gave up may have left its counters half way: they go back to zero with the word
    MOE_CUDA_TRY(cudaMemsetAsync(a->workspace, 0, a->zeroed_bytes, st));
    MOE_CUDA_TRY(cudaStreamSynchronize(st));
    return fail((moe_status)word, word == MOE_ERR_TIMEOUT ? "attention: a bounded device-side wait gave up"
                                                          : "attention: a slot, page, position or length out of range");
  });
}
