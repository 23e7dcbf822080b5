// attention_prefill.cu — causal attention of a ragged batch of prompt chunks over a paged key/value cache,
// on the 5th-generation tensor cores.
//
//   x_ij = scale * (q_i . k_j)  (or softcap * tanh(x_ij / softcap)),  pos_i - window < j <= pos_i
//   y_i  = sum_j exp(x_ij - m_i) v_j / sum_j exp(x_ij - m_i),   lse_i = m_i + log sum_j exp(x_ij - m_i)
//
// A tile is 128 rows = (128 / group) tokens x the group's query heads, so the heads that share keys and
// values share their loads. A CTA owns two tiles (256 rows, consecutive tokens of one sequence and one
// key/value head) and walks the keys 128 at a time:
//   * one warp loads K and V pages by TMA (64 values x a page's tokens per box, SWIZZLE_128B) into rings of
//     STAGES tiles;
//   * one thread issues S_i = Q_i K^T (128 x 128, f32 in tensor memory) and O_i += P_i V, alternating the
//     two tiles, so the tensor cores work on one tile while the other's softmax runs;
//   * four warps per tile hold one row per thread: maximum, exponentials and sum in f32, P rounded to the
//     values' type and written over S in tensor memory, from where the second product reads it. O is
//     rescaled only when a row's maximum grows by more than 2^RESCALE (rare after the first tiles), which leaves
//     P below 2^RESCALE: sums stay exact enough in f32 and the quotient does not change.
// Bound by the tensor cores and by the exponentials (16 per clock and SM against 128 x 128 per 1024 clocks of MMA).
//
// Every wait is bounded: one that runs out sets MOE_ERR_TIMEOUT, the CTA stops issuing work, waits for its
// own MMAs and copies, frees its tensor memory and returns.
#include <algorithm>
#include <type_traits>

#include "attention_internal.cuh"

namespace moe {
namespace attn {

constexpr int BM = 128;      // rows of a tile
constexpr int BN = 128;      // keys of a tile
constexpr int NQ = 2;        // tiles of a CTA
constexpr int STAGES = 2;    // K tiles and V tiles in flight
constexpr int SOFTMAX_WARPS = 4 * NQ;
constexpr int MMA_WARP = SOFTMAX_WARPS;
constexpr int LOAD_WARP = SOFTMAX_WARPS + 1;
constexpr int PF_THREADS = (SOFTMAX_WARPS + 2) * 32;
constexpr int TMEM_COLS = 512;
constexpr int S_COL = 0;            // S_i / P_i at columns BN * i
constexpr int O_COL = NQ * BN;      // O_i at columns O_COL + D * i
constexpr float RESCALE = 8.0f;     // log2 of how far a row's reference may lag behind its maximum

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// SWIZZLE_128B shared-memory matrix descriptor, slabs of 64 values x n rows of 128 bytes, 8-row groups 1024 bytes
// apart. Q and K: K-major (the leading offset is not used). V: MN-major, the next 64 output columns lie
// `leading` bytes on.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t leading) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16 instruction descriptor: f32 accumulator, A and B both bf16 or both f16, M = 128, N = n.
template <class T>
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn_major) {
  const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(BM >> 4) << 24);
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{.reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{.reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// 32 columns of this warp's 32 tensor-memory lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

template <int D>
struct PfShape {
  static constexpr int SLAB = BN * 128;            // 64 values x 128 rows
  static constexpr int TILE = (D / 64) * SLAB;     // a Q, K or V tile
  static constexpr int BYTES = (NQ + 2 * STAGES) * TILE + 1024;
};

struct Bars {
  uint64_t k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES];
  uint64_t s_full[NQ], p_full[NQ], o_full[NQ], drained;
};

template <class T, int D, bool CAP>
__global__ void __launch_bounds__(PF_THREADS, 1)
    prefill_kernel(PrefillParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using S = PfShape<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sQ = smem;
  unsigned char* sK = sQ + NQ * S::TILE;
  unsigned char* sV = sK + STAGES * S::TILE;
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ int s_scan[PF_THREADS / 32];
  __shared__ int s_b, s_tile, s_k_issued, s_v_issued;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &s_abort;

  pdl_wait();
  pdl_trigger();
  if (*reinterpret_cast<volatile int32_t*>(p.err) == (int32_t)MOE_ERR_TIMEOUT) return;

  // ---- which sequence and which token tile: CTAs in order of sequence, the last tiles (the most keys) first ----
  const int tq = BM / p.group, span = NQ * tq;  // tokens of a tile, of a CTA
  const int kvh = blockIdx.x % p.kv_heads;
  const int u = gridDim.x / p.kv_heads - 1 - blockIdx.x / p.kv_heads;
  {
    const int per = (p.B + PF_THREADS - 1) / PF_THREADS;
    int mine = 0;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    for (int b = b0; b < b1; ++b) mine += (max(0, __ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b)) + span - 1) / span;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(FULL, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    if (tid == 0) s_b = -1;
    __syncthreads();
    int before = incl - mine;
    for (int w = 0; w < warp; ++w) before += s_scan[w];
    if (u >= before && u < before + mine) {
      int b = b0, at = before;
      for (;; ++b) {
        const int n = (max(0, __ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b)) + span - 1) / span;
        if (u < at + n) break;
        at += n;
      }
      s_b = b;
      s_tile = u - at;
    }
  }
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.k_free[i], 1);
      mbar_init(&bars.v_free[i], 1);
    }
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    s_k_issued = s_v_issued = 0;
  }
  __syncthreads();
  const int b = s_b;
  if (b < 0) return;  // uniform over the CTA: no tile left
  const int row0 = __ldg(p.cu_q + b), news = min(__ldg(p.cu_q + b + 1), p.T) - row0;
  const int asked = __ldg(p.seq_lens + b);
  const int len = max(0, min(asked, p.max_pages << p.page_shift));
  const int past = len - news;  // position of the chunk's first row (negative: rows before position 0 see nothing)
  if ((asked != len || past < 0 || row0 < 0) && tid == 0) latch(p.err, MOE_ERR_BAD_IDS);
  if (row0 < 0) return;
  const int t0 = s_tile * span;                         // first token of the CTA within the chunk
  const int t1 = min(news, t0 + span);                  // one past its last
  const int hi = max(0, past + t1);                     // keys [lo, hi)
  const int lo = p.window > 0 ? max(0, past + t0 - p.window + 1) : 0;
  const int j0 = lo / BN;
  const int tiles = hi > lo ? (hi + BN - 1) / BN - j0 : 0;

  // ---- Q into shared memory, swizzled as TMA would ----
  for (int e = tid; e < NQ * BM * (D / 8); e += PF_THREADS) {
    const int c = e % (D / 8), r = e / (D / 8), i = r / BM, rr = r % BM;
    const int tok = t0 + i * tq + rr / p.group;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (rr < tq * p.group && tok < t1)
      v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (int64_t)(row0 + tok) * p.q_token_stride +
                                          (int64_t)(kvh * p.group + rr % p.group) * p.q_head_stride + c * 8);
    *reinterpret_cast<uint4*>(sQ + i * S::TILE + (c / 8) * S::SLAB + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v;
  }
  proxy_fence();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s_tmem;

  if (warp == LOAD_WARP) {
    // ---------------- K and V tiles: each lane loads the boxes of its pages ----------------
    const int box_rows = 1 << p.page_shift;
    const int pages = BN >> p.page_shift;  // per tile
    const int boxes = pages * (D / 64);    // at most 16
    for (int j = 0; j < tiles; ++j) {
      const int base = (j0 + j) * BN;
      const int live = min(pages, (len - base + box_rows - 1) >> p.page_shift);  // pages that hold tokens
      const int st = j % STAGES;
      int page = 0;
      const int my = lane % pages;  // this lane's page and 64-value half
      const int half = lane / pages;
      const bool on = lane < boxes && my < live;
      if (on) page = __ldg(p.page_table + (int64_t)b * p.max_pages + (base >> p.page_shift) + my);
      if (on && (unsigned)page >= (unsigned)p.num_pages) {
        latch(p.err, MOE_ERR_BAD_IDS);
        page = p.num_pages;  // out of the map: the box reads as zeros
      }
      bool ok = true;
      for (int kv = 0; kv < 2 && ok; ++kv) {
        uint64_t* full = kv ? &bars.v_full[st] : &bars.k_full[st];
        uint64_t* free_ = kv ? &bars.v_free[st] : &bars.k_free[st];
        ok = j < STAGES || mbar_wait(free_, ((j / STAGES) - 1) & 1, abort);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(full, (uint32_t)(live * box_rows * (D / 64) * 128));
          if (kv) s_v_issued = j + 1;
          else s_k_issued = j + 1;
        }
        __syncwarp();
        if (on)
          tma_load_4d((kv ? sV : sK) + st * S::TILE + half * S::SLAB + my * box_rows * 128, kv ? &v_map : &k_map, half * 64,
                      0, kvh, page, full);
      }
      if (!ok) {
        if (lane == 0) s_abort = 1;
        break;
      }
    }
  } else if (warp == MMA_WARP) {
    // ---------------- MMA issue (lane 0); the whole warp clears values past the length ----------------
    const uint64_t qd = sw128_desc(smem_u32(sQ), 16), kd = sw128_desc(smem_u32(sK), 16);
    const uint64_t vd = sw128_desc(smem_u32(sV), S::SLAB);
    const uint32_t id_s = idesc<T>(BN, false), id_o = idesc<T>(D, true);
    auto qk = [&](int i, int st) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (uint32_t)((k >> 2) * S::SLAB + (k & 3) * 32);
        umma_ss(tmem + S_COL + i * BN, qd + ((i * S::TILE + off) >> 4), kd + ((st * S::TILE + off) >> 4), id_s, k > 0);
      }
      commit(&bars.s_full[i]);
    };
    bool ok = true;
    for (int j = -1; j < tiles && ok && tiles > 0; ++j) {
      const int sv = j % STAGES, sk = (j + 1) % STAGES;
      const bool more = j + 1 < tiles;
      if (more) ok = mbar_wait(&bars.k_full[sk], ((j + 1) / STAGES) & 1, abort);
      if (j >= 0) {
        ok = ok && mbar_wait(&bars.v_full[sv], (j / STAGES) & 1, abort);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        // values past the sequence's length (the rest of its last page, pages not loaded) may be anything, and
        // 0 * NaN is NaN: clear them
        const int valid = len - (j0 + j) * BN;
        if (valid < BN) {
          for (int e = lane; e < (BN - valid) * (D / 8); e += 32) {
            const int r = valid + e / (D / 8), c = e % (D / 8);
            *reinterpret_cast<uint4*>(sV + sv * S::TILE + (c / 8) * S::SLAB + r * 128 + ((c & 7) << 4)) =
                make_uint4(0, 0, 0, 0);
          }
          proxy_fence();
        }
        __syncwarp();
      }
      ok = __all_sync(FULL, ok);
      if (!ok) break;
      for (int i = 0; i < NQ; ++i) {
        if (j >= 0) {
          ok = mbar_wait(&bars.p_full[i], j & 1, abort);
          ok = __all_sync(FULL, ok);
          if (!ok) break;
          tc_after();
          if (lane == 0) {
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              umma_ts(tmem + O_COL + i * D, tmem + S_COL + i * BN + k * 8, vd + ((sv * S::TILE + k * 2048) >> 4), id_o,
                      j > 0 || k > 0);
            commit(&bars.o_full[i]);
            if (i == NQ - 1 && j + STAGES < tiles) commit(&bars.v_free[sv]);
          }
        }
        // S_i of the next keys: issued behind the product that reads P_i from the same columns
        if (more && lane == 0) {
          qk(i, sk);
          if (i == NQ - 1 && j + 1 + STAGES < tiles) commit(&bars.k_free[sk]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (lane == 0) {
        s_abort = 1;
        commit(&bars.drained);  // every MMA issued so far lands before the CTA goes on
        (void)mbar_wait(&bars.drained, 0, nullptr);
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax: one row per thread ----------------
    const int i = warp >> 2, quad = warp & 3;
    const int rr = quad * 32 + lane;
    const int first = t0 + i * tq;  // first token of the tile
    const int tok = first + rr / p.group;
    const bool live = rr < tq * p.group && tok < t1;
    const int pos = past + tok;  // this row sees keys (pos - window, pos]
    const int key_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_at = lane_base + S_COL + i * BN, o_at = lane_base + O_COL + i * D;
    const float c_log2 = p.scale * LOG2E;
    float m = -INFINITY, l = 0.0f;  // reference in units of log2, sum of weights
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      ok = mbar_wait(&bars.s_full[i], j & 1, abort);
      // the product with the previous tile's P has been issued before this S, and finished: its phase is taken
      // note of here, and O may be rescaled
      if (ok && j > 0) ok = mbar_wait(&bars.o_full[i], (j - 1) & 1, abort);
      ok = __all_sync(FULL, ok);
      if (!ok) break;
      tc_after();
      const int base = (j0 + j) * BN;
      // keys that every live row of the tile sees need no mask
      const bool full = base + BN - 1 <= past + first &&
                        (p.window <= 0 || base > past + min(t1, first + tq) - 1 - p.window);
      const int from = full ? 0 : key_lo - base, to = full ? BN : pos + 1 - base;  // columns [from, to)
      auto score = [&](uint32_t raw, int col) {
        float x = __uint_as_float(raw);
        if (CAP) {
          // softcap * tanh(x): 1 - 2 / (e^2x + 1), absolute error about 1e-7 of the cap
          const float e = ex2(x * (2.0f * LOG2E * p.scale / p.softcap));
          x = p.softcap * LOG2E * (1.0f - __fdividef(2.0f, e + 1.0f));
        } else {
          x *= c_log2;
        }
        return (col >= from && col < to) ? x : -INFINITY;
      };
      uint32_t r[32];
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        tmem_ld32(s_at + c * 32, r);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) mx = fmaxf(mx, score(r[k], c * 32 + k));
      }
      const bool grow = mx > m + RESCALE;  // also the first finite maximum
      if (__any_sync(FULL, grow)) {
        const float mn = grow ? mx : m;
        const float f = grow ? ex2(m - mn) : 1.0f;
        m = mn;
        l *= f;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            tmem_ld32(o_at + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * f);
            tmem_st32(o_at + c * 32, r);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        tmem_ld32(s_at + c * 32, r);
        tmem_wait_ld();
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float a = ex2(score(r[2 * k], c * 32 + 2 * k) - ref);
          const float e = ex2(score(r[2 * k + 1], c * 32 + 2 * k + 1) - ref);
          l += a + e;
          w[k] = Elem<T>::pack(a, e);
        }
        tmem_st16(s_at + c * 16, w);  // columns of S that this row has already read
      }
      tmem_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[i]);
    }
    if (ok && tiles > 0) {
      ok = mbar_wait(&bars.o_full[i], (tiles - 1) & 1, abort);
      ok = __all_sync(FULL, ok);
    }
    if (!ok) {
      if (lane == 0) s_abort = 1;
    } else {
      tc_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t row = (int64_t)(row0 + tok) * p.heads + kvh * p.group + rr % p.group;
      T* dst = static_cast<T*>(p.y) + row * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (tiles > 0) {
          tmem_ld32(o_at + c * 32, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        if (live) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)  // a row that saw nothing gives zeros
            w[k] = l == 0.0f ? 0u
                             : Elem<T>::pack(__uint_as_float(r[2 * k]) * inv, __uint_as_float(r[2 * k + 1]) * inv);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(dst + c * 32 + k * 8) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
      }
      if (live && p.lse) p.lse[row] = l == 0.0f ? -INFINITY : m * LN2 + logf(l);
    }
  }
  __syncthreads();
  if (s_abort && tid == 0) {  // the copies still in flight land before the CTA's shared memory goes
    for (int j = max(0, s_k_issued - STAGES); j < s_k_issued; ++j)
      (void)mbar_wait(&bars.k_full[j % STAGES], (j / STAGES) & 1, nullptr);
    for (int j = max(0, s_v_issued - STAGES); j < s_v_issued; ++j)
      (void)mbar_wait(&bars.v_full[j % STAGES], (j / STAGES) & 1, nullptr);
    atomicExch(p.err, (int)MOE_ERR_TIMEOUT);
  }
  tc_before();
  __syncthreads();
  if (warp == MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
}

// f(kernel, dynamic shared memory) for the handle's types and sizes.
template <class F>
static moe_status with_kernel(const moe_attn& a, F&& f) {
  auto by_type = [&](auto zero) -> moe_status {
    using T = decltype(zero);
    const bool cap = a.d.softcap > 0.0f;
    if (a.d.head_dim == 64)
      return cap ? f(prefill_kernel<T, 64, true>, PfShape<64>::BYTES) : f(prefill_kernel<T, 64, false>, PfShape<64>::BYTES);
    return cap ? f(prefill_kernel<T, 128, true>, PfShape<128>::BYTES)
               : f(prefill_kernel<T, 128, false>, PfShape<128>::BYTES);
  };
  return a.d.dtype == MOE_ATTN_BF16 ? by_type(__nv_bfloat16()) : by_type(__half());
}

moe_status prepare_prefill(const moe_attn& a) {
  return with_kernel(a, [](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return MOE_OK;
  });
}

moe_status launch_prefill(const moe_attn& a, const PrefillParams& p, cudaStream_t st) {
  const int span = NQ * (BM / p.group);
  // every sequence wastes less than one tile: CTAs past the last tile leave at once
  const int64_t grid = ((int64_t)p.T / span + std::min(p.B, p.T)) * p.kv_heads;
  if (grid > 0x7fffffffll) return fail(MOE_ERR_INVALID, "moe_attn_prefill: too many rows");
  return with_kernel(a, [&](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)grid), dim3(PF_THREADS), smem, st, p, a.k_map, a.v_map));
    return MOE_OK;
  });
}

moe_status make_page_tmap(CUtensorMap* map, int dtype, const void* pool, int head_dim, int page_size, int kv_heads,
                          int64_t num_pages, int64_t page_stride) {
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)kv_heads, (cuuint64_t)num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)page_size * head_dim * 2,
                                 (cuuint64_t)page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)page_size, 1, 1};
  return encode_tmap_sw128(map, dtype == MOE_ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           4, pool, dims, strides, box);
}

}  // namespace attn
}  // namespace moe
