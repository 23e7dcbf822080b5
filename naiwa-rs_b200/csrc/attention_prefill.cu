// attention_prefill.cu — causal attention of a ragged batch of prompt chunks over a paged key/value cache,
// on the 5th-generation tensor cores.
//
//   x_ij = scale * (q_i . k_j)  (or softcap * tanh(x_ij / softcap)),  pos_i - window < j <= pos_i
//   y_i  = sum_j exp(x_ij - m_i) v_j / sum_j exp(x_ij - m_i),   lse_i = m_i + log sum_j exp(x_ij - m_i)
//
// A tile is 128 rows = (128 / group) tokens x the group's query heads, so the heads that share keys and
// values share their loads. An item is two tiles (256 rows, consecutive tokens of one sequence and one key/value
// head); its keys are walked 128 at a time (a step). Few items are each cut along the keys into equal pieces, whose
// results are joined by the last to arrive, in the pieces' order. The kernel is persistent: one CTA per SM takes
// pieces from a counter, those with the most keys first, and runs its roles over them without a break:
//   * one warp takes the pieces, hands them to the other roles through a small ring, and loads by TMA (SWIZZLE_128B): Q
//     (64 values x the group's heads x a tile's tokens per box) once the piece before has issued its last scores, and K
//     (64 values x a page's tokens per box) into a ring of STAGES tiles; another warp loads V likewise;
//   * one thread issues S_i = Q_i K^T (128 x 128, f32 in tensor memory) and O_i += P_i V, alternating the
//     two tiles, so the tensor cores work on one tile while the other's softmax runs;
//   * four warps per tile hold one row per thread: maximum, exponentials and sum in f32, P rounded to the
//     values' type (what the tensor cores take; the sum is of the unrounded weights) and written over S in tensor
//     memory, from where the second product reads it. O is rescaled only when a row's maximum grows by more than
//     2^RESCALE (rare after the first steps), which leaves P below 2^RESCALE: the quotient does not change. f16 weights
//     take the rest of the type's range, another 2^11, so that only those below 2^-36 of the reference vanish.
// Bound by the tensor cores (1024 clocks of MMA per 128 x 128 step) and as much by the exponentials (16 per clock and SM).
// Measured on a B200: a step of two tiles takes about 3050 clocks of the 2062 that its MMAs need; the rest is the chain from
// scores to weights and back. A 4096-token prompt of 32 + 4 heads of 128: 142 us (0.97 PFLOP/s, 58% of the measured burst
// peak, 69% of the sustained one). The weights' rounding (8 bits in bf16, 11 in f16) is what tcgen05.mma takes: errors
// against 64 bits are 2.0e-3 to 2.3e-3 in bf16 where f32 weights give 1.6e-3, 2.6e-4 against 2.1e-4 in f16. Not taken
// (times of the steps they were weighed in, on a rested GPU): two threads a row (197 us against 157), an MMA warp per tile (137 against
// 129), three stages of K or V (129 against 127), exponentials by polynomials (125 to 131 against 126).
//
// Every wait is bounded (moe_attn_set_wait_limit): one that runs out sets MOE_ERR_TIMEOUT, the CTA stops issuing work, waits for
// its own MMAs and copies, frees its tensor memory and returns.
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
constexpr int V_WARP = SOFTMAX_WARPS + 2;
constexpr int PF_THREADS = (SOFTMAX_WARPS + 4) * 32;  // the last warp writes the rows that no sequence holds
// registers per thread: 168 at launch (384 threads), shared out anew: 2 x 216 + 72 = 3 x 168
constexpr int SOFTMAX_REGS = 216, OTHER_REGS = 72;
constexpr int RING = 4;              // pieces handed out ahead
constexpr int CONSUMERS = SOFTMAX_WARPS + 2;
constexpr int MAX_CUT = 16;          // pieces of an item
constexpr int PIECE_COST = 3;        // what a piece costs beside its steps, in steps (Q, epilogue, join)
constexpr int MOST = BN / 32;        // products of P V (of BN / 16) that start before the rest of P is there
constexpr int TMEM_COLS = 512;
constexpr int S_COL = 0;            // S_i / P_i at columns BN * i
constexpr int O_COL = NQ * BN;      // O_i at columns O_COL + D * i
// log2 of how far a row's reference may lag behind its maximum; f16 weights need the rest of the type's range
template <class T>
constexpr float RESCALE = Elem<T>::kWeightBits ? 4.0f : 8.0f;

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n"
               "cp.async.bulk.commit_group;" ::"l"(map),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 x, y, z;\n"
      "mov.b64 x, {%2, %3};\n"
      "mov.b64 y, {%4, %5};\n"
      "mov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 x, x, y, z;\n"
      "mov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y;\n"
      "mov.b64 x, {%2, %3};\n"
      "mov.b64 y, {%4, %5};\n"
      "add.rn.f32x2 x, x, y;\n"
      "mov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// The bound of this launch's waits: SM clocks, the suspend hint that goes with them, and the flag of a role that gave up.
struct Waits {
  uint32_t limit, suspend;
  volatile int* abort;
};

// Bounded parity wait that sleeps; false once the limit has passed or another role gave up.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, const Waits& w) {
  const uint32_t a = smem_u32(bar);
  uint32_t done;
  asm volatile(
      "{.reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;}"
      : "=r"(done)
      : "r"(a), "r"(parity)
      : "memory");
  if (done) return true;
  const long long t0 = clock64();
#pragma unroll 1
  for (uint32_t i = 0; i < WAIT_POLLS; ++i) {
    if (*w.abort || clock64() - t0 > w.limit) return false;
    if (mbar_try_sleep(a, parity, w.suspend)) return true;
  }
  return false;
}

// The same without the suspend-time hint and in few instructions.
__device__ __forceinline__ bool wait_poll(uint64_t* bar, uint32_t parity, const Waits& w) {
  const uint32_t a = smem_u32(bar);
  uint32_t t0 = 0;
#pragma unroll 1
  while (!mbar_try(a, parity)) {
    const uint32_t t = (uint32_t)clock() | 1u;
    if (t0 == 0) t0 = t;
    if (*w.abort || t - t0 > w.limit) return false;
  }
  return true;
}

// log2 of what the weights of a type are scaled by: with the reference up to RESCALE behind they reach 2^15 in f16.
template <class T>
constexpr float PREFILL_SCALE = Elem<T>::kWeightBits ? Elem<T>::kWeightBits - RESCALE<T> : 0.0f;

// Low word of a SWIZZLE_128B shared-memory matrix descriptor, slabs of 64 values x n rows of 128 bytes, 8-row groups 1024
// bytes apart; the high word is the same for all. Q and K: K-major (the leading offset is not used). V: MN-major, the next
// 64 output columns lie `leading` bytes on. Addresses below 256 KB: adding (bytes >> 4) moves the start.
__device__ __forceinline__ uint32_t sw128_desc(uint32_t addr, uint32_t leading) {
  return ((addr >> 4) & 0x3FFF) | ((leading >> 4) << 16);
}
constexpr uint32_t SW128_HIGH = (1024 >> 4) | (1u << 14) | (2u << 29);

// kind::f16 instruction descriptor: f32 accumulator, A and B both bf16 or both f16, M = 128, N = n.
template <class T>
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(BM >> 4) << 24);
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{.reg .pred p;\n"
      ".reg .b64 x, y;\n"
      "mov.b64 x, {%1, %5};\n"
      "mov.b64 y, {%2, %5};\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(accumulate), "n"(SW128_HIGH)
      : "memory");
}

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{.reg .pred p;\n"
      ".reg .b64 y;\n"
      "mov.b64 y, {%2, %5};\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(accumulate), "n"(SW128_HIGH)
      : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// One lane of the converged warp, the same one each time. The MMA warp runs converged on values made uniform and issues
// inside `if (elect())`, where the compiler keeps the operands in uniform registers. Measured beside 16 warps of
// arithmetic: 64 clocks per tcgen05.mma, its execution time; inside an `if (lane == 0)` 77, with a predicate per
// instruction 87, and 105 with operands that were not made uniform first.
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile(
      "{.reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;}"
      : "=r"(e));
  return e != 0;
}

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(FULL, v, 0); }

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

__device__ __forceinline__ void tmem_ld16u(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <int D>
struct PfShape {
  static constexpr int SLAB = BN * 128;            // 64 values x 128 rows
  static constexpr int TILE = (D / 64) * SLAB;     // a Q, K or V tile
  static constexpr int OUT = 32 * 128;             // a softmax warp's rows x 64 output values, on their way out
  static constexpr int BYTES = (NQ + 2 * STAGES) * TILE + SOFTMAX_WARPS * OUT + 1024;
};

struct Bars {
  uint64_t k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES];
  uint64_t s_full[NQ], p_most[NQ], p_full[NQ], o_full[NQ], q_full, q_free, item_full[RING], item_free[RING], drained;
};

// A piece of work: steps [j0, j0 + steps) over the keys of one item. row0: the sequence's first row; past: the position
// of that row; [t0, t1): the item's tokens; lo: the first key that one of them sees. b < 0: no more work.
struct Piece {
  int b, kvh, row0, past, t0, t1, len, lo, j0, steps, cut, k, item;
};

// The batch as the load warp sees it: each lane holds the tiles of its sequences and their prefix.
struct Batch {
  int per, before, mine, items, cut;
};

__device__ __forceinline__ int tokens_of(const PrefillParams& p, int b) {
  return max(0, min(p.cu_q[b + 1], p.T) - max(0, p.cu_q[b]));
}

__device__ __forceinline__ Batch read_batch(const PrefillParams& p, int span, int lane, int ctas, int join_cost) {
  Batch s;
  s.per = (p.B + 31) / 32;
  s.mine = 0;
  int most = 0;  // steps of the longest item
#pragma unroll 1
  for (int b = min(p.B, lane * s.per); b < min(p.B, (lane + 1) * s.per); ++b) {
    const int n = tokens_of(p, b);
    if (n == 0) continue;
    s.mine += (n + span - 1) / span;
    const int len = min(p.seq_lens[b], p.max_pages << p.page_shift);
    most = max(most, (p.window > 0 ? min(len, p.window + span + BN) : len) / BN + 1);
  }
  int incl = s.mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, incl, o);
    if (lane >= o) incl += v;
  }
  s.before = incl - s.mine;
  s.items = __shfl_sync(FULL, incl, 31) * p.kv_heads;
  most = __reduce_max_sync(FULL, most);
  // The cut that costs the longest CTA least, in half steps: its rounds of pieces, and the join, one CTA's work, that reads
  // every piece's rows.
  s.cut = 1;
  if (s.items > 0) {
    int best = 0x7fffffff;
    const int cut = lane + 1;
    if (cut <= MAX_CUT && (cut == 1 || (int64_t)s.items * cut <= 2 * ctas)) {
      const int rounds = (s.items * cut + ctas - 1) / ctas;
      best = 2 * rounds * ((most + cut - 1) / cut + PIECE_COST) + (cut > 1 ? cut * join_cost : 0);
    }
    const int least = __reduce_min_sync(FULL, best);
    s.cut = __ffs(__ballot_sync(FULL, best == least));  // the smallest such cut
  }
  return s;
}

// Piece number w of the launch (warp-collective): items by sequence, the last tokens (the most keys) first.
__device__ __forceinline__ Piece piece_of(const PrefillParams& p, const Batch& s, int w, int span, int lane) {
  Piece q{};
  q.b = -1;
  if (w >= s.items * s.cut) return q;
  q.cut = s.cut;
  q.item = w / s.cut;
  q.k = w % s.cut;
  q.kvh = q.item % p.kv_heads;
  const int u = s.items / p.kv_heads - 1 - q.item / p.kv_heads;
  const bool here = u >= s.before && u < s.before + s.mine;
  int b = 0, tile = 0;
  if (here) {
    int at = s.before;
#pragma unroll 1
    for (b = lane * s.per;; ++b) {
      const int n = (tokens_of(p, b) + span - 1) / span;
      if (u < at + n) break;
      at += n;
    }
    tile = u - at;
  }
  const int src = __ffs(__ballot_sync(FULL, here)) - 1;
  q.b = __shfl_sync(FULL, b, src);
  tile = __shfl_sync(FULL, tile, src);
  q.row0 = max(0, p.cu_q[q.b]);
  const int news = tokens_of(p, q.b), asked = p.seq_lens[q.b];
  q.len = max(0, min(asked, p.max_pages << p.page_shift));
  q.past = q.len - news;  // negative: rows before position 0 see nothing
  if (lane == 0 && (asked != q.len || q.past < 0)) latch(p.err, MOE_ERR_BAD_IDS);
  q.t0 = tile * span;
  q.t1 = min(news, q.t0 + span);
  const int hi = max(0, q.past + q.t1);  // keys [lo, hi)
  q.lo = p.window > 0 ? max(0, q.past + q.t0 - p.window + 1) : 0;
  const int first = q.lo / BN, all = hi > q.lo ? (hi + BN - 1) / BN - first : 0;
  const int a = all * q.k / q.cut;  // all < 2^24, cut <= MAX_CUT
  q.j0 = first + a;
  q.steps = all * (q.k + 1) / q.cut - a;
  return q;
}

// Half steps that a piece more costs its join (256 rows of D f32 values against a step's products and, capped, three
// exponential-unit results per score). Measured (captured calls, 32 + 4 heads, bf16), costs 0 / 1 / 2 / 3: heads of 128, 64 rows behind
// 4096 tokens 34.2 / 34.1 / 33.8 / 33.8 us, 200 rows 19.3 / 12.2 / 12.1 / 12.1, 128 behind 512 25.8 / 22.4 / 22.3 / 16.9; the same
// capped 40.2 / 44.8 / 49.2 / 49.2, 22.0 / 16.8 / 16.8 / 16.7, 28.6 / 27.2 / 29.8 / 28.5; heads of 64, 64 behind 4096
// 23.2 / 24.0 / 25.4 / 25.4, capped 40 behind 700 19.7 / 21.0 / 24.5 / 30.6.
template <int D, bool CAP>
struct JoinCost {
  static constexpr int value = D == 64 || CAP ? 1 : 3;
};

template <class T, int D, bool CAP>
__global__ void __launch_bounds__(PF_THREADS, 1)
    prefill_kernel(PrefillParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap y_map) {
  using S = PfShape<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sQ = smem;
  unsigned char* sK = sQ + NQ * S::TILE;
  unsigned char* sV = sK + STAGES * S::TILE;
  unsigned char* sO = sV + STAGES * S::TILE;
  __shared__ Bars bars;
  __shared__ Piece s_items[RING];
  __shared__ Batch s_batch[32];  // the load warp's lanes' (registers are short there)
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ int s_k_issued, s_v_issued, s_q_issued;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Waits waits = {p.wait_limit, min(p.wait_limit, SUSPEND_NS), &s_abort};
  // The last CTA to leave puts the counter of pieces back for the next call; a CTA that has nothing to do counts as well.
  auto leave = [&]() {
    __threadfence();
    if (atomicAdd(p.work + 1, 1) == (int)gridDim.x - 1) {
      p.work[0] = 0;
      p.work[1] = 0;
    }
  };
  const int tq = BM / p.group, span = NQ * tq;  // tokens of a tile, of an item

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.k_free[i], 1);
      mbar_init(&bars.v_free[i], 1);
    }
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_most[i], 4);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_full[i], 1);
    }
    for (int i = 0; i < RING; ++i) {
      mbar_init(&bars.item_full[i], 1);
      mbar_init(&bars.item_free[i], CONSUMERS);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_free, 1);
    mbar_init(&bars.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_k_issued = s_v_issued = s_q_issued = 0;
  }
  if (tid == PF_THREADS - 1) {  // the maps' own latency passes behind the set-up
    for (const CUtensorMap* map : {&q_map, &k_map, &v_map})
      asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  // rows of a tile that no box fills (a group that does not divide 128) stay zero
  if (tq * p.group < BM)
    for (int e = tid; e < NQ * S::TILE / 16; e += PF_THREADS) reinterpret_cast<uint4*>(sQ)[e] = make_uint4(0, 0, 0, 0);
  proxy_fence();
  pdl_wait();
  pdl_trigger();
  // after a wait that gave up nothing runs until moe_attn_check; one thread looks, since other CTAs may be setting the word
  if (tid == 0) s_abort = *reinterpret_cast<volatile int32_t*>(p.err) == (int32_t)MOE_ERR_TIMEOUT;
  __syncthreads();
  if (s_abort) {
    if (tid == 0) leave();
    return;
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s_tmem;

  // The n-th piece for a consuming warp; false once a wait gave up. Lane 0 releases the slot.
  auto take = [&](int n, Piece* q) -> bool {
    const int slot = n % RING;
    const bool ok = __all_sync(FULL, wait_for(&bars.item_full[slot], (n / RING) & 1, waits));
    if (!ok) return false;
    *q = s_items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.item_free[slot]);
    return true;
  };

  if (warp >= SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == LOAD_WARP || warp == V_WARP) {
      // One warp takes the pieces and loads their Q and K tiles, another their V tiles: with 16-token pages a tile is 16
      // boxes, one lane each, and they are issued one after the other.
      const bool is_v = warp == V_WARP;
      const int box_rows = 1 << p.page_shift;
      const int pages = BN >> p.page_shift;  // per tile
      const int half = lane / pages;         // this lane's 64-value half and page: at most 16 boxes
      const int my = half < D / 64 ? lane % pages : pages;
      const int box_bytes = box_rows * (D / 64) * 128;
      unsigned char* dst = (is_v ? sV : sK) + half * S::SLAB + my * box_rows * 128;
      uint64_t* full = is_v ? bars.v_full : bars.k_full;
      uint64_t* free_ = is_v ? bars.v_free : bars.k_free;
      const CUtensorMap* map = is_v ? &v_map : &k_map;
      if (!is_v) s_batch[lane] = read_batch(p, span, lane, gridDim.x, JoinCost<D, CAP>::value);
      __syncwarp();
      int g = 0, used = 0, w = blockIdx.x;
      bool ok = true;
#pragma unroll 1
      for (int n = 0; ok; ++n) {
        Piece q;
        if (is_v) {
          ok = take(n, &q);
          if (!ok) break;
        } else {
          q = piece_of(p, s_batch[lane], w, span, lane);
          const int slot = n % RING;
          ok = __all_sync(FULL, n < RING || wait_for(&bars.item_free[slot], ((n / RING) - 1) & 1, waits));
          if (!ok) break;
          if (lane == 0) {
            s_items[slot] = q;
            mbar_arrive(&bars.item_full[slot]);
            if (q.b >= 0) w = gridDim.x + atomicAdd(p.work, 1);
          }
          w = __shfl_sync(FULL, w, 0);
        }
        if (q.b < 0) break;
        const int32_t* table = p.page_table + (int64_t)q.b * p.max_pages + my;
#pragma unroll 1
        for (int j = 0; j < q.steps; ++j, ++g) {
          const int base = (q.j0 + j) * BN, st = g % STAGES;
          // pages that hold tokens which a row sees: not those past the length, nor those wholly behind the window
          const int end = min(pages, (q.len - base + box_rows - 1) >> p.page_shift);
          const int begin = max(0, q.lo - base) >> p.page_shift;
          const bool on = my >= begin && my < end;
          int page = on ? table[base >> p.page_shift] : 0;
          if ((unsigned)page >= (unsigned)p.num_pages) {
            latch(p.err, MOE_ERR_BAD_IDS);
            page = p.num_pages;  // out of the map: the box reads as zeros
          }
          ok = __all_sync(FULL, wait_for(&free_[st], ((g / STAGES) & 1) ^ 1, waits));
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)((end - begin) * box_bytes));
          __syncwarp();
          if (on) tma_load_4d(dst + st * S::TILE, map, half * 64, 0, q.kvh, page, &full[st]);
          if (j == 0 && !is_v) {  // Q behind the first K tile: its place is the last to come free
            ok = __all_sync(FULL, wait_for(&bars.q_free, (used & 1) ^ 1, waits));
            if (!ok) {
              ++g;
              break;
            }
            ++used;
            if (lane == 0) mbar_expect_tx(&bars.q_full, (uint32_t)(NQ * (D / 64) * tq * p.group * 128));
            __syncwarp();
            if (lane < NQ * (D / 64))
              tma_load_3d(sQ + (lane % NQ) * S::TILE + (lane / NQ) * S::SLAB, &q_map, lane / NQ * 64, q.kvh * p.group,
                          q.row0 + q.t0 + (lane % NQ) * tq, &bars.q_full);
          }
        }
      }
      if (lane == 0) {
        if (is_v) {
          s_v_issued = g;
        } else {
          s_k_issued = g;
          s_q_issued = used;
        }
        if (!ok) s_abort = 1;
      }
      // the releases of the last stages have landed before the CTA ends
#pragma unroll 1
      for (int c = max(0, g - STAGES); c < g && ok; ++c) ok = wait_for(&free_[c % STAGES], (c / STAGES) & 1, waits);
      if (ok && used > 0) ok = wait_for(&bars.q_free, (used - 1) & 1, waits);
      if (!ok && lane == 0) s_abort = 1;
      __syncwarp();
    } else if (warp == MMA_WARP) {
      // ---------------- the products; the whole warp clears values past the length ----------------
      const uint32_t tm = (uint32_t)uniform((int)tmem);
      const uint32_t qd = uniform(sw128_desc(smem_u32(sQ), 16)), kd = uniform(sw128_desc(smem_u32(sK), 16));
      const uint32_t vd = uniform(sw128_desc(smem_u32(sV), S::SLAB));
      constexpr uint32_t id_s = idesc<T>(BN, false), id_o = idesc<T>(D, true);
      bool ok = true;
      int g = 0, used = 0;
      uint32_t phase = 0;  // bit i: parity of tile i's next P
      // bits 2 i, 2 i + 1: tile i has committed scores, their last parity; bits 4 + 2 i, 5 + 2 i: outputs
      uint32_t committed = 0xaa;
#pragma unroll 1
      for (int n = 0; ok; ++n) {
        Piece q;
        ok = take(n, &q);
        if (!ok || uniform(q.b) < 0) break;
        const int steps = uniform(q.steps);
        if (steps == 0) continue;
        ok = __all_sync(FULL, wait_for(&bars.q_full, used & 1, waits));
        if (!ok) break;
        ++used;
        tc_after();
        const int tiles = uniform(q.t0 + tq < q.t1 ? 2 : 1);  // tiles with rows
#pragma unroll 1
        for (int j = -1; j < steps && ok; ++j) {
          // step j of this piece is the CTA's step g + j
          const int sv = (g + j + STAGES) % STAGES, sk = (g + j + 1) % STAGES;
          const bool more = j + 1 < steps;
          if (more) ok = wait_for(&bars.k_full[sk], ((g + j + 1) / STAGES) & 1, waits);
          if (j >= 0) {
            ok = ok && wait_for(&bars.v_full[sv], ((g + j) / STAGES) & 1, waits);
            // values past the sequence's length (the rest of its last page, pages not loaded) and behind the window may be
            // anything, and 0 * NaN is NaN: clear them, rows [0, head) and [valid, BN)
            const int valid = min(BN, q.len - (q.j0 + j) * BN), head = max(0, q.lo - (q.j0 + j) * BN);
            if ((valid < BN || head > 0) && __all_sync(FULL, ok)) {
#pragma unroll 1
              for (int e = lane; e < (BN - valid + head) * (D / 8); e += 32) {
                const int at = e / (D / 8), r = at < head ? at : valid + at - head, c = e % (D / 8);
                *reinterpret_cast<uint4*>(sV + sv * S::TILE + (c / 8) * S::SLAB + r * 128 + ((c & 7) << 4)) =
                    make_uint4(0, 0, 0, 0);
              }
              proxy_fence();
            }
            __syncwarp();
          }
          ok = __all_sync(FULL, ok);
          if (!ok) break;
          const uint32_t vb = vd + (uint32_t)(sv * (S::TILE >> 4)), kb = kd + (uint32_t)(sk * (S::TILE >> 4));
          // both tiles unrolled: this warp's own instructions lie on the chain from P to the next S
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if (i >= tiles) break;
            if (j >= 0) {
              // the product starts on the first keys' weights while the last ones are being computed
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                ok = __all_sync(FULL, wait_for(e ? &bars.p_full[i] : &bars.p_most[i], (phase >> i) & 1, waits));
                if (!ok) break;
                tc_after();
                if (elect()) {
#pragma unroll
                  for (int k = e ? MOST : 0; k < (e ? BN / 16 : MOST); ++k)
                    umma_ts(tm + O_COL + i * D, tm + S_COL + i * BN + k * 8, vb + (uint32_t)((k * 2048) >> 4), id_o,
                            j > 0 || k > 0);
                }
                __syncwarp();
              }
              if (!ok) break;
              phase ^= 1u << i;
            }
            // S_i of the next keys: issued behind the product that reads P_i from the same columns. One commit covers both
            // products: a commit costs the issuing warp as much as several products.
            if (elect()) {
              if (more) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  const uint32_t off = (uint32_t)((k >> 2) * S::SLAB + (k & 3) * 32);
                  umma_ss(tm + S_COL + i * BN, qd + ((i * S::TILE + off) >> 4), kb + (off >> 4), id_s, k > 0);
                }
                commit(&bars.s_full[i]);
              } else {
                commit(&bars.o_full[i]);
              }
            }
            __syncwarp();
            const int bit = 2 * i + (more ? 0 : 4);
            committed = (committed | 1u << bit) ^ 2u << bit;
          }
        }
        g += steps;
      }
      if (!ok && lane == 0) s_abort = 1;
      // Every MMA issued and every arrival of a commit lands before the CTA goes on, whichever role gave up (a softmax warp
      // may while the last product runs). A CTA that issued none has none to wait for.
      if (committed & 0x55) {
        if (elect()) commit(&bars.drained);
        (void)mbar_wait(&bars.drained, 0, nullptr);
        for (int i = 0; i < NQ; ++i) {
          if (committed >> (2 * i) & 1) (void)mbar_wait(&bars.s_full[i], committed >> (2 * i + 1) & 1, nullptr);
          if (committed >> (4 + 2 * i) & 1) (void)mbar_wait(&bars.o_full[i], committed >> (5 + 2 * i) & 1, nullptr);
        }
      }
      __syncwarp();
    } else {
      // ---------------- rows before cu_q[0] and from cu_q[B] on: padding, zeros and -inf ----------------
      const int first = p.B > 0 ? min(max(p.cu_q[0], 0), p.T) : 0;
      const int end = p.B > 0 ? min(max(p.cu_q[p.B], first), p.T) : 0;
      for (int r = blockIdx.x; r < p.T - (end - first); r += gridDim.x) {
        const int64_t row = (int64_t)(r < first ? r : r - first + end) * p.heads;
        for (int e = lane; e < p.heads * (D / 8); e += 32)
          reinterpret_cast<uint4*>(static_cast<T*>(p.y) + row * D)[e] = make_uint4(0, 0, 0, 0);
        if (p.lse)
          for (int e = lane; e < p.heads; e += 32) p.lse[row + e] = -INFINITY;
      }
      if (blockIdx.x == 0 && p.B > 0) {
        bool bad = p.cu_q[0] != 0 || p.cu_q[p.B] > p.T;
        for (int b = lane; b < p.B; b += 32) bad |= p.cu_q[b + 1] < p.cu_q[b];
        if (bad) latch(p.err, MOE_ERR_BAD_IDS);
      }
    }
  } else {
    // ---------------- softmax: one row per thread ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    const int i = warp >> 2, quad = warp & 3;
    const int rr = quad * 32 + lane;
    const int my_tok = i * tq + rr / p.group, my_head = rr % p.group;
    const bool my_row = rr < tq * p.group;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_at = lane_base + S_COL + i * BN, o_at = lane_base + O_COL + i * D;
    const float c_log2 = CAP ? 1.0f : p.scale * LOG2E;
    const Cap cap = make_cap(p.scale, CAP ? p.softcap : 1.0f);
    bool ok = true;
    int seen = 0;           // this tile's steps so far
    int g = 0, pieces = 0;  // the CTA's steps so far, this tile's pieces
#pragma unroll 1
    for (int n = 0; ok; ++n) {
      Piece q;
      ok = take(n, &q);
      if (!ok || q.b < 0) break;
      const int first = q.t0 + i * tq;  // first token of the tile
      if (first >= q.t1) {              // no rows in this tile
        g += q.steps;
        continue;
      }
      // the last tile with rows, whose products are issued last, lets go of Q, K and V for both
      const bool frees = (i == NQ - 1 || first + tq >= q.t1) && quad == 0 && lane == 0;
      const int tok = q.t0 + my_tok;
      const bool live = my_row && tok < q.t1;
      const int pos = q.past + tok;  // this row sees keys (pos - window, pos]
      const int key_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      float m = -INFINITY, l = 0.0f;  // reference in units of log2, sum of weights
#pragma unroll 1
      for (int j = 0; j < q.steps; ++j, ++seen) {
        ok = wait_poll(&bars.s_full[i], seen & 1, waits);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        // S complete means that every product issued before it is: the previous step's with P (O may be rescaled), and
        // the reads of its V and of this K
        if (frees) {
          mbar_arrive(&bars.k_free[(g + j) % STAGES]);
          if (j > 0) mbar_arrive(&bars.v_free[(g + j - 1) % STAGES]);
          if (j == q.steps - 1) mbar_arrive(&bars.q_free);
        }
        tc_after();
        uint32_t r[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
          tmem_ld32(s_at + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
        tmem_wait_ld();
        if (CAP) {
          if (cap.wide) {
#pragma unroll
            for (int k = 0; k < BN; ++k) r[k] = __float_as_uint(wide_capped_score(cap, __uint_as_float(r[k])));
          } else {
#pragma unroll
            for (int k = 0; k < BN; ++k) r[k] = __float_as_uint(capped_score(cap, __uint_as_float(r[k])));
          }
        }
        const int base = (q.j0 + j) * BN;
        // keys that every live row of the tile sees need no mask
        const bool masked =
            base + BN - 1 > q.past + first || (p.window > 0 && base <= q.past + min(q.t1, first + tq) - 1 - p.window);
        if (__builtin_expect(masked, 0)) {
          const int from = key_lo - base;
          const unsigned width = (unsigned)max(0, pos + 1 - key_lo);  // columns [from, from + width)
#pragma unroll
          for (int k = 0; k < BN; ++k)
            if ((unsigned)(k - from) >= width) r[k] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < BN; k += 8)
#pragma unroll
          for (int a = 0; a < 4; ++a)
            mx[a] = fmaxf(fmaxf(mx[a], __uint_as_float(r[k + 2 * a])), __uint_as_float(r[k + 2 * a + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c_log2;  // scale > 0
        const bool grow = top > m + RESCALE<T>;  // also the first finite maximum
        if (__builtin_expect(__any_sync(FULL, grow), 0)) {
          const float mn = grow ? top : m;
          const float f = grow ? ex2(m - mn) : 1.0f;
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16u(o_at + c * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(o_at + c * 16, o);
            }
          }
        }
        const float ref = (m == -INFINITY ? 0.0f : m) - PREFILL_SCALE<T>;
        // The weights, 32 columns at a time. The exponential unit sets the pace (a pair per 16 clocks): its instructions are
        // kept in program order, and the packing and summing of a pair follow AHEAD pairs behind, so that no chunk waits for
        // the unit's latency.
        constexpr int PAIRS = BN / 2, AHEAD = 4;
        float2 sum = make_float2(0.0f, 0.0f);
        float2 x[PAIRS];
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < PAIRS + AHEAD; ++k) {
          if (k < PAIRS) {
            x[k] = fma2(make_float2(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1])), make_float2(c_log2, c_log2),
                        make_float2(-ref, -ref));
            x[k].x = ex2_ordered(x[k].x);
            x[k].y = ex2_ordered(x[k].y);
          }
          const int e = k - AHEAD;
          if (e < 0) continue;
          sum = add2(sum, x[e]);
          w[e % 16] = Elem<T>::pack(x[e].x, x[e].y);
          if (e % 16 == 15) {
            tmem_st16(s_at + e / 16 * 16, w);  // columns of S, all of which this row has read
            if (e == MOST * 8 - 1) {
              tmem_wait_st();
              tc_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars.p_most[i]);
            }
          }
        }
        l += sum.x + sum.y;
        tmem_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[i]);
      }
      if (ok && q.steps > 0) {
        ok = __all_sync(FULL, wait_poll(&bars.o_full[i], pieces & 1, waits));
        ++pieces;
        if (ok && frees) mbar_arrive(&bars.v_free[(g + q.steps - 1) % STAGES]);
      }
      if (!ok) break;
      g += q.steps;
      tc_after();
      // ---- the piece's rows: out, or into the workspace ----
      const int64_t row = (int64_t)(q.row0 + tok) * p.heads + q.kvh * p.group + my_head;
      T* dst = static_cast<T*>(p.y) + row * D;
      const int64_t slot = (int64_t)q.item * q.cut * NQ + i;  // piece k of this tile at slot + k * NQ
      float4* part = p.partial + slot * (D / 4) * BM + rr;  // [D / 4][BM] of a slot
      const float inv = q.cut > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      // A warp whose 32 rows are whole tokens, all of them live, sends them out by TMA, 64 values of each at a time (32 / group
      // tokens x the group's heads): a store of a row per lane touches 32 lines, and 16 of them per warp took 4300
      // clocks of a piece.
      if (q.cut == 1 && q.steps > 0 && 32 % p.group == 0 && __all_sync(FULL, live)) {
        unsigned char* stage = sO + warp * S::OUT;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the stage has been read
          __syncwarp();
          uint32_t o2[2][32];
          tmem_ld32(o_at + c * 64, o2[0]);
          tmem_ld32(o_at + c * 64 + 32, o2[1]);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t(&o)[32] = o2[e];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int h = 0; h < 4; ++h)
                w[h] = Elem<T>::pack(__uint_as_float(o[8 * k + 2 * h]) * inv, __uint_as_float(o[8 * k + 2 * h + 1]) * inv);
              if (l == 0.0f) w[0] = w[1] = w[2] = w[3] = 0;  // nothing seen: zeros
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * e + k) ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          proxy_fence();
          __syncwarp();
          if (lane == 0)
            tma_store_3d(&y_map, stage, c * 64, q.kvh * p.group, q.row0 + first + quad * (32 / p.group));
        }
        if (p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (m - PREFILL_SCALE<T>) * LN2 + logf(l);
        continue;
      }
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        if (q.steps > 0) {
          tmem_ld16u(o_at + c * 16, o);
          tmem_wait_ld();
        }
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k] = l == 0.0f ? 0.0f : __uint_as_float(o[k]) * inv;  // nothing seen: zeros
        if (q.cut > 1) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            __stcg(part + ((int64_t)q.k * NQ * (D / 4) + c * 4 + k) * BM,
                   make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]));
        } else if (live) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<uint4*>(dst + c * 16 + k * 8) =
                make_uint4(Elem<T>::pack(f[8 * k], f[8 * k + 1]), Elem<T>::pack(f[8 * k + 2], f[8 * k + 3]),
                           Elem<T>::pack(f[8 * k + 4], f[8 * k + 5]), Elem<T>::pack(f[8 * k + 6], f[8 * k + 7]));
        }
      }
      if (q.cut == 1) {
        if (live && p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (m - PREFILL_SCALE<T>) * LN2 + logf(l);
        continue;
      }
      // ---- the last of the item's pieces to arrive joins them in order, each warp its own rows ----
      float2* ml = p.partial_ml + slot * BM + rr;  // piece k at k * NQ * BM
      constexpr int MLS = NQ * BM;
      __stcg(ml + q.k * MLS, make_float2(m, l));
      __threadfence();
      __syncwarp();
      int last = 0;
      if (lane == 0) {
        int32_t* cnt = p.counters + (q.item * NQ + i) * 4 + quad;
        last = atomicAdd(cnt, 1) == q.cut - 1;
        if (last) *cnt = 0;  // ready for the next call
      }
      if (__shfl_sync(FULL, last, 0)) {
        __threadfence();
        float M = -INFINITY, L = 0.0f;
#pragma unroll 4
        for (int k = 0; k < q.cut; ++k) M = fmaxf(M, ld_l2(ml + k * MLS).x);
        const float at = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
        for (int k = 0; k < q.cut; ++k) {
          const float2 v = ld_l2(ml + k * MLS);
          L += v.y * ex2(v.x - at);
        }
        const float il = L == 0.0f ? 0.0f : 1.0f / L;
        // 32 values at a time, two pieces' loads in flight together: the join is behind everything else, and its time is its
        // trips to L2
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float4 o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = make_float4(0, 0, 0, 0);
#pragma unroll 2
          for (int k = 0; k < q.cut; ++k) {
            float4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ld_l2(part + ((int64_t)k * NQ * (D / 4) + c * 8 + e) * BM);
            const float f = ex2(ld_l2(ml + k * MLS).x - at);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              o[e].x = fmaf(v[e].x, f, o[e].x), o[e].y = fmaf(v[e].y, f, o[e].y);
              o[e].z = fmaf(v[e].z, f, o[e].z), o[e].w = fmaf(v[e].w, f, o[e].w);
            }
          }
          if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) = make_uint4(
                  Elem<T>::pack(o[2 * e].x * il, o[2 * e].y * il), Elem<T>::pack(o[2 * e].z * il, o[2 * e].w * il),
                  Elem<T>::pack(o[2 * e + 1].x * il, o[2 * e + 1].y * il),
                  Elem<T>::pack(o[2 * e + 1].z * il, o[2 * e + 1].w * il));
          }
        }
        if (live && p.lse) p.lse[row] = L == 0.0f ? -INFINITY : (M - PREFILL_SCALE<T>) * LN2 + logf(L);
      }
    }
    if (!ok && lane == 0) s_abort = 1;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the rows on their way out are out
  }
  __syncthreads();
  if (tid == 0) {
    if (s_abort) {
      if (s_q_issued) (void)mbar_wait(&bars.q_full, (s_q_issued - 1) & 1, nullptr);
      // the copies still in flight land before the CTA's shared memory goes
#pragma unroll 1
      for (int j = max(0, s_k_issued - STAGES); j < s_k_issued; ++j)
        (void)mbar_wait(&bars.k_full[j % STAGES], (j / STAGES) & 1, nullptr);
#pragma unroll 1
      for (int j = max(0, s_v_issued - STAGES); j < s_v_issued; ++j)
        (void)mbar_wait(&bars.v_full[j % STAGES], (j / STAGES) & 1, nullptr);
      atomicExch(p.err, (int)MOE_ERR_TIMEOUT);
    }
    leave();
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

static CUtensorMapDataType map_type(int dtype) {
  return dtype == MOE_ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

moe_status prepare_prefill(const moe_attn& a) {
  return with_kernel(a, [](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return MOE_OK;
  });
}

moe_status launch_prefill(const moe_attn& a, const PrefillParams& p, cudaStream_t st) {
  const int tq = BM / p.group, span = NQ * tq;
  // every sequence wastes less than one item
  const int64_t items = ((int64_t)p.T / span + std::min(p.B, p.T)) * p.kv_heads;
  if (items > 0x3fffffff) return fail(MOE_ERR_INVALID, "moe_attn_prefill: too many rows");
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(a.sms, items * MAX_CUT));
  // strides of dimensions of size 1 are never used and may be anything
  const int64_t ts = p.T > 1 ? p.q_token_stride : (int64_t)p.heads * a.d.head_dim;
  const int64_t hs = p.heads > 1 ? p.q_head_stride : a.d.head_dim;
  if (ts <= 0 || hs <= 0 || ts >= (1ll << 38) || hs >= (1ll << 38))
    return fail(MOE_ERR_INVALID, "moe_attn_prefill: q strides must be positive");
  const cuuint64_t dims[3] = {(cuuint64_t)a.d.head_dim, (cuuint64_t)p.heads, (cuuint64_t)p.T};
  const cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)tq};
  CUtensorMap q_map;
  MOE_TRY(encode_tmap_sw128(&q_map, map_type(a.d.dtype), 3, p.q, dims, strides, box));
  // y: a softmax warp's whole tokens (the kernel stores by rows where a warp's rows are not)
  const cuuint64_t y_strides[2] = {(cuuint64_t)a.d.head_dim * 2, (cuuint64_t)p.heads * a.d.head_dim * 2};
  const bool whole = 32 % p.group == 0;
  const cuuint32_t y_box[3] = {64, whole ? (cuuint32_t)p.group : 1, whole ? 32u / p.group : 1};
  CUtensorMap y_map;
  MOE_TRY(encode_tmap_sw128(&y_map, map_type(a.d.dtype), 3, p.y, dims, y_strides, y_box));
  return with_kernel(a, [&](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(PF_THREADS), smem, st, p, q_map, a.k_map, a.v_map, y_map));
    return MOE_OK;
  });
}

size_t prefill_partial_bytes(const moe_attn& a) { return (size_t)2 * a.sms * NQ * BM * a.d.head_dim * sizeof(float); }
size_t prefill_ml_bytes(const moe_attn& a) { return (size_t)2 * a.sms * NQ * BM * sizeof(float2); }
size_t prefill_counters(const moe_attn& a) { return (size_t)2 * a.sms * NQ * 4; }

moe_status make_page_tmap(CUtensorMap* map, int dtype, const void* pool, int head_dim, int page_size, int kv_heads,
                          int64_t num_pages, int64_t page_stride) {
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)kv_heads, (cuuint64_t)num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)page_size * head_dim * 2,
                                 (cuuint64_t)page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)page_size, 1, 1};
  return encode_tmap_sw128(map, map_type(dtype), 4, pool, dims, strides, box);
}

}  // namespace attn
}  // namespace moe
