// attention_decode.cu — attention of one new token per sequence over a paged key/value cache.
//
//   x_j = scale * (q . k_j)  (or softcap * tanh(x_j / softcap)),  j in the sequence's last `window` slots
//   y   = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),   lse = m + log sum_j exp(x_j - m),   m = max_j x_j
//
// Bound by the cache bytes: 2 * length * kv_heads * head_dim * 2 per sequence, each read once. What the
// kernel must do is keep enough of them in flight on every SM whatever the batch and its lengths.
//
// Split. The batch's work is one line of 16-token blocks, ordered by (sequence, key/value head, block).
// Every CTA takes an equal slice of that line, so a single long sequence, a large batch and a ragged one
// all fill the GPU alike. The part of a slice that lies in one (sequence, head) is a piece: a piece that is
// the whole (sequence, head) is written out by its CTA; otherwise each CTA leaves its running maximum, sum
// and weighted values in the workspace, and the one that arrives last (a counter per (sequence, head))
// joins them in CTA order, so results do not depend on timing. The slices follow from the lengths on
// the device: no host read, one launch.
//
// Inside a CTA each warp runs alone over every WARPS-th block with its own ring of STAGES blocks filled by
// 16-byte cp.async: no CTA barrier until the end of a piece. Scores are computed transposed, S^T (16 tokens x 8 query heads)
// = K Q^T with m16n8k16, so the 8 heads of a group fill the N side and nothing is padded; P^T returns to
// the B operand of O^T = V^T P^T by a register transpose (movmatrix). P is rounded to 16 bits in two parts,
// hi + lo, each with its own MMA: the weights keep 16 or more bits and the kernel, bound by loads, does
// not notice the extra MMAs. In f16 they are scaled by 2^14 first, so that a weight's parts stay above the type's
// smallest value down to 2^-39 of the largest weight; sums are scaled alike and the quotient is the same.
//
// "Each byte once" holds for groups of up to 16 query heads; a larger group's heads are taken 16 at a time, and each 16 read the
// cache again (through L2 where it still holds it).
//
// Measured on a B200, whole calls, bf16, 32 + 4 heads of 128: 128 sequences of 1 to 8191 tokens 176 us (6.1 TB/s, 95% of a
// measured copy), one of 131071 53 us (5.1 TB/s), 32 of 128 to 2304 23 us, one of 129 8 us (5.4 on the device).
// Four warps and two CTAs per SM against eight and one: 170 against 183 us for the batch (one CTA's joins leave its SM idle).
#include <algorithm>

#include "attention_internal.cuh"

namespace moe {
namespace attn {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int BLK = 16;      // tokens of a block
constexpr int CTAS_PER_SM = 2;
constexpr int MIN_SLICE = 2 * WARPS;  // blocks
constexpr int JOIN = 8;               // parts joined at once
constexpr int ONE_JOIN = 2 * JOIN;    // more parts than these are joined in two steps, in groups of JOIN
constexpr int SHORT = 4 * WARPS;      // blocks up to which a (sequence, head) is never split

int decode_max_ctas(int sms) { return sms * CTAS_PER_SM; }

template <int D>
struct Shape {
  static constexpr int ROW_BYTES = D * 2;
  static constexpr int HALF = BLK * ROW_BYTES;     // the K (or V) bytes of a block
  static constexpr int STAGES = 24576 / (2 * HALF);  // 24 KB in flight per warp
  static constexpr int CHUNKS = D / 8;             // 16-byte chunks of a row
};

template <int D>
constexpr int decode_smem() {
  // rings, the warps' results for 8 heads (padded against bank conflicts), their {m, l}
  return WARPS * Shape<D>::STAGES * 2 * Shape<D>::HALF + WARPS * 8 * (D + 4) * 4 + WARPS * 8 * 8;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: the 16 bytes are zero-filled and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The blocks of sequence b: first block, one past its last token, block count (0: nothing to attend to).
struct Seq {
  int len, lo, first, nb;
};

// pad > 0: every sequence with a token counts that many blocks (the ones past its last token are empty).
__device__ __forceinline__ Seq seq_of(const DecodeParams& p, int b, int pad) {
  Seq s;
  const int cap = p.max_pages << p.pools.page_shift;
  s.len = max(0, min(p.seq_lens[b], cap));
  s.lo = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.first = s.lo / BLK;
  s.nb = (s.len + BLK - 1) / BLK - s.first;
  if (pad > 0 && s.nb > 0) s.nb = pad;
  return s;
}

// A place on the line of blocks: sequence, virtual head (key/value head x row block) and block.
struct Cursor {
  int b, h, j;
  Seq s;
};

__device__ __forceinline__ void advance(const DecodeParams& p, Cursor& c, int n, int vheads, int pad) {
  c.j += n;
  while (c.j >= c.s.nb && c.b < p.B) {
    c.j -= c.s.nb;
    if (++c.h == vheads) {
      c.h = 0;
      do {
        ++c.b;
        if (c.b >= p.B) return;
        c.s = seq_of(p, c.b, pad);
      } while (c.s.nb == 0);
    }
  }
}

// log2 of what the weights of a type are scaled by.
template <class T>
constexpr float DECODE_SCALE = Elem<T>::kWeightBits ? Elem<T>::kWeightBits - 1.0f : 0.0f;

// Four values of an output row from the joined sums (maximum M in units of log2, sum of scaled weights L), and its lse.
template <class T, int D>
__device__ __forceinline__ void store_row(const DecodeParams& p, int64_t row, int d, const float4& o, float M, float L) {
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.y) + row * D + d) =
      make_uint2(Elem<T>::pack(o.x * inv, o.y * inv), Elem<T>::pack(o.z * inv, o.w * inv));
  if (p.lse && d == 0) p.lse[row] = L == 0.0f ? -INFINITY : (M - DECODE_SCALE<T>) * LN2 + logf(L);
}

// Workspace slot of part k of a (sequence, head) whose first CTA is c0: a CTA's part that began in an earlier
// CTA's slice goes to its slot 0, one that begins in its own slice to slot 1.
__device__ __forceinline__ int part_slot(int c0, int k) { return (c0 + k) * 2 + (k == 0 ? 1 : 0); }

// A (sequence, head) that several CTAs share: their number, the first one, its counter, its first output row.
struct Split {
  int parts, c0, unit;
  int64_t out_row;
  int rows;
};

// Counts an arrival of the whole CTA (after a barrier); true for the last of `need`, which leaves the counter at zero for
// the next call. Release and acquire: what the CTA wrote before the barrier is visible to the last one's threads behind
// their next barrier.
__device__ __forceinline__ bool arrive(int32_t* counter, int need) {
  int before;
  __threadfence();
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  const bool last = before == need - 1;
  if (last) *counter = 0;
  return last;
}

__device__ __forceinline__ bool arrive_first(const DecodeParams& p, const Split& sp, int k) {
  if (sp.parts <= ONE_JOIN) return arrive(p.counters + sp.unit, sp.parts);
  const int g0 = k / JOIN * JOIN;
  return arrive(p.group_counters + part_slot(sp.c0, g0), min(JOIN, sp.parts - g0));
}

// Joins parts k0, k0 + step, .. (n of them, in this order; ml: their maxima and sums) into the output, or, with to_ml,
// into part k0's slot of the workspace. A join is one CTA's work behind everything else, so its time is the number of
// dependent trips to L2: all of a thread's loads of JOIN parts are in flight together.
template <class T, int D, int ROWS>
__device__ __forceinline__ void join(const DecodeParams& p, const Split& sp, int k0, int step, int n, const float2* ml,
                                     float2* to_ml) {
  constexpr int EACH = 8 * (D / 4) / THREADS;  // values (of 4) of 8 rows per thread
  static_assert(EACH >= 1 && 8 * (D / 4) % THREADS == 0, "whole passes");
#pragma unroll 1
  for (int r0 = 0; r0 < sp.rows; r0 += 8) {
    float M[EACH], L[EACH];
    float4 o[EACH];
#pragma unroll
    for (int c = 0; c < EACH; ++c) M[c] = -INFINITY, L[c] = 0.0f, o[c] = make_float4(0, 0, 0, 0);
#pragma unroll 1
    for (int k = 0; k < n; k += JOIN) {
      float2 s[EACH][JOIN];
      float4 v[EACH][JOIN];
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        const int e = threadIdx.x + c * THREADS, row = r0 + e / (D / 4), d = (e % (D / 4)) * 4;
#pragma unroll
        for (int i = 0; i < JOIN; ++i) {
          s[c][i] = make_float2(-INFINITY, 0.0f);
          v[c][i] = make_float4(0, 0, 0, 0);
          if (k + i < n && row < sp.rows) {
            const int64_t at = (int64_t)part_slot(sp.c0, k0 + (k + i) * step) * ROWS + row;
            s[c][i] = ld_l2(ml + at);
            v[c][i] = ld_l2(reinterpret_cast<const float4*>(p.partial + at * D + d));
          }
        }
      }
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        float mx = M[c];
#pragma unroll
        for (int i = 0; i < JOIN; ++i) mx = fmaxf(mx, s[c][i].x);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float f = ex2(M[c] - ref);
        M[c] = mx;
        L[c] *= f;
        o[c].x *= f, o[c].y *= f, o[c].z *= f, o[c].w *= f;
#pragma unroll
        for (int i = 0; i < JOIN; ++i) {
          const float w = ex2(s[c][i].x - ref);
          L[c] = fmaf(s[c][i].y, w, L[c]);
          o[c].x = fmaf(v[c][i].x, w, o[c].x), o[c].y = fmaf(v[c][i].y, w, o[c].y);
          o[c].z = fmaf(v[c][i].z, w, o[c].z), o[c].w = fmaf(v[c][i].w, w, o[c].w);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < EACH; ++c) {
      const int e = threadIdx.x + c * THREADS, row = r0 + e / (D / 4), d = (e % (D / 4)) * 4;
      if (row >= sp.rows) continue;
      if (!to_ml) {
        store_row<T, D>(p, sp.out_row + row, d, o[c], M[c], L[c]);
      } else {  // the slot's own values are read by this thread alone, its ml by others: that goes elsewhere
        const int64_t at = (int64_t)part_slot(sp.c0, k0) * ROWS + row;
        __stcg(reinterpret_cast<float4*>(p.partial + at * D + d), o[c]);
        if (d == 0) __stcg(to_ml + at, make_float2(M[c], L[c]));
      }
    }
  }
}

template <class T, int D, int NT>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) decode_kernel(DecodeParams p) {
  using S = Shape<D>;
  constexpr int ROWS = 8 * NT;
  constexpr int RED = D + 4;  // row pitch of the warps' results
  extern __shared__ __align__(128) unsigned char smem[];
  float* red = reinterpret_cast<float*>(smem + WARPS * S::STAGES * 2 * S::HALF);
  float2* red_ml = reinterpret_cast<float2*>(red + WARPS * 8 * RED);
  __shared__ int s_last[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vheads = p.kv_heads * p.row_blocks;
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's slice [start, end) of the line, and the sequence it starts in ----
  // (every warp finds it for itself, its lanes sharing the sequences: no barrier)
  const int per = (p.B + 31) / 32;
  const int b0 = min(p.B, lane * per), b1 = min(p.B, b0 + per);
  int mine = 0;  // blocks of this lane's sequences; their number and the longest one ride along
  int most = 0, some = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const int nb = seq_of(p, b, 0).nb;
    mine += nb;
    most = max(most, nb);
    some += nb > 0;
    if (blockIdx.x == 0 && p.seq_lens[b] > (p.max_pages << p.pools.page_shift)) latch(p.err, MOE_ERR_BAD_IDS);
  }
  most = __reduce_max_sync(FULL, most);
  // Short sequences are not split: each counts as many blocks as the longest, and slices hold whole (sequence, head)s.
  // The join of a split costs about as much as the blocks it would spread out.
  const int pad = most <= SHORT ? most : 0;
  if (pad) mine = some * pad;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, incl, o);
    if (lane >= o) incl += v;
  }
  const int total = __shfl_sync(FULL, incl, 31) * vheads, before = (incl - mine) * vheads;
  mine *= vheads;
  int slice = max(total / (int)gridDim.x + (total % (int)gridDim.x ? 1 : 0), MIN_SLICE);
  if (pad) slice = (slice + pad - 1) / pad * pad;
  const bool slice_past = (int64_t)slice * blockIdx.x >= total;
  const int start = slice_past ? total : slice * blockIdx.x, end = slice_past ? total : total - start > slice ? start + slice : total;

  // sequences without a token: zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (seq_of(p, b, 0).nb > 0) continue;
    for (int i = tid; i < p.heads * (D / 8); i += THREADS)
      reinterpret_cast<uint4*>(static_cast<T*>(p.y) + (int64_t)b * p.heads * D)[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int i = tid; i < p.heads; i += THREADS) p.lse[(int64_t)b * p.heads + i] = -INFINITY;
  }
  if (start >= total) return;  // uniform over the CTA
  const bool here = start >= before && start - before < mine;
  int first_b = b0, first_base = before;
  if (here) {
    for (;; ++first_b) {
      const int n = seq_of(p, first_b, pad).nb * vheads;
      if (start - first_base < n) break;
      first_base += n;
    }
  }
  const int src = __ffs(__ballot_sync(FULL, here)) - 1;
  first_b = __shfl_sync(FULL, first_b, src);
  first_base = __shfl_sync(FULL, first_base, src);

  Cursor pre;  // the next block this warp looks up
  pre.b = first_b;
  pre.s = seq_of(p, pre.b, pad);
  pre.h = (start - first_base) / pre.s.nb;
  pre.j = (start - first_base) % pre.s.nb;
  Cursor cur = pre;  // the piece being computed (j: its first block in this slice)
  int pre_idx = start + warp;
  advance(p, pre, warp, vheads, pad);

  unsigned char* ring = smem + warp * S::STAGES * 2 * S::HALF;
  const uint32_t ring_a = smem_u32(ring);
  int fill = 0, batch = 32;
  int issued = start + warp;  // the block that the next load fetches
  int64_t my_at = 0;  // lane i: where the warp's i-th block of the batch lies in the pools, and its rows [lo, hi)
  int my_rows = 0;
  // Loads the warp's next block into ring stage `fill` (one cp.async group, empty past the slice's end). The places of
  // 32 blocks are looked up at once, one per lane, so that the page table's latency is paid once for them.
  auto load_next = [&]() {
    if (batch == 32) {
      batch = 0;
      my_rows = 0;
      const int idx = pre_idx + lane * WARPS;
      if (idx < end) {
        Cursor c = pre;
        advance(p, c, lane * WARPS, vheads, pad);
        const int tok = (c.s.first + c.j) * BLK;
        if (tok < c.s.len) {  // not a padding block
          const int page = p.page_table[(int64_t)c.b * p.max_pages + (tok >> p.pools.page_shift)];
          if ((unsigned)page < (unsigned)p.pools.num_pages) {
            my_rows = max(0, c.s.lo - tok) | min(BLK, c.s.len - tok) << 16;
            my_at = (int64_t)page * p.pools.page_stride +
                    ((((int64_t)(c.h / p.row_blocks)) << p.pools.page_shift) + (tok & ((1 << p.pools.page_shift) - 1))) * D;
          } else {
            latch(p.err, MOE_ERR_BAD_IDS);  // its tokens read as zeros
          }
        }
      }
      __syncwarp();
      pre_idx += 32 * WARPS;
      if (pre_idx < end) advance(p, pre, 32 * WARPS, vheads, pad);
    }
    const int64_t at = __shfl_sync(FULL, my_at, batch);
    const int rows = __shfl_sync(FULL, my_rows, batch);
    ++batch;
    if (issued < end) {
      const int lo = rows & 0xffff, hi = rows >> 16;
      const T* ks = static_cast<const T*>(p.pools.k) + at;
      const T* vs = static_cast<const T*>(p.pools.v) + at;
      const uint32_t dst = ring_a + fill * 2 * S::HALF;
#pragma unroll
      for (int i = 0; i < BLK * S::CHUNKS / 32; ++i) {
        const int r = (i * 32 + lane) / S::CHUNKS, c = lane % S::CHUNKS;
        const bool in = r >= lo && r < hi;
        const uint32_t to = dst + r * S::ROW_BYTES + ((c ^ (r & 7)) << 4);
        cp_async16(to, ks + r * D + c * 8, in);
        cp_async16(to + S::HALF, vs + r * D + c * 8, in);
      }
    }
    issued += WARPS;
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  };
#pragma unroll 1
  for (int i = 0; i < S::STAGES - 1; ++i) load_next();

  const float c_log2 = p.scale * LOG2E;
  const bool capped = p.softcap > 0.0f;
  const Cap cap = make_cap(p.scale, capped ? p.softcap : 1.0f);
  const int g8 = lane >> 2, t4 = lane & 3;
  int use = 0;
  int idx = start;  // first block of the piece
  Split ahead{}, behind{};  // the pieces shared with the CTAs before and behind this one
  while (idx < end) {
    const int piece_end = end - idx > cur.s.nb - cur.j ? idx + (cur.s.nb - cur.j) : end;
    const int kvh = cur.h / p.row_blocks, row0 = (cur.h % p.row_blocks) * ROWS;
    const int live_rows = min(ROWS, p.group - row0);
    // q as the B operand: head n = g8, values 2 t4, +1 and + 8
    uint32_t qf[D / 16][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + g8;
      const T* src = static_cast<const T*>(p.q) + cur.b * p.q_token_stride +
                     (int64_t)(kvh * p.group + row0 + (n < live_rows ? n : 0)) * p.q_head_stride + 2 * t4;
#pragma unroll
      for (int kt = 0; kt < D / 16; ++kt) {
        qf[kt][nt][0] = n < live_rows ? *reinterpret_cast<const uint32_t*>(src + kt * 16) : 0u;
        qf[kt][nt][1] = n < live_rows ? *reinterpret_cast<const uint32_t*>(src + kt * 16 + 8) : 0u;
      }
    }
    float acc[D / 16][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[dt][nt][i] = 0.0f;
    }
    // first block of this warp at or after idx
    int w_idx = idx + ((warp - (idx - start) % WARPS + WARPS) % WARPS);
    for (; w_idx < piece_end; w_idx += WARPS) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
      __syncwarp();
      load_next();  // refills the stage that the previous block left
      const uint32_t kb = ring_a + use * 2 * S::HALF, vb = kb + S::HALF;
      use = use + 1 == S::STAGES ? 0 : use + 1;
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.0f;
      {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int kt = 0; kt < D / 16; ++kt) {
          uint32_t a[4];
          ldsm4(a, kb + r * S::ROW_BYTES + (((2 * kt + (lane >> 4)) ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Elem<T>::mma(kt & 1 ? s2[nt] : s[nt], a, qf[kt][nt][0], qf[kt][nt][1]);
        }
      }
      // this lane: tokens g8 and g8 + 8 of the block, heads 8 nt + 2 t4 and + 1
      const int tok = (cur.s.first + cur.j + (int)(w_idx - idx)) * BLK;
      const bool in0 = tok + g8 >= cur.s.lo && tok + g8 < cur.s.len;
      const bool in1 = tok + g8 + 8 >= cur.s.lo && tok + g8 + 8 < cur.s.len;
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[nt][i] + s2[nt][i];
          v = !capped ? v * c_log2 : cap.wide ? wide_capped_score(cap, v) : capped_score(cap, v);
          s[nt][i] = (i < 2 ? in0 : in1) ? v : -INFINITY;  // in units of log2
        }
        float corr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(s[nt][i], s[nt][i + 2]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
          const float mn = fmaxf(m[nt][i], mx);
          const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: exp2(-inf - 0) = 0, no NaN
          corr[i] = ex2(m[nt][i] - ref);
          m[nt][i] = mn;
          s[nt][i] = ex2(s[nt][i] - (ref - DECODE_SCALE<T>));
          s[nt][i + 2] = ex2(s[nt][i + 2] - (ref - DECODE_SCALE<T>));
          l[nt][i] = l[nt][i] * corr[i] + (s[nt][i] + s[nt][i + 2]);
        }
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          acc[dt][nt][0] *= corr[0];
          acc[dt][nt][1] *= corr[1];
          acc[dt][nt][2] *= corr[0];
          acc[dt][nt][3] *= corr[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // Both parts above zero, so that an infinite value stays one (0 * inf and inf - inf are NaN): hi is rounded down, and
          // each part is at least the type's smallest value, 2^-38 of the largest weight in f16. Values of tokens that are
          // not seen are zeros in shared memory.
          constexpr float LEAST = Elem<T>::kLeast;
          const float a = fmaxf(s[nt][2 * i], LEAST), b = fmaxf(s[nt][2 * i + 1], LEAST);
          const uint32_t hi = Elem<T>::pack_down(a, b);
          const float2 back = Elem<T>::unpack(hi);
          ph[nt][i] = movmatrix_t(hi);
          pl[nt][i] = movmatrix_t(Elem<T>::pack(fmaxf(a - back.x, LEAST), fmaxf(b - back.y, LEAST)));
        }
      }
      {
        const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          uint32_t a[4];
          ldsm4t(a, vb + r * S::ROW_BYTES + (((2 * dt + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Elem<T>::mma(acc[dt][nt], a, ph[nt][0], ph[nt][1]);
            Elem<T>::mma(acc[dt][nt], a, pl[nt][0], pl[nt][1]);
          }
        }
      }
    }

    // ---- end of the piece: join the warps, 8 heads at a time ----
    const int u0 = idx - cur.j;  // the whole (sequence, head) starts here on the line
    const int c0 = u0 / slice, n_parts = (u0 + (cur.s.nb - 1)) / slice - c0 + 1;
    const int my_slot = part_slot(c0, blockIdx.x - c0);
    const int64_t out_row = (int64_t)cur.b * p.heads + kvh * p.group + row0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][i] += __shfl_xor_sync(FULL, l[nt][i], o);
        const int n = 2 * t4 + i;
        if (g8 == 0) red_ml[warp * 8 + n] = make_float2(m[nt][i], l[nt][i]);
        float* dst = red + (warp * 8 + n) * RED + g8;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          dst[dt * 16] = acc[dt][nt][i];
          dst[dt * 16 + 8] = acc[dt][nt][i + 2];
        }
      }
      __syncthreads();
      for (int e = tid; e < min(8, live_rows - nt * 8) * (D / 4); e += THREADS) {
        const int n = e / (D / 4), d = (e % (D / 4)) * 4, row = nt * 8 + n;
        float2 ml[WARPS];
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          ml[w] = red_ml[w * 8 + n];
          M = fmaxf(M, ml[w].x);
        }
        const float ref = M == -INFINITY ? 0.0f : M;
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float f = ex2(ml[w].x - ref);
          const float4 v = *reinterpret_cast<const float4*>(red + (w * 8 + n) * RED + d);
          L += ml[w].y * f;
          o.x += v.x * f, o.y += v.y * f, o.z += v.z * f, o.w += v.w * f;
        }
        if (n_parts == 1) {
          store_row<T, D>(p, out_row + row, d, o, M, L);
        } else {
          __stcg(reinterpret_cast<float4*>(p.partial + ((int64_t)my_slot * ROWS + row) * D + d), o);
          if (d == 0) __stcg(p.partial_ml + (int64_t)my_slot * ROWS + row, make_float2(M, L));
        }
      }
      __syncthreads();  // red is free again
    }
    if (n_parts > 1) {  // at most two pieces of a slice: the one it begins in and the one it ends in
      const Split sp = {n_parts, c0, cur.b * vheads + cur.h, out_row, live_rows};
      if (blockIdx.x == c0) behind = sp;
      else ahead = sp;
    }
    const int step = piece_end - idx;
    idx = piece_end;
    if (idx < end) advance(p, cur, step, vheads, pad);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- arrivals: the last CTA of a (sequence, head) joins its parts, or of a group of parts when there are many ----
  if (ahead.parts == 0 && behind.parts == 0) return;
  __syncthreads();
  if (lane == 0 && warp < 2) {
    const Split& sp = warp ? behind : ahead;
    s_last[warp] = sp.parts > 0 && arrive_first(p, sp, blockIdx.x - sp.c0);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (!s_last[i]) continue;  // uniform over the CTA
    const Split sp = i ? behind : ahead;
    if (sp.parts <= ONE_JOIN) {
      join<T, D, ROWS>(p, sp, 0, 1, sp.parts, p.partial_ml, nullptr);
      continue;
    }
    const int g0 = (blockIdx.x - sp.c0) / JOIN * JOIN;
    join<T, D, ROWS>(p, sp, g0, 1, min(JOIN, sp.parts - g0), p.partial_ml, p.group_ml);
    __syncthreads();
    if (tid == 0) s_last[i] = arrive(p.counters + sp.unit, (sp.parts + JOIN - 1) / JOIN);
    __syncthreads();
    if (s_last[i]) {
      join<T, D, ROWS>(p, sp, 0, JOIN, (sp.parts + JOIN - 1) / JOIN, p.group_ml, nullptr);
    }
  }
}

// f(kernel, dynamic shared memory) for the handle's types and sizes.
template <class F>
static moe_status with_kernel(const moe_attn& a, F&& f) {
  const bool wide = decode_rows(a.group) == 16;
  static_assert(decode_smem<128>() <= 233472 / CTAS_PER_SM - 1024 - 256 && decode_smem<64>() <= decode_smem<128>(),
                "shared memory of an SM");
  auto by_type = [&](auto zero) -> moe_status {
    using T = decltype(zero);
    if (a.d.head_dim == 64)
      return wide ? f(decode_kernel<T, 64, 2>, decode_smem<64>()) : f(decode_kernel<T, 64, 1>, decode_smem<64>());
    return wide ? f(decode_kernel<T, 128, 2>, decode_smem<128>()) : f(decode_kernel<T, 128, 1>, decode_smem<128>());
  };
  return a.d.dtype == MOE_ATTN_BF16 ? by_type(__nv_bfloat16()) : by_type(__half());
}

moe_status prepare_decode(const moe_attn& a) {
  return with_kernel(a, [](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return MOE_OK;
  });
}

moe_status launch_decode(const moe_attn& a, const DecodeParams& p, cudaStream_t st) {
  // no more CTAs than the widest table's blocks give work to
  const int64_t widest = ((int64_t)p.max_pages << p.pools.page_shift) / BLK;
  const int64_t bound = (widest * p.B * p.kv_heads * p.row_blocks + MIN_SLICE - 1) / MIN_SLICE;
  if (widest * p.B * p.kv_heads * p.row_blocks > 0x3fffffffll)
    return fail(MOE_ERR_INVALID, "moe_attn_decode: B * num_kv_heads * max_pages * page_size / 16 must be below 2^30");
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(decode_max_ctas(a.sms), bound));
  return with_kernel(a, [&](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(THREADS), smem, st, p));
    return MOE_OK;
  });
}

}  // namespace attn
}  // namespace moe
