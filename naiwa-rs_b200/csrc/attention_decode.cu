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
// not notice the extra MMAs.
#include <algorithm>

#include "attention_internal.cuh"

namespace moe {
namespace attn {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int BLK = 16;      // tokens of a block
constexpr int CTAS_PER_SM = 2;
constexpr int MIN_SLICE = 2 * WARPS;  // blocks

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

__device__ __forceinline__ Seq seq_of(const DecodeParams& p, int b) {
  Seq s;
  const int cap = p.max_pages << p.pools.page_shift;
  s.len = max(0, min(__ldg(p.seq_lens + b), cap));
  s.lo = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.first = s.lo / BLK;
  s.nb = (s.len + BLK - 1) / BLK - s.first;
  return s;
}

// A place on the line of blocks: sequence, virtual head (key/value head x row block) and block.
struct Cursor {
  int b, h, j;
  Seq s;
};

__device__ __forceinline__ void advance(const DecodeParams& p, Cursor& c, int n, int vheads) {
  c.j += n;
  while (c.j >= c.s.nb && c.b < p.B) {
    c.j -= c.s.nb;
    if (++c.h == vheads) {
      c.h = 0;
      do {
        ++c.b;
        if (c.b >= p.B) return;
        c.s = seq_of(p, c.b);
      } while (c.s.nb == 0);
    }
  }
}

// The page of cursor c's block (one out of range is latched, and its tokens read as zeros).
__device__ __forceinline__ int page_of(const DecodeParams& p, const Cursor& c) {
  const int tok = (c.s.first + c.j) * BLK;
  return __ldg(p.page_table + (int64_t)c.b * p.max_pages + (tok >> p.pools.page_shift));
}

// Four values of an output row from the joined sums (maximum M in units of log2, sum of weights L), and its lse.
template <class T, int D>
__device__ __forceinline__ void store_row(const DecodeParams& p, int64_t row, int d, const float4& o, float M, float L) {
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.y) + row * D + d) =
      make_uint2(Elem<T>::pack(o.x * inv, o.y * inv), Elem<T>::pack(o.z * inv, o.w * inv));
  if (p.lse && d == 0) p.lse[row] = L == 0.0f ? -INFINITY : M * LN2 + logf(L);
}

template <class T, int D, int NT>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) decode_kernel(DecodeParams p) {
  using S = Shape<D>;
  constexpr int ROWS = 8 * NT;
  constexpr int RED = D + 4;  // row pitch of the warps' results
  extern __shared__ __align__(128) unsigned char smem[];
  float* red = reinterpret_cast<float*>(smem + WARPS * S::STAGES * 2 * S::HALF);
  float2* red_ml = reinterpret_cast<float2*>(red + WARPS * 8 * RED);
  __shared__ long long s_scan[WARPS];
  __shared__ int s_b;
  __shared__ long long s_base;
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vheads = p.kv_heads * p.row_blocks;
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's slice [start, end) of the line, and the sequence it starts in ----
  const int per = (p.B + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
    const Seq s = seq_of(p, b);
    mine += s.nb;
    if (blockIdx.x == 0 && __ldg(p.seq_lens + b) > (p.max_pages << p.pools.page_shift)) latch(p.err, MOE_ERR_BAD_IDS);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(FULL, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  long long total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  total *= vheads;
  before *= vheads;
  mine *= vheads;
  const long long slice = max((total + gridDim.x - 1) / gridDim.x, (long long)MIN_SLICE);
  const long long start = slice * blockIdx.x, end = min(total, start + slice);

  // sequences without a token: zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (seq_of(p, b).nb > 0) continue;
    for (int i = tid; i < p.heads * (D / 8); i += THREADS)
      reinterpret_cast<uint4*>(static_cast<T*>(p.y) + (int64_t)b * p.heads * D)[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int i = tid; i < p.heads; i += THREADS) p.lse[(int64_t)b * p.heads + i] = -INFINITY;
  }
  if (start >= total) return;  // uniform over the CTA
  if (start >= before && start < before + mine) {
    int b = tid * per;
    long long base = before;
    for (;; ++b) {
      const long long n = (long long)seq_of(p, b).nb * vheads;
      if (start < base + n) break;
      base += n;
    }
    s_b = b;
    s_base = base;
  }
  __syncthreads();

  Cursor pre;  // the next block this warp loads
  pre.b = s_b;
  pre.s = seq_of(p, pre.b);
  const long long rem = start - s_base;
  pre.h = (int)(rem / pre.s.nb);
  pre.j = (int)(rem % pre.s.nb);
  Cursor cur = pre;  // the piece being computed (j: its first block in this slice)
  long long pre_idx = start + warp;
  advance(p, pre, warp, vheads);
  int next_page = pre_idx < end ? page_of(p, pre) : 0;

  unsigned char* ring = smem + warp * S::STAGES * 2 * S::HALF;
  const uint32_t ring_a = smem_u32(ring);
  int fill = 0;
  // Loads the block at `pre` into ring stage `fill` (one cp.async group, empty past the slice's end) and moves
  // `pre` on; the page of the block after it is fetched now, so its latency passes behind the loads.
  auto load_next = [&]() {
    if (pre_idx < end) {
      const int page = next_page;
      const bool page_ok = (unsigned)page < (unsigned)p.pools.num_pages;
      if (!page_ok && lane == 0) latch(p.err, MOE_ERR_BAD_IDS);
      const int tok = (pre.s.first + pre.j) * BLK;
      const int lo = pre.s.lo - tok, hi = page_ok ? pre.s.len - tok : 0;  // rows lo <= r < hi are loaded
      const int off = tok & ((1 << p.pools.page_shift) - 1);
      const int64_t at = (int64_t)(page_ok ? page : 0) * p.pools.page_stride +
                         ((((int64_t)(pre.h / p.row_blocks)) << p.pools.page_shift) + off) * D;
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
      pre_idx += WARPS;
      advance(p, pre, WARPS, vheads);
      if (pre_idx < end) next_page = page_of(p, pre);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  };
#pragma unroll 1
  for (int i = 0; i < S::STAGES - 1; ++i) load_next();

  const float c_log2 = p.scale * LOG2E;
  const int g8 = lane >> 2, t4 = lane & 3;
  int use = 0;
  long long idx = start;  // first block of the piece
  while (idx < end) {
    const long long piece_end = min(end, idx + (cur.s.nb - cur.j));
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
        qf[kt][nt][0] = n < live_rows ? __ldg(reinterpret_cast<const uint32_t*>(src + kt * 16)) : 0u;
        qf[kt][nt][1] = n < live_rows ? __ldg(reinterpret_cast<const uint32_t*>(src + kt * 16 + 8)) : 0u;
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
    long long w_idx = idx + ((warp - (int)((idx - start) % WARPS) + WARPS) % WARPS);
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
          v = p.softcap > 0.0f ? p.softcap * LOG2E * tanhf(v * p.scale / p.softcap) : v * c_log2;
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
          s[nt][i] = ex2(s[nt][i] - ref);
          s[nt][i + 2] = ex2(s[nt][i + 2] - ref);
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
          const uint32_t hi = Elem<T>::pack(s[nt][2 * i], s[nt][2 * i + 1]);
          const float2 back = Elem<T>::unpack(hi);
          ph[nt][i] = movmatrix_t(hi);
          pl[nt][i] = movmatrix_t(Elem<T>::pack(s[nt][2 * i] - back.x, s[nt][2 * i + 1] - back.y));
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
    const long long u0 = idx - cur.j, u1 = u0 + cur.s.nb;  // the whole (sequence, head) on the line
    const int c0 = (int)(u0 / slice), n_parts = (int)((u1 - 1) / slice) - c0 + 1;
    const int my_slot = blockIdx.x * 2 + (blockIdx.x == c0 ? 1 : 0);
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
    if (n_parts > 1) {
      // the last of the piece's CTAs to arrive joins them
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int32_t* cnt = p.counters + (int64_t)cur.b * vheads + cur.h;
        s_last = atomicAdd(cnt, 1) == n_parts - 1;
        if (s_last) *cnt = 0;  // ready for the next call
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int e = tid; e < live_rows * (D / 4); e += THREADS) {
          const int n = e / (D / 4), d = (e % (D / 4)) * 4;
          float M = -INFINITY, L = 0.0f;
          float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
          for (int k = 0; k < n_parts; ++k) {
            const int64_t at = (int64_t)((c0 + k) * 2 + (k == 0 ? 1 : 0)) * ROWS + n;
            const float2 ml = __ldcg(p.partial_ml + at);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.partial + at * D + d));
            const float mn = fmaxf(M, ml.x);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float f0 = ex2(M - ref), f1 = ex2(ml.x - ref);
            M = mn;
            L = L * f0 + ml.y * f1;
            o.x = o.x * f0 + v.x * f1, o.y = o.y * f0 + v.y * f1;
            o.z = o.z * f0 + v.z * f1, o.w = o.w * f0 + v.w * f1;
          }
          store_row<T, D>(p, out_row + n, d, o, M, L);
        }
      }
    }
    const int step = (int)(piece_end - idx);
    idx = piece_end;
    if (idx < end) advance(p, cur, step, vheads);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// f(kernel, dynamic shared memory) for the handle's types and sizes.
template <class F>
static moe_status with_kernel(const moe_attn& a, F&& f) {
  const bool wide = decode_rows(a.group) == 16;
  static_assert(decode_smem<128>() <= 233472 / CTAS_PER_SM - 1024 - 128 && decode_smem<64>() <= decode_smem<128>(),
                "two CTAs per SM");
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
  const int grid = (int)std::min<int64_t>(decode_max_ctas(a.sms), bound);
  return with_kernel(a, [&](auto kernel, int smem) -> moe_status {
    MOE_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(THREADS), smem, st, p));
    return MOE_OK;
  });
}

}  // namespace attn
}  // namespace moe
