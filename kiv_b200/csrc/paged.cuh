// What the kernels over a paged cache share: argument checks, the geometry of
// a sequence, and the division of a batch's work among the blocks of a grid.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace kiv {

#ifndef __CUDA_ARCH__
using std::max;
using std::min;
#endif

kiv_status check_paged(const kiv_paged *pc);

__device__ __forceinline__ void paged_error(int64_t *errors, int64_t bit) {
  if (errors) atomicOr(reinterpret_cast<unsigned long long *>(errors), (unsigned long long)bit);
}

// One sequence: its new tokens' first packed row and count, and its length.
// Lengths and row ranges are clamped to what the arrays hold, so nothing a
// device array says can lead out of bounds.
struct PagedSeq {
  int b;
  int64_t q0;
  int n;
  int len;
};

__device__ __forceinline__ PagedSeq paged_seq(const kiv_paged &pc, int b) {
  PagedSeq s;
  s.b = b;
  const int64_t t0 = min((int64_t)max(pc.q_starts[b], 0), pc.num_tokens);
  const int64_t t1 = min((int64_t)max(pc.q_starts[b + 1], 0), pc.num_tokens);
  s.q0 = t0;
  s.n = t1 > t0 ? (int)(t1 - t0) : 0;
  s.len = (int)min((int64_t)max(pc.seq_lens[b], 0), pc.table_width * pc.page_size);
  return s;
}

// The first sequence that ends behind packed row `tok`, found by the whole
// block in one round trip: how many end at or before it.
__device__ __forceinline__ int paged_find_seq(const kiv_paged &pc, int64_t tok) {
  int before = 0;
  for (int b0 = 0; b0 < pc.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    before += __syncthreads_count(b < pc.batch && (int64_t)pc.q_starts[b + 1] <= tok);
  }
  return before;
}

// ---------------------------------------------------------------------------
// Division of the work.
//
// An item is one row tile of one sequence and one key head: `tpt` new tokens
// with all the query heads of the key head (cut into `hs` parts where there
// are more of them than a tile has rows).  Its work is the tiles of `kt` keys
// that some row of it sees.  The items of the batch, in the order (sequence,
// head part, row tile), make one line of tiles, and block c of G takes the
// tiles [c N / G, (c + 1) N / G) of it (G at most N: the other blocks leave):
// every block streams the same number of key tiles (within one), whatever the
// lengths.  An item inside one block
// is finished there; one that blocks share leaves its parts (running maximum,
// sum, unscaled output) in the workspace, at most two per block -- slot 2c for
// an item that began in an earlier block, slot 2c + 1 for one that began in
// this block and goes on -- and the combine kernel joins them in block order,
// so the result does not depend on timing.
//
// N, and where a block begins, follow from the lengths alone; each block works
// them out for itself at its start (one read of the lengths, one block scan).
// ---------------------------------------------------------------------------
struct PagedPlan {
  kiv_paged pc;
  kiv_paged_query q;
  int grp;       // query heads per head part
  int hs;        // head parts per key head
  int tpt;       // tokens per row tile
  int kt;        // keys per key tile
  int rows;      // rows per part in the workspace: tpt * grp <= rows
  float *part;   // [2 * G][rows][D + 2 (rounded to 4)]
  struct PagedCut *cut;     // [G]
};

// What block c says about the item it began and did not finish (b = -1: none)
struct PagedCut {
  int32_t b, hp, rt, pad;
  int64_t end, total;       // the place past the item's last tile; N
  int64_t blocks;           // blocks that took part
};

// sum over i < n of floor((a i + b) / m), a and b not negative: lattice points
// under a line, counted by exchanging the axes (Euclid's steps).  a n + b stays
// below 2^32 here (places of tokens), so the divisions have 32 bits.
__host__ __device__ inline int64_t floor_sum(int64_t count, uint32_t m, uint32_t a, int64_t b64) {
  int64_t ans = 0;
  if (count <= 0) return 0;
  uint32_t n = (uint32_t)count, b = (uint32_t)b64;
  for (;;) {
    const uint32_t qa = a / m, qb = b / m;
    ans += (int64_t)((uint64_t)n * (n - 1) / 2) * qa + (int64_t)n * qb;
    a -= qa * m;
    b -= qb * m;
    const uint32_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y - n * m;
    const uint32_t x = a;
    a = m;
    m = x;
  }
  return ans;
}

kiv_status launch_paged_combine(const PagedPlan &p, int blocks, cudaStream_t s);
// few rows per key head, 16-bit rows (paged_mma.cu); plan rows 16, 32 or 64, kt 64
bool paged_mma_head(int dtype, int D);
int paged_mma_blocks(int D, int rows);
kiv_status launch_paged_mma(const PagedPlan &p, int blocks, cudaStream_t s);

// chunks, 16-bit rows, tcgen05 (paged_tc.cu, paged_tc256.cu); plan rows 256 (head_dim 256: 128), kt 128, whole
// tokens per 128 rows
bool paged_tc_eligible(const kiv_paged *pc, const kiv_paged_query *q);
kiv_status launch_paged_tc(const PagedPlan &p, int blocks, cudaStream_t s);

struct PagedItems {      // the items of one sequence
  PagedSeq s;
  int nrt;               // row tiles
  int base;              // place of new token 0 (causal), or the length
};

__device__ __forceinline__ PagedItems paged_items(const PagedPlan &p, int b) {
  PagedItems it;
  it.s = paged_seq(p.pc, b);
  it.nrt = (it.s.n + p.tpt - 1) / p.tpt;
  it.base = p.q.causal ? it.s.len - it.s.n : it.s.len;
  return it;
}

// keys [lo, hi) that some row of row tile rt sees; at least one (masked) key,
// so that every item has a tile and its rows are written
__host__ __device__ inline void paged_range(const PagedPlan &p, const PagedItems &it, int rt, int &lo, int &hi) {
  lo = 0;
  if (p.q.causal) {
    const int64_t h = (int64_t)it.base + (int64_t)(rt + 1) * p.tpt;
    hi = (int)max((int64_t)1, min((int64_t)it.s.len, h));
    if (p.q.window > 0) {
      const int64_t l = (int64_t)it.base + (int64_t)rt * p.tpt - p.q.window + 1;
      lo = (int)min(max(l, (int64_t)0), (int64_t)hi - 1);
    }
  } else {
    hi = max(1, it.s.len);
  }
}

__host__ __device__ inline int paged_tiles(const PagedPlan &p, const PagedItems &it, int rt) {
  int lo, hi;
  paged_range(p, it, rt, lo, hi);
  return (hi + p.kt - 1) / p.kt - lo / p.kt;
}

// tiles of the row tiles [0, x) of one head part
__host__ __device__ inline int64_t paged_prefix(const PagedPlan &p, const PagedItems &it, int x) {
  if (x <= 4) {
    int64_t r = 0;
    for (int i = 0; i < x; ++i) r += paged_tiles(p, it, i);
    return r;
  }
  if (!p.q.causal) return (int64_t)x * paged_tiles(p, it, 0);
  // the last row tile may end at the length, the others end at whole tiles of tokens
  int64_t r = 0;
  if (x == it.nrt) r = paged_tiles(p, it, --x);
  const int64_t base = it.base;
  const uint32_t t = p.tpt, k = p.kt;
  const int64_t k0 = base >= 1 ? 0 : min((int64_t)x, (1 - base) / t);   // row tiles with hi = 1
  r += k0 + floor_sum(x - k0, k, t, base + (k0 + 1) * t + k - 1);
  if (p.q.window > 0) {
    const int64_t need = p.q.window - 1 - base;                           // lo > 0 from there on
    const int64_t i0 = need <= 0 ? 0 : min((int64_t)x, (need + t - 1) / t);
    r -= floor_sum(x - i0, k, t, base + i0 * t - p.q.window + 1);
  }
  return r;
}

struct PagedSpot {       // a place on the line of tiles
  PagedItems it;
  int hp;                // key head * hs + head part
  int rt;
  int64_t off;           // tiles into the item
  int64_t total;         // N
  int64_t blocks;        // G
  int64_t unit;          // the place itself
  int64_t end;           // where the block's stretch ends
};

// The stretch of this block (blockIdx.x), found by the whole block.  `sm`:
// shared, 40 words of 8 bytes.  b = -1 in the result: nothing to do.
template <int NT>
__device__ __forceinline__ PagedSpot paged_locate(const PagedPlan &p, int64_t *sm) {
  const int H = p.pc.num_kv_heads * p.hs;
  const int per = (p.pc.batch + NT - 1) / NT;
  const int b0 = threadIdx.x * per, b1 = min(b0 + per, p.pc.batch);
  int64_t mine = 0;
  PagedItems first;
  for (int b = b0; b < b1; ++b) {
    const PagedItems it = paged_items(p, b);
    if (b == b0) first = it;
    if (it.nrt > 0) mine += H * paged_prefix(p, it, it.nrt);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(KIV_FULL_MASK, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = inc;
  if (threadIdx.x == 0) sm[32] = -1;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += sm[w];
    total += sm[w];
  }
  const int64_t G = min((int64_t)gridDim.x, total), c = blockIdx.x;
  const int64_t unit = c < G ? c * total / G : total;   // below 2^63: N counts tiles, c blocks
  int64_t at = unit - (before + inc - mine);
  if (at >= 0 && at < mine) {
    for (int b = b0; b < b1; ++b) {
      const PagedItems it = b == b0 ? first : paged_items(p, b);
      const int64_t c = it.nrt > 0 ? H * paged_prefix(p, it, it.nrt) : 0;
      if (at < c) {
        sm[32] = b;
        sm[33] = at;
        break;
      }
      at -= c;
    }
  }
  __syncthreads();
  PagedSpot r;
  r.total = total;
  r.blocks = G;
  r.unit = unit;
  r.end = c < G ? (c + 1) * total / G : total;
  r.hp = r.rt = 0;
  r.off = 0;
  const int b = (int)sm[32];
  if (b < 0) {
    r.it.s.b = -1;
    r.it.nrt = 0;
    return r;
  }
  r.it = paged_items(p, b);
  int64_t rem = sm[33];
  const int64_t per_head = paged_prefix(p, r.it, r.it.nrt);
  r.hp = (int)(rem / per_head);
  rem -= (int64_t)r.hp * per_head;
  // largest rt with prefix(rt) <= rem: the lanes try 32 places at a time
  int a = 0, z = r.it.nrt;
  while (z - a > 1) {
    const int stride = (z - a + 31) / 32, x = a + lane * stride;
    const unsigned under = __ballot_sync(KIV_FULL_MASK, x < z && paged_prefix(p, r.it, x) <= rem);
    a += (31 - __clz(under)) * stride;           // lane 0 always holds
    z = min(z, a + stride);
  }
  r.rt = a;
  r.off = rem - paged_prefix(p, r.it, a);
  return r;
}

// The item after this one (b = -1: none)
__device__ __forceinline__ void paged_next(const PagedPlan &p, PagedSpot &s) {
  s.off = 0;
  if (++s.rt < s.it.nrt) return;
  s.rt = 0;
  if (++s.hp < p.pc.num_kv_heads * p.hs) return;
  s.hp = 0;
  for (int b = s.it.s.b + 1; b < p.pc.batch; ++b) {
    s.it = paged_items(p, b);
    if (s.it.nrt > 0) return;
  }
  s.it.s.b = -1;
}

// One segment of a block's stretch [at.unit, at.end): the item's tiles [t0, t1)
struct PagedSegment {
  int t0, t1;
  bool head, tail;       // the item began in an earlier block / goes on in a later one
};

__device__ __forceinline__ PagedSegment paged_segment(const PagedPlan &p, const PagedSpot &at) {
  PagedSegment g;
  const int nt = paged_tiles(p, at.it, at.rt);
  g.t0 = (int)at.off;
  g.t1 = (int)min((int64_t)nt, at.off + (at.end - at.unit));
  g.head = g.t0 > 0;
  g.tail = g.t1 < nt;
  return g;
}

// Block c records the item that its stretch cuts (called by one thread).
__device__ __forceinline__ void paged_record(const PagedPlan &p, int c, const PagedSpot &at, const PagedSegment &g) {
  PagedCut r = {};
  r.b = -1;
  if (g.tail && !g.head) {
    r.b = at.it.s.b;
    r.hp = at.hp;
    r.rt = at.rt;
    r.end = at.unit - at.off + paged_tiles(p, at.it, at.rt);
    r.total = at.total;
    r.blocks = at.blocks;
  }
  p.cut[c] = r;
}

__device__ __forceinline__ void paged_check_lens(const kiv_paged &pc, const PagedSeq &s) {
  const int64_t len = pc.seq_lens[s.b];
  if (len < s.n || len > pc.table_width * pc.page_size) paged_error(pc.errors, KIV_ERRBIT_SEQ_LEN);
}

__device__ __forceinline__ float *paged_part(const PagedPlan &p, int64_t slot, int row) {
  return p.part + (slot * p.rows + row) * partial_stride(p.pc.head_dim);
}

// Row r of an item's tile: token (in the sequence) and query head, or false
__device__ __forceinline__ bool paged_row(const PagedPlan &p, const PagedItems &it, int hp, int rt, int r, int &i, int &head) {
  const int ti = r / p.grp, g = r - ti * p.grp;
  i = rt * p.tpt + ti;
  const int per = p.q.num_query_heads / p.pc.num_kv_heads;
  const int gi = (hp % p.hs) * p.grp + g;
  head = (hp / p.hs) * per + gi;
  return ti < p.tpt && i < it.s.n && gi < per;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Capped scores: s <- cap * tanh(scaling * s / cap), N per lane of a converged
// warp.  tanh(x) = 1 - 2 / (1 + e^2x) costs two special-function operations per
// score, twice what the softmax itself does, so where no score of the warp
// passes 0.7 of the cap an odd polynomial serves: x P(x^2), P the degree-5
// Chebyshev fit of tanh(x) / x on [0, 0.49] (relative error 3e-8 in fp32).
template <int N>
__device__ __forceinline__ void cap_scores(float *s, float cap, float scaling) {
  const float k = scaling / cap;
  float most = 0.f;
#pragma unroll
  for (int x = 0; x < N; ++x) most = fmaxf(most, fabsf(s[x]));
  if (__all_sync(KIV_FULL_MASK, most * fabsf(k) <= 0.7f)) {
    const float2 k2 = make_float2(k, k), c2 = make_float2(scaling, scaling);
#pragma unroll
    for (int x = 0; x < N; x += 2) {
      const float2 v = make_float2(s[x], s[x + 1]);
      const float2 t = __fmul2_rn(v, k2), u = __fmul2_rn(t, t);
      float2 y = make_float2(-0.005094828f, -0.005094828f);
      y = __ffma2_rn(y, u, make_float2(0.020032447f, 0.020032447f));
      y = __ffma2_rn(y, u, make_float2(-0.053529456f, -0.053529456f));
      y = __ffma2_rn(y, u, make_float2(0.133284763f, 0.133284763f));
      y = __ffma2_rn(y, u, make_float2(-0.333331347f, -0.333331347f));
      y = __ffma2_rn(y, u, make_float2(1.f, 1.f));
      y = __fmul2_rn(y, __fmul2_rn(v, c2));
      s[x] = y.x;
      s[x + 1] = y.y;
    }
  } else {
    const float e = 2.f * 1.44269504f * k;
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] = cap * (1.f - __fdividef(2.f, 1.f + ex2(s[x] * e)));
  }
}

// Where a finished row goes
template <typename T>
__device__ __forceinline__ T *paged_out(const PagedPlan &p, const PagedItems &it, int i, int head) {
  return static_cast<T *>(p.q.out) + (it.s.q0 + i) * p.q.out_stride_t + head * p.q.out_stride_h;
}
__device__ __forceinline__ void paged_lse(const PagedPlan &p, const PagedItems &it, int i, int head, float m, float l) {
  if (p.q.lse) p.q.lse[(it.s.q0 + i) * p.q.num_query_heads + head] = l > 0.f ? m + logf(l) : -INFINITY;
}

// Element offsets of key j's rows in k and v, or -1 where it has no page
__device__ __forceinline__ void paged_key(const kiv_paged &pc, int b, int64_t j, int kvh, int64_t &ko, int64_t &vo) {
  const int32_t page = pc.block_table[b * pc.table_stride + j / pc.page_size];
  const int64_t r = j % pc.page_size;
  const bool ok = page >= 0 && page < pc.num_pages;
  ko = ok ? page * pc.k_stride_p + kvh * pc.k_stride_h + r * pc.k_stride_t : -1;
  vo = ok ? page * pc.v_stride_p + kvh * pc.v_stride_h + r * pc.v_stride_t : -1;
}

}  // namespace kiv
