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

// After a wait that ran out, copies may still be on the way to the block's shared
// memory, in phases of their barriers that nobody counted: holds the block for as
// long as the wait itself was given (2^31 cycles).
__device__ __forceinline__ void paged_linger() {
  const long long t0 = clock64();
  while (clock64() - t0 < (1ll << 31)) __nanosleep(1000);
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
// An item is one or two row tiles of one sequence and one key head: `tpt` new
// tokens with all the query heads of the key head (cut into `hs` parts where
// there are more of them than a tile has rows).  Its work is the tiles of `kt`
// keys that some row of it sees, each counted once per row tile: two row tiles
// take about twice as long over a key tile as one.  The items of the batch, in
// the order (sequence, head part, item), make one line of N units, and block c
// of G takes the key tiles that begin in its stretch [c N / G, (c + 1) N / G)
// (G at most N, or N / 2 with two row tiles, so that no stretch inside an item
// is empty: the other blocks leave): every block does the same work (within a
// tile), whatever the lengths.  An item inside one block
// is finished there; one that blocks share leaves its parts (running maximum,
// sum, unscaled output) in the workspace, at most two per block -- slot 2c for
// an item that began in an earlier block, slot 2c + 1 for one that began in
// this block and goes on -- and the combine kernel joins them in block order,
// so the result does not depend on timing.
//
// N, and where a block begins, follow from the lengths alone; each block works
// them out for itself at its start (one read of the lengths, one warp scan).
// ---------------------------------------------------------------------------
struct PagedPlan {
  kiv_paged pc;
  kiv_paged_query q;
  int grp;       // query heads per head part
  int hs;        // head parts per key head
  int tpt;       // tokens per item
  int tps;       // tokens per row tile: an item has one (tps = tpt) or two (tpt = 2 tps)
  int kt;        // keys per key tile: a power of two
  int kt_log2;
  int rows;      // rows per part in the workspace: tpt * grp <= rows
  int slots;     // 2 G
  // [rows / 8][slots][8][D + 2 (rounded to 4)]: the few rows of single tokens
  // share a few memory pages over all slots, whose first touches cost most of a
  // short call's join
  float *part;
  struct PagedCut *cut;     // [G], in front of them
};

// What block c says about the item it began and did not finish (b = -1: none)
struct PagedCut {
  int32_t b, hp, rt, n;     // n: new tokens of the sequence
  int64_t q0;               // packed row of its first
  int32_t last, pad;        // the last block that holds a part
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
// fp32 rows (paged_f32.cu); plan rows 16, 32 or 64, kt 32
bool paged_f32_head(int dtype, int D);
int paged_f32_blocks(int D, int rows);
kiv_status launch_paged_f32(const PagedPlan &p, int blocks, cudaStream_t s);
// 16-bit rows (paged_mma.cu); plan rows 16, 32 or 64, kt 64
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
  it.nrt = (uint32_t)(it.s.n + p.tpt - 1) / (uint32_t)p.tpt;
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
  return ((hi + p.kt - 1) >> p.kt_log2) - (lo >> p.kt_log2);
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

// a / b, b > 0: mostly small numbers, and a 64-bit division takes four times a 32-bit one
__host__ __device__ inline int64_t paged_div(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Row tiles of item rt: 1 or 2; its work
__host__ __device__ inline int paged_weight(const PagedPlan &p, const PagedItems &it, int rt) {
  return p.tps < p.tpt && it.s.n - rt * p.tpt > p.tps ? 2 : 1;
}
__host__ __device__ inline int64_t paged_units(const PagedPlan &p, const PagedItems &it, int rt) {
  return (int64_t)paged_tiles(p, it, rt) * paged_weight(p, it, rt);
}
// work of the items [0, x) of one head part: only the last may have one row tile of two
__host__ __device__ inline int64_t paged_line(const PagedPlan &p, const PagedItems &it, int x) {
  const int64_t r = paged_prefix(p, it, x);
  if (p.tps == p.tpt || x == 0) return r;
  return 2 * r - (x == it.nrt && paged_weight(p, it, x - 1) == 1 ? paged_tiles(p, it, x - 1) : 0);
}

struct PagedSpot {       // a place on the line
  PagedItems it;
  int hp;                // key head * hs + head part
  int rt;
  int64_t off;           // units into the item
  int64_t total;         // N
  int64_t blocks;        // G
  int64_t unit;          // the place itself
  int64_t end;           // where the block's stretch ends
};

// The stretch of this block (blockIdx.x), found by one whole warp.  b = -1 in
// the result: nothing to do.
__device__ __forceinline__ PagedSpot paged_locate(const PagedPlan &p) {
  const int H = p.pc.num_kv_heads * p.hs, lane = threadIdx.x & 31;
  const int per = (p.pc.batch + 31) / 32;
  const int b0 = lane * per, b1 = min(b0 + per, p.pc.batch);
  int64_t mine = 0;
  PagedItems own;                                // with up to 32 sequences, the lane's only one
  own.nrt = 0;
  for (int b = b0; b < b1; ++b) {
    own = paged_items(p, b);
    if (own.nrt > 0) mine += H * paged_line(p, own, own.nrt);
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(KIV_FULL_MASK, inc, o);
    if (lane >= o) inc += y;
  }
  const int64_t total = __shfl_sync(KIV_FULL_MASK, inc, 31);
  const int64_t G = min((int64_t)gridDim.x, p.tps < p.tpt ? (total + 1) / 2 : total), c = blockIdx.x;
  PagedSpot r;
  r.total = total;
  r.blocks = G;
  r.unit = c < G ? paged_div(c * total, G) : total;   // below 2^63: N counts tiles, c blocks
  r.end = c < G ? paged_div((c + 1) * total, G) : total;
  r.hp = r.rt = 0;
  r.off = 0;
  r.it.s.b = -1;
  r.it.nrt = 0;
  if (c >= G) return r;
  // the lane whose sequences hold the place, then the sequence among them
  int64_t at = r.unit - (inc - mine);
  const int owner = __ffs(__ballot_sync(KIV_FULL_MASK, at >= 0 && at < mine)) - 1;
  if (lane == owner && per > 1) {
    for (int b = b0; b < b1; ++b) {
      own = paged_items(p, b);
      const int64_t n = own.nrt > 0 ? H * paged_line(p, own, own.nrt) : 0;
      if (at < n) break;
      at -= n;
    }
  }
  int64_t rem = __shfl_sync(KIV_FULL_MASK, at, owner);
  r.it.s.b = __shfl_sync(KIV_FULL_MASK, own.s.b, owner);
  r.it.s.q0 = __shfl_sync(KIV_FULL_MASK, own.s.q0, owner);
  r.it.s.n = __shfl_sync(KIV_FULL_MASK, own.s.n, owner);
  r.it.s.len = __shfl_sync(KIV_FULL_MASK, own.s.len, owner);
  r.it.nrt = __shfl_sync(KIV_FULL_MASK, own.nrt, owner);
  r.it.base = __shfl_sync(KIV_FULL_MASK, own.base, owner);
  const int64_t per_head = paged_line(p, r.it, r.it.nrt);
  r.hp = (int)paged_div(rem, per_head);
  rem -= (int64_t)r.hp * per_head;
  // largest rt with prefix(rt) <= rem: the lanes try 32 places at a time
  int a = 0, z = r.it.nrt;
  while (z - a > 1) {
    const int stride = (z - a + 31) / 32, x = a + lane * stride;
    const unsigned under = __ballot_sync(KIV_FULL_MASK, x < z && paged_line(p, r.it, x) <= rem);
    a += (31 - __clz(under)) * stride;           // lane 0 always holds
    z = min(z, a + stride);
  }
  r.rt = a;
  r.off = rem - paged_line(p, r.it, a);
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
  int t0, t1;            // equal: the stretch ends on the item's first units, without a whole tile
  bool head, tail;       // the item began in an earlier block / goes on in a later one
};

__device__ __forceinline__ PagedSegment paged_segment(const PagedPlan &p, const PagedSpot &at) {
  PagedSegment g;
  const int nt = paged_tiles(p, at.it, at.rt), shift = paged_weight(p, at.it, at.rt) - 1;
  g.t0 = (int)(at.off >> shift);
  g.t1 = (int)min((int64_t)nt, (at.off + (at.end - at.unit)) >> shift);
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
    r.n = at.it.s.n;
    r.q0 = at.it.s.q0;
    // the block of the item's last tile: the last c' whose stretch begins
    // (c' N / G) before the item's end
    const int64_t end = at.unit - at.off + paged_units(p, at.it, at.rt);
    r.last = (int)((end * at.blocks - 1) / at.total);
  }
  p.cut[c] = r;
}

// On to the next item of the stretch, or to its end (b = -1)
__device__ __forceinline__ void paged_advance(const PagedPlan &p, PagedSpot &at, const PagedSegment &g) {
  if (g.tail) {
    at.it.s.b = -1;
    return;
  }
  at.unit += paged_units(p, at.it, at.rt) - at.off;
  paged_next(p, at);
}

__device__ __forceinline__ void paged_check_lens(const kiv_paged &pc, const PagedSeq &s) {
  const int64_t len = pc.seq_lens[s.b];
  if (len < s.n || len > pc.table_width * pc.page_size) paged_error(pc.errors, KIV_ERRBIT_SEQ_LEN);
}

__device__ __forceinline__ float *paged_part(const PagedPlan &p, int64_t slot, int row) {
  return p.part + (((int64_t)(row >> 3) * p.slots + slot) * 8 + (row & 7)) * partial_stride(p.pc.head_dim);
}

// Row r of an item's tile: token (in the sequence) and query head, or false
__device__ __forceinline__ bool paged_row(const PagedPlan &p, const PagedItems &it, int hp, int rt, int r, int &i, int &head) {
  const int ti = (uint32_t)r / (uint32_t)p.grp, g = r - ti * p.grp;
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
// A row's factor and log-sum-exp from its maximum and sum.  A row that has seen
// no key has the sum 0; a sum that is NaN (a NaN in the query or in a key that it
// sees) stays one.
__device__ __forceinline__ float paged_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float paged_log(float m, float l) { return l == 0.f ? -INFINITY : m + logf(l); }
__device__ __forceinline__ void paged_lse(const PagedPlan &p, const PagedItems &it, int i, int head, float m, float l) {
  if (p.q.lse) p.q.lse[(it.s.q0 + i) * p.q.num_query_heads + head] = paged_log(m, l);
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
