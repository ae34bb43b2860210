// What the two tcgen05 kernels over a paged cache share (paged_tc.cu for head
// dimensions up to 128, paged_tc256.cu for 256).
#pragma once

#include "paged.cuh"
#include "tc.cuh"

namespace kiv {

constexpr int PT_KEYS = 128;
constexpr int PT_ROWS = 128;                   // of one row tile
constexpr int PT_THREADS = 384;                // three warpgroups: two of softmax, one with the TMA and the MMA warp
// registers per thread: 168 at launch, (2 x 208 + 88) x 128 = 168 x 384 after the split
constexpr int PT_REGS_SOFTMAX = 208, PT_REGS_OTHER = 88;
constexpr int PT_HEAD = 96;                    // keys of a tile whose P V product begins before the rest of P is there
// The tensor cores' accumulation cuts instead of rounding: a sum drifts towards
// zero by 1e-7 of itself with every 16 keys (1.2e-3 after 200 k).  After this
// many key tiles (1e-4) the output moves to a row of the workspace, added by
// ordinary additions, and the products begin at zero again.
constexpr int PT_FLUSH = 128;
// Growth (log2) that a row's reference may lag behind, and the power of two by
// which every weight, its sum and so the reference are scaled.  fp16 weights
// would be subnormal below 2^-14 and vanish below 2^-25 of the reference while
// the sum still counted them: one key 17 above a long tail lost the tail.  At
// 2^11 they are whole down to 2^-25 and vanish below 2^-36 (128 k keys of those
// hold 2e-6 of the row); the largest is 2^4 2^11, half of what fp16 holds.
template <bool BF> constexpr float PT_LAZY = BF ? 8.f : 4.f;
template <bool BF> constexpr float PT_BIAS = BF ? 0.f : 11.f;

struct PagedTcGeom {
  int tps;       // tokens per row tile
  int br;        // rows per TMA box of a page: a power of two dividing page_size, at most 128
};

namespace tc {
// A [TMEM, 16-bit pairs per column] x B [smem]
__device__ __forceinline__ void mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major operand (rows = K index, contiguous along N) of a swizzled tile:
// column blocks `block` bytes apart, 8-row groups 8 * row bytes apart
template <int ROWB>
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t addr, uint32_t block) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(block >> 4) << 16;
  d |= (uint64_t)((8 * ROWB) >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(ROWB == 128 ? 2 : 4) << 61;
  return d;
}
__device__ __forceinline__ void ld_32x32(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void st_32x32(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void st_32x16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// completion of the loads into r: the registers are operands, so no use of
// them can move before it
__device__ __forceinline__ void wait_ld32(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void wait_ld16(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
}  // namespace tc

// whether the phase of this parity is over, without waiting for it
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}

// one lane of the (converged) warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

template <bool BF>
__device__ __forceinline__ uint32_t pt_pack(float x, float y) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

// What a row's score times c is added to in the exponent of its weight, m being
// the reference.  Rounded down, so that no weight passes 2^(PT_LAZY + PT_BIAS)
// however large the scores.
template <bool BF>
__device__ __forceinline__ float pt_shift(float m, float c) {
  if (m == -INFINITY) return 0.f;
  return BF ? -m * c : __fmaf_rd(-m, c, PT_BIAS<BF>);
}
// The natural logarithm of what the weights of reference m count in
template <bool BF>
__device__ __forceinline__ float pt_reference(float m, float c) {
  return (BF ? m * c : m * c - PT_BIAS<BF>) * 0.693147181f;
}

// Waits, with a limit, for the copies that are on the way to a ring of N stages
// whose next turn is `turn`.
template <int N>
__device__ __forceinline__ void pt_drain(uint64_t *full, uint32_t turn) {
#pragma unroll 1
  for (uint32_t k = 1; k <= N && k <= turn; ++k)
    if (!mbar_wait_bounded(&full[(turn - k) % N], ((turn - k) / N) & 1)) return;
}

// Where a wait ran out, a role goes on without its waits or leaves, so copies and
// products on the way may outlast the roles.  End of the kernel, all threads:
// waits for them, again with a limit, before the block's memory is given back.
// turn, qturn: the ring's turns and the query tiles that this lane's warp asked
// TMA for; mma: the lane of an MMA warp that issued its products.
template <int SLOTS>
__device__ __forceinline__ void pt_finish(bool ok, uint64_t *kv_full, uint32_t turn, uint64_t *q_full, uint32_t qturn, bool mma,
                                          uint64_t *halt) {
  if (__syncthreads_or(ok ? 0 : 1) == 0) return;
  if (qturn > 0) mbar_wait_bounded(q_full, (qturn - 1) & 1);
  pt_drain<SLOTS>(kv_full, turn);
  if (mma) {
    tc::commit(halt);
    mbar_wait_bounded(halt, 0);
  }
  __syncthreads();
}

// One segment of the block's stretch, as the TMA warp tells the others.
struct PtSeg {
  int ntile;       // 0: no more
  int nsub;        // row tiles that have tokens
  int lo, hi;      // live keys
  int64_t j00;     // first key of its first key tile
  int64_t q0;      // packed row of token 0 of the item's first row tile
  int tok;         // tokens from there on
  int base;        // place of that token (causal), or the length
  int head0, heads;   // its query heads
  int part;        // workspace slot, or -1: the rows are finished here
};

// Descriptor of the segment at `at` (not past the block's stretch).  `tps`:
// whole tokens per row tile, an item being one or two of them.
__device__ __forceinline__ PtSeg pt_segment(const PagedPlan &p, const PagedSpot &at, int tps, PagedSegment &cut, int &kvh) {
  PtSeg sg = {};
  const int per = p.q.num_query_heads / p.pc.num_kv_heads;
  cut = paged_segment(p, at);
  paged_range(p, at.it, at.rt, sg.lo, sg.hi);
  sg.hi = min(sg.hi, at.it.s.len);
  sg.j00 = ((int64_t)(sg.lo / PT_KEYS) + cut.t0) * PT_KEYS;
  sg.ntile = cut.t1 - cut.t0;
  const int first = at.rt * p.tpt;
  sg.q0 = at.it.s.q0 + first;
  sg.tok = min(at.it.s.n - first, p.tpt);
  sg.nsub = sg.tok > tps ? 2 : 1;
  sg.base = p.q.causal ? at.it.base + first : at.it.s.len;
  const int part = p.hs == 1 ? 0 : at.hp % p.hs;
  kvh = p.hs == 1 ? at.hp : at.hp / p.hs;
  sg.head0 = kvh * per + part * p.grp;
  sg.heads = min(p.grp, per - part * p.grp);
  sg.part = cut.head ? 2 * (int)blockIdx.x : cut.tail ? 2 * (int)blockIdx.x + 1 : -1;
  return sg;
}

// Page and row of the `br` keys from key j on of sequence b; page -1: no live
// key, or no page: the box reads as zeros.
__device__ __forceinline__ void pt_lookup(const PagedPlan &p, const int32_t *table, const PtSeg &sg, int64_t j, int br, int32_t &page,
                                          int32_t &row) {
  page = -1;
  row = 0;
  if (j < sg.hi && j + br > sg.lo) {
    const uint32_t pg = (uint32_t)j / (uint32_t)p.pc.page_size;
    row = (int32_t)((uint32_t)j - pg * (uint32_t)p.pc.page_size);
    page = table[pg];
    if (page < 0 || page >= p.pc.num_pages) {
      paged_error(p.pc.errors, KIV_ERRBIT_BLOCK_TABLE);
      page = -1;
    }
  }
}

// Adds N columns of a row's output in TMEM to its row in the workspace: acc <-
// acc f + o (f = 0: what is there does not count).  The whole warp; only lanes
// with a row touch memory.
template <int N>
__device__ __forceinline__ void pt_flush(uint32_t to, float *acc, float f, bool row) {
#pragma unroll 1
  for (int x = 0; x < N; x += 16) {
    uint32_t o[16];
    tc::ld_32x16(to + x, o);
    tc::wait_ld16(o);
    if (row) {
#pragma unroll
      for (int y = 0; y < 16; y += 4) {
        float4 *at = reinterpret_cast<float4 *>(acc + x + y);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (f != 0.f) v = *at;
        v.x = fmaf(v.x, f, __uint_as_float(o[y]));
        v.y = fmaf(v.y, f, __uint_as_float(o[y + 1]));
        v.z = fmaf(v.z, f, __uint_as_float(o[y + 2]));
        v.w = fmaf(v.w, f, __uint_as_float(o[y + 3]));
        *at = v;
      }
    }
  }
}

kiv_status pt_maps(const PagedPlan &p, int box, int br, int tps, CUtensorMapSwizzle sw, CUtensorMap *qm, CUtensorMap *km, CUtensorMap *vm);
kiv_status launch_paged_tc256(const PagedPlan &p, int blocks, cudaStream_t s);

}  // namespace kiv
