// Paged attention on tcgen05, head dimension 256.
//
// The output of one row tile (128 x 256 fp32) fills half of TMEM, so an item is
// one row tile and the two halves of the other 256 columns hold the scores of
// two key tiles in turn: S(j+1) is computed while the softmax works on S(j).
// Warp roles:
//   warps 8, 11  TMA: the query tile, then K and V of 128 keys through a ring of
//            five 32 KB slots (K: two halves of the columns, V: two halves of
//            the rows, so that every product finds its operand at one stride);
//   warp 9   S(j+1) = Q K^T;    warp 10   O += P(j) V(j);
//   warps 0-3 and 4-7: softmax, a thread per row and half of the columns; the
//            row's maximum meets in shared memory once per tile.
// Per key tile the tensor cores need 1024 cycles for each product, the special
// function units 1024 for the exponentials, and 128 KB come from L2: 62 bytes a
// cycle, so the tensor cores and L2 share the bound.  Measured: two chunks of up
// to 2047 tokens over up to 18 k keys, 8/1 x 256: 290 us, 1.0 PFLOP/s; single
// tokens of 64 sequences of 32 k keys in pages of 16 read at 6.2 TB/s (one TMA
// warp: 4.0).
//
// The rest (lazy rescale, dead rows, P over S in TMEM) is as in paged_tc.cu.
#include <algorithm>

#include "internal.h"
#include "paged_tc.cuh"

namespace kiv {

constexpr int P2_D = 256;
constexpr int P2_SLOT = 32768;
constexpr int P2_SLOTS = 5;
constexpr int P2_QBYTES = PT_ROWS * P2_D * 2;
constexpr size_t P2_SMEM = P2_QBYTES + (size_t)P2_SLOTS * P2_SLOT + 2 * 2 * PT_ROWS * sizeof(float);   // + maxima: all there is

// ring positions: K(0), then K(t + 1) (while there is one) and V(t), two slots each
struct P2Ring {
  uint32_t n = 0;        // position of the next slot
  __device__ __forceinline__ uint32_t slot(uint32_t h) const { return (n + h) % P2_SLOTS; }
  __device__ __forceinline__ uint32_t parity(uint32_t h) const { return ((n + h) / P2_SLOTS) & 1; }
  __device__ __forceinline__ void skip() { n += 2; }
};

template <bool BF>
__global__ void __launch_bounds__(PT_THREADS, 1)
paged_tc256_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedPlan p, PagedTcGeom g) {
  using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t p2_dyn[];
  __shared__ uint64_t q_full, q_empty, kv_full[P2_SLOTS], kv_empty[P2_SLOTS], s_full[2], p_full[2], pv_done[2], halt[2];
  __shared__ uint32_t s_tmem;
  __shared__ PtSeg seg[2];
  const int warp = __shfl_sync(KIV_FULL_MASK, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  uint8_t *qmem = p2_dyn, *ring = p2_dyn + P2_QBYTES;
  float(*s_max)[2][PT_ROWS] = reinterpret_cast<float(*)[2][PT_ROWS]>(ring + P2_SLOTS * P2_SLOT);   // [tile parity][column half][row]

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 10);                   // last scores, last product, and the softmax warps have read `seg`
    for (int i = 0; i < P2_SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
      mbar_init(&halt[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == 9) {
    tc::tmem_alloc(&s_tmem, 512);
    tc::tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tc::prefetch_map(&qmap);
    tc::prefetch_map(&kmap);
    tc::prefetch_map(&vmap);
  }
  // rows of the row tile that no query box covers stay zero
  for (int x = threadIdx.x; x < P2_QBYTES / 16; x += PT_THREADS) reinterpret_cast<uint4 *>(qmem)[x] = make_uint4(0, 0, 0, 0);
  tc::fence_proxy_async_smem();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;                // scores [0, 256), output [256, 512)
  griddep_wait();
  bool ok = true, mma = false;
  uint32_t turn = 0, qturn = 0;                // what this warp asked TMA for
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (ok && !mbar_wait_bounded(bar, parity)) ok = false;
  };
  const int rows = g.tps * p.grp;

  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_OTHER));
   if (warp == 8 || warp == 11) {
    // ------------------------------------------------ TMA (two warps share the boxes of every slot)
    const int me = warp == 8 ? 0 : 1;
    const bool leader = elect_one();
    PagedSpot at = paged_locate(p);
    P2Ring r;
    const int nbox = PT_KEYS / g.br, half = 64 / g.br;    // boxes of a K tile; of a V half
    if (me == 0 && lane == 0) p.cut[blockIdx.x].b = -1;
    uint32_t items = 0;
    for (;; ++items) {
      PtSeg sg = {};
      PagedSegment cut = {};
      int kvh = 0;
      if (at.it.s.b >= 0 && at.unit < at.end) sg = pt_segment(p, at, g.tps, cut, kvh);
      const int ntile = sg.ntile;              // 0: done
      // lane l brings rows [l br, (l + 1) br) of every tile
      const int32_t *table = p.pc.block_table + (ntile > 0 ? at.it.s.b : 0) * p.pc.table_stride;
      auto lookup = [&](int t, int32_t &page, int32_t &row) {
        page = -1;
        row = 0;
        if (t < ntile && lane < nbox) pt_lookup(p, table, sg, sg.j00 + (int64_t)t * PT_KEYS + lane * g.br, g.br, page, row);
      };
      int32_t page, row;
      lookup(0, page, row);
      // as in paged_tc.cu: this item's first slots may come before its queries
      bool told = me != 0;
      int slots = 0;
      auto tell = [&](bool must) {
        if (told) return;
        if (items > 0 && !must && !__shfl_sync(KIV_FULL_MASK, (int)mbar_test(&q_empty, (items - 1) & 1), 0)) return;
        if (items > 0) wait(&q_empty, (items - 1) & 1);
        if (lane == 0 && ok) {
          seg[items & 1] = sg;
          if (ntile == 0) {
            mbar_arrive(&q_full);
          } else {
            mbar_arrive_tx(&q_full, (uint32_t)rows * P2_D * 2);
            for (int c = 0; c < 4; ++c)
              tc::tma_load_3d(qmem + c * (PT_ROWS * 128), &qmap, c * 64, sg.head0, (int32_t)sg.q0, &q_full);
          }
        }
        __syncwarp();
        told = true;
      };
      if (ntile == 0) {
        tell(true);
        break;
      }
      auto begin = [&](uint32_t h) {           // nullptr: a wait ran out, nothing more is asked for
        tell(slots++ >= P2_SLOTS);
        if (r.n + h >= P2_SLOTS) wait(&kv_empty[r.slot(h)], r.parity(h) ^ 1);
        if (!__all_sync(KIV_FULL_MASK, ok)) {
          turn = turn > 0 ? turn : r.n + h;
          return (uint8_t *)nullptr;
        }
        if (me == 0 && leader) mbar_arrive_tx(&kv_full[r.slot(h)], P2_SLOT);
        return ring + r.slot(h) * P2_SLOT;
      };
      auto load_k = [&](int32_t page, int32_t row) {   // slot h: columns [128 h, 128 h + 128) of all rows
        for (uint32_t h = 0; h < 2; ++h) {
          uint8_t *dst = begin(h);
          if (!dst) break;
          for (int l = 0; l < nbox; ++l) {
            const int32_t bp = __shfl_sync(KIV_FULL_MASK, page, l), br = __shfl_sync(KIV_FULL_MASK, row, l);
            if (leader) tc::tma_load_4d(dst + me * (PT_KEYS * 128) + l * g.br * 128, &kmap, (2 * h + me) * 64, br, kvh, bp, &kv_full[r.slot(h)]);
          }
        }
        r.skip();
      };
      auto load_v = [&](int32_t page, int32_t row) {   // slot h: rows [64 h, 64 h + 64)
        for (uint32_t h = 0; h < 2; ++h) {
          uint8_t *dst = begin(h);
          if (!dst) break;
          for (int l = 0; l < half; ++l) {
            const int32_t bp = __shfl_sync(KIV_FULL_MASK, page, h * half + l), br = __shfl_sync(KIV_FULL_MASK, row, h * half + l);
            if (leader) {
              for (int c = 2 * me; c < 2 * me + 2; ++c)
                tc::tma_load_4d(dst + c * (64 * 128) + l * g.br * 128, &vmap, c * 64, br, kvh, bp, &kv_full[r.slot(h)]);
            }
          }
        }
        r.skip();
      };
      int32_t npage, nrow;
      load_k(page, row);
      lookup(1, npage, nrow);
      for (int t = 0; t < ntile; ++t) {
        int32_t ppage, prow;
        lookup(t + 2, ppage, prow);
        if (t + 1 < ntile) load_k(npage, nrow);
        load_v(page, row);
        page = npage;
        row = nrow;
        npage = ppage;
        nrow = prow;
      }
      tell(true);
      if (me == 0 && lane == 0) {
        if (!cut.head) paged_check_lens(p.pc, at.it.s);
        if (cut.tail) paged_record(p, blockIdx.x, at, cut);
      }
      if (!__all_sync(KIV_FULL_MASK, ok)) break;
      paged_advance(p, at, cut);
    }
    if (__all_sync(KIV_FULL_MASK, ok)) turn = r.n;
    qturn = items + 1;                         // a query tile not asked for: its wait ends at the limit
   } else if (warp == 9) {
    // ------------------------------------------------ S = Q K^T
    constexpr uint32_t id_s = tc::idesc_f16(BF, PT_ROWS, PT_KEYS);
    const uint64_t qd = tc::sdesc_k128(smem_u32(qmem)), kd = tc::sdesc_k128(smem_u32(ring));
    const bool leader = elect_one();
    mma = leader;
    P2Ring r;
    uint32_t tiles = 0;
    for (uint32_t items = 0;; ++items) {
      wait(&q_full, items & 1);
      const int ntile = __shfl_sync(KIV_FULL_MASK, ok ? seg[items & 1].ntile : 0, 0);
      if (ntile == 0) break;
      for (int t = 0; t < ntile; ++t, ++tiles) {
        // the buffer's last P is used (and with it the ring's V slot that the K tile follows)
        if (tiles >= 2) wait(&pv_done[tiles & 1], ((tiles >> 1) - 1) & 1);
        for (uint32_t h = 0; h < 2; ++h) {
          wait(&kv_full[r.slot(h)], r.parity(h));
          tc::fence_after_sync();
          if (leader) {
            const uint64_t b = kd + r.slot(h) * (P2_SLOT >> 4), a = qd + h * 2 * ((PT_ROWS * 128) >> 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t off = ((uint32_t)(k / 4) * (PT_KEYS * 128) + (uint32_t)(k % 4) * 32) >> 4;
              tc::mma_f16(tmem + (tiles & 1) * PT_KEYS, a + off, b + off, id_s, (h > 0 || k > 0) ? 1u : 0u);
            }
            tc::commit(&kv_empty[r.slot(h)]);
          }
        }
        if (leader) {
          tc::commit(&s_full[tiles & 1]);
          if (t + 1 == ntile) tc::commit(&q_empty);
        }
        r.skip();
        if (t > 0) r.skip();                   // V(t - 1) lies behind K(t)
      }
      r.skip();                                // V of the last tile
    }
   } else if (warp == 10) {
    // ------------------------------------------------ O += P V
    constexpr uint32_t id_o = tc::idesc_f16(BF, PT_ROWS, P2_D) | (1u << 16);   // B is MN-major
    const uint64_t vd = tc::sdesc_mn<128>(smem_u32(ring), 64 * 128);
    const bool leader = elect_one();
    mma = leader;
    P2Ring r;
    uint32_t tiles = 0;
    for (uint32_t items = 0;; ++items) {
      wait(&q_full, items & 1);
      const int ntile = __shfl_sync(KIV_FULL_MASK, ok ? seg[items & 1].ntile : 0, 0);
      if (ntile == 0) break;
      r.skip();                                // K(0)
      for (int t = 0; t < ntile; ++t, ++tiles) {
        if (t + 1 < ntile) r.skip();           // K(t + 1)
        wait(&p_full[tiles & 1], (tiles >> 1) & 1);
        for (uint32_t h = 0; h < 2; ++h) {
          wait(&kv_full[r.slot(h)], r.parity(h));
          tc::fence_after_sync();
          if (leader) {
            const uint64_t b = vd + r.slot(h) * (P2_SLOT >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc::mma_f16_ta(tmem + 2 * PT_KEYS, tmem + (tiles & 1) * PT_KEYS + (h * 4 + k) * 8, b + k * ((16 * 128) >> 4), id_o,
                             (t % PT_FLUSH > 0 || h > 0 || k > 0) ? 1u : 0u);
            tc::commit(&kv_empty[r.slot(h)]);
          }
        }
        if (leader) {
          tc::commit(&pv_done[tiles & 1]);
          if (t + 1 == ntile) tc::commit(&q_empty);
        }
        r.skip();
      }
    }
   }
  } else {
    // ------------------------------------------------ softmax: row `r`, keys [64 w, 64 w + 64) of a tile
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    constexpr int COLS = PT_KEYS / 2;
    const int w = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t to = tmem + lanes + 2 * PT_KEYS + w * (P2_D / 2);     // this thread's half of the output row
    const bool cap = p.q.softcap > 0.f;
    const float c = (cap ? 1.f : p.q.scaling) * 1.44269504f;
    const int ti = r / p.grp, gi = r - ti * p.grp;
    P2Ring vr;
    uint32_t tiles = 0;
    for (uint32_t items = 0;; ++items) {
      wait(&q_full, items & 1);
      const PtSeg sg = seg[items & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty);
      // a wait that ran out in one warp ends the loop in all: they share barriers
      uint32_t failed;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 1, 256, q;\n selp.u32 %0, 1, 0, p;\n}\n"
                   : "=r"(failed)
                   : "r"(ok ? 0u : 1u)
                   : "memory");
      if (failed || sg.ntile == 0) break;
      const bool have = ti < g.tps && gi < sg.heads && ti < sg.tok;
      const int place = p.q.causal ? sg.base + ti : 0x7fffffff;
      const int64_t free_hi = p.q.causal ? min((int64_t)sg.hi - 1, (int64_t)sg.base) : (int64_t)sg.hi - 1;
      const int64_t free_lo = max((int64_t)sg.lo, p.q.window > 0 ? (int64_t)sg.base + g.tps - p.q.window : (int64_t)0);
      const bool idle = (warp & 3) * 32 >= min(rows, sg.tok * p.grp);   // a warp without rows keeps the beat
      float m = -INFINITY, l = 0.f;
      // the row that the output moves to, as in paged_tc.cu
      const bool row = r < rows;
      float *const acc = paged_part(p, sg.part >= 0 ? sg.part : 2 * (int)blockIdx.x + 1, r) + w * (P2_D / 2);
      bool moved = false;
      float m_at = m;
      vr.skip();                               // K(0)
      for (int t = 0; t < sg.ntile; ++t, ++tiles) {
        if (t + 1 < sg.ntile) vr.skip();       // K(t + 1); now at V(t)
        const uint32_t ts = tmem + lanes + (tiles & 1) * PT_KEYS;
        wait(&s_full[tiles & 1], (tiles >> 1) & 1);
        tc::fence_after_sync();
        const int64_t j0 = sg.j00 + (int64_t)t * PT_KEYS;
        if (j0 < sg.lo || j0 + PT_KEYS > sg.hi) {
          // Dead rows of V half w, after the product before this one (which
          // used the slot's turn before) and before this one's, which waits
          // for p_full below.
          if (tiles > 0) wait(&pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1);
          wait(&kv_full[vr.slot(w)], vr.parity(w));
          const int dl = (int)max((int64_t)0, sg.lo - j0), dh = (int)max((int64_t)0, min((int64_t)PT_KEYS, sg.hi - j0));
          const int row = w * 64 + (r >> 1);
          if (row < dl || row >= dh) {
#pragma unroll 1
            for (int y = (r & 1) * 16; y < (r & 1) * 16 + 16; ++y)
              *reinterpret_cast<uint4 *>(ring + vr.slot(w) * P2_SLOT + (y / 8) * (64 * 128) + (r >> 1) * 128 + (y % 8) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
        }
        vr.skip();
        if (idle) {                            // what P holds for these rows stays in their own rows
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (lane == 0) mbar_arrive(&p_full[tiles & 1]);
          continue;
        }
        uint32_t su[COLS];
        tc::ld_32x32(ts + w * COLS, su);
        tc::ld_32x32(ts + w * COLS + 32, su + 32);
        tc::wait_ld32(su);
        tc::wait_ld32(su + 32);
        if (cap) cap_scores<COLS>(reinterpret_cast<float *>(su), p.q.softcap, p.q.scaling);
        if (j0 < free_lo || j0 + PT_KEYS - 1 > free_hi) {
          // of this thread's columns [bot, top] are seen
          const int top = (int)min((int64_t)PT_KEYS, min((int64_t)sg.hi - 1, (int64_t)place) - j0) - w * COLS;
          const int bot = (int)max((int64_t)0, max((int64_t)sg.lo, p.q.window > 0 ? (int64_t)place - p.q.window + 1 : (int64_t)0) - j0) - w * COLS;
#pragma unroll
          for (int x = 0; x < COLS; ++x)
            if (x > top || x < bot) su[x] = 0xff800000u;
        }
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int x = 0; x < COLS; x += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            mx[y] = fmaxf(mx[y], fmaxf(__uint_as_float(su[x + 2 * y]), __uint_as_float(su[x + 2 * y + 1])));
        }
        float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        s_max[tiles & 1][w][r] = mn;
        // both halves of the scores are read and both maxima written (the
        // previous tile's are read before this barrier's next turn)
        tc::fence_before_sync();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tc::fence_after_sync();
        mn = fmaxf(mn, s_max[tiles & 1][w ^ 1][r]);
        if (t == 0) {
          m = mn;
        } else if (__any_sync(KIV_FULL_MASK, (mn - m) * c > PT_LAZY<BF>)) {   // the same in both groups
          const float f = mn == -INFINITY ? 1.f : ex2((m - mn) * c);
          l *= f;
          m = mn;
          wait(&pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1);
          tc::fence_after_sync();
#pragma unroll 1
          for (int x = 0; x < P2_D / 2; x += 16) {
            uint32_t o[16];
            tc::ld_32x16(to + x, o);
            tc::wait_ld16(o);
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tc::st_32x16(to + x, o);
          }
        }
        if (t > 0 && t % PT_FLUSH == 0) {
          wait(&pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1);
          tc::fence_after_sync();
          pt_flush<P2_D / 2>(to, acc, !moved ? 0.f : m_at == m ? 1.f : ex2((m_at - m) * c), row);
          moved = true;
          m_at = m;
        }
        const float2 c2 = make_float2(c, c);
        const float neg = pt_shift<BF>(m, c);
        const float2 n2 = make_float2(neg, neg);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[COLS / 2];
#pragma unroll
        for (int y = 0; y < COLS; y += 2) {
          float2 e = __ffma2_rn(make_float2(__uint_as_float(su[y]), __uint_as_float(su[y + 1])), c2, n2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(y >> 1) & 1] = __fadd2_rn(sum[(y >> 1) & 1], e);
          pk[y / 2] = pt_pack<BF>(e.x, e.y);
        }
        tc::st_32x32(ts + w * (COLS / 2), pk);
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[tiles & 1]);
      }
      // ---- the item's rows
      // sums meet where the last maxima did, once those are read
      float(*sum_at)[PT_ROWS] = s_max[(tiles - 1) & 1];
      asm volatile("bar.sync 1, 256;" ::: "memory");
      sum_at[w][r] = l;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      l += sum_at[w ^ 1][r];                   // a + b in both groups: the same
      wait(&pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1);
      tc::fence_after_sync();
      const float mnat = pt_reference<BF>(m, c);
      const bool whole = sg.part < 0;
      const float inv = paged_inv(l);
      const float fa = moved ? (m_at == m ? 1.f : ex2((m_at - m) * c)) : 0.f;
      const int head = sg.head0 + gi;
      T *dst = static_cast<T *>(p.q.out) + (sg.q0 + ti) * p.q.out_stride_t + head * p.q.out_stride_h + w * (P2_D / 2);
      float *part = paged_part(p, sg.part, r) + w * (P2_D / 2);
#pragma unroll
      for (int x = 0; x < P2_D / 2; x += 32) {
        uint32_t o[32];
        tc::ld_32x32(to + x, o);
        tc::wait_ld32(o);
        if (!have) continue;
        if (fa != 0.f) {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(fmaf(acc[x + y], fa, __uint_as_float(o[y])));
        }
        if (whole) {
#pragma unroll
          for (int y = 0; y < 32; y += 8) {
            uint4 u;
            u.x = pt_pack<BF>(__uint_as_float(o[y]) * inv, __uint_as_float(o[y + 1]) * inv);
            u.y = pt_pack<BF>(__uint_as_float(o[y + 2]) * inv, __uint_as_float(o[y + 3]) * inv);
            u.z = pt_pack<BF>(__uint_as_float(o[y + 4]) * inv, __uint_as_float(o[y + 5]) * inv);
            u.w = pt_pack<BF>(__uint_as_float(o[y + 6]) * inv, __uint_as_float(o[y + 7]) * inv);
            st16(dst + x + y, u);
          }
        } else {
#pragma unroll
          for (int y = 0; y < 32; y += 4) st16(part + x + y, make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]));
        }
      }
      if (have && w == 0) {
        if (whole) {
          if (p.q.lse) p.q.lse[(sg.q0 + ti) * p.q.num_query_heads + head] = paged_log(mnat, l);
        } else {
          part[P2_D] = mnat;
          part[P2_D + 1] = l;
        }
      }
      tc::fence_before_sync();                 // the next item's products overwrite the output
    }
  }
  if (!ok) paged_error(p.pc.errors, KIV_ERRBIT_WAIT_TIMEOUT);
  tc::fence_before_sync();
  pt_finish<P2_SLOTS>(ok, kv_full, turn, &q_full, qturn, mma, &halt[warp == 10]);
  tc::fence_after_sync();
  if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

template <bool BF>
static kiv_status launch_tc256(const PagedPlan &p, int blocks, cudaStream_t s) {
  PagedTcGeom g;
  g.tps = PT_ROWS / p.grp;
  g.br = 8;
  while (g.br < 64 && p.pc.page_size % (2 * g.br) == 0) g.br *= 2;
  CUtensorMap qm, km, vm;
  KIV_CHECK(pt_maps(p, 64, g.br, g.tps, CU_TENSOR_MAP_SWIZZLE_128B, &qm, &km, &vm));
  cudaFuncSetAttribute(paged_tc256_kernel<BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P2_SMEM);
  KIV_CHECK(cuda_status(launch_pdl(paged_tc256_kernel<BF>, dim3((unsigned)blocks), dim3(PT_THREADS), P2_SMEM, s, 1, qm, km, vm, p, g),
                        "paged_attend (chunk, 256)"));
  return launch_paged_combine(p, blocks, s);
}

kiv_status launch_paged_tc256(const PagedPlan &p, int blocks, cudaStream_t s) {
  return p.pc.dtype == KIV_DTYPE_BF16 ? launch_tc256<true>(p, blocks, s) : launch_tc256<false>(p, blocks, s);
}

}  // namespace kiv
