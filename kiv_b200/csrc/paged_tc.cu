// Paged attention on tcgen05, head dimensions 64, 96 and 128: chunks of new
// tokens (bound by the tensor cores) and single ones (bound by memory).
//
//   S = Q K^T and O += P V as 128 x 128 x D and 128 x D x 128 products with
//   fp32 accumulators in TMEM; the softmax in between is one pass with the
//   running maximum and sum of each row in registers.
//
// A block takes items of two row tiles of 128 rows: a row is (token, query
// head of the key head), so the heads of a group share every K and V tile
// (`tps` = 128 / heads whole tokens per tile).  Warp roles:
//   warps 8, 11  TMA: the query tiles, then K and V tiles of 128 keys through a
//            ring, one box of `br` rows per page piece;
//   warps 9, 10  MMA of row tile 0 and 1: O += P(j) V(j), then S(j+1);
//   warps 0-3 and 4-7: softmax of row tile 0 and 1, a thread per row.
// An item with one row tile (a single token's heads, a few drafted tokens, a
// short prompt) would leave one group idle and the other one's chain scores ->
// softmax -> product exposed: there both take the same rows, one over the even
// key tiles and one over the odd ones, and join at the end ("twins").  So the
// same kernel serves decode, bound by memory: warps without rows only keep the
// beat, and the tensor cores' empty rows cost nothing that is missed.  Measured
// over 16 sequences of 16 k keys, one token each, pages of 128: 32/8 x 128 211 us
// (5.1 TB/s) and 32/4 x 64 79 us, against 250 and 103 us for m16n8k16 products
// split over the keys (paged_mma.cu); with pages of 16, 227 and 82 against 241
// and 103; four times the sequences, 850 against 838.  Without twins 32/4 x 64
// took 97 us where it took 76.
// While one row tile's softmax runs, the tensor cores work on the other's
// products, so both are kept busy: per tile pair the tensor cores need 4 x 512
// cycles (D = 128) and the 2 x 16384 exponentials 2048 cycles of the special
// function units.  Measured: 4096 tokens over 36864 keys, 32/8 x 128: 2.4-2.5 ms,
// 0.93-0.97 PFLOP/s at the power limit (1.3-1.4 GHz); with the softmax taken out
// the products alone take 1.6 ms.  One warp issuing both row tiles' products
// took 3950 cycles per tile pair where this takes 3240.
//
// P (16-bit) overwrites S in TMEM and is the A operand from there; V is read
// as an MN-major B operand straight from its row-major tile.  The output in
// TMEM is rescaled only when a row's maximum has grown by more than 2^8 (fp16
// 2^4) since the reference it was scaled with (weights up to 256 are as exact as
// weights up to 1: rounding is relative), which after the first tiles is almost
// never.  Rounding is relative as long as a weight is a normal number of its
// type: fp16 weights carry a power of two for that (PT_BIAS).
//
// Key tiles that hold the end of a sequence (or keys before a window) may hold
// anything in the dead rows, NaN too: scores there are replaced, not added to,
// and the softmax groups clear the dead V rows before their products.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"
#include "paged_tc.cuh"

namespace kiv {

template <int D>
struct TcShape {
  static constexpr int BOX = D % 64 == 0 ? 64 : 32;      // elements per TMA box: 128- or 64-byte swizzle
  static constexpr int NB = D / BOX;
  static constexpr int BOXB = BOX * 2;                   // bytes of a box row
  static constexpr int TILE = PT_KEYS * D * 2;           // bytes of a K, V or Q tile
  static constexpr int SLOTS = (232448 - 2048 - 2 * TILE) / TILE < 8 ? (232448 - 2048 - 2 * TILE) / TILE : 8;
  static constexpr size_t SMEM = 1024 + 2 * TILE + (size_t)SLOTS * TILE;
};

template <bool BF, int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedPlan p, PagedTcGeom g) {
  using S = TcShape<D>;
  using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
  constexpr int SLOTS = S::SLOTS;
  extern __shared__ uint8_t pt_dyn[];
  __shared__ uint64_t q_full, q_empty, kv_full[SLOTS], kv_empty[SLOTS], s_full[2], p_full[2], p_tail[2], o_full[2], halt[2];
  __shared__ uint32_t s_tmem;
  __shared__ PtSeg seg[2];
  __shared__ float s_ml[2][PT_ROWS];           // of the second of two twins
  // broadcast: the compiler then knows that a role's control flow is the warp's
  const int warp = __shfl_sync(KIV_FULL_MASK, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  uint8_t *smem = pt_dyn + ((1024 - (smem_u32(pt_dyn) & 1023)) & 1023);
  uint8_t *qmem = smem, *ring = smem + 2 * S::TILE;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 10);                   // each row tile's last scores; the softmax warps have read `seg`
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_tail[i], 4);
      mbar_init(&o_full[i], 1);
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
  // rows of a row tile that no query box covers stay zero
  for (int x = threadIdx.x; x < 2 * S::TILE / 16; x += PT_THREADS) reinterpret_cast<uint4 *>(qmem)[x] = make_uint4(0, 0, 0, 0);
  tc::fence_proxy_async_smem();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  griddep_wait();
  bool ok = true, mma = false;
  uint32_t turn = 0, qturn = 0;                // what this warp asked TMA for
  const int rows = g.tps * p.grp;              // of a row tile
  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_OTHER));
   if (warp == 8 || warp == 11) {
    // ------------------------------------------------ TMA
    // Two warps share the boxes of every tile: with pages of 16 tokens a tile
    // is 16 copies, and one warp issued them at 5.0 TB/s, no faster.
    const int me = warp == 8 ? 0 : 1;
    const bool leader = elect_one();
    PagedSpot at = paged_locate(p);
    uint32_t n = 0, items = 0;
    const int nbox = PT_KEYS / g.br;
    if (me == 0 && lane == 0) p.cut[blockIdx.x].b = -1;
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
      // The queries and `seg` replace the previous item's when those are used
      // up; until then this item's first keys and values can come.
      bool told = me != 0;
      auto tell = [&](bool must) {
        if (told) return;
        if (items > 0 && !must && !__shfl_sync(KIV_FULL_MASK, (int)mbar_test(&q_empty, (items - 1) & 1), 0)) return;
        if (items > 0 && ok && !mbar_wait_bounded(&q_empty, (items - 1) & 1)) ok = false;
        if (lane == 0 && ok) {
          seg[items & 1] = sg;
          if (ntile == 0) {
            mbar_arrive(&q_full);
          } else {
            mbar_arrive_tx(&q_full, (uint32_t)sg.nsub * rows * D * 2);
            for (int i = 0; i < sg.nsub; ++i)
              for (int c = 0; c < S::NB; ++c)
                tc::tma_load_3d(qmem + i * S::TILE + c * (PT_ROWS * S::BOXB), &qmap, c * S::BOX, sg.head0,
                                (int32_t)(sg.q0 + i * g.tps), &q_full);
          }
        }
        __syncwarp();
        told = true;
      };
      if (ntile == 0) {
        tell(true);
        break;
      }
      for (int t = 0; t < ntile; ++t) {
        const int32_t pg = page, rw = row;
        lookup(t + 1, page, row);
        for (int kv = 0; kv < 2; ++kv, ++n) {
          tell(2 * t + kv >= SLOTS);           // from there on a slot waits for this item's own tiles
          const uint32_t s = n % SLOTS;
          if (n >= SLOTS && ok && !mbar_wait_bounded(&kv_empty[s], (n / SLOTS - 1) & 1)) ok = false;
          if (!__all_sync(KIV_FULL_MASK, ok)) goto halted;     // nothing more is asked for
          if (me == 0 && leader) mbar_arrive_tx(&kv_full[s], S::TILE);
          const CUtensorMap *map = kv ? &vmap : &kmap;
          for (int x = me; x < nbox * S::NB; x += 2) {      // box x / NB, columns x % NB
            const int l = x / S::NB, c = x % S::NB;
            const int32_t bp = __shfl_sync(KIV_FULL_MASK, pg, l), br = __shfl_sync(KIV_FULL_MASK, rw, l);
            if (leader)
              tc::tma_load_4d(ring + s * S::TILE + c * (PT_KEYS * S::BOXB) + l * g.br * S::BOXB, map, c * S::BOX, br, kvh, bp, &kv_full[s]);
          }
        }
      }
      tell(true);
      if (me == 0 && lane == 0) {
        if (!cut.head) paged_check_lens(p.pc, at.it.s);
        if (cut.tail) paged_record(p, blockIdx.x, at, cut);
      }
      paged_advance(p, at, cut);
    }
   halted:
    turn = n;
    qturn = items + 1;                         // a query tile not asked for: its wait ends at the limit
   } else if (warp < 11) {
    // ------------------------------------------------ MMA of row tile i
    // The tensor pipe takes few products ahead, so what an issuing warp does
    // between them is lost time; with a warp per row tile, one's waits pass
    // under the other's products.  The whole warp walks the loop and one lane
    // issues, so that descriptors stay in uniform registers.
    const int i = warp - 9;
    constexpr uint32_t id_s = tc::idesc_f16(BF, PT_ROWS, PT_KEYS);
    constexpr uint32_t id_o = tc::idesc_f16(BF, PT_ROWS, D) | (1u << 16);     // B is MN-major
    constexpr uint32_t TILE16 = S::TILE >> 4;
    const uint64_t qd = S::BOX == 64 ? tc::sdesc_k128(smem_u32(qmem)) : tc::sdesc_k64(smem_u32(qmem));
    const uint64_t kd = S::BOX == 64 ? tc::sdesc_k128(smem_u32(ring)) : tc::sdesc_k64(smem_u32(ring));
    const uint64_t vd = tc::sdesc_mn<S::BOXB>(smem_u32(ring), PT_KEYS * S::BOXB);
    const uint32_t ts = tmem + i * PT_KEYS, to = tmem + 2 * PT_KEYS + i * D;
    uint32_t slot = 0, phase = 0;              // of the next K or V tile
    uint32_t tiles = 0;
    const bool leader = elect_one();
    mma = leader;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      if (ok && !mbar_wait_bounded(bar, parity)) ok = false;
    };
    auto bump = [&]() {
      if (++slot == SLOTS) {
        slot = 0;
        phase ^= 1;
      }
    };
    auto scores = [&](uint64_t qa) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = ((uint32_t)(k * 16 / S::BOX) * (PT_ROWS * S::BOXB) + (uint32_t)(k * 16 % S::BOX) * 2) >> 4;
        tc::mma_f16(ts, qa + off, kd + slot * TILE16 + off, id_s, k > 0 ? 1u : 0u);
      }
      tc::commit(&s_full[i]);
      tc::commit(&kv_empty[slot]);
    };
    auto pass = [&]() {                        // a tile that is the other warp's
      wait(&kv_full[slot], phase);
      __syncwarp();
      if (leader) mbar_arrive(&kv_empty[slot]);
      bump();
    };
    for (uint32_t items = 0;; ++items) {
      wait(&q_full, items & 1);
      const int ntile = __shfl_sync(KIV_FULL_MASK, ok ? seg[items & 1].ntile : 0, 0);
      const int nsub = __shfl_sync(KIV_FULL_MASK, seg[items & 1].nsub, 0);
      const bool twin = nsub == 1 && ntile > 1;
      if (ntile == 0) break;
      if (i > 0 && nsub == 1 && !twin) {       // one tile of one row tile: nothing for this warp
        if (leader) mbar_arrive(&q_empty);
        pass();
        pass();
        continue;
      }
      const int step = twin ? 2 : 1, first = twin ? i : 0;
      const uint64_t qa = qd + (twin ? 0u : (uint32_t)i * TILE16);
      if (first > 0) {
        pass();
        pass();
      }
      wait(&kv_full[slot], phase);
      tc::fence_after_sync();
      if (leader) {
        scores(qa);
        if (first + step >= ntile) tc::commit(&q_empty);
      }
      bump();
      for (int t = first; t < ntile; t += step, ++tiles) {
        const bool more = t + step < ntile;
        const uint32_t vs = slot;
        wait(&kv_full[vs], phase);
        bump();
        if (twin && t + 1 < ntile) {
          pass();
          pass();
        }
        if (more) wait(&kv_full[slot], phase);
        const uint64_t b = vd + vs * TILE16;
        const bool fresh = (uint32_t)(t - first) / step % PT_FLUSH == 0;
        wait(&p_full[i], tiles & 1);
        tc::fence_after_sync();
        if (leader) {
#pragma unroll
          for (int k = 0; k < PT_HEAD / 16; ++k) tc::mma_f16_ta(to, ts + k * 8, b + k * S::BOXB, id_o, (!fresh || k > 0) ? 1u : 0u);
        }
        wait(&p_tail[i], tiles & 1);
        tc::fence_after_sync();
        if (leader) {
#pragma unroll
          for (int k = PT_HEAD / 16; k < PT_KEYS / 16; ++k) tc::mma_f16_ta(to, ts + k * 8, b + k * S::BOXB, id_o, 1u);
          if (!more) tc::commit(&o_full[i]);
          if (more) scores(qa);
          tc::commit(&kv_empty[vs]);
          if (more && t + 2 * step >= ntile) tc::commit(&q_empty);
        }
        if (more) bump();
      }
    }
   }
  } else {
    // ------------------------------------------------ softmax of row tile `sub`
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int grp = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + grp * PT_KEYS, to = tmem + lanes + 2 * PT_KEYS + grp * D;
    const bool cap = p.q.softcap > 0.f;
    const float c = (cap ? 1.f : p.q.scaling) * 1.44269504f;              // scores are powers of two of s c
    const int ti = r / p.grp, gi = r - ti * p.grp;
    uint32_t tiles = 0, outs = 0, next = 0, before;   // before: tiles of the block's earlier segments
    for (uint32_t items = 0;; ++items) {
      if (ok && !mbar_wait_bounded(&q_full, items & 1)) ok = false;
      const PtSeg w = seg[items & 1];
      before = next;
      next += w.ntile;
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty);
      // a wait that ran out in one warp ends the loop in all: they share barriers
      uint32_t failed;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 1, 256, q;\n selp.u32 %0, 1, 0, p;\n}\n"
                   : "=r"(failed)
                   : "r"(ok ? 0u : 1u)
                   : "memory");
      if (failed || w.ntile == 0) break;
      const bool twin = w.nsub == 1 && w.ntile > 1;
      if (grp >= w.nsub && !twin) continue;
      const int step = twin ? 2 : 1, first = twin ? grp : 0, sub = twin ? 0 : grp;   // sub: the row tile
      const int tok = sub * g.tps + ti;
      const bool have = ti < g.tps && gi < w.heads && tok < w.tok;
      const int place = p.q.causal ? w.base + tok : 0x7fffffff;
      // key tiles inside [free_lo, free_hi] are seen by every row of this row tile
      const int64_t t0 = (int64_t)w.base + sub * g.tps;
      const int64_t free_hi = p.q.causal ? min((int64_t)w.hi - 1, t0) : (int64_t)w.hi - 1;
      const int64_t free_lo = max((int64_t)w.lo, p.q.window > 0 ? t0 + g.tps - p.q.window : (int64_t)0);
      const bool idle = (warp & 3) * 32 >= min(rows, (w.tok - sub * g.tps) * p.grp);   // a warp without rows keeps the beat
      float m = -INFINITY, l = 0.f;
      // the row that the output moves to (PT_FLUSH), as of reference m_at; a
      // whole item borrows the slot of a later cut one
      const bool row = r < rows;
      float *const acc = paged_part(p, w.part >= 0 ? w.part : 2 * (int)blockIdx.x + 1, twin ? grp * PT_ROWS + r : sub * rows + r);
      bool moved = false;
      float m_at = m;
      for (int t = first; t < w.ntile; t += step, ++tiles) {
        if (ok && !mbar_wait_bounded(&s_full[grp], tiles & 1)) ok = false;
        tc::fence_after_sync();
        const int64_t j0 = w.j00 + (int64_t)t * PT_KEYS;
        if (j0 < w.lo || j0 + PT_KEYS > w.hi) {
          // Dead rows of the V tile: each group clears them for its own
          // product, which waits for p_full below.
          const uint32_t n = 2 * (before + t) + 1, vs = n % SLOTS;
          if (ok && !mbar_wait_bounded(&kv_full[vs], (n / SLOTS) & 1)) ok = false;
          const int dl = (int)max((int64_t)0, w.lo - j0), dh = (int)max((int64_t)0, min((int64_t)PT_KEYS, w.hi - j0));
          if (r < dl || r >= dh) {
#pragma unroll 1
            for (int y = 0; y < D / 8; ++y)
              *reinterpret_cast<uint4 *>(ring + vs * S::TILE + (y / (S::BOX / 8)) * (PT_KEYS * S::BOXB) + r * S::BOXB +
                                         (y % (S::BOX / 8)) * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
        }
        if (idle) {                            // what P holds for these rows stays in their own rows
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&p_full[grp]);
            mbar_arrive(&p_tail[grp]);
          }
          continue;
        }
        uint32_t su[PT_KEYS];
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 32) tc::ld_32x32(ts + x, su + x);
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 32) tc::wait_ld32(su + x);
        if (cap) cap_scores<PT_KEYS>(reinterpret_cast<float *>(su), p.q.softcap, p.q.scaling);
        if (j0 < free_lo || j0 + PT_KEYS - 1 > free_hi) {
          // columns [bot, top] are seen
          const int top = (int)min((int64_t)PT_KEYS, min((int64_t)w.hi - 1, (int64_t)place) - j0);
          const int bot = (int)max((int64_t)0, max((int64_t)w.lo, p.q.window > 0 ? (int64_t)place - p.q.window + 1 : (int64_t)0) - j0);
#pragma unroll
          for (int x = 0; x < PT_KEYS; ++x)
            if (x > top || x < bot) su[x] = 0xff800000u;
        }
        float mx[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) mx[y] = m;
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 16) {
#pragma unroll
          for (int y = 0; y < 8; ++y)
            mx[y] = fmaxf(mx[y], fmaxf(__uint_as_float(su[x + 2 * y]), __uint_as_float(su[x + 2 * y + 1])));
        }
        const float mn = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
        if (t == first) {
          m = mn;
        } else if (__any_sync(KIV_FULL_MASK, (mn - m) * c > PT_LAZY<BF>)) {   // (-inf) - (-inf) is NaN: no growth
          const float f = mn == -INFINITY ? 1.f : ex2((m - mn) * c);
          l *= f;
          m = mn;
#pragma unroll 1
          for (int x = 0; x < D; x += 16) {
            uint32_t o[16];
            tc::ld_32x16(to + x, o);
            tc::wait_ld16(o);
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tc::st_32x16(to + x, o);
          }
        }
        if (t > first && (uint32_t)(t - first) / step % PT_FLUSH == 0) {
          pt_flush<D>(to, acc, !moved ? 0.f : m_at == m ? 1.f : ex2((m_at - m) * c), row);
          moved = true;
          m_at = m;
        }
        const float2 c2 = make_float2(c, c);
        const float neg = pt_shift<BF>(m, c);
        const float2 n2 = make_float2(neg, neg);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            float2 e = __ffma2_rn(make_float2(__uint_as_float(su[x + y]), __uint_as_float(su[x + y + 1])), c2, n2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[(y >> 1) & 1] = __fadd2_rn(sum[(y >> 1) & 1], e);
            pk[y / 2] = pt_pack<BF>(e.x, e.y);
          }
          tc::st_32x16(ts + x / 2, pk);
          if (x + 32 == PT_HEAD) {             // the product of these keys can begin
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[grp]);
          }
        }
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_tail[grp]);
      }
      // ---- the item's rows
      if (ok && !mbar_wait_bounded(&o_full[grp], outs & 1)) ok = false;
      ++outs;
      tc::fence_after_sync();
      // Twins: two groups hold the same rows, over the even and the odd key
      // tiles.  The second leaves maximum and sum in shared memory and its
      // output in TMEM, where the first one's threads reach the same lanes.
      float f0 = 1.f, f1 = 0.f, fa = moved ? (m_at == m ? 1.f : ex2((m_at - m) * c)) : 0.f;
      if (twin) {
        if (grp == 1) {
          s_ml[0][r] = m;
          s_ml[1][r] = l;
          // what has moved once moves whole, as of m
          if (moved && !idle) pt_flush<D>(to, acc, m_at == m ? 1.f : ex2((m_at - m) * c), row);
          tc::fence_before_sync();
          asm volatile("bar.sync 1, 256;" ::: "memory");
          asm volatile("bar.sync 1, 256;" ::: "memory");     // read: the next item may overwrite it
          tc::fence_after_sync();
          continue;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tc::fence_after_sync();
        const float m1 = s_ml[0][r], l1 = s_ml[1][r], top = fmaxf(m, m1);
        f0 = m == -INFINITY ? 0.f : ex2((m - top) * c);
        f1 = m1 == -INFINITY ? 0.f : ex2((m1 - top) * c);
        m = top;
        l = l * f0 + l1 * f1;
      }
      // of the other twin's row, and of what moved before
      const bool moved1 = twin && w.ntile / 2 > PT_FLUSH;
      const float *acc1 = paged_part(p, w.part >= 0 ? w.part : 2 * (int)blockIdx.x + 1, PT_ROWS + r);
      const float mnat = pt_reference<BF>(m, c);
      const bool whole = w.part < 0;
      const float inv = whole ? paged_inv(l) : 1.f;
      f0 *= inv;
      f1 *= inv;
      fa *= f0;
      const int head = w.head0 + gi;
      T *dst = static_cast<T *>(p.q.out) + (w.q0 + tok) * p.q.out_stride_t + head * p.q.out_stride_h;
      float *part = paged_part(p, w.part, sub * rows + r);
      if (!idle) {
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          uint32_t o[32];
          tc::ld_32x32(to + x, o);
          tc::wait_ld32(o);
          float *of = reinterpret_cast<float *>(o);
#pragma unroll
          for (int y = 0; y < 32; ++y) of[y] = f0 == 0.f ? 0.f : of[y] * f0;   // nothing seen: what is there does not count
          if (moved && have && fa != 0.f) {
#pragma unroll
            for (int y = 0; y < 32; ++y) of[y] = fmaf(acc[x + y], fa, of[y]);
          }
          if (twin) {
            uint32_t o1[32];
            tc::ld_32x32(to + D + x, o1);
            tc::wait_ld32(o1);
            if (moved1 && have) {
#pragma unroll
              for (int y = 0; y < 32; ++y) o1[y] = __float_as_uint(acc1[x + y]);
            }
#pragma unroll
            for (int y = 0; y < 32; ++y) of[y] = f1 == 0.f ? of[y] : fmaf(__uint_as_float(o1[y]), f1, of[y]);
          }
          if (!have) continue;
          if (whole) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) st16(dst + x + y, Elem<T>::pack(of + y));
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 4) st16(part + x + y, make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]));
          }
        }
        if (have) {
          if (whole) {
            if (p.q.lse) p.q.lse[(w.q0 + tok) * p.q.num_query_heads + head] = paged_log(mnat, l);
          } else {
            part[D] = mnat;
            part[D + 1] = l;
          }
        }
      }
      if (twin) {
        tc::fence_before_sync();
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      tc::fence_before_sync();                 // the next item's products overwrite the output
    }
  }
  if (!ok) paged_error(p.pc.errors, KIV_ERRBIT_WAIT_TIMEOUT);
  tc::fence_before_sync();
  pt_finish<SLOTS>(ok, kv_full, turn, &q_full, qturn, mma, &halt[warp == 10]);
  tc::fence_after_sync();
  if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ host
bool paged_tc_eligible(const kiv_paged *pc, const kiv_paged_query *q) {
  const int D = pc->head_dim, per = q->num_query_heads / pc->num_kv_heads;
  if (pc->dtype == KIV_DTYPE_F32 || !(D == 64 || D == 96 || D == 128 || D == 256) || pc->page_size % 8 != 0 || per > PT_ROWS) return false;
  if (!(q->scaling > 0.f) || pc->num_pages < 1) return false;   // the row maximum is taken before the scale
  // a dimension that is stepped needs a stride (an expanded one has 0)
  const bool k = (pc->num_pages == 1 || pc->k_stride_p > 0) && (pc->num_kv_heads == 1 || pc->k_stride_h > 0) && pc->k_stride_t > 0;
  const bool v = (pc->num_pages == 1 || pc->v_stride_p > 0) && (pc->num_kv_heads == 1 || pc->v_stride_h > 0) && pc->v_stride_t > 0;
  const bool qs = (pc->num_tokens == 1 || q->stride_t > 0) && (q->num_query_heads == 1 || q->stride_h > 0);
  return k && v && qs && getenv("KIV_DISABLE_TCGEN05") == nullptr;
}

// Tensor maps of the queries (box: `box` elements x the heads of a part x tps
// tokens) and of the pages (`box` elements x br rows of one head and page).
kiv_status pt_maps(const PagedPlan &p, int box, int br, int tps, CUtensorMapSwizzle sw, CUtensorMap *qm, CUtensorMap *km, CUtensorMap *vm) {
  const int D = p.pc.head_dim;
  auto stride = [D](int64_t size, int64_t st) { return (uint64_t)(size == 1 && st <= 0 ? D : st) * 2; };
  {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.q.num_query_heads, (uint64_t)p.pc.num_tokens};
    const uint64_t st[2] = {stride(p.q.num_query_heads, p.q.stride_h), stride(p.pc.num_tokens, p.q.stride_t)};
    const uint32_t b[3] = {(uint32_t)box, (uint32_t)p.grp, (uint32_t)tps};
    KIV_CHECK(encode_tiled(qm, p.pc.dtype, 3, p.q.q, dims, st, b, sw));
  }
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.pc.page_size, (uint64_t)p.pc.num_kv_heads, (uint64_t)p.pc.num_pages};
  const uint32_t b[4] = {(uint32_t)box, (uint32_t)br, 1, 1};
  {
    const uint64_t st[3] = {stride(p.pc.page_size, p.pc.k_stride_t), stride(p.pc.num_kv_heads, p.pc.k_stride_h),
                            stride(p.pc.num_pages, p.pc.k_stride_p)};
    KIV_CHECK(encode_tiled(km, p.pc.dtype, 4, p.pc.k, dims, st, b, sw));
  }
  const uint64_t st[3] = {stride(p.pc.page_size, p.pc.v_stride_t), stride(p.pc.num_kv_heads, p.pc.v_stride_h),
                          stride(p.pc.num_pages, p.pc.v_stride_p)};
  return encode_tiled(vm, p.pc.dtype, 4, p.pc.v, dims, st, b, sw);
}

template <bool BF, int D>
static kiv_status launch_tc(const PagedPlan &p, int blocks, cudaStream_t s) {
  using S = TcShape<D>;
  PagedTcGeom g;
  g.tps = PT_ROWS / p.grp;
  g.br = 8;
  while (g.br < PT_KEYS && p.pc.page_size % (2 * g.br) == 0) g.br *= 2;
  CUtensorMap qm, km, vm;
  KIV_CHECK(pt_maps(p, S::BOX, g.br, g.tps, S::BOX == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, &qm, &km, &vm));
  cudaFuncSetAttribute(paged_tc_kernel<BF, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
  KIV_CHECK(cuda_status(launch_pdl(paged_tc_kernel<BF, D>, dim3((unsigned)blocks), dim3(PT_THREADS), S::SMEM, s, 1, qm, km, vm, p, g),
                        "paged_attend (chunk)"));
  return launch_paged_combine(p, blocks, s);
}

kiv_status launch_paged_tc(const PagedPlan &p, int blocks, cudaStream_t s) {
  const bool bf = p.pc.dtype == KIV_DTYPE_BF16;
  switch (p.pc.head_dim) {
    case 64: return bf ? launch_tc<true, 64>(p, blocks, s) : launch_tc<false, 64>(p, blocks, s);
    case 96: return bf ? launch_tc<true, 96>(p, blocks, s) : launch_tc<false, 96>(p, blocks, s);
    case 256: return launch_paged_tc256(p, blocks, s);
    default: return bf ? launch_tc<true, 128>(p, blocks, s) : launch_tc<false, 128>(p, blocks, s);
  }
}

}  // namespace kiv
