// Paged attention of chunks (many query rows per key head) on tcgen05.
//
//   S = Q K^T and O += P V as 128 x 128 x D and 128 x D x 128 products with
//   fp32 accumulators in TMEM; the softmax in between is one pass with the
//   running maximum and sum of each row in registers.
//
// A block takes items of two row tiles of 128 rows: a row is (token, query
// head of the key head), so the heads of a group share every K and V tile
// (`tps` = 128 / heads whole tokens per tile).  Warp roles:
//   warp 8   TMA: the query tiles, then K and V tiles of 128 keys through a
//            ring, one box of `br` rows per page piece;
//   warp 9   MMA: S_i(j+1) right behind O_i += P_i(j) V(j) for i = 0, 1;
//   warps 0-3 and 4-7: softmax of row tile 0 and 1, a thread per row.
// While one row tile's softmax runs, the tensor cores work on the other's
// products, so both are kept busy: per tile pair the tensor cores need 4 x 512
// cycles (D = 128) and the 2 x 16384 exponentials 2048 cycles of the special
// function units.
//
// P (16-bit) overwrites S in TMEM and is the A operand from there; V is read
// as an MN-major B operand straight from its row-major tile.  The output in
// TMEM is rescaled only when a row's maximum has grown by more than 2^8 since
// the reference it was scaled with (weights up to 256 are as exact as weights
// up to 1: rounding is relative), which after the first tiles is almost never.
//
// Key tiles that hold the end of a sequence (or keys before a window) may hold
// anything in the dead rows, NaN too: scores there are replaced, not added to,
// and the MMA warp clears the dead V rows before the product.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"
#include "tc.cuh"

namespace kiv {

constexpr int PT_KEYS = 128;
constexpr int PT_ROWS = 128;                   // of one row tile
constexpr int PT_THREADS = 320;
constexpr float PT_LAZY = 8.f;                 // growth (log2) that a row's reference may lag behind

struct PagedTcGeom {
  int tps;       // tokens per row tile
  int br;        // rows per TMA box of a page: a power of two dividing page_size, at most 128
};

template <int D>
struct TcShape {
  static constexpr int BOX = D % 64 == 0 ? 64 : 32;      // elements per TMA box: 128- or 64-byte swizzle
  static constexpr int NB = D / BOX;
  static constexpr int BOXB = BOX * 2;                   // bytes of a box row
  static constexpr int TILE = PT_KEYS * D * 2;           // bytes of a K, V or Q tile
  static constexpr int SLOTS = (232448 - 2048 - 2 * TILE) / TILE < 8 ? (232448 - 2048 - 2 * TILE) / TILE : 8;
  static constexpr size_t SMEM = 1024 + 2 * TILE + (size_t)SLOTS * TILE;
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
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
}  // namespace tc

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// Walks the segments of a block's stretch, the same for every warp role.
struct PtWalk {
  PagedSpot at;
  PagedSegment sg;
  int lo, hi;
  int64_t j00;
  int ntile, nsub;
  __device__ __forceinline__ bool live() const { return at.it.s.b >= 0 && at.unit < at.end; }
  __device__ __forceinline__ void open(const PagedPlan &p, int tps) {
    sg = paged_segment(p, at);
    paged_range(p, at.it, at.rt, lo, hi);
    hi = min(hi, at.it.s.len);
    j00 = ((int64_t)lo / PT_KEYS + sg.t0) * PT_KEYS;
    ntile = sg.t1 - sg.t0;
    nsub = at.it.s.n - at.rt * p.tpt > tps ? 2 : 1;
  }
  __device__ __forceinline__ void next(const PagedPlan &p) {
    at.unit += ntile;
    if (sg.tail) {
      at.it.s.b = -1;
      return;
    }
    paged_next(p, at);
  }
};

template <bool BF, int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedPlan p, PagedTcGeom g) {
  using S = TcShape<D>;
  using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
  constexpr int SLOTS = S::SLOTS;
  extern __shared__ uint8_t pt_dyn[];
  __shared__ uint64_t q_full, q_empty, kv_full[SLOTS], kv_empty[SLOTS], s_full[2], p_full[2], o_full[2];
  __shared__ int64_t sm[40];
  __shared__ uint32_t s_tmem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t *smem = pt_dyn + ((1024 - (smem_u32(pt_dyn) & 1023)) & 1023);
  uint8_t *qmem = smem, *ring = smem + 2 * S::TILE;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
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
  PtWalk w;
  w.at = paged_locate<PT_THREADS>(p, sm);
  if (threadIdx.x == 0) p.cut[blockIdx.x].b = -1;
  bool ok = true;
  const int rows = g.tps * p.grp;              // of a row tile
  const int per = p.q.num_query_heads / p.pc.num_kv_heads;

  if (warp == 8) {
    // ------------------------------------------------ TMA
    uint32_t n = 0, items = 0;
    for (; w.live(); w.next(p), ++items) {
      w.open(p, g.tps);
      const int kvh = w.at.hp / p.hs, head0 = kvh * per + (w.at.hp % p.hs) * p.grp;
      if (lane == 0) {
        if (!w.sg.head) paged_check_lens(p.pc, w.at.it.s);
        if (w.sg.tail) paged_record(p, blockIdx.x, w.at, w.sg);
        if (items > 0 && ok && !mbar_wait_bounded(&q_empty, (items - 1) & 1)) ok = false;
        mbar_arrive_tx(&q_full, (uint32_t)w.nsub * rows * D * 2);
        for (int i = 0; i < w.nsub; ++i)
          for (int c = 0; c < S::NB; ++c)
            tc::tma_load_3d(qmem + i * S::TILE + c * (PT_ROWS * S::BOXB), &qmap, c * S::BOX, head0,
                            (int32_t)(w.at.it.s.q0 + (int64_t)w.at.rt * p.tpt + i * g.tps), &q_full);
      }
      __syncwarp();
      // lane l brings rows [l br, (l + 1) br) of every tile
      const int nbox = PT_KEYS / g.br;
      const int32_t *table = p.pc.block_table + w.at.it.s.b * p.pc.table_stride;
      auto lookup = [&](int t, int32_t &page, int32_t &row) {
        page = -1;                             // outside: the box reads as zeros
        row = 0;
        const int64_t j = w.j00 + (int64_t)t * PT_KEYS + lane * g.br;
        if (t < w.ntile && lane < nbox && j < w.hi && j + g.br > w.lo) {
          const uint32_t pg = (uint32_t)j / (uint32_t)p.pc.page_size;
          row = (int32_t)((uint32_t)j - pg * (uint32_t)p.pc.page_size);
          page = table[pg];
          if (page < 0 || page >= p.pc.num_pages) {
            paged_error(p.pc.errors, KIV_ERRBIT_BLOCK_TABLE);
            page = -1;
          }
        }
      };
      int32_t page, row;
      lookup(0, page, row);
      for (int t = 0; t < w.ntile; ++t) {
        const int32_t pg = page, rw = row;
        lookup(t + 1, page, row);
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t s = n % SLOTS;
          if (n >= SLOTS && ok && !mbar_wait_bounded(&kv_empty[s], (n / SLOTS - 1) & 1)) ok = false;
          if (lane == 0) mbar_arrive_tx(&kv_full[s], S::TILE);
          __syncwarp();
          if (lane < nbox)
            for (int c = 0; c < S::NB; ++c)
              tc::tma_load_4d(ring + s * S::TILE + c * (PT_KEYS * S::BOXB) + lane * g.br * S::BOXB, kv ? &vmap : &kmap, c * S::BOX,
                              rw, kvh, pg, &kv_full[s]);
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------ MMA
    const uint32_t id_s = tc::idesc_f16(BF, PT_ROWS, PT_KEYS);
    const uint32_t id_o = tc::idesc_f16(BF, PT_ROWS, D) | (1u << 16);     // B is MN-major
    uint32_t n = 0, items = 0, tiles[2] = {0, 0};
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      if (ok && !mbar_wait_bounded(bar, parity)) ok = false;
      tc::fence_after_sync();
    };
    auto scores = [&](int i, uint32_t slot) {
      if (lane != 0) return;
      const uint32_t a0 = smem_u32(qmem + i * S::TILE), b0 = smem_u32(ring + slot * S::TILE);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (uint32_t)(k * 16 / S::BOX) * (PT_ROWS * S::BOXB) + (uint32_t)(k * 16 % S::BOX) * 2;
        const uint64_t ad = S::BOX == 64 ? tc::sdesc_k128(a0 + off) : tc::sdesc_k64(a0 + off);
        const uint64_t bd = S::BOX == 64 ? tc::sdesc_k128(b0 + off) : tc::sdesc_k64(b0 + off);
        tc::mma_f16(tmem + i * PT_KEYS, ad, bd, id_s, k > 0 ? 1u : 0u);
      }
      tc::commit(&s_full[i]);
    };
    for (; w.live(); w.next(p), ++items) {
      w.open(p, g.tps);
      wait(&q_full, items & 1);
      wait(&kv_full[n % SLOTS], (n / SLOTS) & 1);
      for (int i = 0; i < w.nsub; ++i) scores(i, n % SLOTS);
      if (lane == 0) {
        tc::commit(&kv_empty[n % SLOTS]);
        if (w.ntile == 1) tc::commit(&q_empty);
      }
      for (int t = 0; t < w.ntile; ++t, n += 2) {
        const uint32_t vs = (n + 1) % SLOTS, ks = (n + 2) % SLOTS;
        wait(&kv_full[vs], ((n + 1) / SLOTS) & 1);
        // dead rows of the V tile
        const int64_t j0 = w.j00 + (int64_t)t * PT_KEYS;
        const int dl = (int)max((int64_t)0, w.lo - j0), dh = (int)min((int64_t)PT_KEYS, w.hi - j0);
        if (dl > 0 || dh < PT_KEYS) {
          for (int x = lane; x < PT_KEYS * S::NB * (S::BOXB / 16); x += 32) {
            const int r = x / (S::NB * (S::BOXB / 16)), c = x % (S::NB * (S::BOXB / 16));
            if (r < dl || r >= dh)
              *reinterpret_cast<uint4 *>(ring + vs * S::TILE + (c / (S::BOXB / 16)) * (PT_KEYS * S::BOXB) + r * S::BOXB +
                                         (c % (S::BOXB / 16)) * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
        }
        const bool more = t + 1 < w.ntile;
        for (int i = 0; i < w.nsub; ++i) {
          wait(&p_full[i], tiles[i] & 1);
          ++tiles[i];
          if (lane == 0) {
            const uint32_t b0 = smem_u32(ring + vs * S::TILE);
#pragma unroll
            for (int k = 0; k < PT_KEYS / 16; ++k)
              tc::mma_f16_ta(tmem + 2 * PT_KEYS + i * D, tmem + i * PT_KEYS + k * 8,
                             tc::sdesc_mn<S::BOXB>(b0 + k * 16 * S::BOXB, PT_KEYS * S::BOXB), id_o, (t > 0 || k > 0) ? 1u : 0u);
            if (!more) tc::commit(&o_full[i]);
            if (i == w.nsub - 1) tc::commit(&kv_empty[vs]);
          }
          if (more) {
            if (i == 0) wait(&kv_full[ks], ((n + 2) / SLOTS) & 1);
            scores(i, ks);
            if (i == w.nsub - 1 && lane == 0) {
              tc::commit(&kv_empty[ks]);
              if (t + 2 == w.ntile) tc::commit(&q_empty);
            }
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------ softmax of row tile `sub`
    const int sub = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + sub * PT_KEYS, to = tmem + lanes + 2 * PT_KEYS + sub * D;
    const bool cap = p.q.softcap > 0.f;
    const float c = (cap ? 1.f : p.q.scaling) * 1.44269504f;              // scores are powers of two of s c
    const float cap_in = cap ? 2.f * 1.44269504f * p.q.scaling / p.q.softcap : 0.f;
    uint32_t tiles = 0, items = 0;
    for (; w.live(); w.next(p)) {
      w.open(p, g.tps);
      if (sub >= w.nsub) continue;
      int i, head;
      const bool have = paged_row(p, w.at.it, w.at.hp, w.at.rt, sub * rows + r, i, head) && r < rows;
      const int place = p.q.causal ? w.at.it.base + i : 0x7fffffff;
      // key tiles inside [free_lo, free_hi] are seen by every row of this row tile
      const int64_t t0 = (int64_t)w.at.rt * p.tpt + sub * g.tps;
      const int64_t free_hi = p.q.causal ? min((int64_t)w.hi - 1, (int64_t)w.at.it.base + t0) : (int64_t)w.hi - 1;
      const int64_t free_lo = max((int64_t)w.lo, p.q.window > 0 ? (int64_t)w.at.it.base + t0 + g.tps - p.q.window : (int64_t)0);
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < w.ntile; ++t, ++tiles) {
        if (ok && !mbar_wait_bounded(&s_full[sub], tiles & 1)) ok = false;
        tc::fence_after_sync();
        // The scores are read twice, 32 columns at a time (the second time as
        // exponents): a row of 128 does not fit the registers next to the rest.
        uint32_t buf[2][32];
        const int64_t j0 = w.j00 + (int64_t)t * PT_KEYS;
        const bool masked = j0 < free_lo || j0 + PT_KEYS - 1 > free_hi;
        // columns [bot, top] are seen
        const int top = (int)min((int64_t)PT_KEYS, min((int64_t)w.hi - 1, (int64_t)place) - j0);
        const int bot = (int)max((int64_t)0, max((int64_t)w.lo, p.q.window > 0 ? (int64_t)place - p.q.window + 1 : (int64_t)0) - j0);
        float mx[4] = {m, m, m, m};
        tc::ld_32x32(ts, buf[0]);
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 32) {
          uint32_t *su = buf[(x / 32) & 1];
          tc::wait_ld32(su);
          if (x + 32 < PT_KEYS) tc::ld_32x32(ts + x + 32, buf[(x / 32 + 1) & 1]);
          if (masked || cap) {                 // put the score itself back
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              float v = __uint_as_float(su[y]);
              if (cap) v = p.q.softcap * (1.f - __fdividef(2.f, 1.f + ex2(v * cap_in)));
              if (x + y > top || x + y < bot) v = -INFINITY;
              su[y] = __float_as_uint(v);
            }
            tc::st_32x32(ts + x, su);
          }
#pragma unroll
          for (int y = 0; y < 32; y += 8) {
#pragma unroll
            for (int z = 0; z < 4; ++z)
              mx[z] = fmaxf(mx[z], fmaxf(__uint_as_float(su[y + 2 * z]), __uint_as_float(su[y + 2 * z + 1])));
          }
        }
        if (masked || cap) tc::wait_st();
        tc::ld_32x32(ts, buf[0]);
        const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (t == 0) {
          m = mn;
        } else if (__any_sync(KIV_FULL_MASK, (mn - m) * c > PT_LAZY)) {   // (-inf) - (-inf) is NaN: no growth
          const float f = mn == -INFINITY ? 1.f : ex2((m - mn) * c);
          l *= f;
          m = mn;
#pragma unroll 1
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tc::ld_32x32(to + x, o);
            tc::wait_ld32(o);
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tc::st_32x32(to + x, o);
          }
        }
        const float2 c2 = make_float2(c, c);
        const float neg = m == -INFINITY ? 0.f : -m * c;
        const float2 n2 = make_float2(neg, neg);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int x = 0; x < PT_KEYS; x += 32) {
          uint32_t *su = buf[(x / 32) & 1];
          tc::wait_ld32(su);
          if (x + 32 < PT_KEYS) tc::ld_32x32(ts + x + 32, buf[(x / 32 + 1) & 1]);
          uint32_t pk[16];
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            float2 e = __ffma2_rn(make_float2(__uint_as_float(su[y]), __uint_as_float(su[y + 1])), c2, n2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[(y >> 1) & 1] = __fadd2_rn(sum[(y >> 1) & 1], e);
            pk[y / 2] = pt_pack<BF>(e.x, e.y);
          }
          tc::st_32x16(ts + x / 2, pk);        // over columns that were read before
        }
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[sub]);
      }
      // ---- the item's rows
      if (ok && !mbar_wait_bounded(&o_full[sub], items & 1)) ok = false;
      ++items;
      tc::fence_after_sync();
      const float mnat = m * c * 0.693147181f;
      const bool whole = !w.sg.head && !w.sg.tail;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      T *dst = have && whole ? paged_out<T>(p, w.at.it, i, head) : nullptr;
      float *part = paged_part(p, 2 * (int64_t)blockIdx.x + (w.sg.head ? 0 : 1), sub * rows + r);
#pragma unroll
      for (int x = 0; x < D; x += 32) {
        uint32_t o[32];
        tc::ld_32x32(to + x, o);
        tc::wait_ld32(o);
        if (!have) continue;
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
      if (have) {
        if (whole) {
          paged_lse(p, w.at.it, i, head, mnat, l);
        } else {
          part[D] = mnat;
          part[D + 1] = l;
        }
      }
      tc::fence_before_sync();                 // the next item's products overwrite the output
    }
  }
  if (!ok) paged_error(p.pc.errors, KIV_ERRBIT_WAIT_TIMEOUT);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ host
bool paged_tc_eligible(const kiv_paged *pc, const kiv_paged_query *q) {
  const int D = pc->head_dim, per = q->num_query_heads / pc->num_kv_heads;
  if (pc->dtype == KIV_DTYPE_F32 || !(D == 64 || D == 96 || D == 128) || pc->page_size % 8 != 0 || per > PT_ROWS) return false;
  if (!(q->scaling > 0.f) || pc->num_pages < 1) return false;   // the row maximum is taken before the scale
  // a dimension that is stepped needs a stride (an expanded one has 0)
  const bool k = (pc->num_pages == 1 || pc->k_stride_p > 0) && (pc->num_kv_heads == 1 || pc->k_stride_h > 0) && pc->k_stride_t > 0;
  const bool v = (pc->num_pages == 1 || pc->v_stride_p > 0) && (pc->num_kv_heads == 1 || pc->v_stride_h > 0) && pc->v_stride_t > 0;
  const bool qs = (pc->num_tokens == 1 || q->stride_t > 0) && (q->num_query_heads == 1 || q->stride_h > 0);
  return k && v && qs && getenv("KIV_DISABLE_TCGEN05") == nullptr;
}

template <bool BF, int D>
static kiv_status launch_tc(const PagedPlan &p, int blocks, cudaStream_t s) {
  using S = TcShape<D>;
  PagedTcGeom g;
  g.tps = PT_ROWS / p.grp;
  g.br = 8;
  while (g.br < PT_KEYS && p.pc.page_size % (2 * g.br) == 0) g.br *= 2;
  const CUtensorMapSwizzle sw = S::BOX == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap qm, km, vm;
  auto stride = [](int64_t size, int64_t st) { return (uint64_t)(size == 1 && st <= 0 ? D : st) * 2; };
  {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.q.num_query_heads, (uint64_t)p.pc.num_tokens};
    const uint64_t st[2] = {stride(p.q.num_query_heads, p.q.stride_h), stride(p.pc.num_tokens, p.q.stride_t)};
    const uint32_t box[3] = {S::BOX, (uint32_t)p.grp, (uint32_t)g.tps};
    KIV_CHECK(encode_tiled(&qm, p.pc.dtype, 3, p.q.q, dims, st, box, sw));
  }
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.pc.page_size, (uint64_t)p.pc.num_kv_heads, (uint64_t)p.pc.num_pages};
  const uint32_t box[4] = {S::BOX, (uint32_t)g.br, 1, 1};
  {
    const uint64_t st[3] = {stride(p.pc.page_size, p.pc.k_stride_t), stride(p.pc.num_kv_heads, p.pc.k_stride_h),
                            stride(p.pc.num_pages, p.pc.k_stride_p)};
    KIV_CHECK(encode_tiled(&km, p.pc.dtype, 4, p.pc.k, dims, st, box, sw));
  }
  {
    const uint64_t st[3] = {stride(p.pc.page_size, p.pc.v_stride_t), stride(p.pc.num_kv_heads, p.pc.v_stride_h),
                            stride(p.pc.num_pages, p.pc.v_stride_p)};
    KIV_CHECK(encode_tiled(&vm, p.pc.dtype, 4, p.pc.v, dims, st, box, sw));
  }
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
    default: return bf ? launch_tc<true, 128>(p, blocks, s) : launch_tc<false, 128>(p, blocks, s);
  }
}

}  // namespace kiv
