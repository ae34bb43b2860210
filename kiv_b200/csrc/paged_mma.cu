// Paged attention of 16-bit rows with warp-level tensor-core MMAs, for what the
// tcgen05 kernels do not take (plan_call in paged.cu): pages whose size is no
// multiple of 8, head dimensions 80 and 192, large groups, expanded strides.
// 32 sequences of 16 k keys, one token each, 32/8: x 80 390-440 us (3.0-3.4 TB/s),
// x 192 1.0 ms, x 128 in pages of 10 484 us (4.4 TB/s).
//
// Made for few query rows: with r of them a key head's K and V rows carry 2 r
// FLOP per byte, and HBM is the limit.  A block streams tiles of 64 keys through
// a ring of shared memory, one bulk copy per row (any page size, any row stride): each of the
// 128 threads brings one K or V row of every tile, whose page number it read a
// step before.  With 16-byte cp.async instead, the address arithmetic alone
// was a third of the instructions and the kernel issue-bound at 2.4 TB/s, where
// this reaches 4.9 (64 sequences of up to 32 k keys, 32/8 x 128).  The blocks
// share the batch's tiles evenly (paged.cuh).
//
// WM x WN = 4 warps: WM groups of 16 query rows, WN groups of keys.  Each warp
// runs its own softmax over its keys (maximum, sum and output in registers);
// the WN parts of a row meet in shared memory at the end of an item.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"

namespace kiv {

constexpr int MM_KEYS = 64;
constexpr int MM_THREADS = 128;

template <int D, int ROWS>
struct MmaShape {
  static constexpr int LD = D * 2 + 16;                    // bytes per row: 16 B of padding spread ldmatrix over the banks
  static constexpr int STAGE = 2 * MM_KEYS * LD;           // K and V tile
  // as many blocks per SM as registers allow, each with its next tile on the
  // way: latency x bandwidth asks for some 45 KB in flight per SM
  static constexpr int STAGES = D <= 128 ? 2 : (D == 256 && ROWS == 64 ? 2 : 3);
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + (size_t)ROWS * LD;
  // 228 KB per SM, 1 KB of each block reserved, half a KB static; 170 or 255
  // registers a thread
  static constexpr int FIT = (int)(233472 / (SMEM + 1536)), REGS = ROWS == 16 && D <= 192 ? 3 : 2;
  static constexpr int BLOCKS = FIT < REGS ? FIT : REGS;
};

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
template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
// what the rounding in pack2 lost
template <bool BF>
__device__ __forceinline__ uint32_t pack2_rest(float x, float y, uint32_t p) {
  float a, b;
  if constexpr (BF) {
    a = __uint_as_float(p << 16);
    b = __uint_as_float(p & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p));
    a = f.x;
    b = f.y;
  }
  return pack2<BF>(x - a, y - b);
}

template <bool BF, int D, int WM>
__global__ void __launch_bounds__(MM_THREADS, MmaShape<D, 16 * WM>::BLOCKS) paged_mma_kernel(const __grid_constant__ PagedPlan p) {
  using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
  constexpr int WN = 4 / WM, ROWS = 16 * WM;
  using S = MmaShape<D, ROWS>;
  constexpr int NK = MM_KEYS / WN;             // keys per warp and tile
  constexpr int CH = D / 8;                    // 16-byte chunks per row
  constexpr int STAGES = S::STAGES;
  // The probabilities keep their type's bits twice, in a second product: their
  // rounding would be the largest error of the result.  With 16 rows (bound by
  // memory) it is free; with 64 rows it takes 4 to 19 % (2048 tokens over 16384,
  // 32/8 x 80: 2.91 ms from 2.79; x 192: 7.7 from 6.8).  All row counts do it, as
  // a call's tiling goes by what the host knows of the lengths, and that must not
  // decide how exact a row is.
  // fp16 weights are subnormal below 2^-14 and vanish below 2^-25 of the row's
  // largest; 2^15 of them and of their sum keep those down to 2^-29 whole
  constexpr float BIAS = BF ? 0.f : 15.f;
  constexpr bool QREG = D <= 128;              // query fragments stay in registers
  extern __shared__ __align__(128) uint8_t mm_dyn[];
  __shared__ uint64_t full[STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wm = warp % WM, wn = warp / WM;
  const int g = lane >> 2, tq = lane & 3;
  const uint32_t ring = smem_u32(mm_dyn), sq = ring + STAGES * S::STAGE;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], MM_THREADS);
    mbar_fence_init();
  }
  griddep_wait();
  PagedSpot at = paged_locate(p);              // every warp for itself
  if (threadIdx.x == 0) p.cut[blockIdx.x].b = -1;
  const float scale = p.q.scaling;
  // this thread's row of every tile
  const bool isv = threadIdx.x >= MM_KEYS;
  const int myrow = threadIdx.x % MM_KEYS;
  const T *base = static_cast<const T *>(isv ? p.pc.v : p.pc.k);
  const int64_t sp = isv ? p.pc.v_stride_p : p.pc.k_stride_p, sh = isv ? p.pc.v_stride_h : p.pc.k_stride_h,
                st = isv ? p.pc.v_stride_t : p.pc.k_stride_t;
  uint8_t *const mydst = mm_dyn + threadIdx.x * S::LD;
  uint32_t used = 0;                           // tiles that went through the ring so far
  bool ok = true;

  while (at.it.s.b >= 0 && at.unit < at.end) {
    const PagedSegment sg = paged_segment(p, at);
    const int kvh = at.hp / p.hs;
    int lo, hi;
    paged_range(p, at.it, at.rt, lo, hi);
    if (threadIdx.x == 0) {
      if (!sg.head) paged_check_lens(p.pc, at.it.s);
      if (sg.tail) paged_record(p, blockIdx.x, at, sg);
    }
    hi = min(hi, at.it.s.len);
    const int64_t j00 = ((int64_t)lo / MM_KEYS + sg.t0) * MM_KEYS;   // first key of the segment's first tile
    const int ntile = sg.t1 - sg.t0;

    const int32_t *table = p.pc.block_table + at.it.s.b * p.pc.table_stride;
    const int lo_t = (int)max((int64_t)0, lo - j00), hi_t = (int)(hi - j00);   // live keys, counted from j00
    // where this thread's row of tile t lies: page (-2: not a live key) and row
    auto lookup = [&](int t, int32_t &page, int32_t &row) {
      const int x = t * MM_KEYS + myrow;
      page = -2;
      row = 0;
      if (t < ntile && x >= lo_t && x < hi_t) {
        const uint32_t j = (uint32_t)(j00 + x), pg = j / (uint32_t)p.pc.page_size;
        row = (int32_t)(j - pg * (uint32_t)p.pc.page_size);
        page = table[pg];
      }
    };
    auto load_row = [&](int t, int32_t page, int32_t row) {
      if (t >= ntile) return;
      const uint32_t n = used + t;
      uint8_t *dst = mydst + (n % STAGES) * S::STAGE;
      uint64_t *bar = &full[n % STAGES];
      if (page >= 0 && page < p.pc.num_pages) {
        mbar_arrive_tx(bar, D * 2);
        bulk_g2s(dst, base + page * sp + kvh * sh + row * st, D * 2, bar);
      } else {                                 // reads as zeros
        if (page != -2) paged_error(p.pc.errors, KIV_ERRBIT_BLOCK_TABLE);
        for (int c = 0; c < CH; ++c) *reinterpret_cast<uint4 *>(dst + c * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // a later bulk copy writes here again
        mbar_arrive(bar);
      }
    };

    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();                           // the previous item is done with the ring
    int32_t page, row;
    for (int t = 0; t < STAGES - 1; ++t) {
      lookup(t, page, row);
      load_row(t, page, row);
    }
    lookup(STAGES - 1, page, row);
    for (int x = threadIdx.x; x < ROWS * CH; x += MM_THREADS) {
      const int r = x / CH, c = x - r * CH;
      int i, head;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (paged_row(p, at.it, at.hp, at.rt, r, i, head))
        v = ld16(static_cast<const T *>(p.q.q) + (at.it.s.q0 + i) * p.q.stride_t + head * p.q.stride_h + c * 8);
      *reinterpret_cast<uint4 *>(mm_dyn + STAGES * S::STAGE + r * S::LD + c * 16) = v;
    }
    __syncthreads();

    uint32_t qf[QREG ? D / 16 : 1][4];
    const uint32_t qaddr = sq + (wm * 16 + (lane & 15)) * S::LD + (lane >> 4) * 16;
    if (QREG) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) ldsm4(qf[QREG ? k : 0], qaddr + k * 32);
    }
    // this lane's rows: wm * 16 + g and + 8
    int place[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      int i, head;
      paged_row(p, at.it, at.hp, at.rt, wm * 16 + g + 8 * a, i, head);
      place[a] = p.q.causal ? at.it.base + i : 0x7fffffff;
    }
    // every key of a tile in [free_lo, free_hi] is seen by every row of the item's tile
    const int64_t free_hi = p.q.causal ? min((int64_t)hi - 1, (int64_t)at.it.base + (int64_t)at.rt * p.tpt) : (int64_t)hi - 1;
    const int64_t free_lo = p.q.window > 0 ? (int64_t)at.it.base + (int64_t)(at.rt + 1) * p.tpt - p.q.window : (int64_t)0;

    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;

    for (int t = 0; t < ntile; ++t) {
      if (t > 0) __syncthreads();              // tile t - 1 is read: its stage is free
      load_row(t + STAGES - 1, page, row);
      lookup(t + STAGES, page, row);           // the table entry arrives while the MMAs run
      const uint32_t n = used + t;
      if (ok && !mbar_wait_bounded(&full[n % STAGES], (n / STAGES) & 1)) ok = false;
      const uint32_t kt = ring + (n % STAGES) * S::STAGE, vt = kt + MM_KEYS * S::LD;
      float s[NK / 8][4];
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
      const uint32_t kaddr = kt + (wn * NK + ((lane >> 4) << 3) + (lane & 7)) * S::LD + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if (!QREG) ldsm4(qf[0], qaddr + k * 32);
#pragma unroll
        for (int n = 0; n < NK / 16; ++n) {
          uint32_t b[4];
          ldsm4(b, kaddr + n * 16 * S::LD + k * 32);
          mma16816<BF>(s[2 * n], qf[QREG ? k : 0], b[0], b[1]);
          mma16816<BF>(s[2 * n + 1], qf[QREG ? k : 0], b[2], b[3]);
        }
      }
      const int64_t j0 = j00 + (int64_t)t * MM_KEYS;
      const bool open = j0 >= free_lo && j0 + MM_KEYS - 1 <= free_hi;
      const bool cap = p.q.softcap > 0.f;
      if (cap) cap_scores<NK / 2>(&s[0][0], p.q.softcap, scale);
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < NK / 8; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = cap ? s[n][e] : s[n][e] * scale;
          if (!open) {
            const int64_t j = j0 + wn * NK + n * 8 + 2 * tq + (e & 1);
            const int pl = place[e >> 1];
            if (j >= hi || j > pl || (p.q.window > 0 && j <= (int64_t)pl - p.q.window)) x = -INFINITY;
          }
          s[n][e] = x;
          mx[e >> 1] = fmaxf(mx[e >> 1], x);
        }
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        mx[a] = fmaxf(mx[a], __shfl_xor_sync(KIV_FULL_MASK, mx[a], 1));
        mx[a] = fmaxf(mx[a], __shfl_xor_sync(KIV_FULL_MASK, mx[a], 2));
      }
      if (mx[0] != m[0] || mx[1] != m[1]) {
        float keep[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          keep[a] = mx[a] == -INFINITY ? 1.f : ex2((m[a] - mx[a]) * 1.44269504f);
          l[a] *= keep[a];
          m[a] = mx[a];
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][0] *= keep[0];
          o[d][1] *= keep[0];
          o[d][2] *= keep[1];
          o[d][3] *= keep[1];
        }
      }
      float shift[2];                          // fp16: rounded down, so that no weight passes 2^15
#pragma unroll
      for (int a = 0; a < 2; ++a)
        shift[a] = m[a] == -INFINITY ? 0.f : BF ? -m[a] * 1.44269504f : __fmaf_rd(-m[a], 1.44269504f, BIAS);
      // a tile's weights first: one at a time, like ones would round the long sum
      // the same way each time, and small ones not reach it at all
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = ex2(fmaf(s[n][e], 1.44269504f, shift[e >> 1]));
          sum[e >> 1] += s[n][e];
        }
      l[0] += sum[0];
      l[1] += sum[1];
      const uint32_t vaddr = vt + (wn * NK + (lane & 15)) * S::LD + (lane >> 4) * 16;
      uint32_t a[NK / 16][4], ar[NK / 16][4];
#pragma unroll
      for (int c = 0; c < NK / 16; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[2 * c + (e >> 1)][2 * (e & 1)], y = s[2 * c + (e >> 1)][2 * (e & 1) + 1];
          a[c][e] = pack2<BF>(x, y);
          ar[c][e] = pack2_rest<BF>(x, y, a[c][e]);
        }
      }
      // The MMAs' accumulation cuts instead of rounding and would drift over
      // many keys: they sum one tile, an ordinary addition the tiles.
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        float part[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) part[0][e] = part[1][e] = 0.f;
#pragma unroll
        for (int c = 0; c < NK / 16; ++c) {
          uint32_t b[4];
          ldsm4t(b, vaddr + c * 16 * S::LD + d * 32);
          mma16816<BF>(part[0], ar[c], b[0], b[1]);
          mma16816<BF>(part[1], ar[c], b[2], b[3]);
          mma16816<BF>(part[0], a[c], b[0], b[1]);
          mma16816<BF>(part[1], a[c], b[2], b[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[2 * d][e] += part[0][e];
          o[2 * d + 1][e] += part[1][e];
        }
      }
    }
    used += ntile;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      l[a] += __shfl_xor_sync(KIV_FULL_MASK, l[a], 1);
      l[a] += __shfl_xor_sync(KIV_FULL_MASK, l[a], 2);
    }
    // ---- the warps' parts of a row meet in shared memory: [WN][ROWS][D + 4]
    __syncthreads();                           // the ring is free
    float *sx = reinterpret_cast<float *>(mm_dyn);
    constexpr int XLD = D + 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      float *row = sx + (wn * ROWS + wm * 16 + g + 8 * a) * XLD;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2 *>(row + d * 8 + 2 * tq) = make_float2(o[d][2 * a], o[d][2 * a + 1]);
      if (tq == 0) {
        row[D] = m[a] - BIAS * 0.693147181f;   // what the weights count in
        row[D + 1] = l[a];
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < ROWS * (D / 8); x += MM_THREADS) {
      const int r = x / (D / 8), c = (x - r * (D / 8)) * 8;
      int i, head;
      if (!paged_row(p, at.it, at.hp, at.rt, r, i, head)) continue;
      float mm = -INFINITY, ll = 0.f, acc[8];
#pragma unroll
      for (int w = 0; w < WN; ++w) mm = fmaxf(mm, sx[(w * ROWS + r) * XLD + D]);
      const float ms = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < WN; ++w) {
        const float *row = sx + (w * ROWS + r) * XLD;
        const float f = ex2((row[D] - ms) * 1.44269504f);
        ll = fmaf(row[D + 1], f, ll);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(row[c + e], f, acc[e]);
      }
      if (!sg.head && !sg.tail) {
        const float inv = paged_inv(ll);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= inv;
        st16(paged_out<T>(p, at.it, i, head) + c, Elem<T>::pack(acc));
        if (c == 0) paged_lse(p, at.it, i, head, mm, ll);
      } else {
        float *dst = paged_part(p, 2 * (int64_t)blockIdx.x + (sg.head ? 0 : 1), r);
        *reinterpret_cast<float4 *>(dst + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *reinterpret_cast<float4 *>(dst + c + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (c == 0) {
          dst[D] = mm;
          dst[D + 1] = ll;
        }
      }
    }
    paged_advance(p, at, sg);
  }
  if (!ok) {
    paged_error(p.pc.errors, KIV_ERRBIT_WAIT_TIMEOUT);
    paged_linger();
  }
}

// ------------------------------------------------------------------ host
template <int D>
static int mma_blocks_per_sm(int rows) {
  return rows == 16 ? MmaShape<D, 16>::BLOCKS : rows == 32 ? MmaShape<D, 32>::BLOCKS : MmaShape<D, 64>::BLOCKS;
}

bool paged_mma_head(int dtype, int D) {
  return dtype != KIV_DTYPE_F32 && (D == 64 || D == 80 || D == 96 || D == 128 || D == 192 || D == 256);
}

int paged_mma_blocks(int D, int rows) {
  switch (D) {
    case 64: return sm_count() * mma_blocks_per_sm<64>(rows);
    case 80: return sm_count() * mma_blocks_per_sm<80>(rows);
    case 96: return sm_count() * mma_blocks_per_sm<96>(rows);
    case 128: return sm_count() * mma_blocks_per_sm<128>(rows);
    case 192: return sm_count() * mma_blocks_per_sm<192>(rows);
    default: return sm_count() * mma_blocks_per_sm<256>(rows);
  }
}

template <bool BF, int D, int WM>
static cudaError_t launch_mma(const PagedPlan &p, int blocks, cudaStream_t s) {
  constexpr size_t smem = MmaShape<D, 16 * WM>::SMEM;
  cudaFuncSetAttribute(paged_mma_kernel<BF, D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return launch_pdl(paged_mma_kernel<BF, D, WM>, dim3((unsigned)blocks), dim3(MM_THREADS), smem, s, 1, p);
}
template <bool BF, int D>
static cudaError_t launch_mma_w(const PagedPlan &p, int blocks, cudaStream_t s) {
  if (p.rows == 16) return launch_mma<BF, D, 1>(p, blocks, s);
  if (p.rows == 32) return launch_mma<BF, D, 2>(p, blocks, s);
  return launch_mma<BF, D, 4>(p, blocks, s);
}
template <bool BF>
static cudaError_t launch_mma_d(const PagedPlan &p, int blocks, cudaStream_t s) {
  switch (p.pc.head_dim) {
    case 64: return launch_mma_w<BF, 64>(p, blocks, s);
    case 80: return launch_mma_w<BF, 80>(p, blocks, s);
    case 96: return launch_mma_w<BF, 96>(p, blocks, s);
    case 128: return launch_mma_w<BF, 128>(p, blocks, s);
    case 192: return launch_mma_w<BF, 192>(p, blocks, s);
    default: return launch_mma_w<BF, 256>(p, blocks, s);
  }
}

kiv_status launch_paged_mma(const PagedPlan &p, int blocks, cudaStream_t s) {
  const cudaError_t e = p.pc.dtype == KIV_DTYPE_BF16 ? launch_mma_d<true>(p, blocks, s) : launch_mma_d<false>(p, blocks, s);
  KIV_CHECK(cuda_status(e, "paged_attend"));
  return launch_paged_combine(p, blocks, s);
}

}  // namespace kiv
