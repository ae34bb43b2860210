// Paged attention of fp32 rows with warp-level tensor-core MMAs.
//
// TF32 products alone would leave 11 bits of the rows.  So every operand x is
// split in two, hi = x rounded to TF32 and lo = (x - hi) rounded to TF32, and
// a product is hi hi + hi lo + lo hi, accumulated in fp32: what is dropped is
// 2^-22 of each product, as small as the fp32 sums' own rounding.  Three
// m16n8k8 MMAs stand against CUDA-core FMAs that needed 16 bytes of shared
// memory for every 8 of them (paged.cu keeps that kernel for other head dimensions):
// 197 us against 214 for 3 sequences of up to 130 tokens over 4096, 32/4 x 64,
// and 137 against 225 for single tokens of 32 sequences of up to 8192.  An
// infinite element of a live row gives NaN (inf - inf in the split).
//
// The MMAs' own fp32 accumulation cuts instead of rounding: a sum carried through
// thousands of them drifts towards zero (1e-4 after 20 k keys).  So they only sum
// 16 columns of a score, or the keys of one tile, and what they give is added
// to the score or the output by ordinary, rounding additions.  The sum of the
// weights grows by key tiles too: off by at most 2^-25 of itself per tile (over
// 262144 like weights added one by one it was 4.2e-4 off).
//
// The structure is that of paged_mma.cu: a ring of key tiles (32 keys), one
// bulk copy per row, WM x WN = 4 warps over query rows and keys, the parts of a
// row joined in shared memory.  The scores leave their MMA as columns 2t and
// 2t + 1 of a lane; taking key 2t for the k index t and 2t + 1 for t + 4 makes
// them the next product's A operand as they are, with V's rows read in the same
// order.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"

namespace kiv {

constexpr int MF_KEYS = 32;
constexpr int MF_THREADS = 128;

template <int D, int ROWS>
struct F32Shape {
  static constexpr int LD = D * 4 + 16;                    // bytes per row: 16 B of padding spread ldmatrix over the banks
  static constexpr int STAGE = 2 * MF_KEYS * LD;           // K and V tile
  // as many blocks per SM as registers allow, each with its next tile on the way
  static constexpr int STAGES = D <= 64 ? 3 : 2;
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + (size_t)ROWS * LD;
  // 228 KB per SM, 1 KB of each block reserved, half a KB static; 170 or 255
  // registers a thread
  static constexpr int FIT = (int)(233472 / (SMEM + 1536)), REGS = D <= 96 ? 3 : 2;
  static constexpr int BLOCKS = FIT < REGS ? FIT : REGS;
};

__device__ __forceinline__ void ldsm4f(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t &hi, uint32_t &lo) {
  const float f = __uint_as_float(x);
  hi = to_tf32(f);
  lo = to_tf32(f - __uint_as_float(hi));
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b with both operands split: the small products first
__device__ __forceinline__ void mma_split(float (&c)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t b0, uint32_t b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  mma1688(c, ah, l0, l1);
  mma1688(c, al, h0, h1);
  mma1688(c, ah, h0, h1);
}

template <int D, int WM>
__global__ void __launch_bounds__(MF_THREADS, F32Shape<D, 16 * WM>::BLOCKS) paged_f32_kernel(const __grid_constant__ PagedPlan p) {
  using T = float;
  constexpr int WN = 4 / WM, ROWS = 16 * WM;
  using S = F32Shape<D, ROWS>;
  constexpr int NK = MF_KEYS / WN;             // keys per warp and tile
  constexpr int CH = D / 4;                    // 16-byte chunks per row
  constexpr int STAGES = S::STAGES;
  extern __shared__ __align__(128) uint8_t mf_dyn[];
  __shared__ uint64_t full[STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wm = warp % WM, wn = warp / WM;
  const int g = lane >> 2, tq = lane & 3;
  const uint32_t ring = smem_u32(mf_dyn), sq = ring + STAGES * S::STAGE;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 2 * MF_KEYS);
    mbar_fence_init();
  }
  griddep_wait();
  PagedSpot at = paged_locate(p);              // every warp for itself
  if (threadIdx.x == 0) p.cut[blockIdx.x].b = -1;
  const float scale = p.q.scaling;
  // this thread's row of every tile (the first half of the threads)
  const bool isv = threadIdx.x >= MF_KEYS;
  const int myrow = threadIdx.x % MF_KEYS;
  const T *base = static_cast<const T *>(isv ? p.pc.v : p.pc.k);
  const int64_t sp = isv ? p.pc.v_stride_p : p.pc.k_stride_p, sh = isv ? p.pc.v_stride_h : p.pc.k_stride_h,
                st = isv ? p.pc.v_stride_t : p.pc.k_stride_t;
  uint8_t *const mydst = mf_dyn + threadIdx.x * S::LD;
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
    const int64_t j00 = ((int64_t)lo / MF_KEYS + sg.t0) * MF_KEYS;   // first key of the segment's first tile
    const int ntile = sg.t1 - sg.t0;

    const int32_t *table = p.pc.block_table + at.it.s.b * p.pc.table_stride;
    const int lo_t = (int)max((int64_t)0, lo - j00), hi_t = (int)(hi - j00);   // live keys, counted from j00
    // where this thread's row of tile t lies: page (-2: not a live key) and row
    auto lookup = [&](int t, int32_t &page, int32_t &row) {
      const int x = t * MF_KEYS + myrow;
      page = -2;
      row = 0;
      if (t < ntile && threadIdx.x < 2 * MF_KEYS && x >= lo_t && x < hi_t) {
        const uint32_t j = (uint32_t)(j00 + x), pg = j / (uint32_t)p.pc.page_size;
        row = (int32_t)(j - pg * (uint32_t)p.pc.page_size);
        page = table[pg];
      }
    };
    auto load_row = [&](int t, int32_t page, int32_t row) {
      if (t >= ntile || threadIdx.x >= 2 * MF_KEYS) return;
      const uint32_t n = used + t;
      uint8_t *dst = mydst + (n % STAGES) * S::STAGE;
      uint64_t *bar = &full[n % STAGES];
      if (page >= 0 && page < p.pc.num_pages) {
        mbar_arrive_tx(bar, D * 4);
        bulk_g2s(dst, base + page * sp + kvh * sh + row * st, D * 4, bar);
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
    for (int x = threadIdx.x; x < ROWS * CH; x += MF_THREADS) {
      const int r = x / CH, c = x - r * CH;
      int i, head;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (paged_row(p, at.it, at.hp, at.rt, r, i, head))
        v = ld16(static_cast<const T *>(p.q.q) + (at.it.s.q0 + i) * p.q.stride_t + head * p.q.stride_h + c * 4);
      *reinterpret_cast<uint4 *>(mf_dyn + STAGES * S::STAGE + r * S::LD + c * 16) = v;
    }
    __syncthreads();

    const uint32_t qaddr = sq + (wm * 16 + (lane & 15)) * S::LD + (lane >> 4) * 16;
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
      const uint32_t kt = ring + (n % STAGES) * S::STAGE;
      float s[NK / 8][4];
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
      const uint32_t kaddr = kt + (wn * NK + (lane & 7)) * S::LD + (lane >> 3) * 16;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[NK / 8][4];                 // of two steps of 8 columns
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) ldsm4f(b[n], kaddr + n * 8 * S::LD + k * 64);
        float part[NK / 8][4];                 // of 16 columns: see above
#pragma unroll
        for (int n = 0; n < NK / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[n][e] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4], ah[4], al[4];
          ldsm4f(a, qaddr + k * 64 + h * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) split_tf32(a[e], ah[e], al[e]);
#pragma unroll
          for (int n = 0; n < NK / 8; ++n) mma_split(part[n], ah, al, b[n][2 * h], b[n][2 * h + 1]);
        }
#pragma unroll
        for (int n = 0; n < NK / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] += part[n][e];
      }
      const int64_t j0 = j00 + (int64_t)t * MF_KEYS;
      const bool open = j0 >= free_lo && j0 + MF_KEYS - 1 <= free_hi;
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
      const float ms[2] = {m[0] == -INFINITY ? 0.f : m[0] * 1.44269504f, m[1] == -INFINITY ? 0.f : m[1] * 1.44269504f};
      // a tile's weights first: one at a time, like ones would round the long sum
      // the same way each time, and small ones not reach it at all
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = ex2(fmaf(s[n][e], 1.44269504f, -ms[e >> 1]));
          sum[e >> 1] += s[n][e];
        }
      l[0] += sum[0];
      l[1] += sum[1];
      const float *vrow = reinterpret_cast<const float *>(mf_dyn + (n % STAGES) * S::STAGE + (MF_KEYS + wn * NK + 2 * tq) * S::LD) + g;
      uint32_t ph[NK / 8][4], pl[NK / 8][4];   // k index t is key 2t, t + 4 is key 2t + 1
#pragma unroll
      for (int c = 0; c < NK / 8; ++c) {
        split_tf32(__float_as_uint(s[c][0]), ph[c][0], pl[c][0]);
        split_tf32(__float_as_uint(s[c][2]), ph[c][1], pl[c][1]);
        split_tf32(__float_as_uint(s[c][1]), ph[c][2], pl[c][2]);
        split_tf32(__float_as_uint(s[c][3]), ph[c][3], pl[c][3]);
      }
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NK / 8; ++c)
          mma_split(part, ph[c], pl[c], __float_as_uint(vrow[c * 8 * (S::LD / 4) + d * 8]),
                    __float_as_uint(vrow[(c * 8 + 1) * (S::LD / 4) + d * 8]));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] += part[e];
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
    float *sx = reinterpret_cast<float *>(mf_dyn);
    constexpr int XLD = D + 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      float *row = sx + (wn * ROWS + wm * 16 + g + 8 * a) * XLD;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2 *>(row + d * 8 + 2 * tq) = make_float2(o[d][2 * a], o[d][2 * a + 1]);
      if (tq == 0) {
        row[D] = m[a];
        row[D + 1] = l[a];
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < ROWS * (D / 8); x += MF_THREADS) {
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
        T *dst = paged_out<T>(p, at.it, i, head) + c;
        st16(dst, Elem<T>::pack(acc));
        st16(dst + 4, Elem<T>::pack(acc + 4));
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
static int f32_blocks(int rows) {
  return rows == 16 ? F32Shape<D, 16>::BLOCKS : rows == 32 ? F32Shape<D, 32>::BLOCKS : F32Shape<D, 64>::BLOCKS;
}

bool paged_f32_head(int dtype, int D) {
  return dtype == KIV_DTYPE_F32 && (D == 64 || D == 80 || D == 96 || D == 128 || D == 192 || D == 256);
}

int paged_f32_blocks(int D, int rows) {
  switch (D) {
    case 64: return sm_count() * f32_blocks<64>(rows);
    case 80: return sm_count() * f32_blocks<80>(rows);
    case 96: return sm_count() * f32_blocks<96>(rows);
    case 128: return sm_count() * f32_blocks<128>(rows);
    case 192: return sm_count() * f32_blocks<192>(rows);
    default: return sm_count() * f32_blocks<256>(rows);
  }
}

template <int D, int WM>
static cudaError_t launch_f32(const PagedPlan &p, int blocks, cudaStream_t s) {
  constexpr size_t smem = F32Shape<D, 16 * WM>::SMEM;
  cudaFuncSetAttribute(paged_f32_kernel<D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return launch_pdl(paged_f32_kernel<D, WM>, dim3((unsigned)blocks), dim3(MF_THREADS), smem, s, 1, p);
}
template <int D>
static cudaError_t launch_f32_w(const PagedPlan &p, int blocks, cudaStream_t s) {
  if (p.rows == 16) return launch_f32<D, 1>(p, blocks, s);
  if (p.rows == 32) return launch_f32<D, 2>(p, blocks, s);
  return launch_f32<D, 4>(p, blocks, s);
}

kiv_status launch_paged_f32(const PagedPlan &p, int blocks, cudaStream_t s) {
  cudaError_t e;
  switch (p.pc.head_dim) {
    case 64: e = launch_f32_w<64>(p, blocks, s); break;
    case 80: e = launch_f32_w<80>(p, blocks, s); break;
    case 96: e = launch_f32_w<96>(p, blocks, s); break;
    case 128: e = launch_f32_w<128>(p, blocks, s); break;
    case 192: e = launch_f32_w<192>(p, blocks, s); break;
    default: e = launch_f32_w<256>(p, blocks, s); break;
  }
  KIV_CHECK(cuda_status(e, "paged_attend (fp32)"));
  return launch_paged_combine(p, blocks, s);
}

}  // namespace kiv
