// Attention of new tokens over a paged cache (kiv_paged_attend): checks,
// choice of kernel, the CUDA-core kernel, and the join of split items.
//
//   out = softmax(score(q k^T)) v over the keys a token sees, one pass over
//   the keys with the running maximum and sum of each row in fp32.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"

namespace kiv {

kiv_status check_paged(const kiv_paged *pc) {
  if (!pc) { set_error("paged cache is NULL"); return KIV_ERR_ARG; }
  if (pc->dtype < 0 || pc->dtype > 2) { set_error("unknown dtype %d", pc->dtype); return KIV_ERR_UNSUPPORTED; }
  const int eb = elem_bytes(pc->dtype);
  if (pc->batch < 0 || pc->num_kv_heads < 1 || pc->head_dim < 1 || pc->page_size < 1 || pc->num_pages < 0 ||
      pc->table_width < 0 || pc->table_stride < 0 || pc->num_tokens < 0 || pc->max_query_len < 0) {
    set_error("bad paged cache sizes");
    return KIV_ERR_ARG;
  }
  if ((pc->head_dim * eb) % 16 != 0) {
    set_error("head_dim %d: rows must be a multiple of 16 bytes", pc->head_dim);
    return KIV_ERR_UNSUPPORTED;
  }
  if (pc->num_tokens > 0x7fffffff || pc->num_pages > 0x7fffffff || pc->table_width > 0x7fffffff / pc->page_size ||
      pc->batch > (1 << 20)) {
    set_error("paged cache too large: tokens, pages and table_width * page_size stay below 2^31, batch at most 2^20");
    return KIV_ERR_UNSUPPORTED;
  }
  if (pc->num_tokens > 0 && pc->batch > 0 &&
      (!pc->seq_lens || !pc->q_starts || (pc->table_width > 0 && !pc->block_table))) {
    set_error("block_table, seq_lens or q_starts missing");
    return KIV_ERR_ARG;
  }
  const int64_t strides[6] = {pc->k_stride_p, pc->k_stride_h, pc->k_stride_t, pc->v_stride_p, pc->v_stride_h, pc->v_stride_t};
  for (int64_t s : strides)
    if (s < 0 || (s * eb) % 16) { set_error("page strides must be multiples of 16 bytes"); return KIV_ERR_ARG; }
  if (pc->num_pages > 0 && (!pc->k || !pc->v || (reinterpret_cast<uintptr_t>(pc->k) & 15) || (reinterpret_cast<uintptr_t>(pc->v) & 15))) {
    set_error("pages missing or not 16-byte aligned");
    return KIV_ERR_ARG;
  }
  return KIV_OK;
}

static kiv_status check_paged_query(const kiv_paged *pc, const kiv_paged_query *q) {
  if (!q) { set_error("paged query is NULL"); return KIV_ERR_ARG; }
  const int eb = elem_bytes(pc->dtype);
  if (q->num_query_heads < 1 || q->num_query_heads % pc->num_kv_heads != 0) {
    set_error("query heads %d are not a multiple of key heads %d", q->num_query_heads, pc->num_kv_heads);
    return KIV_ERR_ARG;
  }
  if (pc->head_dim > 256) { set_error("paged attention: head_dim %d above 256", pc->head_dim); return KIV_ERR_UNSUPPORTED; }
  if (q->window < 0 || (q->window > 0 && !q->causal)) { set_error("window must not be negative, and needs causal"); return KIV_ERR_ARG; }
  if (!(q->softcap >= 0.f)) { set_error("softcap must not be negative"); return KIV_ERR_ARG; }
  if (pc->num_tokens > 0 &&
      (!q->q || !q->out || (reinterpret_cast<uintptr_t>(q->q) & 15) || (reinterpret_cast<uintptr_t>(q->out) & 15) ||
       (q->stride_t * eb) % 16 || (q->stride_h * eb) % 16 || (q->out_stride_t * eb) % 16 || (q->out_stride_h * eb) % 16)) {
    set_error("query or output rows missing or not 16-byte aligned");
    return KIV_ERR_ARG;
  }
  return KIV_OK;
}

// ---------------------------------------------------------------------------
// CUDA-core kernel: head dimensions outside the tensor-core kernels' set.
// R rows x 64 keys per step; 16 threads share a row, each with 4 keys of the
// scores and a sixteenth of the output row.  Bound by the shared-memory reads
// that feed the FMAs (a 4 x 4 register tile: 8 FMAs per 16 bytes read).  512 tokens
// over 16384, 32/8 x 112 in 16 bits: 6.1 ms, 19 TFLOP/s; 32 sequences of 16 k keys,
// one token each, x 112: 2.8 ms, x 40 in fp32: 1.3 ms.
// ---------------------------------------------------------------------------
constexpr int CC_KEYS = 64;
constexpr int CC_THREADS = 256;

// fp32 rows up to 128: the next tile comes while this one is used
template <typename T, int DM>
__host__ __device__ constexpr int cc_buffers() { return sizeof(T) == 4 && DM <= 128 ? 2 : 1; }

static size_t cc_smem(int rows, int D, int dtype) {
  const int buffers = dtype == KIV_DTYPE_F32 && D <= 128 ? 2 : 1;
  return sizeof(float) * ((size_t)(rows + buffers * 2 * CC_KEYS) * (D + 4) + (size_t)rows * (CC_KEYS + 4));
}

template <typename T, int R, int DM>
__global__ void __launch_bounds__(CC_THREADS, DM <= 64 || (R == 16 && DM <= 128) ? 2 : 1) paged_cc_kernel(const __grid_constant__ PagedPlan p) {
  constexpr int V = Elem<T>::V;
  constexpr int RPT = R / 16;          // rows per thread
  constexpr int NBUF = cc_buffers<T, DM>();
  constexpr int DC = (DM + 63) / 64;   // 4-element slices of an output row per thread
  extern __shared__ float4 cc_dyn[];
  __shared__ int64_t s_ko[3][CC_KEYS], s_vo[3][CC_KEYS];
  const int D = p.pc.head_dim, nv = D / V, ld = D + 4;
  float *sq = reinterpret_cast<float *>(cc_dyn);
  float *const sk0 = sq + R * ld, *const sp = sk0 + NBUF * 2 * CC_KEYS * ld;   // [buffer][K, V][key]
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  griddep_wait();
  PagedSpot at = paged_locate(p);              // every warp for itself
  if (threadIdx.x == 0) p.cut[blockIdx.x].b = -1;
  while (at.it.s.b >= 0 && at.unit < at.end) {
    const PagedSegment g = paged_segment(p, at);
    const int kvh = at.hp / p.hs;
    int lo, hi;
    paged_range(p, at.it, at.rt, lo, hi);
    if (threadIdx.x == 0) {
      if (!g.head) paged_check_lens(p.pc, at.it.s);
      if (g.tail) paged_record(p, blockIdx.x, at, g);
    }
    hi = min(hi, at.it.s.len);
    __syncthreads();
    for (int x = threadIdx.x; x < R * nv; x += CC_THREADS) {
      const int r = x / nv, vi = x - r * nv;
      float f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = 0.f;
      int i, head;
      if (paged_row(p, at.it, at.hp, at.rt, r, i, head))
        Elem<T>::unpack(ld16(static_cast<const T *>(p.q.q) + (at.it.s.q0 + i) * p.q.stride_t + head * p.q.stride_h + vi * V), f);
#pragma unroll
      for (int e = 0; e < V; ++e) sq[r * ld + vi * V + e] = f[e];
    }
    int place[RPT];                    // of each row's token; -1: no such row
    bool have[RPT];
    float m[RPT], l[RPT];
    float4 o[RPT][DC];
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
      int i, head;
      have[a] = paged_row(p, at.it, at.hp, at.rt, tr * RPT + a, i, head);
      place[a] = p.q.causal ? at.it.base + i : 0x7fffffff;
      m[a] = -INFINITY;
      l[a] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) o[a][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int64_t j00 = ((int64_t)(lo / CC_KEYS) + g.t0) * CC_KEYS;
    const int ntile = g.t1 - g.t0;
    // where tile t's rows lie (-1: they read as zeros), a thread per key; three
    // tiles' places are kept, so that the next one's are there when its copies go
    auto places = [&](int t, int64_t &ko, int64_t &vo) {
      const int64_t j = j00 + (int64_t)t * CC_KEYS + threadIdx.x;
      ko = vo = -1;
      if (t < ntile && threadIdx.x < CC_KEYS && j >= lo && j < hi) {
        paged_key(p.pc, at.it.s.b, j, kvh, ko, vo);
        if (ko < 0) paged_error(p.pc.errors, KIV_ERRBIT_BLOCK_TABLE);
      }
    };
    auto keep = [&](int t, int64_t ko, int64_t vo) {
      if (threadIdx.x < CC_KEYS) {
        s_ko[t % 3][threadIdx.x] = ko;
        s_vo[t % 3][threadIdx.x] = vo;
      }
    };
    auto load = [&](int t) {                   // 16 threads per row
      if (t < ntile) {
        float *bk = sk0 + (t % NBUF) * 2 * CC_KEYS * ld, *bv = bk + CC_KEYS * ld;
#pragma unroll
        for (int y = 0; y < 2 * CC_KEYS / 16; ++y) {
          const int r = (tr + 16 * y) % CC_KEYS;
          const bool isv = tr + 16 * y >= CC_KEYS;
          const int64_t off = isv ? s_vo[t % 3][r] : s_ko[t % 3][r];
          const T *src = static_cast<const T *>(isv ? p.pc.v : p.pc.k) + (off < 0 ? 0 : off);
          float *dst = (isv ? bv : bk) + r * ld;
          for (int vi = tc; vi < nv; vi += 16) {
            if constexpr (sizeof(T) == 4) {
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + vi * V)), "l"(src + vi * V),
                           "r"(off < 0 ? 0 : 16)
                           : "memory");
            } else {
              float f[V];
#pragma unroll
              for (int e = 0; e < V; ++e) f[e] = 0.f;
              if (off >= 0) Elem<T>::unpack(ld16(src + vi * V), f);
#pragma unroll
              for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(dst + vi * V + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();                           // the previous item's readers are done
    int64_t nko, nvo;
    for (int t = 0; t < 2; ++t) {
      places(t, nko, nvo);
      keep(t, nko, nvo);
    }
    __syncthreads();
    load(0);
    for (int t = 0; t < ntile; ++t) {
      const int64_t j0 = j00 + (int64_t)t * CC_KEYS;
      if (NBUF == 1 && t > 0) {
        __syncthreads();                       // tile t - 1 is read
        load(t);
      }
      places(t + 2, nko, nvo);
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();                         // tile t is there; with two buffers, tile t - 1 is read
      if (NBUF == 2) load(t + 1);
      const float *sk = sk0 + (t % NBUF) * 2 * CC_KEYS * ld, *sv = sk + CC_KEYS * ld;
      float2 s2[RPT][4];                       // even and odd columns apart: two FMAs per instruction
#pragma unroll
      for (int a = 0; a < RPT; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) s2[a][c] = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 kk[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) kk[c] = *reinterpret_cast<const float4 *>(sk + (tc + 16 * c) * ld + d);
#pragma unroll
        for (int a = 0; a < RPT; ++a) {
          const float4 qq = *reinterpret_cast<const float4 *>(sq + (tr * RPT + a) * ld + d);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s2[a][c] = __ffma2_rn(make_float2(qq.x, qq.y), make_float2(kk[c].x, kk[c].y), s2[a][c]);
            s2[a][c] = __ffma2_rn(make_float2(qq.z, qq.w), make_float2(kk[c].z, kk[c].w), s2[a][c]);
          }
        }
      }
      float s[RPT][4];
#pragma unroll
      for (int a = 0; a < RPT; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[a][c] = s2[a][c].x + s2[a][c].y;
#pragma unroll
      for (int a = 0; a < RPT; ++a) {
        float mx = m[a];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t j = j0 + tc + 16 * c;
          float x = s[a][c] * p.q.scaling;
          if (p.q.softcap > 0.f) x = p.q.softcap * tanhf(x / p.q.softcap);
          const bool seen = j < hi && j <= place[a] && (p.q.window == 0 || j > (int64_t)place[a] - p.q.window);
          s[a][c] = seen ? x : -INFINITY;
          mx = fmaxf(mx, s[a][c]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(KIV_FULL_MASK, mx, w));
        const float ms = mx == -INFINITY ? 0.f : mx;     // a row that has seen nothing yet: exp(-inf) = 0
        const float keep = ex2((m[a] - ms) * 1.44269504f);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float e = ex2((s[a][c] - ms) * 1.44269504f);
          sp[(tr * RPT + a) * (CC_KEYS + 4) + tc + 16 * c] = e;
          sum += e;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(KIV_FULL_MASK, sum, w);
        l[a] = l[a] * keep + sum;
        m[a] = mx;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          o[a][c].x *= keep;
          o[a][c].y *= keep;
          o[a][c].z *= keep;
          o[a][c].w *= keep;
        }
      }
      __syncwarp();                    // a row's 16 threads are in one warp
#pragma unroll 2
      for (int j = 0; j < CC_KEYS; j += 4) {
        float4 pp[RPT];
#pragma unroll
        for (int a = 0; a < RPT; ++a) pp[a] = *reinterpret_cast<const float4 *>(sp + (tr * RPT + a) * (CC_KEYS + 4) + j);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const int d = 4 * tc + 64 * c;
            if (d < D) {
              const float4 vv = *reinterpret_cast<const float4 *>(sv + (j + jj) * ld + d);
#pragma unroll
              for (int a = 0; a < RPT; ++a) {
                const float e = jj == 0 ? pp[a].x : jj == 1 ? pp[a].y : jj == 2 ? pp[a].z : pp[a].w;
                const float2 e2 = make_float2(e, e);
                float2 lo2 = __ffma2_rn(e2, make_float2(vv.x, vv.y), make_float2(o[a][c].x, o[a][c].y));
                float2 hi2 = __ffma2_rn(e2, make_float2(vv.z, vv.w), make_float2(o[a][c].z, o[a][c].w));
                o[a][c] = make_float4(lo2.x, lo2.y, hi2.x, hi2.y);
              }
            }
          }
        }
      }
      keep(t + 2, nko, nvo);                   // over tile t - 1's
    }
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
      if (!have[a]) continue;
      const int r = tr * RPT + a;
      int i, head;
      paged_row(p, at.it, at.hp, at.rt, r, i, head);
      if (!g.head && !g.tail) {
        const float inv = paged_inv(l[a]);
        T *dst = paged_out<T>(p, at.it, i, head);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const int d = 4 * tc + 64 * c;
          if (d < D) {
            dst[d] = Elem<T>::from_f(o[a][c].x * inv);
            dst[d + 1] = Elem<T>::from_f(o[a][c].y * inv);
            dst[d + 2] = Elem<T>::from_f(o[a][c].z * inv);
            dst[d + 3] = Elem<T>::from_f(o[a][c].w * inv);
          }
        }
        if (tc == 0) paged_lse(p, at.it, i, head, m[a], l[a]);
      } else {
        float *dst = paged_part(p, 2 * (int64_t)blockIdx.x + (g.head ? 0 : 1), r);
#pragma unroll
        for (int c = 0; c < DC; ++c)
          if (4 * tc + 64 * c < D) *reinterpret_cast<float4 *>(dst + 4 * tc + 64 * c) = o[a][c];
        if (tc == 0) {
          dst[D] = m[a];
          dst[D + 1] = l[a];
        }
      }
    }
    paged_advance(p, at, g);
  }
}

// ---------------------------------------------------------------------------
// Join of the items that blocks share.  Block (c, y) takes the item that block
// c of the attention kernel began and did not finish; a warp takes a row's
// slice of 128 columns: the parts' maxima and sums by lane, then the scaled sum
// of the parts in block order.
// ---------------------------------------------------------------------------
constexpr int CB_WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(CB_WARPS * 32) paged_combine_kernel(const __grid_constant__ PagedPlan p) {
  griddep_wait();
  const PagedCut cut = p.cut[blockIdx.x];
  if (cut.b < 0) return;
  const int D = p.pc.head_dim, lane = threadIdx.x & 31;
  const int slices = (D + 127) / 128;
  PagedItems it;
  it.s.b = cut.b;
  it.s.q0 = cut.q0;
  it.s.n = cut.n;
  const int warp = (blockIdx.y * CB_WARPS + (threadIdx.x >> 5)), nwarps = gridDim.y * CB_WARPS;
  // parts: slot 2c + 1, then slot 2c' of the later blocks up to the last
  const int c0 = blockIdx.x, last = cut.last;
  const int64_t stride = 2 * 8 * (int64_t)partial_stride(D);       // two slots
  const int tasks = min(p.tpt, cut.n - cut.rt * p.tpt) * p.grp * slices;   // rows that have tokens
  for (int x = warp; x < tasks; x += nwarps) {
    const int r = slices == 1 ? x : x / slices, slice = x - r * slices, col = slice * 128 + 4 * lane;
    int i, head;
    if (!paged_row(p, it, cut.hp, cut.rt, r, i, head)) continue;
    // lane k holds maximum and sum of part k of 32 at a time; the parts' values
    // are asked for eight at a time, the first of them before the maxima
    float mx = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c1 = c0; c1 <= last; c1 += 32) {
      const int n = min(32, last - c1 + 1);
      const float *src = paged_part(p, 2 * (int64_t)c1, r);
      const int64_t shift = c1 == c0 ? stride / 2 : 0;           // of part 0
      const float *mine = src + lane * stride + (lane == 0 ? shift : 0);
      const float2 ml = lane < n ? *reinterpret_cast<const float2 *>(mine + D) : make_float2(-INFINITY, 0.f);
      float4 v[8];
      auto ask = [&](int k0) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          v[k] = k0 + k < n && col < D ? *reinterpret_cast<const float4 *>(src + (k0 + k) * stride + (k0 + k == 0 ? shift : 0) + col)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      ask(0);
      float top = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(KIV_FULL_MASK, top, o));
      top = fmaxf(top, mx);
      const float ms = top == -INFINITY ? 0.f : top, keep = ex2((mx - ms) * 1.44269504f);
      const float w = ex2((ml.x - ms) * 1.44269504f);
      float sum = ml.y * w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(KIV_FULL_MASK, sum, o);
      l = l * keep + sum;
      mx = top;
      acc.x *= keep;
      acc.y *= keep;
      acc.z *= keep;
      acc.w *= keep;
#pragma unroll 1
      for (int k0 = 0; k0 < n; k0 += 8) {
        if (k0 > 0) ask(k0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float f = __shfl_sync(KIV_FULL_MASK, w, k0 + k);
          acc.x = fmaf(v[k].x, f, acc.x);
          acc.y = fmaf(v[k].y, f, acc.y);
          acc.z = fmaf(v[k].z, f, acc.z);
          acc.w = fmaf(v[k].w, f, acc.w);
        }
      }
    }
    const float inv = paged_inv(l);
    if (col < D) {
      T *dst = paged_out<T>(p, it, i, head) + col;
      dst[0] = Elem<T>::from_f(acc.x * inv);
      dst[1] = Elem<T>::from_f(acc.y * inv);
      dst[2] = Elem<T>::from_f(acc.z * inv);
      dst[3] = Elem<T>::from_f(acc.w * inv);
    }
    if (lane == 0 && slice == 0) paged_lse(p, it, i, head, mx, l);
  }
}

kiv_status launch_paged_combine(const PagedPlan &p, int blocks, cudaStream_t s) {
  if (blocks < 2) return KIV_OK;
  const int slices = (int)ceil_div(p.pc.head_dim, 128);
  const int64_t rows = std::min<int64_t>(p.tpt, p.pc.num_tokens) * p.grp;    // of an item at most
  const int y = (int)std::min<int64_t>(ceil_div(rows * slices, CB_WARPS), 32);
  const dim3 grid((unsigned)blocks, (unsigned)y), block(CB_WARPS * 32);
  cudaError_t e;
  if (p.pc.dtype == KIV_DTYPE_F32) e = launch_pdl(paged_combine_kernel<float>, grid, block, 0, s, 1, p);
  else if (p.pc.dtype == KIV_DTYPE_BF16) e = launch_pdl(paged_combine_kernel<__nv_bfloat16>, grid, block, 0, s, 1, p);
  else e = launch_pdl(paged_combine_kernel<__half>, grid, block, 0, s, 1, p);
  return cuda_status(e, "paged_combine");
}

// ------------------------------------------------------------------ host
// Tiling of one kernel's items: `rows` rows per tile, `kt` keys per tile.
static PagedPlan make_plan(const kiv_paged *pc, const kiv_paged_query *q, int rows, int kt) {
  PagedPlan p = {};
  p.pc = *pc;
  p.q = *q;
  const int per = q->num_query_heads / pc->num_kv_heads;
  p.hs = (int)ceil_div(per, rows);
  p.grp = (int)ceil_div(per, p.hs);
  p.tpt = p.tps = rows / p.grp;
  p.kt = kt;
  p.kt_log2 = kt == 32 ? 5 : kt == 64 ? 6 : 7;
  p.rows = rows;
  return p;
}

enum PagedKernel { PAGED_CC, PAGED_F32, PAGED_MMA, PAGED_TC };

struct PagedCall {
  PagedKernel kernel;
  PagedPlan p;
  int blocks;
  size_t bytes;        // of its workspace
  size_t part_offset;
};

// The kernel of a call and its tiling.  tcgen05 wherever TMA can bring the
// pages (paged_tc.cu): for single tokens too, 211 us against 250 (16 sequences of
// 16 k keys, 32/8 x 128) and 63 against 89 (8/1 x 256) by the split kernel, which
// keeps the pages of odd sizes and strides, the head dimensions 80 and 192 and
// heads in groups above 128; fp32 by split TF32 products (paged_f32.cu); CUDA
// cores for what is left.  The lengths are on the device, so the row tiles of
// all but the first go by what the host knows: the rows of the longest sequence
// (max_query_len), or the mean.
static PagedCall plan_call(const kiv_paged *pc, const kiv_paged_query *q) {
  PagedCall c;
  const int D = pc->head_dim;
  const int64_t per = q->num_query_heads / pc->num_kv_heads;
  const int64_t mean = ceil_div(pc->num_tokens, std::max(1, pc->batch));
  const int64_t likely = per * (pc->max_query_len > 0 ? std::min<int64_t>(pc->max_query_len, pc->num_tokens) : mean);
  if (paged_tc_eligible(pc, q)) {
    c.kernel = PAGED_TC;
    c.p = make_plan(pc, q, 128, 128);
    if (D <= 128) {                 // two row tiles per item; at 256 TMEM holds the output of one
      c.p.tpt *= 2;
      c.p.rows = 256;
    }
    c.blocks = sm_count();
  } else if (paged_mma_head(pc->dtype, D)) {
    c.kernel = PAGED_MMA;
    const int rows = likely <= 16 ? 16 : likely <= 32 ? 32 : 64;
    c.p = make_plan(pc, q, rows, 64);
    c.blocks = paged_mma_blocks(D, rows);
  } else if (paged_f32_head(pc->dtype, D)) {
    c.kernel = PAGED_F32;
    const int rows = likely <= 16 ? 16 : likely <= 32 ? 32 : 64;
    c.p = make_plan(pc, q, rows, 32);
    c.blocks = paged_f32_blocks(D, rows);
  } else {
    c.kernel = PAGED_CC;
    const int rows = likely <= 16 ? 16 : 64;
    c.p = make_plan(pc, q, rows, CC_KEYS);
    const size_t most = D <= 64 || (rows == 16 && D <= 128) ? 2 : 1;       // as the kernel's launch bounds
    c.blocks = sm_count() * (int)std::max<size_t>(1, std::min<size_t>(most, 233472 / (cc_smem(rows, D, pc->dtype) + 4608)));
  }
  c.p.slots = 2 * c.blocks;
  c.part_offset = (size_t)align_up((int64_t)c.blocks * sizeof(PagedCut), 256);
  c.bytes = c.part_offset + (size_t)align_up((int64_t)c.p.slots * c.p.rows * partial_stride(D) * 4, 256);
  return c;
}

template <typename T, int R, int DM>
static cudaError_t launch_cc(const PagedCall &c, cudaStream_t s) {
  const size_t smem = cc_smem(R, c.p.pc.head_dim, c.p.pc.dtype);
  cudaFuncSetAttribute(paged_cc_kernel<T, R, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return launch_pdl(paged_cc_kernel<T, R, DM>, dim3((unsigned)c.blocks), dim3(CC_THREADS), smem, s, 1, c.p);
}
template <typename T, int R>
static cudaError_t launch_cc_d(const PagedCall &c, cudaStream_t s) {
  const int D = c.p.pc.head_dim;
  return D <= 64 ? launch_cc<T, R, 64>(c, s) : D <= 128 ? launch_cc<T, R, 128>(c, s) : launch_cc<T, R, 256>(c, s);
}
template <typename T>
static cudaError_t launch_cc_r(const PagedCall &c, cudaStream_t s) {
  return c.p.rows == 16 ? launch_cc_d<T, 16>(c, s) : launch_cc_d<T, 64>(c, s);
}

static kiv_status run_call(PagedCall c, char *ws, cudaStream_t s) {
  c.p.cut = reinterpret_cast<PagedCut *>(ws);
  c.p.part = reinterpret_cast<float *>(ws + c.part_offset);
  if (c.kernel == PAGED_MMA) return launch_paged_mma(c.p, c.blocks, s);
  if (c.kernel == PAGED_F32) return launch_paged_f32(c.p, c.blocks, s);
  if (c.kernel == PAGED_TC) return launch_paged_tc(c.p, c.blocks, s);
  cudaError_t e;
  if (c.p.pc.dtype == KIV_DTYPE_F32) e = launch_cc_r<float>(c, s);
  else if (c.p.pc.dtype == KIV_DTYPE_BF16) e = launch_cc_r<__nv_bfloat16>(c, s);
  else e = launch_cc_r<__half>(c, s);
  KIV_CHECK(cuda_status(e, "paged_attend"));
  return launch_paged_combine(c.p, c.blocks, s);
}

}  // namespace kiv

using namespace kiv;

extern "C" {

size_t kiv_paged_workspace_bytes(const kiv_paged *pc, const kiv_paged_query *q) {
  if (check_paged(pc) != KIV_OK || !q || q->num_query_heads < 1 || q->num_query_heads % pc->num_kv_heads || pc->head_dim > 256) return 0;
  return plan_call(pc, q).bytes;
}

kiv_status kiv_paged_attend(const kiv_paged *pc, const kiv_paged_query *q, void *ws, size_t ws_bytes, void *stream) {
  KIV_CHECK(check_paged(pc));
  KIV_CHECK(check_paged_query(pc, q));
  if (pc->num_tokens == 0 || pc->batch == 0) return KIV_OK;
  const PagedCall c = plan_call(pc, q);
  if (!ws || ws_bytes < c.bytes || (reinterpret_cast<uintptr_t>(ws) & 255)) {
    set_error("workspace too small or misaligned (%zu < %zu)", ws_bytes, c.bytes);
    return KIV_ERR_CAPACITY;
  }
  return run_call(c, static_cast<char *>(ws), (cudaStream_t)stream);
}

}  // extern "C"
