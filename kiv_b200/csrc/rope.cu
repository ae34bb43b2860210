// Norms of the query and key rows of each head with their position rotation
// in one pass (kiv_qk_norm_rope), and the same turn of the keys on their way
// into the pages of a paged cache (kiv_paged_append).
//
//   y = x * rsqrt(mean(x^2) + eps) * (offset + w),   then per pair (a, b):
//   (a cos - b sin, b cos + a sin),   fp32 throughout, one rounding at the end.
//
// Bound by memory: every row is read once and written once, the rest (cos and
// sin rows, weights) is shared by the heads of a token.  A group of GL lanes
// takes one token and `hc` of its heads: it asks for its first rows, then loads
// the token's cos and sin and its weight elements into registers -- 16 bytes at
// a time where they line up -- and walks the heads, a 16-byte vector per lane
// and row (two for rows of more than 512 bytes), UN rows in flight.  The
// partner of a half-split pair sits rot_dim / 2 elements away, i.e. in another
// lane of the group: one shuffle, with no shared memory.  (A block per token,
// rows asked for after cos and sin, ran at 1.7 TB/s: three dependent round
// trips for one row per thread.)
#include <algorithm>

#include "internal.h"
#include "paged.cuh"

namespace kiv {

constexpr int RP_THREADS = 256;

struct TurnArgs {
  kiv_turn t;
  int turned;            // 1: norm or rotation to do (rows that are only copied skip both)
  kiv_rows in[2], out[2];  // rope: q, k.  append: k, v ([tokens, heads, D]: stride_b unused)
  int rows[2];             // heads of each
  int tokens;              // per batch row (rope) / packed (append)
  int head_dim;
  int64_t ntok;            // all of them
  int hc, nch;             // heads per group; groups per token
  int vec_cs, vec_w;       // cos / sin rows, weights can be read 16 (interleaved: 8 or 16) bytes at a time
  int64_t *errors;
  kiv_paged pc;            // append only
};

template <typename T>
__device__ __forceinline__ float ld_as_float(const void *p, int64_t i, bool f32) {
  return f32 ? static_cast<const float *>(p)[i] : Elem<T>::to_f(static_cast<const T *>(p)[i]);
}

__device__ __forceinline__ int64_t ld_pos(const kiv_turn &t, int axis, int64_t b, int64_t i) {
  const int64_t o = axis * t.pos_stride_a + b * t.pos_stride_b + i * t.pos_stride_t;
  return t.pos_is_i64 ? static_cast<const int64_t *>(t.positions)[o] : (int64_t)static_cast<const int32_t *>(t.positions)[o];
}

// N consecutive values at p[i ..), read as vectors (16-bit: T)
template <typename T, int N>
__device__ __forceinline__ void ld_vec(const void *p, int64_t i, bool f32, float *out) {
  if (f32) {
    const float *q = static_cast<const float *>(p) + i;
#pragma unroll
    for (int e = 0; e < N; e += (N % 4 == 0 ? 4 : 2)) {
      if constexpr (N % 4 == 0) {
        const float4 v = *reinterpret_cast<const float4 *>(q + e);
        out[e] = v.x;
        out[e + 1] = v.y;
        out[e + 2] = v.z;
        out[e + 3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2 *>(q + e);
        out[e] = v.x;
        out[e + 1] = v.y;
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    const T *q = static_cast<const T *>(p) + i;
    if constexpr (N == 8) {
      Elem<T>::unpack(ld16(q), out);
    } else {
      static_assert(N == 4, "8 or 4 values");
      const uint2 v = *reinterpret_cast<const uint2 *>(q);
      float f[8];
      Elem<T>::unpack(make_uint4(v.x, v.y, 0, 0), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = f[e];
    }
  }
}

// GL lanes per row, VPL vectors per lane.  APPEND: in/out 0 are keys (turned),
// 1 are values (copied), and the destination row comes from the block table.
template <typename T, int GL, int VPL, bool APPEND>
__global__ void __launch_bounds__(RP_THREADS) turn_kernel(const __grid_constant__ TurnArgs a) {
  constexpr int V = Elem<T>::V;
  constexpr int GROUPS = RP_THREADS / GL;
  constexpr int UN = VPL == 1 ? 4 : 2;
  // rows of pairs that do not line up with the vectors trade partners here
  __shared__ float s_row[GROUPS][GL * VPL * V];
  const int D = a.head_dim, nv = D / V;
  const int lane = threadIdx.x % GL, grp = threadIdx.x / GL;
  const unsigned gmask = GL == 32 ? KIV_FULL_MASK : ((1u << GL) - 1) << ((threadIdx.x & 31) / GL * GL);
  griddep_wait();
  const int64_t gid = (int64_t)blockIdx.x * GROUPS + grp, tok = gid / a.nch;
  const int ch = (int)(gid - tok * a.nch);
  const kiv_turn &t = a.t;
  bool live = tok < a.ntok;
  const int total = a.rows[0] + a.rows[1], r_end = min(total, (ch + 1) * a.hc);
  const int64_t b = APPEND || !live ? 0 : tok / a.tokens, i = live ? tok - b * a.tokens : 0;

  auto source = [&](int r) {
    const int which = r < a.rows[0] ? 0 : 1;
    const kiv_rows &in = a.in[which];
    return static_cast<const T *>(in.p) + b * in.stride_b + (r - (which ? a.rows[0] : 0)) * in.stride_h + i * in.stride_t;
  };
  uint4 raw[UN][VPL];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int vi = lane + j * GL;
        raw[u][j] = make_uint4(0, 0, 0, 0);
        if (live && r0 + u < r_end && vi < nv) raw[u][j] = ld16(source(r0 + u) + vi * V);
      }
    }
  };
  fetch(ch * a.hc);

  // ---- where the token belongs
  int64_t place = tok, koff = 0, voff = 0;
  if (APPEND) {
    int sb = paged_find_seq(a.pc, (int64_t)blockIdx.x * GROUPS / a.nch);   // of the block's first token
    while (live && sb < a.pc.batch && (int64_t)a.pc.q_starts[sb + 1] <= tok) ++sb;
    const bool mine = live && sb < a.pc.batch && (int64_t)a.pc.q_starts[sb] <= tok;   // else: in no sequence
    live = mine;
    if (mine) {
      place = (int64_t)a.pc.seq_lens[sb] - a.pc.q_starts[sb + 1] + tok;
      live = place >= 0 && place < a.pc.table_width * a.pc.page_size;
      if (!live && lane == 0) paged_error(a.errors, KIV_ERRBIT_SEQ_LEN);
    }
    if (live) {
      const int32_t page = a.pc.block_table[sb * a.pc.table_stride + place / a.pc.page_size];
      const int64_t r = place % a.pc.page_size;
      if (page < 0 || page >= a.pc.num_pages) {
        live = false;
        if (lane == 0) paged_error(a.errors, KIV_ERRBIT_BLOCK_TABLE);
      } else {
        koff = page * a.pc.k_stride_p + r * a.pc.k_stride_t;
        voff = page * a.pc.v_stride_p + r * a.pc.v_stride_t;
      }
    }
  }

  // ---- cos, sin (sign of the pair's side folded in) of this lane's elements
  const int half = t.rot_dim / 2;
  const bool rotate = a.turned && t.cos != nullptr;
  const bool lined = t.interleaved ? t.rot_dim % V == 0 : half % V == 0;   // pairs line up with the vectors
  float c[VPL][V], s[VPL][V];
#pragma unroll
  for (int j = 0; j < VPL; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[j][e] = 1.f;
      s[j][e] = 0.f;
    }
  bool poison = false;
  if (rotate) {
    const bool f32 = t.cs_dtype == KIV_DTYPE_F32;
    bool bad = false;
    if (live) {
      const int64_t row0 = t.positions ? (t.pair_axes ? 0 : ld_pos(t, 0, b, i)) : place;
      bad = row0 < 0 || row0 >= t.cs_rows;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int x0 = (lane + j * GL) * V;
        if (bad || x0 >= t.rot_dim) continue;
        if (a.vec_cs && lined && !t.pair_axes) {
          if (t.interleaved) {
            float cc[V / 2], ss[V / 2];
            ld_vec<T, V / 2>(t.cos, row0 * t.cs_stride + x0 / 2, f32, cc);
            ld_vec<T, V / 2>(t.sin, row0 * t.cs_stride + x0 / 2, f32, ss);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              c[j][e] = cc[e / 2];
              s[j][e] = e & 1 ? ss[e / 2] : -ss[e / 2];
            }
          } else {
            const bool second = x0 >= half;
            ld_vec<T, V>(t.cos, row0 * t.cs_stride + (second ? x0 - half : x0), f32, c[j]);
            ld_vec<T, V>(t.sin, row0 * t.cs_stride + (second ? x0 - half : x0), f32, s[j]);
            if (!second) {
#pragma unroll
              for (int e = 0; e < V; ++e) s[j][e] = -s[j][e];
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int x = x0 + e;
            if (x >= t.rot_dim) continue;
            const int pair = t.interleaved ? x >> 1 : (x < half ? x : x - half);
            const bool second = t.interleaved ? (x & 1) != 0 : x >= half;
            int64_t row = row0;
            if (t.pair_axes) {
              const int ax = t.pair_axes[pair];
              const bool okay = ax >= 0 && ax < t.axes;
              row = !okay ? -1 : t.positions ? ld_pos(t, ax, b, i) : place;
            }
            if (row < 0 || row >= t.cs_rows) {
              bad = true;
            } else {
              c[j][e] = ld_as_float<T>(t.cos, row * t.cs_stride + pair, f32);
              const float sn = ld_as_float<T>(t.sin, row * t.cs_stride + pair, f32);
              s[j][e] = second ? sn : -sn;
            }
          }
        }
      }
    }
    // every row of the token shares the verdict, whichever lane saw it
    poison = (__ballot_sync(KIV_FULL_MASK, bad) & gmask) != 0;
    if (poison) {
      if (lane == 0) paged_error(a.errors, KIV_ERRBIT_POSITION);
      if (APPEND) live = false;
    }
  }

  float w[VPL][V];
  int w_of = -1;   // whose weight is in the registers
  for (int r0 = ch * a.hc; r0 < (ch + 1) * a.hc; r0 += UN) {      // the same count in every group
    if (r0 > ch * a.hc) fetch(r0);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int r = r0 + u, which = r < a.rows[0] ? 0 : 1;
      if (r0 - ch * a.hc + u >= a.hc) break;       // the same in every group
      float x[VPL][V];
#pragma unroll
      for (int j = 0; j < VPL; ++j) Elem<T>::unpack(raw[u][j], x[j]);
      const bool turn = a.turned && !(APPEND && which == 1);
      if (a.turned && t.norm) {   // the same for the whole block: the shuffles below are the whole warp's
        const void *wp = which == 0 && !APPEND ? t.q_weight : t.k_weight;
        if (w_of != which) {
          w_of = which;
          const bool f32 = t.weight_dtype == KIV_DTYPE_F32;
#pragma unroll
          for (int j = 0; j < VPL; ++j) {
            const int x0 = (lane + j * GL) * V;
            if (wp && a.vec_w && x0 < D) {
              ld_vec<T, V>(wp, x0, f32, w[j]);
#pragma unroll
              for (int e = 0; e < V; ++e) w[j][e] += t.weight_offset;
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) w[j][e] = wp && x0 + e < D ? t.weight_offset + ld_as_float<T>(wp, x0 + e, f32) : 1.f;
            }
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) ss = fmaf(x[j][e], x[j][e], ss);
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(KIV_FULL_MASK, ss, o);
        const float rs = rsqrtf(ss / (float)D + t.eps);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) x[j][e] = x[j][e] * rs * w[j][e];
      }
      if (rotate) {
        float p[VPL][V];
        if (t.interleaved) {
#pragma unroll
          for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) p[j][e] = x[j][e ^ 1];
        } else if (lined) {
          const int hv = half / V;
#pragma unroll
          for (int j = 0; j < VPL; ++j) {
            const int vi = lane + j * GL;
            const int pv = vi < hv ? vi + hv : (vi < 2 * hv ? vi - hv : vi);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              p[j][e] = __shfl_sync(KIV_FULL_MASK, x[0][e], pv % GL, GL);
              if (VPL > 1) {
                const float q1 = __shfl_sync(KIV_FULL_MASK, x[VPL - 1][e], pv % GL, GL);
                if (pv >= GL) p[j][e] = q1;
              }
            }
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) s_row[grp][(lane + j * GL) * V + e] = x[j][e];
          __syncwarp();
#pragma unroll
          for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const int xi = (lane + j * GL) * V + e;
              const int pi = xi < half ? xi + half : (xi < 2 * half ? xi - half : xi);
              p[j][e] = s_row[grp][pi];
            }
        }
        if (turn) {
#pragma unroll
          for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e)
              if ((lane + j * GL) * V + e < t.rot_dim) x[j][e] = x[j][e] * c[j][e] + p[j][e] * s[j][e];
        }
      }
      if (poison && turn) {
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) x[j][e] = __int_as_float(0x7fc00000);
      }
      if (live && r < r_end) {
        const int head = r - (which ? a.rows[0] : 0);
        T *dst;
        if (APPEND) {
          dst = which == 0 ? static_cast<T *>(a.pc.k) + koff + head * a.pc.k_stride_h
                           : static_cast<T *>(a.pc.v) + voff + head * a.pc.v_stride_h;
        } else {
          const kiv_rows &o = a.out[which];
          dst = static_cast<T *>(o.p) + b * o.stride_b + head * o.stride_h + i * o.stride_t;
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          const int vi = lane + j * GL;
          if (vi < nv) st16(dst + vi * V, turn ? Elem<T>::pack(x[j]) : raw[u][j]);
        }
      }
    }
  }
}

template <typename T, bool APPEND>
static kiv_status launch_turn(TurnArgs a, int64_t tokens, cudaStream_t s) {
  constexpr int V = Elem<T>::V;
  const int nv = a.head_dim / V;
  const int total = a.rows[0] + a.rows[1];
  const int gl = nv <= 8 ? 8 : (nv <= 16 ? 16 : 32), groups = RP_THREADS / gl;
  // Heads per group: many rows share a load of cos and sin, few keep the SMs
  // filled -- about three blocks on each, down to one row per group, where the
  // call is one chain of loads
  a.hc = 8;
  while (a.hc > 1 && tokens * ceil_div(total, a.hc) < (int64_t)3 * groups * sm_count()) a.hc /= 2;
  a.nch = (int)ceil_div(total, a.hc);
  a.ntok = tokens;
  const int64_t blocks = ceil_div(tokens * a.nch, groups);
  if (blocks > 0x7fffffff) {
    set_error("too many rows for one call");
    return KIV_ERR_UNSUPPORTED;
  }
  auto lines = [](const void *p, int dtype, int64_t per) {   // `per` values from p on, and from multiples of `per` on
    const int64_t bytes = std::min<int64_t>(16, per * elem_bytes(dtype));
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
  };
  const kiv_turn &t = a.t;
  const int per_cs = t.interleaved ? V / 2 : V;
  a.vec_cs = t.cos && lines(t.cos, t.cs_dtype, per_cs) && lines(t.sin, t.cs_dtype, per_cs) && t.cs_stride % per_cs == 0;
  a.vec_w = (!t.q_weight || lines(t.q_weight, t.weight_dtype, V)) && (!t.k_weight || lines(t.k_weight, t.weight_dtype, V));
  const dim3 grid((unsigned)blocks);
  cudaError_t e;
  if (gl == 8) e = launch_pdl(turn_kernel<T, 8, 1, APPEND>, grid, dim3(RP_THREADS), 0, s, 1, a);
  else if (gl == 16) e = launch_pdl(turn_kernel<T, 16, 1, APPEND>, grid, dim3(RP_THREADS), 0, s, 1, a);
  else if (nv <= 32) e = launch_pdl(turn_kernel<T, 32, 1, APPEND>, grid, dim3(RP_THREADS), 0, s, 1, a);
  else e = launch_pdl(turn_kernel<T, 32, 2, APPEND>, grid, dim3(RP_THREADS), 0, s, 1, a);
  return cuda_status(e, APPEND ? "paged_append" : "qk_norm_rope");
}

template <bool APPEND>
static kiv_status launch_any(int dtype, const TurnArgs &a, int64_t tokens, cudaStream_t s) {
  if (tokens == 0 || a.rows[0] + a.rows[1] == 0) return KIV_OK;
  if (dtype == KIV_DTYPE_F32) return launch_turn<float, APPEND>(a, tokens, s);
  if (dtype == KIV_DTYPE_BF16) return launch_turn<__nv_bfloat16, APPEND>(a, tokens, s);
  return launch_turn<__half, APPEND>(a, tokens, s);
}

static kiv_status check_head(int dtype, int head_dim) {
  if (dtype < 0 || dtype > 2) { set_error("unknown dtype %d", dtype); return KIV_ERR_UNSUPPORTED; }
  const int eb = elem_bytes(dtype);
  if (head_dim < 1 || (head_dim * eb) % 16 != 0 || head_dim * eb > 1024) {
    set_error("head_dim %d: rows must be a multiple of 16 bytes, at most 1024", head_dim);
    return KIV_ERR_UNSUPPORTED;
  }
  return KIV_OK;
}

static kiv_status check_turn(const kiv_turn *t, int dtype, int head_dim) {
  if (!t) return KIV_OK;
  if (t->cos || t->sin) {
    if (!t->cos || !t->sin) { set_error("cos and sin come together"); return KIV_ERR_ARG; }
    if (t->rot_dim < 2 || t->rot_dim % 2 || t->rot_dim > head_dim) {
      set_error("rot_dim %d must be even and at most head_dim %d", t->rot_dim, head_dim);
      return KIV_ERR_ARG;
    }
    if (t->cs_dtype != KIV_DTYPE_F32 && t->cs_dtype != dtype) {
      set_error("cos and sin must be float32 or of the rows' dtype");
      return KIV_ERR_ARG;
    }
    if (t->cs_rows < 0 || t->axes < 1) { set_error("bad cos/sin rows %lld or axes %d", (long long)t->cs_rows, t->axes); return KIV_ERR_ARG; }
  }
  if (t->norm && t->weight_dtype != KIV_DTYPE_F32 && t->weight_dtype != dtype && (t->q_weight || t->k_weight)) {
    set_error("norm weights must be float32 or of the rows' dtype");
    return KIV_ERR_ARG;
  }
  if (t->norm && !(t->eps >= 0.f)) { set_error("eps must not be negative"); return KIV_ERR_ARG; }
  return KIV_OK;
}

static kiv_status check_rows(const kiv_rows *r, int eb, const char *what) {
  if (!r->p || (reinterpret_cast<uintptr_t>(r->p) & 15) || (r->stride_b * eb) % 16 || (r->stride_h * eb) % 16 ||
      (r->stride_t * eb) % 16) {
    set_error("%s rows missing or not 16-byte aligned", what);
    return KIV_ERR_ARG;
  }
  return KIV_OK;
}

}  // namespace kiv

using namespace kiv;

extern "C" {

kiv_status kiv_qk_norm_rope(int32_t dtype, int32_t batch, int32_t tokens, int32_t head_dim, const kiv_rows *q,
                            const kiv_rows *k, const kiv_rows *q_out, const kiv_rows *k_out, const kiv_turn *turn,
                            int64_t *errors, void *stream) {
  KIV_CHECK(check_head(dtype, head_dim));
  if (!q || !q_out || !turn || (k != nullptr) != (k_out != nullptr)) {
    set_error("qk_norm_rope: q, q_out and turn are needed, k and k_out come together");
    return KIV_ERR_ARG;
  }
  if (batch < 0 || tokens < 0 || q->heads < 0 || (k && k->heads < 0) || q_out->heads != q->heads ||
      (k && k_out->heads != k->heads)) {
    set_error("qk_norm_rope: bad sizes");
    return KIV_ERR_ARG;
  }
  KIV_CHECK(check_turn(turn, dtype, head_dim));
  if ((int64_t)batch * tokens == 0) return KIV_OK;
  if ((int64_t)batch * tokens > 0x7fffffff) { set_error("qk_norm_rope: more than 2^31 - 1 tokens"); return KIV_ERR_UNSUPPORTED; }
  const int eb = elem_bytes(dtype);
  KIV_CHECK(check_rows(q, eb, "q"));
  KIV_CHECK(check_rows(q_out, eb, "q_out"));
  if (k) {
    KIV_CHECK(check_rows(k, eb, "k"));
    KIV_CHECK(check_rows(k_out, eb, "k_out"));
  }
  TurnArgs a = {};
  a.t = *turn;
  a.turned = turn->norm != 0 || turn->cos != nullptr;
  a.in[0] = *q;
  a.out[0] = *q_out;
  a.rows[0] = q->heads;
  if (k) {
    a.in[1] = *k;
    a.out[1] = *k_out;
    a.rows[1] = k->heads;
  }
  a.tokens = tokens;
  a.head_dim = head_dim;
  a.errors = errors;
  return launch_any<false>(dtype, a, (int64_t)batch * tokens, (cudaStream_t)stream);
}

kiv_status kiv_paged_append(const kiv_paged *pc, const void *k, int64_t k_stride_t, int64_t k_stride_h, const void *v,
                            int64_t v_stride_t, int64_t v_stride_h, const kiv_turn *turn, void *stream) {
  KIV_CHECK(check_paged(pc));
  KIV_CHECK(check_head(pc->dtype, pc->head_dim));
  KIV_CHECK(check_turn(turn, pc->dtype, pc->head_dim));
  if (pc->num_tokens == 0) return KIV_OK;
  const int eb = elem_bytes(pc->dtype);
  TurnArgs a = {};
  if (turn) a.t = *turn;
  a.turned = turn && (turn->norm != 0 || turn->cos != nullptr);
  a.in[0] = kiv_rows{const_cast<void *>(k), 0, k_stride_h, k_stride_t, pc->num_kv_heads, 0};
  a.in[1] = kiv_rows{const_cast<void *>(v), 0, v_stride_h, v_stride_t, pc->num_kv_heads, 0};
  KIV_CHECK(check_rows(&a.in[0], eb, "new key"));
  KIV_CHECK(check_rows(&a.in[1], eb, "new value"));
  a.rows[0] = a.rows[1] = pc->num_kv_heads;
  a.tokens = (int)pc->num_tokens;
  a.head_dim = pc->head_dim;
  a.errors = pc->errors;
  a.pc = *pc;
  return launch_any<true>(pc->dtype, a, pc->num_tokens, (cudaStream_t)stream);
}

}  // extern "C"
