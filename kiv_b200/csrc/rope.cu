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
// a time where they line up -- and walks the heads, RP_UN rows in flight.  A
// lane holds two 16-byte vectors of a row, and for half-split pairs these are
// the two sides of the same pairs: no exchange between lanes, and one cos and
// sin per pair.  Measured: 2 x 4099 tokens of 28/4 x 128 (bf16, no norm, 139 MB)
// 30 us, 4.6 TB/s; one vector per lane and the other side by shuffles took 2.2
// times the instructions and 53 us, a block per token 82 us.
#include <algorithm>

#include "internal.h"
#include "paged.cuh"

namespace kiv {

constexpr int RP_THREADS = 256;
constexpr int RP_UN = 4;         // rows in flight: 512 threads x 4 x 32 B = 64 KB per SM

struct TurnArgs {
  kiv_turn t;
  int turned;            // 1: norm or rotation to do (rows that are only copied skip both)
  kiv_rows in[2], out[2];  // rope: q, k.  append: k, v ([tokens, heads, D]: stride_b unused)
  int rows[2];             // heads of each
  int tokens;              // per batch row (rope) / packed (append)
  int head_dim;
  uint32_t ntok;           // all of them
  int hc;                  // heads per group
  int vec_cs, vec_w;       // cos / sin rows, weights can be read 16 bytes at a time
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

// N consecutive values at p[i ..), read as vectors (N values fill a 16-byte row vector)
template <typename T, int N>
__device__ __forceinline__ void ld_vec(const void *p, int64_t i, bool f32, float *out) {
  if (f32) {
    const float *q = static_cast<const float *>(p) + i;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(q + e);
      out[e] = v.x;
      out[e + 1] = v.y;
      out[e + 2] = v.z;
      out[e + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 2) {
    Elem<T>::unpack(ld16(static_cast<const T *>(p) + i), out);
  }
}

// GL lanes per row, two vectors per lane.  APPEND: in/out 0 are keys (turned),
// 1 are values (copied), and the destination row comes from the block table.
template <typename T, int GL, bool APPEND, bool NORM>
__global__ void __launch_bounds__(RP_THREADS, !NORM && sizeof(T) == 4 ? 3 : 2) turn_kernel(const __grid_constant__ TurnArgs a) {
  constexpr int V = Elem<T>::V;
  constexpr int GROUPS = RP_THREADS / GL;
  // rows of pairs that do not line up with the vectors trade partners here
  __shared__ float s_row[GROUPS][GL * 2 * V];
  const int D = a.head_dim, nv = D / V;
  const int lane = threadIdx.x % GL, grp = threadIdx.x / GL;
  const unsigned gmask = GL == 32 ? KIV_FULL_MASK : ((1u << GL) - 1) << ((threadIdx.x & 31) / GL * GL);
  griddep_wait();
  const kiv_turn &t = a.t;
  const uint32_t tok = blockIdx.x * GROUPS + grp;
  const int r_first = blockIdx.y * a.hc, r_end = min(a.rows[0] + a.rows[1], r_first + a.hc);
  bool live = tok < a.ntok;
  const uint32_t b = APPEND || !live ? 0 : tok / (uint32_t)a.tokens, i = live ? tok - b * (uint32_t)a.tokens : 0;

  // ---- this lane's vectors: the sides of a pair (half-split), else neighbours
  const int half = t.rot_dim / 2;
  const bool rotate = a.turned && t.cos != nullptr;
  const bool lined = t.interleaved ? t.rot_dim % V == 0 : half % V == 0;   // pairs line up with the vectors
  const int hv = rotate && lined && !t.interleaved ? half / V : 0;
  const int va = lane < hv ? lane : 2 * hv + 2 * (lane - hv), vb = lane < hv ? lane + hv : va + 1;
  const bool has_a = live && va < nv, has_b = live && vb < nv;

  const T *src[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) src[k] = static_cast<const T *>(a.in[k].p) + b * a.in[k].stride_b + i * a.in[k].stride_t;
  uint4 ra[RP_UN], rb[RP_UN];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int u = 0; u < RP_UN; ++u) {
      const int r = r0 + u;
      const T *row = r < a.rows[0] ? src[0] + r * a.in[0].stride_h : src[1] + (r - a.rows[0]) * a.in[1].stride_h;
      ra[u] = rb[u] = make_uint4(0, 0, 0, 0);
      if (r < r_end) {
        if (has_a) ra[u] = ld16(row + va * V);
        if (has_b) rb[u] = ld16(row + vb * V);
      }
    }
  };
  fetch(r_first);

  // ---- where the token belongs
  T *dst[2];
  int64_t place = tok;
  if (APPEND) {
    int sb = paged_find_seq(a.pc, (int64_t)blockIdx.x * GROUPS);   // of the block's first token
    while (live && sb < a.pc.batch && (int64_t)a.pc.q_starts[sb + 1] <= (int64_t)tok) ++sb;
    live = live && sb < a.pc.batch && (int64_t)a.pc.q_starts[sb] <= (int64_t)tok;   // else: in no sequence
    if (live) {
      place = (int64_t)a.pc.seq_lens[sb] - a.pc.q_starts[sb + 1] + tok;
      live = place >= 0 && place < a.pc.table_width * a.pc.page_size;
      if (!live && lane == 0) paged_error(a.errors, KIV_ERRBIT_SEQ_LEN);
    }
    dst[0] = dst[1] = nullptr;
    if (live) {
      const uint32_t pi = (uint32_t)place / (uint32_t)a.pc.page_size;
      const int64_t r = (uint32_t)place - pi * (uint32_t)a.pc.page_size;
      const int32_t page = a.pc.block_table[sb * a.pc.table_stride + pi];
      if (page < 0 || page >= a.pc.num_pages) {
        live = false;
        if (lane == 0) paged_error(a.errors, KIV_ERRBIT_BLOCK_TABLE);
      } else {
        dst[0] = static_cast<T *>(a.pc.k) + page * a.pc.k_stride_p + r * a.pc.k_stride_t;
        dst[1] = static_cast<T *>(a.pc.v) + page * a.pc.v_stride_p + r * a.pc.v_stride_t;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) dst[k] = static_cast<T *>(a.out[k].p) + b * a.out[k].stride_b + i * a.out[k].stride_t;
  }

  // ---- cos, sin of this lane's pairs: pair e of (a, b), or, interleaved, pairs
  // e < V / 2 of a and the others of b
  float c[V], s[V];
  bool poison = false, turns = false;          // turns: this lane has pairs
  auto pair_of = [&](int e) { return t.interleaved ? (e < V / 2 ? va * (V / 2) + e : vb * (V / 2) + e - V / 2) : va * V + e; };
  auto row_of = [&](int pair, int64_t row0) -> int64_t {   // of the tables, -1: none
    if (!t.pair_axes) return row0;
    const int ax = t.pair_axes[pair];
    if (ax < 0 || ax >= t.axes) return -1;
    return t.positions ? ld_pos(t, ax, b, i) : place;
  };
  int64_t row0 = place;
  int ax[V];
  if (rotate) {
    const bool f32 = t.cs_dtype == KIV_DTYPE_F32;
    bool bad = false;
    if (live) {
      if (t.positions) row0 = t.pair_axes ? 0 : ld_pos(t, 0, b, i);
      bad = row0 < 0 || row0 >= t.cs_rows;
      if (lined) {
        turns = t.interleaved ? va * V < t.rot_dim : lane < hv;
        const bool both = !t.interleaved || vb * V < t.rot_dim;      // interleaved: b may lie behind the pairs
        bool same = true;                                            // this lane's pairs turn by one row
        if (turns && t.pair_axes) {
          // the axes' positions and the pairs' axes in one round trip
          int64_t at[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) at[k] = t.positions ? (k < t.axes ? ld_pos(t, k, b, i) : -1) : place;
#pragma unroll
          for (int e = 0; e < V; ++e) ax[e] = both || e < V / 2 ? t.pair_axes[pair_of(e)] : -1;
#pragma unroll
          for (int e = 1; e < V; ++e) same = same && ax[e] == ax[0];
          if (same) {
            const int k = ax[0];
            row0 = k < 0 || k >= t.axes ? -1 : !t.positions ? place : k == 0 ? at[0] : k == 1 ? at[1] : k == 2 ? at[2] : k == 3 ? at[3] : ld_pos(t, k, b, i);
            bad = row0 < 0 || row0 >= t.cs_rows;
          }
        }
        if (turns && !bad && a.vec_cs && same && both) {
          ld_vec<T, V>(t.cos, row0 * t.cs_stride + pair_of(0), f32, c);
          ld_vec<T, V>(t.sin, row0 * t.cs_stride + pair_of(0), f32, s);
        } else if (turns && !bad) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            c[e] = 1.f;
            s[e] = 0.f;
            if (both || e < V / 2) {
              const int pair = pair_of(e);
              const int64_t row = row_of(pair, row0);
              if (row < 0 || row >= t.cs_rows) {
                bad = true;
              } else {
                c[e] = ld_as_float<T>(t.cos, row * t.cs_stride + pair, f32);
                s[e] = ld_as_float<T>(t.sin, row * t.cs_stride + pair, f32);
              }
            }
          }
        }
      } else if (!bad && t.pair_axes) {
        for (int pair = lane; pair < half; pair += GL) {
          const int64_t row = row_of(pair, row0);
          bad = bad || row < 0 || row >= t.cs_rows;
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

  float w[NORM ? 2 * V : 1];
  int w_of = -1;   // whose weight is in the registers
  for (int r0 = r_first; r0 < r_first + a.hc; r0 += RP_UN) {       // the same count in every group
    if (r0 > r_first) fetch(r0);
#pragma unroll
    for (int u = 0; u < RP_UN; ++u) {
      if (r0 - r_first + u >= a.hc) break;     // the same in every group
      const int r = r0 + u, which = r < a.rows[0] ? 0 : 1;
      const bool turn = a.turned && !(APPEND && which == 1);
      float x[2 * V];
      Elem<T>::unpack(ra[u], x);
      Elem<T>::unpack(rb[u], x + V);
      if constexpr (NORM) {
        const void *wp = which == 0 && !APPEND ? t.q_weight : t.k_weight;
        if (w_of != which) {
          w_of = which;
          const bool f32 = t.weight_dtype == KIV_DTYPE_F32;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int x0 = (k ? vb : va) * V;
            if (wp && a.vec_w && x0 < D) {
              ld_vec<T, V>(wp, x0, f32, w + k * V);
#pragma unroll
              for (int e = 0; e < V; ++e) w[k * V + e] += t.weight_offset;
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) w[k * V + e] = wp && x0 + e < D ? t.weight_offset + ld_as_float<T>(wp, x0 + e, f32) : 1.f;
            }
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(KIV_FULL_MASK, ss, o);
        const float rs = rsqrtf(ss / (float)D + t.eps);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) x[e] = x[e] * rs * w[e];
      }
      if (rotate && !lined) {
        // any pair of any row of the tables: through shared memory, an element at a time
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) s_row[grp][((e < V ? va : vb) * V + e % V) % (GL * 2 * V)] = x[e];
        __syncwarp();
        if (turn && live && !poison) {
          const bool f32 = t.cs_dtype == KIV_DTYPE_F32;
#pragma unroll 1
          for (int e = 0; e < 2 * V; ++e) {
            const int xi = (e < V ? va : vb) * V + e % V;
            if (xi >= t.rot_dim) continue;
            const int pair = t.interleaved ? xi >> 1 : (xi < half ? xi : xi - half);
            const bool second = t.interleaved ? (xi & 1) != 0 : xi >= half;
            const int64_t row = row_of(pair, row0);
            const float cc = ld_as_float<T>(t.cos, row * t.cs_stride + pair, f32);
            const float sn = ld_as_float<T>(t.sin, row * t.cs_stride + pair, f32);
            const float me = s_row[grp][xi], other = s_row[grp][t.interleaved ? xi ^ 1 : (second ? xi - half : xi + half)];
            const float y = fmaf(me, cc, second ? other * sn : -other * sn);
#pragma unroll
            for (int k = 0; k < 2 * V; ++k)
              if (k == e) x[k] = y;
          }
        }
      } else if (turn && turns) {
        if (t.interleaved) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float p = x[2 * e], q = x[2 * e + 1];
            if (e < V / 2 || vb * V < t.rot_dim) {
              x[2 * e] = p * c[e] - q * s[e];
              x[2 * e + 1] = q * c[e] + p * s[e];
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float p = x[e], q = x[V + e];
            x[e] = p * c[e] - q * s[e];
            x[V + e] = q * c[e] + p * s[e];
          }
        }
      }
      if (poison && turn) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) x[e] = __int_as_float(0x7fc00000);
      }
      if (live && r < r_end) {
        T *row;
        if (APPEND)
          row = which == 0 ? dst[0] + r * a.pc.k_stride_h : dst[1] + (r - a.rows[0]) * a.pc.v_stride_h;
        else
          row = which == 0 ? dst[0] + r * a.out[0].stride_h : dst[1] + (r - a.rows[0]) * a.out[1].stride_h;
        if (va < nv) st16(row + va * V, turn ? Elem<T>::pack(x) : ra[u]);
        if (vb < nv) st16(row + vb * V, turn ? Elem<T>::pack(x + V) : rb[u]);
      }
    }
  }
}

template <typename T, bool APPEND>
static kiv_status launch_turn(TurnArgs a, int64_t tokens, cudaStream_t s) {
  constexpr int V = Elem<T>::V;
  const int lanes = (a.head_dim / V + 1) / 2;
  const int total = a.rows[0] + a.rows[1];
  const int gl = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32, groups = RP_THREADS / gl;
  // Heads per group: many rows share a load of cos and sin, few keep the SMs
  // filled -- two blocks on each, down to one row per group, where the call is
  // one chain of loads
  a.hc = 16;
  while (a.hc > 1 && ceil_div(tokens, groups) * ceil_div(total, a.hc) < (int64_t)2 * sm_count()) a.hc /= 2;
  while (ceil_div(total, a.hc) > 65535) a.hc *= 2;
  a.ntok = (uint32_t)tokens;
  const dim3 grid((unsigned)ceil_div(tokens, groups), (unsigned)ceil_div(total, a.hc));
  auto lines = [](const void *p, int dtype) {   // V values from p on, and from multiples of V on
    return reinterpret_cast<uintptr_t>(p) % std::min<int64_t>(16, (int64_t)V * elem_bytes(dtype)) == 0;
  };
  const kiv_turn &t = a.t;
  a.vec_cs = t.cos && lines(t.cos, t.cs_dtype) && lines(t.sin, t.cs_dtype) && t.cs_stride % V == 0;
  a.vec_w = (!t.q_weight || lines(t.q_weight, t.weight_dtype)) && (!t.k_weight || lines(t.k_weight, t.weight_dtype));
  cudaError_t e;
#define KIV_TURN(GL)                                                                                               \
  (a.turned && t.norm ? launch_pdl(turn_kernel<T, GL, APPEND, true>, grid, dim3(RP_THREADS), 0, s, 1, a)           \
                      : launch_pdl(turn_kernel<T, GL, APPEND, false>, grid, dim3(RP_THREADS), 0, s, 1, a))
  if (gl == 4) e = KIV_TURN(4);
  else if (gl == 8) e = KIV_TURN(8);
  else if (gl == 16) e = KIV_TURN(16);
  else e = KIV_TURN(32);
#undef KIV_TURN
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
