// Append to a paged KV cache with the q/k prologue applied on the way, one launch for a ragged batch.
//
// For token t of sequence b (own position o = kv_len[b] - n_b + i, rotary position p = prefix + o):
//   y = x / sqrt(mean(x^2) + eps) * gamma            (gamma given)
//   r[d] = y[d] cos[p][d] + h[d] sin[p][d],  h = (-y[d + rot/2] | y[d - rot/2])   for d < rot
//   q_out = r(q);  K[slot] = codec(r(k));  V[slot] = codec(v)
// Bound: HBM for prompts (each source read once, each result written once), launch and the dependent
// lookups (offsets -> length -> page) for single tokens.
//
// append_pairs_kernel takes a rotation apart into pairs that one lane owns: a lane has four dims d and the
// four partners d + rot/2 (dims behind rot are paired among themselves, with cos = 1 and sin = 0), so that
// nothing is exchanged between lanes but the row's sum of squares and the block maxima of q8.  With the norm
// folded into the rotation's factors (gamma * cos and gamma * sin, once per token) a value costs three
// instructions:  r_a = inv (x_a (g_a c_a) - x_b (g_b s_a)),  r_b = inv (x_b (g_b c_b) + x_a (g_a s_b)).
// A warp has rows of one token and one kind (q, k or v); it issues the source loads before its lookups and
// the next rows' loads before it works on these.  7424 tokens of 32 q and 8 kv heads, f16 into a q8 cache:
// 51 us (97 us with contiguous values per lane and exchanged partners, all kinds in a warp), 3.4 TB/s.
// append_kernel is the form for everything else: rotation widths that are not multiples of 8, q8 blocks that a
// pair's halves would share, and sources that do not start on 16-byte boundaries.
#include <type_traits>

#include "paged.h"

namespace bg {
namespace {

static __device__ int g_append_error = 0;

template <typename T, int N>
__device__ __forceinline__ void load_row(const T *src, bool vec, float (&x)[N]) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      load_f32<N>(src, x);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = src[i];
    }
  } else {
    if (vec) {
      load_f16<N>(src, x);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __half2float(src[i]);
    }
  }
}

template <int N>
__device__ __forceinline__ void store_f32(float *dst, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}

template <int N>
__device__ __forceinline__ void store_f16(__half *dst, const float (&x)[N]) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    __half2 h = __floats2half2_rn(x[i], x[i + 1]);
    w[i / 2] = *reinterpret_cast<uint32_t *>(&h);
  }
  if constexpr (N == 8) *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
}

// snorm8_encode(v, s) with |v| <= s and r = 1 / s rounded: the correctly rounded quotient by one product, its
// exact remainder and one correction (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000", 1990: correct where r is the rounded reciprocal), instead of a division per value.  A
// remainder that underflows belongs to a quotient far below half a code.
__device__ __forceinline__ uint32_t encode(float v, float s, float r) {
  const float q = v * r, e = fmaf(fmaf(-q, s, v), r, q);
  return (uint32_t)(uint8_t)(int8_t)(int)floorf(0.5f + 127.0f * fminf(fmaxf(e, -1.0f), 1.0f));
}

template <typename SRC, int D>
struct ApCfg {
  static constexpr int EPL = sizeof(SRC) == 2 || D == 256 ? 8 : 4;  // values per lane
  static constexpr int LPR = D / EPL;                               // lanes per row
  static constexpr int RPW = 32 / LPR;                              // rows per warp pass
  static constexpr int U = 2;                                       // passes of one task
};

// Rotary position of token t and the pool row (before the kv-head factor) of its slot, -1 where it has no page
// (then q alone is written).  False: the token is padding, or its length or the tables leave it no position.
__device__ __forceinline__ bool place_token(const PagedAppendArgs &a, uint32_t t, uint32_t lane, uint32_t &pos,
                                            int64_t &slot) {
  const int32_t b = find_seq_warp(a.bv, t, lane);
  if (b < 0) return false;
  uint32_t begin = t, n = 1;
  if (a.bv.cu_q) {
    begin = (uint32_t)__ldg(a.bv.cu_q + b);
    n = (uint32_t)__ldg(a.bv.cu_q + b + 1) - begin;
  }
  const int32_t o = __ldg(a.bv.kv_len + b) - (int32_t)n + (int32_t)(t - begin);
  if (o < 0) return false;
  pos = a.bv.prefix_len + (uint32_t)o;
  if (a.cosT && pos >= a.table_rows) {
    if (lane == 0) atomicExch(&g_append_error, BG_EINVAL);
    return false;
  }
  slot = -1;
  if ((uint32_t)o / a.kv.page_size < a.bv.table_stride)
    slot = paged_row(a.kv, a.bv.table + (uint64_t)b * a.bv.table_stride, (uint32_t)o);
  if (slot < 0 && lane == 0) atomicExch(&g_append_error, BG_EINVAL);
  return true;
}

// ---- pairs ---------------------------------------------------------------------------------------
struct PairPlan {
  uint32_t tq, tk;      // warps per token for q, and for k (as many for v)
  uint32_t passes;      // passes of a warp
};

// Four source values as they are loaded, and as floats.
template <typename SRC>
struct Raw4;
template <>
struct Raw4<float> {
  float4 v = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void load(const float *p) { v = __ldg(reinterpret_cast<const float4 *>(p)); }
  __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
template <>
struct Raw4<__half> {
  uint2 v = {0u, 0u};
  __device__ __forceinline__ void load(const __half *p) { v = __ldg(reinterpret_cast<const uint2 *>(p)); }
  __device__ __forceinline__ void get(float (&x)[4]) const {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
};

__device__ __forceinline__ void store4(float *p, const float (&x)[4]) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__half *p, const float (&x)[4]) {
  __half2 u = __floats2half2_rn(x[0], x[1]), v = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&u), *reinterpret_cast<uint32_t *>(&v));
}

// Four values of one 32-value block (eight lanes' together) as q8 codes; the first of the lanes stores the scale.
__device__ __forceinline__ void store4_q8(int8_t *p, float *scale, bool first, const float (&x)[4], bool live) {
  float am = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
  for (int m = 4; m > 0; m >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, m));
  const float s = fmaxf(am, 1e-30f), r = __frcp_rn(s);
  if (!live) return;
  *reinterpret_cast<uint32_t *>(p) =
      encode(x[0], s, r) | encode(x[1], s, r) << 8 | encode(x[2], s, r) << 16 | encode(x[3], s, r) << 24;
  if (first) *scale = s;
}

template <typename SRC, int D, int MODE>
__global__ void __launch_bounds__(128) append_pairs_kernel(PagedAppendArgs a, PairPlan pl) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, U = 2;
  const uint32_t lane = threadIdx.x & 31, per = pl.tq + 2 * pl.tk;
  const uint64_t task = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t t = (uint32_t)(task / per), w = (uint32_t)(task % per);
  if (t >= a.bv.T) return;
  const uint32_t kind = w < pl.tq ? 0 : w < pl.tq + pl.tk ? 1 : 2;  // q, k, v: the same for the whole warp
  const uint32_t heads = kind == 0 ? a.H : a.kv.KV;
  uint32_t row = (kind == 0 ? w : (w - pl.tq) % pl.tk) * pl.passes * RPW + lane / LPR;
  const uint32_t end = min(heads, row - lane / LPR + pl.passes * RPW);
  const uint64_t hs = kind == 0 ? a.q_hs : kind == 1 ? a.k_hs : a.v_hs;
  const SRC *src = static_cast<const SRC *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                   t * (kind == 0 ? a.q_ts : kind == 1 ? a.k_ts : a.v_ts);
  // this lane's dims: a .. a + 3 and their partners b .. b + 3
  const uint32_t i = lane % LPR, half = a.rot / 2, turned = half / 4;
  const uint32_t da = i < turned ? 4 * i : a.rot + 4 * (i - turned);
  const uint32_t db = i < turned ? da + half : da + (D - a.rot) / 2;
  // the rows' source values; the next rows' are under way while these are worked on
  Raw4<SRC> cur[U][2], nxt[U][2];
  auto load = [&](Raw4<SRC> (&x)[U][2], uint32_t first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = first + u * RPW;
      if (r < end) {
        x[u][0].load(src + r * hs + da);
        x[u][1].load(src + r * hs + db);
      }
    }
  };
  load(cur, row);

  uint32_t pos;
  int64_t slot;
  if (!place_token(a, t, lane, pos, slot)) return;

  // gamma * cos and gamma * sin of this token
  const float *gamma = kind == 0 ? a.q_gamma : kind == 1 ? a.k_gamma : nullptr;
  float fa[4], fb[4], ga[4], gb[4];  // r_a = x_a fa - x_b ga,  r_b = x_b fb + x_a gb
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fa[j] = fb[j] = 1.f;
    ga[j] = gb[j] = 0.f;
  }
  if (kind < 2) {
    if (i < turned) {
      const float *c = a.cosT + (uint64_t)pos * a.rot, *s = a.sinT + (uint64_t)pos * a.rot;
      load_f32<4>(c + da, fa);
      load_f32<4>(c + db, fb);
      load_f32<4>(s + da, ga);
      load_f32<4>(s + db, gb);
    }
    if (gamma) {
      float na[4], nb[4];
      load_f32<4>(gamma + da, na);
      load_f32<4>(gamma + db, nb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fa[j] *= na[j];
        ga[j] *= nb[j];
        fb[j] *= nb[j];
        gb[j] *= na[j];
      }
    }
  }
  for (;;) {
    load(nxt, row + U * RPW);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = row + u * RPW;
      const bool live = r < end;
      float x[2][4];
      cur[u][0].get(x[0]);
      cur[u][1].get(x[1]);
      float inv = 1.f;
      if (gamma) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(x[0][j], x[0][j], fmaf(x[1][j], x[1][j], ss));
#pragma unroll
        for (int m = LPR / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        inv = rsqrtf(ss * (1.0f / D) + a.eps);
      }
      float ya[4], yb[4];
      if (kind < 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ya[j] = inv * fmaf(x[0][j], fa[j], -(x[1][j] * ga[j]));
          yb[j] = inv * fmaf(x[1][j], fb[j], x[0][j] * gb[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ya[j] = x[0][j];
          yb[j] = x[1][j];
        }
      }
      if (kind == 0) {
        if (!live) continue;
        const uint64_t off = ((uint64_t)t * a.H + r) * D;
        if (a.out_f16) {
          store4(static_cast<__half *>(a.q_out) + off + da, ya);
          store4(static_cast<__half *>(a.q_out) + off + db, yb);
        } else {
          store4(static_cast<float *>(a.q_out) + off + da, ya);
          store4(static_cast<float *>(a.q_out) + off + db, yb);
        }
      } else if (slot >= 0) {
        void *dst = kind == 1 ? a.kv.K : a.kv.V;
        const uint64_t at = (uint64_t)slot * a.kv.KV + r, off = at * D;
        if constexpr (MODE == BG_KV_Q8) {
          int8_t *p = static_cast<int8_t *>(dst) + off;
          float *s = (kind == 1 ? a.kv.Ks : a.kv.Vs) + at * (D / 32);
          store4_q8(p + da, s + da / 32, (lane & 7) == 0, ya, live);
          store4_q8(p + db, s + db / 32, (lane & 7) == 0, yb, live);
        } else {
          if (!live) continue;
          using OUT = typename std::conditional<MODE == BG_KV_F32, float, __half>::type;
          store4(static_cast<OUT *>(dst) + off + da, ya);
          store4(static_cast<OUT *>(dst) + off + db, yb);
        }
      }
    }
    row += U * RPW;
    if (row - lane / LPR >= end) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      cur[u][0] = nxt[u][0];
      cur[u][1] = nxt[u][1];
    }
  }
}

template <typename SRC, int D, int MODE>
__global__ void __launch_bounds__(128) append_kernel(PagedAppendArgs a, uint32_t tasks_per_token, int vec) {
  using C = ApCfg<SRC, D>;
  constexpr int EPL = C::EPL, LPR = C::LPR, RPW = C::RPW, U = C::U;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t task = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t t = (uint32_t)(task / tasks_per_token), grp = (uint32_t)(task % tasks_per_token);
  if (t >= a.bv.T) return;
  const uint32_t Hq = a.q ? a.H : 0, KV = a.kv.KV, NR = Hq + 2 * KV;
  const uint32_t sub = lane / LPR, li = lane % LPR, d0 = li * EPL;

  // rows of this task: kind 0 = q, 1 = k, 2 = v, 3 = none
  float x[U][EPL];
  uint32_t kind[U], head[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = (grp * U + u) * RPW + sub;
    kind[u] = r < Hq ? 0 : r < Hq + KV ? 1 : r < NR ? 2 : 3;
    head[u] = r < Hq ? r : r < Hq + KV ? r - Hq : r - Hq - KV;
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[u][i] = 0.f;
    if (kind[u] < 3) {
      const SRC *base = static_cast<const SRC *>(kind[u] == 0 ? a.q : kind[u] == 1 ? a.k : a.v);
      const uint64_t ts = kind[u] == 0 ? a.q_ts : kind[u] == 1 ? a.k_ts : a.v_ts;
      const uint64_t hs = kind[u] == 0 ? a.q_hs : kind[u] == 1 ? a.k_hs : a.v_hs;
      load_row<SRC, EPL>(base + t * ts + head[u] * hs + d0, vec, x[u]);
    }
  }

  uint32_t pos;
  int64_t slot;
  if (!place_token(a, t, lane, pos, slot)) return;

  // this lane's rotation factors, shared by all rows of the token
  float c[EPL], s[EPL];
  const uint32_t half = a.rot / 2;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (a.cosT) {
    const float *cp = a.cosT + (uint64_t)pos * a.rot, *sp = a.sinT + (uint64_t)pos * a.rot;
    if (d0 + EPL <= a.rot && (a.rot & 3) == 0) {
      load_f32<EPL>(cp + d0, c);
      load_f32<EPL>(sp + d0, s);
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (d0 + i < a.rot) {
          c[i] = __ldg(cp + d0 + i);
          s[i] = __ldg(sp + d0 + i);
        }
    }
  }
  const bool by_lane = half % EPL == 0;  // the partner values are another lane's, in the same order
  const uint32_t partner = sub * LPR + (d0 < half ? li + half / EPL : li - half / EPL) % LPR;

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float *gamma = kind[u] == 0 ? a.q_gamma : kind[u] == 1 ? a.k_gamma : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) ss = fmaf(x[u][i], x[u][i], ss);
#pragma unroll
    for (int m = LPR / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    if (gamma) {
      const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[u][i] = x[u][i] * inv * __ldg(gamma + d0 + i);
    }
    float y[EPL];
    if (by_lane) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float p = __shfl_sync(0xffffffffu, x[u][i], partner);
        const float h = d0 < half ? -p : p;
        // two products and one sum, each rounded: what the formula says, not a fused form of it
        y[i] = kind[u] < 2 && d0 + i < a.rot ? __fadd_rn(__fmul_rn(x[u][i], c[i]), __fmul_rn(h, s[i])) : x[u][i];
      }
    } else {
      // a rotation width whose half is not a whole number of lanes: fetch each partner on its own
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const uint32_t d = d0 + i, pd = d < half ? d + half : d - half;
        float p = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const float v = __shfl_sync(0xffffffffu, x[u][j], sub * LPR + (pd / EPL) % LPR);
          if (pd % EPL == j) p = v;
        }
        const float h = d < half ? -p : p;
        y[i] = kind[u] < 2 && d < a.rot ? __fadd_rn(__fmul_rn(x[u][i], c[i]), __fmul_rn(h, s[i])) : x[u][i];
      }
    }
    // q8 block scale: the largest magnitude of 32 values, which 32 / EPL neighbouring lanes hold
    float am = 0.f;
    if constexpr (MODE == BG_KV_Q8) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) am = fmaxf(am, fabsf(y[i]));
#pragma unroll
      for (int m = 16 / EPL; m > 0; m >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, m));
    }
    if (kind[u] == 0) {
      const uint64_t off = ((uint64_t)t * a.H + head[u]) * D + d0;
      if (a.out_f16) store_f16<EPL>(static_cast<__half *>(a.q_out) + off, y);
      else store_f32<EPL>(static_cast<float *>(a.q_out) + off, y);
    } else if (kind[u] < 3 && slot >= 0) {
      const uint64_t row = (uint64_t)slot * KV + head[u], off = row * D + d0;
      void *dst = kind[u] == 1 ? a.kv.K : a.kv.V;
      if constexpr (MODE == BG_KV_F32) {
        store_f32<EPL>(static_cast<float *>(dst) + off, y);
      } else if constexpr (MODE == BG_KV_F16) {
        store_f16<EPL>(static_cast<__half *>(dst) + off, y);
      } else {
        const float sc = fmaxf(am, 1e-30f), rc = __frcp_rn(sc);
        uint32_t w[EPL / 4] = {};
#pragma unroll
        for (int i = 0; i < EPL; ++i) w[i / 4] |= encode(y[i], sc, rc) << (8 * (i % 4));
        int8_t *d = static_cast<int8_t *>(dst) + off;
        if constexpr (EPL == 8) *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(d) = w[0];
        if (d0 % 32 == 0) (kind[u] == 1 ? a.kv.Ks : a.kv.Vs)[row * (D / 32) + d0 / 32] = sc;
      }
    }
  }
}

template <typename SRC, int D>
int launch_pairs(const PagedAppendArgs &a, cudaStream_t st) {
  constexpr uint32_t RPW = 32 / (D / 8), U = 2;
  const uint32_t H = a.q ? a.H : 0, KV = a.kv.KV;
  // passes per warp: the lookups cost three dependent loads, so up to 8 where that leaves 64 warps for every SM
  // (7424 tokens, f16 into q8: 2 passes 91 us, 4 62 us, 8 51 us, 16 56 us; 1321 of head_dim 256: 4 18.8, 8 21.3)
  const uint64_t least = (uint64_t)a.bv.T * ((H + RPW * U - 1) / (RPW * U) + 2 * ((KV + RPW * U - 1) / (RPW * U)));
  uint32_t passes = U;
  while (passes < 8 && least * U / (2 * passes) >= 148 * 64) passes *= 2;
  PairPlan pl;
  pl.passes = passes;
  pl.tq = (H + RPW * passes - 1) / (RPW * passes);
  pl.tk = (KV + RPW * passes - 1) / (RPW * passes);
  const uint64_t blocks = ((uint64_t)a.bv.T * (pl.tq + 2 * pl.tk) + 3) / 4;
  if (blocks > 0x7fffffffull) return BG_EUNSUPPORTED;
  switch (a.mode) {
    case BG_KV_F32: append_pairs_kernel<SRC, D, BG_KV_F32><<<(unsigned)blocks, 128, 0, st>>>(a, pl); break;
    case BG_KV_F16: append_pairs_kernel<SRC, D, BG_KV_F16><<<(unsigned)blocks, 128, 0, st>>>(a, pl); break;
    case BG_KV_Q8: append_pairs_kernel<SRC, D, BG_KV_Q8><<<(unsigned)blocks, 128, 0, st>>>(a, pl); break;
    default: return BG_EUNSUPPORTED;
  }
  return cudaGetLastError() == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

template <typename SRC, int D>
int launch_mode(const PagedAppendArgs &a, cudaStream_t st) {
  using C = ApCfg<SRC, D>;
  const uint32_t NR = (a.q ? a.H : 0) + 2 * a.kv.KV, per = C::RPW * C::U;
  const uint32_t tpt = (NR + per - 1) / per;
  const uint64_t blocks = ((uint64_t)a.bv.T * tpt + 3) / 4;
  if (blocks > 0x7fffffffull) return BG_EUNSUPPORTED;
  // 16-byte loads need every row of every source to start on a 16-byte boundary
  constexpr uint64_t per16 = 16 / sizeof(SRC);
  const uint64_t strides = a.k_ts | a.k_hs | a.v_ts | a.v_hs | (a.q ? a.q_ts | a.q_hs : 0);
  const uintptr_t ptrs = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q;
  const int vec = strides % per16 == 0 && ptrs % 16 == 0;
  const uintptr_t gammas = (uintptr_t)a.q_gamma | (uintptr_t)a.k_gamma;
  if (vec && gammas % 16 == 0 && a.rot % 8 == 0 && (a.mode != BG_KV_Q8 || (a.rot % 64 == 0 && (D - a.rot) % 64 == 0)))
    return launch_pairs<SRC, D>(a, st);
  switch (a.mode) {
    case BG_KV_F32: append_kernel<SRC, D, BG_KV_F32><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
    case BG_KV_F16: append_kernel<SRC, D, BG_KV_F16><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
    case BG_KV_Q8: append_kernel<SRC, D, BG_KV_Q8><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
    default: return BG_EUNSUPPORTED;
  }
  return cudaGetLastError() == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

}  // namespace

int launch_paged_append(const PagedAppendArgs &a, cudaStream_t st) {
  switch (a.D) {
    case 64: return a.src_f16 ? launch_mode<__half, 64>(a, st) : launch_mode<float, 64>(a, st);
    case 128: return a.src_f16 ? launch_mode<__half, 128>(a, st) : launch_mode<float, 128>(a, st);
    case 256: return a.src_f16 ? launch_mode<__half, 256>(a, st) : launch_mode<float, 256>(a, st);
    default: return BG_EUNSUPPORTED;
  }
}

int poll_device_error_paged_append() {
  int v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_append_error, sizeof(int)) != cudaSuccess) return BG_ELAUNCH;
  if (v) cudaMemcpyToSymbol(g_append_error, &z, sizeof(int));
  return v;
}

}  // namespace bg
