// Append to a paged KV cache with the q/k prologue applied on the way, one launch for a ragged batch.
//
// For token t of sequence b (own position o = kv_len[b] - n_b + i, rotary position p = prefix + o):
//   y = x / sqrt(mean(x^2) + eps) * gamma            (gamma given)
//   r[d] = y[d] cos[p][d] + h[d] sin[p][d],  h = (-y[d + rot/2] | y[d - rot/2])   for d < rot
//   q_out = r(q);  K[slot] = codec(r(k));  V[slot] = codec(v)
// Bound: HBM for prompts (each source read once, each result written once), launch and the dependent
// lookups (offsets -> length -> page) for single tokens.  So a row of head_dim values is spread over as
// many lanes as give each one 16 bytes of the source, a warp takes two groups of rows of ONE token
// (its lookups and its cos / sin values are fetched once for all of them), and the source loads are
// issued before the lookups.  The rotation's partner value sits a fixed number of lanes away.
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

template <typename SRC, int D>
struct ApCfg {
  static constexpr int EPL = sizeof(SRC) == 2 || D == 256 ? 8 : 4;  // values per lane
  static constexpr int LPR = D / EPL;                               // lanes per row
  static constexpr int RPW = 32 / LPR;                              // rows per warp pass
  static constexpr int U = 2;                                       // passes of one task
};

template <typename SRC, int D, int MODE>
__global__ void __launch_bounds__(128) paged_append_kernel(PagedAppendArgs a, uint32_t tasks_per_token, int vec) {
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

  // where the token belongs
  const int32_t b = find_seq_warp(a.bv, t, lane);
  if (b < 0) return;  // a row behind the last sequence
  int32_t o;
  {
    uint32_t begin = t, n = 1;
    if (a.bv.cu_q) {
      begin = (uint32_t)__ldg(a.bv.cu_q + b);
      n = (uint32_t)__ldg(a.bv.cu_q + b + 1) - begin;
    }
    o = __ldg(a.bv.kv_len + b) - (int32_t)n + (int32_t)(t - begin);
  }
  if (o < 0) return;  // the length leaves no position for this token
  const uint32_t pos = a.bv.prefix_len + (uint32_t)o;
  if (a.cosT && pos >= a.table_rows) {
    if (lane == 0) atomicExch(&g_append_error, BG_EINVAL);
    return;
  }
  int64_t slot = -1;
  if ((uint32_t)o / a.kv.page_size < a.bv.table_stride)
    slot = paged_row(a.kv, a.bv.table + (uint64_t)b * a.bv.table_stride, (uint32_t)o);
  if (slot < 0 && lane == 0) atomicExch(&g_append_error, BG_EINVAL);  // no such page: q only

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
        const float sc = fmaxf(am, 1e-30f);
        uint32_t w[EPL / 4] = {};
#pragma unroll
        for (int i = 0; i < EPL; ++i) w[i / 4] |= (uint32_t)(uint8_t)snorm8_encode(y[i], sc) << (8 * (i % 4));
        int8_t *d = static_cast<int8_t *>(dst) + off;
        if constexpr (EPL == 8) *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(d) = w[0];
        if (d0 % 32 == 0) (kind[u] == 1 ? a.kv.Ks : a.kv.Vs)[row * (D / 32) + d0 / 32] = sc;
      }
    }
  }
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
  switch (a.mode) {
    case BG_KV_F32: paged_append_kernel<SRC, D, BG_KV_F32><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
    case BG_KV_F16: paged_append_kernel<SRC, D, BG_KV_F16><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
    case BG_KV_Q8: paged_append_kernel<SRC, D, BG_KV_Q8><<<(unsigned)blocks, 128, 0, st>>>(a, tpt, vec); break;
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
