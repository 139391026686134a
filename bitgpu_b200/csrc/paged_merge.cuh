// Log-sum-exp join of partial attention rows, one warp per (row, slice of pieces).
//
// A partial row is (o[D], m, l): o = sum_j 2^(s_j - m) V_j and l = sum_j 2^(s_j - m) over the positions
// of the piece, s_j the scores in log2 units; a piece that attends nothing has l = 0 (its o is not
// read).  Joined:  M = max m,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
#pragma once
#include "common.cuh"

namespace bg {

// Join pieces first, first + step, ... < n of one row; piece k's row index comes from `at(k)`.  The
// lane owns columns 4*lane + 128*j.  Weights of 32 pieces at a time are fetched lane-parallel, and the
// rows in batches of four, so the warp waits for memory once per batch.
template <int D, typename At>
__device__ __forceinline__ void join_pieces(const float *po, const float2 *pml, uint32_t first, uint32_t step, uint32_t n,
                                            uint32_t lane, At at, float (&acc)[(D + 127) / 128][4], float &M, float &L) {
  constexpr int NJ = (D + 127) / 128;
  M = -INFINITY;
  L = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  const bool mine = D >= 128 || lane * 4 < D;
  for (uint32_t k0 = first; k0 < n; k0 += 32 * step) {
    const uint32_t k = k0 + lane * step;
    float2 ml = make_float2(-INFINITY, 0.f);
    uint64_t idx = 0;
    if (k < n) {
      idx = at(k);
      ml = __ldcg(pml + idx);
    }
    const bool some = ml.y != 0.f;  // a sum that is not a number counts: it has to reach the result
    const float m = some ? ml.x : -INFINITY;
    float mx = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(M, mx);
    if (mn == -INFINITY) continue;  // nothing attended so far (the same on every lane)
    const float corr = exp2f(M - mn), w = some ? exp2f(m - mn) : 0.f;
    M = mn;
    float lw = some ? w * ml.y : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
    L = fmaf(L, corr, lw);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] *= corr;
    const uint32_t cnt = min(32u, (n - k0 + step - 1) / step);
    for (uint32_t c0 = 0; c0 < cnt; c0 += 4) {
      float4 v[4][NJ];
      float ws[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ws[u] = __shfl_sync(0xffffffffu, w, (c0 + u) & 31);
        if (c0 + u >= cnt) ws[u] = 0.f;
        const uint64_t id = __shfl_sync(0xffffffffu, idx, (c0 + u) & 31);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          v[u][j] = ws[u] != 0.f && mine ? __ldcg(reinterpret_cast<const float4 *>(po + id * D) + lane + 32 * j)
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          acc[j][0] = fmaf(v[u][j].x, ws[u], acc[j][0]);
          acc[j][1] = fmaf(v[u][j].y, ws[u], acc[j][1]);
          acc[j][2] = fmaf(v[u][j].z, ws[u], acc[j][2]);
          acc[j][3] = fmaf(v[u][j].w, ws[u], acc[j][3]);
        }
    }
  }
}

// 1 / (1 + exp(-g)) to 7 * 2^-24 of its value (two units for the exponential, the sum, one unit for the reciprocal), and
// 0 from -88 on, where it is below 2^-126.  The product g log2(e) comes in two parts, log2(e) in two numbers, so that
// its rounding does not grow with |g|.  One arithmetic for every paged kernel.  (The tcgen05 kernel's threads have
// head_dim of them each: 7 gated prompts of 899 tokens, head_dim 256, take 187 us, with expf and a division 327.)
__device__ __forceinline__ float sigmoid(float g) {
  float p, r;
  asm("{\n .reg .f32 t;\n max.NaN.f32 t, %1, 0fC2B00000;\n min.NaN.f32 %0, t, 0f42B00000;\n}\n" : "=f"(g) : "f"(g));  // +-88
  const float x = -kLog2e * g, rest = fmaf(g, -1.92596299e-8f, fmaf(-kLog2e, g, -x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(x));
  p = fmaf(p, rest * kLn2, p);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + p));
  return r;
}

// Four consecutive columns of one output row: out = o / L, times the sigmoid gate.
__device__ __forceinline__ void write_out4(void *out, int out_f16, const float *gate, uint64_t off, const float (&o)[4],
                                           float L) {
  const float inv = L != 0.f ? 1.0f / L : 0.f;  // a row that attends nothing is zero
  float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if (gate) {
    const float4 g = __ldg(reinterpret_cast<const float4 *>(gate + off));
    v[0] *= sigmoid(g.x);
    v[1] *= sigmoid(g.y);
    v[2] *= sigmoid(g.z);
    v[3] *= sigmoid(g.w);
  }
  if (out_f16) {
    __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(static_cast<__half *>(out) + off) =
        make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
  } else {
    *reinterpret_cast<float4 *>(static_cast<float *>(out) + off) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// The whole block joins one row's n pieces (warps take every (blockDim / 32)-th piece) and writes it.
// `sm`: (blockDim / 32) * (D + 2) floats.
template <int D, int NW, typename At>
__device__ __forceinline__ void join_row_block(const float *po, const float2 *pml, uint32_t n, At at, float *sm, void *out,
                                               int out_f16, const float *gate, uint64_t off) {
  constexpr int NJ = (D + 127) / 128;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float acc[NJ][4], M, L;
  join_pieces<D>(po, pml, warp, NW, n, lane, at, acc, M, L);
  float *ml = sm + NW * D;
  if (lane == 0) {
    ml[2 * warp] = M;
    ml[2 * warp + 1] = L;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if (D >= 128 || lane * 4 < D)
      *reinterpret_cast<float4 *>(sm + warp * D + 4 * lane + 128 * j) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
  __syncthreads();
  for (uint32_t d = threadIdx.x * 4; d < D; d += NW * 128) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, ml[2 * w]);
    float o[4] = {0.f, 0.f, 0.f, 0.f}, Ls = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = ml[2 * w] > -INFINITY ? exp2f(ml[2 * w] - mx) : 0.f;
      Ls = fmaf(ml[2 * w + 1], f, Ls);
      const float4 v = *reinterpret_cast<const float4 *>(sm + w * D + d);
      o[0] = fmaf(v.x, f, o[0]);
      o[1] = fmaf(v.y, f, o[1]);
      o[2] = fmaf(v.z, f, o[2]);
      o[3] = fmaf(v.w, f, o[3]);
    }
    write_out4(out, out_f16, gate, off + d, o, Ls);
  }
}

}  // namespace bg
