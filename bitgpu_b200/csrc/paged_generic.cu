// Ragged attention over a paged cache on the CUDA cores: every cache type (f32, f16, q8), head size and
// page size, any number of query heads per kv head, an optional shared prefix in front of the own
// positions.  It is the kernel of f32 caches and the fallback of the tensor-core ones.
//
//   out[t][h] = sum_j p_j V[j],  p_j = 2^(s_j - m) / sum,  s_j = q . K[j] * scale * log2(e)
//   over j in the prefix and the own positions up to the token's own.
//
// One block of four warps serves one token and up to four query heads of one kv head.  A warp takes
// eight positions at a time: each lane multiplies its head_dim / 32 dims for the 8 x 4 (position, head)
// pairs, and the 32 partial dots are reduced together -- five exchange steps that halve the number of
// values, 31 shuffles for 32 sums -- which leaves pair (head = lane / 8, position = lane % 8) in its
// own lane, where the running maximum and sum of the softmax are kept.  Bound: issue (about 450 slots for 8
// positions of head_dim 128): 32 streams of up to 8192 positions over an f32 pool 478 us, 2.2 TB/s, a third of the copy's
// rate; head_dim 64 366 us (f16 371, q8 851).  Nothing is shared between tokens: one prompt of 2048 takes 3510 us.
#include "paged.h"
#include "paged_merge.cuh"

namespace bg {
namespace {

static __device__ int g_generic_error = 0;

constexpr int kHeads = 4;  // query heads per block
constexpr int kPos = 8;    // positions per warp step

template <int DPL, int MODE>
__device__ __forceinline__ void load_kv(const void *data, const float *scales, uint64_t row, uint32_t lane,
                                        float (&x)[DPL]) {
  constexpr int D = DPL * 32;
  const uint64_t off = row * D + lane * DPL;
  if constexpr (MODE == BG_KV_F32) {
    load_f32<DPL>(static_cast<const float *>(data) + off, x);
  } else if constexpr (MODE == BG_KV_F16) {
    load_f16<DPL>(static_cast<const __half *>(data) + off, x);
  } else {
    int8_t c[DPL];
    load_i8<DPL>(static_cast<const int8_t *>(data) + off, c);
    const float s = __ldg(scales + row * (D / 32) + lane * DPL / 32);
#pragma unroll
    for (int i = 0; i < DPL; ++i) x[i] = snorm8(c[i]) * s;
  }
}

template <int DPL, int MODE>
__global__ void __launch_bounds__(128) paged_generic_kernel(PagedAttnArgs a, uint32_t nsplit) {
  constexpr int D = DPL * 32;
  __shared__ __align__(16) float so[4][kHeads][D];
  __shared__ float sm[4][kHeads], sl[4][kHeads];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t nch = (a.G + kHeads - 1) / kHeads, KV = a.kv.KV;
  const uint32_t ch = blockIdx.x % nch, kvh = blockIdx.x / nch % KV, t = blockIdx.x / nch / KV;
  const uint32_t split = blockIdx.y;
  const uint32_t nr = min((uint32_t)kHeads, a.G - ch * kHeads);
  const int32_t b = find_seq_warp(a.bv, t, lane);
  if (b < 0) return;
  const SeqRange sr = seq_range(a.bv, b, a.kv.page_size);
  const uint32_t P = a.bv.prefix_len;
  if (threadIdx.x == 0 && sr.too_long()) atomicExch(&g_generic_error, BG_EINVAL);
  const int32_t own = sr.attended(t - sr.begin);
  const uint32_t total = P + (uint32_t)own;
  const uint32_t chunk = ((total + nsplit - 1) / nsplit + 31) / 32 * 32;
  const uint32_t lo = min(total, split * chunk), hi = min(total, lo + chunk);
  const int32_t *table = a.bv.table + (uint64_t)b * a.bv.table_stride;

  float q[kHeads][DPL];
  const uint64_t qrow = (uint64_t)t * a.H + kvh * a.G + ch * kHeads;
#pragma unroll
  for (int r = 0; r < kHeads; ++r) {
#pragma unroll
    for (int i = 0; i < DPL; ++i) q[r][i] = 0.f;
    if (r < nr) {
      const uint64_t off = (qrow + r) * D + lane * DPL;
      if (a.q_f16) load_f16<DPL>(static_cast<const __half *>(a.q) + off, q[r]);
      else load_f32<DPL>(static_cast<const float *>(a.q) + off, q[r]);
#pragma unroll
      for (int i = 0; i < DPL; ++i) q[r][i] *= a.sl2;
    }
  }
  float o[kHeads][DPL], m = kNegBig, l = 0.f;
#pragma unroll
  for (int r = 0; r < kHeads; ++r)
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[r][i] = 0.f;

  for (uint32_t base = lo + warp * kPos; base < hi; base += 4 * kPos) {
    // pool rows of the eight positions; a page id outside the pool reads as zeros
    int64_t row[kPos];
    float s[32];
#pragma unroll
    for (int j = 0; j < kPos; ++j) {
      const uint32_t p = base + j;
      row[j] = -1;
      if (p < hi) {
        row[j] = p < P ? paged_row(a.kv, a.bv.prefix_pages, p) : paged_row(a.kv, table, p - P);
        if (row[j] < 0) atomicExch(&g_generic_error, BG_EINVAL);
        else row[j] = row[j] * KV + kvh;
      }
    }
#pragma unroll
    for (int j = 0; j < kPos; ++j) {
      float k[DPL];
#pragma unroll
      for (int i = 0; i < DPL; ++i) k[i] = 0.f;
      if (row[j] >= 0) load_kv<DPL, MODE>(a.kv.K, a.kv.Ks, row[j], lane, k);
#pragma unroll
      for (int r = 0; r < kHeads; ++r) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) d = fmaf(q[r][i], k[i], d);
        s[r * kPos + j] = d;
      }
    }
#pragma unroll
    for (int st = 16; st > 0; st >>= 1) {
      const bool up = lane & st;
#pragma unroll
      for (int i = 0; i < st; ++i) {
        const float keep = up ? s[i + st] : s[i], give = up ? s[i] : s[i + st];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, st);
      }
    }
    const bool valid = base + (lane & 7) < hi;
    const float x = valid ? s[0] : -INFINITY;
    float mx = x;
#pragma unroll
    for (int st = 4; st > 0; st >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, st));
    const float mn = fmaxf(m, mx), corr = exp2f(m - mn), p = exp2f(x - mn);
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int r = 0; r < kHeads; ++r) {
      const float f = __shfl_sync(0xffffffffu, corr, r * kPos);
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[r][i] *= f;
    }
#pragma unroll
    for (int j = 0; j < kPos; ++j) {
      float v[DPL];
#pragma unroll
      for (int i = 0; i < DPL; ++i) v[i] = 0.f;
      if (row[j] >= 0) load_kv<DPL, MODE>(a.kv.V, a.kv.Vs, row[j], lane, v);
#pragma unroll
      for (int r = 0; r < kHeads; ++r) {
        const float w = __shfl_sync(0xffffffffu, p, r * kPos + j);
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[r][i] = fmaf(w, v[i], o[r][i]);
      }
    }
  }
  // join the four warps
#pragma unroll
  for (int st = 4; st > 0; st >>= 1) l += __shfl_xor_sync(0xffffffffu, l, st);
  if ((lane & 7) == 0) {
    sm[warp][lane >> 3] = m;
    sl[warp][lane >> 3] = l;
  }
#pragma unroll
  for (int r = 0; r < kHeads; ++r)
#pragma unroll
    for (int i = 0; i < DPL; ++i) so[warp][r][lane * DPL + i] = o[r][i];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < nr * (D / 4); i += 128) {
    const uint32_t r = i / (D / 4), d = i % (D / 4) * 4;
    float M = kNegBig, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w][r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(sm[w][r] - M);
      L = fmaf(sl[w][r], f, L);
      const float4 x = *reinterpret_cast<const float4 *>(&so[w][r][d]);
      v[0] = fmaf(x.x, f, v[0]);
      v[1] = fmaf(x.y, f, v[1]);
      v[2] = fmaf(x.z, f, v[2]);
      v[3] = fmaf(x.w, f, v[3]);
    }
    if (nsplit == 1) {
      write_out4(a.out, a.out_f16, a.gate, (qrow + r) * D + d, v, L);
    } else {
      const uint64_t idx = (uint64_t)split * a.bv.T * a.H + qrow + r;
      *reinterpret_cast<float4 *>(a.part_o + idx * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) a.part_ml[idx] = make_float2(M, L);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(128) join_splits_kernel(PagedAttnArgs a, uint32_t nsplit) {
  __shared__ __align__(16) float sm[4 * (D + 2)];
  const uint64_t rows = (uint64_t)a.bv.T * a.H, row = blockIdx.x;
  if (find_seq_warp(a.bv, (uint32_t)(row / a.H), threadIdx.x & 31) < 0) return;
  join_row_block<D, 4>(
      a.part_o, a.part_ml, nsplit, [&](uint32_t k) { return k * rows + row; }, sm, a.out, a.out_f16, a.gate, row * D);
}

template <int DPL>
int launch_d(const PagedAttnArgs &a, uint32_t nsplit, cudaStream_t st) {
  const uint64_t bx = (uint64_t)a.bv.T * a.kv.KV * ((a.G + kHeads - 1) / kHeads);
  if (bx > 0x7fffffffull || (uint64_t)a.bv.T * a.H > 0x7fffffffull) return BG_EUNSUPPORTED;
  const dim3 grid((unsigned)bx, nsplit);
  switch (a.mode) {
    case BG_KV_F32: paged_generic_kernel<DPL, BG_KV_F32><<<grid, 128, 0, st>>>(a, nsplit); break;
    case BG_KV_F16: paged_generic_kernel<DPL, BG_KV_F16><<<grid, 128, 0, st>>>(a, nsplit); break;
    case BG_KV_Q8: paged_generic_kernel<DPL, BG_KV_Q8><<<grid, 128, 0, st>>>(a, nsplit); break;
    default: return BG_EUNSUPPORTED;
  }
  if (nsplit > 1) join_splits_kernel<DPL * 32><<<a.bv.T * a.H, 128, 0, st>>>(a, nsplit);
  return cudaGetLastError() == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

}  // namespace

// Enough blocks for four to an SM where there are few rows; a split is never shorter than 64 positions
// of what the page tables can hold.
uint32_t paged_generic_splits(uint32_t T, uint32_t H, uint32_t KV, uint64_t max_positions) {
  const uint64_t blocks = (uint64_t)T * KV * ((H / KV + kHeads - 1) / kHeads);
  uint64_t n = (148 * 4 + blocks - 1) / blocks;
  n = n < 64 ? n : 64;
  const uint64_t most = (max_positions + 63) / 64;
  return (uint32_t)(n < most ? n : most ? most : 1);
}

int launch_paged_generic(const PagedAttnArgs &a, uint32_t nsplit, cudaStream_t st) {
  switch (a.D) {
    case 64: return launch_d<2>(a, nsplit, st);
    case 128: return launch_d<4>(a, nsplit, st);
    case 256: return launch_d<8>(a, nsplit, st);
    default: return BG_EUNSUPPORTED;
  }
}

int poll_device_error_paged_generic() {
  int v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_generic_error, sizeof(int)) != cudaSuccess) return BG_ELAUNCH;
  if (v) cudaMemcpyToSymbol(g_generic_error, &z, sizeof(int));
  return v;
}

}  // namespace bg
