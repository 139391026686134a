// Join of partial attention rows: of units that a block border cut, and of every row's own part with its
// part over a shared prefix.  One block per row; launched as a programmatic dependent of the attention
// kernel, so its launch is hidden behind that kernel's tail.
#include "paged.h"
#include "paged_merge.cuh"

namespace bg {
namespace {

constexpr int kWarps = 4;
constexpr uint32_t kMostPieces = 1024;  // more than any grid has blocks: bounds the loop whatever memory holds

// blockIdx.x: block whose last piece starts a cut unit; blockIdx.y: row of the unit.
template <int D>
__global__ void __launch_bounds__(128) join_cuts_kernel(PagedAttnArgs a, uint32_t ru) {
  __shared__ __align__(16) float sm[kWarps * (D + 2)];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint4 d = __ldcg(reinterpret_cast<const uint4 *>(a.cuts + blockIdx.x));
  const CutUnit c{d.x, d.y, d.z, d.w};
  const uint32_t r = blockIdx.y;
  if (c.npieces == 0 || r >= c.rows) return;
  const uint32_t R = c.R0 + r, t = R / a.G;
  const uint64_t off = ((uint64_t)t * a.H + c.kvh * a.G + R % a.G) * D;
  const uint32_t idx0 = a.slot0 + (2 * blockIdx.x + 1) * ru + r;
  join_row_block<D, kWarps>(
      a.part_o, a.part_ml, min(c.npieces, gridDim.x - blockIdx.x),
      [&](uint32_t k) { return (uint64_t)piece_index(idx0, ru, k); }, sm, a.out, a.out_f16, a.gate, off);
}

// The same for units of many rows and few pieces (tcgen05 kernel): one warp per row.
template <int D>
__global__ void __launch_bounds__(128) join_cuts_wide_kernel(PagedAttnArgs a, uint32_t ru) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t lane = threadIdx.x & 31, r = blockIdx.y * kWarps + (threadIdx.x >> 5);
  const uint4 d = __ldcg(reinterpret_cast<const uint4 *>(a.cuts + blockIdx.x));
  const CutUnit c{d.x, d.y, d.z, d.w};
  if (c.npieces == 0 || r >= c.rows) return;
  const uint32_t R = c.R0 + r, t = R / a.G, idx0 = a.slot0 + (2 * blockIdx.x + 1) * ru + r;
  const uint64_t off = ((uint64_t)t * a.H + c.kvh * a.G + R % a.G) * D;
  constexpr int NJ = (D + 127) / 128;
  float acc[NJ][4], M, L;
  join_pieces<D>(
      a.part_o, a.part_ml, 0, 1, min(c.npieces, gridDim.x - blockIdx.x), lane,
      [&](uint32_t k) { return (uint64_t)piece_index(idx0, ru, k); }, acc, M, L);
#pragma unroll
  for (int j = 0; j < NJ; ++j) write_out4(a.out, a.out_f16, a.gate, off + 4 * lane + 128 * j, acc[j], L);
}

template <int D>
__global__ void __launch_bounds__(128) join_rows_kernel(PagedAttnArgs a) {
  __shared__ __align__(16) float sm[kWarps * (D + 2)];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t t = blockIdx.x / a.H, h = blockIdx.x % a.H;
  if (find_seq_warp(a.bv, t, threadIdx.x & 31) < 0) return;
  const uint64_t at = (uint64_t)(h / a.G) * a.bv.T * a.G + (uint64_t)t * a.G + h % a.G;
  const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(a.own_pieces + at));
  const uint4 y = __ldcg(reinterpret_cast<const uint4 *>(a.pre_pieces + at));
  const uint32_t nx = min(x.y, kMostPieces), ny = min(y.y, kMostPieces), last = (uint32_t)a.part_rows - 1;
  join_row_block<D, kWarps>(
      a.part_o, a.part_ml, nx + ny,
      [&](uint32_t k) { return (uint64_t)min(last, k < nx ? piece_index(x.x, x.z, k) : piece_index(y.x, y.z, k - nx)); },
      sm, a.out, a.out_f16, a.gate, (uint64_t)blockIdx.x * D);
}

template <typename K, typename... A>
int launch_dependent(K kern, dim3 grid, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

}  // namespace

int launch_paged_join_cuts(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, cudaStream_t st) {
  if (ru > 16) {  // a tcgen05 kernel's
    const dim3 wide(blocks, (ru + kWarps - 1) / kWarps);
    if (a.D == 128) return launch_dependent(join_cuts_wide_kernel<128>, wide, st, a, ru);
    if (a.D == 256) return launch_dependent(join_cuts_wide_kernel<256>, wide, st, a, ru);
    return BG_EUNSUPPORTED;
  }
  const dim3 grid(blocks, ru);
  if (a.D == 128) return launch_dependent(join_cuts_kernel<128>, grid, st, a, ru);
  if (a.D == 256) return launch_dependent(join_cuts_kernel<256>, grid, st, a, ru);
  return BG_EUNSUPPORTED;
}

int launch_paged_join_rows(const PagedAttnArgs &a, cudaStream_t st) {
  const dim3 grid(a.bv.T * a.H);
  if (a.D == 128) return launch_dependent(join_rows_kernel<128>, grid, st, a);
  if (a.D == 256) return launch_dependent(join_rows_kernel<256>, grid, st, a);
  return BG_EUNSUPPORTED;
}

}  // namespace bg
