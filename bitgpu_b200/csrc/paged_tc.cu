// Attention of many rows over a paged cache on the 5th-generation tensor cores (tcgen05 + TMEM): chunked
// prefill of a ragged batch, and the rows of a whole batch against its shared prefix.
//
// A unit (paged.h) is 128 or 256 rows R = token*G + g of one kv head -- queries of several tokens and all
// heads of the group, so K and V are shared by all of them -- against a page list; blocks take even shares
// of the units' K/V tiles and leave partial rows where a border cuts a unit.
//
// Two streams keep the tensor pipe and the softmax warps busy at once.  Each has its own score tile S_t,
// output tile O_t (TMEM, f32) and softmax warpgroup:
//   NQT = 2 (256 rows): stream t is rows [128 t, 128 t + 128) and both use every K/V tile;
//   NQT = 1 (128 rows): the streams take even and odd K/V tiles of the same rows, and their outputs are
//           joined at the end (stream 0 reads both from TMEM).
// Softmax works in steps of 64 columns and hands each part of P over at once, so PV of the first part runs
// under the softmax of the second (f16 pool: tiles of 128 positions, one score tile per stream; q8: tiles of
// 64, two score tiles).  PV_t and, behind it, the S_t that takes over its columns (P overwrote the scores in
// place) come from one warp: MMAs of one thread execute in order.
//
// Precision, by the types of the call:
//   f16 rows, f16 pool: operands are exact, P is rounded once to f16 (kept 2^6 up, away from subnormals);
//   f32 rows (LO): q, without the power of two of its row's largest value, and p are split into two f16 halves (22
//           bits) -- two products for S, two for O; the softmax scale gives each row its power back; weights
//           below 2^-31 of a row's largest fall under f16's smallest step and are lost;
//   q8 pool: code * scale has more than 11 bits, so K and V are split too when they are dequantised into
//           the operand tiles: one more product each.  (A single f16 rounding of K and V would double the
//           error of f16 rows; the extra products cost less than that here, because the softmax warps
//           and not the tensor pipe set the pace of the single-product form.)  The halves hold code * scale
//           without the scales' magnitude: K without the power of two of the largest scale of its page list, which
//           the scores get back with the softmax scale, V without one per 32 channels, which the output gets back.
//           top_scales_kernel finds them beforehand: prefix of 32768 q8 positions 211 -> 224 us, 512 f32 tokens
//           behind as many 1180 -> 1220, 977 alone 77 -> 81.  (Found in this kernel, by the dequantising warps or by an
//           idle one, per tile or per run of tiles, they cost the first two 230 to 250 and 1430 to 1600.)
//
// The MMA drops the low bits of what it accumulates (a rounding towards zero a step, measured 0.8 * 2^-24 of the
// sum), so an accumulator that runs over a whole unit of many tiles errs in proportion to their number: 4e-4 after
// 120000 positions.  So a run is bounded (TcCfg::RUN): the softmax warps then add O to a sum in global memory, one
// rounded addition a run, and the next PV starts from zero.  It costs f32 rows 5 to 15 % (512 tokens behind 32768
// positions 660 -> 735 us, q8 1025 -> 1180) and f16 rows of head_dim 128 up to 4 % (mixed prompts 195 -> 202), where
// the code alone, which such short units never reach, does.
//
// Warp roles: warp 0 TMA producer of K and V (f16 pool; page boxes, 128-byte swizzle), warp 1 MMA issuer,
// warps 2-3 ask for the next unit's query rows as soon as the last S of the current one is done, warps 4-11
// softmax (one row per thread), warps 12-15 and 16-19 (q8 pool) dequantise K and V, a tile ahead in registers.
// All waits are bounded; on expiry the block records BG_ETIMEOUT, stops issuing, waits for what it issued,
// frees its TMEM and exits.
#include <cuda.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged.h"
#include "paged_merge.cuh"
#include "umma.cuh"

namespace bg {
namespace {

constexpr int kM = 128;             // rows of a UMMA tile
constexpr float kRescale = 8.0f;    // lazy rescale threshold, log2 units
constexpr float kUp = 6.0f;         // p carries 2^6: at most 2^14 with the lazy rescale

template <int D, bool Q8, bool LO, int NQT>
struct TcCfg {
  static constexpr int NQ = LO ? 2 : 1, NK = Q8 ? 2 : 1;     // operand halves
  static constexpr int QT = kM * D * 2;                      // bytes of one f16 query tile
  // positions of a K/V tile, as shared memory allows beside the query halves
  static constexpr int KT = D == 128 ? (Q8 ? 64 : 128) : (Q8 || LO ? 32 : 64);
  static constexpr int SW = KT < 64 ? KT : 64;               // columns of a softmax step
  static constexpr int PARTS = KT / SW, SLOTS = 3 - PARTS;   // steps per score tile; score tiles per stream
  static constexpr int NS = D == 128 ? 2 : 1;                // streams (TMEM holds one O of 256 columns)
  static_assert(D == 128 || NQT == 1, "head_dim 256: one stream");
  static constexpr int KVT = KT * D * 2;                     // bytes of one f16 K (or V) tile
  static constexpr int LEAD = Q8 ? 2 : 1;                    // a unit's own cost, in tiles
  static constexpr int NST = D == 256 && Q8 && LO ? 1 : 2;   // ring stages of K and of V
  static constexpr int oQ = 0, oK = NQT * NQ * QT, oV = oK + NST * NK * KVT, oB = oV + NST * NK * KVT;
  static constexpr int oInfo = oB + 384, oVP = oInfo + 64, oQP = oVP + 64, oML = oQP + 2 * kM * 4, oScan = oML + kM * 8;
  static constexpr int SMEM = oScan + 24 * 8;
  // a stream's tiles in one accumulator run: at most 64 MMAs for f32 rows (3e-6), 512 for f16 rows (2.5e-5, a
  // twentieth of the result's rounding)
  static constexpr int RUN = (LO ? 64 : 512) / (KT / 16 * (NQ + NK - 1)) & (LO ? ~3 : ~0);
  static constexpr int THREADS = Q8 ? 640 : 384;
  // TMEM columns: part x of stream t at (2t + x) * SW, outputs behind them
  static constexpr uint32_t O0 = 256, O1 = 384;
  static_assert(SMEM <= 232448, "shared memory");
};

struct TcParams {
  PagedAttnArgs a;
  UnitShape u;
  uint32_t box, ppt;  // positions of a page box, boxes per tile
  uint32_t join_rows;
  uint32_t page_shift;  // log2(page_size), or 32
  uint32_t rpt;       // rows of a query tile: whole tokens, at most 128
  uint32_t wide;      // out and the partial rows start on 32-byte boundaries
};

struct alignas(16) TcInfo {
  uint32_t R0, rows, kvh, tile0, ntiles, len;
  int32_t lim_base;
  uint32_t dest, row0;
  float k_pow2;  // of K's scales (q8 pool)
};
constexpr uint32_t kDirect = 0xffffffffu, kRowBuf = 0xfffffffeu;

// 16-byte chunk `ch` (8 f16) of row r in a 128B-swizzled K-major operand tile of R rows
template <int R>
__device__ __forceinline__ uint32_t sw_off(int r, int ch) {
  return (uint32_t)((ch >> 3) * (R * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// eight values as f16 and what the rounding left over
__device__ __forceinline__ void split8(const float (&x)[8], uint4 &hi, uint4 &lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 p = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    const float2 f = __half22float2(p);
    h[i] = *reinterpret_cast<const uint32_t *>(&p);
    l[i] = pack_half2(x[2 * i] - f.x, x[2 * i + 1] - f.y);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Largest block scales (as bits, which order like the magnitudes) of each page list and kv head: V's blocks, K's at
// kTopK.
constexpr uint32_t kTopK = 8;
__device__ __forceinline__ uint32_t top_scale(const PagedAttnArgs &a, const Piece &pc, uint32_t which) {
  return __ldcg(a.tops + ((uint64_t)pc.list * a.kv.KV + pc.kvh) * kTopRow + which);
}

// Codes of one block as two f16 halves of code * x, x below 2^14 / 127, in packed f16 arithmetic.  With
// x = m 2^e and m = mh + ml in f16:  c' = code 2^e is exact (byte + 128 under the pattern 0x64xx is
// 1152 + code, and one fused multiply-add removes the 1152 and applies 2^e);  hi = c' mh rounded;
// c' mh - hi is exact in f16, so  lo = c' ml + (c' mh - hi)  carries the rest, to 2^-22 of the value or half of f16's
// smallest step: 2^-25.
struct CodeScale {
  __half2 p2, bias, least, mh, ml;
  __device__ __forceinline__ explicit CodeScale(float x) {
    const int e = min(4, max(-20, (int)((__float_as_uint(x) >> 23) & 255) - 127));
    const float m = x * __uint_as_float((uint32_t)(127 - e) << 23), f = __uint_as_float((uint32_t)(127 + e) << 23);
    p2 = __float2half2_rn(f);
    bias = __float2half2_rn(-1152.0f * f);
    least = __float2half2_rn(-127.0f * f);  // code -128 stands for -1 too
    mh = __float2half2_rn(m);
    ml = __float2half2_rn(m - __low2float(mh));
  }
  // the four codes of a word, in order
  __device__ __forceinline__ void split4(uint32_t w, uint32_t &h0, uint32_t &h1, uint32_t &l0, uint32_t &l1) const {
    const uint32_t b = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = __byte_perm(b, 0x64646464u, i ? 0x4342 : 0x4140);
      const __half2 c = __hmax2(__hfma2(*reinterpret_cast<const __half2 *>(&x), p2, bias), least);
      const __half2 h = __hmul2(c, mh), r = __hfma2(c, mh, __hneg2(h)), l = __hfma2(c, ml, r);
      (i ? h1 : h0) = *reinterpret_cast<const uint32_t *>(&h);
      (i ? l1 : l0) = *reinterpret_cast<const uint32_t *>(&l);
    }
  }
};

// N consecutive words of one row.  A row belongs to one thread, so a store instruction touches 32 rows:
// 32-byte stores fill whole sectors (16-byte ones write every sector twice: 5.5 -> 2.5 us per 256 rows).
template <int N>
__device__ __forceinline__ void store_words(void *dst, const uint32_t (&w)[N], uint32_t wide) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint32_t *>(dst) + i),
                   "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]),
                   "r"(w[i + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<uint4 *>(static_cast<uint32_t *>(dst) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// A row's O in TMEM joins its run sum, whose weights are f times those of O now.  Only this thread adds to the row,
// so reductions (which it need not wait for) happen in its order.
template <int D>
__device__ __forceinline__ void add_run(uint32_t obase, float4 *sum, float f, bool summed) {
  if (summed && __any_sync(0xffffffffu, f != 1.0f)) {  // rare: the reference moved since the last run
#pragma unroll 4
    for (int i = 0; i < D / 4; ++i) {
      const float4 v = __ldcg(sum + i * kM);
      __stcg(sum + i * kM, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
  }
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(obase + c * 32, o);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float4 *at = sum + (c * 8 + i) * kM;
      const float4 x = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                   __uint_as_float(o[4 * i + 3]));
      if (summed)
        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(x.x), "f"(x.y), "f"(x.z),
                     "f"(x.w)
                     : "memory");
      else __stcg(at, x);
    }
  }
}

// The whole sum, f times, to O.
template <int D>
__device__ __forceinline__ void add_sum(uint32_t obase, const float4 *sum, float f) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(obase + c * 32, o);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 v = __ldcg(sum + (c * 8 + i) * kM);
      o[4 * i] = __float_as_uint(fmaf(v.x, f, __uint_as_float(o[4 * i])));
      o[4 * i + 1] = __float_as_uint(fmaf(v.y, f, __uint_as_float(o[4 * i + 1])));
      o[4 * i + 2] = __float_as_uint(fmaf(v.z, f, __uint_as_float(o[4 * i + 2])));
      o[4 * i + 3] = __float_as_uint(fmaf(v.w, f, __uint_as_float(o[4 * i + 3])));
    }
    tmem_st32(obase + c * 32, o);
  }
  tmem_wait_st();
}

template <int D, bool Q8, bool LO, int NQT>
__global__ void __launch_bounds__(TcCfg<D, Q8, LO, NQT>::THREADS, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ TcParams p) {
  using C = TcCfg<D, Q8, LO, NQT>;
  constexpr int KT = C::KT, SW = C::SW, NQ = C::NQ, NK = C::NK;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::oB);
  uint64_t *k_full = bars, *k_empty = bars + 4, *v_full = bars + 8, *v_empty = bars + 12;
  uint64_t *q_full = bars + 16, *q_free = bars + 17, *info_free = bars + 18;
  uint64_t *s_full = bars + 19, *p_full = bars + 23;  // per score slot 2t + u
  uint64_t *pv_done = bars + 27, *o_free = bars + 29; // per stream
  uint64_t *b_done = bars + 31, *tail = bars + 32, *mma_done = bars + 33;
  uint32_t *tmem_at = reinterpret_cast<uint32_t *>(bars + 35);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 36);
  TcInfo *info = reinterpret_cast<TcInfo *>(smem + C::oInfo);
  volatile float *q_pow2 = reinterpret_cast<float *>(smem + C::oQP);  // [2][kM], by piece (f32 rows)
  volatile float *v_pow2 = reinterpret_cast<float *>(smem + C::oVP);  // [2][8], by piece (q8 pool)
  float2 *ml_s = reinterpret_cast<float2 *>(smem + C::oML);
  const PagedAttnArgs &a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023) {
    atomicExch(&g_device_error, BG_ELAUNCH);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&k_full[i], Q8 ? 4 : 1);
      mbar_init(&v_full[i], Q8 ? 4 : 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);  // one arrival per warp: 128 single ones on one word are serialised
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(mma_done, 1);
    mbar_init(info_free, 4 * C::NS);
    mbar_init(b_done, 4);
    mbar_init(tail, 1);
    *abort_flag = 0;
    fence_barrier_init();
    if (!Q8) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // (a q8 pool's kernel follows top_scales_kernel, which lets it begin when all before is done: only what that one
  // writes has to be waited for)
  if (!Q8) asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_before();
  const TileSpan span = block_span<C::THREADS>(a.bv, p.u, a.kv.page_size, a.min_tiles,
                                               reinterpret_cast<uint32_t *>(smem + C::oScan), &g_device_error);
  if (Q8) asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem = *tmem_at;
  const uint32_t sQ = smem_u32(smem + C::oQ), sK = smem_u32(smem + C::oK), sV = smem_u32(smem + C::oV);
  const uint32_t ps = a.kv.page_size;

  // registers: 384 threads: 128*72 + 256*216 = 384*168; 640: 128*64 + 256*128 + 256*80 = 640*96
  if (warp < 4) {
    if constexpr (Q8) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;" ::: "memory");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
    if (warp == 0) {
      // ---------------- TMA producer (f16 pool) ----------------
      if constexpr (!Q8) {
        PieceWalk walk;
        walk.init(span, a.bv, p.u, ps);
        Piece pc;
        bool ok = true;
        int it = 0, tails = 0, kdone = 0, vdone = 0;
        while (ok && walk.next(pc, a.bv, p.u, ps)) {
          auto page_of = [&](uint32_t tile) -> uint32_t {
            const uint32_t pos = (pc.tile0 + tile) * KT + lane * p.box;
            if ((uint32_t)lane >= p.ppt || tile >= pc.ntiles || pos >= pc.len) return a.kv.num_pages;
            const uint32_t pg = (uint32_t)__ldg(pc.pages + pos / ps);
            if (pg < a.kv.num_pages) return pg;
            atomicExch(&g_device_error, BG_EINVAL);
            return a.kv.num_pages;
          };
          uint32_t pg_next = page_of(0);
          for (uint32_t t = 0; ok && t < pc.ntiles; ++t, ++it) {
            const uint32_t pg = pg_next;
            pg_next = page_of(t + 1);
            const int s = it % C::NST;
            const uint32_t pos0 = (pc.tile0 + t) * KT, par = ((it / C::NST) - 1) & 1;
            const int y = (int)((pos0 + lane * p.box) % ps);
            if (it >= C::NST) ok = mbar_wait_warp(&k_empty[s], par);
            if (!ok || __any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
            if (lane == 0) mbar_expect_tx(&k_full[s], C::KVT);
            __syncwarp();
            if ((uint32_t)lane < p.ppt)
              for (int cb = 0; cb < D / 64; ++cb)
                tma_load_4d(smem + C::oK + s * C::KVT + cb * KT * 128 + lane * p.box * 128, &tmK, &k_full[s], cb * 64,
                            (int)pc.kvh, y, (int)pg);
            kdone = it + 1;
            if (it >= C::NST) ok = mbar_wait_warp(&v_empty[s], par);
            if (!ok || __any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
            // slots of the last page behind the length may hold NaN, and 0 * NaN is NaN: such a tile
            // arrives on its own barrier, its rows behind the length are cleared, then it is handed on
            const bool last = pos0 + KT > pc.len && pc.len > pos0 && pc.len % p.box;
            uint64_t *bar = last ? tail : &v_full[s];
            if (lane == 0) mbar_expect_tx(bar, C::KVT);
            __syncwarp();
            unsigned char *dst = smem + C::oV + s * C::KVT;
            if ((uint32_t)lane < p.ppt)
              for (int cb = 0; cb < D / 64; ++cb)
                tma_load_4d(dst + cb * KT * 128 + lane * p.box * 128, &tmV, bar, cb * 64, (int)pc.kvh, y, (int)pg);
            if (last) {
              ok = mbar_wait_warp(tail, tails++ & 1);
              if (!ok) break;
              const uint32_t r0 = pc.len - pos0, r1 = (r0 + p.box - 1) / p.box * p.box, n = (r1 - r0) * 8;
              for (uint32_t i = lane; i < n * (D / 64); i += 32) {
                const uint32_t cb = i / n, x = i % n;
                *reinterpret_cast<uint4 *>(dst + cb * KT * 128 + r0 * 128 + x * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&v_full[s]);
            }
            vdone = it + 1;
          }
        }
        if (!ok && lane == 0) *abort_flag = 1;
        // no copy may still be in flight when the block exits
        if (lane == 0) {
          for (int i = max(0, kdone - C::NST); i < kdone; ++i) mbar_wait(&k_full[i % C::NST], (i / C::NST) & 1);
          for (int i = max(0, vdone - C::NST); i < vdone; ++i) mbar_wait(&v_full[i % C::NST], (i / C::NST) & 1);
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      // The whole warp runs the loop and one elected lane issues: so the compiler knows every operand to be
      // uniform (run by one lane under a branch, each MMA first moves its descriptors to uniform registers:
      // 2900 -> 1720 cycles for a tile's 24 MMAs and their barriers).  One warp for both streams on purpose:
      // it serves them in turn, which keeps them half a step apart, one on the tensor pipe under the other's
      // softmax.  (With a warp each they fall into step, wait for the pipe together and then for the exp unit.)
      const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
      constexpr uint32_t idS = idesc_f16(KT, false), idO = idesc_f16(D, true);
      constexpr uint32_t kHi = umma_desc_hi(1024);
      const uint32_t q_lo = umma_desc_lo(sQ, 16), k_lo = umma_desc_lo(sK, 16), v_lo = umma_desc_lo(sV, KT * 128);
      // one product over D (K steps of 16 values, 32 bytes of a 128-byte swizzle row)
      auto one_s = [&](uint32_t slot, uint32_t q, uint32_t k, auto acc) {
        umma_ss_lo<kHi, decltype(acc)::value>(slot, q, k, idS);
#pragma unroll
        for (int kk = 1; kk < D / 16; ++kk)
          umma_ss_lo<kHi, true>(slot, q + ((kk >> 2) * (kM * 128) + (kk & 3) * 32) / 16,
                                k + ((kk >> 2) * (KT * 128) + (kk & 3) * 32) / 16, idS);
      };
      // S = Q K^T into score tile u: small products first, so that they are added up among themselves
      auto issue_s = [&](int t, int u, int s) {
        const uint32_t slot = tmem + (2 * t + u) * SW, k = k_lo + s * (NK * C::KVT / 16);
        const uint32_t q = q_lo + (NQT == 2 ? t : 0) * (NQ * C::QT / 16);
        if constexpr (LO) one_s(slot, q + C::QT / 16, k, std::false_type{});
        if constexpr (Q8) one_s(slot, q, k + C::KVT / 16, std::bool_constant<LO>{});
        one_s(slot, q, k, std::bool_constant<LO || Q8>{});
      };
      auto one_pv = [&](uint32_t o, uint32_t pa, uint32_t v, bool acc) {
        if (acc) umma_ts_lo<kHi, true>(o, pa, v, idO);
        else umma_ts_lo<kHi, false>(o, pa, v, idO);
#pragma unroll
        for (int kk = 1; kk < SW / 16; ++kk) umma_ts_lo<kHi, true>(o, pa + kk * 8, v + kk * (16 * 128 / 16), idO);
      };
      // O_t += P V for the SW positions of part h of a tile (P from the columns of part x)
      auto issue_pv = [&](int t, int x, int s, int h, bool acc) {
        const uint32_t slot = tmem + (2 * t + x) * SW, v = v_lo + s * (NK * C::KVT / 16) + h * (SW * 128 / 16);
        const uint32_t o = tmem + (t ? C::O1 : C::O0);
        if constexpr (LO) one_pv(o, slot + SW / 2, v, acc);
        if constexpr (Q8) one_pv(o, slot, v + C::KVT / 16, LO || acc);
        one_pv(o, slot, v, LO || Q8 || acc);
      };
      // a stream's tiles are STEP apart; AHEAD tiles' S come before the first PV, as far as the ring holds their K
      constexpr int STEP = NQT == 2 ? 1 : C::NS, AHEAD = C::SLOTS * STEP < C::NST ? C::SLOTS * STEP : C::NST;
      static_assert(AHEAD % STEP == 0, "the next S belongs to the same stream");
      bool ok = true;
      int it = 0;         // tiles of all pieces before this one
      uint32_t pp = 0;    // next phase parity of p_full, one bit per part
      for (uint32_t piece = 0; ok; ++piece) {
        if (!mbar_wait_warp(q_full, piece & 1)) { ok = false; break; }
        const int n = (int)__shfl_sync(0xffffffffu, info->ntiles, 0);
        if (n == 0) break;
        auto stage = [&](int i) { return (it + i) % C::NST; };
        auto wait_k = [&](int i) { return mbar_wait_warp(&k_full[stage(i)], ((it + i) / C::NST) & 1); };
        auto wait_v = [&](int i) { return mbar_wait_warp(&v_full[stage(i)], ((it + i) / C::NST) & 1); };
        // (one lane) S of stream t, tile i; the last reader of K_i frees it, the last S of the piece frees Q
        auto send_s = [&](int t, int u, int i) {
          issue_s(t, u, stage(i));
          umma_commit(&s_full[2 * t + u]);
          if (NQT == 1 || t == 1) {
            umma_commit(&k_empty[stage(i)]);
            if (i + 1 == n) umma_commit(q_free);
          }
        };
        for (int i = 0; ok && i < AHEAD && i < n; ++i) {
          ok = wait_k(i);
          if (!ok) break;
          const int u = (i / STEP) % C::SLOTS;
          tc_fence_after();
          if (elect_one()) {
            send_s(NQT == 1 && C::NS == 2 ? i & 1 : 0, u, i);
            if (NQT == 2) send_s(1, u, i);
          }
          __syncwarp();
        }
        // the PVs of stream t, tile i, and behind them the S that takes over its columns: in-order execution
        // keeps P safe.  The ring's waits come before P's, under the softmax: K(i + AHEAD) and V(i) only need what
        // earlier steps issued.
        auto step = [&](int t, int i, int u) {
          const bool more = i + AHEAD < n;
          if (NQT == 1 || t == 0) ok = wait_v(i) && (!more || wait_k(i + AHEAD));
          if (ok && i < STEP && piece > 0) ok = mbar_wait_warp(&o_free[NQT == 2 ? t : 0], (piece - 1) & 1);
#pragma unroll
          for (int h = 0; h < C::PARTS; ++h) {
            const int x = C::PARTS == 2 ? h : u, b = 2 * t + x;
            ok = ok && mbar_wait_warp(&p_full[b], (pp >> b) & 1);
            if (!ok) return;
            pp ^= 1u << b;
            tc_fence_after();
            if (elect_one()) {
              issue_pv(t, x, stage(i), h, i / STEP % C::RUN != 0 || h > 0);
              umma_commit(&pv_done[t]);
              if (h == C::PARTS - 1) {
                if (NQT == 1 || t == 1) umma_commit(&v_empty[stage(i)]);
                if (more) send_s(t, ((i + AHEAD) / STEP) % C::SLOTS, i + AHEAD);
              }
            }
            __syncwarp();
          }
        };
        for (int i = 0; ok && i < n; ++i) {
          const int u = (i / STEP) % C::SLOTS;
          if (NQT == 2) {
            step(0, i, u);
            if (ok) step(1, i, u);
          } else if (C::NS == 2 && (i & 1)) {
            step(1, i, u);
          } else {
            step(0, i, u);
          }
        }
        it += n;
      }
      if (!ok) *abort_flag = 1;
      // every MMA must complete before the block frees its TMEM
      if (elect_one()) umma_commit(mma_done);
      __syncwarp();
      mbar_wait_warp(mma_done, 0);
    } else {
      // ---------------- query rows and descriptions ----------------
      const int gt = (warp - 2) * 32 + lane;
      PieceWalk walk;
      walk.init(span, a.bv, p.u, ps);
      Piece pc;
      bool ok = true;
      uint32_t loaded = 0;  // pieces whose query tile was asked for
      if (a.cuts && gt == 0) a.cuts[blockIdx.x].npieces = 0;
      for (uint32_t piece = 0; ok; ++piece) {
        const bool more = walk.next(pc, a.bv, p.u, ps);
        uint32_t top = 0;
        if (Q8 && more && gt <= kTopK) top = top_scale(a, pc, gt);
        float qp[4];  // warp 2: of the piece's rows
        if (LO && more && warp == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t R = pc.R0 + min(lane + 32u * i, pc.rows - 1);
            qp[i] = __ldcg(a.q_pow2 + (uint64_t)(R / a.G) * a.H + pc.kvh * a.G + R % a.G);
          }
        }
        if (piece > 0) {
          ok = mbar_wait_warp(q_free, (piece - 1) & 1) && mbar_wait_warp(info_free, (piece - 1) & 1);
          if (!ok || __any_sync(0xffffffffu, *abort_flag != 0)) break;
        }
        if (!more) {
          if (gt == 0) info->ntiles = 0;
          if (gt == 0) mbar_arrive(q_full);
          break;
        }
        const bool whole = pc.npieces == 1;
        const uint32_t slot = a.slot0 + (2 * blockIdx.x + (pc.starts ? 1 : 0)) * p.u.RU;
        const uint32_t row0 = pc.own ? a.own_row0 : a.pre_row0;
        if (gt == 0) {
          info->R0 = pc.R0;
          info->rows = pc.rows;
          info->kvh = pc.kvh;
          info->tile0 = pc.tile0;
          info->ntiles = pc.ntiles;
          info->len = pc.len;
          info->lim_base = pc.lim_base;
          info->dest = !whole ? slot : p.join_rows ? kRowBuf : kDirect;
          info->row0 = row0;
          if (!p.join_rows && !whole && pc.starts) a.cuts[blockIdx.x] = CutUnit{pc.R0, pc.rows, pc.kvh, pc.npieces};
        }
        if (p.join_rows && pc.starts) {
          RowPieces *rp = (pc.own ? a.own_pieces : a.pre_pieces) + (uint64_t)pc.kvh * a.bv.T * a.G + pc.R0;
          for (uint32_t r = gt; r < pc.rows; r += 64) {
            const uint32_t R = pc.R0 + r;
            rp[r] = RowPieces{whole ? row0 + R / a.G * a.H + pc.kvh * a.G + R % a.G : slot + r, pc.npieces, p.u.RU, 0};
          }
        }
        if constexpr (Q8) {
          if (gt < kTopK) v_pow2[(piece & 1) * 8 + gt] = pow2_of(top);
          if (gt == kTopK) info->k_pow2 = pow2_of(top);
        }
        if (LO && warp == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q_pow2[(piece & 1) * kM + lane + 32 * i] = qp[i];
        }
        __syncwarp();
        // rows come by TMA as boxes of whole tokens' heads; tokens behind the unit's are other sequences' (or
        // zeros) and the tile's last rows stay as they were: computed along, never written
        loaded = piece + 1;
        if (gt == 0) {
          mbar_expect_tx(q_full, NQT * C::NQ * p.rpt * D * 2);
          const int tok = (int)(pc.R0 / a.G), per = (int)(p.rpt / a.G);
          for (int q = 0; q < NQT * C::NQ; ++q)
            for (int cb = 0; cb < D / 64; ++cb)
              tma_load_4d(smem + C::oQ + q * C::QT + cb * kM * 128, &tmQ, q_full, cb * 64, 0, (int)pc.kvh,
                          LO ? tok + q * (int)a.bv.T : tok + q * per);
        }
      }
      if (!ok) {
        *abort_flag = 1;
        // no query tile may still be in flight when the block exits (otherwise q_free is behind it)
        if (gt == 0 && loaded) mbar_wait(q_full, (loaded - 1) & 1);
      }
    }
  } else if (warp < 12) {
    // ---------------- softmax (one row per thread) ----------------
    if constexpr (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;" ::: "memory");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;" ::: "memory");
    const int t = (warp - 4) >> 2;                // stream
    const int row = ((warp & 3) << 5) + lane;     // TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) << 5) << 16;
    const uint32_t obase = (tmem + (t ? C::O1 : C::O0)) | lane_off;
    float sl2 = a.sl2;
    bool ok = true;
    if (t < C::NS) {
      uint32_t sp = 0;           // next phase parity of s_full, one bit per slot of this stream
      uint32_t nv = 0;           // this stream's PVs of the pieces before
      // sums of this stream's runs: four columns of the 128 rows after one another
      constexpr int SUM = D / 4 * kM;
      float4 *const my_sums = a.run_sums + ((uint64_t)blockIdx.x * C::NS + t) * SUM + row;
      for (uint32_t piece = 0;; ++piece) {
        if (!mbar_wait_warp(q_full, piece & 1)) { ok = false; break; }
        const TcInfo in = *info;
        if (in.ntiles == 0) break;
        release_read(info_free);
        const uint32_t r = (NQT == 2 ? t * p.rpt : 0) + row;
        const uint32_t R = in.R0 + min(r, in.rows - 1);
        const int lim = min(in.lim_base + (int)(R / a.G), (int)in.len - 1);
        if (a.gate && in.dest == kDirect && (NQT == 2 || t == 0)) {
          // the gates of the row, to L2: the epilogue would wait for HBM
          const float *g = a.gate + ((uint64_t)(R / a.G) * a.H + in.kvh * a.G + R % a.G) * D;
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) asm volatile("prefetch.global.L2 [%0];" ::"l"(g + 32 * i));
        }
        // (never so small that a masked score times it is not -infinity)
        if constexpr (LO || Q8)
          sl2 = fmaxf(a.sl2 * (LO ? q_pow2[(piece & 1) * kM + row] : 1.f) * (Q8 ? in.k_pow2 : 1.f), 0x1p-126f);
        float m_used = kNegBig, l = 0.f;
        float m_sum = kNegBig;     // what the run sum's weights refer to
        bool summed = false;       // whether there is one (the same for the whole stream)
        const int step = NQT == 2 ? 1 : C::NS;
        const int first = NQT == 2 ? 0 : t;
        for (int j0 = first; ok && j0 < (int)in.ntiles; j0 += C::RUN * step) {
          if (j0 != first) {
            // the run's end: O joins the sum before the next PV overwrites it
            if (!mbar_wait_warp(&pv_done[t], (nv + j0 / step * C::PARTS - 1) & 1)) { ok = false; break; }
            tc_fence_after();
            add_run<D>(obase, my_sums, ex2_approx(m_sum - m_used), summed);
            tc_fence_before();
            m_sum = m_used;
            summed = true;
          }
          const int j1 = min((int)in.ntiles, j0 + C::RUN * step);
          for (int j = j0; j < j1; j += step) {
            const int jj = NQT == 2 ? j : j / C::NS;  // tile of this stream
#pragma unroll 1
            for (int h = 0; h < C::PARTS; ++h) {
              const int g = jj * C::PARTS + h, part = g & 1;  // step of this stream, and where its scores lie
              if (h == 0) {
                const int u = C::PARTS == 2 ? 0 : part;
                if (!mbar_wait_warp(&s_full[2 * t + u], (sp >> u) & 1)) { ok = false; break; }
                sp ^= 1u << u;
                tc_fence_after();
              }
              const uint32_t sbase = (tmem + (2 * t + part) * SW) | lane_off;
              const int key0 = (int)(in.tile0 + j) * KT + h * SW;
              const int nvalid = min(SW, max(0, lim - key0 + 1));
              uint32_t x[SW / 32][32];  // the step's scores of the row: one TMEM wait
#pragma unroll
              for (int c = 0; c < SW / 32; ++c) tmem_ld32(sbase + c * 32, x[c]);
              tmem_wait_ld();
              if (nvalid < SW) {
#pragma unroll
                for (int c = 0; c < SW / 32; ++c)
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (c * 32 + i >= nvalid) x[c][i] = __float_as_uint(-INFINITY);
              }
              float mx8[8];  // eight independent chains
#pragma unroll
              for (int k = 0; k < 8; ++k) mx8[k] = -INFINITY;
#pragma unroll
              for (int c = 0; c < SW / 32; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  const int k = (c * 16 + i / 2) & 7;
                  mx8[k] = fmax3(mx8[k], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
                }
              const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]),
                                     fmax3(mx8[3], mx8[4], fmaxf(mx8[5], fmaxf(mx8[6], mx8[7]))));
              const float mt = mx * sl2;
              // lazy rescale: the whole warp takes the TMEM round trip when any of its rows moved far; rows
              // that did not use the factor 1.  The PV before must have completed.
              // Phases of pv_done are only ever waited for before this tile's P is handed over (or, after a run's
              // last one, by the waits at its end): the barrier cannot have moved on by two.
              bool waited = g == 0;
              const bool need = mt > m_used + kRescale;
              if (__any_sync(0xffffffffu, need)) {
                if (g > 0) {
                  if (!mbar_wait_warp(&pv_done[t], (nv + g - 1) & 1)) { ok = false; break; }
                  waited = true;
                  tc_fence_after();
                  const float f = need ? ex2_approx(m_used - mt) : 1.0f;
#pragma unroll 1
                  for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(obase + c * 32, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st32(obase + c * 32, o);
                  }
                  l *= f;
                }
                if (need) m_used = mt;
              }
              const float mneg = kUp - m_used;
              const uint64_t sl2x2 = pack2(sl2, sl2), mneg2 = pack2(mneg, mneg);
              uint64_t sums[2] = {0, 0};
#pragma unroll
              for (int c = 0; c < SW / 32; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const uint64_t s2 = pack2(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1]));
                  const float2 e = unpack2(fma2(s2, sl2x2, mneg2));
                  const float p0 = ex2_approx(e.x), p1 = ex2_approx(e.y);
                  const uint64_t pp = pack2(p0, p1);
                  sums[i & 1] = add2(sums[i & 1], pp);
                  hi[i] = pack_half2(p0, p1);
                  if constexpr (LO) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
                    lo[i] = pack_half2(p0 - f.x, p1 - f.y);
                  }
                }
                tmem_st16(sbase + c * 16, hi);
                if constexpr (LO) tmem_st16(sbase + SW / 2 + c * 16, lo);
              }
              const float2 sum = unpack2(add2(sums[0], sums[1]));
              l += sum.x + sum.y;
              tmem_wait_st();
              const bool last = j + step >= j1 && h == C::PARTS - 1;
              if (last && !waited && !mbar_wait_warp(&pv_done[t], (nv + g - 1) & 1)) { ok = false; break; }
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[2 * t + part]);
            }
            if (!ok) break;
          }
        }
        if (!ok) break;
        // ---- the piece's rows ----
        const int mine = NQT == 2 || C::NS == 1 ? (int)in.ntiles : ((int)in.ntiles + 1 - t) >> 1;  // this stream's tiles
        const bool some = mine > 0;
        if (some && !mbar_wait_warp(&pv_done[t], (nv + mine * C::PARTS - 1) & 1)) { ok = false; break; }
        nv += mine * C::PARTS;
        if (summed) {
          tc_fence_after();
          add_sum<D>(obase, my_sums, ex2_approx(m_sum - m_used));
        }
        float f0 = 1.f, f1 = 0.f, M = m_used, L = l;
        if constexpr (NQT == 1 && C::NS == 2) {
          if (t == 1) {
            // stream 0 still reads the last piece's (m, l) until it frees O
            tc_fence_after();
            if (piece > 0 && !mbar_wait_warp(&o_free[0], (piece - 1) & 1)) { ok = false; break; }
            ml_s[row] = make_float2(m_used, some ? l : 0.f);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_done);
            continue;
          }
          if (!mbar_wait_warp(b_done, piece & 1)) { ok = false; break; }
          // (stream 1 has seen its last PV done before it counted in)
          const float2 ml = ml_s[row];
          M = fmaxf(m_used, ml.x);
          f0 = ex2_approx(m_used - M);
          f1 = in.ntiles > 1 ? ex2_approx(ml.x - M) : 0.f;
          L = l * f0 + ml.y * f1;
        }
        tc_fence_after();
        const float inv = L != 0.f ? 1.0f / L : 0.f;  // a row that attends nothing is zero
        const bool valid = (uint32_t)row < p.rpt && r < in.rows;
        const uint64_t orow = (uint64_t)(R / a.G) * a.H + in.kvh * a.G + R % a.G;
        const uint64_t prow = in.dest == kRowBuf ? in.row0 + orow : in.dest + r;
        const bool gated = a.gate && in.dest == kDirect && valid;
        const float4 *gate = reinterpret_cast<const float4 *>(a.gate + orow * D);
        // the next chunk's gate travels while a chunk is written, where there are registers for it (otherwise
        // 128 streams behind 32768 shared q8 positions, without any gate, take 211 us for 208)
        constexpr bool AHEAD_GATE = !Q8 || (D == 256 && !LO);
        float4 gn[8];
        if (AHEAD_GATE && gated) {
#pragma unroll
          for (int i = 0; i < 8; ++i) gn[i] = __ldg(gate + i);
        }
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(obase + c * 32, o);
          tmem_wait_ld();
          if constexpr (NQT == 1 && C::NS == 2) {
            if (in.ntiles > 1) {  // uniform: O_1 holds something
              uint32_t o1[32];
              tmem_ld32(((tmem + C::O1) | lane_off) + c * 32, o1);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(o1[i]) * f1);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f0);
            }
          }
          if (!valid) continue;
          if constexpr (Q8) {
            const float v2 = v_pow2[(piece & 1) * 8 + c];
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * v2);
          }
          if (in.dest != kDirect) {
            store_words<32>(a.part_o + prow * D + c * 32, o, p.wide);
            continue;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
          if (gated) {
            if (!AHEAD_GATE) {
#pragma unroll
              for (int i = 0; i < 8; ++i) gn[i] = __ldg(gate + 8 * c + i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[4 * i] = __float_as_uint(__uint_as_float(o[4 * i]) * sigmoid(gn[i].x));
              o[4 * i + 1] = __float_as_uint(__uint_as_float(o[4 * i + 1]) * sigmoid(gn[i].y));
              o[4 * i + 2] = __float_as_uint(__uint_as_float(o[4 * i + 2]) * sigmoid(gn[i].z));
              o[4 * i + 3] = __float_as_uint(__uint_as_float(o[4 * i + 3]) * sigmoid(gn[i].w));
            }
            if (AHEAD_GATE && c + 1 < D / 32) {
#pragma unroll
              for (int i = 0; i < 8; ++i) gn[i] = __ldg(gate + 8 * (c + 1) + i);
            }
          }
          if (a.out_f16) {
            uint32_t h[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) h[i] = pack_half2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
            store_words<16>(static_cast<__half *>(a.out) + orow * D + c * 32, h, p.wide);
          } else {
            store_words<32>(static_cast<float *>(a.out) + orow * D + c * 32, o, p.wide);
          }
        }
        if (valid && in.dest != kDirect) a.part_ml[prow] = make_float2(M - kUp, L);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[NQT == 2 ? t : 0]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else {
    // ---------------- dequantising producers (q8 pool): warps 12-15 for K, 16-19 for V ----------------
    if constexpr (Q8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
      const int v = warp >= 16, gt = tid - (v ? 512 : 384);
      uint64_t *full = v ? v_full : k_full, *empty = v ? v_empty : k_empty;
      const int8_t *codes = static_cast<const int8_t *>(v ? a.kv.V : a.kv.K);
      const float *scales = v ? a.kv.Vs : a.kv.Ks;
      unsigned char *ring = smem + (v ? C::oV : C::oK);
      constexpr int CPR = D / 16;                // 16-code chunks per row
      constexpr int NCH = KT * CPR / 128;        // chunks per thread of one tile
      PieceWalk walk;
      walk.init(span, a.bv, p.u, ps);
      Piece pc;
      uint32_t t = 0;
      bool have = walk.next(pc, a.bv, p.u, ps), ok = true;
      uint4 w[NCH], wn[NCH];
      float sc[NCH], sn[NCH];
      // codes and block scales of the walk's current tile (zeros behind the length), and on to the next
      static_assert(128 % CPR == 0, "a thread's chunks lie in one block of 32 channels");
      float pow2 = 1.f;  // of the walk's current piece
      if (have) pow2 = pow2_of(top_scale(a, pc, v ? gt % CPR / 2 : kTopK));
      auto fetch = [&](uint4 (&x)[NCH], float (&s)[NCH], float &inv) {
        inv = pow2_inv(pow2) * (1.0f / 127.0f);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const uint32_t idx = gt + i * 128, c = idx % CPR, pos = (pc.tile0 + t) * KT + idx / CPR;
          x[i] = make_uint4(0, 0, 0, 0);
          s[i] = 0.f;
          if (pos < pc.len) {
            const uint32_t pg = (uint32_t)__ldg(pc.pages + (p.page_shift < 32 ? pos >> p.page_shift : pos / ps));
            if (pg < a.kv.num_pages) {
              const uint64_t row = ((uint64_t)pg * ps + (p.page_shift < 32 ? pos & (ps - 1) : pos % ps)) * a.kv.KV + pc.kvh;
              x[i] = __ldg(reinterpret_cast<const uint4 *>(codes + row * D + c * 16));
              s[i] = __ldg(scales + row * (D / 32) + c / 2);
            } else {
              atomicExch(&g_device_error, BG_EINVAL);
            }
          }
        }
        if (++t == pc.ntiles) {
          t = 0;
          have = walk.next(pc, a.bv, p.u, ps);
          if (have) pow2 = pow2_of(top_scale(a, pc, v ? gt % CPR / 2 : kTopK));
        }
      };
      bool more = have;
      float inv = 0.f, inv_next = 0.f;
      if (more) fetch(w, sc, inv);
      for (int it = 0; more; ++it) {
        const bool next = have;
        if (next) fetch(wn, sn, inv_next);  // travels while this tile is converted
        const int s = it % C::NST;
        if (it >= C::NST) ok = mbar_wait_warp(&empty[s], ((it / C::NST) - 1) & 1);
        if (!ok) break;
        unsigned char *dst = ring + s * 2 * C::KVT;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const uint32_t idx = gt + i * 128, r = idx / CPR, c = idx % CPR;
          const CodeScale cs(sc[i] * inv);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // the lanes of a row's second half take their two chunks in the other order: a quarter warp's
            // stores then fall on all banks
            const uint32_t hh = h ^ ((c >> 2) & 1);
            uint4 hi, lo;
            cs.split4(hh ? w[i].z : w[i].x, hi.x, hi.y, lo.x, lo.y);
            cs.split4(hh ? w[i].w : w[i].y, hi.z, hi.w, lo.z, lo.w);
            unsigned char *d = dst + sw_off<KT>(r, 2 * c + hh);
            *reinterpret_cast<uint4 *>(d) = hi;
            *reinterpret_cast<uint4 *>(d + C::KVT) = lo;
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
        more = next;
        inv = inv_next;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          w[i] = wn[i];
          sc[i] = sn[i];
        }
      }
      if (!ok) *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// The largest block scales of the page lists that the tcgen05 kernels read (q8 pool): list blockIdx.z (the sequences
// of more than rows_lo rows, then the prefix), kv head blockIdx.y, by a cluster of kParts blocks.  Reads 1/9 of what
// the lists' K and V have.
constexpr uint32_t kParts = 8;
template <int NB>
__global__ void __cluster_dims__(kParts, 1, 1) __launch_bounds__(512)
    top_scales_kernel(PagedAttnArgs a, uint32_t rows_lo, uint32_t first) {
  __shared__ uint32_t top[kTopRow];
  const uint32_t list = first + blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 31, ps = a.kv.page_size;
  if (threadIdx.x < kTopRow) top[threadIdx.x] = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int32_t *pages = a.bv.prefix_pages;
  uint32_t len = a.bv.prefix_len;
  if (list < a.bv.B) {
    const SeqRange sr = seq_range(a.bv, list, ps);
    pages = a.bv.table + (uint64_t)list * a.bv.table_stride;
    len = sr.n * a.G > rows_lo ? (uint32_t)sr.held : 0;
  }
  constexpr uint32_t abs = 0x7fffffffu;
  uint32_t k = 0, v[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) v[b] = 0;
#pragma unroll 4
  for (uint32_t pos = blockIdx.x * 512 + threadIdx.x; pos < len; pos += kParts * 512) {
    const uint32_t pg = (uint32_t)__ldg(pages + pos / ps);
    if (pg >= a.kv.num_pages) continue;
    const uint64_t row = ((uint64_t)pg * ps + pos % ps) * a.kv.KV + kvh;
    const uint4 *ks = reinterpret_cast<const uint4 *>(a.kv.Ks + row * NB), *vs = reinterpret_cast<const uint4 *>(a.kv.Vs + row * NB);
#pragma unroll
    for (int q = 0; q < NB / 4; ++q) {
      const uint4 x = __ldg(ks + q), y = __ldg(vs + q);
      k = max(k, max(max(x.x & abs, x.y & abs), max(x.z & abs, x.w & abs)));
      v[4 * q] = max(v[4 * q], y.x & abs);
      v[4 * q + 1] = max(v[4 * q + 1], y.y & abs);
      v[4 * q + 2] = max(v[4 * q + 2], y.z & abs);
      v[4 * q + 3] = max(v[4 * q + 3], y.w & abs);
    }
  }
  __syncwarp();
  k = __reduce_max_sync(0xffffffffu, k);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t x = __reduce_max_sync(0xffffffffu, v[b]);
    if (lane == 0) atomicMax(top + b, x);
  }
  if (lane == 0) atomicMax(top + kTopK, k);
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x <= kTopK) {
    uint32_t mx = 0;
#pragma unroll
    for (uint32_t i = 0; i < kParts; ++i) mx = max(mx, cluster.map_shared_rank(top, i)[threadIdx.x]);
    a.tops[((uint64_t)list * a.kv.KV + kvh) * kTopRow + threadIdx.x] = mx;
  }
  cluster.sync();  // nobody's shared memory goes before it is read
}

// Rows of f32 (or, beside an f32 result, f16) as two f16 halves, high ones first, of the row without the power of two
// that its largest value asks for (f32 holds values that f16 does not).  n: values / 8, lpr: a row's (16 or 32 lanes).
// One pass for all kv heads' units, which then fetch their tiles by TMA: loaded and split by two warps of
// the attention kernel, a unit's rows took 8 us at head_dim 128.
__global__ void __launch_bounds__(256) split_rows_kernel(const void *q, int q_f16, uint4 *halves, float *pow2, uint64_t n, uint32_t lpr) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint64_t step = (uint64_t)gridDim.x * 256;
  const uint32_t lane = threadIdx.x & 31;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i - lane < n; i += step) {  // (the same for a whole warp)
    float x[8] = {};
    if (i < n) {
      if (q_f16) load_f16<8>(static_cast<const __half *>(q) + i * 8, x);
      else load_f32<8>(static_cast<const float *>(q) + i * 8, x);
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    for (uint32_t m = lpr >> 1; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    const float p = pow2_of(top), inv = pow2_inv(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= inv;
    if (i >= n) continue;
    uint4 hi, lo;
    split8(x, hi, lo);
    halves[i] = hi;
    halves[n + i] = lo;
    if (lane % lpr == 0) pow2[i / lpr] = p;
  }
}

template <int D, bool Q8, bool LO, int NQT>
int launch_cfg(const PagedAttnArgs &a, uint32_t blocks, uint32_t rows_lo, bool prefix, cudaStream_t st) {
  using C = TcCfg<D, Q8, LO, NQT>;
  const uint32_t ps = a.kv.page_size;
  TcParams p;
  p.a = a;
  // a launch has either the prefix's units or the sequences' own
  p.rpt = kM / a.G * a.G;
  p.u = unit_shape(a.G, a.kv.KV, NQT * p.rpt, C::KT, C::LEAD, prefix ? 0xffffffffu : rows_lo, 0xffffffffu, prefix);
  p.box = page_box(ps, C::KT);
  p.ppt = C::KT / p.box;
  p.page_shift = 32;
  for (uint32_t i = 0; i < 31; ++i)
    if (1u << i == ps) p.page_shift = i;
  p.join_rows = a.own_pieces != nullptr;
  CUtensorMap tk = {}, tv = {}, tq = {};
  p.wide = (((uintptr_t)a.out | (uintptr_t)a.part_o) & 31) == 0;
  // f32 rows: the halves that split_rows_kernel left, the low ones T tokens behind the high ones
  const uint64_t qdims[4] = {D, a.G, a.kv.KV, (uint64_t)C::NQ * a.bv.T};
  const uint64_t qstrides[3] = {D * 2, (uint64_t)a.G * D * 2, (uint64_t)a.H * D * 2};
  const uint32_t qbox[4] = {64, a.G, 1, p.rpt / a.G};
  if (make_tmap_4d(&tq, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, LO ? a.q_halves : a.q, qdims, qstrides, qbox,
                   CU_TENSOR_MAP_SWIZZLE_128B))
    return BG_EUNSUPPORTED;
  if (!Q8) {
    const uint64_t rb = (uint64_t)D * 2;
    const uint64_t dims[4] = {D, a.kv.KV, ps, a.kv.num_pages};
    const uint64_t strides[3] = {rb, rb * a.kv.KV, rb * a.kv.KV * ps};
    const uint32_t box[4] = {64, 1, p.box, 1};
    if (make_tmap_4d(&tk, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.kv.K, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) ||
        make_tmap_4d(&tv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.kv.V, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return BG_EUNSUPPORTED;
  }
  auto kern = paged_tc_kernel<D, Q8, LO, NQT>;
  static unsigned long long allowed = 0;
  if (!allow_smem(kern, C::SMEM, allowed)) return BG_ELAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, tk, tv, tq, p) == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

template <bool Q8>
int launch_q(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_lo, bool prefix, cudaStream_t st) {
  const bool lo = !(a.q_f16 && a.out_f16);
  if (a.D == 256) {
    if (!lo) return launch_cfg<256, Q8, false, 1>(a, blocks, rows_lo, prefix, st);
    return launch_cfg<256, Q8, true, 1>(a, blocks, rows_lo, prefix, st);
  }
  if (lo) return launch_cfg<128, Q8, true, 1>(a, blocks, rows_lo, prefix, st);
  return ru > kM ? launch_cfg<128, Q8, false, 2>(a, blocks, rows_lo, prefix, st)
                   : launch_cfg<128, Q8, false, 1>(a, blocks, rows_lo, prefix, st);
}

}  // namespace

// Page boxes of at least 8 positions keep the 128-byte swizzle's pattern.
bool paged_tc_supported(int mode, uint32_t D, uint32_t G, uint32_t KV, uint32_t page_size) {
  return G <= kM && KV <= 65535 && page_size % 8 == 0 && (D == 128 || D == 256) && (mode == BG_KV_F16 || mode == BG_KV_Q8);
}

// Rows of a unit: whole tokens' heads, two query tiles where there are rows for them and memory for both (f16
// rows of head_dim 128).
uint32_t paged_tc_rows(uint32_t D, uint32_t G, bool lo, uint64_t rows) {
  const uint32_t tile = kM / G * G;
  return D == 128 && !lo && rows > tile ? 2 * tile : tile;
}

int launch_paged_split_rows(const PagedAttnArgs &a, cudaStream_t st) {
  const uint64_t n = (uint64_t)a.bv.T * a.H * a.D / 8, blocks = (n + 255) / 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((uint32_t)(blocks < 148 * 8 ? blocks : 148 * 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, split_rows_kernel, a.q, a.q_f16, static_cast<uint4 *>(a.q_halves), a.q_pow2, n, a.D / 8) ==
                 cudaSuccess
             ? BG_OK
             : BG_ELAUNCH;
}

int launch_paged_top_scales(const PagedAttnArgs &a, uint32_t rows_lo, bool own, bool prefix, cudaStream_t st) {
  const uint32_t first = own ? 0 : a.bv.B, end = a.bv.B + (prefix ? 1 : 0);
  for (uint32_t l = first; l < end; l += 65535) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kParts, a.kv.KV, end - l < 65535 ? end - l : 65535);
    cfg.blockDim = dim3(512);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = a.D == 128 ? cudaLaunchKernelEx(&cfg, top_scales_kernel<4>, a, rows_lo, l)
                                     : cudaLaunchKernelEx(&cfg, top_scales_kernel<8>, a, rows_lo, l);
    if (e != cudaSuccess) return BG_ELAUNCH;
  }
  return BG_OK;
}

int launch_paged_tc(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_lo, bool prefix, cudaStream_t st) {
  return a.mode == BG_KV_Q8 ? launch_q<true>(a, blocks, ru, rows_lo, prefix, st)
                            : launch_q<false>(a, blocks, ru, rows_lo, prefix, st);
}

int poll_device_error_paged_tc() {
  int v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return BG_ELAUNCH;
  if (v) cudaMemcpyToSymbol(g_device_error, &z, sizeof(int));
  return v;
}

}  // namespace bg
