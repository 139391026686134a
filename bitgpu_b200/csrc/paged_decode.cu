// Tensor-core attention over a paged cache for few rows a unit (decode, verification, small shared
// prefixes), f16 and q8 pools, head_dim 128 and 256.
//
//   s_j = q . K[j] * scale * log2(e),  out = sum_j 2^(s_j - m) V[j] / sum_j 2^(s_j - m)
//
// Bound: HBM -- each K/V position is read once for up to 16 rows.  Layout of the work:
//   * the batch's K/V tiles (64 positions of one kv head) form one line that the blocks share out
//     evenly (TileSpan in paged.h), so lengths need not be alike and nothing waits for the longest;
//   * a producer warp walks the block's pieces of units, fetches page ids a tile ahead, and streams
//     K and V page by page with 4-D TMA boxes (128-byte swizzle) into an mbarrier ring; q8 block scales
//     (16-byte rows) come by cp.async.  It also stages each unit's query rows and its description, so
//     the consumers never wait for global memory.  Positions behind the length are not fetched: their
//     boxes lie outside the tensor map and read as zeros;
//   * four consumer warps take 16 positions of a tile each.  Scores are computed transposed (m16n8k16
//     with positions on M, up to 8 query rows on N), and so is the output, O^T = V^T P^T; P reaches the
//     B operand in registers through movmatrix;
//   * f32 rows (LO): q, without the power of two of its row's largest value (which the softmax scale puts back), and p
//     are split into two f16 operands (22 bits).  Up to four rows a unit (PK; one
//     token of a group of four heads) the halves share one product, hi in columns 0-3 and lo in 4-7 of the
//     MMA's eight; otherwise both products run twice.  f16 rows: q is exact and p is rounded once to f16,
//     which costs about as much as the rounding of the result.  p carries a factor 2^14, which cancels in the
//     quotient and keeps small weights out of f16's subnormals;
//   * q8: the weights of V's codes are p * block scale / 127, of any magnitude.  Each warp's 16 positions and each
//     block of 32 channels have a power of two that brings the largest to [2^14, 2^15); their products start from
//     zero and join the output by one fused multiply-add that puts the power back;
//   * q8 codes enter the products as exact f16 integers, -128 as -127: byte + 128 under the f16 pattern 0x64xx is
//     1152 + code; less 1025, cut at 0, it is code + 127, and one more packed subtraction leaves the code (32 streams
//     75 us; 71 without the cut, 77 with a packed maximum instead, which is not the FMA pipe's).  (Cancelling what is
//     left inside the MMA instead costs accuracy: the f32 accumulator then holds sums 1152 / |code| times as large.)
#include <cuda.h>
#include <string.h>

#include "mma.cuh"
#include "paged.h"
#include "paged_merge.cuh"
#include "tma.cuh"

namespace bg {
namespace {

constexpr int kTile = 64;    // positions per tile
constexpr int kConsumers = 4;
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kUnits = 2;    // staged units
// tiles' time that a unit costs beside its tiles (64 short own parts: 0 55.8 us a call, 1 52.1, 2 52.1)
constexpr int kLead = 1;

struct DecodeParams {
  PagedAttnArgs a;
  UnitShape u;
  uint32_t ppt;         // page boxes per tile
  uint32_t box;         // positions per box
  uint32_t join_rows;   // 1: every unit leaves partial rows (a shared prefix exists)
};

struct alignas(16) UnitInfo {
  uint32_t R0, rows, kvh, tile0, ntiles, len;
  int32_t lim_base;
  uint32_t dest;  // partial row of the unit's row 0, kDirect or kRowBuf
  uint32_t row0;  // kRowBuf: first partial row of the row-indexed area
};
constexpr uint32_t kDirect = 0xffffffffu, kRowBuf = 0xfffffffeu;

template <int MODE, int D, int NT>
struct DecCfg {
  static constexpr int ES = MODE == BG_KV_F16 ? 2 : 1;
  static constexpr int ROWB = D * ES;
  static constexpr int NCB = ROWB / 128;
  static constexpr int KVT = kTile * ROWB;
  static constexpr int NB = D / 32;
  static constexpr int SCT = MODE == BG_KV_Q8 ? kTile * NB * 4 : 0;
  static constexpr int STAGE = 2 * KVT + 2 * SCT;
  static constexpr int NN = NT * 8;
  static constexpr int QROW = D * 4 + 32;             // f32 row + 32 bytes: rows on distinct banks
  static constexpr int DP = D + 4;
  static constexpr int QSLOT = NN * QROW;             // also holds half of the epilogue's sums
  static constexpr int EPI = NN * DP * 4;
  static constexpr int CTAS = D == 256 ? 1 : MODE == BG_KV_Q8 && NT == 1 ? 3 : 2;  // blocks per SM
  static constexpr int FIXED = kUnits * QSLOT + EPI + 10 * NN * 4 + kUnits * 64 + 512;
  static constexpr int ROOM = (232448 / CTAS - 1024) / 16 * 16 - FIXED;
  static constexpr int NST_RAW = ROOM / STAGE;
  static constexpr int NST = NST_RAW > 6 ? 6 : NST_RAW;
  static_assert(NST >= 2, "ring");
  static constexpr int oQ = NST * STAGE, oE = oQ + kUnits * QSLOT, oM = oE + EPI, oU = oM + 10 * NN * 4,
                       oB = (oU + kUnits * 64 + 15) / 16 * 16;
  static constexpr int SMEM = oB + 384;
};

template <int MODE, int D, int NT, bool LO, bool PK>
__global__ void __launch_bounds__(kThreads, DecCfg<MODE, D, NT>::CTAS)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, DecodeParams p) {
  using C = DecCfg<MODE, D, NT>;
  constexpr int NST = C::NST, NB = C::NB, KS = D / 16, NN = C::NN;
  static_assert(!PK || (LO && NT == 1), "packed halves");
  constexpr bool TWO = LO && !PK;  // the low halves have products of their own
  constexpr float kShift = MODE == BG_KV_F16 ? 14.f : 0.f;  // log2 of the factor that p carries
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::oB);
  uint64_t *empty = full + NST, *ufull = empty + NST, *uempty = ufull + kUnits;
  uint64_t *meet = uempty + kUnits;  // the consumer warps' barrier
  uint32_t *scan = reinterpret_cast<uint32_t *>(meet + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedAttnArgs &a = p.a;
  if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; dynamic shared memory starts on such a border
    atomicExch(&g_device_error, BG_ELAUNCH);
    return;
  }

  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], MODE == BG_KV_Q8 ? 33 : 1);
      mbar_init(&empty[s], kConsumers);
    }
    for (int s = 0; s < kUnits; ++s) {
      mbar_init(&ufull[s], 33);  // 32 lanes' copies of the query rows, and the description
      mbar_init(&uempty[s], kConsumers);
    }
    mbar_init(meet, kConsumers);
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const TileSpan span = block_span<kThreads>(a.bv, p.u, a.kv.page_size, a.min_tiles, scan, &g_device_error);

  if (warp == kConsumers) {  // ---------------- producer ----------------
    PieceWalk walk;
    walk.init(span, a.bv, p.u, a.kv.page_size);
    if (a.cuts && lane == 0) a.cuts[blockIdx.x].npieces = 0;
    Piece pc;
    bool ok = true;
    int it = 0, un = 0;
    const uint32_t ps = a.kv.page_size;
    while (ok && walk.next(pc, a.bv, p.u, ps)) {
      // page id of this lane's box of tile `tile` (num_pages: outside the pool, reads as zeros)
      auto page_of = [&](uint32_t tile) -> uint32_t {
        const uint32_t pos = (pc.tile0 + tile) * kTile + lane * p.box;
        if ((uint32_t)lane >= p.ppt || tile >= pc.ntiles || pos >= pc.len) return a.kv.num_pages;
        const uint32_t pg = (uint32_t)__ldg(pc.pages + pos / ps);
        if (pg < a.kv.num_pages) return pg;
        atomicExch(&g_device_error, BG_EINVAL);
        return a.kv.num_pages;
      };
      uint32_t pg_next = page_of(0);
      // ---- its tiles ----
      // A sequence's own K and V are read once and leave L2 first (64 streams of up to 32768: 640 -> 628 us).
      const uint64_t policy = l2_policy(pc.own);
      for (uint32_t t = 0; t < pc.ntiles; ++t) {
        const uint32_t pg = pg_next;
        pg_next = page_of(t + 1);
        const int s = it % NST;
        if (it >= NST) ok = mbar_wait_warp(&empty[s], ((it / NST) - 1) & 1);
        if (!ok) break;
        unsigned char *st = smem + s * C::STAGE;
        const uint32_t pos0 = (pc.tile0 + t) * kTile;
        if (lane == 0) mbar_expect_tx(&full[s], 2 * C::KVT);
        __syncwarp();
        if ((uint32_t)lane < p.ppt) {
          const int slot_y = (int)((pos0 + lane * p.box) % ps);
          unsigned char *dst = st + lane * p.box * 128;
#pragma unroll
          for (int cb = 0; cb < C::NCB; ++cb) {
            tma_load_4d_hint(dst + cb * kTile * 128, &tmK, &full[s], cb * (128 / C::ES), (int)pc.kvh, slot_y, (int)pg, policy);
            tma_load_4d_hint(dst + C::KVT + cb * kTile * 128, &tmV, &full[s], cb * (128 / C::ES), (int)pc.kvh, slot_y, (int)pg,
                             policy);
          }
        }
        if constexpr (MODE == BG_KV_Q8) {
          constexpr int CPR = NB / 4;  // 16-byte chunks per scale row
          const uint32_t sbase = smem_u32(st + 2 * C::KVT);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t r = lane + 32 * i, pos = pos0 + r;
            const uint32_t rp = __shfl_sync(0xffffffffu, pg, p.ppt > 1 ? r / p.box : 0);
            const bool valid = pos < pc.len && rp < a.kv.num_pages;
            const uint64_t row = valid ? ((uint64_t)rp * ps + pos % ps) * a.kv.KV + pc.kvh : 0;
#pragma unroll
            for (int c = 0; c < 2 * CPR; ++c) {
              const int which = c / CPR, gc = c % CPR;
              const float *src = (which ? a.kv.Vs : a.kv.Ks) + row * NB + gc * 4;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sbase + which * C::SCT + (r * NB + gc * 4) * 4),
                           "l"(src), "r"(valid ? 16u : 0u)
                           : "memory");
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
        }
        ++it;
        if (t > 0) continue;
        // the first tile travels while the unit is made ready: its description and query rows
        const int us = un % kUnits;
        if (un >= kUnits) ok = mbar_wait_warp(&uempty[us], ((un / kUnits) - 1) & 1);
        if (!ok) break;
        const bool whole = pc.npieces == 1;
        const uint32_t slot = a.slot0 + (2 * blockIdx.x + (pc.starts ? 1 : 0)) * p.u.RU;
        if (lane == 0) {
          UnitInfo *ui = reinterpret_cast<UnitInfo *>(smem + C::oU + us * 64);
          ui->R0 = pc.R0;
          ui->rows = pc.rows;
          ui->kvh = pc.kvh;
          ui->tile0 = pc.tile0;
          ui->ntiles = pc.ntiles;
          ui->len = pc.len;
          ui->lim_base = pc.lim_base;
          ui->dest = !whole ? slot : p.join_rows ? kRowBuf : kDirect;
          ui->row0 = pc.own ? a.own_row0 : a.pre_row0;
        }
        if (p.join_rows) {
          if (pc.starts && (uint32_t)lane < pc.rows) {  // where the row's pieces will be
            const uint32_t R = pc.R0 + lane;
            RowPieces rp;
            rp.idx0 = whole ? (pc.own ? a.own_row0 : a.pre_row0) + R / a.G * a.H + pc.kvh * a.G + R % a.G : slot + lane;
            rp.npieces = pc.npieces;
            rp.step = p.u.RU;
            rp.pad = 0;
            (pc.own ? a.own_pieces : a.pre_pieces)[(uint64_t)pc.kvh * a.bv.T * a.G + R] = rp;
          }
        } else if (!whole && pc.starts && lane == 0) {
          a.cuts[blockIdx.x] = CutUnit{pc.R0, pc.rows, pc.kvh, pc.npieces};
        }
        {
          const uint32_t cpr = a.q_f16 ? D / 8 : D / 4;  // 16-byte chunks per query row
          const uint32_t qb = smem_u32(smem + C::oQ + us * C::QSLOT);
          const uint32_t stride = a.q_f16 ? D * 2 + 16 : C::QROW;
          const uint32_t tok0 = pc.R0 / a.G, g0 = pc.R0 % a.G;
          for (uint32_t idx = lane; idx < NN * cpr; idx += 32) {
            const uint32_t r = idx / cpr, c = idx % cpr;
            uint32_t tok = tok0, g = g0 + r;
            while (g >= a.G) {
              g -= a.G;
              ++tok;
            }
            const bool there = r < pc.rows;
            const uint64_t off = there ? ((uint64_t)tok * a.H + pc.kvh * a.G + g) * cpr + c : 0;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(qb + r * stride + c * 16),
                         "l"(static_cast<const uint4 *>(a.q) + off), "r"(there ? 16u : 0u)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ufull[us])) : "memory");
          if (lane == 0) mbar_arrive(&ufull[us]);
        }
        ++un;
      }
    }
    // the end: a unit without tiles
    if (ok) {
      const int us = un % kUnits;
      if (un >= kUnits) ok = mbar_wait_warp(&uempty[us], ((un / kUnits) - 1) & 1);
      if (ok) {
        if (lane == 0) reinterpret_cast<UnitInfo *>(smem + C::oU + us * 64)->ntiles = 0;
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ufull[us])) : "memory");
        if (lane == 0) mbar_arrive(&ufull[us]);
      }
    }
    // never leave the block with copies in flight: wait (bounded) for the last stages
    if (lane == 0)
      for (int i = max(0, it - NST); i < it; ++i) mbar_wait(&full[i % NST], (i / NST) & 1);
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ---------------- consumers ----------------
  const int lrow = (((lane >> 3) & 1) << 3) + (lane & 7);  // ldmatrix row for matrices {0,1},{2,3}
  const int lhi = lane >> 4;
  const int trow = ((lane >> 4) << 3) + (lane & 7);        // transposed f16 V: matrices (pos, d) order
  const int tcol = (lane >> 3) & 1;
  float *mw = reinterpret_cast<float *>(smem + C::oM);  // [4][NN] m, [4][NN] l, [NN] M, [NN] L
  float *lw = mw + 4 * NN, *mrow = lw + 4 * NN, *lrow_s = mrow + NN;
  const float sl2 = a.sl2;
  int it = 0;
  uint32_t met = 0;
  // all consumer warps; bounded like every wait, so that a warp that gave up leaves no other hanging
  auto meet_all = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(meet);
    return mbar_wait_warp(meet, met++ & 1);
  };
  for (int un = 0;; ++un) {
    const int us = un % kUnits;
    if (!mbar_wait_warp(&ufull[us], (un / kUnits) & 1)) return;
    const UnitInfo ui = *reinterpret_cast<const UnitInfo *>(smem + C::oU + us * 64);
    if (ui.ntiles == 0) return;

    // Q^T operand fragments (B of m16n8k16): column n = lane / 4, k pairs
    uint32_t qh[NT][KS][2], ql[TWO ? NT : 1][TWO ? KS : 1][2];
    int32_t lim[NT][2];  // last attended position of the lane's score columns
    float sl[NT][2];     // and their softmax scale, times their row's power of two
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = PK ? (lane >> 2) & 3 : nt * 8 + (lane >> 2);
      const unsigned char *qr = smem + C::oQ + us * C::QSLOT + r * (a.q_f16 ? D * 2 + 16 : C::QROW);
      float pow2 = 1.f, inv = 1.f;  // of the row's values
      if (LO && !a.q_f16) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {  // four lanes have a quarter each
          const uint4 v = *reinterpret_cast<const uint4 *>(qr + (4 * i + (lane & 3)) * 16);
          constexpr uint32_t abs = 0x7fffffffu;
          top = max(top, max(max(v.x & abs, v.y & abs), max(v.z & abs, v.w & abs)));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        pow2 = pow2_of(top);
        inv = pow2_inv(pow2);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // f16 pool: k slots 2j,2j+1 (+8) <-> dims 2j,2j+1 (+8); q8: the byte-pair order of the int8
          // fragments, dims 4j,4j+1 (half 0) and 4j+2,4j+3 (half 1), j = lane % 4
          const int d = MODE == BG_KV_Q8 ? ks * 16 + 4 * (lane & 3) + 2 * half : ks * 16 + 2 * (lane & 3) + 8 * half;
          if (a.q_f16) {
            qh[nt][ks][half] = PK && lane >= 16 ? 0u : *reinterpret_cast<const uint32_t *>(qr + d * 2);
            if constexpr (TWO) ql[nt][ks][half] = 0;
          } else {
            float2 v = *reinterpret_cast<const float2 *>(qr + d * 4);
            v.x *= inv;
            v.y *= inv;
            const uint32_t h = pack_f16(v.x, v.y);
            qh[nt][ks][half] = h;
            if constexpr (LO) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
              const uint32_t lo = pack_f16(v.x - f.x, v.y - f.y);
              if constexpr (TWO) ql[nt][ks][half] = lo;
              else if (lane >= 16) qh[nt][ks][half] = lo;
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t col = nt * 8 + 2 * (lane & 3) + j, rc = min(PK ? col & 3 : col, ui.rows - 1);
        sl[nt][j] = LO ? sl2 * __shfl_sync(0xffffffffu, pow2, 8 * (lane & 3) + 4 * j) : sl2;
        lim[nt][j] = min(ui.lim_base + (int32_t)((ui.R0 + rc) / a.G), (int32_t)ui.len - 1);
      }
    }

    float m[NT][2], l[NT][2];
    float oacc[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kNegBig;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) oacc[nt][mt][i] = 0.f;
    }

    for (uint32_t t = 0; t < ui.ntiles; ++t, ++it) {
      const int s = it % NST;
      if (!mbar_wait_warp(&full[s], (it / NST) & 1)) return;
      const uint32_t kb = smem_u32(smem + s * C::STAGE), vb = kb + C::KVT;
      const int row0 = warp * 16;
      const int32_t base = (int32_t)((ui.tile0 + t) * kTile) + row0;
      const int32_t pa = base + (lane >> 2), pb = pa + 8;

      // ---- scores S^T[pos][n] ----
      float sc[NT][4];
      if constexpr (MODE == BG_KV_F16) {
        // two accumulator chains (the halves of Q, or even and odd steps) instead of one long one
        float acc[NT][4], acl[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][i] = acl[nt][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t f[4];
          ldsm_x4(f, swz<kTile>(kb, row0 + lrow, 2 * ks + lhi));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (TWO) {
              mma16816(acc[nt], f, qh[nt][ks][0], qh[nt][ks][1]);
              mma16816(acl[nt], f, ql[nt][ks][0], ql[nt][ks][1]);
            } else {
              mma16816(ks & 1 ? acl[nt] : acc[nt], f, qh[nt][ks][0], qh[nt][ks][1]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[nt][i] = (acc[nt][i] + acl[nt][i]) * sl[nt][i & 1];
            if constexpr (PK) sc[nt][i] += __shfl_xor_sync(0xffffffffu, sc[nt][i], 2);
          }
      } else {
        const float *ksc = reinterpret_cast<const float *>(smem + s * C::STAGE + 2 * C::KVT);
        const __half2 one = __float2half2_rn(1.f), bias = __float2half2_rn(-1025.f), least = __float2half2_rn(127.f);
        auto code = [&](uint32_t w, uint32_t sel) {
          const uint32_t x = i8pair_biased(w, sel);
          const __half2 h = __hsub2(__hfma2_relu(*reinterpret_cast<const __half2 *>(&x), one, bias), least);
          return *reinterpret_cast<const uint32_t *>(&h);
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
#pragma unroll
        for (int bk = 0; bk < NB; ++bk) {
          uint32_t r[4];
          ldsm_x4(r, swz<kTile>(kb, row0 + lrow, 2 * bk + lhi));
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
          const uint32_t a0[4] = {code(r[0], kSelLo), code(r[1], kSelLo), code(r[0], kSelHi), code(r[1], kSelHi)};
          const uint32_t a1[4] = {code(r[2], kSelLo), code(r[3], kSelLo), code(r[2], kSelHi), code(r[3], kSelHi)};
          const float sa = ksc[(row0 + (lane >> 2)) * NB + bk] * (LO ? 1.0f / 127.0f : sl2 * (1.0f / 127.0f));
          const float sb = ksc[(row0 + (lane >> 2) + 8) * NB + bk] * (LO ? 1.0f / 127.0f : sl2 * (1.0f / 127.0f));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(acc, a0, qh[nt][2 * bk][0], qh[nt][2 * bk][1]);
            mma16816(acc, a1, qh[nt][2 * bk + 1][0], qh[nt][2 * bk + 1][1]);
            if constexpr (TWO) {
              mma16816(acc, a0, ql[nt][2 * bk][0], ql[nt][2 * bk][1]);
              mma16816(acc, a1, ql[nt][2 * bk + 1][0], ql[nt][2 * bk + 1][1]);
            }
            sc[nt][0] = fmaf(acc[0], sa, sc[nt][0]);
            sc[nt][1] = fmaf(acc[1], sa, sc[nt][1]);
            sc[nt][2] = fmaf(acc[2], sb, sc[nt][2]);
            sc[nt][3] = fmaf(acc[3], sb, sc[nt][3]);
          }
        }
        if constexpr (LO) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][i] *= sl[nt][i & 1];
        }
        if constexpr (PK) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[0][i] += __shfl_xor_sync(0xffffffffu, sc[0][i], 2);
        }
      }

      // ---- online softmax (columns 2(lane%4) + j; rows pa, pb) ----
      float pr[NT][4], cr[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x0 = pa <= lim[nt][j] ? sc[nt][j] : -INFINITY;
          const float x1 = pb <= lim[nt][j] ? sc[nt][2 + j] : -INFINITY;
          float mx = fmaxf(x0, x1);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[nt][j], mx), corr = exp2f(m[nt][j] - mn), mo = mn - kShift;
          const float p0 = exp2f(x0 - mo), p1 = exp2f(x1 - mo);
          l[nt][j] = l[nt][j] * corr + (p0 + p1);
          m[nt][j] = mn;
          pr[nt][j] = p0;
          pr[nt][2 + j] = p1;
          cr[nt][j] = corr;
          moved |= corr != 1.0f;
        }
      }
      // f16 rows, q8 pool: rescale the output only when a running max of this warp moved.  f32 rows: every tile's
      // products start from zero and are added to the rescaled output by one fused multiply-add per
      // value -- the MMA truncates what it accumulates, and over the ~100 tiles of a long split that bias
      // alone (3e-6 at 131072 positions) is more than all other errors together.
      if ((!LO || MODE == BG_KV_Q8) && __any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[nt][mt][i] *= cr[nt][i & 1];
      }

      // ---- O^T += V^T . P^T ----
      auto split = [&](float x, float y, uint32_t &hi, uint32_t &lo) {
        uint32_t h = pack_f16(x, y);
        if constexpr (LO) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
          const uint32_t l = pack_f16(x - f.x, y - f.y);
          if constexpr (TWO) lo = movm_t(l);
          else if (lane & 2) h = l;  // columns 4-7
        }
        hi = movm_t(h);
      };
      if constexpr (MODE == BG_KV_F16) {
        uint32_t pb0[NT], pb1[NT], pl0[NT], pl1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          split(pr[nt][0], pr[nt][1], pb0[nt], pl0[nt]);
          split(pr[nt][2], pr[nt][3], pb1[nt], pl1[nt]);
        }
        // slots behind the length may hold NaN, and 0 * NaN is NaN: clear their V values
        const int32_t left = (int32_t)ui.len - base - 2 * (lane & 3);
        const bool tail = base + 16 > (int32_t)ui.len;
        uint32_t mk0 = 0xffffffffu, mk1 = 0xffffffffu;
        if (tail) {
          mk0 = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
          mk1 = left >= 10 ? 0xffffffffu : left == 9 ? 0xffffu : 0u;
        }
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          uint32_t f[4];
          ldsm_x4_t(f, swz<kTile>(vb, row0 + trow, 2 * mt + tcol));
          if (tail) {
            f[0] &= mk0;
            f[1] &= mk0;
            f[2] &= mk1;
            f[3] &= mk1;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (LO) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              if constexpr (TWO) mma16816(acc, f, pl0[nt], pl1[nt]);
              mma16816(acc, f, pb0[nt], pb1[nt]);
#pragma unroll
              for (int i = 0; i < 4; ++i) oacc[nt][mt][i] = fmaf(oacc[nt][mt][i], cr[nt][i & 1], acc[i]);
            } else {
              mma16816(oacc[nt][mt], f, pb0[nt], pb1[nt]);
            }
          }
        }
      } else {
        const float *vsc = reinterpret_cast<const float *>(smem + s * C::STAGE + 2 * C::KVT + C::SCT);
        const __half2 one = __float2half2_rn(1.f), bias = __float2half2_rn(-1025.f), least = __float2half2_rn(127.f);
        auto code = [&](uint32_t w, uint32_t sel) {
          const uint32_t x = i8pair_biased(w, sel);
          const __half2 h = __hsub2(__hfma2_relu(*reinterpret_cast<const __half2 *>(&x), one, bias), least);
          return *reinterpret_cast<const uint32_t *>(&h);
        };
#pragma unroll
        for (int bk = 0; bk < NB; ++bk) {
          const float va = vsc[(row0 + (lane >> 2)) * NB + bk] * (1.0f / 127.0f);
          const float vbb = vsc[(row0 + (lane >> 2) + 8) * NB + bk] * (1.0f / 127.0f);
          float w[NT][4], top = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            w[nt][0] = pr[nt][0] * va;
            w[nt][1] = pr[nt][1] * va;
            w[nt][2] = pr[nt][2] * vbb;
            w[nt][3] = pr[nt][3] * vbb;
            top = fmaxf(fmaxf(top, fmaxf(fabsf(w[nt][0]), fabsf(w[nt][1]))), fmaxf(fabsf(w[nt][2]), fabsf(w[nt][3])));
          }
          // `back`: the power of two of the largest weight, over 2^14 (at least 2^-126); `fore`: its inverse
          const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
          const uint32_t e = (uint32_t)max((int)(bits & 0x7f800000u) - (14 << 23), 1 << 23);
          const float back = __uint_as_float(e), fore = __uint_as_float(0x7f000000u - e);
          uint32_t pb0[NT], pb1[NT], pl0[NT], pl1[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            split(w[nt][0] * fore, w[nt][1] * fore, pb0[nt], pl0[nt]);
            split(w[nt][2] * fore, w[nt][3] * fore, pb1[nt], pl1[nt]);
          }
          uint32_t r[4];
          ldsm_x4_t(r, swz<kTile>(vb, row0 + lrow, 2 * bk + lhi));
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
          const uint32_t a0[4] = {code(r[0], kSelEven), code(r[0], kSelOdd), code(r[1], kSelEven), code(r[1], kSelOdd)};
          const uint32_t a1[4] = {code(r[2], kSelEven), code(r[2], kSelOdd), code(r[3], kSelEven), code(r[3], kSelOdd)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float x0[4] = {0.f, 0.f, 0.f, 0.f}, x1[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (TWO) {
              mma16816(x0, a0, pl0[nt], pl1[nt]);
              mma16816(x1, a1, pl0[nt], pl1[nt]);
            }
            mma16816(x0, a0, pb0[nt], pb1[nt]);
            mma16816(x1, a1, pb0[nt], pb1[nt]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              oacc[nt][2 * bk][i] = fmaf(x0[i], back, oacc[nt][2 * bk][i]);
              oacc[nt][2 * bk + 1][i] = fmaf(x1[i], back, oacc[nt][2 * bk + 1][i]);
            }
          }
        }
      }
      release_read(&empty[s]);
    }

    // ---- the four warps' states meet ----
    // each warp publishes (m, l) per column and scales its own o by 2^(m_warp - M); warps 2 and 3
    // store theirs, warps 0 and 1 add their own to them in place, and every thread adds the two halves
    float *e0 = reinterpret_cast<float *>(smem + C::oE);
    float *e1 = reinterpret_cast<float *>(smem + C::oQ + us * C::QSLOT);  // the unit's query rows are in registers
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float lt = l[nt][j];
        lt += __shfl_xor_sync(0xffffffffu, lt, 4);
        lt += __shfl_xor_sync(0xffffffffu, lt, 8);
        lt += __shfl_xor_sync(0xffffffffu, lt, 16);
        const int n = nt * 8 + 2 * (lane & 3) + j;
        if (lane < 4) {
          mw[warp * NN + n] = m[nt][j];
          lw[warp * NN + n] = lt;
        }
      }
    }
    if (!meet_all()) return;
    float fs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = nt * 8 + 2 * (lane & 3) + j;
        float M = kNegBig, L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, mw[w * NN + n]);
        fs[nt][j] = exp2f(mw[warp * NN + n] - M);
        if (warp == 0 && lane < 4) {
#pragma unroll
          for (int w = 0; w < 4; ++w) L = fmaf(lw[w * NN + n], exp2f(mw[w * NN + n] - M), L);
          mrow[n] = M - kShift;
          lrow_s[n] = L;
        }
      }
    }
    float *mine = warp & 1 ? e1 : e0;
    auto each = [&](auto f) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const int d = MODE == BG_KV_F16 ? mt * 16 + (lane >> 2) + 8 * hh : mt * 16 + 2 * (lane >> 2) + hh;
              f(mine + (nt * 8 + 2 * (lane & 3) + j) * C::DP + d, oacc[nt][mt][2 * hh + j] * fs[nt][j]);
            }
    };
    if (warp >= 2) each([](float *x, float v) { *x = v; });
    if (!meet_all()) return;
    if (warp < 2) each([](float *x, float v) { *x += v; });
    if (!meet_all()) return;
    for (uint32_t idx = tid; idx < ui.rows * (D / 4); idx += kConsumers * 32) {
      const uint32_t n = idx / (D / 4), d = idx % (D / 4) * 4;
      const float4 x = *reinterpret_cast<const float4 *>(e0 + n * C::DP + d);
      const float4 y = *reinterpret_cast<const float4 *>(e1 + n * C::DP + d);
      float o[4] = {x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w};
      if constexpr (PK) {  // the low halves' columns
        const float4 z = *reinterpret_cast<const float4 *>(e0 + (n + 4) * C::DP + d);
        const float4 w = *reinterpret_cast<const float4 *>(e1 + (n + 4) * C::DP + d);
        o[0] += z.x + w.x;
        o[1] += z.y + w.y;
        o[2] += z.z + w.z;
        o[3] += z.w + w.w;
      }
      const uint32_t R = ui.R0 + n;
      const uint64_t row = (uint64_t)(R / a.G) * a.H + ui.kvh * a.G + R % a.G;
      if (ui.dest == kDirect) {
        write_out4(a.out, a.out_f16, a.gate, row * D + d, o, lrow_s[n]);
      } else {
        const uint64_t idx_p = ui.dest == kRowBuf ? ui.row0 + row : ui.dest + n;
        *reinterpret_cast<float4 *>(a.part_o + idx_p * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) a.part_ml[idx_p] = make_float2(mrow[n], lrow_s[n]);
      }
    }
    release_read(&uempty[us]);
    if (!meet_all()) return;  // mw .. and e0 are free again
  }
}

template <int MODE, int D, int NT, bool LO, bool PK = false>
int launch_cfg(const PagedAttnArgs &a, uint32_t blocks, uint32_t rows_hi, bool prefix, cudaStream_t st) {
  using C = DecCfg<MODE, D, NT>;
  const uint32_t ps = a.kv.page_size;
  DecodeParams p;
  p.a = a;
  p.u = unit_shape(a.G, a.kv.KV, PK ? 4 : 8 * NT, kTile, kLead, 0, rows_hi, prefix);
  p.box = page_box(ps, kTile);
  p.ppt = kTile / p.box;
  p.join_rows = a.own_pieces != nullptr;
  CUtensorMap tk, tv;
  const uint64_t rb = (uint64_t)D * C::ES;
  const uint64_t dims[4] = {D, a.kv.KV, ps, a.kv.num_pages};
  const uint64_t strides[3] = {rb, rb * a.kv.KV, rb * a.kv.KV * ps};
  const uint32_t box[4] = {128 / C::ES, 1, p.box, 1};
  const CUtensorMapDataType dt = MODE == BG_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  // L2 fetches no more than a head's row: promoted to 256 bytes, a 128-byte q8 row brings its neighbour head's,
  // whose block comes by much later (32 streams: 423 MB read for caches of 321 MB)
  const auto fetch = rb >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
  if (make_tmap_4d(&tk, dt, a.kv.K, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, fetch)) return BG_EUNSUPPORTED;
  if (make_tmap_4d(&tv, dt, a.kv.V, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, fetch)) return BG_EUNSUPPORTED;
  auto kern = paged_decode_kernel<MODE, D, NT, LO, PK>;
  static unsigned long long allowed = 0;
  if (!allow_smem(kern, C::SMEM, allowed)) return BG_ELAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, tk, tv, p) == cudaSuccess ? BG_OK : BG_ELAUNCH;
}

template <int MODE, int D>
int launch_md(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_hi, bool prefix, cudaStream_t st) {
  const bool lo = !(a.q_f16 && a.out_f16);
  if (ru == 4) return launch_cfg<MODE, D, 1, true, true>(a, blocks, rows_hi, prefix, st);
  if (ru == 8)
    return lo ? launch_cfg<MODE, D, 1, true>(a, blocks, rows_hi, prefix, st)
              : launch_cfg<MODE, D, 1, false>(a, blocks, rows_hi, prefix, st);
  if constexpr (D == 128)  // f32 rows of head_dim 256 come in units of 8
    if (lo) return launch_cfg<MODE, D, 2, true>(a, blocks, rows_hi, prefix, st);
  return launch_cfg<MODE, D, 2, false>(a, blocks, rows_hi, prefix, st);
}

}  // namespace

// Page boxes of at least 8 positions keep the 128-byte swizzle's pattern.
bool paged_decode_supported(int mode, uint32_t D, uint32_t page_size) {
  return (mode == BG_KV_F16 || mode == BG_KV_Q8) && (D == 128 || D == 256) && page_size % 8 == 0;
}

uint32_t paged_decode_blocks(int mode, uint32_t D, uint32_t ru) {
  return 148 * (D == 256 ? 1 : mode == BG_KV_Q8 && ru <= 8 ? 3 : 2);
}

int launch_paged_decode(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_hi, bool prefix,
                        cudaStream_t st) {
  if (a.mode == BG_KV_F16)
    return a.D == 128 ? launch_md<BG_KV_F16, 128>(a, blocks, ru, rows_hi, prefix, st)
                      : launch_md<BG_KV_F16, 256>(a, blocks, ru, rows_hi, prefix, st);
  return a.D == 128 ? launch_md<BG_KV_Q8, 128>(a, blocks, ru, rows_hi, prefix, st)
                    : launch_md<BG_KV_Q8, 256>(a, blocks, ru, rows_hi, prefix, st);
}

int poll_device_error_paged_decode() {
  int v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return BG_ELAUNCH;
  if (v) cudaMemcpyToSymbol(g_device_error, &z, sizeof(int));
  return v;
}

}  // namespace bg
