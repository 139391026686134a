// Shared pieces of the paged-cache operators (append, ragged attention, shared prefix): the device
// views of a page pool and of a ragged batch, the sequence lookup and the internal launch interface.
//
// Rows.  Token t of the batch has H query rows; the G = H / KV rows that read one kv head are numbered
// R = t*G + g, so the rows of one sequence (and of the whole batch) are contiguous in R and any run
// [R0, R0 + n) of them can share the K/V tiles of one kv head.
#pragma once
#include "common.cuh"

namespace bg {

struct PagedView {
  void *K, *V;
  float *Ks, *Vs;
  uint32_t num_pages, page_size, KV;
};

struct BatchView {
  const int32_t *cu_q, *kv_len, *table, *prefix_pages;
  uint32_t B, T, table_stride, prefix_len;
};

// Tokens [begin, end) of sequence b.  Device-side values are never trusted to be in range: offsets
// are clamped to [0, T], lengths to what the sequence's page-table row can hold -- but a token's position follows
// from the length as it was given, as in the append.
struct SeqRange {
  uint32_t begin, n;  // first token, number of tokens
  int32_t len;        // own positions, the new tokens among them
  int32_t held;       // those that the page table has room for
  // Own positions that token i of the sequence attends.
  __device__ __forceinline__ int32_t attended(uint32_t i) const {
    return min(held, max(0, len - (int32_t)n + (int32_t)i + 1));
  }
  // The page table has no room for the length: reported as BG_EINVAL.
  __device__ __forceinline__ bool too_long() const { return n > 0 && held < len; }
};

__device__ __forceinline__ SeqRange seq_range(const BatchView &bv, uint32_t b, uint32_t page_size) {
  SeqRange r;
  if (bv.cu_q) {
    const int32_t a = __ldg(bv.cu_q + b), e = __ldg(bv.cu_q + b + 1);
    const uint32_t ua = (uint32_t)min(max(a, 0), (int32_t)bv.T), ue = (uint32_t)min(max(e, 0), (int32_t)bv.T);
    r.begin = ua;
    r.n = ue > ua ? ue - ua : 0;
  } else {
    r.begin = b;
    r.n = 1;
  }
  r.len = max(__ldg(bv.kv_len + b), 0);
  r.held = min(r.len, (int32_t)(bv.table_stride * page_size));
  return r;
}

// Sequence of token t by a 32-way search over cu_q (whole warp; the offsets do not decrease), or -1
// for a token behind the last sequence.
__device__ __forceinline__ int32_t find_seq_warp(const BatchView &bv, uint32_t t, uint32_t lane) {
  if (!bv.cu_q) return (int32_t)t;
  uint32_t lo = 0, n = bv.B + 1;
  for (;;) {
    const uint32_t step = (n + 31) / 32, i = lo + lane * step;
    const bool le = i < lo + n && __ldg(bv.cu_q + i) <= (int32_t)t;
    const uint32_t cnt = __popc(__ballot_sync(0xffffffffu, le));
    if (cnt == 0) return -1;
    lo += (cnt - 1) * step;
    if (step == 1) break;
    n = min(step, bv.B + 1 - lo);
  }
  return lo < bv.B ? (int32_t)lo : -1;
}

// Pool row (before the kv-head factor) of position j of a page list, or -1 when its page id lies
// outside the pool.
__device__ __forceinline__ int64_t paged_row(const PagedView &kv, const int32_t *pages, uint32_t j) {
  const uint32_t pg = (uint32_t)__ldg(pages + j / kv.page_size);
  return pg < kv.num_pages ? (int64_t)pg * kv.page_size + j % kv.page_size : -1;
}

// ---- the work of a ragged batch as one line of K/V tiles --------------------------------------------
// A unit is up to RU rows R of one kv head against the positions they attend: of the shared prefix (rows
// of the whole batch) or of one sequence's own positions.  Units lie one behind the other, each as many
// tiles of KT positions as its last token attends (at least one, so that rows that attend nothing are
// written too), and block c of the grid takes tiles [c*per, (c+1)*per).  So every block has the same
// work whatever the lengths, decided on the device from the lengths of this very call.  A unit that a
// border cuts leaves partial rows: the piece that starts in block c in slot 2c+1, the piece that block
// c goes on with in slot 2c.  Only a block's first and last piece can be cut, so two slots suffice.
// A unit also costs its queries, its first scores and its epilogue: `lead` tiles' time, counted as empty
// tiles in front of its own, so that blocks with many short units get fewer tiles.
struct UnitShape {
  uint32_t G, KV, RU, KT;
  uint32_t tokens;  // RU / G where that is whole, else 0
  uint32_t shift;   // log2(KT)
  uint32_t lead;
  uint32_t rows_lo, rows_hi;  // own sequences of rows_lo < n*G <= rows_hi rows (others are another kernel's)
  int prefix;                 // whether the prefix's units are this kernel's
};

struct TileSpan {
  uint32_t total, per, t0, t1;  // all tiles, tiles of a block, this block's [t0, t1)
  uint32_t pre;                 // tiles of the prefix's units, which come first
  uint32_t b0;                  // sequence that tile max(t0, pre) belongs to
  uint32_t off0;                // its index among that sequence's tiles
};

inline UnitShape unit_shape(uint32_t G, uint32_t KV, uint32_t RU, uint32_t KT, uint32_t lead, uint32_t rows_lo,
                            uint32_t rows_hi, bool prefix) {
  UnitShape u{G, KV, RU, KT, RU % G ? 0 : RU / G, 0, lead, rows_lo, rows_hi, prefix};
  while ((1u << u.shift) < KT) ++u.shift;
  return u;
}

// An upper bound of all tiles of a call, from what the host knows.
inline uint64_t most_tiles(const UnitShape &u, uint64_t tokens, uint64_t batch, uint64_t capacity, uint64_t prefix) {
  const uint64_t units = tokens * u.G / u.RU + batch + 1;
  return u.KV * units * ((capacity + u.KT - 1) / u.KT + 1 + u.lead + (prefix + u.KT - 1) / u.KT);
}

// Positions that the last row of chunk ch attends (own part of a sequence), and the chunk's tiles.
__device__ __forceinline__ uint32_t chunk_tiles(const SeqRange &s, const UnitShape &u, uint32_t ch) {
  const uint32_t end = u.tokens ? min((ch + 1) * u.tokens, s.n) : (min((ch + 1) * u.RU, s.n * u.G) - 1) / u.G + 1;
  return max(1u, ((uint32_t)s.attended(end - 1) + u.KT - 1) >> u.shift);
}

// Tiles of one kv head of a sequence's own units, their leads among them (0: none of this kernel's).
__device__ __forceinline__ uint32_t seq_tiles(const SeqRange &s, const UnitShape &u) {
  const uint32_t rows = s.n * u.G;
  if (rows <= u.rows_lo || rows > u.rows_hi) return 0;
  uint32_t n = 0;
  for (uint32_t ch = 0; ch * u.RU < rows; ++ch) n += u.lead + chunk_tiles(s, u, ch);
  return n;
}

// Rows R that the prefix's units cover: every row of a token of some sequence.
__device__ __forceinline__ uint32_t batch_rows(const BatchView &bv, uint32_t G) {
  const int32_t t = bv.cu_q ? __ldg(bv.cu_q + bv.B) : (int32_t)bv.B;
  return (uint32_t)min(max(t, 0), (int32_t)bv.T) * G;
}

// All NTHR threads of the block: the block's span; `bad` is set where a length exceeds its table.  `sh`: NTHR / 32 + 2 words of shared memory.  Tile
// numbers have 32 bits: most_tiles() of the call's bounds says whether that is enough.
template <int NTHR>
__device__ __forceinline__ TileSpan block_span(const BatchView &bv, const UnitShape &u, uint32_t page_size,
                                               uint32_t min_tiles, uint32_t *sh, int *bad) {
  constexpr int NW = NTHR / 32;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t per_thread = (bv.B + NTHR - 1) / NTHR;
  const uint32_t lo = min(bv.B, tid * per_thread), hi = min(bv.B, lo + per_thread);
  uint32_t mine = 0;
  uint32_t first = 0;
  for (uint32_t b = lo; b < hi; ++b) {
    const SeqRange sr = seq_range(bv, b, page_size);
    if (sr.too_long() && blockIdx.x == 0) atomicExch(bad, BG_EINVAL);
    const uint32_t n = u.KV * seq_tiles(sr, u);
    if (b == lo) first = n;
    mine += n;
  }
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh[warp] = incl;
  if (tid == 0) sh[NW] = 0;
  __syncthreads();
  uint32_t before = incl - mine, own = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < (int)warp) before += sh[w];
    own += sh[w];
  }
  TileSpan s;
  s.pre = 0;
  if (u.prefix && bv.prefix_len) {
    const uint32_t nch = (batch_rows(bv, u.G) + u.RU - 1) / u.RU;
    s.pre = u.KV * nch * (u.lead + ((bv.prefix_len + u.KT - 1) >> u.shift));
  }
  s.total = s.pre + own;
  const uint32_t even = s.total / gridDim.x + (s.total % gridDim.x != 0);
  s.per = even > min_tiles ? even : min_tiles;
  s.t0 = (uint32_t)min((uint64_t)s.total, (uint64_t)s.per * blockIdx.x);
  s.t1 = s.t0 + min(s.per, s.total - s.t0);
  const uint32_t want = s.t0 > s.pre ? s.t0 - s.pre : 0;  // among the own tiles
  if (mine && want >= before && want < before + mine) {
    uint32_t x = want - before;
    uint32_t b = lo, n = first;
    while (x >= n) {
      x -= n;
      ++b;
      n = u.KV * seq_tiles(seq_range(bv, b, page_size), u);
    }
    sh[NW] = b;
    sh[NW + 1] = x;
  }
  __syncthreads();
  s.b0 = sh[NW];
  s.off0 = sh[NW + 1];
  return s;
}

// One block's pieces of units, in order (uniform over the calling threads).
struct Piece {
  uint32_t R0, rows, kvh;   // rows [R0, R0 + rows) of kv head kvh
  uint32_t tile0, ntiles;   // tiles of the unit
  uint32_t len;             // positions of the list (the prefix's or the sequence's)
  uint32_t list;            // the sequence, or B for the prefix
  int32_t lim_base;         // token t attends positions <= lim_base + t
  const int32_t *pages;
  uint32_t npieces;         // pieces of the unit
  bool own, starts;         // own part (or prefix); whether the unit starts in this block
};

struct PieceWalk {
  uint32_t cur, t1, per, pre;  // next tile, end of the span
  uint32_t b, kvh, ch, in;           // own part: sequence, kv head, chunk, tiles (and lead) before `cur` in the unit
  SeqRange sr;

  __device__ __forceinline__ void seek(const BatchView &bv, const UnitShape &u, uint32_t page_size, uint32_t off) {
    // position inside sequence b: (kvh, chunk, tile)
    sr = seq_range(bv, b, page_size);
    const uint32_t s = seq_tiles(sr, u);
    kvh = off / s;
    uint32_t x = off % s;
    ch = 0;
    for (;;) {
      const uint32_t n = u.lead + chunk_tiles(sr, u, ch);
      if (x < n) break;
      x -= n;
      ++ch;
    }
    in = x;
  }

  __device__ __forceinline__ void init(const TileSpan &s, const BatchView &bv, const UnitShape &u, uint32_t page_size) {
    cur = s.t0;
    t1 = s.t1;
    per = s.per;
    pre = s.pre;
    b = s.b0;
    kvh = ch = in = 0;
    sr = SeqRange{0, 0, 0, 0};
    if (cur < t1 && t1 > pre) seek(bv, u, page_size, s.off0);
  }

  __device__ __forceinline__ bool next(Piece &p, const BatchView &bv, const UnitShape &u, uint32_t page_size) {
    if (cur >= t1) return false;
    uint32_t at, n, done;  // where the unit's first tile lies, its tiles, those before this block's
    if (cur < pre) {
      const uint32_t rows = batch_rows(bv, u.G), nch = (rows + u.RU - 1) / u.RU;
      n = (bv.prefix_len + u.KT - 1) >> u.shift;
      const uint32_t unit = cur / (n + u.lead);
      at = unit * (n + u.lead) + u.lead;
      p.kvh = unit / nch;
      p.R0 = unit % nch * u.RU;
      p.rows = min(u.RU, rows - p.R0);
      p.len = bv.prefix_len;
      p.lim_base = 0x40000000;
      p.pages = bv.prefix_pages;
      p.list = bv.B;
      p.own = false;
      if (cur < at) cur = min(at, t1);
      if (cur >= t1) return false;  // only (some of) the lead is this block's
      done = cur - at;
      p.ntiles = min(n - done, t1 - cur);
    } else {
      const uint32_t rows = sr.n * u.G;
      n = chunk_tiles(sr, u, ch);
      if (in < u.lead) {
        const uint32_t skip = min(u.lead - in, t1 - cur);
        cur += skip;
        in += skip;
        if (cur >= t1) return false;
      }
      done = in - u.lead;
      at = cur - done;
      p.kvh = kvh;
      p.R0 = sr.begin * u.G + ch * u.RU;
      p.rows = min(u.RU, rows - ch * u.RU);
      p.len = (uint32_t)sr.held;
      p.lim_base = sr.len - (int32_t)sr.n - (int32_t)sr.begin;
      p.pages = bv.table + (uint64_t)b * bv.table_stride;
      p.list = b;
      p.own = true;
      p.ntiles = min(n - done, t1 - cur);
      in += p.ntiles;
      if (done + p.ntiles == n) {  // on to the next unit: chunk, kv head, sequence
        in = 0;
        if (++ch * u.RU >= rows) {
          ch = 0;
          if (++kvh == u.KV) {
            kvh = 0;
            if (cur + p.ntiles < t1) {
              do {
                ++b;
                sr = seq_range(bv, b, page_size);
              } while (seq_tiles(sr, u) == 0);
            }
          }
        }
      }
    }
    p.tile0 = done;
    p.npieces = (at + n - 1) / per - at / per + 1;
    p.starts = done == 0;
    cur += p.ntiles;
    return true;
  }
};

// Where a unit's rows wait to be joined.  Without a prefix only cut units leave any: one CutUnit per
// block (npieces 0: none).  With a prefix every row joins two lists of pieces: one RowPieces per (kv
// head, R) and part; piece 0 is partial row idx0, piece k row idx0 + (2k - 1) * step.
struct CutUnit {
  uint32_t R0, rows, kvh, npieces;
};
struct RowPieces {
  uint32_t idx0, npieces, step, pad;
};
__host__ __device__ __forceinline__ uint32_t piece_index(uint32_t idx0, uint32_t step, uint32_t k) {
  return k ? idx0 + (2 * k - 1) * step : idx0;
}

// Positions of a page box: the largest number that divides pages and tiles alike, so that a box that
// starts on a multiple of it never leaves its page.
inline uint32_t page_box(uint32_t page_size, uint32_t tile) {
  uint32_t x = page_size, y = tile;
  while (y) {
    const uint32_t z = x % y;
    x = y;
    y = z;
  }
  return x;
}

// Raise a kernel's dynamic shared memory limit once per device (`done`: one bit per device).
template <typename K>
inline bool allow_smem(K kern, int bytes, unsigned long long &done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  return true;
}

struct PagedAppendArgs {
  PagedView kv;
  BatchView bv;
  int mode, src_f16, out_f16;
  uint32_t H, D, rot, table_rows;
  const void *q, *k, *v;
  uint64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides in elements
  const float *q_gamma, *k_gamma, *cosT, *sinT;
  float eps;
  void *q_out;  // [T][H][D]
};

constexpr uint32_t kTopRow = 16;  // a row of largest scales: V's blocks, K's
constexpr size_t kRunSums = 2 * 128 * 128;  // two streams of 128 columns, or one of 256, for 128 rows

struct PagedAttnArgs {
  PagedView kv;
  BatchView bv;
  int mode, q_f16, out_f16;
  uint32_t H, G, D;
  float sl2;  // softmax scale * log2(e)
  const void *q;
  // tcgen05 kernels, rows that are not f16 in and out: q as two f16 halves [2][T][H][D] and each row's power of two
  void *q_halves;
  float *q_pow2;  // [T][H]
  const float *gate;
  void *out;
  // partial rows: o [n][D] unnormalised, ml [n] (running max in log2 units, sum); n = part_rows
  float *part_o;
  float2 *part_ml;
  uint64_t part_rows;
  uint32_t *tops;    // tcgen05 kernels, q8 pool: [list: sequences, prefix][kv head][kTopRow]
  float4 *run_sums;  // tcgen05 kernels: kRunSums values of each block
  // pieces to join: of the own parts (RowPieces or, without a prefix, CutUnit) and of the prefix
  CutUnit *cuts;
  RowPieces *own_pieces, *pre_pieces;
  uint32_t slot0, own_row0, pre_row0;  // first partial row of this kernel's slots, of whole own / prefix units
  uint32_t min_tiles;
};

int launch_paged_append(const PagedAppendArgs &a, cudaStream_t st);

// CUDA-core kernel for every mode, head size and page size.
uint32_t paged_generic_splits(uint32_t T, uint32_t H, uint32_t KV, uint64_t max_positions);
int launch_paged_generic(const PagedAttnArgs &a, uint32_t nsplit, cudaStream_t st);

// Tensor-core decode kernel (mma.sync): few rows a sequence, f16 and q8 pools.
bool paged_decode_supported(int mode, uint32_t D, uint32_t page_size);

uint32_t paged_decode_blocks(int mode, uint32_t D, uint32_t ru);  // blocks that fill the GPU
int launch_paged_decode(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_hi, bool prefix, cudaStream_t st);
// tcgen05 kernel: many rows a sequence (own part), or the rows of the batch against the shared prefix.
bool paged_tc_supported(int mode, uint32_t D, uint32_t G, uint32_t KV, uint32_t page_size);
int launch_paged_top_scales(const PagedAttnArgs &a, uint32_t rows_lo, bool own, bool prefix, cudaStream_t st);
uint32_t paged_tc_rows(uint32_t D, uint32_t G, bool lo, uint64_t rows);
int launch_paged_split_rows(const PagedAttnArgs &a, cudaStream_t st);
int launch_paged_tc(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, uint32_t rows_lo, bool prefix, cudaStream_t st);
// Join the cut units of `blocks` blocks of ru rows (no prefix), or every row's pieces (prefix).
int launch_paged_join_cuts(const PagedAttnArgs &a, uint32_t blocks, uint32_t ru, cudaStream_t st);
int launch_paged_join_rows(const PagedAttnArgs &a, cudaStream_t st);

int poll_device_error_paged_decode();
int poll_device_error_paged_tc();
int poll_device_error_paged();  // of all paged operators
bool generic_forced();  // bg_force_generic
int poll_device_error_paged_append();
int poll_device_error_paged_generic();

}  // namespace bg
