// extern "C" entry points of the paged-cache operators: argument checks and the choice of kernels.
#include <math.h>

#include "paged.h"

using namespace bg;

namespace {

bool d_ok(uint32_t D) { return D == 64 || D == 128 || D == 256; }

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_paged(const bg_paged_cache *kv, const bg_paged_batch *b, uint32_t KV, uint32_t D) {
  if (!kv || !b || KV == 0) return BG_EINVAL;
  if (!d_ok(D)) return BG_EUNSUPPORTED;
  if (kv->mode == BG_KV_Q8R) return BG_EUNSUPPORTED;
  if (kv->mode > BG_KV_Q8R) return BG_EINVAL;
  if (!kv->K || !kv->V || !aligned16(kv->K) || !aligned16(kv->V)) return BG_EINVAL;
  if (kv->mode == BG_KV_Q8 && (!kv->Ks || !kv->Vs || !aligned16(kv->Ks) || !aligned16(kv->Vs))) return BG_EINVAL;
  if (kv->num_pages == 0 || kv->num_pages > 0x7fffffffull || kv->page_size == 0) return BG_EINVAL;
  if (b->batch == 0 || b->tokens == 0) return BG_OK;
  if (!b->kv_len || !b->page_table || b->table_stride == 0 || b->max_q == 0) return BG_EINVAL;
  if (!b->cu_q && b->tokens != b->batch) return BG_EINVAL;
  if (b->batch > 0x7ffffffeu || b->tokens > 0x7fffffffu) return BG_EINVAL;
  if (b->prefix_len && !b->prefix_pages) return BG_EINVAL;
  if ((uint64_t)b->table_stride * kv->page_size + b->prefix_len > 0x7fffffffull) return BG_EINVAL;
  return BG_OK;
}

PagedView view(const bg_paged_cache *kv, uint32_t KV) {
  return PagedView{kv->K, kv->V, kv->Ks, kv->Vs, (uint32_t)kv->num_pages, kv->page_size, KV};
}

BatchView view(const bg_paged_batch *b) {
  return BatchView{b->cu_q, b->kv_len, b->page_table, b->prefix_pages, b->batch, b->tokens, b->table_stride,
                   b->prefix_len};
}

constexpr uint32_t kSMs = 148;
constexpr uint64_t kManyTiles = 8;

// The kernels of one call and the layout of its workspace: partial rows o [part_rows][D] f32, then ml
// [part_rows] float2, then the descriptions of what is to be joined, then (tcgen05) the blocks' run sums, the
// largest block scales of a q8 pool, the halves of f32 rows and their powers of two.
//   join        a shared prefix: every row joins its parts
//   tc_pre      the prefix's units run on tcgen05
//   tc_own      sequences of more than 16 rows run on tcgen05
//               Both where the decode kernel would walk more than kManyTiles tiles of 16 rows a block instead:
//               that kernel takes ~0.6 us a tile, a tcgen05 launch ~12 us before its first result (f16, 8
//               kv heads of 4; decode kernel and tcgen05: 26 streams behind 206 shared positions 16 and
//               23 us, 64 behind 8192 103 and 43; 4 prompts of 64 tokens after 236 positions 31 and 23).
//               What a sequence holds is bounded by its row of the page table, all that the host knows of it (4
//               prompts of 24 tokens after 60 to 120 positions: 15.0 us in a tight table, 14.0 in one for 131072).
//   decode      the decode kernel has the rest: sequences of at most 16 rows beside tc_own -- not launched
//               where tokens == batch * max_q says that there are none; were it wrong, tc_own has them
struct Plan {
  bool fast, join, tc_pre, tc_own, decode;
  uint32_t nsplit;                  // CUDA-core kernel: splits of every row
  uint32_t ru, blocks;              // decode kernel: rows of a unit, blocks
  uint32_t ru_own, ru_pre;          // tcgen05 kernels: rows of a unit
  uint32_t slot_own, slot_pre;      // first partial row of each kernel's slots (the decode kernel's: 0)
  uint32_t row_own, row_pre;        // ... of the whole units behind a prefix
  uint64_t rows, part_rows;         // tokens * H; all partial rows
  size_t desc, sums, tops, halves, bytes;  // offsets of the descriptions, run sums, scales and q's halves (0: none), size
};

Plan make_plan(const bg_paged_cache *kv, const bg_paged_batch *b, uint32_t H, uint32_t KV, uint32_t D, bool fast, bool lo) {
  Plan p = {};
  const uint32_t G = H / KV;
  const uint64_t cap = (uint64_t)b->table_stride * kv->page_size;
  p.rows = (uint64_t)b->tokens * H;
  p.join = b->prefix_len > 0;
  const UnitShape small = unit_shape(G, KV, 8, 64, 4, 0, 0, false);  // the most units and tiles that any kernel may count
  p.fast = fast && paged_decode_supported((int)kv->mode, D, kv->page_size) && p.rows < 0x10000000ull &&
           most_tiles(small, b->tokens, b->batch, cap, b->prefix_len) < 0xffffffffull;
  if (!p.fast) {
    p.nsplit = paged_generic_splits(b->tokens, H, KV, cap + b->prefix_len);
    p.part_rows = p.nsplit > 1 ? (uint64_t)p.nsplit * p.rows : 0;
    p.bytes = (size_t)p.part_rows * (D * 4 + 8);
    return p;
  }
  const uint64_t group = (uint64_t)b->max_q * G, all = (uint64_t)b->tokens * G;
  const bool tc = paged_tc_supported((int)kv->mode, D, G, KV, kv->page_size);
  const uint64_t own_tiles = (all + 15) / 16 * KV * ((cap + 63) / 64);
  const uint64_t pre_tiles = (all + 15) / 16 * KV * ((uint64_t)(b->prefix_len + 63) / 64);
  const uint64_t many = kManyTiles * paged_decode_blocks((int)kv->mode, D, 16);
  // f32 rows over a q8 pool of head_dim 256 have a ring of one stage: 36 rows a sequence behind 953 positions take
  // 154 us there and 137 with the decode kernel, 60 behind 13388 shared ones 74 and 104
  const uint64_t few = lo && D == 256 && kv->mode == BG_KV_Q8 ? 48 : 16;
  p.tc_own = tc && group > few && own_tiles > many;
  p.tc_pre = tc && p.join && all > few && pre_tiles > many;
  p.decode = !p.tc_own || (p.join && !p.tc_pre) || b->tokens < (uint64_t)b->batch * b->max_q;
  // rows of a unit: as many as a sequence's rows (or, behind a prefix, all rows) fill; f32 rows have a form for 4
  const uint64_t fill = p.tc_own ? 16 : p.join && !p.tc_pre ? (all > group ? all : group) : group;
  // (16 f32 rows of head_dim 256 do not fit the registers: two units of 8 read the positions twice, but sooner)
  p.ru = fill <= 4 && lo ? 4 : fill <= 8 || (lo && D == 256) ? 8 : 16;
  p.blocks = paged_decode_blocks((int)kv->mode, D, p.ru);
  p.ru_own = paged_tc_rows(D, G, lo, group);
  p.ru_pre = paged_tc_rows(D, G, lo, all);
  uint64_t at = p.decode ? 2ull * p.blocks * p.ru : 0;
  p.slot_own = (uint32_t)at;
  if (p.tc_own) at += 2ull * kSMs * p.ru_own;
  p.slot_pre = (uint32_t)at;
  if (p.tc_pre) at += 2ull * kSMs * p.ru_pre;
  p.row_own = (uint32_t)at;
  p.row_pre = (uint32_t)(at + p.rows);
  if (p.join) at += 2 * p.rows;
  p.part_rows = at;
  p.desc = (size_t)p.part_rows * (D * 4 + 8);
  p.bytes = p.desc + (p.join ? 2 * p.rows * sizeof(RowPieces) : (p.blocks + kSMs) * sizeof(CutUnit));
  if (p.tc_own || p.tc_pre) {
    p.sums = (p.bytes + 127) / 128 * 128;  // of one launch at a time: they follow one another
    p.bytes = p.sums + kSMs * kRunSums * sizeof(float);
    if (kv->mode == BG_KV_Q8) {
      p.tops = p.bytes;
      p.bytes += ((uint64_t)b->batch + 1) * KV * kTopRow * 4;
      p.bytes = (p.bytes + 127) / 128 * 128;
    }
    if (lo) {
      p.halves = p.bytes;
      p.bytes += p.rows * (D * 4 + 4);
    }
  }
  return p;
}

// Enough for either kind of kernel and either type of rows, so that what a caller needs does not change with
// bg_force_generic or with the types of one call.
size_t workspace_bytes_for(const bg_paged_cache *kv, const bg_paged_batch *b, uint32_t H, uint32_t KV, uint32_t D) {
  size_t n = 0;
  for (int i = 0; i < 3; ++i) {
    const size_t m = make_plan(kv, b, H, KV, D, i < 2, i == 1).bytes;
    n = m > n ? m : n;
  }
  return n;
}

}  // namespace

namespace bg {
int poll_device_error_paged() {
  // each one is read and cleared: several kernels of one call may have seen the same fault
  const int e[] = {poll_device_error_paged_append(), poll_device_error_paged_generic(), poll_device_error_paged_decode(),
                   poll_device_error_paged_tc()};
  for (int i = 0; i < 4; ++i)
    if (e[i]) return e[i];
  return 0;
}
}  // namespace bg

extern "C" {

int bg_paged_append(const bg_paged_cache *kv, const bg_paged_batch *batch, uint32_t H, uint32_t KV, uint32_t D,
                    const bg_rows *q, const bg_rows *k, const bg_rows *v, uint32_t src_dtype, const float *q_gamma,
                    const float *k_gamma, float eps, const float *cosT, const float *sinT, uint32_t rot,
                    uint32_t table_rows, void *q_out, uint32_t q_out_dtype, bg_stream_t stream) {
  if (int rc = check_paged(kv, batch, KV, D)) return rc;
  if (!k || !v || !k->x || !v->x || src_dtype > BG_DT_F16 || q_out_dtype > BG_DT_F16) return BG_EINVAL;
  if (q && (!q->x || !q_out || H == 0 || !aligned16(q_out))) return BG_EINVAL;
  if ((cosT == nullptr) != (sinT == nullptr)) return BG_EINVAL;
  if (cosT && (rot == 0 || rot % 2 || rot > D || !aligned16(cosT) || !aligned16(sinT))) return BG_EINVAL;
  if (batch->batch == 0 || batch->tokens == 0) return BG_OK;
  PagedAppendArgs a;
  a.kv = view(kv, KV);
  a.bv = view(batch);
  a.mode = (int)kv->mode;
  a.src_f16 = src_dtype == BG_DT_F16;
  a.out_f16 = q_out_dtype == BG_DT_F16;
  a.H = q ? H : 0;
  a.D = D;
  a.rot = cosT ? rot : 0;
  a.table_rows = table_rows;
  a.q = q ? q->x : nullptr;
  a.q_ts = q ? q->token_stride : 0;
  a.q_hs = q ? q->head_stride : 0;
  a.k = k->x;
  a.k_ts = k->token_stride;
  a.k_hs = k->head_stride;
  a.v = v->x;
  a.v_ts = v->token_stride;
  a.v_hs = v->head_stride;
  a.q_gamma = q_gamma;
  a.k_gamma = k_gamma;
  a.cosT = cosT;
  a.sinT = sinT;
  a.eps = eps;
  a.q_out = q_out;
  return launch_paged_append(a, (cudaStream_t)stream);
}

size_t bg_paged_attention_workspace_size(const bg_paged_cache *kv, const bg_paged_batch *batch, uint32_t H, uint32_t KV,
                                         uint32_t D) {
  if (check_paged(kv, batch, KV, D) || H == 0 || H % KV || batch->batch == 0 || batch->tokens == 0) return 0;
  return workspace_bytes_for(kv, batch, H, KV, D);
}

int bg_paged_attention(const bg_paged_cache *kv, const bg_paged_batch *batch, uint32_t H, uint32_t KV, uint32_t D,
                       const void *q, uint32_t q_dtype, float scale, const float *gate, void *out, uint32_t out_dtype,
                       void *workspace, size_t workspace_bytes, bg_stream_t stream) {
  if (int rc = check_paged(kv, batch, KV, D)) return rc;
  if (H == 0 || H % KV || q_dtype > BG_DT_F16 || out_dtype > BG_DT_F16) return BG_EINVAL;
  if (!(scale >= 0.f && scale < INFINITY)) return BG_EINVAL;
  if (batch->batch == 0 || batch->tokens == 0) return BG_OK;
  if (!q || !out || !aligned16(q) || !aligned16(out) || !aligned16(gate) || !aligned16(workspace)) return BG_EINVAL;
  const Plan plan = make_plan(kv, batch, H, KV, D, !generic_forced(), !(q_dtype == BG_DT_F16 && out_dtype == BG_DT_F16));
  const size_t need = workspace_bytes_for(kv, batch, H, KV, D);
  if (need && (!workspace || workspace_bytes < need)) return BG_ENOMEM;
  cudaStream_t st = (cudaStream_t)stream;
  PagedAttnArgs a = {};
  a.kv = view(kv, KV);
  a.bv = view(batch);
  a.mode = (int)kv->mode;
  a.q_f16 = q_dtype == BG_DT_F16;
  a.out_f16 = out_dtype == BG_DT_F16;
  a.H = H;
  a.G = H / KV;
  a.D = D;
  a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf((float)D)) * kLog2e;
  a.q = q;
  a.gate = gate;
  a.out = out;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + plan.part_rows * D);
  a.part_rows = plan.part_rows;
  a.min_tiles = 1;
  if (!plan.fast) return launch_paged_generic(a, plan.nsplit, st);
  unsigned char *desc = static_cast<unsigned char *>(workspace) + plan.desc;
  CutUnit *cuts = reinterpret_cast<CutUnit *>(desc);
  if (plan.sums) a.run_sums = reinterpret_cast<float4 *>(static_cast<unsigned char *>(workspace) + plan.sums);
  if (plan.tops) a.tops = reinterpret_cast<uint32_t *>(static_cast<unsigned char *>(workspace) + plan.tops);
  if (plan.halves) {
    a.q_halves = static_cast<unsigned char *>(workspace) + plan.halves;
    a.q_pow2 = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + plan.halves + plan.rows * D * 4);
  }
  if (plan.join) {
    a.own_pieces = reinterpret_cast<RowPieces *>(desc);
    a.pre_pieces = a.own_pieces + plan.rows;
    a.own_row0 = plan.row_own;
    a.pre_row0 = plan.row_pre;
  }
  auto with = [&](uint32_t slot0, CutUnit *c) {
    PagedAttnArgs x = a;
    x.slot0 = slot0;
    x.cuts = plan.join ? nullptr : c;
    return x;
  };
  const PagedAttnArgs dec = with(0, cuts), own = with(plan.slot_own, cuts + plan.blocks), pre = with(plan.slot_pre, nullptr);
  if (plan.halves)
    if (int rc = launch_paged_split_rows(a, st)) return rc;
  const uint32_t rows_lo = plan.decode ? 16 : 0;  // sequences of more rows are the tcgen05 kernel's
  if (plan.tops)
    if (int rc = launch_paged_top_scales(a, rows_lo, plan.tc_own, plan.tc_pre, st)) return rc;
  if (plan.tc_pre)
    if (int rc = launch_paged_tc(pre, kSMs, plan.ru_pre, 0, true, st)) return rc;
  if (plan.tc_own)
    if (int rc = launch_paged_tc(own, kSMs, plan.ru_own, rows_lo, false, st)) return rc;
  if (plan.decode)
    if (int rc = launch_paged_decode(dec, plan.blocks, plan.ru, plan.tc_own ? 16 : 0xffffffffu, plan.join && !plan.tc_pre, st))
      return rc;
  if (plan.join) return launch_paged_join_rows(a, st);
  if (plan.tc_own)
    if (int rc = launch_paged_join_cuts(own, kSMs, plan.ru_own, st)) return rc;
  if (plan.decode)
    if (int rc = launch_paged_join_cuts(dec, plan.blocks, plan.ru, st)) return rc;
  return BG_OK;
}

}  // extern "C"
