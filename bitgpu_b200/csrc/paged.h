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
// are clamped to [0, T], lengths to what the sequence's page-table row can hold.
struct SeqRange {
  uint32_t begin, n;  // first token, number of tokens
  int32_t len;        // own positions, the new tokens among them
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
  r.len = min(max(__ldg(bv.kv_len + b), 0), (int32_t)(bv.table_stride * page_size));
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

struct PagedAttnArgs {
  PagedView kv;
  BatchView bv;
  int mode, q_f16, out_f16;
  uint32_t H, G, D, max_q;
  float sl2;  // softmax scale * log2(e)
  const void *q;
  const float *gate;
  void *out;
  // partial rows: o [n][D] unnormalised, ml [n] (running max in log2 units, sum); n = part_rows
  float *part_o;
  float2 *part_ml;
  uint64_t part_rows;
};

int launch_paged_append(const PagedAppendArgs &a, cudaStream_t st);

// CUDA-core kernel for every mode, head size and page size.
uint32_t paged_generic_splits(uint32_t T, uint32_t H, uint32_t KV, uint64_t max_positions);
int launch_paged_generic(const PagedAttnArgs &a, uint32_t nsplit, cudaStream_t st);

int poll_device_error_paged();  // of all paged operators
int poll_device_error_paged_append();
int poll_device_error_paged_generic();

}  // namespace bg
