// paged.h -- the paged INT8 KV cache as the kernels see it: pages of
// `page` tokens in a pool, a table of page numbers per sequence, and a batch
// of new tokens packed sequence after sequence.
#pragma once

#include "common.h"

namespace sparkq {

// The batch's metadata lives on the device and is never read by the host, so
// the kernels bound everything that they take from it: a page number outside
// the pool stands for no page, starts outside the packed rows are clamped,
// and a length reaches no further than its table row.
struct PagedBatch {
  const int32_t* table;    // [B, width], rows table_stride apart
  const int32_t* starts;   // [B + 1]
  const int32_t* lengths;  // [B], the new tokens included
  int64_t table_stride;
  int B, T;          // sequences, packed rows of new tokens
  int width, pages;  // pages per table row, pages in the pool
  int page_log2;
};

// One of the pool's two code tensors with its scales: strides of codes in
// bytes, of scales in elements.
struct PagedSide {
  uint8_t* codes;
  uint16_t* scales;
  int64_t c_page, c_head, c_tok;
  int64_t s_page, s_head, s_tok;
};

constexpr int64_t kMaxGrid = 0x7FFFFFFF / 256;  // workgroups of 256 threads: fewer than 2^31 threads

struct SeqRows {
  int first, count;  // packed rows [first, first + count)
  int length;        // tokens in the cache, the new ones included
};

__device__ __forceinline__ SeqRows seq_rows(const PagedBatch& p, int b) {
  SeqRows r;
  r.first = min(max(p.starts[b], 0), p.T);
  r.count = min(max(p.starts[b + 1], r.first), p.T) - r.first;
  r.length = (int)min((int64_t)max(p.lengths[b], 0), (int64_t)p.width << p.page_log2);
  return r;
}

// Page of token `pos` of sequence b, or -1 where it has none. 0 <= pos <
// width << page_log2.
__device__ __forceinline__ int page_of(const PagedBatch& p, int b, int pos) {
  const int id = p.table[b * p.table_stride + (pos >> p.page_log2)];
  return (unsigned)id < (unsigned)p.pages ? id : -1;
}

// the sequence whose rows hold packed row t, or -1
__device__ __forceinline__ int seq_of_row(const PagedBatch& p, int t) {
  int lo = 0, hi = p.B;  // the first b with starts[b + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid + 1] > t)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo < p.B ? lo : -1;
}

// The sequence whose rows hold packed row t, or b = -1: a round trip for the ends of every
// 64 sequences' rows, and one for what is there of the one that has it (the compiler puts
// those loads behind the ballot). All lanes of a wave ask for the same row.
struct RowOf {
  int b;
  SeqRows s;
};
__device__ __forceinline__ RowOf wave_row(const PagedBatch& p, int t) {
  const int lane = threadIdx.x & 63;
  RowOf r{-1, {0, 0, 0}};
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = min(b0 + lane, p.B - 1);
    const SeqRows s = seq_rows(p, b);
    const unsigned long long past = __ballot(b0 + lane < p.B && p.starts[b + 1] > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      r = RowOf{b0 + l, {__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.count, l),
                         __builtin_amdgcn_readlane(s.length, l)}};
      break;
    }
  }
  // (the compiler does not see that a loop left on a ballot leaves scalars)
  for (int* f : {&r.b, &r.s.first, &r.s.count, &r.s.length}) *f = __builtin_amdgcn_readfirstlane(*f);
  return r;
}

// last token that row i of a sequence's new tokens sees (-1: none)
__device__ __forceinline__ int last_seen_by(const SeqRows& s, int i, int causal) {
  return causal ? min(max(s.length - s.count + i, -1), s.length - 1) : s.length - 1;
}

}  // namespace sparkq
