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

}  // namespace sparkq
