// paged.hip -- what keeps a paged INT8 KV cache: the quantized append of new
// tokens, and forking and compacting of its pages (gfx950).
//
// A cache is two code tensors [P, Hkv, page, D] (symmetric s8) with one fp16
// scale per (page, KV head, token). Sequence b's token t lies in page
// table[b, t / page], slot t % page.
#include <algorithm>

#include "paged.h"

namespace sparkq {
namespace {

// ---------------------------------------------------------------------------
// quantize-on-append
// ---------------------------------------------------------------------------
// Row t of the packed new tokens is token length - count + (t - first) of the
// sequence that it falls to. The formula is kv_append's: scale = fp16(amax /
// 127), 1 where that is zero, code = clamp(rint(x / scale), -127, 127).
struct PagedAppendArgs {
  PagedBatch p;
  const void *k, *v;
  int64_t k_tok, k_head, v_tok, v_head;  // input strides (elements)
  PagedSide ks, vs;
  int H, D, x_dtype;
};

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

// v / s for rounding to a whole number, with inv = 1 / s to a unit of fp32 or so:
// the quotient's error (2^-22) after one correction is far below what matters.
// A quotient of a 16-bit v (11 bits) and an fp16 s that is not half-way between
// two whole numbers of 7 bits lies at least 2^-19 of itself from there, and one
// that is there comes out exactly: q + (v - q s) inv differs from it by the square
// of q's error, and rounds to it. A third of the division's instructions: 3501
// tokens of 4 heads of 256 14.4 -> 12.8 us.
__device__ __forceinline__ float near_quotient(float v, float s, float inv) {
  const float q = v * inv;
  return fmaf(fmaf(-q, s, v), inv, q);
}

// D / 8 lanes a row, 8 values (one or two 16-byte loads) and 8 codes (one store)
// a lane, U rows in flight. A workgroup's tokens are placed by a thread each while
// the rows' loads are under way; a decode step, where row t is sequence t's, finds
// its place at once. A chain of five loads and a store, so bound by latency: one
// row a lane where the rows fill the chip no more than once over, else two (3501
// tokens of 4 heads of 256, 21 MB: 11.1 us, 1.9 TB/s; one row 11.9, four 12.0).
template <int LPR, int U>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
  constexpr int RPP = 256 / LPR;
  __shared__ int s_page[RPP * U / 2 + 2], s_slot[RPP * U / 2 + 2];
  const int l = threadIdx.x % LPR;
  // rows are counted in 32 bits, unsigned: T * H is less than 2^31
  const uint32_t heads = 2 * (uint32_t)a.H, total = (uint32_t)a.p.T * heads, row0 = blockIdx.x * (RPP * U);
  const int t0 = (int)(row0 / heads);
  const int t1 = (int)((min(total - row0, (uint32_t)(RPP * U)) - 1 + row0) / heads);  // the last token
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t row = row0 + min(total - row0 - 1, u * RPP + threadIdx.x / LPR);
    const int t = (int)(row / heads), hv = (int)(row - t * heads);
    const bool isv = hv >= a.H;
    const int h = isv ? hv - a.H : hv;
    const int64_t x0 = (isv ? t * a.v_tok + h * a.v_head : t * a.k_tok + h * a.k_head) + 8 * l;
    const void* x = isv ? a.v : a.k;
    if (a.x_dtype == SPARKQ_F32) {
      const f32x4_t* p = reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(x) + x0);
      const f32x4_t lo = p[0], hi = p[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[u][i] = lo[i];
        v[u][4 + i] = hi[i];
      }
    } else {
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(x) + x0);
      const bool bf = a.x_dtype == SPARKQ_BF16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[u][2 * i] = bf ? lo16<BF16>(w[i]) : lo16<F16>(w[i]);
        v[u][2 * i + 1] = bf ? hi16<BF16>(w[i]) : hi16<F16>(w[i]);
      }
    }
  }
  if ((int)threadIdx.x <= t1 - t0) {
    const int t = t0 + threadIdx.x;
    const bool own = t < a.p.B && a.p.starts[t] == t && a.p.starts[t + 1] == t + 1;
    const int b = own ? t : seq_of_row(a.p, t);
    int id = -1, slot = 0;
    if (b >= 0) {
      const SeqRows s = seq_rows(a.p, b);
      const int pos = s.length - s.count + (t - s.first);
      if (t >= s.first && t < s.first + s.count && pos >= 0) id = page_of(a.p, b, pos);
      slot = pos & ((1 << a.p.page_log2) - 1);
    }
    s_page[threadIdx.x] = id;
    s_slot[threadIdx.x] = slot;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t rel = u * RPP + threadIdx.x / LPR, row = row0 + min(total - row0 - 1, rel);
    const bool live = rel < total - row0;
    const int t = (int)(row / heads), hv = (int)(row - t * heads);
    const bool isv = hv >= a.H;
    const int h = isv ? hv - a.H : hv;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[u][i]));
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    uint16_t s16 = f32_to_f16(amax / 127.0f);
    if (f16_to_f32(s16) == 0.0f) s16 = 0x3C00u;
    const float sc = f16_to_f32(s16), inv = __builtin_amdgcn_rcpf(sc);
    const bool divide = a.x_dtype == SPARKQ_F32 || sc > 65504.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = __builtin_rintf(divide ? v[u][i] / sc : near_quotient(v[u][i], sc, inv));
      w[i / 4] |= ((uint32_t)(int)fminf(fmaxf(q, -127.0f), 127.0f) & 255u) << (8 * (i % 4));
    }
    const int64_t id = s_page[t - t0], slot = s_slot[t - t0];
    if (!live || id < 0) continue;
    const PagedSide& side = isv ? a.vs : a.ks;
    if (l == 0) side.scales[id * side.s_page + h * side.s_head + slot * side.s_tok] = s16;
    *reinterpret_cast<uint2*>(side.codes + id * side.c_page + h * side.c_head + slot * side.c_tok + 8 * l) =
        make_uint2(w[0], w[1]);
  }
}

template <int LPR>
void launch_append(const PagedAppendArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.p.T * a.H * 2, groups = cdiv(rows, 256 / LPR);
  if (groups <= 8 * device_cus())
    hipLaunchKernelGGL((paged_append_kernel<LPR, 1>), dim3((unsigned)groups), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<LPR, 2>), dim3((unsigned)cdiv(groups, 2)), dim3(256), 0, st, a);
}

// ---------------------------------------------------------------------------
// pages: who holds them, which are free, and moving them
// ---------------------------------------------------------------------------
// Everything that decides (who holds a page, who gets which free one) is done
// by one workgroup, so that free pages are dealt in order with no host and no
// second pass; the tables and the pages themselves are written by a second
// launch over the whole chip. Counts are integer atomics, so their order does
// not matter.
constexpr int kPlanThreads = 1024;

// Workspace, in ints: head, then arrays of P (held, first, list) and of rows
// (base, src, dst). kOverfull is the caller's to read.
enum { kPairs = 0, kOverfull = 1, kFree = 2, kHead = 16 };
struct PageScratch {
  int* head;
  int *held, *first, *list;
  int *base, *src, *dst;
};

__host__ __device__ inline PageScratch page_scratch(int* ws, int64_t pages, int64_t rows) {
  PageScratch s;
  s.head = ws;
  s.held = ws + kHead;
  s.first = s.held + pages;
  s.list = s.first + pages;
  s.base = s.list + pages;
  s.src = s.base + rows;
  s.dst = s.src + rows;
  return s;
}

// One of the cache's four tensors, by its bytes: layers and pages of it.
struct PageBuf {
  uint8_t* p;
  int64_t layer, page;  // strides (bytes)
};

struct PageArgs {
  const int32_t* table;    // [B, width] before
  const int32_t* lengths;  // [B]
  const int32_t* parents;  // [rows] or null: row i continues sequence i
  const int32_t* fresh;    // [rows] new tokens, or null: none
  int32_t* out_table;      // [rows, width]
  int32_t* out_lengths;    // [rows] (fork)
  int32_t* out_count;      // [1] pages short (fork), pages in use (compact)
  int64_t table_stride;
  int B, rows, width, pages, page_log2;
  PageScratch s;
  PageBuf buf[4];       // codes, codes, scales, scales
  int vec_codes, vec_scales;  // 16-byte pieces of a page in one layer
  int layers, table_blocks;
};

struct RowPlan {
  int src;            // sequence that the row continues, or -1
  int before, after;  // tokens before and after the step
  int held, need;     // pages before and after
  bool over;          // more tokens than its pages have room for
};

__device__ __forceinline__ RowPlan row_plan(const PageArgs& a, int i) {
  RowPlan r;
  r.src = a.parents ? a.parents[i] : i;
  if ((unsigned)r.src >= (unsigned)a.B) r.src = -1;
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int64_t was = r.src < 0 ? 0 : max(a.lengths[r.src], 0), n = min(was, room);
  const int64_t more = a.fresh ? max(a.fresh[i], 0) : 0, m = min(n + more, room);
  r.before = (int)n;
  r.after = (int)m;
  const int64_t up = (1 << a.page_log2) - 1;
  r.held = (int)((n + up) >> a.page_log2);
  r.need = (int)((m + up) >> a.page_log2);
  r.over = was + more > room;
  return r;
}

// entry j < held of row r, or -1
__device__ __forceinline__ int held_page(const PageArgs& a, const RowPlan& r, int j) {
  const int id = a.table[r.src * a.table_stride + j];
  return (unsigned)id < (unsigned)a.pages ? id : -1;
}

// the partly filled last page that the row's new tokens go to, or -1
__device__ __forceinline__ int write_page(const PageArgs& a, const RowPlan& r) {
  if (r.after <= r.before || (r.before & ((1 << a.page_log2) - 1)) == 0) return -1;
  return held_page(a, r, r.held - 1);
}

// Counters of a plan's pages, in LDS (up to kLdsPages) or, of larger pools, in
// the workspace: there through device-scope atomics, which are coherent whatever
// the vector cache holds (a fork of 256 rows in 2048 pages 27.8 us, with counters in
// the workspace 38.0; of 1024 rows in 16384 pages 37.3 and 62.3).
constexpr int kLdsPages = 16384;
template <bool LDS>
struct Counters {
  int* p;
  __device__ void put(int i, int v) const {
    if (LDS)
      p[i] = v;
    else
      splitk_store(p + i, v);
  }
  __device__ int get(int i) const { return LDS ? p[i] : splitk_load(p + i); }
  __device__ void add(int i, int v) const { atomicAdd(p + i, v); }
  __device__ void min(int i, int v) const { atomicMin(p + i, v); }
};

template <bool LDS>
__device__ __forceinline__ void plan_sync() {
  if (!LDS) __threadfence();
  __syncthreads();
}

// exclusive prefix of v over the workgroup's threads; total in every thread
__device__ __forceinline__ int block_prefix(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last call's readers are done with s_wave
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int below = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int n = s_wave[w];
    below += w < wave ? n : 0;
    total += n;
  }
  return below + x - v;
}

// held[p] = rows' entries that name page p. Rows are planned a thread each (`mine`
// is the plan of row tid) and their entries counted by `per` lanes each, four rows'
// loads in flight.
template <bool LDS>
__device__ __forceinline__ void count_held(const PageArgs& a, const Counters<LDS>& held, const RowPlan& mine,
                                           int (&s_src)[kPlanThreads], int (&s_held)[kPlanThreads]) {
  const int tid = threadIdx.x;
  for (int p = tid; p < a.pages; p += kPlanThreads) held.put(p, 0);
  int per = 1;
  while (per < a.width && per < 64) per <<= 1;
  const int step = kPlanThreads / per, l = tid % per;
  for (int i0 = 0; i0 < a.rows; i0 += kPlanThreads) {
    const int n = min(a.rows - i0, kPlanThreads);
    plan_sync<LDS>();  // held is cleared; the last rows are counted
    if (tid < n) {
      const RowPlan r = i0 == 0 ? mine : row_plan(a, i0 + tid);
      s_src[tid] = r.src;
      s_held[tid] = r.held;
    }
    __syncthreads();
    for (int j0 = 0; j0 < a.width; j0 += per) {
      for (int i = tid / per; i < n; i += 4 * step) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int k = min(i + u * step, n - 1), j = j0 + l;
          id[u] = i + u * step < n && j < s_held[k] ? a.table[s_src[k] * a.table_stride + j] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if ((unsigned)id[u] < (unsigned)a.pages) held.add(id[u], 1);
      }
    }
  }
  plan_sync<LDS>();
}

// One workgroup. Three passes over the pages' counters, two over the rows: bound by
// latency, 4.6 us for 8 rows of 512 pages, 6 us for 256 rows of 2048.
template <bool LDS>
__global__ __launch_bounds__(kPlanThreads) void pages_fork_plan_kernel(PageArgs a) {
  extern __shared__ int s_pages[];
  __shared__ int s_wave[kPlanThreads / 64], s_src[kPlanThreads], s_held[kPlanThreads];
  const Counters<LDS> held{LDS ? s_pages : a.s.held}, first{LDS ? s_pages + a.pages : a.s.first};
  const int tid = threadIdx.x;
  // the first rows' plans and the pages they write are looked up once
  RowPlan mine{};
  int mine_w = -1;
  if (tid < a.rows) {
    mine = row_plan(a, tid);
    mine_w = write_page(a, mine);
  }
  for (int p = tid; p < a.pages; p += kPlanThreads) first.put(p, 0x7FFFFFFF);
  count_held<LDS>(a, held, mine, s_src, s_held);
  // free pages in order: each thread takes a run of pages
  const int per = (a.pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(tid * per, a.pages), p1 = min(p0 + per, a.pages);
  int n = 0, nfree;
  for (int p = p0; p < p1; ++p) n += held.get(p) == 0;
  int at = block_prefix(n, s_wave, nfree);
  for (int p = p0; p < p1; ++p)
    if (held.get(p) == 0) a.s.list[at++] = p;
  __syncthreads();
  // holders that do not write: what is left of held without the writers
  for (int i = tid; i < a.rows; i += kPlanThreads) {
    const int w = i == tid ? mine_w : write_page(a, row_plan(a, i));
    if (w >= 0) {
      held.add(w, -1);
      first.min(w, i);
    }
  }
  plan_sync<LDS>();
  int wanted = 0, pairs = 0, overfull = 0;
  for (int i0 = 0; i0 < a.rows; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int copy = 0, w = -1, want = 0, over = 0;
    if (i < a.rows) {
      const RowPlan r = i0 == 0 ? mine : row_plan(a, i);
      w = i0 == 0 ? mine_w : write_page(a, r);
      copy = w >= 0 && (held.get(w) > 0 || first.get(w) != i);
      want = copy + (r.need - r.held);
      over = r.over;
    }
    int t_want, t_copy;
    const int base = wanted + block_prefix(want, s_wave, t_want);
    // (copies and overfull rows in one: of either no more than kPlanThreads)
    const int pair = pairs + (block_prefix(over << 16 | copy, s_wave, t_copy) & 0xFFFF);
    if (i < a.rows) a.s.base[i] = copy ? ~base : base;  // negative: its first page is a copy
    if (copy) {
      a.s.src[pair] = w;
      a.s.dst[pair] = base;  // of the list
    }
    wanted += t_want;
    pairs += t_copy & 0xFFFF;
    overfull += t_copy >> 16;
  }
  if (tid == 0) {
    const int missing = max(wanted - nfree, 0);
    a.s.head[kPairs] = missing ? 0 : pairs;
    a.s.head[kOverfull] = overfull;
    a.s.head[kFree] = nfree;
    *a.out_count = missing;
  }
}

// One workgroup. A page that moves keeps in held the (inverted) place of its new
// number in the list. 3.5 us for 4 rows of 256 pages, 4.7 us for 96 of 2048.
template <bool LDS>
__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan_kernel(PageArgs a) {
  extern __shared__ int s_pages[];
  __shared__ int s_wave[kPlanThreads / 64], s_src[kPlanThreads], s_held[kPlanThreads];
  const Counters<LDS> held{LDS ? s_pages : a.s.held};
  const int tid = threadIdx.x;
  count_held<LDS>(a, held, tid < a.rows ? row_plan(a, tid) : RowPlan{}, s_src, s_held);
  const int per = (a.pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(tid * per, a.pages), p1 = min(p0 + per, a.pages);
  int n = 0, used, movers;
  for (int p = p0; p < p1; ++p) n += held.get(p) != 0;
  const int below = block_prefix(n, s_wave, used);
  int m = 0;  // pages in use at or past `used`
  for (int p = max(p0, used); p < p1; ++p) m += held.get(p) != 0;
  int mover = block_prefix(m, s_wave, movers);
  int hole = p0 - below;  // free pages before p0
  for (int p = p0; p < p1; ++p) {
    const bool live = held.get(p) != 0;
    if (p < used && !live) a.s.list[hole] = p;
    int to = 0;
    if (p >= used && live) {
      a.s.first[mover] = p;
      to = ~mover++;
    }
    a.s.held[p] = to;
    hole += !live;
  }
  if (tid == 0) {
    a.s.head[kPairs] = movers;
    *a.out_count = used;
  }
}

// Copies page src[i] to dst[i] in every layer of the four tensors, in pieces
// of 16 KB dealt over the workgroups, past the caches (read and written once).
// Bound by HBM: 0.87 GB read and written in 161 us, 5.4 TB/s; half the workgroups
// 205 us, cached accesses 171. No page is both a source and a
// destination. The destination is dst[i], or list[dst[i]] where a list is given.
__device__ void copy_pages(const PageArgs& a, const int* src, const int* dst, const int* list, int pairs,
                           int block, int blocks) {
  const int vecs = 2 * (a.vec_codes + a.vec_scales), units = (vecs + 1023) / 1024;
  const int64_t total = (int64_t)pairs * a.layers * units;
  for (int64_t u = block; u < total; u += blocks) {
    const int piece = (int)(u % units);
    const int64_t pl = u / units;
    const int layer = (int)(pl % a.layers), pair = (int)(pl / a.layers);
    const int64_t from = src[pair], to = list ? list[dst[pair]] : dst[pair];
    u32x4_t v[4];
    uint8_t* out[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int e = piece * 1024 + k * 256 + threadIdx.x;
      out[k] = nullptr;
      if (e < vecs) {
        const bool sc = e >= 2 * a.vec_codes;
        if (sc) e -= 2 * a.vec_codes;
        const int n = sc ? a.vec_scales : a.vec_codes, second = e >= n;
        const PageBuf& b = a.buf[2 * sc + second];
        uint8_t* at = b.p + layer * b.layer + 16 * (int64_t)(e - second * n);
        v[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(at + from * b.page));
        out[k] = at + to * b.page;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (out[k]) __builtin_nontemporal_store(v[k], reinterpret_cast<u32x4_t*>(out[k]));
  }
}

__global__ __launch_bounds__(256) void pages_fork_kernel(PageArgs a) {
  if ((int)blockIdx.x >= a.table_blocks) {
    copy_pages(a, a.s.src, a.s.dst, a.s.list, a.s.head[kPairs], blockIdx.x - a.table_blocks,
               gridDim.x - a.table_blocks);
    return;
  }
  const int nfree = a.s.head[kFree];
  for (int i = blockIdx.x; i < a.rows; i += a.table_blocks) {
    const RowPlan r = row_plan(a, i);
    const int b = a.s.base[i], copy = b < 0, base = copy ? ~b : b;
    if (threadIdx.x == 0) a.out_lengths[i] = r.after;
    for (int j = threadIdx.x; j < a.width; j += 256) {
      int id = -1, k = -1;
      if (j < r.held - copy)
        id = held_page(a, r, j);
      else if (j < r.need)
        k = base + (j - (r.held - copy));
      if (k >= 0 && k < nfree) id = a.s.list[k];
      a.out_table[(int64_t)i * a.width + j] = id;
    }
  }
}

__global__ __launch_bounds__(256) void pages_compact_kernel(PageArgs a) {
  if ((int)blockIdx.x >= a.table_blocks) {
    copy_pages(a, a.s.first, a.s.list, nullptr, a.s.head[kPairs], blockIdx.x - a.table_blocks,
               gridDim.x - a.table_blocks);
    return;
  }
  for (int i = blockIdx.x; i < a.rows; i += a.table_blocks) {
    const RowPlan r = row_plan(a, i);
    for (int j = threadIdx.x; j < a.width; j += 256) {
      int id = j < r.held ? held_page(a, r, j) : -1;
      if (id >= 0 && a.s.held[id] < 0) id = a.s.list[~a.s.held[id]];
      a.out_table[(int64_t)i * a.width + j] = id;
    }
  }
}

}  // namespace

int paged_kv_append(const PagedBatch& p, const void* k, const void* v, const int64_t* xst,
                    const PagedSide& ks, const PagedSide& vs, int64_t H, int64_t D, int xdt,
                    hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  const PagedAppendArgs a{p, k, v, xst[0], xst[1], xst[2], xst[3], ks, vs, (int)H, (int)D, xdt};
  if (D == 64)
    launch_append<8>(a, st);
  else if (D == 128)
    launch_append<16>(a, st);
  else
    launch_append<32>(a, st);
  return check_launch("paged_append_kernel");
}

size_t kv_pages_workspace(int64_t rows, int64_t pages) {
  return (size_t)(kHead + 3 * pages + 3 * rows) * sizeof(int);
}

// what fork and compact have in common; the output pointers are theirs
static PageArgs page_args(const int32_t* table, int64_t table_stride, const int32_t* lengths,
                          int64_t B, int64_t rows, int64_t width, int64_t pages, int page_size,
                          int64_t layers, void* const* bufs, const int64_t* strides,
                          int64_t code_bytes, int64_t scale_bytes, void* ws) {
  PageArgs a{};
  a.table = table;
  a.lengths = lengths;
  a.table_stride = table_stride;
  a.B = (int)B;
  a.rows = (int)rows;
  a.width = (int)width;
  a.pages = (int)pages;
  a.page_log2 = __builtin_ctz((unsigned)page_size);
  a.s = page_scratch((int*)ws, pages, rows);
  for (int i = 0; i < 4; ++i)
    a.buf[i] = PageBuf{(uint8_t*)bufs[i], strides[2 * i], strides[2 * i + 1]};
  a.vec_codes = (int)(code_bytes / 16);
  a.vec_scales = (int)(scale_bytes / 16);
  a.layers = (int)layers;
  a.table_blocks = (int)std::min<int64_t>(std::max<int64_t>(rows, 1), 512);
  return a;
}

static dim3 page_grid(const PageArgs& a) { return dim3((unsigned)(a.table_blocks + 8 * device_cus())); }

int kv_pages_fork(const int32_t* table, int64_t table_stride, const int32_t* lengths,
                  const int32_t* parents, const int32_t* fresh, int32_t* out_table,
                  int32_t* out_lengths, int32_t* missing, int64_t B, int64_t rows, int64_t width,
                  int64_t pages, int page_size, int64_t layers, void* const* bufs,
                  const int64_t* strides, int64_t code_bytes, int64_t scale_bytes, void* ws,
                  hipStream_t st) {
  PageArgs a = page_args(table, table_stride, lengths, B, rows, width, pages, page_size, layers, bufs,
                         strides, code_bytes, scale_bytes, ws);
  a.parents = parents;
  a.fresh = fresh;
  a.out_table = out_table;
  a.out_lengths = out_lengths;
  a.out_count = missing;
  if (pages <= kLdsPages)
    hipLaunchKernelGGL(pages_fork_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 2 * pages * sizeof(int), st, a);
  else
    hipLaunchKernelGGL(pages_fork_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, st, a);
  hipLaunchKernelGGL(pages_fork_kernel, page_grid(a), dim3(256), 0, st, a);
  return check_launch("pages_fork_kernel");
}

int kv_pages_compact(const int32_t* table, int64_t table_stride, const int32_t* lengths,
                     int32_t* out_table, int32_t* used, int64_t B, int64_t width, int64_t pages,
                     int page_size, int64_t layers, void* const* bufs, const int64_t* strides,
                     int64_t code_bytes, int64_t scale_bytes, void* ws, hipStream_t st) {
  PageArgs a = page_args(table, table_stride, lengths, B, B, width, pages, page_size, layers, bufs,
                         strides, code_bytes, scale_bytes, ws);
  a.out_table = out_table;
  a.out_count = used;
  if (pages <= kLdsPages)
    hipLaunchKernelGGL(pages_compact_plan_kernel<true>, dim3(1), dim3(kPlanThreads), pages * sizeof(int), st, a);
  else
    hipLaunchKernelGGL(pages_compact_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, st, a);
  hipLaunchKernelGGL(pages_compact_kernel, page_grid(a), dim3(256), 0, st, a);
  return check_launch("pages_compact_kernel");
}

}  // namespace sparkq
