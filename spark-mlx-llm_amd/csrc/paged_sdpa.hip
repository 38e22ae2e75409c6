// paged_sdpa.hip -- attention of packed new tokens over a paged INT8 KV cache
// (symmetric s8 codes, one fp16 scale per token and KV head) on gfx950.
//
//   o[t,h] = sum_n p_n v_n / sum_n p_n,  p_n = exp(scale * q[t,h] . k_n - max)
//
// over the tokens n that row t of sequence b sees: n <= length - count + (t -
// first) under the causal mask, n < length without. Tokens of an absent page
// are hidden, and a row that sees nothing is zero.
//
// Rows. The query rows of a (sequence, KV head) are its (position, query head)
// pairs, rr = position * Hq/Hkv + head: they share every key and value.
//   paged_few_kernel   at most 16 of them (decode, a few drafted tokens): the
//                      waves of a workgroup take turns at 32-token blocks and
//                      combine at the end.
//   paged_tile_kernel  tiles of 128 rows (64 at D = 256): a block is turned to
//                      fp16 in LDS once for all of them.
//   paged_merge_kernel joins the parts of a context that was split.
//
// Work. The lengths live on the device, so every workgroup works out from the
// batch's starts and lengths which (sequence, tile, part of the context) is
// its own (find_item): a context is split so that about `target` parts of equal
// length fill the chip however the lengths differ, and a grid sized by the
// host for the worst case has nothing left over but idle workgroups.
//
// Numerics. Both products are fp16 MFMAs with fp32 sums. Codes are exact in
// fp16; a query row is shifted by a power of two to be exact too. The weight
// of a value, p_n times its scale, is rounded to fp16 once (at most 2^-11 of it,
// what an fp16 output's own rounding is and an eighth of a bf16 output's), under
// a power of two that puts the largest one near 2^7: 2^8 of room for the running
// maximum, which moves only when a block exceeds it by that much, and full
// precision down to 2^-19 of the largest. The running maximum, the normalizer and the
// sums are fp32.
#include <algorithm>
#include <type_traits>

#include "paged.h"
#include "sdpa_common.h"

namespace sparkq {
namespace {

// The cache as the attention addresses it. Keys and values lie alike, so that one
// offset serves both; the page strides are in units of 16 bytes (codes) and 8
// scales, so that a page's offset is one 32-bit product, and a head's tokens
// within a page span less than 32 bits.
struct CodeLayout {
  const uint8_t *k, *v;
  const uint16_t *ks, *vs;
  int64_t c_head, s_head;
  uint32_t c_page, s_page, c_tok;
};

struct PagedSdpaArgs {
  PagedBatch p;
  const uint16_t* q;
  int64_t q_tok, q_head;  // elements
  CodeLayout c;
  void* out;  // [T, Hq, D]
  float *pm, *pz, *pacc;  // [Hkv][slots][rows], [...], [...][D]: parts of split contexts
  int Hq, Hkv, max_new, causal, q_dtype, out_dtype;
  int target;      // parts of the whole batch, about, per KV head
  int slots;       // parts of split contexts, at most, per KV head
  int min_part;    // tokens of a part, at least
  float scale_log2;
};

constexpr int kFewBlock = 32;  // tokens of a block

// ---------------------------------------------------------------------------
// which work is whose
// ---------------------------------------------------------------------------
struct Item {
  int b;               // sequence, or -1: nothing left
  int tile;            // of `rows` / R
  int part, parts;     // of the tile's context
  int slot;            // of the first part (parts > 1)
  int first, count, length, rows;
};

struct SeqWork {
  int first, count, length, rows, tiles;
};

template <int R>  // rows of a tile: 16, 64 or 128
__device__ __forceinline__ SeqWork seq_work(const PagedSdpaArgs& a, int b) {
  SeqWork w{0, 0, 0, 0, 0};
  if (b < a.p.B) {
    const SeqRows s = seq_rows(a.p, b);
    w.first = s.first;
    w.count = s.count;
    w.length = s.length;
    w.rows = min(s.count, a.max_new) * (a.Hq / a.Hkv);
    w.tiles = (w.rows + R - 1) / R;
  }
  return w;
}

// inclusive prefix over the wave's lanes: row shifts, then the rows' totals
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// Reorders the sequences of up to 64 lanes, the longest first: a batch's short
// tiles come last and fill the gaps that the long ones leave.
__device__ __forceinline__ void longest_first(SeqWork& w, int& b, int n) {
  const int lane = threadIdx.x & 63, key = w.tiles ? w.length : -1;
  int rank = 0;
  for (int j = 0; j < n; ++j) {
    const int k = __builtin_amdgcn_readlane(key, j);
    rank += k > key || (k == key && j < lane);
  }
  const int to = 4 * (lane < n ? rank : lane);
  for (int* f : {&w.first, &w.count, &w.length, &w.rows, &w.tiles, &b}) *f = __builtin_amdgcn_ds_permute(to, *f);
}

// Item x of the batch's items in order (SPLIT false: every tile and part), or
// tile x of those whose context is split. A context of n tokens is split into
// ceil(n / C) parts, C = max(min_part, W / target + 1), W all tiles' tokens: fewer
// than `target` contexts are longer than C, and these have fewer than 2 target
// parts together. (W is summed in fp32, to 2^-17 of itself, which C is enlarged
// by.) All lanes of a wave take part, and every wave gets the same answers.
template <int R, bool SPLIT>
__device__ Item find_item(const PagedSdpaArgs& a, int x) {
  const int lane = threadIdx.x & 63;
  int b_of = lane;
  SeqWork w0 = seq_work<R>(a, lane);
  if (R > 16 && a.p.B > 1 && a.p.B <= 64) longest_first(w0, b_of, a.p.B);
  float all = (float)w0.tiles * (float)w0.length;
  for (int b0 = 64; b0 < a.p.B; b0 += 64) {
    const SeqWork w = seq_work<R>(a, b0 + lane);
    all = fmaf((float)w.tiles, (float)w.length, all);
  }
  const float share = wave_sum(all) / (float)a.target;
  const int C = (int)fminf(fmaxf(share + share * 0x1p-16f + 1.0f, (float)a.min_part), 0x1p30f);
  Item it{-1, 0, 0, 1, 0, 0, 0, 0, 0};
  int items = 0, slots = 0;
  for (int b0 = 0; b0 < a.p.B; b0 += 64) {
    const SeqWork w = b0 == 0 ? w0 : seq_work<R>(a, b0 + lane);
    const int parts = w.length > C ? (w.length - 1) / C + 1 : 1;
    const int own = SPLIT ? (parts > 1 ? w.tiles : 0) : w.tiles * parts;
    const int used = parts > 1 ? w.tiles * parts : 0;
    const int end = items + wave_prefix(own), slot_end = slots + wave_prefix(used);
    const unsigned long long hit = __ballot(x < end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      it.b = b0 + of(b_of);
      it.first = of(w.first);
      it.count = of(w.count);
      it.length = of(w.length);
      it.rows = of(w.rows);
      it.parts = of(parts);
      const int i = x - of(end - own), tiles = of(w.tiles);
      const int k = SPLIT ? i : i / it.parts;
      it.part = SPLIT ? 0 : i - k * it.parts;
      it.tile = tiles - 1 - k;  // the last tiles see the most: they start first
      it.slot = of(slot_end - used) + k * it.parts;
      // sequences whose starts overlap are more than the workspace is for, and may be
      // more than 32 bits count
      if ((it.parts > 1 && it.slot + it.parts > a.slots) || (unsigned)i >= (unsigned)of(own)) it.b = -1;
      break;
    }
    items = __builtin_amdgcn_readlane(end, 63);
    slots = __builtin_amdgcn_readlane(slot_end, 63);
  }
  // (the compiler does not see that a loop left on a ballot leaves scalars)
  for (int* f : {&it.b, &it.tile, &it.part, &it.parts, &it.slot, &it.first, &it.count, &it.length, &it.rows})
    *f = __builtin_amdgcn_readfirstlane(*f);
  return it;
}

// last token that row rr of the item sees (-1: none)
__device__ __forceinline__ int last_seen(const PagedSdpaArgs& a, const Item& it, int rr, int gqa) {
  if (rr >= it.rows) return -1;
  if (!a.causal) return it.length - 1;
  return min(max(it.length - it.count + rr / gqa, -1), it.length - 1);
}

// ---------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------
// 8 codes -> fp16, exactly: under the fp16 pattern of 1024 the byte c ^ 0x80
// reads 1024 + 128 + c
__device__ __forceinline__ u32x4_t s8x8_exact(uint32_t lo, uint32_t hi) {
  const uint32_t x = lo ^ 0x80808080u, y = hi ^ 0x80808080u;
  auto pair = [](uint32_t w, uint32_t sel) {
    return exact_f16_pair<128>(__builtin_amdgcn_perm(0x64646464u, w, sel));
  };
  return u32x4_t{pair(x, 0x04010400u), pair(x, 0x04030402u), pair(y, 0x04010400u), pair(y, 0x04030402u)};
}

// max / sum over a row's lanes (l, l ^ 32 and, in four groups of 16, l ^ 16 and
// l ^ 48), the same value in all of them
template <int G>
__device__ __forceinline__ float max_groups(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  if (G == 2) return v;
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int G>
__device__ __forceinline__ float sum_groups(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  if (G == 2) return v;
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A row's query values as exact fp16 under a power of two: chunk c of this lane
// holds dims dim0(c) .. +8. Returns the factor that undoes the shift.
template <int NK, int G, typename F>
__device__ __forceinline__ float load_query(const PagedSdpaArgs& a, const uint16_t* row, bool live, F dim0,
                                            u32x4_t qb[NK]) {
  float top = 0.0f;
  auto value = [&](u32x4_t w, int i) {
    const uint16_t bits = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    return live ? (a.q_dtype == SPARKQ_BF16 ? bf16_to_f32(bits) : f16_to_f32(bits)) : 0.0f;
  };
#pragma unroll
  for (int c = 0; c < NK; ++c) {
    qb[c] = *reinterpret_cast<const u32x4_t*>(row + dim0(c));
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(value(qb[c], i)));
  }
  top = max_groups<G>(top);
  const int e = top > 0.0f && top <= 3.4028235e38f ? ilogbf(top) - 14 : 0;
#pragma unroll
  for (int c = 0; c < NK; ++c) {
    const u32x4_t w = qb[c];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qb[c][i] = pack_round<F16>(ldexpf(value(w, 2 * i), -e), ldexpf(value(w, 2 * i + 1), -e));
  }
  return ldexpf(1.0f, e);
}

// v, in a way that what depends on it stays in its branch: the compiler would
// otherwise rescale the sums of every block and select, at twice the registers
__device__ __forceinline__ float pinned(float v) {
  asm volatile("" : "+v"(v));
  return v;
}

// two values rounded (to nearest even) into packed fp16: one instruction
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_t));
}

// ---------------------------------------------------------------------------
// online softmax of one block for one row per lane
// ---------------------------------------------------------------------------
// The state counts in units of 2^-M, M = m + e - 6: m the running maximum of
// the scores (log2 units) and 2^e .. 2^(e+1) the largest finite value scale that
// the row has seen, so that exp2(s - M) * v_scale < 2^7 at s = m.
struct RowState {
  float m = kNegInf;  // -inf: nothing seen
  float z = 0.0f;
  float e = -24.0f;  // of the smallest fp16
};
constexpr float kRoom = 8.0f;

__device__ __forceinline__ float unit(const RowState& st) { return st.m + (st.e - 6.0f); }

// |scale|, 0 where it does not count or is not finite
__device__ __forceinline__ float scale_size(float v, bool counts) {
  v = fabsf(v);
  return counts && v <= 65504.0f ? v : 0.0f;
}

// What a part of a row's context hands on: its M, or -inf where it saw nothing
// (scores that are all NaN leave no maximum, but a sum that is not 0).
__device__ __forceinline__ float part_max(const RowState& st, float z) {
  return st.m != kNegInf ? unit(st) : (z != 0.0f ? 0.0f : kNegInf);
}

// A block's N scores of this lane's row (raw sums times the key scales times
// the softmax scale: s * mul is in log2 units), of which those in `ok` are
// visible where MASK; `size` is the block's largest finite value scale, used
// where all of it is visible. Writes the packed fp16 weights of the lane's N
// values; returns the factor for what is summed so far (up: it is not 1).
template <int N, int G>
__device__ __forceinline__ float row_block(RowState& st, const float s[N], float mul, const float vsc[N],
                                           float size, u32x4_t w[N / 8], bool& up) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, s[i]);
  top = max_groups<G>(top) * mul;
  const float e = fmaxf(st.e, (float)((int)(__float_as_uint(size) >> 23) - 127));
  const bool raise = top > st.m + kRoom;
  up = raise || e != st.e;
  const float old = unit(st);
  if (raise) st.m = ceilf(top);
  st.e = e;
  const float M = st.m == kNegInf ? 0.0f : unit(st);
  const float alpha = old == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(old - M);
  float p[N], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], mul, -M));
    sum += p[i];
    p[i] *= vsc[i];
  }
  st.z = fmaf(st.z, up ? alpha : 1.0f, sum);
#pragma unroll
  for (int i = 0; i < N; i += 2) w[i / 8][i / 2 % 4] = pack_f16(p[i], p[i + 1]);
  return alpha;
}

// A value scale as the tile kernel keeps it: what is not finite is -0, so that a
// hidden token's weight of 0 times its scale is 0, and a visible one is found.
__device__ __forceinline__ float kept_scale(float v) {
  return fabsf(v) <= 65504.0f ? v + 0.0f : -0.0f;
}

// Hides the scores that are not in `ok` and turns those of values that are not
// finite to NaN; returns the largest value scale of the others.
template <int N, int G>
__device__ __forceinline__ float hide(uint32_t ok, float s[N], const float vsc[N]) {
  float size = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool live = (ok >> i) & 1u;
    s[i] = live ? (__float_as_uint(vsc[i]) == 0x80000000u ? __builtin_nanf("") : s[i]) : kNegInf;
    size = fmaxf(size, live ? fabsf(vsc[i]) : 0.0f);
  }
  return max_groups<G>(size);
}

// Four outputs (dims d .. d + 3) of a row.
__device__ __forceinline__ void store_row4(const PagedSdpaArgs& a, int64_t at, f32x4_t v) {
  if (a.out_dtype == SPARKQ_F32) {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(a.out) + at) = v;
  } else {
    const bool bf = a.out_dtype == SPARKQ_BF16;
    uint2 w;
    w.x = bf ? pack_round<BF16>(v[0], v[1]) : pack_round<F16>(v[0], v[1]);
    w.y = bf ? pack_round<BF16>(v[2], v[3]) : pack_round<F16>(v[2], v[3]);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at) = w;
  }
}

__device__ __forceinline__ int64_t out_row(const PagedSdpaArgs& a, const Item& it, int kh, int rr, int gqa) {
  return ((int64_t)(it.first + rr / gqa) * a.Hq + kh * gqa + rr % gqa);
}

// Offsets within a KV head's codes (bytes) and scales (elements) of a page's slot
__device__ __forceinline__ uint64_t code_at(const CodeLayout& c, int id, int slot) {
  return ((uint64_t)(uint32_t)id * c.c_page << 4) + (uint32_t)slot * c.c_tok;
}
__device__ __forceinline__ uint64_t scale_at(const CodeLayout& c, int id, int slot) {
  return ((uint64_t)(uint32_t)id * c.s_page << 3) + (uint32_t)slot;
}

// Pages of a block's Q runs of 16 tokens; a run without one reads page 0 and is
// hidden (ok). Past the table's row the last entry stands in (those tokens lie
// past every length).
template <int Q>
struct BlockPages {
  int id[Q];
  uint32_t ok;
};
//
// The table is read by scalar loads (its constant address space says that no
// store of this kernel changes it): a vector load among those of the codes
// would be waited for in their order.
typedef const __attribute__((address_space(4))) int32_t* TableRow;
__device__ __forceinline__ TableRow table_row(const PagedSdpaArgs& a, int b) {
  return (TableRow)(uintptr_t)(a.p.table + b * a.p.table_stride);
}
template <int Q>
__device__ __forceinline__ BlockPages<Q> block_pages(const PagedSdpaArgs& a, TableRow row, int t0) {
  BlockPages<Q> r;
  auto look = [&](int h) {
    const int id = row[min((t0 + 16 * h) >> a.p.page_log2, a.p.width - 1)];
    return id;
  };
  auto keep = [&](int h, int id) {
    const bool in = (unsigned)id < (unsigned)a.p.pages;
    r.ok |= (uint32_t)in << h;
    r.id[h] = in ? id : 0;
  };
  r.ok = 0;
  if ((1 << a.p.page_log2) >= 16 * Q) {  // blocks do not straddle pages
    keep(0, look(0));
#pragma unroll
    for (int h = 1; h < Q; ++h) r.id[h] = r.id[0];
    r.ok = r.ok ? (1u << Q) - 1 : 0;
  } else {
#pragma unroll
    for (int h = 0; h < Q; ++h) keep(h, look(h));
  }
  return r;
}

// ---------------------------------------------------------------------------
// at most 16 rows
// ---------------------------------------------------------------------------
// S^T (16 tokens x 16 rows) = K . Q^T twice a block, O^T (16 dims x 16 rows) +=
// V^T . P^T. Row m of the first product's operand is token 8 (m / 4) + m % 4
// (+ 4 in the second), so that the lane with a row's scores of tokens 8g ..
// 8g+7 holds just the k-slots of the second product's operand: weights never
// leave their lane. V goes through a wave's own LDS to be read transposed.
template <int D>
struct FewLds {
  static constexpr int VROW = D + 16;
  static constexpr int VT = kFewBlock * VROW;          // one wave's V block
  static constexpr int LOOP = 4 * VT;
  static constexpr int JOIN = 4 * 16 * (2 + D) * 4;  // the waves' maxima, sums and outputs
  static constexpr int BYTES = LOOP > JOIN ? LOOP : JOIN;
};

template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 3 : 2) void paged_few_kernel(PagedSdpaArgs a) {
  constexpr int NK = D / 32, PL = D / 64, NJ = D / 16, VL = D / 32;
  using L = FewLds<D>;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int kBlock = kFewBlock;
  const int n16 = lane & 15, grp = lane >> 4;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<16, false>(a, blockIdx.x / a.Hkv);
  if (it.b < 0) return;
  const int rows = min(it.rows - 16 * it.tile, 16);
  const int rr = 16 * it.tile + min(n16, rows - 1);
  const int lim = last_seen(a, it, rr, gqa);
  const int seen = last_seen(a, it, 16 * it.tile + rows - 1, gqa) + 1;  // by the last row: the most
  const int nblocks = (seen + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const TableRow trow = table_row(a, it.b);
  unsigned char* vtile = smem + wave * L::VT;

  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + (it.first + rr / gqa) * a.q_tok + (kh * gqa + rr % gqa) * a.q_head;
  // chunk c: dims 16 (g + 4 (c / 2)) + 8 (c % 2), as the 16-byte pieces of K lie
  const float mul = load_query<NK, 4>(a, qrow, true, [&](int c) { return 16 * (grp + 4 * (c >> 1)) + 8 * (c & 1); }, qb);

  u32x4_t kr[2][PL], vr[VL], skr, svr;
  BlockPages<2> next;
  uint32_t pages_ok;
  const int ktok = 8 * (n16 >> 2) + (n16 & 3);
  const uint32_t koff = (ktok & 15) * a.c.c_tok + 16 * grp;
  const uint8_t *const khead = a.c.k + kh * a.c.c_head, *const vhead = a.c.v + kh * a.c.c_head;
  const uint16_t *const kshead = a.c.ks + kh * a.c.s_head, *const vshead = a.c.vs + kh * a.c.s_head;
  const int slot_mask = (1 << a.p.page_log2) - 1;
  const int last = ib1 - 1;
  // block ib (no further than the last) through the pages found for it
  auto load = [&](int ib, const BlockPages<2>& bp) {
    const int t0 = kBlock * min(ib, last);
    const int s0 = t0 & slot_mask, s1 = (t0 + 16) & slot_mask;
    const uint64_t o0 = code_at(a.c, bp.id[0], s0), o1 = code_at(a.c, bp.id[1], s1);
    const uint8_t *kp = khead + (n16 < 8 ? o0 : o1) + koff, *v0 = vhead + o0, *v1 = vhead + o1;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < PL; ++i)
        kr[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kp + (4 * t * a.c.c_tok + 64 * i)));
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      vr[v] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>((2 * v >= VL ? v1 : v0) + ((tok & 15) * a.c.c_tok + 16 * pc)));
    }
    const bool h = grp >= 2;
    const uint64_t so = scale_at(a.c, h ? bp.id[1] : bp.id[0], (h ? s1 : s0) + 8 * (grp & 1));
    skr = *reinterpret_cast<const u32x4_t*>(kshead + so);
    svr = *reinterpret_cast<const u32x4_t*>(vshead + so);
    pages_ok = bp.ok;
  };

  RowState st;
  f32x4_t acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto block = [&](int ib) {
    const int t0 = kBlock * ib;
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      *reinterpret_cast<u32x4_t*>(vtile + tok * L::VROW + 16 * pc) = vr[v];
    }
    f32x4_t sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const u32x4_t kp = kr[t][c >> 1];
        sc[t] = mfma16x16x32_f16((c & 1) ? s8x8_exact(kp.z, kp.w) : s8x8_exact(kp.x, kp.y), qb[c], sc[t]);
      }
    }
    float s[8], vsc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kw = skr[i >> 1], vw = svr[i >> 1];
      s[i] = sc[i >> 2][i & 3] * (((i & 1) ? hi16<F16>(kw) : lo16<F16>(kw)) * a.scale_log2);
      vsc[i] = (i & 1) ? hi16<F16>(vw) : lo16<F16>(vw);
    }
    uint32_t ok = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ok |= (uint32_t)(t0 + 8 * grp + i <= lim) << i;
    if (!((pages_ok >> (grp >> 1)) & 1u)) ok = 0;
    load(ib + 4, next);
    next = block_pages<2>(a, trow, kBlock * min(ib + 8, last));
    u32x4_t w;
    bool up;
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool live = (ok >> i) & 1u;
      s[i] = live ? s[i] : kNegInf;
      vsc[i] = live ? vsc[i] : 0.0f;
      size = fmaxf(size, scale_size(vsc[i], true));
    }
    size = max_groups<4>(size);
    const float alpha = row_block<8, 4>(st, s, mul, vsc, size, &w, up);
    if (__ballot(up)) {
      const float f = pinned(up ? alpha : 1.0f);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
    const unsigned char* vaddr = vtile + (8 * grp + (n16 >> 1)) * L::VROW + 8 * (n16 & 1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      typedef int v2i_t __attribute__((ext_vector_type(2)));
      const v2i_t t8 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (__attribute__((address_space(3))) v2i_t*)(vaddr + 16 * j));
      acc[j] = mfma16x16x32_f16(s8x8_exact((uint32_t)t8.x, (uint32_t)t8.y), w, acc[j]);
    }
  };

  int ib = ib0 + wave;
  if (ib < ib1) {
    load(ib, block_pages<2>(a, trow, kBlock * ib));
    next = block_pages<2>(a, trow, kBlock * min(ib + 4, last));
    for (; ib < ib1; ib += 4) block(ib);
  }

  // combine the waves
  const float z = sum_groups<4>(st.z);
  __syncthreads();
  float* wm = reinterpret_cast<float*>(smem);  // [4][16]
  float* wz = wm + 64;                         // [4][16]
  float* wacc = wz + 64;                       // [4][16][D]
  if (n16 < rows) {
    if (grp == 0) {
      wm[wave * 16 + n16] = part_max(st, z);
      wz[wave * 16 + n16] = z;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      *reinterpret_cast<f32x4_t*>(wacc + (wave * 16 + n16) * D + 16 * j + 4 * grp) = acc[j];
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += 256) {
    const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
    float mm = kNegInf, zz = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, wm[w * 16 + r]);
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float m = wm[w * 16 + r];
      if (m == kNegInf) continue;
      const float f = __builtin_amdgcn_exp2f(m - mm);
      zz = fmaf(wz[w * 16 + r], f, zz);
      o += *reinterpret_cast<const f32x4_t*>(wacc + (w * 16 + r) * D + d) * f;
    }
    if (it.parts == 1) {
      if (zz != 0.0f) o /= zz;
      store_row4(a, out_row(a, it, kh, 16 * it.tile + r, gqa) * D + d, o);
    } else {
      const int64_t at = ((int64_t)kh * a.slots + it.slot + it.part) * 16 + r;
      *reinterpret_cast<f32x4_t*>(a.pacc + at * D + d) = o;
      if (d == 0) {
        a.pm[at] = mm;
        a.pz[at] = zz;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// tiles of 128 or 64 rows
// ---------------------------------------------------------------------------
// Four waves of MT rows each. The products run as above on the MT x MT MFMA: 32
// rows a wave up to D = 128, 16 at 256, with blocks of 64 and 32 tokens, which is
// what fits two workgroups a CU in registers and LDS. These are at different
// places of their blocks, so that one's products and LDS reads run beside the
// other's softmax (at D = 256 eight waves of 16 rows in one workgroup a CU, all in
// step, took 368 us for 24 sequences of up to 1000 new tokens, two of four 356).
// A lane has one row, and of a block the scores i of tokens 4 G (i / 4) + 4 g + i %
// 4, g its group of the G = 64 / MT: scores 8 s .. +8 are its k-slots of the second
// product's step s.
//
// A block of codes is read once by the workgroup and written to LDS as fp16,
// token-major, two buffers deep: the next block's codes are converted while this
// one is computed, and the one after is in flight. K rows are padded by 16 bytes,
// or at D = 256 their 16-byte chunks XOR-swizzled by the token, so that any 16
// lanes of a read that the LDS takes together hit different banks; V rows, read
// transposed, are padded to the same end.
template <int D>
struct TileShape {
  static constexpr int MT = D <= 128 ? 32 : 16, G = 64 / MT;
  static constexpr int ROWS = 4 * MT;                 // of a workgroup
  static constexpr int BLOCK = D <= 128 ? 64 : 32;    // tokens
  static constexpr int N = BLOCK * MT / 64;           // scores a lane
  static constexpr int KROW = 2 * D + (MT == 32 ? 16 : 0), VROW = 2 * D + (MT == 32 ? 64 : 32);
  static constexpr int V = BLOCK * KROW;
  static constexpr int SCALES = V + BLOCK * VROW;     // of keys, of values, the largest of each 16 of these
  static constexpr int BUF = SCALES + 2 * BLOCK * 4 + 16;
  static constexpr int BYTES = 2 * BUF;
};

template <int MT>
struct TileSum {
  typedef f32x4_t type;
};
template <>
struct TileSum<32> {
  typedef f32x16_t type;
};
__device__ __forceinline__ f32x4_t tile_mfma(u32x4_t x, u32x4_t y, f32x4_t c) { return mfma16x16x32_f16(x, y, c); }
__device__ __forceinline__ f32x16_t tile_mfma(u32x4_t x, u32x4_t y, f32x16_t c) { return mfma32x32x16<F16>(x, y, c); }

template <int D>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedSdpaArgs a) {
  using S = TileShape<D>;
  constexpr int MT = S::MT, G = S::G, R = S::ROWS, kBlock = S::BLOCK, N = S::N, Q = kBlock / 16;
  constexpr int NK = D / (8 * G), NJ = D / MT, NT = kBlock / MT, NV = MT * MT / 64;
  constexpr int PPT = kBlock * D / 16 / 256;  // 16-code pieces of a K (or V) block per thread
  using Sum = typename TileSum<MT>::type;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, row = lane % MT, grp = lane / MT;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<R, false>(a, blockIdx.x / a.Hkv);
  if (it.b < 0) return;
  const int rw0 = R * it.tile;
  const int rows = min(it.rows - rw0, R);
  const int seen = last_seen(a, it, rw0 + rows - 1, gqa) + 1;
  const int nblocks = (seen + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const TableRow trow = table_row(a, it.b);

  const int wr0 = rw0 + MT * wave;  // the wave's first row
  const int rr = wr0 + row, rq = min(rr, it.rows - 1);
  const int lim = last_seen(a, it, rr, gqa);
  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + (it.first + rq / gqa) * a.q_tok + (kh * gqa + rq % gqa) * a.q_head;
  const float mul = load_query<NK, G>(a, qrow, rr < it.rows, [&](int c) { return 8 * G * c + 8 * grp; }, qb);
  // what every row of the tile sees
  const int all = __builtin_amdgcn_readfirstlane(last_seen(a, it, rw0, gqa) + 1);

  // Piece p = tid + 256 i of a block: token p / (D / 16), codes 16 (p % (D / 16)).
  // All tokens of a wave's i-th piece lie in one run of 16, and so in one page.
  // Wave w < Q also takes the scales of run w: keys in its first 16 lanes, values
  // in the next. Where blocks do not straddle pages all of a block's addresses are
  // one offset and the lane's own.
  const int slot_mask = (1 << a.p.page_log2) - 1;
  const bool one_page = slot_mask + 1 >= kBlock;
  u32x4_t kcr[PPT], vcr[PPT];
  uint16_t sr;
  const int last = ib1 - 1;
  const uint8_t *const khead = a.c.k + kh * a.c.c_head, *const vhead = a.c.v + kh * a.c.c_head;
  const uint16_t* const shead = (lane < 16 ? a.c.ks : a.c.vs) + kh * a.c.s_head + n16;
  const int tk0 = tid / (D / 16), jb = tid % (D / 16);
  constexpr int TPP = 256 / (D / 16);  // tokens of a round of pieces
  const uint32_t run_off = (tk0 & 15) * a.c.c_tok + 16 * jb;
  uint32_t off[PPT];
#pragma unroll
  for (int i = 0; i < PPT; ++i) off[i] = (tk0 + i * TPP) * a.c.c_tok + 16 * jb;
  auto load = [&](int ib, const BlockPages<Q>& bp) {
    const int t0 = kBlock * min(ib, last);
    if (one_page) {
      const uint64_t at = code_at(a.c, bp.id[0], t0 & slot_mask);
      const uint8_t *kp = khead + at, *vp = vhead + at;
#pragma unroll
      for (int i = 0; i < PPT; ++i) {
        kcr[i] = *reinterpret_cast<const u32x4_t*>(kp + off[i]);
        vcr[i] = *reinterpret_cast<const u32x4_t*>(vp + off[i]);
      }
      if (wave < Q) sr = shead[scale_at(a.c, bp.id[0], (t0 & slot_mask) + 16 * wave)];
    } else {
      auto page_id = [&](int run) {
        return run == 0 ? bp.id[0] : Q == 2 || run == 1 ? bp.id[1] : run == 2 ? bp.id[Q - 2] : bp.id[Q - 1];
      };
#pragma unroll
      for (int i = 0; i < PPT; ++i) {
        const int run = wave * 64 / D + i * (TPP / 16);
        const uint64_t at = code_at(a.c, page_id(run), (t0 + 16 * run) & slot_mask);
        kcr[i] = *reinterpret_cast<const u32x4_t*>(khead + at + run_off);
        vcr[i] = *reinterpret_cast<const u32x4_t*>(vhead + at + run_off);
      }
      if (wave < Q) sr = shead[scale_at(a.c, page_id(wave), (t0 + 16 * wave) & slot_mask)];
    }
  };
  auto kswz = [](int t) { return MT == 32 ? 0 : t & 15; };
  unsigned char* const kput0 = smem + tk0 * S::KROW + 16 * ((2 * jb) ^ kswz(tk0));
  unsigned char* const kput1 = smem + tk0 * S::KROW + 16 * ((2 * jb + 1) ^ kswz(tk0));
  unsigned char* const vput = smem + S::V + tk0 * S::VROW + 32 * jb;
  auto stage = [&](auto bufc) {
    constexpr int at = decltype(bufc)::value * S::BUF;
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      *reinterpret_cast<u32x4_t*>(kput0 + at + i * TPP * S::KROW) = s8x8_exact(kcr[i].x, kcr[i].y);
      *reinterpret_cast<u32x4_t*>(kput1 + at + i * TPP * S::KROW) = s8x8_exact(kcr[i].z, kcr[i].w);
      unsigned char* vt = vput + at + i * TPP * S::VROW;
      *reinterpret_cast<u32x4_t*>(vt) = s8x8_exact(vcr[i].x, vcr[i].y);
      *reinterpret_cast<u32x4_t*>(vt + 16) = s8x8_exact(vcr[i].z, vcr[i].w);
    }
    if (wave < Q) {
      float* sc = reinterpret_cast<float*>(smem + at + S::SCALES);
      const float v = f16_to_f32(sr);
      const float big = max_row16(fabsf(v) <= 65504.0f ? fabsf(v) : __builtin_huge_valf());
      if (lane < 32) sc[(lane < 16 ? 0 : kBlock) + 16 * wave + n16] = lane < 16 ? v * a.scale_log2 : kept_scale(v);
      if (lane == 16) sc[2 * kBlock + wave] = big;
    }
  };

  // chunk G kk + g of token `row`; swizzled chunks kk and kk + 4 are 256 bytes apart
  constexpr int KP = MT == 32 ? 1 : 4;
  const unsigned char* kget[KP];
#pragma unroll
  for (int kk = 0; kk < KP; ++kk) kget[kk] = smem + row * S::KROW + 16 * ((G * kk + grp) ^ kswz(row));
  const unsigned char* const vget = smem + S::V + (4 * grp + (n16 >> 2)) * S::VROW + 8 * (n16 & 3) +
                                    (MT == 32 ? 32 * ((lane >> 4) & 1) : 0);
  const float* const sget = reinterpret_cast<const float*>(smem + S::SCALES) + 4 * grp;
  RowState st;
  Sum acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = Sum{};

  auto compute = [&](auto bufc, int t0, uint32_t pages_ok) {
    constexpr int at = decltype(bufc)::value * S::BUF;
    Sum sc[NT];
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      sc[tt] = Sum{};
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const unsigned char* kp = kget[kk % KP] + at + tt * MT * S::KROW + 16 * G * KP * (kk / KP);
        sc[tt] = tile_mfma(*reinterpret_cast<const u32x4_t*>(kp), qb[kk], sc[tt]);
      }
    }
    const float* scl = sget + at / 4;
    float vsc[N], s[N];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(scl + G * i);
      const f32x4_t v4 = *reinterpret_cast<const f32x4_t*>(scl + kBlock + G * i);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vsc[i + r] = v4[r];
        s[i + r] = sc[i / NV][i % NV + r] * k4[r];
      }
    }
    const float* big = reinterpret_cast<const float*>(smem + at + S::SCALES) + 2 * kBlock;
    float size = big[0];
#pragma unroll
    for (int i = 1; i < Q; ++i) size = fmaxf(size, big[i]);
    if (__builtin_expect(t0 + kBlock > all || pages_ok != (1u << Q) - 1 || size > 65504.0f, 0)) {
      uint32_t ok = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int t = 4 * G * (i >> 2) + 4 * grp + (i & 3);
        ok |= (uint32_t)(t0 + t <= lim && ((pages_ok >> (t / 16)) & 1u)) << i;
      }
      size = hide<N, G>(__float_as_uint(pinned(__uint_as_float(ok))), s, vsc);
    }
    u32x4_t w[N / 8];
    bool up;
    const float alpha = row_block<N, G>(st, s, mul, vsc, size, w, up);
    if (__builtin_expect(__ballot(up) != 0, 0)) {
      const float f = pinned(up ? alpha : 1.0f);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < N / 8; ++k)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const unsigned char* vp = vget + at + 8 * G * k * S::VROW + 2 * MT * j;
        const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(vp)));
        const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(vp + 4 * G * S::VROW)));
        acc[j] = tile_mfma(u32x4_t{lo.x, lo.y, hi.x, hi.y}, w[k], acc[j]);
      }
  };

  if (ib0 < ib1) {
    BlockPages<Q> bp = block_pages<Q>(a, trow, kBlock * ib0);
    uint32_t ok_now = bp.ok, ok_next;
    load(ib0, bp);
    bp = block_pages<Q>(a, trow, kBlock * min(ib0 + 1, last));
    stage(std::integral_constant<int, 0>{});
    load(ib0 + 1, bp);
    ok_next = bp.ok;
    __syncthreads();
    auto step = [&](int ib, auto cur) {
      const BlockPages<Q> after = block_pages<Q>(a, trow, kBlock * min(ib + 2, last));
      if (wr0 < it.rows) compute(cur, kBlock * ib, ok_now);
      stage(std::integral_constant<int, 1 - decltype(cur)::value>{});
      load(ib + 2, after);
      ok_now = ok_next;
      ok_next = after.ok;
      __syncthreads();
    };
    int ib = ib0;
    for (; ib + 2 <= ib1; ib += 2) {
      step(ib, std::integral_constant<int, 0>{});
      step(ib + 1, std::integral_constant<int, 1>{});
    }
    if (ib < ib1 && wr0 < it.rows) compute(std::integral_constant<int, 0>{}, kBlock * ib, ok_now);
  }

  const float z = sum_groups<G>(st.z);
  const int r = MT * wave + row;
  if (r >= rows) return;
  if (it.parts == 1) {
    const int64_t at = out_row(a, it, kh, rw0 + r, gqa) * D;
    const float inv = z != 0.0f ? 1.0f / z : 1.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < NV; v += 4)
        store_row4(a, at + MT * j + G * v + 4 * grp,
                   f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]} * inv);
  } else {
    const int64_t at = ((int64_t)kh * a.slots + it.slot + it.part) * R + r;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < NV; v += 4)
        *reinterpret_cast<f32x4_t*>(a.pacc + at * D + MT * j + G * v + 4 * grp) =
            f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]};
    if (grp == 0) {
      a.pm[at] = part_max(st, z);
      a.pz[at] = z;
    }
  }
}

// Joins the parts of split contexts: workgroup (x, kh) takes 16 rows of a split
// tile. A wave per row finds the parts' weights (a lane each, one round trip);
// then a thread sums four dims of a row over every `ways`-th part, eight loads
// in flight, and the ways are summed through LDS.
constexpr int kMaxParts = 512;
template <int D, int R>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedSdpaArgs a) {
  constexpr int GROUPS = R / 16, D4 = D / 4;
  __shared__ float wts[16][kMaxParts];
  __shared__ f32x4_t sums[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kh = blockIdx.x % a.Hkv, x = blockIdx.x / a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<R, true>(a, x / GROUPS);
  if (it.b < 0) return;
  const int r0 = 16 * (x % GROUPS);
  const int rows = min(it.rows - R * it.tile - r0, 16), parts = it.parts;
  const int64_t base = ((int64_t)kh * a.slots + it.slot) * R + r0;
  for (int r = wave; r < rows; r += 4) {
    float mm = kNegInf, z = 0.0f;
    for (int k = lane; k < parts; k += 64) {
      const float m = a.pm[base + (int64_t)k * R + r];
      wts[r][k] = m;
      mm = fmaxf(mm, m);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    for (int k = lane; k < parts; k += 64) {
      const float m = wts[r][k];
      const float f = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
      const float pz = a.pz[base + (int64_t)k * R + r];
      z = m == kNegInf ? z : fmaf(pz, f, z);
      wts[r][k] = f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o);
    const float inv = z != 0.0f ? 1.0f / z : 0.0f;
    for (int k = lane; k < parts; k += 64) wts[r][k] *= inv;
  }
  __syncthreads();
  // as many ways over the parts as the threads allow: a power of two
  const int items = rows * D4;
  int ways = 1;
  while (2 * ways * items <= 256 && 2 * ways <= parts) ways *= 2;
  const int per = 256 / ways, way = tid / per;
  for (int i0 = 0; i0 < items; i0 += per) {
    const int i = i0 + tid % per;
    const int r = min(i, items - 1) / D4, d = 4 * (min(i, items - 1) % D4);
    const float* p = a.pacc + (base + r) * D + d;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = way; k0 < parts; k0 += 8 * ways) {
      f32x4_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = *reinterpret_cast<const f32x4_t*>(p + (int64_t)min(k0 + u * ways, parts - 1) * R * D);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = wts[r][min(k0 + u * ways, parts - 1)];
        if (k0 + u * ways < parts && f != 0.0f) o += v[u] * f;
      }
    }
    if (ways > 1) {
      __syncthreads();
      sums[tid] = o;
      __syncthreads();
      if (way == 0)
        for (int w = 1; w < ways; ++w) o += sums[tid + w * per];
    }
    if (way == 0 && i < items) store_row4(a, out_row(a, it, kh, R * it.tile + r0 + r, gqa) * D + d, o);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct PagedPlan {
  bool few;
  int rows;           // of a tile
  int64_t max_tiles;  // of the whole batch, at most
  int64_t target, slots, split;  // parts to aim at, parts and tiles of split contexts at most
  int min_part;
};

PagedPlan paged_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                     int64_t max_tokens) {
  PagedPlan p;
  const int64_t gqa = Hq / Hkv;
  max_new = std::min(max_new, T);
  p.few = max_new * gqa <= 16;
  p.rows = p.few ? 16 : D <= 128 ? TileShape<128>::ROWS : TileShape<256>::ROWS;
  p.min_part = 128;
  p.max_tiles = std::min(T * gqa / p.rows + B, B * cdiv(max_new * gqa, p.rows));
  p.target = std::min<int64_t>(cdiv((p.few ? 4 : 2) * device_cus(), Hkv), kMaxParts);
  p.split = max_tokens > p.min_part ? std::min(p.max_tiles, p.target) : 0;
  p.slots = std::min(2 * p.target, p.split * cdiv(max_tokens, p.min_part));
  return p;
}

template <int D>
void launch_paged(const PagedSdpaArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.slots + p.max_tiles) * a.Hkv));  // of an unsplit tile or a part each
  const dim3 merge((unsigned)(p.split * (p.rows / 16) * a.Hkv));
  if (p.few)
    hipLaunchKernelGGL(paged_few_kernel<D>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(paged_tile_kernel<D>, grid, dim3(256), 0, st, a);
  if (merge.x == 0) return;
  if (p.few)
    hipLaunchKernelGGL((paged_merge_kernel<D, 16>), merge, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, TileShape<D>::ROWS>), merge, dim3(256), 0, st, a);
}

}  // namespace

// Parts of split contexts: their outputs, then maxima and sums.
size_t paged_sdpa_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                            int64_t max_tokens) {
  const PagedPlan p = paged_plan(T, B, Hq, Hkv, D, max_new, max_tokens);
  return (size_t)(Hkv * p.slots * p.rows * (D + 2)) * sizeof(float);
}

int paged_sdpa(const PagedBatch& p, const void* q, const int64_t* qst, const PagedSide& ks,
               const PagedSide& vs, void* out, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
               int causal, int qdt, int odt, float scale, void* ws, size_t wsb, hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  const int64_t max_tokens = (int64_t)p.width << p.page_log2;
  const PagedPlan plan = paged_plan(p.T, p.B, Hq, Hkv, D, max_new, max_tokens);
  const size_t need = paged_sdpa_workspace(p.T, p.B, Hq, Hkv, D, max_new, max_tokens);
  if (need > 0 && (!ws || wsb < need))
    return set_error(SPARKQ_ERR_WORKSPACE, "paged_sdpa needs a workspace of %zu bytes (got %zu)", need,
                     ws ? wsb : (size_t)0);
  if (!aligned(ws, 16)) return set_error(SPARKQ_ERR_INVALID, "paged_sdpa: workspace must be 16-byte aligned");
  const int64_t n = Hkv * plan.slots * plan.rows;
  float* acc = (float*)ws;
  const CodeLayout c{ks.codes, vs.codes, ks.scales, vs.scales, ks.c_head, ks.s_head, (uint32_t)(ks.c_page / 16),
                     (uint32_t)(ks.s_page / 8), (uint32_t)ks.c_tok};
  const PagedSdpaArgs a{p, (const uint16_t*)q, qst[0], qst[1], c, out, acc + n * D, acc + n * (D + 1), acc,
                        (int)Hq, (int)Hkv, (int)std::min<int64_t>(max_new, p.T), causal, qdt, odt,
                        (int)plan.target, (int)plan.slots, plan.min_part, scale * 1.44269504088896340736f};
  if (D == 64)
    launch_paged<64>(a, plan, st);
  else if (D == 128)
    launch_paged<128>(a, plan, st);
  else
    launch_paged<256>(a, plan, st);
  return check_launch("paged_sdpa");
}

}  // namespace sparkq
