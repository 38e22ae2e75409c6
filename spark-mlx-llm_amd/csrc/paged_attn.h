// paged_attn.h -- what the attention kernels over a paged INT8 KV cache share:
// their arguments, whose work is whose, operands of the matrix instructions and
// the online softmax of a block.
#pragma once

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
  void* out;   // [T, Hq, D]
  float* lse;  // [T, Hq] logarithms of the rows' sums, or null
  float *pm, *pz, *pacc;  // [Hkv][slots][rows], [...], [...][D]: parts of split contexts
  int Hq, Hkv, max_new, causal, q_dtype, out_dtype;
  int target;      // parts of the whole batch, about, per KV head
  int slots;       // parts of split contexts, at most, per KV head
  int min_part;    // tokens of a part, at least
  int snake;       // items that the chip's CUs take a round of, per KV head (0: in order)
  float scale_log2, sign;  // size (log2 units) and sign of the softmax scale
};

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

constexpr int kFewBlock = 32;    // tokens of a block
constexpr int kTileRows = 128;  // rows of a tile

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

template <int R>  // rows of a tile
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
// by.) All lanes of a wave take part, and every wave gets the same answers: no
// counters, and no launch before this one (two round trips to L2, about 1.5 us).
template <int R, bool SPLIT>
__device__ __forceinline__ Item find_item(const PagedSdpaArgs& a, int x) {
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

// two values rounded (to nearest even) into packed fp16: one instruction
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_t));
}

// A row's query values as exact fp16: chunk c of this lane holds dims dim0(c) ..
// +8. bf16 rows are shifted by a power of two for that; returns the factor that
// undoes it, times the softmax scale: what takes the row's sums times the key scales
// to log2 units. (Scaled sooner, rows of the smallest queries could pass fp32's
// range; where it ends under 2^-126, every score is next to 0, and stays so. What
// bf16 can hold below 2^-28 of the row's largest is rounded.)
template <int NK, int G, typename F>
__device__ __forceinline__ float load_query(const PagedSdpaArgs& a, const uint16_t* row, bool live, F dim0,
                                            u32x4_t qb[NK]) {
#pragma unroll
  for (int c = 0; c < NK; ++c) {
    qb[c] = *reinterpret_cast<const u32x4_t*>(row + dim0(c));
    if (!live) qb[c] = u32x4_t{0, 0, 0, 0};
  }
  if (a.q_dtype == SPARKQ_F16) return fmaxf(a.scale_log2, 0x1p-126f);
  u16x2_t most = {0, 0};
#pragma unroll
  for (int c = 0; c < NK; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, qb[c][i] & 0x7FFF7FFFu));
  const float top = max_groups<G>(bf16_to_f32(most[0] > most[1] ? most[0] : most[1]));
  const int e = top > 0.0f && top <= 3.4028235e38f ? ilogbf(top) - 14 : 0;
#pragma unroll
  for (int c = 0; c < NK; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qb[c][i] = pack_f16(ldexpf(lo16<BF16>(qb[c][i]), -e), ldexpf(hi16<BF16>(qb[c][i]), -e));
  return fmaxf(ldexpf(a.scale_log2, e), 0x1p-126f);
}

// v, in a way that what depends on it stays in its branch: the compiler would
// otherwise rescale the sums of every block and select, at twice the registers
__device__ __forceinline__ float pinned(float v) {
  asm volatile("" : "+v"(v));
  return v;
}

// ---------------------------------------------------------------------------
// online softmax of one block for one row per lane
// ---------------------------------------------------------------------------
// The state counts in units of 2^(t - TOP), t the largest score (log2 units) plus
// exponent of the value's scale (2^e <= scale < 2^(e+1)) when it last moved: with
// TOP = kTopFew or kTopTile, and ROOM for t to be exceeded by, weights stay under
// 2^15.
struct RowState {
  float t = kNegInf;  // -inf: nothing seen
  float z = 0.0f;
};
constexpr int kTopFew = 13, kTopTile = 6;

template <int TOP>
__device__ __forceinline__ float unit(const RowState& st) { return st.t - (float)TOP; }

// The exponent of a value scale's size; no less than -60 (fp16 ends at -24: 0 is
// meant), so that a row whose best token has no value keeps a finite normalizer, and no
// more than 16 (fp16 ends at 15: what is not finite is meant), so that the scores of
// the other tokens still count in it.
__device__ __forceinline__ float scale_exp(float v) {
  return (float)min(max((int)(__float_as_uint(v) >> 23 & 255u), 127 - 60), 127 + 16) - 127.0f;
}

// What a part of a row's context hands on: its unit, or -inf where it saw nothing
// (scores that are all NaN leave no maximum, but a sum that is not 0). Its sums are NaN
// where it saw a value that is not finite, and count whatever their weight: 0 times NaN
// is NaN.
template <int TOP>
__device__ __forceinline__ float part_max(const RowState& st, float z) {
  return st.t != kNegInf ? unit<TOP>(st) : (z != 0.0f ? 0.0f : kNegInf);
}

// A block's N scores of this lane's row (raw sums times the key scales and the
// softmax scale's sign: s * mul is in log2 units; -inf where hidden), `t` the largest
// score plus scale exponent of those that are visible, or up to log2(kSpread) more.
// The state's moves where it is exceeded by more than ROOM: 0 with
// few rows; in tiles, whose sums are dear to scale, 8. Writes the packed fp16 weights
// of the lane's N values (with TWO also what their rounding left of them); returns
// the factor for what is summed so far (up: it is not 1).
template <int N, int TOP, int ROOM, bool TWO>
__device__ __forceinline__ float row_block(RowState& st, const float s[N], float mul, const float vsc[N], float t,
                                           u32x4_t w[N / 8], u32x4_t rest[N / 8], bool& up) {
  up = t > st.t + ROOM;
  const float old = unit<TOP>(st);
  if (up) st.t = t;
  const float M = st.t == kNegInf ? 0.0f : unit<TOP>(st);
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
  for (int i = 0; i < N; i += 2) {
    const uint32_t h = pack_f16(p[i], p[i + 1]);
    w[i / 8][i / 2 % 4] = h;
    if (TWO) rest[i / 8][i / 2 % 4] = pack_f16(p[i] - lo16<F16>(h), p[i + 1] - hi16<F16>(h));
  }
  return alpha;
}

// A value scale as the tile kernel keeps it: what is not finite is -0, so that a
// hidden token's weight of 0 times its scale is 0, and a visible one is found.
__device__ __forceinline__ float kept_scale(float v) {
  return fabsf(v) <= 65504.0f ? v + 0.0f : -0.0f;
}

// The largest and least value scale of 16 tokens, for blocks that are taken whole
// (no row hides any of them, and one exponent stands for all). A scale that is not
// finite makes the largest infinite and the least 0.
__device__ __forceinline__ float most_of(float v) {
  return max_row16(fabsf(v) <= 65504.0f ? fabsf(v) : __builtin_huge_valf());
}
__device__ __forceinline__ float least_of(float v) { return -max_row16(-fabsf(kept_scale(v))); }
constexpr float kSpread = 16.0f;  // of the largest to the least that one exponent stands for

// Hides the scores that are not in `ok`; returns the largest score plus scale exponent
// of those that are visible. `odd` is NaN where the row sees a value that is not finite,
// and takes its sums with it, but not its normalizer.
template <int N, int G>
__device__ __forceinline__ float hide(uint32_t ok, float s[N], float mul, const float vsc[N], float& odd) {
  float t = kNegInf;
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool live = (ok >> i) & 1u;
    s[i] = live ? s[i] : kNegInf;
    t = fmaxf(t, fmaf(s[i], mul, scale_exp(vsc[i])));
    bad |= live ? (uint32_t)(__float_as_uint(vsc[i]) == 0x80000000u) : 0u;
  }
  odd = sum_groups<G>(bad ? __builtin_nanf("") : 0.0f);
  return max_groups<G>(t);
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

// The logarithm of a row's sum of exponentiated scores, from its unit and its
// normalizer in that unit.
__device__ __forceinline__ float row_lse(float unit, float z) {
  return z != 0.0f ? (unit + log2f(z)) * 0.69314718055994530942f : kNegInf;
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

// Which of TOK (16 or 32) tokens have value codes of nothing but 0, a bit each, `p`
// being a lane's share of token lane % TOK's: 16 PIECES bytes. Such a row is stored
// with scale 1, which says nothing of its size: it would take the unit away from
// values that are small beside 1, so its scale is taken for 0. Called where a scale
// is 1, which is rare: the codes are read again, 64 / TOK lanes a token.
template <int D, int TOK>
__device__ __forceinline__ uint32_t zero_rows(const uint8_t* p) {
  constexpr int LPT = 64 / TOK, PIECES = D / 16 / LPT;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p + 16 * i);
    any |= x.x | x.y | x.z | x.w;
  }
  uint64_t zero = __ballot(any == 0);
#pragma unroll
  for (int n = 32; n >= TOK; n /= 2) zero &= zero >> n;
  return (uint32_t)zero & (uint32_t)((1ull << TOK) - 1);
}
// of a sequence's tokens from t0 on
template <int D, int TOK>
__device__ __forceinline__ uint32_t zero_values(const PagedSdpaArgs& a, TableRow row, const uint8_t* vhead, int t0) {
  constexpr int LPT = 64 / TOK, PIECES = D / 16 / LPT;
  const int lane = threadIdx.x & 63, t = t0 + lane % TOK;
  const int id = row[min(t >> a.p.page_log2, a.p.width - 1)];
  return zero_rows<D, TOK>(vhead + code_at(a.c, (unsigned)id < (unsigned)a.p.pages ? id : 0, t & ((1 << a.p.page_log2) - 1)) +
                           16 * PIECES * (lane / TOK));
}

}  // namespace
}  // namespace sparkq
