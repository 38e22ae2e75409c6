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
//   paged_tile_kernel  tiles of 128 rows, 32 a wave: a block is turned to fp16
//                      in LDS once for all of them.
//   paged_merge_kernel joins the parts of a context that was split.
//
// Work. The lengths live on the device, so every workgroup works out from the
// batch's starts and lengths which (sequence, tile, part of the context) is
// its own (find_item): a context is split so that about `slots` parts of equal
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

struct PagedSdpaArgs {
  PagedBatch p;
  const uint16_t* q;
  int64_t q_tok, q_head;  // elements
  PagedSide ks, vs;
  void* out;  // [T, Hq, D]
  float *pm, *pz, *pacc;  // [Hkv][slots][rows], [...], [...][D]: parts of split contexts
  int Hq, Hkv, max_new, causal, q_dtype, out_dtype;
  int slots;       // parts of split contexts, at most, per KV head
  int min_blocks;  // blocks of a part, at least
  float scale_log2;
};

constexpr int kBlock = 32;  // tokens of a block

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
  int first, count, length, rows, tiles, blocks;
};

template <int R>
__device__ __forceinline__ SeqWork seq_work(const PagedSdpaArgs& a, int b) {
  SeqWork w{0, 0, 0, 0, 0, 0};
  if (b < a.p.B) {
    const SeqRows s = seq_rows(a.p, b);
    w.first = s.first;
    w.count = s.count;
    w.length = s.length;
    w.rows = min(s.count, a.max_new) * (a.Hq / a.Hkv);
    w.tiles = (w.rows + R - 1) / R;
    w.blocks = (s.length + kBlock - 1) / kBlock;
  }
  return w;
}

__device__ __forceinline__ int wave_prefix(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Item x of the batch's items in order (SPLIT false: every tile and part), or
// tile x of those whose context is split. A context of n blocks is split into
// floor(n / C) parts, C = max(min_blocks, ceil(all tiles' blocks / slots)), so
// split contexts have no more than `slots` parts together. All lanes of a wave
// take part and get the same answer.
template <int R, bool SPLIT>
__device__ Item find_item(const PagedSdpaArgs& a, int x) {
  const int lane = threadIdx.x & 63;
  long long all = 0;
  for (int b0 = 0; b0 < a.p.B; b0 += 64) {
    const SeqWork w = seq_work<R>(a, b0 + lane);
    all += (long long)w.tiles * w.blocks;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
  const long long C = max((all + a.slots - 1) / a.slots, (long long)a.min_blocks);
  Item it{-1, 0, 0, 1, 0, 0, 0, 0, 0};
  int items = 0, slots = 0;
  for (int b0 = 0; b0 < a.p.B; b0 += 64) {
    const SeqWork w = seq_work<R>(a, b0 + lane);
    const int parts = max(1, (int)(w.blocks / C));
    const int own = SPLIT ? (parts > 1 ? w.tiles : 0) : w.tiles * parts;
    const int used = parts > 1 ? w.tiles * parts : 0;
    const int end = items + wave_prefix(own, lane), slot_end = slots + wave_prefix(used, lane);
    const unsigned long long hit = __ballot(x < end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      it.b = b0 + l;
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
      return it;
    }
    items = __builtin_amdgcn_readlane(end, 63);
    slots = __builtin_amdgcn_readlane(slot_end, 63);
  }
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

// A row's query values as exact fp16 under a power of two: chunk c of lane
// group g holds dims dim0(c) .. +8. The row's lanes are l, l^16, l^32, l^48.
// Returns the factor that undoes the shift.
template <int NK, typename F>
__device__ __forceinline__ float load_query(const PagedSdpaArgs& a, const uint16_t* row, bool live, F dim0,
                                            u32x4_t qb[NK]) {
  float qv[NK][8], top = 0.0f;
#pragma unroll
  for (int c = 0; c < NK; ++c) {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + dim0(c));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t bits = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      qv[c][i] = live ? (a.q_dtype == SPARKQ_BF16 ? bf16_to_f32(bits) : f16_to_f32(bits)) : 0.0f;
      top = fmaxf(top, fabsf(qv[c][i]));
    }
  }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const int e = top > 0.0f && top <= 3.4028235e38f ? ilogbf(top) - 14 : 0;
#pragma unroll
  for (int c = 0; c < NK; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qb[c][i] = pack_round<F16>(ldexpf(qv[c][2 * i], -e), ldexpf(qv[c][2 * i + 1], -e));
  return ldexpf(1.0f, e);
}

// max / sum over the four 16-lane rows of a wave, the same value in all of them
__device__ __forceinline__ float max_groups(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
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

// The block's 8 scores of this lane's row (raw sums times the key scales times
// the softmax scale: s * mul is in log2 units), `ok` where visible; `size` is
// the block's largest finite value scale, used where all of it is visible.
// Writes the packed fp16 weights of its 8 values; returns the factor for what
// is summed so far (up: it is not 1).
template <bool MASK>
__device__ __forceinline__ float row_block(RowState& st, const float s[8], const bool ok[8], float mul,
                                           const float vsc[8], float size, u32x4_t& w, bool& up) {
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, MASK ? (ok[i] ? s[i] : kNegInf) : s[i]);
  top = max_groups(top) * mul;
  if (MASK) {
    size = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) size = fmaxf(size, scale_size(vsc[i], ok[i]));
    size = max_groups(size);
  }
  const float e = fmaxf(st.e, (float)((int)(__float_as_uint(size) >> 23) - 127));
  const bool raise = top > st.m + kRoom;
  up = raise || e != st.e;
  const float old = unit(st);
  if (raise) st.m = ceilf(top);
  st.e = e;
  const float M = st.m == kNegInf ? 0.0f : unit(st);
  const float alpha = old == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(old - M);
  float p[8], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], mul, -M));
    if (MASK) p[i] = ok[i] ? p[i] : 0.0f;
    sum += p[i];
    p[i] *= vsc[i];
    if (MASK) p[i] = ok[i] ? p[i] : 0.0f;
  }
  st.z = fmaf(st.z, up ? alpha : 1.0f, sum);
  w = u32x4_t{pack_round<F16>(p[0], p[1]), pack_round<F16>(p[2], p[3]), pack_round<F16>(p[4], p[5]),
              pack_round<F16>(p[6], p[7])};
  return alpha;
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

// Pages of a block's two 16-token halves; a half without one reads page 0 and
// is hidden. Past the table's row the last entry stands in (those tokens lie
// past every length).
struct BlockPages {
  int id[2];
  bool ok[2];
};
__device__ __forceinline__ BlockPages block_pages(const PagedSdpaArgs& a, const int32_t* row, int t0) {
  BlockPages r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int id = row[min((t0 + 16 * h) >> a.p.page_log2, a.p.width - 1)];
    r.ok[h] = (unsigned)id < (unsigned)a.p.pages;
    r.id[h] = r.ok[h] ? id : 0;
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
  static constexpr int VT = kBlock * VROW;          // one wave's V block
  static constexpr int LOOP = 4 * VT;
  static constexpr int JOIN = 4 * 16 * (2 + D) * 4;  // the waves' maxima, sums and outputs
  static constexpr int BYTES = LOOP > JOIN ? LOOP : JOIN;
};

template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void paged_few_kernel(PagedSdpaArgs a) {
  constexpr int NK = D / 32, PL = D / 64, NJ = D / 16, VL = D / 32;
  using L = FewLds<D>;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, grp = lane >> 4;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<16, false>(a, blockIdx.x / a.Hkv);
  if (it.b < 0) return;
  const int rows = min(it.rows - 16 * it.tile, 16);
  const int rr = 16 * it.tile + min(n16, rows - 1);
  const int lim = last_seen(a, it, rr, gqa);
  const int seen = last_seen(a, it, 16 * it.tile + rows - 1, gqa) + 1;  // by the last row: the most
  const int all = last_seen(a, it, 16 * it.tile, gqa) + 1;              // by every row
  const int nblocks = (seen + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const int32_t* trow = a.p.table + it.b * a.p.table_stride;
  unsigned char* vtile = smem + wave * L::VT;

  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + (it.first + rr / gqa) * a.q_tok + (kh * gqa + rr % gqa) * a.q_head;
  // chunk c: dims 16 (g + 4 (c / 2)) + 8 (c % 2), as the 16-byte pieces of K lie
  const float mul = load_query<NK>(a, qrow, true, [&](int c) { return 16 * (grp + 4 * (c >> 1)) + 8 * (c & 1); }, qb);

  u32x4_t kr[2][2][PL], vr[2][VL], skr[2], svr[2];
  BlockPages pg[2], next;
  const int ktok = 8 * (n16 >> 2) + (n16 & 3);
  const int slot_mask = (1 << a.p.page_log2) - 1;
  const int last = ib1 - 1;
  // block ib (no further than the last) through the pages found for it
  auto load = [&](int set, int ib, const BlockPages& bp) {
    const int t0 = kBlock * min(ib, last);
    const int s0 = t0 & slot_mask, s1 = (t0 + 16) & slot_mask;
    auto base = [&](const PagedSide& s, int h) {
      return s.codes + bp.id[h] * s.c_page + kh * s.c_head + (h ? s1 : s0) * s.c_tok;
    };
    const uint8_t *k0 = base(a.ks, 0), *k1 = base(a.ks, 1), *v0 = base(a.vs, 0), *v1 = base(a.vs, 1);
    const uint8_t* kp = (n16 < 8 ? k0 : k1) + (ktok & 15) * a.ks.c_tok;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < PL; ++i)
        kr[set][t][i] = *reinterpret_cast<const u32x4_t*>(kp + 4 * t * a.ks.c_tok + 16 * (grp + 4 * i));
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      vr[set][v] = *reinterpret_cast<const u32x4_t*>((2 * v >= VL ? v1 : v0) + (tok & 15) * a.vs.c_tok + 16 * pc);
    }
    auto scales = [&](const PagedSide& s) {
      const int h = grp >> 1;
      const uint16_t* p = s.scales + (h ? bp.id[1] : bp.id[0]) * s.s_page + kh * s.s_head + (h ? s1 : s0) + 8 * (grp & 1);
      return *reinterpret_cast<const u32x4_t*>(p);
    };
    skr[set] = scales(a.ks);
    svr[set] = scales(a.vs);
    pg[set] = bp;
  };

  RowState st;
  f32x4_t acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto block = [&](int ib, auto setc) {
    constexpr int set = decltype(setc)::value;
    const int t0 = kBlock * ib;
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      *reinterpret_cast<u32x4_t*>(vtile + tok * L::VROW + 16 * pc) = vr[set][v];
    }
    f32x4_t sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const u32x4_t kp = kr[set][t][c >> 1];
        sc[t] = mfma16x16x32_f16((c & 1) ? s8x8_exact(kp.z, kp.w) : s8x8_exact(kp.x, kp.y), qb[c], sc[t]);
      }
    }
    float s[8], vsc[8];
    bool ok[8];
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kw = skr[set][i >> 1], vw = svr[set][i >> 1];
      s[i] = sc[i >> 2][i & 3] * (((i & 1) ? hi16<F16>(kw) : lo16<F16>(kw)) * a.scale_log2);
      vsc[i] = (i & 1) ? hi16<F16>(vw) : lo16<F16>(vw);
    }
    const bool half_ok[2] = {pg[set].ok[0], pg[set].ok[1]};
    const bool whole = t0 + kBlock <= all && half_ok[0] && half_ok[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ok[i] = whole || (t0 + 8 * grp + i <= lim && (grp < 2 ? half_ok[0] : half_ok[1]));
      big = fmaxf(big, scale_size(vsc[i], true));
    }
    load(set, ib + 8, next);
    next = block_pages(a, trow, kBlock * min(ib + 12, last));
    u32x4_t w;
    bool up;
    const float alpha = whole ? row_block<false>(st, s, ok, mul, vsc, max_groups(big), w, up)
                              : row_block<true>(st, s, ok, mul, vsc, 0.0f, w, up);
    if (__ballot(up)) {
      const float f = up ? alpha : 1.0f;
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
    load(0, ib, block_pages(a, trow, kBlock * ib));
    load(1, ib + 4, block_pages(a, trow, kBlock * min(ib + 4, last)));
    next = block_pages(a, trow, kBlock * min(ib + 8, last));
    for (; ib + 4 < ib1; ib += 8) {
      block(ib, std::integral_constant<int, 0>{});
      block(ib + 4, std::integral_constant<int, 1>{});
    }
    if (ib < ib1) block(ib, std::integral_constant<int, 0>{});
  }

  // combine the waves
  const float z = sum_groups(st.z);
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
// tiles of 128 rows
// ---------------------------------------------------------------------------
// The products run as above with 2 x 16 rows a wave; the lane with a row's
// scores of tokens 16 t + 4 g + r holds those k-slots. A block of codes is read
// once by the workgroup and written to LDS as fp16, K token-major with its
// 16-byte chunks XOR-swizzled by the token, V token-major with its 32-byte runs
// swizzled (read transposed), two buffers deep: the next block's codes are
// converted while this one is computed, and the one after is in flight.
template <int D>
struct TileLds {
  static constexpr int ROW = 2 * D;
  static constexpr int TILE = kBlock * ROW;
  static constexpr int BUF = 2 * TILE + 2 * kBlock * 4 + 16;  // K, V, key and value scales, the largest of these
  static constexpr int BYTES = 2 * BUF;
};
template <int D>
__device__ __forceinline__ int kswz(int t) { return D >= 128 ? (t & 15) : ((t >> 1) & 7); }
template <int D>
__device__ __forceinline__ int vswz(int t) { return D >= 128 ? (t & 7) : ((t >> 1) & 3); }

template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void paged_tile_kernel(PagedSdpaArgs a) {
  using L = TileLds<D>;
  constexpr int NK = D / 32, NJ = D / 16;
  constexpr int PIECES = 2 * D;  // 16-code pieces of a K (or V) block
  constexpr int PPT = PIECES >= 256 ? PIECES / 256 : 1;
  constexpr int NVB = NJ < 8 ? NJ : 8;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, grp = lane >> 4;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<128, false>(a, blockIdx.x / a.Hkv);
  if (it.b < 0) return;
  const int rw0 = 128 * it.tile;
  const int rows = min(it.rows - rw0, 128);
  const int seen = last_seen(a, it, rw0 + rows - 1, gqa) + 1;
  const int nblocks = (seen + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const int32_t* trow = a.p.table + it.b * a.p.table_stride;

  u32x4_t qb[2][NK];
  int lim[2];
  float mul[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int rr = rw0 + 32 * wave + 16 * rt + n16, rq = min(rr, it.rows - 1);
    lim[rt] = last_seen(a, it, rr, gqa);
    const uint16_t* qrow = a.q + (it.first + rq / gqa) * a.q_tok + (kh * gqa + rq % gqa) * a.q_head;
    mul[rt] = load_query<NK>(a, qrow, rr < it.rows, [&](int c) { return 32 * c + 8 * grp; }, qb[rt]);
  }
  // what every row of the wave sees, and what its last one does
  const int wr0 = rw0 + 32 * wave;
  const int all = last_seen(a, it, wr0, gqa) + 1 > 0 && wr0 + 31 < it.rows ? last_seen(a, it, wr0, gqa) + 1 : 0;
  const int most = wr0 < it.rows ? last_seen(a, it, min(wr0 + 31, it.rows - 1), gqa) + 1 : 0;

  const int slot_mask = (1 << a.p.page_log2) - 1;
  const bool stager = PIECES >= 256 || tid < PIECES;  // wave-uniform
  u32x4_t kcr[PPT], vcr[PPT];
  uint16_t sr;
  const int last = ib1 - 1;
  // piece p = tid + 256 i: token p / (D / 16), codes 16 (p % (D / 16)); thread
  // t < 64 also takes a scale: key t, or value t - 32
  auto load = [&](int ib, const BlockPages& bp) {
    const int t0 = kBlock * min(ib, last);
    const int s0 = t0 & slot_mask, s1 = (t0 + 16) & slot_mask;
    if (stager) {
#pragma unroll
      for (int i = 0; i < PPT; ++i) {
        const int p = tid + 256 * i, tk = p / (D / 16), jb = p % (D / 16), h = tk >> 4;
        const int64_t id = h ? bp.id[1] : bp.id[0];
        const int64_t slot = (h ? s1 : s0) + (tk & 15);
        kcr[i] = *reinterpret_cast<const u32x4_t*>(a.ks.codes + id * a.ks.c_page + kh * a.ks.c_head + slot * a.ks.c_tok + 16 * jb);
        vcr[i] = *reinterpret_cast<const u32x4_t*>(a.vs.codes + id * a.vs.c_page + kh * a.vs.c_head + slot * a.vs.c_tok + 16 * jb);
      }
    }
    if (wave == 0) {
      const PagedSide& s = lane < 32 ? a.ks : a.vs;
      const int h = (lane >> 4) & 1;
      sr = s.scales[(h ? bp.id[1] : bp.id[0]) * s.s_page + kh * s.s_head + (h ? s1 : s0) + (lane & 15)];
    }
  };
  auto stage = [&](unsigned char* buf) {
    if (stager) {
#pragma unroll
      for (int i = 0; i < PPT; ++i) {
        const int p = tid + 256 * i, tk = p / (D / 16), jb = p % (D / 16), ks = kswz<D>(tk);
        unsigned char* kt = buf + tk * L::ROW;
        *reinterpret_cast<u32x4_t*>(kt + ((2 * jb) ^ ks) * 16) = s8x8_exact(kcr[i].x, kcr[i].y);
        *reinterpret_cast<u32x4_t*>(kt + ((2 * jb + 1) ^ ks) * 16) = s8x8_exact(kcr[i].z, kcr[i].w);
        unsigned char* vt = buf + L::TILE + tk * L::ROW + (jb ^ vswz<D>(tk)) * 32;
        *reinterpret_cast<u32x4_t*>(vt) = s8x8_exact(vcr[i].x, vcr[i].y);
        *reinterpret_cast<u32x4_t*>(vt + 16) = s8x8_exact(vcr[i].z, vcr[i].w);
      }
    }
    if (wave == 0) {
      float* sc = reinterpret_cast<float*>(buf + 2 * L::TILE);
      const float v = f16_to_f32(sr);
      sc[lane] = lane < 32 ? v * a.scale_log2 : v;
      const float big = max_groups(max_row16(scale_size(v, lane >= 32)));
      if (lane == 0) sc[64] = big;
    }
  };

  int ka[NK], va[NVB];
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) ka[kk] = n16 * L::ROW + ((4 * kk + grp) ^ kswz<D>(n16)) * 16;
  {
    const int tv = 4 * grp + (n16 >> 2), sw = vswz<D>(tv);
#pragma unroll
    for (int v = 0; v < NVB; ++v) va[v] = L::TILE + tv * L::ROW + ((v ^ sw) * 32) + 8 * (n16 & 3);
  }
  RowState st[2];
  f32x4_t acc[2][NJ];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[rt][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](const unsigned char* buf, int t0, bool ok0, bool ok1) {
    f32x4_t sc[2][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) sc[tt][rt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(buf + ka[kk] + tt * 16 * L::ROW);
        sc[tt][0] = mfma16x16x32_f16(kf, qb[0][kk], sc[tt][0]);
        sc[tt][1] = mfma16x16x32_f16(kf, qb[1][kk], sc[tt][1]);
      }
    const float* scl = reinterpret_cast<const float*>(buf + 2 * L::TILE);
    float ksc[8], vsc[8];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(scl + 16 * tt + 4 * grp);
      const f32x4_t v4 = *reinterpret_cast<const f32x4_t*>(scl + 32 + 16 * tt + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ksc[4 * tt + r] = k4[r];
        vsc[4 * tt + r] = v4[r];
      }
    }
    const float size = scl[64];
    const bool whole = t0 + kBlock <= all && ok0 && ok1;
    u32x4_t pb[2];
    float alpha[2];
    bool up[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      float s[8];
      bool ok[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = sc[i >> 2][rt][i & 3] * ksc[i];
        ok[i] = t0 + 16 * (i >> 2) + 4 * grp + (i & 3) <= lim[rt] && (i < 4 ? ok0 : ok1);
      }
      alpha[rt] = whole ? row_block<false>(st[rt], s, ok, mul[rt], vsc, size, pb[rt], up[rt])
                        : row_block<true>(st[rt], s, ok, mul[rt], vsc, 0.0f, pb[rt], up[rt]);
    }
    if (__ballot(up[0] || up[1])) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const float f = up[rt] ? alpha[rt] : 1.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[rt][j] *= f;
      }
    }
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const unsigned char* vp = buf + va[j % NVB] + 256 * (j / NVB);
      const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4_t*)(vp)));
      const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4_t*)(vp + 16 * L::ROW)));
      const u32x4_t vf = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      acc[0][j] = mfma16x16x32_f16(vf, pb[0], acc[0][j]);
      acc[1][j] = mfma16x16x32_f16(vf, pb[1], acc[1][j]);
    }
  };

  if (ib0 < ib1) {
    BlockPages now = block_pages(a, trow, kBlock * ib0);
    BlockPages next = block_pages(a, trow, kBlock * min(ib0 + 1, last));
    load(ib0, now);
    stage(smem);
    load(ib0 + 1, next);
    BlockPages after = block_pages(a, trow, kBlock * min(ib0 + 2, last));
    __syncthreads();
    for (int ib = ib0; ib < ib1; ++ib) {
      const int cur = (ib - ib0) & 1;
      if (kBlock * ib < most) compute(smem + cur * L::BUF, kBlock * ib, now.ok[0], now.ok[1]);
      stage(smem + (cur ^ 1) * L::BUF);
      load(ib + 2, after);
      now = next;
      next = after;
      after = block_pages(a, trow, kBlock * min(ib + 3, last));
      __syncthreads();
    }
  }

#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const float z = sum_groups(st[rt].z);
    const int r = 32 * wave + 16 * rt + n16;
    if (r >= rows) continue;
    if (it.parts == 1) {
      const int64_t at = out_row(a, it, kh, rw0 + r, gqa) * D;
      const float inv = z != 0.0f ? 1.0f / z : 0.0f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) store_row4(a, at + 16 * j + 4 * grp, z != 0.0f ? acc[rt][j] * inv : acc[rt][j]);
    } else {
      const int64_t at = ((int64_t)kh * a.slots + it.slot + it.part) * 128 + r;
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4_t*>(a.pacc + at * D + 16 * j + 4 * grp) = acc[rt][j];
      if (grp == 0) {
        a.pm[at] = part_max(st[rt], z);
        a.pz[at] = z;
      }
    }
  }
}

// Joins the parts of split contexts: workgroup (x, kh) takes 16 rows of a split
// tile, each thread four dims of a row at a time, eight parts in flight.
template <int D, int R>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedSdpaArgs a) {
  constexpr int GROUPS = R / 16;
  const int kh = blockIdx.x % a.Hkv, x = blockIdx.x / a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<R, true>(a, x / GROUPS);
  if (it.b < 0) return;
  const int r0 = 16 * (x % GROUPS);
  const int rows = min(it.rows - R * it.tile - r0, 16);
  const int64_t base = ((int64_t)kh * a.slots + it.slot) * R + r0;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 256) {
    const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
    float mm = kNegInf, z = 0.0f;
    for (int k = 0; k < it.parts; ++k) mm = fmaxf(mm, a.pm[base + (int64_t)k * R + r]);
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < it.parts; k0 += 8) {
      f32x4_t v[8];
      float f[8];
      bool live[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t at = base + (int64_t)min(k0 + u, it.parts - 1) * R + r;
        const float m = a.pm[at];
        live[u] = k0 + u < it.parts && m != kNegInf;
        f[u] = __builtin_amdgcn_exp2f(m - mm);
        v[u] = *reinterpret_cast<const f32x4_t*>(a.pacc + at * D + d);
        z = live[u] ? fmaf(a.pz[at], f[u], z) : z;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (live[u]) o += v[u] * f[u];
    }
    if (z != 0.0f) o /= z;
    store_row4(a, out_row(a, it, kh, R * it.tile + r0 + r, gqa) * D + d, o);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct PagedPlan {
  bool few;
  int rows;           // of a tile
  int64_t max_tiles;  // of the whole batch, at most
  int64_t slots;
  int min_blocks;
};

PagedPlan paged_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t max_tokens) {
  PagedPlan p;
  const int64_t gqa = Hq / Hkv;
  max_new = std::min(max_new, T);
  p.few = max_new * gqa <= 16;
  p.rows = p.few ? 16 : 128;
  p.min_blocks = 4;
  p.max_tiles = std::min(T * gqa / p.rows + B, B * cdiv(max_new * gqa, p.rows));
  const int64_t blocks = p.max_tiles * cdiv(max_tokens, kBlock);
  p.slots = std::max<int64_t>(1, std::min<int64_t>(cdiv(env_int("SPARKQ_PAGED_WGS", 4) * device_cus(), Hkv), cdiv(blocks, p.min_blocks)));
  return p;
}

template <int D>
void launch_paged(const PagedSdpaArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.slots + p.max_tiles) * a.Hkv));
  const dim3 merge((unsigned)(p.slots / 2 * (p.rows / 16) * a.Hkv));
  if (p.few)
    hipLaunchKernelGGL(paged_few_kernel<D>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(paged_tile_kernel<D>, grid, dim3(256), 0, st, a);
  if (merge.x == 0) return;
  if (p.few)
    hipLaunchKernelGGL((paged_merge_kernel<D, 16>), merge, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, 128>), merge, dim3(256), 0, st, a);
}

}  // namespace

// Parts of split contexts: their outputs, then maxima and sums.
size_t paged_sdpa_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                            int64_t max_tokens) {
  const PagedPlan p = paged_plan(T, B, Hq, Hkv, max_new, max_tokens);
  return p.slots < 2 ? 0 : (size_t)(Hkv * p.slots * p.rows * (D + 2)) * sizeof(float);
}

int paged_sdpa(const PagedBatch& p, const void* q, const int64_t* qst, const PagedSide& ks,
               const PagedSide& vs, void* out, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
               int causal, int qdt, int odt, float scale, void* ws, size_t wsb, hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  const int64_t max_tokens = (int64_t)p.width << p.page_log2;
  const PagedPlan plan = paged_plan(p.T, p.B, Hq, Hkv, max_new, max_tokens);
  const size_t need = paged_sdpa_workspace(p.T, p.B, Hq, Hkv, D, max_new, max_tokens);
  if (need > 0 && (!ws || wsb < need))
    return set_error(SPARKQ_ERR_WORKSPACE, "paged_sdpa needs a workspace of %zu bytes (got %zu)", need,
                     ws ? wsb : (size_t)0);
  if (!aligned(ws, 16)) return set_error(SPARKQ_ERR_INVALID, "paged_sdpa: workspace must be 16-byte aligned");
  const int64_t n = Hkv * plan.slots * plan.rows;
  float* acc = (float*)ws;
  const PagedSdpaArgs a{p, (const uint16_t*)q, qst[0], qst[1], ks, vs, out, acc + n * D, acc + n * (D + 1), acc,
                        (int)Hq, (int)Hkv, (int)std::min<int64_t>(max_new, p.T), causal, qdt, odt,
                        (int)plan.slots, plan.min_blocks, scale * 1.44269504088896340736f};
  if (D == 64)
    launch_paged<64>(a, plan, st);
  else if (D == 128)
    launch_paged<128>(a, plan, st);
  else
    launch_paged<256>(a, plan, st);
  return check_launch("paged_sdpa");
}

}  // namespace sparkq
