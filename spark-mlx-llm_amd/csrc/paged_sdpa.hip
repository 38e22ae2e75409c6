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
//   paged_tile_kernel  tiles of 128 rows, D up to 128: a block of 64 tokens is
//                      turned to fp16 in LDS once for all of them.
//   paged_pair_kernel  the same at D = 256, where a pair of waves shares its rows.
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
// of a value, p_n times its scale, goes in as two fp16 operands, what the first's
// rounding leaves being the second (22 bits), with few rows, where the matrix cores
// idle (64 sequences 66.9 -> 67.5 us), and in tiles with fp32 outputs. With 16-bit
// outputs tiles take one, off by at most 2^-11, what an fp16 output's own rounding is
// and an eighth of a bf16 output's: the second product costs a quarter of the time
// (2048 new tokens 315 -> 392 us, 24 sequences at D = 256 290 -> 343). All of them in a
// unit that the largest of these weights sets, so that neither tokens of small
// values and much weight nor those of large values and little cost the others their
// bits: near 2^14 with few rows, near 2^7 in tiles, which move their unit only when
// a block exceeds it by 2^8. In the products the scales' exponents stand for the
// scales. So the unit is a power of two beside the score of the token that it comes
// from, whose weight is then its value's scale times a power of two, which one fp16
// holds: where one token outweighs the rest nothing is lost (fp16 outputs of sharp
// rows in tiles: 1.07 to 1.13 times the error of rounding the exact ones, where a power
// of two above the maximum had 1.41). The running maximum, the normalizer and the
// sums are fp32.
#include <algorithm>
#include <type_traits>

#include "paged_attn.h"

namespace sparkq {
namespace {

// ---------------------------------------------------------------------------
// at most 16 rows
// ---------------------------------------------------------------------------
// S^T (16 tokens x 16 rows) = K . Q^T twice a block, O^T (16 dims x 16 rows) +=
// V^T . P^T. Row m of the first product's operand is token 8 (m / 4) + m % 4
// (+ 4 in the second), so that the lane with a row's scores of tokens 8g ..
// 8g+7 holds just the k-slots of the second product's operand: weights never
// leave their lane. V goes through a wave's own LDS to be read transposed.
//
// The waves of a workgroup take turns at blocks of 32 tokens, each with the next
// block's loads in flight and no barrier until they join; keys and values, read
// once, go past the caches. Bound by HBM where there is much: 64 sequences of up to
// 8192 tokens, 8 heads of 128, 304 MB in 62.5 us, 4.9 TB/s (of an earlier form that
// took 61.5: two workgroups a CU 68, four, which spill, 99, cached loads 64); by the
// latency of its steps where there is little: one of 4095 tokens 7 us, of which
// find_item and the first loads are half.
//
// Up to 16 rows: 16 sequences of 8192 tokens (4 heads to each of 8 of 128) with one
// new one each 61 us a call, with 4 new ones 66, by tiles 84 and 82; with 8 new ones,
// which would be two passes over the cache here, 83 by tiles.
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
  const int all = last_seen(a, it, 16 * it.tile, gqa) + 1;              // by every row
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
    u16x2_t most = {0, 0};  // the largest scale's bits: finite below those of infinity
    u16x2_t one = {1, 1};   // 0 where a scale is 1
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kw = skr[i >> 1], vw = svr[i >> 1];
      s[i] = sc[i >> 2][i & 3] * (((i & 1) ? hi16<F16>(kw) : lo16<F16>(kw)) * a.sign);
      vsc[i] = (i & 1) ? hi16<F16>(vw) : lo16<F16>(vw);
      if (i & 1) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, vw & 0x7FFF7FFFu));
        one = __builtin_elementwise_min(one, __builtin_bit_cast(u16x2_t, vw ^ 0x3C003C00u));
      }
    }
    const bool odd = most[0] >= 0x7C00 || most[1] >= 0x7C00 || one[0] == 0 || one[1] == 0;
    if (__builtin_expect(t0 + kBlock > all || pages_ok != 3 || __ballot(odd) != 0, 0)) {
      uint32_t ok = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) ok |= (uint32_t)(t0 + 8 * grp + i <= lim) << i;
      if (!((pages_ok >> (grp >> 1)) & 1u)) ok = 0;
      ok = __float_as_uint(pinned(__uint_as_float(ok)));
      uint32_t zero = 0;
      if (__ballot(one[0] == 0 || one[1] == 0)) zero = zero_values<D, 32>(a, trow, vhead, t0) >> (8 * grp);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool live = (ok >> i) & 1u;
        s[i] = live ? s[i] : kNegInf;
        vsc[i] = live && !(((zero >> i) & 1u) && vsc[i] == 1.0f) ? vsc[i] : 0.0f;
      }
    }
    float t = kNegInf;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaxf(t, fmaf(s[i], mul, scale_exp(vsc[i])));
    t = max_groups<4>(t);
    load(ib + 4, next);
    next = block_pages<2>(a, trow, kBlock * min(ib + 8, last));
    u32x4_t w, rest;
    bool up;
    const float alpha = row_block<8, kTopFew, 0, true>(st, s, mul, vsc, t, &w, &rest, up);
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
      const u32x4_t v8 = s8x8_exact((uint32_t)t8.x, (uint32_t)t8.y);
      acc[j] = mfma16x16x32_f16(v8, w, acc[j]);
      acc[j] = mfma16x16x32_f16(v8, rest, acc[j]);
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
      wm[wave * 16 + n16] = part_max<kTopFew>(st, z);
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
      if (a.lse && d == 0) a.lse[out_row(a, it, kh, 16 * it.tile + r, gqa)] = row_lse(mm, zz);
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
// Four waves of 32 rows each. The products run as above on the 32 x 32 MFMA, a
// lane has one row, and of a block the scores i of tokens 8 (i / 4) + 4 g + i % 4, g
// its half of the wave: scores 8 s .. +8 are its k-slots of the second product's
// step s. 16-row waves read every K and V operand from LDS for half the work: 334
// us where these took 309 (2048 new tokens of 8192, 32 heads).
//
// A block of codes is read once by the workgroup and written to LDS as fp16,
// token-major, two buffers deep: the next block's codes are converted while this
// one is computed, and the one after is in flight. K rows are padded by 16 bytes, so
// that any 16 lanes of a read that the LDS takes together hit different banks; V
// rows, read transposed, are padded to the same end.
//
// Two workgroups a CU is what registers (240) and LDS (76 KB) allow; being at
// different places of their blocks, one's products and LDS reads run beside the
// other's softmax. 2048 new tokens of 8192, 32 heads of 128, 240 GFLOP: 314 us, 764
// TFLOP/s. Nothing is full: of the cycles the matrix cores are busy in 34%, the LDS in
// 44%, vector instructions issue in 53%, and waves wait in 26% of theirs. What is short
// is the overlap of two waves a SIMD, each of which needs some 3000 cycles for a block
// of 64 tokens with 32 products (1024 cycles of the matrix cores), about 370 vector and
// 75 LDS instructions; and the clock falls to 2.2 GHz. Scores one block ahead, so that
// products and exponentials are independent neighbours in one wave, saved 4% of the
// cycles and lost as much in clock.
template <int D>
struct TileShape {
  static constexpr int BLOCK = 64;                    // tokens
  static constexpr int KROW = 2 * D + 16, VROW = 2 * D + 64;
  static constexpr int V = BLOCK * KROW;
  static constexpr int SCALES = V + BLOCK * VROW;     // of keys, of values, the largest and least of each 16 of these
  static constexpr int BUF = SCALES + 2 * BLOCK * 4 + 64;  // (as many again that are not read)
  static constexpr int BYTES = 2 * BUF;
};

// The pages of a block of 64 tokens, PG of them (1, 2 or 4), as offsets into a
// head's codes and scales: of a wave's pieces i, which lie in runs run0 + i * step
// of 16 tokens, and of the run srun whose scales it takes. A lane's own offset
// counts from the block's first token where PG is 1, else from its page's.
// `ok` says which runs have a page; page 0 stands in for the others, whose tokens
// are hidden. (2048 new tokens of 8192, 32 heads of 128: one page to a block 314 us,
// two 316, four 319.)
template <int PG, int PPT>
struct TilePages {
  uint64_t at[PG == 1 ? 1 : PPT], sat;
  uint32_t ok;
};
template <int PG, int PPT>
__device__ __forceinline__ TilePages<PG, PPT> tile_pages(const PagedSdpaArgs& a, TableRow row, int t0, int run0,
                                                         int step, int srun) {
  // the block's entries in one load; those past the table's row stand behind every
  // length, and are the last one
  typedef int entries_t __attribute__((ext_vector_type(PG), aligned(4)));
  typedef const __attribute__((address_space(4))) entries_t* Entries;
  const int mask = (1 << a.p.page_log2) - 1, j0 = t0 >> a.p.page_log2;
  entries_t id;
  if (PG == 1 || j0 + PG <= a.p.width) {
    id = *(Entries)(row + (PG == 1 ? min(j0, a.p.width - 1) : j0));
  } else {
#pragma unroll
    for (int h = 0; h < PG; ++h) id[h] = row[min(j0 + h, a.p.width - 1)];
  }
  constexpr uint32_t runs = (1u << 4 / PG) - 1;
  TilePages<PG, PPT> r;
  r.ok = 0;
#pragma unroll
  for (int h = 0; h < PG; ++h) {
    const bool valid = (unsigned)id[h] < (unsigned)a.p.pages;
    r.ok |= (valid ? runs : 0) << (4 / PG * h);
    id[h] = valid ? id[h] : 0;
  }
  auto of = [&](int run) __attribute__((always_inline)) {
    const int h = run * PG / 4;
    int v = id[0];
#pragma unroll
    for (int k = 1; k < PG; ++k) v = h == k ? id[k] : v;
    return v;
  };
  if constexpr (PG == 1) {
    r.at[0] = code_at(a.c, id[0], t0 & mask);
    r.sat = scale_at(a.c, id[0], (t0 & mask) + 16 * srun);
  } else {
#pragma unroll
    for (int i = 0; i < PPT; ++i) r.at[i] = code_at(a.c, of(run0 + i * step), 0);
    r.sat = scale_at(a.c, of(srun), 16 * srun & mask);
  }
  return r;
}

__device__ __forceinline__ f32x16_t tile_mfma(u32x4_t x, u32x4_t y, f32x16_t c) { return mfma32x32x16<F16>(x, y, c); }

template <int D, int PG, bool TWO>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedSdpaArgs a) {
  using S = TileShape<D>;
  constexpr int R = kTileRows, kBlock = S::BLOCK, G = 2, N = kBlock / G, Q = kBlock / 16;
  constexpr int NK = D / 16, NJ = D / 32, NT = kBlock / 32;
  constexpr int PPT = kBlock * D / 16 / 256;  // 16-code pieces of a K (or V) block per thread
  using Sum = f32x16_t;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, row = lane & 31, grp = lane >> 5;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  // the CUs' second workgroups in reverse order: the longest with the shortest
  const int x = blockIdx.x / a.Hkv;
  const Item it = find_item<R, false>(a, x >= a.snake && x < 2 * a.snake ? 3 * a.snake - 1 - x : x);
  if (it.b < 0) return;
  const int rw0 = R * it.tile;
  const int rows = min(it.rows - rw0, R);
  const int seen = last_seen(a, it, rw0 + rows - 1, gqa) + 1;
  const int nblocks = (seen + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const TableRow trow = table_row(a, it.b);

  const int wr0 = rw0 + 32 * wave;  // the wave's first row
  const int rr = wr0 + row, rq = min(rr, it.rows - 1);
  const int lim = last_seen(a, it, rr, gqa);
  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + (it.first + rq / gqa) * a.q_tok + (kh * gqa + rq % gqa) * a.q_head;
  const float mul = load_query<NK, G>(a, qrow, rr < it.rows, [&](int c) { return 16 * c + 8 * grp; }, qb);
  // what every row of the tile sees
  const int all = __builtin_amdgcn_readfirstlane(last_seen(a, it, rw0, gqa) + 1);

  // Piece i of a block: token tk0 + i TPP, codes 16 jb .. +16. All tokens of a
  // wave's piece lie in one run of 16, and so in one page. Wave w also takes the
  // scales of run w: keys in its first 16 lanes, values in the next, and the same
  // again in the upper half, which spares branches.
  u32x4_t kcr[PPT], vcr[PPT];
  uint16_t sr;
  const int last = ib1 - 1;
  const uint8_t *const khead = a.c.k + kh * a.c.c_head, *const vhead = a.c.v + kh * a.c.c_head;
  const bool ks_lane = !(lane & 16);
  const uint16_t* const shead = (ks_lane ? a.c.ks : a.c.vs) + kh * a.c.s_head + n16;
  const int tk0 = tid / (D / 16), jb = tid % (D / 16);
  constexpr int TPP = 256 / (D / 16);  // tokens of a round of pieces
  uint32_t off[PPT];
#pragma unroll
  for (int i = 0; i < PPT; ++i) off[i] = ((tk0 + i * TPP) & (kBlock / PG - 1)) * a.c.c_tok + 16 * jb;
  using Pages = TilePages<PG, PPT>;
  auto pages = [&](int ib) {
    return tile_pages<PG, PPT>(a, trow, kBlock * min(ib, last), wave * 64 / D, TPP / 16, wave);
  };
  auto load = [&](const Pages& bp) {
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      kcr[i] = *reinterpret_cast<const u32x4_t*>(khead + bp.at[PG == 1 ? 0 : i] + off[i]);
      vcr[i] = *reinterpret_cast<const u32x4_t*>(vhead + bp.at[PG == 1 ? 0 : i] + off[i]);
    }
    sr = shead[bp.sat];
  };
  unsigned char* const kput = smem + tk0 * S::KROW + 32 * jb;
  unsigned char* const vput = smem + S::V + tk0 * S::VROW + 32 * jb;
  float* const sput = reinterpret_cast<float*>(smem + S::SCALES) + (ks_lane ? 0 : kBlock) + 16 * wave + n16;
  float* const bput = reinterpret_cast<float*>(smem + S::SCALES) + 2 * kBlock + (ks_lane ? 4 : 0) + wave;
  auto stage = [&](auto bufc, int ib) {  // block ib, no further than the last
    constexpr int at = decltype(bufc)::value * S::BUF;
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      unsigned char *kt = kput + at + i * TPP * S::KROW, *vt = vput + at + i * TPP * S::VROW;
      *reinterpret_cast<u32x4_t*>(kt) = s8x8_exact(kcr[i].x, kcr[i].y);
      *reinterpret_cast<u32x4_t*>(kt + 16) = s8x8_exact(kcr[i].z, kcr[i].w);
      *reinterpret_cast<u32x4_t*>(vt) = s8x8_exact(vcr[i].x, vcr[i].y);
      *reinterpret_cast<u32x4_t*>(vt + 16) = s8x8_exact(vcr[i].z, vcr[i].w);
    }
    float v = f16_to_f32(sr);
    if (__builtin_expect(__ballot(!ks_lane && v == 1.0f) != 0, 0)) {
      const uint32_t zero = zero_values<D, 16>(a, trow, vhead, kBlock * min(ib, last) + 16 * wave);
      if (!ks_lane && v == 1.0f && ((zero >> n16) & 1u)) v = 0.0f;
    }
    sput[at / 4] = ks_lane ? v * a.sign : kept_scale(v);
    bput[at / 4] = most_of(v);
    bput[at / 4 + 8] = least_of(v);
  };

  const unsigned char* const kget = smem + row * S::KROW + 16 * grp;  // chunk 2 kk + g of token `row`
  const unsigned char* const vget = smem + S::V + (4 * grp + (n16 >> 2)) * S::VROW + 8 * (n16 & 3) +
                                    32 * ((lane >> 4) & 1);
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
      for (int kk = 0; kk < NK; ++kk)
        sc[tt] = tile_mfma(*reinterpret_cast<const u32x4_t*>(kget + at + tt * 32 * S::KROW + 32 * kk), qb[kk], sc[tt]);
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
        s[i + r] = sc[i / 16][i % 16 + r] * k4[r];
      }
    }
    const float* big = reinterpret_cast<const float*>(smem + at + S::SCALES) + 2 * kBlock;
    float size = big[0], least = big[8];
#pragma unroll
    for (int i = 1; i < Q; ++i) {
      size = fmaxf(size, big[i]);
      least = fminf(least, big[8 + i]);
    }
    float t;
    if (__builtin_expect(t0 + kBlock > all || pages_ok != (1u << Q) - 1 || size > kSpread * least, 0)) {
      uint32_t ok = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = 4 * G * (i >> 2) + 4 * grp + (i & 3);
        ok |= (uint32_t)(t0 + j <= lim && ((pages_ok >> (j / 16)) & 1u)) << i;
      }
      float odd;
      t = hide<N, G>(__float_as_uint(pinned(__uint_as_float(ok))), s, mul, vsc, odd);
      if (__ballot(odd != odd)) {
        const float f = pinned(odd != odd ? odd : 1.0f);
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] *= f;
      }
    } else {
      t = s[0];
#pragma unroll
      for (int i = 1; i < N; ++i) t = fmaxf(t, s[i]);
      t = fmaf(max_groups<G>(t), mul, scale_exp(size));
    }
    u32x4_t w[N / 8], rest[N / 8];
    bool up;
    const float alpha = row_block<N, kTopTile, 8, TWO>(st, s, mul, vsc, t, w, rest, up);
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
        const unsigned char* vp = vget + at + 16 * k * S::VROW + 64 * j;
        const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(vp)));
        const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(vp + 8 * S::VROW)));
        acc[j] = tile_mfma(u32x4_t{lo.x, lo.y, hi.x, hi.y}, w[k], acc[j]);
        if (TWO) acc[j] = tile_mfma(u32x4_t{lo.x, lo.y, hi.x, hi.y}, rest[k], acc[j]);
      }
  };

  if (ib0 < ib1) {
    Pages bp = pages(ib0);
    uint32_t ok_now = bp.ok, ok_next;
    load(bp);
    bp = pages(ib0 + 1);
    stage(std::integral_constant<int, 0>{}, ib0);
    load(bp);
    ok_next = bp.ok;
    __syncthreads();
    auto step = [&](int ib, auto cur) {
      const Pages after = pages(ib + 2);
      if (wr0 < it.rows) compute(cur, kBlock * ib, ok_now);
      stage(std::integral_constant<int, 1 - decltype(cur)::value>{}, ib + 1);
      load(after);
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
  const int r = 32 * wave + row;
  if (r >= rows) return;
  if (it.parts == 1) {
    const int64_t at = out_row(a, it, kh, rw0 + r, gqa) * D;
    if (a.lse && grp == 0) a.lse[at / D] = row_lse(part_max<kTopTile>(st, z), z);
    const float inv = z != 0.0f ? 1.0f / z : 1.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        store_row4(a, at + 32 * j + 2 * v + 4 * grp,
                   f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]} * inv);
  } else {
    const int64_t at = ((int64_t)kh * a.slots + it.slot + it.part) * R + r;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4_t*>(a.pacc + at * D + 32 * j + 2 * v + 4 * grp) =
            f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]};
    if (grp == 0) {
      a.pm[at] = part_max<kTopTile>(st, z);
      a.pz[at] = z;
    }
  }
}

// ---------------------------------------------------------------------------
// tiles of 128 rows, D = 256
// ---------------------------------------------------------------------------
// The outputs of 32 rows of 256 take 128 registers a lane and their queries 64: one
// wave a SIMD. So a pair of waves shares 32 rows: each scores one half of a block's
// 64 tokens over all dims, hands its weights to the other through LDS, and sums all
// 64 tokens' values of its half of the dims. Eight waves a CU, every operand from
// LDS is used for 32 rows, and a block's conversion is shared by 512 threads.
// (24 sequences of up to 1000 new tokens, 166 GFLOP, 16 heads of 256: 289 us, 575
// TFLOP/s. With maxima rounded up to whole numbers, which need no second pass over the
// sums below but cost bits, 18 us less; an earlier form of 296, where waves of 16 rows
// with all dims took 346, and waves of 32 rows alone on their SIMDs 376.)
//
// Both waves weigh in the units of their own running maxima; where these differ
// after a block (its first, and hardly ever later: they move by 2^8 or more) both go
// on with the larger.
//
// A block has two phases. In the first its keys are read and its values are written
// to LDS, in the second the values are read and the next keys are written: one buffer
// of each and a barrier after each phase. (Half the waves a phase behind the others,
// with two buffers, took 306 us for these 296.) Bound by the latency of a wave's own
// chain through these phases: matrix cores busy in 24% of the cycles, the LDS in 32%,
// waves wait in 30% of theirs, and a CU has no other workgroup to run meanwhile.
template <bool TWO>
struct PairShape {
  static constexpr int D = 256, BLOCK = 64;
  static constexpr int KROW = 2 * D + 16, VROW = 2 * D + 64;
  static constexpr int V = BLOCK * KROW, P = V + BLOCK * VROW;
  static constexpr int STATE = P + 8 * 2 * 1024 * (TWO ? 2 : 1);  // of each wave's rows: t
  static constexpr int SCALES = STATE + 8 * 32 * 4;   // of keys, of values, the largest and least of each 16 of these
  static constexpr int BYTES = SCALES + 2 * BLOCK * 4 + 32;
};

template <int PG, bool TWO>  // pages that a block lies in: 1, 2 or 4
__global__ __launch_bounds__(512, 2) void paged_pair_kernel(PagedSdpaArgs a) {
  using S = PairShape<TWO>;
  constexpr int D = S::D, R = kTileRows, kBlock = S::BLOCK, N = 16, Q = kBlock / 16, G = 2;
  constexpr int NK = D / 16, NJ = 4, PPT = 2;
  using Sum = f32x16_t;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave & 1;
  const int n16 = lane & 15, row = lane & 31, grp = lane >> 5;
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

  const int wr0 = rw0 + 32 * (wave >> 1);  // the pair's first row
  const int rr = wr0 + row, rq = min(rr, it.rows - 1);
  const int lim = last_seen(a, it, rr, gqa);
  const bool live = wr0 < it.rows;
  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + (it.first + rq / gqa) * a.q_tok + (kh * gqa + rq % gqa) * a.q_head;
  const float mul = load_query<NK, G>(a, qrow, rr < it.rows, [&](int c) { return 16 * c + 8 * grp; }, qb);
  const int all = __builtin_amdgcn_readfirstlane(last_seen(a, it, rw0, gqa) + 1);

  // Piece i of a block: token tk0 + 32 i, codes 16 jb .. +16. A wave's pieces lie in
  // runs 2 i + wave / 4 of 16 tokens, and it takes the scales of run wave % 4.
  u32x4_t kcr[PPT], vcr[PPT];
  uint16_t skr, svr;
  const int last = ib1 - 1, srun = wave & 3;
  const uint8_t *const khead = a.c.k + kh * a.c.c_head, *const vhead = a.c.v + kh * a.c.c_head;
  const uint16_t *const kshead = a.c.ks + kh * a.c.s_head + n16, *const vshead = a.c.vs + kh * a.c.s_head + n16;
  const int tk0 = tid >> 4, jb = tid & 15;
  uint32_t off[PPT];
#pragma unroll
  for (int i = 0; i < PPT; ++i) off[i] = ((tk0 + 32 * i) & (kBlock / PG - 1)) * a.c.c_tok + 16 * jb;
  using Pages = TilePages<PG, PPT>;
  auto pages = [&](int ib) __attribute__((always_inline)) {
    return tile_pages<PG, PPT>(a, trow, kBlock * min(ib, last), wave >> 2, 2, srun);
  };
  auto load_codes = [&](const uint8_t* head, const Pages& bp, u32x4_t (&r)[PPT]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PPT; ++i)
      r[i] = *reinterpret_cast<const u32x4_t*>(head + bp.at[PG == 1 ? 0 : i] + off[i]);
  };
  auto load_scales = [&](const Pages& bp) __attribute__((always_inline)) {
    skr = kshead[bp.sat];
    svr = vshead[bp.sat];
  };
  unsigned char* const kput = smem + tk0 * S::KROW + 32 * jb;
  unsigned char* const vput = smem + S::V + tk0 * S::VROW + 32 * jb;
  auto stage = [&](unsigned char* t, u32x4_t c) __attribute__((always_inline)) {
    *reinterpret_cast<u32x4_t*>(t) = s8x8_exact(c.x, c.y);
    *reinterpret_cast<u32x4_t*>(t + 16) = s8x8_exact(c.z, c.w);
  };
  float* const scl = reinterpret_cast<float*>(smem + S::SCALES);
  auto stage_scales = [&](int ib) __attribute__((always_inline)) {  // block ib, no further than the last
    float v = f16_to_f32(svr);
    if (__builtin_expect(__ballot(v == 1.0f) != 0, 0)) {
      const uint32_t zero = zero_values<D, 16>(a, trow, vhead, kBlock * min(ib, last) + 16 * srun);
      if (v == 1.0f && ((zero >> n16) & 1u)) v = 0.0f;
    }
    scl[16 * srun + n16] = f16_to_f32(skr) * a.sign;
    scl[kBlock + 16 * srun + n16] = kept_scale(v);
    scl[2 * kBlock + srun] = most_of(v);
    scl[2 * kBlock + 4 + srun] = least_of(v);
  };

  const unsigned char* const kget = smem + (32 * half + row) * S::KROW + 16 * grp;
  const unsigned char* const vget = smem + S::V + (4 * grp + (n16 >> 2)) * S::VROW + 8 * (n16 & 3) +
                                    32 * ((lane >> 4) & 1) + 256 * half;
  constexpr int WAVE = TWO ? 4096 : 2048;
  unsigned char* const pput = smem + S::P + wave * WAVE + lane * 16;
  const unsigned char* const pget = smem + S::P + (wave ^ 1) * WAVE + lane * 16;
  float* const state = reinterpret_cast<float*>(smem + S::STATE);
  const int own = 32 * half * S::VROW, other = 32 * (half ^ 1) * S::VROW;
  RowState st;
  Sum acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = Sum{};
  u32x4_t w[4], rest[4];  // of the half of this wave, of the other

  // scores and weights of this wave's 32 tokens, and values into LDS
  auto first = [&](int t0, uint32_t pages_ok) __attribute__((always_inline)) {
    Sum sc = Sum{};
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      sc = tile_mfma(*reinterpret_cast<const u32x4_t*>(kget + 32 * kk), qb[kk], sc);
      if (kk == 4 || kk == 8) stage(vput + (kk / 4 - 1) * 32 * S::VROW, vcr[kk / 4 - 1]);
    }
    const float* ks = scl + 32 * half + 4 * grp;
    float s[N], vsc[N];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(ks + G * i);
      const f32x4_t v4 = *reinterpret_cast<const f32x4_t*>(ks + kBlock + G * i);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vsc[i + r] = v4[r];
        s[i + r] = sc[i + r] * k4[r];
      }
    }
    const f32x4_t big = *reinterpret_cast<const f32x4_t*>(scl + 2 * kBlock);
    const f32x4_t low = *reinterpret_cast<const f32x4_t*>(scl + 2 * kBlock + 4);
    const float size = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
    const float least = fminf(fminf(low[0], low[1]), fminf(low[2], low[3]));
    float t;
    if (__builtin_expect(t0 + kBlock > all || pages_ok != (1u << Q) - 1 || size > kSpread * least, 0)) {
      uint32_t ok = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = 32 * half + 4 * G * (i >> 2) + 4 * grp + (i & 3);
        ok |= (uint32_t)(t0 + j <= lim && ((pages_ok >> (j / 16)) & 1u)) << i;
      }
      float odd;
      t = hide<N, G>(__float_as_uint(pinned(__uint_as_float(ok))), s, mul, vsc, odd);
      if (__ballot(odd != odd)) {
        const float f = pinned(odd != odd ? odd : 1.0f);
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] *= f;
      }
    } else {
      t = s[0];
#pragma unroll
      for (int i = 1; i < N; ++i) t = fmaxf(t, s[i]);
      t = fmaf(max_groups<G>(t), mul, scale_exp(size));
    }
    bool up;
    const float alpha = row_block<N, kTopTile, 8, TWO>(st, s, mul, vsc, t, w, rest, up);
    if (__builtin_expect(__ballot(up) != 0, 0)) {
      const float f = pinned(up ? alpha : 1.0f);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
    *reinterpret_cast<u32x4_t*>(pput) = w[0];
    *reinterpret_cast<u32x4_t*>(pput + 1024) = w[1];
    if (TWO) {
      *reinterpret_cast<u32x4_t*>(pput + 2048) = rest[0];
      *reinterpret_cast<u32x4_t*>(pput + 3072) = rest[1];
    }
    state[32 * wave + row] = st.t;
  };
  // the outputs of this wave's 128 dims, and the next keys into LDS
  auto second = [&](int) __attribute__((always_inline)) {
    w[2] = *reinterpret_cast<const u32x4_t*>(pget);
    w[3] = *reinterpret_cast<const u32x4_t*>(pget + 1024);
    if (TWO) {
      rest[2] = *reinterpret_cast<const u32x4_t*>(pget + 2048);
      rest[3] = *reinterpret_cast<const u32x4_t*>(pget + 3072);
    }
    const float o = state[32 * (wave ^ 1) + row];
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    auto product = [&](int k, int j) __attribute__((always_inline)) {
      const unsigned char* vp = vget + (k < 2 ? own : other) + 16 * (k & 1) * S::VROW + 64 * j;
      const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4_t*)(vp)));
      const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4_t*)(vp + 8 * S::VROW)));
      acc[j] = tile_mfma(u32x4_t{lo.x, lo.y, hi.x, hi.y}, w[k], acc[j]);
      if (TWO) acc[j] = tile_mfma(u32x4_t{lo.x, lo.y, hi.x, hi.y}, rest[k], acc[j]);
    };
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        product(k, j);
        if (k == 1 && j < PPT) stage(kput + j * 32 * S::KROW, kcr[j]);
      }
    const float mine = st.t, theirs = o;
    const bool differ = __ballot(mine != theirs) != 0;
    float after = 1.0f;
    if (__builtin_expect(differ, 0)) {
      // The sums go into the other's unit while its weights are added, so that these
      // stay as they were rounded; weights whose unit is 2^-60 of the row's own do not
      // count. (A half that has seen nothing has the unit 2^-inf.)
      st.t = fmaxf(mine, theirs);
      const float now = st.t, gap = mine - theirs;
      const bool near = gap <= 60.0f;
      const float own_factor = mine == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mine - now);
      const float before = pinned(near ? __builtin_amdgcn_exp2f(gap) : 1.0f);
      after = near ? __builtin_amdgcn_exp2f(theirs - now) : own_factor;
      if (!near) w[2] = w[3] = rest[2] = rest[3] = u32x4_t{0, 0, 0, 0};
      st.z *= own_factor;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= before;
    }
#pragma unroll
    for (int k = 2; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < NJ; ++j) product(k, j);
    if (__builtin_expect(differ, 0)) {
      const float f = pinned(after);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
  };

  if (ib0 < ib1) {
    Pages now = pages(ib0), next = pages(ib0 + 1);
    load_codes(khead, now, kcr);
    load_scales(now);
#pragma unroll
    for (int i = 0; i < PPT; ++i) stage(kput + i * 32 * S::KROW, kcr[i]);
    stage_scales(ib0);
    load_codes(vhead, now, vcr);
    load_codes(khead, next, kcr);
    load_scales(next);
    __syncthreads();
    auto block = [&](int ib, auto one, auto two) __attribute__((always_inline)) {
      const Pages after = pages(ib + 2);
      one();
      load_codes(vhead, next, vcr);
      __syncthreads();
      two();
      stage_scales(ib + 1);
      load_codes(khead, after, kcr);
      load_scales(after);
      now = next;
      next = after;
      __syncthreads();
    };
    if (live) {
      for (int ib = ib0; ib < ib1; ++ib)
        block(ib, [&]() __attribute__((always_inline)) { first(kBlock * ib, now.ok); },
              [&]() __attribute__((always_inline)) { second(ib); });
    } else {
      for (int ib = ib0; ib < ib1; ++ib)
        block(ib,
              [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < PPT; ++i) stage(vput + i * 32 * S::VROW, vcr[i]);
              },
              [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < PPT; ++i) stage(kput + i * 32 * S::KROW, kcr[i]);
              });
    }
  }

  // the halves' sums (every wave is past its last read of the states and the weights); a
  // wave that weighed a value that is not finite has NaN in its dims, and here the other
  // learns of it
  float z = sum_groups<G>(st.z);
  float* const some = reinterpret_cast<float*>(smem + S::P);
  state[32 * wave + row] = z;
  if (grp == 0) some[32 * wave + row] = acc[0][0];
  __syncthreads();
  z += state[32 * (wave ^ 1) + row];
  const float odd = some[32 * (wave ^ 1) + row];
  if (__builtin_expect(odd != odd, 0)) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] *= odd;
  }
  const int r = 32 * (wave >> 1) + row;
  if (r >= rows) return;
  if (it.parts == 1) {
    const int64_t at = out_row(a, it, kh, rw0 + r, gqa) * D + 128 * half;
    if (a.lse && grp == 0 && half == 0) a.lse[at / D] = row_lse(part_max<kTopTile>(st, z), z);
    const float inv = z != 0.0f ? 1.0f / z : 1.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        store_row4(a, at + 32 * j + 2 * v + 4 * grp,
                   f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]} * inv);
  } else {
    const int64_t at = ((int64_t)kh * a.slots + it.slot + it.part) * R + r;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4_t*>(a.pacc + at * D + 128 * half + 32 * j + 2 * v + 4 * grp) =
            f32x4_t{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]};
    if (grp == 0 && half == 0) {
      a.pm[at] = part_max<kTopTile>(st, z);
      a.pz[at] = z;
    }
  }
}

// Joins the parts of split contexts: workgroup (x, kh) takes 16 rows of a split
// tile. A wave per row finds the parts' weights (a lane each, one round trip);
// then a thread sums four dims of a row over every `ways`-th part, eight loads
// in flight, and the ways are summed through LDS. A chain of round trips: 4.2 us
// where nothing was split, 4.6 us for 32 parts of one sequence's 32 heads. What weighs
// nothing is added all the same, which NaN needs and which lets the eight loads go out
// together (where each was behind a test of its weight 5.5). A join by the last part to
// end would need counters, in memory of their own that threads and captured graphs share.
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
  if (rows <= 0) return;
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
    if (a.lse && lane == 0) a.lse[out_row(a, it, kh, R * it.tile + r0 + r, gqa)] = row_lse(mm, z);
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
        o += v[u] * (k0 + u * ways < parts ? f : 0.0f);
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
  int min_part, snake;
};

PagedPlan paged_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                     int64_t max_tokens) {
  PagedPlan p;
  const int64_t gqa = Hq / Hkv;
  max_new = std::min(max_new, T);
  p.few = max_new * gqa <= 16;
  p.rows = p.few ? 16 : kTileRows;
  p.min_part = 128;
  p.max_tiles = std::min(T * gqa / p.rows + B, B * cdiv(max_new * gqa, p.rows));
  // a part for each workgroup that the chip holds at once (two tiles a CU, one pair
  // tile: 294 us with two parts a CU where one took 271); with few rows, where three
  // workgroups fit, four, as ragged lengths leave uneven ends (64 sequences 67.5 us,
  // three parts 70.2, six 67.0; 16 of 8192 tokens with 4 new ones 66.1, 63.1 and 72.9)
  p.target = std::min<int64_t>(cdiv((p.few ? 4 : D <= 128 ? 2 : 1) * device_cus(), Hkv), kMaxParts);
  p.split = max_tokens > p.min_part ? std::min(p.max_tiles, p.target) : 0;
  p.slots = std::min(2 * p.target, p.split * cdiv(max_tokens, p.min_part));
  // where the heads' items are dealt to the CUs evenly, and the grid holds the
  // round that is reversed
  p.snake = D <= 128 && device_cus() % Hkv == 0 && p.slots + p.max_tiles >= 2 * device_cus() / Hkv
                ? (int)(device_cus() / Hkv) : 0;
  return p;
}

template <int D, int PG, bool TWO>
void launch_tile(const PagedSdpaArgs& a, dim3 grid, hipStream_t st) {
  if constexpr (D <= 128)
    hipLaunchKernelGGL((paged_tile_kernel<D, PG, TWO>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_pair_kernel<PG, TWO>), grid, dim3(512), 0, st, a);
}

template <int D, bool TWO>
void launch_tiles(const PagedSdpaArgs& a, dim3 grid, hipStream_t st) {
  if (a.p.page_log2 >= 6)
    launch_tile<D, 1, TWO>(a, grid, st);
  else if (a.p.page_log2 == 5)
    launch_tile<D, 2, TWO>(a, grid, st);
  else
    launch_tile<D, 4, TWO>(a, grid, st);
}

template <int D>
void launch_paged(const PagedSdpaArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.slots + p.max_tiles) * a.Hkv));  // of an unsplit tile or a part each
  const dim3 merge((unsigned)(p.split * (p.rows / 16) * a.Hkv));
  if (p.few)
    hipLaunchKernelGGL(paged_few_kernel<D>, grid, dim3(256), 0, st, a);
  else if (a.out_dtype == SPARKQ_F32)
    launch_tiles<D, true>(a, grid, st);
  else
    launch_tiles<D, false>(a, grid, st);
  if (merge.x == 0) return;
  if (p.few)
    hipLaunchKernelGGL((paged_merge_kernel<D, 16>), merge, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, kTileRows>), merge, dim3(256), 0, st, a);
}

}  // namespace

// Parts of split contexts: their outputs, then maxima and sums.
size_t paged_sdpa_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                            int64_t max_tokens) {
  const PagedPlan p = paged_plan(T, B, Hq, Hkv, D, max_new, max_tokens);
  return (size_t)(Hkv * p.slots * p.rows * (D + 2)) * sizeof(float);
}

int paged_sdpa(const PagedBatch& p, const void* q, const int64_t* qst, const PagedSide& ks,
               const PagedSide& vs, void* out, float* lse, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
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
  const PagedSdpaArgs a{p, (const uint16_t*)q, qst[0], qst[1], c, out, lse, acc + n * D, acc + n * (D + 1), acc,
                        (int)Hq, (int)Hkv, (int)std::min<int64_t>(max_new, p.T), causal, qdt, odt,
                        (int)plan.target, (int)plan.slots, plan.min_part, plan.snake,
                        fabsf(scale) * 1.44269504088896340736f, scale < 0.0f ? -1.0f : 1.0f};
  if (D == 64)
    launch_paged<64>(a, plan, st);
  else if (D == 128)
    launch_paged<128>(a, plan, st);
  else
    launch_paged<256>(a, plan, st);
  return check_launch("paged_sdpa");
}

}  // namespace sparkq
