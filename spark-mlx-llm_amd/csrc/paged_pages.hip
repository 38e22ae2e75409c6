// paged_pages.hip -- what a query needs to choose pages of a paged INT8 KV cache:
// the bounds of each page's keys, and scores of the pages for each new token
// (gfx950).
//
// A page's keys lie between lo[d] and hi[d] in every channel d, so no logit of a
// query head with one of them is larger than
//
//   scale * sum_d max(q[d] lo[d], q[d] hi[d])  =  scale * (q+ . hi + q- . lo)
//
// with q+ and q- the positive and negative values of q (scale >= 0; q takes its
// sign): a product of depth 2 D, in fp32 sums (so but for (2 D + 2) 2^-24 of its terms'
// sizes).
#include <algorithm>

#include "paged.h"
#include "sdpa_common.h"

namespace sparkq {
namespace {

typedef short s16x2_t __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------
struct BoundsArgs {
  PagedBatch p;
  const uint8_t* codes;
  const uint16_t* scales;
  int64_t c_page, c_head, c_tok, s_page, s_head, s_tok;  // bytes, elements
  uint16_t* bounds;
  int64_t b_page, b_head;  // elements; [2][D] behind them is contiguous
  int H, per_row;          // KV heads; pages that a sequence's new tokens lie in, at most
};

// fp32 to bf16, away from zero where it is not exact (`away`), else towards it
__device__ __forceinline__ uint32_t bf16_outward(float v, bool away) {
  const uint32_t u = __float_as_uint(v);
  return (away && (u & 0xFFFFu) ? u + 0x10000u : u) >> 16;
}

// A workgroup per (page that holds new tokens, KV head): the page's tokens are read
// again from its codes, so that the bounds are right whatever stood there (a page
// that a fork copied, tokens that were taken back). D / 4 lanes a token, a lane the
// least and largest key of 4 channels, U tokens a thread in flight; the waves' are
// joined through LDS. A token whose scale is not finite bounds nothing: the page's
// bounds are then bf16's largest numbers.
// Latency bounds it, lengths, table and codes one after the other: 16 decoded tokens
// (128 workgroups) take 4.4 us, 3 x 2000 new tokens (5.1 MB, 768 workgroups) 5.8.
template <int D>
__global__ __launch_bounds__(256) void paged_bounds_kernel(BoundsArgs a) {
  constexpr int LPR = D / 4, TPP = 256 / LPR, U = 8;
  __shared__ float s_lo[4][D], s_hi[4][D];
  __shared__ int s_odd[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % a.H, x = blockIdx.x / a.H, b = x / a.per_row;
  const SeqRows s = seq_rows(a.p, b);
  if (s.count == 0) return;
  const int j = (max(s.length - s.count, 0) >> a.p.page_log2) + (x - b * a.per_row);
  const int64_t t0 = (int64_t)j << a.p.page_log2;
  if (t0 >= s.length) return;
  const int id = page_of(a.p, b, (int)t0);
  if (id < 0) return;
  const int n = min(1 << a.p.page_log2, s.length - (int)t0);
  const uint8_t* codes = a.codes + id * a.c_page + h * a.c_head + 4 * (tid % LPR);
  const uint16_t* scales = a.scales + id * a.s_page + h * a.s_head;
  float lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = __builtin_huge_valf();
    hi[i] = -__builtin_huge_valf();
  }
  bool odd = false;
  for (int k0 = tid / LPR; k0 < n; k0 += U * TPP) {
    uint32_t w[U];
    uint16_t sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(k0 + u * TPP, n - 1);  // the last token again changes nothing
      w[u] = *reinterpret_cast<const uint32_t*>(codes + k * a.c_tok);
      sc[u] = scales[k * a.s_tok];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = f16_to_f32(sc[u]);
      odd |= (sc[u] & 0x7C00u) == 0x7C00u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = (float)(int8_t)(w[u] >> (8 * i)) * f;  // exact: 7 + 11 bits
        lo[i] = fminf(lo[i], v);
        hi[i] = fmaxf(hi[i], v);
      }
    }
  }
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = fminf(lo[i], __shfl_xor(lo[i], o));
      hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], o));
    }
  if (lane < LPR) {
    *reinterpret_cast<f32x4_t*>(&s_lo[wave][4 * lane]) = f32x4_t{lo[0], lo[1], lo[2], lo[3]};
    *reinterpret_cast<f32x4_t*>(&s_hi[wave][4 * lane]) = f32x4_t{hi[0], hi[1], hi[2], hi[3]};
  }
  const bool any_odd = __ballot(odd) != 0;
  if (lane == 0) s_odd[wave] = any_odd;
  __syncthreads();
  if (tid >= D) return;
  const int side = tid >= D / 2, d = 2 * (tid % (D / 2));
  const float(*v)[D] = side ? s_hi : s_lo;
  const bool open = s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3];
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float m = v[0][d + i];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = side ? fmaxf(m, v[w][d + i]) : fminf(m, v[w][d + i]);
    const uint32_t r = open ? (side ? 0x7F7Fu : 0xFF7Fu) : bf16_outward(m, side ? m > 0.0f : m < 0.0f);
    out |= r << (16 * i);
  }
  *reinterpret_cast<uint32_t*>(a.bounds + id * a.b_page + h * a.b_head + side * D + d) = out;
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
struct ScoreArgs {
  PagedBatch p;
  const uint16_t* q;
  int64_t q_tok, q_head;  // elements
  const uint16_t* bounds;
  int64_t b_page, b_head;
  float* scores;  // [T, Hkv, width]
  int32_t* seen;  // [T] pages that each row sees
  int Hq, Hkv, max_new, causal, chunks;
  float scale;     // its size
  uint32_t flip;   // bits that give a packed pair the scale's sign
};

template <typename T>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t x, u32x4_t y, f32x4_t c) {
  if constexpr (T::code == SPARKQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y), c,
                                                   0, 0, 0);
  else
    return mfma16x16x32_f16(x, y, c);
}

// A lane's share of the bounds of a page: dims 32 c + 8 grp .. + 8, and what the
// scores have to be multiplied by. For fp16 queries the bounds are turned to fp16,
// shifted by a power of two for that: exact but for what bf16 holds below 2^-28 of
// the page's largest, which is rounded, by 2^-39 of the largest at most (to nearest: a
// bound may come out that much too narrow).
template <typename T, int D>
struct PageOperand {
  u32x4_t lo[D / 32], hi[D / 32];
  float mul;
};
template <typename T, int D>
__device__ __forceinline__ void load_bounds(const uint16_t* at, PageOperand<T, D>& b) {
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    b.lo[c] = *reinterpret_cast<const u32x4_t*>(at + 32 * c);
    b.hi[c] = *reinterpret_cast<const u32x4_t*>(at + D + 32 * c);
  }
}
template <typename T, int D>
__device__ __forceinline__ void turn_bounds(PageOperand<T, D>& b) {
  b.mul = 1.0f;
  if constexpr (T::code == SPARKQ_F16) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t most = {0, 0};
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, b.lo[c][i] & 0x7FFF7FFFu));
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, b.hi[c][i] & 0x7FFF7FFFu));
      }
    uint32_t top = max((uint32_t)most[0], (uint32_t)most[1]);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    // 2^e <= the largest < 2^(e + 1); 0, and infinities, stay as they are
    const int e = (int)(top >> 7) - 127, shift = top >= 0x80u && top < 0x7F80u ? 14 - e : 0;
    auto turn = [&](uint32_t w) {
      return (uint32_t)f32_to_f16(ldexpf(lo16<BF16>(w), shift)) | (uint32_t)f32_to_f16(ldexpf(hi16<BF16>(w), shift)) << 16;
    };
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b.lo[c][i] = turn(b.lo[c][i]);
        b.hi[c][i] = turn(b.hi[c][i]);
      }
    b.mul = ldexpf(1.0f, -shift);
  }
}

// scores of 16 pages (4 grp + r in a lane's result) for 16 rows of query values, raw
template <typename T, int D>
__device__ __forceinline__ f32x4_t page_scores(const PageOperand<T, D>& b, const u32x4_t (&raw)[D / 32],
                                               uint32_t flip) {
  f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    u32x4_t pos, neg;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // (16-bit floats' bits have the sign of whole numbers)
      const s16x2_t v = __builtin_bit_cast(s16x2_t, raw[c][i] ^ flip), zero = {0, 0};
      pos[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(v, zero));
      neg[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(v, zero));
    }
    s = mfma16<T>(b.lo[c], neg, s);
    s = mfma16<T>(b.hi[c], pos, s);
  }
  return s;
}

// One new token a sequence: a group's query heads are the product's 16 columns, and
// the largest of their scores is taken over a row of 16 lanes. A wave has 16 pages of
// one KV head, a workgroup 64. A chain of three round trips, starts, then length and table,
// then bounds and queries: one sequence of 512 pages takes 4.2 us, 64 of up to 512 (39 MB)
// 14.0 to 15.1 (with 32 pages a wave 5.3 and 15.9), where the grid, which the table's width
// makes, is twice what the chip holds and mostly idle.
constexpr int kOnePages = 64;
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_scores_one_kernel(ScoreArgs a) {
  constexpr int NK = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = blockIdx.x % a.Hkv, x = blockIdx.x / a.Hkv, b = x / a.chunks, chunk = x - b * a.chunks;
  const int gqa = a.Hq / a.Hkv;
  const int j0 = chunk * kOnePages + 16 * wave, j = j0 + n16;
  // (asked for beside the length, which says whether it is a page)
  const int id = a.p.table[b * a.p.table_stride + min(j, a.p.width - 1)];
  const SeqRows s = seq_rows(a.p, b);
  if (s.count == 0) return;
  const int t = s.first, lim = last_seen_by(s, 0, a.causal);
  const int pages = lim < 0 ? 0 : (lim >> a.p.page_log2) + 1;
  if (kh == 0 && chunk == 0 && tid == 0) a.seen[t] = pages;
  float* out = a.scores + ((int64_t)t * a.Hkv + kh) * a.p.width;
  if (j0 >= pages) {
    if (grp == 0 && j < a.p.width) out[j] = kNegInf;
    return;
  }
  const bool in = j < pages && (unsigned)id < (unsigned)a.p.pages;
  PageOperand<T, D> page;
  load_bounds<T, D>(a.bounds + (in ? id : 0) * a.b_page + kh * a.b_head + 8 * grp, page);
  f32x4_t most = {kNegInf, kNegInf, kNegInf, kNegInf};
  for (int g0 = 0; g0 < gqa; g0 += 16) {
    const int g = min(g0 + n16, gqa - 1);  // (the last head again for what is past it)
    const uint16_t* row = a.q + t * a.q_tok + (kh * gqa + g) * a.q_head + 8 * grp;
    u32x4_t raw[NK];
#pragma unroll
    for (int c = 0; c < NK; ++c) raw[c] = *reinterpret_cast<const u32x4_t*>(row + 32 * c);
    if (g0 == 0) turn_bounds<T, D>(page);
    const f32x4_t v = page_scores<T, D>(page, raw, a.flip);
#pragma unroll
    for (int r = 0; r < 4; ++r) most[r] = fmaxf(most[r], v[r]);
  }
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = max_row16(most[r]);
  const int k = 4 * grp + n16;  // lane n16 < 4 of a group stores score n16
  const float mul = __shfl(page.mul, k & 63) * a.scale;
  const uint64_t present = __ballot(in);
  if (n16 < 4 && j0 + k < a.p.width) {
    const float m = n16 == 0 ? v[0] : n16 == 1 ? v[1] : n16 == 2 ? v[2] : v[3];
    out[j0 + k] = ((present >> k) & 1) && m != kNegInf ? m * mul : kNegInf;
  }
}

// The tile of 16 new tokens that is number x of the batch's, or b = -1.
struct TokenTile {
  int b, row0;  // sequence, first of its rows
  SeqRows s;
};
__device__ __forceinline__ TokenTile find_tokens(const PagedBatch& p, int max_new, int x) {
  const int lane = threadIdx.x & 63;
  TokenTile t{-1, 0, {0, 0, 0}};
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    SeqRows s{0, 0, 0};
    if (b0 + lane < p.B) s = seq_rows(p, b0 + lane);
    const int tiles = (min(s.count, max_new) + 15) / 16;
    int end = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(end, o);
      if (lane >= o) end += y;
    }
    const unsigned long long hit = __ballot(x < before + end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      t.b = b0 + l;
      t.row0 = 16 * (x - before - __builtin_amdgcn_readlane(end - tiles, l));
      t.s.first = __builtin_amdgcn_readlane(s.first, l);
      t.s.count = __builtin_amdgcn_readlane(s.count, l);
      t.s.length = __builtin_amdgcn_readlane(s.length, l);
      break;
    }
    before += __builtin_amdgcn_readlane(end, 63);
  }
  // (the compiler does not see that a loop left on a ballot leaves scalars)
  for (int* f : {&t.b, &t.row0, &t.s.first, &t.s.count, &t.s.length}) *f = __builtin_amdgcn_readfirstlane(*f);
  return t;
}

// Several new tokens a sequence: 16 of them are the product's columns, one query
// head at a time, and the largest over the group's heads stays in the lane. A wave
// holds the bounds of 32 pages in registers, a workgroup takes 128. 512 new tokens of
// 16384 (512 pages of 32, 20 heads on 4, fp16) take 13.4 us, 200 TFLOP/s: 512 workgroups,
// each a chain of lengths, the first tile's page, its bounds beside the second's page, that
// one's bounds, and then a round trip a head: the compiler loads a head's queries right
// before its products, not beside the ones before. Bounds turned to fp16 (once a wave) and
// queries parted by sign are most of its instructions.
constexpr int kManyPages = 128;
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_scores_many_kernel(ScoreArgs a) {
  constexpr int NK = D / 32, TILES = 2;
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = blockIdx.x % a.Hkv, x = blockIdx.x / a.Hkv, chunk = x % a.chunks;
  const int gqa = a.Hq / a.Hkv;
  const TokenTile tt = find_tokens(a.p, a.max_new, x / a.chunks);
  if (tt.b < 0) return;
  const int rows = min(min(tt.s.count, a.max_new) - tt.row0, 16);
  const int i_row = tt.row0 + min(n16, rows - 1), t = tt.s.first + i_row;
  const int lim = last_seen_by(tt.s, i_row, a.causal);
  const int pages = lim < 0 ? 0 : (lim >> a.p.page_log2) + 1;
  const int most_lim = last_seen_by(tt.s, tt.row0 + rows - 1, a.causal);
  const int most_pages = most_lim < 0 ? 0 : (most_lim >> a.p.page_log2) + 1;
  if (kh == 0 && chunk == 0 && wave == 0 && lane < rows) a.seen[t] = pages;
  const int j0 = chunk * kManyPages + 32 * wave;
  if (j0 >= a.p.width) return;
  f32x4_t most[TILES];
#pragma unroll
  for (int i = 0; i < TILES; ++i) most[i] = f32x4_t{kNegInf, kNegInf, kNegInf, kNegInf};
  float mul[TILES][4] = {};
  uint64_t present[TILES] = {0, 0};
  if (j0 < most_pages) {
    PageOperand<T, D> page[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int j = j0 + 16 * i + n16;
      const int id = j < most_pages ? a.p.table[tt.b * a.p.table_stride + j] : -1;
      const bool in = (unsigned)id < (unsigned)a.p.pages;
      present[i] = __ballot(in);
      load_bounds<T, D>(a.bounds + (in ? id : 0) * a.b_page + kh * a.b_head + 8 * grp, page[i]);
    }
    const uint16_t* row = a.q + t * a.q_tok + kh * gqa * a.q_head + 8 * grp;
    u32x4_t next[NK];
    auto load = [&](int g) {
#pragma unroll
      for (int c = 0; c < NK; ++c) next[c] = *reinterpret_cast<const u32x4_t*>(row + g * a.q_head + 32 * c);
    };
    load(0);
#pragma unroll
    for (int i = 0; i < TILES; ++i) turn_bounds<T, D>(page[i]);
    for (int g = 0; g < gqa; ++g) {
      u32x4_t raw[NK];
#pragma unroll
      for (int c = 0; c < NK; ++c) raw[c] = next[c];
      load(min(g + 1, gqa - 1));
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const f32x4_t v = page_scores<T, D>(page[i], raw, a.flip);
#pragma unroll
        for (int r = 0; r < 4; ++r) most[i][r] = fmaxf(most[i][r], v[r]);
      }
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) mul[i][r] = __shfl(page[i].mul, 4 * grp + r) * a.scale;
  }
  if (n16 >= rows) return;
  float* out = a.scores + ((int64_t)t * a.Hkv + kh) * a.p.width;
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const int j = j0 + 16 * i + 4 * grp;
    f32x4_t v;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      v[r] = j + r < pages && ((present[i] >> (4 * grp + r)) & 1) && most[i][r] != kNegInf ? most[i][r] * mul[i][r] : kNegInf;
    if ((a.p.width & 3) == 0) {
      if (j < a.p.width) *reinterpret_cast<f32x4_t*>(out + j) = v;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j + r < a.p.width) out[j + r] = v[r];
    }
  }
}

template <typename T, int D>
void launch_scores(const ScoreArgs& a, int64_t groups, hipStream_t st) {
  if (a.max_new == 1)
    hipLaunchKernelGGL((paged_scores_one_kernel<T, D>), dim3((unsigned)groups), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_scores_many_kernel<T, D>), dim3((unsigned)groups), dim3(256), 0, st, a);
}

}  // namespace

int paged_key_bounds(const PagedBatch& p, const PagedSide& ks, void* bounds, const int64_t* bst, int64_t H, int64_t D,
                     int64_t max_new, hipStream_t st) {
  if (p.B == 0) return SPARKQ_OK;
  // n new tokens lie in at most ceil((n - 1) / page) + 1 pages
  const int64_t page = 1LL << p.page_log2;
  const int64_t per_row = std::min<int64_t>(cdiv(std::min(max_new, (int64_t)p.width * page) - 1, page) + 1, p.width);
  if (p.B > kMaxGrid / (per_row * H)) return set_error(SPARKQ_ERR_INVALID, "paged_key_bounds: shape too large");
  const BoundsArgs a{p, ks.codes, ks.scales, ks.c_page, ks.c_head, ks.c_tok, ks.s_page, ks.s_head, ks.s_tok,
                     (uint16_t*)bounds, bst[0], bst[1], (int)H, (int)per_row};
  const dim3 grid((unsigned)(p.B * per_row * H));
  if (D == 64)
    hipLaunchKernelGGL(paged_bounds_kernel<64>, grid, dim3(256), 0, st, a);
  else if (D == 128)
    hipLaunchKernelGGL(paged_bounds_kernel<128>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(paged_bounds_kernel<256>, grid, dim3(256), 0, st, a);
  return check_launch("paged_bounds_kernel");
}

int paged_page_scores(const PagedBatch& p, const void* q, const int64_t* qst, const void* bounds, const int64_t* bst,
                      float* scores, int32_t* seen, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int causal,
                      int qdt, float scale, hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  max_new = std::min<int64_t>(max_new, p.T);
  const int64_t chunks = cdiv(p.width, max_new == 1 ? kOnePages : kManyPages);
  const int64_t tiles = max_new == 1 ? p.B : std::min(p.T / 16 + (int64_t)p.B, p.B * cdiv(max_new, 16));
  if (tiles > kMaxGrid / (chunks * Hkv)) return set_error(SPARKQ_ERR_INVALID, "paged_page_scores: shape too large");
  const ScoreArgs a{p, (const uint16_t*)q, qst[0], qst[1], (const uint16_t*)bounds, bst[0], bst[1], scores, seen,
                    (int)Hq, (int)Hkv, (int)max_new, causal, (int)chunks, fabsf(scale),
                    scale < 0.0f ? 0x80008000u : 0u};
  const int64_t groups = tiles * chunks * Hkv;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (D == 64)
      launch_scores<T, 64>(a, groups, st);
    else if (D == 128)
      launch_scores<T, 128>(a, groups, st);
    else
      launch_scores<T, 256>(a, groups, st);
  };
  if (qdt == SPARKQ_BF16)
    go(BF16{});
  else
    go(F16{});
  return check_launch("paged_scores_kernel");
}

}  // namespace sparkq
