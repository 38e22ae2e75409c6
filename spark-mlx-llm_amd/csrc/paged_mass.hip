// paged_mass.hip -- the attention weight that the cached tokens of a paged INT8 KV
// cache gather from a batch's new tokens (gfx950):
//
//   mass[b,h,n] += sum_t sum_g exp(scale * q[t,g] . k[h,n] - lse[t,g])
//
// over sequence b's new tokens t that see token n and the query heads g of KV head
// h, with the logarithms of the rows' sums that the attention returned. A batch's
// new tokens start from 0. One workgroup has all rows that see its tokens: every sum
// has one order, and there are no atomics.
#include <algorithm>
#include <type_traits>

#include "paged_attn.h"

namespace sparkq {
namespace {

struct MassArgs {
  PagedSdpaArgs a;   // (no values, no outputs)
  const float* lse;  // [T, Hq]
  float* mass;       // [B, Hkv, tokens], tokens contiguous
  int64_t m_row, m_head;
  int tokens;        // of a row of it
  float scale;       // the softmax scale in log2 units, signed
};

// What a row's logarithm is in log2 units; a row that sees nothing weighs nothing.
__device__ __forceinline__ float row_base(float lse) {
  return lse == kNegInf ? __builtin_huge_valf() : lse * 1.44269504088896340736f;
}

// ---------------------------------------------------------------------------
// at most 64 rows a (sequence, KV head)
// ---------------------------------------------------------------------------
// S^T (16 tokens x 16 rows) = K . Q^T twice a block of 32 tokens and once for each of
// the TILES of 16 rows, the lane with a row's scores of tokens 8g .. 8g+7; the rows'
// weights are summed over the tiles and then over 16 lanes. The waves of a workgroup
// take turns at blocks, each with the next one's loads in flight. Contexts are split
// like the attention's.
// It reads the keys once, D + 2 bytes a token and KV head, and the sums it adds to: of
// one new token each of 64 sequences of up to 8192 (8 KV heads of 128) 103 MB in 28 us,
// where latency and the first blocks' table lookups are what is left. More tiles take
// more products and exponentials a key, and the bytes cease to bind: 48 sequences of 8 new
// tokens and up to 12000 (32 rows) 33 us, the kernel for more rows 93. At 64 rows the two
// meet: 2 sequences of 16 new tokens and up to 12000 17.3 us, there 19.8; with 4 KV heads
// of 256 18.4 and 18.8.
template <int D, int TILES>
__global__ __launch_bounds__(256) void paged_mass_few_kernel(MassArgs s) {
  constexpr int NK = D / 32, PL = D / 64, kBlock = kFewBlock;
  const PagedSdpaArgs& a = s.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, grp = lane >> 4;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  const Item it = find_item<16 * TILES, false>(a, blockIdx.x / a.Hkv);
  if (it.b < 0) return;
  const int rows = it.rows;
  const int all = last_seen(a, it, 0, gqa) + 1;  // seen by every row
  const int nblocks = (it.length + kBlock - 1) / kBlock;
  const int ib0 = (int)((int64_t)it.part * nblocks / it.parts);
  const int ib1 = (int)((int64_t)(it.part + 1) * nblocks / it.parts);
  const TableRow trow = table_row(a, it.b);

  u32x4_t qb[TILES][NK];
  float mul[TILES], base[TILES];
  int lim[TILES];  // (of a row that is none: -1)
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const int r = 16 * i + n16, rr = min(r, rows - 1), rt = rr / gqa;
    const int64_t t = it.first + rt;
    const int head = kh * gqa + rr - rt * gqa;
    mul[i] = a.sign * load_query<NK, 4>(a, a.q + t * a.q_tok + head * a.q_head, true,
                                        [&](int c) { return 16 * (grp + 4 * (c >> 1)) + 8 * (c & 1); }, qb[i]);
    // (a row that is none has the last one's scores, and no weight)
    base[i] = r < rows ? row_base(s.lse[t * a.Hq + head]) : __builtin_huge_valf();
    lim[i] = r < rows ? last_seen(a, it, rr, gqa) : -1;
  }

  u32x4_t kr[2][PL], skr;
  float2 old;
  BlockPages<2> next;
  uint32_t pages_ok;
  const int ktok = 8 * (n16 >> 2) + (n16 & 3);
  const uint32_t koff = (ktok & 15) * a.c.c_tok + 16 * grp;
  const uint8_t* const khead = a.c.k + kh * a.c.c_head;
  const uint16_t* const kshead = a.c.ks + kh * a.c.s_head;
  const int slot_mask = (1 << a.p.page_log2) - 1;
  const int last = ib1 - 1;
  // lane q < 4 of a group has the sums of tokens 8 grp + 2 q, + 1 of a block
  const int off = 8 * grp + 2 * (n16 & 3);
  float* const mine = s.mass + it.b * s.m_row + kh * s.m_head + off;
  const int fresh = it.length - it.count;  // tokens from it on start from 0
  auto load = [&](int ib, const BlockPages<2>& bp) {
    const int t0 = kBlock * min(ib, last);
    const int s0 = t0 & slot_mask, s1 = (t0 + 16) & slot_mask;
    const uint64_t o0 = code_at(a.c, bp.id[0], s0), o1 = code_at(a.c, bp.id[1], s1);
    const uint8_t* kp = khead + (n16 < 8 ? o0 : o1) + koff;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < PL; ++i)
        kr[h][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kp + (4 * h * a.c.c_tok + 64 * i)));
    const bool h = grp >= 2;
    skr = *reinterpret_cast<const u32x4_t*>(kshead + scale_at(a.c, h ? bp.id[1] : bp.id[0], (h ? s1 : s0) + 8 * (grp & 1)));
    old = *reinterpret_cast<const float2*>(mine + (min(t0 + off, s.tokens - 2) - off));
    pages_ok = bp.ok;
  };

  auto block = [&](int ib) {
    const int t0 = kBlock * ib;
    // (one tile's products take the keys as they come, several of them converted once)
    u32x4_t kf[2][NK];
    auto key = [&](int h, int c) {
      const u32x4_t kp = kr[h][c >> 1];
      return (c & 1) ? s8x8_exact(kp.z, kp.w) : s8x8_exact(kp.x, kp.y);
    };
    float ksc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) ksc[i] = (i & 1) ? hi16<F16>(skr[i >> 1]) : lo16<F16>(skr[i >> 1]);
    const uint32_t ok = pages_ok;
    const float2 was = old;
    auto ahead = [&]() {
      load(ib + 4, next);
      next = block_pages<2>(a, trow, kBlock * min(ib + 8, last));
    };
    if constexpr (TILES > 1) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NK; ++c) kf[h][c] = key(h, c);
      ahead();
    }
    const bool hidden = t0 + kBlock > all || ok != 3;
    float p[8];
#pragma unroll
    for (int r = 0; r < TILES; ++r) {
      f32x4_t sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NK; ++c) sc[h] = mfma16x16x32_f16(TILES > 1 ? kf[h][c] : key(h, c), qb[r][c], sc[h]);
      }
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(sc[i >> 2][i & 3] * ksc[i], mul[r], -base[r]));
      if (hidden) {
        const int rel = (ok >> (grp >> 1)) & 1u ? lim[r] - t0 - 8 * grp : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i <= rel ? e[i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = r == 0 ? e[i] : p[i] + e[i];
    }
    if constexpr (TILES == 1) ahead();
    // sums over the 16 lanes: lanes 4k + q end with tokens 2q, 2q + 1
    float h4[4], h2[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // lanes with bit 1 keep tokens 4 .. 7
      const bool up = n16 & 2;
      const float keep = up ? p[4 + i] : p[i], give = up ? p[i] : p[4 + i];
      h4[i] = keep + dpp_row<0x4E>(give);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // bit 0: the upper two of these
      const bool up = n16 & 1;
      const float keep = up ? h4[2 + i] : h4[i], give = up ? h4[i] : h4[2 + i];
      h2[i] = keep + dpp_row<0xB1>(give);
      h2[i] += dpp_row<0x124>(h2[i]);
      h2[i] += dpp_row<0x128>(h2[i]);
    }
    const int at = t0 + 8 * grp + 2 * n16;
    if (n16 < 4) {
      if (at + 1 < it.length) {
        *reinterpret_cast<float2*>(mine + t0) =
            make_float2((at < fresh ? was.x : 0.0f) + h2[0], (at + 1 < fresh ? was.y : 0.0f) + h2[1]);
      } else if (at < it.length) {
        mine[t0] = (at < fresh ? was.x : 0.0f) + h2[0];
      }
    }
  };

  int ib = ib0 + wave;
  if (ib < ib1) {
    load(ib, block_pages<2>(a, trow, kBlock * ib));
    next = block_pages<2>(a, trow, kBlock * min(ib + 4, last));
    for (; ib < ib1; ib += 4) block(ib);
  }
}

// ---------------------------------------------------------------------------
// more rows
// ---------------------------------------------------------------------------
// A wave has 32 tokens of one KV head, their codes in registers as the first operand
// of the 32 x 32 products. The workgroup goes over the rows that see its tokens, kRows
// at a time: it brings their queries into LDS, in one of two buffers, and a wave takes
// tiles of 32 of them as second operands. A lane then has one row's scores of 16
// tokens, and sums its rows' weights in registers; lanes (and waves) are joined at the
// end through LDS. Codes are exact in either 16-bit type, so queries stay as they are.
// WAYS waves share 32 tokens and take turns at the tiles: two, or four where that gives
// less than two workgroups a CU (500 new tokens of 1000, 8 KV heads: four 22 us, two 28;
// 3 sequences of 300 and 6000, 4 KV heads of 256: two 33, four 49). What counts is what the
// tables have room for, as lengths are on the device: those 500 take 28 in a table of 128
// pages of 64.
// What it has to do is the product and an exponential a score: 2048 new tokens of 8192, 32
// heads of 128 on 8, take 150 to 155 us, 780 to 800 TFLOP/s. Nothing is full (vector units
// 65 %, matrix units 42 %, waves wait in 39 % of their time). The next rows' loads are issued
// before this round's tiles, but do not run beside them: the compiler cannot tell the
// buffer that they fill from the one that is read, and waits for them before a tile's first
// read, so each round of two tiles a wave has a round trip to memory in it. Queries go
// straight into LDS: through registers the same tiles take 164 us, as 11 of them spill.
template <typename T>
__device__ __forceinline__ u32x4_t codes_as(uint32_t lo, uint32_t hi);
template <>
__device__ __forceinline__ u32x4_t codes_as<F16>(uint32_t lo, uint32_t hi) {
  return s8x8_exact(lo, hi);
}
template <>
__device__ __forceinline__ u32x4_t codes_as<BF16>(uint32_t lo, uint32_t hi) {
  auto pair = [](uint32_t w, int i) {
    return pack_round<BF16>((float)(int8_t)(w >> (8 * i)), (float)(int8_t)(w >> (8 * i + 8)));
  };
  return u32x4_t{pair(lo, 0), pair(lo, 2), pair(hi, 0), pair(hi, 2)};
}

// The block of `size` tokens that is number x of the batch's sequences with new tokens
struct TokenBlock {
  int b, t0;
  SeqRows s;
};
__device__ __forceinline__ TokenBlock find_block(const PagedBatch& p, int size, int x) {
  const int lane = threadIdx.x & 63;
  TokenBlock r{-1, 0, {0, 0, 0}};
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    SeqRows s{0, 0, 0};
    if (b0 + lane < p.B) s = seq_rows(p, b0 + lane);
    const int n = s.count > 0 ? (s.length + size - 1) / size : 0;
    const int end = before + wave_prefix(n);
    const unsigned long long hit = __ballot(x < end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      r.b = b0 + l;
      r.t0 = size * (x - __builtin_amdgcn_readlane(end - n, l));
      r.s.first = __builtin_amdgcn_readlane(s.first, l);
      r.s.count = __builtin_amdgcn_readlane(s.count, l);
      r.s.length = __builtin_amdgcn_readlane(s.length, l);
      break;
    }
    before = __builtin_amdgcn_readlane(end, 63);
  }
  for (int* f : {&r.b, &r.t0, &r.s.first, &r.s.count, &r.s.length}) *f = __builtin_amdgcn_readfirstlane(*f);
  return r;
}

constexpr int kMassHeads = 128;  // rows of a new token, at most: a round of them
constexpr int mass_tokens(int ways) { return 256 / ways; }  // of a workgroup

template <int D, int WAYS>
struct MassShape {
  static constexpr int ROWS = 128;         // queries in LDS at a time
  static constexpr int BUF = ROWS * 2 * D;
  static constexpr int JOIN = 8 * 32 * 33 * 4;
  static constexpr int BYTES = 2 * BUF > JOIN ? 2 * BUF : JOIN;
  static constexpr int ALIGN = 2 * D;  // of the buffers: a row's pieces are addressed by xor
  static_assert(BUF % ALIGN == 0 && ROWS * ALIGN == BUF, "rows lie at multiples of their size");
  // 16-byte piece p of row r lies at place p ^ turn(r) of its row: any 16 rows' pieces p
  // hit different banks
  static __device__ __forceinline__ int turn(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
};

// Wait for this thread's loads into LDS.
__device__ __forceinline__ void wait_loads() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

template <typename T, int D, int WAYS>
__global__ __launch_bounds__(512, D <= 128 ? 4 : 2) void paged_mass_many_kernel(MassArgs s, int blocks) {
  using S = MassShape<D, WAYS>;
  constexpr int NK = D / 16, N = mass_tokens(WAYS), kRows = S::ROWS;
  constexpr int PPR = D / 8, PPT = kRows * PPR / 512;  // 16-byte pieces of a row, of a thread
  const PagedSdpaArgs& a = s.a;
  __shared__ __attribute__((aligned(S::ALIGN))) unsigned char smem[S::BYTES];
  __shared__ float s_base[2][kRows];
  __shared__ int s_lim[2][kRows];
  __shared__ __attribute__((aligned(16))) float s_scale[N];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, grp = lane >> 5, group = wave / WAYS, way = wave % WAYS;
  const int gqa = a.Hq / a.Hkv, kh = blockIdx.x % a.Hkv;
  const int per = kRows / gqa;  // new tokens of a round
  for (int x = blockIdx.x / a.Hkv; x < blocks; x += gridDim.x / a.Hkv) {
    const TokenBlock tb = find_block(a.p, N, x);
    if (tb.b < 0) return;
    const int t0 = tb.t0, count = min(tb.s.count, a.max_new);
    // the first new token that sees the block's first token
    const int first = min(a.causal ? max(t0 - (tb.s.length - tb.s.count), 0) : 0, count);

    u32x4_t kf[NK];
    const int w0 = t0 + 32 * group, pos = w0 + col;
    {
      const int id = pos < tb.s.length ? page_of(a.p, tb.b, pos) : -1;
      const int at = max(id, 0), slot = pos & ((1 << a.p.page_log2) - 1);
      const uint8_t* kp = a.c.k + kh * a.c.c_head + code_at(a.c, at, slot) + 8 * grp;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const uint2 w = *reinterpret_cast<const uint2*>(kp + 16 * k);
        kf[k] = codes_as<T>(w.x, w.y);
      }
      if (way == 0 && grp == 0)
        s_scale[32 * group + col] = f16_to_f32(a.c.ks[kh * a.c.s_head + scale_at(a.c, at, slot)]) * s.scale;
    }

    // A round is of whole new tokens: `per` of them, all heads of each. Piece i of a
    // thread lies at place tid + 512 i of a buffer. The first kRows threads also bring a
    // row's logarithm and what it sees; rows past a round's own, and past the last new
    // token, see nothing.
    int qt[PPT], qo[PPT];
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int r = (tid + 512 * i) / PPR, rr = min(r, per * gqa - 1);
      qt[i] = rr / gqa;
      qo[i] = (rr - qt[i] * gqa) * (int)a.q_head + 8 * ((tid % PPR) ^ S::turn(r));
    }
    const uint16_t* const qbase = a.q + tb.s.first * a.q_tok + (int64_t)kh * gqa * a.q_head;
    const int q_tok = (int)a.q_tok, lt = tid / gqa;
    const float* const lp = s.lse + (int64_t)tb.s.first * a.Hq + kh * gqa + tid - lt * gqa;
    float base_r;
    int lim_r;
    auto load = [&](int i0, int buf) {  // new tokens i0 .. i0 + per - 1
#pragma unroll
      for (int i = 0; i < PPT; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(qbase + ((int64_t)min(i0 + qt[i], count - 1) * q_tok + qo[i])),
            (__attribute__((address_space(3))) void*)(smem + buf * S::BUF + 8192 * i + 1024 * wave), 16, 0, 0);
      if (tid < kRows) {
        const bool live = lt < per && i0 + lt < count;
        base_r = live ? row_base(lp[(int64_t)(i0 + lt) * a.Hq]) : __builtin_huge_valf();
        lim_r = live ? last_seen_by(tb.s, i0 + lt, a.causal) : -1;
      }
    };
    auto stage = [&](int buf) {
      if (tid < kRows) {
        s_base[buf][tid] = base_r;
        s_lim[buf][tid] = lim_r;
      }
      wait_loads();
    };
    float sum[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) sum[v] = 0.0f;
    auto tile = [&](int buf, int r, bool whole) {  // rows r .. r + 31 of a buffer
      // (16 ((2 k + grp) ^ turn) is 32 k ^ 16 (grp ^ turn), and below the 2 D that rows are
      // aligned to: one address, where the compiler would keep one for each k)
      uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem + buf * S::BUF +
                    (r + col) * 2 * D + 16 * (grp ^ S::turn(r + col));
      asm volatile("" : "+v"(at));
      constexpr int AHEAD = 4;  // operands on the way
      u32x4_t q[AHEAD];
      auto read = [&](int k) { return *(__attribute__((address_space(3))) const u32x4_t*)(uintptr_t)(at ^ (32 * k)); };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) q[k] = read(k);
      const float base = s_base[buf][r + col];
      // (in the compiler's own order every product waits for its operand)
      __builtin_amdgcn_sched_barrier(0);
      f32x16_t sc = f32x16_t{};
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        sc = mfma32x32x16<T>(kf[k], q[k % AHEAD], sc);
        if (k + AHEAD < NK) q[k % AHEAD] = read(k + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(s_scale + 32 * group + 2 * v + 4 * grp);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[v + i] = __builtin_amdgcn_exp2f(fmaf(sc[v + i], k4[i], -base));
      }
      if (__builtin_expect(!whole, 0)) {
        const int rel = s_lim[buf][r + col] - w0 - 4 * grp;  // of this lane's tokens (mfma32_row)
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = 8 * (v >> 2) + (v & 3) <= rel ? sc[v] : 0.0f;
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) sum[v] += sc[v];
    };
    if (first < count) {
      load(first, 0);
      stage(0);
      __syncthreads();
      for (int i0 = first, buf = 0; i0 < count; i0 += per, buf ^= 1) {
        load(i0 + per, buf ^ 1);
        // whether these rows see all of this wave's tokens: the first sees the least
        const bool whole = i0 + per <= count && last_seen_by(tb.s, i0, a.causal) >= w0 + 31;
        const int live = min(per, count - i0) * gqa;
#pragma unroll 1
        for (int r = 32 * way; r < live; r += 32 * WAYS) tile(buf, r, whole);
        stage(buf ^ 1);
        __syncthreads();
      }
    }
    float(*join)[32][33] = reinterpret_cast<float(*)[32][33]>(smem);
#pragma unroll
    for (int v = 0; v < 16; ++v) join[wave][mfma32_row(lane, v)][col] = sum[v];
    __syncthreads();
    // 512 / N threads a token: half of a wave's sums each
    const int tok = tid / (512 / N), h = tid % (512 / N);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += join[tok / 32 * WAYS + h / 2][tok % 32][16 * (h & 1) + i];
    v += dpp_row<0xB1>(v);
    v += dpp_row<0x4E>(v);
    if (WAYS == 4) v += dpp_row<0x141>(v);
    if (h == 0 && t0 + tok < tb.s.length) {
      float* m = s.mass + tb.b * s.m_row + kh * s.m_head + t0 + tok;
      const bool in = page_of(a.p, tb.b, t0 + tok) >= 0;
      *m = (t0 + tok < tb.s.length - tb.s.count ? *m : 0.0f) + (in ? v : 0.0f);
    }
    __syncthreads();
  }
}

template <int D>
void launch_few(const MassArgs& s, int tiles, int64_t items, hipStream_t st) {
  const dim3 grid((unsigned)(items * s.a.Hkv));
  if (tiles == 1)
    hipLaunchKernelGGL((paged_mass_few_kernel<D, 1>), grid, dim3(256), 0, st, s);
  else if (tiles == 2)
    hipLaunchKernelGGL((paged_mass_few_kernel<D, 2>), grid, dim3(256), 0, st, s);
  else
    hipLaunchKernelGGL((paged_mass_few_kernel<D, 4>), grid, dim3(256), 0, st, s);
}
template <typename T, int D>
void launch_many(const MassArgs& s, bool share, int64_t items, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)(items * s.a.Hkv));
  if (share)
    hipLaunchKernelGGL((paged_mass_many_kernel<T, D, 4>), grid, dim3(512), 0, st, s, (int)blocks);
  else
    hipLaunchKernelGGL((paged_mass_many_kernel<T, D, 2>), grid, dim3(512), 0, st, s, (int)blocks);
}

}  // namespace

int paged_kv_mass(const PagedBatch& p, const void* q, const int64_t* qst, const float* lse, const PagedSide& ks,
                  float* mass, const int64_t* mst, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int causal,
                  int qdt, float scale, hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  max_new = std::min<int64_t>(max_new, p.T);
  const int64_t gqa = Hq / Hkv, max_tokens = (int64_t)p.width << p.page_log2;
  if (gqa > kMassHeads)
    return set_error(SPARKQ_ERR_UNSUPPORTED, "paged_kv_mass: at most %d query heads to a KV head (got %lld)", kMassHeads,
                     (long long)gqa);
  MassArgs s{};
  s.a.p = p;
  s.a.q = (const uint16_t*)q;
  s.a.q_tok = qst[0];
  s.a.q_head = qst[1];
  s.a.c = CodeLayout{ks.codes, nullptr, ks.scales, nullptr, ks.c_head, ks.s_head, (uint32_t)(ks.c_page / 16),
                     (uint32_t)(ks.s_page / 8), (uint32_t)ks.c_tok};
  s.a.Hq = (int)Hq;
  s.a.Hkv = (int)Hkv;
  s.a.max_new = (int)max_new;
  s.a.causal = causal;
  s.a.q_dtype = qdt;
  s.a.scale_log2 = fabsf(scale) * 1.44269504088896340736f;
  s.a.sign = scale < 0.0f ? -1.0f : 1.0f;
  s.lse = lse;
  s.mass = mass;
  s.m_row = mst[0];
  s.m_head = mst[1];
  s.tokens = (int)max_tokens;
  s.scale = scale * 1.44269504088896340736f;
  if (max_new * gqa <= 64) {
    const int tiles = max_new * gqa <= 16 ? 1 : max_new * gqa <= 32 ? 2 : 4;
    // (as the attention's plan: B sequences of one tile, and the parts of split contexts,
    // about as many as the chip holds at once)
    s.a.min_part = 128;
    s.a.target = (int)std::min<int64_t>(cdiv((tiles == 1 ? 4 : 2) * device_cus(), Hkv), 512);
    const int64_t split = max_tokens > 128 ? std::min<int64_t>(p.B, s.a.target) : 0;
    s.a.slots = (int)std::min<int64_t>(2 * s.a.target, split * cdiv(max_tokens, 128));
    const int64_t items = s.a.slots + p.B;
    if (items > kMaxGrid / Hkv) return set_error(SPARKQ_ERR_INVALID, "paged_kv_mass: shape too large");
    if (D == 64)
      launch_few<64>(s, tiles, items, st);
    else if (D == 128)
      launch_few<128>(s, tiles, items, st);
    else
      launch_few<256>(s, tiles, items, st);
    return check_launch("paged_mass_few_kernel");
  }
  const bool share = p.B * cdiv(max_tokens, mass_tokens(2)) * Hkv < 2 * device_cus();
  const int64_t blocks = p.B * cdiv(max_tokens, mass_tokens(share ? 4 : 2));
  if (blocks > 0x7FFFFFFF) return set_error(SPARKQ_ERR_INVALID, "paged_kv_mass: shape too large");
  // no more workgroups than the chip holds a few times over; they take further blocks
  const int64_t items = std::min(blocks, cdiv(8 * device_cus(), Hkv));
  auto go = [&](auto t) {
    using T = decltype(t);
    if (D == 64)
      launch_many<T, 64>(s, share, items, blocks, st);
    else if (D == 128)
      launch_many<T, 128>(s, share, items, blocks, st);
    else
      launch_many<T, 256>(s, share, items, blocks, st);
  };
  if (qdt == SPARKQ_BF16)
    go(BF16{});
  else
    go(F16{});
  return check_launch("paged_mass_many_kernel");
}

}  // namespace sparkq
