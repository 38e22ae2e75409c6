// paged_sparse.hip -- attention of packed new tokens over pages that were selected
// for each of them, from a paged INT8 KV cache (symmetric s8 codes, one fp16 scale
// per token and KV head) on gfx950.
//
//   o[t,h] = sum_n p_n v_n / sum_n p_n,  p_n = exp(scale * q[t,h] . k_n - max)
//
// over the tokens n of the pages that row t's list for its KV head names and that
// it sees. A page that is named twice counts twice; one that lies outside the row's
// table, has no place in the pool or is not seen counts for nothing, and a row that
// is left with nothing is zero.
//
// The query heads of a KV head share a row's list, and so its keys and values: they
// are the 16 columns of the products. Lists differ from token to token, and nothing
// is shared between these.
#include <algorithm>

#include "paged_attn.h"

namespace sparkq {
namespace {

struct SparseArgs {
  PagedSdpaArgs a;      // (of the parts: [row, KV head, tile, part][rows_held])
  const int32_t* list;  // [T, Hkv, count], ascending where select_top made it
  int64_t l_tok, l_head;
  int count, tiles, parts;  // entries; tiles of 16 query heads; parts of a list
  int rows_held;            // rows of a tile that parts have room for
};

constexpr int kListed = 512;  // pages that a workgroup looks up at a time

// The pages of a list that are there, in order: number in the pool, first position.
struct Listed {
  int id[kListed], pos[kListed];
  int n;
};

// Entries [e0, e1) of a list, no more than kListed, looked up by the first wave; j are
// its first 64.
__device__ __forceinline__ void look_up(const SparseArgs& s, Listed& l, const int32_t* list, int b, int lim, int e0,
                                        int e1, int j) {
  const PagedBatch& p = s.a.p;
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int e = e0; e < e1; e += 64) {
    bool in = e + lane < e1 && (unsigned)j < (unsigned)p.width && ((int64_t)j << p.page_log2) <= lim;
    const int id = p.table[b * p.table_stride + (in ? j : 0)];
    in = in && (unsigned)id < (unsigned)p.pages;
    const int at_j = j;
    j = list[min(e + 64 + lane, e1 - 1)];
    const unsigned long long m = __ballot(in);
    if (in) {
      const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
      l.id[at] = id;
      l.pos[at] = at_j << p.page_log2;
    }
    n += __builtin_popcountll(m);
  }
  if (lane == 0) l.n = n;
}

template <int D>
struct SparseLds {
  static constexpr int VROW = D + 16;
  static constexpr int VT = kFewBlock * VROW;        // one wave's V block
  static constexpr int LOOP = 4 * VT;
  static constexpr int JOIN = 4 * 16 * (2 + D) * 4;  // the waves' maxima, sums and outputs
  static constexpr int BYTES = LOOP > JOIN ? LOOP : JOIN;
};

// A block's two runs of 16 tokens: page (0 where there is none, with its bit in ok
// clear), slot, position.
struct Runs {
  int id[2], slot[2], pos[2];
  uint32_t ok;
};

// S^T (16 tokens x 16 rows) = K . Q^T twice a block, O^T (16 dims x 16 rows) += V^T .
// P^T; row m of the first product's operand is token 8 (m / 4) + m % 4 (+ 4 in the
// second), so that the lane with a row's scores of tokens 8g .. 8g+7 holds just the
// k-slots of the second product's operand. The waves take turns at blocks of 32
// tokens of the listed pages, each with the next block's loads in flight and no
// barrier until they join.
// Bytes bound it, 2 (D + 2) a listed token and KV head: 56 decoded tokens with lists of
// 77 pages of 32, 4 KV heads of 256 (196 MB), take 51 us, 3.85 TB/s of the 5.1 that a
// copy reaches: 224 workgroups of four waves are what keeps loads in flight (eight waves:
// 54 us). One sequence of 32 pages of 64, 8 KV heads of 128 (4.3 MB), is latency: 7.3 us,
// and 3.8 for the parts' join; unsplit lists, which need no join, take 24 there with four
// waves, 21 with eight, as a block's 380 vector instructions then follow each other.
template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 3 : 2) void paged_sparse_kernel(SparseArgs s) {
  constexpr int NK = D / 32, PL = D / 64, NJ = D / 16, VL = D / 32;
  using L = SparseLds<D>;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::BYTES];
  __shared__ Listed lst;
  const PagedSdpaArgs& a = s.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, grp = lane >> 4;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv;
  int x = blockIdx.x / a.Hkv;
  const int part = x % s.parts;
  x /= s.parts;
  const int tile = x % s.tiles, t = x / s.tiles;
  const int32_t* list = s.list + t * s.l_tok + kh * s.l_head;
  const int e_first = (int)((int64_t)part * s.count / s.parts), e_end = (int)((int64_t)(part + 1) * s.count / s.parts);
  // (asked for before it is known whose row this is)
  const int j_first = list[min(e_first + lane, s.count - 1)];
  const RowOf ro = wave_row(a.p, t);
  const int b = ro.b;
  if (b < 0) return;
  const SeqRows sq = ro.s;
  const int i_row = t - sq.first;
  if (i_row < 0 || i_row >= min(sq.count, a.max_new)) return;
  const int lim = last_seen_by(sq, i_row, a.causal);
  const int rows = min(gqa - 16 * tile, 16);
  const int head = kh * gqa + 16 * tile + min(n16, rows - 1);
  unsigned char* vtile = smem + wave * L::VT;

  u32x4_t qb[NK];
  const uint16_t* qrow = a.q + t * a.q_tok + head * a.q_head;
  // chunk c: dims 16 (g + 4 (c / 2)) + 8 (c % 2), as the 16-byte pieces of K lie
  const float mul = load_query<NK, 4>(a, qrow, true, [&](int c) { return 16 * (grp + 4 * (c >> 1)) + 8 * (c & 1); }, qb);

  u32x4_t kr[2][PL], vr[VL], skr, svr;
  const int ktok = 8 * (n16 >> 2) + (n16 & 3);
  const uint32_t koff = (ktok & 15) * a.c.c_tok + 16 * grp;
  const uint8_t *const khead = a.c.k + kh * a.c.c_head, *const vhead = a.c.v + kh * a.c.c_head;
  const uint16_t *const kshead = a.c.ks + kh * a.c.s_head, *const vshead = a.c.vs + kh * a.c.s_head;
  const int slot_mask = (1 << a.p.page_log2) - 1;
  int last = 0, listed = 0;  // the wave's last block, pages that are there
  auto runs = [&](int ib) {
    Runs r;
    r.ok = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int v = kFewBlock * ib + 16 * h, e = v >> a.p.page_log2;
      const bool in = e < listed;
      const int at = in ? e : 0;
      r.id[h] = __builtin_amdgcn_readfirstlane(lst.id[at]);
      r.slot[h] = v & slot_mask;
      r.pos[h] = __builtin_amdgcn_readfirstlane(lst.pos[at]) + r.slot[h];
      r.ok |= (uint32_t)in << h;
    }
    return r;
  };
  Runs now, next;
  auto load = [&](const Runs& r) {
    const uint64_t o0 = code_at(a.c, r.id[0], r.slot[0]), o1 = code_at(a.c, r.id[1], r.slot[1]);
    const uint8_t *kp = khead + (n16 < 8 ? o0 : o1) + koff, *v0 = vhead + o0, *v1 = vhead + o1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < PL; ++i)
        kr[h][i] = *reinterpret_cast<const u32x4_t*>(kp + (4 * h * a.c.c_tok + 64 * i));
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      vr[v] = *reinterpret_cast<const u32x4_t*>((2 * v >= VL ? v1 : v0) + ((tok & 15) * a.c.c_tok + 16 * pc));
    }
    const bool h = grp >= 2;
    const uint64_t so = scale_at(a.c, h ? r.id[1] : r.id[0], (h ? r.slot[1] : r.slot[0]) + 8 * (grp & 1));
    skr = *reinterpret_cast<const u32x4_t*>(kshead + so);
    svr = *reinterpret_cast<const u32x4_t*>(vshead + so);
  };

  RowState st;
  f32x4_t acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto block = [&](int ib) {
#pragma unroll
    for (int v = 0; v < VL; ++v) {
      const int f = lane + 64 * v, tok = f / (D / 16), pc = f % (D / 16);
      *reinterpret_cast<u32x4_t*>(vtile + tok * L::VROW + 16 * pc) = vr[v];
    }
    f32x4_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const u32x4_t kp = kr[h][c >> 1];
        sc[h] = mfma16x16x32_f16((c & 1) ? s8x8_exact(kp.z, kp.w) : s8x8_exact(kp.x, kp.y), qb[c], sc[h]);
      }
    }
    float sv[8], vsc[8];
    u16x2_t most = {0, 0};  // the largest scale's bits: finite below those of infinity
    u16x2_t one = {1, 1};   // 0 where a scale is 1
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kw = skr[i >> 1], vw = svr[i >> 1];
      sv[i] = sc[i >> 2][i & 3] * (((i & 1) ? hi16<F16>(kw) : lo16<F16>(kw)) * a.sign);
      vsc[i] = (i & 1) ? hi16<F16>(vw) : lo16<F16>(vw);
      if (i & 1) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, vw & 0x7FFF7FFFu));
        one = __builtin_elementwise_min(one, __builtin_bit_cast(u16x2_t, vw ^ 0x3C003C00u));
      }
    }
    const bool odd = most[0] >= 0x7C00 || most[1] >= 0x7C00 || one[0] == 0 || one[1] == 0;
    if (__builtin_expect(now.pos[0] + 15 > lim || now.pos[1] + 15 > lim || now.ok != 3 || __ballot(odd) != 0, 0)) {
      uint32_t ok = 0;
      const int pos = (grp >= 2 ? now.pos[1] : now.pos[0]) + 8 * (grp & 1);
#pragma unroll
      for (int i = 0; i < 8; ++i) ok |= (uint32_t)(pos + i <= lim) << i;
      if (!((now.ok >> (grp >> 1)) & 1u)) ok = 0;
      ok = __float_as_uint(pinned(__uint_as_float(ok)));
      uint32_t zero = 0;
      if (__ballot(one[0] == 0 || one[1] == 0)) {
        const bool h = (lane & 31) >= 16;
        zero = zero_rows<D, 32>(vhead + code_at(a.c, h ? now.id[1] : now.id[0], (h ? now.slot[1] : now.slot[0]) + n16) +
                                D / 2 * (lane / 32)) >> (8 * grp);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool live = (ok >> i) & 1u;
        sv[i] = live ? sv[i] : kNegInf;
        vsc[i] = live && !(((zero >> i) & 1u) && vsc[i] == 1.0f) ? vsc[i] : 0.0f;
      }
    }
    float top = kNegInf;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaf(sv[i], mul, scale_exp(vsc[i])));
    top = max_groups<4>(top);
    load(next);
    now = next;
    next = runs(min(ib + 8, last));
    u32x4_t w, rest;
    bool up;
    const float alpha = row_block<8, kTopFew, 0, true>(st, sv, mul, vsc, top, &w, &rest, up);
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

  for (int e = e_first; e < e_end; e += kListed) {
    if (e != e_first) __syncthreads();  // the pages looked up before are done with
    if (wave == 0) look_up(s, lst, list, b, lim, e, min(e + kListed, e_end), e == e_first ? j_first : list[min(e + lane, e_end - 1)]);
    __syncthreads();
    listed = __builtin_amdgcn_readfirstlane(lst.n);
    const int blocks = ((listed << a.p.page_log2) + kFewBlock - 1) / kFewBlock;
    last = blocks - 1;
    int ib = wave;
    if (ib >= blocks) continue;
    now = runs(ib);
    load(now);
    next = runs(min(ib + 4, last));
    for (; ib < blocks; ib += 4) block(ib);
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
    if (s.parts == 1) {
      if (zz != 0.0f) o /= zz;
      store_row4(a, ((int64_t)t * a.Hq + kh * gqa + 16 * tile + r) * D + d, o);
    } else {
      const int64_t at = ((((int64_t)t * a.Hkv + kh) * s.tiles + tile) * s.parts + part) * s.rows_held + r;
      *reinterpret_cast<f32x4_t*>(a.pacc + at * D + d) = o;
      if (d == 0) {
        a.pm[at] = mm;
        a.pz[at] = zz;
      }
    }
  }
}

// Joins the parts of a row's list: a workgroup per (row, KV head, tile), a thread
// four dims of one of its heads, eight parts' loads in flight.
template <int D>
__global__ __launch_bounds__(256) void paged_sparse_merge_kernel(SparseArgs s) {
  const PagedSdpaArgs& a = s.a;
  const int kh = blockIdx.x % a.Hkv, gqa = a.Hq / a.Hkv, x = blockIdx.x / a.Hkv;
  const int tile = x % s.tiles, t = x / s.tiles;
  const RowOf ro = wave_row(a.p, t);
  const SeqRows sq = ro.s;
  if (ro.b < 0) return;
  if (t < sq.first || t - sq.first >= min(sq.count, a.max_new)) return;
  const int rows = min(gqa - 16 * tile, 16);
  const int64_t base = ((((int64_t)t * a.Hkv + kh) * s.tiles + tile) * s.parts) * s.rows_held;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 256) {
    const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
    const float *pm = a.pm + base + r, *pz = a.pz + base + r, *pacc = a.pacc + (base + r) * D + d;
    float mm = kNegInf, zz = 0.0f;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < s.parts; k0 += 8) {
      float m[8], z[8];
      f32x4_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t k = (int64_t)min(k0 + u, s.parts - 1) * s.rows_held;
        m[u] = pm[k];
        z[u] = pz[k];
        v[u] = *reinterpret_cast<const f32x4_t*>(pacc + k * D);
      }
      float top = mm;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, m[u]);
      if (top == kNegInf) continue;
      const float f0 = mm == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mm - top);
      zz *= f0;
      o *= f0;
      mm = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (k0 + u >= s.parts || m[u] == kNegInf) continue;
        const float f = __builtin_amdgcn_exp2f(m[u] - top);
        zz = fmaf(z[u], f, zz);
        o += v[u] * f;
      }
    }
    if (zz != 0.0f) o /= zz;
    store_row4(a, ((int64_t)t * a.Hq + kh * gqa + 16 * tile + r) * D + d, o);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct SparsePlan {
  int64_t tiles, parts, rows_held;
};

SparsePlan sparse_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t count, int64_t page) {
  SparsePlan p;
  const int64_t gqa = Hq / Hkv;
  p.tiles = cdiv(gqa, 16);
  p.rows_held = std::min<int64_t>(gqa, 16);
  // Lists are split where there are no more of them than half the CUs, into parts of no
  // less than 128 tokens (a block for each wave). More parts fill the chip better, but joining
  // them costs 4 us: 224 lists of 77 pages of 32 tokens at D = 256 take 51 us whole, 53
  // + 5 in two parts; 56 lists of 32 pages of 64 at D = 128 15 + 4 in four, 17 + 4 in ten.
  // Lists that four waves take about as long for as a join stay whole, one launch less: 8
  // lists of 512 tokens at D = 128 10.6 us (split 9.7), of 256 at D = 256 10.9 (11.7).
  const int64_t most =
      count * page <= (D <= 128 ? 512 : 256) ? 1 : std::min(cdiv(count * page, 128), count);
  p.parts = std::max<int64_t>(std::min(device_cus() / std::max<int64_t>(T * Hkv * p.tiles, 1), most), 1);
  return p;
}

template <int D>
void launch_sparse(const SparseArgs& s, hipStream_t st) {
  const int64_t rows = (int64_t)s.a.p.T * s.a.Hkv * s.tiles;
  hipLaunchKernelGGL(paged_sparse_kernel<D>, dim3((unsigned)(rows * s.parts)), dim3(256), 0, st, s);
  if (s.parts > 1) hipLaunchKernelGGL(paged_sparse_merge_kernel<D>, dim3((unsigned)rows), dim3(256), 0, st, s);
}

}  // namespace

size_t paged_sparse_workspace(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t count, int64_t page) {
  const SparsePlan p = sparse_plan(T, Hq, Hkv, D, count, page);
  return p.parts == 1 ? 0 : (size_t)(T * Hkv * p.tiles * p.parts * p.rows_held * (D + 2)) * sizeof(float);
}

int paged_sparse_sdpa(const PagedBatch& p, const void* q, const int64_t* qst, const PagedSide& ks, const PagedSide& vs,
                      const int32_t* list, const int64_t* lst, int64_t count, void* out, int64_t Hq, int64_t Hkv,
                      int64_t D, int64_t max_new, int causal, int qdt, int odt, float scale, void* ws, size_t wsb,
                      hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  const int64_t page = 1LL << p.page_log2;
  const SparsePlan plan = sparse_plan(p.T, Hq, Hkv, D, count, page);
  const size_t need = paged_sparse_workspace(p.T, Hq, Hkv, D, count, page);
  if (need > 0 && (!ws || wsb < need))
    return set_error(SPARKQ_ERR_WORKSPACE, "paged_sparse_sdpa needs a workspace of %zu bytes (got %zu)", need,
                     ws ? wsb : (size_t)0);
  if (!aligned(ws, 16)) return set_error(SPARKQ_ERR_INVALID, "paged_sparse_sdpa: workspace must be 16-byte aligned");
  if ((int64_t)p.T * Hkv * plan.tiles > kMaxGrid / plan.parts)
    return set_error(SPARKQ_ERR_INVALID, "paged_sparse_sdpa: shape too large");
  const int64_t n = (int64_t)p.T * Hkv * plan.tiles * plan.parts * plan.rows_held;
  float* acc = (float*)ws;
  const CodeLayout c{ks.codes, vs.codes, ks.scales, vs.scales, ks.c_head, ks.s_head, (uint32_t)(ks.c_page / 16),
                     (uint32_t)(ks.s_page / 8), (uint32_t)ks.c_tok};
  SparseArgs s{};
  s.a.p = p;
  s.a.q = (const uint16_t*)q;
  s.a.q_tok = qst[0];
  s.a.q_head = qst[1];
  s.a.c = c;
  s.a.out = out;
  s.a.pacc = acc;
  s.a.pm = acc + n * D;
  s.a.pz = acc + n * (D + 1);
  s.a.Hq = (int)Hq;
  s.a.Hkv = (int)Hkv;
  s.a.max_new = (int)std::min<int64_t>(max_new, p.T);
  s.a.causal = causal;
  s.a.q_dtype = qdt;
  s.a.out_dtype = odt;
  s.a.scale_log2 = fabsf(scale) * 1.44269504088896340736f;
  s.a.sign = scale < 0.0f ? -1.0f : 1.0f;
  s.list = list;
  s.l_tok = lst[0];
  s.l_head = lst[1];
  s.count = (int)count;
  s.tiles = (int)plan.tiles;
  s.parts = (int)plan.parts;
  s.rows_held = (int)plan.rows_held;
  if (D == 64)
    launch_sparse<64>(s, st);
  else if (D == 128)
    launch_sparse<128>(s, st);
  else
    launch_sparse<256>(s, st);
  return check_launch("paged_sparse_sdpa");
}

}  // namespace sparkq
