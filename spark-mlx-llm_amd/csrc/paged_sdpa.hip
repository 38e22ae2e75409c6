// paged_sdpa.hip -- attention of packed new tokens over a paged INT8 KV cache
// (symmetric s8 codes, one fp16 scale per token and KV head) on gfx950.
//
//   o[t,h] = sum_n p_n v_n / sum_n p_n,  p_n = exp(scale * q[t,h] . k_n - max)
//
// over the tokens n that row t of sequence b sees: n <= length - count + (t -
// first) under the causal mask, n < length without. Tokens of an absent page
// are hidden, and a row that sees nothing is zero.
#include <algorithm>

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
  int Hq, Hkv, max_new, causal, q_dtype, out_dtype;
  float scale_log2;
};

// One wave per (packed row, query head), 64 tokens at a time: lane n scores
// token n, then lane d sums dim d over the 64 weighted values.
template <int D>
__global__ __launch_bounds__(256) void paged_sdpa_row_kernel(PagedSdpaArgs a) {
  constexpr int E = D / 64;
  __shared__ float sq[4][D];
  __shared__ float sp[4][64];
  __shared__ int64_t sv[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  const int t = (int)(row / a.Hq), h = (int)(row - (int64_t)t * a.Hq), kh = h / (a.Hq / a.Hkv);
  int b = -1;
  SeqRows s{0, 0, 0};
  if (t < a.p.T)
    for (int i = 0; i < a.p.B; ++i) {
      s = seq_rows(a.p, i);
      if (t >= s.first && t < s.first + min(s.count, a.max_new)) {
        b = i;
        break;
      }
    }
  const int end = b < 0 ? 0 : (a.causal ? s.length - s.count + (t - s.first) + 1 : s.length);
  if (b >= 0)
    for (int d = lane; d < D; d += 64)
      sq[wave][d] = load_in(a.q, t * a.q_tok + h * a.q_head + d, a.q_dtype) * a.scale_log2;
  float m = kNegInf, z = 0.0f, acc[E] = {};
  for (int n0 = 0; n0 < end; n0 += 64) {
    const int n = n0 + lane;
    const int id = n < end ? page_of(a.p, b, n) : -1;
    const int slot = n & ((1 << a.p.page_log2) - 1);
    float sc = kNegInf, vs = 0.0f;
    int64_t vo = 0;
    if (id >= 0) {
      const int8_t* kp = (const int8_t*)a.ks.codes + id * a.ks.c_page + kh * a.ks.c_head + slot * a.ks.c_tok;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(sq[wave][d], (float)kp[d], dot);
      sc = dot * f16_to_f32(a.ks.scales[id * a.ks.s_page + kh * a.ks.s_head + slot * a.ks.s_tok]);
      vs = f16_to_f32(a.vs.scales[id * a.vs.s_page + kh * a.vs.s_head + slot * a.vs.s_tok]);
      vo = id * a.vs.c_page + kh * a.vs.c_head + slot * a.vs.c_tok;
    }
    float mb = sc;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mb = fmaxf(mb, __shfl_xor(mb, o));
    mb = fmaxf(mb, m);
    const float alpha = exp2_guarded(m - mb, m != kNegInf);
    m = mb;
    const float p = id >= 0 ? exp2_guarded(sc - mb, sc != kNegInf) : 0.0f;
    z = z * alpha + wave_sum(p);
    sp[wave][lane] = id >= 0 ? p * vs : 0.0f;
    sv[wave][lane] = vo;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= alpha;
    const int live = min(64, end - n0);
    for (int i = 0; i < live; ++i) {
      const int8_t* vp = (const int8_t*)a.vs.codes + sv[wave][i];
      const float w = sp[wave][i];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(w, (float)vp[lane + 64 * e], acc[e]);
    }
  }
  if (b < 0) return;
#pragma unroll
  for (int e = 0; e < E; ++e)
    store_out(a.out, row * D + lane + 64 * e, z != 0.0f ? acc[e] / z : 0.0f, a.out_dtype);
}

}  // namespace

size_t paged_sdpa_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int paged_sdpa(const PagedBatch& p, const void* q, const int64_t* qst, const PagedSide& ks,
               const PagedSide& vs, void* out, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
               int causal, int qdt, int odt, float scale, void* ws, size_t wsb, hipStream_t st) {
  if (p.T == 0 || p.B == 0) return SPARKQ_OK;
  const PagedSdpaArgs a{p, (const uint16_t*)q, qst[0], qst[1], ks, vs, out, (int)Hq, (int)Hkv,
                        (int)max_new, causal, qdt, odt, scale * 1.44269504088896340736f};
  const dim3 grid((unsigned)cdiv((int64_t)p.T * Hq, 4));
  if (D == 64)
    hipLaunchKernelGGL(paged_sdpa_row_kernel<64>, grid, dim3(256), 0, st, a);
  else if (D == 128)
    hipLaunchKernelGGL(paged_sdpa_row_kernel<128>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(paged_sdpa_row_kernel<256>, grid, dim3(256), 0, st, a);
  return check_launch("paged_sdpa_row_kernel");
}

}  // namespace sparkq
