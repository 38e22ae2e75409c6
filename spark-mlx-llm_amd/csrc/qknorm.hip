// qknorm.hip -- RMS norm of every query and key head with the rotary position
// embedding in the same pass (gfx950).
//
//   y = x * rsqrt(mean(x^2) + eps) * w            over one head's D values
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t),
//   t = scale * pos * base^(-2i/dims),  pair i = (i, i + dims/2) or (2i, 2i+1)
//
// Everything is fp32 and rounded to the 16-bit type once, at the store. The
// angle is taken in turns in fp64 and reduced there: at position 131071 an
// fp32 product alone is off by 0.008 rad.
#include <algorithm>

#include "common.h"

namespace sparkq {
namespace {

struct QkArgs {
  const uint16_t *q, *k, *wq, *wk;
  const void* pos;
  uint16_t *qo, *ko;
  int64_t q_tok, q_head, k_tok, k_head;  // input strides (elements)
  int64_t T;
  int Hq, Hkv, D, dims, pos64, traditional;
  float eps;
  double log2_base, turns;  // turns = scale / (2 pi)
};

__device__ __forceinline__ double position(const QkArgs& a, int64_t t) {
  return a.pos64 ? (double)reinterpret_cast<const int64_t*>(a.pos)[t]
                 : (double)reinterpret_cast<const int32_t*>(a.pos)[t];
}

// cos and sin of pair i at a position
__device__ __forceinline__ float2 rotation(const QkArgs& a, double pos, int i) {
  double t = pos * a.turns * exp2(-2.0 * i / a.dims * a.log2_base);
  t -= rint(t);
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  return make_float2(c, s);
}

// Any head dim, any even dims, any alignment: one wave per head.
template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_row_kernel(QkArgs a) {
  const int lane = threadIdx.x & 63, H = a.Hq + a.Hkv, half = a.dims >> 1;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.T * H) return;
  const int64_t t = row / H;
  const int h = (int)(row - t * H);
  const bool isq = h < a.Hq;
  const uint16_t* x = isq ? a.q + t * a.q_tok + h * a.q_head : a.k + t * a.k_tok + (h - a.Hq) * a.k_head;
  const uint16_t* w = isq ? a.wq : a.wk;
  uint16_t* out = isq ? a.qo + (t * a.Hq + h) * a.D : a.ko + (t * a.Hkv + h - a.Hq) * a.D;
  float ss = 0.0f;
  for (int d = lane; d < a.D; d += 64) {
    const float v = T::to_f32(x[d]);
    ss = fmaf(v, v, ss);
  }
  const float r = rsqrtf(wave_sum(ss) / (float)a.D + a.eps);
  const double pos = position(a, t);
  for (int i = lane; i < half + (a.D - a.dims); i += 64) {
    if (i >= half) {
      const int d = a.dims + (i - half);
      out[d] = T::from_f32(T::to_f32(x[d]) * r * T::to_f32(w[d]));
      continue;
    }
    const int da = a.traditional ? 2 * i : i, db = a.traditional ? 2 * i + 1 : i + half;
    const float2 cs = rotation(a, pos, i);
    const float ya = T::to_f32(x[da]) * r * T::to_f32(w[da]), yb = T::to_f32(x[db]) * r * T::to_f32(w[db]);
    out[da] = T::from_f32(ya * cs.x - yb * cs.y);
    out[db] = T::from_f32(ya * cs.y + yb * cs.x);
  }
}

}  // namespace

int qk_norm_rope(const void* q, const void* k, const void* wq, const void* wk, const void* pos,
                 int pos64, void* qo, void* ko, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                 int dims, int traditional, float eps, double base, double scale, int dt,
                 const int64_t* st, hipStream_t stream) {
  if (T == 0) return SPARKQ_OK;
  const QkArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)wq, (const uint16_t*)wk,
                 pos, (uint16_t*)qo, (uint16_t*)ko, st[0], st[1], st[2], st[3], T, (int)Hq,
                 (int)Hkv, (int)D, dims, pos64, traditional, eps, log2(base),
                 scale * 0.15915494309189533577};
  const dim3 grid((unsigned)cdiv(T * (Hq + Hkv), 4));
  if (dt == SPARKQ_BF16)
    hipLaunchKernelGGL(qk_norm_rope_row_kernel<BF16>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(qk_norm_rope_row_kernel<F16>, grid, dim3(256), 0, stream, a);
  return check_launch("qk_norm_rope_row_kernel");
}

}  // namespace sparkq
