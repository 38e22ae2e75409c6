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
  int Hq, Hkv, D, dims;
  bool pos64, traditional;
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

// Head dims of 64 to 512 (a power of two), dims a multiple of 8, 8-byte aligned
// heads: D / 8 lanes a head, each with both halves of four rotary pairs (or, past
// the rotated dims, eight plain values), so that a head is one load, one
// reduction over its lanes and one store. A workgroup takes 256 / (dims / 2)
// tokens (at least one), computes their angles once into LDS, one per thread and
// pair (an fp64 power and a sine: as dear as a head's whole work), and shares
// them among all heads; with few tokens a token's heads are dealt to several
// workgroups. Four heads of loads in flight a lane. Bound by HBM at length: 4096
// tokens of 32 + 8 heads of 128 (84 MB read and written) in 18.1 us, 4.6 TB/s, where
// the kernel below, which finds every head's angles itself, takes 61; one token 3.9 us.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs a, int toks) {
  constexpr int RPP = 256 / LPR, U = 4;
  __shared__ float2 cs[256];
  const int tid = threadIdx.x, l = tid % LPR, half = a.dims >> 1, H = a.Hq + a.Hkv;
  const int64_t t0 = (int64_t)blockIdx.x * toks;
  const int n = (int)min((int64_t)toks, a.T - t0), rows = n * H;
  if (tid < n * half) cs[tid] = rotation(a, position(a, t0 + tid / half), tid % half);
  // this lane's dims: da .. +4 and db .. +4; pairs i0 .. +4 where it rotates
  const bool rot = 8 * l < a.dims;
  const int i0 = 4 * l;
  const int da = a.traditional || !rot ? 8 * l : i0, db = a.traditional || !rot ? 8 * l + 4 : half + i0;
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wq[i] = T::to_f32(a.wq[da + i]);
    wq[4 + i] = T::to_f32(a.wq[db + i]);
    wk[i] = T::to_f32(a.wk[da + i]);
    wk[4 + i] = T::to_f32(a.wk[db + i]);
  }
  __syncthreads();
  for (int r0 = blockIdx.y * (RPP * U) + tid / LPR; r0 < rows; r0 += gridDim.y * (RPP * U)) {
    uint2 xa[U], xb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = min(r0 + u * RPP, rows - 1), t = r / H, h = r - t * H;
      const uint16_t* x = h < a.Hq ? a.q + (t0 + t) * a.q_tok + h * a.q_head
                                   : a.k + (t0 + t) * a.k_tok + (h - a.Hq) * a.k_head;
      xa[u] = *reinterpret_cast<const uint2*>(x + da);
      xb[u] = *reinterpret_cast<const uint2*>(x + db);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = min(r0 + u * RPP, rows - 1), t = r / H, h = r - t * H;
      float y[8] = {lo16<T>(xa[u].x), hi16<T>(xa[u].x), lo16<T>(xa[u].y), hi16<T>(xa[u].y),
                    lo16<T>(xb[u].x), hi16<T>(xb[u].x), lo16<T>(xb[u].y), hi16<T>(xb[u].y)};
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
      const float inv = rsqrtf(ss / (float)(8 * LPR) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= inv * (h < a.Hq ? wq[i] : wk[i]);
      if (rot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 c = cs[t * half + i0 + i];
          float& ya = a.traditional ? y[2 * i] : y[i];
          float& yb = a.traditional ? y[2 * i + 1] : y[4 + i];
          const float za = ya * c.x - yb * c.y;
          yb = ya * c.y + yb * c.x;
          ya = za;
        }
      }
      if (r0 + u * RPP < rows) {
        uint16_t* out = h < a.Hq ? a.qo + ((t0 + t) * a.Hq + h) * a.D : a.ko + ((t0 + t) * a.Hkv + h - a.Hq) * a.D;
        *reinterpret_cast<uint2*>(out + da) = make_uint2(pack_round<T>(y[0], y[1]), pack_round<T>(y[2], y[3]));
        *reinterpret_cast<uint2*>(out + db) = make_uint2(pack_round<T>(y[4], y[5]), pack_round<T>(y[6], y[7]));
      }
    }
  }
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

template <typename T, int LPR>
void launch_lanes(const QkArgs& a, hipStream_t st) {
  const int64_t H = a.Hq + a.Hkv;
  // half <= 256 as D <= 512; fewer tokens a workgroup where there are few
  const int64_t toks = std::min<int64_t>(256 / (a.dims / 2), a.T), groups = cdiv(a.T, toks);
  const int64_t y = std::min(cdiv(4 * device_cus(), groups), cdiv(toks * H, 256 / LPR * 4));
  hipLaunchKernelGGL((qk_norm_rope_kernel<T, LPR>), dim3((unsigned)groups, (unsigned)y), dim3(256), 0, st, a,
                     (int)toks);
}

template <typename T>
void launch_qk(const QkArgs& a, hipStream_t st) {
  const bool even = ((a.q_tok | a.q_head | a.k_tok | a.k_head) & 3) == 0 && aligned(a.q, 8) && aligned(a.k, 8) &&
                    aligned(a.qo, 8) && aligned(a.ko, 8);
  if (even && a.dims % 8 == 0 && a.T * (a.Hq + a.Hkv) <= 0x7FFFFFFF) {
    if (a.D == 64) return launch_lanes<T, 8>(a, st);
    if (a.D == 128) return launch_lanes<T, 16>(a, st);
    if (a.D == 256) return launch_lanes<T, 32>(a, st);
    if (a.D == 512) return launch_lanes<T, 64>(a, st);
  }
  hipLaunchKernelGGL(qk_norm_rope_row_kernel<T>, dim3((unsigned)cdiv(a.T * (a.Hq + a.Hkv), 4)), dim3(256), 0, st, a);
}

}  // namespace

int qk_norm_rope(const void* q, const void* k, const void* wq, const void* wk, const void* pos,
                 int pos64, void* qo, void* ko, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                 int dims, int traditional, float eps, double base, double scale, int dt,
                 const int64_t* st, hipStream_t stream) {
  if (T == 0) return SPARKQ_OK;
  const QkArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)wq, (const uint16_t*)wk,
                 pos, (uint16_t*)qo, (uint16_t*)ko, st[0], st[1], st[2], st[3], T, (int)Hq,
                 (int)Hkv, (int)D, dims, pos64 != 0, traditional != 0, eps, log2(base),
                 scale * 0.15915494309189533577};
  if (dt == SPARKQ_BF16)
    launch_qk<BF16>(a, stream);
  else
    launch_qk<F16>(a, stream);
  return check_launch("qk_norm_rope");
}

}  // namespace sparkq
