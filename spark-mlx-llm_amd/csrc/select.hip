// select.hip -- the largest values of many rows, as a list of their places
// (gfx950): pages for a query to attend, tokens for a cache to keep.
//
// A row's values are ordered as whole numbers (`key`), and the k-th largest key is
// found from its leading bits on, by counting. What is larger than that key is taken,
// and of what is equal to it the first that there is room for, so ties go to the
// lowest place. Counts are whole numbers: nothing depends on an order of additions.
#include <algorithm>

#include "common.h"

namespace sparkq {
namespace {

struct SelectArgs {
  const float* x;          // [layers, rows, heads, n], n contiguous
  const int32_t* lengths;  // [rows] or null
  int32_t* out;            // [layers, rows, heads, count]
  int64_t x_layer, x_row, x_head;  // elements
  int64_t total;                   // layers * rows * heads
  int rows, heads, n, count, first, last;
};

// Whole numbers in the order of the values; 0 is left for what is no value. -inf
// stands for NaN, 0 for -0; a place that has to be taken comes before +inf.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v == v)) v = -__builtin_huge_valf();
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectRow {
  const float* x;
  int32_t* out;
  int n, k;  // values, how many of them are taken
  int late;  // the first of the last places, which have to be taken
};
__device__ __forceinline__ SelectRow select_row(const SelectArgs& a, int64_t i) {
  const int64_t lr = i / a.heads, h = i - lr * a.heads, l = lr / a.rows, r = lr - l * a.rows;
  SelectRow s;
  s.x = a.x + l * a.x_layer + r * a.x_row + h * a.x_head;
  s.out = a.out + i * a.count;
  s.n = a.lengths ? min(max(a.lengths[r], 0), a.n) : a.n;
  s.k = min(a.count, s.n);
  s.late = s.n - a.last;
  return s;
}
__device__ __forceinline__ uint32_t key_at(const SelectArgs& a, const SelectRow& s, int i, float v) {
  return i >= s.n ? 0u : (i < a.first || i >= s.late) ? 0xFFFFFFFFu : key_of(v);
}

__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// ---------------------------------------------------------------------------
// a wave a row: rows of up to 64 * KPT values, which stay in registers
// ---------------------------------------------------------------------------
// A bit at a time: it is set in the k-th key if k keys have it and the bits so far.
template <int KPT>
__global__ __launch_bounds__(256) void select_wave_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= a.total) return;
  const SelectRow s = select_row(a, i);
  if (s.n <= s.k) {
    for (int j = lane; j < a.count; j += 64) s.out[j] = j < s.k ? j : -1;
    return;
  }
  uint32_t key[KPT];
  {
    float v[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) v[u] = s.x[min(64 * u + lane, s.n - 1)];
#pragma unroll
    for (int u = 0; u < KPT; ++u) key[u] = key_at(a, s, 64 * u + lane, v[u]);
  }
  uint32_t theta = 0;
  int taken = 0;  // keys that are at least theta (once a bit is set)
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = theta | 1u << bit;
    int c = 0;
#pragma unroll
    for (int u = 0; u < KPT; ++u) c += __builtin_popcountll(__ballot(key[u] >= cand));
    if (c >= s.k) {
      theta = cand;
      taken = c;
      if (c == s.k) break;
    }
  }
  // taken > k: theta is the k-th key itself, and the last of its equals are left out
  int equal = 0x7FFFFFFF;
  if (taken != s.k) {
    equal = s.k;
#pragma unroll
    for (int u = 0; u < KPT; ++u) equal -= __builtin_popcountll(__ballot(key[u] > theta));
  }
  int at = 0;
#pragma unroll
  for (int u = 0; u < KPT; ++u) {
    const unsigned long long eq = __ballot(key[u] == theta);
    const bool take = key[u] > theta || (key[u] == theta && lanes_below(eq) < equal);
    equal -= __builtin_popcountll(eq);
    const unsigned long long m = __ballot(take);
    if (take) s.out[at + lanes_below(m)] = 64 * u + lane;
    at += __builtin_popcountll(m);
  }
  for (int j = s.k + lane; j < a.count; j += 64) s.out[j] = -1;
}

// ---------------------------------------------------------------------------
// a workgroup a row
// ---------------------------------------------------------------------------
// Wave w has the places [w per, (w + 1) per), 64 KPT of them at a time: rows of up to
// 1024 KPT values stay in registers, longer ones are read again for every pass.
constexpr int kSelectWaves = 16, kBins = 2048;
template <int KPT, bool HELD>
struct SelectKeys {
  uint32_t key[KPT];
  int w0, w1;  // this wave's places

  __device__ __forceinline__ void load(const SelectArgs& a, const SelectRow& s, int i0, int lane) {
    float v[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) v[u] = s.x[min(i0 + 64 * u + lane, s.n - 1)];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int i = i0 + 64 * u + lane;
      key[u] = i < w1 ? key_at(a, s, i, v[u]) : 0u;
    }
  }
  // f(keys' place, this) for the wave's keys in order
  template <typename F>
  __device__ __forceinline__ void each(const SelectArgs& a, const SelectRow& s, int lane, F f) {
    if (HELD) {
      f(w0);
    } else {
      for (int i0 = w0; i0 < w1; i0 += 64 * KPT) {
        load(a, s, i0, lane);
        f(i0);
      }
    }
  }
};

template <int KPT, bool HELD>
__global__ __launch_bounds__(64 * kSelectWaves) void select_group_kernel(SelectArgs a) {
  __shared__ int s_bins[kBins], s_pick[3], s_count[2][kSelectWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SelectRow s = select_row(a, blockIdx.x);
  if (s.n <= s.k) {
    for (int j = tid; j < a.count; j += 64 * kSelectWaves) s.out[j] = j < s.k ? j : -1;
    return;
  }
  SelectKeys<KPT, HELD> keys;
  const int per = (s.n + 64 * kSelectWaves - 1) / (64 * kSelectWaves) * 64;
  keys.w0 = min(wave * per, s.n);
  keys.w1 = min(keys.w0 + per, s.n);
  if (HELD) keys.load(a, s, keys.w0, lane);
  // The k-th largest key by digits of 11, 11 and 10 bits: how many of the keys with
  // the digits found so far have each next one, and down from the largest which digit
  // the k-th has.
  uint32_t prefix = 0, theta = 0;
  int need = s.k;  // its place among the keys with the digits so far
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int above = 32 - 11 * pass, shift = max(above - 11, 0);
    for (int d = tid; d < kBins; d += 64 * kSelectWaves) s_bins[d] = 0;
    __syncthreads();
    keys.each(a, s, lane, [&](int) {
#pragma unroll
      for (int u = 0; u < KPT; ++u) {
        const uint32_t key = keys.key[u];
        const bool in = pass == 0 ? key != 0 : key >> above == prefix;
        if (in) atomicAdd(&s_bins[(key >> shift) & ((1u << (above - shift)) - 1)], 1);
      }
    });
    __syncthreads();
    // two digits a thread, from the largest down
    const int d = kBins - 1 - 2 * tid;
    const int c0 = s_bins[d], c1 = s_bins[d - 1];
    int before = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(before, o);
      if (lane >= o) before += y;
    }
    if (lane == 63) s_count[0][wave] = before;
    __syncthreads();
    before -= c0 + c1;
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) before += w < wave ? s_count[0][w] : 0;
    if (before < need && need <= before + c0 + c1) {
      const bool second = need > before + c0;
      s_pick[0] = d - second;
      s_pick[1] = need - before - (second ? c0 : 0);
      s_pick[2] = second ? c1 : c0;
    }
    __syncthreads();
    prefix = pass == 0 ? s_pick[0] : prefix << (above - shift) | s_pick[0];
    need = s_pick[1];
    theta = prefix << shift;
    if (need == s_pick[2]) {  // all keys with these digits are taken
      --theta;
      break;
    }
  }
  // what each wave has that is larger, and equal
  int more = 0, same = 0;
  keys.each(a, s, lane, [&](int) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      more += __builtin_popcountll(__ballot(keys.key[u] > theta));
      same += __builtin_popcountll(__ballot(keys.key[u] == theta));
    }
  });
  __syncthreads();
  if (lane == 0) {
    s_count[0][wave] = more;
    s_count[1][wave] = same;
  }
  __syncthreads();
  int all_more = 0, more_before = 0, same_before = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const int m = s_count[0][w], e = s_count[1][w];
    all_more += m;
    more_before += w < wave ? m : 0;
    same_before += w < wave ? e : 0;
  }
  const int room = s.k - all_more;  // of the equal ones (all of them where k are at least theta)
  int at = more_before + min(same_before, room), equal = room - same_before;
  keys.each(a, s, lane, [&](int i0) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const unsigned long long eq = __ballot(keys.key[u] == theta);
      const bool take = keys.key[u] > theta || (keys.key[u] == theta && lanes_below(eq) < equal);
      equal -= __builtin_popcountll(eq);
      const unsigned long long m = __ballot(take);
      if (take) s.out[at + lanes_below(m)] = i0 + 64 * u + lane;
      at += __builtin_popcountll(m);
    }
  });
  for (int j = s.k + tid; j < a.count; j += 64 * kSelectWaves) s.out[j] = -1;
}

template <int KPT>
void launch_wave(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(select_wave_kernel<KPT>, dim3((unsigned)cdiv(a.total, 4)), dim3(256), 0, st, a);
}
template <int KPT, bool HELD>
void launch_group(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((select_group_kernel<KPT, HELD>), dim3((unsigned)a.total), dim3(64 * kSelectWaves), 0, st, a);
}

}  // namespace

int select_top(const float* x, const int32_t* lengths, int32_t* out, int64_t layers, int64_t rows, int64_t heads,
               int64_t n, int64_t count, int64_t first, int64_t last, const int64_t* st, hipStream_t stream) {
  const int64_t total = layers * rows * heads;
  if (total == 0) return SPARKQ_OK;
  const SelectArgs a{x, lengths, out, st[0], st[1], st[2], total, (int)rows, (int)heads, (int)n, (int)count,
                     (int)first, (int)last};
  if (n <= 256)
    launch_wave<4>(a, stream);
  else if (n <= 512)
    launch_wave<8>(a, stream);
  else if (n <= 1024)
    launch_wave<16>(a, stream);
  else if (n <= 4096)
    launch_group<4, true>(a, stream);
  else if (n <= 8192)
    launch_group<8, true>(a, stream);
  else if (n <= 16384)
    launch_group<16, true>(a, stream);
  else if (n <= 32768)
    launch_group<32, true>(a, stream);
  else
    launch_group<32, false>(a, stream);
  return check_launch("select_top");
}

}  // namespace sparkq
