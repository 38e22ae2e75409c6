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
  uint32_t total;                  // layers * rows * heads, below 2^22
  int rows, heads, n, count, first, last;
};

// Whole numbers in the order of the values; 0 is left for what is no value. -inf
// stands for NaN, 0 for -0; a place that has to be taken comes before +inf.
__device__ __forceinline__ uint32_t key_of(float v) {
  const int u = __float_as_int(v == v ? v + 0.0f : -__builtin_huge_valf());
  return (uint32_t)(u ^ (u >> 31 | (int)0x80000000));
}

struct SelectRow {
  const float* x;
  int32_t* out;
  int n, k;  // values, how many of them are taken
  int late;  // the first of the last places, which have to be taken
};
__device__ __forceinline__ SelectRow select_row(const SelectArgs& a, uint32_t i) {
  const uint32_t lr = i / (uint32_t)a.heads, h = i - lr * a.heads, l = lr / (uint32_t)a.rows, r = lr - l * a.rows;
  SelectRow s;
  s.x = a.x + l * a.x_layer + r * a.x_row + h * a.x_head;
  s.out = a.out + (int64_t)i * a.count;
  // (a scalar load, which what follows from it is scalar by: nothing here writes lengths)
  typedef const __attribute__((address_space(4))) int32_t* Lengths;
  s.n = a.lengths ? min(max(((Lengths)(uintptr_t)a.lengths)[r], 0), a.n) : a.n;
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

// A wave's k-th largest key, of those with theta's bits above bit `bit`, or one less
// than all that are taken: those that are larger than the result are taken, and of
// those that are equal to it as many as are still wanted. A bit at a time: it is set in
// the k-th key if k keys have it and the bits so far.
template <int KPT>
__device__ __forceinline__ uint32_t kth_key(const uint32_t (&key)[KPT], int k, uint32_t theta, int bit) {
  for (; bit >= 0; --bit) {
    const uint32_t cand = theta | 1u << bit;
    int c = 0;
#pragma unroll
    for (int u = 0; u < KPT; ++u) c += __builtin_popcountll(__ballot(key[u] >= cand));
    if (c >= k) theta = cand;
    if (c == k) return theta - 1;
  }
  return theta;
}

// ---------------------------------------------------------------------------
// a wave a row: rows of up to 64 * KPT values, which stay in registers
// ---------------------------------------------------------------------------
// A chain of at most 32 counts, each KPT ballots: 128 rows of up to 512 (0.1 MB) take
// 5.8 us, about 3 of them a launch's and the load's latency.
template <int KPT>
__global__ __launch_bounds__(256) void select_wave_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  const uint32_t theta = kth_key<KPT>(key, s.k, 0, 31);
  int equal = s.k;  // of the keys that are theta, how many are taken
#pragma unroll
  for (int u = 0; u < KPT; ++u) equal -= __builtin_popcountll(__ballot(key[u] > theta));
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
// Wave w of W has the places [w per, (w + 1) per), 64 KPT of them at a time: the keys
// of rows of up to 64 W KPT values stay in registers (HELD), those of others are made
// again from the values in every pass. (In LDS they let three workgroups on a CU where
// four fit.)
//
// The k-th largest key is found by digits of 11, 11 and 10 bits: how many of the keys
// with the digits found so far have each next one, and down from the largest which
// digit the k-th has. Where few enough keys share its first digit they are listed, and
// one wave finds it among them.
// 1024 rows of up to 8192 values (30 MB) take 19.8 us, where a copy of them takes 6: four
// workgroups a CU go through one chain of barriers each and fill the vector units to 62%.
constexpr int kBins = 2048, kListed = 512;

template <int W, int KPT, bool HELD>
__global__ __launch_bounds__(64 * W, KPT > 16 ? 4 : 8) void select_group_kernel(SelectArgs a) {
  __shared__ int s_bins[kBins], s_pick[3], s_count[2][W], s_listed;
  __shared__ uint32_t s_list[kListed], s_theta;
  __shared__ uint8_t s_owner[kListed];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SelectRow s = select_row(a, blockIdx.x);
  if (s.n <= s.k) {
    for (int j = tid; j < a.count; j += 64 * W) s.out[j] = j < s.k ? j : -1;
    return;
  }
  const int per = (s.n + 64 * W - 1) / (64 * W) * 64, w0 = wave * per, w1 = min(w0 + per, s.n);
  uint32_t key[KPT];
  // (offsets in 32 bits beside scalar addresses: n and count are below 2^30)
  auto value = [&](int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(s.x) + (uint32_t)i * 4u);
  };
  auto make = [&](int i0) __attribute__((always_inline)) {
    float v[KPT];
    if (i0 + 64 * KPT <= s.n) {
#pragma unroll
      for (int u = 0; u < KPT; ++u) v[u] = value(i0 + lane + 64 * u);
    } else {
#pragma unroll
      for (int u = 0; u < KPT; ++u) v[u] = value(min(i0 + lane + 64 * u, s.n - 1));
    }
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int i = i0 + 64 * u;
      if (i >= a.first && i + 64 <= min(s.late, w1))
        key[u] = key_of(v[u]);
      else
        key[u] = i < w1 ? key_at(a, s, i + lane, v[u]) : 0u;
    }
  };
  // f(place of lane 0's, key) for the wave's keys in order, 64 at a time
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    for (int i0 = w0; i0 < w1; i0 += 64 * KPT) {
      if (!HELD) make(i0);
#pragma unroll
      for (int u = 0; u < KPT; ++u) {
        // (or the compiler keeps one pass's comparisons for the next, and spills them)
        asm volatile("" : "+v"(key[u]));
        if (i0 + 64 * u < w1) f(i0 + 64 * u, key[u]);
      }
      if (HELD) break;
    }
  };
  if (HELD) make(w0);
  for (int d = tid; d < kBins; d += 64 * W) s_bins[d] = 0;
  if (tid < W) s_count[0][tid] = s_count[1][tid] = 0;
  if (tid == 0) s_listed = 0;
  __syncthreads();
  // (what is no value is counted as digit 0, which no k-th key has)
  each([&](int, uint32_t key) __attribute__((always_inline)) { atomicAdd(&s_bins[key >> 21], 1); });
  uint32_t prefix = 0, theta = 0;
  int need = s.k;        // its place among the keys with the digits so far
  bool counted = false;  // s_count is what each wave has that is larger than theta, and equal
  for (int pass = 0; pass < 3; ++pass) {
    const int above = 32 - 11 * pass, shift = max(above - 11, 0);
    if (pass > 0)
      each([&](int, uint32_t key) __attribute__((always_inline)) {
        if (key >> above == prefix) atomicAdd(&s_bins[(key >> shift) & ((1u << (above - shift)) - 1)], 1);
      });
    __syncthreads();
    // BPT digits a thread, from the largest down
    constexpr int BPT = kBins / (64 * W);
    __shared__ int s_sum[W];
    const int d = kBins - 1 - BPT * tid;
    int own = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) own += s_bins[d - i];
    int before = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(before, o);
      if (lane >= o) before += y;
    }
    if (lane == 63) s_sum[wave] = before;
    __syncthreads();
    before -= own;
#pragma unroll
    for (int w = 0; w < W; ++w) before += w < wave ? s_sum[w] : 0;
    if (before < need && need <= before + own) {
      int i = 0;
      while (need > before + s_bins[d - i]) before += s_bins[d - i++];
      s_pick[0] = d - i;
      s_pick[1] = need - before;
      s_pick[2] = s_bins[d - i];
    }
    __syncthreads();
    prefix = pass == 0 ? s_pick[0] : prefix << (above - shift) | s_pick[0];
    need = s_pick[1];
    const int alike = s_pick[2];
    theta = prefix << shift;
    if (need == alike) {  // all keys with these digits are taken
      --theta;
      break;
    }
    if (pass == 0 && alike <= kListed) {
      int more = 0, own = 0;  // of the wave, of the lane
      const uint32_t next = theta + (1u << 21) - 1;  // the last key with this digit
      each([&](int, uint32_t key) __attribute__((always_inline)) {
        more += __builtin_popcountll(__ballot(key > next));
        own += key - theta < 1u << 21;
      });
      int at = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(at, o);
        if (lane >= o) at += y;
      }
      int base = 0;
      if (lane == 63) base = atomicAdd(&s_listed, at);
      at += __shfl(base, 63) - own;
      each([&](int, uint32_t key) __attribute__((always_inline)) {
        if (key - theta < 1u << 21) {
          s_list[at] = key;
          s_owner[at++] = (uint8_t)wave;
        }
      });
      if (lane == 0) s_count[0][wave] = more;
      __syncthreads();
      if (wave == 0) {
        uint32_t key[kListed / 64];
#pragma unroll
        for (int u = 0; u < kListed / 64; ++u) key[u] = 64 * u + lane < alike ? s_list[64 * u + lane] : 0u;
        theta = kth_key<kListed / 64>(key, need, theta, 20);
#pragma unroll
        for (int u = 0; u < kListed / 64; ++u)
          if (64 * u + lane < alike && key[u] >= theta) atomicAdd(&s_count[key[u] == theta][s_owner[64 * u + lane]], 1);
        if (lane == 0) s_theta = theta;
      }
      __syncthreads();
      theta = s_theta;
      counted = true;
      break;
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) s_bins[d - i] = 0;
    __syncthreads();
  }
  if (!counted) {
    int more = 0, same = 0;
    each([&](int, uint32_t key) __attribute__((always_inline)) {
      more += __builtin_popcountll(__ballot(key > theta));
      same += __builtin_popcountll(__ballot(key == theta));
    });
    if (lane == 0) {
      s_count[0][wave] = more;
      s_count[1][wave] = same;
    }
    __syncthreads();
  }
  int all_more = 0, more_before = 0, same_before = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int m = s_count[0][w], e = s_count[1][w];
    all_more += m;
    more_before += w < wave ? m : 0;
    same_before += w < wave ? e : 0;
  }
  const int room = s.k - all_more;  // of the equal ones (none of them where theta is no key)
  int at = more_before + min(same_before, room), equal = room - same_before;
  each([&](int i0, uint32_t key) __attribute__((always_inline)) {
    bool take = key > theta;
    const unsigned long long eq = __ballot(key == theta);
    if (eq) {
      take = take || (key == theta && lanes_below(eq) < equal);
      equal -= __builtin_popcountll(eq);
    }
    const unsigned long long m = __ballot(take);
    const uint32_t slot = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, at));
    if (take) *reinterpret_cast<int32_t*>(reinterpret_cast<char*>(s.out) + slot * 4u) = i0 + lane;
    at += __builtin_popcountll(m);
  });
  for (int j = s.k + tid; j < a.count; j += 64 * W) s.out[j] = -1;
}

template <int KPT>
void launch_wave(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(select_wave_kernel<KPT>, dim3((unsigned)cdiv(a.total, 4)), dim3(256), 0, st, a);
}
template <int W, int KPT, bool HELD>
void launch_group(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((select_group_kernel<W, KPT, HELD>), dim3((unsigned)a.total), dim3(64 * W), 0, st, a);
}

}  // namespace

int select_top(const float* x, const int32_t* lengths, int32_t* out, int64_t layers, int64_t rows, int64_t heads,
               int64_t n, int64_t count, int64_t first, int64_t last, const int64_t* st, hipStream_t stream) {
  const int64_t total = layers * rows * heads;
  if (total == 0) return SPARKQ_OK;
  const SelectArgs a{x, lengths, out, st[0], st[1], st[2], (uint32_t)total, (int)rows, (int)heads, (int)n, (int)count,
                     (int)first, (int)last};
  // Up to 1024 values a wave a row: 2048 rows of 1000 take 10.7 us, with a workgroup each
  // 12.6 or more; rows of 2000 13.4 with a workgroup, 17.4 with a wave. The smallest
  // workgroup that holds the keys of longer ones; without (rows of 16000) 2048 rows take
  // 83 us, with them 62. 32 keys a thread let one workgroup on a CU: 256 rows of 20000 take
  // 20 us, 512 35, where keys that are made again take 32 and 45; 2048 rows 131 and 117.
  // It goes by what a row has room for, as lengths are on the device: 1024 rows of 2000 take
  // 12 us in 2000 places, 14 in 8192, 27 in 16384 and 40 in 40000.
  if (n <= 256)
    launch_wave<4>(a, stream);
  else if (n <= 512)
    launch_wave<8>(a, stream);
  else if (n <= 1024)
    launch_wave<16>(a, stream);
  else if (n <= 4096)
    launch_group<4, 16, true>(a, stream);
  else if (n <= 8192)
    launch_group<8, 16, true>(a, stream);
  else if (n <= 16384)
    launch_group<16, 16, true>(a, stream);
  else if (n <= 32768 && total <= 2 * device_cus())
    launch_group<16, 32, true>(a, stream);
  else
    launch_group<16, 16, false>(a, stream);
  return check_launch("select_top");
}

}  // namespace sparkq
