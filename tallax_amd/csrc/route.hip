// Routing tokens to experts: scores, the choice of groups, the choice of
// experts and their weights, a wave for each token.
#include <math.h>

#include <type_traits>

#include "tx_common.h"
#include "tx_host.h"

#include "tallax_hip.h"

namespace tx {

constexpr int kMostExperts = 1024, kMostGroups = 64, kMostChosen = 64;
constexpr int kRouteWaves = 4;

struct RouteArgs {
  const void* logits;
  int64_t tokens, row_stride;
  int experts, k, groups, per_group, top_groups, group_top, sigmoid, renormalise;
  int shift, vectors;  // a group's lanes are 1 << shift; logits may be read four at a time
  const float* bias;
  double scale;
  float* weights;
  int32_t* ids;
};

__device__ __forceinline__ double lane_xor_d(double x, int d) {
  return __longlong_as_double((long long)shfl_xor_u64((uint64_t)__double_as_longlong(x), d));
}

// The largest key of the wave and, of its equals, the lowest index; the same in all lanes.
__device__ __forceinline__ void wave_first(double& key, int& at) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double k = lane_xor_d(key, d);
    const int i = (int)lane_xor((uint32_t)at, d);
    const bool other = (k > key) | ((k == key) & (i < at));
    key = other ? k : key;
    at = other ? i : at;
  }
}

constexpr double kGone = -1.0e300;    // the key of an expert that is not there: below every score plus bias
constexpr double kTaken = -INFINITY;  // of one that is chosen already, or of no chosen group

constexpr float kMost = 3.4028234663852886e38f;

template <bool BF16>
__device__ __forceinline__ float logit_at(const RouteArgs& a, int64_t token, int e) {
  if constexpr (BF16) return __uint_as_float((uint32_t)((const uint16_t*)a.logits)[token * a.row_stride + e] << 16);
  return ((const float*)a.logits)[token * a.row_stride + e];
}

// A token by a wave, all in 64 bits.  keys: [experts] in LDS, where there are groups.
template <bool BF16, int NJ>
__device__ __forceinline__ void route_exactly(const RouteArgs& a, int64_t token, double* keys) {
  const int lane = lane_id();
  float x[NJ];
  double s[NJ], key[NJ];
  bool here[NJ];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + j * kWave;
    const float v = e < a.experts ? logit_at<BF16>(a, token, e) : -INFINITY;
    here[j] = v > -INFINITY;  // not NaN either
    x[j] = here[j] ? fminf(v, kMost) : -kMost;
    if (here[j]) top = fmaxf(top, x[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = here[j] ? 1.0 / (1.0 + exp(-(double)x[j])) : 0.0;
  } else {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, lane_xor_f(top, d));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) sum += s[j] = here[j] ? exp((double)x[j] - (double)top) : 0.0;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) sum += lane_xor_d(sum, d);
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sum > 0.0 ? s[j] / sum : 0.0;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + j * kWave;
    double b = 0.0;
    if (a.bias && e < a.experts) {
      const float f = a.bias[e];
      here[j] = here[j] && f == f;
      b = fminf(fmaxf(f, -kMost), kMost);
    }
    if (!here[j]) s[j] = 0.0;
    // of a group's sum; for the choice without a bias it is the logit itself, which no rounding ties
    key[j] = here[j] ? s[j] + b : kGone;
  }
  uint64_t open = ~0ull;  // groups that are chosen
  if (a.groups > 1) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = lane + j * kWave;
      // alone it stands for the group's rank: the logit, without a bias
      if (e < a.experts) keys[e] = !a.bias && a.group_top == 1 && here[j] ? (double)x[j] : key[j];
    }
    __builtin_amdgcn_wave_barrier();
    double rank = kTaken;
    if (lane < a.groups) {
      double first = kGone, second = kGone;
      for (int i = 0; i < a.per_group; ++i) {
        const double y = keys[lane * a.per_group + i];
        second = fmax(second, fmin(first, y));
        first = fmax(first, y);
      }
      rank = a.group_top == 2 && second > kGone ? first + second : first;
    }
    open = 0;
    for (int i = 0; i < a.top_groups; ++i) {
      double r = rank;
      int g = lane;
      wave_first(r, g);
      open |= 1ull << g;
      if (lane == g) rank = kTaken;
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + j * kWave;
    const double y = !a.bias & here[j] ? (double)x[j] : key[j];
    const bool out = (e >= a.experts) | !((open >> (e / a.per_group & 63)) & 1);
    key[j] = out ? kTaken : y;
  }
  double mine = 0.0, sum = 0.0;  // lane i: the score of choice i
  int id = 0;
  for (int i = 0; i < a.k; ++i) {
    double best = key[0], score = s[0];
    int at = lane;
#pragma unroll
    for (int j = 1; j < NJ; ++j) {
      if (key[j] > best) {
        best = key[j];
        at = lane + j * kWave;
        score = s[j];
      }
    }
    const int own = at;
    wave_first(best, at);
    const uint64_t who = __ballot(own == at);
    const int src = __ffsll((long long)who) - 1;
    const uint32_t lo = readlane_u32((uint32_t)__double_as_longlong(score), src);
    const uint32_t hi = readlane_u32((uint32_t)((uint64_t)__double_as_longlong(score) >> 32), src);
    const double w = __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
    sum += w;
    if (lane == i) {
      mine = w;
      id = at;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (at == lane + j * kWave) key[j] = kTaken;
  }
  if (lane < a.k) {
    if (a.renormalise) mine = sum > 0.0 ? mine / sum : 0.0;
    a.weights[token * a.k + lane] = (float)(mine * a.scale);
    a.ids[token * a.k + lane] = id;
  }
}

template <bool BF16, int NJ>
__global__ __launch_bounds__(kRouteWaves * kWave) void route_exactly_kernel(RouteArgs a) {
  extern __shared__ double lds[];  // [waves][experts], where there are groups
  const int wave = threadIdx.x / kWave;
  const int64_t token = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (token < a.tokens) route_exactly<BF16, NJ>(a, token, lds + wave * a.experts);
}

// Comparators of Batcher's odd-even merge sort of N values.
template <int N>
struct SortNet {
  int lo[80] = {}, hi[80] = {}, n = 0;
  constexpr SortNet() {
    for (int p = 1; p < N; p *= 2)
      for (int k = p; k >= 1; k /= 2)
        for (int j = k % p; j + k < N; j += 2 * k)
          for (int i = 0; i < k && i + j + k < N; ++i)
            if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) {
              lo[n] = i + j;
              hi[n++] = i + j + k;
            }
  }
};

__device__ __forceinline__ void larger_first(int& x, int& y) {
  const int m = max(x, y);
  y = min(x, y);
  x = m;
}

template <int N>
__device__ __forceinline__ void sort_down(int* v) {
  constexpr SortNet<N> net;
#pragma unroll
  for (int i = 0; i < net.n; ++i) larger_first(v[net.lo[i]], v[net.hi[i]]);
}

// The L largest of two descending lists of L, descending, in the first.
template <int L>
__device__ __forceinline__ void keep_largest(int* x, const int* y) {
#pragma unroll
  for (int i = 0; i < L; ++i) x[i] = max(x[i], y[L - 1 - i]);
#pragma unroll
  for (int d = L / 2; d >= 1; d /= 2)
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (!(i & d)) larger_first(x[i], x[i + d]);
}

// A float's order as a signed integer, and back.
__device__ __forceinline__ int ordered(float f) {
  const int i = __float_as_int(f);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// Value of lane (l - N) % 16 of the same 16 lanes.
template <int N>
__device__ __forceinline__ int row_ror(int x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xF, 0xF, false);
}

__device__ __forceinline__ int row_max(int v) {  // of 16 lanes, in all of them
  v = max(v, row_ror<8>(v));
  v = max(v, row_ror<4>(v));
  v = max(v, row_ror<2>(v));
  return max(v, row_ror<1>(v));
}
template <int N>
__device__ __forceinline__ float row_ror_f(float x) {
  return __int_as_float(row_ror<N>(__float_as_int(x)));
}
__device__ __forceinline__ float row_max_f(float v) {
  v = fmaxf(v, row_ror_f<8>(v));
  v = fmaxf(v, row_ror_f<4>(v));
  v = fmaxf(v, row_ror_f<2>(v));
  return fmaxf(v, row_ror_f<1>(v));
}
__device__ __forceinline__ float row_sum_f(float v) {
  v += lane_xor_f(v, 8);
  v += lane_xor_f(v, 4);
  v += lane_xor_f(v, 2);
  return v + lane_xor_f(v, 1);
}
__device__ __forceinline__ double row_sum_d(double v) {
  v += lane_xor_d(v, 8);
  v += lane_xor_d(v, 4);
  v += lane_xor_d(v, 2);
  return v + lane_xor_d(v, 1);
}

// A group's rank, the same in all of its lanes.
struct Rank {
  int whole;          // where it is exact
  float value, room;  // else, and how far any two of the token may be off
};

// Compares it with that of the group N lanes before: counts those that come first, and sees whether any is too near to
// tell.
template <int N>
__device__ __forceinline__ void count_before(const Rank& r, bool exact, int l, int shift, int& before, bool& near) {
  if (N & ((1 << shift) - 1)) return;
  const bool lower = (((l - N) & 15) >> shift) < (l >> shift);
  if (exact) {
    const int o = row_ror<N>(r.whole);
    before += (o > r.whole) | ((o == r.whole) & lower);
  } else {
    const float o = row_ror_f<N>(r.value);
    before += (o > r.value) | ((o == r.value) & lower);
    near = near | (fabsf(o - r.value) <= r.room);
  }
}

// Whether it matters: one of the two is chosen and the other is not.
template <int N>
__device__ __forceinline__ void across(const Rank& r, int open, int shift, bool& near) {
  if (N & ((1 << shift) - 1)) return;
  near = near | ((fabsf(row_ror_f<N>(r.value) - r.value) <= r.room) & (row_ror<N>(open) != open));
}

template <int N>
__device__ __forceinline__ void count_larger(double key, int at, int l, int k, int& before) {
  const uint64_t u = (uint64_t)__double_as_longlong(key);
  const uint32_t lo = (uint32_t)row_ror<N>((int)(uint32_t)u), hi = (uint32_t)row_ror<N>((int)(uint32_t)(u >> 32));
  const double o = __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
  const int i = row_ror<N>(at);
  before += (((l - N) & 15) < k) & ((o > key) | ((o == key) & (i < at)));
}

template <class F>
__device__ __forceinline__ void for_rotations(F f) {  // of 16 lanes
  f(std::integral_constant<int, 1>());
  f(std::integral_constant<int, 2>());
  f(std::integral_constant<int, 3>());
  f(std::integral_constant<int, 4>());
  f(std::integral_constant<int, 5>());
  f(std::integral_constant<int, 6>());
  f(std::integral_constant<int, 7>());
  f(std::integral_constant<int, 8>());
  f(std::integral_constant<int, 9>());
  f(std::integral_constant<int, 10>());
  f(std::integral_constant<int, 11>());
  f(std::integral_constant<int, 12>());
  f(std::integral_constant<int, 13>());
  f(std::integral_constant<int, 14>());
  f(std::integral_constant<int, 15>());
}

constexpr int kNone = INT32_MIN;

// e^x for weights, to 2^-32 of itself: in 64 bits by its Taylor series to r^8, |r| <= ln 2 / 2; from 2^-1000 to 2^1000.
__device__ __forceinline__ double power(double x) {
  const double t = fmin(fmax(x * 1.4426950408889634, -1000.0), 1000.0), n = rint(t), r = (t - n) * 0.6931471805599453;
  double p = 1.0 / 40320.0;
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  return ldexp(fma(p, r, 1.0), (int)n);
}

// 1 / x to 2^-40, of normal numbers.
__device__ __forceinline__ double reciprocal(double x) {
  const double r = __builtin_amdgcn_rcp(x);
  return fma(fma(-x, r, 1.0), r, r);
}

// Four tokens a wave, 16 lanes each, a lane with up to EPL neighbouring experts
// of one group; 1 << shift lanes hold a group.  Keys (scores plus bias, or
// logits) are 32 bits, in the order of integers, their last bits the expert's
// place in the lane.  Each lane sorts its keys and keeps the L largest; the
// largest head of 16 lanes is the next choice, and the lane it is from moves on.
// Where two choices lie within their keys' rounding, their order is found in 64
// bits; where the last choice and the next, or a group that is chosen and one
// that is not, do, or there are not enough experts, the token goes to the whole
// wave in 64 bits.  bfloat16 logits without a bias have room for the whole
// expert's number in the key, which then is exact.
template <bool BF16, int EPL, int L>
__global__ __launch_bounds__(kRouteWaves * kWave) void route_kernel(RouteArgs a) {
  extern __shared__ double lds[];  // [waves][experts], where there are groups
  constexpr int kPlace = EPL - 1;
  constexpr float kLog2e = 1.44269504088896340736f;
  // How far apart two keys must lie: the place takes up to EPL - 1 last bits of 24 of each; a score is off by the rounding
  // of its exponent (at most .3 of 2^-23 of the largest score, since s |x| has a maximum), of its exponential, sum and
  // reciprocal (2^-23 of itself each) and of the sum with the bias: by less than 2^-21 of the largest, two by 2^-20.
  constexpr float kCut = EPL / 8388608.0f, kOff = 9.5367432e-7f;
  const int wave = threadIdx.x / kWave, lane = lane_id(), l = lane & 15;
  const int64_t first = ((int64_t)blockIdx.x * kRouteWaves + wave) * 4, token = first + lane / 16;
  if (first >= a.tokens) return;
  const bool valid = token < a.tokens, exact = BF16 && !a.bias;
  const int group = l >> a.shift, within = (l & ((1 << a.shift) - 1)) * EPL;
  const int e0 = group * a.per_group + within;
  const int n = valid && group < a.groups ? a.per_group - within : 0;  // experts of this lane, if positive
  float x[EPL], bias[EPL];
  if (a.vectors) {
#pragma unroll
    for (int j = 0; j < EPL; j += 4) {
      const bool some = j < n;
      const int64_t at = some ? token * a.row_stride + e0 + j : 0;
      if constexpr (BF16) {
        const uint2 u = *(const uint2*)((const uint16_t*)a.logits + at);
        x[j] = __uint_as_float(u.x << 16);
        x[j + 1] = __uint_as_float(u.x & 0xffff0000u);
        x[j + 2] = __uint_as_float(u.y << 16);
        x[j + 3] = __uint_as_float(u.y & 0xffff0000u);
      } else {
        const float4 u = *(const float4*)((const float*)a.logits + at);
        x[j] = u.x;
        x[j + 1] = u.y;
        x[j + 2] = u.z;
        x[j + 3] = u.w;
      }
      const float4 u = a.bias ? *(const float4*)(a.bias + (some ? e0 + j : 0)) : make_float4(0.f, 0.f, 0.f, 0.f);
      bias[j] = u.x;
      bias[j + 1] = u.y;
      bias[j + 2] = u.z;
      bias[j + 3] = u.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j + i] = some ? x[j + i] : -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const bool some = j < n;
      x[j] = logit_at<BF16>(a, some ? token : 0, some ? e0 + j : 0);
      bias[j] = a.bias ? a.bias[some ? e0 + j : 0] : 0.0f;
      x[j] = some ? x[j] : -INFINITY;
    }
  }
  // softmax: the sum over all experts, where scores are compared or given as they are
  const bool scores = a.bias || (a.groups > 1 && a.group_top == 2);
  float top = 0.0f, sum = 1.0f;  // top: 0 for sigmoid scores
  if (!a.sigmoid && (scores || !a.renormalise)) {
    top = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) top = x[j] > top ? fminf(x[j], kMost) : top;
    top = row_max_f(top);
    top = top == -INFINITY ? 0.0f : top;
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      part += x[j] > -INFINITY ? __builtin_amdgcn_exp2f((fminf(x[j], kMost) - top) * kLog2e) : 0.0f;
    sum = row_sum_f(part);
  }
  const float inverse = 1.0f / sum, largest = a.sigmoid ? 1.0f : inverse;  // of all scores
  auto score_of = [&](float v) {
    return a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e))
                     : __builtin_amdgcn_exp2f((v - top) * kLog2e) * inverse;
  };
  int key[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    bool here = x[j] > -INFINITY;  // not NaN either
    x[j] += 0.0f;  // -0 is 0
    if (exact) {
      key[j] = here ? (ordered(x[j]) & (int)0xffff0000) | (0xffff - (e0 + j)) : kNone;
    } else {
      float f = fminf(x[j], kMost);
      if (a.bias) {
        here = here & (bias[j] == bias[j]);
        f = score_of(f) + fminf(fmaxf(bias[j], -kMost), kMost);
      }
      key[j] = here ? (ordered(f) & ~kPlace) | (kPlace - j) : kNone;
    }
  }
  constexpr int S = L < EPL ? L : EPL;
#pragma unroll
  for (int i = 0; i < EPL; i += S) {
    sort_down<S>(key + i);
    if (i > 0) keep_largest<S>(key, key + i);
  }
  bool near = false;
  auto value = [&](int k) { return from_ordered(k & (exact ? (int)0xffff0000 : ~kPlace)); };
  if (a.groups > 1) {
    int k0 = key[0], k1 = key[1];
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      if (d >> a.shift) continue;
      const int o0 = (int)lane_xor((uint32_t)k0, d), o1 = (int)lane_xor((uint32_t)k1, d);
      k1 = max(min(k0, o0), max(k1, o1));
      k0 = max(k0, o0);
    }
    Rank r;
    const bool whole = a.group_top == 1 && exact;
    r.whole = group < a.groups ? k0 : kNone;
    float v0 = value(k0), v1 = value(k1);
    if (a.group_top == 1) {
      r.value = v0;
      // logits, as they are but for their last bits
      r.room = a.bias ? kCut * fabsf(v0) + kOff * largest : kCut * fabsf(v0);
    } else if (a.bias) {
      r.value = v0 + (k1 == kNone ? 0.0f : v1);
      r.room = kCut * (fabsf(v0) + (k1 == kNone ? 0.0f : fabsf(v1))) + 2.0f * kOff * largest;
    } else {
      const float far = fmaxf(fabsf(v0), k1 == kNone ? 0.0f : fabsf(v1)) + fabsf(top);
      r.value = score_of(v0) + (k1 == kNone ? 0.0f : score_of(v1));
      r.room = (kCut + kOff) * r.value * (1.0f + far);
    }
    if (k0 == kNone || group >= a.groups) r.value = -INFINITY, r.room = 0.0f;
    r.room = 2.0f * row_max_f(r.room);
    int before = 0;
    bool close = false;
    for_rotations([&](auto i) { count_before<i.value>(r, whole, l, a.shift, before, close); });
    if (__ballot(close)) for_rotations([&](auto i) { across<i.value>(r, before < a.top_groups, a.shift, near); });
    if (before >= a.top_groups) {
#pragma unroll
      for (int i = 0; i < S; ++i) key[i] = kNone;
    }
  }
  int mine = kNone, from = 0;  // lane i: choice i, and the lane it is from
#pragma unroll 1
  for (int i = 0; i < a.k; ++i) {
    const int best = row_max(key[0]);
    const int src = __ffs((int)(uint32_t)((__ballot(key[0] == best) >> (lane & 48)) & 0xffff)) - 1;
    mine = l == i ? best : mine;
    from = l == i ? src : from;
    // by masks: of a choice between two places of an array the compiler makes a search through all of it
    const int pop = l == src ? -1 : 0;
#pragma unroll
    for (int j = 0; j < S; ++j) key[j] = (pop & (j + 1 < S ? key[j + 1 < S ? j + 1 : 0] : kNone)) | (~pop & key[j]);
  }
  near = near | ((l < a.k) & (mine == kNone));
  bool order = false;  // of this choice and the one before it is open
  if (!exact) {
    const int next = row_max(key[0]);
    auto close = [&](int larger, int smaller) {
      const float p = value(larger), q = value(smaller);
      return (smaller != kNone) & (a.bias ? p - q <= kCut * (fabsf(p) + fabsf(q)) + kOff * largest : p == q);
    };
    order = (l > 0) & (l < a.k) & close(row_ror<1>(mine), mine);
    // 32 bits of a softmax's sum leave it open what a score adds to a bias
    near = near | (order & (a.bias && !a.sigmoid)) | ((l == a.k - 1) & close(mine, next));
  }
  const int at = exact ? 0xffff - (mine & 0xffff)
                       : (from >> a.shift) * a.per_group + (from & ((1 << a.shift) - 1)) * EPL + kPlace - (mine & kPlace);
  const bool picked = valid & (l < a.k) & (mine != kNone);
  const float logit = picked ? fminf(logit_at<BF16>(a, token, at), kMost) : -INFINITY;
  // scores that 64 bits may not hold, and whose sum may be 0
  if (a.renormalise && (a.sigmoid || scores)) near = near | (picked & (logit - top < -700.0f));
  const uint64_t unsure = __ballot(near & valid);
  const bool chosen = picked && ((unsure >> (lane & 48)) & 0xffff) == 0;
  double w = 0.0;
  if (a.sigmoid) {
    w = reciprocal(1.0 + power(-(double)logit));
  } else {
    const float base = a.renormalise ? row_max_f(logit) : top;
    w = power((double)logit - (double)base);
    if (!a.renormalise) w *= reciprocal((double)sum);
  }
  w = chosen ? w : 0.0;
  if (a.renormalise) {
    const double all = row_sum_d(w);
    w = all > 0.0 ? w * reciprocal(all) : 0.0;
  }
  int place = l;
  if (__ballot(order & chosen)) {
    const double score = 1.0 / (1.0 + exp(-(double)logit));
    const double exactly = !a.bias ? (double)logit : chosen ? score + (double)fminf(fmaxf(a.bias[at], -kMost), kMost) : 0.0;
    place = 0;
    for_rotations([&](auto i) { count_larger<i.value>(exactly, at, l, a.k, place); });
  }
  if (chosen) {
    a.weights[token * a.k + place] = (float)(w * a.scale);
    a.ids[token * a.k + place] = at;
  }
  for (int r = 0; r < 4; ++r)
    if ((unsure >> (16 * r)) & 0xffff) route_exactly<BF16, EPL / 4>(a, first + r, lds + wave * a.experts);
}

template <bool BF16, int EPL, int L>
static int launch_rows(const RouteArgs& a, size_t lds, hipStream_t s) {
  constexpr int kTokens = kRouteWaves * 4;
  route_kernel<BF16, EPL, L><<<(unsigned)((a.tokens + kTokens - 1) / kTokens), kRouteWaves * kWave, lds, s>>>(a);
  return launch_status("route");
}

template <bool BF16>
static int launch_route(RouteArgs a, hipStream_t s) {
  const size_t lds = a.groups > 1 ? (size_t)kRouteWaves * a.experts * 8 : 0;
  // lanes of a group: a power of two, all groups in 16
  int shift = 4;
  while (shift > 0 && a.groups << shift > 16) --shift;
  const int each = (a.per_group + (1 << shift) - 1) >> shift;
  if (a.groups <= 16 && a.k <= 16 && each <= 32) {
    const int bytes = BF16 ? 2 : 4;
    a.shift = shift;
    a.vectors = ((uintptr_t)a.logits | (uintptr_t)(a.row_stride * bytes)) % (4 * bytes) == 0 && (uintptr_t)a.bias % 16 == 0 &&
                a.per_group % 4 == 0;
    if (each <= 4) return launch_rows<BF16, 4, 4>(a, lds, s);
    if (each <= 8) return launch_rows<BF16, 8, 8>(a, lds, s);
    if (each <= 16) return a.k <= 8 ? launch_rows<BF16, 16, 8>(a, lds, s) : launch_rows<BF16, 16, 16>(a, lds, s);
    return a.k <= 8 ? launch_rows<BF16, 32, 8>(a, lds, s) : launch_rows<BF16, 32, 16>(a, lds, s);
  }
  const unsigned grid = (unsigned)((a.tokens + kRouteWaves - 1) / kRouteWaves);
  const int threads = kRouteWaves * kWave;
  if (a.experts <= 256) route_exactly_kernel<BF16, 4><<<grid, threads, lds, s>>>(a);
  else route_exactly_kernel<BF16, 16><<<grid, threads, lds, s>>>(a);
  return launch_status("route");
}

}  // namespace tx

using namespace tx;

extern "C" {

int tallax_route(const void* logits, int logits_dtype, int64_t tokens, int64_t experts, int64_t row_stride, int64_t k,
                 int sigmoid, const float* bias, int64_t groups, int64_t top_groups, int group_top, int renormalise,
                 double scale, float* out_weights, int32_t* out_ids, tallax_stream_t stream) {
  if (logits_dtype != TALLAX_F32 && logits_dtype != TALLAX_BF16) {
    set_error("route: logits of dtype %d (float32 or bfloat16)", logits_dtype);
    return kUnsupported;
  }
  if (tokens < 0 || experts < 1 || groups < 1 || experts % groups || top_groups < 1 || top_groups > groups || k < 1 ||
      k > top_groups * (experts / groups) || (group_top != 1 && group_top != 2) || row_stride < 0) {
    set_error("route: %lld of %lld experts in %lld of %lld groups, ranked by %d, row stride %lld", (long long)k,
              (long long)experts, (long long)top_groups, (long long)groups, group_top, (long long)row_stride);
    return kInvalidArgument;
  }
  if (!(fabs(scale) <= 3.4028234e38)) {
    set_error("route: scale must be finite in float32");
    return kInvalidArgument;
  }
  if (experts > kMostExperts || groups > kMostGroups || k > kMostChosen || tokens > ((int64_t)1 << 31) ||
      row_stride > ((int64_t)1 << 31)) {
    set_error("route: up to %d experts, %d groups, %d chosen, 2^31 tokens", kMostExperts, kMostGroups, kMostChosen);
    return kUnsupported;
  }
  if (tokens == 0) return kOk;
  if (!logits || !out_weights || !out_ids) {
    set_error("route: null pointer");
    return kInvalidArgument;
  }
  RouteArgs a;
  a.logits = logits;
  a.tokens = tokens;
  a.row_stride = row_stride;
  a.experts = (int)experts;
  a.k = (int)k;
  a.groups = (int)groups;
  a.per_group = (int)(experts / groups);
  a.top_groups = (int)top_groups;
  a.group_top = group_top;
  a.sigmoid = sigmoid;
  a.renormalise = renormalise;
  a.bias = bias;
  a.scale = scale;
  a.weights = out_weights;
  a.ids = out_ids;
  hipStream_t s = (hipStream_t)stream;
  return logits_dtype == TALLAX_BF16 ? launch_route<true>(a, s) : launch_route<false>(a, s);
}

}  // extern "C"
