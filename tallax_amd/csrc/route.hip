// Routing tokens to experts: scores s = softmax(x) or 1 / (1 + exp(-x)), keys
// s + bias, the choice of groups by their largest key or the sum of two, the choice
// of the k largest keys in them, and the weights s (over their sum) times scale.
// What is chosen is what 64-bit keys choose.
//
// Four tokens a wave and 32-bit keys, for up to 16 chosen of up to 16 groups
// (route_kernel); a wave for each token, all in 64 bits, for others and for the
// tokens whose 32-bit keys leave a choice open (route_exactly).  A row of logits is
// read once or twice, the second time from the cache, and little else: 16384 tokens
// of 256 float32 experts in 8 groups, sigmoid with a bias, the two largest, 17.8 MB,
// take 13.2 us, where reading them takes 3.7.  What bounds it is its instructions: 1151
// vector ones a wave, four waves to a SIMD, whose vector unit they keep busy 85 % of the
// time that they are there; 2.3 us are the few waves with a comparison in 64 bits.  130
// tokens take 6.5 us, one of 64 experts 3.  A softmax with a bias takes 15.7 us (its sum,
// and more comparisons in 64 bits, since that sum is of 32), unnormalised 12.0 (10.2 with a
// sum of 32 bits), bfloat16 without either 7.9.
#include <math.h>

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
  int shift, each, places, vectors;  // a group's lanes are 1 << shift, with `each` experts; logits may be read four at a time
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

__device__ __forceinline__ void larger_first(int& x, int& y) {
  const int m = max(x, y);
  y = min(x, y);
  x = m;
}

// The L largest of a descending list of L and four values, descending.
template <int L>
__device__ __forceinline__ void insert_four(int (&x)[L], int (&y)[4]) {
  larger_first(y[0], y[1]);
  larger_first(y[2], y[3]);
  larger_first(y[0], y[2]);
  larger_first(y[1], y[3]);
  larger_first(y[1], y[2]);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[L - 1 - i] = max(x[L - 1 - i], y[i]);
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

__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)x);
}
__device__ __forceinline__ double from_lane_d(double x, int lane) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = from_lane((uint32_t)u, lane), hi = from_lane((uint32_t)(u >> 32), lane);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// How many of lanes l + step, l + 2 step, .. (mod 16) of the same 16, below n, come before this one: by the larger key,
// of equal ones by the lower number.
__device__ __forceinline__ int count_before(double key, int number, int l, int step, int n) {
  int before = 0;
#pragma unroll 1
  for (int r = step; r < 16; r += step) {
    const int from = (l + r) & 15, lane = (lane_id() & 48) | from;
    const double o = from_lane_d(key, lane);
    const int i = (int)from_lane((uint32_t)number, lane);
    before += (from < n) & ((o > key) | ((o == key) & (i < number)));
  }
  return before;
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

// Four tokens a wave, 16 lanes each, a lane with a.each neighbouring experts of
// one group; 1 << shift lanes hold a group.  Keys (scores plus bias, or logits)
// are 32 bits, in the order of integers, their last bits the expert's place in
// the lane.  Each lane keeps its L largest, sorted; the largest head of 16 lanes
// is the next choice, and the lane it is from moves on.
// Where two choices, or the last and the next, lie within their keys' rounding,
// those are compared in 64 bits, and where a group that is chosen and one that is
// not do, the groups are.  Where the one after the next is as near, or there are
// not enough experts, the token goes to the whole wave in 64 bits.  bfloat16 logits
// without a bias have room for the whole expert's number in the key, which then is
// exact.
//
// Every wave runs through here once, and what it waits for is its instructions, some
// 16 cycles each with four waves to a SIMD.  Loops hold little code (16384 tokens of 256
// experts in 8 groups took 17.2 us with everything unrolled).
template <bool BF16, int L, int NJ>
__global__ __launch_bounds__(kRouteWaves * kWave) void route_kernel(RouteArgs a) {
  extern __shared__ double lds[];  // [waves][experts], where there are groups
  constexpr float kLog2e = 1.44269504088896340736f;
  // How far apart two keys must lie: the place takes the last bits of 24 of each, so that both are too small, by up to
  // `cut` of themselves; a score is off by the rounding of its exponent (at most .6 of 2^-23 of the largest score, since
  // s |x| has a maximum), of its exponential and reciprocal (2^-23 of itself each) and of the sum with the bias: by less
  // than 2^-21 of the largest, two by 2^-20.  A softmax's sum is off by up to `each` half steps for as many additions of a
  // lane, by three for each of its rescalings, of which there is one in four experts at most, and by less than 13 steps
  // for its terms' exponents (of up to 7, where 1024 of them make half of the sum), the lanes' join and the quotient.  That
  // moves all scores alike, two of them apart by as much of the largest.
  const float cut = (a.places + 1) * 1.1920929e-7f;
  const float off = 9.5367432e-7f + (a.sigmoid ? 0.0f : (a.each + 16) * 1.1920929e-7f);
  const int wave = threadIdx.x / kWave, lane = lane_id(), l = lane & 15;
  const int64_t first = ((int64_t)blockIdx.x * kRouteWaves + wave) * 4, token = first + lane / 16;
  if (first >= a.tokens) return;
  const bool valid = token < a.tokens, exact = BF16 && !a.bias;
  const int group = l >> a.shift, within = (l & ((1 << a.shift) - 1)) * a.each;
  const int e0 = group * a.per_group + within;
  const int n = valid && group < a.groups ? min(a.per_group - within, a.each) : 0;  // experts of this lane, if positive
  const int64_t row = valid ? token * a.row_stride : 0;

  // logits and biases of four experts; -inf where there are none
  auto four = [&](int j, float (&x)[4], float (&b)[4]) {
    if (a.vectors) {
      const int at = j < n ? e0 + j : 0;
      if constexpr (BF16) {
        const uint2 u = *(const uint2*)((const uint16_t*)a.logits + row + at);
        x[0] = __uint_as_float(u.x << 16);
        x[1] = __uint_as_float(u.x & 0xffff0000u);
        x[2] = __uint_as_float(u.y << 16);
        x[3] = __uint_as_float(u.y & 0xffff0000u);
      } else {
        const float4 u = *(const float4*)((const float*)a.logits + row + at);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      }
      const float4 u = a.bias ? *(const float4*)(a.bias + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = j + i < n ? e0 + j + i : 0;
        x[i] = BF16 ? __uint_as_float((uint32_t)((const uint16_t*)a.logits)[row + at] << 16) : ((const float*)a.logits)[row + at];
        b[i] = a.bias ? a.bias[at] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = j + i < n ? x[i] : -INFINITY;
  };

  // softmax: the sum over all experts, where scores are compared
  const bool scores = a.bias || (a.groups > 1 && a.group_top == 2);
  float top = 0.0f, sum = 1.0f;  // top: 0 for sigmoid scores
  if (!a.sigmoid && scores) {
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll 1
    for (int j = 0; j < a.each; j += 4) {
      float x[4], b[4];
      four(j, x, b);
      float m = top;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = x[i] > m ? fminf(x[i], kMost) : m;
      const float base = m == -INFINITY ? 0.0f : m;
      sum *= __builtin_amdgcn_exp2f((top - base) * kLog2e);
      top = m;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sum += x[i] > -INFINITY ? __builtin_amdgcn_exp2f((fminf(x[i], kMost) - base) * kLog2e) : 0.0f;
    }
    const float m = row_max_f(top), base = m == -INFINITY ? 0.0f : m;
    sum = row_sum_f(sum * __builtin_amdgcn_exp2f((top - base) * kLog2e));
    top = base;
  }
  const float inverse = 1.0f / sum, largest = a.sigmoid ? 1.0f : inverse;  // of all scores
  auto score_of = [&](float v) {
    return a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e))
                     : __builtin_amdgcn_exp2f((v - top) * kLog2e) * inverse;
  };

  int key[L];
#pragma unroll
  for (int i = 0; i < L; ++i) key[i] = kNone;
#pragma unroll 1
  for (int j = 0; j < a.each; j += 4) {
    float x[4], b[4];
    int k[4];
    four(j, x, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool here = (x[i] > -INFINITY) & (b[i] == b[i]);  // not NaN either
      const float v = x[i] + 0.0f;                            // -0 is 0
      if (exact) {
        k[i] = (ordered(v) & (int)0xffff0000) | (0xffff - (e0 + j + i));
      } else {
        float f = fminf(v, kMost);
        if (a.bias) f = score_of(f) + __builtin_amdgcn_fmed3f(b[i], -kMost, kMost);
        k[i] = (ordered(f) & ~a.places) | (a.places - (j + i));
      }
      k[i] = here ? k[i] : kNone;
    }
    insert_four<L>(key, k);
  }
  bool near = false;
  // A key's logit, or score plus bias, without the expert's place: as it is where bfloat16 left its bits free (a negative
  // number's are ones in its order), else the end of what the key stands for.
  auto value = [&](int k) { return from_ordered(!exact ? k & ~a.places : k < 0 ? k | 0xffff : k & (int)0xffff0000); };
  // in 64 bits, for the few tokens that need it
  auto exact_sum = [&]() {
    double all = 0.0;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const float v = logit_at<BF16>(a, token, e0 + j);
      all += v > -INFINITY ? exp((double)fminf(v, kMost) - (double)top) : 0.0;
    }
    return row_sum_d(all);
  };
  auto exact_key = [&](float v, float b, double all) {
    const double e = exp(a.sigmoid ? -(double)v : (double)v - (double)top);
    return (a.sigmoid ? 1.0 / (1.0 + e) : e / all) + (double)__builtin_amdgcn_fmed3f(b, -kMost, kMost);
  };
  // whether two keys, in this order, are too near to tell
  auto close = [&](int larger, int smaller) {
    const float p = value(larger), q = value(smaller);
    return (smaller != kNone) & (a.bias ? p - q <= cut * fmaxf(fabsf(p), fabsf(q)) + off * largest : p == q);
  };
  auto expert_of = [&](int k, int lane_of) {
    return exact ? 0xffff - (k & 0xffff)
                 : (lane_of >> a.shift) * a.per_group + (lane_of & ((1 << a.shift) - 1)) * a.each + a.places - (k & a.places);
  };
  if (a.groups > 1) {
    int k0 = key[0], k1 = key[1];
#pragma unroll 1
    for (int d = 1; d >> a.shift == 0; d <<= 1) {
      const int o0 = (int)from_lane((uint32_t)k0, lane ^ d), o1 = (int)from_lane((uint32_t)k1, lane ^ d);
      k1 = max(min(k0, o0), max(k1, o1));
      k0 = max(k0, o0);
    }
    // the group's rank, and how far any two of the token may be off; whole: integers, which are exact
    const bool whole = a.group_top == 1 && exact, two = a.group_top == 2 && k1 != kNone;
    float rank = value(k0), room = cut * fabsf(rank);
    const float v1 = two ? value(k1) : 0.0f;
    if (a.bias) {
      room += cut * fabsf(v1);
      rank += v1;
      if (!(fabsf(rank) <= kMost)) room = INFINITY;  // past float32: only 64 bits tell it from others
    } else if (a.group_top == 2) {
      const float far = fmaxf(fabsf(rank), fabsf(v1)) + fabsf(top);
      rank = score_of(rank) + (two ? score_of(v1) : 0.0f);
      room = 2.0f * (cut + off) * rank * (1.0f + far);
    }
    const bool none = k0 == kNone || group >= a.groups;
    if (whole) rank = __int_as_float(0);
    rank = none ? -INFINITY : rank;
    room = row_max_f(none ? 0.0f : room) + (a.bias ? a.group_top * off * largest : 0.0f);
    const int number = none ? kNone : k0;
    int before = 0;
    float over = INFINITY, under = INFINITY;  // to the nearest group that comes before, and after
#pragma unroll 1
    for (int r = 1 << a.shift; r < 16; r += 1 << a.shift) {
      const int from = (l + r) & 15, other = (lane & 48) | from;
      const bool lower = from >> a.shift < group;
      const float o = __uint_as_float(from_lane(__float_as_uint(rank), other));
      const int i = (int)from_lane((uint32_t)number, other);
      const bool first_ = whole ? (i > number) | ((i == number) & lower) : (o > rank) | ((o == rank) & lower);
      before += first_;
      const float d = fabsf(o - rank);  // NaN where both have none
      over = first_ ? fminf(over, d) : over;
      under = first_ ? under : fminf(under, d);
    }
    // too near: the last group that is chosen and the first that is not
    const bool border = before == a.top_groups - 1 ? under <= room : before == a.top_groups && over <= room;
    if (!whole && __ballot(border & valid)) {
      // of each lane's first four: its two largest are among them, unless the second and the fifth are as near
      const double all = a.sigmoid || !scores ? 1.0 : exact_sum();
      double m0 = kGone, m1 = kGone;
      near = near | close(key[1], key[4]);
      int k[4] = {key[0], key[1], key[2], key[3]};
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int e = expert_of(k[0], l);
        const float v = k[0] != kNone ? fminf(logit_at<BF16>(a, token, e), kMost) : 0.0f;
        const double y = !scores ? (double)v : exact_key(v, a.bias && k[0] != kNone ? a.bias[e] : 0.0f, all);
        if (k[0] != kNone) {
          m1 = fmax(m1, fmin(m0, y));
          m0 = fmax(m0, y);
        }
        k[0] = k[1], k[1] = k[2], k[2] = k[3];
      }
#pragma unroll 1
      for (int d = 1; d >> a.shift == 0; d <<= 1) {
        const double o0 = from_lane_d(m0, lane ^ d), o1 = from_lane_d(m1, lane ^ d);
        m1 = fmax(fmin(m0, o0), fmax(m1, o1));
        m0 = fmax(m0, o0);
      }
      if (a.group_top == 2 && m1 > kGone) m0 += m1;
      before = count_before(group < a.groups ? m0 : kTaken, group, l, 1 << a.shift, 16);
    }
    if (before >= a.top_groups) {
#pragma unroll
      for (int i = 0; i < L; ++i) key[i] = kNone;
    }
  }
  // the lists' ends: what a lane had no room for comes after its own
  const int end = n > L ? key[L - 1] : kNone;
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
    for (int j = 0; j < L; ++j) key[j] = (pop & (j + 1 < L ? key[j + 1 < L ? j + 1 : 0] : kNone)) | (~pop & key[j]);
  }
  near = near | ((l < a.k) & (mine == kNone));
  bool order = false;  // of this choice and the one before it is open
  int picks = a.k;     // lanes that hold one
  if (!exact) {
    const int next = row_max(key[0]);
    const bool edge = (l == a.k - 1) & close(mine, next);  // of the last choice and the next
    // where a lane's whole list may be chosen, or next: whether the last choice is as near to what it had no room for
    if (a.k >= L - 1) near = near | ((l == a.k - 1) & close(mine, row_max(end)));
    order = (l > 0) & (l < a.k) & close(row_ror<1>(mine), mine);
    const uint64_t edges = __ballot(edge & valid);
    if (edges) {  // then the next is a choice too, of which one is left out; of other tokens of the wave it is not
      if (a.k == 16) {
        near = near | edge;
      } else {
        const int src = __ffs((int)(uint32_t)((__ballot(key[0] == next) >> (lane & 48)) & 0xffff)) - 1;
        const int third = row_max(l == src ? key[1] : key[0]);
        near = near | (edge & close(mine, third));
        const bool here = (edges >> (lane & 48)) & 0xffff;
        mine = here & (l == a.k) ? next : mine;
        from = here & (l == a.k) ? src : from;
        picks = a.k + (here & (next != kNone));
        order = order | edge;
      }
    }
  }
  const int at = expert_of(mine, from);
  const bool picked = valid & (l < picks) & (mine != kNone);
  const float logit = picked ? fminf(logit_at<BF16>(a, token, at), kMost) : -INFINITY;
  // scores that 64 bits may not hold, and whose sum may be 0, or that power() does not reach (2^-1000 is e^-693.1)
  if (a.renormalise && (a.sigmoid || scores)) near = near | (picked & (logit - top < -690.0f));
  const uint64_t unsure = __ballot(near & valid);
  const bool chosen = picked && ((unsure >> (lane & 48)) & 0xffff) == 0;
  double w = 0.0;
  if (a.sigmoid) {
    w = reciprocal(1.0 + power(-(double)logit));
  } else {
    // without a bias the largest logit of all is among the choices
    const float base = a.renormalise || !scores ? row_max_f(logit) : top;
    w = power((double)logit - (double)base);
    if (!a.renormalise) {  // a sum of 32 bits would be off by some steps of the weight
      double all = 0.0;
#pragma unroll 1
      for (int j = 0; j < a.each; j += 4) {
        float x[4], b[4];
        four(j, x, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) all += x[i] > -INFINITY ? power((double)fminf(x[i], kMost) - (double)base) : 0.0;
      }
      w *= reciprocal(row_sum_d(all));
    }
  }
  int place = chosen ? l : 16;
  if (__ballot(order & chosen)) {
    const double all = a.sigmoid || !a.bias ? 1.0 : exact_sum();
    const double exactly = !a.bias ? (double)logit : exact_key(logit, picked ? a.bias[at] : 0.0f, all);
    const int before = count_before(exactly, at, l, 1, picks);
    place = chosen ? before : 16;
  }
  const bool kept = place < a.k;
  w = kept ? w : 0.0;
  if (a.renormalise) {
    const double all = row_sum_d(w);
    w = all > 0.0 ? w * reciprocal(all) : 0.0;
  }
  if (kept) {
    a.weights[token * a.k + place] = (float)(w * a.scale);
    a.ids[token * a.k + place] = at;
  }
#pragma unroll 1
  for (int r = 0; r < 4; ++r)
    if ((unsure >> (16 * r)) & 0xffff) route_exactly<BF16, NJ>(a, first + r, lds + wave * a.experts);
}

template <bool BF16, int L>
static int launch_rows(const RouteArgs& a, size_t lds, hipStream_t s) {
  constexpr int kTokens = kRouteWaves * 4, kThreads = kRouteWaves * kWave;
  const unsigned grid = (unsigned)((a.tokens + kTokens - 1) / kTokens);
  if (a.experts <= 256) route_kernel<BF16, L, 4><<<grid, kThreads, lds, s>>>(a);
  else route_kernel<BF16, L, 16><<<grid, kThreads, lds, s>>>(a);
  return launch_status("route");
}

template <bool BF16>
static int launch_route(RouteArgs a, hipStream_t s) {
  const size_t lds = a.groups > 1 ? (size_t)kRouteWaves * a.experts * 8 : 0;
  // lanes of a group: a power of two, all groups in 16
  int shift = 4;
  while (shift > 0 && a.groups << shift > 16) --shift;
  if (a.groups <= 16 && a.k <= 16) {
    const int bytes = BF16 ? 2 : 4;
    a.shift = shift;
    a.each = (((a.per_group + (1 << shift) - 1) >> shift) + 3) / 4 * 4;  // at most 116: 9 groups of 113, with 127 places
    a.places = 3;
    while (a.places < a.each - 1) a.places = 2 * a.places + 1;
    a.vectors = ((uintptr_t)a.logits | (uintptr_t)(a.row_stride * bytes)) % (4 * bytes) == 0 && (uintptr_t)a.bias % 16 == 0 &&
                a.per_group % 4 == 0;
    return a.k <= 8 ? launch_rows<BF16, 8>(a, lds, s) : launch_rows<BF16, 16>(a, lds, s);
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
  if (experts > kMostExperts || groups > kMostGroups || k > kMostChosen || tokens > (1 << 25) ||
      row_stride > ((int64_t)1 << 37)) {  // the logits' addresses are 64 bits wide
    set_error("route: up to %d experts, %d groups, %d chosen, 2^25 tokens, rows up to 2^37 elements apart", kMostExperts,
              kMostGroups, kMostChosen);
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
