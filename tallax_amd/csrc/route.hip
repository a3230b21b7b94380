// Routing tokens to experts: scores, the choice of groups, the choice of
// experts and their weights, a wave for each token.
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
  int experts, k, groups, per_group, top_groups, group_top, renormalise;
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

template <bool BF16, bool SIGMOID, int NJ>
__global__ __launch_bounds__(kRouteWaves * kWave) void route_kernel(RouteArgs a) {
  extern __shared__ double lds[];  // [waves][experts] keys, where there are groups
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int64_t token = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (token >= a.tokens) return;
  constexpr float kMost = 3.4028234663852886e38f;
  float x[NJ];
  double s[NJ], key[NJ];
  bool here[NJ];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + j * kWave;
    float v = -INFINITY;
    if (e < a.experts) {
      if constexpr (BF16)
        v = __uint_as_float((uint32_t)((const uint16_t*)a.logits)[token * a.row_stride + e] << 16);
      else
        v = ((const float*)a.logits)[token * a.row_stride + e];
    }
    here[j] = v > -INFINITY;  // not NaN either
    x[j] = here[j] ? fminf(v, kMost) : -kMost;
    if (here[j]) top = fmaxf(top, x[j]);
  }
  if constexpr (SIGMOID) {
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
    double* keys = lds + wave * a.experts;
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

template <bool BF16, bool SIGMOID>
static int launch_route(const RouteArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((a.tokens + kRouteWaves - 1) / kRouteWaves);
  const size_t lds = a.groups > 1 ? (size_t)kRouteWaves * a.experts * 8 : 0;
  const int threads = kRouteWaves * kWave;
  if (a.experts <= 64) route_kernel<BF16, SIGMOID, 1><<<grid, threads, lds, s>>>(a);
  else if (a.experts <= 128) route_kernel<BF16, SIGMOID, 2><<<grid, threads, lds, s>>>(a);
  else if (a.experts <= 256) route_kernel<BF16, SIGMOID, 4><<<grid, threads, lds, s>>>(a);
  else if (a.experts <= 512) route_kernel<BF16, SIGMOID, 8><<<grid, threads, lds, s>>>(a);
  else route_kernel<BF16, SIGMOID, 16><<<grid, threads, lds, s>>>(a);
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
  a.renormalise = renormalise;
  a.bias = bias;
  a.scale = scale;
  a.weights = out_weights;
  a.ids = out_ids;
  hipStream_t s = (hipStream_t)stream;
  if (logits_dtype == TALLAX_BF16) return sigmoid ? launch_route<true, true>(a, s) : launch_route<true, false>(a, s);
  return sigmoid ? launch_route<false, true>(a, s) : launch_route<false, false>(a, s);
}

}  // extern "C"
