// Verification of drafted tokens against the target's softmax, and the draw of
// the next token.
//
// Three launches.  verify_stats reads every row of logits once: maximum and sum
// of weights of each chunk (and the place of the maximum for greedy rows).
// verify_race joins them for a sequence's rows, finds how many drafts are
// accepted, and races the elements of the one row that the next token comes
// from, a chunk per workgroup.  verify_finish joins the chunks and writes the
// tokens.
//
// A token hangs on every comparison, so comparisons are made in 64 bits:
// sums of 32-bit weights are joined in 64, an accepted draft's probability is
// computed in 64, and the race computes 32-bit scores with a bound on their
// error and evaluates in 64 bits only those that may be the largest.
#include <float.h>
#include <math.h>

#include "tx_common.h"
#include "tx_host.h"

#include "tallax_hip.h"

namespace tx {

constexpr int kVerThreads = 256;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr int kMaxDrafted = 63;
constexpr int kRaceItems = 16;                           // elements of a thread in the race
constexpr int kRaceChunk = kVerThreads * kRaceItems;
constexpr float kGreedy = 1e-5f;

struct RowPart {  // a chunk of a row
  double sum;     // of exp((l - max) / temperature)
  float max;
  int32_t at;     // greedy rows: the first place of max
};

struct RacePart {
  double score;
  int64_t at;  // -1: no positive weight
};

struct VerifyArgs {
  const int32_t* draft;
  const void* logits;
  int64_t vocab;
  int batch, drafted;
  const int32_t* counts;
  const float* temperature;
  const void* probs;
  int probs_bf16;
  const float* uniforms;
  const float* noise;
  int32_t* tokens;
  int32_t* accepted;
  RowPart* parts;  // [batch * (drafted + 1)][stat_chunks]
  int stat_chunks;
  int64_t stat_vecs;  // 16-byte blocks of a chunk
  RacePart* race;     // [batch][race_chunks]
  int race_chunks;
};

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.drafted) : a.drafted;
}

// NaN counts as -inf, and +inf as the largest number, so that +inf logits
// share the whole weight.
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -INFINITY), FLT_MAX); }

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if constexpr (DT == kBF16) return clean(__uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16));
  return clean(((const float*)p)[i]);
}

// log2(e) / temperature in two parts, so that a weight's exponent is off by its
// own rounding alone (a rounded factor would shift every sum the same way).
struct Scale {
  float hi, lo;
  __device__ __forceinline__ explicit Scale(float temperature) {
    const double f = 1.4426950408889634 / (double)temperature;
    hi = (float)f;
    lo = (float)(f - (double)hi);
    if (!(fabsf(lo) <= FLT_MAX)) lo = 0.0f;
  }
  // exp((l - max) / temperature); d = l - max <= 0
  __device__ __forceinline__ float weight(float d) const {
    const float x = d * hi;
    const float y = __builtin_fmaf(d, lo, __builtin_fmaf(d, hi, -x));
    // below 2^-150 (also where the product is -inf, or NaN for -inf at an infinite temperature) the weight is 0
    return !(x >= -150.0f) ? 0.0f : __builtin_amdgcn_exp2f(x + y);
  }
};

__device__ __forceinline__ double lane_xor_d(double x, int d) {
  return __longlong_as_double((long long)shfl_xor_u64((uint64_t)__double_as_longlong(x), d));
}

template <int DT>
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyArgs a) {
  constexpr int N = DT == kBF16 ? 8 : 4;  // elements of 16 bytes
  constexpr int V = 4;                    // blocks of a thread at a time
  __shared__ float red_max[kVerWaves];
  __shared__ double red_sum[kVerWaves];
  __shared__ int red_at[kVerWaves];
  const int row = blockIdx.y, b = row / (a.drafted + 1), i = row - b * (a.drafted + 1);
  if (i > drafts_of(a, b)) return;
  const float temperature = a.temperature[b];
  const bool greedy = temperature < kGreedy;
  const Scale scale(greedy ? 1.0f : temperature);
  const int tid = threadIdx.x, wave = tid / kWave;
  const char* base = (const char*)a.logits + (int64_t)row * a.vocab * (16 / N);
  const RowVec<16 / N> rv(base);
  const int64_t blocks = (a.vocab + rv.mis + N - 1) / N;
  const int64_t first = blockIdx.x * a.stat_vecs, last = min(first + a.stat_vecs, blocks);
  float m = -INFINITY, s = 0.0f;
  int32_t at = INT32_MAX;
  for (int64_t v0 = first + tid; v0 < last; v0 += kVerThreads * V) {
    float x[V * N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t blk = v0 + v * kVerThreads;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (blk < last) w = load_once(rv.base + blk);
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = DT == kBF16 ? __uint_as_float((e & 1) ? ww[e / 2] & 0xFFFF0000u : ww[e / 2] << 16)
                                    : __uint_as_float(ww[e & 3]);
        const int64_t el = blk * N + e - rv.mis;
        x[v * N + e] = blk < last && el >= 0 && el < a.vocab ? clean(l) : -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < V * N; ++e) top = fmaxf(top, x[e]);
    if (greedy) {
      if (top > m) {
        m = top;
        at = INT32_MAX;
#pragma unroll
        for (int e = V * N - 1; e >= 0; --e)
          if (x[e] == top) at = (int32_t)((v0 + (e / N) * kVerThreads) * N + e % N - rv.mis);
      }
    } else if (top > -INFINITY) {
      if (top > m) {
        s = m == -INFINITY ? 0.0f : s * scale.weight(m - top);
        m = top;
      }
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < V * N; ++e) t += scale.weight(x[e] - m);
      s += t;
    }
  }
  float wm = m;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) wm = fmaxf(wm, lane_xor_f(wm, d));
  if (lane_id() == 0) red_max[wave] = wm;
  __syncthreads();
  float bm = red_max[0];
#pragma unroll
  for (int w = 1; w < kVerWaves; ++w) bm = fmaxf(bm, red_max[w]);
  double sum = m == -INFINITY ? 0.0 : (double)s * (double)scale.weight(m - bm);
  int first_at = m == bm ? at : INT32_MAX;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    sum += lane_xor_d(sum, d);
    first_at = min(first_at, (int)lane_xor((uint32_t)first_at, d));
  }
  if (lane_id() == 0) {
    red_sum[wave] = sum;
    red_at[wave] = first_at;
  }
  __syncthreads();
  if (tid == 0) {
    RowPart p;
    p.max = bm;
    p.sum = 0.0;
    p.at = INT32_MAX;
    for (int w = 0; w < kVerWaves; ++w) {
      p.sum += red_sum[w];
      p.at = min(p.at, red_at[w]);
    }
    a.parts[(int64_t)row * a.stat_chunks + blockIdx.x] = p;
  }
}

// Maximum, sum of weights and place of the maximum of a row, by 16 lanes (`l`
// of them this one); the same in all of them.
struct RowStat {
  double sum;
  float max;
  int32_t at;
};

__device__ __forceinline__ RowStat join_row(const VerifyArgs& a, int64_t row, int l, double inv_t) {
  const RowPart* p = a.parts + row * a.stat_chunks;
  float m = -INFINITY;
  for (int c = l; c < a.stat_chunks; c += 16) m = fmaxf(m, p[c].max);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, lane_xor_f(m, d));
  RowStat r;
  r.max = m;
  r.sum = 0.0;
  r.at = INT32_MAX;
  for (int c = l; c < a.stat_chunks; c += 16) {
    const RowPart x = p[c];
    if (x.max == m) r.at = min(r.at, x.at);
    if (x.max > -INFINITY) r.sum += x.sum * exp(((double)x.max - (double)m) * inv_t);
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    r.sum += lane_xor_d(r.sum, d);
    r.at = min(r.at, (int)lane_xor((uint32_t)r.at, d));
  }
  return r;
}

__device__ __forceinline__ double prob_of_draft(const VerifyArgs& a, int64_t row, int64_t v) {
  const int64_t at = row * a.vocab + v;
  if (a.probs_bf16) return (double)__uint_as_float((uint32_t)((const uint16_t*)a.probs)[at] << 16);
  return (double)((const float*)a.probs)[at];
}

// What a sequence draws its next token from.
struct Drawn {
  int n;        // accepted drafts
  int refused;  // whether draft n was refused
  RowStat row;  // of row n
};

// By the whole workgroup (its first waves hold 16 rows at a time).
template <int DT>
__device__ __forceinline__ Drawn accept_drafts(const VerifyArgs& a, int b, Drawn* shared, RowStat* stats, int* ok) {
  const int cnt = drafts_of(a, b), tid = threadIdx.x;
  const float temperature = a.temperature[b];
  const bool greedy = temperature < kGreedy;
  const double inv_t = greedy ? 1.0 : 1.0 / (double)temperature;
  for (int i = tid / 16; i <= cnt; i += kVerThreads / 16) {
    const int64_t row = (int64_t)b * (a.drafted + 1) + i;
    const RowStat r = join_row(a, row, tid & 15, inv_t);
    if ((tid & 15) == 0) {
      stats[i] = r;
      bool good = false;
      if (i < cnt) {
        const int64_t at = (int64_t)b * a.drafted + i;
        const int32_t x = a.draft[at];
        if (x >= 0 && x < a.vocab && r.max > -INFINITY) {
          if (greedy) {
            good = x == r.at;
          } else {
            const char* base = (const char*)a.logits + row * a.vocab * (DT == kBF16 ? 2 : 4);
            const double p = exp(((double)logit_at<DT>(base, x) - (double)r.max) * inv_t) / r.sum;
            const double q = a.probs ? prob_of_draft(a, at, x) : 1.0;
            good = (double)a.uniforms[at] * q < p;
          }
        }
      }
      ok[i] = good;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    while (n < cnt && ok[n]) ++n;
    shared->n = n;
    shared->refused = n < cnt;
    shared->row = stats[n];
  }
  __syncthreads();
  return *shared;
}

// One element of the race in 64 bits: (p - q) / noise, or p / noise.
template <int DT>
__device__ __forceinline__ double exact_score(const VerifyArgs& a, const char* logits, double inv_t, const RowStat& r,
                                              double q, float noise, int64_t v) {
  const double p = exp(((double)logit_at<DT>(logits, v) - (double)r.max) * inv_t) / r.sum;
  return (p - q) / (double)noise;
}

__device__ __forceinline__ void take_better(double& s, int64_t& at, double os, int64_t oat) {
  if (oat >= 0 && (at < 0 || os > s || (os == s && oat < at))) {
    s = os;
    at = oat;
  }
}

template <int DT>
__device__ __forceinline__ RacePart race_chunk(const VerifyArgs& a, int b, const Drawn& d, int64_t first, bool plain,
                                               float* red, RacePart* red_best) {
  const int tid = threadIdx.x, wave = tid / kWave;
  const float temperature = a.temperature[b];
  const double inv_t = 1.0 / (double)temperature;
  const Scale scale(temperature);
  const int64_t row = (int64_t)b * (a.drafted + 1) + d.n;
  const char* logits = (const char*)a.logits + row * a.vocab * (DT == kBF16 ? 2 : 4);
  const float* noise = a.noise + (int64_t)b * a.vocab;
  const int64_t qrow = (int64_t)b * a.drafted + d.n;
  const bool with_q = d.refused && !plain;
  const int64_t certain = with_q && !a.probs ? a.draft[qrow] : -1;
  const float inv_sum = (float)(1.0 / d.row.sum);
  float hi[kRaceItems];
  float low = 0.0f;
#pragma unroll
  for (int k = 0; k < kRaceItems; ++k) {
    const int64_t v = first + k * kVerThreads + tid;
    hi[k] = 0.0f;
    if (v >= a.vocab) continue;
    const float p = scale.weight(logit_at<DT>(logits, v) - d.row.max) * inv_sum;
    const float q = !with_q ? 0.0f : a.probs ? (float)prob_of_draft(a, qrow, v) : v == certain ? 1.0f : 0.0f;
    const float e = noise[v];
    // p is off by at most 2^-17 of itself (its exponent is as low as -150 and rounded to half of 2^-16; exp2
    // and four roundings add little) and by what lies below the normal numbers, the quotient by 2^-22 more
    const float slack = p * 0x1p-16f + 0x1p-120f;
    hi[k] = (p - q + slack) / e * (1.0f + 0x1p-20f);
    low = fmaxf(low, (p - q - slack) / e * (1.0f - 0x1p-20f));
  }
#pragma unroll
  for (int x = 1; x < kWave; x <<= 1) low = fmaxf(low, lane_xor_f(low, x));
  if (lane_id() == 0) red[wave] = low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w) low = fmaxf(low, red[w]);
  double best = 0.0;
  int64_t at = -1;
#pragma unroll
  for (int k = 0; k < kRaceItems; ++k) {
    if (hi[k] > 0.0f && hi[k] >= low) {
      const int64_t v = first + k * kVerThreads + tid;
      const double q = !with_q ? 0.0 : a.probs ? prob_of_draft(a, qrow, v) : v == certain ? 1.0 : 0.0;
      const double s = exact_score<DT>(a, logits, inv_t, d.row, q, noise[v], v);
      if (s > 0.0) take_better(best, at, s, v);
    }
  }
#pragma unroll
  for (int x = 1; x < kWave; x <<= 1) {
    const double os = lane_xor_d(best, x);
    const int64_t oat = (int64_t)shfl_xor_u64((uint64_t)at, x);
    take_better(best, at, os, oat);
  }
  if (lane_id() == 0) red_best[wave] = {best, at};
  __syncthreads();
  RacePart r = red_best[0];
#pragma unroll
  for (int w = 1; w < kVerWaves; ++w) take_better(r.score, r.at, red_best[w].score, red_best[w].at);
  __syncthreads();
  return r;
}

struct VerifyShared {
  Drawn drawn;
  RowStat stats[kMaxDrafted + 1];
  int ok[kMaxDrafted + 1];
  float red[kVerWaves];
  RacePart best[kVerWaves];
};

template <int DT>
__global__ __launch_bounds__(kVerThreads) void verify_race_kernel(VerifyArgs a) {
  __shared__ VerifyShared sh;
  const int b = blockIdx.y;
  if (a.temperature[b] < kGreedy) return;
  const Drawn d = accept_drafts<DT>(a, b, &sh.drawn, sh.stats, sh.ok);
  RacePart r = {0.0, -1};
  if (d.row.max > -INFINITY)
    r = race_chunk<DT>(a, b, d, (int64_t)blockIdx.x * kRaceChunk, false, sh.red, sh.best);
  if (threadIdx.x == 0) a.race[(int64_t)b * a.race_chunks + blockIdx.x] = r;
}

template <int DT>
__global__ __launch_bounds__(kVerThreads) void verify_finish_kernel(VerifyArgs a) {
  __shared__ VerifyShared sh;
  const int b = blockIdx.x, tid = threadIdx.x;
  const Drawn d = accept_drafts<DT>(a, b, &sh.drawn, sh.stats, sh.ok);
  int64_t token = -1;
  if (a.temperature[b] < kGreedy) {
    if (d.row.max > -INFINITY) token = d.row.at;
  } else if (d.row.max > -INFINITY) {
    double best = 0.0;
    int64_t at = -1;
    for (int c = tid; c < a.race_chunks; c += kVerThreads) {
      const RacePart r = a.race[(int64_t)b * a.race_chunks + c];
      take_better(best, at, r.score, r.at);
    }
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) {
      const double os = lane_xor_d(best, x);
      const int64_t oat = (int64_t)shfl_xor_u64((uint64_t)at, x);
      take_better(best, at, os, oat);
    }
    if (lane_id() == 0) sh.best[tid / kWave] = {best, at};
    __syncthreads();
    RacePart r = sh.best[0];
    for (int w = 1; w < kVerWaves; ++w) take_better(r.score, r.at, sh.best[w].score, sh.best[w].at);
    __syncthreads();
    if (r.at < 0) {  // p - q is nowhere positive (rounded probabilities): drawn from p
      for (int c = 0; c < a.race_chunks; ++c) {
        const RacePart o = race_chunk<DT>(a, b, d, (int64_t)c * kRaceChunk, true, sh.red, sh.best);
        take_better(r.score, r.at, o.score, o.at);
      }
    }
    token = r.at;
  }
  for (int t = tid; t <= a.drafted; t += kVerThreads)
    a.tokens[(int64_t)b * (a.drafted + 1) + t] =
        t < d.n ? a.draft[(int64_t)b * a.drafted + t] : t == d.n ? (int32_t)token : -1;
  if (tid == 0) a.accepted[b] = d.n;
}

struct VerifyPlan {
  int stat_chunks, race_chunks;
  int64_t stat_vecs;
  size_t part_bytes, race_bytes;
};

static VerifyPlan plan_verify(int64_t batch, int64_t drafted, int64_t vocab, int dtype) {
  VerifyPlan p;
  const int64_t n = dtype == TALLAX_BF16 ? 8 : 4;
  const int64_t blocks = (vocab + n - 1) / n + 1;  // a row may begin inside a block
  p.stat_vecs = kVerThreads * 4;
  p.stat_chunks = (int)((blocks + p.stat_vecs - 1) / p.stat_vecs);
  p.race_chunks = (int)((vocab + kRaceChunk - 1) / kRaceChunk);
  p.part_bytes = align_up((size_t)(batch * (drafted + 1)) * p.stat_chunks * sizeof(RowPart), 256);
  p.race_bytes = (size_t)batch * p.race_chunks * sizeof(RacePart);
  return p;
}

template <int DT>
static int launch_verify(const VerifyArgs& a, hipStream_t s) {
  verify_stats_kernel<DT><<<dim3(a.stat_chunks, a.batch * (a.drafted + 1)), kVerThreads, 0, s>>>(a);
  verify_race_kernel<DT><<<dim3(a.race_chunks, a.batch), kVerThreads, 0, s>>>(a);
  verify_finish_kernel<DT><<<a.batch, kVerThreads, 0, s>>>(a);
  return launch_status("verify");
}

}  // namespace tx

using namespace tx;

extern "C" {

size_t tallax_verify_workspace_size(int64_t batch, int64_t drafted, int64_t vocab, int logits_dtype) {
  if (batch < 0 || drafted < 0 || vocab < 1) return 0;
  const VerifyPlan p = plan_verify(batch, drafted, vocab, logits_dtype);
  return p.part_bytes + p.race_bytes;
}

int tallax_verify(const int32_t* draft, const void* logits, int logits_dtype, int64_t batch, int64_t drafted,
                  int64_t vocab, const int32_t* counts, const float* temperature, const void* draft_probs,
                  int probs_dtype, const float* uniforms, const float* noise, int32_t* out_tokens,
                  int32_t* out_accepted, void* workspace, size_t workspace_bytes, tallax_stream_t stream) {
  if (batch < 0 || drafted < 0 || vocab < 1 || vocab > INT32_MAX) {
    set_error("verify: batch %lld, drafted %lld, vocab %lld", (long long)batch, (long long)drafted, (long long)vocab);
    return kInvalidArgument;
  }
  if (drafted > kMaxDrafted || batch * (drafted + 1) > 65535) {
    set_error("verify: %lld drafted tokens (at most %d), %lld rows of logits (at most 65535)", (long long)drafted,
              kMaxDrafted, (long long)(batch * (drafted + 1)));
    return kUnsupported;
  }
  if ((logits_dtype != TALLAX_F32 && logits_dtype != TALLAX_BF16) ||
      (draft_probs && probs_dtype != TALLAX_F32 && probs_dtype != TALLAX_BF16)) {
    set_error("verify: logits and draft probabilities are float32 or bfloat16");
    return kUnsupported;
  }
  if (batch == 0) return kOk;
  if (!logits || !temperature || !noise || !out_tokens || !out_accepted || (drafted > 0 && (!draft || !uniforms))) {
    set_error("verify: null pointer");
    return kInvalidArgument;
  }
  const VerifyPlan p = plan_verify(batch, drafted, vocab, logits_dtype);
  if (!workspace || workspace_bytes < p.part_bytes + p.race_bytes) {
    set_error("verify: workspace of %zu bytes, %zu needed", workspace_bytes, p.part_bytes + p.race_bytes);
    return kWorkspaceTooSmall;
  }
  VerifyArgs a;
  a.draft = draft;
  a.logits = logits;
  a.vocab = vocab;
  a.batch = (int)batch;
  a.drafted = (int)drafted;
  a.counts = counts;
  a.temperature = temperature;
  a.probs = draft_probs;
  a.probs_bf16 = probs_dtype == TALLAX_BF16;
  a.uniforms = uniforms;
  a.noise = noise;
  a.tokens = out_tokens;
  a.accepted = out_accepted;
  a.parts = (RowPart*)workspace;
  a.stat_chunks = p.stat_chunks;
  a.stat_vecs = p.stat_vecs;
  a.race = (RacePart*)((char*)workspace + p.part_bytes);
  a.race_chunks = p.race_chunks;
  return logits_dtype == TALLAX_BF16 ? launch_verify<kBF16>(a, (hipStream_t)stream)
                                     : launch_verify<kF32>(a, (hipStream_t)stream);
}

}  // extern "C"
