// Verification of drafted tokens against the target's softmax, and the draw of
// the next token.
//
// Two launches, or three.  verify_stats reads every row of logits once: maximum
// and sum of weights of each chunk (and the place of the maximum for greedy
// rows); one more workgroup a sequence looks up the drafts' logits and
// probabilities.  verify_accept joins a sequence's rows and finds how many
// drafts are accepted; where the race is small its workgroups do that
// themselves.  verify_race races the elements of the one row that the next token
// comes from, a chunk per workgroup; the last workgroup of a sequence to finish
// joins the chunks and writes the tokens.
//
// Bound by memory: 64 sequences of 5 rows of 128256 bfloat16, with the draft's
// probabilities, 42 us for the 136 MB that it reads, rows past a sequence's
// drafts left out (3.2 TB/s: 19 us for the rows, 5 and 20 for the rest); 130 of 8
// rows of 151937 float32, drafts without, 116 us for 666 MB (5.7 TB/s).  At one
// sequence (14 us) each launch is a chain of loads that wait for each other.
//
// A token hangs on every comparison, so comparisons are made in 64 bits: an
// accepted draft's probability is computed in 64, and the race computes 32-bit
// scores with a bound on their error and evaluates in 64 bits only those that
// may be the largest.  A row's sum is of 32-bit weights, added up in 32 bits by
// each thread and joined in 64: 64-bit exponentials of every logit would take
// longer than reading it.  The sum is off by some 1e-7 of itself, so a draft
// whose u q is as near as that to p may fall on either side.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "tx_common.h"
#include "tx_host.h"

#include "tallax_hip_testing.h"

namespace tx {

constexpr int kVerThreads = 256;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr int kMaxDrafted = 63;
constexpr int kRaceVec = 8;  // neighbouring elements of a thread in a step of the race
// A counter has its cache lines to itself: 63 workgroups of each of 64 sequences
// raising counters side by side took 20 us longer.
constexpr int kDoneStride = 64;
// Up to this many workgroups of the race each finds the accepted drafts itself,
// beyond it a launch of its own does: 16 sequences of 50257 elements (400
// workgroups) take 16.8 us against 19.1, 64 of 128256 (4032) 46.2 against 43.6.
constexpr int kAcceptInRace = 1024;
constexpr float kGreedy = 1e-5f;

struct RowPart {  // a chunk of a row
  double sum;     // of exp((l - max) / temperature)
  float max;
  int32_t at;     // greedy rows: the first place of max
};

struct DraftPart {    // a drafted token
  double uq;          // uniform * q(token)
  float logit;
  int32_t token;      // -1: outside the vocabulary
};

// What a sequence draws its next token from.
struct Drawn {
  double inv_t;        // 1 / temperature
  double inv_sum;      // of the row's weights
  float max;
  float hi, lo;        // its Scale
  int32_t n;           // accepted drafts: the row
  int32_t what;        // kDone, kTarget, kRest
  int32_t certain;     // kRest without probabilities: the draft, else -1
};

constexpr int kDone = 0;    // no race: the tokens are written
constexpr int kTarget = 1;  // from p
constexpr int kRest = 2;    // from max(p - q, 0)

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
  DraftPart* drafts;  // [batch][drafted]
  Drawn* drawn;       // [batch]
  RacePart* race;     // [batch][race_chunks]
  int32_t* done;      // [batch][kDoneStride]: workgroups of the race that have written their part
  int race_chunks;
  int64_t race_size;  // elements of a chunk
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
// own rounding alone (a rounded factor would shift every sum the same way).  lo
// is positive, so that -inf stays -inf in the sum of both products.
struct Scale {
  float hi, lo;
  bool plain;  // weight_fast may be used: no product below overflows, or is 0 times infinity
  __device__ __forceinline__ explicit Scale(float temperature) {
    const double f = 1.4426950408889634 / (double)temperature;
    hi = (float)f;
    if ((double)hi > f) hi = __uint_as_float(__float_as_uint(hi) - 1);
    lo = (float)(f - (double)hi);
    plain = hi > 1e-20f && hi < 1e20f;
    lo = plain ? fmaxf(lo, 1e-37f) : lo <= FLT_MAX ? lo : 0.0f;
  }
  __device__ __forceinline__ Scale(float h, float l) : hi(h), lo(l), plain(false) {}
  // exp((l - max) / temperature); d = l - max <= 0
  __device__ __forceinline__ float weight(float d) const {
    const float x = d * hi;
    const float y = __builtin_fmaf(d, lo, __builtin_fmaf(d, hi, -x));
    // below 2^-150 (also where the product is -inf, or NaN for -inf at an infinite temperature) the weight is 0
    return !(x >= -150.0f) ? 0.0f : __builtin_amdgcn_exp2f(x + y);
  }
};

// A call: inlined, the constants of each exp stay in registers of their own
// through the kernel's loops (126 instead of 64 registers, half the waves).
__device__ __attribute__((noinline)) double exp_64(double x) { return exp(x); }

__device__ __forceinline__ double lane_xor_d(double x, int d) {
  return __longlong_as_double((long long)shfl_xor_u64((uint64_t)__double_as_longlong(x), d));
}

__device__ __forceinline__ double prob_of_draft(const VerifyArgs& a, int64_t row, int64_t v) {
  const int64_t at = row * a.vocab + v;
  if (a.probs_bf16) return (double)__uint_as_float((uint32_t)((const uint16_t*)a.probs)[at] << 16);
  return (double)((const float*)a.probs)[at];
}

// Elements of V 16-byte blocks kVerThreads apart from blk on; `last` blocks in all.
template <int DT, int V>
__device__ __forceinline__ void load_blocks(const uint4* base, int64_t blk, int64_t last, uint4 (&w)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = make_uint4(0, 0, 0, 0);
    if (blk + v * kVerThreads < last) w[v] = load_once(base + blk + v * kVerThreads);
  }
}

template <int DT>
__device__ __forceinline__ float element(const uint4& w, int e) {
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
  return DT == kBF16 ? __uint_as_float((e & 1) ? ww[e / 2] & 0xFFFF0000u : ww[e / 2] << 16) : __uint_as_float(ww[e & 3]);
}

// One row's chunk.  Inside a row, and where no element is NaN or +inf, an
// element takes its maximum, the difference d = l - m to the largest of its
// thread so far, two products for its exponent d * f = fma(d, hi, d * lo), exp2
// and an addition: about 10 issue slots of the 14 that a bf16 element has at the
// rate of memory.  The difference comes first: m may be a mask's -1e9 or a
// forced token's 1e9, of which m * f alone is rounded by more than a whole
// exponent.  It is at most 0, so that neither product nor their sum is NaN.
// Everything else takes the second form, element by element.
template <int DT>
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyArgs a) {
  constexpr int N = DT == kBF16 ? 8 : 4;  // elements of 16 bytes
  constexpr int V = 4;                    // blocks of a thread at a time
  __shared__ float red_max[kVerWaves];
  __shared__ double red_sum[kVerWaves];
  __shared__ int red_at[kVerWaves];
  const int row = blockIdx.y, b = row / (a.drafted + 1), i = row - b * (a.drafted + 1);
  const int tid = threadIdx.x, wave = tid / kWave;
  if ((int)blockIdx.x == a.stat_chunks) {  // the drafts, by one workgroup of the sequence
    if (i != 0) return;
    if (tid == 0) a.done[b * kDoneStride] = 0;
    if (tid < a.drafted) {
      const int64_t at = (int64_t)b * a.drafted + tid;
      const int32_t x = a.draft[at];
      DraftPart d = {0.0, 0.0f, -1};
      if (x >= 0 && x < a.vocab) {
        d.token = x;
        d.logit = logit_at<DT>(a.logits, ((int64_t)row + tid) * a.vocab + x);
        d.uq = (double)a.uniforms[at] * (a.probs ? prob_of_draft(a, at, x) : 1.0);
      }
      a.drafts[at] = d;
    }
    return;
  }
  if (i > drafts_of(a, b)) return;
  const char* base = (const char*)a.logits + (int64_t)row * a.vocab * (16 / N);
  const RowVec<16 / N> rv(base);
  const int64_t blocks = (a.vocab + rv.mis + N - 1) / N;
  const int64_t first = blockIdx.x * a.stat_vecs, last = min(first + a.stat_vecs, blocks);
  // blocks that lie in the row whole
  const int64_t whole0 = rv.mis ? 1 : 0, whole1 = (a.vocab + rv.mis) / N;
  uint4 next[V];
  load_blocks<DT, V>(rv.base, first + tid, last, next);
  const float temperature = a.temperature[b];
  const bool greedy = temperature < kGreedy;
  const Scale scale(greedy ? 1.0f : temperature);
  float m = -INFINITY, s = 0.0f;
  int32_t at = INT32_MAX;
  for (int64_t w0 = first; w0 < last; w0 += kVerThreads * V) {
    uint4 w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = next[v];
    load_blocks<DT, V>(rv.base, w0 + kVerThreads * V + tid, last, next);
    const int64_t v0 = w0 + tid;
    bool slow = true;
    if (scale.plain && w0 >= whole0 && w0 + kVerThreads * V <= min(last, whole1)) {
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < N; e += 2) top = raw_max3(element<DT>(w[v], e), element<DT>(w[v], e + 1), top);
      slow = !(top <= FLT_MAX);  // +inf, or a signalling NaN
      if (!slow && !greedy && top > -INFINITY) {
        const float nm = fmaxf(m, top);
        float t = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float d = element<DT>(w[v], e) - nm;
            t += __builtin_amdgcn_exp2f(__builtin_fmaf(d, scale.hi, d * scale.lo));
          }
        slow = !(t <= FLT_MAX);  // a NaN among them
        if (!slow) {
          if (nm > m) {
            s = m == -INFINITY ? 0.0f : s * scale.weight(m - nm);
            m = nm;
          }
          s += t;
        }
      } else if (!slow && greedy && top > m) {
        m = top;
        at = INT32_MAX;
#pragma unroll
        for (int e = V * N - 1; e >= 0; --e)
          if (element<DT>(w[e / N], e % N) == top) at = (int32_t)((v0 + (e / N) * kVerThreads) * N + e % N - rv.mis);
      }
    }
    if (__builtin_expect(slow, 0)) {
#pragma unroll 1
      for (int64_t blk = v0; blk < min(last, w0 + kVerThreads * V); blk += kVerThreads) {
        const uint4 w1 = load_once(rv.base + blk);
        float top = -INFINITY;
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int64_t el = blk * N + e - rv.mis;
          x[e] = el >= 0 && el < a.vocab ? clean(element<DT>(w1, e)) : -INFINITY;
          top = fmaxf(top, x[e]);
        }
        if (greedy) {
          if (top > m) {
            m = top;
            at = INT32_MAX;
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
              if (x[e] == top) at = (int32_t)(blk * N + e - rv.mis);
          }
        } else if (top > -INFINITY) {
          if (top > m) {
            s = m == -INFINITY ? 0.0f : s * scale.weight(m - top);
            m = top;
          }
          float t = 0.0f;
#pragma unroll
          for (int e = 0; e < N; ++e) t += scale.weight(x[e] - m);
          s += t;
        }
      }
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
// of them this one; `mine` its first part); the same in all of them.
struct RowStat {
  double sum;
  float max;
  int32_t at;
};

__device__ __forceinline__ RowStat join_row(const VerifyArgs& a, int64_t row, int l, RowPart x, double inv_t) {
  const RowPart* p = a.parts + row * a.stat_chunks;
  float m = x.max;
  for (int c = l + 16; c < a.stat_chunks; c += 16) m = fmaxf(m, p[c].max);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, lane_xor_f(m, d));
  RowStat r;
  r.max = m;
  r.sum = 0.0;
  r.at = INT32_MAX;
  for (int c = l;;) {
    if (x.max == m) r.at = min(r.at, x.at);
    if (x.max > -INFINITY) r.sum += x.sum * exp_64(((double)x.max - (double)m) * inv_t);
    c += 16;
    if (c >= a.stat_chunks) break;
    x = p[c];
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    r.sum += lane_xor_d(r.sum, d);
    r.at = min(r.at, (int)lane_xor((uint32_t)r.at, d));
  }
  return r;
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int n, int64_t token) {
  for (int t = threadIdx.x; t <= a.drafted; t += kVerThreads)
    a.tokens[(int64_t)b * (a.drafted + 1) + t] =
        t < n ? a.draft[(int64_t)b * a.drafted + t] : t == n ? (int32_t)token : -1;
  if (threadIdx.x == 0) a.accepted[b] = n;
}

struct AcceptShared {
  RowStat stats[kMaxDrafted + 1];
  int ok[kMaxDrafted + 1];
};

// What a sequence draws from, by the whole workgroup, 16 lanes a row; `token`:
// the next token of a row without a race.  Rows past the sequence's drafts have
// no statistics: what is read there is not used.
__device__ __forceinline__ Drawn accept_drafts(const VerifyArgs& a, int b, int64_t& token, AcceptShared& sh) {
  const int cnt = drafts_of(a, b), tid = threadIdx.x;
  const float temperature = a.temperature[b];
  const bool greedy = temperature < kGreedy;
  const double inv_t = greedy ? 1.0 : 1.0 / (double)temperature;
  for (int i = tid / 16; i <= a.drafted; i += kVerThreads / 16) {
    const int64_t row = (int64_t)b * (a.drafted + 1) + i;
    DraftPart d = {0.0, 0.0f, -1};
    RowPart p = {0.0, -INFINITY, INT32_MAX};
    if (i < a.drafted) d = a.drafts[(int64_t)b * a.drafted + i];
    if ((tid & 15) < a.stat_chunks) p = a.parts[row * a.stat_chunks + (tid & 15)];
    const RowStat r = join_row(a, row, tid & 15, p, inv_t);
    if ((tid & 15) == 0) {
      sh.stats[i] = r;
      bool good = false;
      if (i < cnt && d.token >= 0 && r.max > -INFINITY)
        good = greedy ? d.token == r.at : d.uq < exp_64(((double)d.logit - (double)r.max) * inv_t) / r.sum;
      sh.ok[i] = good;
    }
  }
  __syncthreads();
  const int lane = lane_id();
  const uint64_t good = __ballot(lane < cnt && sh.ok[lane]);
  const int n = (int)__builtin_ctzll(~good);  // at most 63 drafts: a bit is 0
  const RowStat row = sh.stats[n];
  const bool any = row.max > -INFINITY;
  const Scale scale(greedy ? 1.0f : temperature);
  Drawn d;
  d.inv_t = inv_t;
  d.inv_sum = any ? 1.0 / row.sum : 0.0;
  d.max = row.max;
  d.hi = scale.hi;
  d.lo = scale.lo;
  d.n = n;
  d.what = greedy || !any ? kDone : n < cnt ? kRest : kTarget;
  d.certain = n < cnt && !a.probs ? a.drafts[(int64_t)b * a.drafted + n].token : -1;
  token = any ? row.at : -1;
  return d;
}

__global__ __launch_bounds__(kVerThreads) void verify_accept_kernel(VerifyArgs a) {
  __shared__ AcceptShared sh;
  int64_t token;
  const Drawn d = accept_drafts(a, blockIdx.x, token, sh);
  if (threadIdx.x == 0) a.drawn[blockIdx.x] = d;
  if (d.what == kDone) write_tokens(a, blockIdx.x, d.n, token);
}

struct RaceShared {
  float low[2][kVerWaves];
  RacePart best[kVerWaves];
  int last;
};

__device__ __forceinline__ void take_better(double& s, int64_t& at, double os, int64_t oat) {
  if (oat >= 0 && (at < 0 || os > s || (os == s && oat < at))) {
    s = os;
    at = oat;
  }
}

// VEC neighbouring elements of a row from element v on, as floats.  Rows begin
// on any element: the load is as wide as the hardware takes it at the element's
// alignment.
template <bool BF16, int VEC>
__device__ __forceinline__ void load_elements(const void* row, int64_t v, float (&x)[VEC]) {
  if constexpr (BF16) {
    uint16_t h[VEC];
    __builtin_memcpy(h, (const uint16_t*)row + v, sizeof(h));
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = __uint_as_float((uint32_t)h[e] << 16);
  } else {
    __builtin_memcpy(x, (const float*)row + v, sizeof(x));
  }
}

// A thread's elements of a step of the race: `from` is the first of the VEC that
// are loaded, those below `own` belong to the thread before (a row's last
// vector is loaded whole, so it overlaps).
template <int VEC>
struct RaceSpan {
  int64_t own, from;
  bool any;
  __device__ __forceinline__ RaceSpan(int64_t vocab, int64_t step) {
    own = step + (int64_t)threadIdx.x * VEC;
    any = own < vocab;
    from = min(own, vocab - VEC);
  }
};

// Races the elements first .. end - 1; e: the noise of this thread's first ones.
template <int DT, int VEC>
__device__ __forceinline__ RacePart race_chunk(const VerifyArgs& a, int b, const Drawn& d, int64_t first, int64_t end,
                                               bool with_q, float (&e)[VEC], RaceShared& sh) {
  constexpr int kStep = kVerThreads * VEC;
  const int wave = threadIdx.x / kWave;
  const Scale scale(d.hi, d.lo);
  const int64_t row = (int64_t)b * (a.drafted + 1) + d.n;
  const char* logits = (const char*)a.logits + row * a.vocab * (DT == kBF16 ? 2 : 4);
  const int64_t qrow = (int64_t)b * a.drafted + d.n;
  const char* probs = (const char*)a.probs + qrow * a.vocab * (a.probs_bf16 ? 2 : 4);
  const float inv_sum = (float)d.inv_sum;
  double best = 0.0;
  int64_t at = -1;
  float low = 0.0f;  // some element's score is at least this
  int turn = 0;
  for (int64_t step = first; step < end; step += kStep, turn ^= 1) {
    const RaceSpan<VEC> span(a.vocab, step);
    float l[VEC], q[VEC], hi[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      l[k] = -INFINITY;
      q[k] = with_q && span.from + k == d.certain ? 1.0f : 0.0f;
    }
    if (span.any) {
      if (step > first) load_elements<false, VEC>(a.noise + (int64_t)b * a.vocab, span.from, e);
      load_elements<DT == kBF16, VEC>(logits, span.from, l);
      if (with_q && a.probs) {
        if (a.probs_bf16)
          load_elements<true, VEC>(probs, span.from, q);
        else
          load_elements<false, VEC>(probs, span.from, q);
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      l[k] = span.from + k >= span.own ? clean(l[k]) : -INFINITY;
      const float p = scale.weight(l[k] - d.max) * inv_sum;
      // p is off by at most 1.2e-5 of itself, below 2^-16: its exponent is as low as -150 and rounded to half of
      // 2^-16 (ln 2 of which is 5.3e-6), l - max by 2^-24 of itself (150 ln 2 2^-24 = 6.2e-6), and exp2, the sum's
      // reciprocal and three roundings add 4e-7; and by what lies below the normal numbers, the quotient by 2^-21 more.
      // The reciprocal of noise below the normal numbers may be infinite: it bounds from above only.
      const float slack = p * 0x1p-16f + 0x1p-120f;
      const float r = __builtin_amdgcn_rcpf(e[k]);
      const bool in = l[k] > -INFINITY;
      hi[k] = in ? (p - q[k] + slack) * r * (1.0f + 0x1p-19f) : 0.0f;
      const float lo = (p - q[k] - slack) * r * (1.0f - 0x1p-19f);
      low = in && e[k] >= FLT_MIN ? fmaxf(low, lo) : low;
    }
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) low = fmaxf(low, lane_xor_f(low, x));
    if (lane_id() == 0) sh.low[turn][wave] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) low = fmaxf(low, sh.low[turn][w]);
    uint32_t may = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) may |= (uint32_t)(hi[k] > 0.0f && hi[k] >= low) << k;
    while (may) {  // seldom more than one element of a workgroup
      const int at_k = __builtin_ctz(may);
      may &= may - 1;
      float lk = l[0], qk = q[0], ek = e[0];
#pragma unroll
      for (int k = 1; k < VEC; ++k) {
        lk = k == at_k ? l[k] : lk;
        qk = k == at_k ? q[k] : qk;
        ek = k == at_k ? e[k] : ek;
      }
      const double p = exp_64(((double)lk - (double)d.max) * d.inv_t) * d.inv_sum;
      const double s = (p - (double)qk) / (double)ek;
      if (s > 0.0) take_better(best, at, s, span.from + at_k);
    }
  }
#pragma unroll
  for (int x = 1; x < kWave; x <<= 1) {
    const double os = lane_xor_d(best, x);
    const int64_t oat = (int64_t)shfl_xor_u64((uint64_t)at, x);
    take_better(best, at, os, oat);
  }
  if (lane_id() == 0) sh.best[wave] = {best, at};
  __syncthreads();
  RacePart r = sh.best[0];
#pragma unroll
  for (int w = 1; w < kVerWaves; ++w) take_better(r.score, r.at, sh.best[w].score, sh.best[w].at);
  __syncthreads();
  return r;
}

// A part passes from one workgroup to another in the same launch.  Both sides
// use accesses of device scope, which go past the caches that one XCD has to
// itself, and the store has come back before the counter is raised.  (A fence
// of device scope would write back the whole L2: 60 us a launch of 2000
// workgroups.)
__device__ __forceinline__ void store_part(RacePart* to, const RacePart& r) {
  __hip_atomic_store((uint64_t*)&to->score, (uint64_t)__double_as_longlong(r.score), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store((uint64_t*)&to->at, (uint64_t)r.at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
__device__ __forceinline__ RacePart load_part(RacePart* from) {
  RacePart r;
  r.score = __longlong_as_double((long long)__hip_atomic_load((uint64_t*)&from->score, __ATOMIC_RELAXED,
                                                              __HIP_MEMORY_SCOPE_AGENT));
  r.at = (int64_t)__hip_atomic_load((uint64_t*)&from->at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return r;
}

template <int DT, int VEC, bool ACCEPT>
__global__ __launch_bounds__(kVerThreads) void verify_race_kernel(VerifyArgs a) {
  __shared__ RaceShared sh;
  __shared__ std::conditional_t<ACCEPT, AcceptShared, int> accept;  // not used: takes no space
  const int b = blockIdx.y;
  Drawn d;
  if constexpr (ACCEPT) {
    int64_t drawn;
    d = accept_drafts(a, b, drawn, accept);
    if (d.what == kDone) {
      if (blockIdx.x == 0) write_tokens(a, b, d.n, drawn);
      return;
    }
  } else {
    d = a.drawn[b];
    if (d.what == kDone) return;
  }
  int64_t first = (int64_t)blockIdx.x * a.race_size, end = min(first + a.race_size, a.vocab);
  int64_t token;
  for (bool with_q = d.what == kRest;;) {
    float e[VEC];
    const RaceSpan<VEC> span(a.vocab, first);
#pragma unroll
    for (int k = 0; k < VEC; ++k) e[k] = 1.0f;
    if (span.any) load_elements<false, VEC>(a.noise + (int64_t)b * a.vocab, span.from, e);
    RacePart r = race_chunk<DT, VEC>(a, b, d, first, end, with_q, e, sh);
    if (a.race_chunks > 1 && end - first <= a.race_size) {
      RacePart* parts = a.race + (int64_t)b * a.race_chunks;
      if (threadIdx.x == 0) {
        store_part(parts + blockIdx.x, r);
        sh.last = atomicAdd(&a.done[b * kDoneStride], 1) == a.race_chunks - 1;
      }
      __syncthreads();
      if (!sh.last) return;
      r = {0.0, -1};
      for (int c = lane_id(); c < a.race_chunks; c += kWave) {  // every wave the same
        const RacePart o = load_part(parts + c);
        take_better(r.score, r.at, o.score, o.at);
      }
#pragma unroll
      for (int x = 1; x < kWave; x <<= 1) {
        const double os = lane_xor_d(r.score, x);
        const int64_t oat = (int64_t)shfl_xor_u64((uint64_t)r.at, x);
        take_better(r.score, r.at, os, oat);
      }
    }
    token = r.at;
    if (token >= 0 || !with_q) break;
    // p - q is nowhere positive (rounded probabilities): drawn from p, the whole row by this workgroup
    with_q = false;
    first = 0;
    end = a.vocab;
  }
  write_tokens(a, b, d.n, token);
}

struct VerifyPlan {
  int stat_chunks, race_chunks;
  int64_t stat_vecs, race_size;
  size_t part_bytes, draft_bytes, drawn_bytes, race_bytes, bytes;
};

// stat_steps, race_steps: steps of a workgroup (0: as many as are best).
static VerifyPlan plan_verify(int64_t batch, int64_t drafted, int64_t vocab, int dtype, int stat_steps = 0,
                              int race_steps = 0) {
  VerifyPlan p;
  const int64_t n = dtype == TALLAX_BF16 ? 8 : 4;
  const int64_t blocks = (vocab + n - 1) / n + 1;  // a row may begin inside a block
  // up to about 8192 workgroups of whole steps (a thread's 4 blocks): at 1040 rows of 151937 float32 86 us,
  // with 4096 of them 86 to 92, with 2048 129 (the last ones of uneven rows run alone)
  const int64_t step = kVerThreads * 4, rows = batch * (drafted + 1);
  int64_t steps = stat_steps ? stat_steps : blocks * rows / (8192 * step);
  if (steps < 1) steps = 1;
  p.stat_vecs = steps * step;
  p.stat_chunks = (int)((blocks + p.stat_vecs - 1) / p.stat_vecs);
  // and of the race about 2048: the same rows 31 us, with 512 49
  const int64_t size = kVerThreads * (vocab < kRaceVec ? 1 : kRaceVec);
  steps = race_steps ? race_steps : (vocab * batch + 1024 * size) / (2048 * size);
  p.race_size = (steps < 1 ? 1 : steps) * size;
  p.race_chunks = (int)((vocab + p.race_size - 1) / p.race_size);
  p.part_bytes = align_up((size_t)rows * p.stat_chunks * sizeof(RowPart), 256);
  p.draft_bytes = align_up((size_t)(batch * drafted) * sizeof(DraftPart), 256);
  p.drawn_bytes = align_up((size_t)batch * sizeof(Drawn), 256);
  p.race_bytes = align_up((size_t)batch * p.race_chunks * sizeof(RacePart), 256);
  p.bytes = p.part_bytes + p.draft_bytes + p.drawn_bytes + p.race_bytes + (size_t)batch * kDoneStride * sizeof(int32_t);
  return p;
}

template <int DT, int VEC>
static void launch_race(const VerifyArgs& a, hipStream_t s) {
  const dim3 grid(a.race_chunks, a.batch);
  if ((int64_t)a.batch * a.race_chunks <= kAcceptInRace) {
    verify_race_kernel<DT, VEC, true><<<grid, kVerThreads, 0, s>>>(a);
  } else {
    verify_accept_kernel<<<a.batch, kVerThreads, 0, s>>>(a);
    verify_race_kernel<DT, VEC, false><<<grid, kVerThreads, 0, s>>>(a);
  }
}

template <int DT>
static int launch_verify(const VerifyArgs& a, hipStream_t s) {
  verify_stats_kernel<DT><<<dim3(a.stat_chunks + 1, a.batch * (a.drafted + 1)), kVerThreads, 0, s>>>(a);
  if (a.vocab < kRaceVec)
    launch_race<DT, 1>(a, s);
  else
    launch_race<DT, kRaceVec>(a, s);
  return launch_status("verify");
}

static int verify(const int32_t* draft, const void* logits, int logits_dtype, int64_t batch, int64_t drafted,
                  int64_t vocab, const int32_t* counts, const float* temperature, const void* draft_probs,
                  int probs_dtype, const float* uniforms, const float* noise, int32_t* out_tokens,
                  int32_t* out_accepted, void* workspace, size_t workspace_bytes, tallax_stream_t stream,
                  int stat_steps, int race_steps) {
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
  const VerifyPlan p = plan_verify(batch, drafted, vocab, logits_dtype, stat_steps, race_steps);
  const int st = check_workspace("verify", workspace, workspace_bytes, p.bytes);
  if (st != kOk) return st;
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
  a.drafts = (DraftPart*)((char*)workspace + p.part_bytes);
  a.drawn = (Drawn*)((char*)a.drafts + p.draft_bytes);
  a.race = (RacePart*)((char*)a.drawn + p.drawn_bytes);
  a.done = (int32_t*)((char*)a.race + p.race_bytes);
  a.race_chunks = p.race_chunks;
  a.race_size = p.race_size;
  return logits_dtype == TALLAX_BF16 ? launch_verify<kBF16>(a, (hipStream_t)stream)
                                     : launch_verify<kF32>(a, (hipStream_t)stream);
}

}  // namespace tx

using namespace tx;

extern "C" {

size_t tallax_verify_workspace_size(int64_t batch, int64_t drafted, int64_t vocab, int logits_dtype) {
  if (batch < 0 || drafted < 0 || vocab < 1) return 0;
  const VerifyPlan p = plan_verify(batch, drafted, vocab, logits_dtype);
  return p.bytes;
}

int tallax_verify(const int32_t* draft, const void* logits, int logits_dtype, int64_t batch, int64_t drafted,
                  int64_t vocab, const int32_t* counts, const float* temperature, const void* draft_probs,
                  int probs_dtype, const float* uniforms, const float* noise, int32_t* out_tokens,
                  int32_t* out_accepted, void* workspace, size_t workspace_bytes, tallax_stream_t stream) {
  return verify(draft, logits, logits_dtype, batch, drafted, vocab, counts, temperature, draft_probs, probs_dtype,
                uniforms, noise, out_tokens, out_accepted, workspace, workspace_bytes, stream, 0, 0);
}

int tallax_testing_verify_steps(const int32_t* draft, const void* logits, int logits_dtype, int64_t batch,
                                int64_t drafted, int64_t vocab, const int32_t* counts, const float* temperature,
                                const void* draft_probs, int probs_dtype, const float* uniforms, const float* noise,
                                int32_t* out_tokens, int32_t* out_accepted, void* workspace, size_t workspace_bytes,
                                tallax_stream_t stream, int stat_steps, int race_steps) {
  if (stat_steps < 0 || race_steps < 0 || stat_steps > 65536 || race_steps > 65536) {
    set_error("verify: %d and %d steps (0 to 65536)", stat_steps, race_steps);
    return kInvalidArgument;
  }
  return verify(draft, logits, logits_dtype, batch, drafted, vocab, counts, temperature, draft_probs, probs_dtype,
                uniforms, noise, out_tokens, out_accepted, workspace, workspace_bytes, stream, stat_steps, race_steps);
}

}  // extern "C"
