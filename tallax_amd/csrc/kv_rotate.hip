// Appending tokens to a paged cache with the rotation of their positions on the
// way: pair i of a query's or key's elements is turned by the angle p f_i of its
// token's position p,
//   y0 = x0 cos a - x1 sin a,   y1 = x1 cos a + x0 sin a,
// in float32, rounded once to the tensors' type; values are only moved.
//
// A workgroup takes a few tokens of one sequence.  Its threads first work out
// the tokens' places in the cache and the cosines and sines of all pairs, which
// the heads share, into LDS; then each moves 16 bytes at a time.
#include "tx_common.h"
#include "tx_kv.h"

namespace tx {

struct RotateArgs {
  KvView c;
  const int32_t* lens;
  const int32_t* counts;
  const char* in[3];                       // q, k, v of the new tokens
  int64_t batch_at[3], token_at[3], head_at[3];  // their strides in bytes
  char* out_q;
  int tokens, heads, kv_heads, pairs, axes;
  int per_wg;       // tokens of a workgroup
  const float* frequencies;
  const int32_t* places;     // [batch, tokens, axes] or null
  const int32_t* pair_axes;  // [pairs] or null
  float* scores;
  int32_t* positions;
  const int32_t* seen;
  int32_t* out_lens;
  PageDiv per_token, per_head, per_value;  // items of a token, of a rotated head, of a value's head
};

constexpr int kRotateTokens = 4;  // of a workgroup, at most
constexpr int kMostPairs = 128;

// cos and sin of 2 pi r for r in turns, in 64 bits: the angle of a far position
// is right to 2^-52 of its turns, and so many of them may be whole.  r less its
// nearest quarter is at most an eighth of a turn, where the Taylor series to
// x^12 and x^11 are off by less than 2^-40.
__device__ __forceinline__ float2 cos_sin_turns(double r) {
  r -= rint(r);
  const double quarter = rint(4.0 * r);
  const double x = (r - 0.25 * quarter) * 6.283185307179586477, z = x * x;
  double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, -1.0 / 5040.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, -1.0 / 6.0);
  s = fma(s * z, x, x);
  c = fma(c, z, -1.0 / 3628800.0);
  c = fma(c, z, 1.0 / 40320.0);
  c = fma(c, z, -1.0 / 720.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int n = (int)quarter & 3;
  const float cf = (float)c, sf = (float)s;
  const float cc = n & 1 ? sf : cf, ss = n & 1 ? cf : sf;
  return make_float2(n == 1 || n == 2 ? -cc : cc, n & 2 ? -ss : ss);
}

template <bool F32>
struct Vec {  // 16 bytes of elements as float32
  static constexpr int kE = F32 ? 4 : 8;
  float x[kE];
  __device__ __forceinline__ void load(const char* p) {
    const uint4 u = *(const uint4*)p;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      if constexpr (F32)
        x[i] = __uint_as_float(w[i]);
      else
        x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
  }
  __device__ __forceinline__ uint4 bits() const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F32) {
        w[i] = __float_as_uint(x[i]);
      } else {
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        bf16x2_t r;  // to nearest, ties to even
        r[0] = (__bf16)x[2 * i];
        r[1] = (__bf16)x[2 * i + 1];
        w[i] = __builtin_bit_cast(uint32_t, r);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <bool F32>
__device__ __forceinline__ float element(const char* p, int i) {
  if constexpr (F32) return ((const float*)p)[i];
  return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

// How pairs lie: (i, i + pairs) in whole vectors, in any number, or (2i, 2i + 1).
enum PairsAre { kHalves = 0, kHalvesAny = 1, kNeighbours = 2 };

template <bool F32, int HOW>
__global__ __launch_bounds__(256) void kv_rotate_kernel(RotateArgs a) {
  constexpr int E = Vec<F32>::kE;
  __shared__ float2 turn[kRotateTokens * kMostPairs];
  __shared__ int64_t k_to[kRotateTokens], v_to[kRotateTokens];  // the token's slot in the pools, -1: in none
  const int b = blockIdx.y, tid = threadIdx.x, t0 = blockIdx.x * a.per_wg;
  const int n = min(a.per_wg, a.tokens - t0);
  const int len = max(a.lens[b], 0);
  const int cnt = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  const int first = a.seen ? a.seen[b] : len;
  if (blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) a.out_lens[b] = (int)min((int64_t)len + cnt, (int64_t)a.c.capacity);
  if (tid < n) {
    const int64_t slot = (int64_t)len + t0 + tid;
    int64_t k = -1, v = -1;
    if (t0 + tid < cnt && slot < a.c.capacity) {
      const int page = page_id(a.c, a.c.table + (int64_t)b * a.c.width, (int)slot);
      if (page >= 0) {
        const int off = (int)slot - (int)page_of(a.c.div, (uint32_t)slot) * a.c.div.size;
        k = page * a.c.k_page + off * a.c.k_slot;
        v = page * a.c.v_page + off * a.c.v_slot;
      }
    }
    k_to[tid] = k;
    v_to[tid] = v;
  }
  for (int i = tid; i < n * a.pairs; i += 256) {
    const int t = i / a.pairs, pair = i - t * a.pairs;
    const int axis = a.pair_axes ? min(max(a.pair_axes[pair], 0), a.axes - 1) : 0;
    const int64_t p = a.places ? a.places[((int64_t)b * a.tokens + t0 + t) * a.axes + axis] : (int64_t)first + t0 + t;
    turn[t * a.pairs + pair] = cos_sin_turns((double)p * ((double)a.frequencies[pair] * 0.15915494309189533577));
  }
  __syncthreads();
  const int dim = a.c.dim, vecs = dim / E, rotated = a.heads + a.kv_heads;
  const int from_values = rotated * a.per_head.size;
  const int items = n * a.per_token.size;
  for (int i = blockIdx.z * 256 + tid; i < items; i += gridDim.z * 256) {
    const int t = (int)page_of(a.per_token, i);
    int r = i - t * a.per_token.size;
    const int64_t k_slot = k_to[t], v_slot = v_to[t];
    if (r >= from_values) {
      r -= from_values;
      const int head = (int)page_of(a.per_value, r), v = r - head * a.per_value.size;
      if (v_slot >= 0)
        *(uint4*)(a.c.v + v_slot + head * a.c.v_head + v * 16) =
            *(const uint4*)(a.in[2] + b * a.batch_at[2] + (t0 + t) * a.token_at[2] + head * a.head_at[2] + v * 16);
      continue;
    }
    int head = (int)page_of(a.per_head, r);
    const int v = r - head * a.per_head.size;
    const bool key = head >= a.heads;
    head -= key ? a.heads : 0;
    char* to;
    if (key) {
      if (k_slot < 0) continue;
      to = a.c.k + k_slot + head * a.c.k_head;
      if (a.scores && v == 0) {
        const int64_t at = ((int64_t)b * a.kv_heads + head) * a.c.capacity + len + t0 + t;
        a.scores[at] = 0.0f;
        a.positions[at] = a.seen[b] + t0 + t;
      }
    } else {
      to = a.out_q + (((int64_t)b * a.tokens + t0 + t) * a.heads + head) * dim * (F32 ? 4 : 2);
      if (t0 + t >= cnt) {  // a token that does not count
        const int half = HOW == kHalves ? a.pairs / E : 0;
        if (v < half) *(uint4*)(to + v * 16) = make_uint4(0, 0, 0, 0);
        *(uint4*)(to + (v + half) * 16) = make_uint4(0, 0, 0, 0);
        continue;
      }
    }
    const char* from = a.in[key] + b * a.batch_at[key] + (t0 + t) * a.token_at[key] + head * a.head_at[key];
    const float2* tr = turn + t * a.pairs;
    Vec<F32> x;
    if constexpr (HOW == kHalves) {
      // the first pairs / E items are vectors of both halves, the others what is not rotated
      const int half = a.pairs / E;
      if (v < half) {
        Vec<F32> y;
        x.load(from + v * 16);
        y.load(from + (v + half) * 16);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 cs = tr[v * E + e];
          const float x0 = x.x[e], x1 = y.x[e];
          x.x[e] = x0 * cs.x - x1 * cs.y;
          y.x[e] = x1 * cs.x + x0 * cs.y;
        }
        *(uint4*)(to + v * 16) = x.bits();
        *(uint4*)(to + (v + half) * 16) = y.bits();
      } else {
        *(uint4*)(to + (v + half) * 16) = *(const uint4*)(from + (v + half) * 16);
      }
    } else {
      x.load(from + v * 16);
      if (v * E < 2 * a.pairs) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int d = v * E + e;
          if constexpr (HOW == kNeighbours) {
            if (e & 1 || d >= 2 * a.pairs) continue;
            const float2 cs = tr[d / 2];
            const float x0 = x.x[e], x1 = x.x[e | 1];
            x.x[e] = x0 * cs.x - x1 * cs.y;
            x.x[e | 1] = x1 * cs.x + x0 * cs.y;
          } else if (d < a.pairs) {
            const float2 cs = tr[d];
            x.x[e] = x.x[e] * cs.x - element<F32>(from, d + a.pairs) * cs.y;
          } else if (d < 2 * a.pairs) {
            const float2 cs = tr[d - a.pairs];
            x.x[e] = x.x[e] * cs.x + element<F32>(from, d - a.pairs) * cs.y;
          }
        }
      }
      *(uint4*)(to + v * 16) = x.bits();
    }
  }
}

}  // namespace tx

using namespace tx;

extern "C" {

int tallax_kv_append_rotated(const tallax_kv_cache* cache, const int32_t* lens, const int32_t* counts,
                             const tallax_kv_tokens* fresh, const tallax_rotation* turn, float* scores,
                             int32_t* positions, const int32_t* seen, void* out_q, int32_t* out_lens,
                             tallax_stream_t stream) {
  RotateArgs a;
  int st = make_kv_view(cache, "kv_append_rotated", &a.c);
  if (st != kOk) return st;
  if (!fresh || !turn) {
    set_error("kv_append_rotated: null tokens or rotation");
    return kInvalidArgument;
  }
  if (fresh->tokens < 0 || fresh->tokens > (1 << 24) || fresh->heads < 1 || turn->pairs < 1 ||
      2 * turn->pairs > cache->dim || turn->axes < 1) {
    set_error("kv_append_rotated: %lld tokens (0 to 2^24), %lld heads, %lld pairs of %d elements, %lld axes",
              (long long)fresh->tokens, (long long)fresh->heads, (long long)turn->pairs, cache->dim,
              (long long)turn->axes);
    return kInvalidArgument;
  }
  if (fresh->heads > 65535 || turn->axes > 1024) {
    set_error("kv_append_rotated: up to 65535 heads and 1024 axes");
    return kUnsupported;
  }
  if (turn->axes > 1 && (!turn->pair_axes || !turn->places)) {
    set_error("kv_append_rotated: several axes need the axis of each pair and the places of the tokens");
    return kInvalidArgument;
  }
  if (cache->batch == 0) return kOk;
  if (!lens || !out_lens || lens == out_lens || (!scores != !positions) || (scores && !seen) ||
      (fresh->tokens > 0 && (!fresh->q || !fresh->k || !fresh->v || !out_q || !turn->frequencies))) {
    set_error("kv_append_rotated: null pointer, out_lens the same as lens, or scores without positions and seen");
    return kInvalidArgument;
  }
  const int64_t es = cache->dtype == TALLAX_F32 ? 4 : 2;
  const void* in[3] = {fresh->q, fresh->k, fresh->v};
  bool ok = ((uintptr_t)out_q & 15) == 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t s[3] = {fresh->stride_batch[i], fresh->stride_token[i], fresh->stride_head[i]};
    for (int64_t x : s) ok = ok && x >= 0 && x * es % 16 == 0 && x < ((int64_t)1 << 40);
    ok = ok && ((uintptr_t)in[i] & 15) == 0;
    a.in[i] = (const char*)in[i];
    a.batch_at[i] = s[0] * es;
    a.token_at[i] = s[1] * es;
    a.head_at[i] = s[2] * es;
  }
  if (!ok) {
    set_error("kv_append_rotated: q, k, v, their strides and out_q must be multiples of 16 bytes");
    return kUnsupported;
  }
  a.lens = lens;
  a.counts = counts;
  a.out_q = (char*)out_q;
  a.tokens = (int)fresh->tokens;
  a.heads = (int)fresh->heads;
  a.kv_heads = (int)cache->kv_heads;
  a.pairs = (int)turn->pairs;
  a.axes = (int)turn->axes;
  a.frequencies = turn->frequencies;
  a.places = turn->places;
  a.pair_axes = turn->pair_axes;
  a.scores = scores;
  a.positions = positions;
  a.seen = seen;
  a.out_lens = out_lens;
  const int e = 16 / (int)es, vecs = cache->dim / e;
  const PairsAre how = turn->neighbours ? kNeighbours : turn->pairs % e == 0 ? kHalves : kHalvesAny;
  const int per_head = how == kHalves ? vecs - a.pairs / e : vecs;
  const int64_t per_token = (int64_t)(a.heads + a.kv_heads) * per_head + (int64_t)a.kv_heads * vecs;
  a.per_head = make_page_div(per_head);
  a.per_value = make_page_div(vecs);
  a.per_token = make_page_div(per_token);
  // One token a workgroup while that gives the card no more than it has room for, and then several workgroups to a
  // token's heads.
  const int64_t all = (int64_t)cache->batch * a.tokens;
  a.per_wg = all >= 8192 ? kRotateTokens : 1;
  const int64_t blocks = a.tokens > 0 ? (a.tokens + a.per_wg - 1) / a.per_wg : 1;
  int64_t split = (per_token * a.per_wg + 255) / 256;
  const int64_t room = all > 0 ? 512 / all : 1;
  split = split < room ? split : room;
  const dim3 grid((unsigned)blocks, (unsigned)cache->batch, (unsigned)(split < 1 ? 1 : split));
  hipStream_t s = (hipStream_t)stream;
  if (es == 4) {
    if (how == kHalves) kv_rotate_kernel<true, kHalves><<<grid, 256, 0, s>>>(a);
    else if (how == kHalvesAny) kv_rotate_kernel<true, kHalvesAny><<<grid, 256, 0, s>>>(a);
    else kv_rotate_kernel<true, kNeighbours><<<grid, 256, 0, s>>>(a);
  } else {
    if (how == kHalves) kv_rotate_kernel<false, kHalves><<<grid, 256, 0, s>>>(a);
    else if (how == kHalvesAny) kv_rotate_kernel<false, kHalvesAny><<<grid, 256, 0, s>>>(a);
    else kv_rotate_kernel<false, kNeighbours><<<grid, 256, 0, s>>>(a);
  }
  return launch_status("kv_append_rotated");
}

}  // extern "C"
