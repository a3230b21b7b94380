// Appending tokens to a paged cache with the rotation of their positions on the
// way: pair i of a query's or key's elements is turned by the angle p f_i of its
// token's position p,
//   y0 = x0 cos a - x1 sin a,   y1 = x1 cos a + x0 sin a,
// in float32, rounded once to the tensors' type; values are only moved.
//
// A workgroup takes one to four tokens of one sequence, a whole number of waves
// each.  Its threads first work out the tokens' places in the cache and the
// cosines and sines of all pairs, which the heads share, into LDS; then each
// moves 16 bytes of a head at a time, or 32.  A token's addresses are the same
// in a wave: what is left to each vector is its head and its place in it.
//
// Bound by memory: 4 x 4096 tokens of 32 + 2 x 8 heads of 128, bfloat16, 403 MB,
// 76 us (5.3 TB/s; a copy of 4 GiB reaches 4.8); 3 x 2501 tokens of 12 + 2 x 12 heads
// of 80, float32, three axes, 173 MB, 31 us by itself and 45 among other calls, whose
// data then are in the caches.  A token each of 64 sequences takes 4.6 us, the launch
// and a chain of loads (length, table, tokens); 65 pairs of 192 elements, partners
// off the vectors' alignment, 395 MB in 101 us (3.9 TB/s).
#include "tx_common.h"
#include "tx_kv.h"

namespace tx {

struct RotateArgs {
  KvView c;
  const int32_t* lens;
  const int32_t* counts;
  const char* in[3];                       // q, k, v of the new tokens
  uint32_t batch_at[3], token_at[3];       // their strides, of heads in bytes, else in sixteens of them
  uint32_t head_at[3];
  char* out_q;
  int tokens, heads, kv_heads, pairs, axes;
  int log_tokens;   // 1 << log_tokens tokens a workgroup, 256 >> log_tokens threads each
  const float* frequencies;
  const int32_t* places;     // [batch, tokens, axes] or null
  const int32_t* pair_axes;  // [pairs] or null
  float* scores;
  int32_t* positions;
  const int32_t* seen;
  int32_t* out_lens;
  PageDiv per_head, per_value, per_token;  // items of a rotated head, of a value's head; pairs of a token
};

constexpr int kRotateTokens = 4;  // of a workgroup, at most
constexpr int kMostPairs = 128;

// cos and sin of 2 pi r for r in turns, in 64 bits: the angle of a far position
// is right to 2^-52 of its turns, and so many of them may be whole.  r less its
// nearest quarter is at most an eighth of a turn, where the Taylor series to
// x^12 and x^13 are off by less than 2^-41 and 2^-45.
__device__ __forceinline__ float2 cos_sin_turns(double r) {
  r -= rint(r);
  const double quarter = rint(4.0 * r);
  const double x = (r - 0.25 * quarter) * 6.283185307179586477, z = x * x;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;
  s = fma(s, z, -1.0 / 39916800.0);
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
  __device__ __forceinline__ void load(const char* p) { unpack(*(const uint4*)p); }
  __device__ __forceinline__ void unpack(uint4 u) {
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

// 16 bytes at any address.
__device__ __forceinline__ uint4 load_any(const char* p) {
  uint4 u;
  __builtin_memcpy(&u, p, 16);
  return u;
}
__device__ __forceinline__ void store_any(char* p, uint4 u) { __builtin_memcpy(p, &u, 16); }

// How pairs lie: (i, i + pairs) in whole vectors, in any number, or (2i, 2i + 1); kHalvesOver: in any number that fills a
// vector, and so does what is not rotated, or there is nothing.
enum PairsAre { kHalves = 0, kHalvesAny = 1, kNeighbours = 2, kHalvesOver = 3 };

template <bool F32, int HOW>
__global__ __launch_bounds__(256) void kv_rotate_kernel(RotateArgs a) {
  constexpr int E = Vec<F32>::kE, ES = F32 ? 4 : 2;
  __shared__ float2 turn[kRotateTokens * kMostPairs];
  const int b = blockIdx.y, tid = threadIdx.x, t0 = blockIdx.x << a.log_tokens;
  const int n = min(1 << a.log_tokens, a.tokens - t0);
  const int len = max(a.lens[b], 0);
  const int cnt = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  const int first = a.seen ? a.seen[b] : len;
  if (blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) a.out_lens[b] = (int)min((int64_t)len + cnt, (int64_t)a.c.capacity);
  // this wave's token, and its slot in the pools
  const int log_threads = 8 - a.log_tokens, t = __builtin_amdgcn_readfirstlane(tid >> log_threads), token = t0 + t;
  const bool counts = token < cnt;
  const int64_t slot = (int64_t)len + token;
  int page = -1, off = 0;
  if (counts && slot < a.c.capacity) {
    const uint32_t in_row = page_of(a.c.div, (uint32_t)slot);
    page = a.c.table[(uint64_t)(uint32_t)b * (uint32_t)a.c.width + in_row];
    page = (uint32_t)page < (uint32_t)a.c.pages ? page : -1;
    off = (int)slot - (int)in_row * a.c.div.size;
  }
  for (int i = tid; i < n * a.pairs; i += 256) {
    const int u = (int)page_of(a.per_token, (uint32_t)i), pair = i - u * a.pairs;
    int64_t p = (int64_t)first + t0 + u;
    if (a.places) {
      const int axis = a.pair_axes ? min(max(a.pair_axes[pair], 0), a.axes - 1) : 0;
      p = a.places[((int64_t)b * a.tokens + t0 + u) * a.axes + axis];
    }
    turn[i] = cos_sin_turns((double)p * ((double)a.frequencies[pair] * 0.15915494309189533577));
  }
  __syncthreads();
  if (t >= n) return;
  const int dim = a.c.dim, vecs = a.per_value.size, half = a.pairs / E;
  const int from_values = (a.heads + a.kv_heads) * a.per_head.size, items = from_values + a.kv_heads * vecs;
  const char* in[3];
#pragma unroll
  for (int i = 0; i < 3; ++i)
    in[i] = a.in[i] + (((uint64_t)(uint32_t)b * a.batch_at[i] + (uint64_t)(uint32_t)token * a.token_at[i]) << 4);
  char* out_q = a.out_q + ((uint64_t)(uint32_t)b * (uint32_t)a.tokens + (uint32_t)token) * (uint32_t)(a.heads * vecs) * 16;
  char* k_to = a.c.k + (uint64_t)(uint32_t)page * (uint64_t)a.c.k_page + (uint32_t)off * a.c.k_slot;
  char* v_to = a.c.v + (uint64_t)(uint32_t)page * (uint64_t)a.c.v_page + (uint32_t)off * a.c.v_slot;
  const float2* tr = turn + t * a.pairs;
  for (int i = (blockIdx.z << log_threads) + (tid & ((1 << log_threads) - 1)); i < items; i += gridDim.z << log_threads) {
    if (i >= from_values) {
      const int r = i - from_values, head = (int)page_of(a.per_value, r), v = r - head * vecs;
      if (page >= 0)
        *(uint4*)(v_to + head * a.c.v_head + v * 16) = *(const uint4*)(in[2] + (uint64_t)(uint32_t)head * a.head_at[2] + v * 16);
      continue;
    }
    int head = (int)page_of(a.per_head, i);
    const int v = i - head * a.per_head.size;
    const bool key = head >= a.heads;
    head -= key ? a.heads : 0;
    if (key && page < 0) continue;
    char* to = key ? k_to + head * a.c.k_head : out_q + (uint32_t)(head * vecs) * 16;
    if (!counts) {  // a token that does not count: its query is 0, its key has no slot
      const uint4 none = make_uint4(0, 0, 0, 0);
      *(uint4*)(to + v * 16) = none;
      if (v + a.per_head.size < vecs) *(uint4*)(to + (v + a.per_head.size) * 16) = none;
      continue;
    }
    if (key && v == 0 && a.scores) {
      const int64_t s = ((int64_t)b * a.kv_heads + head) * a.c.capacity + slot;
      a.scores[s] = 0.0f;
      a.positions[s] = a.seen[b] + token;
    }
    const char* from = key ? in[1] + (uint64_t)(uint32_t)head * a.head_at[1] : in[0] + (uint64_t)(uint32_t)head * a.head_at[0];
    Vec<F32> x;
    if constexpr (HOW == kHalves) {
      // the first pairs / E items are vectors of both halves, the others what is not rotated
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
    } else if constexpr (HOW == kNeighbours) {
      x.load(from + v * 16);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const int pair = (v * E + e) / 2;
        if (pair < a.pairs) {
          const float2 cs = tr[pair];
          const float x0 = x.x[e], x1 = x.x[e + 1];
          x.x[e] = x0 * cs.x - x1 * cs.y;
          x.x[e + 1] = x1 * cs.x + x0 * cs.y;
        }
      }
      *(uint4*)(to + v * 16) = x.bits();
    } else if constexpr (HOW == kHalvesOver) {
      // both halves, then what is not rotated, each in whole vectors at any alignment; the last of them begins inside the
      // one before it, and writes the same there
      const int low = (a.pairs + E - 1) / E, rest = 2 * a.pairs;
      if (v < low) {
        const int d = min(v * E, a.pairs - E);
        Vec<F32> y;
        x.unpack(load_any(from + d * ES));
        y.unpack(load_any(from + (d + a.pairs) * ES));
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 cs = tr[d + e];
          const float x0 = x.x[e], x1 = y.x[e];
          x.x[e] = x0 * cs.x - x1 * cs.y;
          y.x[e] = x1 * cs.x + x0 * cs.y;
        }
        store_any(to + d * ES, x.bits());
        store_any(to + (d + a.pairs) * ES, y.bits());
      } else {
        const int d = min(rest + (v - low) * E, dim - E);
        store_any(to + d * ES, load_any(from + d * ES));
      }
    } else {
      // the partners of a vector's elements are as many elements before or after it, at any alignment
      x.load(from + v * 16);
      const int d = v * E;
      Vec<F32> y;
      const bool low = d + E <= a.pairs && d + a.pairs + E <= dim, high = d >= a.pairs && d + E <= 2 * a.pairs;
      if (low || high) {
        y.unpack(load_any(from + (low ? d + a.pairs : d - a.pairs) * ES));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int p = d + e < a.pairs ? d + e + a.pairs : d + e < 2 * a.pairs ? d + e - a.pairs : d + e;
          y.x[e] = element<F32>(from, p);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int pair = d + e < a.pairs ? d + e : d + e - a.pairs;
        if (pair < a.pairs) {
          const float2 cs = tr[pair];
          const float other = y.x[e] * cs.y;
          x.x[e] = x.x[e] * cs.x + (d + e < a.pairs ? -other : other);
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
  if (fresh->tokens < 0 || fresh->tokens > (1 << 23) || fresh->heads < 1 || turn->pairs < 1 ||
      2 * turn->pairs > cache->dim || turn->axes < 1) {
    set_error("kv_append_rotated: %lld tokens (0 to 2^23), %lld heads, %lld pairs of %d elements, %lld axes",
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
    for (int64_t x : s) ok = ok && x >= 0 && x < ((int64_t)1 << 35) && x * es % 16 == 0 && x * es / 16 <= UINT32_MAX;
    ok = ok && s[2] * es <= UINT32_MAX;
    ok = ok && ((uintptr_t)in[i] & 15) == 0;
    a.in[i] = (const char*)in[i];
    a.batch_at[i] = (uint32_t)(s[0] * es / 16);
    a.token_at[i] = (uint32_t)(s[1] * es / 16);
    a.head_at[i] = (uint32_t)(s[2] * es);
  }
  if (!ok) {
    set_error("kv_append_rotated: q, k, v, their strides and out_q must be multiples of 16 bytes, below 2^36, of heads 2^32");
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
  // Halves that are no whole vectors: in vectors over each other in bfloat16 (4 x 4096 tokens of 32 + 2 x 8 heads of 128, 33
  // pairs 96 us, each vector as itself and as a partner 121; of 80, 36 pairs 44 and 61), not in float32, whose vectors hold
  // half as many elements and whose other way is at the memory's rate (35 of 128 83 and 80.5), nor where single elements are
  // left (63 of 128 109 and 103, 5 121 and 108).
  const int left = cache->dim - 2 * a.pairs;
  const bool over = es == 2 && a.pairs >= e && (left == 0 || left >= e);
  const PairsAre how = turn->neighbours ? kNeighbours : a.pairs % e == 0 ? kHalves : over ? kHalvesOver : kHalvesAny;
  const int per_head = how == kHalves       ? vecs - a.pairs / e
                       : how == kHalvesOver ? (a.pairs + e - 1) / e + (left + e - 1) / e
                                            : vecs;
  const int64_t items = (int64_t)(a.heads + a.kv_heads) * per_head + (int64_t)a.kv_heads * vecs;
  a.per_head = make_page_div(per_head);
  a.per_value = make_page_div(vecs);
  // A token's threads: 256 unless it has fewer items than that; and several workgroups to one where they are few.
  const int64_t all = (int64_t)cache->batch * a.tokens;
  a.per_token = make_page_div(a.pairs);
  a.log_tokens = items <= 192 ? 2 : items <= 300 ? 1 : 0;
  while (a.log_tokens > 0 && 1 << (a.log_tokens - 1) >= a.tokens) --a.log_tokens;
  const int64_t blocks = a.tokens > 0 ? (a.tokens + (1 << a.log_tokens) - 1) >> a.log_tokens : 1;
  int64_t split = ((items << a.log_tokens) + 255) / 256;
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
    else if (how == kHalvesOver) kv_rotate_kernel<false, kHalvesOver><<<grid, 256, 0, s>>>(a);
    else if (how == kHalvesAny) kv_rotate_kernel<false, kHalvesAny><<<grid, 256, 0, s>>>(a);
    else kv_rotate_kernel<false, kNeighbours><<<grid, 256, 0, s>>>(a);
  }
  return launch_status("kv_append_rotated");
}

}  // extern "C"
