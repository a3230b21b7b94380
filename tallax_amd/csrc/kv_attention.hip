// Attention of the newest tokens over a paged key-value cache.
//
// One workgroup of four waves takes one kv head of one sequence, up to 16 * MT
// of its query rows (row = query * group + head in the group) and one chunk of
// the length; a wave takes every fourth tile of the chunk and keeps its own
// running maximum, sum and output, joined in LDS at the chunk's end.  Chunks
// are joined by a second kernel.
//
// Both products have the tokens of a tile as a matrix dimension and are laid
// out so that nothing is exchanged between lanes, and neither keys nor values go
// through LDS:
//   S^T = K Q^T   operand A: lane (n, g) holds 16 bytes of token n's key,
//                 B: of row n's query (from LDS); the result has row n's scores
//                 of tokens 4g .. 4g + 3 in lane (n, g)
//                 (n = lane % 16, g = lane / 16);
//   O^T = V^T P^T operand B: those scores as they lie; operand A: the values of
//                 the same tokens, which lane (n, g) has loaded (dim / 16 of
//                 each token, so 16 lanes read a token's value in one piece) and
//                 transposes in its own registers.  out_dim has the order in
//                 which the outputs then lie.
// bfloat16 takes the 16x16x32 products on tiles of 32 tokens (above dim 128
// 16x16x16 ones on 16), float32 the 16x16x4 ones on tiles of 16.
//
// Bound by memory.  64 sequences of up to 4096 slots, 8 kv heads of 128
// (bfloat16), 685 MB: 148 us here and 13 in the join, 4.2 TB/s; 4 of up to
// 131071, 1.54 GB: 285 and 5 us, 5.3 TB/s; the loads alone take 136 and 277 us.
// Float32, 9 of up to 2050, 12 heads of 80, 90 MB: 26 and 5 us, loads alone 22.
//
// The length is split by max_len, which is the table's width unless the caller
// knows a smaller bound: 4 sequences of up to 4096 slots with 8 kv heads take 16 us,
// also in a table of 131072 slots with max_len 4096, and 54 there without it.
#include <math.h>

#include "tx_common.h"
#include "tx_kv.h"

namespace tx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = 4;

struct AttnArgs {
  KvView c;
  const char* q;
  int64_t q_batch, q_query, q_head;  // strides in bytes
  const int32_t* lens;
  const int32_t* counts;
  char* out;
  float* lse;
  int queries, heads, kv_heads, group;  // group = heads / kv_heads
  int rows;                             // queries * group
  int max_len, chunk, chunks;
  int row_groups;                       // workgroups that share a kv head's rows
  int shift;                            // offsets in the pools are in units of 2^shift bytes
  uint32_t k_page, k_slot, v_page, v_slot;
  float scale2;                         // scale * log2 e
  float2* part_ml;                      // [batch * kv_heads][chunks][rows]: maximum (base 2), sum
  float* part_o;                        // [batch * kv_heads][chunks][rows][dim]
  float* raw;                           // [batch * kv_heads][rows][raw_ld]: scores (base 2), or null
  int raw_ld;
  const float* scores;
  float* out_scores;
  int vector_scores;                    // their rows are whole 16-byte vectors
};

// What a sequence's rows see: row of query t sees slots below limit(t).
struct Seen {
  int len, cnt, first;  // first + t = limit of query t
  __device__ __forceinline__ Seen(const AttnArgs& a, int b) {
    len = min(max(a.lens[b], 0), a.max_len);
    cnt = a.queries;
    if (a.counts) cnt = min(max(a.counts[b], 0), a.queries);
    first = len - cnt + 1;
  }
  __device__ __forceinline__ int limit(int t) const { return t < cnt ? min(first + t, len) : 0; }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // round to nearest even
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  bf16x2_t r;
  r[0] = (__bf16)lo;
  r[1] = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ bool bf16_pair_not_finite(uint32_t w) {
  return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
}

template <bool F32, int DP>
struct Tile {
  static constexpr int kTokens = F32 || DP > 128 ? 16 : 32;    // 16 where keys and values of 32 would fill the registers
  static constexpr int kParts = kTokens / 16;                  // 16-token parts
  static constexpr int kKeyVecs = F32 ? DP / 16 : DP / 32;     // 16-byte vectors of a key per lane and 16 tokens
  static constexpr int kValueTokens = kTokens / 4;             // tokens whose values a lane holds
  static constexpr int kValueWords = F32 ? DP / 16 : DP / 32;  // 32-bit words of each
  static constexpr int kAcc = DP / 16;                         // products (and f32x4 accumulators) per 16 rows
};

// A tile's keys (16 tokens, 16-byte vectors) and values (tokens, words) in a lane's registers.
template <bool F32, int DP>
using Key = uint4[Tile<F32, DP>::kKeyVecs];
template <bool F32, int DP>
using Value = uint32_t[Tile<F32, DP>::kValueWords];
template <bool F32, int DP>
using Keys = uint4[Tile<F32, DP>::kParts][Tile<F32, DP>::kKeyVecs];
template <bool F32, int DP>
using Values = uint32_t[Tile<F32, DP>::kValueTokens][Tile<F32, DP>::kValueWords];

// x of 16 tokens for 16 rows: S^T in the accumulator layout.  q: this lane's
// vectors of the rows' queries in LDS, one every 64 lanes.
template <bool F32, int DP>
__device__ __forceinline__ void scores_of(const Keys<F32, DP>& key, const uint4* q, int dim, f32x4 (&s)[Tile<F32, DP>::kParts]) {
  using T = Tile<F32, DP>;
#pragma unroll
  for (int u = 0; u < T::kParts; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < T::kKeyVecs; ++i) {
    if (F32 && 16 * i >= dim) continue;
    const uint4 qi = q[i * kWave];
#pragma unroll
    for (int u = 0; u < T::kParts; ++u) {
      const uint4 k = key[u][i];
      if constexpr (F32) {
        s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.x), __uint_as_float(qi.x), s[u], 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.y), __uint_as_float(qi.y), s[u], 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.z), __uint_as_float(qi.z), s[u], 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.w), __uint_as_float(qi.w), s[u], 0, 0, 0);
      } else {
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, qi),
                                                       s[u], 0, 0, 0);
      }
    }
  }
}

// O^T += V^T P^T for 16 * MT rows
template <bool F32, int DP, int MT>
__device__ __forceinline__ void add_values(const Values<F32, DP>& v, const float (&p)[MT][Tile<F32, DP>::kTokens / 4],
                                           int dim, f32x4 (&acc)[MT][Tile<F32, DP>::kAcc]) {
  if constexpr (F32) {
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      if (32 * (j / 2) >= dim) continue;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][j]), p[mt][r], acc[mt][j], 0, 0, 0);
    }
  } else {
    // Element j of a lane's tokens by the rows' weights: 32 tokens a product, or 16.  The product takes both sides in
    // bfloat16: the weights, at most 1, are rounded to it (by 2^-8 of each at most), and their sum, by which the output
    // is divided, is of the unrounded ones.  The roundings are of either sign and meet the output's own to bfloat16:
    // against 64 bits the output is off by 5 to 8 % more than with 32-bit weights, which would take two products or
    // the float32 ones at an eighth of the rate.
    constexpr int kPairs = Tile<F32, DP>::kValueTokens / 2;
    uint32_t pb[MT][kPairs];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int k = 0; k < kPairs; ++k) pb[mt][k] = pack_bf16(p[mt][2 * k], p[mt][2 * k + 1]);
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
      uint32_t t[kPairs];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) t[k] = __builtin_amdgcn_perm(v[2 * k + 1][j / 2], v[2 * k][j / 2], sel);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (kPairs == 4)
          acc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, make_uint4(t[0], t[1], t[2], t[3])),
              __builtin_bit_cast(bf16x8_t, make_uint4(pb[mt][0], pb[mt][1], pb[mt][2], pb[mt][3])), acc[mt][j], 0, 0, 0);
        else
          acc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
              __builtin_bit_cast(bf16x4, make_uint2(t[0], t[1])), __builtin_bit_cast(bf16x4, make_uint2(pb[mt][0], pb[mt][1])),
              acc[mt][j], 0, 0, 0);
      }
    }
  }
}

// d of accumulator j, register r, lane group g.  bfloat16: a lane holds DP / 16
// neighbouring elements of a value; float32: two of each 32.
template <bool F32, int DP>
__device__ __forceinline__ int out_dim(int j, int r, int g) {
  return F32 ? 32 * (j / 2) + 2 * (4 * g + r) + (j & 1) : (DP / 16) * (4 * g + r) + j;
}

__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)x);
}

// Every load of a tile is issued, in the same order, whatever there is to load:
// waiting for one then does not mean waiting for those after it.  Elements past
// dim are read from the token's first ones.
template <bool F32, int DP>
__device__ __forceinline__ void load_key(Key<F32, DP>& k, const char* p, int g, int dim) {
#pragma unroll
  for (int i = 0; i < Tile<F32, DP>::kKeyVecs; ++i) {
    const int d = F32 ? 16 * i + 4 * g : 32 * i + 8 * g;
    k[i] = *(const uint4*)(p + (d < dim ? d : 0) * (F32 ? 4 : 2));
  }
}

template <bool F32, int DP>
__device__ __forceinline__ void load_value(Value<F32, DP>& w, const char* p, int n, int dim) {
  if constexpr (F32 || DP == 64) {
    constexpr int E = F32 ? 2 : 4;  // elements of 8 bytes
#pragma unroll
    for (int c = 0; c < Tile<F32, DP>::kValueWords / 2; ++c) {
      const int d = 16 * E * c + E * n;
      const uint2 x = *(const uint2*)(p + (d < dim ? d : 0) * (8 / E));
      w[2 * c] = x.x;
      w[2 * c + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int c = 0; c < DP / 128; ++c) {
      const int d = (DP / 16) * n + 8 * c;
      const uint4 x = *(const uint4*)(p + 2 * (d < dim ? d : 0));
      w[4 * c] = x.x;
      w[4 * c + 1] = x.y;
      w[4 * c + 2] = x.z;
      w[4 * c + 3] = x.w;
    }
  }
}

// Adds weight times value where the value is not finite, for tokens from..to - 1
// of the tile at t0, to those of 16 rows that see the token.
template <bool F32>
__device__ __forceinline__ void add_strange(const AttnArgs& a, const Seen& seen, const char* vbase, uint32_t v_at,
                                            uint64_t gone, int t0, int from, int to, int row0, float* outs, int ld,
                                            const float* weights) {
#pragma unroll 1
  for (int in = from; in < to; ++in) {
    const char* p = vbase + ((uint64_t)from_lane(v_at, in) << a.shift);
    if ((gone >> in) & 1) continue;
#pragma unroll 1
    for (int d = lane_id(); d < a.c.dim; d += kWave) {
      const float v = F32 ? ((const float*)p)[d] : __uint_as_float((uint32_t)((const uint16_t*)p)[d] << 16);
      if ((__float_as_uint(v) & 0x7f800000u) != 0x7f800000u) continue;
#pragma unroll 1
      for (int r = 0; r < 16 && row0 + r < a.rows; ++r)
        if (t0 + in < seen.limit((row0 + r) / a.group)) outs[r * ld + d] += weights[in * 16 + r] * v;
    }
  }
}

// Waves of a SIMD that the registers of an instance are held to.  Left to itself
// the compiler takes 350 registers for <bfloat16, 128, 2>, which is one wave: 32
// sequences of up to 8191 slots with 5 queries 231 us without scores, against 142
// with two; a third spills (414 us).  Instances for one query leave out what takes
// values that are not finite apart (half of the code and 35 registers), and those
// of 16 rows hold three waves.  In float32 that pays where two would leave
// workgroups waiting for a place on the card.  Of 152 cases of one query, those
// with 769 to 1152 workgroups are 2 to 19 % faster with three in 13 of 14 (9
// sequences of up to 2050 slots with 12 heads of 80 31.1 us, with two 38.3), and
// those with more by 2 % in the mean; those with 513 to 768, three to a CU, are 4
// to 21 % slower in 14 of 16 (7 of 2985 with 8 of 128 36.8, with two 31.9), and
// those with fewer the same.  With several queries two are faster in 35 of 41, by
// 2 % in the mean.
template <bool F32, int DP, int MT, bool MANY>
constexpr int kWavesHeld = F32 && DP > 128 ? 1 : DP == 128 && MT == 1 && !MANY ? 3 : 2;
constexpr int64_t kTwoWavesUpTo = 3 * 256;  // workgroups of a float32 launch of one query

// MANY: more queries than one, so that some rows do not see the newest tokens.
template <bool F32, int DP, int MT, bool MANY, int WAVES>
__global__ __launch_bounds__(kAttnThreads, WAVES) void kv_decode_kernel(AttnArgs a) {
  using T = Tile<F32, DP>;
  constexpr int ES = F32 ? 4 : 2;
  constexpr int STEP = kAttnWaves * T::kTokens;
  extern __shared__ float lds[];  // [kAttnWaves][16][DP + 4], m and l of the waves, the queries, weights
  uint4* queries = (uint4*)(lds + kAttnWaves * 16 * (DP + 4) + (kAttnWaves + 1) * 32);  // [MT][kKeyVecs][64]

  const int rg = blockIdx.x % a.row_groups;
  const int unit = blockIdx.x / a.row_groups;  // sequence * kv_heads + kv head
  const int b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
  const int wave = threadIdx.x / kWave, lane = lane_id(), n = lane & 15, g = lane >> 4;
  const Seen seen(a, b);
  const int start = blockIdx.y * a.chunk;
  if (start >= seen.len && a.chunks > 1) return;
  const int end = min(start + a.chunk, seen.len);
  const int row0 = rg * 16 * MT;

  const char* kbase = a.c.k + kvh * a.c.k_head;
  const char* vbase = a.c.v + kvh * a.c.v_head;
  const int32_t* table = a.c.table + (int64_t)b * a.c.width;
  const int mine = lane & (T::kTokens - 1);
  auto page_at = [&](int t0) { return t0 + mine < end ? page_id(a.c, table, t0 + mine) : -1; };
  int t0 = start + wave * T::kTokens;
  // Each lane works out the place of one token and hands it to those that load
  // from it.  Tokens past the end or in no page are read from a query.
  const char* safe = a.q + b * a.q_batch + (int64_t)(kvh * a.group) * a.q_head;
  struct Places {
    int page;
    uint32_t k, v;
  };
  auto places_of = [&](int t, int page) {
    const int off = t + mine - (int)page_of(a.c.div, (uint32_t)(t + mine)) * a.c.div.size;
    return Places{page, (uint32_t)page * a.k_page + (uint32_t)off * a.k_slot,
                  (uint32_t)page * a.v_page + (uint32_t)off * a.v_slot};
  };
  Keys<F32, DP> key;
  auto load_keys = [&](const Places& pl) {
#pragma unroll
    for (int u = 0; u < T::kParts; ++u) {
      const char* p = kbase + ((uint64_t)from_lane(pl.k, 16 * u + n) << a.shift);
      load_key<F32, DP>(key[u], (int)from_lane((uint32_t)pl.page, 16 * u + n) >= 0 ? p : safe, g, a.c.dim);
    }
  };
  Places next = places_of(t0, page_at(t0));
  load_keys(next);
  int next_page = page_at(t0 + STEP);

  for (int i = threadIdx.x; i < MT * T::kKeyVecs * kWave; i += kAttnThreads) {
    const int l = i % kWave, v = i / kWave % T::kKeyVecs, mt = i / (kWave * T::kKeyVecs);
    const int row = row0 + 16 * mt + (l & 15), t = row / a.group;
    const int d = F32 ? 16 * v + 4 * (l >> 4) : 32 * v + 8 * (l >> 4);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row < a.rows && d < a.c.dim)
      x = *(const uint4*)(a.q + b * a.q_batch + t * a.q_query +
                          (int64_t)(kvh * a.group + row - t * a.group) * a.q_head + d * ES);
    queries[i] = x;
  }
  f32x4 acc[MT][T::kAcc];
  float wm[MT], wl[MT];
  int limit[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + n;
    limit[mt] = row < a.rows ? seen.limit(row / a.group) : 0;
    wm[mt] = -INFINITY;
    wl[mt] = 0.0f;
#pragma unroll
    for (int j = 0; j < T::kAcc; ++j) acc[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // below this every row of a query that counts sees every slot
  const int open = min(seen.first, end);
  __syncthreads();

  for (; t0 < end; t0 += STEP) {
    const Places here = next;
    const uint32_t v_at = here.v;
    const uint64_t gone = __ballot(here.page < 0);  // bit i: token i of the tile is past the end or in no page
    const bool plain = t0 + T::kTokens <= open && gone == 0;
    Values<F32, DP> val;
#pragma unroll
    for (int j = 0; j < T::kValueTokens; ++j) {
      const int in = 16 * (j / 4) + 4 * g + (j & 3);
      const char* p = vbase + ((uint64_t)from_lane(v_at, in) << a.shift);
      load_value<F32, DP>(val[j], (gone >> in) & 1 ? safe : p, n, a.c.dim);
    }
    next = places_of(t0 + STEP, next_page);
    next_page = page_at(t0 + 2 * STEP);
    if (DP != a.c.dim) {
#pragma unroll
      for (int u = 0; u < T::kParts; ++u)
#pragma unroll
        for (int i = 0; i < T::kKeyVecs; ++i)
          if ((F32 ? 16 * i + 4 * g : 32 * i + 8 * g) >= a.c.dim) key[u][i] = make_uint4(0, 0, 0, 0);
    }
    float x[MT][4 * T::kParts];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4 s[T::kParts];
      scores_of<F32, DP>(key, queries + mt * T::kKeyVecs * kWave + lane, a.c.dim, s);
#pragma unroll
      for (int u = 0; u < T::kParts; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[mt][4 * u + r] = s[u][r] * a.scale2;
    }
    // the next tile's keys take the registers of these
    __builtin_amdgcn_sched_barrier(0);
    load_keys(next);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (!plain) {
#pragma unroll
        for (int u = 0; u < T::kParts; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int in = 16 * u + 4 * g + r;
            if (((gone >> in) & 1) || t0 + in >= limit[mt]) x[mt][4 * u + r] = -INFINITY;
          }
      }
      if (a.raw) {
        const int row = row0 + 16 * mt + n;
        if (limit[mt] > 0) {
          float* rp = a.raw + ((int64_t)unit * a.rows + row) * a.raw_ld + t0 + 4 * g;
#pragma unroll
          for (int u = 0; u < T::kParts; ++u)
            *(float4*)(rp + 16 * u) = make_float4(x[mt][4 * u], x[mt][4 * u + 1], x[mt][4 * u + 2], x[mt][4 * u + 3]);
        }
      }
      float top = x[mt][0];
#pragma unroll
      for (int i = 1; i < 4 * T::kParts; ++i) top = fmaxf(top, x[mt][i]);
      top = fmaxf(top, lane_xor_f(top, 16));
      top = fmaxf(top, lane_xor_f(top, 32));
      const float m = fmaxf(wm[mt], top);
      const float base = m == -INFINITY ? 0.0f : m;  // nothing seen yet: every weight is exp2(-inf) = 0
      if (__ballot(m > wm[mt])) {  // seldom, after the first tiles
        const float shrink = __builtin_amdgcn_exp2f(wm[mt] - base);
        wm[mt] = m;
        wl[mt] *= shrink;
#pragma unroll
        for (int j = 0; j < T::kAcc; ++j) acc[mt][j] *= shrink;
      }
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * T::kParts; ++i) {
        x[mt][i] = __builtin_amdgcn_exp2f(x[mt][i] - base);
        sum += x[mt][i];
      }
      wl[mt] += sum;
    }
    // A value that is not finite would reach rows that do not see its token
    // through 0 * inf: those are taken out of the product and added to the rows
    // that see them one by one.
    if (!plain) {
#pragma unroll
      for (int j = 0; j < T::kValueTokens; ++j)
#pragma unroll
        for (int i = 0; i < T::kValueWords; ++i)
          val[j][i] = (gone >> (16 * (j / 4) + 4 * g + (j & 3))) & 1 ? 0u : val[j][i];
    }
    if (MANY && !plain) {
      bool strange = false;
#pragma unroll
      for (int j = 0; j < T::kValueTokens; ++j)
#pragma unroll
        for (int i = 0; i < T::kValueWords; ++i)
          strange = strange || (F32 ? (val[j][i] & 0x7f800000u) == 0x7f800000u : bf16_pair_not_finite(val[j][i]));
      if (__ballot(strange)) {
        // not a constant to the compiler: it would keep the addresses below in registers through the whole loop
        int here = wave;
        asm volatile("" : "+v"(here));
        float* outs = lds + here * 16 * (DP + 4);                              // [row][DP + 4]
        float* weights = (float*)(queries + MT * T::kKeyVecs * kWave) + here * 16 * T::kTokens;  // [token][row]
        const int row_at = (lane & 15) * (DP + 4);
#pragma unroll
        for (int j = 0; j < T::kValueTokens; ++j) {
          const bool all = t0 + 16 * (j / 4) + 4 * g + (j & 3) < open;
#pragma unroll
          for (int i = 0; i < T::kValueWords; ++i) {
            uint32_t v = val[j][i];
            if constexpr (F32) {
              v = (v & 0x7f800000u) == 0x7f800000u ? 0u : v;
            } else {
              v = (v & 0x7f800000u) == 0x7f800000u ? v & 0xffffu : v;
              v = (v & 0x7f80u) == 0x7f80u ? v & 0xffff0000u : v;
            }
            val[j][i] = all ? val[j][i] : v;
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int j = 0; j < T::kAcc; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) outs[row_at + out_dim<F32, DP>(j, r, g)] = acc[mt][j][r];
#pragma unroll
          for (int i = 0; i < 4 * T::kParts; ++i) weights[(16 * (i / 4) + 4 * g + (i & 3)) * 16 + n] = x[mt][i];
          add_strange<F32>(a, seen, vbase, v_at, gone, t0, max(open - t0, 0), T::kTokens, row0 + 16 * mt, outs, DP + 4,
                           weights);
#pragma unroll
          for (int j = 0; j < T::kAcc; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[mt][j][r] = outs[row_at + out_dim<F32, DP>(j, r, g)];
        }
      }
    }
    add_values<F32, DP, MT>(val, x, a.c.dim, acc);
  }
  // join the four waves
  float* ml = lds + kAttnWaves * 16 * (DP + 4);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float l = wl[mt];
    l += lane_xor_f(l, 16);
    l += lane_xor_f(l, 32);
    if (limit[mt] <= 0) {  // a row that sees nothing
      wm[mt] = -INFINITY;
      l = 0.0f;
    }
    if (g == 0) {
      ml[(wave * 16 + n) * 2] = wm[mt];
      ml[(wave * 16 + n) * 2 + 1] = l;
    }
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kAttnWaves; ++i) m = fmaxf(m, ml[(i * 16 + n) * 2]);
    const float base = m == -INFINITY ? 0.0f : m;
    const float mine = __builtin_amdgcn_exp2f(wm[mt] - base);
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < kAttnWaves; ++i)
      l += ml[(i * 16 + n) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(i * 16 + n) * 2] - base);
    float* mo = lds + (wave * 16 + n) * (DP + 4);
    // four neighbouring outputs are one register of four products, or two registers of two (out_dim)
    const bool none = wm[mt] == -INFINITY;
    if (row0 + 16 * mt + n < a.rows) {
#pragma unroll
      for (int i = 0; i < T::kAcc; ++i) {
        const int j = F32 ? i / 2 * 2 : i / 4 * 4, r = F32 ? i % 2 * 2 : i % 4;
        const f32x4(&o)[T::kAcc] = acc[mt];
        const float4 x = F32 ? make_float4(o[j][r], o[j + 1][r], o[j][r + 1], o[j + 1][r + 1])
                             : make_float4(o[j][r], o[F32 ? 0 : j + 1][r], o[F32 ? 0 : j + 2][r], o[F32 ? 0 : j + 3][r]);
        *(float4*)(mo + out_dim<F32, DP>(j, r, g)) =
            none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * mine, x.y * mine, x.z * mine, x.w * mine);
      }
    }
    if (wave == 0 && g == 0) {  // for the threads that write the rows
      ml[kAttnWaves * 32 + 2 * n] = m;
      ml[kAttnWaves * 32 + 2 * n + 1] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (DP / 4); i += kAttnThreads) {
      const int rn = i / (DP / 4), d = (i - rn * (DP / 4)) * 4;
      const int row = row0 + 16 * mt + rn;
      if (row >= a.rows || d >= a.c.dim) continue;
      if (a.chunks > 1 && seen.limit(row / a.group) <= 0) continue;  // nor does the second kernel read it
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kAttnWaves; ++k) {
        const float4 x = *(const float4*)(lds + (k * 16 + rn) * (DP + 4) + d);
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      const float rm = ml[kAttnWaves * 32 + 2 * rn], rl = ml[kAttnWaves * 32 + 2 * rn + 1];
      if (a.chunks > 1) {
        const int64_t at = ((int64_t)unit * a.chunks + blockIdx.y) * a.rows + row;
        *(float4*)(a.part_o + at * a.c.dim + d) = o;
        if (d == 0) a.part_ml[at] = make_float2(rm, rl);
      } else {
        const float inv = rl == 0.0f ? 0.0f : 1.0f / rl;
        const int t = row / a.group;
        const int64_t head = ((int64_t)b * a.queries + t) * a.heads + kvh * a.group + (row - t * a.group);
        const bool none = rl == 0.0f;
        o.x = none ? 0.f : o.x * inv, o.y = none ? 0.f : o.y * inv, o.z = none ? 0.f : o.z * inv,
        o.w = none ? 0.f : o.w * inv;
        if constexpr (F32)
          *(float4*)(a.out + (head * a.c.dim + d) * 4) = o;
        else
          *(uint2*)(a.out + (head * a.c.dim + d) * 2) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
        if (d == 0) {
          if (a.lse) a.lse[head] = none ? -INFINITY : (rm + __builtin_amdgcn_logf(rl)) * kLn2;
          if (a.raw) a.part_ml[(int64_t)unit * a.rows + row] = make_float2(rm, rl);
        }
      }
    }
    __syncthreads();
  }
}

// Maximum and sum of a row over its chunks, by `width` neighbouring lanes (a
// power of two, `l` of them this one); the same in all of them.
__device__ __forceinline__ float2 join_row(const float2* ml, int nch, int rows, int row, int l, int width) {
  float m = -INFINITY, s = 0.0f;
  auto add = [&](float om, float os) {
    const float t = fmaxf(m, om), base = t == -INFINITY ? 0.0f : t;
    s = s * __builtin_amdgcn_exp2f(m - base) + os * __builtin_amdgcn_exp2f(om - base);
    m = t;
  };
  for (int c = l; c < nch; c += width) {
    const float2 x = ml[(int64_t)c * rows + row];
    add(x.x, x.y);
  }
  for (int d = 1; d < width; d <<= 1) {
    const float om = __uint_as_float(from_lane(__float_as_uint(m), lane_id() ^ d));
    const float os = __uint_as_float(from_lane(__float_as_uint(s), lane_id() ^ d));
    add(om, os);
  }
  return make_float2(m, s);
}

// Joins the chunks.  The first `rows` workgroups of a sequence's kv head (where
// there is more than one chunk) take an output row each, the chunks shared out
// over groups of lanes; the others sum 1024 slots' weights over the rows.
__global__ __launch_bounds__(256) void kv_decode_join_kernel(AttnArgs a, int f32, int out_blocks) {
  extern __shared__ float lds[];  // an output row: 256 x 4 sums; weights: base and 1 / sum of each row
  const int unit = blockIdx.x, b = unit / a.kv_heads, kvh = unit - b * a.kv_heads, tid = threadIdx.x;
  const Seen seen(a, b);
  const int chunks = a.chunks > 1 ? (seen.len + a.chunk - 1) / a.chunk : 1;
  const float2* ml = a.part_ml + (int64_t)unit * a.chunks * a.rows;
  if ((int)blockIdx.y < out_blocks) {
    const int row = blockIdx.y, t = row / a.group;
    const int64_t head = ((int64_t)b * a.queries + t) * a.heads + kvh * a.group + (row - t * a.group);
    const int nch = seen.limit(t) > 0 ? chunks : 0;
    const float2 j = join_row(ml, nch, a.rows, row, lane_id(), kWave);
    const float base = j.x == -INFINITY ? 0.0f : j.x;
    const int width = a.c.dim <= 64 ? 16 : a.c.dim <= 128 ? 32 : 64;  // lanes that hold a row
    const int d = (tid & (width - 1)) * 4, groups = 256 / width;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < a.c.dim) {
#pragma unroll 4
      for (int c = tid / width; c < nch; c += groups) {
        const int64_t at = ((int64_t)unit * a.chunks + c) * a.rows + row;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[at].x - base);
        const float4 x = *(const float4*)(a.part_o + at * a.c.dim + d);
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
      }
    }
    float4* sums = (float4*)lds;
    sums[tid] = o;
    __syncthreads();
    if (tid < width && d < a.c.dim) {
      for (int k = 1; k < groups; ++k) {
        const float4 x = sums[k * width + tid];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      const float inv = j.y == 0.0f ? 0.0f : 1.0f / j.y;
      const bool none = j.y == 0.0f;
      o.x = none ? 0.f : o.x * inv, o.y = none ? 0.f : o.y * inv, o.z = none ? 0.f : o.z * inv,
      o.w = none ? 0.f : o.w * inv;
      if (f32)
        *(float4*)(a.out + (head * a.c.dim + d) * 4) = o;
      else
        *(uint2*)(a.out + (head * a.c.dim + d) * 2) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
      if (tid == 0 && a.lse) a.lse[head] = none ? -INFINITY : (j.x + __builtin_amdgcn_logf(j.y)) * kLn2;
    }
    return;
  }
  const int slot0 = ((int)blockIdx.y - out_blocks) * 1024 + tid * 4;
  const bool some = slot0 - tid * 4 < seen.len;  // else this workgroup's slots are copied
  if (some) {
    int width = 1;  // lanes of a row
    while (width < chunks && width < kWave) width <<= 1;
    const int used = seen.cnt * a.group, at_once = kWave / width;
    for (int row0 = tid / kWave * at_once; row0 < used; row0 += 4 * at_once) {
      const int row = row0 + lane_id() / width, l = lane_id() & (width - 1);
      const bool sees = row < used && seen.limit(row / a.group) > 0;
      const float2 j = join_row(ml, sees ? chunks : 0, a.rows, row, l, width);
      if (l == 0 && row < used) {
        lds[2 * row] = j.x == -INFINITY ? 0.0f : j.x;
        lds[2 * row + 1] = j.y == 0.0f ? -1.0f : 1.0f / j.y;
      }
    }
    __syncthreads();
  }
  if (slot0 >= a.c.capacity) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (some && slot0 < seen.len) {  // raw rows are whole tiles: what lies past len in one is dropped below
    const float* raw = a.raw + (int64_t)unit * a.rows * a.raw_ld + slot0;
    // eight rows are asked for before the first is used
    const int used = seen.cnt * a.group;
    for (int row0 = 0; row0 < used; row0 += 8) {
      float4 x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = *(const float4*)(raw + (int64_t)min(row0 + r, used - 1) * a.raw_ld);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (row0 + r >= used || lds[2 * (row0 + r) + 1] == -1.0f) continue;  // a row that sees nothing
        const float base = lds[2 * (row0 + r)], inv = lds[2 * (row0 + r) + 1];
        s.x += __builtin_amdgcn_exp2f(x[r].x - base) * inv;
        s.y += __builtin_amdgcn_exp2f(x[r].y - base) * inv;
        s.z += __builtin_amdgcn_exp2f(x[r].z - base) * inv;
        s.w += __builtin_amdgcn_exp2f(x[r].w - base) * inv;
      }
    }
  }
  const int64_t at = (int64_t)unit * a.c.capacity + slot0;
  if (a.vector_scores) {
    float4 o = *(const float4*)(a.scores + at);
    if (slot0 < seen.len) o.x += s.x;
    if (slot0 + 1 < seen.len) o.y += s.y;
    if (slot0 + 2 < seen.len) o.z += s.z;
    if (slot0 + 3 < seen.len) o.w += s.w;
    *(float4*)(a.out_scores + at) = o;
  } else {
    const float ss[4] = {s.x, s.y, s.z, s.w};
    for (int k = 0; k < 4 && slot0 + k < a.c.capacity; ++k)
      a.out_scores[at + k] = a.scores[at + k] + (slot0 + k < seen.len ? ss[k] : 0.0f);
  }
}

struct AttnPlan {
  int mt, row_groups, chunk, chunks, max_len, rows, raw_ld;
  size_t ml_bytes, o_bytes, raw_bytes;
};

static void plan_attention(int64_t batch, int64_t kv_heads, int64_t rows, int dim, int dtype, int64_t max_len,
                           bool with_scores, AttnPlan* p) {
  const int tiles = (int)((rows + 15) / 16), most = dtype != TALLAX_F32 && dim > 128 ? 1 : 2;
  // 32 rows of a kv head to a workgroup, or 16: rows beyond are a workgroup of their own, which reads the keys and
  // values again.  Its registers cost more than that: with 64 rows of dim 128 and 32 of dim 256 (bfloat16) a SIMD
  // holds one wave, and 16 sequences x 48 rows take 207 us, against 125; 13 x 40 rows of dim 192 226, against 124.
  p->mt = tiles < most ? 1 : most;
  p->row_groups = (tiles + p->mt - 1) / p->mt;
  p->rows = (int)rows;
  p->max_len = (int)max_len;
  const int64_t units = batch * kv_heads * p->row_groups;
  // Chunks of about 2048 workgroups: sequences of uneven length leave some without work, and the rest still fill the
  // card.  With few kv heads in all 512 longer ones lose less to their beginnings and ends: 32 of 131071 slots 289 us
  // against 303, 128 of 4000 34 against 40; with 512 of 4096 they take 170 against 162, and 108 float32 ones of 2050,
  // whose products take longer, 44 against 35; 26 with three workgroups of rows each 138 against 127.  Chunks of 128 slots, not 256, where those are too few for the card:
  // 5 kv heads of 2756 slots 11.2 us against 12.6; but up to 256 slots are one chunk, which needs no second launch
  // (2 kv heads of 200 slots 6.4 us against 9.6).
  const int64_t target = p->row_groups == 1 && units <= (dtype == TALLAX_F32 ? 32 : 128) ? 512 : 2048;
  const int64_t least = max_len > 256 && max_len * units < 256 * 256 ? 128 : 256;
  int64_t chunk = (max_len * units / target + 127) / 128 * 128;
  if (chunk < least) chunk = least;
  p->chunk = (int)chunk;
  p->chunks = max_len <= chunk ? 1 : (int)((max_len + chunk - 1) / chunk);
  p->raw_ld = (int)((max_len + 31) / 32 * 32);
  const int64_t kv = batch * kv_heads;
  p->ml_bytes = align_up((size_t)(kv * p->chunks * rows) * sizeof(float2), 256);
  p->o_bytes = p->chunks > 1 ? align_up((size_t)(kv * p->chunks * rows) * dim * 4, 256) : 0;
  p->raw_bytes = with_scores ? align_up((size_t)(kv * rows) * p->raw_ld * 4, 256) : 0;
  if (p->chunks == 1 && !with_scores) p->ml_bytes = 0;
}

template <bool F32, int DP, int MT, bool MANY, int WAVES = kWavesHeld<F32, DP, MT, MANY>>
static int launch_decode_mt(const AttnArgs& a, const AttnPlan& p, int64_t units, hipStream_t s) {
  if constexpr (F32 && WAVES == 3)
    if (units * p.row_groups * p.chunks <= kTwoWavesUpTo) return launch_decode_mt<F32, DP, MT, MANY, 2>(a, p, units, s);
  const int bytes = (kAttnWaves * 16 * (DP + 4) + (kAttnWaves + 1) * 32) * 4 + MT * Tile<F32, DP>::kKeyVecs * kWave * 16 +
                    (MANY ? kAttnWaves * 16 * Tile<F32, DP>::kTokens * 4 : 0);
  if (bytes > 65536) {
    const hipError_t e = set_dynamic_lds_limit((const void*)kv_decode_kernel<F32, DP, MT, MANY, WAVES>, bytes, s);
    if (e != hipSuccess) {
      set_error("kv_decode: %s", hipGetErrorString(e));
      return kHipError;
    }
  }
  kv_decode_kernel<F32, DP, MT, MANY, WAVES>
      <<<dim3((unsigned)(units * p.row_groups), (unsigned)p.chunks), kAttnThreads, bytes, s>>>(a);
  return launch_status("kv_decode");
}

template <bool F32, int DP>
static int launch_decode(const AttnArgs& a, const AttnPlan& p, int64_t units, hipStream_t s) {
  if constexpr (F32 || DP <= 128) {
    if (p.mt == 2)
      return a.queries > 1 ? launch_decode_mt<F32, DP, 2, true>(a, p, units, s)
                           : launch_decode_mt<F32, DP, 2, false>(a, p, units, s);
  }
  return a.queries > 1 ? launch_decode_mt<F32, DP, 1, true>(a, p, units, s)
                       : launch_decode_mt<F32, DP, 1, false>(a, p, units, s);
}

}  // namespace tx

using namespace tx;

extern "C" {

size_t tallax_kv_decode_workspace_size(const tallax_kv_cache* cache, int64_t queries, int64_t heads, int64_t max_len,
                                       int with_scores) {
  KvView v;
  if (make_kv_view(cache, "kv_decode", &v) != kOk || queries < 1 || heads < 1 || heads % cache->kv_heads) return 0;
  if (max_len > v.capacity || max_len < 0) max_len = v.capacity;
  AttnPlan p;
  plan_attention(cache->batch, cache->kv_heads, queries * (heads / cache->kv_heads), v.dim, cache->dtype, max_len,
                 with_scores != 0, &p);
  return p.ml_bytes + p.o_bytes + p.raw_bytes;
}

int tallax_kv_decode(const tallax_kv_cache* cache, const void* q, int64_t q_stride_batch, int64_t q_stride_query,
                     int64_t q_stride_head, int64_t queries, int64_t heads, double scale, const int32_t* lens,
                     const int32_t* counts, int64_t max_len, const float* scores, void* out, float* out_lse,
                     float* out_scores, void* workspace, size_t workspace_bytes, tallax_stream_t stream) {
  AttnArgs a;
  int st = make_kv_view(cache, "kv_decode", &a.c);
  if (st != kOk) return st;
  if (queries < 1 || queries > 1024 || heads < 1 || heads % cache->kv_heads) {
    set_error("kv_decode: %lld queries (1 to 1024), %lld heads over %lld kv heads (a multiple)", (long long)queries,
              (long long)heads, (long long)cache->kv_heads);
    return kInvalidArgument;
  }
  const int64_t group = heads / cache->kv_heads, rows = queries * group;
  if (rows > 4096) {
    set_error("kv_decode: %lld queries x %lld heads of a kv head: at most 4096 rows", (long long)queries,
              (long long)group);
    return kUnsupported;
  }
  if (!(scale == scale) || scale - scale != 0.0) {
    set_error("kv_decode: scale must be finite");
    return kInvalidArgument;
  }
  if (cache->batch == 0) return kOk;
  if (!q || !lens || !out || (!scores != !out_scores)) {
    set_error("kv_decode: null pointer, or scores without out_scores");
    return kInvalidArgument;
  }
  const int64_t es = cache->dtype == TALLAX_F32 ? 4 : 2;
  if (((uintptr_t)q | (uintptr_t)out) & 15 || q_stride_batch * es % 16 || q_stride_query * es % 16 ||
      q_stride_head * es % 16 || q_stride_batch < 0 || q_stride_query < 0 || q_stride_head < 0) {
    set_error("kv_decode: q, its strides and out must be multiples of 16 bytes");
    return kUnsupported;
  }
  if (max_len < 0 || max_len > a.c.capacity) {
    set_error("kv_decode: max_len %lld must be in [0, %d], the slots of a table row", (long long)max_len,
              a.c.capacity);
    return kInvalidArgument;
  }
  AttnPlan p;
  plan_attention(cache->batch, cache->kv_heads, rows, a.c.dim, cache->dtype, max_len, scores != nullptr, &p);
  st = check_workspace("kv_decode", workspace, workspace_bytes, p.ml_bytes + p.o_bytes + p.raw_bytes);
  if (st != kOk) return st;
  a.q = (const char*)q;
  a.q_batch = q_stride_batch * es;
  a.q_query = q_stride_query * es;
  a.q_head = q_stride_head * es;
  a.lens = lens;
  a.counts = counts;
  a.out = (char*)out;
  a.lse = out_lse;
  a.queries = (int)queries;
  a.heads = (int)heads;
  a.kv_heads = (int)cache->kv_heads;
  a.group = (int)group;
  a.rows = p.rows;
  a.max_len = p.max_len;
  a.chunk = p.chunk;
  a.chunks = p.chunks;
  a.row_groups = p.row_groups;
  a.scale2 = (float)(scale * 1.4426950408889634);
  char* ws = (char*)workspace;
  a.part_ml = (float2*)ws;
  a.part_o = (float*)(ws + p.ml_bytes);
  a.raw = scores ? (float*)(ws + p.ml_bytes + p.o_bytes) : nullptr;
  a.raw_ld = p.raw_ld;
  a.scores = scores;
  a.out_scores = out_scores;
  a.vector_scores = scores && a.c.capacity % 4 == 0 && !(((uintptr_t)scores | (uintptr_t)out_scores) & 15);
  uint64_t bits = 1 << 20;  // offsets in units of the largest power of two that the strides share
  for (int64_t x : {a.c.k_page, a.c.k_slot, a.c.v_page, a.c.v_slot}) bits |= (uint64_t)x;
  a.shift = __builtin_ctzll(bits);
  const uint64_t far_page = cache->pages > 0 ? cache->pages - 1 : 0, far_slot = cache->page_size - 1;
  if ((far_page * a.c.k_page + far_slot * a.c.k_slot) >> a.shift >> 32 ||
      (far_page * a.c.v_page + far_slot * a.c.v_slot) >> a.shift >> 32) {
    set_error("kv_decode: a pool may span up to 2^32 times the largest power of two that divides its strides (%d bytes)",
              1 << a.shift);
    return kUnsupported;
  }
  a.k_page = (uint32_t)(a.c.k_page >> a.shift);
  a.k_slot = (uint32_t)(a.c.k_slot >> a.shift);
  a.v_page = (uint32_t)(a.c.v_page >> a.shift);
  a.v_slot = (uint32_t)(a.c.v_slot >> a.shift);
  const int64_t units = cache->batch * cache->kv_heads;
  if (units * p.row_groups > INT32_MAX || p.chunks > 65535) {
    set_error("kv_decode: too many workgroups");
    return kUnsupported;
  }
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = cache->dtype == TALLAX_F32;
  if (a.c.dim <= 64)
    st = f32 ? launch_decode<true, 64>(a, p, units, s) : launch_decode<false, 64>(a, p, units, s);
  else if (a.c.dim <= 128)
    st = f32 ? launch_decode<true, 128>(a, p, units, s) : launch_decode<false, 128>(a, p, units, s);
  else
    st = f32 ? launch_decode<true, 256>(a, p, units, s) : launch_decode<false, 256>(a, p, units, s);
  if (st != kOk) return st;
  const int out_blocks = p.chunks > 1 ? p.rows : 0;
  const int blocks = out_blocks + (scores ? (a.c.capacity + 1023) / 1024 : 0);
  if (blocks == 0) return kOk;
  const size_t lds = (size_t)p.rows * 8 > 4096 ? (size_t)p.rows * 8 : 4096;
  kv_decode_join_kernel<<<dim3((unsigned)units, (unsigned)blocks), 256, lds, s>>>(a, f32, out_blocks);
  return launch_status("kv_decode");
}

}  // extern "C"
