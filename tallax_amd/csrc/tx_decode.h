// The attention of a few rows over a chunk of a list of slots, by one workgroup
// of four waves: up to 16 * MT rows (queries of a kv head), of which a wave takes
// every fourth tile of the chunk and keeps its own running maximum, sum and
// output, joined in LDS at the chunk's end.
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
#pragma once
#include "tx_attention.h"

namespace tx {

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = 4;

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
template <bool F32, class Rows>
__device__ __forceinline__ void add_strange(const AttnArgs& a, const Rows& rows, const char* vbase, uint32_t v_at,
                                            uint64_t gone, int t0, int from, int to, int row0, float* outs, int ld,
                                            const float* weights) {
#pragma unroll 1
  for (int in = from; in < to; ++in) {
    const char* p = vbase + ((uint64_t)from_lane(v_at, in) << a.at.shift);
    if ((gone >> in) & 1) continue;
#pragma unroll 1
    for (int d = lane_id(); d < a.c.dim; d += kWave) {
      const float v = F32 ? ((const float*)p)[d] : __uint_as_float((uint32_t)((const uint16_t*)p)[d] << 16);
      if ((__float_as_uint(v) & 0x7f800000u) != 0x7f800000u) continue;
#pragma unroll 1
      for (int r = 0; r < 16 && row0 + r < rows.count(); ++r)
        if (t0 + in < rows.limit(row0 + r)) outs[r * ld + d] += weights[in * 16 + r] * v;
    }
  }
}

// A sequence's own slots, as its queries' rows see them.
struct OwnRows {
  static constexpr bool kOutputs = true;  // one chunk's results are the outputs themselves
  const AttnArgs& a;
  int unit, b, kvh;
  Seen seen;
  __device__ __forceinline__ OwnRows(const AttnArgs& args, int u)
      : a(args), unit(u), b(u / args.kv_heads), kvh(u - u / args.kv_heads * args.kv_heads), seen(args, u / args.kv_heads) {}
  __device__ __forceinline__ int count() const { return a.rows; }
  __device__ __forceinline__ int len() const { return seen.len; }
  __device__ __forceinline__ int chunk() const { return a.chunk; }
  __device__ __forceinline__ bool parts() const { return a.chunks > 1; }
  __device__ __forceinline__ int limit(int row) const { return seen.limit(row / a.group); }
  __device__ __forceinline__ int open() const { return seen.first; }
  __device__ __forceinline__ const int32_t* table() const { return a.c.table + (int64_t)b * a.c.width; }
  // where token t of the list lies: in which table's row (of the one above, or another), and in which slot of it
  __device__ __forceinline__ const int32_t* table_of(const int32_t* own, int) const { return own; }
  __device__ __forceinline__ int slot_of(int t) const { return t; }
  __device__ __forceinline__ const char* query(int row) const {
    const int t = row / a.group;
    return a.q + b * a.q_batch + t * a.q_query + (int64_t)(kvh * a.group + row - t * a.group) * a.q_head;
  }
  __device__ __forceinline__ int64_t output(int row) const {
    const int t = row / a.group;
    return ((int64_t)b * a.queries + t) * a.heads + kvh * a.group + (row - t * a.group);
  }
  // what belongs to an output beside these slots: elements d .. d + 3, maximum and sum of a row
  __device__ __forceinline__ void merge(int, int, float4&, float&, float&) const {}
  __device__ __forceinline__ int64_t part(int c) const { return ((int64_t)unit * a.chunks + c) * a.rows; }
  __device__ __forceinline__ float2* part_ml() const { return a.part_ml; }
  __device__ __forceinline__ float* part_o() const { return a.part_o; }
};

template <bool F32, int DP, int MT, bool MANY>
constexpr int decode_lds_bytes() {
  return (kAttnWaves * 16 * (DP + 4) + (kAttnWaves + 1) * 32) * 4 + MT * Tile<F32, DP>::kKeyVecs * kWave * 16 +
         (MANY ? kAttnWaves * 16 * Tile<F32, DP>::kTokens * 4 : 0);
}

// Rows 16 MT rg and on, over chunk number `chunk`.  MANY: some rows may not see
// the newest tokens.  lds: [kAttnWaves][16][DP + 4], m and l of the waves, the
// queries, weights.
template <bool F32, int DP, int MT, bool MANY, class Rows>
__device__ __forceinline__ void decode_chunk(const AttnArgs& a, const Rows& rows, int rg, int chunk, float* lds) {
  using T = Tile<F32, DP>;
  constexpr int ES = F32 ? 4 : 2;
  constexpr int STEP = kAttnWaves * T::kTokens;
  uint4* queries = (uint4*)(lds + kAttnWaves * 16 * (DP + 4) + (kAttnWaves + 1) * 32);  // [MT][kKeyVecs][64]

  const int wave = threadIdx.x / kWave, lane = lane_id(), n = lane & 15, g = lane >> 4;
  const int start = chunk * rows.chunk();
  if (start >= rows.len() && rows.parts()) return;
  const int end = min(start + rows.chunk(), rows.len());
  const int row0 = rg * 16 * MT;

  const char* kbase = a.c.k + rows.kvh * a.c.k_head;
  const char* vbase = a.c.v + rows.kvh * a.c.v_head;
  const int32_t* table = rows.table();
  const int mine = lane & (T::kTokens - 1);
  auto page_at = [&](int t0) {
    const int t = t0 + mine;
    return t < end ? page_id(a.c, rows.table_of(table, t), rows.slot_of(t)) : -1;
  };
  int t0 = start + wave * T::kTokens;
  // Each lane works out the place of one token and hands it to those that load
  // from it.  Tokens past the end or in no page are read from a query.
  const char* safe = rows.query(0);
  struct Places {
    int page;
    uint32_t k, v;
  };
  auto places_of = [&](int t, int page) {
    const int slot = rows.slot_of(t + mine), off = slot - (int)page_of(a.c.div, (uint32_t)slot) * a.c.div.size;
    return Places{page, (uint32_t)page * a.at.k_page + (uint32_t)off * a.at.k_slot,
                  (uint32_t)page * a.at.v_page + (uint32_t)off * a.at.v_slot};
  };
  Keys<F32, DP> key;
  auto load_keys = [&](const Places& pl) {
#pragma unroll
    for (int u = 0; u < T::kParts; ++u) {
      const char* p = kbase + ((uint64_t)from_lane(pl.k, 16 * u + n) << a.at.shift);
      load_key<F32, DP>(key[u], (int)from_lane((uint32_t)pl.page, 16 * u + n) >= 0 ? p : safe, g, a.c.dim);
    }
  };
  Places next = places_of(t0, page_at(t0));
  load_keys(next);
  int next_page = page_at(t0 + STEP);

  for (int i = threadIdx.x; i < MT * T::kKeyVecs * kWave; i += kAttnThreads) {
    const int l = i % kWave, v = i / kWave % T::kKeyVecs, mt = i / (kWave * T::kKeyVecs);
    const int row = row0 + 16 * mt + (l & 15);
    const int d = F32 ? 16 * v + 4 * (l >> 4) : 32 * v + 8 * (l >> 4);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row < rows.count() && d < a.c.dim) x = *(const uint4*)(rows.query(row) + d * ES);
    queries[i] = x;
  }
  f32x4 acc[MT][T::kAcc];
  float wm[MT], wl[MT];
  int limit[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + n;
    limit[mt] = row < rows.count() ? rows.limit(row) : 0;
    wm[mt] = -INFINITY;
    wl[mt] = 0.0f;
#pragma unroll
    for (int j = 0; j < T::kAcc; ++j) acc[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // below this every row of a query that counts sees every slot
  const int open = min(rows.open(), end);
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
      const char* p = vbase + ((uint64_t)from_lane(v_at, in) << a.at.shift);
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
      if (Rows::kOutputs && a.raw) {
        const int row = row0 + 16 * mt + n;
        if (limit[mt] > 0) {
          float* rp = a.raw + ((int64_t)rows.unit * a.rows + row) * a.raw_ld + t0 + 4 * g;
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
          add_strange<F32>(a, rows, vbase, v_at, gone, t0, max(open - t0, 0), T::kTokens, row0 + 16 * mt, outs, DP + 4,
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
    if (row0 + 16 * mt + n < rows.count()) {
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
      if (row >= rows.count() || d >= a.c.dim) continue;
      if (rows.parts() && rows.limit(row) <= 0) continue;  // nor does the second kernel read it
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kAttnWaves; ++k) {
        const float4 x = *(const float4*)(lds + (k * 16 + rn) * (DP + 4) + d);
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      float rm = ml[kAttnWaves * 32 + 2 * rn], rl = ml[kAttnWaves * 32 + 2 * rn + 1];
      if (rows.parts()) {
        const int64_t at = rows.part(chunk) + row;
        *(float4*)(rows.part_o() + at * a.c.dim + d) = o;
        if (d == 0) rows.part_ml()[at] = make_float2(rm, rl);
      } else if constexpr (Rows::kOutputs) {
        rows.merge(row, d, o, rm, rl);
        const float inv = rl == 0.0f ? 0.0f : 1.0f / rl;
        const int64_t head = rows.output(row);
        const bool none = rl == 0.0f;
        o.x = none ? 0.f : o.x * inv, o.y = none ? 0.f : o.y * inv, o.z = none ? 0.f : o.z * inv,
        o.w = none ? 0.f : o.w * inv;
        if constexpr (F32)
          *(float4*)(a.out + (head * a.c.dim + d) * 4) = o;
        else
          *(uint2*)(a.out + (head * a.c.dim + d) * 2) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
        if (d == 0) {
          if (a.lse) a.lse[head] = none ? -INFINITY : (rm + __builtin_amdgcn_logf(rl)) * kLn2;
          if (a.raw) a.part_ml[(int64_t)rows.unit * a.rows + row] = make_float2(rm, rl);
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace tx
