// Attention of the newest tokens of sequences that begin with a shared prefix:
// x = scale q.k over the prefix's slots and the sequence's own, w = exp(x - lse),
// out = sum w v.  A chunk of either gives its rows' maximum m, l = sum 2^(x - m)
// and sum 2^(x - m) v (x in base 2); two of them join as m = max, l = l1 2^(m1 - m)
// + l2 2^(m2 - m), and so the outputs.
//
// The prefix's slots are taken for all its sequences at once: the rows of a kv
// head (sequence, query and head of the group, in this order) are the columns
// of two matrix products,
//   S^T = K Q^T   (tokens x rows),   O^T = V^T P^T   (dim x rows).
// Short prefixes are read by each sequence (kv_shared_whole_kernel): one launch.
// Up to 32 rows (16 in bfloat16 above dim 128): kv_shared_rows_kernel, by the
// products of tx_decode.h.  More: kv_shared_tiles_kernel, of which a workgroup
// computes 32 * RG rows over a chunk of the prefix.  The sequences' own slots are
// always tx_decode.h's: in the same launch (kv_shared_rows_kernel,
// kv_shared_both_kernel), or after the prefix's (kv_shared_last_kernel, which makes
// the outputs, and kv_decode_kernel); plan_shared has the rules.  Where nothing
// else does, kv_shared_join_kernel makes the outputs.
//
// A workgroup of tiles has RG * TG waves: wave (rg, tg) takes 32 rows and every
// TG-th tile of WT tokens, which its RG waves bring into LDS together, through
// registers and one tile ahead.  In S^T a lane holds one row's scores, so that
// weights are the second operand of the second product as they lie; its first
// operand, values by dim, is read transposed from LDS (bfloat16), or in single
// elements (float32).
//
// Up to some 100 rows the bytes bound it, beyond that the products, whose weights
// take as many cycles of the vector units (an exponential of 16, and some eight
// operations of 4, to each 64 scores): 20 rows of each of 128 sequences behind 4099
// slots of 8 heads of 128, 43 GFLOP, 72 us in the tiles, 600 TFLOP/s, the matrix
// units busy a quarter of the cycles; 16 x 64 / 8 heads behind 131071 slots with up
// to 300 of their own, 69 GFLOP and 550 MB, 114 us and 10.5 in the join (reading
// alone 115); 64 x 32 / 8 heads behind 8192 with up to 1024, 203 MB, 51 and 10.5;
// float32, 3 x 12 heads of 80 behind three times 2050 slots with up to 333, 18 and 5.
#include "tallax_hip_testing.h"
#include "tx_decode.h"

namespace tx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct SharedArgs {
  AttnArgs own;
  const int32_t* table;  // [prefixes, width]
  const int32_t* lens;   // [prefixes]
  int width, max_len;
  int per;               // sequences of a prefix
  int rows;              // of a prefix's kv head
  int row_tiles, chunk, chunks;
  int pieces;            // chunks of all kv heads of all prefixes
  int own_units;         // workgroups of a chunk of the sequences' own slots
  int own_from;          // the first of them, where the prefix's are tiles
  uint32_t flip;         // sign bits of q, where the scale is negative
  float scale2;          // its size, above 0: -inf, of what is not seen, stays -inf
  float2* part_ml;       // [prefixes * kv_heads][chunks][rows]: maximum (base 2), sum
  float* part_o;         // [prefixes * kv_heads][chunks][rows][dim]
};

// Places of 16-byte vectors in a tile: vector c of a token's row is stored at
// c ^ swizzle(token), so that the lanes of a read, which take the same vectors
// of neighbouring tokens, meet different banks.  A swizzle is made of single
// bits of the token, so that it may be taken of parts of a token's number.
template <int VECS>
__host__ __device__ constexpr int key_swizzle(int token) {
  return VECS >= 16 ? token & 15 : (token >> 1) & 7;
}

template <bool F32, int VECS>
__host__ __device__ constexpr int value_swizzle(int token) {
  return F32 ? 8 * ((token >> 2) & 1) : VECS >= 16 ? 4 * (token & 3) : 4 * ((token >> 1) & 1);
}

typedef __attribute__((address_space(3))) char lds_char;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(lds_char*)at;
}

template <bool F32, int DP, int RG, int TG, int WT>
struct Prefix {
  static constexpr int ES = F32 ? 4 : 2, NW = RG * TG, kThreads = NW * kWave;
  static constexpr int VECS = DP * ES / 16;               // 16-byte vectors of a token's key
  static constexpr int ROW = VECS * 16;
  static constexpr int LOADS = WT * VECS / (kWave * RG);  // of a tile's keys, per lane
  static constexpr int TPL = kWave / VECS;                // tokens of a load
  static constexpr int QV = VECS / 2;                     // of a row's query, per lane
  static constexpr int NB = WT / 32, ACC = DP / 32, STEP = TG * WT, PAD = 36;
  static constexpr int kTile = 2 * WT * ROW;  // bytes of a tile: keys, then values
  static constexpr int kRoom = 2 * TG * kTile, kJoin = NW * 32 * (8 + PAD * 4);
  static constexpr int kBytes = kRoom > kJoin ? kRoom : kJoin;
  static_assert(kBytes <= 160 * 1024, "LDS");
  static_assert(VECS <= kWave && LOADS >= 1, "whole tokens in a load");

  const SharedArgs& a;
  int lane, n, h, end;
  int source;           // lane that works out the place of this lane's token of a tile's first load
  const char *kbase, *vbase;  // with this lane's vector of a token
  const int32_t* table;
  uint4 q[QV];
  uint4 staged[2 * LOADS];  // of a tile on its way to LDS: keys and values in turn
  f32x16 acc[ACC];
  float m, l;  // of q.k, which times scale2 is the exponent of a weight

  __device__ __forceinline__ explicit Prefix(const SharedArgs& args) : a(args) {}

  // The table's entry of this lane's token of the tile at t0.
  __device__ __forceinline__ int entry_at(int t0) const {
    return table[page_of(a.own.c.div, (uint32_t)min(t0 + (lane & (WT - 1)), end - 1))];
  }

  // Where a tile's tokens lie: each lane works out the place of one token and
  // hands it to those that load from it.  Tokens that are not there are read
  // from the pool's first slot, and cleared on the way to LDS.
  struct Places {
    uint32_t k, v;
    uint64_t gone;
  };
  __device__ __forceinline__ Places places_of(int t0, int entry) const {
    const AttnArgs& o = a.own;
    const int t = t0 + (lane & (WT - 1));
    const bool there = (t < end) & ((uint32_t)entry < (uint32_t)o.c.pages);
    const uint32_t off = (uint32_t)t - page_of(o.c.div, (uint32_t)t) * (uint32_t)o.c.div.size;
    return Places{there ? (uint32_t)entry * o.at.k_page + off * o.at.k_slot : 0u,
                  there ? (uint32_t)entry * o.at.v_page + off * o.at.v_slot : 0u, __ballot(!there)};
  }

  __device__ __forceinline__ uint32_t place(int i, const Places& at) const {
    return from_lane(i & 1 ? at.v : at.k, source + i / 2 * TPL);
  }

  __device__ __forceinline__ void load(int i, uint32_t place) {
    staged[i] = *(const uint4*)((i & 1 ? vbase : kbase) + ((uint64_t)place << a.own.at.shift));
  }

  // to: this lane's place of the first load in the tile's keys, or values.  What is not there must not be infinite or NaN
  // in values, where its weight is 0, nor in what queries do not have; scores of tokens that are not there are masked.
  __device__ __forceinline__ void store(int i, uint64_t gone, uint32_t to) const {
    const int j = i / 2;
    uint4 x = staged[i];
    if (((i & 1) && gone != 0) || DP != a.own.c.dim) {
      const int c = lane % VECS;
      if (((gone >> (source + j * TPL)) & 1) || c * 16 >= a.own.c.dim * ES) x = make_uint4(0, 0, 0, 0);
    }
    const int turn = i & 1 ? value_swizzle<F32, VECS>(j * TPL) : key_swizzle<VECS>(j * TPL);
    *(__attribute__((address_space(3))) u32x4*)(lds_char*)((to ^ (turn << 4)) + j * TPL * ROW) = __builtin_bit_cast(u32x4, x);
  }

  // One tile's keys and values into this wave's rows.  Meanwhile the next tile
  // goes from registers to LDS and the one after it is asked for, a vector at a
  // time between the products: loads that are asked for all at once hold a wave
  // up until the memory has taken them.
  // keys, values: this lane's first places in the tile that is read; next_k, next_v: in the one that is written
  __device__ __forceinline__ void round(uint32_t keys, uint32_t values, uint32_t next_k, uint32_t next_v, uint64_t gone,
                                        uint64_t next_gone, const Places& after) {
    f32x16 s[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
    // Vectors are read a group of products ahead: a read's way through LDS takes longer than a product.
    constexpr int GROUP = 4 / NB < QV ? 4 / NB : QV;
    constexpr int JG = ACC < 4 ? ACC : 4, STEPS = F32 ? 4 * NB : 2 * NB * (ACC / JG), SLOTS = QV / GROUP + STEPS;
    // A place is handed over in the slot before its load: it comes through LDS, behind the reads that were made before.
    constexpr int EACH = (2 * LOADS + SLOTS - 1) / SLOTS;
    uint32_t places[2][EACH];
    auto hand_over = [&](int slot) {
#pragma unroll
      for (int i = 0; i < 2 * LOADS; ++i)
        if (i / EACH == slot) places[slot & 1][i % EACH] = place(i, after);
    };
    auto pass_on = [&](int slot) {
#pragma unroll
      for (int i = 0; i < 2 * LOADS; ++i) {
        if (i / EACH != slot) continue;
        store(i, next_gone, i & 1 ? next_v : next_k);
        load(i, places[slot & 1][i % EACH]);
      }
    };
    hand_over(0);
    uint4 kv[2][GROUP][NB];
    // float32: products of elements past dim, all zeros, are left out in blocks, where the instance has such.  64
    // sequences x 4 rows of dim 80 behind 8192 slots 53 us, with them 60; in bfloat16 they cost nothing (25.5, 25.6).
    const int dim = a.own.c.dim;
    constexpr int SPAN = GROUP * 32 / ES;  // elements of a group of the first product
    auto in_keys = [&](int g) { return !F32 || g * SPAN <= DP / 2 || g * SPAN < dim; };
    auto in_values = [&](int j) { return !F32 || 32 * j <= DP / 2 || 32 * j < dim; };
    auto read_keys = [&](int g) {
      if (!in_keys(g)) return;
#pragma unroll
      for (int i = 0; i < GROUP; ++i)
#pragma unroll
        for (int u = 0; u < NB; ++u)
          kv[g & 1][i][u] = __builtin_bit_cast(uint4, lds_read<u32x4>((keys ^ (2 * (g * GROUP + i) << 4)) + 32 * u * ROW));
    };
    read_keys(0);
#pragma unroll
    for (int g = 0; g < QV / GROUP; ++g) {
      hand_over(g + 1);
      if (g + 1 < QV / GROUP) read_keys(g + 1);
      pass_on(g);
      __builtin_amdgcn_sched_barrier(0);
      if (!in_keys(g)) continue;
#pragma unroll
      for (int i = 0; i < GROUP; ++i)
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const uint4 k = kv[g & 1][i][u], x = q[g * GROUP + i];
          if constexpr (F32) {
            s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.x), __uint_as_float(x.x), s[u], 0, 0, 0);
            s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.y), __uint_as_float(x.y), s[u], 0, 0, 0);
            s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.z), __uint_as_float(x.z), s[u], 0, 0, 0);
            s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.w), __uint_as_float(x.w), s[u], 0, 0, 0);
          } else {
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                           __builtin_bit_cast(bf16x8_t, x), s[u], 0, 0, 0);
          }
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    // lane (n, h) holds row n's scores of tokens 32 u + 8 (r / 4) + 4 h + r % 4
    if (gone != 0) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const uint32_t here = (uint32_t)(gone >> (32 * u)) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = (here >> (8 * (r / 4) + r % 4)) & 1 ? -INFINITY : s[u][r];
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    top = fmaxf(top, lane_xor_f(top, 32));
    const float next = fmaxf(m, top);
    const float base = next == -INFINITY ? 0.0f : next * a.scale2;  // nothing seen yet: every weight is exp2(-inf) = 0
    if (__ballot(next > m)) {  // seldom, after the first tiles
      const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m * a.scale2 - base);
      m = next;
      l *= shrink;
#pragma unroll
      for (int j = 0; j < ACC; ++j) acc[j] *= shrink;
    }
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], a.scale2, -base));
        sum += s[u][r];
      }
    l += sum;
    if constexpr (F32) {
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (r % 4 == 0) {
            hand_over(QV / GROUP + 4 * u + r / 4 + 1);
            pass_on(QV / GROUP + 4 * u + r / 4);
          }
#pragma unroll
          for (int j = 0; j < ACC; ++j)
            if (in_values(j)) acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                lds_read<float>((values ^ (8 * j << 4)) + (32 * u + 8 * (r / 4) + r % 4) * ROW), s[u][r], acc[j], 0, 0, 0);
        }
    } else {
      // The product takes both sides in bfloat16: the weights, at most 1, are rounded to it (by 2^-8 of each at most);
      // their sum, by which the output is divided, is of the unrounded ones.
      uint2 vv[2][JG][2];
      auto read_values = [&](int i) {  // of 16 tokens and 32 JG elements
        typedef __attribute__((address_space(3))) bf16x4 lds_x4;
        // 16 lanes read 16 neighbouring elements of four tokens, and get four tokens of one element each
#pragma unroll
        for (int j = 0; j < JG; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            vv[i & 1][j][half] = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (lds_x4*)(lds_char*)((values ^ (4 * (i % (ACC / JG) * JG + j) << 4)) +
                                                (16 * (i / (ACC / JG)) + 8 * half) * ROW)));
      };
      read_values(0);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        hand_over(QV / GROUP + i + 1);
        if (i + 1 < STEPS) read_values(i + 1);
        pass_on(QV / GROUP + i);
        const int u = i / (ACC / JG) / 2, r = 8 * (i / (ACC / JG) % 2);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = pack_bf16(s[u][r + 2 * k], s[u][r + 2 * k + 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < JG; ++j) {
          f32x16& to = acc[i % (ACC / JG) * JG + j];
          to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8_t, make_uint4(vv[i & 1][j][0].x, vv[i & 1][j][0].y, vv[i & 1][j][1].x, vv[i & 1][j][1].y)),
              __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3])), to, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// Rows 32 RG times the tile's number and on of a prefix's kv head, over one chunk: workgroup f of those for prefixes.
template <bool F32, int DP, int RG, int TG, int WT>
__device__ __forceinline__ void prefix_chunk(const SharedArgs& a, int f, uint4* tiles) {
  using P = Prefix<F32, DP, RG, TG, WT>;
  constexpr int NW = P::NW, PAD = P::PAD, STEP = P::STEP;

  // The row tiles of a piece (chunk of a prefix's kv head) are workgroups of one XCD, that follow one another: their
  // numbers are the same modulo 8.
  const int step = f >> 3, piece = (step / a.row_tiles) * 8 + (f & 7);
  if (piece >= a.pieces) return;
  const int unit = piece / a.chunks, chunk = piece - unit * a.chunks;
  const AttnArgs& o = a.own;
  const int p = unit / o.kv_heads, kvh = unit - p * o.kv_heads;
  const int len = min(max(a.lens[p], 0), a.max_len);
  const int start = chunk * a.chunk;
  if (start >= len) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), tg = wave / RG;
  P w(a);
  const int rg = wave % RG;
  w.lane = lane_id();
  w.n = w.lane & 31;
  w.h = w.lane >> 5;
  w.end = min(start + a.chunk, len);
  w.source = rg * P::LOADS * P::TPL + w.lane / P::VECS;
  const int c0 = w.lane % P::VECS, c = c0 * 16 < o.c.dim * P::ES ? c0 : 0;  // vectors past dim are cleared too
  w.kbase = o.c.k + kvh * o.c.k_head + c * 16;
  w.vbase = o.c.v + kvh * o.c.v_head + c * 16;
  w.table = a.table + (int64_t)p * a.width;
  const int n = w.n, h = w.h, row0 = (step % a.row_tiles) * 32 * RG + rg * 32;

  // this lane's first places in the first of two tiles; the other is TG * kTile away
  const uint32_t keys = (uint32_t)(uintptr_t)(lds_char*)(char*)tiles + tg * P::kTile, values = keys + WT * P::ROW;
  const uint32_t put_k = keys + w.source * P::ROW + ((c0 ^ key_swizzle<P::VECS>(w.source)) << 4);
  const uint32_t put_v = values + w.source * P::ROW + ((c0 ^ value_swizzle<F32, P::VECS>(w.source)) << 4);
  const uint32_t get_k = keys + n * P::ROW + ((h ^ key_swizzle<P::VECS>(n)) << 4);
  // bfloat16: token 4 h + (lane % 16) / 4, 8 bytes of its elements each; float32: token 4 h, an element each
  const int first = F32 ? 4 * h : 4 * h + (w.lane & 15) / 4;
  const int vec = F32 ? n / 4 : 2 * ((w.lane >> 4) & 1) + (w.lane & 3) / 2;
  const uint32_t get_v = values + first * P::ROW + ((vec ^ value_swizzle<F32, P::VECS>(first)) << 4) +
                         (F32 ? n % 4 * 4 : (w.lane & 1) * 8);

  int t0 = start + tg * WT;
  typename P::Places at = w.places_of(t0, w.entry_at(t0));
#pragma unroll
  for (int i = 0; i < 2 * P::LOADS; ++i) w.load(i, w.place(i, at));
  int entry = w.entry_at(t0 + STEP);
  {
    const int row = row0 + n, seq = row / o.rows, rr = row - seq * o.rows, t = rr / o.group;
    const char* at = o.q + (int64_t)(p * a.per + seq) * o.q_batch + t * o.q_query +
                     (int64_t)(kvh * o.group + rr - t * o.group) * o.q_head;
#pragma unroll
    for (int i = 0; i < P::QV; ++i) {
      const int c = 2 * i + h;
      w.q[i] = make_uint4(0, 0, 0, 0);
      if (row < a.rows && c * 16 < o.c.dim * P::ES) {
        const uint4 x = *(const uint4*)(at + c * 16);
        w.q[i] = make_uint4(x.x ^ a.flip, x.y ^ a.flip, x.z ^ a.flip, x.w ^ a.flip);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < P::ACC; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) w.acc[j][r] = 0.0f;
  w.m = -INFINITY;
  w.l = 0.0f;

  const int rounds = (w.end - start + STEP - 1) / STEP;
  uint64_t gone = at.gone;
  at = w.places_of(t0 + STEP, entry);
  entry = w.entry_at(t0 + 2 * STEP);
#pragma unroll
  for (int i = 0; i < 2 * P::LOADS; ++i) {
    w.store(i, gone, i & 1 ? put_v : put_k);
    w.load(i, w.place(i, at));
  }
#pragma unroll 1
  for (int it = 0; it < rounds; ++it, t0 += STEP) {
    // One barrier a round: the tile that is written in it was read in the round before.
    lds_barrier();
    const uint64_t next_gone = at.gone;
    at = w.places_of(t0 + 2 * STEP, entry);
    entry = w.entry_at(t0 + 3 * STEP);
    const uint32_t here = (it & 1) * TG * P::kTile, there = TG * P::kTile - here;
    w.round(get_k + here, get_v + here, put_k + there, put_v + there, gone, next_gone, at);
    gone = next_gone;
  }
  f32x16(&acc)[P::ACC] = w.acc;
  const float m = w.m;
  float l = w.l;
  // join the token groups, 32 elements of the outputs at a time
  l += lane_xor_f(l, 32);
  const float m2 = m == -INFINITY ? m : m * a.scale2;
  float2* ml = (float2*)tiles;                 // [NW][32]
  float* sums = (float*)(tiles + NW * 32 / 2);  // [NW][32][PAD]
  __syncthreads();
  if (h == 0) ml[wave * 32 + n] = make_float2(m2, l);
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (int i = 0; i < TG; ++i) all = fmaxf(all, ml[(i * RG + rg) * 32 + n].x);
  const float base = all == -INFINITY ? 0.0f : all;
  const float mine = __builtin_amdgcn_exp2f(m2 - base);
  const int64_t out = ((int64_t)unit * a.chunks + chunk) * a.rows;
  if (tg == 0 && h == 0 && row0 + n < a.rows) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < TG; ++i) {
      const float2 x = ml[(i * RG + rg) * 32 + n];
      total += x.y * __builtin_amdgcn_exp2f(x.x - base);
    }
    a.part_ml[out + row0 + n] = make_float2(all, total);
  }
  const bool none = m2 == -INFINITY;
  const int row1 = (step % a.row_tiles) * 32 * RG;
#pragma unroll
  for (int j = 0; j < P::ACC; ++j) {
    float* mo = sums + (wave * 32 + n) * PAD;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4 x = make_float4(acc[j][4 * i] * mine, acc[j][4 * i + 1] * mine, acc[j][4 * i + 2] * mine,
                             acc[j][4 * i + 3] * mine);
      if (none) x = make_float4(0.f, 0.f, 0.f, 0.f);
      *(float4*)(mo + 8 * i + 4 * h) = x;
    }
    __syncthreads();
    for (int i = tid; i < RG * 32 * 8; i += P::kThreads) {
      const int row = i / 8, d = 32 * j + i % 8 * 4;
      if (row1 + row >= a.rows || d >= o.c.dim) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < TG; ++k) {
        const float4 y = *(const float4*)(sums + (k * RG * 32 + row) * PAD + i % 8 * 4);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      *(float4*)(a.part_o + (out + row1 + row) * o.c.dim + d) = x;
    }
    __syncthreads();
  }
}

// A prefix's slots, as its sequences' rows see them: all of them.
struct PrefixRows {
  static constexpr bool kOutputs = false;
  const SharedArgs& a;
  int unit, p, kvh, length;
  __device__ __forceinline__ PrefixRows(const SharedArgs& args, int u) : a(args), unit(u) {
    p = u / a.own.kv_heads;
    kvh = u - p * a.own.kv_heads;
    length = min(max(a.lens[p], 0), a.max_len);
  }
  __device__ __forceinline__ int count() const { return a.rows; }
  __device__ __forceinline__ int len() const { return length; }
  __device__ __forceinline__ int chunk() const { return a.chunk; }
  __device__ __forceinline__ bool parts() const { return true; }
  __device__ __forceinline__ int limit(int) const { return length; }
  __device__ __forceinline__ int open() const { return length; }
  __device__ __forceinline__ const int32_t* table() const { return a.table + (int64_t)p * a.width; }
  __device__ __forceinline__ const int32_t* table_of(const int32_t* own, int) const { return own; }
  __device__ __forceinline__ int slot_of(int t) const { return t; }
  __device__ __forceinline__ const char* query(int row) const {
    const AttnArgs& o = a.own;
    const int seq = row / o.rows, rr = row - seq * o.rows, t = rr / o.group;
    return o.q + (int64_t)(p * a.per + seq) * o.q_batch + t * o.q_query + (int64_t)(kvh * o.group + rr - t * o.group) * o.q_head;
  }
  __device__ __forceinline__ int64_t output(int) const { return 0; }
  __device__ __forceinline__ int64_t part(int c) const { return ((int64_t)unit * a.chunks + c) * a.rows; }
  __device__ __forceinline__ float2* part_ml() const { return a.part_ml; }
  __device__ __forceinline__ float* part_o() const { return a.part_o; }
};

// A sequence's own slots in one chunk, joined with the parts of its prefix: what comes out are the outputs.
struct LastRows : OwnRows {
  const SharedArgs& s;
  __device__ __forceinline__ LastRows(const SharedArgs& args, int u) : OwnRows(args.own, u), s(args) {}
  __device__ __forceinline__ bool parts() const { return false; }
  __device__ __forceinline__ void merge(int row, int d, float4& x, float& m, float& l) const {
    if (row / a.group >= seen.cnt) return;
    const int p = b / s.per, len = min(max(s.lens[p], 0), s.max_len), chunks = (len + s.chunk - 1) / s.chunk;
    const int64_t first = ((int64_t)(p * a.kv_heads + kvh) * s.chunks) * s.rows + (b - p * s.per) * a.rows + row;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) {
      const int64_t i = first + (int64_t)c * s.rows;
      const float2 y = s.part_ml[i];
      const float4 z = *(const float4*)(s.part_o + i * a.c.dim + d);
      const float top = fmaxf(m, y.x), base = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(y.x - base);
      m = top;
      l = l * f + y.y * g;
      x.x = x.x * f + z.x * g;
      x.y = x.y * f + z.y * g;
      x.z = x.z * f + z.z * g;
      x.w = x.w * f + z.w * g;
    }
  }
};

// A sequence's prefix and its own slots, one after the other, as its queries' rows see them.
struct WholeRows : OwnRows {
  const int32_t* front;
  int first;  // slots of the prefix
  __device__ __forceinline__ WholeRows(const SharedArgs& s, int u) : OwnRows(s.own, u) {
    const int p = b / s.per;
    front = s.table + (int64_t)p * s.width;
    first = min(max(s.lens[p], 0), s.max_len);
  }
  __device__ __forceinline__ int len() const { return first + seen.len; }
  __device__ __forceinline__ int chunk() const { return first + seen.len; }
  __device__ __forceinline__ bool parts() const { return false; }
  __device__ __forceinline__ int limit(int row) const {
    const int t = row / a.group;
    return t < seen.cnt ? first + max(seen.limit(t), 0) : 0;
  }
  __device__ __forceinline__ int open() const { return first + max(seen.first, 0); }
  __device__ __forceinline__ const int32_t* table_of(const int32_t* own, int t) const { return t < first ? front : own; }
  __device__ __forceinline__ int slot_of(int t) const { return t < first ? t : t - first; }
};

// Short prefixes and lengths: each sequence reads all of its own.
template <bool F32, int DP, int MT, bool MANY, int WAVES>
__global__ __launch_bounds__(kAttnThreads, WAVES) void kv_shared_whole_kernel(SharedArgs a) {
  extern __shared__ float lds[];
  const int rg = blockIdx.x % a.own.row_groups, unit = blockIdx.x / a.own.row_groups;
  decode_chunk<F32, DP, MT, MANY>(a.own, WholeRows(a, unit), rg, 0, lds);
}

template <bool F32, int DP, int MT, bool MANY, int WAVES>
__global__ __launch_bounds__(kAttnThreads, WAVES) void kv_shared_last_kernel(SharedArgs a) {
  extern __shared__ float lds[];
  const int rg = blockIdx.x % a.own.row_groups, unit = blockIdx.x / a.own.row_groups;
  decode_chunk<F32, DP, MT, MANY>(a.own, LastRows(a, unit), rg, 0, lds);
}

// Many rows behind a prefix.
template <bool F32, int DP, int RG, int TG, int WT, int WAVES>
__global__ __launch_bounds__(RG * TG * kWave, WAVES) void kv_shared_tiles_kernel(SharedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint4 tiles[];  // [2][TG][keys, values][WT * VECS]
  prefix_chunk<F32, DP, RG, TG, WT>(a, blockIdx.x, tiles);
}

// The same, and the sequences' own slots in the same launch.
template <bool F32, int DP, int RG, int TG, int WT, int MT, int WAVES>
__global__ __launch_bounds__(RG * TG * kWave, WAVES) void kv_shared_both_kernel(SharedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint4 tiles[];
  const int i = (int)blockIdx.x - a.own_from;
  if (i < 0) {
    prefix_chunk<F32, DP, RG, TG, WT>(a, blockIdx.x, tiles);
  } else {
    const int chunk = i / a.own_units, k = i - chunk * a.own_units, unit = k / a.own.row_groups;
    decode_chunk<F32, DP, MT, true>(a.own, OwnRows(a.own, unit), k - unit * a.own.row_groups, chunk, (float*)tiles);
  }
}

// Few rows behind a prefix, and the sequences' own slots in the same launch.
template <bool F32, int DP, int MT, bool MANY, int WAVES>
__global__ __launch_bounds__(kAttnThreads, WAVES) void kv_shared_rows_kernel(SharedArgs a) {
  extern __shared__ float lds[];
  const int i = blockIdx.x;
  if (i < a.pieces) {
    const int unit = i / a.chunks;
    decode_chunk<F32, DP, MT, false>(a.own, PrefixRows(a, unit), 0, i - unit * a.chunks, lds);
  } else {
    const int j = i - a.pieces, chunk = j / a.own_units, k = j - chunk * a.own_units, unit = k / a.own.row_groups;
    decode_chunk<F32, DP, MT, MANY>(a.own, OwnRows(a.own, unit), k - unit * a.own.row_groups, chunk, lds);
  }
}

// Joins the chunks of the prefix and of the sequence's own slots.  A row's
// parts are shared out over `split` groups of lanes, each of which holds a row.
__global__ __launch_bounds__(256) void kv_shared_join_kernel(SharedArgs a, int f32, int split, int64_t total) {
  __shared__ float4 sums[256];
  __shared__ float2 stats[256];
  const AttnArgs& o = a.own;
  const int dim = o.c.dim, width = dim <= 64 ? 16 : dim <= 128 ? 32 : 64, groups = 256 / width;
  const int group = threadIdx.x / width, l = threadIdx.x & (width - 1), d = l * 4;
  const int64_t at = (int64_t)blockIdx.x * (groups / split) + group / split;  // output row: sequence, query, head
  const int part = group % split;
  float m = -INFINITY, s = 0.0f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (at < total) {
    const int head = (int)(at % o.heads), t = (int)(at / o.heads % o.queries), b = (int)(at / o.heads / o.queries);
    const int kvh = head / o.group, own_row = t * o.group + head - kvh * o.group;
    const int p = b / a.per, row = (b - p * a.per) * o.rows + own_row;
    const Seen seen(o, b);
    const int len = min(max(a.lens[p], 0), a.max_len);
    const int front = t < seen.cnt ? (len + a.chunk - 1) / a.chunk : 0;
    const int both = front + (seen.limit(t) > 0 ? (seen.len + o.chunk - 1) / o.chunk : 0);
    const int64_t front_at = ((int64_t)p * o.kv_heads + kvh) * a.chunks * a.rows + row;
    const int64_t own_at = ((int64_t)b * o.kv_heads + kvh) * o.chunks * o.rows + own_row;
#pragma unroll 4
    for (int c = part; c < both; c += split) {
      const int64_t i = c < front ? front_at + (int64_t)c * a.rows : own_at + (int64_t)(c - front) * o.rows;
      const float2 y = c < front ? a.part_ml[i] : o.part_ml[i];
      float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d < dim) z = *(const float4*)((c < front ? a.part_o : o.part_o) + i * dim + d);
      const float top = fmaxf(m, y.x), base = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(y.x - base);
      m = top;
      s = s * f + y.y * g;
      x.x = x.x * f + z.x * g;
      x.y = x.y * f + z.y * g;
      x.z = x.z * f + z.z * g;
      x.w = x.w * f + z.w * g;
    }
  }
  if (split > 1) {
    sums[threadIdx.x] = x;
    stats[threadIdx.x] = make_float2(m, s);
    __syncthreads();
    if (part != 0) return;
    for (int k = 1; k < split; ++k) {
      const float2 y = stats[threadIdx.x + k * width];
      const float4 z = sums[threadIdx.x + k * width];
      const float top = fmaxf(m, y.x), base = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(y.x - base);
      m = top;
      s = s * f + y.y * g;
      x.x = x.x * f + z.x * g;
      x.y = x.y * f + z.y * g;
      x.z = x.z * f + z.z * g;
      x.w = x.w * f + z.w * g;
    }
  }
  if (at >= total || d >= dim) return;
  const bool none = s == 0.0f;
  const float inv = none ? 0.0f : 1.0f / s;
  x = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  if (f32)
    *(float4*)(o.out + (at * dim + d) * 4) = x;
  else
    *(uint2*)(o.out + (at * dim + d) * 2) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
  if (l == 0 && o.lse) o.lse[at] = none ? -INFINITY : (m + __builtin_amdgcn_logf(s)) * kLn2;
}

struct SharedPlan {
  int rg;  // groups of 32 rows to a workgroup; 0: few rows
  int step, row_tiles, chunk, chunks;
  AttnPlan own;
  bool whole;  // each sequence's prefix and own slots in one chunk: of the others own.mt and own.row_groups count alone
  bool both;  // tiles, and the sequences' own slots in the same launch
  bool last;  // the sequences' own slots are one chunk each, whose workgroup makes the outputs
  int own_chunks;
  size_t ml_bytes, o_bytes, own_ml_bytes, own_o_bytes;
  size_t bytes() const { return ml_bytes + o_bytes + own_ml_bytes + own_o_bytes; }
};

// Tokens of a tile.
constexpr int tile_tokens(bool f32, int dim, int rg) { return !f32 && dim <= 128 && rg == 4 ? 64 : 32; }

// Waves of a SIMD that its registers leave room for.
constexpr int tile_waves(bool f32, int dim, int rg) { return dim > 128 || (f32 && dim > 64 && rg == 2) ? 1 : 2; }

static void plan_shared(const tallax_kv_cache* c, int64_t prefixes, int64_t queries, int64_t group, int64_t max_prefix,
                        int64_t max_len, SharedPlan* p) {
  const int64_t rows = queries * group;
  const bool f32 = c->dtype == TALLAX_F32;
  const int64_t all = c->batch / prefixes * rows, units = prefixes * c->kv_heads;
  const int most = f32 || c->dim <= 128 ? 2 : 1;  // sixteens of rows that the kernel for few takes
  plan_attention(c->batch, c->kv_heads, rows, c->dim, c->dtype, max_len, false, &p->own);
  // One workgroup for a sequence's prefix and own slots, without parts and their join, takes some 5.4 us and 1 us for 100
  // slots in bfloat16 at dim 128 (0.7 at 64, 2 at 256; two to three times that in float32), and longer where there are more of
  // them than the card holds; the other ways take 10 to 11 us with few rows and 14 and more with tiles.  Sequences of 32 / 8
  // heads of 128 behind 250 slots with up to 60 of their own: 4 of them 8.6 us, else 11.4, 32 8.9 and 15.8, 128 20.4 and 25.4;
  // behind 1000 with up to 100: 4 16.4 and 10.9, 16 16.6 and 15.5; 16 in float32 behind 250 15.7 and 19.7, 500 25.4 and 20.4.
  const int64_t units_all = c->batch * c->kv_heads * p->own.row_groups;
  const double most_slots = (all <= 16 * most ? 105e3 : 210e3) / (c->dim + 64) / (f32 ? 3 : 1) / (1 + units_all / 1024.0);
  p->whole = (double)(max_prefix + max_len) <= most_slots;
  if (p->whole) {
    const AttnPlan own = p->own;
    *p = SharedPlan{};
    p->own = own;
    p->whole = true;
    return;
  }
  if (all <= 16 * most) {
    p->rg = 0;
    p->own.mt = all <= 16 ? 1 : 2;
    p->own.row_groups = 1;
    AttnPlan front;
    plan_attention(prefixes, c->kv_heads, all, c->dim, c->dtype, max_prefix, false, &front);
    p->row_tiles = 1;
    p->step = 1;
    p->chunk = front.chunk;
    p->chunks = front.chunks;
  } else {
    p->rg = all <= 64 && !(f32 && c->dim > 128) ? 2 : 4;  // float32 above dim 128 has no room for two groups' tiles
    p->step = kAttnWaves / p->rg * tile_tokens(f32, c->dim, p->rg);
    p->row_tiles = (int)((all + 32 * p->rg - 1) / (32 * p->rg));
    // Chunks: of those that make one to eight workgroups to a CU, what takes the least by these measurements (bfloat16,
    // dim 128): a workgroup alone on its CU takes 2.3 us a step, two of them 3.9, some two steps more for their beginning
    // and end; and each chunk's parts are written and read, at some 5 TB/s.  64 sequences, 32 / 8 heads, behind 8192
    // slots 31 us with 16 chunks, 33 with 32; 16 with 64 / 8 heads behind 131071 145 with 64 and 167 with 32.
    const int64_t steps = (max_prefix + p->step - 1) / p->step, pieces = units * p->row_tiles;
    const bool two = tile_waves(f32, c->dim, p->rg) == 2;
    const double dims = c->dim <= 64 ? 64 : c->dim <= 128 ? 128 : 256, tokens = tile_tokens(f32, c->dim, p->rg);
    const double step_us = (f32 ? 7.4 : 2.3) * dims / 128 * tokens / 64, part_us = (double)(units * all) * c->dim * 8 / 5e6;
    double best = 1e300;
    p->chunks = 1;
    p->chunk = (int)(steps > 0 ? steps : 1) * p->step;
    for (int k = 1; k <= 8; ++k) {
      int64_t n = 256 * k / pieces;
      n = n > steps ? steps : n;
      n = n < 1 ? 1 : n;
      const int64_t each = (steps + n - 1) / n, groups = pieces * n, room = two ? 512 : 256, rest = groups % room;
      const double turns = groups / room * (two ? 1.7 : 1.0) + (rest > 256 ? 1.7 : rest ? 1.0 : 0.0);
      const double cost = turns * (each + 2) * step_us + n * part_us;
      if (steps > 0 && cost < best) {
        best = cost;
        p->chunk = (int)(each * p->step);
        p->chunks = (int)((steps + each - 1) / each);
      }
    }
  }
  // The sequences' own slots, behind tiles.  In the same launch, where the tiles' workgroups are all on the card at once:
  // both take each other's time (32 / 8 heads of 128 behind 2048 slots, up to 512 of their own: 31 sequences 27.8 us, one
  // launch after the other 33.8; 64 behind 8192 42.9 and 45.3 in one chunk each, 128 66.4 and 75.9), but not where a
  // workgroup has a CU for itself and there is one on each (64 sequences, 4 / 2 heads of 256: 47.7 and 44.7).
  // Or each sequence in one chunk after the tiles, where there are enough of them to fill the card: their workgroups make
  // the outputs, which spares the join and their parts' way.  So where the prefix is short next to its rows (128 sequences
  // behind 512: 49.6 and 56.0), or the decode kernel needs the registers that tiles leave it less of: two sixteens of
  // rows (128 x 5 queries behind 4099: 137 and 162), float32 (50 x 8 heads, one a kv head, behind 1024: 55 and 65).
  // Both sides were measured with own slots of up to some 1000.  Longer ones that are alike in length fill the card as
  // well (32 x 5 queries, 32 / 8 heads, lengths of 65536 down to a quarter: 1182 us, where their bytes take 1151; float32,
  // one query, 16384: 828 and 578).  One long sequence among short ones is what this plan is slow for: its one chunk is what
  // the call takes (of 31 x 500 slots and one of 4096 90 us, of 16384 242, of 65536 997, where kv_decode's chunks take 33, 59
  // and 199 for the own slots).
  p->last = p->rg && max_len > 0 && c->batch * c->kv_heads * p->own.row_groups >= 256 &&
            (f32 || p->own.mt == 2 || max_prefix < 4 * all);
  if (p->last) {
    p->own.chunk = (int)max_len;
    p->own.chunks = 1;
  }
  p->both = p->rg && max_len > 0 && !p->last && units * p->row_tiles * p->chunks <= (tile_waves(f32, c->dim, p->rg) == 2 ? 512 : 255);
  p->own_chunks = p->last ? 1 : p->own.chunks > 1 ? p->own.chunks : 2;  // with one the kernel would write outputs, not parts
  p->ml_bytes = align_up((size_t)(units * p->chunks * all) * sizeof(float2), 256);
  p->o_bytes = align_up((size_t)(units * p->chunks * all) * c->dim * 4, 256);
  const int64_t own = max_len > 0 && !p->last ? c->batch * c->kv_heads * p->own_chunks * rows : 0;
  p->own_ml_bytes = align_up((size_t)own * sizeof(float2), 256);
  p->own_o_bytes = align_up((size_t)own * c->dim * 4, 256);
}

// The plan of a call; false where its arguments are not those of one.
static bool plan_call(const tallax_kv_cache* cache, int64_t prefixes, int64_t prefix_width, int64_t queries, int64_t heads,
                      int64_t max_prefix, int64_t max_len, SharedPlan* p) {
  KvView v;
  if (make_kv_view(cache, "kv_decode_shared", &v) != kOk || cache->batch < 1 || queries < 1 || queries > 1024 ||
      heads < 1 || heads % cache->kv_heads || prefixes < 1 || cache->batch % prefixes || prefix_width < 0 ||
      prefix_width > (1 << 25) / cache->page_size)
    return false;
  if (max_len < 0 || max_len > v.capacity) max_len = v.capacity;
  const int64_t most = prefix_width * cache->page_size;
  if (max_prefix < 0 || max_prefix > most) max_prefix = most;
  plan_shared(cache, prefixes, queries, heads / cache->kv_heads, max_prefix, max_len, p);
  return true;
}

template <class K>
static int launch_shared(K kernel, const SharedArgs& a, int64_t groups, int bytes, hipStream_t s) {
  if (bytes > 48 * 1024) {
    const hipError_t e = set_dynamic_lds_limit((const void*)kernel, bytes, s);
    if (e != hipSuccess) {
      set_error("kv_decode_shared: %s", hipGetErrorString(e));
      return kHipError;
    }
  }
  kernel<<<(unsigned)groups, kAttnThreads, bytes, s>>>(a);
  return launch_status("kv_decode_shared");
}

template <bool F32, int DP, int RG>
static int launch_tiles(const SharedArgs& a, const SharedPlan& p, int64_t groups, hipStream_t s) {
  constexpr int TG = kAttnWaves / RG, WT = tile_tokens(F32, DP, RG), WAVES = tile_waves(F32, DP, RG);
  constexpr int kBytes = Prefix<F32, DP, RG, TG, WT>::kBytes;
  if (!p.both) return launch_shared(kv_shared_tiles_kernel<F32, DP, RG, TG, WT, WAVES>, a, groups, kBytes, s);
  constexpr int kOwn = decode_lds_bytes<F32, DP, 1, true>(), kMost = kBytes > kOwn ? kBytes : kOwn;
  if constexpr (F32 || DP <= 128) {
    constexpr int kOwn2 = decode_lds_bytes<F32, DP, 2, true>();
    if (p.own.mt == 2)
      return launch_shared(kv_shared_both_kernel<F32, DP, RG, TG, WT, 2, WAVES>, a, groups, kBytes > kOwn2 ? kBytes : kOwn2, s);
  }
  return launch_shared(kv_shared_both_kernel<F32, DP, RG, TG, WT, 1, WAVES>, a, groups, kMost, s);
}

template <bool F32, int DP, int MT>
static int launch_rows(const SharedArgs& a, int64_t groups, hipStream_t s) {
  constexpr int WAVES = F32 && DP > 128 ? 1 : 2;
  if (a.own.queries > 1)
    return launch_shared(kv_shared_rows_kernel<F32, DP, MT, true, WAVES>, a, groups, decode_lds_bytes<F32, DP, MT, true>(), s);
  return launch_shared(kv_shared_rows_kernel<F32, DP, MT, false, WAVES>, a, groups, decode_lds_bytes<F32, DP, MT, false>(), s);
}

template <bool F32, int DP>
static int launch_dim(const SharedArgs& a, const SharedPlan& p, int64_t groups, hipStream_t s) {
  if (p.rg == 4) return launch_tiles<F32, DP, 4>(a, p, groups, s);
  if constexpr (!F32 || DP <= 128)
    if (p.rg == 2) return launch_tiles<F32, DP, 2>(a, p, groups, s);
  if constexpr (F32 || DP <= 128)
    if (p.own.mt == 2) return launch_rows<F32, DP, 2>(a, groups, s);
  return launch_rows<F32, DP, 1>(a, groups, s);
}

template <bool F32, int DP, int MT>
static int launch_last_mt(const SharedArgs& a, const SharedPlan& p, int64_t groups, hipStream_t s) {
  constexpr int W1 = F32 && DP > 128 ? 1 : 2, W3 = DP == 128 && MT == 1 ? 3 : W1;
  if (p.whole && a.own.queries > 1)
    return launch_shared(kv_shared_whole_kernel<F32, DP, MT, true, W1>, a, groups, decode_lds_bytes<F32, DP, MT, true>(), s);
  if (p.whole)
    return launch_shared(kv_shared_whole_kernel<F32, DP, MT, false, W3>, a, groups, decode_lds_bytes<F32, DP, MT, false>(), s);
  if (a.own.queries > 1)
    return launch_shared(kv_shared_last_kernel<F32, DP, MT, true, W1>, a, groups, decode_lds_bytes<F32, DP, MT, true>(), s);
  return launch_shared(kv_shared_last_kernel<F32, DP, MT, false, W3>, a, groups, decode_lds_bytes<F32, DP, MT, false>(), s);
}

template <bool F32, int DP>
static int launch_last(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  if constexpr (F32 || DP <= 128)
    if (p.own.mt == 2) return launch_last_mt<F32, DP, 2>(a, p, a.own_units, s);
  return launch_last_mt<F32, DP, 1>(a, p, a.own_units, s);
}

template <bool F32>
static int launch_prefix(const SharedArgs& a, const SharedPlan& p, int64_t groups, hipStream_t s) {
  if (a.own.c.dim <= 64) return launch_dim<F32, 64>(a, p, groups, s);
  return a.own.c.dim <= 128 ? launch_dim<F32, 128>(a, p, groups, s) : launch_dim<F32, 256>(a, p, groups, s);
}

}  // namespace tx

using namespace tx;

extern "C" {

size_t tallax_kv_decode_shared_workspace_size(const tallax_kv_cache* cache, int64_t prefixes, int64_t prefix_width,
                                              int64_t queries, int64_t heads, int64_t max_prefix, int64_t max_len) {
  SharedPlan p;
  return plan_call(cache, prefixes, prefix_width, queries, heads, max_prefix, max_len, &p) ? p.bytes() : 0;
}

int tallax_testing_shared_plan(const tallax_kv_cache* cache, int64_t prefixes, int64_t prefix_width, int64_t queries,
                               int64_t heads, int64_t max_prefix, int64_t max_len, int32_t* out) {
  SharedPlan p;
  if (!out || !plan_call(cache, prefixes, prefix_width, queries, heads, max_prefix, max_len, &p)) {
    set_error("bad arguments");
    return kInvalidArgument;
  }
  out[0] = p.whole ? 0 : !p.rg ? 1 : p.both ? 2 : p.last ? 3 : 4;
  out[1] = p.rg;
  out[2] = p.own.mt;
  out[3] = p.own.row_groups;
  out[4] = p.whole ? 1 : p.chunks;
  out[5] = p.whole ? 1 : p.own.chunks;
  return kOk;
}

int tallax_kv_decode_shared(const tallax_kv_cache* cache, const int32_t* prefix_table, int64_t prefixes,
                            int64_t prefix_width, const int32_t* prefix_lens, const void* q, int64_t q_stride_batch,
                            int64_t q_stride_query, int64_t q_stride_head, int64_t queries, int64_t heads, double scale,
                            const int32_t* lens, const int32_t* counts, int64_t max_prefix, int64_t max_len, void* out,
                            float* out_lse, void* workspace, size_t workspace_bytes, tallax_stream_t stream) {
  SharedArgs a;
  AttnArgs& o = a.own;
  int st = make_kv_view(cache, "kv_decode_shared", &o.c);
  if (st != kOk) return st;
  if (queries < 1 || queries > 1024 || heads < 1 || heads % cache->kv_heads) {
    set_error("kv_decode_shared: %lld queries (1 to 1024), %lld heads over %lld kv heads (a multiple)",
              (long long)queries, (long long)heads, (long long)cache->kv_heads);
    return kInvalidArgument;
  }
  if (prefix_width < 0 || prefixes < 0 || (cache->batch > 0 && (prefixes < 1 || cache->batch % prefixes))) {
    set_error("kv_decode_shared: a batch of %lld over %lld prefixes (a multiple) of %lld pages", (long long)cache->batch,
              (long long)prefixes, (long long)prefix_width);
    return kInvalidArgument;
  }
  const int64_t group = heads / cache->kv_heads, rows = queries * group;
  if (rows > 4096 || prefix_width > (1 << 25) / cache->page_size) {
    set_error("kv_decode_shared: %lld queries x %lld heads of a kv head (at most 4096 rows), a prefix of up to 2^25 slots",
              (long long)queries, (long long)group);
    return kUnsupported;
  }
  if (!(fabs(scale) * 1.4426950408889634 <= 3.4028234e38)) {
    set_error("kv_decode_shared: scale must be finite in float32");
    return kInvalidArgument;
  }
  if (cache->batch == 0) return kOk;
  const int64_t room = prefix_width * cache->page_size;
  if (!q || !lens || !out || !prefix_lens || (room > 0 && (!prefix_table || (cache->pages > 0 && (!cache->k || !cache->v))))) {
    set_error("kv_decode_shared: null pointer");
    return kInvalidArgument;
  }
  const int64_t es = cache->dtype == TALLAX_F32 ? 4 : 2;
  if (((uintptr_t)q | (uintptr_t)out) & 15 || q_stride_batch * es % 16 || q_stride_query * es % 16 ||
      q_stride_head * es % 16 || q_stride_batch < 0 || q_stride_query < 0 || q_stride_head < 0) {
    set_error("kv_decode_shared: q, its strides and out must be multiples of 16 bytes");
    return kUnsupported;
  }
  if (max_len < 0 || max_len > o.c.capacity || max_prefix < 0 || max_prefix > room) {
    set_error("kv_decode_shared: max_len %lld must be in [0, %d] and max_prefix %lld in [0, %lld], the slots of a table row",
              (long long)max_len, o.c.capacity, (long long)max_prefix, (long long)room);
    return kInvalidArgument;
  }
  SharedPlan p;
  plan_shared(cache, prefixes, queries, group, max_prefix, max_len, &p);
  st = check_workspace("kv_decode_shared", workspace, workspace_bytes, p.bytes());
  if (st != kOk) return st;
  st = pool_offsets(cache, o.c, "kv_decode_shared", &o.at);
  if (st != kOk) return st;
  const int64_t units = cache->batch * cache->kv_heads, pieces = prefixes * cache->kv_heads * p.chunks;
  const int64_t all = cache->batch * queries * heads;
  const int64_t most = (1 << 24) - 1;  // workgroups of 256 threads, of which HIP counts below 2^32
  if (units * p.own.row_groups * p.own.chunks + (pieces + 8) * p.row_tiles > most || all > most || p.own.chunks > 65535) {
    set_error("kv_decode_shared: too many workgroups");
    return kUnsupported;
  }
  char* ws = (char*)workspace;
  a.part_ml = (float2*)ws;
  a.part_o = (float*)(ws + p.ml_bytes);
  o.part_ml = (float2*)(ws + p.ml_bytes + p.o_bytes);
  o.part_o = (float*)(ws + p.ml_bytes + p.o_bytes + p.own_ml_bytes);
  o.q = (const char*)q;
  o.q_batch = q_stride_batch * es;
  o.q_query = q_stride_query * es;
  o.q_head = q_stride_head * es;
  o.lens = lens;
  o.counts = counts;
  o.out = (char*)out;
  o.lse = out_lse;
  o.queries = (int)queries;
  o.heads = (int)heads;
  o.kv_heads = (int)cache->kv_heads;
  o.group = (int)group;
  o.rows = (int)rows;
  o.max_len = (int)max_len;
  o.chunk = p.own.chunk;
  o.chunks = p.own_chunks;
  o.row_groups = p.own.row_groups;
  o.scale2 = (float)(scale * 1.4426950408889634);
  o.raw = nullptr;
  o.raw_ld = 0;
  o.scores = nullptr;
  o.out_scores = nullptr;
  o.vector_scores = 0;
  a.table = prefix_table;
  a.lens = prefix_lens;
  a.width = (int)prefix_width;
  a.max_len = cache->pages > 0 ? (int)max_prefix : 0;  // without a page there is nothing to see, nor to read
  a.per = (int)(cache->batch / prefixes);
  a.rows = (int)(a.per * rows);
  a.row_tiles = p.row_tiles;
  a.chunk = p.chunk;
  a.chunks = p.chunks;
  a.flip = scale < 0 ? (es == 4 ? 0x80000000u : 0x80008000u) : 0u;
  a.scale2 = fmaxf(fabsf(o.scale2), 1.1754944e-38f);
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = cache->dtype == TALLAX_F32;
  a.pieces = a.max_len > 0 ? (int)pieces : 0;
  a.own_units = (int)(units * p.own.row_groups);
  const int64_t own = max_len > 0 ? (int64_t)a.own_units * p.own.chunks : 0;
  a.own_from = (int)(((int64_t)a.pieces + 7) / 8 * 8 * p.row_tiles);
  const int64_t groups = p.whole ? 0 : !p.rg ? a.pieces + own : p.both ? a.own_from + own : a.own_from;
  if (groups > 0) {
    st = f32 ? launch_prefix<true>(a, p, groups, s) : launch_prefix<false>(a, p, groups, s);
    if (st != kOk) return st;
  }
  if (p.last || p.whole) {
    if (o.c.dim <= 64) return f32 ? launch_last<true, 64>(a, p, s) : launch_last<false, 64>(a, p, s);
    if (o.c.dim <= 128) return f32 ? launch_last<true, 128>(a, p, s) : launch_last<false, 128>(a, p, s);
    return f32 ? launch_last<true, 256>(a, p, s) : launch_last<false, 256>(a, p, s);
  }
  if (p.rg && !p.both && own > 0) {
    st = launch_attention(o, p.own, units, f32, s);
    if (st != kOk) return st;
  }
  const int slots = o.c.dim <= 64 ? 16 : o.c.dim <= 128 ? 8 : 4;
  const int64_t parts = p.chunks + p.own.chunks;
  int split = 1;  // enough workgroups for the card, and no more groups of lanes to a row than parts
  while (split < slots && split < parts && all * split / slots < 1024) split *= 2;
  const int64_t each = slots / split;
  kv_shared_join_kernel<<<(unsigned)((all + each - 1) / each), 256, 0, s>>>(a, f32, split, all);
  return launch_status("kv_decode_shared");
}

}  // extern "C"
