// Attention of the newest tokens of sequences that begin with a shared prefix.
//
// The prefix's slots are taken for all its sequences at once: the rows of a kv
// head (sequence, query and head of the group, in this order) are the columns
// of two matrix products,
//   S^T = K Q^T   (tokens x rows),   O^T = V^T P^T   (dim x rows),
// of which a workgroup computes 32 * RG rows over a chunk of the prefix.  The
// sequences' own slots are kv_attention.hip's; the join puts both together.
//
// A workgroup has RG * TG waves: wave (rg, tg) takes 32 rows and every TG-th
// tile of WT tokens, which its RG waves bring into LDS together, through
// registers and one tile ahead.  In S^T a lane holds one row's scores, so that
// weights are the second operand of the second product as they lie; its first
// operand, values by dim, is read transposed from LDS (bfloat16), or in single
// elements (float32).
#include "tx_attention.h"

namespace tx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct SharedArgs {
  AttnArgs own;
  const int32_t* table;  // [prefixes, width]
  const int32_t* lens;   // [prefixes]
  int width, max_len;
  int per;               // sequences of a prefix
  int rows;              // of a prefix's kv head
  int row_tiles, chunk, chunks, pieces;
  uint32_t flip;         // sign bits of q, where the scale is negative
  float scale2;          // its size, above 0: -inf, of what is not seen, stays -inf
  float2* part_ml;       // [prefixes * kv_heads][chunks][rows]: maximum (base 2), sum
  float* part_o;         // [prefixes * kv_heads][chunks][rows][dim]
};

// Places of 16-byte vectors in a tile: vector c of a token's row is stored at
// c ^ swizzle, so that the lanes of a read, which take the same vectors of
// neighbouring tokens, meet different banks.
template <int VECS>
__device__ __forceinline__ int key_place(int token, int c) {
  return token * VECS + (c ^ (VECS >= 16 ? token & 15 : (token >> 1) & 7));
}

template <bool F32, int VECS>
__device__ __forceinline__ int value_place(int token, int c) {
  if (F32) return token * VECS + (c ^ (8 * ((token >> 2) & 1)));
  return token * VECS + (c ^ (VECS >= 16 ? 4 * (token & 3) : 4 * ((token >> 1) & 1)));
}

template <bool F32, int DP, int RG, int TG, int WT, int WAVES>
__global__ __launch_bounds__(RG * TG * kWave, WAVES) void kv_prefix_kernel(SharedArgs a) {
  constexpr int ES = F32 ? 4 : 2, NW = RG * TG, kThreads = NW * kWave;
  constexpr int VECS = DP * ES / 16;               // 16-byte vectors of a token's key
  constexpr int LOADS = WT * VECS / (kWave * RG);  // of a tile's keys, per lane
  constexpr int QV = VECS / 2;                     // of a row's query, per lane
  constexpr int NB = WT / 32, ACC = DP / 32, STEP = TG * WT, PAD = 36;
  extern __shared__ uint4 tiles[];  // [2][TG][keys, values][WT * VECS]

  // The row tiles of a piece (chunk of a prefix's kv head) are workgroups of one XCD, that follow one another: their
  // numbers are the same modulo 8.
  const int step = blockIdx.x >> 3, piece = (step / a.row_tiles) * 8 + (blockIdx.x & 7);
  if (piece >= a.pieces) return;
  const int unit = piece / a.chunks, chunk = piece - unit * a.chunks;
  const AttnArgs& o = a.own;
  const int p = unit / o.kv_heads, kvh = unit - p * o.kv_heads;
  const int len = min(max(a.lens[p], 0), a.max_len);
  const int start = chunk * a.chunk;
  if (start >= len) return;
  const int end = min(start + a.chunk, len);
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), n = lane & 31, h = lane >> 5;
  const int rg = wave % RG, tg = wave / RG;
  const int row0 = (step % a.row_tiles) * 32 * RG + rg * 32;

  const char* kbase = o.c.k + kvh * o.c.k_head;
  const char* vbase = o.c.v + kvh * o.c.v_head;
  const int32_t* table = a.table + (int64_t)p * a.width;
  const char* safe = o.q;  // what is read in the place of a vector that is not there

  uint4 ks[LOADS], vs[LOADS];
  uint32_t holes = 0;  // bit j: vectors j of this lane are not there
  uint64_t gone = 0, next_gone = 0;
  auto load_tile = [&](int t0) {
    const int t = t0 + (lane & (WT - 1));
    const int page = t < end ? page_id(o.c, table, t) : -1;
    const int off = t - (int)page_of(o.c.div, (uint32_t)t) * o.c.div.size;
    const uint32_t k_at = (uint32_t)page * o.at.k_page + (uint32_t)off * o.at.k_slot;
    const uint32_t v_at = (uint32_t)page * o.at.v_page + (uint32_t)off * o.at.v_slot;
    next_gone = __ballot(page < 0);
    holes = 0;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = (rg * LOADS + j) * kWave + lane, token = i / VECS, c = i % VECS;
      const char* pk = kbase + ((uint64_t)from_lane(k_at, token) << o.at.shift) + c * 16;
      const char* pv = vbase + ((uint64_t)from_lane(v_at, token) << o.at.shift) + c * 16;
      const bool hole = ((next_gone >> token) & 1) || c * 16 >= o.c.dim * ES;
      holes |= (uint32_t)hole << j;
      ks[j] = *(const uint4*)(hole ? safe : pk);
      vs[j] = *(const uint4*)(hole ? safe : pv);
    }
  };
  load_tile(start + tg * WT);

  uint4 q[QV];
  {
    const int row = row0 + n, seq = row / o.rows, rr = row - seq * o.rows, t = rr / o.group;
    const char* at = o.q + (int64_t)(p * a.per + seq) * o.q_batch + t * o.q_query +
                     (int64_t)(kvh * o.group + rr - t * o.group) * o.q_head;
#pragma unroll
    for (int i = 0; i < QV; ++i) {
      const int c = 2 * i + h;
      q[i] = make_uint4(0, 0, 0, 0);
      if (row < a.rows && c * 16 < o.c.dim * ES) {
        q[i] = *(const uint4*)(at + c * 16);
        q[i] = make_uint4(q[i].x ^ a.flip, q[i].y ^ a.flip, q[i].z ^ a.flip, q[i].w ^ a.flip);
      }
    }
  }
  f32x16 acc[ACC];
#pragma unroll
  for (int j = 0; j < ACC; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // of q.k, which times scale2 is the exponent of a weight

  const int rounds = (end - start + STEP - 1) / STEP;
  for (int it = 0; it < rounds; ++it) {
    const int t0 = start + it * STEP + tg * WT;
    uint4* keys = tiles + ((it & 1) * TG + tg) * 2 * WT * VECS;
    uint4* values = keys + WT * VECS;
    gone = next_gone;
    if (gone != 0 || DP != o.c.dim) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        if ((holes >> j) & 1) ks[j] = vs[j] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = (rg * LOADS + j) * kWave + lane, token = i / VECS, c = i % VECS;
      keys[key_place<VECS>(token, c)] = ks[j];
      values[value_place<F32, VECS>(token, c)] = vs[j];
    }
    if (it + 1 < rounds) load_tile(t0 + STEP);
    // One barrier a round: what is written in the next round was read in the last one, before this.
    lds_barrier();
    f32x16 s[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < QV; ++i) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const uint4 k = keys[key_place<VECS>(32 * u + n, 2 * i + h)];
        if constexpr (F32) {
          s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.x), __uint_as_float(q[i].x), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.y), __uint_as_float(q[i].y), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.z), __uint_as_float(q[i].z), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.w), __uint_as_float(q[i].w), s[u], 0, 0, 0);
        } else {
          s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                         __builtin_bit_cast(bf16x8_t, q[i]), s[u], 0, 0, 0);
        }
      }
    }
    // lane (n, h) holds row n's scores of tokens 32 u + 8 (r / 4) + 4 h + r % 4
    if (gone != 0) {
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((gone >> (32 * u + 8 * (r / 4) + 4 * h + r % 4)) & 1) s[u][r] = -INFINITY;
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
      const float* v = (const float*)values;
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int j = 0; j < ACC; ++j) {
            const int token = 32 * u + 8 * (r / 4) + 4 * h + r % 4;
            acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[value_place<true, VECS>(token, 8 * j + n / 4) * 4 + n % 4],
                                                          s[u][r], acc[j], 0, 0, 0);
          }
    } else {
      // The product takes both sides in bfloat16: the weights, at most 1, are rounded to it (by 2^-8 of each at most);
      // their sum, by which the output is divided, is of the unrounded ones.
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_bf16(s[u][8 * kk + 2 * i], s[u][8 * kk + 2 * i + 1]);
          const bf16x8_t weights = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
          for (int j = 0; j < ACC; ++j) {
            // 16 lanes read 16 neighbouring elements of four tokens, and get four tokens of one element each
            typedef __attribute__((address_space(3))) bf16x4 lds_x4;
            const int token = 32 * u + 16 * kk + 4 * h + (lane & 15) / 4;
            const int c = 4 * j + 2 * ((lane >> 4) & 1) + (lane & 3) / 2;
            const char* lo = (const char*)(values + value_place<false, VECS>(token, c)) + (lane & 1) * 8;
            const char* hi = (const char*)(values + value_place<false, VECS>(token + 8, c)) + (lane & 1) * 8;
            const bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_x4*)lo);
            const bf16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_x4*)hi);
            const uint2 xu = __builtin_bit_cast(uint2, x), yu = __builtin_bit_cast(uint2, y);
            acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(bf16x8_t, make_uint4(xu.x, xu.y, yu.x, yu.y)), weights, acc[j], 0, 0, 0);
          }
        }
    }
  }
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
  const int first = (step % a.row_tiles) * 32 * RG;
#pragma unroll
  for (int j = 0; j < ACC; ++j) {
    float* mo = sums + (wave * 32 + n) * PAD;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4 x = make_float4(acc[j][4 * i] * mine, acc[j][4 * i + 1] * mine, acc[j][4 * i + 2] * mine,
                             acc[j][4 * i + 3] * mine);
      if (none) x = make_float4(0.f, 0.f, 0.f, 0.f);
      *(float4*)(mo + 8 * i + 4 * h) = x;
    }
    __syncthreads();
    for (int i = tid; i < RG * 32 * 8; i += kThreads) {
      const int row = i / 8, d = 32 * j + i % 8 * 4;
      if (first + row >= a.rows || d >= o.c.dim) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < TG; ++k) {
        const float4 y = *(const float4*)(sums + (k * RG * 32 + row) * PAD + i % 8 * 4);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      *(float4*)(a.part_o + (out + first + row) * o.c.dim + d) = x;
    }
    __syncthreads();
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
  int rg, step, row_tiles, chunk, chunks;
  AttnPlan own;
  int own_chunks;
  size_t ml_bytes, o_bytes, own_ml_bytes, own_o_bytes;
  size_t bytes() const { return ml_bytes + o_bytes + own_ml_bytes + own_o_bytes; }
};

static void plan_shared(const tallax_kv_cache* c, int64_t prefixes, int64_t rows, int64_t max_prefix, int64_t max_len,
                        SharedPlan* p) {
  const bool f32 = c->dtype == TALLAX_F32;
  const int64_t all = c->batch / prefixes * rows, units = prefixes * c->kv_heads;
  p->rg = all <= 32 && !(f32 && c->dim > 128) ? 1 : all <= 64 ? 2 : 4;
  const int tg = c->dim > 128 ? (f32 || p->rg == 4 ? 1 : 2) : f32 ? (c->dim > 64 ? 2 : p->rg == 4 ? 2 : 4) : p->rg == 4 ? 2 : 4;
  const int wt = !f32 && c->dim <= 128 && p->rg == 4 ? 64 : 32;
  p->step = tg * wt;
  p->row_tiles = (int)((all + 32 * p->rg - 1) / (32 * p->rg));
  int64_t chunk = (max_prefix * units * p->row_tiles + 255) / 256;
  if (chunk < p->step) chunk = p->step;
  chunk = (chunk + p->step - 1) / p->step * p->step;
  p->chunk = (int)chunk;
  p->chunks = (int)((max_prefix + chunk - 1) / chunk);
  if (p->chunks < 1) p->chunks = 1;
  plan_attention(c->batch, c->kv_heads, rows, c->dim, c->dtype, max_len, false, &p->own);
  p->own_chunks = p->own.chunks > 1 ? p->own.chunks : 2;  // with one the kernel would write outputs, not parts
  p->ml_bytes = align_up((size_t)(units * p->chunks * all) * sizeof(float2), 256);
  p->o_bytes = align_up((size_t)(units * p->chunks * all) * c->dim * 4, 256);
  const int64_t own = max_len > 0 ? c->batch * c->kv_heads * p->own_chunks * rows : 0;
  p->own_ml_bytes = align_up((size_t)own * sizeof(float2), 256);
  p->own_o_bytes = align_up((size_t)own * c->dim * 4, 256);
}

template <bool F32, int DP, int RG, int TG, int WT, int WAVES>
static int launch_prefix(const SharedArgs& a, int step, hipStream_t s) {
  if (step != TG * WT) {  // the plan and the instance must agree
    set_error("kv_decode_shared: no kernel for steps of %d", step);
    return kUnsupported;
  }
  constexpr int kTiles = 2 * TG * 2 * WT * DP * (F32 ? 4 : 2), kJoin = RG * TG * 32 * (8 + 36 * 4);
  constexpr int kBytes = kTiles > kJoin ? kTiles : kJoin;
  static_assert(kBytes <= 160 * 1024, "LDS");
  if (kBytes > 48 * 1024) {
    const hipError_t e = set_dynamic_lds_limit((const void*)kv_prefix_kernel<F32, DP, RG, TG, WT, WAVES>, kBytes, s);
    if (e != hipSuccess) {
      set_error("kv_decode_shared: %s", hipGetErrorString(e));
      return kHipError;
    }
  }
  const unsigned grid = (unsigned)((a.pieces + 7) / 8 * 8) * (unsigned)a.row_tiles;
  kv_prefix_kernel<F32, DP, RG, TG, WT, WAVES><<<grid, RG * TG * kWave, kBytes, s>>>(a);
  return launch_status("kv_decode_shared");
}

static int launch_prefix_any(const SharedArgs& a, int rg, int step, bool f32, hipStream_t s) {
  const int dim = a.own.c.dim;
  if (f32) {
    if (dim <= 64)
      return rg == 1   ? launch_prefix<true, 64, 1, 4, 32, 1>(a, step, s)
             : rg == 2 ? launch_prefix<true, 64, 2, 4, 32, 2>(a, step, s)
                       : launch_prefix<true, 64, 4, 2, 32, 2>(a, step, s);
    if (dim <= 128)
      return rg == 1   ? launch_prefix<true, 128, 1, 2, 32, 1>(a, step, s)
             : rg == 2 ? launch_prefix<true, 128, 2, 2, 32, 1>(a, step, s)
                       : launch_prefix<true, 128, 4, 2, 32, 2>(a, step, s);
    return rg == 2 ? launch_prefix<true, 256, 2, 1, 32, 1>(a, step, s) : launch_prefix<true, 256, 4, 1, 32, 1>(a, step, s);
  }
  if (dim <= 64)
    return rg == 1   ? launch_prefix<false, 64, 1, 4, 32, 1>(a, step, s)
           : rg == 2 ? launch_prefix<false, 64, 2, 4, 32, 2>(a, step, s)
                     : launch_prefix<false, 64, 4, 2, 64, 2>(a, step, s);
  if (dim <= 128)
    return rg == 1   ? launch_prefix<false, 128, 1, 4, 32, 1>(a, step, s)
           : rg == 2 ? launch_prefix<false, 128, 2, 4, 32, 2>(a, step, s)
                     : launch_prefix<false, 128, 4, 2, 64, 2>(a, step, s);
  return rg == 1   ? launch_prefix<false, 256, 1, 2, 32, 1>(a, step, s)
         : rg == 2 ? launch_prefix<false, 256, 2, 2, 32, 1>(a, step, s)
                   : launch_prefix<false, 256, 4, 1, 32, 1>(a, step, s);
}

}  // namespace tx

using namespace tx;

extern "C" {

size_t tallax_kv_decode_shared_workspace_size(const tallax_kv_cache* cache, int64_t prefixes, int64_t prefix_width,
                                              int64_t queries, int64_t heads, int64_t max_prefix, int64_t max_len) {
  KvView v;
  if (make_kv_view(cache, "kv_decode_shared", &v) != kOk || cache->batch < 1 || queries < 1 || queries > 1024 ||
      heads < 1 || heads % cache->kv_heads || prefixes < 1 || cache->batch % prefixes || prefix_width < 0 ||
      prefix_width > (1 << 25) / cache->page_size)
    return 0;
  if (max_len < 0 || max_len > v.capacity) max_len = v.capacity;
  const int64_t most = prefix_width * cache->page_size;
  if (max_prefix < 0 || max_prefix > most) max_prefix = most;
  SharedPlan p;
  plan_shared(cache, prefixes, queries * (heads / cache->kv_heads), max_prefix, max_len, &p);
  return p.bytes();
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
  plan_shared(cache, prefixes, rows, max_prefix, max_len, &p);
  st = check_workspace("kv_decode_shared", workspace, workspace_bytes, p.bytes());
  if (st != kOk) return st;
  st = pool_offsets(cache, o.c, "kv_decode_shared", &o.at);
  if (st != kOk) return st;
  const int64_t units = cache->batch * cache->kv_heads, pieces = prefixes * cache->kv_heads * p.chunks;
  const int64_t all = cache->batch * queries * heads;
  if (units * p.own.row_groups > INT32_MAX || p.own.chunks > 65535 || cache->batch * rows > INT32_MAX / 64 ||
      (pieces + 8) * p.row_tiles > INT32_MAX || all > INT32_MAX) {
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
  a.max_len = (int)max_prefix;
  a.per = (int)(cache->batch / prefixes);
  a.rows = (int)(a.per * rows);
  a.row_tiles = p.row_tiles;
  a.chunk = p.chunk;
  a.chunks = p.chunks;
  a.pieces = (int)pieces;
  a.flip = scale < 0 ? (es == 4 ? 0x80000000u : 0x80008000u) : 0u;
  a.scale2 = fmaxf(fabsf(o.scale2), 1.1754944e-38f);
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = cache->dtype == TALLAX_F32;
  if (max_prefix > 0) {
    st = launch_prefix_any(a, p.rg, p.step, f32, s);
    if (st != kOk) return st;
  }
  if (max_len > 0) {
    st = launch_attention(o, p.own, units, f32, s);
    if (st != kOk) return st;
  }
  const int groups = o.c.dim <= 64 ? 16 : o.c.dim <= 128 ? 8 : 4;
  const int64_t parts = p.chunks + p.own.chunks;
  int split = 1;  // enough workgroups for the card, and no more groups of lanes to a row than parts
  while (split < groups && split < parts && all * split / groups < 1024) split *= 2;
  const int64_t each = groups / split;
  kv_shared_join_kernel<<<(unsigned)((all + each - 1) / each), 256, 0, s>>>(a, f32, split, all);
  return launch_status("kv_decode_shared");
}

}  // extern "C"
