// Attention of the newest tokens over a paged key-value cache.
//
// One workgroup of four waves takes one kv head of one sequence, up to 16 * MT
// of its query rows (row = query * group + head in the group) and one chunk of
// the length (tx_decode.h).  Chunks are joined by a second kernel.
//
// Bound by memory.  64 sequences of up to 4096 slots, 8 kv heads of 128
// (bfloat16), 685 MB: 148 us here and 13 in the join, 4.2 TB/s; 4 of up to
// 131071, 1.54 GB: 285 and 5 us, 5.3 TB/s; the loads alone take 136 and 277 us.
// Float32, 9 of up to 2050, 12 heads of 80, 90 MB: 26 and 5 us, loads alone 22.
//
// The length is split by max_len, which is the table's width unless the caller
// knows a smaller bound: 4 sequences of up to 4096 slots with 8 kv heads take 16 us,
// also in a table of 131072 slots with max_len 4096, and 54 there without it.
#include "tx_decode.h"

namespace tx {

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

template <bool F32, int DP, int MT, bool MANY, int WAVES>
__global__ __launch_bounds__(kAttnThreads, WAVES) void kv_decode_kernel(AttnArgs a) {
  extern __shared__ float lds[];
  const int rg = blockIdx.x % a.row_groups, unit = blockIdx.x / a.row_groups;  // sequence * kv_heads + kv head
  decode_chunk<F32, DP, MT, MANY>(a, OwnRows(a, unit), rg, blockIdx.y, lds);
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

void plan_attention(int64_t batch, int64_t kv_heads, int64_t rows, int dim, int dtype, int64_t max_len, bool with_scores,
                    AttnPlan* p) {
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
  constexpr int bytes = decode_lds_bytes<F32, DP, MT, MANY>();
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

int launch_attention(const AttnArgs& a, const AttnPlan& p, int64_t units, bool f32, hipStream_t s) {
  if (a.c.dim <= 64) return f32 ? launch_decode<true, 64>(a, p, units, s) : launch_decode<false, 64>(a, p, units, s);
  if (a.c.dim <= 128) return f32 ? launch_decode<true, 128>(a, p, units, s) : launch_decode<false, 128>(a, p, units, s);
  return f32 ? launch_decode<true, 256>(a, p, units, s) : launch_decode<false, 256>(a, p, units, s);
}

int pool_offsets(const tallax_kv_cache* cache, const KvView& c, const char* what, PoolOffsets* out) {
  uint64_t bits = 1 << 20;  // offsets in units of the largest power of two that the strides share
  for (int64_t x : {c.k_page, c.k_slot, c.v_page, c.v_slot}) bits |= (uint64_t)x;
  out->shift = __builtin_ctzll(bits);
  const uint64_t far_page = cache->pages > 0 ? cache->pages - 1 : 0, far_slot = cache->page_size - 1;
  if ((far_page * c.k_page + far_slot * c.k_slot) >> out->shift >> 32 ||
      (far_page * c.v_page + far_slot * c.v_slot) >> out->shift >> 32) {
    set_error("%s: a pool may span up to 2^32 times the largest power of two that divides its strides (%d bytes)", what,
              1 << out->shift);
    return kUnsupported;
  }
  out->k_page = (uint32_t)(c.k_page >> out->shift);
  out->k_slot = (uint32_t)(c.k_slot >> out->shift);
  out->v_page = (uint32_t)(c.v_page >> out->shift);
  out->v_slot = (uint32_t)(c.v_slot >> out->shift);
  return kOk;
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
  st = pool_offsets(cache, a.c, "kv_decode", &a.at);
  if (st != kOk) return st;
  const int64_t units = cache->batch * cache->kv_heads;
  if (units * p.row_groups > INT32_MAX || p.chunks > 65535) {
    set_error("kv_decode: too many workgroups");
    return kUnsupported;
  }
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = cache->dtype == TALLAX_F32;
  st = launch_attention(a, p, units, f32, s);
  if (st != kOk) return st;
  const int out_blocks = p.chunks > 1 ? p.rows : 0;
  const int blocks = out_blocks + (scores ? (a.c.capacity + 1023) / 1024 : 0);
  if (blocks == 0) return kOk;
  const size_t lds = (size_t)p.rows * 8 > 4096 ? (size_t)p.rows * 8 : 4096;
  kv_decode_join_kernel<<<dim3((unsigned)units, (unsigned)blocks), 256, lds, s>>>(a, f32, out_blocks);
  return launch_status("kv_decode");
}

}  // extern "C"
