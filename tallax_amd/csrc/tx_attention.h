// Attention over a paged cache: what its kernels share.
#pragma once
#include <math.h>

#include "tx_common.h"
#include "tx_kv.h"

namespace tx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr float kLn2 = 0.693147180559945309417f;

// Strides in a pool, in units of 2^shift bytes, which 32 bits hold.
struct PoolOffsets {
  int shift;
  uint32_t k_page, k_slot, v_page, v_slot;
};

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
  PoolOffsets at;
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

__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)x);
}

struct AttnPlan {
  int mt, row_groups, chunk, chunks, max_len, rows, raw_ld;
  size_t ml_bytes, o_bytes, raw_bytes;
};

// How the attention of each sequence over its own slots is split over workgroups.
void plan_attention(int64_t batch, int64_t kv_heads, int64_t rows, int dim, int dtype, int64_t max_len, bool with_scores,
                    AttnPlan* p);

// The chunks of that attention (outputs themselves where a.chunks is 1).
int launch_attention(const AttnArgs& a, const AttnPlan& p, int64_t units, bool f32, hipStream_t s);

// The pool's strides as its offsets are counted, or a Status with the message set.
int pool_offsets(const tallax_kv_cache* cache, const KvView& c, const char* what, PoolOffsets* out);

}  // namespace tx
