// Paged key-value cache: appending tokens and evicting them by accumulated
// attention weight.
#include "tx_kv.h"

#include "tx_common.h"
#include "tx_scan.h"

namespace tx {

// moves x vectors and slots x heads of one row stay below 2^31
constexpr int64_t kMaxCapacity = 1 << 25;

int make_kv_view(const tallax_kv_cache* c, const char* what, KvView* out) {
  if (!c) {
    set_error("%s: null cache", what);
    return kInvalidArgument;
  }
  if (c->dtype != TALLAX_F32 && c->dtype != TALLAX_BF16) {
    set_error("%s: cache dtype %d (float32 or bfloat16)", what, c->dtype);
    return kUnsupported;
  }
  if (c->batch < 0 || c->pages < 0 || c->table_width < 0 || c->kv_heads < 1 || c->page_size < 1) {
    set_error("%s: batch %lld, pages %lld, table width %lld, kv_heads %lld, page_size %lld", what, (long long)c->batch,
              (long long)c->pages, (long long)c->table_width, (long long)c->kv_heads, (long long)c->page_size);
    return kInvalidArgument;
  }
  if (c->dim < 8 || c->dim > 256 || c->dim % 8) {
    set_error("%s: dim %d must be a multiple of 8 in [8, 256]", what, c->dim);
    return kUnsupported;
  }
  if (c->batch > 65535 || c->kv_heads > 65535 || c->pages > INT32_MAX || c->page_size > (1 << 20) ||
      c->table_width > kMaxCapacity / c->page_size || c->batch * c->kv_heads > INT32_MAX / 256) {
    set_error("%s: batch and kv_heads up to 65535, pages below 2^31, a table of up to 2^25 slots, page_size up to 2^20", what);
    return kUnsupported;
  }
  if (c->batch > 0 && c->table_width > 0 && (!c->block_table || (c->pages > 0 && (!c->k || !c->v)))) {
    set_error("%s: null cache pointer", what);
    return kInvalidArgument;
  }
  const int64_t es = c->dtype == TALLAX_F32 ? 4 : 2;
  const int64_t st[6] = {c->k_stride_page, c->k_stride_head, c->k_stride_slot,
                         c->v_stride_page, c->v_stride_head, c->v_stride_slot};
  bool ok = (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0;
  for (int64_t s : st) ok = ok && s >= 0 && s * es % 16 == 0 && s < ((int64_t)1 << 40);
  // inside a page the kernels' offsets are 32 bits wide
  ok = ok && st[2] * es * c->page_size < ((int64_t)1 << 31) && st[5] * es * c->page_size < ((int64_t)1 << 31);
  if (!ok) {
    set_error("%s: cache bases and strides must be multiples of 16 bytes, a head's slots of a page within 2 GiB", what);
    return kUnsupported;
  }
  out->k = (char*)c->k;
  out->v = (char*)c->v;
  out->k_page = st[0] * es;
  out->k_head = st[1] * es;
  out->k_slot = st[2] * es;
  out->v_page = st[3] * es;
  out->v_head = st[4] * es;
  out->v_slot = st[5] * es;
  out->table = c->block_table;
  out->width = (int)c->table_width;
  out->capacity = (int)(c->table_width * c->page_size);
  out->pages = (int)c->pages;
  out->dim = c->dim;
  out->div = make_page_div(c->page_size);
  return kOk;
}

// ---------------------------------------------------------------------------
// Append: one thread per 16 bytes of a new key and of its value.
// ---------------------------------------------------------------------------
struct AppendArgs {
  KvView c;
  const int32_t* lens;
  const int32_t* counts;
  const uint4* k_new;
  const uint4* v_new;
  int tokens, heads, vecs;  // vecs: 16-byte vectors of one head's key
  float* scores;
  int32_t* positions;
  const int32_t* seen;
  int32_t* out_lens;
};

__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const int b = blockIdx.y;
  const int len = max(a.lens[b], 0);
  int cnt = a.tokens;
  if (a.counts) cnt = min(max(a.counts[b], 0), a.tokens);
  if (blockIdx.x == 0 && threadIdx.x == 0)
    a.out_lens[b] = (int)min((int64_t)len + cnt, (int64_t)a.c.capacity);
  const int line = a.heads * a.vecs;  // vectors of one token
  const int64_t n = (int64_t)cnt * line;
  const int64_t base = (int64_t)b * a.tokens * line;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int t = (int)(i / line);
    const int r = (int)(i - (int64_t)t * line);
    const int h = r / a.vecs, d = r - h * a.vecs;
    const int64_t slot = (int64_t)len + t;
    if (slot >= a.c.capacity) continue;
    const int page = page_id(a.c, a.c.table + (int64_t)b * a.c.width, (int)slot);
    if (page < 0) continue;
    const int off = (int)slot - (int)page_of(a.c.div, (uint32_t)slot) * a.c.div.size;
    *(uint4*)(a.c.k + page * a.c.k_page + h * a.c.k_head + off * a.c.k_slot + d * 16) = a.k_new[base + i];
    *(uint4*)(a.c.v + page * a.c.v_page + h * a.c.v_head + off * a.c.v_slot + d * 16) = a.v_new[base + i];
    if (a.scores && d == 0) {
      const int64_t at = ((int64_t)b * a.heads + h) * a.c.capacity + slot;
      a.scores[at] = 0.0f;
      a.positions[at] = a.seen[b] + t;
    }
  }
}

// ---------------------------------------------------------------------------
// Evict, choice: one workgroup per (sequence, kv head).  Every slot has a key
// (all ones where it is always kept, else the order-preserving integer of its
// score); four 8-bit radix steps find the key of the budget-th largest, then
// one pass in slot order marks what is kept, writes the scores and positions
// that stay and lists the free places and the slots that move into them.
// ---------------------------------------------------------------------------
struct EvictArgs {
  KvView c;
  const int32_t* lens;
  const float* scores;
  const int32_t* positions;
  const int32_t* seen;
  int heads, budget, recent, sinks;
  int32_t* out_lens;
  float* out_scores;
  int32_t* out_positions;
  int32_t* moves;  // [rows]: how many, then [rows][2][budget]: from, to
  int rows;
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;

__global__ __launch_bounds__(kEvictThreads) void kv_evict_select_kernel(EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int red[kEvictWaves];
  __shared__ int found[2];
  const int row = blockIdx.x, b = row / a.heads, tid = threadIdx.x;
  const int cap = a.c.capacity;
  const int len = min(max(a.lens[b], 0), cap);
  const int nlen = min(len, a.budget);
  const int64_t at = (int64_t)row * cap;
  const float* sc = a.scores + at;
  const int32_t* ps = a.positions + at;
  float* osc = a.out_scores + at;
  int32_t* ops = a.out_positions + at;
  if (row % a.heads == 0 && tid == 0) a.out_lens[b] = nlen;
  for (int i = nlen + tid; i < cap; i += kEvictThreads) {
    osc[i] = 0.0f;
    ops[i] = -1;
  }
  if (len <= a.budget) {
    if (tid == 0) a.moves[row] = 0;
    for (int i = tid; i < nlen; i += kEvictThreads) {
      osc[i] = sc[i];
      ops[i] = ps[i];
    }
    return;
  }
  const int64_t newest = (int64_t)a.seen[b] - a.recent;
  auto key_of = [&](int i) -> uint32_t {
    const int32_t p = ps[i];
    return p < a.sinks || p >= newest ? 0xFFFFFFFFu : select_key(__float_as_uint(sc[i]));
  };
  // the budget-th largest key, and how many of its equals are kept
  uint32_t prefix = 0;
  int need = a.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < len; i += kEvictThreads) {
      const uint32_t k = key_of(i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < kWave) {  // lane l: digits 255 - 4l down to 252 - 4l
      int c[4], s = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += c[j] = hist[255 - 4 * tid - j];
      int total;
      int above = wave_exscan_i32(s, total);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (above < need && need <= above + c[j]) {
          found[0] = 255 - 4 * tid - j;
          found[1] = need - above;
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    __syncthreads();
  }
  int32_t* from = a.moves + a.rows + (int64_t)row * 2 * a.budget;
  int32_t* to = from + a.budget;
  int ties = 0, holes = 0, movers = 0;
  for (int i0 = 0; i0 < len; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < len ? key_of(i) : 0u;
    const bool tie = i < len && k == prefix;
    int total;
    const int rank = ties + block_exscan<kEvictWaves>(tie, red, total);
    ties += total;
    const bool keep = i < len && (k > prefix || (tie && rank < need));
    const bool hole = i < nlen && !keep, mover = i >= nlen && keep;
    const int pre = block_exscan<kEvictWaves>((int)hole + ((int)mover << 16), red, total);
    if (hole) to[holes + (pre & 0xFFFF)] = i;
    if (mover) from[movers + (pre >> 16)] = i;
    if (i < nlen && keep) {
      osc[i] = sc[i];
      ops[i] = ps[i];
    }
    holes += total & 0xFFFF;
    movers += total >> 16;
  }
  if (tid == 0) a.moves[row] = movers;
  __threadfence_block();
  __syncthreads();
  for (int j = tid; j < movers; j += kEvictThreads) {
    osc[to[j]] = sc[from[j]];
    ops[to[j]] = ps[from[j]];
  }
}

// Evict, moves: keys and values of the listed slots, 16 bytes a thread.
__global__ __launch_bounds__(256) void kv_evict_move_kernel(EvictArgs a, int vecs) {
  const int row = blockIdx.x, b = row / a.heads, h = row - b * a.heads;
  const int n = a.moves[row] * vecs;
  const int32_t* from = a.moves + a.rows + (int64_t)row * 2 * a.budget;
  const int32_t* to = from + a.budget;
  const int32_t* table = a.c.table + (int64_t)b * a.c.width;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < n; i += gridDim.y * 256) {
    const int j = i / vecs, d = (i - j * vecs) * 16;
    const int s = from[j], t = to[j];
    const int ps = page_id(a.c, table, s), pt = page_id(a.c, table, t);
    if (ps < 0 || pt < 0) continue;
    const int so = s - (int)page_of(a.c.div, s) * a.c.div.size, to_ = t - (int)page_of(a.c.div, t) * a.c.div.size;
    const uint4 k = *(const uint4*)(a.c.k + ps * a.c.k_page + h * a.c.k_head + so * a.c.k_slot + d);
    const uint4 v = *(const uint4*)(a.c.v + ps * a.c.v_page + h * a.c.v_head + so * a.c.v_slot + d);
    *(uint4*)(a.c.k + pt * a.c.k_page + h * a.c.k_head + to_ * a.c.k_slot + d) = k;
    *(uint4*)(a.c.v + pt * a.c.v_page + h * a.c.v_head + to_ * a.c.v_slot + d) = v;
  }
}

// No sequence can be longer than the table's capacity.
static int64_t clamp_budget(int64_t budget, int64_t capacity) {
  return budget > capacity ? (capacity > 0 ? capacity : 1) : budget;
}

}  // namespace tx

using namespace tx;

extern "C" {

int tallax_kv_append(const tallax_kv_cache* cache, const int32_t* lens, const int32_t* counts, const void* k_new,
                     const void* v_new, int64_t tokens, float* scores, int32_t* positions, const int32_t* seen,
                     int32_t* out_lens, tallax_stream_t stream) {
  AppendArgs a;
  int st = make_kv_view(cache, "kv_append", &a.c);
  if (st != kOk) return st;
  if (tokens < 0 || tokens > (1 << 24)) {
    set_error("kv_append: %lld tokens (0 to 2^24)", (long long)tokens);
    return kInvalidArgument;
  }
  if (cache->batch == 0) return kOk;
  if (!lens || !out_lens || lens == out_lens || (tokens > 0 && (!k_new || !v_new)) || (!scores != !positions) ||
      (scores && !seen)) {
    set_error("kv_append: null pointer, out_lens the same as lens, or scores without positions and seen");
    return kInvalidArgument;
  }
  if (((uintptr_t)k_new | (uintptr_t)v_new) & 15) {
    set_error("kv_append: k_new and v_new must be 16-byte aligned");
    return kUnsupported;
  }
  a.lens = lens;
  a.counts = counts;
  a.k_new = (const uint4*)k_new;
  a.v_new = (const uint4*)v_new;
  a.tokens = (int)tokens;
  a.heads = (int)cache->kv_heads;
  a.vecs = cache->dim * (cache->dtype == TALLAX_F32 ? 4 : 2) / 16;
  a.scores = scores;
  a.positions = positions;
  a.seen = seen;
  a.out_lens = out_lens;
  const int64_t blocks = (tokens * a.heads * a.vecs + 255) / 256;
  const int64_t most = 65536 / cache->batch + 1;  // enough workgroups to fill the card, then strides
  const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks > most ? most : blocks), (unsigned)cache->batch);
  kv_append_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(a);
  return launch_status("kv_append");
}

size_t tallax_kv_evict_workspace_size(const tallax_kv_cache* cache, int64_t budget) {
  if (!cache || budget < 0 || cache->batch < 0 || cache->kv_heads < 0 || cache->table_width < 0) return 0;
  budget = clamp_budget(budget, cache->table_width * cache->page_size);
  return (size_t)(cache->batch * cache->kv_heads) * (1 + 2 * (size_t)budget) * 4;
}

int tallax_kv_evict(const tallax_kv_cache* cache, const int32_t* lens, const float* scores, const int32_t* positions,
                    const int32_t* seen, int64_t budget, int64_t recent, int64_t sinks, int32_t* out_lens,
                    float* out_scores, int32_t* out_positions, void* workspace, size_t workspace_bytes,
                    tallax_stream_t stream) {
  EvictArgs a;
  int st = make_kv_view(cache, "kv_evict", &a.c);
  if (st != kOk) return st;
  if (budget < 1 || budget > INT32_MAX || recent < 0 || sinks < 0 || recent + sinks > budget) {
    set_error("kv_evict: budget %lld, recent %lld, sinks %lld (budget >= 1, recent + sinks <= budget)",
              (long long)budget, (long long)recent, (long long)sinks);
    return kInvalidArgument;
  }
  if (cache->batch == 0) return kOk;
  if (!lens || !seen || !out_lens || (a.c.capacity && (!scores || !positions || !out_scores || !out_positions)) ||
      (scores && scores == out_scores) || (positions && positions == out_positions)) {
    set_error("kv_evict: null pointer, or an output that is its input");
    return kInvalidArgument;
  }
  budget = clamp_budget(budget, a.c.capacity);
  const size_t bytes = tallax_kv_evict_workspace_size(cache, budget);
  if (!workspace || workspace_bytes < bytes) {
    set_error("kv_evict: workspace of %zu bytes, %zu needed", workspace_bytes, bytes);
    return kWorkspaceTooSmall;
  }
  a.lens = lens;
  a.scores = scores;
  a.positions = positions;
  a.seen = seen;
  a.heads = (int)cache->kv_heads;
  a.budget = (int)budget;
  a.recent = (int)recent;
  a.sinks = (int)sinks;
  a.out_lens = out_lens;
  a.out_scores = out_scores;
  a.out_positions = out_positions;
  a.moves = (int32_t*)workspace;
  a.rows = (int)(cache->batch * cache->kv_heads);
  hipStream_t s = (hipStream_t)stream;
  kv_evict_select_kernel<<<a.rows, kEvictThreads, 0, s>>>(a);
  st = launch_status("kv_evict");
  if (st != kOk) return st;
  const int vecs = cache->dim * (cache->dtype == TALLAX_F32 ? 4 : 2) / 16;
  const int64_t room = a.c.capacity - budget;  // at most this many slots move
  const int64_t most = (budget < room ? budget : room) * vecs;
  const int64_t want = (most + 255) / 256, cap = 4096 / a.rows + 1;
  if (want > 0)
    kv_evict_move_kernel<<<dim3(a.rows, (unsigned)(want < cap ? want : cap)), 256, 0, s>>>(a, vecs);
  return launch_status("kv_evict");
}

}  // extern "C"
