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
// Append: one thread per 16 bytes of a new key and of its value.  Bound by
// memory: 8 sequences x 2047 tokens x 8 heads of 128, 135 MB, 28 us (4.8 TB/s).
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
// score), read once, four neighbours a lane, and held in LDS (those past what LDS
// holds, 32 for each of 1024 threads, are read again in every pass); three radix
// steps of 11, 11 and 10 bits find the key of the budget-th largest.  (The first digit is a score's
// exponent and two bits more: with 8 bits most lanes of a wave raise the same
// counter of LDS, one after the other.)  A wave holds neighbouring slots, so
// that places in slot order are popcounts in the wave and one exchange of the
// waves' totals.  What is kept in place is written here, the free places and
// the slots that move into them are listed for the second kernel.
// [8 x 8 heads, 32768 slots, 4095 kept]: 36 us on 64 workgroups, and 54 us for the
// moves (230 MB, 4.3 TB/s); [64 x 8, 2176 slots, 2048 kept]: 15 and 9 us.
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
  int vecs;        // 16-byte vectors of a slot's key
};

// What follows the choice, by threads first, first + step, ...: keys and values
// of the listed slots, 16 bytes a thread, with their scores and positions; and
// what no choice was needed for: rows within the budget are copied, slots past
// the new length cleared.
__device__ __forceinline__ void finish_row(const EvictArgs& a, int row, int first, int step) {
  const int b = row / a.heads, h = row - b * a.heads, vecs = a.vecs;
  const int n = a.moves[row] * vecs, cap = a.c.capacity;
  const int len = min(max(a.lens[b], 0), cap);
  const int64_t at = (int64_t)row * cap;
  const int32_t* from = a.moves + a.rows + (int64_t)row * 2 * a.budget;
  const int32_t* to = from + a.budget;
  const int32_t* table = a.c.table + (int64_t)b * a.c.width;
  for (int i = first; i < n; i += step) {
    const int j = i / vecs, d = (i - j * vecs) * 16;
    const int s = from[j], t = to[j];
    if (d == 0) {
      a.out_scores[at + t] = a.scores[at + s];
      a.out_positions[at + t] = a.positions[at + s];
    }
    const int ps = page_id(a.c, table, s), pt = page_id(a.c, table, t);
    if (ps < 0 || pt < 0) continue;
    const int so = s - (int)page_of(a.c.div, s) * a.c.div.size, to_ = t - (int)page_of(a.c.div, t) * a.c.div.size;
    const uint4 k = *(const uint4*)(a.c.k + ps * a.c.k_page + h * a.c.k_head + so * a.c.k_slot + d);
    const uint4 v = *(const uint4*)(a.c.v + ps * a.c.v_page + h * a.c.v_head + so * a.c.v_slot + d);
    *(uint4*)(a.c.k + pt * a.c.k_page + h * a.c.k_head + to_ * a.c.k_slot + d) = k;
    *(uint4*)(a.c.v + pt * a.c.v_page + h * a.c.v_head + to_ * a.c.v_slot + d) = v;
  }
  const int whole = len <= a.budget ? len : 0;
  for (int i = first; i < whole; i += step) {
    a.out_scores[at + i] = a.scores[at + i];
    a.out_positions[at + i] = a.positions[at + i];
  }
  for (int i = min(len, a.budget) + first; i < cap; i += step) {
    a.out_scores[at + i] = 0.0f;
    a.out_positions[at + i] = -1;
  }
}

// Lanes below this one whose bit is set.
__device__ __forceinline__ int lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// NW waves; `room` groups of four slots of each thread in LDS.  MOVE: the moves
// are made here too.
template <int NW, bool MOVE>
__global__ __launch_bounds__(NW * kWave) void kv_evict_select_kernel(EvictArgs a, int room) {
  constexpr int kThreads = NW * kWave, kBins = 2048, kBinsOf = kBins / kThreads, kGroup = 4 * kWave;
  extern __shared__ uint4 held[];  // [room][kThreads]
  __shared__ int hist[kBins];
  __shared__ int red[NW], red2[NW];
  __shared__ int found[3];
  const int row = blockIdx.x, b = row / a.heads, tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const int cap = a.c.capacity;
  const int len = min(max(a.lens[b], 0), cap);
  const int nlen = min(len, a.budget);
  const int64_t at = (int64_t)row * cap;
  const float* sc = a.scores + at;
  const int32_t* ps = a.positions + at;
  if (row % a.heads == 0 && tid == 0) a.out_lens[b] = nlen;
  if (len <= a.budget) {
    if (tid == 0) a.moves[row] = 0;
    if constexpr (MOVE) {
      __syncthreads();
      finish_row(a, row, tid, kThreads);
    }
    return;
  }
  // this wave's slots: first + 256 j + 4 lane + k, j < count, k < 4
  const int count = (len + 4 * kThreads - 1) / (4 * kThreads);
  const int first = wave * count * kGroup + 4 * lane;
  const int64_t newest = (int64_t)a.seen[b] - a.recent;
  struct Four {
    float x[4];
    int32_t p[4];
  };
  auto read_four = [&](int i, Four& f) {
    if (i + 4 <= len) {
      __builtin_memcpy(f.x, sc + i, 16);
      __builtin_memcpy(f.p, ps + i, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f.x[k] = sc[min(i + k, len - 1)];
        f.p[k] = ps[min(i + k, len - 1)];
      }
    }
  };
  auto keys_from = [&](int i, const Four& f) -> uint4 {
    uint32_t key[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      key[k] = f.p[k] < a.sinks || f.p[k] >= newest ? 0xFFFFFFFFu : select_key(__float_as_uint(f.x[k]));
      if (i + k >= len) key[k] = 0u;  // below every key
    }
    return make_uint4(key[0], key[1], key[2], key[3]);
  };
  const int in_lds = min(count, room);
  {
    Four next = {};
    if (in_lds > 0) read_four(first, next);
#pragma unroll 2
    for (int j = 0; j < in_lds; ++j) {
      const Four now = next;
      if (j + 1 < in_lds) read_four(first + (j + 1) * kGroup, next);
      held[j * kThreads + tid] = keys_from(first + j * kGroup, now);
    }
  }
  // f(slot, keys, scores and positions of four) for this thread's slots in order; all lanes of a wave take part in
  // every call.  Scores and positions are there for slots below `with` and where the keys are not held; they are
  // asked for one call ahead.  The loop is not unrolled: a workgroup runs it a few times, and what it waits for then
  // is its instructions.
  auto each = [&](int with, auto f) {
    Four next = {};
    if (in_lds == 0 || first < with) read_four(first, next);
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const Four now = next;
      const int i = first + j * kGroup;
      if (j + 1 < count && (j + 1 >= in_lds || i + kGroup < with)) read_four(i + kGroup, next);
      const uint4 four = j < in_lds ? held[j * kThreads + tid] : keys_from(i, now);
      const uint32_t key[4] = {four.x, four.y, four.z, four.w};
      f(i, key, now);
    }
  };
  // the budget-th largest key, and how many of its equals are kept
  uint32_t prefix = 0, fixed = 0;  // bits below `fixed` are 0 in the prefix: any key from it on is kept
  int need = a.budget;
  bool all = false;  // of its equals
#pragma unroll 1
  for (int shift = 21; shift >= 0 && !all; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
    const uint32_t digit = shift ? 2047u : 1023u;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    each(0, [&](int i, const uint32_t (&key)[4], const Four&) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < len && ((key[k] ^ prefix) & fixed) == 0) atomicAdd(&hist[(key[k] >> shift) & digit], 1);
    });
    __syncthreads();
    int c[kBinsOf], s = 0;  // bins from the largest digit down
#pragma unroll
    for (int j = 0; j < kBinsOf; ++j) s += c[j] = hist[kBins - 1 - tid * kBinsOf - j];
    int total;
    int above = block_exscan<NW>(s, red, total);
#pragma unroll
    for (int j = 0; j < kBinsOf; ++j) {
      if (above < need && need <= above + c[j]) {
        found[0] = kBins - 1 - tid * kBinsOf - j;
        found[1] = need - above;
        found[2] = c[j];
      }
      above += c[j];
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    fixed = ~0u << shift;
    need = found[1];
    all = need == found[2];
  }
  // places in slot order: of the ties, then of the free places and of the slots that move
  auto before = [&](int mine, int* shared) {
    if (lane == 0) shared[wave] = mine;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) n += w < wave ? shared[w] : 0;
    return n;
  };
  int first_tie = 0;
  if (!all) {
    int ties = 0;
    each(0, [&](int i, const uint32_t (&key)[4], const Four&) {
#pragma unroll
      for (int k = 0; k < 4; ++k) ties += __popcll(__ballot(i + k < len && key[k] == prefix));
    });
    __syncthreads();  // red has been read
    first_tie = before(ties, red);
  }
  int32_t* from = a.moves + a.rows + (int64_t)row * 2 * a.budget;
  int32_t* to = from + a.budget;
  float* osc = a.out_scores + at;
  int32_t* ops = a.out_positions + at;
  int hole = 0, mover = 0;
  // the first time only counts the free places and the slots that move
#pragma unroll 1
  for (int write = 0; write < 2; ++write) {
    int tie = first_tie;
    each(write ? nlen : 0, [&](int i, const uint32_t (&key)[4], const Four& here) {
      bool keep[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = i + k < len && key[k] >= prefix;
      if (!all) {
        int rank = tie;
        bool equal[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          equal[k] = i + k < len && key[k] == prefix;
          const uint64_t e = __ballot(equal[k]);
          rank += lanes_below(e);
          tie += __popcll(e);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          keep[k] = keep[k] && (!equal[k] || rank < need);
          rank += equal[k];
        }
      }
      int h = hole, m = mover;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t bh = __ballot(i + k < nlen && !keep[k]), bm = __ballot(i + k >= nlen && keep[k]);
        h += lanes_below(bh);
        m += lanes_below(bm);
        hole += __popcll(bh);
        mover += __popcll(bm);
      }
      if (!write) return;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i + k < nlen) {
          if (keep[k]) {
            osc[i + k] = here.x[k];
            ops[i + k] = here.p[k];
          } else {
            to[h++] = i + k;
          }
        } else if (keep[k]) {
          from[m++] = i + k;
        }
      }
    });
    if (write) break;
    __syncthreads();  // red has been read
    const int total = mover;
    hole = before(hole, red);
    mover = before(mover, red2);
    if (wave == NW - 1 && lane == 0) a.moves[row] = mover + total;
  }
  if constexpr (MOVE) {
    __syncthreads();  // the lists are written
    finish_row(a, row, tid, kThreads);
  }
}

// Evict, moves, by workgroups of their own.
__global__ __launch_bounds__(256) void kv_evict_move_kernel(EvictArgs a) {
  finish_row(a, blockIdx.x, blockIdx.y * 256 + threadIdx.x, gridDim.y * 256);
}

template <int NW, bool MOVE>
static int launch_select(const EvictArgs& a, hipStream_t s) {
  constexpr int kThreads = NW * kWave, kMost = 8;
  const int64_t each = ((int64_t)a.c.capacity + 4 * kThreads - 1) / (4 * kThreads);
  const int room = (int)(each < kMost ? each : kMost), bytes = room * kThreads * 16;
  if (bytes > 48 * 1024) {
    const hipError_t e = set_dynamic_lds_limit((const void*)kv_evict_select_kernel<NW, MOVE>, kMost * kThreads * 16, s);
    if (e != hipSuccess) {
      set_error("kv_evict: %s", hipGetErrorString(e));
      return kHipError;
    }
  }
  kv_evict_select_kernel<NW, MOVE><<<a.rows, kThreads, bytes, s>>>(a, room);
  return launch_status("kv_evict");
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
  st = check_workspace("kv_evict", workspace, workspace_bytes, tallax_kv_evict_workspace_size(cache, budget));
  if (st != kOk) return st;
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
  a.vecs = cache->dim * (cache->dtype == TALLAX_F32 ? 4 : 2) / 16;
  const int64_t room = a.c.capacity - budget;  // at most this many slots move
  const int64_t most = (budget < room ? budget : room) * a.vecs;
  // Short rows whose moves are few make them in the same launch: 2 x 2 rows of 100 slots 8.0 us against 12.9, 2048 of
  // 700 24.1 against 27.3.  (Many moves are shared out over more workgroups, each of which moves some 30 GB/s.)
  if (a.c.capacity <= 1024 && most <= 4096) return launch_select<4, true>(a, s);
  st = a.c.capacity <= 1024   ? launch_select<4, false>(a, s)
       : a.c.capacity <= 4096 ? launch_select<8, false>(a, s)
                              : launch_select<16, false>(a, s);
  if (st != kOk) return st;
  const int64_t want = ((most > a.c.capacity ? most : a.c.capacity) + 255) / 256, limit = 4096 / a.rows + 1;
  kv_evict_move_kernel<<<dim3(a.rows, (unsigned)(want < limit ? want : limit)), 256, 0, s>>>(a);
  return launch_status("kv_evict");
}

}  // extern "C"
