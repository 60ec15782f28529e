// Eviction from a paged cache by accumulated weight: for each sequence and key/value head the first `sink` slots, the
// last `recent` ones and those with the largest sums in between, `budget` in all (equal sums: the lowest slots), move in
// their order to the slots 0, 1, ... of the destination.  A sequence of at most `budget` slots keeps them all.
//
// Two launches.  select: a block per (sequence, head) finds the smallest sum that stays by a radix selection, 11, 11 and 10
// bits of an order-preserving integer form of the float at a time, then walks the slots once in order and writes the list of
// those kept and their sums.  move: copies the rows of the list.  In place a row's new slot is never above its old one,
// so rows may be written in ascending order once all rows up to them have been read; the columns of a row are
// independent of one another, and a block takes a few columns of all rows of one (sequence, head).  Into another cache
// the rows are independent too and are split over blocks.
//
// What bounds it: the rows kept are read and written once; the selection holds up to 8192
// sums in registers and reads longer ones again from L2.
#pragma once

#include "paged_kv.cuh"

namespace w4a4 {
namespace evict {

using namespace kv;

constexpr int SELECT_THREADS = 1024, SELECT_WARPS = SELECT_THREADS / 32, BINS = 2048;
constexpr int KEYS = 8;                                      // keys a thread holds; longer sequences are read again every pass
constexpr int MOVE_THREADS = 256, MOVE_CHUNKS = 8, MOVE_UNROLL = 8, MOVE_ROWS = MOVE_THREADS / MOVE_CHUNKS * MOVE_UNROLL;
static_assert(MOVE_ROWS == MOVE_THREADS, "a thread locates one row of a batch");

struct SelectParams {
  const int32_t* lengths;
  const float* sums;
  long long sums_seq, sums_head;
  int32_t* kept;              // (n_seqs, n_kv, budget)
  int32_t* new_lengths;
  float* new_sums;            // (n_seqs, n_kv, new_slots)
  int n_kv, max_slots, new_slots, budget, sink, recent;
};

// Unsigned integers in the order of the floats: both zeros alike, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(const SelectParams p) {
  __shared__ int hist[BINS];
  __shared__ int warp_sums[2][2][SELECT_WARPS];
  __shared__ int s_bin, s_left, s_count;
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / p.n_kv, g = blockIdx.x % p.n_kv;
  grid_dependency_wait();
  const int len = ld_plain(p.lengths + b), n = min(max(len, 0), p.max_slots);
  if (n != len && tid == 0) record_error(SITE_KV_SEQ, b);
  const int n_new = min(n, p.budget);
  if (g == 0 && tid == 0) p.new_lengths[b] = n_new;
  const float* sums = p.sums + (long long)b * p.sums_seq + (long long)g * p.sums_head;
  int32_t* kept = p.kept + ((long long)b * p.n_kv + g) * p.budget;
  float* out = p.new_sums + ((long long)b * p.n_kv + g) * p.new_slots;

  if (n <= p.budget) {
    for (int j = tid; j < n; j += SELECT_THREADS) {
      kept[j] = j;
      out[j] = ld_plain(sums + j);
    }
  } else {
    const int lo = p.sink, hi = n - p.recent;              // candidates; the rest stays anyway (sink + recent <= budget < n)
    int left = p.budget - p.sink - p.recent;               // how many of them stay
    const bool any = left > 0, held = n <= KEYS * SELECT_THREADS;
    float v[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = i * SELECT_THREADS + tid;
      v[i] = held && j < n ? ld_plain(sums + j) : 0.f;
    }
    uint32_t prefix = 0;                                   // leading bits of the smallest key that stays
#pragma unroll 1
    for (int pass = 0; any && pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < BINS; i += SELECT_THREADS) hist[i] = 0;
      __syncthreads();
      auto count = [&](int j, float x) {
        if (j < lo || j >= hi) return;
        const uint32_t k = order_key(x);
        if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1);
      };
      if (held) {
#pragma unroll
        for (int i = 0; i < KEYS; ++i) count(i * SELECT_THREADS + tid, v[i]);
      } else {
        for (int j = lo + tid; j < hi; j += SELECT_THREADS) count(j, ld_plain(sums + j));
      }
      __syncthreads();
      // bins from the top, two a thread: the one in which the count reaches `left`
      const int h0 = hist[BINS - 1 - 2 * tid], h1 = hist[BINS - 2 - 2 * tid];
      int above = h0 + h1;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += a;
      }
      if (lane == 31) warp_sums[0][0][warp] = above;
      __syncthreads();
      above += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[0][0][lane] : 0) - h0 - h1;
      if (above < left && left <= above + h0 + h1) {
        const bool second = left > above + h0;
        s_bin = BINS - 1 - 2 * tid - (second ? 1 : 0);
        s_left = left - above - (second ? h0 : 0);
        s_count = second ? h1 : h0;
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      left = s_left;
      if (left == s_count) break;                          // the whole bin stays: its lowest key is the border
    }
    // Now `prefix` is the smallest key that stays, or below it and above all that go, and `left` how many slots with
    // just that leading part stay: the first ones.
    int done = 0, ties = 0;                                // slots kept, and slots with the border's key, before this round
    auto place = [&](int j, float x, int round) {
      bool sure = false, tie = false;
      if (j < n) {
        const uint32_t k = order_key(x);
        const bool free = j >= lo && j < hi;
        sure = !free || (any && k > prefix);
        tie = free && any && k == prefix;
      }
      const unsigned ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie), before = (1u << lane) - 1;
      int(*sums_of)[SELECT_WARPS] = warp_sums[round & 1];  // (two in turn: one barrier a round)
      if (lane == 0) { sums_of[0][warp] = __popc(ms); sums_of[1][warp] = __popc(mt); }
      __syncthreads();
      const int ws = sums_of[0][lane], wt = sums_of[1][lane];
      const int s_before = __reduce_add_sync(0xffffffffu, lane < warp ? ws : 0) + __popc(ms & before);
      const int t_before = ties + __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0) + __popc(mt & before);
      const int s_all = __reduce_add_sync(0xffffffffu, ws), t_all = __reduce_add_sync(0xffffffffu, wt);
      if (sure || (tie && t_before < left)) {
        const int to = done + s_before + min(t_before, left) - min(ties, left);
        kept[to] = j;
        out[to] = x;
      }
      done += s_all + min(ties + t_all, left) - min(ties, left);
      ties += t_all;
    };
    __syncthreads();
    if (held) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i)
        if (i * SELECT_THREADS < n) place(i * SELECT_THREADS + tid, v[i], i);
    } else {
      for (int base = 0, r = 0; base < n; base += SELECT_THREADS, ++r) place(base + tid, base + tid < n ? ld_plain(sums + base + tid) : 0.f, r);
    }
  }
  for (int j = n_new + tid; j < p.budget; j += SELECT_THREADS) kept[j] = -1;
  for (int j = n_new + tid; j < p.new_slots; j += SELECT_THREADS) out[j] = 0.f;
}

struct MoveParams {
  Cache from, to;
  const int32_t* kept;
  const int32_t* new_lengths;
  int budget;
  int parts, rows_per_part;   // blocks over the rows of one (sequence, head); one when the caches share memory
  int in_place;
};

// A block moves MOVE_CHUNKS 16-byte chunks of each of its rows, MOVE_ROWS rows at a time.  Thread i finds out where row i
// comes from and goes to (list, page tables, divisions: once per row, one batch ahead), then every thread has
// MOVE_UNROLL loads under way before it stores.  Measured (32 x 8 x 2048 rows of 256 bytes, keys and values, into
// another cache): 78 us; with addresses per chunk and four loads under way 173.
__global__ void __launch_bounds__(MOVE_THREADS, 4) evict_move_kernel(const MoveParams p) {
  __shared__ long long s_src[2][MOVE_ROWS], s_dst[2][MOVE_ROWS];      // element offsets; negative: nothing to move
  grid_launch_dependents();
  const int tid = threadIdx.x;
  const int row_chunks = p.from.dim / 8;                   // of a key or value row
  const int slices = 2 * row_chunks / MOVE_CHUNKS;
  const int part = blockIdx.x % p.parts, rest = blockIdx.x / p.parts;
  const int slice = rest % slices, unit = rest / slices;
  const int b = unit / p.from.n_kv, g = unit % p.from.n_kv;
  const bool is_v = slice * MOVE_CHUNKS >= row_chunks;
  const int d = (slice * MOVE_CHUNKS % row_chunks + tid % MOVE_CHUNKS) * 8;
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.from.v : p.from.k) + d;
  uint16_t* dst = static_cast<uint16_t*>(is_v ? p.to.v : p.to.k) + d;
  grid_dependency_wait();
  const int n = min(ld_plain(p.new_lengths + b), p.budget);
  const int first = part * p.rows_per_part, end = min(n, first + p.rows_per_part);
  const int32_t* kept = p.kept + (long long)unit * p.budget;

  long long from = -1, to = -1;
  auto locate = [&](int row0) {
    const int i = row0 + tid;
    from = to = -1;
    if (i >= end) return;
    const int j = ld_plain(kept + i);
    if (p.in_place && j == i) return;
    const int sp = page_of(p.from, b, j / p.from.page), dp = page_of(p.to, b, i / p.to.page);
    if (sp < 0 || dp < 0) return;
    from = is_v ? sp * p.from.v_page + (j % p.from.page) * p.from.v_slot + g * p.from.v_head
                : sp * p.from.k_page + (j % p.from.page) * p.from.k_slot + g * p.from.k_head;
    to = is_v ? dp * p.to.v_page + (i % p.to.page) * p.to.v_slot + g * p.to.v_head
              : dp * p.to.k_page + (i % p.to.page) * p.to.k_slot + g * p.to.k_head;
  };
  locate(first);
  // In place a batch is stored once every thread has loaded its rows of it; rows of later batches lie at or above the
  // batch's end, so the stores touch none that is still to be read.
  for (int row0 = first, buf = 0; row0 < end; row0 += MOVE_ROWS, buf ^= 1) {
    s_src[buf][tid] = from;
    s_dst[buf][tid] = to;
    __syncthreads();
    locate(row0 + MOVE_ROWS);
    uint4 x[MOVE_UNROLL];
#pragma unroll
    for (int u = 0; u < MOVE_UNROLL; ++u) {
      const long long o = s_src[buf][u * (MOVE_ROWS / MOVE_UNROLL) + tid / MOVE_CHUNKS];
      if (o >= 0) x[u] = ld_plain(reinterpret_cast<const uint4*>(src + o));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MOVE_UNROLL; ++u) {
      const int r = u * (MOVE_ROWS / MOVE_UNROLL) + tid / MOVE_CHUNKS;
      if (s_src[buf][r] >= 0) *reinterpret_cast<uint4*>(dst + s_dst[buf][r]) = x[u];
    }
  }
}

}  // namespace evict
}  // namespace w4a4
