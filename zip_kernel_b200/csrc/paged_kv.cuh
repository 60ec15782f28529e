// The paged key/value cache as kernels see it, and the sequences of a call.
//
// A page holds `page` slots of every key/value head; sequence b's slot j is slot j % page of page table[b][j / page].
// The lengths count the slots in use with the call's new tokens among them, so new token i of sequence b has slot
// lengths[b] - q_len + i and sees the slots up to its own.  Table, lengths and offsets are data on the device that no
// host check has seen: every kernel clamps what it reads from them and records the device error word where it had to.
#pragma once

#include <cuda_bf16.h>

#include <cstring>
#include <type_traits>

#include "common.cuh"

namespace w4a4 {
namespace kv {

enum : int { SITE_KV_PAGE = 32, SITE_KV_SEQ, SITE_KV_POS };

struct Cache {
  void* k;
  void* v;
  long long k_page, k_head, k_slot;      // strides in elements; the elements of a row are neighbours
  long long v_page, v_head, v_slot;
  const int32_t* table;
  long long table_stride;
  int n_pages, page, n_kv, dim, n_seqs, max_pages;
};

// New tokens and cache lengths of the sequences of a call.
struct Seqs {
  const int32_t* cu;        // n_seqs + 1: first token of each sequence, and the end of the last
  const int32_t* lengths;   // n_seqs
  int n, T, max_slots, max_q;
};

struct Seq {
  int q0, q_len, len;
};

// Reads sequence b.  What cannot be true is cut to what can and reported; `n` is the length as it was given.
__device__ __forceinline__ Seq load_seq(const Seqs& s, int b, int& n) {
  const int c0 = ld_plain(s.cu + b), c1 = ld_plain(s.cu + b + 1);
  n = ld_plain(s.lengths + b);
  Seq r;
  r.q0 = min(max(c0, 0), s.T);
  r.q_len = min(max(c1, r.q0), s.T) - r.q0;
  r.len = min(max(n, 0), s.max_slots);
  if (r.q0 != c0 || r.q0 + r.q_len != c1 || r.len != n || r.q_len > s.max_q) record_error(SITE_KV_SEQ, b);
  r.q_len = min(r.q_len, s.max_q);
  return r;
}
__device__ __forceinline__ Seq load_seq(const Seqs& s, int b) {
  int n;
  return load_seq(s, b, n);
}

// Page number of `slot` of sequence b, or -1 (reported) when the table holds none of the cache's.
__device__ __forceinline__ int page_of(const Cache& c, int b, int slot_page) {
  const int p = ld_plain(c.table + (long long)b * c.table_stride + slot_page);
  if ((unsigned)p < (unsigned)c.n_pages) return p;
  record_error(SITE_KV_PAGE, b);
  return -1;
}

// Position in the row of all tiles of a call that a persistent kernel cuts into equal runs: sequences in order, in each
// the key/value heads, in each the row tiles, in each the slot tiles.  Params has a cache c and sequences s;
// unit_shape(p, seq, row_tiles, tiles) beside it says how many of each a sequence has.
template <typename Params>
struct Walk {
  int b, head, row_tile, tile;
  int row_tiles, tiles;
  Seq q;
  long long at;               // global tile number

  __device__ __forceinline__ void set_seq(const Params& p, int seq) {
    b = seq;
    q = load_seq(p.s, b);
    unit_shape(p, q, row_tiles, tiles);
  }
  // Whole warp: all tiles of the call, run c of min(grid, total), and this walk at its first tile; false when there is
  // no such run.  The first 32 sequences are read once for both.
  __device__ __forceinline__ bool start(const Params& p, int grid, int c, long long& total, long long& runs, long long& begin, long long& end) {
    const int lane = threadIdx.x & 31;
    Seq first{};
    int rt0 = 0, n0 = 0;
    if (lane < p.s.n) {
      first = load_seq(p.s, lane);
      unit_shape(p, first, rt0, n0);
    }
    long long w0 = (long long)rt0 * n0 * p.c.n_kv;
    scan(w0);
    total = 0;
    for (int i = 32 + lane; i < p.s.n; i += 32) {
      int rt, n;
      unit_shape(p, load_seq(p.s, i), rt, n);
      total += (long long)rt * n * p.c.n_kv;
    }
    if (p.s.n > 32)
#pragma unroll
      for (int o = 16; o > 0; o /= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
    const long long head0 = __shfl_sync(0xffffffffu, w0, 31);
    total += head0;
    runs = min((long long)grid, total);
    if (c >= runs) return false;
    begin = c * total / runs;
    end = (c + 1) * total / runs;
    at = begin;
    if (begin < head0) {
      const int i = __ffs(__ballot_sync(0xffffffffu, w0 > begin)) - 1;
      const long long before = __shfl_sync(0xffffffffu, w0, (i - 1) & 31);
      b = i;
      q.q0 = __shfl_sync(0xffffffffu, first.q0, i);
      q.q_len = __shfl_sync(0xffffffffu, first.q_len, i);
      q.len = __shfl_sync(0xffffffffu, first.len, i);
      unit_shape(p, q, row_tiles, tiles);
      inside(begin - (i ? before : 0));
      return true;
    }
    long long before = head0;
    for (int base = 32; base < p.s.n; base += 32) {
      int rt = 0, n = 0;
      if (base + lane < p.s.n) unit_shape(p, load_seq(p.s, base + lane), rt, n);
      long long w = (long long)rt * n * p.c.n_kv;
      scan(w);
      const unsigned past = __ballot_sync(0xffffffffu, before + w > begin);
      if (past) {
        const int i = __ffs(past) - 1;
        const long long w1 = __shfl_sync(0xffffffffu, w, (i - 1) & 31);
        set_seq(p, base + i);
        inside(begin - before - (i ? w1 : 0));
        return true;
      }
      before += __shfl_sync(0xffffffffu, w, 31);
    }
    return false;                                            // (not reached: begin is below the total)
  }
  __device__ __forceinline__ static void scan(long long& w) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long a = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += a;
    }
  }
  __device__ __forceinline__ void inside(long long rem) {
    const long long per_head = (long long)row_tiles * tiles;
    head = (int)(rem / per_head);
    const long long r2 = rem - head * per_head;
    row_tile = (int)(r2 / tiles);
    tile = (int)(r2 - (long long)row_tile * tiles);
  }
  // to the first tile of the next unit (there is one)
  __device__ __forceinline__ void next_unit(const Params& p) {
    at += tiles - tile;
    tile = 0;
    if (++row_tile < row_tiles) return;
    row_tile = 0;
    if (++head < p.c.n_kv) return;
    head = 0;
    do set_seq(p, b + 1); while (row_tiles == 0);
  }
  __device__ __forceinline__ long long unit_first() const { return at - tile; }
};

// Page numbers of a sequence's copy boxes (`box` slots each, none crosses a page), 32 at a time in the lanes of the warp
// that issues the copies, and the next 32 already asked for: a look-up per tile would put a load's latency, longer than a
// tile takes to arrive, between any two tiles.
struct PagesAhead {
  int b = -1, base = 0, cur = 0, nxt = 0;

  __device__ __forceinline__ int load(const Cache& c, int len, int box, int i) const {
    const long long slot = (long long)i * box;
    if (slot >= len) return -1;
    const int page = page_of(c, b, (int)(slot / c.page));
    return page < 0 ? c.n_pages : page;                      // past the end of the map: reads zeros
  }
  // Whole warp: the page of box first + lane of sequence seq, for lane < TILE / box; -1 where no slot is in use.  `first`
  // is a multiple of TILE / box, a power of two up to 32.
  __device__ __forceinline__ int get(const Cache& c, int seq, int len, int box, int first) {
    const int lane = threadIdx.x & 31, want = first & ~31;
    if (seq != b || want != base) {
      const bool next = seq == b && want == base + 32;
      b = seq;
      base = want;
      cur = next ? nxt : load(c, len, box, want + lane);
      nxt = load(c, len, box, want + 32 + lane);
    }
    return __shfl_sync(0xffffffffu, cur, (first - base + lane) & 31);
  }
};

// ---------------------------------------------------------------- 16-bit float types
template <typename T> struct Half2Of;
template <> struct Half2Of<__half> { typedef __half2 type; };
template <> struct Half2Of<__nv_bfloat16> { typedef __nv_bfloat162 type; };

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  typename Half2Of<T>::type h;
  memcpy(&h, &v, 4);
  if constexpr (std::is_same<T, __half>::value) return __half22float2(h);
  else return __bfloat1622float2(h);
}
// two floats, each rounded once to nearest even; `lo` in the lower half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t v;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// Weights are taken relative to a base below the maximum of their row, so that the largest is 2^SHIFT.  As fp16 relative to
// the maximum itself, weights below 2^-25 would be lost, and in a long history with one slot far ahead whose values
// are near zero they can be all there is to see.  Sums and outputs are larger by the same factor, which the quotient removes.
// The subtraction rounds up: where a step of the maximum is coarse, no weight may exceed the type's range.
template <typename T> constexpr float WEIGHT_SHIFT = std::is_same<T, __half>::value ? 15.f : 0.f;
__device__ __forceinline__ float below_max(float top, float shift) { return __fadd_ru(top, -shift); }
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// cp.async.bulk.tensor of a 4-D box {element, slot, head, page}
__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const void* tmap, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

}  // namespace kv
}  // namespace w4a4
