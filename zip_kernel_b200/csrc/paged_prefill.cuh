// Attention of many query rows per key/value head over a paged cache: prompts and chunks of them.
//
//   o[r] = sum_j p[r,j] v[j] / sum_j p[r,j],  p[r,j] = exp(scale q[r].k[j] - m[r]),  j up to the row's own slot,
//
// in one pass over 128-slot tiles.  A row = (new token, head of the group that shares the key/value head): a tile of 128
// rows holds whole tokens, so the heads of a group share every key and value tile, and a block has two row tiles, whose
// products and softmax alternate: while the tensor cores work on one, the other's softmax warps have the CUDA cores.
//
// Roles: a warp that plans (finds the CTA's next unit of work and writes it to shared memory), a warp that issues copies
// (TMA boxes of one page each), a thread that issues MMAs, four warps of softmax per row tile.  Scores are 128 x 128 fp32
// in tensor memory, thread = row; the weights go back there as 16-bit pairs over the scores and are the A operand of the
// second product, whose B operand is the value tile as it lands (slots x elements, read along the elements).  The output
// stays in tensor memory; it is multiplied by exp(m_old - m_new) only when some row's maximum has grown by more than a
// factor of 2^8, until when the weights are simply larger (2^8 at most; fp16 weights are 2^7 times as large besides).  A
// weight is rounded to the 16-bit type of the values, as the product demands: half a step of the output's own type.
//
// The order PV(j), S(j + 1) in the issuing thread makes one barrier do for two things: the scores of step j + 1 are
// complete only after the product that reads the weights of step j and writes the output, so the softmax warps may
// overwrite the one and multiply the other.
//
// What bounds it: products and exponentials alike at dim 128, 2048 clocks each per step of both row tiles if each had the SM to
// itself.  A row tile's own chain is longer - scores read 100, maximum 400, weights 1300 to 1500 beside the other tile's,
// then the hand-over and its products - and tensor memory is full (scores and outputs of both row tiles), so the next
// scores cannot be made ahead: a step takes about 3200 clocks.  Measured: 8192-token prompt, 32/8 heads, 495 us, 1110
// TFLOP/s at 1965 MHz (60 calls in a row); 569 us in a row of seconds, in which the power limit holds the clock at 1627 MHz.
// One thread issues the products of both row tiles, in turn: with a thread for each the two fall into step and
// no longer fill each other's pauses (607 us).
#pragma once

#include "cache_sums.cuh"

namespace w4a4 {
namespace ppre {

using namespace kv;
using csum::add_f32x2;
using csum::idesc_f16;
using csum::umma_f16;

constexpr int TILE = 128, ROWS = 128;                        // slots of a tile, rows of a row tile
constexpr int WARP_COPY = 8, WARP_MMA = 9, WARP_PLAN = 10, THREADS = 12 * 32;
constexpr int WORKS = 4;                                     // units planned ahead
constexpr int REG_ISSUE = 88, REG_SOFTMAX = 208;
static_assert(REG_ISSUE + 2 * REG_SOFTMAX <= 3 * 168, "the warpgroups share the registers of the launch");
constexpr int TMEM_COLS = 512, TMEM_O = 256;
// Scores (log2) from which on their product with the scale is rounded before the maximum is taken off: a weight is made with
// one rounding for both, the maximum is a rounded product, and from here on the two may differ by more than half a step of 2.
constexpr float HUGE_SCORE = 4194304.f;
constexpr float GROWTH = 8.f;                                // (log2) of a row's maximum before the output follows
// Below the maximum by less than elsewhere, for the weights may grow by 2^GROWTH: fp16 loses what is below 2^-32 of the largest.
template <typename T> constexpr float SHIFT = WEIGHT_SHIFT<T> > 0.f ? WEIGHT_SHIFT<T> - GROWTH : 0.f;

enum : int { SITE_PPRE_EMPTY = 80, SITE_PPRE_Q, SITE_PPRE_K, SITE_PPRE_V, SITE_PPRE_P, SITE_PPRE_S, SITE_PPRE_VZERO, SITE_PPRE_O, SITE_PPRE_QEMPTY, SITE_PPRE_OEMPTY, SITE_PPRE_WORK, SITE_PPRE_WFREE };

template <int DIM>
struct Layout {
  static constexpr int HALVES = DIM / 64;
  static constexpr int SLOT = TILE * DIM * 2;                // a tile of keys, or of values, or of query rows
  static constexpr int STAGES = DIM == 128 ? 5 : 10;
  static constexpr int q = STAGES * SLOT;
  static constexpr int works = q + 2 * SLOT;                 // Work [WORKS]
  static constexpr int bars = works + WORKS * 64;
  static constexpr int total = bars + (2 * STAGES + 14 + 2 * WORKS) * 8 + 16;
  static constexpr int PART = 2 * ROWS * (DIM + 2);          // of a unit in the workspace: float2 m, l [row], float4 [dim / 4][row]
  static_assert(1024 + total <= 232448, "shared memory of one SM");
};
template <int DIM> inline size_t smem_bytes() { return 1024 + Layout<DIM>::total; }

struct Params {
  Cache c;
  Seqs s;
  void* out;
  long long o_tok, o_head;
  float* lse;                 // (T, n_heads), or NULL
  float* parts;               // [2 * grid][Layout::PART]
  void* joins;                // Join [grid]
  int n_heads, group, box, toks, min_rows;
  float scale_log2;
};

// A unit is a pair of row tiles of one (sequence, key/value head).  All units lie end to end, measured in slots: those that
// a unit's last row sees and PAD more for what a unit costs besides its tiles; the row is cut into one equal run per
// CTA.  A unit that falls into several runs leaves its parts in the workspace, and a second launch joins them in their
// order, spread over the card.  (Joined by the CTA that finished a unit's last part, 64 tokens of 32/8 heads over 8192
// slots took 48 us, half of it one CTA's reads of sixteen parts of 133 KB.)  An 8192-token prompt takes 534, 515, 499 and 495 us
// with a PAD of 192, 256, 320 and 448, chunks of 500, 333 and 166 tokens over up to 7001 slots 112, 100, 93 and 97.
constexpr int PAD = 320;
// Shorter runs cost more in joining than they save: 128 tokens of 32/8 heads over 1024 slots take 23.0 us with two tiles at
// least, 26.3 with four and 32.8 with eight, 64 tokens over 8192 slots 34.6, 33.3 and 36.4.
constexpr int MIN_RUN = 2 * TILE;

struct Unit {
  int b, head, blk, blocks;
  long long past;             // slots before the sequence's new tokens, not below zero
  long long u0, weight;       // place in the row
  Seq q;
};

// Units of sequence b for each head in this kernel.
__device__ __forceinline__ int seq_blocks(const Params& p, const Seq& q) {
  return (long long)q.q_len * p.group > p.min_rows ? (q.q_len + 2 * p.toks - 1) / (2 * p.toks) : 0;
}
// Weight of the first `blk` units of a head, all of them whole.
__device__ __forceinline__ long long blocks_weight(const Params& p, long long past, long long blk) {
  return blk * (PAD + past) + (long long)p.toks * blk * (blk + 1);
}
__device__ __forceinline__ long long head_weight(const Params& p, const Seq& q, int blocks) {
  const long long past = max(q.len - q.q_len, 0);
  return blocks > 0 ? blocks_weight(p, past, blocks - 1) + PAD + past + q.q_len : 0;
}

struct Units {
  long long total, count;     // weight and number of all units (whole warp)
  __device__ __forceinline__ void sum(const Params& p) {
    total = count = 0;
    for (int b = threadIdx.x & 31; b < p.s.n; b += 32) {
      const Seq q = load_seq(p.s, b);
      const int n = seq_blocks(p, q);
      total += head_weight(p, q, n) * p.c.n_kv;
      count += (long long)n * p.c.n_kv;
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
  }
};

__device__ __forceinline__ void unit_weight(const Params& p, Unit& u) {
  u.weight = PAD + u.past + min((u.blk + 1) * 2 * p.toks, u.q.q_len);
}
// The unit at place x of the row, x below the total (whole warp).
__device__ __forceinline__ Unit unit_at(const Params& p, long long x) {
  const int lane = threadIdx.x & 31;
  Unit u{};
  long long before = 0;
  for (int base = 0; base < p.s.n; base += 32) {
    long long w = 0;
    if (base + lane < p.s.n) {
      const Seq q = load_seq(p.s, base + lane);
      w = head_weight(p, q, seq_blocks(p, q)) * p.c.n_kv;
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long a = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += a;
    }
    const unsigned over = __ballot_sync(0xffffffffu, before + w > x);
    if (over) {
      const int i = __ffs(over) - 1;
      const long long w1 = __shfl_sync(0xffffffffu, w, (i - 1) & 31);
      before += i ? w1 : 0;
      u.b = base + i;
      u.q = load_seq(p.s, u.b);
      u.blocks = seq_blocks(p, u.q);
      u.past = max(u.q.len - u.q.q_len, 0);
      const long long per_head = head_weight(p, u.q, u.blocks);
      u.head = (int)((x - before) / per_head);
      const long long start = before + u.head * per_head;
      int lo = 0, hi = u.blocks - 1;                         // the last block that does not start behind x
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (start + blocks_weight(p, u.past, mid) <= x) lo = mid;
        else hi = mid - 1;
      }
      u.blk = lo;
      u.u0 = start + blocks_weight(p, u.past, lo);
      unit_weight(p, u);
      return u;
    }
    before += __shfl_sync(0xffffffffu, w, 31);
  }
  return u;
}
// The next unit (there is one).
__device__ __forceinline__ void next_unit(const Params& p, Unit& u) {
  u.u0 += u.weight;
  if (++u.blk == u.blocks) {
    u.blk = 0;
    if (++u.head == p.c.n_kv) {
      u.head = 0;
      do {
        u.q = load_seq(p.s, ++u.b);
        u.blocks = seq_blocks(p, u.q);
      } while (u.blocks == 0);
      u.past = max(u.q.len - u.q.q_len, 0);
    }
  }
  unit_weight(p, u);
}

// What a run has of a unit, as the planning warp leaves it in shared memory: tiles j0 .. of it, for either row tile up to
// n_row (none when that is j0).
struct Work {
  int live;                   // 0: the run has ended
  int b, head, tok0;          // sequence, key/value head, first token (of the sequence) of the unit
  int q0, q_len, len;
  int j0, n_row[2];
  int whole;                  // the unit is in this run alone
  int part;                   // else its part in the workspace
  int pad[4];
};
static_assert(sizeof(Work) == 64, "the place of one");

// What the second launch needs to know of the unit that is cut for the first time at a run's end (there is one at most).
struct Join {
  int parts;                  // 0: none
  int head, q0, q_len, tok0;
  int pad[3];
};
static_assert(sizeof(Join) == 32, "the place of one");

// descriptor of a B operand whose rows in shared memory are the K side (slots) and run along N (elements): 64 elements
// under the 128-byte swizzle, 8 slots 1024 bytes apart, the next 64 elements `halves` bytes on
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t halves) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(halves >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16 with the A operand in tensor memory (row = lane, two 16-bit values a column)
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t accumulate, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 columns of the calling thread's lane, not waited for
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16_issue(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8_issue(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Largest of three; NaN when one is (unlike fmaxf)
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Slots whose weights are handed over first: late enough that the thread that issues the products is not held up by the
// rest, which the other row tile then waits for.  Measured, 8192-token prompt and chunks of 500, 333 and 166 tokens: 64
// slots 521 and 107 us, 96 503 and 104, 112 494 and 101.
constexpr int EARLY = 112;
// The weights 2^(x * scale - base) of N scores of a row, as 16-bit pairs to tensor memory; returns their sum.  (With one pair
// of four by a polynomial on the multiply-add pipe, to spare the unit for 2^x: prompts the same, chunks 99 us for 96.)
template <typename T, int N>
__device__ __forceinline__ float weights(const uint32_t* x, float scale, float base, uint32_t tp) {
  const f32x2_t scale2 = pack_f32x2(scale, scale), base2 = pack_f32x2(-base, -base);
  f32x2_t sum[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
  static_assert(N % 32 == 0 || N % 32 == 16, "whole chunks");
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const f32x2_t v = fma_f32x2(pack_f32x2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, base2);
    float2 e = unpack_f32x2(v);
    e = make_float2(ex2(e.x), ex2(e.y));
    sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(e.x, e.y));
    w[i % 16] = pack2<T>(e.x, e.y);
    if (i % 16 == 15) tmem_st16_issue(tp + i - 15, w);
    else if (i == N / 2 - 1) tmem_st8_issue(tp + i - 7, w);
  }
  tmem_st_wait();
  const float2 s = unpack_f32x2(add_f32x2(sum[0], sum[1]));
  return s.x + s.y;
}

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_q, const Params p) {
  using L = Layout<DIM>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);    // ring of key and value tiles in turn
  uint64_t* empty = full + L::STAGES;
  uint64_t* q_full = empty + L::STAGES;                          // [2] per row tile, as the next five
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;
  uint64_t* p_full = s_full + 2;                                 // [2][2 halves of the slots]
  uint64_t* o_full = p_full + 4;
  uint64_t* o_empty = o_full + 2;
  uint64_t* w_full = o_empty + 2;                                // [WORKS]
  uint64_t* w_empty = w_full + WORKS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(w_empty + WORKS);
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < L::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < WORKS; ++i) { mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], 10); }
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_q);
  }
  if (warp == WARP_MMA) pre::tmem_alloc(tmem_slot, TMEM_COLS);
  pre::tc_fence_before();
  __syncthreads();
  pre::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (warp == WARP_COPY) grid_dependency_wait_for_async_reads();
  else grid_dependency_wait();

  Work* works = reinterpret_cast<Work*>(sm + L::works);
  bool ok = true;                                          // no wait of this thread has given up
  uint32_t nw = 0;                                         // units taken so far
  // The next unit of work (whole warp), nullptr after the last; handed back with work_done.
  auto next_work = [&]() -> const Work* {
    if (ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&w_full[nw % WORKS], nw / WORKS & 1, SITE_PPRE_WORK));
    return ok && works[nw % WORKS].live ? &works[nw % WORKS] : nullptr;
  };
  auto work_done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&w_empty[nw % WORKS]);
    ++nw;
  };

  if (warp >= WARP_COPY) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_ISSUE));
    if (warp == WARP_PLAN) {
      // ---------------------------------------------------------- planning
      Units all;
      all.sum(p);
      const long long runs = min((long long)gridDim.x, max(all.count, all.total / MIN_RUN)), run = blockIdx.x;
      auto put = [&](const Work& w) {
        if (nw >= WORKS) ok = __all_sync(0xffffffffu, wide::wait_suspend(&w_empty[nw % WORKS], (nw / WORKS - 1) & 1, SITE_PPRE_WFREE));
        if (!ok) return;
        if (lane == 0) {
          works[nw % WORKS] = w;
          mbar_arrive(&w_full[nw % WORKS]);                // (releases the writes before it)
        }
        __syncwarp();
        ++nw;
      };
      Join join{};
      if (run < runs) {
        const long long begin = run * all.total / runs, end = (run + 1) * all.total / runs;
        Unit u = unit_at(p, begin);
        while (ok) {
          Work w{};
          w.live = 1;
          w.b = u.b;
          w.head = u.head;
          w.q0 = u.q.q0;
          w.q_len = u.q.q_len;
          w.len = u.q.len;
          w.tok0 = u.blk * 2 * p.toks;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int t0 = w.tok0 + t * p.toks, t1 = min(t0 + p.toks, w.q_len);
            w.n_row[t] = t0 < w.q_len ? max(0, (w.len - w.q_len + t1 + TILE - 1) / TILE) : 0;
          }
          const int n = max(1, max(w.n_row[0], w.n_row[1]));       // (a unit that sees nothing still has zeros to write)
          const long long first = u.u0 + PAD;              // where the unit's first tile lies in the row
          const int j1 = (int)min((max(end - first, 0LL) + TILE - 1) / TILE, (long long)n);
          w.j0 = (int)min((max(begin - first, 0LL) + TILE - 1) / TILE, (long long)n);
#pragma unroll
          for (int t = 0; t < 2; ++t) w.n_row[t] = max(w.j0, min(j1, w.n_row[t]));
          w.whole = w.j0 == 0 && j1 == n;
          w.part = (int)(2 * run) + (first < begin ? 0 : 1);
          if (w.j0 == 0 && j1 > 0 && j1 < n) {
            // parts: the runs that the unit's tiles fall into; run(x) = the c with c * total / runs <= x < (c + 1) * total / runs
            join.parts = (int)(((first + (long long)(n - 1) * TILE + 1) * runs - 1) / all.total - run) + 1;
            join.head = u.head;
            join.q0 = u.q.q0;
            join.q_len = u.q.q_len;
            join.tok0 = w.tok0;
          }
          if (j1 > w.j0) put(w);
          if (u.u0 + u.weight >= end) break;
          next_unit(p, u);
        }
      }
      if (lane == 0) static_cast<Join*>(p.joins)[run] = join;
      if (ok) put(Work{});
    } else if (warp == WARP_COPY) {
      // ---------------------------------------------------------- copies
      int s = 0;
      uint32_t ph = 1, uses[2] = {0, 0};
      bool lap = false;
      const int boxes = TILE / p.box;                      // at most 8
      PagesAhead pages;
      while (const Work* w = next_work()) {
        const int b = w->b, head = w->head, len = w->len, j0 = w->j0, n_row[2] = {w->n_row[0], w->n_row[1]}, tok = w->q0 + w->tok0;
        work_done();
        for (int t = 0; ok && t < 2; ++t) {
          if (n_row[t] == j0) continue;
          if (uses[t] > 0) ok = __all_sync(0xffffffffu, wide::wait_suspend(&q_empty[t], (uses[t] - 1) & 1, SITE_PPRE_QEMPTY));
          if (!ok) break;
          ++uses[t];
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[t], p.toks * p.group * DIM * 2);
            for (int h = 0; h < L::HALVES; ++h)
              tma_load_3d(sm + L::q + t * L::SLOT + h * ROWS * 128, &tm_q, h * 64, head * p.group, tok + t * p.toks, &q_full[t]);
          }
          __syncwarp();
        }
        const int j_end = max(n_row[0], n_row[1]);
        for (int j = j0; ok && j < j_end; ++j) {
          const int slot = j * TILE + lane * p.box;
          const bool mine = lane < boxes && slot < len;
          const int page = pages.get(p.c, b, len, p.box, j * boxes);
          const int live = __popc(__ballot_sync(0xffffffffu, mine)), in_page = slot % p.c.page;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (lap && ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&empty[s], ph, SITE_PPRE_EMPTY));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], live * p.box * DIM * 2);
            __syncwarp();
            if (mine)
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h)
                tma_load_4d(smem_u32(sm) + s * L::SLOT + h * TILE * 128 + lane * p.box * 128, kv ? &tm_v : &tm_k, h * 64, in_page,
                            head, page, &full[s]);
            if (++s == L::STAGES) { s = 0; ph ^= 1; lap = true; }
          }
        }
      }
    } else if (warp == WARP_MMA && csum::elected()) {
      // ---------------------------------------------------------- MMAs: one thread
      const uint32_t id_s = idesc_f16<T>(TILE), id_o = idesc_f16<T>(DIM) | (1u << 16);
      int s = 0;
      uint32_t ph = 0, uses[2] = {0, 0}, steps[2] = {0, 0};
      auto next = [&]() { if (++s == L::STAGES) { s = 0; ph ^= 1; } };
      auto scores = [&](int t, int slot, bool last) {
#pragma unroll
        for (int h = 0; h < L::HALVES; ++h) {
          const uint64_t a = pre::smem_desc_sw128(sm + L::q + t * L::SLOT + h * ROWS * 128);
          const uint64_t bd = pre::smem_desc_sw128(sm + slot * L::SLOT + h * TILE * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16(tmem_base + t * TILE, a + 2 * k, bd + 2 * k, h > 0 || k > 0, id_s);
        }
        pre::umma_commit(&s_full[t]);
        if (last) pre::umma_commit(&q_empty[t]);
      };
      auto release = [&](int slot) { pre::umma_commit(&empty[slot]); };
      while (ok) {
        ok = wide::wait_suspend(&w_full[nw % WORKS], nw / WORKS & 1, SITE_PPRE_WORK);
        const Work* w = &works[nw % WORKS];
        if (!ok || !w->live) break;
        const int j0 = w->j0, n_row[2] = {w->n_row[0], w->n_row[1]};
        mbar_arrive(&w_empty[nw++ % WORKS]);
        const int j_end = max(n_row[0], n_row[1]);
        if (j0 < j_end) {
          ok = wide::wait_suspend(&full[s], ph, SITE_PPRE_K);
          for (int t = 0; ok && t < 2; ++t) {
            if (n_row[t] == j0) continue;
            ok = wide::wait_suspend(&q_full[t], uses[t] & 1, SITE_PPRE_Q);
            if (!ok) break;
            pre::tc_fence_after();
            scores(t, s, j0 + 1 == n_row[t]);
          }
          if (ok) release(s);
          next();
        }
        for (int j = j0; ok && j < j_end; ++j) {
          const int vs = s;
          ok = wide::wait_suspend(&full[s], ph, SITE_PPRE_V);
          next();
          const int ks = s;
          const uint32_t kph = ph;
          bool k_here = false;
          for (int t = 0; ok && t < 2; ++t) {
            if (j >= n_row[t]) continue;
            if (j == j0) {                                 // the output of the unit before has been read
              if (uses[t] > 0) ok = wide::wait_suspend(&o_empty[t], (uses[t] - 1) & 1, SITE_PPRE_OEMPTY);
              ++uses[t];
            }
            const uint64_t bd = smem_desc_mn_sw128(smem_u32(sm + vs * L::SLOT), TILE * 128);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (ok) ok = wide::wait_suspend(&p_full[2 * t + h], steps[t] & 1, SITE_PPRE_P);
              if (!ok) break;
              pre::tc_fence_after();
#pragma unroll
              for (int k = h == 0 ? 0 : EARLY / 16; k < (h == 0 ? EARLY : TILE) / 16; ++k)
                umma_f16_ta(tmem_base + TMEM_O + t * DIM, tmem_base + t * TILE + k * 8, bd + k * (2048 >> 4), j > j0 || k > 0, id_o);
            }
            if (!ok) break;
            ++steps[t];
            if (j == n_row[t] - 1) pre::umma_commit(&o_full[t]);
            if (j + 1 < n_row[t]) {
              if (!k_here) ok = wide::wait_suspend(&full[ks], kph, SITE_PPRE_K);
              k_here = true;
              if (!ok) break;
              pre::tc_fence_after();
              scores(t, ks, j + 2 == n_row[t]);
            }
          }
          if (ok) release(vs);
          if (j + 1 < j_end) {
            if (ok) release(ks);
            next();
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFTMAX));
    // -------------------------------------------------------------- softmax: thread = row
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_base + lanes + t * TILE, to = tmem_base + lanes + TMEM_O + t * DIM;
    uint32_t steps = 0, uses = 0, ring = 0;                // ring: key and value tiles before this unit's
    while (const Work* w = next_work()) {
      const int j0 = w->j0, n = w->n_row[t], len = w->len;
      float m = neg_inf(), l = 0.f;
      {
        const int tok = w->tok0 + t * p.toks + row / p.group;
        const int limit = row / p.group < p.toks && tok < w->q_len ? len - w->q_len + tok : -1;    // last slot this row sees
        const int limit_all = __reduce_min_sync(0xffffffffu, limit);
        for (int j = j0; j < n; ++j) {
          if (ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&s_full[t], steps & 1, SITE_PPRE_S));
          ++steps;
          if (!ok) break;
          pre::tc_fence_after();
          uint32_t x[TILE];
#pragma unroll
          for (int c = 0; c < TILE; c += 32) tmem_ld32_issue(ts + c, x + c);
          tmem_ld_wait();
          if ((j + 1) * TILE - 1 > limit_all) {
            const int last = limit - j * TILE;             // last visible column
#pragma unroll
            for (int c = 0; c < TILE; ++c) x[c] = c <= last ? x[c] : 0xff800000u;
          }
          float top[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = __uint_as_float(x[i]);
#pragma unroll
          for (int c = 4; c + 8 <= TILE; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = max3_nan(top[i], __uint_as_float(x[c + i]), __uint_as_float(x[c + 4 + i]));
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3_nan(top[i], __uint_as_float(x[TILE - 4 + i]), neg_inf());
          const float all_top = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], neg_inf());
          const float scaled = all_top * p.scale_log2;     // (a NaN leaves the maximum alone and the weights are NaN)
          const float mx = below_max(scaled, SHIFT<T>);
          float scale = p.scale_log2;
          const bool huge = fabsf(scaled) > HUGE_SCORE && scaled != neg_inf();
          if (__any_sync(0xffffffffu, mx > __fadd_rd(m, GROWTH) || huge)) {
            if (__any_sync(0xffffffffu, huge)) {
#pragma unroll
              for (int c = 0; c < TILE; ++c) x[c] = __float_as_uint(__fmul_rn(__uint_as_float(x[c]), scale));
              scale = 1.f;
            }
            const float a = mx > m ? ex2(m - mx) : 1.f;    // (m still minus infinity: zero)
            m = fmaxf(m, mx);
            l *= a;
            if (j > j0) {
#pragma unroll
              for (int c = 0; c < DIM; c += 16) {
                uint32_t o[16];
                csum::tmem_ld16(to + c, o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                tmem_st16_issue(to + c, o);
              }
              tmem_st_wait();
            }
          }
          const float base = m == neg_inf() ? 0.f : m;
          if ((j + 1) * TILE > len) {
            // the sequence ends in this tile: values behind it become zero before a product reads them
            const uint32_t k = ring + 2 * (j - j0) + 1, s = k % L::STAGES;
            ok = __all_sync(0xffffffffu, wide::wait_suspend(&full[s], (k / L::STAGES) & 1, SITE_PPRE_VZERO));
            if (!ok) break;
            if (j * TILE + row >= len) {
#pragma unroll
              for (int ch = 0; ch < DIM / 8; ++ch)
                sts_v4(smem_u32(sm) + s * L::SLOT + (ch >> 3) * TILE * 128 + row * 128 + ((ch & 7) << 4), make_uint4(0, 0, 0, 0));
            }
            fence_proxy_async_smem();
          }
          // The product with the first slots' values starts while the other weights are made; it reads only rows of
          // values that this warp's row tile has zeroed where need be (all four warps arrive for either part).
          l += weights<T, EARLY>(x, scale, base, ts);
          pre::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t]);
          l += weights<T, TILE - EARLY>(x + EARLY, scale, base, ts + EARLY / 2);
          pre::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + 1]);
        }
      }
      ring += 2 * (max(w->n_row[0], w->n_row[1]) - j0);
      // ------------------------------------------------------------ output
      const bool any = n > j0;
      if (any && ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&o_full[t], uses & 1, SITE_PPRE_O));
      if (any) ++uses;
      pre::tc_fence_after();
      const int tok = w->tok0 + t * p.toks + row / p.group;
      const bool live = row / p.group < p.toks && tok < w->q_len;
      const long long tr = w->q0 + tok;
      const int hd = w->head * p.group + row % p.group;
      T* dst_row = static_cast<T*>(p.out) + tr * p.o_tok + (long long)hd * p.o_head;
      auto write_row = [&](int c, const float (&o)[16], float f) {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
          reinterpret_cast<uint4*>(dst_row + c)[i / 8] = make_uint4(pack2<T>(o[i] * f, o[i + 1] * f), pack2<T>(o[i + 2] * f, o[i + 3] * f),
                                                                    pack2<T>(o[i + 4] * f, o[i + 5] * f), pack2<T>(o[i + 6] * f, o[i + 7] * f));
      };
      const int pr = t * ROWS + row;                       // row of a part
      float* part = p.parts + (long long)w->part * L::PART;
      const bool whole = w->whole;
      const float f = l > 0.f ? 1.f / l : 1.f;
#pragma unroll
      for (int c = 0; c < DIM; c += 16) {
        uint32_t x[16];
        float o[16];
        if (any && ok) csum::tmem_ld16(to + c, x);
        // where nothing was summed (or a NaN was) what the accumulator holds does not count; a NaN stays one
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = l > 0.f ? __uint_as_float(x[i]) : l;
        if (whole) {
          if (live && ok) write_row(c, o, f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            reinterpret_cast<float4*>(part + 4 * ROWS)[(c + i) / 4 * (2 * ROWS) + pr] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      if (any) {
        pre::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
      if (whole) {
        if (live && ok && p.lse) p.lse[tr * p.n_heads + hd] = l > 0.f ? (m + log2f(l)) * LN2 : l == l ? neg_inf() : l;
      } else {
        reinterpret_cast<float2*>(part)[pr] = make_float2(m, l);
      }
      work_done();
    }
  }
  // Common exit, then the allocating warp frees tensor memory.  After a wait that gave up copies and MMAs may still be
  // in flight: the block stays for a millisecond, many times what they need, before its memory is handed on.
  pre::tc_fence_before();
  if (__syncthreads_or(!ok)) {
    if (tid == 0)
      for (const uint64_t t0 = wide::timer_ns(); wide::timer_ns() - t0 < 1000000;) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == WARP_MMA) {
    pre::tc_fence_after();
    pre::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Joins the parts of the units that the runs cut: a block takes JOIN_ROWS rows of the unit that is cut first in its run, a
// thread EACH times four neighbouring elements.
constexpr int JOIN_ROWS = 32, JOIN_THREADS = 256;
template <typename T, int DIM>
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const Params p) {
  using L = Layout<DIM>;
  constexpr int STEP = JOIN_THREADS / JOIN_ROWS * 4;       // elements between a thread's fours
  constexpr int EACH = DIM / STEP;
  grid_launch_dependents();
  grid_dependency_wait();
  const int run = blockIdx.x;
  const Join u = static_cast<const Join*>(p.joins)[run];
  const int row = blockIdx.y * JOIN_ROWS + threadIdx.x % JOIN_ROWS, c = threadIdx.x / JOIN_ROWS * 4;
  const int t = row / ROWS, r = row % ROWS, tok = u.tok0 + t * p.toks + r / p.group;
  if (u.parts == 0 || r / p.group >= p.toks || tok >= u.q_len) return;
  // the first part is the second of its run's two (the unit begins in that run), the others their run's first
  auto part_of = [&](int k) { return p.parts + (2 * (long long)(run + k) + (k == 0 ? 1 : 0)) * L::PART; };
  float m = neg_inf(), l = 0.f;
#pragma unroll 4
  for (int k = 0; k < u.parts; ++k) m = fmaxf(m, reinterpret_cast<const float2*>(part_of(k))[row].x);
  float4 acc[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int k = 0; k < u.parts; ++k) {
    const float2 ml = reinterpret_cast<const float2*>(part_of(k))[row];
    const float a = ml.x == neg_inf() ? (ml.y == ml.y ? 0.f : 1.f) : ex2(ml.x - m);
    l += a * ml.y;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float4 o = reinterpret_cast<const float4*>(part_of(k) + 4 * ROWS)[(c + i * STEP) / 4 * (2 * ROWS) + row];
      acc[i].x += a * o.x;
      acc[i].y += a * o.y;
      acc[i].z += a * o.z;
      acc[i].w += a * o.w;
    }
  }
  const float f = l > 0.f ? 1.f / l : 1.f;                 // (nothing summed: the sums are zero; a NaN stays one)
  const long long tr = u.q0 + tok;
  const int hd = u.head * p.group + r % p.group;
  T* dst = static_cast<T*>(p.out) + tr * p.o_tok + (long long)hd * p.o_head + c;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    *reinterpret_cast<uint2*>(dst + i * STEP) = make_uint2(pack2<T>(acc[i].x * f, acc[i].y * f), pack2<T>(acc[i].z * f, acc[i].w * f));
  if (p.lse && c == 0) p.lse[tr * p.n_heads + hd] = l > 0.f ? (m + log2f(l)) * LN2 : l == l ? neg_inf() : l;
}

}  // namespace ppre
}  // namespace w4a4
