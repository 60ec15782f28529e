// Attention weight that each cache slot has received from a call's new tokens:
//
//   sums[b, g, j] += sum over new tokens i that see j, heads h of group g of exp(scale q[i,h].k[j] - lse[i,h]).
//
// The product is taken transposed, scores[slot, row] = K Q^T with 128 slots on the M side: a slot is then one lane of
// tensor memory and one thread, which adds its weights up in a register without talking to anybody - one order of
// additions, no atomics - and few rows make a narrow product (N = 16 for a decode step) instead of an empty tall one.
//
// What bounds it: with few rows the one read of the keys; from about 64 rows on the exponentials, 16 per clock and SM.
// The 128-slot tiles of all (sequence, head) units are laid end to end, each weighing its row tiles and each unit PAD
// more, and cut into one equal run per CTA; a tile goes through all row tiles before the next one, so its sums are
// finished in one place.  Roles: a warp that issues copies, a thread that issues MMAs, two teams of four warps that read
// the accumulators out, a team a tile.  Up to NARROW rows the queries' buffers are small and the keys' ring is deeper.
// Measured: a decode step of 32 sequences up to 4096 slots 31 us, the last 64 tokens of four prompts up to 8000 slots
// 20.6 us, sums fresh; zeroed by a launch of their own, with one team and four key tiles ahead, 40 and 31.
#pragma once

#include "paged_kv.cuh"
#include "prefill_wide_gemm.cuh"

namespace w4a4 {
namespace csum {

using namespace kv;

constexpr int TILE = 128, MAX_COLS = 128, NARROW = 32;
constexpr int TEAMS = 2, WARPS = 4 * TEAMS, WARP_COPY = WARPS, WARP_MMA = WARPS + 1;
constexpr int THREADS = (WARPS + 2) * 32;
constexpr int Q_STAGES = 2, ACCS = 2;                       // accumulators of a team
constexpr int PAD = 2;                                     // what a unit costs besides its tiles, in steps

enum : int { SITE_SUMS_KEMPTY = 38, SITE_SUMS_QEMPTY, SITE_SUMS_KFULL, SITE_SUMS_QFULL, SITE_SUMS_ACCEMPTY, SITE_SUMS_ACCFULL };

// COLS: rows of a row tile that there is room for, NARROW or MAX_COLS
template <int DIM, int COLS>
struct Layout {
  static constexpr int HALVES = DIM / 64;
  static constexpr int K_BYTES = TILE * DIM * 2, Q_BYTES = COLS * DIM * 2;
  static constexpr int K_STAGES = (COLS == NARROW ? 6 : 4) * 128 / DIM;
  static constexpr int TMEM_COLS = TEAMS * ACCS * COLS;
  static constexpr int q = K_STAGES * K_BYTES;
  static constexpr int cols = q + Q_STAGES * Q_BYTES;            // float minus lse, int limit: [TEAMS][2][COLS] each
  static constexpr int bars = cols + TEAMS * 2 * COLS * 8;
  static constexpr int total = bars + (2 * K_STAGES + 2 * Q_STAGES + 2 * TEAMS * ACCS) * 8 + 16;
  static_assert(1024 + total <= 232448, "shared memory of one SM");
};
template <int DIM, int COLS> inline size_t smem_bytes() { return 1024 + Layout<DIM, COLS>::total; }

struct Params {
  Cache c;
  Seqs s;
  const float* lse;           // (T, n_heads)
  float* sums;
  long long sums_seq, sums_head;
  int n_heads, group, box;
  int cols, toks;             // rows of a row tile on the N side, and whole tokens in it
  int fresh;                  // sums holds nothing yet: every slot is written, zero where nothing is added
  float scale_log2;
};

// Steps of sequence b: PAD, and one for each slot tile and row tile.
__device__ __forceinline__ int row_tiles_of(const Params& p, const Seq& q) { return (q.q_len + p.toks - 1) / p.toks; }
__device__ __forceinline__ void unit_shape(const Params& p, const Seq& q, int& row_tiles, int& tiles) {
  row_tiles = q.q_len > 0 && q.len > 0 ? 1 : 0;
  tiles = row_tiles ? PAD + (q.len + TILE - 1) / TILE * row_tiles_of(p, q) : 0;
}
// What a run that ends at `end` has of the unit it stands in: row tiles, and slot tiles first .. stop - 1.
struct Part {
  int n_rt, first, stop;
  bool more;
  __device__ __forceinline__ Part(const Params& p, const Walk<Params>& w, long long end) {
    n_rt = row_tiles_of(p, w.q);
    const int stop_step = (int)min((long long)w.tiles, w.tile + (end - w.at));
    first = (max(w.tile - PAD, 0) + n_rt - 1) / n_rt;
    stop = (max(stop_step - PAD, 0) + n_rt - 1) / n_rt;
    more = w.at - w.tile + stop_step < end;
  }
};

// Zeros behind the lengths, and in all of a sequence without a new token, of sums that hold nothing yet.  The read-out
// warps write them while the first keys are on their way.  Measured, a decode step of 32 sequences up to 4096 slots of 8
// heads, 31 us; 33 with a launch before that zeroes all of sums.
__device__ __forceinline__ void zero_rest(const Params& p) {
  constexpr int CHUNK = 4096;
  const int n_chunks = (p.s.max_slots - 1) / CHUNK + 1;      // (there is a slot, and up to 2^31 - 1025 of them)
  const long long all = (long long)p.s.n * p.c.n_kv * n_chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const int row = (int)(i / n_chunks), c0 = (int)(i - (long long)row * n_chunks) * CHUNK, b = row / p.c.n_kv;
    const Seq q = load_seq(p.s, b);
    float* s = p.sums + (long long)b * p.sums_seq + (long long)(row % p.c.n_kv) * p.sums_head;
    const int end = c0 + min(CHUNK, p.s.max_slots - c0);
    for (int j = max(c0, q.q_len > 0 ? q.len : 0) + threadIdx.x; j < end; j += WARPS * 32) s[j] = 0.f;
  }
}

// kind::f16: 16-bit operands K-major in shared memory, M = 128, fp32 accumulation
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n) {
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t accumulate, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ f32x2_t add_f32x2(f32x2_t a, f32x2_t b) {
  f32x2_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// One lane of a converged warp, the same every time.  MMAs are issued under this rather than under lane == 0: the compiler
// then knows that one thread runs the branch and keeps descriptors in uniform registers.  Measured, scores and weights
// x values of 128 x 128 x 128 back to back: 1025 against 1111 clocks alone, and twice that beside busy softmax warps.
__device__ __forceinline__ bool elected() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <typename T, int DIM, int COLS>
__global__ void __launch_bounds__(THREADS, 1)
cache_sums_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const Params p) {
  using L = Layout<DIM, COLS>;
  constexpr int K_STAGES = L::K_STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* k_empty = k_full + K_STAGES;
  uint64_t* q_full = k_empty + K_STAGES;
  uint64_t* q_empty = q_full + Q_STAGES;
  uint64_t* acc_full = q_empty + Q_STAGES;                       // [TEAMS][ACCS]: a barrier belongs to one team, which waits for all its phases
  uint64_t* acc_empty = acc_full + TEAMS * ACCS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + TEAMS * ACCS);
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < K_STAGES; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < Q_STAGES; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); }
    for (int i = 0; i < TEAMS * ACCS; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4); }
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_q);
  }
  // rows of a row tile that no whole token fills are never copied: zero, once
  for (int i = tid; i < Q_STAGES * L::Q_BYTES / 16; i += THREADS) sts_v4(smem_u32(sm) + L::q + i * 16, make_uint4(0, 0, 0, 0));
  fence_proxy_async_smem();
  if (warp == WARP_MMA) pre::tmem_alloc(tmem_slot, L::TMEM_COLS);
  pre::tc_fence_before();
  __syncthreads();
  pre::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (warp == WARP_COPY) grid_dependency_wait_for_async_reads();
  else grid_dependency_wait();

  bool ok = true;                                          // no wait of this thread has given up
  if (p.fresh && warp < WARPS) zero_rest(p);
  Walk<Params> w;
  long long total, runs, begin, end;
  if (w.start(p, gridDim.x, blockIdx.x, total, runs, begin, end)) {
    if (warp == WARP_COPY) {
      // ---------------------------------------------------------- copies
      PagesAhead pages;
      int ks = 0, qs = 0;                                  // ring places and their phases
      uint32_t kph = 0, qph = 0;
      bool k_lap = false, q_lap = false;                   // the ring has been walked once: its places must be free
      while (ok) {
        const Part u(p, w, end);
        for (int t = u.first; ok && t < u.stop; ++t) {
          if (k_lap) ok = __all_sync(0xffffffffu, wide::wait_suspend(&k_empty[ks], kph ^ 1, SITE_SUMS_KEMPTY));
          if (!ok) break;
          const int boxes = TILE / p.box, slot = t * TILE + lane * p.box;      // (at most 8 boxes)
          const bool mine = lane < boxes && slot < w.q.len;
          const int page = pages.get(p.c, w.b, w.q.len, p.box, t * boxes);
          const int live = __popc(__ballot_sync(0xffffffffu, mine));
          if (lane == 0) mbar_arrive_expect_tx(&k_full[ks], live * p.box * DIM * 2);
          __syncwarp();
          if (mine)
#pragma unroll
            for (int h = 0; h < L::HALVES; ++h)
              tma_load_4d(smem_u32(sm) + ks * L::K_BYTES + h * TILE * 128 + lane * p.box * 128, &tm_k, h * 64,
                          slot % p.c.page, w.head, page, &k_full[ks]);
          if (++ks == K_STAGES) { ks = 0; kph ^= 1; k_lap = true; }
          for (int r = 0; r < u.n_rt; ++r) {
            if (u.n_rt == 1 && t != u.first) continue;     // one row tile: copied once for all tiles of the unit
            if (q_lap) ok = __all_sync(0xffffffffu, wide::wait_suspend(&q_empty[qs], qph ^ 1, SITE_SUMS_QEMPTY));
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[qs], p.toks * p.group * DIM * 2);
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h)
                tma_load_3d(sm + L::q + qs * L::Q_BYTES + h * COLS * 128, &tm_q, h * 64, w.head * p.group,
                            w.q.q0 + r * p.toks, &q_full[qs]);
            }
            __syncwarp();
            if (++qs == Q_STAGES) { qs = 0; qph ^= 1; q_lap = true; }
          }
        }
        if (!u.more) break;
        w.next_unit(p);
      }
    } else if (warp == WARP_MMA) {
      // ---------------------------------------------------------- MMAs: one thread
      if (elected()) {
        const uint32_t idesc = idesc_f16<T>(p.cols);
        int ks = 0, qs = 0, team = 0;
        uint32_t kph = 0, qph = 0, steps[TEAMS] = {0, 0};
        while (ok) {
          const Part u(p, w, end);
          for (int t = u.first; ok && t < u.stop; ++t) {
            ok = wide::wait_suspend(&k_full[ks], kph, SITE_SUMS_KFULL);
            for (int r = 0; ok && r < u.n_rt; ++r) {
              const uint32_t step = team ? steps[1]++ : steps[0]++;
              const int acc = team * ACCS + (int)(step % ACCS);
              if (u.n_rt > 1 || t == u.first) ok = wide::wait_suspend(&q_full[qs], qph, SITE_SUMS_QFULL);
              if (ok && step >= ACCS) ok = wide::wait_suspend(&acc_empty[acc], (step / ACCS - 1) & 1, SITE_SUMS_ACCEMPTY);
              if (!ok) break;
              pre::tc_fence_after();
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h) {
                const uint64_t a = pre::smem_desc_sw128(sm + ks * L::K_BYTES + h * TILE * 128);
                const uint64_t b = pre::smem_desc_sw128(sm + L::q + qs * L::Q_BYTES + h * COLS * 128);
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_f16(tmem_base + acc * COLS, a + 2 * j, b + 2 * j, h > 0 || j > 0, idesc);
              }
              pre::umma_commit(&acc_full[acc]);
              if (r == u.n_rt - 1) pre::umma_commit(&k_empty[ks]);
              if (u.n_rt > 1 || t == u.stop - 1) {
                pre::umma_commit(&q_empty[qs]);
                if (++qs == Q_STAGES) { qs = 0; qph ^= 1; }
              }
            }
            if (++ks == K_STAGES) { ks = 0; kph ^= 1; }
            team ^= 1;
          }
          if (!u.more) break;
          // (next_unit uses no warp operation)
          w.next_unit(p);
        }
      }
    } else {
      // ---------------------------------------------------------- read-out: thread = slot of the tile
      const int team = warp / 4, row = tid % 128;
      const uint32_t table = smem_u32(sm + L::cols) + team * 2 * COLS * 8;      // [2] of COLS floats, then COLS ints
      const f32x2_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
      uint32_t steps = 0, tables = 0;
      int turn = 0;                                        // team of the next tile
      // this thread's column of row tile r: minus the logarithm (base 2) of its sum, and the last slot it sees (-1: no row)
      auto column = [&](int r, float& nl, int& limit) {
        const int tok = r * p.toks + row / p.group, hd = w.head * p.group + row % p.group;
        nl = neg_inf();
        limit = -1;
        if (row < p.toks * p.group && tok < w.q.q_len) {
          const float lse = ld_plain(p.lse + (long long)(w.q.q0 + tok) * p.n_heads + hd);
          if (lse != neg_inf()) { nl = -lse * LOG2E; limit = w.q.len - w.q.q_len + tok; }
        }
      };
      while (true) {
        const Part u(p, w, end);
        float nl;
        int limit;
        const bool mine = (u.stop - u.first > 1) || turn == team;
        bool written = false;                              // one row tile: its table serves all tiles of the unit
        uint32_t at = 0;
        if (mine && u.stop > u.first) column(0, nl, limit);
        for (int t = u.first; t < u.stop; ++t, turn ^= 1) {
          if (turn != team) continue;
          const int slot = t * TILE + row;
          f32x2_t sum2[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
          float sum = 0.f;
          for (int r = 0; r < u.n_rt; ++r) {
            if (u.n_rt > 1 || !written) {
              written = true;
              at = table + (tables & 1) * COLS * 8;
              if (row < COLS) {
                sts_f1(at + row * 4, nl);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + COLS * 4 + row * 4), "r"(limit) : "memory");
              }
              asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory");
              ++tables;
              if (u.n_rt > 1) column(r + 1 < u.n_rt ? r + 1 : 0, nl, limit);
            }
            const int acc = team * ACCS + (int)(steps % ACCS);
            if (ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&acc_full[acc], steps / ACCS & 1, SITE_SUMS_ACCFULL));
            ++steps;
            if (ok) {
              pre::tc_fence_after();
              const uint32_t ta = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * COLS;
              // every row of the tile exists and sees the whole slot tile
              const bool clear = (r + 1) * p.toks <= w.q.q_len && (t + 1) * TILE - 1 <= w.q.len - w.q.q_len + r * p.toks;
              for (int c0 = 0; c0 < p.cols; c0 += 16) {
                uint32_t a[16];
                tmem_ld16(ta + c0, a);
                if (clear) {
#pragma unroll
                  for (int i = 0; i < 16; i += 4) {
                    f32x2_t n0, n1;
                    lds_f32x2_pair(at + (c0 + i) * 4, n0, n1);
                    const float2 e0 = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(a[i]), __uint_as_float(a[i + 1])), scale2, n0));
                    const float2 e1 = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(a[i + 2]), __uint_as_float(a[i + 3])), scale2, n1));
                    sum2[0] = add_f32x2(sum2[0], pack_f32x2(ex2(e0.x), ex2(e0.y)));
                    sum2[1] = add_f32x2(sum2[1], pack_f32x2(ex2(e1.x), ex2(e1.y)));
                  }
                } else {
#pragma unroll
                  for (int i = 0; i < 16; i += 4) {
                    const float4 nl4 = lds_f4(at + (c0 + i) * 4);
                    const uint4 lim = lds_v4(at + COLS * 4 + (c0 + i) * 4);
                    sum += slot <= (int)lim.x ? ex2(fmaf(__uint_as_float(a[i]), p.scale_log2, nl4.x)) : 0.f;
                    sum += slot <= (int)lim.y ? ex2(fmaf(__uint_as_float(a[i + 1]), p.scale_log2, nl4.y)) : 0.f;
                    sum += slot <= (int)lim.z ? ex2(fmaf(__uint_as_float(a[i + 2]), p.scale_log2, nl4.z)) : 0.f;
                    sum += slot <= (int)lim.w ? ex2(fmaf(__uint_as_float(a[i + 3]), p.scale_log2, nl4.w)) : 0.f;
                  }
                }
              }
              pre::tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[acc]);
            }
          }
          if (ok && slot < w.q.len) {
            const float2 s = unpack_f32x2(add_f32x2(sum2[0], sum2[1]));
            float* to = p.sums + (long long)w.b * p.sums_seq + (long long)w.head * p.sums_head + slot;
            *to = (p.fresh ? 0.f : *to) + (sum + (s.x + s.y));
          }
        }
        if (!u.more) break;
        w.next_unit(p);
      }
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
    pre::tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
}

}  // namespace csum
}  // namespace w4a4
