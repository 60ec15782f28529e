// Attention weight that each cache slot has received from a call's new tokens:
//
//   sums[b, g, j] += sum over new tokens i that see j, heads h of group g of exp(scale q[i,h].k[j] - lse[i,h]).
//
// The product is taken transposed, scores[slot, row] = K Q^T with 128 slots on the M side: a slot is then one lane of
// tensor memory and one thread, which adds its weights up in a register without talking to anybody - one order of
// additions, no atomics - and few rows make a narrow product (N = 16 for a decode step) instead of an empty tall one.
//
// What bounds it: with few rows the one read of the keys; from about 64 rows on the exponentials, 16 per clock and SM.
// The 128-slot tiles of all (sequence, head) units are laid end to end and cut into one equal run per CTA; a tile goes
// through all row tiles before the next one, so its sums are finished in one place.  Roles: a warp that issues copies,
// a thread that issues MMAs into two accumulators in turn, four warps that read them out.
#pragma once

#include "paged_kv.cuh"
#include "prefill_wide_gemm.cuh"

namespace w4a4 {
namespace csum {

using namespace kv;

constexpr int TILE = 128, MAX_COLS = 128, WARPS = 4, WARP_COPY = 4, WARP_MMA = 5;
constexpr int THREADS = 6 * 32;
constexpr int K_STAGES = 4, Q_STAGES = 2, ACCS = 2;
constexpr int TMEM_COLS = ACCS * MAX_COLS;

enum : int { SITE_SUMS_KEMPTY = 38, SITE_SUMS_QEMPTY, SITE_SUMS_KFULL, SITE_SUMS_QFULL, SITE_SUMS_ACCEMPTY, SITE_SUMS_ACCFULL };

template <int DIM>
struct Layout {
  static constexpr int HALVES = DIM / 64;
  static constexpr int K_BYTES = TILE * DIM * 2, Q_BYTES = MAX_COLS * DIM * 2;
  static constexpr int q = K_STAGES * K_BYTES;
  static constexpr int cols = q + Q_STAGES * Q_BYTES;            // {float lse, int limit} [2][MAX_COLS]
  static constexpr int bars = cols + 2 * MAX_COLS * 8;
  static constexpr int total = bars + (2 * K_STAGES + 2 * Q_STAGES + 2 * ACCS) * 8 + 16;
  static_assert(1024 + total <= 232448, "shared memory of one SM");
};
template <int DIM> inline size_t smem_bytes() { return 1024 + Layout<DIM>::total; }

struct Params {
  Cache c;
  Seqs s;
  const float* lse;           // (T, n_heads)
  float* sums;
  long long sums_seq, sums_head;
  int n_heads, group, box;
  int cols, toks;             // rows of a row tile on the N side, and whole tokens in it
  float scale_log2;
};

__device__ __forceinline__ void unit_shape(const Params& p, const Seq& q, int& row_tiles, int& tiles) {
  row_tiles = 1;
  tiles = q.q_len > 0 ? (q.len + TILE - 1) / TILE : 0;
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

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS, 1)
cache_sums_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const Params p) {
  using L = Layout<DIM>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* k_empty = k_full + K_STAGES;
  uint64_t* q_full = k_empty + K_STAGES;
  uint64_t* q_empty = q_full + Q_STAGES;
  uint64_t* acc_full = q_empty + Q_STAGES;
  uint64_t* acc_empty = acc_full + ACCS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + ACCS);
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < K_STAGES; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < Q_STAGES; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); }
    for (int i = 0; i < ACCS; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], WARPS); }
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_q);
  }
  if (warp == WARP_MMA) pre::tmem_alloc(tmem_slot, TMEM_COLS);
  pre::tc_fence_before();
  __syncthreads();
  pre::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (warp == WARP_COPY) grid_dependency_wait_for_async_reads();
  else grid_dependency_wait();

  const long long total = total_tiles(p);
  const long long runs = min((long long)gridDim.x, total), c = blockIdx.x;
  bool ok = true;                                          // no wait of this thread has given up
  if (c < runs) {
    const long long begin = c * total / runs, end = (c + 1) * total / runs;
    Walk<Params> w;
    w.start(p, begin);
    int ks = 0, qs = 0, acc = 0;                           // ring places and their phases, walked alike by every role
    uint32_t kph = 0, qph = 0, aph = 0;
    bool k_lap = false, q_lap = false, a_lap = false;      // the ring has been walked once: its places must be free
    if (warp == WARP_COPY) {
      // ---------------------------------------------------------- copies
      PagesAhead pages;
      while (ok) {
        const int stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
        const int n_rt = (w.q.q_len + p.toks - 1) / p.toks;
        for (int t = w.tile; ok && t < stop; ++t) {
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
          for (int r = 0; r < n_rt; ++r) {
            if (n_rt == 1 && t != w.tile) continue;        // one row tile: copied once for all tiles of the unit
            if (q_lap) ok = __all_sync(0xffffffffu, wide::wait_suspend(&q_empty[qs], qph ^ 1, SITE_SUMS_QEMPTY));
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[qs], p.toks * p.group * DIM * 2);
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h)
                tma_load_3d(sm + L::q + qs * L::Q_BYTES + h * MAX_COLS * 128, &tm_q, h * 64, w.head * p.group,
                            w.q.q0 + r * p.toks, &q_full[qs]);
            }
            __syncwarp();
            if (++qs == Q_STAGES) { qs = 0; qph ^= 1; q_lap = true; }
          }
        }
        if (w.at - w.tile + stop >= end) break;
        w.next_unit(p);
      }
    } else if (warp == WARP_MMA) {
      // ---------------------------------------------------------- MMAs
      const uint32_t idesc = idesc_f16<T>(p.cols);
      while (ok) {
        const int stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
        const int n_rt = (w.q.q_len + p.toks - 1) / p.toks;
        for (int t = w.tile; ok && t < stop; ++t) {
          ok = __all_sync(0xffffffffu, wide::wait_suspend(&k_full[ks], kph, SITE_SUMS_KFULL));
          for (int r = 0; ok && r < n_rt; ++r) {
            if (n_rt > 1 || t == w.tile) ok = __all_sync(0xffffffffu, wide::wait_suspend(&q_full[qs], qph, SITE_SUMS_QFULL));
            if (ok && a_lap) ok = __all_sync(0xffffffffu, wide::wait_suspend(&acc_empty[acc], aph ^ 1, SITE_SUMS_ACCEMPTY));
            if (!ok) break;
            pre::tc_fence_after();
            if (elected()) {
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h) {
                const uint64_t a = pre::smem_desc_sw128(sm + ks * L::K_BYTES + h * TILE * 128);
                const uint64_t b = pre::smem_desc_sw128(sm + L::q + qs * L::Q_BYTES + h * MAX_COLS * 128);
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_f16(tmem_base + acc * MAX_COLS, a + 2 * j, b + 2 * j, h > 0 || j > 0, idesc);
              }
              pre::umma_commit(&acc_full[acc]);
              if (r == n_rt - 1) pre::umma_commit(&k_empty[ks]);
              if (n_rt > 1 || t == stop - 1) pre::umma_commit(&q_empty[qs]);
            }
            __syncwarp();
            if (++acc == ACCS) { acc = 0; aph ^= 1; a_lap = true; }
            if (n_rt > 1 || t == stop - 1) { if (++qs == Q_STAGES) { qs = 0; qph ^= 1; } }
          }
          if (++ks == K_STAGES) { ks = 0; kph ^= 1; }
        }
        if (w.at - w.tile + stop >= end) break;
        w.next_unit(p);
      }
    } else {
      // ---------------------------------------------------------- read-out: thread = slot of the tile
      const uint32_t cols_a = smem_u32(sm + L::cols);
      int step = 0;                                        // column tables written so far
      // this thread's column of row tile r: logarithm (base 2) of its sum, and the last slot it sees
      auto column = [&](int r) {
        const int tok = r * p.toks + tid / p.group, hd = w.head * p.group + tid % p.group;
        const bool live = tid < p.toks * p.group && tok < w.q.q_len;
        float2 v = make_float2(0.f, __int_as_float(-1));
        if (live) {
          const float lse = ld_plain(p.lse + (long long)(w.q.q0 + tok) * p.n_heads + hd) * LOG2E;
          if (lse != neg_inf()) v = make_float2(lse, __int_as_float(w.q.len - w.q.q_len + tok));
        }
        return v;
      };
      while (true) {
        const int stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
        const int n_rt = (w.q.q_len + p.toks - 1) / p.toks;
        float2 col = column(0);
        for (int t = w.tile; t < stop; ++t) {
          const int slot = t * TILE + tid;
          float sum = 0.f;
          for (int r = 0; r < n_rt; ++r) {
            if (n_rt > 1 || t == w.tile) {
              sts_f2(cols_a + (((step & 1) * MAX_COLS) + tid) * 8, col);
              asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
              ++step;
              if (n_rt > 1) col = column(r + 1 < n_rt ? r + 1 : 0);
            }
            const uint32_t ct = cols_a + ((step - 1) & 1) * MAX_COLS * 8;
            if (ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&acc_full[acc], aph, SITE_SUMS_ACCFULL));
            if (ok) {
              pre::tc_fence_after();
              const uint32_t ta = tmem_base + ((uint32_t)(warp * 32) << 16) + acc * MAX_COLS;
              for (int c0 = 0; c0 < p.cols; c0 += 16) {
                uint32_t a[16];
                tmem_ld16(ta + c0, a);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  const float4 cc = lds_f4(ct + (c0 + i) * 8);
                  const float p0 = ex2(__uint_as_float(a[i]) * p.scale_log2 - cc.x), p1 = ex2(__uint_as_float(a[i + 1]) * p.scale_log2 - cc.z);
                  sum += slot <= __float_as_int(cc.y) ? p0 : 0.f;
                  sum += slot <= __float_as_int(cc.w) ? p1 : 0.f;
                }
              }
              pre::tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[acc]);
            }
            if (++acc == ACCS) { acc = 0; aph ^= 1; }
          }
          if (ok && slot < w.q.len) {
            float* dst = p.sums + (long long)w.b * p.sums_seq + (long long)w.head * p.sums_head + slot;
            *dst += sum;
          }
        }
        if (w.at - w.tile + stop >= end) break;
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
    pre::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace csum
}  // namespace w4a4
