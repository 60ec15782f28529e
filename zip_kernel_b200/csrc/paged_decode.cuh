// Attention of few query rows per key/value head over a paged cache: decode steps, and chunks of a few tokens.
//
//   o[r] = sum_j p[r,j] v[j] / sum_j p[r,j],  p[r,j] = exp(scale q[r].k[j] - m[r]),  j up to the row's own slot,
//
// the running maximum m, the sum and o carried through one pass over the slots (o and the sum are multiplied by
// exp(m_old - m_new) when the maximum grows).  A row = (new token, head of the group that shares the key/value head);
// up to 16 rows fill the M side of an m16n8k16 product.
//
// What bounds it: every key and value is read once from HBM, 2 * dim * 2 bytes for 4 * 16 * dim multiply-adds at most.
// So the whole card must stream, whatever the number and lengths of the sequences: the 64-slot tiles of all (sequence,
// head, row tile) units are laid end to end and cut into one equal run per CTA.  A unit that falls into several runs
// is joined by the CTA that finishes its last part (the parts' order, and so the result's bits, depend on the lengths
// alone).
//
// A CTA is one warp that issues copies (TMA boxes of one page each, 128-byte swizzle, a ring of tiles) and four that
// compute, each on 16 slots of a tile with a maximum, sum and output of its own, joined at the end of a unit: no
// barrier between the warps inside a unit.
//
// Rows of values past the sequence's last slot are set to zero in shared memory first: a stale NaN there times a
// weight of zero would be NaN.  Scores there are replaced, not added to.  Weights enter the second product as 16-bit
// values; for bfloat16, whose step is 2^-8, as the sum of two (the value and what its rounding left), which costs
// tensor time that this kernel has to spare.
#pragma once

#include "paged_kv.cuh"
#include "prefill_wide_gemm.cuh"

namespace w4a4 {
namespace pdec {

using namespace kv;

constexpr int TILE = 64, WARPS = 4, WK = TILE / WARPS, ROWS = 16;
constexpr int THREADS = (WARPS + 1) * 32;

enum : int { SITE_PDEC_FULL = 35, SITE_PDEC_EMPTY, SITE_PDEC_DRAIN };

template <int DIM>
struct Layout {
  static constexpr int HALVES = DIM / 64;                    // 128-byte wide column blocks
  static constexpr int KV_BYTES = TILE * DIM * 2;            // one tile of keys, or of values
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int STAGES = DIM == 128 ? 5 : 10;
  // a part of a unit in the workspace: m and l of the rows, then their outputs
  static constexpr int PART = ROWS * (2 + DIM);
  static constexpr int joined = STAGES * STAGE;              // float [WARPS][ROWS][DIM]
  static constexpr int ml = joined + WARPS * ROWS * DIM * 4; // float [WARPS][ROWS][2]
  static constexpr int bars = ml + WARPS * ROWS * 2 * 4;
  static constexpr int total = bars + 2 * STAGES * 8 + 16;
  static_assert(1024 + total <= 232448, "shared memory of one SM");
};
template <int DIM> inline size_t smem_bytes() { return 1024 + Layout<DIM>::total; }

struct Params {
  Cache c;
  Seqs s;
  const void* q;
  long long q_tok, q_head;
  void* out;
  long long o_tok, o_head;
  float* lse;                 // (T, n_heads), or NULL
  float* parts;               // [2 * grid][Layout::PART]
  int* arrived;               // [grid]: finished parts of the unit that is cut first in that run; zero between calls
  int n_heads, group, box, max_rows;
  float scale_log2;
};

// Row tiles and key tiles of sequence b in this kernel: none when it has no new token or more rows than max_rows.
__device__ __forceinline__ void unit_shape(const Params& p, const Seq& q, int& row_tiles, int& tiles) {
  const long long rows = (long long)q.q_len * p.group;
  const bool mine = q.q_len > 0 && rows <= p.max_rows;
  row_tiles = mine ? (int)((rows + ROWS - 1) / ROWS) : 0;
  tiles = mine ? max(1, (q.len + TILE - 1) / TILE) : 0;
}

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); }

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p,
                    const uint32_t zero) {
  using L = Layout<DIM>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* empty = full + L::STAGES;
  int* last_flag = reinterpret_cast<int*>(empty + L::STAGES);
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WARPS);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncthreads();
  if (warp == WARPS) grid_dependency_wait_for_async_reads();
  else grid_dependency_wait();

  const long long total = total_tiles(p);
  const long long runs = min((long long)gridDim.x, total), c = blockIdx.x;
  if (c >= runs) return;
  const long long begin = c * total / runs, end = (c + 1) * total / runs;
  const uint32_t ring = smem_u32(sm);
  bool ok = true;                                            // no wait of this thread has given up

  if (warp == WARPS) {
    // ------------------------------------------------------------ copies
    Walk<Params> w;
    w.start(p, begin);
    int s = 0;
    uint32_t ph = 1;
    long long n = 0;
    while (ok) {
      const int stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
      for (int t = w.tile; t < stop; ++t, ++n) {
        if (n >= L::STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ph, SITE_PDEC_EMPTY));
        if (!ok) break;
        // one lane per box; boxes with no slot in use are not copied
        const int boxes = TILE / p.box, slot = t * TILE + lane * p.box;
        const bool mine = lane < boxes && slot < w.q.len;
        int page = 0;
        if (mine) {
          page = page_of(p.c, w.b, slot / p.c.page);
          if (page < 0) page = p.c.n_pages;                  // past the end of the map: reads zeros
        }
        const int live = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], live * p.box * DIM * 4);
        __syncwarp();
        if (mine) {
          const uint32_t dst = ring + s * L::STAGE + lane * p.box * 128;
          const int in_page = slot % p.c.page;
#pragma unroll
          for (int h = 0; h < L::HALVES; ++h) tma_load_4d(dst + h * TILE * 128, &tm_k, h * 64, in_page, w.head, page, &full[s]);
#pragma unroll
          for (int h = 0; h < L::HALVES; ++h)
            tma_load_4d(dst + L::KV_BYTES + h * TILE * 128, &tm_v, h * 64, in_page, w.head, page, &full[s]);
        }
        if (++s == L::STAGES) { s = 0; ph ^= 1; }
      }
      if (w.at - w.tile + stop >= end) break;
      w.next_unit(p);
    }
  } else {
    // ------------------------------------------------------------ arithmetic
    const int g = lane >> 2, c2 = (lane & 3) * 2;            // fragment row (and row + 8), first of two columns
    Walk<Params> w;
    w.start(p, begin);
    int s = 0;
    uint32_t ph = 0;
    // addresses inside a tile: this lane's ldmatrix row and the swizzle of its 16-byte chunks
    const int k_row = warp * WK + (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;
    const int v_row = warp * WK + (lane & 15), v_chunk = lane >> 4;
    while (true) {
      const int row0 = w.row_tile * ROWS, rows = min(ROWS, w.q.q_len * p.group - row0);
      // A fragments of the rows; rows that do not exist are zero
      uint32_t qf[DIM / 16][4];
      int limit[2];                                          // last slot the fragment's two rows see
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h, tok = (row0 + r) / p.group, hd = (row0 + r) % p.group;
        const bool live = r < rows;
        const T* src = static_cast<const T*>(p.q) + (long long)(w.q.q0 + (live ? tok : 0)) * p.q_tok + (long long)(w.head * p.group + (live ? hd : 0)) * p.q_head;
        limit[h] = live ? w.q.len - w.q.q_len + tok : -1;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          qf[k][h] = live ? ld_plain(reinterpret_cast<const uint32_t*>(src + k * 16 + c2)) : 0;
          qf[k][h + 2] = live ? ld_plain(reinterpret_cast<const uint32_t*>(src + k * 16 + 8 + c2)) : 0;
        }
      }
      float o[DIM / 8][4], m[2] = {neg_inf(), neg_inf()}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DIM / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

      const int first = w.tile, stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
      for (int t = first; t < stop; ++t) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[s], ph, SITE_PDEC_FULL));
        if (!ok) break;
        const uint32_t kt = ring + s * L::STAGE, vt = kt + L::KV_BYTES;
        const int slot0 = t * TILE + warp * WK;
        if (slot0 + WK > w.q.len) {
          // the sequence ends inside these 16 slots, or before them
          const int from = max(0, w.q.len - slot0);
          for (int i = lane; i < (WK - from) * (DIM / 8); i += 32) {
            const int r = warp * WK + from + i / (DIM / 8), ch = i % (DIM / 8);
            sts_v4(vt + (ch >> 3) * TILE * 128 + r * 128 + ((ch & 7) << 4), make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();                          // ordered before the copy that reuses the place
          __syncwarp();
        }
        float sc[2][4] = {};
        uint32_t dep = 0;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          uint32_t b[4];
          ldmatrix_x4(b, kt + (k >> 2) * TILE * 128 + k_row * 128 + ((((k & 3) * 2 + k_chunk) ^ (k_row & 7)) << 4));
          mma_16x8x16<T>(sc[0], qf[k], b[0], b[1]);
          mma_16x8x16<T>(sc[1], qf[k], b[2], b[3]);
        }
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int slot = slot0 + i * 8 + c2 + (e & 1);
            sc[i][e] = slot <= limit[e >> 1] ? sc[i][e] * p.scale_log2 : neg_inf();
            top[e >> 1] = fmaxf(top[e >> 1], sc[i][e]);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = top[h] > m[h] ? ex2(m[h] - top[h]) : 1.f;      // (m still minus infinity: zero)
            m[h] = top[h];
            l[h] *= a;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) { o[i][2 * h] *= a; o[i][2 * h + 1] *= a; }
          }
        }
        const float base[2] = {m[0] == neg_inf() ? 0.f : m[0], m[1] == neg_inf() ? 0.f : m[1]};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[i][e] = ex2(sc[i][e] - base[e >> 1]);
            l[e >> 1] += sc[i][e];
          }
        const uint32_t pf[4] = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]),
                                pack2<T>(sc[1][0], sc[1][1]), pack2<T>(sc[1][2], sc[1][3])};
        uint32_t pl[4];
        if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 hi = unpack2<T>(pf[i]);
            pl[i] = pack2<T>(sc[i >> 1][(i & 1) * 2] - hi.x, sc[i >> 1][(i & 1) * 2 + 1] - hi.y);
          }
        }
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
          uint32_t b[4];
          ldmatrix_x4_t(b, vt + (d >> 2) * TILE * 128 + v_row * 128 + ((((d & 3) * 2 + v_chunk) ^ (v_row & 7)) << 4));
          mma_16x8x16<T>(o[2 * d], pf, b[0], b[1]);
          mma_16x8x16<T>(o[2 * d + 1], pf, b[2], b[3]);
          if constexpr (!std::is_same<T, __half>::value) {
            mma_16x8x16<T>(o[2 * d], pl, b[0], b[1]);
            mma_16x8x16<T>(o[2 * d + 1], pl, b[2], b[3]);
          }
          dep ^= b[0] ^ b[3];
        }
        // handed back once the loads have returned (their registers are an input of the arrival's address); those of
        // the keys have, their products are inputs of what came since
        __syncwarp();
        if (lane == 0) mbar_arrive_after(&empty[s], dep, zero);
        if (++s == L::STAGES) { s = 0; ph ^= 1; }
      }
      // ---------------------------------------------------------- join the four warps
      float* joined = reinterpret_cast<float*>(sm + L::joined);
      float* ml = reinterpret_cast<float*>(sm + L::ml);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) {
          ml[(warp * ROWS + g + 8 * h) * 2] = m[h];
          ml[(warp * ROWS + g + 8 * h) * 2 + 1] = l[h];
        }
        if (g + 8 * h < rows) {
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i)
            *reinterpret_cast<float2*>(joined + (warp * ROWS + g + 8 * h) * DIM + i * 8 + c2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        }
      }
      // (after a wait that gave up the warp still goes to every barrier that the others wait at)
      compute_barrier();
      const bool whole = first == 0 && stop == w.tiles;
      const long long u0 = w.unit_first(), u1 = u0 + w.tiles;
      float* part = p.parts + (2 * c + (u0 < begin ? 0 : 1)) * L::PART;
      for (int e = tid; e < rows * (DIM / 2); e += WARPS * 32) {
        const int r = e / (DIM / 2), d = (e % (DIM / 2)) * 2;
        float mx = neg_inf(), lt = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < WARPS; ++k) mx = fmaxf(mx, ml[(k * ROWS + r) * 2]);
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
          const float mk = ml[(k * ROWS + r) * 2], a = mk == neg_inf() ? 0.f : ex2(mk - mx);
          const float2 v = *reinterpret_cast<const float2*>(joined + (k * ROWS + r) * DIM + d);
          lt += a * ml[(k * ROWS + r) * 2 + 1];
          acc.x += a * v.x;
          acc.y += a * v.y;
        }
        if (whole) {
          const int tok = w.q.q0 + (row0 + r) / p.group, hd = w.head * p.group + (row0 + r) % p.group;
          const float inv = lt > 0.f ? 1.f / lt : 0.f;       // a row that sees nothing is zero
          *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (long long)tok * p.o_tok + (long long)hd * p.o_head + d) = pack2<T>(acc.x * inv, acc.y * inv);
          if (p.lse && d == 0) p.lse[(long long)tok * p.n_heads + hd] = lt > 0.f ? (mx + log2f(lt)) * LN2 : lt == lt ? neg_inf() : lt;
        } else {
          *reinterpret_cast<float2*>(part + 2 * ROWS + r * DIM + d) = acc;
          if (d == 0) { part[2 * r] = mx; part[2 * r + 1] = lt; }
        }
      }
      if (!whole) {
        // runs the unit falls into: run(x) = the c with c * total / runs <= x < (c + 1) * total / runs
        const long long c0 = ((u0 + 1) * runs - 1) / total, c1 = (u1 * runs - 1) / total;
        __threadfence();
        compute_barrier();
        if (tid == 0) {
          int* a = p.arrived + c0;                           // (at most one unit is cut for the first time in a run)
          const bool last = atomicAdd(a, 1) == (int)(c1 - c0);
          if (last) *a = 0;
          __threadfence();
          *last_flag = last;
        }
        compute_barrier();
        if (*last_flag) {
          for (int e = tid; e < rows * (DIM / 2); e += WARPS * 32) {
            const int r = e / (DIM / 2), d = (e % (DIM / 2)) * 2;
            // the first part is the second of its run's two, unless the run starts with the unit's first tile; every
            // later run starts inside the unit
            float mx = neg_inf(), lt = 0.f;
            float2 acc = make_float2(0.f, 0.f);
            for (long long k = c0; k <= c1; ++k) {
              const float* q = p.parts + (2 * k + (k == c0 ? 1 : 0)) * L::PART;
              mx = fmaxf(mx, __ldcg(q + 2 * r));
            }
            for (long long k = c0; k <= c1; ++k) {
              const float* q = p.parts + (2 * k + (k == c0 ? 1 : 0)) * L::PART;
              const float mk = __ldcg(q + 2 * r), a = mk == neg_inf() ? 0.f : ex2(mk - mx);
              const float2 v = __ldcg(reinterpret_cast<const float2*>(q + 2 * ROWS + r * DIM + d));
              lt += a * __ldcg(q + 2 * r + 1);
              acc.x += a * v.x;
              acc.y += a * v.y;
            }
            const int tok = w.q.q0 + (row0 + r) / p.group, hd = w.head * p.group + (row0 + r) % p.group;
            const float inv = lt > 0.f ? 1.f / lt : 0.f;
            *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (long long)tok * p.o_tok + (long long)hd * p.o_head + d) = pack2<T>(acc.x * inv, acc.y * inv);
            if (p.lse && d == 0) p.lse[(long long)tok * p.n_heads + hd] = lt > 0.f ? (mx + log2f(lt)) * LN2 : lt == lt ? neg_inf() : lt;
          }
        }
      }
      compute_barrier();                                     // the joining buffers are free again
      if (u0 + stop >= end) break;
      w.next_unit(p);
    }
  }
  // After a wait that gave up copies may still be in flight: the block stays for a millisecond, many times what they
  // need, before its shared memory is handed on.
  if (__syncthreads_or(!ok)) {
    if (tid == 0)
      for (const uint64_t t0 = wide::timer_ns(); wide::timer_ns() - t0 < 1000000;) __nanosleep(1000);
    __syncthreads();
  }
}

}  // namespace pdec
}  // namespace w4a4
