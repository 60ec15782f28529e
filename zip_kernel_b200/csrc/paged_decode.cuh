// Attention of few query rows per key/value head over a paged cache: decode steps, and chunks of a few tokens.
//
//   o[r] = sum_j p[r,j] v[j] / sum_j p[r,j],  p[r,j] = exp(scale q[r].k[j] - m[r]),  j up to the row's own slot,
//
// the running maximum m, the sum and o carried through one pass over the slots (o and the sum are multiplied by
// exp(m_old - m_new) when the maximum grows; fp16 weights are 2^15 times as large, see WEIGHT_SHIFT).  A row = (new token,
// head of the group that shares the key/value head); up to 16 rows fill the M side of an m16n8k16 product.
//
// What bounds it: every key and value is read once from HBM, 2 * dim * 2 bytes for 4 * 16 * dim multiply-adds at most.
// So the whole card must stream, whatever the number and lengths of the sequences: the 64-slot tiles of all (sequence,
// head, row tile) units are laid end to end and cut into one equal run per CTA.  A unit that falls into several runs
// is joined by the CTA that finishes its last part (the parts' order, and so the result's bits, depend on the lengths
// alone).
//
// A CTA has one warp that issues copies (TMA boxes of one page each, 128-byte swizzle, a ring of tiles) and two teams of
// four that compute on alternate tiles, each warp on 16 slots of a tile with a maximum, sum and output of its own, joined
// at the end of a unit: no barrier between the warps inside a unit.  Measured, 32 histories up to 4096 slots of 8
// key/value heads at dim 128: 55 us, 4.9 TB/s.
//
// Rows of values past the sequence's last slot are set to zero in shared memory first: a stale NaN there times a
// weight of zero would be NaN.  Scores there are replaced, not added to.  Weights enter the second product as the
// sum of two 16-bit values (the rounded one and what its rounding left), so that only the output is rounded to its type; the
// tensor time is there to spare (measured with and without as fp16: 32 histories up to 4096 slots 55.1 and 53.4 us by graph
// replay, 67.6 either way with cold caches, one of 8191 16.4 either way).
#pragma once

#include "paged_kv.cuh"
#include "prefill_wide_gemm.cuh"

namespace w4a4 {
namespace pdec {

using namespace kv;

constexpr int TILE = 64, WK = 16, ROWS = 16;
constexpr int SHARE = TILE / WK, TEAMS = 2, WARPS = TEAMS * SHARE;      // warps that share a tile, teams that take turns
constexpr int THREADS = (WARPS + 4) * 32;                    // a third warpgroup: the copying warp, and three to fill it
// Registers of the launch, 168 a thread, dealt out again: with 168 for the arithmetic the loop over tiles spills (a
// batch of 32 histories up to 4096 slots 72 us with 208 bytes spilled, 57 us with 116).
constexpr int REG_COPY = 72, REG_COMPUTE = 216;
static_assert(REG_COPY + 2 * REG_COMPUTE <= 3 * 168, "the warpgroups share the registers of the launch");
constexpr int MAX_RUNS = 256;                                // CTAs of a launch

enum : int { SITE_PDEC_FULL = 35, SITE_PDEC_EMPTY, SITE_PDEC_DRAIN };

template <int DIM>
struct Layout {
  static constexpr int HALVES = DIM / 64;                    // 128-byte wide column blocks
  static constexpr int KV_BYTES = TILE * DIM * 2;            // one tile of keys, or of values
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int STAGES = DIM == 128 ? 6 : 12;
  // A place of the ring belongs to one team: a team that met a place's barrier only every second phase could take the
  // phase before the last for the last, they have the same parity.
  static_assert(STAGES % TEAMS == 0, "a team waits for every phase of the barriers that it waits for");
  // a part of a unit in the workspace: m and l of the rows, then their outputs
  static constexpr int PART = ROWS * (2 + DIM);
  static constexpr int joined = STAGES * STAGE;              // float [SHARE][ROWS][DIM]; weights of the parts of a unit
  static constexpr int JOINED = SHARE * ROWS * DIM * 4 > MAX_RUNS * ROWS * 4 ? SHARE * ROWS * DIM * 4 : MAX_RUNS * ROWS * 4;
  static constexpr int ml = joined + JOINED;                 // float [SHARE][ROWS][2]
  static constexpr int bars = ml + SHARE * ROWS * 2 * 4;
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

// What a unit costs besides its tiles - its queries, the joining of the warps - in tiles: runs are cut as if every unit
// had that many more.  Measured, 32 sequences of 1 to 4096 slots x 8 heads: SMs busy 49 us on average and 67 us at most
// without.
constexpr int PAD = 3;

// Row tiles and steps (PAD and then the slot tiles) of sequence b in this kernel: none when it has no new token or more
// rows than max_rows.
__device__ __forceinline__ void unit_shape(const Params& p, const Seq& q, int& row_tiles, int& tiles) {
  const long long rows = (long long)q.q_len * p.group;
  const bool mine = q.q_len > 0 && rows <= p.max_rows;
  row_tiles = mine ? (int)((rows + ROWS - 1) / ROWS) : 0;
  tiles = mine ? PAD + max(1, (q.len + TILE - 1) / TILE) : 0;
}

// D(16x8, f32) += A(16x16) B(16x8).  With MH == 1 rows 8 to 15 are empty: d[2] and d[3] neither live nor enter.
#define W4A4_MMA16(TYPE)                                                                                                      \
  if constexpr (MH == 2)                                                                                                      \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"   \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));     \
  else {                                                                                                                      \
    float x, y;                                                                                                               \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"   \
        : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y) : "r"(a[0]), "r"(0), "r"(a[2]), "r"(b0), "r"(b1), "f"(0.f));               \
  }
template <typename T, int MH>
__device__ __forceinline__ void mma_16x8x16(float (&d)[2 * MH], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) { W4A4_MMA16("f16") }
  else { W4A4_MMA16("bf16") }
}
#undef W4A4_MMA16
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); }

// Two elements of a row's output (a row that sees nothing is zero), and its lse with the first.
template <typename T>
__device__ __forceinline__ void write_out(const Params& p, int tok, int hd, int d, const float2& acc, float m, float l) {
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (long long)tok * p.o_tok + (long long)hd * p.o_head + d) = pack2<T>(acc.x * inv, acc.y * inv);
  if (p.lse && d == 0) p.lse[(long long)tok * p.n_heads + hd] = l > 0.f ? (m + log2f(l)) * LN2 : l == l ? neg_inf() : l;
}

// Joins the parts of a unit (all computing warps).
template <typename T, int DIM>
__device__ __forceinline__ void join_parts(const Params& p, long long c0, int parts, int rows, int q0, int head, int row0, float* wt, float* ml) {
  using L = Layout<DIM>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the first part is the second of its run's two (the unit begins in that run), the others their run's first
  auto part_of = [&](int k) { return p.parts + (2 * (c0 + k) + (k == 0 ? 1 : 0)) * L::PART; };
  // the outputs of the first parts are on their way while the weights (wt [row][part]) are made
  constexpr int AHEAD = 16;
  const int elements = rows * (DIM / 2);
  float2 v[AHEAD];
  auto fetch = [&](int e, int k0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (e < elements && k0 + k < parts)
        v[k] = __ldcg(reinterpret_cast<const float2*>(part_of(k0 + k) + 2 * ROWS + e / (DIM / 2) * DIM + (e % (DIM / 2)) * 2));
  };
  fetch(tid, 0);
  for (int r = warp; r < rows; r += WARPS) {
    float mx = neg_inf(), lt = 0.f;
    for (int k = lane; k < parts; k += 32) mx = fmaxf(mx, __ldcg(part_of(k) + 2 * r));
#pragma unroll
    for (int s = 16; s > 0; s /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    for (int k = lane; k < parts; k += 32) {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(part_of(k)) + r);
      const float a = x.x == neg_inf() ? (x.y == x.y ? 0.f : 1.f) : ex2(x.x - mx);
      lt += a * x.y;
      wt[r * MAX_RUNS + k] = a;
    }
#pragma unroll
    for (int s = 16; s > 0; s /= 2) lt += __shfl_xor_sync(0xffffffffu, lt, s);
    if (lane == 0) { ml[2 * r] = mx; ml[2 * r + 1] = lt; }
  }
  compute_barrier();
  for (int e = tid; e < elements; e += WARPS * 32) {
    const int r = e / (DIM / 2), d = (e % (DIM / 2)) * 2;
    float2 acc = make_float2(0.f, 0.f);
    for (int k0 = 0; k0 < parts; k0 += AHEAD) {
      if (e != tid || k0 > 0) fetch(e, k0);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (k0 + k < parts) {
          const float a = wt[r * MAX_RUNS + k0 + k];
          acc.x += a * v[k].x;
          acc.y += a * v[k].y;
        }
    }
    write_out<T>(p, q0 + (row0 + r) / p.group, head * p.group + (row0 + r) % p.group, d, acc, ml[2 * r], ml[2 * r + 1]);
  }
}

// MH: eight-row halves of a row tile that are in use
template <typename T, int DIM, int MH>
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
      mbar_init(&empty[i], SHARE);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncthreads();
  if (warp == WARPS) grid_dependency_wait_for_async_reads();
  else grid_dependency_wait();

  const int c = blockIdx.x;                                  // run; there may be fewer, then the CTA has nothing to do
  const uint32_t ring = smem_u32(sm);
  bool ok = true;                                            // no wait of this thread has given up

  if (warp >= WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_COPY));
    if (warp == WARPS) {
    // ------------------------------------------------------------ copies
    Walk<Params> w;
    long long total, runs, begin, end;
    const bool any = w.start(p, gridDim.x, c, total, runs, begin, end);
    PagesAhead pages;
    int s = 0;
    uint32_t ph = 1;
    long long n = 0;
    while (any && ok) {
      const int stop = (int)min((long long)w.tiles, w.tile + (end - w.at));
      for (int t = max(w.tile - PAD, 0); t < stop - PAD; ++t, ++n) {
        if (n >= L::STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ph, SITE_PDEC_EMPTY));
        if (!ok) break;
        // one lane per box; boxes with no slot in use are not copied
        const int boxes = TILE / p.box, slot = t * TILE + lane * p.box;
        const bool mine = lane < boxes && slot < w.q.len;
        const int page = pages.get(p.c, w.b, w.q.len, p.box, t * boxes);
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
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_COMPUTE));
    // ------------------------------------------------------------ arithmetic
    const int g = lane >> 2, c2 = (lane & 3) * 2;            // fragment row (and row + 8), first of two columns
    Walk<Params> w;
    long long total, runs, begin, end;
    const bool any = w.start(p, gridDim.x, c, total, runs, begin, end);
    const int team = warp / SHARE, share = warp % SHARE;
    uint32_t n = 0;                                          // tiles of the run before this unit
    // addresses inside a tile: this lane's ldmatrix row and the swizzle of its 16-byte chunks
    const int k_row = share * WK + (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;
    const int v_row = share * WK + (lane & 15), v_chunk = lane >> 4;
    // A fragments of a unit's rows (rows that do not exist are zero), and the last slots that they see
    uint32_t qf[DIM / 16][4];
    int limit[MH];
    auto load_rows = [&](const Walk<Params>& u) {
      const int left = u.q.q_len * p.group - u.row_tile * ROWS;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h, tok = (u.row_tile * ROWS + r) / p.group, hd = (u.row_tile * ROWS + r) % p.group;
        const bool live = h < MH && r < left;
        const T* src = static_cast<const T*>(p.q) + (long long)(u.q.q0 + (live ? tok : 0)) * p.q_tok + (long long)(u.head * p.group + (live ? hd : 0)) * p.q_head;
        if (h < MH) limit[h < MH ? h : 0] = live ? u.q.len - u.q.q_len + tok : -1;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          qf[k][h] = live ? ld_plain(reinterpret_cast<const uint32_t*>(src + k * 16 + c2)) : 0;
          qf[k][h + 2] = live ? ld_plain(reinterpret_cast<const uint32_t*>(src + k * 16 + 8 + c2)) : 0;
        }
      }
    };
    if (any) load_rows(w);
    while (any) {
      const int row0 = w.row_tile * ROWS, rows = min(ROWS, w.q.q_len * p.group - row0);
      float o[DIM / 8][2 * MH], m[MH], l[MH];
#pragma unroll
      for (int h = 0; h < MH; ++h) { m[h] = neg_inf(); l[h] = 0.f; }
#pragma unroll
      for (int i = 0; i < DIM / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2 * MH; ++e) o[i][e] = 0.f;

      const int stop_step = (int)min((long long)w.tiles, w.tile + (end - w.at));
      const int first = max(w.tile - PAD, 0), stop = max(stop_step - PAD, 0);
      for (int t = first + ((n ^ team) & 1); t < stop; t += TEAMS) {
        const uint32_t place = n + (t - first), s = place % L::STAGES;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[s], place / L::STAGES & 1, SITE_PDEC_FULL));
        if (!ok) break;
        const uint32_t kt = ring + s * L::STAGE, vt = kt + L::KV_BYTES;
        const int slot0 = t * TILE + share * WK;
        if (slot0 + WK > w.q.len) {
          // the sequence ends inside these 16 slots, or before them
          const int from = max(0, w.q.len - slot0);
          for (int i = lane; i < (WK - from) * (DIM / 8); i += 32) {
            const int r = share * WK + from + i / (DIM / 8), ch = i % (DIM / 8);
            sts_v4(vt + (ch >> 3) * TILE * 128 + r * 128 + ((ch & 7) << 4), make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();                          // ordered before the copy that reuses the place
          __syncwarp();
        }
        float sc[2][2 * MH] = {}, sd[2][2 * MH] = {};                  // two chains of products, added at the end
        uint32_t dep = 0;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          uint32_t b[4];
          ldmatrix_x4(b, kt + (k >> 2) * TILE * 128 + k_row * 128 + ((((k & 3) * 2 + k_chunk) ^ (k_row & 7)) << 4));
          mma_16x8x16<T, MH>(k & 1 ? sd[0] : sc[0], qf[k], b[0], b[1]);
          mma_16x8x16<T, MH>(k & 1 ? sd[1] : sc[1], qf[k], b[2], b[3]);
        }
        float top[MH];
        bool grown = false;
#pragma unroll
        for (int h = 0; h < MH; ++h) top[h] = neg_inf();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 2 * MH; ++e) {
            const int slot = slot0 + i * 8 + c2 + (e & 1);
            sc[i][e] = slot <= limit[e >> 1] ? (sc[i][e] + sd[i][e]) * p.scale_log2 : neg_inf();
            top[e >> 1] = fmaxf(top[e >> 1], sc[i][e]);
          }
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
          top[h] = fmaxf(m[h], below_max(top[h], WEIGHT_SHIFT<T>));
          grown |= top[h] > m[h];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int h = 0; h < MH; ++h) {
            const float a = top[h] > m[h] ? ex2(m[h] - top[h]) : 1.f;      // (m still minus infinity: zero)
            m[h] = top[h];
            l[h] *= a;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) { o[i][2 * h] *= a; o[i][2 * h + 1] *= a; }
          }
        }
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          const float base = m[h] == neg_inf() ? 0.f : m[h];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) {
              sc[i][e] = ex2(sc[i][e] - base);
              l[h] += sc[i][e];
            }
        }
        uint32_t pf[4] = {}, pl[4] = {};                     // (slots 0-7 | 8-15) x (rows 0-7, 8-15): the A fragment
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < MH; ++h) {
            pf[2 * i + h] = pack2<T>(sc[i][2 * h], sc[i][2 * h + 1]);
            const float2 hi = unpack2<T>(pf[2 * i + h]);
            pl[2 * i + h] = pack2<T>(sc[i][2 * h] - hi.x, sc[i][2 * h + 1] - hi.y);
          }
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
          uint32_t b[4];
          ldmatrix_x4_t(b, vt + (d >> 2) * TILE * 128 + v_row * 128 + ((((d & 3) * 2 + v_chunk) ^ (v_row & 7)) << 4));
          mma_16x8x16<T, MH>(o[2 * d], pf, b[0], b[1]);
          mma_16x8x16<T, MH>(o[2 * d + 1], pf, b[2], b[3]);
          mma_16x8x16<T, MH>(o[2 * d], pl, b[0], b[1]);
          mma_16x8x16<T, MH>(o[2 * d + 1], pl, b[2], b[3]);
          dep ^= b[0] ^ b[3];
        }
        // handed back once the loads have returned (their registers are an input of the arrival's address); those of
        // the keys have, their products are inputs of what came since
        __syncwarp();
        if (lane == 0) mbar_arrive_after(&empty[s], dep, zero);
      }
      n += stop - first;
      // the next unit's queries are under way while this one is joined
      const Walk<Params> u = w;
      const bool more = w.at - w.tile + stop_step < end;
      if (more) {
        w.next_unit(p);
        load_rows(w);
      }
      if (stop > first) {
      // ---------------------------------------------------------- join the warps
      float* joined = reinterpret_cast<float*>(sm + L::joined);
      float* ml = reinterpret_cast<float*>(sm + L::ml);
      auto place_of = [&](int h, int i) { return reinterpret_cast<float2*>(joined + (share * ROWS + g + 8 * h) * DIM + i * 8 + c2); };
      auto leave = [&]() {                                   // this warp's m, l and outputs
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + (share * ROWS + g + 8 * h) * 2) = make_float2(m[h], l[h]);
          if (g + 8 * h < rows)
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) *place_of(h, i) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        }
      };
#pragma unroll
      for (int h = 0; h < MH; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      }
      if (team == 1) leave();
      compute_barrier();
      if (team == 0) {
        // takes over what the other team's warp with the same slots of a tile has
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          const float2 other = *reinterpret_cast<const float2*>(ml + (share * ROWS + g + 8 * h) * 2);
          const float mx = fmaxf(m[h], other.x);
          const float a = m[h] == neg_inf() ? 0.f : ex2(m[h] - mx), d = other.x == neg_inf() ? 0.f : ex2(other.x - mx);
          m[h] = mx;
          l[h] = a * l[h] + d * other.y;
          if (g + 8 * h < rows)
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) {
              const float2 v = *place_of(h, i);
              o[i][2 * h] = a * o[i][2 * h] + d * v.x;
              o[i][2 * h + 1] = a * o[i][2 * h + 1] + d * v.y;
            }
        }
        __syncwarp();
        leave();
      }
      // (after a wait that gave up the warp still goes to every barrier that the others wait at)
      compute_barrier();
      const bool whole = first == 0 && stop == u.tiles - PAD;
      const long long u0 = u.unit_first() + PAD, u1 = u0 + u.tiles - PAD;
      float* part = p.parts + (2 * c + (u0 < begin ? 0 : 1)) * L::PART;
      for (int e = tid; e < rows * (DIM / 2); e += WARPS * 32) {
        const int r = e / (DIM / 2), d = (e % (DIM / 2)) * 2;
        float mx = neg_inf(), lt = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < SHARE; ++k) mx = fmaxf(mx, ml[(k * ROWS + r) * 2]);
#pragma unroll
        for (int k = 0; k < SHARE; ++k) {
          const float mk = ml[(k * ROWS + r) * 2], a = mk == neg_inf() ? 0.f : ex2(mk - mx);
          const float2 v = *reinterpret_cast<const float2*>(joined + (k * ROWS + r) * DIM + d);
          lt += a * ml[(k * ROWS + r) * 2 + 1];
          acc.x += a * v.x;
          acc.y += a * v.y;
        }
        if (whole) {
          write_out<T>(p, u.q.q0 + (row0 + r) / p.group, u.head * p.group + (row0 + r) % p.group, d, acc, mx, lt);
        } else {
          *reinterpret_cast<float2*>(part + 2 * ROWS + r * DIM + d) = acc;
          if (d == 0) { part[2 * r] = mx; part[2 * r + 1] = lt; }
        }
      }
      if (!whole) {
        // runs the unit falls into: run(x) = the c with c * total / runs <= x < (c + 1) * total / runs
        const long long c0 = ((u0 + 1) * runs - 1) / total, c1 = (u1 * runs - 1) / total;
        compute_barrier();
        if (tid == 0) {
          __threadfence();                                   // (and with it what the barrier has ordered before)
          int* a = p.arrived + c0;                           // (at most one unit is cut for the first time in a run)
          const bool last = atomicAdd(a, 1) == (int)(c1 - c0);
          if (last) *a = 0;
          __threadfence();
          *last_flag = last;
        }
        compute_barrier();
        if (*last_flag) join_parts<T, DIM>(p, c0, (int)(c1 - c0) + 1, rows, u.q.q0, u.head, row0, joined, ml);
      }
      compute_barrier();                                     // the joining buffers are free again
      }
      if (!more) break;
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
