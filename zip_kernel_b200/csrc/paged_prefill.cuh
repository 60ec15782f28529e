// Attention of many query rows per key/value head over a paged cache: prompts and chunks of them.
//
//   o[r] = sum_j p[r,j] v[j] / sum_j p[r,j],  p[r,j] = exp(scale q[r].k[j] - m[r]),  j up to the row's own slot,
//
// in one pass over 128-slot tiles.  A row = (new token, head of the group that shares the key/value head): a tile of 128
// rows holds whole tokens, so the heads of a group share every key and value tile, and a block has two row tiles, whose
// products and softmax alternate: while the tensor cores work on one, the other's softmax warps have the CUDA cores.
//
// Roles: a warp that issues copies (TMA boxes of one page each), a thread that issues MMAs, four warps of softmax per
// row tile.  Scores are 128 x 128 fp32 in tensor memory, thread = row; the weights go back there as 16-bit pairs over
// the scores and are the A operand of the second product, whose B operand is the value tile as it lands (slots x
// elements, read along the elements).  The output stays in tensor memory; it is multiplied by exp(m_old - m_new) only
// when some row's maximum has grown by more than a factor of 2^8, until when the weights are simply larger than one
// (2^8 at most: exact in the sum, no worse rounded).  What a row's weights are rounded to (16 bits) is half a step of
// the output's own type.
//
// The order PV(j), S(j + 1) in the issuing thread makes one barrier do for two things: the scores of step j + 1 are
// complete only after the product that reads the weights of step j and writes the output, so the softmax warps may
// overwrite the one and multiply the other.
//
// What bounds it: products and exponentials alike, 2048 clocks each per step of both row tiles at dim 128.
#pragma once

#include "cache_sums.cuh"

namespace w4a4 {
namespace ppre {

using namespace kv;
using csum::idesc_f16;
using csum::umma_f16;

constexpr int TILE = 128, ROWS = 128;                        // slots of a tile, rows of a row tile
constexpr int WARP_COPY = 8, WARP_MMA = 9, THREADS = 12 * 32;
constexpr int REG_ISSUE = 56, REG_SOFTMAX = 224;
static_assert(REG_ISSUE + 2 * REG_SOFTMAX <= 3 * 168, "the warpgroups share the registers of the launch");
constexpr int TMEM_COLS = 512, TMEM_O = 256;
constexpr float GROWTH = 8.f;                                // (log2) of a row's maximum before the output follows

enum : int { SITE_PPRE_EMPTY = 80, SITE_PPRE_Q, SITE_PPRE_K, SITE_PPRE_V, SITE_PPRE_P, SITE_PPRE_S, SITE_PPRE_VZERO, SITE_PPRE_O };

template <int DIM>
struct Layout {
  static constexpr int HALVES = DIM / 64;
  static constexpr int SLOT = TILE * DIM * 2;                // a tile of keys, or of values, or of query rows
  static constexpr int STAGES = DIM == 128 ? 5 : 10;
  static constexpr int q = STAGES * SLOT;
  static constexpr int bars = q + 2 * SLOT;
  static constexpr int total = bars + (2 * STAGES + 8) * 8 + 16;
  static_assert(1024 + total <= 232448, "shared memory of one SM");
};
template <int DIM> inline size_t smem_bytes() { return 1024 + Layout<DIM>::total; }

struct Params {
  Cache c;
  Seqs s;
  void* out;
  long long o_tok, o_head;
  float* lse;                 // (T, n_heads), or NULL
  float* parts;               // [splits][T * n_heads][dim], or NULL when splits == 1
  float* parts_ml;            // [splits][T * n_heads][2]
  int n_heads, group, box, toks, min_rows, splits;
  float scale_log2;
};

// Blocks (pairs of row tiles) of sequence b in this kernel.
__device__ __forceinline__ int seq_blocks(const Params& p, const Seq& q) {
  return (long long)q.q_len * p.group > p.min_rows ? (q.q_len + 2 * p.toks - 1) / (2 * p.toks) : 0;
}

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
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_q, const Params p) {
  using L = Layout<DIM>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);    // ring of key and value tiles in turn
  uint64_t* empty = full + L::STAGES;
  uint64_t* q_full = empty + L::STAGES;                          // [2] per row tile, as the next three
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < L::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
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

  // The block's sequence: the last blocks of a sequence, which see most slots, come first.
  int b = -1, blk = 0;
  Seq q{};
  {
    int before = 0;
    const int r = blockIdx.x;
    for (int base = 0; base < p.s.n && b < 0; base += 32) {
      int n = base + lane < p.s.n ? seq_blocks(p, load_seq(p.s, base + lane)) : 0, w = n;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += a;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + w > r);
      if (past) {
        const int i = __ffs(past) - 1;
        b = base + i;
        blk = before + __shfl_sync(0xffffffffu, w, i) - 1 - r;
        q = load_seq(p.s, b);
      }
      before += __shfl_sync(0xffffffffu, w, 31);
    }
  }
  const int head = blockIdx.y, split = blockIdx.z;
  bool ok = true;                                          // no wait of this thread has given up
  if (b >= 0) {
    const int tok0 = blk * 2 * p.toks, past_len = q.len - q.q_len;
    // tiles of either row tile up to its last row's slot; none when it has no row or its rows see nothing
    int n_all[2], n[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int t0 = tok0 + t * p.toks, t1 = min(t0 + p.toks, q.q_len);
      n_all[t] = t0 < q.q_len ? max(0, (past_len + t1 + TILE - 1) / TILE) : 0;
    }
    // this split's share of the tiles of the longer one
    const int n_max = max(n_all[0], n_all[1]);
    const int j0 = (int)((long long)n_max * split / p.splits), j1 = (int)((long long)n_max * (split + 1) / p.splits);
#pragma unroll
    for (int t = 0; t < 2; ++t) n[t] = max(j0, min(j1, n_all[t]));
    const int j_end = max(n[0], n[1]);

    if (warp >= WARP_COPY) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_ISSUE));
      if (warp == WARP_COPY) {
        // ---------------------------------------------------------- copies
        if (lane == 0) {
          for (int t = 0; t < 2; ++t) {
            if (n[t] == j0) continue;
            mbar_arrive_expect_tx(&q_full[t], p.toks * p.group * DIM * 2);
            for (int h = 0; h < L::HALVES; ++h)
              tma_load_3d(sm + L::q + t * L::SLOT + h * ROWS * 128, &tm_q, h * 64, head * p.group, q.q0 + tok0 + t * p.toks, &q_full[t]);
          }
        }
        __syncwarp();
        int s = 0;
        uint32_t ph = 1;
        const int boxes = TILE / p.box;                    // at most 8
        PagesAhead pages;
        for (int j = j0; ok && j < j_end; ++j) {
          const int slot = j * TILE + lane * p.box;
          const bool mine = lane < boxes && slot < q.len;
          const int page = pages.get(p.c, b, q.len, p.box, j * boxes);
          const int live = __popc(__ballot_sync(0xffffffffu, mine)), in_page = slot % p.c.page;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (2 * (j - j0) + kv >= L::STAGES && ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&empty[s], ph, SITE_PPRE_EMPTY));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], live * p.box * DIM * 2);
            __syncwarp();
            if (mine)
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h)
                tma_load_4d(smem_u32(sm) + s * L::SLOT + h * TILE * 128 + lane * p.box * 128, kv ? &tm_v : &tm_k, h * 64, in_page,
                            head, page, &full[s]);
            if (++s == L::STAGES) { s = 0; ph ^= 1; }
          }
        }
      } else if (warp == WARP_MMA) {
        // ---------------------------------------------------------- MMAs
        const uint32_t id_s = idesc_f16<T>(TILE), id_o = idesc_f16<T>(DIM) | (1u << 16);
        int s = 0;
        uint32_t ph = 0;
        auto next = [&]() { if (++s == L::STAGES) { s = 0; ph ^= 1; } };
        auto scores = [&](int t, int slot) {
          if (lane == 0) {
#pragma unroll
            for (int h = 0; h < L::HALVES; ++h) {
              const uint64_t a = pre::smem_desc_sw128(sm + L::q + t * L::SLOT + h * ROWS * 128);
              const uint64_t bd = pre::smem_desc_sw128(sm + slot * L::SLOT + h * TILE * 128);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16(tmem_base + t * TILE, a + 2 * k, bd + 2 * k, h > 0 || k > 0, id_s);
            }
            pre::umma_commit(&s_full[t]);
          }
          __syncwarp();
        };
        auto release = [&](int slot) {
          if (lane == 0) pre::umma_commit(&empty[slot]);
          __syncwarp();
        };
        if (j0 < j_end) {
          ok = __all_sync(0xffffffffu, wide::wait_suspend(&full[s], ph, SITE_PPRE_K));
          for (int t = 0; ok && t < 2; ++t) {
            if (n[t] == j0) continue;
            ok = __all_sync(0xffffffffu, wide::wait_suspend(&q_full[t], 0, SITE_PPRE_Q));
            if (!ok) break;
            pre::tc_fence_after();
            scores(t, s);
          }
          if (ok) release(s);
          next();
        }
        for (int j = j0; ok && j < j_end; ++j) {
          const int vs = s;
          ok = __all_sync(0xffffffffu, wide::wait_suspend(&full[s], ph, SITE_PPRE_V));
          next();
          const int ks = s;
          const uint32_t kph = ph;
          bool k_here = false;
          for (int t = 0; ok && t < 2; ++t) {
            if (j >= n[t]) continue;
            ok = __all_sync(0xffffffffu, wide::wait_suspend(&p_full[t], (j - j0) & 1, SITE_PPRE_P));
            if (!ok) break;
            pre::tc_fence_after();
            if (lane == 0) {
              const uint64_t bd = smem_desc_mn_sw128(smem_u32(sm + vs * L::SLOT), TILE * 128);
#pragma unroll
              for (int k = 0; k < TILE / 16; ++k)
                umma_f16_ta(tmem_base + TMEM_O + t * DIM, tmem_base + t * TILE + k * 8, bd + k * (2048 >> 4), j > j0 || k > 0, id_o);
              if (j == n[t] - 1) pre::umma_commit(&o_full[t]);
            }
            __syncwarp();
            if (j + 1 < n[t]) {
              if (!k_here) ok = __all_sync(0xffffffffu, wide::wait_suspend(&full[ks], kph, SITE_PPRE_K));
              k_here = true;
              if (!ok) break;
              pre::tc_fence_after();
              scores(t, ks);
            }
          }
          if (ok) release(vs);
          if (j + 1 < j_end) {
            if (ok) release(ks);
            next();
          }
        }
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFTMAX));
      // ------------------------------------------------------------ softmax: thread = row
      const int t = warp >> 2, row = tid & 127;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem_base + lanes + t * TILE, to = tmem_base + lanes + TMEM_O + t * DIM;
      const int tok = tok0 + t * p.toks + row / p.group;
      const bool live = row < p.toks * p.group && tok < q.q_len;
      const int limit = live ? past_len + tok : -1;        // last slot this row sees
      float m = neg_inf(), l = 0.f;
      for (int j = j0; j < n[t]; ++j) {
        if (ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&s_full[t], (j - j0) & 1, SITE_PPRE_S));
        if (!ok) break;
        pre::tc_fence_after();
        uint32_t x[TILE];
#pragma unroll
        for (int c = 0; c < TILE; c += 32) tmem_ld32_issue(ts + c, x + c);
        tmem_ld_wait();
        const int last = limit - j * TILE;                 // last visible column
        if (!__all_sync(0xffffffffu, last >= TILE - 1)) {
#pragma unroll
          for (int c = 0; c < TILE; ++c) x[c] = c <= last ? x[c] : 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = __uint_as_float(x[i]);
#pragma unroll
        for (int c = 4; c < TILE; ++c) top[c & 3] = fmaxf(top[c & 3], __uint_as_float(x[c]));
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
        if (__any_sync(0xffffffffu, mx > m + GROWTH)) {
          const float a = mx > m ? ex2(m - mx) : 1.f;      // (m still minus infinity: zero)
          m = fmaxf(m, mx);
          l *= a;
          if (j > j0) {
#pragma unroll
            for (int c = 0; c < DIM; c += 32) {
              uint32_t o[32];
              tmem_ld32_issue(to + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
              pre::tmem_st32(to + c, o);
            }
          }
        }
        const float base = m == neg_inf() ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < TILE; c += 64) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float p0 = ex2(fmaf(__uint_as_float(x[c + i]), p.scale_log2, -base));
            const float p1 = ex2(fmaf(__uint_as_float(x[c + i + 1]), p.scale_log2, -base));
            sum[i & 2] += p0;
            sum[(i & 2) + 1] += p1;
            w[i / 2] = pack2<T>(p0, p1);
          }
          pre::tmem_st32(ts + c / 2, w);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if ((j + 1) * TILE > q.len) {
          // the sequence ends in this tile: values behind it become zero before a product reads them
          const int k = 2 * (j - j0) + 1, s = k % L::STAGES;
          ok = __all_sync(0xffffffffu, wide::wait_suspend(&full[s], (k / L::STAGES) & 1, SITE_PPRE_VZERO));
          if (!ok) break;
          if (j * TILE + row >= q.len) {
#pragma unroll
            for (int ch = 0; ch < DIM / 8; ++ch)
              sts_v4(smem_u32(sm) + s * L::SLOT + (ch >> 3) * TILE * 128 + row * 128 + ((ch & 7) << 4), make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();
        }
        pre::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      // ------------------------------------------------------------ output
      const int hd = head * p.group + row % p.group;
      const bool any = n[t] > j0;
      if (any && ok) ok = __all_sync(0xffffffffu, wide::wait_suspend(&o_full[t], 0, SITE_PPRE_O));
      if (ok) {
        pre::tc_fence_after();
        const long long tr = q.q0 + tok;
        const float inv = l > 0.f ? 1.f / l : 0.f;         // a row that sees nothing is zero
        const long long idx = ((long long)split * p.s.T + tr) * p.n_heads + hd;
        if (live) {
          if (p.splits > 1) {
            *reinterpret_cast<float2*>(p.parts_ml + 2 * idx) = make_float2(m, l);
          } else if (p.lse) {
            p.lse[tr * p.n_heads + hd] = l > 0.f ? (m + log2f(l)) * LN2 : neg_inf();
          }
        }
#pragma unroll
        for (int c = 0; c < DIM; c += 32) {
          uint32_t o[32];
          if (any) {
            tmem_ld32_issue(to + c, o);
            tmem_ld_wait();
          }
          if (!live) continue;
          if (!(l > 0.f)) {
            // nothing was summed (or a NaN was): what the accumulator holds does not count, a NaN stays one
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = l == l ? 0u : 0x7fffffffu;
          }
          if (p.splits > 1) {
            float4* dst = reinterpret_cast<float4*>(p.parts + idx * DIM + c);
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              dst[i / 4] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
          } else {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + tr * p.o_tok + (long long)hd * p.o_head + c);
            const float f = l == l ? inv : 1.f;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              dst[i / 8] = make_uint4(pack2<T>(__uint_as_float(o[i]) * f, __uint_as_float(o[i + 1]) * f), pack2<T>(__uint_as_float(o[i + 2]) * f, __uint_as_float(o[i + 3]) * f),
                                      pack2<T>(__uint_as_float(o[i + 4]) * f, __uint_as_float(o[i + 5]) * f), pack2<T>(__uint_as_float(o[i + 6]) * f, __uint_as_float(o[i + 7]) * f));
          }
        }
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

// Joins the splits of the kernel above: a warp per (token, head), in the order of the splits.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) paged_join_kernel(const Params p) {
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)p.s.T * p.n_heads;
  grid_dependency_wait();
  if (row >= rows) return;
  const int t = (int)(row / p.n_heads), hd = (int)(row % p.n_heads);
  int below = 0;
  for (int i = lane; i <= p.s.n; i += 32) below += ld_plain(p.s.cu + i) <= t;
  const int b = __reduce_add_sync(0xffffffffu, below) - 1;
  if (b < 0 || b >= p.s.n) return;
  const Seq q = load_seq(p.s, b);
  if (seq_blocks(p, q) == 0 || t >= q.q0 + q.q_len) return;
  constexpr int E = DIM / 32;
  float m = neg_inf(), l = 0.f, acc[E] = {};
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.parts_ml[2 * (s * rows + row)]);
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.parts_ml + 2 * (s * rows + row));
    const float a = ml.x == neg_inf() ? (ml.y == ml.y ? 0.f : 1.f) : ex2(ml.x - m);
    l += a * ml.y;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] += a * p.parts[(s * rows + row) * DIM + lane * E + i];
  }
  const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : 1.f;
  T* dst = static_cast<T*>(p.out) + (long long)t * p.o_tok + (long long)hd * p.o_head + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = l > 0.f ? (m + log2f(l)) * LN2 : l == l ? neg_inf() : l;
}

}  // namespace ppre
}  // namespace w4a4
