// Norms of queries and keys, position rotation and cache write, one launch behind the qkv linear.
//
//   x = head row of qkv;  n = x * w / sqrt(mean(x^2) + eps)  (queries and keys, each where a weight is given);
//   (a, b) -> (a c - b s, b c + a s)  for the pairs of the first `rot` elements, c and s of the token's position:
//   neighbours (interleaved) or i and i + rot / 2.  Values go to the cache as they are.
//
// Everything between the load and the one rounding of the result is fp32.  The sum of squares is over at most 128
// elements: 8 per lane in order, then a butterfly over the row's lanes.
//
// What bounds it: memory traffic for prompts, the chain offsets -> length -> page number and angles -> store for
// decode steps.  Eight lanes (dim 64) or sixteen (128) take a head row with one 16-byte load each; the loads of the
// first rows are issued before the chain is walked, whose first step is one round of loads for up to 32 sequences
// (each lane compares one offset).
#pragma once

#include "paged_kv.cuh"

namespace w4a4 {
namespace kv {

constexpr int ROPE_THREADS = 256;

struct RopeParams {
  Cache c;
  Seqs s;
  const void* qkv;
  long long ld_qkv;
  void* q_out;
  long long q_tok, q_head;
  const float* cos;
  const float* sin;
  const void* q_norm;
  const void* k_norm;
  const int32_t* offsets;     // per sequence: position minus slot, or NULL
  int n_heads, rot, max_pos, interleaved;
  int toks;                   // tokens of a block: 1, 2 or 4
  float eps;
};

// How a lane's eight elements lie in the row and where the partner of each is.  In the two usual layouts pairs do not leave
// the lane: PAIRS takes eight neighbours, HALVES four of either half of the row.  APART (halves of a part of the row)
// takes eight neighbours and gets their partners from another lane.  Measured, 16384 tokens of 80 heads with norms,
// halves: 172 us with partners from other lanes (eight exchanges per 16 bytes) and IEEE square root and division.
enum : int { ROPE_PAIRS, ROPE_HALVES, ROPE_APART };

// A block takes `toks` tokens, and each of them ROPE_THREADS / LANES / toks groups of LANES lanes that go through its
// rows in turn with the token's cosines and sines in registers.
template <typename T, int DIM, int MODE>
__global__ void __launch_bounds__(ROPE_THREADS, 4) qkv_rope_kernel(const RopeParams p) {
  constexpr int LANES = DIM / 8, GROUPS = ROPE_THREADS / LANES, UNROLL = 4, ANGLES = MODE == ROPE_APART ? 8 : 4;
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31;
  const int sub = tid % LANES;               // this thread's 8 elements of a head row
  const int per_tok = GROUPS / p.toks;       // groups that share a token
  const int t = blockIdx.x * p.toks + tid / LANES / per_tok, row_first = tid / LANES % per_tok;
  if (t >= p.s.T) return;                    // (a warp's lanes share a token: a token has four groups or more)
  const int n_rows = p.n_heads + 2 * p.c.n_kv;
  const T* src = static_cast<const T*>(p.qkv) + (long long)t * p.ld_qkv;
  auto get = [&](const T* row) -> uint4 {
    if (MODE == ROPE_HALVES) {
      const uint2 a = ld_plain(reinterpret_cast<const uint2*>(row + sub * 4)), b = ld_plain(reinterpret_cast<const uint2*>(row + DIM / 2 + sub * 4));
      return make_uint4(a.x, a.y, b.x, b.y);
    }
    return ld_plain(reinterpret_cast<const uint4*>(row + sub * 8));
  };
  auto put = [&](T* row, const uint4& v) {
    if (MODE == ROPE_HALVES) {
      *reinterpret_cast<uint2*>(row + sub * 4) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(row + DIM / 2 + sub * 4) = make_uint2(v.z, v.w);
    } else {
      *reinterpret_cast<uint4*>(row + sub * 8) = v;
    }
  };
  auto floats = [&](const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 e = unpack2<T>(w[i]);
      f[2 * i] = e.x;
      f[2 * i + 1] = e.y;
    }
  };
  grid_dependency_wait();

  uint4 x[UNROLL];
  auto load = [&](int row0) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int r = row0 + u * per_tok + row_first;
      if (r < n_rows) x[u] = get(src + (long long)r * DIM);
    }
  };
  load(0);

  // the token's sequence: how many of the n + 1 offsets are not above t, less one
  int below = 0;
  for (int i = lane; i <= p.s.n; i += 32) below += ld_plain(p.s.cu + i) <= t;
  const int b = __reduce_add_sync(0xffffffffu, below) - 1;
  if (b < 0 || b >= p.s.n) return;           // behind the last sequence: left as it is
  int length;
  const Seq q = load_seq(p.s, b, length);
  // from the length as it was given: a token of a sequence that has outgrown its table must not take an earlier one's slot
  const long long at = (long long)length - q.q_len + (t - q.q0);
  const int slot = at >= 0 && at < p.s.max_slots ? (int)at : -1;
  const int pos = slot + (p.offsets ? ld_plain(p.offsets + b) : 0);
  if (slot < 0 || (p.rot > 0 && (unsigned)pos >= (unsigned)p.max_pos) || t < q.q0 || t >= q.q0 + q.q_len) {
    if (lane == 0) record_error(SITE_KV_POS, b);
    return;
  }
  const int page = page_of(p.c, b, slot / p.c.page), in_page = slot % p.c.page;

  // cosines and sines of this thread's pairs
  const int half = p.rot / 2;
  const bool rotated = MODE == ROPE_HALVES || sub * 8 < p.rot;
  const int partner = sub * 8 < half ? half / 8 : -(half / 8);
  const int angle0 = MODE != ROPE_APART ? sub * 4 : (sub * 8 < half ? sub * 8 : sub * 8 - half);
  float cs[ANGLES] = {}, sn[ANGLES] = {};
  if (rotated) {
#pragma unroll
    for (int i = 0; i < ANGLES; i += 4) {
      const float4 c4 = ld_plain(reinterpret_cast<const float4*>(p.cos + (long long)pos * half + angle0 + i));
      const float4 s4 = ld_plain(reinterpret_cast<const float4*>(p.sin + (long long)pos * half + angle0 + i));
      cs[i] = c4.x; cs[i + 1] = c4.y; cs[i + 2] = c4.z; cs[i + 3] = c4.w;
      sn[i] = s4.x; sn[i + 1] = s4.y; sn[i + 2] = s4.z; sn[i + 3] = s4.w;
    }
  }

  for (int row0 = 0; row0 < n_rows; row0 += UNROLL * per_tok) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int r = row0 + u * per_tok + row_first;
      const bool live = r < n_rows, is_v = r >= p.n_heads + p.c.n_kv, is_q = r < p.n_heads;
      uint4 y = live ? x[u] : make_uint4(0, 0, 0, 0);
      if (__any_sync(0xffffffffu, live && !is_v)) {
        float f[8];
        floats(y, f);
        const T* nw = static_cast<const T*>(is_q ? p.q_norm : p.k_norm);
        if (p.q_norm != nullptr || p.k_norm != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += f[i] * f[i];
#pragma unroll
          for (int o = LANES / 2; o > 0; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (nw != nullptr) {
            const float r_rms = rsqrtf(ss * (1.f / DIM) + p.eps);      // (two steps of fp32 off at most)
            float w[8];
            floats(get(nw), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] *= r_rms * w[i];
          }
        }
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (MODE == ROPE_PAIRS) {
            g[i] = i & 1 ? f[i] * cs[i / 2] + f[i - 1] * sn[i / 2] : f[i] * cs[i / 2] - f[i + 1] * sn[i / 2];
          } else if (MODE == ROPE_HALVES) {
            g[i] = i >= 4 ? f[i] * cs[i - 4] + f[i - 4] * sn[i - 4] : f[i] * cs[i] - f[i + 4] * sn[i];
          } else {
            const float o = __shfl_sync(0xffffffffu, f[i], (lane & ~(LANES - 1)) | ((sub + partner) & (LANES - 1)));
            g[i] = f[i] * cs[i % ANGLES] + (partner > 0 ? -o : o) * sn[i % ANGLES];
          }
        }
        if (!is_v) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = rotated ? g[i] : f[i];
          y = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
        }
      }
      if (live) {
        if (is_q) {
          put(static_cast<T*>(p.q_out) + (long long)t * p.q_tok + (long long)r * p.q_head, y);
        } else if (page >= 0) {
          const int h = is_v ? r - p.n_heads - p.c.n_kv : r - p.n_heads;
          put(is_v ? static_cast<T*>(p.c.v) + page * p.c.v_page + h * p.c.v_head + in_page * p.c.v_slot
                   : static_cast<T*>(p.c.k) + page * p.c.k_page + h * p.c.k_head + in_page * p.c.k_slot, y);
        }
      }
    }
    load(row0 + UNROLL * per_tok);
  }
}

}  // namespace kv
}  // namespace w4a4
