// dpt_attn_impl.h - the attention kernels, instantiated per element type (dpt_attn_f32.hip, dpt_attn_bf16.hip).
#pragma once
#include "dpt_attn.h"

namespace dptat {

// what a workgroup works on
struct Place {
  int b, hk, q0, nq, k0, nk, rows;
  int64_t pair0;
};

// workgroup -> (block of rows or keys, complex, key head): key heads innermost, so that with 8 of them (or a multiple) a head stays on one XCD and
// its keys in that XCD's L2; the complexes in the caller's order, largest first
__device__ __forceinline__ Place place(const Dev& d, int id, int* tile) {
  Place p;
  p.hk = id % d.a.kv_heads;
  id /= d.a.kv_heads;
  p.b = d.a.order[id % d.a.B];
  *tile = id / d.a.B;
  p.q0 = d.a.q_ptr[p.b];
  p.nq = d.a.q_ptr[p.b + 1] - p.q0;
  p.k0 = d.a.k_ptr[p.b];
  p.nk = d.a.k_ptr[p.b + 1] - p.k0;
  p.pair0 = d.a.pair_ptr[p.b];
  p.rows = p.nq * d.group;
  return p;
}

__device__ __forceinline__ int clampi(int x, int hi) { return x < 0 ? 0 : x < hi ? x : hi; }
// keys that query i of the complex sees
__device__ __forceinline__ int keys_seen(const Dev& d, const Place& p, int i) { return d.a.causal ? clampi(i + 1 + p.nk - p.nq, p.nk) : p.nk; }

// a lane's row: its query and head, and where it lies
struct Row { int i, head; int64_t token; };
__device__ __forceinline__ Row row_at(const Dev& d, const Place& p, int r) {
  Row x;
  x.i = div_group(d, r);
  x.head = p.hk * d.group + (r - x.i * d.group);
  x.token = p.q0 + x.i;
  return x;
}

// scores of 32 keys x the lane's row: scaled, biased, masked.  key0: the tile's first key; lim: keys that the row sees
template <typename T, bool BIAS>
__device__ __forceinline__ void finish_scores(const Dev& d, f16v& s, int key0, int h, int lim, bool part, const T* __restrict__ bias) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int key = key0 + 8 * (e >> 2) + 4 * h + (e & 3);
    float x = s[e] * d.a.scale;
    if constexpr (BIAS) {
      const float bv = key < lim ? (float)bias[key * d.a.bias_pair] : NEG_INF;
      x = bv == NEG_INF ? NEG_INF : x + bv;
    } else {
      if (part) x = key < lim ? x : NEG_INF;
    }
    s[e] = x;
  }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------------------
// NW waves x 32 rows; keys in tiles of BN.  Running maximum and sum per row, one pass over the keys.
template <typename T, int DP, int NW, int BN, bool BIAS>
__global__ __launch_bounds__(64 * NW) void fwd_kernel(Dev d) {
  __shared__ __attribute__((aligned(16))) T kt[BN * DP], vt[BN * DP];
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5, wave = threadIdx.x / 64;
  int id = blockIdx.x, tile;
  const int split = id % d.splits;
  const Place p = place(d, id / d.splits, &tile);
  constexpr int BM = 32 * NW;
  const int tiles = (p.rows + BM - 1) / BM;
  if (tile >= tiles) return;
  if (d.a.causal) tile = tiles - 1 - tile;                   // the longest rows first
  const int r0 = tile * BM, r = r0 + wave * 32 + l31;
  const Row row = row_at(d, p, r < p.rows ? r : p.rows - 1);
  const int lim = keys_seen(d, p, row.i);
  const int lim_lo = keys_seen(d, p, div_group(d, min(r0 + wave * 32, p.rows - 1)));
  const int lim_hi = keys_seen(d, p, div_group(d, min(r0 + wave * 32 + 31, p.rows - 1)));
  const int last = keys_seen(d, p, div_group(d, min(r0 + BM, p.rows) - 1));
  const int ktiles = (last + BN - 1) / BN, per = (ktiles + d.splits - 1) / d.splits;
  const int t0 = split * per, t1 = min(t0 + per, ktiles);

  typename Tr<T>::frag qf[NC<T, DP> / 2];
  {
    const T* q = (const T*)d.a.q + row.token * d.a.q_row + row.head * d.a.q_head;
#pragma unroll
    for (int s = 0; s < NC<T, DP> / 2; ++s) qf[s] = load_chunk<T>(q, 2 * s + h, d.a.dim, d.vec);
  }
  const T* bias = BIAS ? (const T*)d.a.bias + row.head * d.a.bias_head + (p.pair0 + (int64_t)row.i * p.nk) * d.a.bias_pair : nullptr;
  const T* kb = (const T*)d.a.k + (int64_t)p.k0 * d.a.k_row + p.hk * d.a.k_head;
  const T* vb = (const T*)d.a.v + (int64_t)p.k0 * d.a.v_row + p.hk * d.a.v_head;

  f16v o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m = NEG_INF, l = 0.f;
  for (int t = t0; t < t1; ++t) {
    const int key0 = t * BN;
    __syncthreads();
    stage_keys<T, DP, BN, 64 * NW>(kt, kb, d.a.k_row, key0, p.nk, d.a.dim, d.vec);
    stage_keys<T, DP, BN, 64 * NW>(vt, vb, d.a.v_row, key0, p.nk, d.a.dim, d.vec);
    __syncthreads();
    if (key0 >= lim_hi) continue;                            // (wave-uniform; the barriers above are still met by every wave)
    f16v s[BN / 32];
    float top = m;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = 0.f;
      s[j] = rows_times<T, DP>(kt, 32 * j, l31, h, qf, s[j]);
      finish_scores<T, BIAS>(d, s[j], key0 + 32 * j, h, lim, key0 + BN > lim_lo, bias);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[j][e]);
    }
    top = half_max(top);
    const float base = top == NEG_INF ? 0.f : top;           // nothing seen yet: exp of -inf - 0
    const float alpha = __builtin_amdgcn_exp2f((m - base) * LOG2E);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[j][e] = __builtin_amdgcn_exp2f((s[j][e] - base) * LOG2E);
        sum += s[j][e];
      }
    l = l * alpha + half_sum(sum);
    m = top;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j) cols_times<DP>(vt, 32 * j, lane, (const float*)&s[j], o);
  }
  if (r >= p.rows) return;
  const int64_t at = row.token * d.a.heads + row.head, st = (int64_t)row.head * d.a.n_q + row.token, plane = (int64_t)d.a.heads * d.a.n_q;
  if (d.splits == 1) {
    store_col<T, DP>((T*)d.a.out + at * d.a.dim, h, d.a.dim, d.vec, o, l == 0.f ? 0.f : 1.f / l);
    if (h == 0) { d.a.stats[st] = m; d.a.stats[plane + st] = l; }
  } else {
    store_col<float, DP>(d.part_o + (split * plane + at) * d.a.dim, h, d.a.dim, d.a.dim % 4 == 0, o, 1.f);
    if (h == 0) { d.part_ml[2 * split * plane + st] = m; d.part_ml[(2 * split + 1) * plane + st] = l; }
  }
}

// joins the key ranges of a row: one wave per (row, head), in the ranges' order
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Dev d) {
  const int64_t plane = (int64_t)d.a.heads * d.a.n_q, at = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (at >= plane) return;
  const int lane = threadIdx.x & 63, head = (int)(at % d.a.heads);
  const int64_t st = (int64_t)head * d.a.n_q + at / d.a.heads;
  float m = NEG_INF, l = 0.f;
  for (int s = 0; s < d.splits; ++s) m = fmaxf(m, d.part_ml[2 * s * plane + st]);
  const float base = m == NEG_INF ? 0.f : m;
  float acc[2] = {0.f, 0.f};
  for (int s = 0; s < d.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f((d.part_ml[2 * s * plane + st] - base) * LOG2E);
    l += f * d.part_ml[(2 * s + 1) * plane + st];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (lane + 64 * j < d.a.dim) acc[j] += f * d.part_o[(s * plane + at) * d.a.dim + lane + 64 * j];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (lane + 64 * j < d.a.dim) ((T*)d.a.out)[at * d.a.dim + lane + 64 * j] = (T)(acc[j] * inv);
  if (lane == 0) { d.a.stats[st] = m; d.a.stats[plane + st] = l; }
}

// ---- backward: gradients of the queries and of the bias -------------------------------------------------------------------------------------------
// As the forward pass, with the probabilities formed again from the stored statistics: ds = p (do.v - delta), dq += ds k.
// Also writes delta = sum_d do o for the second kernel.
template <typename T, int DP, int NW, int BN, bool BIAS>
__global__ __launch_bounds__(64 * NW) void dq_kernel(Dev d) {
  __shared__ __attribute__((aligned(16))) T kt[BN * DP], vt[BN * DP];
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5, wave = threadIdx.x / 64;
  int tile;
  const Place p = place(d, blockIdx.x, &tile);
  constexpr int BM = 32 * NW;
  const int tiles = (p.rows + BM - 1) / BM;
  if (tile >= tiles) return;
  if (d.a.causal) tile = tiles - 1 - tile;
  const int r0 = tile * BM, r = r0 + wave * 32 + l31;
  const bool live = r < p.rows;
  const Row row = row_at(d, p, live ? r : p.rows - 1);
  const int lim = keys_seen(d, p, row.i);
  const int lim_lo = keys_seen(d, p, div_group(d, min(r0 + wave * 32, p.rows - 1)));
  const int lim_hi = keys_seen(d, p, div_group(d, min(r0 + wave * 32 + 31, p.rows - 1)));
  const int last = keys_seen(d, p, div_group(d, min(r0 + BM, p.rows) - 1));
  // a bias gradient is written for every pair, 0 for those behind the causal edge
  const int end = BIAS && d.a.dbias ? p.nk : last;

  const int64_t at = row.token * d.a.heads + row.head, st = (int64_t)row.head * d.a.n_q + row.token, plane = (int64_t)d.a.heads * d.a.n_q;
  typename Tr<T>::frag qf[NC<T, DP> / 2], gf[NC<T, DP> / 2];
  float delta = 0.f;
  {
    const T* q = (const T*)d.a.q + row.token * d.a.q_row + row.head * d.a.q_head;
    const T* g = (const T*)d.a.dout + row.token * d.a.dout_row + row.head * d.a.dout_head;
    const T* o = (const T*)d.a.out + at * d.a.dim;
#pragma unroll
    for (int s = 0; s < NC<T, DP> / 2; ++s) {
      qf[s] = load_chunk<T>(q, 2 * s + h, d.a.dim, d.vec);
      gf[s] = load_chunk<T>(g, 2 * s + h, d.a.dim, d.vec);
      const typename Tr<T>::frag of = load_chunk<T>(o, 2 * s + h, d.a.dim, d.vec);
#pragma unroll
      for (int e = 0; e < Tr<T>::CH; ++e) delta = fmaf((float)gf[s][e], (float)of[e], delta);
    }
    delta = half_sum(delta);
    if (live && h == 0) d.delta[st] = delta;
  }
  const float m = d.a.stats[st], l = d.a.stats[plane + st];
  const float base = m == NEG_INF ? 0.f : m, inv = l == 0.f ? 0.f : 1.f / l;
  const T* bias = BIAS ? (const T*)d.a.bias + row.head * d.a.bias_head + (p.pair0 + (int64_t)row.i * p.nk) * d.a.bias_pair : nullptr;
  T* dbias = BIAS && d.a.dbias ? (T*)d.a.dbias + row.head * d.a.n_pairs + p.pair0 + (int64_t)row.i * p.nk : nullptr;
  const T* kb = (const T*)d.a.k + (int64_t)p.k0 * d.a.k_row + p.hk * d.a.k_head;
  const T* vb = (const T*)d.a.v + (int64_t)p.k0 * d.a.v_row + p.hk * d.a.v_head;

  f16v dq[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[i][e] = 0.f;
  for (int key0 = 0; key0 < end; key0 += BN) {
    __syncthreads();
    stage_keys<T, DP, BN, 64 * NW>(kt, kb, d.a.k_row, key0, p.nk, d.a.dim, d.vec);
    stage_keys<T, DP, BN, 64 * NW>(vt, vb, d.a.v_row, key0, p.nk, d.a.dim, d.vec);
    __syncthreads();
    if (key0 >= lim_hi && !dbias) continue;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j) {
      f16v s, g;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = g[e] = 0.f;
      s = rows_times<T, DP>(kt, 32 * j, l31, h, qf, s);
      g = rows_times<T, DP>(vt, 32 * j, l31, h, gf, g);
      finish_scores<T, BIAS>(d, s, key0 + 32 * j, h, lim, key0 + BN > lim_lo, bias);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_amdgcn_exp2f((s[e] - base) * LOG2E) * inv;
        s[e] = s[e] == NEG_INF ? 0.f : x * (g[e] - delta);
      }
      if constexpr (BIAS) {
        if (dbias && live) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = key0 + 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
            if (key < p.nk) dbias[key] = (T)s[e];
          }
        }
      }
      cols_times<DP>(kt, 32 * j, lane, (const float*)&s, dq);
    }
  }
  if (live) store_col<T, DP>((T*)d.a.dq + at * d.a.dim, h, d.a.dim, d.vec, dq, d.a.scale);
}

// ---- backward: gradients of the keys and values ---------------------------------------------------------------------------------------------------
// NW waves x 32 keys; the rows of all heads of the group in tiles of BR.  Rows down, keys across: the probability and ds tiles are second operands as
// they stand, dv[d, key] += do[row, d] p[row, key], dk[d, key] += q[row, d] ds[row, key].
template <typename T, int DP, int NW, int BR, bool BIAS>
__global__ __launch_bounds__(64 * NW) void dkv_kernel(Dev d) {
  __shared__ __attribute__((aligned(16))) T qt[BR * DP], gt[BR * DP];
  __shared__ __attribute__((aligned(16))) float sm[BR], sl[BR], sd[BR];
  __shared__ __attribute__((aligned(16))) int slim[BR];
  __shared__ int64_t sb[BIAS ? BR : 1];
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5, wave = threadIdx.x / 64;
  int tile;
  const Place p = place(d, blockIdx.x, &tile);
  constexpr int BM = 32 * NW;
  if (tile * BM >= p.nk) return;
  const int key0 = tile * BM, key = key0 + wave * 32 + l31;
  const bool live = key < p.nk;
  const int64_t token = p.k0 + (live ? key : p.nk - 1), plane = (int64_t)d.a.heads * d.a.n_q;
  typename Tr<T>::frag kf[NC<T, DP> / 2], vf[NC<T, DP> / 2];
#pragma unroll
  for (int s = 0; s < NC<T, DP> / 2; ++s) {
    kf[s] = load_chunk<T>((const T*)d.a.k + token * d.a.k_row + p.hk * d.a.k_head, 2 * s + h, d.a.dim, d.vec);
    vf[s] = load_chunk<T>((const T*)d.a.v + token * d.a.v_row + p.hk * d.a.v_head, 2 * s + h, d.a.dim, d.vec);
  }
  f16v dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[i][e] = dv[i][e] = 0.f;
  // the first query that sees this block's first key
  const int first = d.a.causal ? clampi(key0 + p.nq - p.nk, p.nq) * d.group / BR * BR : 0;
  for (int r0 = first; r0 < p.rows; r0 += BR) {
    __syncthreads();
    for (int i = threadIdx.x; i < BR * NC<T, DP>; i += 64 * NW) {
      constexpr int N = NC<T, DP>;
      const int rr = i / N, c = i % N;
      const Row row = row_at(d, p, min(r0 + rr, p.rows - 1));
      const int to = (rr * N + (c ^ sw<N>(rr))) * Tr<T>::CH;
      *reinterpret_cast<typename Tr<T>::frag*>(qt + to) = load_chunk<T>((const T*)d.a.q + row.token * d.a.q_row + row.head * d.a.q_head, c, d.a.dim, d.vec);
      *reinterpret_cast<typename Tr<T>::frag*>(gt + to) =
          load_chunk<T>((const T*)d.a.dout + row.token * d.a.dout_row + row.head * d.a.dout_head, c, d.a.dim, d.vec);
    }
    for (int i = threadIdx.x; i < BR; i += 64 * NW) {
      const Row row = row_at(d, p, min(r0 + i, p.rows - 1));
      const int64_t st = (int64_t)row.head * d.a.n_q + row.token;
      const float m = d.a.stats[st], l = d.a.stats[plane + st];
      sm[i] = m == NEG_INF ? 0.f : m;
      sl[i] = l == 0.f ? 0.f : 1.f / l;
      sd[i] = d.delta[st];
      slim[i] = r0 + i < p.rows ? keys_seen(d, p, row.i) : 0;
      if constexpr (BIAS) sb[i] = row.head * d.a.bias_head + (p.pair0 + (int64_t)row.i * p.nk) * d.a.bias_pair;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < BR / 32; ++j) {
      f16v s, g;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = g[e] = 0.f;
      s = rows_times<T, DP>(qt, 32 * j, l31, h, kf, s);
      g = rows_times<T, DP>(gt, 32 * j, l31, h, vf, g);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int rr = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
        const bool seen = live && key < slim[rr];
        float x = s[e] * d.a.scale;
        if constexpr (BIAS) {
          const float bv = seen ? (float)((const T*)d.a.bias)[sb[rr] + key * d.a.bias_pair] : NEG_INF;
          x = bv == NEG_INF ? NEG_INF : x + bv;
        } else {
          x = seen ? x : NEG_INF;
        }
        const float pr = __builtin_amdgcn_exp2f((x - sm[rr]) * LOG2E) * sl[rr];
        s[e] = x == NEG_INF ? 0.f : pr;
        g[e] = x == NEG_INF ? 0.f : pr * (g[e] - sd[rr]);
      }
      cols_times<DP>(gt, 32 * j, lane, (const float*)&s, dv);
      cols_times<DP>(qt, 32 * j, lane, (const float*)&g, dk);
    }
  }
  if (live) {
    const int64_t at = (token * d.a.kv_heads + p.hk) * d.a.dim;
    store_col<T, DP>((T*)d.a.dk + at, h, d.a.dim, d.vec, dk, d.a.scale);
    store_col<T, DP>((T*)d.a.dv + at, h, d.a.dim, d.vec, dv, 1.f);
  }
}

template <typename T, int DP>
hipError_t run_fwd(const Dev& d, bool small, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  const unsigned n = (unsigned)((int64_t)d.tiles * d.a.B * d.a.kv_heads * d.splits);
  if (n) {
    if (d.a.bias) {
      if (small) hipLaunchKernelGGL((fwd_kernel<T, DP, 1, BN, true>), dim3(n), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((fwd_kernel<T, DP, 4, BN, true>), dim3(n), dim3(256), 0, st, d);
    } else {
      if (small) hipLaunchKernelGGL((fwd_kernel<T, DP, 1, BN, false>), dim3(n), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((fwd_kernel<T, DP, 4, BN, false>), dim3(n), dim3(256), 0, st, d);
    }
    if (d.splits > 1)
      hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(((int64_t)d.a.heads * d.a.n_q + 3) / 4)), dim3(256), 0, st, d);
  }
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t run_bwd(const Dev& d0, bool small_rows, bool small_keys, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32, BR = 32;
  Dev d = d0;
  const int64_t rows = (int64_t)d.a.max_nq * d.group;
  d.tiles = (int)((rows + (small_rows ? 31 : 127)) / (small_rows ? 32 : 128));
  const unsigned n = (unsigned)((int64_t)d.tiles * d.a.B * d.a.kv_heads);
  if (n) {
    if (d.a.bias) {
      if (small_rows) hipLaunchKernelGGL((dq_kernel<T, DP, 1, BN, true>), dim3(n), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((dq_kernel<T, DP, 4, BN, true>), dim3(n), dim3(256), 0, st, d);
    } else {
      if (small_rows) hipLaunchKernelGGL((dq_kernel<T, DP, 1, BN, false>), dim3(n), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((dq_kernel<T, DP, 4, BN, false>), dim3(n), dim3(256), 0, st, d);
    }
  }
  d.tiles = (d.a.max_nk + (small_keys ? 31 : 127)) / (small_keys ? 32 : 128);
  const unsigned nk = (unsigned)((int64_t)d.tiles * d.a.B * d.a.kv_heads);
  if (nk) {
    if (d.a.bias) {
      if (small_keys) hipLaunchKernelGGL((dkv_kernel<T, DP, 1, BR, true>), dim3(nk), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((dkv_kernel<T, DP, 4, BR, true>), dim3(nk), dim3(256), 0, st, d);
    } else {
      if (small_keys) hipLaunchKernelGGL((dkv_kernel<T, DP, 1, BR, false>), dim3(nk), dim3(64), 0, st, d);
      else hipLaunchKernelGGL((dkv_kernel<T, DP, 4, BR, false>), dim3(nk), dim3(256), 0, st, d);
    }
  }
  return hipGetLastError();
}

template <typename T>
hipError_t fwd_by_dim(const Dev& d, bool small, hipStream_t st) {
  return d.a.dim <= 32 ? run_fwd<T, 32>(d, small, st) : d.a.dim <= 64 ? run_fwd<T, 64>(d, small, st) : run_fwd<T, 128>(d, small, st);
}
template <typename T>
hipError_t bwd_by_dim(const Dev& d, bool sr, bool sk, hipStream_t st) {
  return d.a.dim <= 32 ? run_bwd<T, 32>(d, sr, sk, st) : d.a.dim <= 64 ? run_bwd<T, 64>(d, sr, sk, st) : run_bwd<T, 128>(d, sr, sk, st);
}

}  // namespace dptat
