// dpt_attn_impl.h - the attention kernels, instantiated per element type and padded head dimension (dpt_attn_<type>_<dim>.hip).
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
__device__ __forceinline__ int keys_seen(const Dev& d, const Place& p, int i) { return d.a.causal ? clampi(i + 1 - p.nq + p.nk, p.nk) : p.nk; }

// a lane's row: its query and head, and where it lies
struct Row { int i, head; int64_t token; };
__device__ __forceinline__ Row row_at(const Dev& d, const Place& p, int r) {
  Row x;
  x.i = div_group(d, r);
  x.head = p.hk * d.group + (r - x.i * d.group);
  x.token = p.q0 + x.i;
  return x;
}

// From a product q.k to exp(s - m).  FAST (bf16 without a bias): scores stay unscaled, exp2(fma(x, scale log2 e, -m scale log2 e)) - one operation and the
// exponential, an error of a few 2^-24 |m|, far below the rounding of a bf16 probability.  Otherwise exp2((s - m) log2 e) with the difference first:
// a row of the type's lowest values is then a row of exact zeros under the exponential, and fp32 keeps its last bits.
template <typename T, bool BIAS> constexpr bool FAST = sizeof(T) == 2 && !BIAS;

// scores of 32 keys x the lane's row: scaled and biased unless FAST, masked.  key0: the tile's first key; lim: keys that the row sees; part: some
// row of the wave sees only a part of the tile
template <typename T, bool BIAS>
__device__ __forceinline__ void finish_scores(const Dev& d, f16v& s, int key0, int h, int lim, bool part, const T* __restrict__ bias) {
  if constexpr (BIAS) {
    const bool unit = d.a.bias_pair == 1;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int key = key0 + 8 * g + 4 * h;
      float bv[4];
      if (unit && key + 4 <= lim) {
        const Four<T> f = *reinterpret_cast<const Four<T>*>(bias + key);
#pragma unroll
        for (int i = 0; i < 4; ++i) bv[i] = (float)f.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) bv[i] = key + i < lim ? (float)bias[(key + i) * d.a.bias_pair] : NEG_INF;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * g + i] = bv[i] == NEG_INF ? NEG_INF : s[4 * g + i] * d.a.scale + bv[i];
    }
  } else if constexpr (!FAST<T, BIAS>) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] *= d.a.scale;
  }
  if constexpr (!BIAS) {
    if (part) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = key0 + 8 * (e >> 2) + 4 * h + (e & 3) < lim ? s[e] : NEG_INF;
    }
  }
}

// a row block's view of its keys, common to the forward and the dq kernel
template <int BM>
struct RowBlock {
  Row row;
  bool live;
  int lim, lim_lo, lim_hi, last;   // keys that the lane's row, the wave's first and last row, the block's last row see
  __device__ __forceinline__ RowBlock(const Dev& d, const Place& p, int tile, int lane) {
    const int w0 = tile * BM + (threadIdx.x & ~63) / 2, r = w0 + (lane & 31), end = p.rows - 1;
    live = r <= end;
    row = row_at(d, p, min(r, end));
    lim = keys_seen(d, p, row.i);
    lim_lo = __builtin_amdgcn_readfirstlane(keys_seen(d, p, div_group(d, min(w0, end))));
    lim_hi = __builtin_amdgcn_readfirstlane(keys_seen(d, p, div_group(d, min(w0 + 31, end))));
    last = keys_seen(d, p, div_group(d, min(tile * BM + BM - 1, end)));
  }
};

template <int N>
__device__ __forceinline__ void zero(f16v* x) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) x[i][e] = 0.f;
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------------------
// NW waves x 32 rows; keys in tiles of BN, the next tile on its way into the other LDS buffer while one is worked on.  One pass over the keys with a
// running base and sum per row.  The base follows the row's maximum only when that has moved by more than 2^8 (exp of the difference then still has all its
// bits, and so has a bf16 of it), so the accumulators are rescaled a few times per row instead of once per tile.
// Long rows are bound by the matrix units and the exponentials in equal parts (2 x 4096 causal, 16 heads of 128, bf16: 152 us, 903 TFLOP/s; with one wave per SIMD
// 253 us), single queries by HBM (24 of them against up to 16384 keys: 179 us, 5.1 TB/s), small complexes by latency (40 x (20 x 79) fp32: 11 us).
template <typename T, int DP, int NW, int BN, bool BIAS, bool VEC>
__global__ __launch_bounds__(64 * NW, (FAST<T, BIAS> ? 2 : 1)) void fwd_kernel(Dev d) {
  __shared__ __attribute__((aligned(16))) T kt0[BN * DP], vt0[BN * DP], kt1[BN * DP], vt1[BN * DP];
  constexpr int NT = 64 * NW, BM = 32 * NW, J = BN / 32;
  constexpr float FAR = 8.f;
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  int id = d.first + blockIdx.x, tile;
  const int split = id % d.splits;
  const Place p = place(d, id / d.splits, &tile);
  const int tiles = (p.rows + BM - 1) / BM;
  if (tile >= tiles) return;
  if (d.a.causal) tile = tiles - 1 - tile;                   // the longest rows first
  const RowBlock<BM> rb(d, p, tile, lane);
  const Row row = rb.row;
  const int ktiles = (rb.last + BN - 1) / BN, per = (ktiles + d.splits - 1) / d.splits;
  const int t0 = split * per, t1 = min(t0 + per, ktiles);

  const T* kb = (const T*)d.a.k + (int64_t)p.k0 * d.a.k_row + p.hk * d.a.k_head;
  const T* vb = (const T*)d.a.v + (int64_t)p.k0 * d.a.v_row + p.hk * d.a.v_head;
  // keys behind the last one repeat it: their scores are masked, and it brings in no value that the result does not hold anyway
  auto fetch = [&](T* kt, T* vt, int t) __attribute__((always_inline)) {
    stage<T, DP, BN, NT, VEC>(kt, d.a.dim, kb + (int64_t)t * BN * d.a.k_row, d.a.k_row, p.nk - t * BN);
    stage<T, DP, BN, NT, VEC>(vt, d.a.dim, vb + (int64_t)t * BN * d.a.v_row, d.a.v_row, p.nk - t * BN);
  };
  if (t0 < t1) fetch(kt0, vt0, t0);
  zero_pad<T, DP, BN, NT, VEC>(kt0, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(vt0, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(kt1, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(vt1, d.a.dim);
  typename Tr<T>::frag qf[NC<T, DP> / 2];
  {
    const T* q = (const T*)d.a.q + row.token * d.a.q_row + row.head * d.a.q_head;
#pragma unroll
    for (int s = 0; s < NC<T, DP> / 2; ++s) qf[s] = load_chunk<T, VEC>(q, 2 * s + h, d.a.dim);
  }
  const T* bias = BIAS ? (const T*)d.a.bias + row.head * d.a.bias_head + (p.pair0 + (int64_t)row.i * p.nk) * d.a.bias_pair : nullptr;
  const float c = FAST<T, BIAS> ? d.a.scale * LOG2E : LOG2E;   // exp(s - base) = exp2((x - base) c)

  f16v o[DP / 32];
  zero<DP / 32>(o);
  float m = NEG_INF, base = NEG_INF, l = 0.f;                // of the scores as they are held; l: this half's share of the sum
  auto work = [&](const T* kt, const T* vt, int t) __attribute__((always_inline)) {
    const int key0 = t * BN;
    if (key0 >= rb.lim_hi) return;
    f16v s[J];
    zero<J>(s);
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = rows_times<T, DP>(kt, 32 * j, l31, h, qf, s[j]);
    float top = m;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      finish_scores<T, BIAS>(d, s[j], key0 + 32 * j, h, rb.lim, key0 + BN > rb.lim_lo, bias);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[j][e]);
    }
    m = half_max(top);
    if (__any((m - base) * c > FAR)) {                       // (base -inf: the first keys that the row sees)
      const float nb = fmaxf(base, m), alpha = __builtin_amdgcn_exp2f((base - (nb == NEG_INF ? 0.f : nb)) * c);
      base = nb;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
    }
    const float b0 = base == NEG_INF ? 0.f : base, nbc = -b0 * c;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[j][e] = __builtin_amdgcn_exp2f(FAST<T, BIAS> ? fmaf(s[j][e], c, nbc) : (s[j][e] - b0) * c);
        l += s[j][e];
      }
#pragma unroll
    for (int j = 0; j < J; ++j) cols_times<DP>(vt, 32 * j, lane, (const float*)&s[j], o);
  };
  // one barrier per tile: it waits for the tile's fetch and for the last reads of the buffer that the next fetch overwrites
  for (int t = t0; t < t1; t += 2) {
    tile_barrier();
    if (t + 1 < t1) fetch(kt1, vt1, t + 1);
    work(kt0, vt0, t);
    if (t + 1 >= t1) break;
    tile_barrier();
    if (t + 2 < t1) fetch(kt0, vt0, t + 2);
    work(kt1, vt1, t + 1);
  }
  if (!rb.live) return;
  // the sum in terms of the true maximum
  l = half_sum(l);
  if (l == 0.f) zero<DP / 32>(o);                            // a row that sees nothing: 0, also beside values that are not finite (a NaN row has l = NaN)
  const float lm = m == NEG_INF ? l : l * __builtin_amdgcn_exp2f((base - m) * c), mm = FAST<T, BIAS> ? m * d.a.scale : m;
  const int64_t at = row.token * d.a.heads + row.head, st = (int64_t)row.head * d.a.n_q + row.token, plane = (int64_t)d.a.heads * d.a.n_q;
  if (d.splits == 1) {
    store_col<T, DP, VEC>((T*)d.a.out + at * d.a.dim, h, d.a.dim, o, l == 0.f ? 0.f : 1.f / l);
    if (h == 0) { d.a.stats[st] = mm; d.a.stats[plane + st] = lm; }
  } else {
    const float f = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((base - m) * c);
    store_col<float, DP, VEC>(d.part_o + (split * plane + at) * d.a.dim, h, d.a.dim, o, f);
    if (h == 0) { d.part_ml[2 * split * plane + st] = mm; d.part_ml[(2 * split + 1) * plane + st] = lm; }
  }
}

// joins the key ranges of a row: one wave per (row, head), in the ranges' order; d.first as above
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Dev d) {
  const int64_t plane = (int64_t)d.a.heads * d.a.n_q, at = ((int64_t)d.first + blockIdx.x) * 4 + threadIdx.x / 64;
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
// What the backward kernels make of a row's statistics.  FAST: p = exp2(fma(x, scale log2 e, f0)), f0 = -(m log2 e + log2 l) (-inf for a row that sees nothing);
// otherwise p = exp2((s - f0) log2 e) f1 with f0 = m, f1 = 1 / l (0 and 0).
template <typename T, bool BIAS>
struct Probs {
  float f0, f1;
  __device__ __forceinline__ Probs(float m, float l) {
    if constexpr (FAST<T, BIAS>) {
      f0 = l == 0.f ? NEG_INF : -(m * LOG2E + __builtin_amdgcn_logf(l));
      f1 = 0.f;
    } else {
      f0 = m == NEG_INF ? 0.f : m;
      f1 = l == 0.f ? 0.f : 1.f / l;
    }
  }
  __device__ __forceinline__ bool nothing() const { return FAST<T, BIAS> ? f0 == NEG_INF : f1 == 0.f; }    // the row sees no key
  static __device__ __forceinline__ float p(float x, float c, float f0, float f1) {
    return FAST<T, BIAS> ? __builtin_amdgcn_exp2f(fmaf(x, c, f0)) : __builtin_amdgcn_exp2f((x - f0) * c) * f1;
  }
};

// As the forward pass, with the probabilities formed again from the stored statistics: ds = p (do.v - delta), dq += ds k.  Writes delta = sum_d do o and the
// rows' factors for the second kernel.  Where a complex's keys are one tile, delta is taken as sum_j p_j do.v_j instead: the stored out is rounded to
// its type, and with few keys that rounding does not average out.
// Measured: 223 us for 2 x 4096 causal, 16 heads of 128, bf16 (three products: 925 TFLOP/s; at two waves per SIMD 7 registers of a lane are spilled); 31 us for 512
// complexes of 15 .. 45 x 16 .. 48 with a bias, fp32.  At a head dimension of 128 the instance for short fp32 rows without a bias spills 16 registers, and the
// one-wave instances for rows that are read element by element spill up to 300 scalar ones.
template <typename T, int DP, int NW, int BN, bool BIAS, bool VEC>
__global__ __launch_bounds__(64 * NW, (FAST<T, BIAS> ? 2 : 1)) void dq_kernel(Dev d) {
  __shared__ __attribute__((aligned(16))) T kt0[BN * DP], vt0[BN * DP], kt1[BN * DP], vt1[BN * DP];
  constexpr int NT = 64 * NW, BM = 32 * NW, J = BN / 32;
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  int id = d.first + blockIdx.x, tile;
  const int split = id % d.splits_q;
  const Place p = place(d, id / d.splits_q, &tile);
  const int tiles = (p.rows + BM - 1) / BM;
  if (tile >= tiles) return;
  if (d.a.causal) tile = tiles - 1 - tile;
  const RowBlock<BM> rb(d, p, tile, lane);
  const Row row = rb.row;
  // a bias gradient is written for every pair, 0 for those behind the causal edge
  const int ktiles = ((BIAS && d.a.dbias ? p.nk : rb.last) + BN - 1) / BN, per = (ktiles + d.splits_q - 1) / d.splits_q;
  const int t0 = split * per, t1 = min(t0 + per, ktiles);

  const T* kb = (const T*)d.a.k + (int64_t)p.k0 * d.a.k_row + p.hk * d.a.k_head;
  const T* vb = (const T*)d.a.v + (int64_t)p.k0 * d.a.v_row + p.hk * d.a.v_head;
  auto fetch = [&](T* kt, T* vt, int t) __attribute__((always_inline)) {
    stage<T, DP, BN, NT, VEC>(kt, d.a.dim, kb + (int64_t)t * BN * d.a.k_row, d.a.k_row, p.nk - t * BN);
    stage<T, DP, BN, NT, VEC>(vt, d.a.dim, vb + (int64_t)t * BN * d.a.v_row, d.a.v_row, p.nk - t * BN);
  };
  if (t0 < t1) fetch(kt0, vt0, t0);
  zero_pad<T, DP, BN, NT, VEC>(kt0, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(vt0, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(kt1, d.a.dim);
  zero_pad<T, DP, BN, NT, VEC>(vt1, d.a.dim);

  const int64_t at = row.token * d.a.heads + row.head, st = (int64_t)row.head * d.a.n_q + row.token, plane = (int64_t)d.a.heads * d.a.n_q;
  const bool one = p.nk <= BN && d.splits_q == 1;
  typename Tr<T>::frag qf[NC<T, DP> / 2], gf[NC<T, DP> / 2];
  float delta = 0.f;
  {
    const T* q = (const T*)d.a.q + row.token * d.a.q_row + row.head * d.a.q_head;
    const T* g = (const T*)d.a.dout + row.token * d.a.dout_row + row.head * d.a.dout_head;
    const T* o = (const T*)d.a.out + at * d.a.dim;
#pragma unroll
    for (int s = 0; s < NC<T, DP> / 2; ++s) {
      qf[s] = load_chunk<T, VEC>(q, 2 * s + h, d.a.dim);
      gf[s] = load_chunk<T, VEC>(g, 2 * s + h, d.a.dim);
    }
    if (!one) {
#pragma unroll
      for (int s = 0; s < NC<T, DP> / 2; ++s) {
        const typename Tr<T>::frag of = load_chunk<T, VEC>(o, 2 * s + h, d.a.dim);
#pragma unroll
        for (int e = 0; e < Tr<T>::CH; ++e) delta = fmaf((float)gf[s][e], (float)of[e], delta);
      }
      delta = half_sum(delta);
    }
  }
  const Probs<T, BIAS> f(d.a.stats[st], d.a.stats[plane + st]);
  const float c = FAST<T, BIAS> ? d.a.scale * LOG2E : LOG2E;
  const T* bias = BIAS ? (const T*)d.a.bias + row.head * d.a.bias_head + (p.pair0 + (int64_t)row.i * p.nk) * d.a.bias_pair : nullptr;
  T* dbias = BIAS && d.a.dbias ? (T*)d.a.dbias + row.head * d.a.n_pairs + p.pair0 + (int64_t)row.i * p.nk : nullptr;

  f16v dq[DP / 32];
  zero<DP / 32>(dq);
  auto work = [&](const T* kt, const T* vt, int t) __attribute__((always_inline)) {
    const int key0 = t * BN;
    if (key0 >= rb.lim_hi && !dbias) return;
    const bool part = key0 + BN > rb.lim_lo;
    // probabilities (into s) and do.v (into g) of 32 keys
    auto probs = [&](int j, f16v& s, f16v& g) __attribute__((always_inline)) {
      zero<1>(&s);
      zero<1>(&g);
      s = rows_times<T, DP>(kt, 32 * j, l31, h, qf, s);
      g = rows_times<T, DP>(vt, 32 * j, l31, h, gf, g);
      finish_scores<T, BIAS>(d, s, key0 + 32 * j, h, rb.lim, part, bias);
      if (part || BIAS) {                                    // what is masked may stand beside a do.v that is not finite
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e] = s[e] == NEG_INF ? 0.f : g[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = Probs<T, BIAS>::p(s[e], c, f.f0, f.f1);
    };
    f16v s, g;
    if (one) {
#pragma unroll 1
      for (int j = 0; j < J; ++j) {
        probs(j, s, g);
#pragma unroll
        for (int e = 0; e < 16; ++e) delta = fmaf(s[e], g[e], delta);
      }
      delta = half_sum(delta);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      probs(j, s, g);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= g[e] - delta;
      if constexpr (BIAS) {
        if (dbias && rb.live) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int key = key0 + 32 * j + 8 * q + 4 * h;
            if (key + 4 <= p.nk) {
              *reinterpret_cast<Four<T>*>(dbias + key) = Four<T>{{(T)s[4 * q], (T)s[4 * q + 1], (T)s[4 * q + 2], (T)s[4 * q + 3]}};
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key + i < p.nk) dbias[key + i] = (T)s[4 * q + i];
            }
          }
        }
      }
      cols_times<DP>(kt, 32 * j, lane, (const float*)&s, dq);
    }
  };
  for (int t = t0; t < t1; t += 2) {
    tile_barrier();
    if (t + 1 < t1) fetch(kt1, vt1, t + 1);
    work(kt0, vt0, t);
    if (t + 1 >= t1) break;
    tile_barrier();
    if (t + 2 < t1) fetch(kt0, vt0, t + 2);
    work(kt1, vt1, t + 1);
  }
  if (!rb.live) return;
  // a row that sees nothing: 0, also beside keys that are not finite (a branch around zero() costs the bf16 kernel of 64 dimensions five registers and its third
  // wave per SIMD: 55 -> 64 us for 48 ragged complexes of up to 700 x 900)
  const bool none = f.nothing();
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[i][e] = none ? 0.f : dq[i][e];
  if (d.splits_q == 1) store_col<T, DP, VEC>((T*)d.a.dq + at * d.a.dim, h, d.a.dim, dq, d.a.scale);
  else store_col<float, DP, VEC>(d.part_g + (split * plane + at) * d.a.dim, h, d.a.dim, dq, d.a.scale);
  if (h == 0 && split == 0) {
    d.delta[st] = delta;
    d.fac0[st] = f.f0;
    if (!FAST<T, BIAS>) d.fac1[st] = f.f1;
  }
}

// ---- backward: gradients of the keys and values ---------------------------------------------------------------------------------------------------
// NW waves x 32 keys; the rows of all heads of the group in tiles of BR, the next one on its way.  Rows down, keys across: the probability and ds tiles
// are second operands as they stand, dv[d, key] += do[row, d] p[row, key], dk[d, key] += q[row, d] ds[row, key].
// Measured as above: 402 us (four products: 684 TFLOP/s; at a head dimension of 128 a lane takes 392 of its 512 registers - both sums, the wave's keys and values and
// the tiles being worked on -, so one wave per SIMD) and 34 us.
template <typename T, int DP, int NW, int BR, bool BIAS>
struct RowTile {
  __attribute__((aligned(16))) T q[BR * DP], g[BR * DP];
  __attribute__((aligned(16))) float f0[BR], f1[FAST<T, BIAS> ? 4 : BR], delta[BR];
  int64_t bias[BIAS ? BR : 1];
};

template <typename T, int DP, int NW, int BR, bool BIAS, bool VEC>
__global__ __launch_bounds__(64 * NW, (FAST<T, BIAS> && DP <= 64 ? 2 : 1)) void dkv_kernel(Dev d) {
  __shared__ RowTile<T, DP, NW, BR, BIAS> rt0, rt1;
  constexpr int NT = 64 * NW, BM = 32 * NW, J = BR / 32;
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  int id = d.first + blockIdx.x, tile;
  const int split = id % d.splits_k;
  const Place p = place(d, id / d.splits_k, &tile);
  if (tile * BM >= p.nk) return;
  const int key0 = tile * BM, w0 = key0 + (threadIdx.x & ~63) / 2, key = w0 + l31;
  const bool live = key < p.nk;
  const int64_t token = p.k0 + (live ? key : p.nk - 1);
  // rows that see key j of the complex: from (j + n_queries - n_keys) group on (causal), all otherwise
  auto rows_from = [&](int j) __attribute__((always_inline)) { return d.a.causal ? clampi(j - p.nk + p.nq, p.nq) * d.group : 0; };
  const int rmin = rows_from(key), r_lo = __builtin_amdgcn_readfirstlane(rows_from(w0)), r_hi = __builtin_amdgcn_readfirstlane(rows_from(w0 + 31));
  const int begin = rows_from(key0) / BR, end = (p.rows + BR - 1) / BR, per = (end - begin + d.splits_k - 1) / d.splits_k;
  const int first = begin + split * per, last = min(first + per, end);

  const int li = div_group(d, threadIdx.x / NC<T, DP>), lg = threadIdx.x / NC<T, DP> - li * d.group;
  const uint32_t q_off = (uint32_t)li * (uint32_t)d.a.q_row + (uint32_t)lg * (uint32_t)d.a.q_head, g_off = (uint32_t)li * (uint32_t)d.a.dout_row + (uint32_t)lg * (uint32_t)d.a.dout_head;
  auto fetch = [&](RowTile<T, DP, NW, BR, BIAS>& rt, int t) __attribute__((always_inline)) {
    const int r0 = t * BR;
    auto src = [&](int r) __attribute__((always_inline)) { return row_at(d, p, min(r0 + r, p.rows - 1)); };
    // as stage(): with 1, 2, 4 .. STEP heads in the group, rows STEP apart are the same head of queries STEP / group apart
    constexpr int N = NC<T, DP>, STEP = NT / N;
    const int row0 = threadIdx.x / N;
    if (VEC && r0 + BR <= p.rows && STEP % d.group == 0) {
      const int64_t i0 = p.q0 + r0 / d.group;
      const T* q0 = (const T*)d.a.q + i0 * d.a.q_row + (int64_t)p.hk * d.group * d.a.q_head;
      const T* g0 = (const T*)d.a.dout + i0 * d.a.dout_row + (int64_t)p.hk * d.group * d.a.dout_head;
#pragma unroll
      for (int n = 0; n < BR / STEP; ++n) {
        const int c = (threadIdx.x % N) ^ sw<N>(n * STEP + row0);
        const int64_t di = n * (STEP / d.group);
        stage_chunk<T, DP, NT, VEC>(rt.q, n, c, d.a.dim, q0 + di * d.a.q_row + q_off);
        stage_chunk<T, DP, NT, VEC>(rt.g, n, c, d.a.dim, g0 + di * d.a.dout_row + g_off);
      }
    } else {
#pragma unroll 1
      for (int n = 0; n < BR / STEP; ++n) {
        const Row x = src(n * STEP + row0);
        const int c = (threadIdx.x % N) ^ sw<N>(n * STEP + row0);
        stage_chunk<T, DP, NT, VEC>(rt.q, n, c, d.a.dim, (const T*)d.a.q + x.token * d.a.q_row + x.head * d.a.q_head);
        stage_chunk<T, DP, NT, VEC>(rt.g, n, c, d.a.dim, (const T*)d.a.dout + x.token * d.a.dout_row + x.head * d.a.dout_head);
      }
    }
    if (threadIdx.x < BR) {
      const Row x = src(threadIdx.x);
      const int64_t st = (int64_t)x.head * d.a.n_q + x.token;
      rt.f0[threadIdx.x] = d.fac0[st];
      if constexpr (!FAST<T, BIAS>) rt.f1[threadIdx.x] = d.fac1[st];
      rt.delta[threadIdx.x] = d.delta[st];
      if constexpr (BIAS) rt.bias[threadIdx.x] = x.head * d.a.bias_head + (p.pair0 + (int64_t)x.i * p.nk) * d.a.bias_pair;
    }
  };
  if (first < last) fetch(rt0, first);
  zero_pad<T, DP, BR, NT, VEC>(rt0.q, d.a.dim);
  zero_pad<T, DP, BR, NT, VEC>(rt0.g, d.a.dim);
  zero_pad<T, DP, BR, NT, VEC>(rt1.q, d.a.dim);
  zero_pad<T, DP, BR, NT, VEC>(rt1.g, d.a.dim);

  typename Tr<T>::frag kf[NC<T, DP> / 2], vf[NC<T, DP> / 2];
#pragma unroll
  for (int s = 0; s < NC<T, DP> / 2; ++s) {
    kf[s] = load_chunk<T, VEC>((const T*)d.a.k + token * d.a.k_row + p.hk * d.a.k_head, 2 * s + h, d.a.dim);
    vf[s] = load_chunk<T, VEC>((const T*)d.a.v + token * d.a.v_row + p.hk * d.a.v_head, 2 * s + h, d.a.dim);
  }
  const float c = FAST<T, BIAS> ? d.a.scale * LOG2E : LOG2E;
  f16v dk[DP / 32], dv[DP / 32];
  zero<DP / 32>(dk);
  zero<DP / 32>(dv);
  auto work = [&](const RowTile<T, DP, NW, BR, BIAS>& rt, int t) __attribute__((always_inline)) {
    const int r0 = t * BR;
    if (r0 + BR <= r_lo || w0 >= p.nk) return;
    const bool part = r0 < r_hi || r0 + BR > p.rows || w0 + 32 > p.nk;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      f16v s, g;
      zero<1>(&s);
      zero<1>(&g);
      s = rows_times<T, DP>(rt.q, 32 * j, l31, h, kf, s);
      g = rows_times<T, DP>(rt.g, 32 * j, l31, h, vf, g);
      if constexpr (!FAST<T, BIAS>) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= d.a.scale;
      }
      unsigned seen = 0xffffu;                               // a bit per entry
      if (part || BIAS) {
        seen = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int rr = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3), r = r0 + rr;
          bool in = live && r >= rmin && r < p.rows;
          if constexpr (BIAS) {
            const float bv = in ? (float)((const T*)d.a.bias)[rt.bias[rr] + key * d.a.bias_pair] : NEG_INF;
            s[e] += bv;
            in = bv != NEG_INF;
          }
          seen |= (unsigned)in << e;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int rr = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
        s[e] = Probs<T, BIAS>::p(s[e], c, rt.f0[rr], FAST<T, BIAS> ? 0.f : rt.f1[rr]);
        g[e] = s[e] * (g[e] - rt.delta[rr]);
      }
      if (part || BIAS) {                                    // chosen, not multiplied: scores, statistics and do.v of what is taken out may be anything
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = seen >> e & 1 ? s[e] : 0.f;
          g[e] = seen >> e & 1 ? g[e] : 0.f;
        }
      }
      cols_times<DP>(rt.g, 32 * j, lane, (const float*)&s, dv);
      cols_times<DP>(rt.q, 32 * j, lane, (const float*)&g, dk);
    }
  };
  for (int t = first; t < last; t += 2) {
    tile_barrier();
    if (t + 1 < last) fetch(rt1, t + 1);
    work(rt0, t);
    if (t + 1 >= last) break;
    tile_barrier();
    if (t + 2 < last) fetch(rt0, t + 2);
    work(rt1, t + 1);
  }
  if (live) {
    const int64_t at = (token * d.a.kv_heads + p.hk) * d.a.dim;
    if (d.splits_k == 1) {
      store_col<T, DP, VEC>((T*)d.a.dk + at, h, d.a.dim, dk, d.a.scale);
      store_col<T, DP, VEC>((T*)d.a.dv + at, h, d.a.dim, dv, 1.f);
    } else {
      const int64_t n = (int64_t)d.a.n_k * d.a.kv_heads * d.a.dim;
      store_col<float, DP, VEC>(d.part_g + 2 * split * n + at, h, d.a.dim, dk, d.a.scale);
      store_col<float, DP, VEC>(d.part_g + (2 * split + 1) * n + at, h, d.a.dim, dv, 1.f);
    }
  }
}

// sums the ranges' shares of a gradient, in the ranges' order; blockIdx.y: the second of two gradients that lie side by side in every range
template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(const float* __restrict__ part, int splits, int64_t stride, int64_t n, T* __restrict__ out0, T* __restrict__ out1) {
  T* out = blockIdx.y ? out1 : out0;
  part += blockIdx.y * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float x = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) x += part[s * stride + i];
    out[i] = (T)x;
  }
}

template <typename T, int DP, bool BIAS, bool VEC>
hipError_t run_fwd(const Dev& d0, bool small, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  Dev d = d0;
  const int64_t n = (int64_t)d.tiles * d.a.B * d.a.kv_heads * d.splits;
  hipError_t rc = in_parts(d, n, [&](unsigned part) {
    if (small) hipLaunchKernelGGL((fwd_kernel<T, DP, 1, BN, BIAS, VEC>), dim3(part), dim3(64), 0, st, d);
    else hipLaunchKernelGGL((fwd_kernel<T, DP, 4, BN, BIAS, VEC>), dim3(part), dim3(256), 0, st, d);
  });
  if (rc == hipSuccess && n && d.splits > 1)
    rc = in_parts(d, ((int64_t)d.a.heads * d.a.n_q + 3) / 4, [&](unsigned part) { hipLaunchKernelGGL((join_kernel<T>), dim3(part), dim3(256), 0, st, d); });
  return rc;
}

template <typename T, int DP, bool BIAS, bool VEC>
hipError_t run_bwd(const Dev& d0, bool small_rows, bool small_keys, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32, BR = BN;
  Dev d = d0;
  const int64_t rows = (int64_t)d.a.max_nq * d.group;
  d.tiles = (int)((rows + (small_rows ? 31 : 127)) / (small_rows ? 32 : 128));
  auto sum = [&](int splits, int64_t count, int many, void* a, void* b) {
    if (splits == 1 || count == 0) return hipSuccess;
    const int64_t need = (count + 255) / 256;
    hipLaunchKernelGGL((sum_kernel<T>), dim3((unsigned)(need < 4096 ? need : 4096), many), dim3(256), 0, st, d.part_g, splits, many * count, count, (T*)a, (T*)b);
    return hipGetLastError();
  };
  // (the second kernel reads what the first one wrote: it is not started if a launch of the first failed)
  hipError_t rc = in_parts(d, (int64_t)d.tiles * d.a.B * d.a.kv_heads * d.splits_q, [&](unsigned part) {
    if (small_rows) hipLaunchKernelGGL((dq_kernel<T, DP, 1, BN, BIAS, VEC>), dim3(part), dim3(64), 0, st, d);
    else hipLaunchKernelGGL((dq_kernel<T, DP, 4, BN, BIAS, VEC>), dim3(part), dim3(256), 0, st, d);
  });
  if (rc == hipSuccess) rc = sum(d.splits_q, (int64_t)d.a.n_q * d.a.heads * d.a.dim, 1, d.a.dq, nullptr);
  if (rc != hipSuccess) return rc;
  d.tiles = (d.a.max_nk + (small_keys ? 31 : 127)) / (small_keys ? 32 : 128);
  rc = in_parts(d, (int64_t)d.tiles * d.a.B * d.a.kv_heads * d.splits_k, [&](unsigned part) {
    if (small_keys) hipLaunchKernelGGL((dkv_kernel<T, DP, 1, BR, BIAS, VEC>), dim3(part), dim3(64), 0, st, d);
    else hipLaunchKernelGGL((dkv_kernel<T, DP, 4, BR, BIAS, VEC>), dim3(part), dim3(256), 0, st, d);
  });
  return rc == hipSuccess ? sum(d.splits_k, (int64_t)d.a.n_k * d.a.kv_heads * d.a.dim, 2, d.a.dk, d.a.dv) : rc;
}

template <typename T, int DP>
hipError_t fwd_of(const Dev& d, bool small, hipStream_t st) {
  if (d.a.bias) return d.vec ? run_fwd<T, DP, true, true>(d, small, st) : run_fwd<T, DP, true, false>(d, small, st);
  return d.vec ? run_fwd<T, DP, false, true>(d, small, st) : run_fwd<T, DP, false, false>(d, small, st);
}
template <typename T, int DP>
hipError_t bwd_of(const Dev& d, bool sr, bool sk, hipStream_t st) {
  if (d.a.bias) return d.vec ? run_bwd<T, DP, true, true>(d, sr, sk, st) : run_bwd<T, DP, true, false>(d, sr, sk, st);
  return d.vec ? run_bwd<T, DP, false, true>(d, sr, sk, st) : run_bwd<T, DP, false, false>(d, sr, sk, st);
}

}  // namespace dptat
