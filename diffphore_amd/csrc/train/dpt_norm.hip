// dpt_norm.hip - layer norm over the last dimension, forward and backward.
//
// Both directions are bound by HBM: x is read once, y written once (backward: x, dy read, dx written).  A row stays in the registers of L lanes
// (L = 8 .. 1024: part of a wave, a wave, or a workgroup), so the statistics are taken in two passes over registers, not over memory:
//   m0 = mean x;  d = x - m0;  c = mean d;  d -= c        (c is what the rounding of m0 left: rows whose entries lie close together need it)
//   rstd = 1 / sqrt(mean d^2 + eps);  y = d rstd w + b;  mean = m0 + c
// Backward, with xh = d rstd and g = dy w:  dx = rstd (g - mean g - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy.
// The column sums stay in registers while a group walks over its rows; a workgroup joins its groups in LDS and writes one partial row, a second
// launch adds the partial rows in a fixed order: no atomics, the same bits every time.
// Measured: forward 16384 x 4096 bf16 48 us (5.5 TB/s traced, 4.6 from call to call), backward 32749 x 2048 bf16 89 + 8 us (4.5 TB/s for the rows); a copy
// of 1 GiB runs at 5.0 TB/s.  Backward with three exchanges per row and no row ahead took 188 us.  The widest rows pay for their 1024 lanes (128 registers each: up to 6
// spilled backward, 28 to 32 where a row's length or address does not allow 16-byte reads): 4096 x 16384 bf16 77 forward and 206 us backward, 4096 x 16383 182 and 319.
#include "dpt_dev.h"

namespace dptn {
using namespace dpt;

constexpr int MAX_WIDTH = 16384;
constexpr int PARTS = 1024;           // most partial rows of the column sums

// sum over the L lanes of a row; L > 64: over the workgroup (blockDim.x == L), through LDS.  N sums at a time.
template <int L, int N>
__device__ __forceinline__ void row_sum(float* x, float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = group_sum<(L < 64 ? L : 64)>(x[i]);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    __syncthreads();                 // the last sum's values have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * W + threadIdx.x / 64] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) x[i] += red[i * W + w];
    }
  }
}

// column of element e of a lane: chunks of V consecutive elements, dealt over the lanes
template <int L, int V>
__device__ __forceinline__ int column(int lane, int e) { return ((e / V) * L + lane) * V + e % V; }

template <typename T, int L, int E, int V>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int lane, int width, float* o) {
#pragma unroll
  for (int e = 0; e < E; e += V) {
    const int c = column<L, V>(lane, e);
    if (c < width) {
      load_n<T, V>(p + c, o + e);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) o[e + i] = 0.f;
    }
  }
}

template <typename T, int L, int E, int V>
__device__ __forceinline__ void store_row(T* __restrict__ p, int lane, int width, const float* v) {
#pragma unroll
  for (int e = 0; e < E; e += V) {
    const int c = column<L, V>(lane, e);
    if (c < width) store_n<T, V>(p + c, v + e);
  }
}

// d = x - mean of the row, exact to the rounding of d itself; entries behind the width are 0
template <int L, int E, int V>
__device__ __forceinline__ void centre(float* x, float m0, int lane, int width, float inv, float* mean, float* red) {
  float s[1] = {0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = column<L, V>(lane, e) < width ? x[e] - m0 : 0.f;
    s[0] += x[e];
  }
  row_sum<L, 1>(s, red);
  const float c = s[0] * inv;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = column<L, V>(lane, e) < width ? x[e] - c : 0.f;
  *mean = m0 + c;
}

template <typename T, typename W, int L, int E, int V>
__global__ __launch_bounds__(L > 256 ? L : 256) void fwd_kernel(int64_t rows, int width, const T* __restrict__ x, int64_t xs, const W* __restrict__ w,
                                                                const W* __restrict__ b, float eps, T* __restrict__ y, int64_t ys,
                                                                float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x % L;
  const int64_t groups = (int64_t)gridDim.x * (blockDim.x / L);
  const float inv = 1.f / (float)width;
  // the trip count is the same for every lane of a wave (L <= 64: rows past the end are computed and not stored) and of a workgroup (L > 64)
  for (int64_t r0 = (int64_t)blockIdx.x * (blockDim.x / L); r0 < rows; r0 += groups) {
    const int64_t r = r0 + threadIdx.x / L;
    const bool live = r < rows;
    float v[E], s[1] = {0.f}, m, q[1] = {0.f};
    load_row<T, L, E, V>(x + (live ? r : rows - 1) * xs, lane, width, v);
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += v[e];
    row_sum<L, 1>(s, red);
    centre<L, E, V>(v, s[0] * inv, lane, width, inv, &m, red);
#pragma unroll
    for (int e = 0; e < E; ++e) q[0] = fmaf(v[e], v[e], q[0]);
    row_sum<L, 1>(q, red);
    const float rs = 1.f / sqrtf(q[0] * inv + eps);
#pragma unroll
    for (int e = 0; e < E; e += V) {
      const int c = column<L, V>(lane, e);
      if (c >= width) continue;
      float wv[V], bv[V];
#pragma unroll
      for (int i = 0; i < V; ++i) { wv[i] = 1.f; bv[i] = 0.f; }
      if (w) load_n<W, V>(w + c, wv);
      if (b) load_n<W, V>(b + c, bv);
#pragma unroll
      for (int i = 0; i < V; ++i) v[e + i] = fmaf(v[e + i] * rs, wv[i], bv[i]);
    }
    if (live) {
      store_row<T, L, E, V>(y + r * ys, lane, width, v);
      if (lane == 0) { mean[r] = m; rstd[r] = rs; }
    }
  }
}

// a row's elements of a lane as they lie in memory
template <typename T, int E, int V>
struct Raw {
  typedef __attribute__((ext_vector_type(V))) T vec;
  vec v[E / V];
  template <int L>
  __device__ __forceinline__ void load(const T* __restrict__ p, int lane, int width) {
#pragma unroll
    for (int i = 0; i < E / V; ++i) {
      const int c = column<L, V>(lane, i * V);
      if (c < width) {
        v[i] = *reinterpret_cast<const vec*>(p + c);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = (T)0.f;
      }
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return (float)v[e / V][e % V]; }
};

// One exchange per row: with u = x - mean (as stored) the three sums of u, g and g u give what the rounding of the stored mean left (c = mean u), mean g
// and mean(g xh) = rstd (mean(g u) - c mean g).  The next row is on its way while a row is worked on, and the weight stays in registers (not in the widest
// rows: 1024 lanes have 128 registers each).
template <typename T, typename W, int L, int E, int V>
__global__ __launch_bounds__(L > 256 ? L : 256) void bwd_kernel(int64_t rows, int width, const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
                                                                int64_t xs, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                const W* __restrict__ w, T* __restrict__ dx, int64_t dxs, float* __restrict__ part) {
  constexpr int TPB = L > 256 ? L : 256, G = TPB / L;
  constexpr bool ROOM = L < 1024;
  __shared__ float red[L > 64 ? 3 * (L / 64) : 1];
  __shared__ float cols[G > 1 ? G * L * E : 1];
  const int lane = threadIdx.x % L;
  const int64_t groups = (int64_t)gridDim.x * G;
  const float inv = 1.f / (float)width;
  float wv[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { wv[e] = 1.f; dw[e] = 0.f; db[e] = 0.f; }
  if (ROOM && w) load_row<W, L, E, V>(w, lane, width, wv);
  Raw<T, E, V> xr, gr;
  float mr, rr;
  auto fetch = [&](int64_t r0) __attribute__((always_inline)) {
    const int64_t r = r0 + threadIdx.x / L, at = r < rows ? r : rows - 1;
    xr.template load<L>(x + at * xs, lane, width);
    gr.template load<L>(dy + at * dys, lane, width);
    mr = mean[at];
    rr = rstd[at];
  };
  int64_t r0 = (int64_t)blockIdx.x * G;
  if (ROOM && r0 < rows) fetch(r0);
  for (; r0 < rows; r0 += groups) {
    const int64_t r = r0 + threadIdx.x / L;
    const bool live = r < rows;
    float v[E], g[E], s[3] = {0.f, 0.f, 0.f};
    if constexpr (!ROOM) {
      fetch(r0);
      if (w) load_row<W, L, E, V>(w, lane, width, wv);
    }
    const float rs = rr;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = column<L, V>(lane, e) < width ? xr[e] - mr : 0.f;
      g[e] = gr[e];
      const float t = g[e] * wv[e];
      s[0] += v[e];
      s[1] += t;
      s[2] = fmaf(t, v[e], s[2]);
    }
    if (ROOM && r0 + groups < rows) fetch(r0 + groups);
    row_sum<L, 3>(s, red);
    const float c = s[0] * inv, a = s[1] * inv, q = rs * fmaf(-c, a, s[2] * inv);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float xh = (v[e] - c) * rs;
      if (live) { dw[e] = fmaf(g[e], xh, dw[e]); db[e] += g[e]; }
      v[e] = rs * (g[e] * wv[e] - a - xh * q);
    }
    if (live) store_row<T, L, E, V>(dx + r * dxs, lane, width, v);
  }
  if (!part) return;
  // columns of the workgroup's groups, joined in the groups' order
  float* p = part + (size_t)blockIdx.x * 2 * width;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* a = k ? db : dw;
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) cols[(threadIdx.x / L) * L * E + column<L, V>(lane, e)] = a[e];
      __syncthreads();
      for (int c = threadIdx.x; c < width; c += TPB) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < G; ++q) t += cols[q * L * E + c];
        p[k * width + c] = t;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = column<L, V>(lane, e);
        if (c < width) p[k * width + c] = a[e];
      }
    }
  }
}

// out[c] = sum over the partial rows: 16 columns and 64 strands of rows per workgroup (16 loads one behind the other for the most partial rows), joined in order
template <typename W>
__global__ __launch_bounds__(1024) void cols_kernel(int parts, int width, const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float t[64][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, k = blockIdx.y, strand = threadIdx.x / 16;
  W* out = k ? db : dw;
  if (!out) return;
  float a = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int p = strand; p < parts; p += 64) a += part[((size_t)p * 2 + k) * width + c];
  }
  t[strand][threadIdx.x % 16] = a;
  __syncthreads();
  if (strand == 0 && c < width) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) s += t[i][threadIdx.x];
    out[c] = (W)s;
  }
}

struct Args {
  int64_t rows; int width;
  const void *x, *dy, *w, *b; int64_t xs, dys, ys;
  float eps; void* y; float *mean, *rstd, *part; int blocks; hipStream_t st;
};

template <typename T, typename W, int L, int E, int V, bool BWD>
void launch(const Args& a) {
  constexpr int TPB = L > 256 ? L : 256;
  if constexpr (BWD)
    hipLaunchKernelGGL((bwd_kernel<T, W, L, E, V>), dim3(a.blocks), dim3(TPB), 0, a.st, a.rows, a.width, (const T*)a.dy, a.dys, (const T*)a.x, a.xs, a.mean,
                       a.rstd, (const W*)a.w, (T*)a.y, a.ys, a.part);
  else
    hipLaunchKernelGGL((fwd_kernel<T, W, L, E, V>), dim3(a.blocks), dim3(TPB), 0, a.st, a.rows, a.width, (const T*)a.x, a.xs, (const W*)a.w, (const W*)a.b, a.eps,
                       (T*)a.y, a.ys, a.mean, a.rstd);
}

// lanes and elements per lane by width: the fewest lanes that hold a row in at most 16 registers per array.  (Rows of 1025 .. 2048 with 8 registers in 256
// lanes rather than with 32 in one wave, which leaves one wave per SIMD: backward 32749 x 2048 bf16 88 against 112 us.)
template <typename T, typename W, int V, bool BWD>
void by_width(const Args& a) {
  constexpr int V4 = V == 1 ? 1 : 4;
  if (a.width <= 32) launch<T, W, 8, 4, V4, BWD>(a);
  else if (a.width <= 64) launch<T, W, 16, 4, V4, BWD>(a);
  else if (a.width <= 256) launch<T, W, 64, 4, V4, BWD>(a);
  else if (a.width <= 1024) launch<T, W, 64, 16, V, BWD>(a);
  else if (a.width <= 2048) launch<T, W, 256, 8, V, BWD>(a);
  else if (a.width <= 4096) launch<T, W, 256, 16, V, BWD>(a);
  else if (a.width <= 8192) launch<T, W, 512, 16, V, BWD>(a);
  else launch<T, W, 1024, 16, V, BWD>(a);
}

int groups_per_block(int width) { return width <= 32 ? 32 : width <= 64 ? 16 : width <= 1024 ? 4 : 1; }

bool aligned(const void* p, int64_t stride, int size, int n) { return ((uintptr_t)p % (size * n)) == 0 && stride % n == 0; }

template <bool BWD>
int dispatch(int type, int wtype, const Args& a) {
  const int ws = wtype == DPT_F32 ? 4 : 2;
  if (type == DPT_F32) {
    const bool v = a.width % 4 == 0 && aligned(a.x, a.xs, 4, 4) && aligned(a.y, a.ys, 4, 4) && aligned(a.w, 0, ws, 4) && aligned(a.b, 0, ws, 4) &&
                   (!BWD || aligned(a.dy, a.dys, 4, 4));
    if (v) by_width<float, float, 4, BWD>(a); else by_width<float, float, 1, BWD>(a);
  } else {
    // 8 elements are 16 bytes of x; narrow rows take 4 at a time (by_width), their alignment follows
    const bool v = a.width % 8 == 0 && aligned(a.x, a.xs, 2, 8) && aligned(a.y, a.ys, 2, 8) && aligned(a.w, 0, ws, 4) && aligned(a.b, 0, ws, 4) &&
                   (wtype == DPT_F32 || (aligned(a.w, 0, 2, 8) && aligned(a.b, 0, 2, 8))) && (!BWD || aligned(a.dy, a.dys, 2, 8));
    if (wtype == DPT_F32) {
      if (v) by_width<__bf16, float, 8, BWD>(a); else by_width<__bf16, float, 1, BWD>(a);
    } else {
      if (v) by_width<__bf16, __bf16, 8, BWD>(a); else by_width<__bf16, __bf16, 1, BWD>(a);
    }
  }
  return (int)hipGetLastError();
}

bool bad(int type, int wtype, int64_t rows, int width) {
  return (type != DPT_F32 && type != DPT_BF16) || (wtype != DPT_F32 && wtype != type) || rows < 0 || width < 1;
}

int parts_of(int64_t rows, int width) {
  const int64_t need = (rows + groups_per_block(width) - 1) / groups_per_block(width);
  return (int)(need < PARTS ? need : PARTS);
}

}  // namespace dptn

extern "C" {

int dpt_layer_norm_max_width(void) { return dptn::MAX_WIDTH; }

int dpt_layer_norm_fwd(int32_t type, int32_t wtype, int64_t rows, int32_t width, const void* x, int64_t x_stride, const void* weight, const void* bias,
                       float eps, void* y, int64_t y_stride, float* mean, float* rstd, void* stream) {
  if (dptn::bad(type, wtype, rows, width) || !(eps >= 0.f)) return DPT_E_BADARG;
  if (width > dptn::MAX_WIDTH) return DPT_E_TOOLARGE;
  if (rows == 0) return DPT_OK;
  if (!x || !y || !mean || !rstd || x_stride < 0 || y_stride < width) return DPT_E_BADARG;
  dptn::Args a{};
  a.rows = rows; a.width = width; a.x = x; a.xs = x_stride; a.w = weight; a.b = bias; a.eps = eps; a.y = y; a.ys = y_stride; a.mean = mean; a.rstd = rstd;
  const int64_t need = (rows + dptn::groups_per_block(width) - 1) / dptn::groups_per_block(width);
  a.blocks = (int)(need < 1 << 20 ? need : 1 << 20);
  a.st = (hipStream_t)stream;
  return dptn::dispatch<false>(type, wtype, a);
}

size_t dpt_layer_norm_ws_bytes(int64_t rows, int32_t width) {
  if (rows < 0 || width < 1 || width > dptn::MAX_WIDTH) return 0;
  return (size_t)dptn::parts_of(rows, width) * 2 * (size_t)width * sizeof(float);
}

int dpt_layer_norm_bwd(int32_t type, int32_t wtype, int64_t rows, int32_t width, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                       const float* mean, const float* rstd, const void* weight, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                       void* ws, size_t ws_bytes, void* stream) {
  if (dptn::bad(type, wtype, rows, width)) return DPT_E_BADARG;
  if (width > dptn::MAX_WIDTH) return DPT_E_TOOLARGE;
  const bool cols = dweight || dbias;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx || dy_stride < 0 || x_stride < 0 || dx_stride < width)) return DPT_E_BADARG;
  if (cols && rows > 0 && (!ws || ws_bytes < dpt_layer_norm_ws_bytes(rows, width))) return DPT_E_BADARG;
  const int parts = dptn::parts_of(rows, width);
  if (rows > 0) {
    dptn::Args a{};
    a.rows = rows; a.width = width; a.dy = dy; a.dys = dy_stride; a.x = x; a.xs = x_stride; a.mean = (float*)mean; a.rstd = (float*)rstd; a.w = weight;
    a.y = dx; a.ys = dx_stride; a.part = cols ? (float*)ws : nullptr; a.blocks = parts; a.st = (hipStream_t)stream;
    const int rc = dptn::dispatch<true>(type, wtype, a);
    if (rc) return rc;
  }
  if (cols) {
    const dim3 grid((width + 15) / 16, 2);
    if (wtype == DPT_F32)
      hipLaunchKernelGGL(dptn::cols_kernel<float>, grid, dim3(1024), 0, (hipStream_t)stream, parts, width, (const float*)ws, (float*)dweight, (float*)dbias);
    else
      hipLaunchKernelGGL(dptn::cols_kernel<__bf16>, grid, dim3(1024), 0, (hipStream_t)stream, parts, width, (const float*)ws, (__bf16*)dweight, (__bf16*)dbias);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
