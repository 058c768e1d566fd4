// dpt_attn.h - attention over packed complexes: the pieces its forward and backward kernels share.
//
// One workgroup works on one (complex, key head) and a block of "rows": the queries of the complex times the query heads that share the key head,
// row r = query r / G, head r % G of the group.  So keys and values are staged once for all heads that share them, a single new token of G heads
// is still one row block, and the gradients of shared heads are sums inside a workgroup.
//
// Products run on 32x32 matrix tiles.  Scores are formed transposed where a row's statistics are needed (keys down, rows across): a lane then holds 16 keys of
// ONE row, so maxima and sums are register work plus one exchange between the wave's halves, and the factors of a row are one register.  An
// accumulator tile is the second operand of the next product as it stands: lane half h holds the entries 8 g + 4 h + i (g, i = 0..3) of a 32-long
// axis, and since a product's sum may run in any order, the first operand is read in that same order (bf16: two 4-entry transposing LDS reads;
// fp32: plain reads).  No data moves between lanes.
#pragma once
#include "dpt_dev.h"

namespace dptat {
using namespace dpt;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_INF = -__builtin_huge_valf();

struct Dev {                     // DptAttnArgs plus what every workgroup would derive
  DptAttnArgs a;
  int group, splits;             // query heads per key head; key ranges
  uint32_t magic;                // r / group = mulhi(r, magic) for group > 1
  int tiles;                     // row (backward: key) blocks of the largest complex
  int first;                     // this launch's first workgroup (in_parts)
  int vec;                       // rows of q, k, v, dout may be read, out and gradients written, 16 bytes at a time
  float *delta, *fac0, *fac1;    // backward, [heads, n_q] each: sum_d dout out; what turns a score into a probability (Probs)
  float *part_o, *part_ml;       // forward with splits: [splits, n_q, heads, dim] and [splits, 2, heads, n_q]
  int splits_q, splits_k;        // backward: key ranges of a row block (dq), row ranges of a key block (dk, dv) that are summed afterwards
  float* part_g;                 // [splits_q, n_q, heads, dim], then [splits_k, 2, n_k, kv_heads, dim]: the one is summed before the other is written
};

__device__ __forceinline__ int div_group(const Dev& d, int r) { return d.group == 1 ? r : (int)__umulhi((uint32_t)r, d.magic); }

template <typename T> struct Tr;
template <> struct Tr<__bf16> {
  typedef b8 frag;
  static constexpr int CH = 8;   // elements of a 16-byte chunk
  static __device__ __forceinline__ f16v mma(frag a, frag b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<float> {
  typedef f4 frag;
  static constexpr int CH = 4;
  static __device__ __forceinline__ f16v mma(frag a, frag b, f16v c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// four neighbouring elements at any address (the memory system takes them unaligned)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; };

// 16-byte chunks per row of a tile of DP elements, and the permutation of a row's chunks in LDS that keeps both kinds of reads (32 rows at one
// chunk; 4 rows at 4 neighbouring chunks) on different banks.  Linear over xor, and only the low 4 bits of the row count.
template <typename T, int DP> constexpr int NC = DP * (int)sizeof(T) / 16;
template <int N>
__device__ __forceinline__ constexpr int sw(int row) {
  if constexpr (N == 4) return (row >> 2) & 3;
  else if constexpr (N == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else if constexpr (N == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return (((row >> 2) & 1) << 3) | (((row >> 3) & 1) << 2) | (row & 3);
}

// one chunk of a row in memory; what lies behind the row's dim elements is 0.  VEC: rows may be read 16 bytes at a time (dim is a multiple of a chunk)
template <typename T, bool VEC>
__device__ __forceinline__ typename Tr<T>::frag load_chunk(const T* __restrict__ row, int c, int dim) {
  constexpr int CH = Tr<T>::CH;
  typename Tr<T>::frag v;
  if constexpr (VEC) {
    if (c * CH < dim) return *reinterpret_cast<const typename Tr<T>::frag*>(row + c * CH);
#pragma unroll
    for (int e = 0; e < CH; ++e) v[e] = (T)0.f;
  } else {
#pragma unroll
    for (int e = 0; e < CH; ++e) v[e] = c * CH + e < dim ? row[c * CH + e] : (T)0.f;
  }
  return v;
}

// first / second operand of the row-wise products: chunk 2 s + h of the lane's row
template <typename T, int DP>
__device__ __forceinline__ typename Tr<T>::frag lds_chunk(const T* tile, int row, int c) {
  constexpr int N = NC<T, DP>;
  return *reinterpret_cast<const typename Tr<T>::frag*>(tile + (row * N + (c ^ sw<N>(row))) * Tr<T>::CH);
}

// acc[row of the tile, column] += tile rows (row0 + 0..31) x the lane's column in b
template <typename T, int DP>
__device__ __forceinline__ f16v rows_times(const T* tile, int row0, int l31, int h, const typename Tr<T>::frag* b, f16v acc) {
#pragma unroll
  for (int s = 0; s < NC<T, DP> / 2; ++s) acc = Tr<T>::mma(lds_chunk<T, DP>(tile, row0 + l31, 2 * s + h), b[s], acc);
  return acc;
}

// out[d, column] += sum over the 32 tile rows from row0 of tile[row, d] y[row, column], y an accumulator tile
template <int DP>
__device__ __forceinline__ void cols_times(const __bf16* tile, int row0, int lane, const float* y, f16v* out) {
  constexpr int N = NC<__bf16, DP>;
  typedef __attribute__((address_space(3))) s4* lds4;
  // transposing read: 16 lanes fetch 4 rows x 16 columns and get a column's 4 rows each
  const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), sub = (lane & 1) * 4;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    b8 b;
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (__bf16)y[8 * ks + e];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      b8 a;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = row0 + 16 * ks + 8 * j + r;
        const __bf16* p = tile + (row * N + ((4 * dt + c) ^ sw<N>(row))) * 8 + sub;
        const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p));
        const b4 w = __builtin_bit_cast(b4, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * j + e] = w[e];
      }
      out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, out[dt], 0, 0, 0);
    }
  }
}
template <int DP>
__device__ __forceinline__ void cols_times(const float* tile, int row0, int lane, const float* y, f16v* out) {
  constexpr int N = NC<float, DP>;
  const int h = lane >> 5, l31 = lane & 31;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = row0 + 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      const float a = tile[(row * N + ((8 * dt + (l31 >> 2)) ^ sw<N>(row))) * 4 + (l31 & 3)];
      out[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, y[e], out[dt], 0, 0, 0);
    }
  }
}

// over a lane pair (l, l + 32)
__device__ __forceinline__ float half_max(float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); }
__device__ __forceinline__ float half_sum(float x) { return x + __shfl_xor(x, 32, 64); }

// out[d = 32 dt + 8 g + 4 h + i] of the lane's column into a row of dim elements
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void store_col(T* __restrict__ row, int h, int dim, const f16v* acc, float f) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * h;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[dt][4 * g + i] * f;
      if constexpr (VEC) {
        if (d < dim) store_n<T, 4>(row + d, v);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < dim) row[d + i] = (T)v[i];
      }
    }
}

// A tile of ROWS rows is filled by the workgroup's NT lanes, 16 bytes per lane and turn, in LDS order: turn n of lane t fills chunk n NT + t, so the
// lane's source is the chunk that the permutation puts there.
//   VEC: straight into LDS (no registers; the tile is there after the next tile_barrier).  Chunks behind dim are not
//        fetched: they hold the zeros that zero_pad() put there before the loop.
//   otherwise: through registers, element by element.
template <typename T, int DP, int NT, bool VEC>
__device__ __forceinline__ void stage_chunk(T* tile, int n, int c, int dim, const T* row) {
  constexpr int CH = Tr<T>::CH;
  if constexpr (VEC) {
    T* dst = tile + (n * NT + __builtin_amdgcn_readfirstlane(threadIdx.x & ~63)) * CH;
    if (c * CH < dim)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(row + c * CH), (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
  } else {
    *reinterpret_cast<typename Tr<T>::frag*>(tile + (n * NT + threadIdx.x) * CH) = load_chunk<T, false>(row, c, dim);
  }
}
// rows of a regular array, `there` of them (at least one): row r at src + r stride.  What follows the last one repeats it.
// (VEC: the host has checked that a tile's offsets fit 32 bits; a 64-bit multiplication costs several times as much)
template <typename T, int DP, int ROWS, int NT, bool VEC>
__device__ __forceinline__ void stage(T* tile, int dim, const T* src, int64_t stride, int there) {
  constexpr int N = NC<T, DP>, STEP = NT / N;
  static_assert(NT % N == 0 && ROWS % STEP == 0, "every lane in every turn");
#pragma unroll
  for (int n = 0; n < ROWS / STEP; ++n) {
    const int row = n * STEP + threadIdx.x / N, r = min(row, there - 1);
    const T* p = VEC ? src + (uint32_t)r * (uint32_t)stride : src + (int64_t)r * stride;
    stage_chunk<T, DP, NT, VEC>(tile, n, (threadIdx.x % N) ^ sw<N>(row), dim, p);
  }
}

// The barrier between tiles: every wave waits for its own fetches into LDS, then for the others.  The wait is written out: the compiler orders a workgroup's
// plain LDS accesses at a barrier, but does not hold a barrier back for fetches that go past the registers (seen in its output: none on a loop's way back).
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}
template <typename T, int DP, int ROWS, int NT, bool VEC>
__device__ __forceinline__ void zero_pad(T* tile, int dim) {
  constexpr int N = NC<T, DP>, CH = Tr<T>::CH;
  if (!VEC || dim == DP) return;
  for (int i = threadIdx.x; i < ROWS * N; i += NT) {
    const int row = i / N, c = (i % N) ^ sw<N>(row);
    typename Tr<T>::frag z;
#pragma unroll
    for (int e = 0; e < CH; ++e) z[e] = (T)0.f;
    if (c * CH >= dim) *reinterpret_cast<typename Tr<T>::frag*>(tile + i * CH) = z;
  }
}

// A launch's gridDim.x * blockDim.x has to stay below 2^32, and check() allows up to 2^31 workgroups of 256 lanes: more than MOST go in several launches, each
// with the number of its first workgroup.  Ends at the first launch that fails.
template <typename F>
hipError_t in_parts(Dev& d, int64_t n, F launch) {
  constexpr int64_t MOST = 1 << 23;
  for (int64_t at = 0; at < n; at += MOST) {
    d.first = (int)at;
    launch((unsigned)(n - at < MOST ? n - at : MOST));
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

// dpt_attn_<type>_<padded head dimension>.hip
#define DPT_ATTN_DECL(x)                                          \
  hipError_t fwd_##x(const Dev& d, bool small, hipStream_t st);   \
  hipError_t bwd_##x(const Dev& d, bool small_rows, bool small_keys, hipStream_t st);
DPT_ATTN_DECL(f32_32) DPT_ATTN_DECL(f32_64) DPT_ATTN_DECL(f32_128) DPT_ATTN_DECL(bf16_32) DPT_ATTN_DECL(bf16_64) DPT_ATTN_DECL(bf16_128)
#undef DPT_ATTN_DECL

}  // namespace dptat
