// dpt_adamw.hip - one AdamW step over a list of tensors, states in 32 or 8 bits, with the running average of the parameters.
//
// Bound by HBM: every value is read once and written once.  A wave takes one 256-element block (4 elements per lane: one 16-byte load per fp32
// array); the block's tensor comes from a table, the gradients' addresses come with the launch.  All of a step is ONE launch per 400 tensors.
//
// Step number: b1^t and b2^t live on the device (so a captured graph counts on), every workgroup reads them, and the workgroup that is the last to
// have read them moves them on.
//
// 8-bit states: m' and v' are formed in 64 bits from the decoded values, the parameter's update uses them unrounded, and the stored codes are the
// nearest ones.  "Nearest" is decided exactly: a candidate from a 32-bit root is compared with the borders (c -+ 1/2)^2 resp. ^4, whose products
// with the scale are exact or within 2^-53 - so a code never depends on the rounding of a square root.
#include "dpt_dev.h"

namespace dpta {
using namespace dpt;

constexpr int BLOCK = DPT_ADAMW_BLOCK, WAVES = 4;

struct Grads { const void* p[DPT_ADAMW_MAX_TENSORS]; };

__device__ __forceinline__ double wave_max(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_xor(x, d, 64);
    x = y > x ? y : x;
  }
  return x;
}

// nearest code c in 0..TOP of |x| on the curve scale (c / TOP)^POW
template <int TOP, int POW>
__device__ __forceinline__ int encode(double x, float scale, double inv) {
  constexpr double T = POW == 2 ? (double)TOP * TOP : (double)TOP * TOP * TOP * TOP;
  const float u = (float)(x * inv);
  float root = sqrtf(u);
  if constexpr (POW == 4) root = sqrtf(root);
  int c = (int)(root * (float)TOP + 0.5f);
  c = c > TOP ? TOP : c;
  const double y = x * T, s = scale;
  auto border = [&](int k) {                       // scale (k - 1/2)^POW
    const double h = (double)k - 0.5, h2 = h * h;
    return POW == 2 ? s * h2 : s * (h2 * h2);
  };
  if (c < TOP && y >= border(c + 1)) ++c;
  else if (c > 0 && y < border(c)) --c;
  return c;
}

template <typename P, typename G, int BITS, bool EMA>
__global__ __launch_bounds__(64 * WAVES) void step_kernel(DptAdamWArgs a, Grads grads) {
  // the step's factors, in 64 bits
  const double p1 = a.counter[1] * a.beta1, p2 = a.counter[2] * a.beta2;
  const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
  const float b1 = (float)a.beta1, omb1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, omb2 = (float)(1.0 - a.beta2);
  const float lr1 = (float)(lr / (1.0 - p1)), ic2 = (float)(1.0 / (1.0 - p2)), eps = (float)a.eps;
  const float ema_d = (float)a.ema_decay, ema_o = (float)(1.0 - a.ema_decay), gs = a.grad_scale ? *a.grad_scale : 1.f;
  const int lane = threadIdx.x & 63;
  for (int i = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / 64); i < a.n_blocks; i += gridDim.x * WAVES) {
    const int blk = a.block0 + i, t = __builtin_amdgcn_readfirstlane(a.block_tensor[blk]);
    const int64_t in_tensor = (int64_t)(blk - a.first_block[t]) * BLOCK, at = (int64_t)blk * BLOCK + lane * 4;
    const int64_t left = a.numel[t] - in_tensor;                         // elements of the tensor from this block on
    P* __restrict__ p = (P*)a.param[t] + in_tensor;
    const G* __restrict__ g = (const G*)grads.p[t - a.tensor0] + in_tensor;
    const float shrink = (float)(1.0 - lr * a.weight_decay * (double)a.decay[t]);
    const bool whole = left >= BLOCK && ((uintptr_t)p % (4 * sizeof(P))) == 0 && ((uintptr_t)g % (4 * sizeof(G))) == 0;
    if (!grads.p[t - a.tensor0]) continue;                               // no gradient: the tensor and its state stay as they are
    float gv[4], pv[4];
    if (whole) {
      load_n<G, 4>(g + lane * 4, gv);
      if constexpr (sizeof(P) == 4) load_n<P, 4>(p + lane * 4, pv);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = lane * 4 + e < left;
        gv[e] = in ? (float)g[lane * 4 + e] : 0.f;
        if constexpr (sizeof(P) == 4) pv[e] = in ? (float)p[lane * 4 + e] : 0.f;
      }
    }
    if constexpr (sizeof(P) == 2) load_n<float, 4>(a.master + at, pv);
    float mv[4], vv[4];
    if constexpr (BITS == 32) {
      float* ms = (float*)a.exp_avg + at;
      float* vs = (float*)a.exp_avg_sq + at;
      load_n<float, 4>(ms, mv);
      load_n<float, 4>(vs, vv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = gv[e] * gs;
        mv[e] = mv[e] * b1 + x * omb1;
        vv[e] = vv[e] * b2 + x * x * omb2;
      }
      store_n<float, 4>(ms, mv);
      store_n<float, 4>(vs, vv);
    } else {
      char4* ms = (char4*)((int8_t*)a.exp_avg + at);
      uchar4* vs = (uchar4*)((uint8_t*)a.exp_avg_sq + at);
      const char4 mc = *ms;
      const uchar4 vc = *vs;
      const double ma = (double)a.exp_avg_scale[blk] / (127.0 * 127.0), va = (double)a.exp_avg_sq_scale[blk] / (255.0 * 255.0 * 255.0 * 255.0);
      const int ci[4] = {mc.x, mc.y, mc.z, mc.w}, ui[4] = {vc.x, vc.y, vc.z, vc.w};
      double m[4], v[4], mm = 0.0, vm = 0.0;
      bool fine = true;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double x = (double)gv[e] * (double)gs;
        const int u2 = ui[e] * ui[e];                                     // < 2^16: its square fits 32 unsigned bits
        m[e] = ma * (double)(ci[e] * abs(ci[e])) * a.beta1 + x * (1.0 - a.beta1);
        v[e] = va * (double)((unsigned)u2 * (unsigned)u2) * a.beta2 + x * x * (1.0 - a.beta2);
        mv[e] = (float)m[e];
        vv[e] = (float)v[e];
        fine = fine && __builtin_isfinite(mv[e]) && __builtin_isfinite(vv[e]);
        mm = fmax(mm, fabs(m[e]));
        vm = fmax(vm, v[e]);
      }
      float msc = (float)wave_max(mm), vsc = (float)wave_max(vm);
      int cm[4] = {0, 0, 0, 0}, cv[4] = {0, 0, 0, 0};
      if (__all(fine)) {
        const double mi = 1.0 / (double)msc, vi = 1.0 / (double)vsc;         // inf for a scale of 0: not used then
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (msc > 0.f) {
            cm[e] = encode<127, 2>(fabs(m[e]), msc, mi);
            if (m[e] < 0.0) cm[e] = -cm[e];
          }
          if (vsc > 0.f) {
            cv[e] = encode<255, 4>(v[e], vsc, vi);
            if (cv[e] == 0 && v[e] > 0.0) cv[e] = 1;
          }
        }
      } else {
        msc = vsc = __builtin_nanf("");
      }
      *ms = make_char4((signed char)cm[0], (signed char)cm[1], (signed char)cm[2], (signed char)cm[3]);
      *vs = make_uchar4((unsigned char)cv[0], (unsigned char)cv[1], (unsigned char)cv[2], (unsigned char)cv[3]);
      if (lane == 0) { a.exp_avg_scale[blk] = msc; a.exp_avg_sq_scale[blk] = vsc; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) pv[e] = pv[e] * shrink - lr1 * (mv[e] / (sqrtf(vv[e] * ic2) + eps));
    if constexpr (sizeof(P) == 2) store_n<float, 4>(a.master + at, pv);
    if constexpr (EMA) {
      float ev[4];
      load_n<float, 4>(a.ema + at, ev);
#pragma unroll
      for (int e = 0; e < 4; ++e) ev[e] = ev[e] * ema_d + pv[e] * ema_o;
      store_n<float, 4>(a.ema + at, ev);
    }
    if (whole) {
      store_n<P, 4>(p + lane * 4, pv);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane * 4 + e < left) p[lane * 4 + e] = (P)pv[e];
    }
  }
  if (!a.last) return;
  // Every wave of this workgroup has read the counter (its products p1 and p2 are there); the last workgroup to say so moves it on and leaves the ticket
  // at 0.  No fence: nothing that this launch wrote is read by another workgroup, and the next launch sees it all.  (A device-wide fence here, which
  // writes back the caches of its die, made 85 us of a 16 us step.)
  asm volatile("" ::"v"(p1), "v"(p2));
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* ticket = (unsigned*)(a.counter + 3);
    if (__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
      a.counter[0] += 1.0;
      a.counter[1] = p1;
      a.counter[2] = p2;
      __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

__global__ __launch_bounds__(256) void moments_kernel(const int8_t* __restrict__ mc, const float* __restrict__ ms, const uint8_t* __restrict__ vc,
                                                      const float* __restrict__ vs, int64_t quads, float* __restrict__ m, float* __restrict__ v) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (int64_t)gridDim.x * 256) {
    const char4 c = ((const char4*)mc)[i];
    const uchar4 u = ((const uchar4*)vc)[i];
    const double a = (double)ms[i / (BLOCK / 4)] / (127.0 * 127.0), b = (double)vs[i / (BLOCK / 4)] / (255.0 * 255.0 * 255.0 * 255.0);
    const int ci[4] = {c.x, c.y, c.z, c.w}, ui[4] = {u.x, u.y, u.z, u.w};
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = (float)(a * (double)(ci[e] * abs(ci[e])));
      const unsigned u2 = (unsigned)(ui[e] * ui[e]);
      y[e] = (float)(b * (double)(u2 * u2));
    }
    store_n<float, 4>(m + i * 4, x);
    store_n<float, 4>(v + i * 4, y);
  }
}

template <typename P, typename G, int BITS>
void launch(const DptAdamWArgs& a, const Grads& g, hipStream_t st) {
  const int need = (a.n_blocks + WAVES - 1) / WAVES, blocks = need < 1 ? 1 : need < 2048 ? need : 2048;
  if (a.ema) hipLaunchKernelGGL((step_kernel<P, G, BITS, true>), dim3(blocks), dim3(64 * WAVES), 0, st, a, g);
  else hipLaunchKernelGGL((step_kernel<P, G, BITS, false>), dim3(blocks), dim3(64 * WAVES), 0, st, a, g);
}

template <typename P, typename G>
void by_bits(const DptAdamWArgs& a, const Grads& g, hipStream_t st) {
  if (a.state_bits == 8) launch<P, G, 8>(a, g, st); else launch<P, G, 32>(a, g, st);
}

}  // namespace dpta

extern "C" {

int dpt_adamw_step(const DptAdamWArgs* a, const void* const* grads, void* stream) {
  if (!a || a->n_tensors < 0 || a->n_tensors > DPT_ADAMW_MAX_TENSORS || (a->n_tensors && !grads) || a->n_blocks < 0 || a->block0 < 0) return DPT_E_BADARG;
  if ((a->state_bits != 8 && a->state_bits != 32) || !a->counter) return DPT_E_BADARG;
  if (a->type != DPT_F32 && a->type != DPT_BF16) return DPT_E_BADARG;
  if (a->grad_type != a->type && a->grad_type != DPT_F32) return DPT_E_UNSUPPORTED;
  if (a->n_blocks > 0 && (!a->block_tensor || !a->first_block || !a->numel || !a->param || !a->decay || !a->exp_avg || !a->exp_avg_sq ||
                          (a->type == DPT_BF16 && !a->master) || (a->state_bits == 8 && (!a->exp_avg_scale || !a->exp_avg_sq_scale)))) return DPT_E_BADARG;
  dpta::Grads g{};
  for (int i = 0; i < a->n_tensors; ++i) g.p[i] = grads[i];
  hipStream_t st = (hipStream_t)stream;
  if (a->type == DPT_F32) dpta::by_bits<float, float>(*a, g, st);
  else if (a->grad_type == DPT_BF16) dpta::by_bits<__bf16, __bf16>(*a, g, st);
  else dpta::by_bits<__bf16, float>(*a, g, st);
  return (int)hipGetLastError();
}

int dpt_adamw_moments(const void* exp_avg, const float* exp_avg_scale, const void* exp_avg_sq, const float* exp_avg_sq_scale, int32_t n_blocks,
                      float* m, float* v, void* stream) {
  if (n_blocks < 0 || (n_blocks > 0 && (!exp_avg || !exp_avg_scale || !exp_avg_sq || !exp_avg_sq_scale || !m || !v))) return DPT_E_BADARG;
  if (n_blocks == 0) return DPT_OK;
  const int64_t quads = (int64_t)n_blocks * (DPT_ADAMW_BLOCK / 4), need = (quads + 255) / 256;
  hipLaunchKernelGGL(dpta::moments_kernel, dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, (hipStream_t)stream, (const int8_t*)exp_avg, exp_avg_scale,
                     (const uint8_t*)exp_avg_sq, exp_avg_sq_scale, quads, m, v);
  return (int)hipGetLastError();
}

}  // extern "C"
