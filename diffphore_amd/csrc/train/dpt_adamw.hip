// dpt_adamw.hip - one AdamW step over a list of tensors, states in 32 or 8 bits, with the running average of the parameters.
//
// Bound by HBM: every value is read once and written once.  A wave takes one 256-element block (4 elements per lane: one 16-byte load per fp32
// array); the block's tensor comes from a table, the gradients' addresses come with the launch.  All of a step is ONE launch per 400 tensors.
// Measured: 120 M bf16 parameters with masters and 8-bit states 550 us (3.5 TB/s), the score model's 2.2 M fp32 parameters in 228 tensors with averages 27 us.
//
// Step number: b1^t and b2^t live on the device (so a captured graph counts on), every workgroup reads them, and the workgroup that is the last to
// have read them moves them on.
//
// 8-bit states: m' and v' are formed in 64 bits from the decoded values, the parameter's update uses them unrounded, and the stored codes are the
// nearest ones.  "Nearest" is decided exactly: a 32-bit root gives the code's position, and where some position of the block lies within its own error of a
// border between two codes, the block's values are compared with the borders in 64 bits, (c - 1/2)^2 resp. ^4 times the scale (exact, or within 2^-53) -
// so a code does not depend on the rounding of a root.  This form is bound by instructions as much as by memory (vector units 72 % busy): everything that can be is 32 bits.
#include "dpt_dev.h"

#include <type_traits>

namespace dpta {
using namespace dpt;

constexpr int BLOCK = DPT_ADAMW_BLOCK, WAVES = 4;

struct Grads { const void* p[DPT_ADAMW_MAX_TENSORS]; };

// maximum over the wave of values >= 0, without LDS: shifts inside rows of 16 lanes, then across rows; lane 63 has it in the end
__device__ __forceinline__ float wave_max(float x) {
  auto step = [&](auto ctrl) __attribute__((always_inline)) {
    const int b = __builtin_bit_cast(int, x);
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  step(std::integral_constant<int, 0x111>{});   // row_shr 1, 2, 4, 8
  step(std::integral_constant<int, 0x112>{});
  step(std::integral_constant<int, 0x114>{});
  step(std::integral_constant<int, 0x118>{});
  step(std::integral_constant<int, 0x142>{});   // row_bcast 15, 31
  step(std::integral_constant<int, 0x143>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// Position t = TOP (x / scale)^(1/POW) of a value on its curve.  x (rounded from 64 bits) and its product with 1 / scale are good to 2^-24, 1 / scale and a root
// to an ulp, so |dt| < TOP 2^-24 (4 / POW + 3) < 8e-5 on both curves (NEAR); below TINY the 32-bit values may have lost bits to underflow, and
// above VAST 1 / scale is (the hardware's reciprocal of more than 2^126 is 0): such blocks take the 64-bit codes.
constexpr float NEAR = 1e-4f, TINY = 1e-30f, VAST = 0x1p125f;
template <int TOP, int POW>
__device__ __forceinline__ float position(float x, float inv) {
  float t = __builtin_amdgcn_sqrtf(x * inv);
  if constexpr (POW == 4) t = __builtin_amdgcn_sqrtf(t);
  return t * (float)TOP;
}
__device__ __forceinline__ bool near_border(float t) { return fabsf(__builtin_amdgcn_fractf(t + 0.5f) - 0.5f) > 0.5f - NEAR; }

// Nearest code by comparison with the borders; for values whose root may be off, from a 64-bit root
template <int TOP, int POW>
__device__ __forceinline__ int exact_code(double x, double scale) {
  constexpr double T = POW == 2 ? (double)TOP * TOP : (double)TOP * TOP * TOP * TOP;
  double t = sqrt(x / scale);
  if constexpr (POW == 4) t = sqrt(t);
  const int near = (int)(t * TOP + 0.5);           // right, or one too high or too low by a rounding
  const int c = near > TOP ? TOP : near;
  auto below = [&](int k) { const double h = (double)k - 0.5, h2 = h * h; return x * T < scale * (POW == 2 ? h2 : h2 * h2); };
  return c > 0 && below(c) ? c - 1 : c < TOP && !below(c + 1) ? c + 1 : c;
}

// a block's values on their way
template <typename P, typename G>
struct Values {
  typedef __attribute__((ext_vector_type(4))) G g4;
  DptAdamWBlock b;
  const G* g;                    // nullptr: no gradient, the tensor and its state stay as they are
  bool whole;                    // 256 elements at aligned addresses
  g4 gv;
  f4 pv, mv, vv, ev;
  int mc, vc;                    // four codes each
  float ms, vs;
};

// (six waves per SIMD: 540 us for the 120 M parameters with 8-bit states against 555 with the registers that the compiler takes for four.  It is a trade: at 80 registers
// the 8-bit instances spill 13 to 25 of a lane's, among them values of the block that is on its way, which are waited for when they are spilled)
template <typename P, typename G, int BITS, bool EMA>
__global__ __launch_bounds__(64 * WAVES, 6) void step_kernel(DptAdamWArgs a, Grads grads) {
  // the step's factors, in 64 bits
  const double p1 = a.counter[1] * a.beta1, p2 = a.counter[2] * a.beta2;
  const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
  const float b1 = (float)a.beta1, omb1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, omb2 = (float)(1.0 - a.beta2);
  const float lr1 = (float)(lr / (1.0 - p1)), ic2 = (float)(1.0 / (1.0 - p2)), eps = (float)a.eps;
  const float ema_d = (float)a.ema_decay, ema_o = (float)(1.0 - a.ema_decay), gs = a.grad_scale ? *a.grad_scale : 1.f;
  const double gsd = (double)gs, k1 = 1.0 - a.beta1, k2 = 1.0 - a.beta2;
  const bool scaled = a.grad_scale != nullptr;
  const int lane = threadIdx.x & 63;
  // 8 bits: what the codes stand for, as shares of the scale
  __shared__ double m_of[BITS == 8 ? 256 : 1], v_of[BITS == 8 ? 256 : 1];
  if constexpr (BITS == 8) {
    static_assert(64 * WAVES == 256, "a code per lane");
    const int c = (int)(int8_t)threadIdx.x;
    const double r = (double)threadIdx.x / 255.0, r2 = r * r;
    m_of[threadIdx.x] = (double)(c * abs(c)) / (127.0 * 127.0);
    v_of[threadIdx.x] = r2 * r2;
    __syncthreads();
  }
  typedef const __attribute__((address_space(4))) DptAdamWBlock* Rec;      // constant memory: a wave's record is one scalar load
  auto record = [&](int i) __attribute__((always_inline)) {
    const Rec r = (Rec)(unsigned long long)(a.blocks + a.block0 + min(i, a.n_blocks - 1));
    return DptAdamWBlock{r->param, r->tensor, r->index, r->left, r->decay, {0, 0}};
  };
  auto fetch = [&](int i, const DptAdamWBlock& b) __attribute__((always_inline)) {
    Values<P, G> x;
    x.b = b;
    const G* g = (const G*)grads.p[b.tensor - a.tensor0];
    x.g = g && i < a.n_blocks ? g + (int64_t)b.index * BLOCK : nullptr;
    x.whole = b.left == BLOCK && b.param % (4 * sizeof(P)) == 0 && (uintptr_t)g % (4 * sizeof(G)) == 0;
    if (!x.g) return x;
    const P* p = (const P*)b.param;
    const int64_t blk = a.block0 + i, at = blk * BLOCK + lane * 4;
    if (x.whole) {
      x.gv = *(const typename Values<P, G>::g4*)(x.g + lane * 4);
      if constexpr (sizeof(P) == 4) x.pv = *(const f4*)(p + lane * 4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = lane * 4 + e < b.left;
        x.gv[e] = in ? x.g[lane * 4 + e] : (G)0.f;
        if constexpr (sizeof(P) == 4) x.pv[e] = in ? p[lane * 4 + e] : 0.f;
      }
    }
    if constexpr (sizeof(P) == 2) x.pv = *(const f4*)(a.master + at);
    if constexpr (EMA) x.ev = *(const f4*)(a.ema + at);
    if constexpr (BITS == 32) {
      x.mv = *(const f4*)((const float*)a.exp_avg + at);
      x.vv = *(const f4*)((const float*)a.exp_avg_sq + at);
    } else {
      x.mc = *(const int*)((const int8_t*)a.exp_avg + at);
      x.vc = *(const int*)((const uint8_t*)a.exp_avg_sq + at);
      x.ms = a.exp_avg_scale[blk];
      x.vs = a.exp_avg_sq_scale[blk];
    }
    return x;
  };
  // the next block's values are on their way while a block is worked on, and the record of the one after it: otherwise every turn would wait for a
  // record and then for the values that it points to
  const int stride = gridDim.x * WAVES;
  int i = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  Values<P, G> x;
  DptAdamWBlock ahead;
  if (a.n_blocks > 0) {                                      // (a list of empty tensors has no record to read)
    x = fetch(i, record(i));
    ahead = record(i + stride);
  }
  for (; i < a.n_blocks; i += stride) {
    const Values<P, G> next = fetch(i + stride, ahead);
    ahead = record(i + 2 * stride);
    if (x.g) {
      const int64_t blk = a.block0 + i, at = blk * BLOCK + lane * 4;
      const float shrink = (float)(1.0 - lr * a.weight_decay * (double)x.b.decay);
      P* p = (P*)x.b.param;
      if constexpr (BITS == 32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = (float)x.gv[e] * gs;
          x.mv[e] = x.mv[e] * b1 + g * omb1;
          x.vv[e] = x.vv[e] * b2 + g * omb2 * g;             // (in this order g^2, which may pass the 32-bit numbers where v does not, is never formed)
        }
      } else {
        const double ma = (double)x.ms, va = (double)x.vs;
        double m[4], v[4];
        float mm = 0.f, vm = 0.f, bad = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // Each operation rounded by itself, in the order of the formula.  The new scale is the largest of these rounded to 32 bits, and with betas of one
          // decimal and bf16 gradients about one block in 130 has its largest exactly between two 32-bit numbers: a fused multiplication decides such a tie by
          // its own last bit, and the formula evaluated in 64 bits elsewhere would get another scale.
#pragma clang fp contract(off)
          const double g = scaled ? (double)x.gv[e] * gsd : (double)x.gv[e];
          const double m_old = m_of[(unsigned)(x.mc >> (8 * e)) & 255u] * ma, v_old = v_of[(unsigned)(x.vc >> (8 * e)) & 255u] * va;
          m[e] = m_old * a.beta1 + g * k1;
          v[e] = v_old * a.beta2 + g * g * k2;
          x.mv[e] = (float)m[e];
          x.vv[e] = (float)v[e];
          bad = fmaf(x.mv[e], 0.f, fmaf(x.vv[e], 0.f, bad));             // NaN as soon as one is not finite
          mm = fmaxf(mm, fabsf(x.mv[e]));                                // rounding keeps the order: the rounded maximum is the maximum rounded
          vm = fmaxf(vm, x.vv[e]);
        }
        float msc = wave_max(mm), vsc = wave_max(vm);
        unsigned mc = 0, vc = 0;
        if (__any(bad != 0.f)) {
          msc = vsc = __builtin_nanf("");
        } else {
          const float mi = __builtin_amdgcn_rcpf(msc), vi = __builtin_amdgcn_rcpf(vsc);       // not used below TINY and above VAST
          int cm[4], cv[4];
          int near = (msc < TINY) | (vsc < TINY) | (msc > VAST) | (vsc > VAST);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float tm = position<127, 2>(fabsf(x.mv[e]), mi), tv = position<255, 4>(x.vv[e], vi);
            near |= (int)near_border(tm) | (int)near_border(tv);
            cm[e] = min((int)(tm + 0.5f), 127);
            cv[e] = min((int)(tv + 0.5f), 255);
          }
          if (__any(near)) {
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
              const double me = e == 0 ? m[0] : e == 1 ? m[1] : e == 2 ? m[2] : m[3], ve = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
              const int c = msc > 0.f ? exact_code<127, 2>(fabs(me), (double)msc) : 0, w = vsc > 0.f ? exact_code<255, 4>(ve, (double)vsc) : 0;
#pragma unroll
              for (int f = 0; f < 4; ++f) { cm[f] = f == e ? c : cm[f]; cv[f] = f == e ? w : cv[f]; }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            cm[e] = __builtin_bit_cast(int64_t, m[e]) < 0 ? -cm[e] : cm[e];
            cv[e] = vsc > 0.f && v[e] > 0.0 ? max(cv[e], 1) : cv[e];
            mc |= (unsigned)(uint8_t)cm[e] << (8 * e);
            vc |= (unsigned)cv[e] << (8 * e);
          }
        }
        x.mc = (int)mc; x.vc = (int)vc; x.ms = msc; x.vs = vsc;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // root and quotient to an ulp each, of an update that is itself a small part of the parameter; moments next to underflow are rooted 2^64 times as large,
        // those next to overflow (v / (1 - b2^t) may pass it where v does not) 2^64 times as small
        const float w = x.vv[e] * ic2;
        const bool tiny = w < 0x1p-96f, vast = w > 0x1p96f;
        const float root = __builtin_amdgcn_sqrtf(tiny ? w * 0x1p64f : vast ? x.vv[e] * 0x1p-64f * ic2 : w), den = root * (tiny ? 0x1p-32f : vast ? 0x1p32f : 1.f) + eps;
        const float q = x.mv[e] * __builtin_amdgcn_rcpf(den);
        x.pv[e] = fmaf(-lr1, q, x.pv[e] * shrink);
      }
      if constexpr (EMA) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x.ev[e] = x.ev[e] * ema_d + x.pv[e] * ema_o;
      }
      if (x.b.left < BLOCK) {                                // what pads a tensor's last block stays 0 whatever the factors are (eps 0: 0 / 0; an infinite scale)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (lane * 4 + e < x.b.left) continue;
          x.pv[e] = 0.f;
          if constexpr (EMA) x.ev[e] = 0.f;
          if constexpr (BITS == 32) x.mv[e] = x.vv[e] = 0.f;
        }
      }
      // the next block's values are waited for here, before the stores: loads and stores share a counter, and a wait behind the stores would be one for them too
      __builtin_amdgcn_s_waitcnt(0x0f70);                    // vmcnt(0)
      if constexpr (BITS == 32) {
        *(f4*)((float*)a.exp_avg + at) = x.mv;
        *(f4*)((float*)a.exp_avg_sq + at) = x.vv;
      } else {
        *(int*)((int8_t*)a.exp_avg + at) = x.mc;
        *(int*)((uint8_t*)a.exp_avg_sq + at) = x.vc;
        if (lane == 0) { a.exp_avg_scale[blk] = x.ms; a.exp_avg_sq_scale[blk] = x.vs; }
      }
      if constexpr (sizeof(P) == 2) *(f4*)(a.master + at) = x.pv;
      if constexpr (EMA) *(f4*)(a.ema + at) = x.ev;
      float pv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pv[e] = x.pv[e];
      if (x.whole) {
        store_n<P, 4>(p + lane * 4, pv);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lane * 4 + e < x.b.left) p[lane * 4 + e] = (P)pv[e];
      }
    }
    x = next;
  }
  if (!a.last) return;
  // Every wave of this workgroup has read the counter (its products p1 and p2 are there); the last workgroup to say so moves it on and leaves the ticket
  // at 0.  No fence: nothing that this launch wrote is read by another workgroup, and the next launch sees it all.  (A device-wide fence here, which
  // writes back the caches of its die, made the score model's step 85 us.)
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
  // at most one generation of resident workgroups: each of them pays the counter's atomic once
  constexpr int MOST = 1536;
  const int need = (a.n_blocks + WAVES - 1) / WAVES, blocks = need < 1 ? 1 : need < MOST ? need : MOST;
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
  if (a->n_blocks > 0 && (!a->blocks || !a->exp_avg || !a->exp_avg_sq ||
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
