// dpt_attn.hip - C entry points of the attention operators: checks, workspace, choice of the row blocks (kernels: dpt_attn_impl.h).
#include "dpt_attn.h"

namespace dptat {

constexpr int CUS = 256;
constexpr size_t ALIGN = 256;
constexpr int32_t MOST_ROWS = DPT_ATTN_MAX_ROWS;
size_t up(size_t n) { return (n + ALIGN - 1) / ALIGN * ALIGN; }

int check(const DptAttnArgs* a) {
  if (!a || (a->type != DPT_F32 && a->type != DPT_BF16)) return DPT_E_BADARG;
  if (a->B < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->dim < 1) return DPT_E_BADARG;
  if (!(a->scale >= 0x1p-126f && a->scale <= 0x1p126f)) return DPT_E_BADARG;             // scale log2 e has to be a normal number
  if (a->n_q < 0 || a->n_k < 0 || a->max_nq < 0 || a->max_nk < 0 || a->max_nq > a->n_q || a->max_nk > a->n_k || a->n_pairs < 0 || a->splits < 0) return DPT_E_BADARG;
  if (a->dim > 128 || a->n_q > MOST_ROWS || a->n_k > MOST_ROWS) return DPT_E_TOOLARGE;   // the last block's row numbers, past the end, still fit
  const int64_t group = a->heads / a->kv_heads, rows = (int64_t)a->max_nq * group;
  // 32-bit row numbers, and their division by a multiplication; 32-bit workgroup numbers, over all parts of a launch (32 rows or keys each at the least; ranges()
  // splits few workgroups only)
  const int64_t most = ((int64_t)1 << 31) / (a->splits ? 64 : 1);
  if (rows > MOST_ROWS || rows * group >= (int64_t)1 << 31) return DPT_E_TOOLARGE;
  const int64_t lists = (int64_t)a->B * a->kv_heads, longest = (rows > a->max_nk ? rows : a->max_nk) / 32 + 1;
  if (lists >= most || longest * lists >= most) return DPT_E_TOOLARGE;
  return DPT_OK;
}

// Row blocks of 32 (one wave) where the largest complex has few rows: a block of 128 would leave waves without rows; otherwise 128.
bool small_rows(const DptAttnArgs* a) { return (int64_t)a->max_nq * (a->heads / a->kv_heads) <= 64; }
bool small_keys(const DptAttnArgs* a) { return a->max_nk <= 64; }

// Ranges of an axis of `length` that `blocks` workgroups walk along, each in turn: where they do not fill the chip evenly the axis is split and the ranges'
// results are joined afterwards.  `room`: workgroups that the chip holds at once; a range is no shorter than `least`.  The time is taken as the generations
// of workgroups times the length of a range, plus a join that costs a part of it; whichever number of ranges makes that least.
// (Backward of one fp32 complex of 783 rows and 674 keys, 4 key heads: 92 us against 418 unsplit.)
int ranges(int64_t blocks, int64_t length, int64_t room, int64_t least) {
  if (blocks == 0) return 1;
  const int64_t most = length / least < 64 ? length / least : 64;
  int best = 1;
  double cost = (double)((blocks + room - 1) / room);
  for (int s = 2; s <= most && blocks * s <= 4 * room; ++s) {
    const double c = (double)((blocks * s + room - 1) / room) / s + 0.05 + 0.012 * s;
    if (c < cost) { cost = c; best = s; }
  }
  return best;
}

struct Splits { int fwd, q, k; };
Splits splits_of(const DptAttnArgs* a) {
  const int64_t rows = (int64_t)a->max_nq * (a->heads / a->kv_heads), bm = small_rows(a) ? 32 : 128, bk = small_keys(a) ? 32 : 128;
  // workgroups that have work: by the largest complex, or by the total with half a block lost per complex, whichever is less (ragged batches)
  auto blocks = [&](int64_t largest, int64_t total, int64_t block) {
    const int64_t x = (largest + block - 1) / block * a->B, y = (total + a->B * (block / 2) + block - 1) / block;
    return (x < y ? x : y) * a->kv_heads;
  };
  const int64_t row_blocks = blocks(rows, (int64_t)a->n_q * (a->heads / a->kv_heads), bm), key_blocks = blocks(a->max_nk, a->n_k, bk);
  if (a->splits) {
    const int s = a->splits > 64 ? 64 : a->splits;
    return {s, s, s};
  }
  Splits s;
  // room is taken as four workgroups of one wave to a CU, or one of four waves (two, where a kernel is built for that, share it, but each is then the slower).  Of the
  // one-wave ones LDS lets in ten with heads of up to 32 dimensions, four or five of 64, two of 128: four is a middle, not the limit of each
  s.fwd = a->max_nk < 1024 ? 1 : ranges(row_blocks, a->max_nk, small_rows(a) ? 4 * CUS : CUS, 128);   // (shorter walks take less than a join)
  s.q = ranges(row_blocks, a->max_nk, small_rows(a) ? 4 * CUS : CUS, 128);
  s.k = ranges(key_blocks, rows, small_keys(a) ? 4 * CUS : CUS, 128);
  return s;
}

struct Ws { size_t delta, part_ml, total; };
Ws layout(const DptAttnArgs* a, bool backward, const Splits& s) {
  Ws w{};
  const size_t plane = (size_t)a->heads * a->n_q * sizeof(float);
  if (backward) {
    w.delta = up(plane);                 // one of three planes, the parts of split gradients behind them
    const size_t q = s.q > 1 ? plane * a->dim * s.q : 0, k = s.k > 1 ? (size_t)a->n_k * a->kv_heads * a->dim * sizeof(float) * 2 * s.k : 0;
    w.total = 3 * w.delta + up(q > k ? q : k);
  } else if (s.fwd > 1) {
    w.part_ml = up(plane * a->dim * s.fwd);
    w.total = w.part_ml + up(2 * plane * s.fwd);
  }
  return w;
}

// 16-byte reads of rows of q, k, v, dout and out, 16- or 8-byte stores: the row length, every stride and every address have to allow them
bool vec(const DptAttnArgs* a, bool backward) {
  const int n = a->type == DPT_F32 ? 4 : 8;
  // (strides below 2^24: 64 rows and as many heads apart still fit the 32-bit offset that the kernels use)
  auto ok = [&](const void* p, int64_t r, int64_t h) { return (uintptr_t)p % 16 == 0 && r % n == 0 && h % n == 0 && r < 1 << 24 && h < 1 << 24; };
  bool v = a->dim % n == 0 && ok(a->q, a->q_row, a->q_head) && ok(a->k, a->k_row, a->k_head) && ok(a->v, a->v_row, a->v_head) && ok(a->out, 0, 0);
  if (backward) v = v && ok(a->dout, a->dout_row, a->dout_head) && ok(a->dq, 0, 0) && ok(a->dk, 0, 0) && ok(a->dv, 0, 0);
  return v;
}

Dev dev(const DptAttnArgs* a, bool backward) {
  Dev d{};
  d.a = *a;
  d.group = a->heads / a->kv_heads;
  d.magic = d.group > 1 ? (uint32_t)((((uint64_t)1 << 32) + d.group - 1) / d.group) : 0;
  d.vec = vec(a, backward);
  d.splits = d.splits_q = d.splits_k = 1;
  return d;
}

// kernels by the head dimension, padded to 32, 64 or 128
template <typename F>
F pick(int dim, F f32, F f64, F f128) { return dim <= 32 ? f32 : dim <= 64 ? f64 : f128; }

bool strides_bad(const DptAttnArgs* a) {
  return a->q_row < 0 || a->q_head < 0 || a->k_row < 0 || a->k_head < 0 || a->v_row < 0 || a->v_head < 0 || a->bias_head < 0 || a->bias_pair < 0;
}

}  // namespace dptat

extern "C" {

int dpt_abi_version(void) { return DPT_ABI_VERSION; }

int dpt_struct_sizes(int32_t* out, int32_t n) {
  const int32_t s[2] = {(int32_t)sizeof(DptAttnArgs), (int32_t)sizeof(DptAdamWArgs)};
  for (int i = 0; out && i < n && i < 2; ++i) out[i] = s[i];
  return 2;
}

size_t dpt_attn_ws_bytes(const DptAttnArgs* a, int32_t backward) {
  if (dptat::check(a) != DPT_OK) return 0;
  return dptat::layout(a, backward != 0, dptat::splits_of(a)).total;
}

int dpt_attn_fwd(const DptAttnArgs* a, void* stream) {
  const int rc = dptat::check(a);
  if (rc) return rc;
  if (a->B == 0 || a->n_q == 0) return DPT_OK;
  if (!a->q || !a->out || !a->stats || !a->q_ptr || !a->k_ptr || !a->pair_ptr || !a->order || (a->n_k > 0 && (!a->k || !a->v)) || dptat::strides_bad(a)) return DPT_E_BADARG;
  dptat::Dev d = dptat::dev(a, false);
  const dptat::Splits s = dptat::splits_of(a);
  d.splits = s.fwd;
  const dptat::Ws w = dptat::layout(a, false, s);
  if (w.total && (!a->ws || a->ws_bytes < w.total || (uintptr_t)a->ws % 16)) return DPT_E_BADARG;
  d.part_o = (float*)a->ws;
  d.part_ml = (float*)((char*)a->ws + w.part_ml);
  const bool small = dptat::small_rows(a);
  const int bm = small ? 32 : 128;
  d.tiles = (int)(((int64_t)a->max_nq * d.group + bm - 1) / bm);
  using namespace dptat;
  return (int)(a->type == DPT_F32 ? pick(a->dim, fwd_f32_32, fwd_f32_64, fwd_f32_128) : pick(a->dim, fwd_bf16_32, fwd_bf16_64, fwd_bf16_128))(d, small, (hipStream_t)stream);
}

int dpt_attn_bwd(const DptAttnArgs* a, void* stream) {
  const int rc = dptat::check(a);
  if (rc) return rc;
  if (a->B == 0 || (a->n_q == 0 && a->n_k == 0)) return DPT_OK;
  if (!a->q_ptr || !a->k_ptr || !a->pair_ptr || !a->order || dptat::strides_bad(a) || a->dout_row < 0 || a->dout_head < 0) return DPT_E_BADARG;
  if (a->n_q > 0 && (!a->q || !a->out || !a->stats || !a->dout || !a->dq)) return DPT_E_BADARG;
  if (a->n_k > 0 && (!a->k || !a->v || !a->dk || !a->dv)) return DPT_E_BADARG;
  const dptat::Splits s = dptat::splits_of(a);
  const dptat::Ws w = dptat::layout(a, true, s);
  if (w.total && (!a->ws || a->ws_bytes < w.total || (uintptr_t)a->ws % 16)) return DPT_E_BADARG;
  dptat::Dev d = dptat::dev(a, true);
  d.delta = (float*)a->ws;
  d.fac0 = (float*)((char*)a->ws + w.delta);
  d.fac1 = (float*)((char*)a->ws + 2 * w.delta);
  d.part_g = (float*)((char*)a->ws + 3 * w.delta);
  d.splits_q = s.q;
  d.splits_k = s.k;
  const bool sr = dptat::small_rows(a), sk = dptat::small_keys(a);
  using namespace dptat;
  return (int)(a->type == DPT_F32 ? pick(a->dim, bwd_f32_32, bwd_f32_64, bwd_f32_128) : pick(a->dim, bwd_bf16_32, bwd_bf16_64, bwd_bf16_128))(d, sr, sk, (hipStream_t)stream);
}

}  // extern "C"
