// dpt_attn_f32.hip - attention kernels for f32 (dpt_attn_impl.h)
#include "dpt_attn_impl.h"

namespace dptat {
hipError_t fwd_f32(const Dev& d, bool small, hipStream_t st) { return fwd_by_dim<float>(d, small, st); }
hipError_t bwd_f32(const Dev& d, bool small_rows, bool small_keys, hipStream_t st) { return bwd_by_dim<float>(d, small_rows, small_keys, st); }
}  // namespace dptat
