// dpt_attn_f32_128.hip - attention kernels for f32, head dimensions up to 128 (dpt_attn_impl.h)
#include "dpt_attn_impl.h"

namespace dptat {
hipError_t fwd_f32_128(const Dev& d, bool small, hipStream_t st) { return fwd_of<float, 128>(d, small, st); }
hipError_t bwd_f32_128(const Dev& d, bool small_rows, bool small_keys, hipStream_t st) { return bwd_of<float, 128>(d, small_rows, small_keys, st); }
}  // namespace dptat
