// dpt_attn_bf16.hip - attention kernels for bf16 (dpt_attn_impl.h)
#include "dpt_attn_impl.h"

namespace dptat {
hipError_t fwd_bf16(const Dev& d, bool small, hipStream_t st) { return fwd_by_dim<__bf16>(d, small, st); }
hipError_t bwd_bf16(const Dev& d, bool small_rows, bool small_keys, hipStream_t st) { return bwd_by_dim<__bf16>(d, small_rows, small_keys, st); }
}  // namespace dptat
