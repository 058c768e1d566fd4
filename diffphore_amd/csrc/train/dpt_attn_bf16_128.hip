// dpt_attn_bf16_128.hip - attention kernels for bf16, head dimensions up to 128 (dpt_attn_impl.h)
#include "dpt_attn_impl.h"

namespace dptat {
hipError_t fwd_bf16_128(const Dev& d, bool small, hipStream_t st) { return fwd_of<__bf16, 128>(d, small, st); }
hipError_t bwd_bf16_128(const Dev& d, bool small_rows, bool small_keys, hipStream_t st) { return bwd_of<__bf16, 128>(d, small_rows, small_keys, st); }
}  // namespace dptat
