// The grouped product of 8-bit codes with tiles of 128 x 128, two workgroups of 4 waves per compute unit (int8_gemm.hip says when).
#define MOE_I8_TILE 128
#include "int8_gemm_kernel.h"

int moe_launch_i8_gemm_small(const MoeI8Gemm& p, int64_t R, hipStream_t stream) { return launch_epilogue(p, R, stream); }
