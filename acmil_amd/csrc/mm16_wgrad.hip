// mm16_wgrad.hip -- dW = dz^T x (both operands K strided): instances of mm16_kernel.h
#include "mm16_kernel.h"

int mm_launch_wgrad(const MmArgs& a, bool bf, int epi, int cfg, hipStream_t st) {
    return epi == MM_PART ? mm_go_any<MM_KS, MM_KS, MM_PART, false>(a, bf, cfg, st) : mm_go_any<MM_KS, MM_KS, MM_ACT, false>(a, bf, cfg, st);
}
