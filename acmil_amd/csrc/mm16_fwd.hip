// mm16_fwd.hip -- y = x W^T and the gate / up pair (both operands K contiguous): instances of mm16_kernel.h
#include "mm16_kernel.h"

int mm_launch_fwd(const MmArgs& a, bool bf, int epi, bool dual, int cfg, hipStream_t st) {
    if (dual) return epi == MM_PART ? mm_go_any<MM_KC, MM_KC, MM_PART, true>(a, bf, cfg, st) : mm_go_any<MM_KC, MM_KC, MM_GATE, true>(a, bf, cfg, st);
    return epi == MM_PART ? mm_go_any<MM_KC, MM_KC, MM_PART, false>(a, bf, cfg, st) : mm_go_any<MM_KC, MM_KC, MM_ACT, false>(a, bf, cfg, st);
}
