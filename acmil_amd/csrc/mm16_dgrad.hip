// mm16_dgrad.hip -- dx = dz W (W read K strided) and dh = dy Wd with the gate's backward: instances of mm16_kernel.h
#include "mm16_kernel.h"

int mm_launch_dgrad(const MmArgs& a, bool bf, int epi, int cfg, hipStream_t st) {
    if (epi == MM_PART) return mm_go_any<MM_KS, MM_KC, MM_PART, false>(a, bf, cfg, st);
    if (epi == MM_GATE_BWD) return mm_go_any<MM_KS, MM_KC, MM_GATE_BWD, false>(a, bf, cfg, st);
    return mm_go_any<MM_KS, MM_KC, MM_ACT, false>(a, bf, cfg, st);
}
