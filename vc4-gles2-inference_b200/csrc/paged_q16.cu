// paged_q16.cu -- the split attention kernels over q16 pages (see paged_split.inc).
#define VC4_PFMT vc4::P_Q16
#define VC4_PNAME launch_paged_split_q16
#include "paged_split.inc"
