// paged_q8.cu -- the split attention kernels over q8 pages (see paged_split.inc).
#define VC4_PFMT vc4::P_Q8
#define VC4_PNAME launch_paged_split_q8
#include "paged_split.inc"
