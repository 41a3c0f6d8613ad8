// paged_f16.cu -- the split attention kernels over f16 pages (see paged_split.inc).
#define VC4_PFMT vc4::P_F16
#define VC4_PNAME launch_paged_split_f16
#include "paged_split.inc"
