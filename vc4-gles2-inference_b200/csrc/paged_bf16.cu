// paged_bf16.cu -- the split attention kernels over bf16 pages (see paged_split.inc).
#define VC4_PFMT vc4::P_BF16
#define VC4_PNAME launch_paged_split_bf16
#include "paged_split.inc"
