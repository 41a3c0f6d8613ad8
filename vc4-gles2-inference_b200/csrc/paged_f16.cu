// paged_f16.cu -- the attention kernels over f16 pages (see paged_split.inc, paged_chunk.inc).
#define VC4_PFMT vc4::P_F16
#define VC4_PNAME launch_paged_split_f16
#define VC4_CNAME launch_paged_chunk_f16
#include "paged_split.inc"
#include "paged_chunk.inc"
