// paged_q16.cu -- the attention kernels over q16 pages (see paged_split.inc, paged_chunk.inc).
#define VC4_PFMT vc4::P_Q16
#define VC4_PNAME launch_paged_split_q16
#define VC4_CNAME launch_paged_chunk_q16
#include "paged_split.inc"
#include "paged_chunk.inc"
