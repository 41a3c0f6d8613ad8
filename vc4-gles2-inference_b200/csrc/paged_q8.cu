// paged_q8.cu -- the attention kernels over q8 pages (see paged_split.inc, paged_chunk.inc).
#define VC4_PFMT vc4::P_Q8
#define VC4_PNAME launch_paged_split_q8
#define VC4_CNAME launch_paged_chunk_q8
#include "paged_split.inc"
#include "paged_chunk.inc"
