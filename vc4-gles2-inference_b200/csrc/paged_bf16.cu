// paged_bf16.cu -- the attention kernels over bf16 pages (see paged_split.inc, paged_chunk.inc).
#define VC4_PFMT vc4::P_BF16
#define VC4_PNAME launch_paged_split_bf16
#define VC4_CNAME launch_paged_chunk_bf16
#include "paged_split.inc"
#include "paged_chunk.inc"
