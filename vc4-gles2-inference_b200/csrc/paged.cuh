// paged.cuh -- what the paged-cache kernels share: the launch arguments, where a
// row of a sequence lies, the cached formats as tensor-core operands.
//
// A pool is [page][K, V][kv head][page_len][head_dim] values, so the rows of one
// head inside a page are one contiguous piece, whatever the format.
#pragma once
#include "kernels.cuh"
#include "../../include/vc4b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace vc4 {

// Formats as template arguments.
enum PFmt : int { P_Q8 = 0, P_Q16 = 1, P_BF16 = 2, P_F16 = 3 };

// The pool and the batch, as every paged kernel gets them.
struct PagedArgs {
    uint8_t* data;
    int pages, page_shift, kv_heads, head_dim;
    int seqs, tokens, max_new, table_stride;
    const int *cu, *len, *table;
    int* status;
};

struct PagedAttnArgs {
    PagedArgs p;
    const void* q;
    void* out;
    long long q_stride, out_stride;
    int q_type, out_type, heads, group;
    int fmt;                 // PFmt of the pages
    int row_tiles, splits;   // grid: ((sequence * kv_heads + head) * row_tiles + tile) * splits + split
    float scale2;            // score scale x log2 e x the K grid
    float vscale;            // the V grid
    float* part;             // many-row kernel: [splits][tokens*heads][head_dim] unnormalised sums
    float2* ml;              // [splits][tokens*heads] running maximum (of the unscaled score) and sum
};

// The split kernels of one format (paged_*.cu); wr: 16-row tiles per block (1, 2 or 4).
bool launch_paged_split_q8(const PagedAttnArgs& a, int wr, cudaStream_t st);
bool launch_paged_split_q16(const PagedAttnArgs& a, int wr, cudaStream_t st);
bool launch_paged_split_bf16(const PagedAttnArgs& a, int wr, cudaStream_t st);
bool launch_paged_split_f16(const PagedAttnArgs& a, int wr, cudaStream_t st);
// The many-row kernels; false where no TMA descriptor of the pool can be made.
bool launch_paged_chunk_q8(const PagedAttnArgs& a, cudaStream_t st);
bool launch_paged_chunk_q16(const PagedAttnArgs& a, cudaStream_t st);
bool launch_paged_chunk_bf16(const PagedAttnArgs& a, cudaStream_t st);
bool launch_paged_chunk_f16(const PagedAttnArgs& a, cudaStream_t st);

namespace {

constexpr int kPagedMaxSplits = 64;    // of the many-row kernel
constexpr int kPagedChunkRows = 256;   // rows of its blocks
constexpr int kPagedMaxCluster = 8;    // splits of the few-row kernel: blocks of a cluster

__device__ __forceinline__ void paged_flag(int* status, int code) {
    if (status) atomicMax(status, code);
}

// The sequence that holds row `r`: the last s with cu[s] <= r, by a 32-way
// search of one warp (every lane returns it).  Any contents of cu give an s in
// [0, seqs).
__device__ __forceinline__ int paged_find(const int* cu, int seqs, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = seqs;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool le = lane * step < n && cu[at] <= r;
        // the candidates are ordered: the last lane that holds
        const unsigned m = __ballot_sync(0xffffffffu, le);
        const int last = m ? 31 - __clz(m) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether one of the eight 16-bit floats is infinite or NaN.
template <int FMT>
__device__ __forceinline__ bool any_wild(const uint4 v) {
    constexpr unsigned top = FMT == P_BF16 ? 0x7F807F80u : 0x7C007C00u;   // all exponent bits
    auto wild = [](unsigned w) { return (w & (top & 0xFFFFu)) == (top & 0xFFFFu) || (w & (top & 0xFFFF0000u)) == (top & 0xFFFF0000u); };
    return wild(v.x) || wild(v.y) || wild(v.z) || wild(v.w);
}
// The same values with 0 for those.
template <int FMT>
__device__ __forceinline__ uint4 tamed(uint4 v) {
    constexpr unsigned top = FMT == P_BF16 ? 0x7F807F80u : 0x7C007C00u;
    auto tame = [](unsigned w) {
        if ((w & (top & 0xFFFFu)) == (top & 0xFFFFu)) w &= 0xFFFF0000u;
        if ((w & (top & 0xFFFF0000u)) == (top & 0xFFFF0000u)) w &= 0xFFFFu;
        return w;
    };
    return make_uint4(tame(v.x), tame(v.y), tame(v.z), tame(v.w));
}
// What the taken-out infinite and NaN V add to two values from column d of row r of sequence
// s (rows of a block that starts at row r0): those of the positions the row sees and some
// row of its block does not, read again from their pages; 0 where there are none.
template <int FMT>
__device__ __forceinline__ float2 wild_sum(const PagedArgs& p, int s, int kvh, int group, int r0, int r, int d) {
    const int n = p.cu[s + 1] - p.cu[s], len = max(p.len[s], 0);
    const int end = min(min(len, p.table_stride << p.page_shift), len - n + r / group + 1);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (int pos = max(0, len - n + r0 / group + 1); pos < end; ++pos) {
        const int id = p.table[(size_t)s * p.table_stride + (pos >> p.page_shift)];
        if (id < 0 || id >= p.pages) continue;
        const size_t row = ((((size_t)id * 2 + 1) * p.kv_heads + kvh) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
        const unsigned w = *reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned short*>(p.data) + row * p.head_dim + d);
        float2 x;
        if (FMT == P_BF16) x = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
        else x = __half22float2(*reinterpret_cast<const __half2*>(&w));
        if (!(fabsf(x.x) < INFINITY)) sum.x += x.x;
        if (!(fabsf(x.y) < INFINITY)) sum.y += x.y;
    }
    return sum;
}
// Adds them to the finished rows r0 .. r0 + count - 1: the first `threads` threads of a block.
template <int FMT>
__device__ __forceinline__ void add_wild(const PagedAttnArgs& a, int s, int kvh, int r0, int count, int threads) {
    const int half = a.p.head_dim / 2;
#pragma unroll 1
    for (int e = threadIdx.x; e < count * half; e += threads) {
        const int r = r0 + e / half, d = e % half * 2;
        const float2 w = wild_sum<FMT>(a.p, s, kvh, a.group, r0, r, d);
        const long long i = (long long)(a.p.cu[s] + r / a.group) * a.out_stride + (long long)(kvh * a.group + r % a.group) * a.p.head_dim + d;
        auto add = [](auto* v, float x) {
            if (x != 0.0f) *v = (float)*v + x;
        };
        if (a.out_type == VC4_F32) {
            add(reinterpret_cast<float*>(a.out) + i, w.x);
            add(reinterpret_cast<float*>(a.out) + i + 1, w.y);
        } else if (a.out_type == VC4_BF16) {
            add(reinterpret_cast<__nv_bfloat16*>(a.out) + i, w.x);
            add(reinterpret_cast<__nv_bfloat16*>(a.out) + i + 1, w.y);
        } else {
            add(reinterpret_cast<__half*>(a.out) + i, w.x);
            add(reinterpret_cast<__half*>(a.out) + i + 1, w.y);
        }
    }
}
// A sum of weights, negative where such values belong to its row.
__device__ __forceinline__ float mark_wild(float l) { return __int_as_float(__float_as_int(l) | (int)0x80000000u); }
__device__ __forceinline__ bool marked_wild(float l) { return __float_as_int(l) < 0; }
__device__ __forceinline__ uint4 ld_shared16(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void st_shared16(unsigned addr, const uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// For a block in which a bounded wait gave up, all its threads: the copies and products it
// still has in flight end before its shared memory is used again or given back (warp 0
// waits, the others for it).
__device__ __forceinline__ void wait_for_copies() {
    if (threadIdx.x < 32) {
        const unsigned long long began = global_ns();
        while (global_ns() - began < 2000000ull) __nanosleep(1000);
    }
    __syncthreads();
}

template <int FMT> struct PagedBytes { static constexpr int v = FMT == P_Q8 ? 1 : 2; };

// Two 16-bit operands in one register.
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int FMT>
__device__ __forceinline__ unsigned pack_op(float lo, float hi) {
    return FMT == P_BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}
// Two bf16 query values as f16: exact inside f16's normal range (8 significant
// bits go into 11); beyond +-65504 the largest f16, and below 2^-14 the error is
// at most 2^-25 absolute.  NaN stays NaN.
__device__ __forceinline__ unsigned bf16_to_f16(unsigned w) {
    float lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
    lo = lo > 65504.0f ? 65504.0f : lo < -65504.0f ? -65504.0f : lo;
    hi = hi > 65504.0f ? 65504.0f : hi < -65504.0f ? -65504.0f : hi;
    return pack_f16(lo, hi);
}
// Two q16 levels (big-endian int16 in memory) as f16: 2^23 + (level + 2^15)
// built in the mantissa, so the subtraction is exact; the f16 rounding keeps 11
// of at most 16 bits (2^-12 relative), and `rest` what it drops, exactly.
template <bool REST>
__device__ __forceinline__ unsigned q16_to_f16(unsigned w, unsigned& rest) {
    w ^= 0x00800080u;
    const float bias = 8388608.0f + 32768.0f;
    const float lo = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7601)) - bias;
    const float hi = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7623)) - bias;
    const unsigned r = pack_f16(lo, hi);
    if (REST) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        rest = pack_f16(lo - f.x, hi - f.y);
    }
    return r;
}
__device__ __forceinline__ unsigned q16_to_f16(unsigned w) {
    unsigned none;
    return q16_to_f16<false>(w, none);
}
// Bytes (already xor 0x80) 0,1 / 2,3 of x as f16 levels: 1024 + u in the
// mantissa, minus 1152; exact.
__device__ __forceinline__ unsigned q8_pair(unsigned x, bool high) {
    const unsigned m = __byte_perm(x, 0x64646464u, high ? 0x4342 : 0x4140);
    unsigned r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0x64806480u));
    return r;
}

template <bool BF>
__device__ __forceinline__ void mma_16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- the few-row kernel's tiles (es: bytes of a cached value) ----

// How a tile lies in shared memory.  Rows of 128 bytes (f16, bf16 from head size 64 in
// panels of 64 values; q8 of 128) are in the 128-byte swizzle and rows of 64 (q8) in the
// 64-byte one, so that the lanes' fragment loads spread over the banks; the others are
// packed.
__host__ __device__ constexpr int split_mode(int es, int hd) {   // 0 packed, 1 128-byte, 2 64-byte swizzle
    return es == 2 ? (hd >= 64 ? 1 : 0) : hd == 128 ? 1 : hd == 64 ? 2 : 0;
}
__host__ __device__ constexpr int split_panels(int es, int hd) { return es == 2 && hd > 64 ? 2 : 1; }
__host__ __device__ constexpr int split_pitch(int es, int hd) { return split_mode(es, hd) == 1 ? 128 : hd * es; }
// positions per tile: 128 for short rows of the 16-row kernel (a tile's softmax and
// barriers cost the same for 16 and 32 positions of a warp)
__host__ __device__ constexpr int split_tile(int es, int hd, int wr) { return wr == 1 && hd * es <= 128 ? 128 : 64; }
__host__ __device__ constexpr int split_half(int es, int hd, int wr) { return split_tile(es, hd, wr) * split_pitch(es, hd) * split_panels(es, hd); }
__host__ __device__ constexpr int split_stages(int es, int hd, int wr) {   // about 75 KB: three blocks on an SM
    const int s = (75 * 1024) / (2 * split_half(es, hd, wr));
    return s < 3 ? 3 : s > 6 ? 6 : s;
}
__host__ __device__ constexpr size_t split_smem(int es, int hd, int wr) {
    const size_t ring = (size_t)2 * split_half(es, hd, wr) * split_stages(es, hd, wr), join = 4 * 16 * (size_t)(hd + 4) * 4 + 4 * 16 * 8;
    return 1023 + (ring > join ? ring : join);      // 1023: the ring starts on a swizzle atom
}

// Blocks of the kernel an SM holds: by its launch bounds and by shared memory.
__host__ __device__ constexpr int split_bound(int es, int hd, int wr) { return hd * wr <= 64 ? 4 : wr == 4 && hd >= 96 ? 2 : 3; }
inline int split_blocks(int es, int hd, int wr) {
    return std::max(1, std::min(split_bound(es, hd, wr), (int)(228 * 1024 / (split_smem(es, hd, wr) + 1024))));
}

// The pool as rows of `row_bytes`; a box is `width` bytes of as many rows as a page has
// in a tile; the host's checks keep the rows below 2^31.  False where no descriptor can
// be made.
inline bool paged_map(CUtensorMap* map, const PagedArgs& p, int row_bytes, int width, int tile, CUtensorMapSwizzle swizzle) {
    const auto enc = tmap_encode_fn();
    const int page_len = 1 << p.page_shift, span = page_len < tile ? page_len : tile;
    const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, ((cuuint64_t)p.pages * 2 * p.kv_heads) << p.page_shift};
    const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)width, (cuuint32_t)span}, es[2] = {1, 1};
    return enc &&
           enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.data, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Two floats in one 64-bit register: sm_100's packed float operations take half the
// issue slots.
__device__ __forceinline__ unsigned long long pack2(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// Stores four consecutive floats as `type` from element index i of a row.
__device__ __forceinline__ void store4_as(void* row, int type, long long i, float4 v) {
    if (type == VC4_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(row) + i) = v;
    else if (type == VC4_BF16)
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(row) + i) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    else
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(row) + i) = make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
}

}  // namespace
}  // namespace vc4
