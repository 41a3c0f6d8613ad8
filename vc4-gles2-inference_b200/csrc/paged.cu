// paged.cu -- the paged KV cache: the append kernel (QK-norm, RoPE and the cache
// codec over a projection's rows), the join of split attention, and the C entries.
#include "paged.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <string>

namespace vc4 {
namespace {

int fail(int code, const std::string& msg) { return set_error(code, msg.c_str()); }

// The GPU of a handle as the current device for one call; the caller's after it.
struct OnDevice {
    int before = -1;
    cudaError_t err;
    explicit OnDevice(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else if (err == cudaSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

struct AppendArgs {
    PagedArgs p;
    const void* qkv;
    void* q;
    long long qkv_stride, q_stride;
    const float *q_norm, *k_norm, *cos, *sin;
    float eps;
    int heads, rope_len, half, q_type, per_block;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;    // most tokens of a block (one warp looks one up)
constexpr int kAppendVecs = 4;      // head vectors a group of lanes holds at once
constexpr int kAppendSms = 148;     // SMs the tokens of a block are chosen for

// Four consecutive values of a row, as they lie there and as two float pairs.
template <int TIN> struct Raw4 { uint2 w; };
template <> struct Raw4<VC4_F32> { uint4 w; };
template <int TIN>
__device__ __forceinline__ void load4(const void* row, long long i, Raw4<TIN>& v) {
    if constexpr (TIN == VC4_F32) v.w = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(row) + i));
    else v.w = __ldcs(reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(row) + i));
}
template <int TIN>
__device__ __forceinline__ void pairs4(const Raw4<TIN>& r, unsigned long long (&v)[2]) {
    if constexpr (TIN == VC4_F32) {
        v[0] = pack2(__uint_as_float(r.w.x), __uint_as_float(r.w.y));
        v[1] = pack2(__uint_as_float(r.w.z), __uint_as_float(r.w.w));
    } else if constexpr (TIN == VC4_BF16) {
        v[0] = pack2(__uint_as_float(r.w.x << 16), __uint_as_float(r.w.x & 0xFFFF0000u));
        v[1] = pack2(__uint_as_float(r.w.y << 16), __uint_as_float(r.w.y & 0xFFFF0000u));
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.w.y));
        v[0] = pack2(a.x, a.y);
        v[1] = pack2(b.x, b.y);
    }
}
__device__ __forceinline__ float4 as_float4(const unsigned long long (&v)[2]) {
    float4 f;
    unpack2(v[0], f.x, f.y);
    unpack2(v[1], f.z, f.w);
    return f;
}

// Four consecutive values of a cached row, in the pages' format.
template <int FMT>
__device__ __forceinline__ void store_cache4(uint8_t* row, int i, float4 v) {
    float dec;
    if (FMT == P_Q8) {
        *reinterpret_cast<unsigned*>(row + i) = kv_encode(v.x, 1, &dec) | kv_encode(v.y, 1, &dec) << 8 |
                                                kv_encode(v.z, 1, &dec) << 16 | kv_encode(v.w, 1, &dec) << 24;
    } else if (FMT == P_Q16) {
        *reinterpret_cast<uint2*>(row + 2 * i) = make_uint2(kv_encode(v.x, 2, &dec) | kv_encode(v.y, 2, &dec) << 16,
                                                            kv_encode(v.z, 2, &dec) | kv_encode(v.w, 2, &dec) << 16);
    } else {
        constexpr int F = FMT == P_BF16 ? P_BF16 : P_F16;
        *reinterpret_cast<uint2*>(row + 2 * i) = make_uint2(pack_op<F>(v.x, v.y), pack_op<F>(v.z, v.w));
    }
}

// A group of LPV lanes takes four head vectors of a token at once; a lane holds eight
// values of each as four rotation pairs, so norm, rotation and encoding stay in its
// registers and every load and store is 4 to 16 bytes wide.  Bound by bytes for many
// tokens, by the chain offsets -> length -> page id for a few; the first vectors' loads
// are issued before that chain.  With one vector at a time the square root, the two
// divisions and the sums' shuffles, the same for every lane, took as long as the bytes
// (12332 tokens of 32 + 16 heads of 128 in bf16: 120 us against 80, 3.8 TB/s): four
// vectors' sums are halved across the lanes (10 shuffles for 32), so each lane ends with
// one vector's and takes its root.
// The float operations are the slot cache's (k_attn): squares summed in double,
// 1/sqrt(ss/hd + eps), w*(r*x), the rotation's products and sums rounded one by one, the
// codec's floor(x*grid + 1/2).  (Packed products round like single ones.)
template <int TIN, int FMT, int LPV>
__global__ void __launch_bounds__(kAppendThreads, TIN == VC4_F32 ? 2 : 3) k_paged_append(AppendArgs a) {
    constexpr int N = kAppendVecs, NG = 32 / LPV;   // groups of a warp
    const PagedArgs& p = a.p;
    const int hd = p.head_dim, half = hd / 2, nvec = a.heads + 2 * p.kv_heads, turned = a.heads + p.kv_heads;
    __shared__ int s_pos[kAppendTokens];             // the position, -1: nothing to do
    __shared__ long long s_row[kAppendTokens];       // row index of (page, K, head 0, offset)
    const int tok0 = blockIdx.x * a.per_block, ntok = min(a.per_block, p.tokens - tok0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPV;
    const bool live = sub * 8 < hd;
    const int i0 = a.half ? 4 * sub : 8 * sub, i1 = a.half ? half + 4 * sub : 8 * sub + 4;
    // pieces of four vectors of a token; a warp takes NG of them at a time, in order
    const int pieces = (nvec + N - 1) / N, total = ntok * pieces, step = kAppendThreads / 32 * NG;
    Raw4<TIN> raw[N][2];
    auto fetch = [&](int at) {
        const int t = at / pieces, vec0 = at % pieces * N;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (at < total && live && vec0 + k < nvec) {
                const long long base = (long long)(tok0 + t) * a.qkv_stride + (long long)(vec0 + k) * hd;
                load4<TIN>(a.qkv, base + i0, raw[k][0]);
                load4<TIN>(a.qkv, base + i1, raw[k][1]);
            } else {
                raw[k][0] = raw[k][1] = Raw4<TIN>{};
            }
    };
    const int first = warp * NG + lane / LPV;
    fetch(first);

    if (warp < ntok) {
        const int tok = tok0 + warp, s = paged_find(p.cu, p.seqs, tok);
        const int c0 = p.cu[s], c1 = p.cu[s + 1];
        int pos = -1;
        long long row = 0;
        if (tok >= c0 && tok < c1 && c0 >= 0 && c1 <= p.tokens) {   // rows of no sequence, or of a bad one: none of this
            const int page_len = 1 << p.page_shift;
            pos = max(p.len[s], 0) - (c1 - tok);
            bool bad = pos < 0 || pos >= (long long)p.table_stride * page_len || (a.cos && pos >= a.rope_len) ||
                       c1 - c0 > p.max_new;
            if (!bad) {
                const int page = p.table[(size_t)s * p.table_stride + (pos >> p.page_shift)];
                bad = page < 0 || page >= p.pages;
                row = (((long long)page * 2 * p.kv_heads) << p.page_shift) + (pos & (page_len - 1));
            }
            if (bad) {
                if (lane == 0) paged_flag(p.status, VC4_EINVAL);
                pos = -1;
            }
        }
        if (lane == 0) {
            s_pos[warp] = pos;
            s_row[warp] = row;
        }
    }
    // offsets that start below 0, run backwards or end past the rows: a sequence a lane of the
    // last warp, so that those no token's look-up meets are found too
    if (warp == kAppendThreads / 32 - 1)
        for (long long i = (long long)blockIdx.x * 32 + lane; i < p.seqs; i += (long long)gridDim.x * 32)
            if (p.cu[i] < 0 || p.cu[i + 1] < p.cu[i] || p.cu[i + 1] > p.tokens) paged_flag(p.status, VC4_EINVAL);
    __syncthreads();

    const int es = FMT == P_Q8 ? 1 : 2;
    for (int w = warp * NG; w < total; w += step) {          // (the groups of a warp stay together: the sums shuffle)
        const int at = w + lane / LPV, t = min(at, total - 1) / pieces, vec0 = min(at, total - 1) % pieces * N;
        const int pos = at < total ? s_pos[t] : -1;
        unsigned long long x[N][2][2];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            pairs4<TIN>(raw[k][0], x[k][0]);
            pairs4<TIN>(raw[k][1], x[k][1]);
        }
        fetch(at + step);                                    // on its way during this round
        if (a.q_norm) {
            double ss[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                ss[k] = 0.0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 f = as_float4(x[k][h]);     // a product of two floats is exact in double
                    ss[k] = fma((double)f.x, (double)f.x, ss[k]);
                    ss[k] = fma((double)f.y, (double)f.y, ss[k]);
                    ss[k] = fma((double)f.z, (double)f.z, ss[k]);
                    ss[k] = fma((double)f.w, (double)f.w, ss[k]);
                }
            }
            float r[N];
            auto root = [&](double sum) {
                return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(__double2float_rn(sum), (float)hd), a.eps)));
            };
            if (LPV >= 4) {      // two vectors' halves change places, then one's; then one is summed
                const bool up = lane & (LPV / 2), right = lane & (LPV / 4);
                double keep[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    keep[k] = (up ? ss[2 + k] : ss[k]) + __shfl_xor_sync(0xffffffffu, up ? ss[k] : ss[2 + k], LPV / 2);
                double one = (right ? keep[1] : keep[0]) + __shfl_xor_sync(0xffffffffu, right ? keep[0] : keep[1], LPV / 4);
#pragma unroll
                for (int o = LPV / 8; o; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
                const float mine = root(one);
#pragma unroll
                for (int k = 0; k < N; ++k)
                    r[k] = __shfl_sync(0xffffffffu, mine, (lane & ~(LPV - 1)) + (k >> 1) * (LPV / 2) + (k & 1) * (LPV / 4));
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) r[k] = root(ss[k] + __shfl_xor_sync(0xffffffffu, ss[k], 1));
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int vec = vec0 + k;
                if (vec >= turned || !live) continue;
                const float* w = vec < a.heads ? a.q_norm : a.k_norm;
                const float4 w0 = *reinterpret_cast<const float4*>(w + i0), w1 = *reinterpret_cast<const float4*>(w + i1);
                const unsigned long long rr = pack2(r[k], r[k]);
                x[k][0][0] = mul2(pack2(w0.x, w0.y), mul2(rr, x[k][0][0]));
                x[k][0][1] = mul2(pack2(w0.z, w0.w), mul2(rr, x[k][0][1]));
                x[k][1][0] = mul2(pack2(w1.x, w1.y), mul2(rr, x[k][1][0]));
                x[k][1][1] = mul2(pack2(w1.z, w1.w), mul2(rr, x[k][1][1]));
            }
        }
        if (pos >= 0 && live) {
            if (a.cos) {
                const float4 c = *reinterpret_cast<const float4*>(a.cos + (size_t)pos * half + 4 * sub);
                const float4 s = *reinterpret_cast<const float4*>(a.sin + (size_t)pos * half + 4 * sub);
                // (single operations: a packed product and sum may come out as one rounding)
                auto turn = [](float& u, float& v, float cc, float ss) {
                    const float y = __fsub_rn(__fmul_rn(u, cc), __fmul_rn(v, ss));
                    v = __fadd_rn(__fmul_rn(u, ss), __fmul_rn(v, cc));
                    u = y;
                };
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    if (vec0 + k >= turned) continue;
                    float4 f0 = as_float4(x[k][0]), f1 = as_float4(x[k][1]);
                    if (a.half) {
                        turn(f0.x, f1.x, c.x, s.x);
                        turn(f0.y, f1.y, c.y, s.y);
                        turn(f0.z, f1.z, c.z, s.z);
                        turn(f0.w, f1.w, c.w, s.w);
                    } else {
                        turn(f0.x, f0.y, c.x, s.x);
                        turn(f0.z, f0.w, c.y, s.y);
                        turn(f1.x, f1.y, c.z, s.z);
                        turn(f1.z, f1.w, c.w, s.w);
                    }
                    x[k][0][0] = pack2(f0.x, f0.y);
                    x[k][0][1] = pack2(f0.z, f0.w);
                    x[k][1][0] = pack2(f1.x, f1.y);
                    x[k][1][1] = pack2(f1.z, f1.w);
                }
            }
            const long long qrow = (long long)(tok0 + t) * a.q_stride;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int vec = vec0 + k;
                if (vec >= nvec) continue;
                if (vec < a.heads) {
                    store4_as(a.q, a.q_type, qrow + (long long)vec * hd + i0, as_float4(x[k][0]));
                    store4_as(a.q, a.q_type, qrow + (long long)vec * hd + i1, as_float4(x[k][1]));
                } else {
                    // heads of K, then of V, lie page_len rows apart
                    uint8_t* row = p.data + (s_row[t] + ((long long)(vec - a.heads) << p.page_shift)) * (hd * es);
                    store_cache4<FMT>(row, i0, as_float4(x[k][0]));
                    store_cache4<FMT>(row, i1, as_float4(x[k][1]));
                }
            }
        }
    }
}

template <int FMT, int LPV>
void launch_append_lanes(const AppendArgs& a, int type, unsigned blocks, cudaStream_t st) {
    if (type == VC4_F32) k_paged_append<VC4_F32, FMT, LPV><<<blocks, kAppendThreads, 0, st>>>(a);
    else if (type == VC4_BF16) k_paged_append<VC4_BF16, FMT, LPV><<<blocks, kAppendThreads, 0, st>>>(a);
    else k_paged_append<VC4_F16, FMT, LPV><<<blocks, kAppendThreads, 0, st>>>(a);
}
int append_lanes(int hd) { return hd > 64 ? 16 : hd > 32 ? 8 : hd > 16 ? 4 : 2; }
template <int FMT>
void launch_append(const AppendArgs& a, int type, unsigned blocks, cudaStream_t st) {
    switch (append_lanes(a.p.head_dim)) {
        case 16: launch_append_lanes<FMT, 16>(a, type, blocks, st); break;
        case 8: launch_append_lanes<FMT, 8>(a, type, blocks, st); break;
        case 4: launch_append_lanes<FMT, 4>(a, type, blocks, st); break;
        default: launch_append_lanes<FMT, 2>(a, type, blocks, st); break;
    }
}

// Tokens of a block: what its groups of lanes take in one round, and in three where one
// round each gives more than six blocks an SM: a block's look-up then comes before more
// loads (1, 2, 4, 8 tokens: 12332 of 32/8 heads of 128, three rounds at 4, 114, 95, 80,
// 79 us; 2000 22.7, 22.4, 21.0, 20.5; 600 9.8, 9.4, 11.4, 16.4, one round at 1; 14204 of
// 4/2 heads of 64, one round at 16, 111, 56, 33, 20).
int append_tokens(int tokens, int nvec, int hd) {
    const int groups = kAppendThreads / append_lanes(hd), pieces = (nvec + kAppendVecs - 1) / kAppendVecs;
    const int rounds = (long long)tokens * pieces / groups > 6 * kAppendSms ? 3 : 1;
    return std::max(1, std::min(rounds * groups / pieces, kAppendTokens));
}

// ---------------------------------------------------------------------------
// join of split attention: o = sum_i 2^(c(m_i - m)) O_i / sum_i 2^(c(m_i - m)) l_i
// ---------------------------------------------------------------------------

// One warp per (token, head); lane i holds the weights of splits i and i + 32, then four
// values of the row.  Bound by the partial sums' bytes, which the many-row kernel just
// left in L2 (256 tokens x 16 heads of 128 in 9 parts: 7.8 us).
__global__ void __launch_bounds__(256) k_paged_join(PagedAttnArgs a) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const PagedArgs& p = a.p;
    const int tok = (int)(task / a.heads), head = (int)(task % a.heads);
    if (tok >= p.tokens) return;
    const size_t at = (size_t)task, step = (size_t)p.tokens * a.heads;
    float2 e[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        e[k] = lane + 32 * k < a.splits ? a.ml[at + (lane + 32 * k) * step] : make_float2(-INFINITY, 0.0f);
    // rows of no sequence, of one whose offsets are bad and beyond max_new were not computed:
    // leave them
    const int s = paged_find(p.cu, p.seqs, tok), c0 = p.cu[s], c1 = p.cu[s + 1];
    if (c0 < 0 || tok < c0 || tok >= c1 || c1 > p.tokens || tok - c0 >= p.max_new) return;
    bool wild = false;      // infinite or NaN values were taken out of this row
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        wild |= marked_wild(e[k].y);
        e[k].y = fabsf(e[k].y);
    }
    wild = __any_sync(0xffffffffu, wild);
    float m = fmaxf(e[0].x, e[1].x);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float w[2], l = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        w[k] = e[k].x == -INFINITY ? 0.0f : ex2f((e[k].x - m) * a.scale2);
        if (w[k] != 0.0f) l = __fmaf_rn(w[k], e[k].y, l);
    }
    // NaN statistics (a NaN score) have m_i = -inf or a NaN sum: the sum carries them
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (e[k].y != e[k].y) l = e[k].y;
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float f = l > 0.0f || l != l ? a.vscale / l : 0.0f;
    const int hd = p.head_dim, d = 4 * lane;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < a.splits; i0 += 4) {
        float4 x[4];
        float wi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + k;
            wi[k] = __shfl_sync(0xffffffffu, i < 32 ? w[0] : w[1], i & 31);
            // (an empty split left nothing to read)
            x[k] = i < a.splits && wi[k] != 0.0f && d < hd
                       ? *reinterpret_cast<const float4*>(a.part + (at + i * step) * hd + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v.x = __fmaf_rn(wi[k], x[k].x, v.x);
            v.y = __fmaf_rn(wi[k], x[k].y, v.y);
            v.z = __fmaf_rn(wi[k], x[k].z, v.z);
            v.w = __fmaf_rn(wi[k], x[k].w, v.w);
        }
    }
    if (d < hd) {
        float y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
        if (wild) {
            const int r = (tok - c0) * a.group + head % a.group, r0 = r / kPagedChunkRows * kPagedChunkRows;
            for (int k = 0; k < 4; k += 2) {
                const float2 x = a.fmt == P_BF16 ? wild_sum<P_BF16>(p, s, head / a.group, a.group, r0, r, d + k)
                                                 : wild_sum<P_F16>(p, s, head / a.group, a.group, r0, r, d + k);
                y[k] += x.x;
                y[k + 1] += x.y;
            }
        }
        store4_as(a.out, a.out_type, (long long)tok * a.out_stride + (long long)head * hd + d, make_float4(y[0], y[1], y[2], y[3]));
    }
}

// ---------------------------------------------------------------------------
// argument checks and plans
// ---------------------------------------------------------------------------

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

std::string bad_pages(const vc4_pages* p) {
    if (!p) return "pages is null";
    if (p->format != VC4_KV_Q8 && p->format != VC4_KV_Q16 && p->format != VC4_KV_BF16 && p->format != VC4_KV_F16)
        return "unknown page format " + std::to_string(p->format);
    if (p->page_len != 16 && p->page_len != 32 && p->page_len != 64 && p->page_len != 128 && p->page_len != 256)
        return "page_len must be 16, 32, 64, 128 or 256";
    if (p->pages <= 0 || p->kv_heads <= 0) return "pages and kv_heads must be positive";
    if (p->head_dim <= 0 || p->head_dim > 128 || p->head_dim % 16) return "head_dim must be a multiple of 16, at most 128";
    if (!p->data || !aligned16(p->data)) return "the pool's address must be a multiple of 16";
    if ((long long)p->pages * 2 > 0x7fffffffLL / ((long long)p->kv_heads * p->page_len))
        return "a pool holds at most 2^31 - 1 rows (pages x 2 x kv_heads x page_len)";
    return "";
}

std::string bad_batch(const vc4_paged_batch* b, const vc4_pages* p) {
    if (!b) return "batch is null";
    if (b->seqs <= 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->table_stride <= 0)
        return "seqs and table_stride must be positive, tokens, max_new and max_len not negative";
    if (!b->cu || !b->len || !b->table) return "cu, len and table are required";
    if (((uintptr_t)b->cu | (uintptr_t)b->len | (uintptr_t)b->table | (uintptr_t)b->status) % 4)
        return "cu, len, table and status are aligned to their elements";
    if ((long long)b->max_len > (long long)b->table_stride * p->page_len) return "max_len runs past the page table";
    if ((long long)b->table_stride * p->page_len > (1LL << 30)) return "a page table covers at most 2^30 positions (table_stride x page_len)";
    return "";
}

std::string bad_rows(const char* what, const void* ptr, long long stride, long long width) {
    if (!ptr || !aligned16(ptr)) return std::string(what) + "'s address must be a multiple of 16";
    if (stride < width || stride % 8) return std::string(what) + "'s stride must be a multiple of 8 elements, at least a row";
    return "";
}

// Rows of bytes, `stride` apart, and whether two sets of them share a byte.  Rows that lie
// side by side in one buffer (equal strides) do not; of sets with different strides the
// whole extents count.
struct Extent {
    const void* at;
    size_t rows, stride, width;
};
bool meet(Extent a, Extent b) {
    if (!a.rows || !b.rows) return false;
    if ((uintptr_t)b.at < (uintptr_t)a.at) std::swap(a, b);
    const size_t ahead = (uintptr_t)b.at - (uintptr_t)a.at;
    if (ahead >= (a.rows - 1) * a.stride + a.width) return false;
    if (a.rows == 1 || (b.rows > 1 && b.stride != a.stride)) return true;
    const size_t in = ahead % a.stride;      // where b's rows start in a's
    return in < a.width || a.stride - in < b.width;
}
size_t bytes_of(int type) { return type == VC4_F32 ? 4 : 2; }
Extent pool_of(const vc4_pages* p) {
    const size_t rows = (size_t)p->pages * 2 * p->kv_heads * p->page_len;
    return {p->data, 1, 0, rows * p->head_dim * (p->format == VC4_KV_Q8 ? 1 : 2)};
}

int shift_of(int page_len) { return page_len == 16 ? 4 : page_len == 32 ? 5 : page_len == 64 ? 6 : page_len == 128 ? 7 : 8; }

PagedArgs paged_args(const vc4_pages* p, const vc4_paged_batch* b) {
    PagedArgs a{};
    a.data = (uint8_t*)p->data;
    a.pages = p->pages; a.page_shift = shift_of(p->page_len); a.kv_heads = p->kv_heads; a.head_dim = p->head_dim;
    a.seqs = b->seqs; a.tokens = b->tokens; a.max_new = b->max_new; a.table_stride = b->table_stride;
    a.cu = b->cu; a.len = b->len; a.table = b->table; a.status = b->status;
    return a;
}

int pfmt(int format) {
    return format == VC4_KV_Q8 ? P_Q8 : format == VC4_KV_Q16 ? P_Q16 : format == VC4_KV_BF16 ? P_BF16 : P_F16;
}

struct AttnPlan {
    bool chunk;           // the many-row kernel
    int wr, row_tiles, splits;
    size_t bytes;
};

// Up to 64 rows (new tokens x query heads of a KV head) of a sequence go to the
// few-row kernel, in blocks of the least of 16, 32 and 64 that holds them; more to
// the many-row kernel, 256 a block; of large heads from 33 rows, where every SM has a
// block (32 x 16 tokens over 4000 bf16 positions, 32/8 heads of 128: 133 us in blocks of
// 64 rows, 111 in the many-row kernel; 61 x 5 over 2000, 16/2 of 64: 29 and 35; at 96 and 80
// either may win, 32/8 heads, bf16, 32 x 16 over 4000 113 and 101, 104 and 98, 64 x 10 over
// 1500 91 and 95, 85 and 93).  q16
// pages with an f16 or float output stay with the few-row kernel, which holds a level in
// two operands.
// Splits of the few-row kernel: as many as the GPU holds at once, of three tiles of 64
// positions or more (16 rows, whose four warps share a tile; 32 rows two, 64 rows, where
// each warp takes every tile, one): in a replayed graph, with 1, 2, 3, 6 tiles a split,
// one token over 777 q16 positions 11.6, 11.0, 10.3, 11.3 us, 16 x 8 over 300, 16/4 heads
// of 64, 8.9, 8.3, 8.7, 8.7, 5 over 400, 16/2 of 64, 7.9, 9.9, 10.3, 13.1; a whole
// cluster of eight for long sequences that do not fill the GPU a whole number of times,
// whose ragged lengths then even out (12 x 40k positions: 1, 2, 3, 4, 8 splits 457, 274,
// 283, 278, 244 us).  Of the many-row kernel: what one block on each SM allows, down to
// one tile of 128 (8, 4, 2, 1 tiles or more: 128 tokens over 2000 bf16 positions, 32/8
// heads of 128, 32.9, 26.7, 24.7, 25.0 us; 300 over 1500 q16, 8/4 of 96, 51.5, 29.8,
// 24.1, 24.7; 128 over 700 24.9, 24.9, 24.7, 21.0); they leave partial results in the
// work buffer, for a second kernel.
AttnPlan attn_plan(const vc4_pages* p, const vc4_paged_batch* b, int heads, int sms, int out_type) {
    AttnPlan pl{};
    // (a sequence has no more new tokens than the batch, whatever max_new allows)
    const long long rows = (long long)std::min(b->max_new, b->tokens) * (heads / p->kv_heads);
    const bool many = rows > 64 || (rows > 32 && p->head_dim > 96 && (long long)b->seqs * p->kv_heads >= sms);
    pl.chunk = many && !(p->format == VC4_KV_Q16 && out_type != VC4_BF16);
    pl.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const int per = pl.chunk ? kPagedChunkRows : 16 * pl.wr, tile = pl.chunk ? 128 : 64;
    pl.row_tiles = (int)((rows + per - 1) / per);
    const long long units = (long long)b->seqs * p->kv_heads * std::max(1, pl.row_tiles);
    const int tiles = (b->max_len + tile - 1) / tile;
    if (pl.chunk) {
        pl.splits = (int)std::max(1LL, std::min({sms / units, (long long)tiles, (long long)kPagedMaxSplits}));
    } else {
        const int es = p->format == VC4_KV_Q8 ? 1 : 2;
        const long long fit = (long long)sms * split_blocks(es, p->head_dim, pl.wr);
        const int least = pl.wr == 1 ? 3 : pl.wr == 2 ? 2 : 1;
        pl.splits = (int)std::max(1LL, std::min({fit / units, (long long)tiles / least, (long long)kPagedMaxCluster}));
        if (units < fit && fit / units < kPagedMaxCluster && tiles >= 128 * pl.splits) pl.splits = kPagedMaxCluster;
    }
    if (pl.chunk && pl.splits > 1) pl.bytes = (size_t)pl.splits * b->tokens * heads * ((size_t)p->head_dim * 4 + 8);
    return pl;
}

int sms_of(int device, int* sms) {
    static int have[64] = {};
    static std::mutex mu;
    std::lock_guard<std::mutex> lk(mu);
    if (device < 0 || device >= 64) return fail(VC4_EINVAL, "device index too large");
    if (!have[device]) {
        const cudaError_t e = cudaDeviceGetAttribute(&have[device], cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return fail(VC4_ECUDA, cudaGetErrorString(e));
    }
    *sms = have[device];
    return VC4_OK;
}

}  // namespace
}  // namespace vc4

using namespace vc4;

extern "C" int vc4_paged_append(vc4_gpu* g, const vc4_pages* p, const vc4_paged_batch* b, const void* qkv, int qkv_type,
                                long long qkv_stride, int heads, const float* q_norm, const float* k_norm, float eps,
                                const float* cos, const float* sin, int rope_len, int rope_half, void* q, int q_type,
                                long long q_stride, void* stream) {
    auto refuse = [](const std::string& m) { return fail(VC4_EINVAL, "paged_append: " + m); };
    std::string m = bad_pages(p);
    if (m.empty()) m = bad_batch(b, p);
    if (!m.empty()) return refuse(m);
    if (heads <= 0 || heads % p->kv_heads) return refuse("heads must be a positive multiple of kv_heads");
    if (qkv_type < VC4_F32 || qkv_type > VC4_F16 || q_type < VC4_F32 || q_type > VC4_F16)
        return refuse("qkv and q are VC4_F32, VC4_BF16 or VC4_F16");
    const long long width = ((long long)heads + 2 * p->kv_heads) * p->head_dim, qw = (long long)heads * p->head_dim;
    if (!qkv_stride) qkv_stride = width;
    if (!q_stride) q_stride = qw;
    m = bad_rows("qkv", qkv, qkv_stride, width);
    if (m.empty()) m = bad_rows("q", q, q_stride, qw);
    if (!m.empty()) return refuse(m);
    if (!q_norm != !k_norm) return refuse("q_norm and k_norm go together");
    if (q_norm && (!aligned16(q_norm) || !aligned16(k_norm))) return refuse("the norm weights' addresses must be multiples of 16");
    if (q_norm && !(eps >= 0.0f)) return refuse("eps must not be negative");
    if (!cos != !sin) return refuse("cos and sin go together");
    if (cos && (!aligned16(cos) || !aligned16(sin) || rope_len <= 0))
        return refuse("the rotation tables need rows, their addresses multiples of 16");
    if (!g) return refuse("gpu is null");
    const Extent from{qkv, (size_t)b->tokens, qkv_stride * bytes_of(qkv_type), width * bytes_of(qkv_type)};
    const Extent to{q, (size_t)b->tokens, q_stride * bytes_of(q_type), qw * bytes_of(q_type)};
    if (meet(from, to)) return refuse("q overlaps qkv");
    if (meet(from, pool_of(p)) || meet(to, pool_of(p))) return refuse("the pool overlaps qkv or q");
    if (!b->tokens || !b->max_new) return VC4_OK;
    OnDevice on(gpu_device(g));
    if (on.err != cudaSuccess) return fail(VC4_ECUDA, cudaGetErrorString(on.err));
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : gpu_stream(g);
    AppendArgs a{};
    a.p = paged_args(p, b);
    a.qkv = qkv; a.q = q; a.qkv_stride = qkv_stride; a.q_stride = q_stride;
    a.q_norm = q_norm; a.k_norm = k_norm; a.cos = cos; a.sin = sin; a.eps = eps;
    a.heads = heads; a.rope_len = rope_len; a.half = rope_half ? 1 : 0; a.q_type = q_type;
    a.per_block = append_tokens(b->tokens, heads + 2 * p->kv_heads, p->head_dim);
    const unsigned blocks = (unsigned)(((long long)b->tokens + a.per_block - 1) / a.per_block);
    switch (pfmt(p->format)) {
        case P_Q8: launch_append<P_Q8>(a, qkv_type, blocks, st); break;
        case P_Q16: launch_append<P_Q16>(a, qkv_type, blocks, st); break;
        case P_BF16: launch_append<P_BF16>(a, qkv_type, blocks, st); break;
        default: launch_append<P_F16>(a, qkv_type, blocks, st); break;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(VC4_ECUDA, std::string("paged_append: ") + cudaGetErrorString(e));
    return VC4_OK;
}

extern "C" int vc4_paged_attention_bytes(vc4_gpu* g, const vc4_pages* p, const vc4_paged_batch* b, int heads,
                                         size_t* bytes) {
    auto refuse = [](const std::string& m) { return fail(VC4_EINVAL, "paged_attention_bytes: " + m); };
    std::string m = bad_pages(p);
    if (m.empty()) m = bad_batch(b, p);
    if (!m.empty()) return refuse(m);
    if (heads <= 0 || heads % p->kv_heads) return refuse("heads must be a positive multiple of kv_heads");
    if (!bytes) return refuse("bytes is null");
    if ((long long)b->tokens * heads > 0x7fffffffLL) return refuse("too many rows in one call");
    if (!g) return refuse("gpu is null");
    int sms = 0;
    if (int e = sms_of(gpu_device(g), &sms)) return e;
    *bytes = std::max(attn_plan(p, b, heads, sms, VC4_BF16).bytes, attn_plan(p, b, heads, sms, VC4_F32).bytes);
    return VC4_OK;
}

extern "C" int vc4_paged_attention(vc4_gpu* g, const vc4_pages* p, const vc4_paged_batch* b, const void* q, int q_type,
                                   long long q_stride, int heads, float scale, void* out, int out_type,
                                   long long out_stride, void* work, size_t work_bytes, void* stream) {
    auto refuse = [](const std::string& m) { return fail(VC4_EINVAL, "paged_attention: " + m); };
    std::string m = bad_pages(p);
    if (m.empty()) m = bad_batch(b, p);
    if (!m.empty()) return refuse(m);
    if (heads <= 0 || heads % p->kv_heads) return refuse("heads must be a positive multiple of kv_heads");
    if (q_type != VC4_BF16 && q_type != VC4_F16) return refuse("q is VC4_BF16 or VC4_F16");
    if ((p->format == VC4_KV_BF16 && q_type != VC4_BF16) || (p->format == VC4_KV_F16 && q_type != VC4_F16))
        return refuse("q has the pages' type where that is bf16 or f16");
    if (out_type < VC4_F32 || out_type > VC4_F16) return refuse("out is VC4_F32, VC4_BF16 or VC4_F16");
    const long long width = (long long)heads * p->head_dim;
    if (!q_stride) q_stride = width;
    if (!out_stride) out_stride = width;
    m = bad_rows("q", q, q_stride, width);
    if (m.empty()) m = bad_rows("out", out, out_stride, width);
    if (!m.empty()) return refuse(m);
    if (!(scale >= 0.0f) || !(scale < INFINITY)) return refuse("scale must not be negative (0: 1/sqrt(head_dim))");
    const double grid = p->format == VC4_KV_Q8 ? 1.0 / 16 : p->format == VC4_KV_Q16 ? 1.0 / 2048 : 1.0;
    const double sc = scale > 0.0f ? (double)scale : 1.0 / std::sqrt((double)p->head_dim);
    const float scale2 = (float)(sc * 1.4426950408889634 * grid);
    if (!(scale2 >= FLT_MIN) || !(scale2 < INFINITY)) return refuse("scale's product with the pages' grid leaves float's range");
    if ((long long)b->tokens * heads > 0x7fffffffLL) return refuse("too many rows in one call");
    if (!g) return refuse("gpu is null");
    const Extent from{q, (size_t)b->tokens, q_stride * bytes_of(q_type), width * bytes_of(q_type)};
    const Extent to{out, (size_t)b->tokens, out_stride * bytes_of(out_type), width * bytes_of(out_type)};
    if (meet(from, to)) return refuse("out overlaps q");
    if (meet(to, pool_of(p))) return refuse("out overlaps the pool");
    int sms = 0;
    if (int e = sms_of(gpu_device(g), &sms)) return e;
    const AttnPlan pl = attn_plan(p, b, heads, sms, out_type);
    if (work_bytes < pl.bytes || (pl.bytes && (!work || !aligned16(work))))
        return refuse("the work buffer needs " + std::to_string(pl.bytes) + " bytes at a multiple of 16");
    const Extent parts{work, pl.bytes ? 1u : 0u, 0, pl.bytes};
    if (meet(parts, from) || meet(parts, to) || meet(parts, pool_of(p))) return refuse("the work buffer overlaps q, out or the pool");
    if (!b->tokens || !b->max_new) return VC4_OK;
    if ((long long)b->seqs * p->kv_heads * pl.row_tiles * pl.splits > 0x7fffffffLL) return refuse("too many rows in one call");
    OnDevice on(gpu_device(g));
    if (on.err != cudaSuccess) return fail(VC4_ECUDA, cudaGetErrorString(on.err));
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : gpu_stream(g);
    PagedAttnArgs a{};
    a.p = paged_args(p, b);
    a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride; a.q_type = q_type; a.out_type = out_type;
    a.heads = heads; a.group = heads / p->kv_heads; a.row_tiles = pl.row_tiles; a.splits = pl.splits;
    a.fmt = pfmt(p->format);
    a.scale2 = scale2;
    a.vscale = (float)grid;
    if (pl.bytes) {
        a.part = (float*)work;
        a.ml = (float2*)((char*)work + (size_t)pl.splits * b->tokens * heads * p->head_dim * 4);
    }
    bool ok;
    switch (pfmt(p->format)) {
        case P_Q8: ok = pl.chunk ? launch_paged_chunk_q8(a, st) : launch_paged_split_q8(a, pl.wr, st); break;
        case P_Q16: ok = pl.chunk ? launch_paged_chunk_q16(a, st) : launch_paged_split_q16(a, pl.wr, st); break;
        case P_BF16: ok = pl.chunk ? launch_paged_chunk_bf16(a, st) : launch_paged_split_bf16(a, pl.wr, st); break;
        default: ok = pl.chunk ? launch_paged_chunk_f16(a, st) : launch_paged_split_f16(a, pl.wr, st); break;
    }
    if (!ok) return fail(VC4_ECUDA, "paged_attention: no TMA descriptor for this pool");
    if (pl.bytes) launch_pdl_block(k_paged_join, dim3((unsigned)(((long long)b->tokens * heads + 7) / 8)), 256, 0, st, a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(VC4_ECUDA, std::string("paged_attention: ") + cudaGetErrorString(e));
    return VC4_OK;
}
