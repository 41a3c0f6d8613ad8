// verify.cu -- verification of drafted tokens against the target's probabilities.
//
// Two kernels.  The first reads every row once, a warp per chunk: the maximum, its first
// place and sum exp((l - max)/T); it is bound by those bytes (256 sequences of 8 rows of
// 73448 floats: 94 us, 6.4 TB/s).  The second (72 us there, no unit full: issue 43%, fp64
// 26%; 1024 blocks in 1.7 waves) takes a cluster of blocks per sequence: it
// joins the chunks, walks the drafts, and samples from the row that ends the walk.  A
// sample depends on cumulative sums next to a border, so that row is summed in double, in
// one pass: per warp's slice of ids S = sum e, and over the ids A whose e / S0 exceeds
// the draft's d (in float, S0 the first kernel's sum) E = sum e and D = sum d.  The
// rest's sum over a slice is then E / S - D; an id that 2^-19 of float error puts on the
// wrong side of A changes it by that much of d.  The slice that holds the goal is
// searched again by its block.
// (One kernel per sequence that stops reading where the walk ends reads half the rows
// at 60% accepted drafts, but its joins follow one another: 187 us against 166 for 256
// sequences of 8 rows of 73448.)
#include "kernels.cuh"
#include "../../include/vc4b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>
#include <type_traits>

namespace vc4 {
namespace {

int vfail(int code, const std::string& msg) { return set_error(code, msg.c_str()); }

constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCtas = 8;           // most blocks of a cluster
constexpr int kVerifySms = 148;          // SMs the block counts are chosen for

struct VerifyPart {       // one slice of one row
    float max, sum;
    int first;            // the first id of max
    int bad;              // a NaN was there
};

struct VerifyArgs {
    int seqs, rows, vocab;
    int chunk_words, chunks;      // 16-byte words of a chunk, chunks of a row
    int words;                    // words of a slice of the sampled row
    const int *cu, *fed;
    const void* logits;
    long long stride, probs_stride;
    const float *probs, *u, *u_sample;
    double inv_t, scale256;       // 1 / temperature (0: greedy), 256 log2 e / temperature
    float scale2;                 // log2 e / temperature
    int *next, *accepted, *status;
    float* prob;
    VerifyPart* part;             // [rows][chunks]
};

template <int T>
__device__ __forceinline__ float logit_at(const void* row, long long i) {
    if (T == VC4_F32) return reinterpret_cast<const float*>(row)[i];
    if (T == VC4_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
    if (T == VC4_F16) return __half2float(reinterpret_cast<const __half*>(row)[i]);
    return __fmul_rn((float)reinterpret_cast<const int*>(row)[i], 1.0f / 256.0f);
}
template <int T> __host__ __device__ constexpr int logit_size() { return T == VC4_BF16 || T == VC4_F16 ? 2 : 4; }

// The values of one aligned 16-byte word.
template <int T>
__device__ __forceinline__ void logit_word(const uint4 w, float (&v)[16 / logit_size<T>()]) {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (T == VC4_F32) v[j] = __uint_as_float(u[j]);
        else if (T == VC4_Q16I) v[j] = __fmul_rn((float)(int)u[j], 1.0f / 256.0f);
        else if (T == VC4_BF16) {
            v[2 * j] = __uint_as_float(u[j] << 16);
            v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}

__device__ __forceinline__ float ex2v(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ double warp_sum_d(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Of 128 sums, four a lane in order, the first whose running sum exceeds the goal (the
// last one with anything in it where rounding puts the goal past the end), and the
// running sum before it; every lane returns them.
__device__ __forceinline__ int warp_choose(const double (&x)[4], double goal, double& before) {
    const int lane = threadIdx.x & 31;
    const double mine = (x[0] + x[1]) + (x[2] + x[3]);
    double upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const unsigned any = __ballot_sync(0xffffffffu, mine > 0.0), over = __ballot_sync(0xffffffffu, mine > 0.0 && upto > goal);
    const int owner = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
    double run = upto - mine;
    int pick = 4 * lane;
    bool done = false;
    before = run;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!done && x[i] > 0.0) {
            pick = 4 * lane + i;
            before = run;
            run += x[i];
            done = run > goal;
        }
    before = __shfl_sync(0xffffffffu, before, owner);
    return __shfl_sync(0xffffffffu, pick, owner);
}

// 2^(y/256), y <= 0: y = k + f, k the nearest integer, 2^(f/256) = exp(r) with
// r = f ln 2/256 by its Taylor polynomial of degree 3 (|r| <= 0.00136, so what is left
// out is r^4/24 < 1.5e-13), 2^((k mod 256)/256) from a table in shared memory: 11
// double operations.  Below 2^-1000, and for NaN, 0.
__device__ __forceinline__ double exp2_256(double y, const double* tab) {
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the low word of y + magic is k
    const bool there = y >= -256000.0;         // (y may be above 0 by a rounding)
    const double t = y + magic, f = y - (t - magic);
    const int k = __double2loint(t);
    constexpr double c1 = 0.69314718055994530942 / 256;
    const double q = f * fma(f, fma(f, c1 * c1 * c1 / 6, c1 * c1 / 2), c1);
    const double b = tab[k & 255], e = fma(b, q, b);
    return there ? __hiloint2double(__double2hiint(e) + ((k >> 8) << 20), __double2loint(e)) : 0.0;
}

// A row on its aligned 16-byte grid: word w holds ids w*VEC - head ..; the first and the
// last may reach over the row's ends.
template <int T>
struct RowWords {
    static constexpr int VEC = 16 / logit_size<T>();
    const char* base;
    const uint4* words;
    int head, vocab, w1;       // w1: the slice's end
    __device__ RowWords(const VerifyArgs& a, int row, int slice, int per, int& w0) {
        base = reinterpret_cast<const char*>(a.logits) + (long long)row * a.stride * logit_size<T>();
        head = (int)(((uintptr_t)base & 15) / logit_size<T>());
        words = reinterpret_cast<const uint4*>(base - head * logit_size<T>());
        vocab = a.vocab;
        w0 = slice * per;
        w1 = min(w0 + per, (head + vocab + VEC - 1) / VEC);
    }
    __device__ __forceinline__ bool whole(int w) const { return w < w1 && w * VEC >= head && (w + 1) * VEC - head <= vocab; }
    __device__ __forceinline__ void values(int w, const uint4& raw, float (&v)[VEC]) const {
        if (whole(w)) logit_word<T>(raw, v);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int at = w * VEC - head + j;
                v[j] = w < w1 && at >= 0 && at < vocab ? logit_at<T>(base, at) : -INFINITY;
            }
    }
};

// One warp: maximum, sum and first maximum of a chunk of a row.  Every lane keeps them
// for its own words (the sum rescaled when the maximum moves, once a word), eight loads
// ahead, and the lanes join at the end.  A sum that came out NaN (a NaN logit, or more
// than one infinity) is taken again value by value.
template <int T>
__device__ __forceinline__ VerifyPart chunk_part(const VerifyArgs& a, int row, int slice) {
    constexpr int VEC = 16 / logit_size<T>(), DEEP = 8;
    const int lane = threadIdx.x & 31;
    int w0;
    const RowWords<T> r(a, row, slice, a.chunk_words, w0);
    const bool greedy = a.inv_t == 0.0;
    float m = -INFINITY, sum = 0.0f;
    int first = 0x7fffffff, bad = 0;
    for (int w = w0 + lane; w < r.w1; w += 32 * DEEP) {
        uint4 raw[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (r.whole(w + 32 * i)) raw[i] = __ldcs(r.words + w + 32 * i);
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            if (w + 32 * i >= r.w1) break;
            float v[VEC];
            r.values(w + 32 * i, raw[i], v);
            float wm = v[0];
#pragma unroll
            for (int j = 1; j < VEC; ++j) wm = fmaxf(wm, v[j]);
            if (greedy) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) bad |= v[j] != v[j];
                if (wm > m) {
                    m = wm;
#pragma unroll
                    for (int j = VEC - 1; j >= 0; --j)
                        if (v[j] == wm) first = (w + 32 * i) * VEC - r.head + j;
                }
            } else {
                // (a lane that has seen nothing has m = -inf; -inf - -inf is kept out)
                const float mn = fmaxf(m, wm), from = mn == -INFINITY ? 0.0f : mn;
                sum *= ex2v(__fmul_rn(__fsub_rn(m, from), a.scale2));
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    s0 += ex2v(__fmul_rn(__fsub_rn(v[j], from), a.scale2));
                    s1 += ex2v(__fmul_rn(__fsub_rn(v[j + 1], from), a.scale2));
                }
                sum += s0 + s1;
                m = mn;
            }
        }
    }
    float top = m;          // (a NaN never is a maximum)
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (greedy) {
        if (m != top || top == -INFINITY) first = 0x7fffffff;
        for (int o = 16; o; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    } else {
        sum *= m == -INFINITY ? 0.0f : m == top ? 1.0f : ex2v(__fmul_rn(__fsub_rn(m, top), a.scale2));
        if (__any_sync(0xffffffffu, sum != sum)) {
            sum = 0.0f;
            for (int w = w0 + lane; w < r.w1; w += 32) {
                float v[VEC];
                r.values(w, r.whole(w) ? __ldg(r.words + w) : make_uint4(0, 0, 0, 0), v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    bad |= v[j] != v[j];
                    if (v[j] == top && top != -INFINITY) sum += 1.0f;   // infinite maxima count one each
                    else if (v[j] == v[j] && v[j] != -INFINITY) sum += ex2v(__fmul_rn(__fsub_rn(v[j], top), a.scale2));
                }
            }
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    return VerifyPart{top, sum, first, __any_sync(0xffffffffu, bad)};
}

template <int T>
__global__ void __launch_bounds__(kVerifyThreads) k_verify_stats(VerifyArgs a) {
    const int task = blockIdx.x * kVerifyWarps + (threadIdx.x >> 5);
    pdl_launch_dependents();
    if (task >= a.rows * a.chunks) return;
    const VerifyPart p = chunk_part<T>(a, task / a.chunks, task % a.chunks);
    if ((threadIdx.x & 31) == 0) a.part[task] = p;
}

template <int T>
__global__ void __launch_bounds__(kVerifyThreads, 4) k_verify_pick(VerifyArgs a) {
    namespace cg = cooperative_groups;
    constexpr int W = kVerifyWarps, VEC = 16 / logit_size<T>();
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double s_tab[256], s_sum[3][W], s_all[3][W * kVerifyCtas], s_rowsum[W], s_goal, s_S;
    __shared__ float s_max[W], s_p[W];
    __shared__ int s_first[W], s_ok[W], s_range;
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int s = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = a.cu[s], c1 = a.cu[s + 1], n = c1 - c0, V = a.vocab;
    s_tab[tid] = exp2((double)tid / 256);
    // this sequence's first row of draft_probs: a row for each of the batch before it, but
    // for the last row of every sequence that has any.  Behind offsets that start below 0 or
    // run backwards nobody knows where it is.
    int dbase = 0;
    bool lost = false;
    if (a.probs) {
        const int first = a.cu[0];
        dbase = c0 - first;
        lost = first < 0;
        for (int j = 0; j < s; j += kVerifyThreads) {
            const int i = min(j + tid, s - 1), lo = a.cu[i], hi = a.cu[i + 1];
            lost |= hi < lo;
            dbase -= __syncthreads_count(j + tid < s && hi > lo);
        }
    }
    const bool writes = rank == 0;
    lost = __syncthreads_or(lost);
    pdl_wait();
    if (c0 < 0 || n <= 0 || c1 > a.rows || lost) {   // every block of the cluster leaves here
        if (tid == 0 && writes) a.accepted[s] = 0;
        if (tid == 0 && (n || c0 < 0 || c1 > a.rows) && a.status) atomicMax(a.status, VC4_EINVAL);   // bad offsets
        return;
    }

    // ---- the walk, W rows at a time, the same in every block ----
    int stop = n - 1, row_first = 0;
    float row_max = 0.0f;
    double row_sum = 0.0;
    for (int i0 = 0; i0 < n; i0 += W) {
        const int m = min(W, n - i0), i = i0 + warp;
        if (warp < m) {      // a warp joins a row
            const bool judge = i < n - 1;
            const int x = judge ? a.fed[c0 + i + 1] : 0;
            const bool in = x >= 0 && x < V;
            const float l = judge && in ? logit_at<T>(reinterpret_cast<const char*>(a.logits) +
                                                      (long long)(c0 + i) * a.stride * logit_size<T>(), x) : 0.0f;
            const float d = judge && in && a.probs ? a.probs[(long long)(dbase + i) * a.probs_stride + x] : 1.0f;
            const float u = judge ? a.u[c0 + i] : 0.0f;
            const VerifyPart* part = a.part + (size_t)(c0 + i) * a.chunks;
            float top = -INFINITY;
            int bad = 0, first = 0x7fffffff;
            for (int c = lane; c < a.chunks; c += 32) {
                top = fmaxf(top, part[c].max);
                bad |= part[c].bad;
            }
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            double sum = 0.0;
            for (int c = lane; c < a.chunks; c += 32) {
                const VerifyPart p = part[c];
                if (p.max == top) {
                    sum += (double)p.sum;
                    first = min(first, p.first);
                } else if (p.max != -INFINITY) {
                    sum += (double)p.sum * exp2_256(((double)p.max - (double)top) * a.scale256, s_tab);
                }
            }
            sum = warp_sum_d(sum);
            for (int o = 16; o; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
            bad = __any_sync(0xffffffffu, bad);
            double q = 0.0;
            if (a.inv_t == 0.0) q = first == x ? 1.0 : 0.0;
            else if (sum > 0.0 && l == l) q = (l == top ? 1.0 : exp2_256(((double)l - (double)top) * a.scale256, s_tab)) / sum;
            if (!in) q = 0.0;
            if (lane == 0) {
                s_max[warp] = top;
                s_rowsum[warp] = sum;
                s_first[warp] = first;
                s_ok[warp] = judge && in && (double)u * (double)d < q;
                s_p[warp] = (float)q;
                if (writes && a.status) {
                    if (!in) atomicMax(a.status, VC4_EINVAL);
                    if (bad) atomicMax(a.status, VC4_ERANGE);
                }
            }
        }
        __syncthreads();
        int j = 0;
        while (j < m && s_ok[j]) ++j;
        if (writes && warp == 0 && lane < j) {
            a.next[c0 + i0 + lane] = a.fed[c0 + i0 + lane + 1];
            if (a.prob) a.prob[c0 + i0 + lane] = s_p[lane];
        }
        if (j < m) {          // the last row of the sequence never accepts, so this is reached
            stop = i0 + j;
            row_max = s_max[j];
            row_sum = s_rowsum[j];
            row_first = s_first[j];
            break;
        }
        __syncthreads();
    }
    const int row = c0 + stop;
    if (writes) {
        for (int i = stop + 1 + tid; i < n; i += kVerifyThreads) {
            a.next[c0 + i] = -1;
            if (a.prob) a.prob[c0 + i] = 0.0f;
        }
        if (tid == 0) a.accepted[s] = stop;
    }
    // no finite logit: nothing to sample; greedy: the first maximum, whatever is left of
    // it (the rest holds nothing else, and where it is empty the row itself is meant)
    if (row_max == -INFINITY || a.inv_t == 0.0) {
        if (tid == 0 && writes) {
            const bool none = row_max == -INFINITY;
            a.next[row] = none ? -1 : row_first;
            if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
            if (none && a.status) atomicMax(a.status, VC4_ERANGE);
        }
        return;
    }

    // ---- the row that is sampled from ----
    int w0;
    const RowWords<T> r(a, row, rank * W + warp, a.words, w0);
    const bool refused = stop < n - 1;
    const float* drow = refused && a.probs ? a.probs + (long long)(dbase + stop) * a.probs_stride : nullptr;
    const int cut = refused && !a.probs ? a.fed[row + 1] : -1;
    // exp((l - max)/T), the difference taken first: the maximum's weight is 1 however large
    // it is.  Infinite maxima take all, in equal parts.
    const bool endless = row_max == INFINITY;
    const double scale = a.scale256, most = endless ? 0.0 : (double)row_max;
    auto weight = [&](float l) -> double {
        if (endless) l = l == row_max ? 0.0f : -INFINITY;
        return exp2_256(((double)l - most) * scale, s_tab);
    };
    const float inv0 = (float)(1.0 / row_sum);
    const bool dvec = (((uintptr_t)drow - 4 * r.head) & 15) == 0;   // words of logits meet 16-byte pieces of d
    double S = 0.0, E = 0.0, D = 0.0;
    auto pass = [&](auto which) {         // 0: from the row, 1: less id `cut`, 2: less d
        constexpr int rule = decltype(which)::value;
        constexpr int DEEP = VEC == 4 ? 4 : 2;       // words whose loads go out together
        for (int w = w0 + lane; w < r.w1; w += 32 * DEEP) {
            uint4 raw[DEEP];
            float d[DEEP][VEC];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int wk = w + 32 * k, at = wk * VEC - r.head;
                const bool whole = r.whole(wk);
                raw[k] = whole ? __ldg(r.words + wk) : make_uint4(0, 0, 0, 0);
                if (rule == 2 && whole && dvec) {
#pragma unroll
                    for (int j = 0; j < VEC; j += 4) {
                        const float4 f = __ldg(reinterpret_cast<const float4*>(drow + at + j));
                        d[k][j] = f.x;
                        d[k][j + 1] = f.y;
                        d[k][j + 2] = f.z;
                        d[k][j + 3] = f.w;
                    }
                } else if (rule == 2) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) d[k][j] = wk < r.w1 && at + j >= 0 && at + j < V ? __ldg(drow + at + j) : 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int wk = w + 32 * k;
                if (wk >= r.w1) break;
                float l[VEC];
                r.values(wk, raw[k], l);
                if (endless) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) l[j] = l[j] == row_max ? 0.0f : -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const double e = exp2_256(((double)l[j] - most) * scale, s_tab);
                    S += e;
                    if (rule == 1 && wk * VEC - r.head + j != cut) E += e;
                    if (rule == 2 && (float)e * inv0 > d[k][j]) {
                        E += e;
                        D += (double)d[k][j];
                    }
                }
            }
        }
    };
    if (drow) pass(std::integral_constant<int, 2>());
    else if (refused) pass(std::integral_constant<int, 1>());
    else pass(std::integral_constant<int, 0>());
    S = warp_sum_d(S);
    E = warp_sum_d(E);
    D = warp_sum_d(D);
    if (lane == 0) {
        s_sum[0][warp] = S;
        s_sum[1][warp] = E;
        s_sum[2][warp] = D;
    }
    cluster.sync();
    for (int i = tid; i < 3 * W * C; i += kVerifyThreads) {    // every block holds all sums
        const int k = i / (W * C), e = i % (W * C);
        s_all[k][e] = cluster.map_shared_rank(&s_sum[k][0], e / W)[e % W];
    }
    cluster.sync();            // its own sums were read by all: a block may leave after this
    if (warp == 0) {
        double whole[4], rest[4], all = 0.0, total = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * lane + i;
            whole[i] = e < W * C ? s_all[0][e] : 0.0;
            all += whole[i];
        }
        all = warp_sum_d(all);
        const double inv = 1.0 / all;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * lane + i;
            rest[i] = e < W * C && refused ? fmax(drow ? s_all[1][e] * inv - s_all[2][e] : s_all[1][e], 0.0) : 0.0;
            total += rest[i];
        }
        total = warp_sum_d(total);
        const bool some = total > 0.0;                         // else from the row itself
#pragma unroll
        for (int i = 0; i < 4; ++i) rest[i] = some ? rest[i] : whole[i];
        const double goal = (double)a.u_sample[s] * (some ? total : all);
        double before;
        const int pick = warp_choose(rest, goal, before);
        if (lane == 0) {
            s_range = some ? pick : ~pick;
            s_goal = goal - before;
            s_S = all;
        }
    }
    __syncthreads();
    const bool some = s_range >= 0;
    const int range = some ? s_range : ~s_range;
    if (range / W != rank) return;
    const double inv = 1.0 / s_S;
    auto value = [&](int v) -> double {
        const double w = weight(logit_at<T>(r.base, v));
        if (!some) return w;
        if (drow) return fmax(w * inv - (double)drow[v], 0.0);
        return v == cut ? 0.0 : w;
    };
    const int per = a.words * VEC;
    int x0 = min(V, max(0, range * per - r.head)), x1 = min(V, max(0, (range + 1) * per - r.head));
    double goal = s_goal;
    if (per > 8 * 32) {        // narrowed by all warps first
        const int step = (per + W - 1) / W, v0 = min(x1, x0 + warp * step), v1 = min(x1, v0 + step);
        double mine = 0.0;
        for (int v = v0 + lane; v < v1; v += 32) mine += value(v);
        mine = warp_sum_d(mine);
        if (lane == 0) s_sum[0][warp] = mine;                  // (read by no other block any more)
        __syncthreads();
        double part[4], before;
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = 4 * lane + i < W ? s_sum[0][4 * lane + i] : 0.0;
        const int sub = warp_choose(part, goal, before);
        goal -= before;
        x0 = min(x1, x0 + sub * step);
        x1 = min(x1, x0 + step);
    }
    if (warp) return;
    double run = 0.0;
    int last = -1;                                             // the last id with any weight
    for (int base = x0; base < x1; base += 32) {
        const int v = base + lane;
        const double x = v < x1 ? value(v) : 0.0;
        double sum = x;
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, x > 0.0 && run + sum > goal), any = __ballot_sync(0xffffffffu, x > 0.0);
        if (any) last = base + (over ? __ffs(over) - 1 : 31 - __clz(any));
        if (over) break;
        run += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
        a.next[row] = last;
        if (a.prob) a.prob[row] = last >= 0 ? (float)(weight(logit_at<T>(r.base, last)) * inv) : 0.0f;
    }
}

// Logits of a chunk: 4096, 1024 while that many leave the GPU's warps (32 on an SM)
// without work.
int verify_chunk(int rows, int vocab) { return (long long)rows * vocab < 4096LL * 32 * kVerifySms ? 1024 : 4096; }
int verify_chunks(int rows, int vocab) {   // 7: the words' overhang at the row's start
    const int c = verify_chunk(rows, vocab);
    return (int)(((long long)vocab + 7 + c - 1) / c);
}

std::string bad_sizes(int seqs, int rows, int vocab) {
    if (seqs <= 0 || rows < 0 || vocab <= 0) return "seqs and vocab must be positive, rows not negative";
    if (seqs > (1 << 24) || vocab > (1 << 30) || (long long)rows * verify_chunks(rows, vocab) > 0x7fffffffLL)
        return "too many sequences, rows or ids in one call";
    return "";
}

template <int T>
void launch_verify(VerifyArgs a, cudaStream_t st) {
    constexpr int VEC = 16 / logit_size<T>();
    a.chunk_words = verify_chunk(a.rows, a.vocab) / VEC;
    k_verify_stats<T><<<(unsigned)(((long long)a.rows * a.chunks + kVerifyWarps - 1) / kVerifyWarps), kVerifyThreads, 0, st>>>(a);
    // Blocks per sequence: up to eight for each SM, with 1024 ids or more each (256
    // sequences of 73448: 1, 2, 4, 8 blocks 234, 174, 166, 174 us; 61: 86, 54, 43, 35;
    // one of 6400: 16.7, 13.2, 13.1, 12.9).
    int c = 1;
    while (c < kVerifyCtas && 2 * c * a.seqs <= 8 * kVerifySms && a.vocab > 1024 * c) c *= 2;
    const long long words = ((long long)a.vocab + 2 * VEC - 2) / VEC;   // with the widest head
    a.words = (int)((words + c * kVerifyWarps - 1) / (c * kVerifyWarps));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.seqs * c));
    cfg.blockDim = dim3(kVerifyThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)c;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_verify_pick<T>, a);
}

}  // namespace
}  // namespace vc4

using namespace vc4;

extern "C" int vc4_verify_draft_bytes(int seqs, int rows, int vocab, size_t* bytes) {
    const std::string m = bad_sizes(seqs, rows, vocab);
    if (!m.empty()) return vfail(VC4_EINVAL, "verify_draft_bytes: " + m);
    if (!bytes) return vfail(VC4_EINVAL, "verify_draft_bytes: bytes is null");
    *bytes = (size_t)rows * verify_chunks(rows, vocab) * sizeof(VerifyPart);
    return VC4_OK;
}

extern "C" int vc4_verify_draft(vc4_gpu* g, int seqs, int rows, int vocab, const int* cu, const int* fed,
                                const void* logits, int logits_type, long long logits_stride, const float* draft_probs,
                                long long probs_stride, double temperature, const float* u, const float* u_sample,
                                int* next, int* accepted, float* prob, int* status, void* work, size_t work_bytes,
                                void* stream) {
    auto refuse = [](const std::string& m) { return vfail(VC4_EINVAL, "verify_draft: " + m); };
    const std::string m = bad_sizes(seqs, rows, vocab);
    if (!m.empty()) return refuse(m);
    if (logits_type < VC4_F32 || logits_type > VC4_Q16I) return refuse("unknown logits type");
    if (!logits_stride) logits_stride = vocab;
    if (!probs_stride) probs_stride = vocab;
    if (logits_stride < vocab || probs_stride < vocab) return refuse("a stride is below the vocabulary");
    // (below this the logits' products with 1/T would leave double's whole numbers)
    if (!(temperature == 0.0 || temperature >= 1e-5) || !(temperature < INFINITY))
        return refuse("temperature must be 0 or at least 1e-5");
    if (!cu || !fed || !logits || !u || !u_sample || !next || !accepted) return refuse("a required array is null");
    const int es = logits_type == VC4_BF16 || logits_type == VC4_F16 ? 2 : 4;
    const void* words[] = {cu, fed, draft_probs, u, u_sample, next, accepted, prob, status};
    bool aligned = (uintptr_t)logits % es == 0;
    for (const void* w : words) aligned = aligned && (uintptr_t)w % 4 == 0;
    if (!aligned) return refuse("an array is not aligned to its elements");
    const size_t need = (size_t)rows * verify_chunks(rows, vocab) * sizeof(VerifyPart);
    if (work_bytes < need || (need && (!work || (uintptr_t)work % 16)))
        return refuse("the work buffer needs " + std::to_string(need) + " bytes at a multiple of 16");
    {   // the blocks of a sequence all read the inputs while one of them writes
        struct Span { const void* at; size_t bytes; };
        const size_t r = (size_t)rows, n = (size_t)seqs, whole = r > n ? (r - n - 1) * (size_t)probs_stride * 4 + (size_t)vocab * 4 : 0;
        const Span in[] = {{cu, 4 * (n + 1)}, {fed, 4 * r}, {u, 4 * r}, {u_sample, 4 * n},
                           {draft_probs, whole}, {logits, r ? ((r - 1) * (size_t)logits_stride + vocab) * es : 0}};
        const Span out[] = {{next, 4 * r}, {accepted, 4 * n}, {prob, 4 * r}, {status, 4}, {work, need}};
        auto meet = [](const Span& x, const Span& y) {
            const uintptr_t a0 = (uintptr_t)x.at, b0 = (uintptr_t)y.at;
            return a0 && b0 && a0 < b0 + y.bytes && b0 < a0 + x.bytes;
        };
        for (const Span& o : out) {
            for (const Span& i : in)
                if (meet(o, i)) return refuse("an output overlaps an input");
            for (const Span& w : out)
                if (&w != &o && meet(o, w)) return refuse("two outputs overlap");
        }
    }
    if (!g) return refuse("gpu is null");
    int before = -1;
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != gpu_device(g)) e = cudaSetDevice(gpu_device(g));
    else before = -1;
    if (e != cudaSuccess) return vfail(VC4_ECUDA, cudaGetErrorString(e));
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : gpu_stream(g);
    if (!rows) {     // no sequence has a row: none accepts a draft
        e = cudaMemsetAsync(accepted, 0, (size_t)seqs * sizeof(int), st);
        if (before >= 0) cudaSetDevice(before);
        return e == cudaSuccess ? VC4_OK : vfail(VC4_ECUDA, std::string("verify_draft: ") + cudaGetErrorString(e));
    }
    VerifyArgs a{};
    a.seqs = seqs; a.rows = rows; a.vocab = vocab;
    a.cu = cu; a.fed = fed; a.logits = logits; a.stride = logits_stride; a.probs_stride = probs_stride;
    a.probs = draft_probs; a.u = u; a.u_sample = u_sample; a.next = next; a.accepted = accepted; a.status = status;
    a.prob = prob; a.part = (VerifyPart*)work; a.chunks = verify_chunks(rows, vocab);
    a.inv_t = temperature > 0.0 ? 1.0 / temperature : 0.0;
    a.scale2 = (float)(1.4426950408889634 * a.inv_t);
    a.scale256 = 1.44269504088896340736 * 256 * a.inv_t;
    switch (logits_type) {
        case VC4_F32: launch_verify<VC4_F32>(a, st); break;
        case VC4_BF16: launch_verify<VC4_BF16>(a, st); break;
        case VC4_F16: launch_verify<VC4_F16>(a, st); break;
        default: launch_verify<VC4_Q16I>(a, st); break;
    }
    e = cudaGetLastError();
    if (before >= 0) cudaSetDevice(before);
    if (e != cudaSuccess) return vfail(VC4_ECUDA, std::string("verify_draft: ") + cudaGetErrorString(e));
    return VC4_OK;
}
