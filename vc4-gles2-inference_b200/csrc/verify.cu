// verify.cu -- verification of drafted tokens against the target's probabilities.
//
// Two kernels.  The first reads every row of logits once: per row and chunk the
// maximum, its first place and sum exp((l - max)/T), the chunk's own maximum as
// base.  The second takes one block per sequence: it joins the chunks, walks the
// drafts, and samples from the row that ends the walk.  The samples depend on
// cumulative sums next to a border, so that row is summed in double: the total S,
// the rest max(p - d, 0), then a search that halves nothing but places: 32 warps'
// ranges, 32 sub-ranges of the one that holds the goal, 32 lanes of that one.
#include "kernels.cuh"
#include "../../include/vc4b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

namespace vc4 {
namespace {

int vfail(int code, const std::string& msg) { return set_error(code, msg.c_str()); }

constexpr int kVerifyChunk = 8192;       // logits of a row per block of the first kernel
constexpr int kStatThreads = 256;
constexpr int kPickThreads = 1024;

struct VerifyPart {       // one chunk of one row
    float max, sum;
    int first;            // the first place of max
    int bad;              // a NaN was there
};

struct VerifyArgs {
    int seqs, rows, vocab, chunks;
    const int *cu, *fed;
    const void* logits;
    long long stride, probs_stride;
    const float *probs, *u, *u_sample;
    double inv_t;                 // 1 / temperature; 0: greedy
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
// exp((l - m) / T), the limit for infinities: the row's +inf maxima count one
__device__ __forceinline__ float rel_exp(float l, float m, float scale2) {
    return l == m ? 1.0f : ex2v(__fmul_rn(__fsub_rn(l, m), scale2));
}
__device__ __forceinline__ double rel_exp_d(float l, float m, double inv_t) {
    return l == m ? 1.0 : exp(((double)l - (double)m) * inv_t);
}

template <int T>
__global__ void __launch_bounds__(kStatThreads) k_verify_stats(VerifyArgs a) {
    constexpr int VEC = 16 / logit_size<T>(), PER = kVerifyChunk / (kStatThreads * VEC);
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    pdl_launch_dependents();
    const char* base = reinterpret_cast<const char*>(a.logits) + (long long)row * a.stride * logit_size<T>();
    // words of the row's aligned 16-byte grid: the first and last may reach over its ends
    const int head = (int)(((uintptr_t)base & 15) / logit_size<T>());
    const uint4* words = reinterpret_cast<const uint4*>(base - head * logit_size<T>());
    const int nwords = (head + a.vocab + VEC - 1) / VEC;
    const int w0 = chunk * (kVerifyChunk / VEC);
    float v[PER][VEC];
    float m = -INFINITY;
    int bad = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int w = w0 + i * kStatThreads + threadIdx.x, at = w * VEC - head;
        if (w < nwords && at >= 0 && at + VEC <= a.vocab) logit_word<T>(__ldcs(words + w), v[i]);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                v[i][j] = w < nwords && at + j >= 0 && at + j < a.vocab ? logit_at<T>(base, at + j) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (v[i][j] != v[i][j]) {
                v[i][j] = -INFINITY;
                bad = 1;
            }
            m = fmaxf(m, v[i][j]);
        }
    __shared__ float s_m[kStatThreads / 32], s_sum[kStatThreads / 32];
    __shared__ int s_first[kStatThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_m[warp] = m;
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < kStatThreads / 32; ++w) m = fmaxf(m, s_m[w]);
    float sum = 0.0f;
    int first = 0x7fffffff;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
#pragma unroll
        for (int j = VEC - 1; j >= 0; --j) {
            if (v[i][j] == m) first = (w0 + i * kStatThreads + (int)threadIdx.x) * VEC - head + j;
            if (m != -INFINITY) sum += rel_exp(v[i][j], m, a.scale2);
        }
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    }
    if (lane == 0) {
        s_sum[warp] = sum;
        s_first[warp] = first;
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        for (int w = 1; w < kStatThreads / 32; ++w) {
            sum += s_sum[w];
            first = min(first, s_first[w]);
        }
        a.part[blockIdx.x] = VerifyPart{m, sum, first, bad};
    }
}

// A row's chunks joined, by one warp.
struct RowStat {
    float max;
    double sum;
    int first;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, int row) {
    const int lane = threadIdx.x & 31;
    RowStat r{-INFINITY, 0.0, 0x7fffffff};
    for (int c = lane; c < a.chunks; c += 32) r.max = fmaxf(r.max, a.part[(size_t)row * a.chunks + c].max);
    for (int o = 16; o; o >>= 1) r.max = fmaxf(r.max, __shfl_xor_sync(0xffffffffu, r.max, o));
    for (int c = lane; c < a.chunks; c += 32) {
        const VerifyPart p = a.part[(size_t)row * a.chunks + c];
        if (p.max == -INFINITY) continue;
        r.sum += (double)p.sum * rel_exp_d(p.max, r.max, a.inv_t);
        if (p.max == r.max) r.first = min(r.first, p.first);
    }
    for (int o = 16; o; o >>= 1) {
        r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
        r.first = min(r.first, __shfl_xor_sync(0xffffffffu, r.first, o));
    }
    return r;
}

__device__ __forceinline__ double warp_sum_d(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int T>
__global__ void __launch_bounds__(kPickThreads) k_verify_pick(VerifyArgs a) {
    pdl_wait();
    constexpr int W = kPickThreads / 32;
    __shared__ double s_d[W], s_total, s_goal;
    __shared__ float s_max[W], s_p[W];
    __shared__ int s_first[W], s_ok[W], s_stop, s_lo, s_hi;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = a.cu[s], c1 = min(a.cu[s + 1], a.rows), n = c1 - c0, V = a.vocab;
    // this sequence's first row of draft_probs: a row for each before it, but for
    // the last row of every sequence that has any
    int dbase = c0;
    if (a.probs)
        for (int j = 0; j < s; j += kPickThreads)
            dbase -= __syncthreads_count(j + tid < s && a.cu[j + tid + 1] > a.cu[j + tid]);
    if (c0 < 0 || n <= 0 || dbase < 0) {
        if (tid == 0) a.accepted[s] = 0;
        if (tid == 0 && n > 0 && a.status) atomicMax(a.status, VC4_EINVAL);   // offsets that run backwards
        return;
    }
    // the walk over the drafts, W rows at a time
    int stop = n - 1;
    float row_max = 0.0f;
    int row_first = 0;
    for (int i0 = 0; i0 < n; i0 += W) {
        const int i = i0 + warp;
        if (i < n) {
            const RowStat st = row_stat(a, c0 + i);
            int ok = 0;
            float px = 0.0f;
            if (i < n - 1) {
                const int x = a.fed[c0 + i + 1];
                const bool in = x >= 0 && x < V;
                if (!in && lane == 0 && a.status) atomicMax(a.status, VC4_EINVAL);
                double p = 0.0;
                if (in && a.inv_t == 0.0) p = st.first == x ? 1.0 : 0.0;
                else if (in && st.sum > 0.0) {
                    const float l = logit_at<T>(reinterpret_cast<const char*>(a.logits) +
                                                (long long)(c0 + i) * a.stride * logit_size<T>(), x);
                    p = l == l ? rel_exp_d(l, st.max, a.inv_t) / st.sum : 0.0;
                }
                const double d = a.probs && in ? (double)a.probs[(long long)(dbase + i) * a.probs_stride + x] : 1.0;
                ok = (double)a.u[c0 + i] * d < p;
                px = (float)p;
            }
            if (lane == 0) {
                s_max[warp] = st.max;
                s_first[warp] = st.first;
                s_ok[warp] = ok;
                s_p[warp] = px;
            }
        }
        __syncthreads();
        if (tid == 0) {
            int j = 0;
            const int m = min(W, n - i0);
            while (j < m && s_ok[j]) ++j;
            s_stop = j;
        }
        __syncthreads();
        const int j = s_stop;
        if (warp == 0 && lane < j) {
            a.next[c0 + i0 + lane] = a.fed[c0 + i0 + lane + 1];
            if (a.prob) a.prob[c0 + i0 + lane] = s_p[lane];
        }
        if (j < min(W, n - i0)) {     // the last row of the sequence never accepts, so this is reached
            stop = i0 + j;
            row_max = s_max[j];
            row_first = s_first[j];
            break;
        }
        __syncthreads();
    }
    for (int i = stop + 1 + tid; i < n; i += kPickThreads) {
        a.next[c0 + i] = -1;
        if (a.prob) a.prob[c0 + i] = 0.0f;
    }
    if (tid == 0) a.accepted[s] = stop;

    // the row that is sampled from
    const int row = c0 + stop;
    const char* lrow = reinterpret_cast<const char*>(a.logits) + (long long)row * a.stride * logit_size<T>();
    const bool refused = stop < n - 1;
    const float* drow = refused && a.probs ? a.probs + (long long)(dbase + stop) * a.probs_stride : nullptr;
    const int cut = refused && !a.probs ? a.fed[row + 1] : -1;
    if (row_max == -INFINITY) {       // no finite logit: nothing to sample
        if (tid == 0) {
            a.next[row] = -1;
            if (a.prob) a.prob[row] = 0.0f;
            if (a.status) atomicMax(a.status, VC4_ERANGE);
        }
        return;
    }
    auto weight = [&](int v) -> double {      // exp((l - max)/T), greedy: the first maximum
        if (a.inv_t == 0.0) return v == row_first ? 1.0 : 0.0;
        const float l = logit_at<T>(lrow, v);
        return l == l ? rel_exp_d(l, row_max, a.inv_t) : 0.0;
    };
    const int per = (V + W - 1) / W;          // warp w's ids: [w*per, (w+1)*per)
    const int b0 = min(V, warp * per), b1 = min(V, b0 + per);
    auto block_total = [&](double mine) {     // every warp's sum in s_d, the total to all
        mine = warp_sum_d(mine);
        __syncthreads();
        if (lane == 0) s_d[warp] = mine;
        __syncthreads();
        double t = 0.0;
        for (int w = 0; w < W; ++w) t += s_d[w];
        return t;
    };
    double mine = 0.0;
    for (int v = b0 + lane; v < b1; v += 32) mine += weight(v);
    const double S = block_total(mine);
    bool rest = refused;                      // sample from the rest, unless that is empty
    auto value = [&](int v) -> double {
        const double w = weight(v);
        if (!rest) return w;
        if (drow) return fmax(w / S - (double)drow[v], 0.0);
        return v == cut ? 0.0 : w;
    };
    double total = S;
    if (refused) {
        mine = 0.0;
        for (int v = b0 + lane; v < b1; v += 32) mine += value(v);
        total = block_total(mine);
        if (!(total > 0.0)) {
            rest = false;
            mine = 0.0;
            for (int v = b0 + lane; v < b1; v += 32) mine += weight(v);
            total = block_total(mine);
        }
    }
    // the range of s_d that holds the goal: the first whose running sum exceeds it
    auto choose = [&](int lo, int hi, int step, double goal) {   // thread 0
        double run = 0.0;
        int pick = -1;
        double before = 0.0;
        for (int w = 0; w < W && lo + w * step < hi; ++w) {
            if (s_d[w] > 0.0) {
                pick = w;            // the last range with anything in it, should rounding miss the goal
                before = run;
                if (run + s_d[w] > goal) break;
            }
            run += s_d[w];
        }
        s_goal = goal - before;
        s_lo = lo + max(0, pick) * step;
        s_hi = min(hi, s_lo + step);
    };
    if (tid == 0) choose(0, V, per, (double)a.u_sample[s] * total);
    __syncthreads();
    while (s_hi - s_lo > 32) {
        const int lo = s_lo, hi = s_hi, step = max(32, (hi - lo + W - 1) / W);
        const int r0 = min(hi, lo + warp * step), r1 = min(hi, r0 + step);
        const double goal = s_goal;
        mine = 0.0;
        for (int v = r0 + lane; v < r1; v += 32) mine += value(v);
        block_total(mine);
        if (tid == 0) choose(lo, hi, step, goal);
        __syncthreads();
    }
    if (warp == 0) {
        const int v = s_lo + lane;
        const double x = v < s_hi ? value(v) : 0.0;
        double run = x;
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, x > 0.0 && run > s_goal), any = __ballot_sync(0xffffffffu, x > 0.0);
        const int k = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
        if (lane == k) {
            a.next[row] = v;
            if (a.prob) a.prob[row] = (float)(weight(v) / S);
        }
    }
    for (int i = tid; i < n * a.chunks; i += kPickThreads)
        if (a.part[(size_t)c0 * a.chunks + i].bad && a.status) atomicMax(a.status, VC4_ERANGE);
}

int verify_chunks(int vocab) { return (vocab + 15 + kVerifyChunk - 1) / kVerifyChunk; }   // 15: the words' overhang

std::string bad_sizes(int seqs, int rows, int vocab) {
    if (seqs <= 0 || rows < 0 || vocab <= 0) return "seqs and vocab must be positive, rows not negative";
    if ((long long)rows * verify_chunks(vocab) > 0x7fffffffLL) return "too many rows in one call";
    return "";
}

template <int T>
void launch_verify(const VerifyArgs& a, cudaStream_t st) {
    k_verify_stats<T><<<(unsigned)(a.rows * a.chunks), kStatThreads, 0, st>>>(a);
    launch_pdl_block(k_verify_pick<T>, dim3((unsigned)a.seqs), kPickThreads, 0, st, a);
}

}  // namespace
}  // namespace vc4

using namespace vc4;

extern "C" int vc4_verify_draft_bytes(int seqs, int rows, int vocab, size_t* bytes) {
    const std::string m = bad_sizes(seqs, rows, vocab);
    if (!m.empty()) return vfail(VC4_EINVAL, "verify_draft_bytes: " + m);
    if (!bytes) return vfail(VC4_EINVAL, "verify_draft_bytes: bytes is null");
    *bytes = (size_t)rows * verify_chunks(vocab) * sizeof(VerifyPart);
    return VC4_OK;
}

extern "C" int vc4_verify_draft(vc4_gpu* g, int seqs, int rows, int vocab, const int* cu, const int* fed,
                                const void* logits, int logits_type, long long logits_stride, const float* draft_probs,
                                long long probs_stride, float temperature, const float* u, const float* u_sample,
                                int* next, int* accepted, float* prob, int* status, void* work, size_t work_bytes,
                                void* stream) {
    auto refuse = [](const std::string& m) { return vfail(VC4_EINVAL, "verify_draft: " + m); };
    const std::string m = bad_sizes(seqs, rows, vocab);
    if (!m.empty()) return refuse(m);
    if (logits_type < VC4_F32 || logits_type > VC4_Q16I) return refuse("unknown logits type");
    if (!logits_stride) logits_stride = vocab;
    if (!probs_stride) probs_stride = vocab;
    if (logits_stride < vocab || probs_stride < vocab) return refuse("a stride is below the vocabulary");
    if (!(temperature >= 0.0f) || !(temperature < INFINITY)) return refuse("temperature must not be negative");
    if (!cu || !fed || !logits || !u || !u_sample || !next || !accepted) return refuse("a required array is null");
    const int es = logits_type == VC4_BF16 || logits_type == VC4_F16 ? 2 : 4;
    if ((uintptr_t)logits % es || (uintptr_t)draft_probs % 4) return refuse("an array is not aligned to its elements");
    const size_t need = (size_t)rows * verify_chunks(vocab) * sizeof(VerifyPart);
    if (work_bytes < need || (need && (!work || (uintptr_t)work % 16)))
        return refuse("the work buffer needs " + std::to_string(need) + " bytes at a multiple of 16");
    if (!g) return refuse("gpu is null");
    if (!rows) return VC4_OK;
    int before = -1;
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != gpu_device(g)) e = cudaSetDevice(gpu_device(g));
    else before = -1;
    if (e != cudaSuccess) return vfail(VC4_ECUDA, cudaGetErrorString(e));
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : gpu_stream(g);
    VerifyArgs a{};
    a.seqs = seqs; a.rows = rows; a.vocab = vocab; a.chunks = verify_chunks(vocab);
    a.cu = cu; a.fed = fed; a.logits = logits; a.stride = logits_stride; a.probs_stride = probs_stride;
    a.probs = draft_probs; a.u = u; a.u_sample = u_sample; a.next = next; a.accepted = accepted; a.status = status;
    a.prob = prob; a.part = (VerifyPart*)work;
    a.inv_t = temperature > 0.0f ? 1.0 / (double)temperature : 0.0;
    a.scale2 = (float)(1.4426950408889634 * a.inv_t);
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
