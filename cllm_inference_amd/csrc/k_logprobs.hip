// k_logprobs.hip -- log probabilities from logits: of a given token per row, with its rank, the
// row's entropy and log-sum-exp, and the most likely tokens, in one pass over the logits.
//
//   m = max x,  S = sum exp(x - m),  lse = m + log S,  logprob(t) = (x_t - m) - log S,
//   entropy = log S + sum (m - x) exp(x - m) / S.
// S is held as 1 + S', the sum without one of its largest terms, so that log S = log1p(S') and the
// entropy keep their relative precision where one token has nearly all of the probability; every
// term of the entropy is positive.
//
// What bounds it: the read of the logits. A workgroup takes 8192 logits of one row (grid rows x
// parts) and holds them in registers, 32 a thread, all loads in flight at once: its maximum first,
// then its sums, the tokens ahead of the given one and its largest logits, without reading twice.
// A second launch joins a row's parts.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device_utils.h"
#include "kv4.h"

namespace cllm_hip {
namespace {

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kVecs = 8;                            // four logits each
constexpr int kPart = kThreads * kVecs * 4;         // logits of a part
constexpr int kCand = 1024;                         // candidates a part ranks in LDS
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();

// A part's results: its maximum; the sum of exp(x - max) over the logits below it and how many
// equal it; the sum of (max - x) exp(x - max); how many tokens stand ahead of the given one.
struct Part {
    float max, sum, ent;
    int equal, ahead, pad[3];
};

// Order of the logits: larger first, -0 as 0, NaN behind -inf; absent elements have key 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    if (x != x) return 1u;
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    if (key <= 1u) return __builtin_nanf("");
    return __builtin_bit_cast(float, (key >> 31) ? key & 0x7FFFFFFFu : ~key);
}
// With the token's index: equal logits stand in the order of their ids.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) {
    return ((uint64_t)key << 32) | (uint32_t)~id;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// The wave's 64 values in descending order, lane i the i-th (bitonic).
__device__ __forceinline__ float wave_sort(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float o = __shfl_xor(v, j, 64);
            const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
            v = keep_max ? fmaxf(v, o) : fminf(v, o);
        }
    }
    return v;
}

// Sum over the workgroup, in every thread; buf: a value per wave, free to write.
__device__ __forceinline__ int block_sum(int v, int* buf) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += buf[w];
    return v;
}

// top: [rows][parts][top_k] entries, each part's in descending order, 0 where the part has fewer.
__global__ __launch_bounds__(kThreads) void k_logprobs_part(const float* __restrict__ logits, int64_t stride, int vocab,
                                                            const int32_t* __restrict__ tokens, int top_k, int parts,
                                                            Part* __restrict__ part, uint64_t* __restrict__ top) {
    __shared__ float s_f[4][kWaves];
    __shared__ int s_i[2][kWaves];
    __shared__ int s_count;
    __shared__ uint64_t s_cand[kCand];
    const int row = blockIdx.x / parts, z = blockIdx.x % parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x0 = logits + (int64_t)row * stride;
    const int base = z * kPart;
    const int n = min(kPart, vocab - base);
    if (tid == 0) s_count = 0;

    // -inf past the row's end: adds nothing to a sum, and candidates check the index
    float x[kVecs][4];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = (i * kThreads + tid) * 4;
        if (at + 4 <= n) {
            const f32x4_a4 v = *(const f32x4_a4*)(x0 + base + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = at + j < n ? x0[base + at + j] : kNegInf;
        }
    }
    const int tok = tokens ? tokens[row] : -1;
    const bool have = (unsigned)tok < (unsigned)vocab;
    const float xt = have ? x0[tok] : 0.0f;

    float tmax = kNegInf;  // (NaN never wins)
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) tmax = fmaxf(tmax, x[i][j]);
    const float wmax = wave_max(tmax);
    // a bound that at least top_k of the part's logits reach: each wave's (top_k / 4)-th largest
    // thread maximum is reached by a quarter of them in every wave, its top_k-th by all of them
    float b_all = kNegInf, b_own = kNegInf;
    if (top_k > 0) {
        const float sorted = wave_sort(tmax, lane);
        b_all = __shfl(sorted, (top_k + kWaves - 1) / kWaves - 1, 64);
        b_own = __shfl(sorted, top_k - 1, 64);
    }
    if (lane == 0) {
        s_f[0][wave] = wmax;
        s_f[1][wave] = b_all;
        s_f[2][wave] = b_own;
    }
    __syncthreads();
    float m = s_f[0][0], bound = s_f[1][0], own = s_f[2][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        m = fmaxf(m, s_f[0][w]);
        bound = fminf(bound, s_f[1][w]);
        own = fmaxf(own, s_f[2][w]);
    }
    bound = fmaxf(bound, own);
    const float mu = m == kNegInf ? 0.0f : m;  // (no logit above -inf)

    float sum = 0.0f, ent = 0.0f;
    int equal = 0, ahead = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (exp of -200 and less is 0; NaN passes both selects)
            const float d = x[i][j] - mu;
            const float e = __builtin_amdgcn_exp2f(d * kLog2e);
            equal += d == 0.0f;
            sum += d == 0.0f ? 0.0f : e;
            ent -= (d < -200.0f ? 0.0f : d) * e;
        }
    }
    if (have) {
        const uint32_t kt = key_of(xt);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (i * kThreads + tid) * 4 + j;
                const uint32_t k = key_of(x[i][j]);
                ahead += at < n && (k > kt || (k == kt && base + at < tok));
            }
        }
    }
    sum = wave_sum(sum);
    ent = wave_sum(ent);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        equal += __shfl_xor(equal, d, 64);
        ahead += __shfl_xor(ahead, d, 64);
    }
    __syncthreads();
    if (lane == 0) {
        s_f[0][wave] = sum;
        s_f[1][wave] = ent;
        s_i[0][wave] = equal;
        s_i[1][wave] = ahead;
    }

    // candidates: the logits at the bound or above
    if (top_k > 0) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (i * kThreads + tid) * 4 + j;
                if (x[i][j] >= bound && at < n) {
                    const int c = atomicAdd(&s_count, 1);
                    if (c < kCand) s_cand[c] = entry_of(key_of(x[i][j]), base + at);
                }
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        Part p;
        p.max = m;
        p.sum = p.ent = 0.0f;
        p.equal = p.ahead = 0;
        for (int w = 0; w < kWaves; ++w) {
            p.sum += s_f[0][w];
            p.ent += s_f[1][w];
            p.equal += s_i[0][w];
            p.ahead += s_i[1][w];
        }
        part[(int64_t)row * parts + z] = p;
    }
    if (top_k == 0) return;
    uint64_t* out = top + ((int64_t)row * parts + z) * top_k;
    int count = s_count;
    const int want = min(top_k, n);
    if (count > kCand) {
        // Many logits equal the bound (a mask's -inf, a coarse grid of values): of those only the
        // first by index can be wanted. The index below which top_k of them lie, by bisection.
        int lo = 0, hi = kPart, above = 0;
        for (int step = 0; step < 14; ++step) {
            const int mid = step == 0 ? 0 : (lo + hi) >> 1;  // (first: the logits above the bound)
            int k = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = (i * kThreads + tid) * 4 + j;
                    k += at < n && (step == 0 ? x[i][j] > bound : x[i][j] == bound && at < mid);
                }
            k = block_sum(k, s_i[0]);
            if (step == 0) {
                above = k;
                if (above > kCand - kMaxTopK) break;
            } else if (k >= top_k) {
                hi = mid;
            } else {
                lo = mid;
            }
        }
        if (above <= kCand - kMaxTopK) {
            if (tid == 0) s_count = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = (i * kThreads + tid) * 4 + j;
                    if (at < n && (x[i][j] > bound || (x[i][j] == bound && at < hi))) {
                        const int c = atomicAdd(&s_count, 1);
                        if (c < kCand) s_cand[c] = entry_of(key_of(x[i][j]), base + at);
                    }
                }
            }
            __syncthreads();
            count = s_count;
        }
    }
    if (count >= want && count <= kCand) {
        // a candidate's place is the number of candidates above it
        for (int c = tid; c < count; c += kThreads) {
            const uint64_t e = s_cand[c];
            int above = 0;
            for (int o = 0; o < count; ++o) above += s_cand[o] > e;
            if (above < top_k) out[above] = e;
        }
        for (int c = count + tid; c < top_k; c += kThreads) out[c] = 0;
        return;
    }
    // NaN among the wanted, or the bound far from the top_k-th logit: one after the other
    uint64_t last = ~0ull;
    for (int r = 0; r < top_k; ++r) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (i * kThreads + tid) * 4 + j;
                const uint64_t e = at < n ? entry_of(key_of(x[i][j]), base + at) : 0;
                if (e < last && e > best) best = e;
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)best, d, 64);
            best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) s_cand[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) best = s_cand[w] > best ? s_cand[w] : best;
        if (tid == 0) out[r] = best;
        last = best;
    }
}

// One workgroup per row: the parts' sums, then the row's largest logits out of the parts' lists. An
// entry's place is its place in its own list and, by bisection, the entries above it in the others.
__global__ __launch_bounds__(kThreads) void k_logprobs_join(const float* __restrict__ logits, int64_t stride, int vocab,
                                                            const int32_t* __restrict__ tokens, int top_k, int parts,
                                                            const Part* __restrict__ part,
                                                            const uint64_t* __restrict__ top,
                                                            float* __restrict__ logprobs, int32_t* __restrict__ ranks,
                                                            float* __restrict__ entropy, float* __restrict__ lse,
                                                            int32_t* __restrict__ top_ids,
                                                            float* __restrict__ top_logprobs) {
    __shared__ double s_log;
    __shared__ float s_max;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Part* p = part + (int64_t)row * parts;
    if (tid < 64) {
        float m = kNegInf;
        for (int z = tid; z < parts; z += 64) m = fmaxf(m, p[z].max);
        m = wave_max(m);
        double sum = 0.0, ent = 0.0;
        int equal = 0, ahead = 0;
        for (int z = tid; z < parts; z += 64) {
            const Part a = p[z];
            ahead += a.ahead;
            if (a.max == m) {
                sum += a.sum;
                ent += a.ent;
                equal += a.equal;
            } else if (a.max == kNegInf) {
                sum += a.sum;  // 0, or NaN
            } else {
                const double d = (double)m - a.max, w = exp(-d), s = (double)a.sum + a.equal;
                sum += w * s;
                ent += w * (a.ent + d * s);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            sum += __shfl_xor(sum, d, 64);
            ent += __shfl_xor(ent, d, 64);
            equal += __shfl_xor(equal, d, 64);
            ahead += __shfl_xor(ahead, d, 64);
        }
        if (tid == 0) {
            const bool none = m == kNegInf;
            // without a logit above -inf the sums are of exp(x) = 0, or NaN
            const double rest = sum + (equal - 1), log_s = none ? sum : log1p(rest);
            s_log = log_s;
            s_max = m;
            if (entropy) entropy[row] = (float)(none ? sum : log_s + ent / (1.0 + rest));
            if (lse) lse[row] = none && sum == 0.0 ? kNegInf : (float)(m + log_s);
            const int tok = tokens ? tokens[row] : -1;
            const bool have = (unsigned)tok < (unsigned)vocab;
            if (logprobs) {
                const float xt = have ? logits[(int64_t)row * stride + tok] : kNegInf;
                const double lp = none ? (sum == 0.0 ? (double)kNegInf : sum) : ((double)xt - m) - log_s;
                logprobs[row] = have ? (float)lp : kNegInf;
            }
            if (ranks) ranks[row] = have ? ahead : -1;
        }
    }
    if (top_k == 0) return;
    __syncthreads();
    const uint64_t* t = top + (int64_t)row * parts * top_k;
    for (int i = tid; i < parts * top_k; i += kThreads) {
        const int z = i / top_k;
        const uint64_t e = t[i];
        if (e == 0) continue;
        int above = i - z * top_k;
        for (int o = 0; o < parts && above < top_k; ++o) {
            if (o == z) continue;
            int lo = 0, hi = top_k;  // entries of list o above e
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (t[o * top_k + mid] > e) lo = mid + 1; else hi = mid;
            }
            above += lo;
        }
        if (above >= top_k) continue;
        const float x = value_of((uint32_t)(e >> 32));
        const double lp = s_max == kNegInf ? (s_log == 0.0 ? (double)kNegInf : s_log) : ((double)x - s_max) - s_log;
        if (top_ids) top_ids[(int64_t)row * top_k + above] = (int32_t)~(uint32_t)e;
        if (top_logprobs) top_logprobs[(int64_t)row * top_k + above] = (float)lp;
    }
}

int parts_of(int vocab) { return (vocab + kPart - 1) / kPart; }

}  // namespace

size_t logprobs_ws_bytes(int n_rows, int vocab, int top_k) {
    return (size_t)n_rows * parts_of(vocab) * (sizeof(Part) + (size_t)top_k * sizeof(uint64_t));
}

hipError_t launch_logprobs(const float* logits, int64_t stride, int n_rows, int vocab,
                           const int32_t* tokens, int top_k, float* logprobs, int32_t* ranks,
                           float* entropy, float* lse, int32_t* top_ids, float* top_logprobs,
                           void* ws, hipStream_t stream) {
    const int parts = parts_of(vocab);
    Part* part = (Part*)ws;
    uint64_t* top = (uint64_t*)(part + (size_t)n_rows * parts);
    hipLaunchKernelGGL(k_logprobs_part, dim3((unsigned)n_rows * (unsigned)parts), dim3(kThreads), 0, stream, logits,
                       stride, vocab, tokens, top_k, parts, part, top);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_logprobs_join, dim3((unsigned)n_rows), dim3(kThreads), 0, stream, logits, stride, vocab,
                       tokens, top_k, parts, part, top, logprobs, ranks, entropy, lse, top_ids, top_logprobs);
    return hipGetLastError();
}

}  // namespace cllm_hip
