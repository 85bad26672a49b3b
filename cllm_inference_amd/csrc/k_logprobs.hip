// k_logprobs.hip -- log probabilities from logits: of a given token per row, with its rank, the
// row's entropy and log-sum-exp, and the most likely tokens, in one pass over the logits.
//
//   m = max x,  S = sum exp(x - m),  lse = m + log S,  logprob(t) = (x_t - m) - log S,
//   entropy = log S + sum (m - x) exp(x - m) / S.
// S is held as 1 + S', the sum without one of its largest terms, so that log S = log1p(S') and the
// entropy keep their relative precision where one token has nearly all of the probability; every
// term of the entropy is positive.
//
// What bounds it: VALU work, 22 operations a logit (79% of the cycles in which a CU has work), and the starts
// and ends of two rounds of workgroups, each of which loads all that it reads before it works on it (a CU has
// work in 70% of the launch): 1021 rows of 32003 29 us with the top 20 (4.5 TB/s), 23.6 without a list, 36 with the
// top 64, and 4 to 6 for the join; one row of 128256 6.8 and 4. A workgroup takes 8192 logits of one row (grid
// rows x parts) and holds them in registers, 32 a thread, all loads in flight at once: its maximum
// first, then its sums, the tokens ahead of the given one and its largest logits, without reading twice.
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

// The largest that is no NaN (v_max3_f32; fmaxf would quieten a signalling NaN of each operand first,
// an operation per logit).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Over the wave, in every lane (DPP inside rows of 16, row swaps between them).
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f32<DPP_QUAD_SWAP1>(v));
    v = fmaxf(v, dpp_f32<DPP_QUAD_SWAP2>(v));
    v = fmaxf(v, dpp_f32<DPP_ROW_HALF_MIRROR>(v));
    v = fmaxf(v, dpp_f32<DPP_ROW_MIRROR>(v));
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// A value that at least q (1 .. 64) of the wave's values v (max the largest, none NaN) reach, close to
// the q-th largest: bisection between the smallest above -inf and the largest, on ballots. -inf where
// fewer are above it.
__device__ __forceinline__ float wave_bound(float v, float max, int q) {
    if (__popcll(__ballot(v > kNegInf)) < q) return kNegInf;
    float lo = -wave_max(v > kNegInf ? -v : kNegInf), hi = max;
    if (q == 1) return hi;
    for (int i = 0; i < 12; ++i) {
        const float mid = 0.5f * lo + 0.5f * hi;
        const int c = __popcll(__ballot(v >= mid));
        if (c >= q) lo = mid; else hi = mid;
        if (c == q) break;
    }
    return lo;
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
    __shared__ float s_f[2][kWaves];
    __shared__ int s_i[2][kWaves];
    __shared__ int s_count;
    __shared__ uint64_t s_cand[kCand];
    const int row = blockIdx.x / parts, z = blockIdx.x % parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x0 = logits + (int64_t)row * stride;
    const int base = z * kPart;
    const int n = min(kPart, vocab - base);
    if (tid == 0) s_count = 0;

    // -inf past the row's end: adds nothing to a sum, and is no candidate above a bound
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

    float vmax[kVecs], tmax = kNegInf;  // (NaN never wins)
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        vmax[i] = max3(x[i][0], x[i][1], max3(x[i][2], x[i][3], kNegInf));
        tmax = fmaxf(tmax, vmax[i]);
    }
    // a bound that at least top_k of the part's logits reach: a quarter of them in every wave
    const float wmax = wave_max(tmax);
    if (lane == 0) s_f[0][wave] = wmax;
    if (top_k > 0) {
        const float b = wave_bound(tmax, wmax, (top_k + kWaves - 1) / kWaves);
        if (lane == 0) s_f[1][wave] = b;
    }
    __syncthreads();
    float m = s_f[0][0], bound = s_f[1][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        m = fmaxf(m, s_f[0][w]);
        bound = fminf(bound, s_f[1][w]);
    }

    // candidates: the logits at the bound or above
    if (top_k > 0 && bound > kNegInf) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (vmax[i] >= bound) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (x[i][j] >= bound) {
                        const int c = atomicAdd(&s_count, 1);
                        if (c < kCand) s_cand[c] = entry_of(key_of(x[i][j]), base + (i * kThreads + tid) * 4 + j);
                    }
                }
            }
        }
    }

    // Tokens ahead of the given one: those above it, and its equals with lower ids, which are above the
    // next number below it.
    int ahead = 0;
    if (have && xt > kNegInf) {
        const int rel = tok - base;  // its place in the part, if it is there
        const uint32_t u = __builtin_bit_cast(uint32_t, xt);
        const float below = __builtin_bit_cast(float, xt > 0.0f ? u - 1 : xt < 0.0f ? u + 1 : 0x80000001u);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const float than = (i * kThreads + tid) * 4 + 3 < rel ? below : xt;
#pragma unroll
            for (int j = 0; j < 4; ++j) ahead += __popcll(__ballot(x[i][j] > than));
        }
        ahead = lane == 0 ? ahead : 0;
        if (rel >= 0 && rel < n && (rel >> 8 & (kWaves - 1)) == wave) {  // the wave with the token's own vector
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = (i * kThreads + tid) * 4;
                    ahead += at + 3 >= rel && at + j < rel && x[i][j] == xt;
                }
        }
    } else if (have) {  // -inf, or a NaN: behind all numbers
        const uint32_t kt = key_of(xt);
#pragma unroll 1
        for (int at = tid; at < n; at += kThreads) {
            const uint32_t k = key_of(x0[base + at]);
            ahead += k > kt || (k == kt && base + at < tok);
        }
    }

    // the sums, without the logits that equal the maximum: they are counted
    // (in x's own registers: what is left to do with the logits is rare, and reads them again)
    int equal = 0;
    const float mu = m == kNegInf ? 0.0f : m;  // (no logit above -inf)
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] -= mu;
    if (__any(tmax == mu)) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                equal += x[i][j] == 0.0f;
                x[i][j] = x[i][j] == 0.0f ? kNegInf : x[i][j];
            }
    }
    float sum = 0.0f, ent = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(x[i][j] * kLog2e);
            sum += e;
            // (exp of -200 and less is 0; a NaN stays in e)
            ent = __builtin_fmaf(__builtin_amdgcn_fmed3f(x[i][j], -200.0f, 0.0f), -e, ent);
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
    // What follows up to the ranking is rare; it reads the logits again, one at a time, so that the
    // kernel's registers are those of the work above (64 a thread instead of 109). It is met by masks that leave one
    // stretch of the ids: of 128256 logits -inf but for the first 600, top 20 121 us a call instead of 12, top
    // 64 369 instead of 17; with the type's lowest value for -inf, 97 and 100.
    const auto each = [&](auto f) {
#pragma unroll 1
        for (int at = tid; at < n; at += kThreads) f(at, x0[base + at]);
    };
    if (bound == kNegInf) {
        // Few logits above -inf (a mask, a short part): all of those, and the first ids, of which no
        // more than `above` are no -inf. (A NaN counts as too many.)
        int above = 0;
        each([&](int, float v) { above += v > kNegInf ? 1 : v != v ? kCand : 0; });
        above = block_sum(above, s_i[0]);
        if (above <= kCand / 2 - kMaxTopK) {
            const int first = min(n, want + above);
            each([&](int at, float v) {
                if (v > kNegInf || at < first) s_cand[atomicAdd(&s_count, 1)] = entry_of(key_of(v), base + at);
            });
        }
        __syncthreads();
        count = s_count;
    } else if (count > kCand) {
        // Many logits equal the bound (a coarse grid of values): of those only the first by index can
        // be wanted. The index below which top_k of them lie, by bisection.
        int above = 0;
        each([&](int, float v) { above += v > bound; });
        above = block_sum(above, s_i[0]);
        if (above <= kCand - kMaxTopK) {
            int lo = 0, hi = kPart;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                int k = 0;
                each([&](int at, float v) { k += v == bound && at < mid; });
                if (block_sum(k, s_i[0]) >= top_k) hi = mid; else lo = mid;
            }
            if (tid == 0) s_count = 0;
            __syncthreads();
            each([&](int at, float v) {
                if (v > bound || (v == bound && at < hi)) s_cand[atomicAdd(&s_count, 1)] = entry_of(key_of(v), base + at);
            });
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
        each([&](int at, float v) {
            const uint64_t e = entry_of(key_of(v), base + at);
            if (e < last && e > best) best = e;
        });
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

// One workgroup per row: the parts' sums (the first wave), then the row's largest logits out of the
// parts' lists. The second wave finds a bound that top_k entries of the lists reach: the smallest of
// the lists' ceil(top_k / parts)-th entries, or the largest of their last ones. The entries at the bound
// or above, kCount at most, meet in LDS, and an entry's place is the number of them above it. Where more
// pass (lists of very unlike parts) it is its place in its own list and, by bisection, those in the others.
// (One row of 128256 logits, top 64: 55 us with bisection alone.)
constexpr int kCount = 512;
__global__ __launch_bounds__(kThreads) void k_logprobs_join(const float* __restrict__ logits, int64_t stride, int vocab,
                                                            const int32_t* __restrict__ tokens, int top_k, int parts,
                                                            const Part* __restrict__ part,
                                                            const uint64_t* __restrict__ top,
                                                            float* __restrict__ logprobs, int32_t* __restrict__ ranks,
                                                            float* __restrict__ entropy, float* __restrict__ lse,
                                                            int32_t* __restrict__ top_ids,
                                                            float* __restrict__ top_logprobs) {
    __shared__ uint64_t s_top[kCount], s_bound;
    __shared__ float s_log, s_max;
    __shared__ int s_none, s_count;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Part* p = part + (int64_t)row * parts;
    const uint64_t* t = top + (int64_t)row * parts * top_k;
    const int64_t entries = (int64_t)parts * top_k;
    if (tid >= 64 && tid < 128 && top_k > 0) {
        const int q = (top_k + parts - 1) / parts;
        uint64_t least = ~0ull, most = 0;
        for (int64_t z = tid - 64; z < parts; z += 64) {
            const uint64_t a = t[z * top_k + q - 1], b = t[z * top_k + top_k - 1];
            least = a < least ? a : least;
            most = b > most ? b : most;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t a = __shfl_xor((unsigned long long)least, d, 64), b = __shfl_xor((unsigned long long)most, d, 64);
            least = a < least ? a : least;
            most = b > most ? b : most;
        }
        if (tid == 64) {
            const uint64_t bound = least > most ? least : most;
            s_bound = bound > 0 ? bound : 1;  // (0 is no entry)
            s_count = 0;
        }
    }
    if (tid < 64) {
        const int tok = tokens ? tokens[row] : -1;
        const bool have = (unsigned)tok < (unsigned)vocab;
        const float xt = have && logprobs ? logits[(int64_t)row * stride + tok] : kNegInf;
        float m = kNegInf;
        for (int z = tid; z < parts; z += 64) m = fmaxf(m, p[z].max);
        m = wave_max(m);
        float sum = 0.0f, ent = 0.0f;
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
                // (exp of -200 and less is 0, as in the part; a part of a mask's finite lowest values is farther,
                // and that times its 8192 weights past fp32's range)
                const float d = fminf(m - a.max, 200.0f), s = a.sum + (float)a.equal, w = __builtin_amdgcn_exp2f(-d * kLog2e);
                sum += w * s;
                ent += w * (a.ent + d * s);
            }
        }
        sum = wave_sum(sum);
        ent = wave_sum(ent);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            equal += __shfl_xor(equal, d, 64);
            ahead += __shfl_xor(ahead, d, 64);
        }
        if (tid == 0) {
            // without a logit above -inf the sum is 0, or NaN
            const bool none = m == kNegInf && sum == 0.0f;
            const float rest = sum + (float)(m == kNegInf ? 0 : equal - 1);
            const float log_s = m == kNegInf ? sum : log1pf(rest);
            s_log = log_s;
            s_max = m;
            s_none = none;
            if (entropy) entropy[row] = none ? 0.0f : log_s + ent / (1.0f + rest);
            if (lse) lse[row] = none ? kNegInf : m + log_s;
            if (logprobs) logprobs[row] = none || !have ? kNegInf : (xt - m) - log_s;
            if (ranks) ranks[row] = have ? ahead : -1;
        }
    }
    if (top_k == 0) return;
    __syncthreads();
    const auto put = [&](uint64_t e, int place) {
        const float x = value_of((uint32_t)(e >> 32));
        if (top_ids) top_ids[(int64_t)row * top_k + place] = (int32_t)~(uint32_t)e;
        if (top_logprobs) top_logprobs[(int64_t)row * top_k + place] = s_none ? kNegInf : (x - s_max) - s_log;
    };
    const uint64_t bound = s_bound;
    for (int64_t i = tid; i < entries; i += kThreads) {
        const uint64_t e = t[i];
        if (e < bound) continue;
        const int c = atomicAdd(&s_count, 1);
        if (c < kCount) s_top[c] = e;
    }
    __syncthreads();
    const int count = s_count;
    if (count <= kCount) {
        for (int c = tid; c < count; c += kThreads) {
            const uint64_t e = s_top[c];
            int above = 0;
#pragma unroll 8
            for (int o = 0; o < count; ++o) above += s_top[o] > e;
            if (above < top_k) put(e, above);
        }
        return;
    }
    for (int64_t i = tid; i < entries; i += kThreads) {
        const uint64_t e = t[i];
        if (e < bound) continue;
        const int z = (int)(i / top_k);
        int above = (int)(i - (int64_t)z * top_k);
        for (int o = 0; o < parts && above < top_k; ++o) {
            if (o == z) continue;
            int lo = 0, hi = top_k;  // entries of list o above e
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (t[(int64_t)o * top_k + mid] > e) lo = mid + 1; else hi = mid;
            }
            above += lo;
        }
        if (above < top_k) put(e, above);
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
