// k_route.hip -- a router's choice of experts, and entries sorted by group (gfx950).
//
// What moves is small (a logit row is at most 4 KB); launches and dependent steps are the cost. Sorting
// is by counting: an entry's place is the number of entries with a lower id, plus those of its own id
// before it, so the order is stable and the same every time, without atomics or scratch.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device_utils.h"
#include "experts.h"

namespace cllm_hip {
namespace {

constexpr int kSmallEntries = 64;  // up to here one workgroup can route and sort

// ---- entries sorted by group --------------------------------------------------------------------
// Workgroup g lists the entries of group g (the last one, the entries of none). Its 16 waves take
// consecutive stretches of the ids: each counts its matches and the lower ids, then, behind the sums of the
// waves before it, writes its matches. Every workgroup reads all ids: 32792 ids (131 KB) and 257 workgroups,
// 34 MB from L2, 10 us (one load at a time: 22 us); two dependent passes, not the bytes, bound it.
__global__ __launch_bounds__(1024) void k_group_rows(const int32_t* __restrict__ ids, int n, int groups,
                                                     int32_t* __restrict__ offsets, int32_t* __restrict__ order) {
    __shared__ int lower[16], mine[16];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // 1024 ids to a step of a wave: four loads of four neighbouring ids a lane, all on their way at once
    const int per = ((n + 16 * 1024 - 1) / (16 * 1024)) * 1024;
    const int first = min(wave * per, n), last = min(n, first + per);
    const bool vec = ((uintptr_t)ids & 15u) == 0;
    auto step = [&](int i, int (&k)[16]) {
        if (vec && i + 1024 <= last) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int4 v = *(const int4*)(ids + i + 256 * j + 4 * lane);
                k[4 * j] = v.x, k[4 * j + 1] = v.y, k[4 * j + 2] = v.z, k[4 * j + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int at = i + 256 * (j >> 2) + 4 * lane + (j & 3);
                k[j] = at < last ? ids[at] : -2;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int at = i + 256 * (j >> 2) + 4 * lane + (j & 3);
            k[j] = at >= last ? groups + 1 : (uint32_t)k[j] < (uint32_t)groups ? k[j] : groups;
        }
    };
    int lo = 0, at = 0;
    for (int i = first; i < last; i += 1024) {
        int k[16];
        step(i, k);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            lo += k[j] < g;
            at += k[j] == g;
        }
    }
    for (int d = 32; d > 0; d >>= 1) {
        lo += __shfl_xor(lo, d, 64);
        at += __shfl_xor(at, d, 64);
    }
    if (lane == 0) lower[wave] = lo, mine[wave] = at;
    __syncthreads();
    int base = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        base += lower[w];
        if (w < wave) before += mine[w];
    }
    if (threadIdx.x == 0) offsets[g] = base;
    if (at == 0) return;
    int to = base + before;
    const uint64_t below = (1ull << lane) - 1;
    for (int i = first; i < last; i += 1024) {
        int k[16];
        step(i, k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // neighbouring ids are one lane's: those of the lanes below, then its own before this one
            int ahead = 0, all = 0;
            uint64_t b[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                b[c] = __ballot(k[4 * j + c] == g);
                ahead += __popcll(b[c] & below);
                all += __popcll(b[c]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (k[4 * j + c] == g) order[to + ahead++] = i + 256 * j + 4 * lane + c;
            to += all;
        }
    }
}

// ---- the choice ----------------------------------------------------------------------------------
// The largest of the lanes' values, in every lane (moves between lanes by DPP: no LDS latency).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)u, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(u >> 32), (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double wave_max(double v) {
    v = fmax(v, dpp_f64<DPP_QUAD_SWAP1, 0xF>(v));
    v = fmax(v, dpp_f64<DPP_QUAD_SWAP2, 0xF>(v));
    v = fmax(v, dpp_f64<DPP_ROW_HALF_MIRROR, 0xF>(v));
    v = fmax(v, dpp_f64<DPP_ROW_MIRROR, 0xF>(v));
    v = fmax(v, dpp_f64<0x142, 0xA>(v));  // a row's last lane to the next row
    v = fmax(v, dpp_f64<0x143, 0xC>(v));  // lane 31 to the upper half
    return lane_f64(v, 63);
}
__device__ __forceinline__ double wave_add(double v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// One wave chooses a row's experts. Lane l has experts V l .. V l + V - 1, so that of equal keys the lowest
// lane's lowest slot is the lowest expert. Keys and scores are in 64 bits: scores plus a bias lie close
// together, and the choice is then the definition's whatever the order of sums. keys: this wave's LDS for
// 64 V doubles, used with parts only.
template <int V>
__device__ void choose(const RouteArgs& a, int row, int lane, double* keys) {
    const float* z = a.logits + (size_t)row * a.stride;
    const double none = -__builtin_inf();
    double x[V], key[V];
    double top = none;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = V * lane + j;
        float f = e < a.experts ? z[e] : -__builtin_inff();
        if (f != f) f = -__builtin_inff();
        x[j] = (double)f;
        top = fmax(top, x[j]);
    }
    // an expert's score: the sigmoid, or exp(x - top) (over the row's sum: below)
    auto score = [&](double v) {
        if (a.sigmoid) return 1.0 / (1.0 + exp(-v));
        return v == top ? 1.0 : exp(v - top);
    };
    const bool all = !a.sigmoid && (a.bias || !a.normalise);  // the softmax's sum is needed
    double sum = 1.0;
    if (!a.sigmoid) top = wave_max(top);
    if (all) {
        sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) sum += x[j] == none ? 0.0 : score(x[j]);
        sum = wave_add(sum);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = V * lane + j;
        key[j] = x[j];
        if (a.bias && x[j] != none) {
            key[j] = score(x[j]) / sum + (double)a.bias[e];
            if (key[j] != key[j]) key[j] = none;
        }
    }
    if (a.parts > 1) {
        const int width = a.experts / a.parts;
#pragma unroll
        for (int j = 0; j < V; ++j) keys[V * lane + j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        // `share` neighbouring lanes to a part, every share-th key each, then their two largest joined
        int share = 64;
        while (share * a.parts > 64) share >>= 1;
        const int part = lane / share;
        double best = none, second = none;
        if (part < a.parts)
            for (int i = lane & (share - 1); i < width; i += share) {
                const double v = keys[part * width + i];
                second = fmax(second, fmin(best, v));
                best = fmax(best, v);
            }
        for (int d = 1; d < share; d <<= 1) {
            const double b = __shfl_xor(best, d, 64), s = __shfl_xor(second, d, 64);
            second = fmax(fmin(best, b), fmax(second, s));
            best = fmax(best, b);
        }
        double mine = best;
        if (a.bias && width > 1) mine = best + second;
        if (mine != mine) mine = none;
        int ahead = 0;
        for (int p = 0; p < a.parts; ++p) {
            const double v = lane_f64(mine, p * share);
            ahead += v > mine || (v == mine && p < part);
        }
        const uint64_t kept = __ballot(part < a.parts && ahead < a.top_parts);
        uint64_t keep = 0;  // bit p: part p
        for (int p = 0; p < a.parts; ++p) keep |= ((kept >> (p * share)) & 1) << p;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = V * lane + j;
            if (e >= a.experts || !((keep >> (e / width)) & 1)) key[j] = none;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
    // the k largest, one a round; lane i keeps the i-th
    int id = -1;
    double p = 0.0, mine_x = none;
    for (int i = 0; i < a.top_k; ++i) {
        double best = key[0];
        int slot = 0;
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) best = key[j], slot = j;
        const double m = wave_max(best);
        if (m == none) break;
        const int owner = __ffsll((unsigned long long)__ballot(best == m)) - 1;
        const int s = __builtin_amdgcn_readlane(slot, owner);
        double v = none;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v = j == s ? x[j] : v;
            if (lane == owner && j == s) key[j] = none;
        }
        v = lane_f64(v, owner);
        if (lane == i) id = V * owner + s, mine_x = v;
    }
    if (id >= 0) p = score(mine_x);
    if (a.normalise) sum = wave_add(p);
    if (lane < a.top_k) {
        a.ids[(size_t)row * a.top_k + lane] = id;
        a.weights[(size_t)row * a.top_k + lane] = id < 0 || !(sum > 0.0) ? 0.0f : (float)(p / sum * (double)a.scale);
    }
}

// A wave a row, V keys a lane; SORT: one workgroup for all rows, which then sorts their entries too.
// Measured (MI355X): one row of 8 experts 3.9 us, a launch; 4099 rows of 256, sigmoid with bias, the best 4 of 8 groups,
// top 8: 15.3 us for 4.6 MB. With one round of the eight 10.9, without exponentials and quotients 13.6, without the
// groups 13.1, without all three 5.7: the rounds, each a maximum of 64-bit keys over a wave, are the largest part.
template <int V, bool SORT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_route(RouteArgs a) {
    extern __shared__ double keys[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int row = blockIdx.x * WAVES + wave; row < a.rows; row += gridDim.x * WAVES)
        choose<V>(a, row, lane, keys + wave * 64 * V);
    if constexpr (SORT) {
        __shared__ int key[kSmallEntries];
        __threadfence_block();
        __syncthreads();
        const int n = a.rows * a.top_k;
        for (int i = threadIdx.x; i < n; i += 64 * WAVES) {
            const int v = a.ids[i];
            key[i] = (uint32_t)v < (uint32_t)a.experts ? v : a.experts;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += 64 * WAVES) {
            const int k = key[i];
            int to = 0;
            for (int j = 0; j < n; ++j) to += key[j] < k || (key[j] == k && j < i);
            a.order[to] = i;
        }
        for (int e = threadIdx.x; e <= a.experts; e += 64 * WAVES) {
            int c = 0;
            for (int j = 0; j < n; ++j) c += key[j] < e;
            a.offsets[e] = c;
        }
    }
}

template <int V>
hipError_t route_launch(const RouteArgs& a, hipStream_t s) {
    // One workgroup for all rows, or a wave a row over the chip and a launch that sorts. The second launch costs 3 to 4 us; a
    // second turn of the waves, and comparing every entry with every other, soon as much. MI355X, us, one | two
    // launches: 8 rows top 8 of 64 experts 7.0 | 8.1, of 256 8.4 | 9.1, of 512 11.9 | 11.2; 16 rows 11.9 | 8.2, 14.6 | 9.3; 64
    // rows 41 | 8.8, 53 | 9.8. 1024 experts (four waves) 4 rows 13.0 | 16.9, 5 19.6 | 16.7; top 32 of 64 2 rows 10.2 | 11.6,
    // 4 12.5 | 11.7. Two turns for few entries of few experts: 16 rows top 2 of 8 6.0 | 7.3, top 4 of 32 7.9 | 7.7.
    const int entries = a.rows * a.top_k;
    const bool small = (a.rows <= (V == 16 ? 4 : 8) && entries <= kSmallEntries) || (V == 1 && a.rows <= 16 && entries <= 32);
    const size_t per = a.parts > 1 ? 64 * V * sizeof(double) : 0;
    if (small) {
        if (a.rows <= 4 || V == 16)  // (of 16 experts to a lane, more waves' keys would not fit 64 KB)
            k_route<V, true, 4><<<1, 256, 4 * per, s>>>(a);
        else
            k_route<V, true, 8><<<1, 512, 8 * per, s>>>(a);
        return hipGetLastError();
    }
    // (a grid's threads are counted in 32 bits: more than 2^26 rows take turns)
    k_route<V, false, 4><<<std::min((a.rows + 3) / 4, 1 << 22), 256, 4 * per, s>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_group_rows(a.ids, a.rows * a.top_k, a.experts, a.offsets, a.order, s);
}

}  // namespace

hipError_t launch_group_rows(const int32_t* ids, int n, int groups, int32_t* offsets, int32_t* order, hipStream_t s) {
    k_group_rows<<<groups + 1, 1024, 0, s>>>(ids, n, groups, offsets, order);
    return hipGetLastError();
}

hipError_t launch_route(const RouteArgs& a, hipStream_t s) {
    return a.experts <= 64 ? route_launch<1>(a, s) : a.experts <= 128 ? route_launch<2>(a, s)
         : a.experts <= 256 ? route_launch<4>(a, s) : a.experts <= 512 ? route_launch<8>(a, s) : route_launch<16>(a, s);
}

}  // namespace cllm_hip
