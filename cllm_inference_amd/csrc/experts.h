// experts.h -- products whose weights a row's index chooses (internal to libcllm_hip.so): rows
// grouped by index, a router, feed-forwards of experts over GGUF blocks, low-rank adapters.
//
// Launchers validate nothing: capi.hip checks shapes, types and alignment first. What the device
// arrays hold (offsets, order, ids) is bounded where the kernels read it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cllm_hip {

constexpr int kMaxGroups = 1024;
constexpr int kMaxRouteTopK = 32;
constexpr int kMaxRouteParts = 64;
constexpr int kMaxLoraMats = 4;
constexpr int kMaxLoraRank = 256;

// Parts of a workspace start at multiples of 256 bytes.
inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// Entries grouped by index: order lists them sorted by group, those of group g at
// order[offsets[g]] .. order[offsets[g + 1] - 1], those of no group from offsets[groups] on.
struct Groups {
    const int32_t* offsets;
    const int32_t* order;
    int groups, entries;
};

hipError_t launch_group_rows(const int32_t* ids, int n, int groups, int32_t* offsets, int32_t* order,
                             hipStream_t stream);

struct RouteArgs {
    const float* logits;
    int64_t stride;
    const float* bias;
    int rows, experts, top_k, parts, top_parts;
    bool sigmoid, normalise;
    float scale;
    int32_t* ids;
    float* weights;
    int32_t* offsets;
    int32_t* order;
};
hipError_t launch_route(const RouteArgs& a, hipStream_t stream);

// The experts' products: entry e has activation row e / per_row of x [rows][k]; with two matrices
// y[e] = silu(w[0] x) * (w[1] x), with one y[e] = w[0] x (plus the biases, [groups][n]).
// Matrices are [groups][n] rows of row_bytes.
struct ExpertArgs {
    uint32_t type;
    const uint8_t* w[2];
    const float* bias[2];
    int mats, k, n;
    const float* x;
    int rows, per_row;
    Groups g;
    float* y;
    void* ws;  // expert_act_bytes(type, k, rows)
};
size_t expert_act_bytes(uint32_t type, int k, int rows);
hipError_t launch_experts(const ExpertArgs& a, hipStream_t stream);
// Workgroups (of at most 512 threads) of that launch.
int64_t expert_workgroups(uint32_t type, int mats, int k, int n, int groups, int entries);
void expert_plan_name(uint32_t type, int mats, int k, int n, int groups, int entries, char* buf, size_t cap);
// y[r] = (base[r] +) sum over j of weights[r][j] * p[r top_k + j], the j with an id in range
hipError_t launch_expert_sum(const float* p, const int32_t* ids, const float* weights, int rows, int top_k,
                             int groups, int n, const float* base, float* y, hipStream_t stream);

struct LoraArgs {
    bool half;
    int k, mats, max_rank;
    const void* a[kMaxLoraMats];
    const void* b[kMaxLoraMats];
    int n[kMaxLoraMats];
    const float* base[kMaxLoraMats];
    float* y[kMaxLoraMats];
    const int32_t* ranks;
    const float* scales;
    const float* x;
    Groups g;
    float* ws;
};
size_t lora_ws_bytes(int mats, int k, int max_rank, int groups, int rows);
hipError_t launch_lora(const LoraArgs& a, hipStream_t stream);

#if defined(__HIPCC__)
// The t-th tile of at most M entries of one group. A group's tiles start at id offsets[g] / M + g,
// which leaves room for each (a/M + ceil(b/M) <= (a + b)/M + 1), or, where that is fewer ids, at
// every M-th entry of the group (by_entry). Every id is looked up with one round of loads. extra: 1 to
// take the entries of no group for one more.
struct GroupTile {
    int group, first, count;
};
template <int M>
__host__ __device__ inline bool tiles_by_entry(int groups, int entries) {
    return entries <= entries / M + groups;
}
template <int M>
__host__ __device__ inline int tile_ids(int groups, int entries) {
    return tiles_by_entry<M>(groups, entries) ? entries : entries / M + groups;
}
template <int M>
__device__ __forceinline__ GroupTile find_tile(const Groups& v, int extra, int t, int lane) {
    const int n = v.groups + extra;
    const bool by_entry = tiles_by_entry<M>(n, v.entries);
    int c = 0;
    for (int b = 0; b < n; b += 64) {
        const int g = b + lane;
        bool at = false;
        if (g < n) {
            const int o = v.offsets[g];
            at = (by_entry ? o : o / M + g) <= t;
        }
        c += __popcll(__ballot(at));
    }
    const int g = __builtin_amdgcn_readfirstlane(c) - 1;
    if (g < 0) return {0, 0, 0};
    const int o0 = v.offsets[g], o1 = g == v.groups ? v.entries : v.offsets[g + 1];
    const int first = by_entry ? t : o0 + (t - (o0 / M + g)) * M;
    int count = o1 - first;
    if (first < 0 || first >= v.entries || (by_entry && (t - o0) % M != 0)) count = 0;
    count = count > M ? M : count;
    count = count > v.entries - first ? v.entries - first : count;
    return {g, __builtin_amdgcn_readfirstlane(first), __builtin_amdgcn_readfirstlane(count)};
}
#endif

}  // namespace cllm_hip
