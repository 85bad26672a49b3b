// k_lora.hip -- low-rank adapters of the requests of a batch beside shared projections (gfx950).
//
// y_i[r] = base_i[r] + s_a B_i,a (A_i,a x_r) for row r with adapter a, rows grouped by adapter. Reads of A
// and B (few rows to an adapter) or of x, base and y (prompts) bound it; products are on fp32 MFMA, so that
// fp32 rows meet binary16 or fp32 adapters without a rounding, and 16 x 16 tiles lose nothing that the
// reads would not hide. Two launches: the ranks' sums, split over K where the rows alone do not fill the
// chip (the second launch adds the parts, in order), then the outputs with the shared projection added.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device_utils.h"
#include "experts.h"

namespace cllm_hip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

struct Down {
    const void* a[kMaxLoraMats];
    const int32_t* ranks;
    const float* x;
    Groups g;
    int k, max_rank, parts, k_part;  // k_part: elements of a part, a multiple of 64
    int rank_blocks;                 // of 16 RT ranks
    float* t;                        // [mat][part][entry][max_rank]
};
struct Up {
    const void* b[kMaxLoraMats];
    const float* base[kMaxLoraMats];
    float* y[kMaxLoraMats];
    int n[kMaxLoraMats], block_end[kMaxLoraMats];
    const int32_t* ranks;
    const float* scales;
    const float* t;
    Groups g;
    int mats, max_rank, parts, tiles;  // tiles: 16-column tiles of a wave
};

__device__ __forceinline__ int rank_of(const int32_t* ranks, int max_rank, int group) {
    return ranks ? min(max(ranks[group], 0), max_rank) : max_rank;
}
template <bool HALF>
__device__ __forceinline__ f32x4 load4(const void* p, size_t at) {
    if constexpr (HALF) {
        const h16x4 v = *(const h16x4*)((const _Float16*)p + at);
        return f32x4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
    } else {
        return *(const f32x4*)((const float*)p + at);
    }
}

// Tile of 16 rows of an adapter x RT tiles of 16 ranks x a part of K. Lane (r, q) loads elements 4q .. 4q + 3
// of every 16 of K, of row r and of rank r, which four MFMAs take one by one; the four waves take every fourth
// 64 elements and meet in LDS.
template <bool HALF, int RT>
__global__ __launch_bounds__(256) void k_lora_down(Down a) {
    __shared__ float red[4][RT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const GroupTile t = find_tile<16>(a.g, 0, blockIdx.x, lane);
    if (t.count <= 0) return;
    const int part = blockIdx.y, mat = (int)blockIdx.z / a.rank_blocks;
    const int r0 = 16 * RT * ((int)blockIdx.z - mat * a.rank_blocks);
    const int rank = rank_of(a.ranks, a.max_rank, t.group);
    if (r0 >= rank) return;  // (the second launch takes ranks past it for zero)
    const int r = lane & 15, q = lane >> 4;
    int e = r < t.count ? a.g.order[t.first + r] : -1;
    if ((uint32_t)e >= (uint32_t)a.g.entries) e = -1;
    const float* xp = a.x + (size_t)max(e, 0) * a.k;
    const size_t arow = (size_t)t.group * a.max_rank;
    const int k0 = part * a.k_part, k1 = min(a.k, k0 + a.k_part);
    f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = k0 + 64 * wave; k < k1; k += 256) {
        f32x4 xv[4], av[4][RT];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int at = k + 16 * b + 4 * q;
            const bool in = at < k1;
            xv[b] = in && e >= 0 ? *(const f32x4*)(xp + at) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int row = r0 + 16 * i + r;
                av[b][i] = in && row < rank ? load4<HALF>(a.a[mat], (arow + row) * a.k + at) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[b][j], av[b][i][j], acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) *(f32x4*)&red[wave][i][4 * lane] = acc[i];
    __syncthreads();
    // lane (r, q) had rows 4q + j of rank r
    const int tok = threadIdx.x >> 4, col = threadIdx.x & 15;
    int en = tok < t.count ? a.g.order[t.first + tok] : -1;
    if ((uint32_t)en >= (uint32_t)a.g.entries) return;
    const int at = 4 * (16 * (tok >> 2) + col) + (tok & 3);
    float* out = a.t + (((size_t)mat * a.parts + part) * a.g.entries + en) * a.max_rank + r0 + col;
#pragma unroll
    for (int i = 0; i < RT; ++i)
        if (r0 + 16 * i + col < rank) out[16 * i] = ((red[0][i][at] + red[1][i][at]) + red[2][i][at]) + red[3][i][at];
}

// Tile of 16 rows of an adapter (or of none) x the columns of a workgroup's four waves. The rows' rank sums
// stand in LDS; lane (r, q) loads B's elements 4q .. 4q + 3 of every 16 ranks of output column r, and ends with
// four neighbouring columns of one row.
template <bool HALF>
__global__ __launch_bounds__(256) void k_lora_up(Up a) {
    __shared__ float ts[16][kMaxLoraRank + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const GroupTile t = find_tile<16>(a.g, 1, blockIdx.x, lane);
    if (t.count <= 0) return;
    int mat = 0;
    while (mat + 1 < a.mats && (int)blockIdx.y >= a.block_end[mat]) ++mat;
    const int blk = (int)blockIdx.y - (mat ? a.block_end[mat - 1] : 0);
    const float* base = a.base[mat];
    float* y = a.y[mat];
    const bool none = t.group == a.g.groups;
    if (none && base == y) return;
    const int rank = none ? 0 : rank_of(a.ranks, a.max_rank, t.group);
    const int chunks = (rank + 15) / 16;
    const float scale = none ? 0.0f : a.scales ? a.scales[t.group] : 1.0f;
    const int r = lane & 15, q = lane >> 4, n = a.n[mat];
    for (int i = threadIdx.x; i < 16 * 16 * chunks; i += 256) {
        const int tok = i / (16 * chunks), c = i - tok * 16 * chunks;
        const int en = tok < t.count ? a.g.order[t.first + tok] : -1;
        float v = 0.0f;
        if (c < rank && (uint32_t)en < (uint32_t)a.g.entries) {
            const float* src = a.t + ((size_t)mat * a.parts * a.g.entries + en) * a.max_rank + c;
            for (int p = 0; p < a.parts; ++p) v += src[(size_t)p * a.g.entries * a.max_rank];
        }
        ts[tok][c] = v * scale;
    }
    __syncthreads();
    int e = r < t.count ? a.g.order[t.first + r] : -1;
    if ((uint32_t)e >= (uint32_t)a.g.entries) e = -1;
    const size_t brow = (size_t)t.group * n;
    for (int j = 0; j < a.tiles; ++j) {
        const int n0 = (blk * 4 + wave) * 16 * a.tiles + 16 * j;
        if (n0 >= n) break;
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        const int row = min(n0 + r, n - 1);
        for (int c = 0; c < chunks; ++c) {
            const int at = 16 * c + 4 * q;
            f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
            if (at < rank) {
                w = load4<HALF>(a.b[mat], (brow + row) * a.max_rank + at);
#pragma unroll
                for (int i = 1; i < 4; ++i) w[i] = at + i < rank ? w[i] : 0.0f;
            }
            const f32x4 v = *(const f32x4*)&ts[r][at];
#pragma unroll
            for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i], v[i], s, 0, 0, 0);
        }
        if (e < 0) continue;
        const int col = n0 + 4 * q;
        const size_t at = (size_t)e * n + col;
        if (n % 4 == 0) {
            if (col < n) *(f32x4*)(y + at) = base ? *(const f32x4*)(base + at) + s : s;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < n) y[at + i] = base ? base[at + i] + s[i] : s[i];
        }
    }
}

struct LoraPlan {
    int parts, k_part;
};
LoraPlan lora_plan(int mats, int k, int groups, int rows) {
    const int wgs = std::max(1, std::min(tile_ids<16>(groups, rows), rows)) * mats;
    int parts = std::max(1, std::min((512 + wgs - 1) / wgs, (k + 511) / 512));
    parts = std::min(parts, 8);
    LoraPlan p;
    p.k_part = ((k + parts - 1) / parts + 63) / 64 * 64;
    p.parts = (k + p.k_part - 1) / p.k_part;
    return p;
}

template <bool HALF>
hipError_t lora_launch(const LoraArgs& a, hipStream_t s) {
    const LoraPlan p = lora_plan(a.mats, a.k, a.g.groups, a.g.entries);
    Down d{};
    Up u{};
    for (int i = 0; i < a.mats; ++i) d.a[i] = a.a[i], u.b[i] = a.b[i], u.base[i] = a.base[i], u.y[i] = a.y[i], u.n[i] = a.n[i];
    d.ranks = u.ranks = a.ranks;
    u.scales = a.scales;
    d.x = a.x;
    d.g = u.g = a.g;
    d.k = a.k;
    d.max_rank = u.max_rank = a.max_rank;
    d.parts = u.parts = p.parts;
    d.k_part = p.k_part;
    d.t = a.ws;
    u.t = a.ws;
    u.mats = a.mats;
    const unsigned tiles = (unsigned)tile_ids<16>(a.g.groups, a.g.entries);
    const int rt = a.max_rank <= 16 ? 1 : 2;
    d.rank_blocks = (a.max_rank + 16 * rt - 1) / (16 * rt);
    const dim3 grid(tiles, (unsigned)p.parts, (unsigned)(a.mats * d.rank_blocks));
    if (rt == 1)
        k_lora_down<HALF, 1><<<grid, 256, 0, s>>>(d);
    else
        k_lora_down<HALF, 2><<<grid, 256, 0, s>>>(d);
    if (hipError_t e = hipGetLastError()) return e;
    const unsigned up_tiles = (unsigned)tile_ids<16>(a.g.groups + 1, a.g.entries);
    u.tiles = up_tiles >= 16 ? 4 : 1;
    int blocks = 0;
    for (int i = 0; i < a.mats; ++i) u.block_end[i] = blocks += (a.n[i] + 64 * u.tiles - 1) / (64 * u.tiles);
    if (blocks == 0) return hipSuccess;
    k_lora_up<HALF><<<dim3(up_tiles, (unsigned)blocks), 256, 0, s>>>(u);
    return hipGetLastError();
}

}  // namespace

size_t lora_ws_bytes(int mats, int k, int max_rank, int groups, int rows) {
    return (size_t)mats * lora_plan(mats, k, groups, rows).parts * rows * max_rank * sizeof(float);
}

hipError_t launch_lora(const LoraArgs& a, hipStream_t s) {
    return a.half ? lora_launch<true>(a, s) : lora_launch<false>(a, s);
}

}  // namespace cllm_hip
