// k_lora.hip -- low-rank adapters of the requests of a batch beside shared projections (gfx950).
//
// y_i[r] = base_i[r] + s_a B_i,a (A_i,a x_r) for row r with adapter a, rows grouped by adapter. Reads of A
// and B (few rows to an adapter) or of x, base and y (prompts) are what it cannot do without; products are on fp32 MFMA,
// so that fp32 rows meet binary16 or fp32 adapters without a rounding. Tiles are 16 rows of one adapter: with two rows to an
// adapter seven eighths of the products are for nothing, 8 to 10 us of the second launch for 64 rows. Two launches: the ranks' sums, split over K where the rows alone do not fill the
// chip (the second launch adds the parts, in order), then the outputs with the shared projection added.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "device_utils.h"
#include "experts.h"

namespace cllm_hip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxParts = 8;  // of K

struct Down {
    const void* a[kMaxLoraMats];
    const int32_t* ranks;
    const float* x;
    Groups g;
    int k, max_rank, parts, k_part;  // k_part: elements of a part, a multiple of 256
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
    int mats, max_rank, parts, steps;  // steps: column blocks of a workgroup
};

__device__ __forceinline__ int rank_of(const int32_t* ranks, int max_rank, int group) {
    return ranks ? min(max(ranks[group], 0), max_rank) : max_rank;
}
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

// VL neighbouring elements of a lane: 16 bytes (8 of binary16, 4 of fp32), or 8 where rows of binary16 are no
// multiple of 16 bytes (or 16 ranks at most).
template <bool HALF, int VL>
struct Piece {
    static_assert(VL == 4 || HALF, "fp32: 4");
    std::conditional_t<!HALF, f32x4, std::conditional_t<VL == 8, h16x8, h16x4>> v;
    __device__ __forceinline__ void load(const void* p, size_t at) {
        using V = decltype(v);
        if constexpr (HALF)
            v = *(const V*)((const _Float16*)p + at);
        else
            v = *(const V*)((const float*)p + at);
    }
    __device__ __forceinline__ void zero() { v = decltype(v){}; }
    __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
};

// Tile of 16 rows of an adapter x RT tiles of 16 ranks x a part of K. Lane (r, q) loads VL elements from 4 VL b + q VL
// on, of row r and of rank r, which VL MFMAs take one by one; the four waves take every fourth 64 elements, each
// loaded while the 64 before are multiplied, and meet in LDS.
// Measured (MI355X): 64 rows of 32 adapters (27 named), two matrices of rank 64, K 4096: 21 MB of binary16, 13.9 us; one
// row 4.8; 2045 rows of 5 adapters, rank 32, fp32: 34 MB of x,
// 19 us (1.8 TB/s). Neither is near its bytes; what a workgroup's start and the waves' meeting take was not measured apart.
template <bool HALF, int VL, int RT>
__global__ __launch_bounds__(256) void k_lora_down(Down a) {
    constexpr int NB = 16 / VL;  // pieces of 64 elements
    __shared__ float red[4][RT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const GroupTile t = find_tile<16>(a.g, 0, blockIdx.x, lane);
    if (t.count <= 0) return;
    const int part = blockIdx.y, mat = (int)blockIdx.z / a.rank_blocks;
    const int r0 = 16 * RT * ((int)blockIdx.z - mat * a.rank_blocks);
    const int rank = rank_of(a.ranks, a.max_rank, t.group);
    if (r0 >= rank) return;  // (the second launch takes ranks past it for zero)
    const int r = lane & 15, q = lane >> 4;
    const int k0 = part * a.k_part, k1 = min(a.k, k0 + a.k_part);
    const size_t arow = (size_t)t.group * a.max_rank;
    Piece<HALF, VL> av[2][NB][RT];
    f32x4 xv[2][NB][VL / 4];
    auto load_a = [&](int k, int buf) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int at = k + VL * (4 * b + q), row = r0 + 16 * i + r;
                if (at < k1 && row < rank)
                    av[buf][b][i].load(a.a[mat], (arow + row) * a.k + at);
                else
                    av[buf][b][i].zero();
            }
    };
    load_a(k0 + 64 * wave, 0);  // on its way while the rows are looked up
    int e = r < t.count ? a.g.order[t.first + r] : -1;
    if ((uint32_t)e >= (uint32_t)a.g.entries) e = -1;
    const float* xp = a.x + (size_t)max(e, 0) * a.k;
    auto load_x = [&](int k, int buf) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < VL / 4; ++h) {
                const int at = k + VL * (4 * b + q) + 4 * h;
                xv[buf][b][h] = at < k1 && e >= 0 ? *(const f32x4*)(xp + at) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
    };
    load_x(k0 + 64 * wave, 0);
    f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto step = [&]<int BUF>(int k) {
        if (k + 256 < k1) {
            load_a(k + 256, 1 - BUF);
            load_x(k + 256, 1 - BUF);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < VL; ++j)
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[BUF][b][j / 4][j % 4], av[BUF][b][i].at(j), acc[i], 0, 0, 0);
    };
    for (int k = k0 + 64 * wave; k < k1; k += 512) {
        step.template operator()<0>(k);
        if (k + 256 < k1) step.template operator()<1>(k + 256);
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

// Tile of 16 rows of an adapter (or of none) x the columns of a workgroup: `steps` blocks of four waves' 16 TILES
// each. The rows' rank sums stand in LDS; lane (r, q) loads VL of B's elements of every 4 VL ranks of output column
// r, and ends with four neighbouring columns of one row. A block's elements of B (of the first 4 VL NCH ranks)
// and of the shared projection are on their way while the block before is multiplied, the first ones while the
// rank sums are read.
// Measured (MI355X): 64 rows of 32 adapters (27 named), 2 x 14336 columns: B of all 64 ranks, which is read whatever an
// adapter's rank, 99 MB (of the ranks that count 74), 35 us (2.8 TB/s; the fp32 MFMAs 8 to 10 of it); 2045 rows, rank 32,
// 4096 columns: 67 MB of base and y, 24 us (2.8 TB/s).
template <bool HALF, int VL, int NCH, int TILES>
__global__ __launch_bounds__(256) void k_lora_up(Up a) {
    constexpr int CH = 4 * VL;  // ranks of a chunk
    __shared__ float ts[16][kMaxLoraRank + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const GroupTile t = find_tile<16>(a.g, 1, blockIdx.x, lane);
    if (t.count <= 0) return;
    int mat = 0;
    while (mat + 1 < a.mats && (int)blockIdx.y >= a.block_end[mat]) ++mat;
    const int blk = ((int)blockIdx.y - (mat ? a.block_end[mat - 1] : 0)) * a.steps;
    const float* base = a.base[mat];
    float* y = a.y[mat];
    const bool none = t.group == a.g.groups;
    if (none && base == y) return;
    const int rank = none ? 0 : rank_of(a.ranks, a.max_rank, t.group);
    const int chunks = (rank + CH - 1) / CH;
    const int r = lane & 15, q = lane >> 4, n = a.n[mat];
    const size_t brow = none ? 0 : (size_t)t.group * n;
    const int cols = 64 * TILES, first = blk * cols + wave * 16 * TILES;
    const int steps = min(a.steps, (n - blk * cols + cols - 1) / cols);
    Piece<HALF, VL> w[2][TILES][NCH];
    auto load_b = [&](int n0, int c0, int buf) {
        if (rank == 0) return;
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                // (ranks past the adapter's are dropped where they are used)
                const int at = min(CH * (c0 + c) + VL * q, a.max_rank - VL);
                w[buf][j][c].load(a.b[mat], (brow + min(n0 + 16 * j + r, n - 1)) * a.max_rank + at);
            }
    };
    load_b(first, 0, 0);
    int e = r < t.count ? a.g.order[t.first + r] : -1;
    if ((uint32_t)e >= (uint32_t)a.g.entries) e = -1;
    const bool vec = n % 4 == 0;
    f32x4 s[2][TILES];
    const size_t out = (size_t)max(e, 0) * n + 4 * q;
    // (lanes past the rows or columns read what others read: no branches between the loads)
    const int e0 = __builtin_amdgcn_readfirstlane(max(e, 0));
    const float* from = base ? base + (size_t)(e < 0 ? e0 : e) * n : nullptr;
    auto load_base = [&](int n0, int buf) {
        if (!from || !vec) return;
#pragma unroll
        for (int j = 0; j < TILES; ++j) s[buf][j] = *(const f32x4*)(from + min(n0 + 16 * j + 4 * q, n - 4));
    };
    load_base(first, 0);
    const float scale = none ? 0.0f : a.scales ? a.scales[t.group] : 1.0f;
    // four neighbouring ranks of a row to a thread, every part's on its way at once
    const int tok = threadIdx.x >> 4, en0 = tok < t.count ? a.g.order[t.first + tok] : -1;
    const bool row = (uint32_t)en0 < (uint32_t)a.g.entries;
    for (int c = 4 * (threadIdx.x & 15); c < CH * chunks; c += 64) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row && c < rank) {
            const float* src = a.t + ((size_t)mat * a.parts * a.g.entries + en0) * a.max_rank + c;
            const size_t step = (size_t)a.g.entries * a.max_rank;
            f32x4 u[kMaxParts];
#pragma unroll
            for (int p = 0; p < kMaxParts; ++p)
                u[p] = p < a.parts ? *(const f32x4*)(src + p * step) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < kMaxParts; ++p) v += u[p];
#pragma unroll
            for (int k = 1; k < 4; ++k) v[k] = c + k < rank ? v[k] : 0.0f;  // (ranks past the adapter's are not written)
        }
        *(f32x4*)&ts[tok][c] = v * scale;
    }
    __syncthreads();
    auto step = [&]<int BUF>(int i) {
        const int n0 = first + i * cols;
        if (i + 1 < steps) {
            load_b(n0 + cols, 0, 1 - BUF);
            load_base(n0 + cols, 1 - BUF);
        }
        // the adapter's part apart from the projection's, which may be far larger, and then one addition
        f32x4 d[TILES];
#pragma unroll
        for (int j = 0; j < TILES; ++j) d[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c0 = 0; c0 < chunks; c0 += NCH) {
            if (c0 > 0) load_b(n0, c0, BUF);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (c0 + c >= chunks) break;
                const int at = CH * (c0 + c) + VL * q;
                float v[VL];
#pragma unroll
                for (int k = 0; k < VL; k += 4) {
                    const f32x4 x = *(const f32x4*)&ts[r][at + k];
                    v[k] = x.x, v[k + 1] = x.y, v[k + 2] = x.z, v[k + 3] = x.w;
                }
#pragma unroll
                for (int k = 0; k < VL; ++k)
#pragma unroll
                    for (int j = 0; j < TILES; ++j)  // (ranks past the adapter's: whatever stands there)
                        d[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(at + k < rank ? w[BUF][j][c].at(k) : 0.0f, v[k], d[j], 0, 0, 0);
            }
        }
        if (e < 0) return;
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            const int col = n0 + 16 * j + 4 * q;
            if (vec) {
                if (col < n) *(f32x4*)(y + out + n0 + 16 * j) = base ? s[BUF][j] + d[j] : d[j];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const size_t at = out + n0 + 16 * j + k;
                    if (col + k < n) y[at] = base ? base[at] + d[j][k] : d[j][k];
                }
            }
        }
    };
    for (int i = 0; i < steps; i += 2) {
        step.template operator()<0>(i);
        if (i + 1 < steps) step.template operator()<1>(i + 1);
    }
}

struct LoraPlan {
    int parts, k_part;
};
// K in parts of 512 and more, as many as make 1024 workgroups (at most 8). 512 | 1024 | 2048 workgroups, MI355X, us: 256
// rows of 16 adapters on q, k and v 18.8 | 17.0 | 17.2, 2045 rows of rank 32 43.7 | 42.1 | 42.2; elsewhere no difference.
LoraPlan lora_plan(int mats, int k, int groups, int rows) {
    const int wgs = std::max(1, std::min(tile_ids<16>(groups, rows), rows)) * mats;
    int parts = std::max(1, std::min((1024 + wgs - 1) / wgs, (k + 511) / 512));
    parts = std::min(parts, kMaxParts);
    LoraPlan p;
    p.k_part = ((k + parts - 1) / parts + 255) / 256 * 256;
    p.parts = (k + p.k_part - 1) / p.k_part;
    return p;
}

template <bool HALF, int VL>
hipError_t down_launch(Down& d, dim3 grid, int rt, hipStream_t s) {
    if (rt == 1)
        k_lora_down<HALF, VL, 1><<<grid, 256, 0, s>>>(d);
    else
        k_lora_down<HALF, VL, 2><<<grid, 256, 0, s>>>(d);
    return hipGetLastError();
}
template <bool HALF, int VL, int NCH>
hipError_t up_launch(Up& u, dim3 grid, int tiles, hipStream_t s) {
    if (tiles == 1)
        k_lora_up<HALF, VL, NCH, 1><<<grid, 256, 0, s>>>(u);
    else
        k_lora_up<HALF, VL, NCH, 2><<<grid, 256, 0, s>>>(u);
    return hipGetLastError();
}

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
    hipError_t e = !a.half ? down_launch<false, 4>(d, grid, rt, s)
                 : a.k % 8 == 0 ? down_launch<true, 8>(d, grid, rt, s) : down_launch<true, 4>(d, grid, rt, s);
    if (e != hipSuccess) return e;
    const unsigned up_tiles = (unsigned)tile_ids<16>(a.g.groups + 1, a.g.entries);
    // A wave's columns, 16 or 32 (rank sums read once for both). Few workgroups are better off with 16, as are many of short
    // ranks, whose loads of B then hide; long ranks are bound by the products. MI355X, us, 16 | 32, both launches: 16 rows,
    // 13 tiles 9.3 | 9.4; 300 rows of fp32 rank 32 x 4096 15.7 | 14.5; 128 rows 12.5 | 12.1; 512 rows 22.0 | 23.6, 1000 rows 28.9 |
    // 31.3, 2045 rows 42.2 | 47.2; 64 rows of 32 adapters of rank 64 x 28672 43.7 | 50.5; rank 256, 2045 rows 156 | 142
    int64_t pairs = 0;
    for (int i = 0; i < a.mats; ++i) pairs += (a.n[i] + 127) / 128;
    const int wide = up_tiles >= 16 && (a.max_rank > 64 || pairs * up_tiles < 1024) ? 2 : 1;
    int blocks = 0;
    for (int i = 0; i < a.mats; ++i) blocks += (a.n[i] + 64 * wide - 1) / (64 * wide);
    // column blocks of a workgroup: as many as leave 1024 workgroups, at most 8 (512 | 1024 | 2048 workgroups: 1000 rows
    // of rank 32 x 4096 25.7 | 23.8 | 25.1, 64 adapters of rank 16 in 64 rows 12.8 | 12.1 | 13.9, 2045 rows 42.2 | 42.1 | 44.2)
    u.steps = (int)std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)blocks * up_tiles / 1024));
    blocks = 0;
    for (int i = 0; i < a.mats; ++i)
        u.block_end[i] = blocks += (a.n[i] + 64 * wide * u.steps - 1) / (64 * wide * u.steps);
    if (blocks == 0) return hipSuccess;
    const dim3 up(up_tiles, (unsigned)blocks);
    if (!a.half) return up_launch<false, 4, 2>(u, up, wide, s);
    if (a.max_rank > 16 && a.max_rank % 8 == 0) return up_launch<true, 8, 2>(u, up, wide, s);
    return up_launch<true, 4, 1>(u, up, wide, s);
}

}  // namespace

// Room for the sums of every batch up to `rows`. The parts of K fall in steps as the rows grow, so what a batch writes,
// parts x rows, goes up and down: bounded here by what grows with the rows. A single row's parts are the most of all;
// and as parts < 1024 / workgroups + 1 and a workgroup has 16 rows at most, parts x rows < 16384 / mats + rows.
size_t lora_ws_bytes(int mats, int k, int max_rank, int groups, int rows) {
    const size_t most = (size_t)lora_plan(mats, k, groups, 1).parts * rows, split = (size_t)(16384 + mats - 1) / mats + rows;
    return (size_t)mats * std::min(most, split) * max_rank * sizeof(float);
}

hipError_t launch_lora(const LoraArgs& a, hipStream_t s) { return lora_launch(a, s); }

}  // namespace cllm_hip
