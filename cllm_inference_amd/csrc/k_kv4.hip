// k_kv4.hip -- the 4-bit paged KV cache: rows quantized into pages (with RoPE), pages read back,
// and grouped-query attention over them (kv4.h has the layout).
//
// Attention of query row t of head h, over the keys k_j and values v_j the row sees:
//   s_j = (q . k_j) / sqrt(HD),  y = sum_j exp(s_j) v_j / sum_j exp(s_j),
// in one pass over the cache with the running maximum and sum of each (row, head). The keys and
// values are exact fp16 numbers; the queries and the weights are fp32 and enter the fp16 MFMAs as
// hi + lo pairs (22 significant bits), accumulated in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "device_utils.h"
#include "kv4.h"
#include "launch.h"

namespace cllm_hip {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kTile = 32;  // positions of a tile

__device__ __forceinline__ f32x4 mfma(const h8& a, const h8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight codes of a dword as exact fp16 d * (c - 8): pairs 1024 + c, minus 1032, times d. d[r]
// scales codes 2 r and 2 r + 1. Every step is exact (kv4.h).
__device__ __forceinline__ h8 dequant8(uint32_t w, const h2 (&d)[4]) {
    const h2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    h2 p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t m = ((w >> (4 * r)) & 0x000F000Fu) | 0x64006400u;
        p[r] = (__builtin_bit_cast(h2, m) + off) * d[r];
    }
    return h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

__device__ __forceinline__ h2 pkrtz(float a, float b) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// Eight fp32 values as fp16 hi + lo. hi is rounded towards zero, so the remainder is exact.
__device__ __forceinline__ void split8(const float (&x)[8], h8& hi, h8& lo) {
    h2 a[4], b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        a[r] = pkrtz(x[2 * r], x[2 * r + 1]);
        b[r] = pkrtz(x[2 * r] - (float)a[r].x, x[2 * r + 1] - (float)a[r].y);
    }
    hi = h8{a[0].x, a[0].y, a[1].x, a[1].y, a[2].x, a[2].y, a[3].x, a[3].y};
    lo = h8{b[0].x, b[0].y, b[1].x, b[1].y, b[2].x, b[2].y, b[3].x, b[3].y};
}

__device__ __forceinline__ float max_over_g(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_over_g(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// What lane 16 g + n holds of a tile.
template <int HD>
struct TileRegs {
    static constexpr int KW = HD / 32;            // key dwords of either half
    static constexpr int NT = HD / 16, NB = HD / 32;
    uint32_t k[2][KW];
    uint32_t ks[HD == 256 ? 2 : 1];               // the lane's blocks: scales of both halves
    uint32_t v[NT];
    u32x4 vs[NB];

    __device__ __forceinline__ void load_k(const uint8_t* tile, int lane) {
        constexpr int W = KW < 4 ? KW : 4, C = KW / W;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint8_t* p = tile + ((t * C + c) * 64 + lane) * (4 * W);
                if constexpr (W == 4) {
                    const u32x4 x = *(const u32x4*)p;
                    k[t][4 * c] = x.x; k[t][4 * c + 1] = x.y; k[t][4 * c + 2] = x.z; k[t][4 * c + 3] = x.w;
                } else {
                    const u32x2 x = *(const u32x2*)p;
                    k[t][0] = x.x; k[t][1] = x.y;
                }
            }
        const uint32_t* s = (const uint32_t*)(tile + 32 * HD);
        const int g = lane >> 4, n = lane & 15;
        if constexpr (HD == 64) ks[0] = s[(g >> 1) * 16 + n];
        if constexpr (HD == 128) ks[0] = s[g * 16 + n];
        if constexpr (HD == 256) {
            ks[0] = s[(2 * g) * 16 + n];
            ks[1] = s[(2 * g + 1) * 16 + n];
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t* tile, int lane) {
#pragma unroll
        for (int c = 0; c < NT / 4; ++c) {
            const u32x4 x = *(const u32x4*)(tile + 16 * HD + (c * 64 + lane) * 16);
            v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = x.z; v[4 * c + 3] = x.w;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) vs[b] = *(const u32x4*)(tile + 34 * HD + (b * 4 + (lane >> 4)) * 16);
    }
    // Value scales of positions past `limit` (counted from the tile's start): bytes that no store
    // has written, which may be NaN.
    __device__ __forceinline__ void mask_v(int g, int limit) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = 16 * (r >> 1) + 4 * g + 2 * (r & 1);
            const uint32_t m = (p < limit ? 0x0000FFFFu : 0u) | (p + 1 < limit ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int b = 0; b < NB; ++b) vs[b][r] &= m;
        }
    }
    __device__ __forceinline__ h8 key(int t, int j) const {
        const uint32_t s = HD == 256 && j >= KW / 2 ? ks[HD == 256 ? 1 : 0] : ks[0];
        const uint32_t d = __builtin_amdgcn_perm(s, s, t ? 0x03020302u : 0x01000100u);
        const h2 dd = __builtin_bit_cast(h2, d);
        const h2 d4[4] = {dd, dd, dd, dd};
        return dequant8(k[t][j], d4);
    }
    __device__ __forceinline__ h8 value(int dt) const {
        const u32x4 s = vs[dt / 2];
        const h2 d4[4] = {__builtin_bit_cast(h2, (uint32_t)s.x), __builtin_bit_cast(h2, (uint32_t)s.y),
                          __builtin_bit_cast(h2, (uint32_t)s.z), __builtin_bit_cast(h2, (uint32_t)s.w)};
        return dequant8(v[dt], d4);
    }
};

// The 16 columns of a column tile: (row, head) pairs c = row * G + head in group of one KV head,
// column n of the tile in lanes 16 g + n.
template <int HD>
struct Queries {
    static constexpr int KW = HD / 32;
    h8 hi[KW], lo[KW];
    float sc;  // score in log2 units = product * sc

    // q row scaled by a power of two so that its largest element lies in [2^14, 2^15): hi and lo
    // then keep 22 significant bits of every element that counts.
    __device__ __forceinline__ void load(const float* row, bool valid, int g) {
        float x[KW][8];
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            if (valid) {
                const f32x4 a = *(const f32x4*)(row + g * (HD / 4) + 8 * j);
                const f32x4 b = *(const f32x4*)(row + g * (HD / 4) + 8 * j + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[j][i] = a[i];
                    x[j][4 + i] = b[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[j][i]));
        }
        m = max_over_g(m);
        int sh = 0;
        if (m > 0.0f && m < __builtin_huge_valf())
            sh = min(max(15 - __builtin_amdgcn_frexp_expf(m), -120), 120);
        sc = ldexpf(kLog2e / sqrtf((float)HD), -sh);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = ldexpf(x[j][i], sh);
            split8(x[j], hi[j], lo[j]);
        }
    }
};

// The place of one workgroup's work.
struct Place {
    Kv4Seq s;
    int h, c0;          // KV head, first column
    int n_cols;         // columns of the sequence and head: rows * G
    int kv_end;         // positions the tile's last row sees
    int vis_min;        // positions its first row sees
};
__device__ __forceinline__ Place place_of(const Kv4View& c, const int32_t* slots, const int32_t* q_start,
                                          int seq, int h, int ct, int cols, int G, int n_rows, int max_rows) {
    Place p;
    p.s = kv4_seq(c, slots, q_start, seq, n_rows);
    p.h = h;
    p.c0 = ct * cols;
    const int rows = min(p.s.rows, max_rows);  // rows past max_rows have no column tile
    p.n_cols = rows * G;
    const int t1 = min(rows - 1, (p.c0 + cols - 1) / G), t0 = p.c0 / G;
    p.kv_end = max(0, p.s.len - p.s.rows + t1 + 1);
    p.vis_min = p.s.len - p.s.rows + t0 + 1;
    return p;
}

// Tile tl of the place's sequence and head, null if it has no page.
__device__ __forceinline__ const uint8_t* tile_of(const Kv4View& c, int layer, const Place& p, int tl) {
    const int sub = c.page_shift - 5;
    const int page = c.table[(int64_t)p.s.slot * c.max_pages + (tl >> sub)];
    if ((unsigned)page >= (unsigned)c.n_pages) return nullptr;
    return c.pages + ((int64_t)layer * c.n_pages + page) * c.page_bytes +
           (((int64_t)p.h << sub) + (tl & ((1 << sub) - 1))) * (36 * c.hd);
}

// Partial results of split z for (row, head): unnormalised outputs part[((row * n_head + head) *
// splits + z) * HD], and the running maximum (log2 units) and sum in ml.
struct Parts {
    float* o;
    float* ml;
    int splits;
};

// grid: splits x column tiles x KV heads x sequences, one workgroup of four waves each. The waves
// walk the split's tiles alone (tile w, w + 4, ...), each with its own running maximum, and meet
// once at the end. A wave loads the keys of its next tile when the scores have been formed and the
// values when they have been used, so about 4.6 KB (HD 128) are in flight per wave.
template <int HD>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_kv4_attention(Kv4View c, int layer, const float* __restrict__ q,
                                                          const int32_t* __restrict__ slots,
                                                          const int32_t* __restrict__ q_start, int n_seqs,
                                                          int n_rows, int max_rows, int n_head, int col_tiles,
                                                          int chunk_tiles, Parts parts, float* __restrict__ out) {
    constexpr int NT = HD / 16, KW = HD / 32;
    const int G = n_head / c.n_kv;
    int b = blockIdx.x;
    const int sp = b % parts.splits;
    b /= parts.splits;
    const int ct = b % col_tiles;
    b /= col_tiles;
    const int h = b % c.n_kv;
    const Place pl = place_of(c, slots, q_start, b / c.n_kv, h, ct, 16, G, n_rows, max_rows);
    if (pl.c0 >= pl.n_cols) return;
    const int tiles = (pl.kv_end + kTile - 1) / kTile;
    const int n_splits = min(parts.splits, max(1, (tiles + chunk_tiles - 1) / chunk_tiles));
    if (sp >= n_splits) return;
    const int t_begin = sp * chunk_tiles, t_end = sp == n_splits - 1 ? tiles : t_begin + chunk_tiles;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int col = pl.c0 + n;
    const bool valid = col < pl.n_cols;
    const int row = col / G, head = h * G + (col - row * G);
    const int64_t qrow = (int64_t)(pl.s.r0 + row) * n_head + head;
    const int vis = valid ? pl.s.len - pl.s.rows + row + 1 : 0;

    Queries<HD> qs;
    qs.load(q + qrow * HD, valid, g);

    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNegInf, l = 0.0f;

    TileRegs<HD> r;
    int tl = t_begin + wave;
    const uint8_t* tile = nullptr;
    if (tl < t_end) {
        tile = tile_of(c, layer, pl, tl);
        if (tile) {
            r.load_k(tile, lane);
            r.load_v(tile, lane);
        }
    }
    while (tl < t_end) {
        const int next = tl + 4;
        const uint8_t* tile_next = next < t_end ? tile_of(c, layer, pl, next) : nullptr;
        if (tile) {
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KW; ++j) {
                    const h8 k = r.key(t, j);
                    s[t] = mfma(k, qs.hi[j], s[t]);
                    s[t] = mfma(k, qs.lo[j], s[t]);
                }
            }
            if (tile_next) r.load_k(tile_next, lane);
            const int p0 = tl * kTile;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * qs.sc;
            if (p0 + kTile > pl.vis_min) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (p0 + 16 * (e >> 2) + 4 * g + (e & 3) >= vis) x[e] = kNegInf;
                if (p0 + kTile > pl.s.len) r.mask_v(g, pl.s.len - p0);
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
            mx = max_over_g(mx);
            if (__any(mx > m)) {
                const float m_new = fmaxf(m, mx);
                const float a = m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= a;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i] *= a;
            }
            // weights times 2^15: as fp16 pairs they keep 22 bits down to 2^-29 of the largest
            const float mm = (m == kNegInf ? 0.0f : m) - 15.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(x[e] - mm);
                l += x[e];
            }
            h8 hi, lo;
            split8(x, hi, lo);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const h8 v = r.value(i);
                acc[i] = mfma(v, hi, acc[i]);
                acc[i] = mfma(v, lo, acc[i]);
            }
            if (tile_next) r.load_v(tile_next, lane);
        } else if (tile_next) {
            r.load_k(tile_next, lane);
            r.load_v(tile_next, lane);
        }
        tile = tile_next;
        tl = next;
    }
    l = sum_over_g(l);

    // the four waves' results meet: wave w's outputs of column n, elements 16 i + 4 g .. + 3
    __shared__ float sm[4][16], sl[4][16];
    __shared__ f32x4 so[4][16][HD / 4 + 1];
    if (g == 0) {
        sm[wave][n] = m;
        sl[wave][n] = l;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) so[wave][n][4 * i + g] = acc[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += 256) {
        const int cn = i / (HD / 4), d4 = i % (HD / 4);
        const int cc = pl.c0 + cn;
        if (cc >= pl.n_cols) continue;
        float mm = sm[0][cn];
#pragma unroll
        for (int w = 1; w < 4; ++w) mm = fmaxf(mm, sm[w][cn]);
        float ls = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (mm != kNegInf) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float a = __builtin_amdgcn_exp2f(sm[w][cn] - mm);
                ls += sl[w][cn] * a;
                o += so[w][cn][d4] * a;
            }
        } else {
            // nothing seen, or only NaN scores (their sums are NaN, an empty row's 0)
#pragma unroll
            for (int w = 0; w < 4; ++w) ls += sl[w][cn];
        }
        const int rr = cc / G, hh = h * G + (cc - rr * G);
        const int64_t idx = (int64_t)(pl.s.r0 + rr) * n_head + hh;
        if (n_splits == 1) {
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            *(f32x4*)(out + idx * HD + 4 * d4) = mm == kNegInf ? f32x4{ls, ls, ls, ls} : o * inv;
        } else {
            *(f32x4*)(parts.o + (idx * parts.splits + sp) * HD + 4 * d4) = o;
            if (d4 == 0) {
                parts.ml[(idx * parts.splits + sp) * 2] = mm;
                parts.ml[(idx * parts.splits + sp) * 2 + 1] = ls;
            }
        }
    }
}

// The splits of every (row, head) joined: grid column tiles x KV heads x sequences.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4View c, const int32_t* __restrict__ slots,
                                                  const int32_t* __restrict__ q_start, int n_rows, int max_rows,
                                                  int n_head, int cols, int col_tiles, int chunk_tiles, Parts parts,
                                                  float* __restrict__ out) {
    const int G = n_head / c.n_kv;
    int b = blockIdx.x;
    const int ct = b % col_tiles;
    b /= col_tiles;
    const int h = b % c.n_kv;
    const Place pl = place_of(c, slots, q_start, b / c.n_kv, h, ct, cols, G, n_rows, max_rows);
    if (pl.c0 >= pl.n_cols) return;
    const int tiles = (pl.kv_end + kTile - 1) / kTile;
    const int n_splits = min(parts.splits, max(1, (tiles + chunk_tiles - 1) / chunk_tiles));
    if (n_splits == 1) return;
    for (int i = threadIdx.x; i < cols * (HD / 4); i += 256) {
        const int cc = pl.c0 + i / (HD / 4), d4 = i % (HD / 4);
        if (cc >= pl.n_cols) break;
        const int rr = cc / G, hh = h * G + (cc - rr * G);
        const int64_t idx = (int64_t)(pl.s.r0 + rr) * n_head + hh;
        const float* ml = parts.ml + idx * parts.splits * 2;
        const float* po = parts.o + idx * parts.splits * HD + 4 * d4;
        float mm = kNegInf;
        for (int z = 0; z < n_splits; ++z) mm = fmaxf(mm, ml[2 * z]);
        float ls = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (mm != kNegInf) {
            for (int z = 0; z < n_splits; ++z) {
                const float a = __builtin_amdgcn_exp2f(ml[2 * z] - mm);
                ls += ml[2 * z + 1] * a;
                o += *(const f32x4*)(po + (int64_t)z * HD) * a;
            }
            o *= ls == 0.0f ? 0.0f : 1.0f / ls;
        } else {
            for (int z = 0; z < n_splits; ++z) ls += ml[2 * z + 1];
            o = f32x4{ls, ls, ls, ls};
        }
        *(f32x4*)(out + idx * HD + 4 * d4) = o;
    }
}

// ------------------------------------------------------------------------ store and load

// A segment: the rows of one sequence that fall into one tile. Workgroup `seg` of the grid finds
// its own: every wave counts the sequences' segments, 64 sequences a step, until it passes seg.
struct Segment {
    Kv4Seq s;
    int tile;    // -1: none
    int a, b;    // positions of the tile [a, b) that rows of the batch stand at
    int row;     // batch row of position a
};
__device__ __forceinline__ Segment find_segment(const Kv4View& c, const int32_t* slots,
                                                const int32_t* q_start, int n_seqs, int n_rows, int seg) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    Segment r;
    r.tile = -1;
    for (int i0 = 0; i0 < n_seqs; i0 += 64) {
        int count = 0;
        Kv4Seq s = {0, 0, 0, 0};
        if (i0 + lane < n_seqs) {
            s = kv4_seq(c, slots, q_start, i0 + lane, n_rows);
            const int p0 = max(0, s.len - s.rows);
            count = s.rows > 0 && s.len > p0 ? ((s.len - 1) >> 5) - (p0 >> 5) + 1 : 0;
        }
        int sum = count;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(sum, d, 64);
            if (lane >= d) sum += y;
        }
        const int total = __shfl(sum, 63, 64);
        if (seg < before + total) {
            const uint64_t past = __ballot(before + sum > seg);
            const int w = __builtin_ctzll(past);
            r.s.slot = __shfl(s.slot, w, 64);
            r.s.r0 = __shfl(s.r0, w, 64);
            r.s.rows = __shfl(s.rows, w, 64);
            r.s.len = __shfl(s.len, w, 64);
            const int first = __shfl(sum - count, w, 64) + before;
            const int p0 = max(0, r.s.len - r.s.rows);
            r.tile = (p0 >> 5) + (seg - first);
            const int base = r.tile * kTile;
            r.a = max(0, p0 - base);
            r.b = min(kTile, r.s.len - base);
            r.row = r.s.r0 + (base + r.a) - (r.s.len - r.s.rows);
            return r;
        }
        before += total;
    }
    return r;
}

// max(x) / 8 to 8 significant bits (round to nearest even, twice where fp16 is subnormal).
__device__ __forceinline__ _Float16 scale_of(float mx, float mn) {
    const float a = bf16_val(bf16_bits(fmaxf(mx, -mn) * 0.125f));
    const _Float16 d = (_Float16)fminf(a, 8160.0f);
    return -mn >= mx ? d : (_Float16)-d;
}

// x / d to the nearest integer, ties to even, exactly: the quotient's rounding is checked against
// the remainder, which an FMA gives without error (x and d * q agree to within d).
__device__ __forceinline__ uint32_t code_of(float x, float d, float inv) {
    float t = __builtin_rintf(x * inv);
    if (fabsf(t) < 16.0f) {
        const float rem = __builtin_fmaf(-t, d, x), half = 0.5f * fabsf(d);
        const float up = (rem < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f;  // the next integer on rem's side
        const bool odd = __builtin_fmaf(-2.0f, __builtin_floorf(0.5f * t), t) != 0.0f;
        if (fabsf(rem) > half || (fabsf(rem) == half && odd)) t += up;
    }
    t = fminf(fmaxf(t, -8.0f), 7.0f);
    return (uint32_t)((int)t + 8);
}

// grid (segments at most, KV heads [+ query head groups when q is rotated]). A workgroup reads the
// segment's rows of its head once, quantizes them into LDS and writes the tile's dwords. A dword of
// keys belongs to one position; a dword of values to eight, of which only the segment's change.
// theta_base > 0: keys turn by the NEOX rotation of k_rope_neox at their positions first, and the
// workgroups past the KV heads turn the query rows in place.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_store(Kv4View c, int layer, const float* __restrict__ k,
                                                   const float* __restrict__ v, float* __restrict__ q, int n_head,
                                                   float theta_base, const int32_t* __restrict__ slots,
                                                   const int32_t* __restrict__ q_start, int n_seqs, int n_rows) {
    constexpr int HALF = HD / 2, PER = HD / 8, NB = HD / 32;
    __shared__ float cs[kTile][HALF], sn[kTile][HALF], power[HALF];
    __shared__ uint8_t codes[2][kTile][HD + 4];
    __shared__ _Float16 scales[2][kTile][NB];
    __shared__ int bad[kTile];
    const Segment sg = find_segment(c, slots, q_start, n_seqs, n_rows, blockIdx.x);
    if (sg.tile < 0) return;
    const int tid = threadIdx.x;
    if (theta_base > 0.0f) {
        for (int i = tid; i < HALF; i += 256) power[i] = powf(theta_base, __fdiv_rn((float)i, (float)HALF));
        __syncthreads();
        for (int i = tid; i < (sg.b - sg.a) * HALF; i += 256) {
            const int p = sg.a + i / HALF, j = i % HALF;
            const float theta = __fdiv_rn((float)(sg.tile * kTile + p), power[j]);
            cs[p][j] = cosf(theta);
            sn[p][j] = sinf(theta);
        }
        __syncthreads();
    }
    if ((int)blockIdx.y >= c.n_kv) {  // query heads, as k_rope_neox
        const int h0 = ((int)blockIdx.y - c.n_kv) * 8, heads = min(8, n_head - h0);
        const int per_row = heads * HALF;
        for (int i = tid; i < (sg.b - sg.a) * per_row; i += 256) {
            const int p = i / per_row, hh = (i - p * per_row) / HALF, j = i % HALF;
            float* x = q + ((int64_t)(sg.row + p) * n_head + h0 + hh) * HD + j;
            const float x0 = x[0], x1 = x[HALF], co = cs[sg.a + p][j], si = sn[sg.a + p][j];
            x[0] = __builtin_fmaf(x0, co, -__fmul_rn(x1, si));
            x[HALF] = __builtin_fmaf(x0, si, __fmul_rn(x1, co));
        }
        return;
    }
    const int h = blockIdx.y;
    const int sub = c.page_shift - 5;
    const int page = c.table[(int64_t)sg.s.slot * c.max_pages + (sg.tile >> sub)];
    if ((unsigned)page >= (unsigned)c.n_pages) return;  // no page: the rows have no place
    uint8_t* tile = c.pages + ((int64_t)layer * c.n_pages + page) * c.page_bytes +
                    (((int64_t)h << sub) + (sg.tile & ((1 << sub) - 1))) * (36 * HD);
    if (tid < kTile) bad[tid] = 0;
    __syncthreads();

    // thread: position tid / 8, elements (tid % 8) * PER .. of both rows
    const int p = tid >> 3, d0 = (tid & 7) * PER;
    const bool on = p >= sg.a && p < sg.b;
    const int64_t src = ((int64_t)(sg.row + p - sg.a) * c.n_kv + h) * HD;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        float x[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = 0.0f;
        if (on) {
            const float* base = (kv ? v : k) + src;
#pragma unroll
            for (int i = 0; i < PER; i += 4) *(f32x4*)(x + i) = *(const f32x4*)(base + d0 + i);
            if (kv == 0 && theta_base > 0.0f) {
                const bool upper = d0 >= HALF;
                const int j0 = upper ? d0 - HALF : d0;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const float other = base[upper ? j0 + i : d0 + HALF + i];
                    const float co = cs[p][j0 + i], si = sn[p][j0 + i];
                    x[i] = upper ? __builtin_fmaf(other, si, __fmul_rn(x[i], co))
                                 : __builtin_fmaf(x[i], co, -__fmul_rn(other, si));
                }
            }
        }
        // a block's 32 elements lie in 32 / PER threads
        float mx = x[0], mn = x[0];
        bool finite = true;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            mx = fmaxf(mx, x[i]);
            mn = fminf(mn, x[i]);
            finite &= fabsf(x[i]) < __builtin_huge_valf();
        }
        if constexpr (PER <= 16) {
            mx = fmaxf(mx, dpp_f32<DPP_QUAD_SWAP1>(mx));
            mn = fminf(mn, dpp_f32<DPP_QUAD_SWAP1>(mn));
        }
        if constexpr (PER <= 8) {
            mx = fmaxf(mx, dpp_f32<DPP_QUAD_SWAP2>(mx));
            mn = fminf(mn, dpp_f32<DPP_QUAD_SWAP2>(mn));
        }
        if (on && !finite) bad[p] = 1;  // (every writer writes the same)
        const _Float16 dh = scale_of(mx, mn);
        const float d = (float)dh, inv = d == 0.0f ? 0.0f : 1.0f / d;
        if (on) {
#pragma unroll
            for (int i = 0; i < PER; ++i) codes[kv][p][d0 + i] = (uint8_t)(d == 0.0f ? 8u : code_of(x[i], d, inv));
            if (d0 % 32 == 0) scales[kv][p][d0 / 32] = dh;
        }
    }
    __syncthreads();

    // key dwords, in the tile's order
    constexpr int W = NB < 4 ? NB : 4, C = NB / W;
    for (int i = tid; i < 4 * HD; i += 256) {
        const int w = i % W, nn = i / W % 16, g = i / W / 16 % 4, t = i / W / 64 / C, cc = i / W / 64 % C;
        const int pos = 16 * t + nn;
        if (pos < sg.a || pos >= sg.b) continue;
        const uint8_t* e = &codes[0][pos][g * (HD / 4) + 8 * (cc * W + w)];
        uint32_t x = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) x |= (uint32_t)e[j] << (4 * (j / 2 + 4 * (j % 2)));
        ((uint32_t*)tile)[i] = bad[pos] ? 0x88888888u : x;
    }
    // value dwords
    const bool whole = sg.a == 0 && sg.b == kTile;
    for (int i = tid; i < 4 * HD; i += 256) {
        const int w = i % 4, nn = i / 4 % 16, g = i / 64 % 4, cc = i / 256;
        const int dim = 16 * (4 * cc + w) + nn;
        uint32_t x = 0, mask = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pos = 16 * (j / 4) + 4 * g + j % 4, sh = 4 * (j / 2 + 4 * (j % 2));
            if (pos >= sg.a && pos < sg.b) {
                x |= (uint32_t)(bad[pos] ? 8 : codes[1][pos][dim]) << sh;
                mask |= 15u << sh;
            }
        }
        if (!mask) continue;
        uint32_t* dst = (uint32_t*)(tile + 16 * HD) + i;
        *dst = whole ? x : (*dst & ~mask) | x;
    }
    // scales
    for (int i = tid; i < 2 * kTile * NB; i += 256) {
        const int kv = i / (kTile * NB), b = i / kTile % NB, pos = i % kTile;
        if (pos < sg.a || pos >= sg.b) continue;
        _Float16 d = scales[kv][pos][b];
        if (bad[pos]) d = kv ? (_Float16)0.0f : (_Float16)__builtin_nanf("");
        const int place = kv ? (b * 4 + pos % 16 / 4) * 8 + pos / 16 * 4 + pos % 4 : (b * 16 + pos % 16) * 2 + pos / 16;
        ((_Float16*)(tile + (kv ? 34 : 32) * HD))[place] = d;
    }
}

// The rows of the batch read back as fp32, d * (c - 8); rows without a place are 0.
// grid (segments at most + sequences, KV heads): the workgroups past the segments write the rows of
// sequences with more rows than positions that stand before the first position (0).
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_load(Kv4View c, int layer, const int32_t* __restrict__ slots,
                                                  const int32_t* __restrict__ q_start, int n_seqs, int n_rows,
                                                  int segments, float* __restrict__ k, float* __restrict__ v) {
    constexpr int NB = HD / 32;
    if ((int)blockIdx.x >= segments) {
        const Kv4Seq s = kv4_seq(c, slots, q_start, (int)blockIdx.x - segments, n_rows);
        for (int i = threadIdx.x; i < (s.rows - s.len) * HD; i += 256) {
            const int64_t at = ((int64_t)(s.r0 + i / HD) * c.n_kv + blockIdx.y) * HD + i % HD;
            k[at] = 0.0f;
            v[at] = 0.0f;
        }
        return;
    }
    const Segment sg = find_segment(c, slots, q_start, n_seqs, n_rows, blockIdx.x);
    if (sg.tile < 0) return;
    const int h = blockIdx.y, sub = c.page_shift - 5, tid = threadIdx.x;
    const int page = c.table[(int64_t)sg.s.slot * c.max_pages + (sg.tile >> sub)];
    const bool none = (unsigned)page >= (unsigned)c.n_pages;
    const uint8_t* tile = c.pages + ((int64_t)layer * c.n_pages + (none ? 0 : page)) * c.page_bytes +
                          (((int64_t)h << sub) + (sg.tile & ((1 << sub) - 1))) * (36 * HD);
    constexpr int W = NB < 4 ? NB : 4, C = NB / W;
    for (int i = tid; i < 4 * HD; i += 256) {
        const int w = i % W, nn = i / W % 16, g = i / W / 16 % 4, t = i / W / 64 / C, cc = i / W / 64 % C;
        const int pos = 16 * t + nn, dim = g * (HD / 4) + 8 * (cc * W + w);
        if (pos < sg.a || pos >= sg.b) continue;
        float* dst = k + ((int64_t)(sg.row + pos - sg.a) * c.n_kv + h) * HD + dim;
        float e[8] = {};
        if (!none) {
            const uint32_t x = ((const uint32_t*)tile)[i];
            const float d = (float)((const _Float16*)(tile + 32 * HD))[(dim / 32 * 16 + nn) * 2 + t];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = d * (float)((int)((x >> (4 * (j / 2 + 4 * (j % 2)))) & 15u) - 8);
        }
        *(f32x4*)dst = f32x4{e[0], e[1], e[2], e[3]};
        *(f32x4*)(dst + 4) = f32x4{e[4], e[5], e[6], e[7]};
    }
    for (int i = tid; i < 4 * HD; i += 256) {
        const int w = i / 64 % 4, nn = i % 16, g = i / 16 % 4, cc = i / 256;  // 16 elements side by side
        const int dim = 16 * (4 * cc + w) + nn;
        const uint32_t x = none ? 0 : ((const uint32_t*)(tile + 16 * HD))[((cc * 4 + g) * 16 + nn) * 4 + w];
        const _Float16* ds = (const _Float16*)(tile + 34 * HD) + (dim / 32 * 4 + g) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pos = 16 * (j / 4) + 4 * g + j % 4;
            if (pos < sg.a || pos >= sg.b) continue;
            const float y = none ? 0.0f : (float)ds[j] * (float)((int)((x >> (4 * (j / 2 + 4 * (j % 2)))) & 15u) - 8);
            v[((int64_t)(sg.row + pos - sg.a) * c.n_kv + h) * HD + dim] = y;
        }
    }
}

int segments_at_most(int n_seqs, int n_rows) {
    return (int)std::min<int64_t>(n_rows, (int64_t)n_rows / 32 + 2 * (int64_t)n_seqs);
}

}  // namespace

// ------------------------------------------------------------------------------- launchers

#define KV4_HD(hd, CALL)                   \
    switch (hd) {                          \
        case 64: { constexpr int HD = 64; CALL; } break;   \
        case 128: { constexpr int HD = 128; CALL; } break; \
        default: { constexpr int HD = 256; CALL; } break;  \
    }

hipError_t launch_kv4_store(const Kv4View& c, int layer, const float* k, const float* v, float* q,
                            int n_head, float theta_base, const int32_t* slots,
                            const int32_t* q_start, int n_seqs, int n_rows, hipStream_t stream) {
    const int groups = q && theta_base > 0.0f ? (n_head + 7) / 8 : 0;
    const dim3 grid((unsigned)segments_at_most(n_seqs, n_rows), (unsigned)(c.n_kv + groups));
    KV4_HD(c.hd, hipLaunchKernelGGL((k_kv4_store<HD>), grid, dim3(256), 0, stream, c, layer, k, v, q, n_head,
                                    theta_base, slots, q_start, n_seqs, n_rows));
    return hipGetLastError();
}

hipError_t launch_kv4_load(const Kv4View& c, int layer, const int32_t* slots, const int32_t* q_start,
                           int n_seqs, int n_rows, float* k, float* v, hipStream_t stream) {
    const int segments = segments_at_most(n_seqs, n_rows);
    const dim3 grid((unsigned)(segments + n_seqs), (unsigned)c.n_kv);
    KV4_HD(c.hd, hipLaunchKernelGGL((k_kv4_load<HD>), grid, dim3(256), 0, stream, c, layer, slots, q_start,
                                    n_seqs, n_rows, segments, k, v));
    return hipGetLastError();
}

Kv4AttnPlan kv4_attention_plan(const Kv4View& c, int n_seqs, int max_rows, int max_len, int n_head) {
    Kv4AttnPlan p;
    const int64_t cols = (int64_t)max_rows * (n_head / c.n_kv);
    p.kind = 0;
    p.col_tiles = (int)std::min<int64_t>((cols + 15) / 16, 1 << 30);
    // splits for two workgroups on each of 256 CUs, of four tiles (one per wave) at least
    const int tiles = std::max(1, (max_len + kTile - 1) / kTile);
    const int64_t groups = (int64_t)n_seqs * c.n_kv * p.col_tiles;
    const int want = (int)std::min<int64_t>(std::max<int64_t>(1, 1024 / std::max<int64_t>(1, groups)), tiles);
    p.chunk_tiles = std::max(4, ((tiles + want - 1) / want + 3) / 4 * 4);
    p.chunk_tiles = std::min(p.chunk_tiles, 64);
    p.splits = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
    return p;
}

size_t kv4_attention_ws_bytes(const Kv4AttnPlan& p, int n_rows, int n_head, int hd) {
    return p.splits == 1 ? 0 : (size_t)n_rows * n_head * p.splits * (hd + 2) * sizeof(float);
}

bool kv4_attention_fits(const Kv4AttnPlan& p, const Kv4View& c, int n_seqs) {
    return (double)p.splits * p.col_tiles * c.n_kv * n_seqs < 2147483647.0;
}

hipError_t launch_kv4_attention(const Kv4View& c, const Kv4AttnPlan& p, int layer, const float* q,
                                const int32_t* slots, const int32_t* q_start, int n_seqs, int n_rows,
                                int max_rows, int n_head, float* out, void* ws, hipStream_t stream) {
    Parts parts;
    parts.splits = p.splits;
    parts.o = (float*)ws;
    parts.ml = parts.o + (size_t)n_rows * n_head * p.splits * c.hd;
    const unsigned groups = (unsigned)(p.col_tiles * c.n_kv * n_seqs);
    KV4_HD(c.hd, hipLaunchKernelGGL((k_kv4_attention<HD>), dim3(groups * (unsigned)p.splits), dim3(256), 0, stream, c,
                                    layer, q, slots, q_start, n_seqs, n_rows, max_rows, n_head, p.col_tiles,
                                    p.chunk_tiles, parts, out));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    KV4_HD(c.hd, hipLaunchKernelGGL((k_kv4_join<HD>), dim3(groups), dim3(256), 0, stream, c, slots, q_start, n_rows,
                                    max_rows, n_head, 16, p.col_tiles, p.chunk_tiles, parts, out));
    return hipGetLastError();
}

}  // namespace cllm_hip
