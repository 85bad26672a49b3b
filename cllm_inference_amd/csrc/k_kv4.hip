// k_kv4.hip -- the 4-bit paged KV cache: rows quantized into pages (with RoPE), pages read back,
// and grouped-query attention over them (kv4.h has the layout).
//
// Attention of query row t of head h, over the keys k_j and values v_j the row sees:
//   s_j = (q . k_j) / sqrt(HD),  y = sum_j exp(s_j) v_j / sum_j exp(s_j),
// in one pass over the cache with the running maximum and sum of each (row, head). The keys and
// values are exact fp16 numbers (an MFMA keeps fewer bits of products with subnormal ones: kv4.h); the
// queries and the weights are fp32 and enter the fp16 MFMAs as hi + lo pairs (22 significant bits),
// accumulated in fp32.
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
// Weights are exp2(score - m + kTop), m the running maximum when the accumulators were last rescaled:
// they are not until a score passes m by kSlack (with scores of unit spread, a tile in three raised the
// maximum of some column). Weights stay within 2^15, and the fp16 parts of one that is the largest so far
// reach down to 2^-24, 2^-35 of it. The exponent is one FMA with kTop - m, whose rounding is common to a
// column's weights. From |m| = 2^23 on that and m's own would pass the slack: there the difference with m
// is formed first, of products rounded as m was, so that the largest weight stays within 2^15.
constexpr float kTop = 11.0f, kSlack = 4.0f, kFar = 8388608.0f;
__device__ __forceinline__ float far_from(float score, float sc, float m) {
#pragma clang fp contract(off)
    return score * sc - m;
}

__device__ __forceinline__ f32x4 mfma(const h8& a, const h8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight codes of a dword as exact fp16 d * (c - 8): the pair in bits 0-3 of the halves becomes
// 1024 + c, that in bits 4-7 64 + c (no shift), less 1032 or 72, times d. d[r] scales codes 2 r and
// 2 r + 1. Every step is exact (kv4.h). 13 VALU operations; an instruction reads one scalar
// register or literal, so the or's constants lie in vector registers (Magic): v_and_or_b32.
struct Magic {
    uint32_t m1024, m64;
    float minus1;  // (as a literal it would take v_fma_mix, which reads fp16, out of the products)
    __device__ __forceinline__ Magic() {
        asm("v_mov_b32 %0, 0x64006400" : "=v"(m1024));
        asm("v_mov_b32 %0, 0x54005400" : "=v"(m64));
        asm("v_mov_b32 %0, -1.0" : "=v"(minus1));
    }
};
__device__ __forceinline__ h8 dequant8(uint32_t w, const h2 (&d)[4], const Magic& mg) {
    const h2 off0 = {(_Float16)-1032.0f, (_Float16)-1032.0f}, off1 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t w8 = w >> 8;
    const h2 a = (__builtin_bit_cast(h2, (w & 0x000F000Fu) | mg.m1024) + off0) * d[0];
    const h2 b = (__builtin_bit_cast(h2, (w & 0x00F000F0u) | mg.m64) + off1) * d[1];
    const h2 e = (__builtin_bit_cast(h2, (w8 & 0x000F000Fu) | mg.m1024) + off0) * d[2];
    const h2 f = (__builtin_bit_cast(h2, (w8 & 0x00F000F0u) | mg.m64) + off1) * d[3];
    return h8{a.x, a.y, b.x, b.y, e.x, e.y, f.x, f.y};
}

__device__ __forceinline__ h2 pkrtz(float a, float b) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// Eight fp32 values as fp16 hi + lo. hi is rounded towards zero, so the remainder is exact.
__device__ __forceinline__ void split8(const float (&x)[8], h8& hi, h8& lo, const Magic& mg) {
    h2 a[4], b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        a[r] = pkrtz(x[2 * r], x[2 * r + 1]);
        b[r] = pkrtz(__builtin_fmaf((float)a[r].x, mg.minus1, x[2 * r]), __builtin_fmaf((float)a[r].y, mg.minus1, x[2 * r + 1]));
    }
    hi = h8{a[0].x, a[0].y, a[1].x, a[1].y, a[2].x, a[2].y, a[3].x, a[3].y};
    lo = h8{b[0].x, b[0].y, b[1].x, b[1].y, b[2].x, b[2].y, b[3].x, b[3].y};
}

// The high parts of eight values (low 0), or their low parts (low -1).
__device__ __forceinline__ h8 part8(const float (&x)[8], float low) {
    h2 b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const h2 a = pkrtz(x[2 * r], x[2 * r + 1]);
        b[r] = pkrtz(__builtin_fmaf((float)a.x, low, x[2 * r]), __builtin_fmaf((float)a.y, low, x[2 * r + 1]));
    }
    return h8{b[0].x, b[0].y, b[1].x, b[1].y, b[2].x, b[2].y, b[3].x, b[3].y};
}

// Over the four 16-lane rows of the wave (lanes of one column), in every lane.
__device__ __forceinline__ float max_over_g(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float sum_over_g(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// s_waitcnt vmcnt(N), and lgkmcnt(0) (gfx9 encoding, the other counters at max); no memory access
// moves across either.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}

// A tile loaded straight into LDS (36 * HD bytes at `slot`) by one wave, 16 bytes a lane, the last load
// by part of the lanes. The loads are the wave's own business: the compiler, which would wait for all
// of them before any LDS read, does not see them, and wait_loads orders the reads. (Nor does it see that a
// scalar write of M0 needs a wait state before the load: the s_nop.) ONCE: bytes that no
// other workgroup reads (nontemporal: 64 sequences of 4096-8192 positions 108.6 -> 104.0 us).
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint32_t m0) {
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(from), "s"(m0) : "memory",
                     "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(m0) : "memory", "m0");
}
template <int HD>
struct TileLoads {
    static constexpr int BYTES = 36 * HD, WHOLE = BYTES / 1024, REST = (BYTES - 1024 * WHOLE) / 16;
    static constexpr int COUNT = WHOLE + (REST > 0);
    template <bool ONCE>
    static __device__ __forceinline__ void issue(const uint8_t* tile, const uint8_t* slot, int lane) {
        const uint32_t m0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)slot;
#pragma unroll
        for (int i = 0; i < WHOLE; ++i) load_to_lds<ONCE>(tile + 1024 * i + 16 * lane, m0 + 1024 * i);
        if (REST > 0 && lane < REST) load_to_lds<ONCE>(tile + 1024 * WHOLE + 16 * lane, m0 + 1024 * WHOLE);
    }
};

// What lane 16 g + n reads of a tile in LDS: key fragments (rows are positions 16 t + n) and value
// fragments (rows are elements 16 dt + n), as exact fp16.
template <int HD>
struct TileView {
    static constexpr int KW = HD / 32, W = KW < 4 ? KW : 4, C = KW / W;
    uint8_t* p;
    int lane;

    // Key fragments c W .. c W + W - 1: the lane's elements there lie in one block.
    __device__ __forceinline__ void keys(int t, int c, h8 (&k)[W], const Magic& mg) const {
        const int g = lane >> 4, n = lane & 15;
        const uint32_t b = ((const uint32_t*)(p + 32 * HD))[(HD == 64 ? g >> 1 : HD == 128 ? g : 2 * g + c) * 16 + n];
        const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, b, t ? 0x03020302u : 0x01000100u));
        const h2 d4[4] = {d, d, d, d};
        const uint8_t* w = p + ((t * C + c) * 64 + lane) * (4 * W);
        if constexpr (W == 4) {
            const u32x4 x = *(const u32x4*)w;
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = dequant8(x[j], d4, mg);
        } else {
            const u32x2 x = *(const u32x2*)w;
#pragma unroll
            for (int j = 0; j < 2; ++j) k[j] = dequant8(x[j], d4, mg);
        }
    }
    // The value scales of positions from `limit` of the tile on become 0 in LDS: bytes that no store has
    // written may be NaN.
    __device__ __forceinline__ void mask_scales(int limit) const {
        uint16_t* s = (uint16_t*)(p + 34 * HD);
#pragma unroll
        for (int i = 0; i < HD; i += 64) {
            const int e = lane & 7, g = lane >> 3 & 3;
            if (16 * (e >> 2) + 4 * g + (e & 3) >= limit) s[i + lane] = 0;
        }
    }
    // Value fragments 4 c .. 4 c + 3.
    __device__ __forceinline__ void values(int c, h8 (&v)[4], const Magic& mg) const {
        const u32x4 x = *(const u32x4*)(p + 16 * HD + (c * 64 + lane) * 16);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const u32x4 s = *(const u32x4*)(p + 34 * HD + ((2 * c + b) * 4 + (lane >> 4)) * 16);
            const h2 d4[4] = {__builtin_bit_cast(h2, (uint32_t)s.x), __builtin_bit_cast(h2, (uint32_t)s.y),
                              __builtin_bit_cast(h2, (uint32_t)s.z), __builtin_bit_cast(h2, (uint32_t)s.w)};
            v[2 * b] = dequant8(x[2 * b], d4, mg);
            v[2 * b + 1] = dequant8(x[2 * b + 1], d4, mg);
        }
    }
};

// The 16 columns of the products' second operand. PARTS 1: column n is (row, head) pair n of the unit's
// 16, and there is a second operand for the low parts. PARTS 2: column n is the high (n even) or low part
// of pair n / 2 of the unit's 8, and half the products do.
template <int HD, int PARTS>
struct Queries {
    static constexpr int KW = HD / 32;
    h8 hi[KW], lo[PARTS == 1 ? KW : 1];
    float sc;  // score in log2 units = product * sc

    // q row scaled by a power of two so that its largest element lies in [2^14, 2^15): hi and lo
    // then keep 22 significant bits of every element that counts.
    __device__ __forceinline__ void load(const float* row, bool valid, int g, int n, const Magic& mg) {
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
        const float low = n & 1 ? mg.minus1 : 0.0f;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = ldexpf(x[j][i], sh);
            if constexpr (PARTS == 1) split8(x[j], hi[j], lo[j], mg); else hi[j] = part8(x[j], low);
        }
    }
};

// Sum over the two columns of a pair (neighbouring lanes), in both. (Every lane has a source, so the
// move needs no old value and folds into the addition.)
__device__ __forceinline__ float add_pair(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), DPP_QUAD_SWAP1, 0xF, 0xF, true));
}

// ---------------------------------------------------------------------------- the work's split
//
// A unit is a column tile of a KV head of a sequence: n tiles of positions (one at least, so that
// rows that see nothing are written too). Only the device knows the lengths:
//   direct: `splits` workgroups per unit; a unit of n tiles uses min(splits, ceil(n / kMinShare)) of
//   them, evenly, and the rest end at once. A workgroup finds its place from its index alone; with one
//   split there is nothing to join.
//   stream: the units' tiles lie end to end and workgroup w takes tiles [w Q, (w + 1) Q), found from
//   sums over the sequences that each wave forms 64 at a time: the work is even whatever the lengths
//   are, for a few restarts where a share crosses units and a join (8 to 20 us more than direct where
//   contexts are short).
// Direct up to kDirectUnits units or kDirectLen positions. One row, 8 KV heads of 128, us direct /
// stream: 16 sequences of 1000-8000 31 / 34; 24 of 1000-8000 56 / 41, of 100-6000 37 / 49, of 6000
// 46 / 40, of 4000 35 / 37; 64 of 1000-8000 90 / 77, of 4096-8192 102 / 95, of 6000 83 / 90, of 100-1000
// 17 / 29, of 300 12 / 22; 256 of 100-2000 76 / 133. The host knows max_len only: 24 of 6000 get the slower
// form, and short contexts under a max_len past kDirectLen (a captured call's bound) the stream's times.
// Partial results lie in slots (direct: unit * splits + split; stream: unit + workgroup, which grows
// along the staircase of pairs), and a second launch joins them.
constexpr int kCus = 256;
// Direct: workgroups at most, unless there are more units. 16 sequences of 1000-8000 (8 KV heads of 128), one, two,
// three and four a CU: 40.9, 31.1, 33.3, 35.2 us; 4 of 4000-8000 17.6, 16.9, 18.4, 21.3.
constexpr int kGrid = 2 * kCus;
constexpr int kDirectUnits = 128, kDirectLen = 6144;
// Tiles of a share: one sequence of 600 positions (8 KV heads of 128) 4 9.6 us, 8 10.8, 16 11.4; of 8000
// 15.3, 12.5, 13.7; 16 sequences of up to 2047 (2 KV heads of 64) 10.4, 10.0, 11.6.
constexpr int kMinShare = 8;

struct SeqWork {
    Kv4Seq s;
    int rows;           // computed: rows past max_rows have no column tile
    int units, tiles;   // units of the sequence, tiles of each
};
struct AttnArgs {
    const int32_t* slots;
    const int32_t* q_start;
    int n_seqs, n_rows, max_rows, n_head, G, cols;
};
__device__ __forceinline__ SeqWork seq_work(const Kv4View& c, const AttnArgs& a, int i) {
    SeqWork w;
    if (i >= a.n_seqs) {
        w.s = Kv4Seq{0, 0, 0, 0};
        w.rows = w.units = w.tiles = 0;
        return w;
    }
    w.s = kv4_seq(c, a.slots, a.q_start, i, a.n_rows);
    w.rows = min(w.s.rows, a.max_rows);
    w.units = c.n_kv * ((w.rows * a.G + a.cols - 1) / a.cols);
    w.tiles = max(1, (w.s.len - w.s.rows + w.rows + kTile - 1) / kTile);
    return w;
}
// The value of lane 0 (or of lane `at`), in scalar registers.
__device__ __forceinline__ int64_t scalar(int64_t v) {
    return ((int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ int64_t scalar(int64_t v, int at) {
    return ((int64_t)__builtin_amdgcn_readlane((int)(v >> 32), at) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, at);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up((long long)v, d, 64);
        if (lane >= d) v += y;
    }
    return v;
}

// Stream: the tiles of a share, and the place of tile f: its sequence, unit and tile there.
__device__ __forceinline__ int64_t share_of(const Kv4View& c, const AttnArgs& a, int grid, int64_t& total,
                                            int64_t& n_units, int lane) {
    int64_t tiles = 0, units = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += 64) {
        const SeqWork w = seq_work(c, a, i0 + lane);
        tiles += (int64_t)w.units * w.tiles;
        units += w.units;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        tiles += __shfl_xor((long long)tiles, d, 64);
        units += __shfl_xor((long long)units, d, 64);
    }
    n_units = scalar(units);
    total = scalar(tiles);
    const int64_t q = total < INT32_MAX / 2 ? (int64_t)(((uint32_t)total + (uint32_t)grid - 1) / (uint32_t)grid)
                                            : (total + grid - 1) / grid;
    return max((int64_t)kMinShare, q);
}
struct Found {
    SeqWork w;
    int unit, tile;           // of the sequence, of the unit
    int64_t units_before;     // of the sequences before
    bool ok;
};
__device__ __forceinline__ Found find_tile(const Kv4View& c, const AttnArgs& a, int64_t f, int lane) {
    int64_t items = 0, units = 0;
    Found r;
    r.ok = false;
    for (int i0 = 0; i0 < a.n_seqs; i0 += 64) {
        const SeqWork w = seq_work(c, a, i0 + lane);
        const int64_t mine = (int64_t)w.units * w.tiles;
        const int64_t incl = wave_scan(mine, lane), uincl = wave_scan((int64_t)w.units, lane);
        const uint64_t past = __ballot(items + incl > f);
        if (past) {
            const int at = __builtin_ctzll(past);
            r.w.s.slot = __builtin_amdgcn_readlane(w.s.slot, at);
            r.w.s.r0 = __builtin_amdgcn_readlane(w.s.r0, at);
            r.w.s.rows = __builtin_amdgcn_readlane(w.s.rows, at);
            r.w.s.len = __builtin_amdgcn_readlane(w.s.len, at);
            r.w.rows = __builtin_amdgcn_readlane(w.rows, at);
            r.w.units = __builtin_amdgcn_readlane(w.units, at);
            r.w.tiles = __builtin_amdgcn_readlane(w.tiles, at);
            r.units_before = units + scalar(uincl - w.units, at);
            const int64_t rest = f - items - scalar(incl - mine, at);
            r.unit = __builtin_amdgcn_readfirstlane(
                rest <= INT32_MAX ? (int)((uint32_t)rest / (uint32_t)r.w.tiles) : (int)(rest / r.w.tiles));
            r.tile = __builtin_amdgcn_readfirstlane((int)(rest - (int64_t)r.unit * r.w.tiles));
            r.ok = true;
            return r;
        }
        items += scalar(incl, 63);
        units += scalar(uincl, 63);
    }
    return r;
}

// Partial results of slot i and column n: unnormalised outputs o[(i * cols + n) * HD], the running
// maximum (log2 units) and sum ml[(i * cols + n) * 2].
// map (stream): what the join needs of every unit, and their number.
struct UnitMap {
    int64_t slot;
    int n_split, r0, rows, unit;
};
struct Parts {
    float* o;
    float* ml;
    UnitMap* map;
    int64_t* n_units;
};

// One workgroup of four waves per share. The waves walk a unit's tiles alone (tile w, w + 4, ...),
// each with its own running maximum, tiles coming through a ring of STAGES slots in LDS that the
// wave fills itself, and meet once at the unit's end.
//
// What bounds it: the read of the cache, and beside it about 240 VALU operations per tile and wave for
// dequantization (208 at HD 128) and the softmax of its 16 columns. 64 sequences of 4096-8192 positions,
// 32 + 8 heads of 128 (485 MB): 93 to 103 us with the join over several cards, 4.7 to 5.2 TB/s (its loads
// alone 83, a one-launch read 69); one sequence of 129: 7.2; 16 of up to 2047, 14 + 2 heads of 64: 10 to 11;
// 3 to 5 rows of 8 sequences of 800-4600, 16 + 4 heads of 256: 29, as its 20 columns are two units, each of which
// dequantizes every tile.
template <int HD>
struct AttnLds {
    // waves on a SIMD, which is workgroups on a CU, and slots a wave: within 512 registers and 160 KB
    // (64 sequences of 4096-8192 positions, HD 128: 2 and 4 101 us, 3 and 2 94, 4 and 2 103)
    static constexpr int WAVES = HD == 64 ? 4 : HD == 128 ? 3 : 2, STAGES = HD == 64 ? 4 : 2;
    static constexpr int RING = STAGES * 36 * HD;
    union {
        uint8_t ring[4][RING];
        f32x4 o[4][16][HD / 4 + 1];
    };
    float m[4][16], l[4][16];
};

template <int HD, int PARTS>
__global__ __launch_bounds__(256, AttnLds<HD>::WAVES) void k_kv4_attention(Kv4View c, int layer, const float* __restrict__ q,
                                                          AttnArgs a, int splits, bool once, Parts parts,
                                                          float* __restrict__ out) {
    constexpr int NT = HD / 16, W = TileView<HD>::W, COLS = 16 / PARTS, STAGES = AttnLds<HD>::STAGES, NL = TileLoads<HD>::COUNT;
    extern __shared__ __align__(16) uint8_t lds_bytes[];
    AttnLds<HD>& lds = *(AttnLds<HD>*)lds_bytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const Magic mg;
    const int sub = c.page_shift - 5;
    const uint8_t* const layer_pages = c.pages + (int64_t)layer * c.n_pages * c.page_bytes;
    int64_t f = 0, f_end = 1, share = 0;  // direct: one unit; stream: tiles
    if (splits == 0) {
        int64_t n_units;
        share = share_of(c, a, gridDim.x, f_end, n_units, lane);
        if (blockIdx.x == 0 && threadIdx.x == 0) *parts.n_units = n_units;
        f = blockIdx.x * share;
        f_end = min(f + share, f_end);
    }

    while (f < f_end) {
        // the unit (of its sequence), its tiles [t_begin, t_end) of this workgroup, whether it is split
        SeqWork w;
        int unit, t_begin, t_end;
        int64_t slot;
        bool split;
        if (splits > 0) {
            f = f_end;
            const int u = (int)blockIdx.x / splits, z = (int)blockIdx.x - u * splits;
            const int per_seq = c.n_kv * ((a.max_rows * a.G + COLS - 1) / COLS);
            const int seq = u / per_seq;
            unit = u - seq * per_seq;
            w = seq_work(c, a, seq);
            const int n_split = min(splits, (w.tiles + kMinShare - 1) / kMinShare);
            if (unit >= w.units || z >= n_split) return;
            t_begin = (int)((int64_t)w.tiles * z / n_split);
            t_end = (int)((int64_t)w.tiles * (z + 1) / n_split);
            split = n_split > 1;
            slot = blockIdx.x;
        } else {
            const Found u = find_tile(c, a, f, lane);
            if (!u.ok) return;
            w = u.w;
            unit = u.unit;
            t_begin = u.tile;
            t_end = (int)min((int64_t)w.tiles, t_begin + (f_end - f));
            split = t_begin > 0 || t_end < w.tiles;
            slot = u.units_before + unit + blockIdx.x;
            if (t_begin == 0 && threadIdx.x == 0) {
                const int64_t last = (f + w.tiles - 1) / share;
                parts.map[u.units_before + unit] =
                    UnitMap{slot, (int)(last - blockIdx.x) + 1, w.s.r0, w.rows, unit};
            }
            f += t_end - t_begin;
        }
        const int h = unit % c.n_kv, c0 = unit / c.n_kv * COLS, n_cols = w.rows * a.G;
        const int col = c0 + n / PARTS;
        const bool valid = col < n_cols;
        const int row = col / a.G, head = h * a.G + (col - row * a.G);
        const int vis = valid ? w.s.len - w.s.rows + row + 1 : 0;       // positions the column sees
        const int vis_min = w.s.len - w.s.rows + c0 / a.G + 1;          // and the tile's first row
        // the column tile's last row sees no tile from here on
        const int last_row = min(w.rows - 1, (c0 + COLS - 1) / a.G);
        t_end = min(t_end, max(t_begin, (max(0, w.s.len - w.s.rows + last_row + 1) + kTile - 1) / kTile));

        // The wave's tiles first, first + 4, ...: a lane holds the page id of every 64th. A tile
        // without a page loads the first bytes of page 0 instead, and all of it is masked: holes
        // keeps a bit for each tile in the ring, the one in turn lowest.
        const int first = t_begin + wave;
        const int count = first < t_end ? (t_end - first + 3) / 4 : 0;
        const int32_t* table = c.table + (int64_t)w.s.slot * c.max_pages;
        int ids = -1;
        uint32_t holes = 0;
        const auto issue = [&](int i, int ahead) {
            if ((i & 63) == 0) {
                const int tl = first + 4 * (i + lane);
                ids = tl < t_end ? table[tl >> sub] : -1;
            }
            const int tl = first + 4 * i, page = __builtin_amdgcn_readlane(ids, i & 63);
            const bool none = (unsigned)page >= (unsigned)c.n_pages;
            const uint8_t* p = layer_pages;
            if (!none) p += page * c.page_bytes + (((int64_t)h << sub) + (tl & ((1 << sub) - 1))) * (36 * HD);
            holes |= (none ? 1u : 0u) << ahead;
            const uint8_t* slot_lds = lds.ring[wave] + (i % STAGES) * (36 * HD);
            if (once) TileLoads<HD>::template issue<true>(p, slot_lds, lane);
            else TileLoads<HD>::template issue<false>(p, slot_lds, lane);
        };
        for (int i = 0; i < min(count, STAGES - 1); ++i) issue(i, i);

        Queries<HD, PARTS> qs;
        qs.load(q + ((int64_t)(w.s.r0 + row) * a.n_head + head) * HD, valid, g, n, mg);
        f32x4 acc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = kNegInf, l = 0.0f;
        bool far = false;  // a column's maximum is kFar or more from 0 (of all lanes)
        const float low = n & 1 ? mg.minus1 : 0.0f;  // (PARTS 2)

        // edge: the tile ends past what some column sees, or past the sequence, or has no page (len 0)
        const auto step = [&](const TileView<HD>& tv, int p0, int len, bool edge) {
            if (edge) tv.mask_scales(len - p0);
            f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int kc = 0; kc < TileView<HD>::C; ++kc) {
                h8 k[2][W];
#pragma unroll
                for (int t = 0; t < 2; ++t) tv.keys(t, kc, k[t], mg);
#pragma unroll
                for (int j = 0; j < W; ++j) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) s[t] = mfma(k[t][j], qs.hi[kc * W + j], s[t]);
                    if constexpr (PARTS == 1) {
#pragma unroll
                        for (int t = 0; t < 2; ++t) s[t] = mfma(k[t][j], qs.lo[kc * W + j], s[t]);
                    }
                }
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = PARTS == 1 ? s[e >> 2][e & 3] : add_pair(s[e >> 2][e & 3]);
            if (edge) {
                const int end = min(vis, len) - p0 - 4 * g;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 16 * (e >> 2) + (e & 3) >= end ? kNegInf : x[e];
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
            mx = max_over_g(mx) * qs.sc;
            float sc = qs.sc, mm = kTop - (m == kNegInf ? 0.0f : m);
            if (__any(mx > m + kSlack) || far) {
                const float m_new = fmaxf(m, mx);
                const float r = m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= r;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i] *= r;
                const float base = m == kNegInf ? 0.0f : m;
                mm = kTop - base;
                far = __any(fabsf(base) >= kFar);
                if (__builtin_expect(far, 0)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = far_from(x[e], sc, base);
                    sc = 1.0f;
                    mm = kTop;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], sc, mm));
                l += x[e];
            }
            h8 hi, lo;
            if constexpr (PARTS == 1) split8(x, hi, lo, mg); else hi = part8(x, low);
#pragma unroll
            for (int cc = 0; cc < NT / 4; ++cc) {
                h8 v[4];
                tv.values(cc, v, mg);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[4 * cc + i] = mfma(v[i], hi, acc[4 * cc + i]);
                if constexpr (PARTS == 1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[4 * cc + i] = mfma(v[i], lo, acc[4 * cc + i]);
                }
            }
        };
        for (int i = 0; i < count; ++i) {
            if (i + STAGES - 1 < count) {
                wait_lds();  // the reads of the slot's last tile have returned
                issue(i + STAGES - 1, STAGES - 1);
                wait_loads<(STAGES - 1) * NL>();
            } else {
                wait_loads<0>();
            }
            const bool hole = holes & 1u;
            holes >>= 1;
            const int p0 = (first + 4 * i) * kTile;
            const TileView<HD> tv = {lds.ring[wave] + (i % STAGES) * (36 * HD), lane};
            step(tv, p0, hole ? 0 : w.s.len, hole || p0 + kTile > vis_min || p0 + kTile > w.s.len);
        }
        if constexpr (PARTS == 2) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = add_pair(acc[i][j]);
        }
        l = sum_over_g(l);

        // the four waves' results meet (in the ring's place): outputs of column n, elements 16 i + 4 g
        // .. + 3 of each wave
        if (g == 0 && n % PARTS == 0) {
            lds.m[wave][n / PARTS] = m;
            lds.l[wave][n / PARTS] = l;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (PARTS == 1 || i % 2 == n % 2) lds.o[wave][n / PARTS][4 * i + g] = acc[i];
        __syncthreads();
        for (int i = threadIdx.x; i < COLS * (HD / 4); i += 256) {
            const int cn = i / (HD / 4), d4 = i % (HD / 4);
            const int cc = c0 + cn;
            if (cc >= n_cols) break;
            float mm = lds.m[0][cn];
#pragma unroll
            for (int v = 1; v < 4; ++v) mm = fmaxf(mm, lds.m[v][cn]);
            float ls = 0.0f;
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
            if (mm != kNegInf) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float r = __builtin_amdgcn_exp2f(lds.m[v][cn] - mm);
                    ls += lds.l[v][cn] * r;
                    o += lds.o[v][cn][d4] * r;
                }
            } else {
                // nothing seen, or only NaN scores (their sums are NaN, an empty row's 0)
#pragma unroll
                for (int v = 0; v < 4; ++v) ls += lds.l[v][cn];
            }
            if (!split) {
                const int rr = cc / a.G, hh = h * a.G + (cc - rr * a.G);
                const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                *(f32x4*)(out + ((int64_t)(w.s.r0 + rr) * a.n_head + hh) * HD + 4 * d4) =
                    mm == kNegInf ? f32x4{ls, ls, ls, ls} : o * inv;
            } else {
                *(f32x4*)(parts.o + (slot * COLS + cn) * HD + 4 * d4) = o;
                if (d4 == 0) {
                    parts.ml[(slot * COLS + cn) * 2] = mm;
                    parts.ml[(slot * COLS + cn) * 2 + 1] = ls;
                }
            }
        }
        __syncthreads();  // the LDS is free for the next unit's tiles
    }
}

// ------------------------------------------------------------------------------- many rows
//
// A workgroup of eight waves has COLS (row, head) pairs of a KV head, NC column tiles of 16 to a wave.
// Waves 0-3 take the first half of a turn's TURN tiles, waves 4-7, with the same columns, the second
// half; the two meet at the end. Tiles are dequantized once for all waves, into fp16 fragments in LDS
// (fragment, lane, 16 bytes: no bank is hit twice), a turn at a time in two buffers: the codes of the
// turn after the next are loaded while the next one's fragments are written and the present ones are
// multiplied, with one barrier a turn.
//
// What bounds it: VALU and MFMA work that overlap little, and waiting. 32 positions x 32 columns of HD 128
// take 64 MFMAs of 16 cycles (two parts of the queries, two of the weights) and about 190 VALU operations, 75
// of them the wave's share of the dequantization. Counters, prompt / second turns below: a CU has work in 86 /
// 72% of the time; of a SIMD's cycles then MFMA takes 33 / 39% and VALU 38 / 40%, LDS is busy 13 / 15% without
// conflicts, and a wave waits for 36 / 33% (for the barrier of a turn and the loads). One prompt of 2048, 32 + 8
// heads of 128: 91 us (34.4 GFLOP; 760 TFLOP/s of both parts' products); 288-499 rows of 4 sequences of
// 2345-4744: 217 to 224 us (720). (At the clock of a long run; the first launches of a short one take 103 and
// 246.) Heads of 64 and 256, four sequences of 1500-6000: 135 and 416.
template <int HD>
struct ManyRows {
    static constexpr int NC = HD == 64 ? 4 : HD == 128 ? 2 : 1, COLS = 4 * NC * 16;
    static constexpr int FRAGS = HD / 8;  // of a tile: HD / 16 of keys, then HD / 16 of values
    static constexpr int TURN = HD == 256 ? 2 : 4;
    static constexpr int RING = 2 * TURN * FRAGS * 1024;
    // the second half's results: accumulators, then maxima and sums
    static constexpr int MEET = 4 * NC * (HD / 16) * 1024, LDS = RING > MEET + 4 * NC * 512 ? RING : MEET + 4 * NC * 512;
    // a tile is staged in KINDS pieces of four fragments, HD / 64 of keys and HD / 64 of values
    static constexpr int KINDS = HD / 32, STAGED = TURN * KINDS / 8;
};

// A wave's piece of a tile on its way to LDS: 16 bytes of codes a lane, four fragments. Key pieces are
// chunks (t, c) of the tile's key codes (HD 64: both halves t), value pieces chunks c of its value codes.
template <int HD>
struct Staged {
    static constexpr int KW = HD / 32, KEYS = HD / 64;
    u32x4 x, s0, s1;
    int limit;  // positions of the tile with values (0: no page)

    __device__ __forceinline__ void load(const uint8_t* tile, int limit_, int kind, int lane) {
        limit = tile ? limit_ : 0;
        if (!tile) return;
        const int g = lane >> 4, n = lane & 15;
        if (kind < KEYS) {
            if constexpr (HD == 64) {
                const u32x2 a = *(const u32x2*)(tile + lane * 8), b = *(const u32x2*)(tile + 512 + lane * 8);
                x = u32x4{a.x, a.y, b.x, b.y};
                s0.x = ((const uint32_t*)(tile + 32 * HD))[(g >> 1) * 16 + n];
            } else {
                x = *(const u32x4*)(tile + (kind * 64 + lane) * 16);
                s0.x = ((const uint32_t*)(tile + 32 * HD))[(HD == 128 ? g : 2 * g + (kind & 1)) * 16 + n];
            }
        } else {
            const int c = kind - KEYS;
            x = *(const u32x4*)(tile + 16 * HD + (c * 64 + lane) * 16);
            s0 = *(const u32x4*)(tile + 34 * HD + ((2 * c) * 4 + g) * 16);
            s1 = *(const u32x4*)(tile + 34 * HD + ((2 * c + 1) * 4 + g) * 16);
        }
    }
    __device__ __forceinline__ void store(uint8_t* frags, int kind, int lane, const Magic& mg) {
        if (kind < KEYS) {
            const auto put = [&](uint32_t w, int t, int j) {
                const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(s0.x, s0.x, t ? 0x03020302u : 0x01000100u));
                const h2 d4[4] = {d, d, d, d};
                *(h8*)(frags + (t * KW + j) * 1024 + lane * 16) = dequant8(w, d4, mg);
            };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (HD == 64) put(x[i], i >> 1, i & 1);
                if constexpr (HD == 128) put(x[i], kind, i);
                if constexpr (HD == 256) put(x[i], kind >> 1, (kind & 1) * 4 + i);
            }
        } else {
            if (limit < kTile) {  // bytes that no store has written: their scales may be NaN
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = 16 * (r >> 1) + 4 * (lane >> 4) + 2 * (r & 1);
                    const uint32_t m = (at < limit ? 0x0000FFFFu : 0u) | (at + 1 < limit ? 0xFFFF0000u : 0u);
                    s0[r] &= m;
                    s1[r] &= m;
                }
            }
            const int c = kind - KEYS;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 s = i < 2 ? s0 : s1;
                const h2 d4[4] = {__builtin_bit_cast(h2, (uint32_t)s.x), __builtin_bit_cast(h2, (uint32_t)s.y),
                                  __builtin_bit_cast(h2, (uint32_t)s.z), __builtin_bit_cast(h2, (uint32_t)s.w)};
                *(h8*)(frags + (HD / 16 + 4 * c + i) * 1024 + lane * 16) = dequant8(x[i], d4, mg);
            }
        }
    }
};

// grid units * splits, the heaviest first, so that the last ones to start are short: the sequences by
// their tiles (up to 64 of them), the last rows of a sequence before the first, and all KV heads of a
// column tile side by side.
template <int HD>
__global__ __launch_bounds__(512, 2) void k_kv4_many_rows(Kv4View c, int layer, const float* __restrict__ q,
                                                          AttnArgs a, int splits, Parts parts,
                                                          float* __restrict__ out) {
    using S = ManyRows<HD>;
    constexpr int NT = HD / 16, KW = HD / 32, NC = S::NC, TURN = S::TURN;
    extern __shared__ __align__(16) uint8_t lds_bytes[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = wave >> 2, cw = wave & 3;
    const int g = lane >> 4, n = lane & 15;
    const Magic mg;

    const int cts = (a.max_rows * a.G + S::COLS - 1) / S::COLS;
    int b = blockIdx.x;
    const int h = b % c.n_kv;
    b /= c.n_kv;
    const int z = b % splits;
    b /= splits;
    const int from_last = b % cts;
    int seq = b / cts;
    if (a.n_seqs <= 64) {
        const int mine = lane < a.n_seqs ? seq_work(c, a, lane).tiles : -1;
        int rank = 0;
        for (int j = 0; j < a.n_seqs; ++j) {
            const int t = __builtin_amdgcn_readlane(mine, j);
            rank += t > mine || (t == mine && j < lane);
        }
        seq = __builtin_ctzll(__ballot(rank == seq && lane < a.n_seqs));
    }
    const SeqWork w = seq_work(c, a, seq);
    const int n_cols = w.rows * a.G, my_cts = (n_cols + S::COLS - 1) / S::COLS;
    if (from_last >= my_cts) return;
    const int ct = my_cts - 1 - from_last, c0 = ct * S::COLS;
    const int p0_seq = w.s.len - w.s.rows;  // position of row 0
    const int last_row = min(w.rows - 1, (c0 + S::COLS - 1) / a.G);
    // the unit's own tiles in as many splits as the join counts (by the sequence's)
    const int tiles = max(1, (max(0, p0_seq + last_row + 1) + kTile - 1) / kTile);
    const int n_split = min(splits, (w.tiles + kMinShare - 1) / kMinShare);
    if (z >= n_split) return;
    const int t_begin = (int)((int64_t)tiles * z / n_split), t_end = (int)((int64_t)tiles * (z + 1) / n_split);

    const int sub = c.page_shift - 5;
    const int32_t* table = c.table + (int64_t)w.s.slot * c.max_pages;
    const uint8_t* const layer_pages = c.pages + (int64_t)layer * c.n_pages * c.page_bytes;
    // the wave's pieces of a turn: the same kind of tiles wave / KINDS, + 8 / KINDS
    const int kind = wave % S::KINDS, tile0 = wave / S::KINDS;
    Staged<HD> st[S::STAGED];
    uint32_t holes = 0;  // a bit per tile of the turn
    int ids = -1;        // page ids of 64 tiles, one a lane
    const auto load = [&](int t0) {
        holes = 0;
        const int at = (t0 - t_begin) & 63;
        if (at == 0) ids = t0 + lane < t_end ? table[(t0 + lane) >> sub] : -1;
#pragma unroll
        for (int i = 0; i < TURN; ++i) {
            const int tl = t0 + i, page = __builtin_amdgcn_readlane(ids, at + i);
            const uint8_t* p = nullptr;
            if ((unsigned)page < (unsigned)c.n_pages)
                p = layer_pages + page * c.page_bytes + (((int64_t)h << sub) + (tl & ((1 << sub) - 1))) * (36 * HD);
            holes |= (p == nullptr ? 1u : 0u) << i;
            if (i % (8 / S::KINDS) == tile0) st[i / (8 / S::KINDS)].load(p, min(kTile, w.s.len - tl * kTile), kind, lane);
        }
    };
    const auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < S::STAGED; ++i)
            st[i].store(lds_bytes + (buf * TURN + tile0 + i * (8 / S::KINDS)) * S::FRAGS * 1024, kind, lane, mg);
    };

    load(t_begin);
    uint32_t holes_now = holes;

    // this wave's columns
    Queries<HD, 1> qs[NC];
    int vis[NC];
    int wave_vis = 0, wave_min = INT32_MAX;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int first = c0 + (cw * NC + i) * 16, col = first + n;
        const bool valid = col < n_cols;
        const int row = valid ? col / a.G : 0, head = h * a.G + (valid ? col - row * a.G : 0);
        vis[i] = valid ? max(0, p0_seq + row + 1) : 0;
        qs[i].load(q + ((int64_t)(w.s.r0 + row) * a.n_head + head) * HD, valid, g, n, mg);
        if (first < n_cols) {
            wave_vis = max(wave_vis, max(0, p0_seq + min(w.rows - 1, (first + 15) / a.G) + 1));
            wave_min = min(wave_min, max(0, p0_seq + first / a.G + 1));
        }
    }
    f32x4 acc[NC][NT];
    float m[NC], l[NC];
    bool far = false;  // a column's maximum is kFar or more from 0 (of all lanes)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        m[i] = kNegInf;
        l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const auto step = [&](const uint8_t* frags, int p0, bool hole) {
        // (the wave that forms scores goes first: its neighbour's softmax fills the gaps; 3% less time)
        __builtin_amdgcn_s_setprio(1);
        f32x4 s[NC][2];
#pragma unroll
        for (int i = 0; i < NC; ++i) s[i][0] = s[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KW; ++j) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const h8 k = *(const h8*)(frags + (t * KW + j) * 1024 + lane * 16);
#pragma unroll
                for (int i = 0; i < NC; ++i) s[i][t] = mfma(k, qs[i].hi[j], s[i][t]);
#pragma unroll
                for (int i = 0; i < NC; ++i) s[i][t] = mfma(k, qs[i].lo[j], s[i][t]);
            }
        }
        if (hole || p0 + kTile > wave_min) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int end = hole ? -1 : vis[i] - p0 - 4 * g;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    s[i][e >> 2][e & 3] = 16 * (e >> 2) + (e & 3) >= end ? kNegInf : s[i][e >> 2][e & 3];
            }
        }
        float mx[NC];
        bool grow = false;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            mx[i] = s[i][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx[i] = fmaxf(mx[i], s[i][e >> 2][e & 3]);
            mx[i] = max_over_g(mx[i]) * qs[i].sc;
            grow |= mx[i] > m[i] + kSlack;
        }
        float sc[NC], mm[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            sc[i] = qs[i].sc;
            mm[i] = kTop - (m[i] == kNegInf ? 0.0f : m[i]);
        }
        if (__any(grow) || far) {
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const float m_new = fmaxf(m[i], mx[i]);
                const float r = m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m[i] - m_new);
                m[i] = m_new;
                l[i] *= r;
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] *= r;
                const float base = m[i] == kNegInf ? 0.0f : m[i];
                mm[i] = kTop - base;
                most = fmaxf(most, fabsf(base));
            }
            far = __any(most >= kFar);
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    const float base = m[i] == kNegInf ? 0.0f : m[i];
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[i][e >> 2][e & 3] = far_from(s[i][e >> 2][e & 3], sc[i], base);
                    sc[i] = 1.0f;
                    mm[i] = kTop;
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        h8 hi[NC], lo[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e >> 2][e & 3], sc[i], mm[i]));
                l[i] += x[e];
            }
            split8(x, hi[i], lo[i], mg);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const h8 v = *(const h8*)(frags + (NT + j) * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[i][j] = mfma(v, hi[i], acc[i][j]);
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[i][j] = mfma(v, lo[i], acc[i][j]);
        }
    };

    put(0);
    load(t_begin + TURN);
    __syncthreads();
    int buf = 0;
    for (int t0 = t_begin; t0 < t_end; t0 += TURN, buf ^= 1) {
        // of the two waves on a SIMD (w and w + 4) one writes its fragments before its steps and one
        // after, so that the one's VALU work runs beside the other's MFMAs
        const uint32_t holes_next = holes;
        if (half == 0 && t0 + TURN < t_end) {
            put(buf ^ 1);
            load(t0 + 2 * TURN);
        }
#pragma unroll
        for (int i = 0; i < TURN / 2; ++i) {
            const int tl = t0 + half * (TURN / 2) + i, p0 = tl * kTile;
            if (tl < t_end && p0 < wave_vis)
                step(lds_bytes + (buf * TURN + half * (TURN / 2) + i) * S::FRAGS * 1024, p0,
                     (holes_now >> (half * (TURN / 2) + i)) & 1);
        }
        if (half == 1 && t0 + TURN < t_end) {
            put(buf ^ 1);
            load(t0 + 2 * TURN);
        }
        holes_now = holes_next;
        __syncthreads();
    }

    // the halves meet: waves 4-7 hand over what waves 0-3 hold in the same lanes and registers
    f32x4* const meet = (f32x4*)lds_bytes;
    float2* const meet_ml = (float2*)(lds_bytes + S::MEET);
    if (half == 1) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int j = 0; j < NT; ++j) meet[((cw * NC + i) * NT + j) * 64 + lane] = acc[i][j];
            meet_ml[(cw * NC + i) * 64 + lane] = float2{m[i], l[i]};
        }
    }
    __syncthreads();
    if (half == 1) return;
    const int64_t slot = ((int64_t)(seq * cts + ct) * c.n_kv + h) * splits + z;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const float2 other = meet_ml[(cw * NC + i) * 64 + lane];
        const float m_all = fmaxf(m[i], other.x), base = m_all == kNegInf ? 0.0f : m_all;
        const float r0 = __builtin_amdgcn_exp2f(m[i] - base), r1 = __builtin_amdgcn_exp2f(other.x - base);
        const float ls = sum_over_g((l[i] != l[i] ? l[i] : l[i] * r0) + (other.y != other.y ? other.y : other.y * r1));
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = acc[i][j] * r0 + meet[((cw * NC + i) * NT + j) * 64 + lane] * r1;
        const int cn = (cw * NC + i) * 16 + n, col = c0 + cn;
        if (col >= n_cols) continue;
        if (n_split == 1) {
            const int row = col / a.G, head = h * a.G + (col - row * a.G);
            float* o = out + ((int64_t)(w.s.r0 + row) * a.n_head + head) * HD + 4 * g;
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
#pragma unroll
            for (int j = 0; j < NT; ++j) *(f32x4*)(o + 16 * j) = ls != ls ? f32x4{ls, ls, ls, ls} : acc[i][j] * inv;
        } else {
            float* o = parts.o + (slot * S::COLS + cn) * HD + 4 * g;
#pragma unroll
            for (int j = 0; j < NT; ++j) *(f32x4*)(o + 16 * j) = acc[i][j];
            if (g == 0) {
                parts.ml[(slot * S::COLS + cn) * 2] = m_all;
                parts.ml[(slot * S::COLS + cn) * 2 + 1] = ls;
            }
        }
    }
}

// The splits of a column joined by a group of HD / 4 lanes, four elements each: those z = first, first +
// step, ... below n. A split that saw nothing has a maximum of -inf and adds exp2(-inf) = 0; one whose
// scores were all NaN has a NaN sum, which no factor takes away.
struct Joined {
    float m, l;
    f32x4 o;
    __device__ __forceinline__ void add(float m_add, float l_add, const f32x4& o_add, float base) {
        const float r = __builtin_amdgcn_exp2f(m_add - base);
        l += l_add != l_add ? l_add : l_add * r;
        o += o_add * r;
    }
    // (a NaN sum with nothing else seen: the outputs are it)
    __device__ __forceinline__ f32x4 result() const {
        return l != l ? f32x4{l, l, l, l} : o * (l == 0.0f ? 0.0f : 1.0f / l);
    }
};
template <int HD>
__device__ __forceinline__ Joined join_splits(const Parts& parts, int64_t slot, int cols, int cn, int d4, int first,
                                              int step, int n) {
    const float* ml = parts.ml + (slot * cols + cn) * 2;
    const float* po = parts.o + (slot * cols + cn) * HD + 4 * d4;
    Joined j = {kNegInf, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    for (int z = first; z < n; z += step) j.m = fmaxf(j.m, ml[(int64_t)z * cols * 2]);
    const float base = j.m == kNegInf ? 0.0f : j.m;
#pragma unroll 4
    for (int z = first; z < n; z += step) {
        const int64_t at = (int64_t)z * cols;
        j.add(ml[at * 2], ml[at * 2 + 1], *(const f32x4*)(po + at * HD), base);
    }
    return j;
}

// Up to kFewSplits splits (many rows, or streamed shares): a workgroup has a unit's GROUPS columns, one
// each. More: a workgroup per column, whose groups take every GROUPS-th split, so the loads of a long
// list are in flight together, and meet in LDS.
constexpr int kFewSplits = 4;  // 8 sequences of 96 columns (HD 64): 3 66.6 us, 4 49.2, 6 49.8
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4View c, AttnArgs a, int splits, Parts parts,
                                                  float* __restrict__ out) {
    constexpr int LANES = HD / 4, GROUPS = 256 / LANES;
    __shared__ f32x4 so[GROUPS][LANES];
    __shared__ float sm[GROUPS], sl[GROUPS];
    const int d4 = threadIdx.x % LANES, grp = threadIdx.x / LANES;
    const auto store = [&](int unit, int r0, int rows, int cn, const f32x4& o) {
        const int cc = unit / c.n_kv * a.cols + cn, rr = cc / a.G;
        const int hh = unit % c.n_kv * a.G + (cc - rr * a.G);
        if (rr < rows) *(f32x4*)(out + ((int64_t)(r0 + rr) * a.n_head + hh) * HD + 4 * d4) = o;
    };
    const int per_seq = c.n_kv * ((a.max_rows * a.G + a.cols - 1) / a.cols);
    if (splits <= kFewSplits) {
        const int per_unit = (a.cols + GROUPS - 1) / GROUPS, uu = (int)blockIdx.x / per_unit;
        const int cn = ((int)blockIdx.x - uu * per_unit) * GROUPS + grp;
        UnitMap u;
        if (splits == 0) {
            if (uu >= *parts.n_units) return;
            u = parts.map[uu];
        } else {
            const int seq = uu / per_seq;
            const SeqWork w = seq_work(c, a, seq);
            u.unit = uu - seq * per_seq;
            if (u.unit >= w.units) return;
            u.n_split = min(splits, (w.tiles + kMinShare - 1) / kMinShare);
            u.slot = (int64_t)uu * splits;
            u.r0 = w.s.r0;
            u.rows = w.rows;
        }
        if (u.n_split == 1 || cn >= a.cols || u.unit / c.n_kv * a.cols + cn >= u.rows * a.G) return;
        store(u.unit, u.r0, u.rows, cn, join_splits<HD>(parts, u.slot, a.cols, cn, d4, 0, 1, u.n_split).result());
        return;
    }
    const int uu = (int)blockIdx.x / a.cols, cn = (int)blockIdx.x - uu * a.cols;
    const int seq = uu / per_seq;
    const SeqWork w = seq_work(c, a, seq);
    const int unit = uu - seq * per_seq, n_split = min(splits, (w.tiles + kMinShare - 1) / kMinShare);
    if (unit >= w.units || n_split == 1 || unit / c.n_kv * a.cols + cn >= w.rows * a.G) return;
    const Joined mine = join_splits<HD>(parts, (int64_t)uu * splits, a.cols, cn, d4, grp, GROUPS, n_split);
    so[grp][d4] = mine.o;
    if (d4 == 0) {
        sm[grp] = mine.m;
        sl[grp] = mine.l;
    }
    __syncthreads();
    if (grp > 0) return;
    Joined all = {sm[0], 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) all.m = fmaxf(all.m, sm[i]);
    const float base = all.m == kNegInf ? 0.0f : all.m;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) all.add(sm[i], sl[i], so[i][d4], base);
    store(unit, w.s.r0, w.rows, cn, all.result());
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

// x / d to the nearest integer, ties to even, exactly: the rounded product with 1 / d is checked against
// the remainder, which an FMA gives without error (x and d * t agree to within d), and is at most one
// off, or a tie. (x and d finite, d not 0.)
__device__ __forceinline__ uint32_t code_of(float x, float d, float inv, float half) {
    float t = __builtin_rintf(x * inv);
    const float rem = __builtin_fmaf(-t, d, x);
    if (fabsf(rem) >= half && fabsf(t) < 16.0f) {  // (rare; past 16 the code is 0 or 15 anyway)
        const bool odd = __builtin_fmaf(-2.0f, __builtin_floorf(0.5f * t), t) != 0.0f;
        if (fabsf(rem) > half || odd) t += (rem < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f;
    }
    return (uint32_t)((int)__builtin_amdgcn_fmed3f(t, -8.0f, 7.0f) + 8);
}

// What bounds it: the quantization's VALU work beside the rows' read; 9534 rows of 8 heads of 128 21.5 us
// (78 MB of rows, 4.1 TB/s with the pages); 64 tokens 7.0: two dependent loads (length, page) before the
// first store. With the rotation its sines bind it, which every head's workgroup forms again: 12297 rows 25.6 us
// without, 50 with rotated keys, 154 with 32 query heads too (whose read and write alone are 57 at the one-launch
// read's rate); 64 tokens 7.1, 8.1, 8.3.
// grid (segments at most, KV heads [+ query head groups when q is rotated]). A workgroup reads the
// segment's rows of its head once and quantizes them, eight threads to a position; a dword of keys is
// eight elements of one position, a dword of values one element of eight positions, which meet in LDS.
// theta_base > 0: keys turn by the NEOX rotation of k_rope_neox at their positions first, and the
// workgroups past the KV heads turn the query rows in place.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_store(Kv4View c, int layer, const float* __restrict__ k,
                                                   const float* __restrict__ v, float* __restrict__ q, int n_head,
                                                   float theta_base, const int32_t* __restrict__ slots,
                                                   const int32_t* __restrict__ q_start, int n_seqs, int n_rows) {
    constexpr int HALF = HD / 2, PER = HD / 8, NB = HD / 32;
    __shared__ float cs[kTile][HALF], sn[kTile][HALF], power[HALF];
    __shared__ uint8_t codes[kTile][HD + 4];  // of the values
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
    const bool none = (unsigned)page >= (unsigned)c.n_pages;
    uint8_t* tile = c.pages + ((int64_t)layer * c.n_pages + (none ? 0 : page)) * c.page_bytes +
                    (((int64_t)h << sub) + (sg.tile & ((1 << sub) - 1))) * (36 * HD);
    // thread: position tid / 8, elements (tid % 8) * PER .. of both rows
    const int p = tid >> 3, d0 = (tid & 7) * PER;
    const bool on = p >= sg.a && p < sg.b;
    const int64_t src = ((int64_t)(sg.row + p - sg.a) * c.n_kv + h) * HD;
    // all that is read is on its way before the page id (and with it the tile) is known: both rows,
    // and then the value dwords of which only some positions change
    float both[2][PER];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
        for (int i = 0; i < PER; ++i) both[kv][i] = 0.0f;
        if (on) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) *(f32x4*)(both[kv] + i) = *(const f32x4*)((kv ? v : k) + src + d0 + i);
        }
    }
    if (none) return;  // no page: the rows have no place
    const bool whole = sg.a == 0 && sg.b == kTile;
    uint32_t old[4 * HD / 256];
#pragma unroll
    for (int i = 0; i < 4 * HD / 256; ++i)
        old[i] = whole ? 0u : ((const uint32_t*)(tile + 16 * HD))[i * 256 + tid];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        float (&x)[PER] = both[kv];
        if (on) {
            const float* base = (kv ? v : k) + src;
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
    }
    // a row that is not finite: known to the position's eight threads
    bool finite = true;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        finite &= fabsf(both[0][i]) < __builtin_huge_valf() && fabsf(both[1][i]) < __builtin_huge_valf();
    int bad = finite ? 0 : 1;
    bad |= dpp_i32<DPP_QUAD_SWAP1>(bad);
    bad |= dpp_i32<DPP_QUAD_SWAP2>(bad);
    bad |= dpp_i32<DPP_ROW_HALF_MIRROR>(bad);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        // a block's 32 elements lie in 32 / PER threads (the whole wave takes part)
        float (&x)[PER] = both[kv];
        float mx = x[0], mn = x[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) {
            mx = fmaxf(mx, x[i]);
            mn = fminf(mn, x[i]);
        }
        if constexpr (PER <= 16) {
            mx = fmaxf(mx, dpp_f32<DPP_QUAD_SWAP1>(mx));
            mn = fminf(mn, dpp_f32<DPP_QUAD_SWAP1>(mn));
        }
        if constexpr (PER <= 8) {
            mx = fmaxf(mx, dpp_f32<DPP_QUAD_SWAP2>(mx));
            mn = fminf(mn, dpp_f32<DPP_QUAD_SWAP2>(mn));
        }
        if (!on) continue;
        _Float16 dh = scale_of(mx, mn);
        const float d = (float)dh;
        const bool plain = d != 0.0f && !bad;
        const float inv = plain ? 1.0f / d : 0.0f, half = plain ? 0.5f * fabsf(d) : 1.0f;
        // eight elements are a key dword of the tile, which belongs to the position alone
        constexpr int W = NB < 4 ? NB : 4, C = NB / W;
#pragma unroll
        for (int j = 0; j < PER; j += 8) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t code = plain ? code_of(x[j + i], d, inv, half) : 8u;
                if (kv) codes[p][d0 + j + i] = (uint8_t)code;
                w |= code << (4 * (i / 2 + 4 * (i % 2)));
            }
            const int g = (d0 + j) / (HD / 4), f = (d0 + j) % (HD / 4) / 8;
            if (kv == 0) ((uint32_t*)tile)[(((p / 16 * C + f / W) * 4 + g) * 16 + p % 16) * W + f % W] = w;
        }
        if (d0 % 32 == 0) {
            if (bad) dh = kv ? (_Float16)0.0f : (_Float16)__builtin_nanf("");
            const int b = d0 / 32;
            const int place = kv ? (b * 4 + p % 16 / 4) * 8 + p / 16 * 4 + p % 4 : (b * 16 + p % 16) * 2 + p / 16;
            ((_Float16*)(tile + (kv ? 34 : 32) * HD))[place] = dh;
        }
    }
    __syncthreads();

    // value dwords, of which only the segment's positions change
#pragma unroll
    for (int turn = 0; turn < 4 * HD / 256; ++turn) {
        const int i = turn * 256 + tid;
        const int w = i % 4, nn = i / 4 % 16, g = i / 64 % 4, cc = i / 256;
        const int dim = 16 * (4 * cc + w) + nn;
        uint32_t x = 0, mask = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pos = 16 * (j / 4) + 4 * g + j % 4, sh = 4 * (j / 2 + 4 * (j % 2));
            if (pos >= sg.a && pos < sg.b) {
                x |= (uint32_t)codes[pos][dim] << sh;
                mask |= 15u << sh;
            }
        }
        if (!mask) continue;
        ((uint32_t*)(tile + 16 * HD))[i] = (old[turn] & ~mask) | x;
    }
}

// The rows of the batch read back as fp32, d * (c - 8); rows without a place are 0. Bound by the writes:
// 9534 rows of 8 heads of 128 20.7 us (4.3 TB/s), 64 tokens 5.1.
// grid (segments at most + sequences, KV heads): the workgroups past the segments write the rows of
// sequences with more rows than positions that stand before the first position (0).
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_load(Kv4View c, int layer, const int32_t* __restrict__ slots,
                                                  const int32_t* __restrict__ q_start, int n_seqs, int n_rows,
                                                  int segments, float* __restrict__ k, float* __restrict__ v) {
    constexpr int NB = HD / 32;
    if ((int)blockIdx.x >= segments) {
        const Kv4Seq s = kv4_seq(c, slots, q_start, (int)blockIdx.x - segments, n_rows);
        for (int64_t i = threadIdx.x; i < (int64_t)(s.rows - s.len) * HD; i += 256) {
            const int64_t at = ((s.r0 + i / HD) * c.n_kv + blockIdx.y) * HD + i % HD;
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

#define KV4_HD(hd, ...)                                           \
    switch (hd) {                                                 \
        case 64: { constexpr int HD = 64; __VA_ARGS__; } break;   \
        case 128: { constexpr int HD = 128; __VA_ARGS__; } break; \
        default: { constexpr int HD = 256; __VA_ARGS__; } break;  \
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

// The kernel of one column tile reads the cache once per 16 columns and dequantizes it as often, which
// the many columns of k_kv4_many_rows share; but those fill the chip with few of them. So the former
// takes up to kFewCols columns, and on, where contexts are short, up to kFewColsShort (heads of 64: at any
// length) and what it has workgroups at once for. us, one tile / many rows, 8 KV heads of 4 query heads each:
//   1 sequence of 4000, 64 rows: heads of 64 16.3 / 27.8, 128 20.9 / 29.1, 256 31.6 / 36.8
//   1 of 128, 128 rows: 6.0 / 15.0, 7.5 / 14.7, 10.9 / 16.1; 128 rows of 8000: 48 / 46, 69 / 58, 105 / 97
//   8 of 2000-4000, 24 rows: 35 / 49, 47 / 48, 75 / 91; 8 of 2000-4000, 64 rows: 58 / 57, 88 / 78, 155 / 156
//   16 of 8000, 17 rows: 68 / 153, 103 / 137, 198 / 363; 16 of 8000, 32 rows: 111 / 155, 169 / 142, 343 / 378
//   4 of 12000, 32 rows: 64 / 78, 93 / 71, 165 / 137
// (Between 97 and 128 columns of long contexts one rule serves 4 and 16 sequences: the latter, with heads of
// 256, get the slower form, 378 instead of 343.)
constexpr int kFewCols = 96, kFewColsShort = 128;

Kv4AttnPlan kv4_attention_plan(const Kv4View& c, int n_seqs, int max_rows, int max_len, int n_head) {
    Kv4AttnPlan p;
    const int64_t cols = (int64_t)max_rows * (n_head / c.n_kv);
    const int64_t tiles = std::max(1, (max_len + kTile - 1) / kTile), shares = (tiles + kMinShare - 1) / kMinShare;
    p.cols = cols <= 8 ? 8 : 16;
    p.units = (int64_t)n_seqs * c.n_kv * ((cols + p.cols - 1) / p.cols);
    const bool short_ = max_len <= kDirectLen;
    p.many_rows = cols > kFewCols && (cols > kFewColsShort || (c.hd > 64 && !short_)) && (p.units > kCus || !short_);
    if (p.many_rows) {
        KV4_HD(c.hd, p.cols = ManyRows<HD>::COLS);
        p.units = (int64_t)n_seqs * c.n_kv * ((cols + p.cols - 1) / p.cols);
        p.splits = (int)std::max<int64_t>(1, std::min(shares, kCus / p.units));
        p.grid = p.units * p.splits;
        return p;
    }
    const bool direct = p.units <= kDirectUnits || short_;
    p.splits = direct ? (int)std::max<int64_t>(1, std::min<int64_t>(shares, kGrid / p.units)) : 0;
    KV4_HD(c.hd, p.grid = direct ? p.units * p.splits : kCus * AttnLds<HD>::WAVES);
    return p;
}

// Workgroups of the join: per unit its columns in groups, or one a column (k_kv4_join).
static int64_t join_grid(const Kv4AttnPlan& p, int hd) {
    const int groups = 256 / (hd / 4);
    return p.splits == 1 ? 0 : p.units * (p.splits <= kFewSplits ? (p.cols + groups - 1) / groups : p.cols);
}
// A launch's threads are counted in 32 bits.
bool kv4_attention_fits(const Kv4AttnPlan& p, int hd) {
    return p.units <= INT32_MAX && p.grid <= UINT32_MAX / (p.many_rows ? 512 : 256) && join_grid(p, hd) <= UINT32_MAX / 256;
}

static size_t kv4_attention_slots(const Kv4AttnPlan& p) {
    return (size_t)(p.splits > 0 ? p.grid : p.units + p.grid);
}
size_t kv4_attention_ws_bytes(const Kv4AttnPlan& p, int hd) {
    if (p.splits == 1) return 0;
    const size_t part = kv4_attention_slots(p) * p.cols * (hd + 2) * sizeof(float);
    return p.splits > 0 ? part : part + p.units * sizeof(UnitMap) + sizeof(int64_t);
}

template <int HD, int PARTS>
static hipError_t launch_attention(const Kv4View& c, const Kv4AttnPlan& p, int layer, const float* q, const AttnArgs& a,
                                   const Parts& parts, float* out, hipStream_t stream) {
    static LdsLimit limit;
    const hipError_t e = limit.raise((const void*)k_kv4_attention<HD, PARTS>, sizeof(AttnLds<HD>));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_kv4_attention<HD, PARTS>), dim3((unsigned)p.grid), dim3(256), sizeof(AttnLds<HD>), stream, c,
                       layer, q, a, p.splits, a.max_rows * a.G <= p.cols, parts, out);
    return hipGetLastError();
}

template <int HD>
static hipError_t launch_many_rows(const Kv4View& c, const Kv4AttnPlan& p, int layer, const float* q, const AttnArgs& a,
                                   const Parts& parts, float* out, hipStream_t stream) {
    static LdsLimit limit;
    const hipError_t e = limit.raise((const void*)k_kv4_many_rows<HD>, ManyRows<HD>::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_kv4_many_rows<HD>), dim3((unsigned)p.grid), dim3(512), ManyRows<HD>::LDS, stream, c, layer, q,
                       a, p.splits, parts, out);
    return hipGetLastError();
}

hipError_t launch_kv4_attention(const Kv4View& c, const Kv4AttnPlan& p, int layer, const float* q,
                                const int32_t* slots, const int32_t* q_start, int n_seqs, int n_rows,
                                int max_rows, int n_head, float* out, void* ws, hipStream_t stream) {
    const AttnArgs a = {slots, q_start, n_seqs, n_rows, max_rows, n_head, n_head / c.n_kv, p.cols};
    Parts parts;
    parts.o = (float*)ws;
    parts.ml = parts.o + kv4_attention_slots(p) * p.cols * c.hd;
    parts.map = (UnitMap*)(parts.ml + kv4_attention_slots(p) * p.cols * 2);
    parts.n_units = (int64_t*)(parts.map + p.units);
    hipError_t e = hipSuccess;
    KV4_HD(c.hd, {
        e = p.many_rows ? launch_many_rows<HD>(c, p, layer, q, a, parts, out, stream)
            : p.cols == 16 ? launch_attention<HD, 1>(c, p, layer, q, a, parts, out, stream)
                           : launch_attention<HD, 2>(c, p, layer, q, a, parts, out, stream);
    });
    if (e != hipSuccess || p.splits == 1) return e;
    KV4_HD(c.hd, {
        hipLaunchKernelGGL((k_kv4_join<HD>), dim3((unsigned)join_grid(p, HD)), dim3(256), 0, stream, c, a, p.splits, parts,
                           out);
    });
    return hipGetLastError();
}

}  // namespace cllm_hip
