// k_experts.hip -- products of rows with the matrix of the row's expert, over GGUF blocks (gfx950).
//
// y[e] = W_x . q(x_r) of every entry e = (row r, expert x): the reference's vec_dot terms
// (src/core/quant.cpp:549-687, 706-724) on the Q8_0 blocks of x_r (420-452), with the entries
// grouped by expert on the device; two matrices give silu(gate) * up (src/core/engine.cpp:509-512).
//
// Arithmetic. A Q8_0 element is dx * c. k_expert_act writes it, times a power of two of its row, as
// fp16 hi + lo (22 bits; the Q8_0 product has 24 + 8), the token operand of the fp16 MFMAs; the weight operand holds the blocks'
// integers (times the 6-bit sub-scales of Q4_K / Q5_K: at most 1953, exact in fp16; Q6_K's
// scale * (q - 32) as its fp16 rounding and the exact rest, whose product with lo, 2^-22 of the whole, is left
// out). As dx is inside the operand, nothing is done per block of 32: a super-block's 256 products add up in the MFMA's fp32 accumulators and meet
// the weight row's d once, which with the weights on the column side is one scalar of the lane.
// Blocks of 32 (Q4_0, Q5_0, Q8_0) meet their d once a block. The K-quants' minimum term is one
// more MFMA a super-block: the 8 minima against dx * (sum of the block's codes) in three fp16 parts.
// The order of a super-block's elements in the operands is free, so each lane takes contiguous
// weight bytes and the activations are written in the order that follows.
//
// One power of two for a row holds to those 22 bits only blocks whose loudness (largest element) is within a
// range of 2^kSpread: below it lo is a subnormal and then nothing. A row that spreads further has its range where most of
// its blocks are; the others, often one or two that are far louder, are zeros in the operand and stand beside
// it as their exact codes and dx. far_sums forms their products, a block at a time, for all entries of a tile that
// have any. So no value that fp32 holds is lost, and a tile pays for the blocks apart that it has.
//
// (The weight-row GEMM applies dx per block on the VALU, one FMA per output and block, with half the
// MFMAs; here the MFMAs are doubled and the VALU is left to unpack.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "device_utils.h"
#include "experts.h"
#include "ggml_blocks.h"
#include "launch.h"
#include "mfma_common.h"

namespace cllm_hip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- the activation operand -----------------------------------------------------------------
// Row r: chunks of 256 elements, 1024 bytes of 16-byte fragments (8 fp16: step s, lane group g, hi or lo):
//   K-quants          [g / 2][s 8][hi, lo][g % 2], so that half a super-block is 512 bytes
//   blocks of 32      [s 8][hi, lo][g 4]
// then (K-quants with minima) [row][chunk][3 parts and zeros][8 blocks] fp16, 64 bytes a
// chunk; then the rows' exponents; then, written for rows with blocks apart only, [row] a bit a block (whether it is
// apart), dx and the sum of the codes of each block (fp32), its 32 codes as fp16 in their own order (zeros of
// blocks that are not apart). Fragment (s, g) holds elements
//   Q4_K, Q5_K  64 g + 8 s + e                    (lane group g: the 32 quant bytes of blocks 2g, 2g + 1)
//   Q6_K        128 (g / 2) + 32 (s / 2) + 16 (g % 2) + 8 (s % 2) + e
//   Q8_0        32 s + 8 g + e
//   Q4_0, Q5_0  32 s + 4 g + e (e < 4), 32 s + 16 + 4 g + e - 4 (e >= 4)
// with e = 0, 2, 1, 3 in each four where the low and high 16 bits of a dword are unpacked together.
constexpr int kExpNaN = INT32_MIN;  // exponent of a row with an infinity or a NaN: its results are NaN
constexpr int kExpFar = 1 << 20;    // added to the exponent of a row that has blocks apart
constexpr int kTop = 14;            // rows are scaled to magnitudes below 2^(kTop + 1) (-128 codes of subnormals: 1.01 of it)
constexpr int kMinShift = 5;        // minimum operand: 2^-5 of the scale (a block's codes add up to 4064)
// A block within 2^kSpread of the loudest has an element of 2^5 and more, so a dx of 2^-2 and more, and hi + lo of any of
// its values c dx is within 2^-23 of it (lo's least step is 2^-24, half of it 2^-23 of 2^-2).
constexpr int kSpread = kTop - 5;
constexpr int kLoudness = 288;  // exponents of fp32 values, from -149 on

enum Order { kMin64, kQ6, kByte, kNibble };
__host__ __device__ constexpr Order order_of(uint32_t t) {
    return t == T_Q4_K || t == T_Q5_K ? kMin64 : t == T_Q6_K ? kQ6 : t == T_Q8_0 ? kByte : kNibble;
}
__host__ __device__ constexpr bool has_min(uint32_t t) { return t == T_Q4_K || t == T_Q5_K; }
__host__ __device__ constexpr bool is_kq(uint32_t t) { return has_min(t) || t == T_Q6_K; }

struct Act {
    const uint8_t* frags;
    const uint8_t* mins;
    const int32_t* exps;
    const uint8_t* far;
    uint32_t row;  // bytes of a row's fragments
    int chunks;
    // of a row's blocks apart: the places of dx and of the codes, and all bytes
    __host__ __device__ uint32_t far_scales() const { return ((uint32_t)chunks + 15u) & ~15u; }
    __host__ __device__ uint32_t far_codes() const { return far_scales() + (uint32_t)chunks * 64u; }
    __host__ __device__ size_t far_row() const { return (size_t)far_codes() + (size_t)chunks * 512u; }
};
int chunks_of(int k) { return (k + 255) / 256; }
Act act_of(void* ws, uint32_t type, int k, int rows) {
    Act a;
    a.chunks = chunks_of(k);
    a.row = (uint32_t)a.chunks * 1024u;
    uint8_t* p = (uint8_t*)ws;
    a.frags = p;
    p += (size_t)rows * a.row;
    a.mins = p;
    if (has_min(type)) p += up256((size_t)rows * a.chunks * 64);
    a.exps = (const int32_t*)p;
    p += up256((size_t)rows * 4);
    a.far = p;
    return a;
}

// One workgroup a row: how loud its blocks are, then each quad of lanes one Q8_0 block (eight
// elements a lane, quantize_row_q8_0 bit for bit) as scaled fp16 parts. What a thread reads first it keeps, the rest
// is read again from the caches. 1024 threads for few rows, where one row's latency is what counts. A row is
// read once and 4 bytes an element written: the copy rate bounds it (4096 rows of 14336: 470 MB, 104 us, 4.5
// TB/s); a single row of 14336 takes 5.0 us: two dependent passes over 56 KB by one CU. A row with blocks apart takes two more passes, and writes 2.3 bytes an element more.
template <Order O, int THREADS>
__global__ __launch_bounds__(THREADS) void k_expert_act(const float* __restrict__ x, int k, Act act) {
    __shared__ uint32_t tops[THREADS / 64], lows[THREADS / 64], best;
    __shared__ int loud[kLoudness];
    const int row = blockIdx.x, tid = threadIdx.x, chunks = act.chunks;
    const f32x4* __restrict__ src = (const f32x4*)(x + (size_t)row * k);
    uint8_t* mins = (uint8_t*)act.mins;
    int32_t* exps = (int32_t*)act.exps;
    // the largest of a block, (bits << 1), in a quad of lanes that has its eight elements each: orders magnitudes, and NaN
    // above infinity. (A quad has a block or none: k is a multiple of 32.)
    auto block_top = [&](const f32x4& v, const f32x4& w) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max(__float_as_uint(v[j]) << 1, __float_as_uint(w[j]) << 1));
        m = max(m, (uint32_t)dpp_i32<DPP_QUAD_SWAP1>((int)m));
        return max(m, (uint32_t)dpp_i32<DPP_QUAD_SWAP2>((int)m));
    };
    auto loudness = [&](uint32_t m) {
        int ex;
        (void)frexpf(__builtin_bit_cast(float, m >> 1), &ex);  // magnitude in [2^(ex - 1), 2^ex)
        return ex;
    };
    uint32_t top = 0, low = UINT32_MAX;  // the loudest block, the quietest (less 1) but for blocks of zeros
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 lo0 = zero, hi0 = zero;  // the first eight of this thread, read once
    if (8 * tid < k) lo0 = src[2 * tid], hi0 = src[2 * tid + 1];
    for (int i = tid; i < k / 8; i += THREADS) {
        const uint32_t m = i == tid ? block_top(lo0, hi0) : block_top(src[2 * i], src[2 * i + 1]);
        top = max(top, m);
        low = min(low, m - 1);
    }
    for (int d = 32; d >= 4; d >>= 1) {
        top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
        low = min(low, (uint32_t)__shfl_xor((int)low, d, 64));
    }
    if ((tid & 63) == 0) tops[tid >> 6] = top, lows[tid >> 6] = low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) top = max(top, tops[i]), low = min(low, lows[i]);
    const bool finite = top < 0xFF000000u;
    bool far = false;
    int ex = kTop + 1;  // the range's top: blocks of loudness ex - kSpread to ex
    if (finite && top != 0) {
        ex = loudness(top);
        far = ex - loudness(low + 1) > kSpread;
    }
    if (far) {  // the range with the most blocks; of equal ones the loudest
        for (int i = tid; i < kLoudness; i += THREADS) loud[i] = 0;
        if (tid == 0) best = 0;
        __syncthreads();
        for (int i = tid; i < k / 8; i += THREADS) {
            const uint32_t m = block_top(src[2 * i], src[2 * i + 1]);
            if ((i & 3) == 0 && m != 0) atomicAdd(&loud[loudness(m) + 149], 1);
        }
        __syncthreads();
        for (int i = tid; i < kLoudness; i += THREADS) {
            int n = 0;
            for (int j = max(0, i - kSpread); j <= i; ++j) n += loud[j];
            atomicMax(&best, ((uint32_t)min(n, 65535) << 16) | (uint32_t)i);
        }
        __syncthreads();
        ex = (int)(best & 0xFFFFu) - 149;
    }
    const int e = kTop + 1 - ex;
    if (tid == 0) exps[row] = !finite ? kExpNaN : far ? e + kExpFar : e;
    uint8_t* out = (uint8_t*)act.frags + (size_t)row * act.row;
    uint8_t* apart = (uint8_t*)act.far + (size_t)row * act.far_row();
    // lanes past the row's end write zeros up to the last chunk's end (whole quads: k is a multiple of 32)
    for (int i = tid; i < chunks * 32; i += THREADS) {
        const int c = i >> 5, b = (i >> 2) & 7, p = i & 3;  // chunk, block, eight elements of it
        f32x4 lo = lo0, hi = hi0;
        if (i != tid && 8 * i < k) lo = src[2 * i], hi = src[2 * i + 1];
        if (!finite || 8 * i >= k) lo = hi = zero;
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        uint32_t q[2];
        float d;
        int s8;
        q8_quant_quad(v, q, d, s8);
        if (far) {
            const uint32_t m = block_top(lo, hi);
            const int l = loudness(m);
            const bool out_of = m != 0 && (l > ex || l < ex - kSpread);
            const int s16 = s8 + dpp_i32<DPP_QUAD_SWAP1>(s8);
            const int sum = s16 + dpp_i32<DPP_QUAD_SWAP2>(s16);
            const wu4 none = {0, 0, 0, 0};
            *(wu4*)(apart + act.far_codes() + (size_t)(i >> 2) * 64 + 16 * p) = out_of ? int8x8_to_h8(q[0], q[1]) : none;
            if (p == 0) *(float2*)(apart + act.far_scales() + (size_t)(i >> 2) * 8) = out_of ? make_float2(d, (float)sum) : make_float2(0.0f, 0.0f);
            const uint32_t bits = (uint32_t)(__ballot(out_of) >> (tid & 32));  // four alike a block
            if ((i & 31) == 0) {
                uint32_t byte = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) byte |= ((bits >> (4 * j)) & 1u) << j;
                apart[c] = (uint8_t)byte;
            }
            if (out_of) d = 0.0f;
        }
        const float dx = ldexpf(d, e);
        _Float16 h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (rounded to fp32 first, for both parts alike: else the compiler forms hi from the product
            // in one rounding and lo from the rounded product, and where the two hi differ lo is a step off)
            const float t = pinned(dx * (float)(int8_t)(q[j >> 2] >> (8 * (j & 3))));
            h[j] = (_Float16)t;
            l[j] = (_Float16)(t - (float)h[j]);
        }
        uint8_t* ch = out + (size_t)c * 1024;
        if constexpr (O == kNibble) {
            // elements 8p .. of the block: the first (p < 2) or second four of fragments g and g + 1
            const int g = 2 * (p & 1);
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint8_t* at = ch + b * 128 + (g + j) * 16 + 8 * (p >> 1);
                *(h4*)at = h4{h[4 * j], h[4 * j + 2], h[4 * j + 1], h[4 * j + 3]};
                *(h4*)(at + 64) = h4{l[4 * j], l[4 * j + 2], l[4 * j + 1], l[4 * j + 3]};
            }
        } else {
            int s, g;
            if constexpr (O == kMin64) {
                s = 4 * (b & 1) + p, g = b >> 1;
            } else if constexpr (O == kQ6) {
                s = 2 * (b & 3) + (p & 1), g = 2 * (b >> 2) + (p >> 1);
            } else {
                s = b, g = p;
            }
            constexpr int LO = O == kByte ? 64 : 32;
            uint8_t* at = ch + (O == kByte ? s * 128 + g * 16 : (g >> 1) * 512 + s * 64 + (g & 1) * 16);
            if constexpr (O == kMin64) {
                *(wh8*)at = wh8{h[0], h[2], h[1], h[3], h[4], h[6], h[5], h[7]};
                *(wh8*)(at + LO) = wh8{l[0], l[2], l[1], l[3], l[4], l[6], l[5], l[7]};
            } else {
                *(wh8*)at = wh8{h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[7]};
                *(wh8*)(at + LO) = wh8{l[0], l[1], l[2], l[3], l[4], l[5], l[6], l[7]};
            }
        }
        if constexpr (O == kMin64) {
            const int s16 = s8 + dpp_i32<DPP_QUAD_SWAP1>(s8);
            const int sum = s16 + dpp_i32<DPP_QUAD_SWAP2>(s16);
            float t = pinned(ldexpf(d, e - kMinShift) * (float)sum);
            _Float16* m = (_Float16*)(mins + ((size_t)row * chunks + c) * 64) + b;
            if (p == 0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    const _Float16 part = (_Float16)t;
                    m[8 * j] = part;
                    t -= (float)part;
                }
                m[24] = (_Float16)0.0f;
            }
        }
    }
}

// ---- the weight operand ----------------------------------------------------------------------
// One weight row's share of a lane group g (of 4) of a 256-element chunk: its bytes in registers,
// then fragments of 8 fp16 integers.
__device__ __forceinline__ wh2 as_h2(uint32_t v) { return __builtin_bit_cast(wh2, v); }
__device__ __forceinline__ wh2 both(float v) { return wh2{(_Float16)v, (_Float16)v}; }
__device__ __forceinline__ wh8 cat(wh2 a, wh2 b, wh2 c, wh2 d) {
    return wh8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
template <int BYTES, class V>
__device__ __forceinline__ V ld_any(const uint8_t* p) {  // any alignment: one load instruction
    V v;
    __builtin_memcpy(&v, p, BYTES);
    return v;
}

// 6-bit scales and minima of the super-block's eight blocks, a byte each (get_scale_min_k4,
// quant.cpp:72-80): minima as fp16
__device__ __forceinline__ wh8 k4_minima(const u32x4& hdr) {
    const uint32_t a = hdr.z & 0x3F3F3F3Fu;
    const uint32_t b = ((hdr.w >> 4) & 0x0F0F0F0Fu) | ((hdr.z >> 2) & 0x30303030u);
    const wh2 off = both(-1024.0f);
    return cat(magic_pair(a, 0) + off, magic_pair(a, 1) + off, magic_pair(b, 0) + off, magic_pair(b, 1) + off);
}
// the scales of blocks 2g and 2g + 1
__device__ __forceinline__ void k4_scales2(const u32x4& hdr, int g, float& s0, float& s1) {
    const int sh = 16 * (g & 1);
    const uint32_t lo = (hdr.y >> sh) & 0x3F3Fu;
    const uint32_t hi = ((hdr.w >> sh) & 0x0F0Fu) | ((hdr.y >> (sh + 2)) & 0x3030u);
    const uint32_t s = g < 2 ? lo : hi;
    s0 = (float)(s & 0xFFu);
    s1 = (float)((s >> 8) & 0xFFu);
}

// Lane group g of a super-block: its own bytes (Part) and, with minima, the row's header (16 bytes).
struct Scales2 {  // of blocks 2g and 2g + 1
    wh2 s0, c0, s1, c1;
};

template <uint32_t T>
struct Part;
template <>
struct Part<T_Q4_K> {
    static constexpr int BYTES = Q4_K_BYTES;
    u32x4 q[2];
    __device__ __forceinline__ void load(const uint8_t* p, int g) {
        q[0] = ld_u32x4(p + Q4_K_QS + 32 * g);
        q[1] = ld_u32x4(p + Q4_K_QS + 32 * g + 16);
    }
    static __device__ __forceinline__ Scales2 scale(const u32x4& hdr, int g) {
        float a, b;
        k4_scales2(hdr, g, a, b);
        return Scales2{both(a), both(-1024.0f * a), both(b * 0.0625f), both(-64.0f * b)};
    }
    __device__ __forceinline__ wh8 frag(const Scales2& c, int s, int) const {
        const uint32_t a = q[(s & 3) >> 1][2 * (s & 1)], b = q[(s & 3) >> 1][2 * (s & 1) + 1];
        const uint32_t m = s < 4 ? 0x000F000Fu : 0x00F000F0u, o = 0x64006400u;
        const wh2 k = s < 4 ? c.s0 : c.s1, z = s < 4 ? c.c0 : c.c1;
        return cat(__builtin_elementwise_fma(as_h2((a & m) | o), k, z),
                   __builtin_elementwise_fma(as_h2(((a >> 8) & m) | o), k, z),
                   __builtin_elementwise_fma(as_h2((b & m) | o), k, z),
                   __builtin_elementwise_fma(as_h2(((b >> 8) & m) | o), k, z));
    }
};

template <>
struct Part<T_Q5_K> {
    static constexpr int BYTES = Q5_K_BYTES;
    u32x4 q[2], h[2];
    __device__ __forceinline__ void load(const uint8_t* p, int g) {
        h[0] = ld_u32x4(p + Q5_K_QH);
        h[1] = ld_u32x4(p + Q5_K_QH + 16);
        q[0] = ld_u32x4(p + Q5_K_QS + 32 * g);
        q[1] = ld_u32x4(p + Q5_K_QS + 32 * g + 16);
    }
    static __device__ __forceinline__ Scales2 scale(const u32x4& hdr, int g) {
        float a, b;
        k4_scales2(hdr, g, a, b);
        return Scales2{both(a), both(-1024.0f * a), both(b), both(-1024.0f * b)};
    }
    __device__ __forceinline__ wh8 frag(const Scales2& c, int s, int g) const {
        const int hi = s >> 2;  // block 2g + hi
        const wh2 m = hi ? c.s1 : c.s0, z = hi ? c.c1 : c.c0;
        wh2 f[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t n = q[(s & 3) >> 1][2 * (s & 1) + j], b = h[(s & 3) >> 1][2 * (s & 1) + j];
            const uint32_t v = ((hi ? n >> 4 : n) & 0x0F0F0F0Fu) | (((b >> (2 * g + hi)) & 0x01010101u) << 4);
            f[2 * j] = __builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(0x64646464u, v, 0x04020400u)), m, z);
            f[2 * j + 1] = __builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(0x64646464u, v, 0x04030401u)), m, z);
        }
        return cat(f[0], f[1], f[2], f[3]);
    }
};

template <>
struct Part<T_Q6_K> {
    static constexpr int BYTES = Q6_K_BYTES;
    u32x4 l[2], h;
    u32x2 sc;
    uint32_t db;
    __device__ __forceinline__ void load(const uint8_t* p, int g) {
        const int n = g >> 1, u = g & 1;
        l[0] = ld_any<16, u32x4>(p + 64 * n + 16 * u);
        l[1] = ld_any<16, u32x4>(p + 64 * n + 32 + 16 * u);
        h = ld_any<16, u32x4>(p + Q6_K_QH + 32 * n + 16 * u);
        sc = ld_any<8, u32x2>(p + Q6_K_SC + 8 * n);
        db = ld_u16(p + Q6_K_D);
    }
    // scale * (q - 32): the fp16 rounding and the rest, exact
    __device__ __forceinline__ wh8 frag(int s, int g, wh8& rest) const {
        const int i = s >> 1;
        const wh2 m = both((float)(int8_t)(sc[i >> 1] >> (16 * (i & 1) + 8 * (g & 1))));
        const wh2 off = both(-1056.0f);
        wh2 f[4], r[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t n = l[i & 1][2 * (s & 1) + j], b = h[2 * (s & 1) + j];
            const uint32_t v = ((i < 2 ? n : n >> 4) & 0x0F0F0F0Fu) | (((b >> (2 * i)) & 0x03030303u) << 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const wh2 p = magic_pair(v, e) + off;
                f[2 * j + e] = p * m;
                r[2 * j + e] = __builtin_elementwise_fma(p, m, -f[2 * j + e]);
            }
        }
        rest = cat(r[0], r[1], r[2], r[3]);
        return cat(f[0], f[1], f[2], f[3]);
    }
    __device__ __forceinline__ float d() const { return f16_to_f32(db); }
};

// Blocks of 32: the eight elements of lane group g of one block.
__device__ __forceinline__ wh8 nibbles8(uint32_t v, float off) {
    const uint32_t o = 0x64006400u;
    const wh2 one = both(1.0f), c0 = both(-1024.0f + off), k1 = both(0.0625f), c1 = both(-64.0f + off);
    return cat(__builtin_elementwise_fma(as_h2((v & 0x000F000Fu) | o), one, c0),
               __builtin_elementwise_fma(as_h2(((v >> 8) & 0x000F000Fu) | o), one, c0),
               __builtin_elementwise_fma(as_h2((v & 0x00F000F0u) | o), k1, c1),
               __builtin_elementwise_fma(as_h2(((v >> 8) & 0x00F000F0u) | o), k1, c1));
}
// bits 4 g .. 4 g + 3 (and 16 more) of qh to bit 4 of four bytes
__device__ __forceinline__ uint32_t bits4(uint32_t x) {
    return ((((x & 0xFu) * 0x00204081u) & 0x01010101u) << 4);
}
__device__ __forceinline__ wh8 five8(uint32_t v, uint32_t qh, int g) {
    const uint32_t a = (v & 0x0F0F0F0Fu) | bits4(qh >> (4 * g));
    const uint32_t b = ((v >> 4) & 0x0F0F0F0Fu) | bits4(qh >> (16 + 4 * g));
    const wh2 c = both(-1040.0f);
    return cat(as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04020400u)) + c,
               as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04030401u)) + c,
               as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04020400u)) + c,
               as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04030401u)) + c);
}

template <uint32_t T>
struct Unit;
template <>
struct Unit<T_Q8_0> {
    static constexpr int BYTES = Q8_0_BYTES;
    u32x2 q;
    uint32_t db;
    __device__ __forceinline__ wh8 frag(int) const { return __builtin_bit_cast(wh8, int8x8_to_h8(q.x, q.y)); }
};
template <>
struct Unit<T_Q4_0> {
    static constexpr int BYTES = Q4_0_BYTES;
    uint32_t q, db;
    __device__ __forceinline__ wh8 frag(int) const { return nibbles8(q, -8.0f); }
};
template <>
struct Unit<T_Q5_0> {
    static constexpr int BYTES = Q5_0_BYTES;
    uint32_t q, h, db;
    __device__ __forceinline__ wh8 frag(int g) const { return five8(q, h, g); }
};

// Two neighbouring blocks of a row of 32-row tiles: lane half h loads block h whole, then the halves exchange
// so that each has its 16 elements (lane groups 2h and 2h + 1) of both.
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const auto v = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = v[0], b = v[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
    const auto v = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = v[0], b = v[1];
}
template <uint32_t T>
struct BlockPair {
    static constexpr int BYTES = T == T_Q8_0 ? Q8_0_BYTES : T == T_Q4_0 ? Q4_0_BYTES : Q5_0_BYTES;
    static constexpr int HALF = T == T_Q8_0 ? 4 : 2;  // dwords of half a block's quants
    static constexpr int QS = T == T_Q5_0 ? 6 : 2;
    uint32_t q[2][HALF], d[2], h5[2];  // loaded: this half's block's two halves; after exchange(): of both blocks
    __device__ __forceinline__ void load(const uint8_t* at) {
#pragma unroll
        for (int k = 0; k < HALF / 2; ++k) {
            const u32x4 v = ld_any<16, u32x4>(at + QS + 16 * k);
            uint32_t* to = HALF == 4 ? q[k] : q[0];
            to[0] = v.x, to[1] = v.y;
            if constexpr (HALF == 4)
                to[2] = v.z, to[3] = v.w;
            else
                q[1][0] = v.z, q[1][1] = v.w;
        }
        d[0] = ld_u16(at);
        if constexpr (T == T_Q5_0) h5[0] = ld_any<4, uint32_t>(at + 2);
    }
    __device__ __forceinline__ void exchange() {
#pragma unroll
        for (int k = 0; k < HALF; ++k) swap32(q[0][k], q[1][k]);
        d[1] = d[0];
        swap32(d[0], d[1]);
        if constexpr (T == T_Q5_0) {
            h5[1] = h5[0];
            swap32(h5[0], h5[1]);
        }
    }
    // lane group 2h + i of block b
    __device__ __forceinline__ wh8 frag(int b, int i, int h) const {
        if constexpr (T == T_Q8_0)
            return __builtin_bit_cast(wh8, int8x8_to_h8(q[b][2 * i], q[b][2 * i + 1]));
        else if constexpr (T == T_Q4_0)
            return nibbles8(q[b][i], -8.0f);
        else
            return five8(q[b][i], h5[b], 2 * h + i);
    }
};

template <uint32_t T>
struct Bytes {
    static constexpr uint32_t V = T == T_Q4_K ? Q4_K_BYTES : Q5_K_BYTES;
};

struct Mul {
    const uint8_t* w[2];
    const float* bias[2];
    size_t expert_bytes;
    uint32_t row_bytes;
    int n, nb;  // weight rows, 32-element blocks of a row
    Act act;
    int per_row, rows;
    Groups g;
    int n_blocks;
    float* y;
};

// What a tile's entry needs: its number (-1: none), its activation row.
__device__ __forceinline__ int entry_of(const Mul& a, const GroupTile& t, int i) {
    const int e = i < t.count ? a.g.order[t.first + i] : -1;
    return (uint32_t)e < (uint32_t)a.g.entries && e / a.per_row < a.rows ? e : -1;
}
__device__ __forceinline__ float unscaled(float v, int e) {
    return e == kExpNaN ? __builtin_nanf("") : ldexpf(v, -e);
}
// (of a row with blocks apart: done where those were added)
__device__ __forceinline__ float result(float v, int e) { return e >= kExpFar / 2 ? v : unscaled(v, e); }

// One weight row's share of lane group g of a chunk: 64 elements (16-row tiles).
template <uint32_t T>
struct WeightChunk {
    Part<T> p;
    u32x4 hdr;
    __device__ __forceinline__ void load(const uint8_t* row, int c, int, int g) {
        const uint8_t* at = row + (size_t)c * Part<T>::BYTES;
        if constexpr (has_min(T)) hdr = ld_u32x4(at);
        p.load(at, g);
    }
};
// Blocks of 32: lane group g loads blocks g and 4 + g whole, and the groups then exchange quarters (a 4 x 4
// transposition between lane groups and registers): a third of the loads of each group's own quarters.
// m[j] of lane group b becomes m[b] of lane group j
__device__ __forceinline__ void transpose4(uint32_t (&m)[4]) {
    swap32(m[0], m[2]);
    swap32(m[1], m[3]);
    swap16(m[0], m[1]);
    swap16(m[2], m[3]);
}
template <uint32_t T>
    requires(!is_kq(T))
struct WeightChunk<T> {
    static constexpr int QW = T == T_Q8_0 ? 2 : 1;  // dwords of a quarter
    static constexpr int QS = T == T_Q5_0 ? 6 : 2;  // the quants' place in a block
    u32x4 q[2][QW];
    uint32_t db[2], qh[2];
    __device__ __forceinline__ void load(const uint8_t* row, int c, int nb, int g) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint8_t* at = row + (size_t)min(8 * c + 4 * k + g, nb - 1) * Unit<T>::BYTES;
#pragma unroll
            for (int j = 0; j < QW; ++j) q[k][j] = ld_any<16, u32x4>(at + QS + 16 * j);
            db[k] = ld_u16(at);
            if constexpr (T == T_Q5_0) qh[k] = ld_any<4, uint32_t>(at + 2);
        }
    }
    // blocks 4 k .. 4 k + 3, this lane group's eight elements of each
    __device__ __forceinline__ void units(int k, Unit<T> (&u)[4]) const {
        uint32_t m[4];
        if constexpr (T == T_Q8_0) {
            // quarter j is dwords 2j and 2j + 1
            uint32_t lo[4] = {q[k][0].x, q[k][0].z, q[k][1].x, q[k][1].z};
            uint32_t hi[4] = {q[k][0].y, q[k][0].w, q[k][1].y, q[k][1].w};
            transpose4(lo);
            transpose4(hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j].q = u32x2{lo[j], hi[j]};
        } else {
            uint32_t v[4] = {q[k][0].x, q[k][0].y, q[k][0].z, q[k][0].w};
            transpose4(v);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j].q = v[j];
        }
        if constexpr (T == T_Q5_0) {
            uint32_t v[4] = {qh[k], qh[k], qh[k], qh[k]};
            transpose4(v);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j].h = v[j];
        }
        m[0] = m[1] = m[2] = m[3] = db[k];
        transpose4(m);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j].db = m[j];
    }
};
// acc += a chunk of 16 entries x the NT tiles' rows; frag(s, part): the activations' fragments
template <uint32_t T, int NT, class Frag>
__device__ __forceinline__ void chunk_product(const WeightChunk<T> (&w)[NT], int c, int nb, int g, Frag frag, wh8 am,
                                              f32x4 (&acc)[NT]) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (is_kq(T)) {
        f32x4 sum[NT];
        Scales2 sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            sum[i] = zero;
            if constexpr (has_min(T)) sc[i] = Part<T>::scale(w[i].hdr, g);
        }
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const wh8 ah = frag(s, 0), al = frag(s, 1);
            wh8 f[NT], rest[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if constexpr (T == T_Q6_K)
                    f[i] = w[i].p.frag(s, g, rest[i]);
                else
                    f[i] = w[i].p.frag(sc[i], s, g);
            }
            // (a product waits for the one before it in its accumulator: the tiles in turn)
#pragma unroll
            for (int i = 0; i < NT; ++i) sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, f[i], sum[i], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < NT; ++i) sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, f[i], sum[i], 0, 0, 0);
            if constexpr (T == T_Q6_K) {
#pragma unroll
                for (int i = 0; i < NT; ++i) sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, rest[i], sum[i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (has_min(T)) {
                const float d = f16_to_f32(w[i].hdr.x & 0xFFFFu);
                const f32x4 m = __builtin_amdgcn_mfma_f32_16x16x32_f16(am, k4_minima(w[i].hdr), zero, 0, 0, 0);
                const float dm = -(float)(1 << kMinShift) * f16_to_f32(w[i].hdr.x >> 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(d, sum[i][j], fmaf(dm, m[j], acc[i][j]));
            } else {
                const float d = w[i].p.d();
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(d, sum[i][j], acc[i][j]);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            Unit<T> u[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i) w[i].units(k, u[i]);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int s = 4 * k + b;
                const wh8 ah = frag(s, 0), al = frag(s, 1);
                const bool there = 8 * c + s < nb;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const wh8 f = u[i][b].frag(g);
                    f32x4 sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, f, zero, 0, 0, 0);
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, f, sum, 0, 0, 0);
                    const float d = there ? f16_to_f32(u[i][b].db) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(d, sum[j], acc[i][j]);
                }
            }
        }
    }
}

// ---- blocks apart -------------------------------------------------------------------------------
// Lane group g's eight elements (8 g on) of one block of 32 of a weight row: the bytes, then integers as fp16 (Q6_K:
// scale * (q - 32) as in the operand above), the block's scale and, of types with minima, its minimum.
template <uint32_t T>
struct CodeBlock {
    u32x4 hdr;  // Q4_K, Q5_K: d, dmin and the 6-bit scales; else d and, of Q6_K, the block's scale, of Q5_0 the high bits
    u32x2 q, h;
    __device__ __forceinline__ void load(const uint8_t* row, int b, int g) {
        if constexpr (is_kq(T)) {
            const uint8_t* at = row + (size_t)(b >> 3) * (T == T_Q6_K ? Q6_K_BYTES : T == T_Q4_K ? Q4_K_BYTES : Q5_K_BYTES);
            b &= 7;
            if constexpr (T == T_Q6_K) {
                const int n = b >> 2, i = b & 3;
                q = ld_any<8, u32x2>(at + 64 * n + 32 * (i & 1) + 8 * g);
                h = ld_any<8, u32x2>(at + Q6_K_QH + 32 * n + 8 * g);
                hdr.x = ld_u16(at + Q6_K_D);
                hdr.y = at[Q6_K_SC + 8 * n + 2 * i + (g >> 1)];
            } else {
                hdr = ld_u32x4(at);
                q = ld_any<8, u32x2>(at + (T == T_Q4_K ? Q4_K_QS : Q5_K_QS) + 32 * (b >> 1) + 8 * g);
                if constexpr (T == T_Q5_K) h = ld_any<8, u32x2>(at + Q5_K_QH + 8 * g);
            }
        } else {
            const uint8_t* at = row + (size_t)b * Unit<T>::BYTES;
            hdr.x = ld_u16(at);
            // (elements from 16 on are the high nibbles)
            q = ld_any<8, u32x2>(at + (T == T_Q5_0 ? 6 : 2) + 8 * (T == T_Q8_0 ? g : g & 1));
            if constexpr (T == T_Q5_0) hdr.y = ld_any<4, uint32_t>(at + 2);
        }
    }
    __device__ __forceinline__ wh8 unpack(int b, int g, wh8& rest, float& d, float& m) const {
        uint32_t v[2];
        float off = 0.0f;
        d = f16_to_f32(hdr.x & 0xFFFFu);
        if constexpr (T == T_Q8_0) {
            return __builtin_bit_cast(wh8, int8x8_to_h8(q.x, q.y));
        } else if constexpr (T == T_Q6_K) {
            const int i = b & 3;
            const wh2 sc = both((float)(int8_t)hdr.y);
            wh2 p[4], r[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = ((q[k >> 1] >> (4 * (i >> 1))) & 0x0F0F0F0Fu) | (((h[k >> 1] >> (2 * i)) & 0x03030303u) << 4);
                const wh2 c = magic_pair(u, k & 1) + both(-1056.0f);
                p[k] = c * sc;
                r[k] = __builtin_elementwise_fma(c, sc, -p[k]);
            }
            rest = cat(r[0], r[1], r[2], r[3]);
            return cat(p[0], p[1], p[2], p[3]);
        } else if constexpr (is_kq(T)) {
            int sc, mn;
            k4_scale_min(hdr.y, hdr.z, hdr.w, b & 7, sc, mn);
            d *= (float)sc;
            m = f16_to_f32(hdr.x >> 16) * (float)mn;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v[k] = (q[k] >> (4 * (b & 1))) & 0x0F0F0F0Fu;
                if constexpr (T == T_Q5_K) v[k] |= ((h[k] >> (b & 7)) & 0x01010101u) << 4;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) v[k] = (q[k] >> (4 * (g >> 1))) & 0x0F0F0F0Fu;
            off = T == T_Q5_0 ? -16.0f : -8.0f;
            if constexpr (T == T_Q5_0) {
                v[0] |= bits4(hdr.y >> (8 * g));
                v[1] |= bits4(hdr.y >> (8 * g + 4));
            }
        }
        const wh2 c = both(-1024.0f + off);
        return cat(magic_pair(v[0], 0) + c, magic_pair(v[0], 1) + c, magic_pair(v[1], 0) + c, magic_pair(v[1], 1) + c);
    }
};

// The lane, found anew: what is done for few tiles holds no register over the loop of all.
__device__ __forceinline__ int lane_again() {
    uint32_t zero;
    asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}

// The sums of the blocks apart of a tile's entries, of M entries and two tiles of M weight rows from n0 on (gate and up of the
// same rows, or 2 M rows), as a matrix instruction leaves them (M 16: lane (r, g) has entries 4g + j of row r; 32:
// 8 (j / 4) + 4h + j % 4). The products of a block's codes are whole numbers below 2^24, exact in fp32, and meet
// d and dx once; its minimum meets the sum of the codes. e: the entry of lane r, far: whether its row has blocks
// apart, rows: the tile's entries (lanes past them have them again). The blocks that any entry has apart are taken
// one after another; of KP waves each takes every KP-th. AHEAD: the next one's loads are on their way, where registers allow.
// Measured (MI355X), no row | every 64th row | all rows with one block apart, us: one row, gate and up Q4_K 4096 x 14336
// 36 | 45 | 45, down Q6_K 39 | 47 | 47; 61 rows over 128 experts, 2048 x 768 Q4_K 59 | 61 | 68; 2048 rows over 8, gate
// and up Q4_K 1944 | 1978 | 2019, down Q6_K 1796 | 1815 | 1800. (Whole rows as codes, which needs no range to be
// found: 36 | 148 | 142, 2007 | 5312 | 20269.) Each of 2048 rows with 4 apart in places of its own, so that a tile has most:
// 6.3 and 3.6 ms (without AHEAD 7.8 and 4.3); a block then takes some 1.2 us, most of it the lanes' arithmetic.
template <uint32_t T, int M, int KP, bool AHEAD, bool SWIGLU, class V>
__device__ __forceinline__ void far_sums(const Mul& a, int group, int n0, int e, bool far, int rows, int kp, int lane,
                                         V (&sum)[2]) {
    constexpr int N = M == 16 ? 4 : 16, NT = 2;  // values of a lane
    const int r = lane & (M - 1), g = lane / M;
    const int row = far ? e / a.per_row : 0;
    const size_t bytes = a.act.far_row();
    const uint8_t* own = a.act.far + (size_t)row * bytes;
    const uint32_t set = (uint32_t)(__ballot(far) & ((1ull << rows) - 1));
    const uint8_t* wp[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
        wp[i] = a.w[SWIGLU ? i : 0] + (size_t)group * a.expert_bytes + (size_t)min(n0 + (SWIGLU ? 0 : M * i) + r, a.n - 1) * a.row_bytes;
#pragma unroll
    for (int i = 0; i < NT; ++i) sum[i] = V{};
    // the blocks that any entry has apart, in order: 32 to a lane's word
    int w0 = -64, l = 0;
    uint32_t word = 0, left = 0;
    uint64_t some = 0;
    auto any = [&]() {
        while (left == 0) {
            if (some != 0) {
                l = __ffsll((unsigned long long)some) - 1;
                some &= some - 1;
                left = (uint32_t)__builtin_amdgcn_readlane((int)word, l);
                continue;
            }
            w0 += 64;
            if (4 * w0 >= a.act.chunks) return -1;
            word = 0;
            const uint32_t at = 4u * (uint32_t)min(w0 + lane, (a.act.chunks - 1) >> 2);
            for (int i = 0; i < rows; i += 4) {  // (four rows' words on their way at once; those of no entry are dropped)
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[k] = *(const uint32_t*)(a.act.far + (size_t)__builtin_amdgcn_readlane(row, i + k) * bytes + at);
#pragma unroll
                for (int k = 0; k < 4; ++k) word |= (set >> (i + k)) & 1 ? v[k] : 0u;
            }
            if (4 * (w0 + lane) >= a.act.chunks) word = 0;
            some = __ballot(word != 0);
        }
        const int b = 32 * (w0 + l) + __ffs(left) - 1;
        left &= left - 1;
        return b < a.nb ? b : -1;  // (bits past the last chunk: nothing follows)
    };
    int count = 0;
    auto next = [&]() {
        int b = any();
        while (KP > 1 && b >= 0 && count++ % KP != kp) b = any();
        return b;
    };
    struct Loads {
        CodeBlock<T> w[M / 16][NT];
        wh8 x[M / 16];
        float2 s;
    };
    auto load = [&](int b, Loads& to) {
        to.s = make_float2(0.0f, 0.0f);
        if (far) to.s = *(const float2*)(own + a.act.far_scales() + 8 * (size_t)b);
#pragma unroll
        for (int q = 0; q < M / 16; ++q) {
            const int gq = M == 16 ? g : 2 * q + g;
            to.x[q] = wh8{};
            if (far) to.x[q] = *(const wh8*)(own + a.act.far_codes() + 64 * (size_t)b + 16 * gq);
#pragma unroll
            for (int i = 0; i < NT; ++i) to.w[q][i].load(wp[i], b, gq);
        }
    };
    Loads cur;
    int b = next();
    if (AHEAD && b >= 0) load(b, cur);
    while (b >= 0) {
        if (!AHEAD) load(b, cur);
        const int after = next();
        Loads ahead;
        if (AHEAD) {
            ahead = cur;
            if (after >= 0) load(after, ahead);
        }
        V part[NT];
        float d[NT], m[NT];
#pragma unroll
        for (int q = 0; q < M / 16; ++q)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                wh8 rest;
                const wh8 f = cur.w[q][i].unpack(b, M == 16 ? g : 2 * q + g, rest, d[i], m[i]);
                if (q == 0) part[i] = V{};
                if constexpr (M == 16) {
                    part[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cur.x[q], f, part[i], 0, 0, 0);
                    if constexpr (T == T_Q6_K) part[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cur.x[q], rest, part[i], 0, 0, 0);
                } else {
                    part[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(cur.x[q], f, part[i], 0, 0, 0);
                    if constexpr (T == T_Q6_K) part[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(cur.x[q], rest, part[i], 0, 0, 0);
                }
            }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = M == 16 ? 4 * g + j : 8 * (j >> 2) + 4 * g + (j & 3);
            const float dx = __shfl(cur.s.x, at, 64), codes = __shfl(cur.s.y, at, 64);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                // (the weights' factors first: they overflow only where the term does)
                sum[i][j] = fmaf(d[i] * part[i][j], dx, sum[i][j]);
                if constexpr (has_min(T)) sum[i][j] = fmaf(-(m[i] * codes), dx, sum[i][j]);
            }
        }
        if (AHEAD) cur = ahead;
        b = after;
    }
}

// 64 x 16 bytes straight to LDS at m0 (the same in every lane), lane i's from base + off (the lanes' own) to m0 + 16 i.
// In assembly, as the compiler, which would wait for them before any LDS read, is not to see these loads; nor
// does it see that the load needs a wait state behind the write of M0.
__device__ __forceinline__ void to_lds16(const uint8_t* base, uint32_t off, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane((int)m0)) : "memory", "m0");
}

// ---- few rows to an expert ----------------------------------------------------------------------
// ROWS entries of an expert (16, or 4 of single tokens) and the weight rows of NS waves, two 16-row tiles each
// (gate and up of the same rows, or 32 rows); KP groups of NS waves take every KP-th chunk and meet in LDS, in
// order. A wave's weight bytes go to registers a chunk ahead; a group's activation fragments go to LDS a chunk
// ahead, by direct-to-LDS loads (one an entry). LDS: [entry][64 fragments of 16 bytes], fragment f of entry
// i in place f ^ (i % 8), so that eight entries' reads of one fragment fall on distinct banks.
// What counts is how many bytes are on their way: the weights come from HBM, some 2 us away when all CUs read,
// so a CU needs 40 KB and more in flight. Many rows of 16 entries: NS = 4, KP = 1; single tokens: NS = 1 and K
// split over the workgroup, as their few tiles alone would not fill the chip; long rows: both, as
// neighbouring chunks read at the same time are longer runs of memory.
// Measured (MI355X; a kernel alone is the profiler's median, which carries up to 2 us of its own): one row, two of 8 experts,
// gate and up Q4_K 4096 x 14336: 132 MB, a pass with k_expert_act 37 us (3.5 TB/s), this kernel 38, at least 34; down
// Q6_K 14336 x 4096: 96 MB, 32 (3.0 TB/s), at least 30. 61 rows, eight of 128 experts, 2048 x 768 Q4_K: 226 MB, 68 (3.3 TB/s);
// with no weight loads in its loop still 47, of which the unpacking is 24, the MFMAs 9, the rest starts,
// the entries' look-up and barriers: its 768 columns leave each workgroup 8 chunks to work on.
template <uint32_t T, int KP, int NS, int ROWS, bool SWIGLU>
__global__ __launch_bounds__(64 * KP * NS, KP * NS == 8 ? 4 : 3) void k_expert_few(Mul a) {
    constexpr int NT = 2, LOADS = ROWS / NS, MIN = has_min(T) ? 64 * ROWS : 0, BUF = 1024 * ROWS + MIN;
    extern __shared__ __align__(16) uint8_t lds[];  // [KP][2][BUF]
    // (HELD: in registers, which Q4_0 and Q5_0 have: with 128 bytes more of LDS a CU holds three workgroups, not four)
    constexpr bool HELD = ROWS == 16 && (T == T_Q4_0 || T == T_Q5_0);
    __shared__ int ent[ROWS], exps[ROWS];
    // the sums of blocks apart, each lane's own: kept here over the loop, which has no registers for them
    __shared__ f32x4 apart[NS][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kp = wave / NS, ns = wave % NS;
    const int blk = blockIdx.x % a.n_blocks;
    const GroupTile t = find_tile<ROWS>(a.g, 0, blockIdx.x / a.n_blocks, lane);
    if (t.count <= 0) return;
    const int r = lane & 15, g = lane >> 4;
    const int n0 = (blk * NS + ns) * (SWIGLU ? 16 : 32);
    if (kp == 0) {
#pragma unroll
        for (int i = 0; i < NT; ++i) apart[ns][i][lane] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint8_t* wp[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
        wp[i] = a.w[SWIGLU ? i : 0] + (size_t)t.group * a.expert_bytes +
                (size_t)min(n0 + (SWIGLU ? 0 : 16 * i) + r, a.n - 1) * a.row_bytes;
    const int chunks = a.act.chunks;
    WeightChunk<T> wt[2][NT];
    if (kp < chunks) {
#pragma unroll
        for (int i = 0; i < NT; ++i) wt[0][i].load(wp[i], kp, a.nb, g);  // on their way while the entries are looked up
    }
    const int er = r & (ROWS - 1);
    const int e = entry_of(a, t, er);
    const int arow = e < 0 ? 0 : e / a.per_row;
    const int ex = a.act.exps[arow];
    const bool far = e >= 0 && ex >= kExpFar / 2;
    const int own = far ? ex - kExpFar : ex;
    if (!HELD && threadIdx.x < ROWS) {
        ent[er] = e;
        exps[er] = own;
    }
    if (__builtin_expect(__ballot(far) != 0, 0)) {
        f32x4 sum[NT];
        far_sums<T, 16, KP, false, SWIGLU>(a, t.group, n0, e, far, ROWS, kp, lane, sum);
        f32x4* parts = (f32x4*)lds;  // [wave][NT][64]
        if constexpr (KP > 1) {
#pragma unroll
            for (int i = 0; i < NT; ++i) parts[(wave * NT + i) * 64 + lane] = sum[i];
            __syncthreads();
        }
        if (kp == 0) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int k = 1; k < KP; ++k) sum[i] += parts[((k * NS + ns) * NT + i) * 64 + lane];
                apart[ns][i][lane] = sum[i];
            }
        }
        if constexpr (KP > 1) __syncthreads();
        if (kp < chunks) {
#pragma unroll
            for (int i = 0; i < NT; ++i) wt[0][i].load(wp[i], kp, a.nb, g);  // (once more: not held over it)
        }
    }
    // this wave's loads: entries ns, ns + NS, .. (the rows of those lanes)
    const uint8_t* from[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
        from[j] = a.act.frags + (size_t)(uint32_t)__builtin_amdgcn_readlane(arow, ns + NS * j) * a.act.row;
    const uint32_t m_off = (uint32_t)__shfl(arow, (lane >> 2) & (ROWS - 1), 64) * (uint32_t)(chunks * 64) +
                           16u * (uint32_t)((lane & 3) ^ ((lane >> 3) & 3));
    uint8_t* mine = lds + kp * 2 * BUF;
    const uint32_t m0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)mine;
    auto issue = [&](int c, int buf) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int i = ns + NS * j;
            if (i < t.count)
                to_lds16(from[j] + (size_t)c * 1024, 16u * (uint32_t)(lane ^ (i & 7)),
                         m0 + (uint32_t)(BUF * buf + 1024 * i));
        }
        if (has_min(T) && ns == NS - 1 && lane < 4 * ROWS)
            to_lds16(a.act.mins + (size_t)c * 64, m_off, m0 + (uint32_t)(BUF * buf + 1024 * ROWS));
    };
    // fragment (s, part) of this lane's entry and group: a_at ^ a constant
    const uint32_t a_at = (uint32_t)er * 1024u + 16u * (uint32_t)((is_kq(T) ? (g >> 1) * 32 + (g & 1) : g) ^ (er & 7));
    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (kp < chunks) issue(kp, 0);
    auto chunk = [&]<int PAR>(int c) {
        // this wave's loads are in LDS, and its reads of the other buffer done, which is loaded next (of a group of
        // waves the barrier says both for all)
        __builtin_amdgcn_s_waitcnt(NS > 1 ? 0x0F70 : 0x0070);
        asm volatile("" ::: "memory");
        if constexpr (NS > 1) __syncthreads();
        if (c + KP < chunks) {
            issue(c + KP, 1 - PAR);
#pragma unroll
            for (int i = 0; i < NT; ++i) wt[1 - PAR][i].load(wp[i], c + KP, a.nb, g);
        }
        if (c >= chunks) return;
        const uint8_t* cur = mine + PAR * BUF;
        auto frag = [&](int s, int part) {
            return *(const wh8*)(cur + (a_at ^ (uint32_t)(is_kq(T) ? 64 * s + 32 * part : 128 * s + 64 * part)));
        };
        wh8 am = {};
        if constexpr (has_min(T)) am = *(const wh8*)(cur + 1024 * ROWS + er * 64 + 16 * (g ^ ((er >> 1) & 3)));
        chunk_product<T, NT>(wt[PAR], c, a.nb, g, frag, am, acc);
    };
    for (int c = kp; c - kp < chunks; c += 2 * KP) {
        chunk.template operator()<0>(c);
        if (c - kp + KP < chunks) chunk.template operator()<1>(c + KP);
    }
    // lane (r, g) has entries 4g + j of weight row r of each tile
    if constexpr (KP > 1) {
        float* red = (float*)lds;  // [wave][NT][256]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT; ++i) *(f32x4*)(red + (wave * NT + i) * 256 + 4 * lane) = acc[i];
        __syncthreads();
        if (kp != 0) return;
#pragma unroll
        for (int k = 1; k < KP; ++k)
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] += *(const f32x4*)(red + ((k * NS + ns) * NT + i) * 256 + 4 * lane);
    } else {
        __syncthreads();
    }
    int en4[4], ex4[4];
    if constexpr (HELD) {
#pragma unroll
        for (int j = 0; j < 4; ++j) en4[j] = __shfl(e, 4 * g + j, 64), ex4[j] = __shfl(own, 4 * g + j, 64);
    }
#pragma unroll
    for (int i = 0; i < (SWIGLU ? 1 : NT); ++i) {
        const int row = n0 + 16 * i + r;
        if (row >= a.n) continue;
        const size_t b = (size_t)t.group * a.n + row;
        const float b0 = a.bias[0] ? a.bias[0][b] : 0.0f, b1 = SWIGLU && a.bias[1] ? a.bias[1][b] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int tok = 4 * g + j, en = HELD ? en4[j] : tok < ROWS ? ent[tok & (ROWS - 1)] : -1;
            if (en < 0) continue;
            const int x = HELD ? ex4[j] : exps[tok & (ROWS - 1)];
            float v = unscaled(acc[i][j], x) + apart[ns][i][lane][j] + b0;
            if constexpr (SWIGLU) v = silu_mul(v, unscaled(acc[1][j], x) + apart[ns][1][lane][j] + b1);
            a.y[(size_t)en * a.n + row] = v;
        }
    }
}
template <uint32_t T, int KP, int NS, int ROWS>
constexpr int few_lds() {
    const int buf = KP * 2 * (1024 * ROWS + (has_min(T) ? 64 * ROWS : 0)), red = KP > 1 ? KP * NS * 2048 : 0;
    return buf > red ? buf : red;
}

// ---- many rows to an expert ----------------------------------------------------------------------
// 32 MT entries of an expert and 256 weight rows (128 of gate and of up): four waves of 64 weight rows (two
// 32-column MFMA tiles, gate and up of the same rows, or 64 rows). The waves share the activation
// fragments, which reach LDS in stages of half a chunk, two buffers, by direct-to-LDS loads; each wave
// loads and unpacks its weight rows' bytes a stage ahead in registers (with minima, the rows' headers in LDS).
// LDS: [entry][32 fragments of 16 bytes], fragment f of entry i in place f ^ (i % 32), so that the 32
// entries' reads of one fragment fall on distinct banks.
// Measured (MI355X): 2048 rows, two of 8 experts each, gate and up Q4_K of 4096 x 14336: 1.95 ms, 962 GFLOP,
// 493 TFLOP/s, and as many again for lo: 76% of what the library's fp16 product reaches. With nothing
// loaded in the loop 1.44 ms: the activations' way to LDS (7.3 GB, from L2) is the rest; the weights' is
// hidden. A register spilled into that loop costs much: 2.57 ms with 10. 128 entries to eight waves,
// which halves the weights' unpacking: slower (3.32 | 2.42 ms), as eight waves in step at
// each stage leave the matrix cores idle. Down Q6_K 14336 x 4096, three products: 1.70 ms, 849 TFLOP/s.
template <int MT>
struct Wide {
    static constexpr int BM = 32 * MT;
    static constexpr int FRAGS = BM * 512;                       // a stage's fragments, two buffers
    static constexpr int MINS = 2 * FRAGS, HDRS = MINS + BM * 64;  // minima of a chunk; headers, two buffers
    static constexpr int LDS = HDRS + 2 * 256 * 16;
};

template <uint32_t T, int MT, bool SWIGLU>
__global__ __launch_bounds__(256, 2) void k_expert_wide(Mul a) {
    using C = Wide<MT>;
    constexpr int NT = 2;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int ent[C::BM], exps[C::BM];
    __shared__ uint32_t from_a[C::BM], from_m[C::BM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blk = blockIdx.x % a.n_blocks;
    const GroupTile t = find_tile<C::BM>(a.g, 0, blockIdx.x / a.n_blocks, lane);
    if (t.count <= 0) return;
    const int r = lane & 31, h = lane >> 5;
    for (int i = threadIdx.x; i < C::BM; i += 256) {
        const int e = entry_of(a, t, i);
        const uint32_t row = (uint32_t)(e < 0 ? 0 : e / a.per_row);
        ent[i] = e;
        exps[i] = e < 0 ? 0 : a.act.exps[row];
        from_a[i] = row * a.act.row;
        from_m[i] = row * (uint32_t)(a.act.chunks * 64);
    }
    __syncthreads();
    const uint8_t* wbase[2];
    uint32_t w_at[NT];  // this lane's rows
    const int n0 = blk * (SWIGLU ? 128 : 256) + wave * (SWIGLU ? 32 : 64);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        wbase[i] = a.w[SWIGLU ? i : 0] + (size_t)t.group * a.expert_bytes;
        w_at[i] = (uint32_t)min(n0 + (SWIGLU ? 0 : 32 * i) + r, a.n - 1) * a.row_bytes;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)lds;
    // this wave's direct-to-LDS loads of a stage: two entries each; of the minima's 16, place q of entry i
    // holds part q ^ (i / 2 % 4)
    auto issue = [&](int st, int buf) {
        const uint32_t to = lds0 + (uint32_t)buf * C::FRAGS;
        const uint8_t* from = a.act.frags + (size_t)st * 512;
        uint32_t swz = 16u * (uint32_t)(r ^ (2 * wave + h));  // 16 (r ^ (i % 32)), but for bits 3 and 4 of i
        asm volatile("" : "+v"(swz));                         // (not a register for each j)
#pragma unroll
        for (int j = 0; j < C::BM / 8; ++j) {
            const int k = 4 * j + wave, i = 2 * k + h;
            to_lds16(from, from_a[i] + (swz ^ (128u * (uint32_t)(j & 3))), to + 1024u * (uint32_t)k);
        }
        if (has_min(T) && (st & 1) && 16 * wave < C::BM) {
            const int i = 16 * wave + (lane >> 2);
            to_lds16(a.act.mins + (size_t)(st >> 1) * 64, from_m[i] + 16u * (uint32_t)((lane & 3) ^ ((i >> 1) & 3)),
                     lds0 + C::MINS + 1024u * (uint32_t)wave);
        }
        // the headers of the next chunk: lanes 0-31 the wave's first tile's rows, 32-63 the second's
        if (has_min(T) && !(st & 1)) {
            const uint32_t to_h = lds0 + C::HDRS + 4096u * (uint32_t)((st >> 1) & 1) + 1024u * (uint32_t)wave;
            const size_t chunk = (size_t)(st >> 1) * Bytes<T>::V;
            if (!SWIGLU)
                to_lds16(wbase[0] + chunk, h ? w_at[1] : w_at[0], to_h);
            else if (h == 0)
                to_lds16(wbase[0] + chunk, w_at[0], to_h);
            else
                to_lds16(wbase[1] + chunk, w_at[1], to_h);
        }
    };

    const int stages = 2 * a.act.chunks;
    const wf16 zero = {};
    wf16 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = zero;
    // fragment (s, part) of lane half h of the wave's entry 32 m + r: a_at ^ 16 (4 s + 2 part), plus 16384 m
    // (blocks of 32: (block, part, 2 h + q) at a_at ^ 16 (8 block + 4 part + q))
    const uint32_t a_at = (uint32_t)(r * 512 + 16 * (r ^ (is_kq(T) ? h : 2 * h)));
    auto begin = [&](int st, int half) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's loads of the stage are in LDS
        asm volatile("" ::: "memory");
        __syncthreads();                     // and every wave's; the other buffer is free
        if (st + 1 < stages) issue(st + 1, 1 - half);
    };
    issue(0, 0);

    if constexpr (is_kq(T)) {
        // A stage is 8 steps: 16 elements of K, the 8 of lane half h from lane group g = 2 HALF + h. A step's MFMAs
        // run beside the unpacking of the next; its lo fragments are read beside the products with hi, the
        // next step's hi beside those with lo. Weight bytes are loaded a stage ahead, like the activations.
        constexpr int PARTS = T == T_Q6_K ? 3 : 2;
        constexpr bool AHEAD = T == T_Q4_K || MT == 1;  // (registers; 32 entries, down Q6_K 14336, 120 rows: 378 | 308 us)
        Part<T> pt[AHEAD ? 2 : 1][NT];
        wf16 sum[NT][MT];
        wh8 ah[MT], al[MT], bf[2][NT], rest[2][NT];
        Scales2 sc[NT];
        auto load_part = [&](int st, int half) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if constexpr (T == T_Q4_K)
                    pt[half][i].load(wbase[i] + (size_t)(st >> 1) * Part<T>::BYTES + 64 * half + (w_at[i] + 32u * (uint32_t)h), 0);
                else
                    pt[AHEAD ? half : 0][i].load(wbase[i] + (size_t)(st >> 1) * Part<T>::BYTES + w_at[i], 2 * half + h);
        };
        auto stage = [&]<int HALF>(int st) {
            begin(st, HALF);
            if (AHEAD && st + 1 < stages) load_part(st + 1, 1 - HALF);
            const uint8_t* cur = lds + HALF * C::FRAGS;
            const int g = 2 * HALF + h;
            const uint8_t* hdr = lds + C::HDRS + 4096 * ((st >> 1) & 1) + 1024 * wave + 16 * r;
            uint32_t a_now = a_at;
            if constexpr (has_min(T) || MT == 1) asm volatile("" : "+v"(a_now));  // (not a register for each fragment's place)
            auto read_a = [&](int p, int part, wh8 (&to)[MT]) {
                const uint8_t* from = cur + (a_now ^ (uint32_t)(16 * (4 * p + 2 * part)));
#pragma unroll
                for (int m = 0; m < MT; ++m) to[m] = *(const wh8*)(from + 16384 * m);
            };
            auto unpack = [&](int p) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if constexpr (has_min(T))
                        if (p == 0) sc[i] = Part<T>::scale(*(const u32x4*)(hdr + 512 * i), g);
                    if constexpr (T == T_Q6_K)
                        bf[p & 1][i] = pt[AHEAD ? HALF : 0][i].frag(p, g, rest[p & 1][i]);
                    else
                        bf[p & 1][i] = pt[AHEAD ? HALF : 0][i].frag(sc[i], p, g);
                }
            };
            float dq[NT];
            read_a(0, 0, ah);
            unpack(0);
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                __builtin_amdgcn_sched_barrier(0);
                read_a(p, 1, al);
                if (p < 7) unpack(p + 1);
                if (!AHEAD && p == 7) {
                    if constexpr (T == T_Q6_K) {
#pragma unroll
                        for (int i = 0; i < NT; ++i) dq[i] = pt[0][i].d();
                    }
                    if (st + 1 < stages) load_part(st + 1, 1 - HALF);
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            sum[i][m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                                part == PARTS - 1 ? al[m] : ah[m], PARTS == 3 && part == 1 ? rest[p & 1][i] : bf[p & 1][i],
                                HALF == 0 && p == 0 && part == 0 ? zero : sum[i][m], 0, 0, 0);
                    if (part == PARTS - 2 && p < 7) read_a(p + 1, 0, ah);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, MT, 0);  // lo of this step
#pragma unroll
                for (int g = 0; g < PARTS * NT * MT; ++g) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // an MFMA
                    __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);  // unpacking beside it
                    if (g == (PARTS - 1) * NT * MT - 1) __builtin_amdgcn_sched_group_barrier(0x100, MT, 0);  // the next hi
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (HALF == 1) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float d, dm = 0.0f;
                    wh8 mn;
                    if constexpr (has_min(T)) {
                        const u32x4 v = *(const u32x4*)(hdr + 512 * i);
                        d = f16_to_f32(v.x & 0xFFFFu);
                        dm = -(float)(1 << kMinShift) * f16_to_f32(v.x >> 16);
                        mn = k4_minima(v);
                    } else {
                        d = AHEAD ? pt[AHEAD ? 1 : 0][i].d() : dq[i];
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        if constexpr (has_min(T)) {
                            const uint8_t* row = lds + C::MINS + (32 * m + r) * 64;
                            wf16 f = zero;
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const wh8 x = *(const wh8*)(row + 16 * ((2 * h + q) ^ ((r >> 1) & 3)));
                                f = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, mn, f, 0, 0, 0);
                            }
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                acc[i][m][e] = fmaf(d, sum[i][m][e], fmaf(dm, f[e], acc[i][m][e]));
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[i][m][e] = fmaf(d, sum[i][m][e], acc[i][m][e]);
                        }
                        asm volatile("" : "+v"(acc[i][m]));  // not sunk to where the sums are read next
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        };
        load_part(0, 0);
        for (int st = 0; st < stages; st += 2) {
            stage.template operator()<0>(st);
            stage.template operator()<1>(st + 1);
        }
    } else {
        // A stage is 4 blocks. Items (block, entry tile, weight tile): an item's four MFMAs run beside the
        // multiplication with d of the item before it. Everything is read or unpacked into the registers
        // that the items no longer need: a block's fragments an item or two ahead, a stage's weight
        // bytes a stage ahead.
        constexpr int N = NT * MT;
        BlockPair<T> u[2][NT];
        auto load_pair = [&](int st, int k) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                u[k][i].load(wbase[i] + (size_t)min(4 * st + 2 * k + h, a.nb - 1) * BlockPair<T>::BYTES + w_at[i]);
        };
        load_pair(0, 0);
        load_pair(0, 1);
        auto stage = [&]<int HALF>(int st) {
            begin(st, HALF);
            const uint8_t* cur = lds + HALF * C::FRAGS;
            wh8 af[2][2][2], bf[NT][2];  // [entry tile, or block parity][q][part]
            float d[2][NT];
            wf16 f[2];
            auto read = [&](int s, int m) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        af[MT == 2 ? m : s & 1][q][part] =
                            *(const wh8*)(cur + (a_at ^ (uint32_t)(16 * (8 * s + 4 * part + q))) + 16384 * m);
            };
            auto unpack = [&](int s, int i) {
                if ((s & 1) == 0) u[s >> 1][i].exchange();
#pragma unroll
                for (int q = 0; q < 2; ++q) bf[i][q] = u[s >> 1][i].frag(s & 1, q, h);
                d[s & 1][i] = 4 * st + s < a.nb ? f16_to_f32(u[s >> 1][i].d[s & 1]) : 0.0f;
            };
            auto fold = [&](int it) {
                const int s = it / N, m = it % N / NT, i = it % NT;
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][m][e] = fmaf(d[s & 1][i], f[it & 1][e], acc[i][m][e]);
                asm volatile("" : "+v"(acc[i][m]));  // not sunk to where the sums are read next
            };
            read(0, 0);
            unpack(0, 0);
#pragma unroll
            for (int it = 0; it < 4 * N; ++it) {
                const int s = it / N, m = it % N / NT, i = it % NT;
                __builtin_amdgcn_sched_barrier(0);
                if (it % N == 0) {
                    if (MT == 2) read(s, 1);
                    unpack(s, 1);
                    if (MT == 1 && s < 3) read(s + 1, 0);
                }
                if (it % N == 1 && (s & 1) && st + 1 < stages) load_pair(st + 1, s >> 1);
                if (MT == 2 && it % N == 2 && s < 3) read(s + 1, 0);
                if (it % N == N - 1 && s < 3) unpack(s + 1, 0);
                wf16 z = zero;
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        z = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[MT == 2 ? m : s & 1][q][part], bf[i][q], z, 0, 0, 0);
                f[it & 1] = z;
                if (it > 0) fold(it - 1);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            fold(4 * N - 1);
        };
        for (int st = 0; st < stages; st += 2) {
            stage.template operator()<0>(st);
            stage.template operator()<1>(st + 1);
        }
    }

#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int again = lane_again(), x = exps[32 * m + (again & 31)];
        if (__builtin_expect(__ballot(x >= kExpFar / 2) != 0, 0)) {
            wf16 sum[NT];
            far_sums<T, 32, 1, MT == 2, SWIGLU>(a, t.group, n0, ent[32 * m + (again & 31)], x >= kExpFar / 2, 32, 0, again, sum);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int of = exps[32 * m + 8 * (e >> 2) + 4 * (again >> 5) + (e & 3)];
                    if (of >= kExpFar / 2) acc[i][m][e] = unscaled(acc[i][m][e], of - kExpFar) + sum[i][e];
                }
        }
    }
    // lane (r, h) has entries 8 (e / 4) + 4 h + e % 4 of weight row r of each tile
#pragma unroll
    for (int i = 0; i < (SWIGLU ? 1 : NT); ++i) {
        const int row = n0 + 32 * i + r;
        if (row >= a.n) continue;
        const size_t b = (size_t)t.group * a.n + row;
        const float b0 = a.bias[0] ? a.bias[0][b] : 0.0f, b1 = SWIGLU && a.bias[1] ? a.bias[1][b] : 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int tok = 32 * m + 8 * (e >> 2) + 4 * h + (e & 3);
                const int en = ent[tok];
                if (en < 0) continue;
                float v = result(acc[i][m][e], exps[tok]) + b0;
                if constexpr (SWIGLU) v = silu_mul(v, result(acc[1][m][e], exps[tok]) + b1);
                a.y[(size_t)en * a.n + row] = v;
            }
    }
}

// ---- the sum over a row's experts ----------------------------------------------------------------
// Bound by its bytes: 2048 rows x 2 of 4096 and the sums 100 MB, 17 us (5.9 TB/s, partly from caches); one row 4.7 us.
__global__ __launch_bounds__(256) void k_expert_sum(const float* __restrict__ p, const int32_t* __restrict__ ids,
                                                    const float* __restrict__ weights, int top_k, int groups, int n,
                                                    const float* base, float* y) {
    const int row = blockIdx.y;
    const int i = (blockIdx.x * 256 + threadIdx.x);
    if (n % 4 == 0) {
        if (4 * i >= n) return;
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j = 0; j < top_k; ++j) {
            if ((uint32_t)ids[row * top_k + j] >= (uint32_t)groups) continue;
            const float w = weights[row * top_k + j];
            const f32x4 v = *(const f32x4*)(p + ((size_t)row * top_k + j) * n + 4 * i);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c] = fmaf(w, v[c], s[c]);
        }
        const size_t at = (size_t)row * n + 4 * i;
        if (base) s += *(const f32x4*)(base + at);
        *(f32x4*)(y + at) = s;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int col = (blockIdx.x * 4 + c) * 256 + threadIdx.x;
            if (col >= n) return;
            float s = 0.0f;
            for (int j = 0; j < top_k; ++j) {
                if ((uint32_t)ids[row * top_k + j] >= (uint32_t)groups) continue;
                s = fmaf(weights[row * top_k + j], p[((size_t)row * top_k + j) * n + col], s);
            }
            const size_t at = (size_t)row * n + col;
            y[at] = base ? s + base[at] : s;
        }
    }
}

template <Order O>
hipError_t act_launch(const ExpertArgs& a, const Act& act, hipStream_t s) {
    if (a.rows <= 64)
        k_expert_act<O, 1024><<<a.rows, 1024, 0, s>>>(a.x, a.k, act);
    else
        k_expert_act<O, 256><<<a.rows, 256, 0, s>>>(a.x, a.k, act);
    return hipGetLastError();
}

struct Plan {
    int rows;  // entries of a tile: 4, 8 or 16 (k_expert_few), 32 or 64 (k_expert_wide)
    int kp;    // K parts of k_expert_few's workgroups (tiles of 8: 4)
    int n_blocks, tiles;
};
Plan plan_of(uint32_t type, int mats, int k, int n, int groups, int entries) {
    Plan p{};
    const int live = std::max(1, std::min(groups, entries)), per = (entries + live - 1) / live;
    // By the mean number of entries of an expert (MI355X, us, tile of fewer | of more entries):
    //  4 | 16  16 entries over 8 experts, gate and up Q4_K 4096 x 14336: 117 | 132; rows of 2048, 256 over 128: 66 | 59
    //  8       rows of 8192 and more: 24 over 8, down Q4_K 14336: 78, on tiles of 16 114; 80 Q6_K: 236, 257
    // 16 | 32  128 over 8, gate and up Q4_K 4096: 209 | 188; 2048 over 128, rows of 2048: 103 | 112
    //          down 14336: 180 over 8: Q4_K 186 | 205, Q6_K 347 | 306, 120 Q6_K 256 | 305
    // 32 | 64  gate and up Q4_K 4096: 260 over 8: 296 | 279, 400: 336 | 343, 512: 410 | 387, 1024: 678 | 617; Q5_K, 400:
    //          443 | 422, 280: 369 | 362; Q8_0 1408 x 1376, 2036 over 60: 160 | 144;
    //          Q6_K, whose bytes stay ahead in a tile of 32 only: down 14336, 280: 308 | 440, 400: 478 | 441; 4800 over 128
    //          experts of 2048 x 768: 225 | 239
    const int chunks = chunks_of(k);
    p.rows = per <= (chunks >= 12 ? 2 : 1) ? 4 : per <= 12 && chunks >= 32 ? 8 : per <= (chunks >= 32 && type != T_Q6_K ? 24 : 16) ? 16
           : per <= (type == T_Q6_K ? 40 : 32) ? 32 : 64;
    p.kp = p.rows == 8 ? 4 : 1;
    const int block = (p.rows == 4 ? 32 : p.rows == 8 ? 64 : p.rows == 16 ? 128 : 256) / mats;
    p.n_blocks = (n + block - 1) / block;
    p.tiles = p.rows == 4 ? tile_ids<4>(groups, entries) : p.rows == 8 ? tile_ids<8>(groups, entries) : p.rows == 16 ? tile_ids<16>(groups, entries)
            : p.rows == 32 ? tile_ids<32>(groups, entries) : tile_ids<64>(groups, entries);
    if (p.rows == 4) {
        // K in 8 parts where 4 would leave a CU fewer than 16 waves and have long ways each (3 rows over 8 experts,
        // down Q4_0 14336: 73 us, 80 in 4 parts; one row, gate and up Q4_K 4096: 43 and 38)
        const long waves = (long)std::min(p.tiles, entries) * p.n_blocks;
        p.kp = chunks >= 32 && waves * 4 < 4096 ? 8 : 4;
    }
    return p;
}

template <uint32_t T, int KP, int NS, int ROWS, bool SWIGLU>
hipError_t few_launch(Mul& m, uint32_t grid, hipStream_t s) {
    constexpr int LDS = few_lds<T, KP, NS, ROWS>();
    auto* kern = k_expert_few<T, KP, NS, ROWS, SWIGLU>;
    if constexpr (LDS > 60 * 1024) {
        static LdsLimit limit;
        if (hipError_t e = limit.raise((const void*)kern, LDS)) return e;
    }
    kern<<<grid, 64 * KP * NS, LDS, s>>>(m);
    return hipGetLastError();
}

template <uint32_t T, int MT, bool SWIGLU>
hipError_t wide_launch(Mul& m, uint32_t grid, hipStream_t s) {
    static LdsLimit limit;
    auto* kern = k_expert_wide<T, MT, SWIGLU>;
    if (hipError_t e = limit.raise((const void*)kern, Wide<MT>::LDS)) return e;
    kern<<<grid, 256, Wide<MT>::LDS, s>>>(m);
    return hipGetLastError();
}

template <uint32_t T, bool SWIGLU>
hipError_t mul_launch(Mul& m, const Plan& p, hipStream_t s) {
    const uint32_t grid = (uint32_t)p.n_blocks * (uint32_t)p.tiles;
    if (p.rows == 64) return wide_launch<T, 2, SWIGLU>(m, grid, s);
    if (p.rows == 32) return wide_launch<T, 1, SWIGLU>(m, grid, s);
    if (p.rows == 8) return few_launch<T, 4, 2, 8, SWIGLU>(m, grid, s);
    if (p.rows == 16) return few_launch<T, 1, 4, 16, SWIGLU>(m, grid, s);
    if (p.kp == 8) return few_launch<T, 8, 1, 4, SWIGLU>(m, grid, s);
    return few_launch<T, 4, 1, 4, SWIGLU>(m, grid, s);
}
template <uint32_t T>
hipError_t mul_launch2(Mul& m, int mats, const Plan& p, hipStream_t s) {
    return mats == 2 ? mul_launch<T, true>(m, p, s) : mul_launch<T, false>(m, p, s);
}

}  // namespace

size_t expert_act_bytes(uint32_t type, int k, int rows) {
    const Act a = act_of(nullptr, type, k, rows);
    return up256((size_t)(uintptr_t)a.far + (size_t)rows * a.far_row());
}

hipError_t launch_experts(const ExpertArgs& a, hipStream_t s) {
    const Act act = act_of(a.ws, a.type, a.k, a.rows);
    hipError_t e;
    switch (order_of(a.type)) {
        case kMin64: e = act_launch<kMin64>(a, act, s); break;
        case kQ6: e = act_launch<kQ6>(a, act, s); break;
        case kByte: e = act_launch<kByte>(a, act, s); break;
        default: e = act_launch<kNibble>(a, act, s); break;
    }
    if (e != hipSuccess) return e;
    const Plan p = plan_of(a.type, a.mats, a.k, a.n, a.g.groups, a.g.entries);
    Mul m{};
    m.w[0] = a.w[0], m.w[1] = a.w[1];
    m.bias[0] = a.bias[0], m.bias[1] = a.bias[1];
    m.row_bytes = (uint32_t)(a.k / block_elems(a.type) * (int)block_bytes(a.type));
    m.expert_bytes = (size_t)a.n * m.row_bytes;
    m.n = a.n;
    m.nb = a.k / 32;
    m.act = act;
    m.per_row = a.per_row;
    m.rows = a.rows;
    m.g = a.g;
    m.n_blocks = p.n_blocks;
    m.y = a.y;
    switch (a.type) {
        case T_Q4_0: return mul_launch2<T_Q4_0>(m, a.mats, p, s);
        case T_Q5_0: return mul_launch2<T_Q5_0>(m, a.mats, p, s);
        case T_Q8_0: return mul_launch2<T_Q8_0>(m, a.mats, p, s);
        case T_Q4_K: return mul_launch2<T_Q4_K>(m, a.mats, p, s);
        case T_Q5_K: return mul_launch2<T_Q5_K>(m, a.mats, p, s);
        case T_Q6_K: return mul_launch2<T_Q6_K>(m, a.mats, p, s);
        default: return hipErrorInvalidValue;
    }
}

void expert_plan_name(uint32_t type, int mats, int k, int n, int groups, int entries, char* buf, size_t cap) {
    if (!has_kernel(type) || n <= 0 || entries <= 0) {
        snprintf(buf, cap, "none");
        return;
    }
    const Plan p = plan_of(type, mats, k, n, groups, entries);
    if (p.rows <= 16)
        snprintf(buf, cap, "k_expert_few<%d,%d> workgroups=%lld", p.kp, p.rows, (long long)p.n_blocks * p.tiles);
    else
        snprintf(buf, cap, "k_expert_wide<%d> workgroups=%lld", p.rows, (long long)p.n_blocks * p.tiles);
}

int64_t expert_workgroups(uint32_t type, int mats, int k, int n, int groups, int entries) {
    const Plan p = plan_of(type, mats, k, n, groups, entries);
    return (int64_t)p.n_blocks * p.tiles;
}

hipError_t launch_expert_sum(const float* p, const int32_t* ids, const float* weights, int rows, int top_k, int groups,
                             int n, const float* base, float* y, hipStream_t s) {
    k_expert_sum<<<dim3((unsigned)((n + 1023) / 1024), (unsigned)rows), 256, 0, s>>>(p, ids, weights, top_k, groups, n,
                                                                                    base, y);
    return hipGetLastError();
}

}  // namespace cllm_hip
