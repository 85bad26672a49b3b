// kv4.h -- the paged key/value cache held in 4 bits: its layout, shared by the kernels that store,
// read, attend over and move its pages (internal to libcllm_hip.so).
//
// A page holds page_size positions of every KV head of one layer, as [n_kv][page_size / 32] tiles;
// the pool is [n_layers][n_pages][page]. A tile is 32 positions of one head, 36 * HD bytes:
//   key codes    at 0       dwords of 8 codes, [t 2][c][g 4][n 16][w W]: position 16 t + n, elements
//                           g HD/4 + 8 (c W + w) + e; W = min(4, HD / 32)
//   value codes  at 16 HD   dwords of 8 codes, [c HD/64][g 4][n 16][w 4]: element 16 (4 c + w) + n,
//                           positions 16 (e / 4) + 4 g + e % 4
//   key scales   at 32 HD   fp16 [HD / 32][n 16][t 2]: position 16 t + n
//   value scales at 34 HD   fp16 [HD / 32][g 4][e 8]: positions as the value codes'
// Code e of a dword lies in nibble e / 2 + 4 (e % 2), so that each (dword >> 4 r) & 0x000F000F is
// the fp16 pair of codes 2 r and 2 r + 1 after an or with 0x6400 (1024 + code).
//
// The order is the MFMA operands': for v_mfma_f32_16x16x32_f16, lane 16 g + n reads its key dwords
// as row n of a keys x queries product and its value dwords as row n of a values x weights product,
// whose weights (positions 4 g .. 4 g + 3 of either half of the tile) are the lane's own scores,
// so neither codes nor weights move between lanes; every load of a wave is contiguous.
//
// An element is d * (c - 8). The scale d has 8 significant bits, so the product (8 bits by a 3-bit
// magnitude, or 8) is exact in fp16: dequantization adds no error to the quantization's. d is at
// most 8160, so no element passes 65280. (Elements below 2^-14 are fp16 subnormals, exact too, but an
// MFMA does not normalise them and keeps fewer bits of their products: outputs from values of 1e-5 are
// off by 5e-7 in the root mean square, like any, from 1e-6 by 3e-6, from 3e-7 by 1e-5; keys of 1e-6 add
// 3e-7.) A position whose key or value row held an infinity or a NaN has NaN as its key scales and 0 as
// its value scales: whatever sees it becomes NaN through its score, and rows that do not see it stay
// clean (a NaN among the values would not: 0 * NaN is NaN).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cllm_hip {

// The cache as the kernels see it (cllm_hip_kv4_cache, checked).
struct Kv4View {
    uint8_t* pages;
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    int32_t* work;
    int n_layers, n_pages, n_kv, hd, max_seqs, max_pages;
    int page_shift;      // log2(page_size)
    int64_t page_bytes;  // of one layer
};

// Sequence i of a batch: its slot, its rows [r0, r0 + rows) of the batch and its length, each held
// to what the buffers have (malformed values read as an empty sequence, never out of range).
struct Kv4Seq {
    int slot, r0, rows, len;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4View& c, const int32_t* slots,
                                          const int32_t* q_start, int i, int n_rows) {
    Kv4Seq s;
    s.slot = slots ? slots[i] : i;
    s.r0 = min(max(q_start[i], 0), n_rows);
    s.rows = min(max(q_start[i + 1], s.r0), n_rows) - s.r0;
    if ((unsigned)s.slot >= (unsigned)c.max_seqs) {
        s.slot = 0;
        s.rows = 0;
    }
    s.len = min(max(c.lens[s.slot], 0), c.max_pages << c.page_shift);
    return s;
}

// Attention (k_kv4.hip). ws: kv4_attention_ws_bytes bytes.
struct Kv4AttnPlan {
    bool many_rows; // the kernel for many rows
    int splits;     // workgroups per unit, 0: shares across units (k_kv4.hip)
    int cols;       // (row, head) pairs of a workgroup
    int64_t units;  // column tiles of the KV heads of the sequences, at most
    int64_t grid;   // workgroups
};
Kv4AttnPlan kv4_attention_plan(const Kv4View& c, int n_seqs, int max_rows, int max_len, int n_head);
bool kv4_attention_fits(const Kv4AttnPlan& p, int hd);
size_t kv4_attention_ws_bytes(const Kv4AttnPlan& p, int hd);
hipError_t launch_kv4_attention(const Kv4View& c, const Kv4AttnPlan& p, int layer, const float* q,
                                const int32_t* slots, const int32_t* q_start, int n_seqs, int n_rows,
                                int max_rows, int n_head, float* out, void* ws, hipStream_t stream);
hipError_t launch_kv4_store(const Kv4View& c, int layer, const float* k, const float* v, float* q,
                            int n_head, float theta_base, const int32_t* slots,
                            const int32_t* q_start, int n_seqs, int n_rows, hipStream_t stream);
hipError_t launch_kv4_load(const Kv4View& c, int layer, const int32_t* slots, const int32_t* q_start,
                           int n_seqs, int n_rows, float* k, float* v, hipStream_t stream);

// Page work (k_pages.hip).
int64_t kv4_work_ints(int n_pages, int max_seqs, int max_pages);
hipError_t launch_kv4_extend(const Kv4View& c, const int32_t* slots, const int32_t* counts, int n,
                             int32_t* status, hipStream_t stream);
hipError_t launch_kv4_fork(const Kv4View& c, const int32_t* src, const int32_t* dst, int n,
                           hipStream_t stream);
hipError_t launch_kv4_truncate(const Kv4View& c, const int32_t* slots, const int32_t* new_lens, int n,
                               hipStream_t stream);
hipError_t launch_kv4_compact(const Kv4View& c, int32_t* n_live, hipStream_t stream);
hipError_t launch_kv4_copy_pages(const Kv4View& c, const int32_t* src, const int32_t* dst, int n,
                                 hipStream_t stream);

// Log probabilities (k_logprobs.hip).
constexpr int kMaxTopK = 64;
size_t logprobs_ws_bytes(int n_rows, int vocab, int top_k);
hipError_t launch_logprobs(const float* logits, int64_t stride, int n_rows, int vocab,
                           const int32_t* tokens, int top_k, float* logprobs, int32_t* ranks,
                           float* entropy, float* lse, int32_t* top_ids, float* top_logprobs,
                           void* ws, hipStream_t stream);

}  // namespace cllm_hip
