// Arguments and shared pieces of the gated delta rule over packed sequences
// (scan.hip: token by token; scan_chunk.hip: in chunks, and the gradient).
#pragma once

#include <algorithm>

#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {

struct ScanArgs {
    int seqs, tokens, heads, key_heads, group, dim, value_dim, pool;
    int normalize, beta_fp32, clear;
    int token_wise;   // sequences of up to so many tokens go token by token
    float scale;
    const uint16_t *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;   // strides in elements
    const float* g;
    const void* beta;
    int64_t g_token, beta_token;
    const int32_t *starts, *from, *into;
    const uint8_t* fresh;
    const float* initial;
    float* final;
    uint16_t* out;
    int64_t out_token, out_head;
    uint8_t* tape;   // what the gradient needs: the chunks' first states and w, or NULL
};
struct ScanGradArgs {
    const uint16_t* d_out;
    int64_t d_out_token, d_out_head;
    const float* d_final;
    const uint8_t* tape;
    uint16_t *dq, *dk, *dv;
    float* dg;
    void* dbeta;
    float* d_initial;
};
hipError_t launch_delta_scan(ScanArgs a, bool fp16, int max_new, void* workspace, hipStream_t stream);
size_t delta_scan_workspace_bytes(ScanArgs a, bool fp16, int max_new);

size_t delta_scan_tape_bytes(const ScanArgs& a);
size_t delta_scan_grad_workspace_bytes(const ScanArgs& a, bool fp16);
hipError_t launch_delta_scan_grad(const ScanArgs& a, const ScanGradArgs& d, bool fp16, void* workspace,
                                  hipStream_t stream);

// The chunked form (scan_chunk.hip).
size_t scan_chunk_bytes(const ScanArgs& a, bool fp16);
hipError_t launch_scan_chunks(const ScanArgs& a, bool fp16, void* workspace, const uint32_t** flags,
                              hipStream_t stream);

// ---- chunks ------------------------------------------------------------------
//
// Sequences are cut into chunks of 64 tokens.  Sequence s has the chunk slots
// from min(starts[s] / c, starts[s] / 64 + s) on (rounded down), with c the fewest
// tokens of a sequence that goes in chunks, 32 at most: with n >= c tokens either
// number grows by ceil(n / 64) or more up to the next sequence, so that slots
// never meet, whatever the counts, and need no scan over the sequences.  Those of
// the tokens' end are enough for all: empty sequences and those that go token by
// token cost none where there are few tokens.
constexpr int kChunk = 64;

__host__ __device__ __forceinline__ int scan_slot_tokens(const ScanArgs& a) { return a.token_wise < 31 ? a.token_wise + 1 : 32; }
__device__ __forceinline__ int scan_first_chunk(const ScanArgs& a, int s) {
    return min(a.starts[s] / scan_slot_tokens(a), (a.starts[s] >> 6) + s);
}
__host__ __forceinline__ int scan_slots(const ScanArgs& a) {
    return std::max(std::min(a.tokens / scan_slot_tokens(a), a.tokens / kChunk + a.seqs), 1);
}

// Fragments of 16 bytes per lane, as the matrix instructions' A operands.  The
// tokens of a chunk, where they are summed over, come in this order: step ks
// (of 32), lane group g (of 16 lanes), element j: token 32 ks + 4 g + j for
// j < 4, 32 ks + 16 + 4 g + j - 4 from there on: what a lane of the waves 2 ks
// and 2 ks + 1 holds of a product's rows.  Of a lower triangular 64 x 64 matrix
// the blocks (ks, row tile w) with 2 ks <= w are kept, of an upper one those
// with 2 ks + 1 >= w: six each.
constexpr int kBlocks = 6;
constexpr int kFragBytes = 1024;
__host__ __device__ __forceinline__ constexpr int lower_block(int ks, int w) { return ks == 0 ? w : 2 + w; }
__host__ __device__ __forceinline__ constexpr int upper_block(int ks, int w) { return ks == 1 ? w : 4 + w; }

constexpr int kVec = 4 * kChunk + 64;   // (whole cache lines)

// What the first launch leaves the second, per chunk slot and value head (or
// key head), in this order in the workspace.
struct ScanChunks {
    int slots, parts;      // parts: bf16 numbers that a q or k is (1, or 2 for fp16)
    uint8_t *t, *p;        // [slots][heads]: 3 parts of 6 blocks
    float* vec;            // [slots][heads][kVec]: factors of K S, of Q S, of K^T U and beta per token, then the chunk's decay
    uint8_t *kt, *qt;      // [slots][key_heads][dim / 16][2][parts]: K^T, and for the gradient Q^T
    uint8_t *kf, *qf;      // [slots][key_heads][4][dim / 32][parts]: rows of K, and for the outputs of Q
    uint32_t* flags;       // [seqs][heads][value_dim / 16]
    // For the gradient: t and p hold the transposed matrices, and
    double* sums;          // [slots][heads][64]: running sums of g
    float* norms;          // [slots][key_heads][128]: factors of k and of q
    float *ds, *du;        // [slots][heads][dim][value_dim], [slots][heads][64][value_dim]
    f32x4* pairs;          // [slots][key_heads][4][512]: q . k and k . k, by threads
};

// The tape, fp32: states [slots][heads][dim][value_dim], then w [slots][heads][64]
// [value_dim] (u = beta w).
__host__ __device__ __forceinline__ int64_t tape_states(int64_t slots, int heads, int dim, int value_dim) {
    return slots * heads * dim * value_dim;
}

// An fp32 number as the sum of bf16 ones, each the rest rounded to nearest: two
// hold an fp16 number, three all of fp32's 24 bits.
struct Split2 {
    uint32_t part[3];   // pairs
};
template <int PARTS>
__device__ __forceinline__ Split2 split2(float lo, float hi) {
    Split2 s;
    s.part[0] = pack_bf2(lo, hi);
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
        lo -= lo_bf(s.part[p - 1]), hi -= hi_bf(s.part[p - 1]);
        s.part[p] = pack_bf2(lo, hi);
    }
    return s;
}

// Tokens of a sequence: [a, b), empty where starts do not lie in order within
// [0, tokens].
struct ScanSeq {
    int a, n;
};
__device__ __forceinline__ ScanSeq scan_seq(const int32_t* starts, int s, int tokens) {
    const int a = starts[s], b = starts[s + 1];
    const bool ok = a >= 0 && b >= a && b <= tokens;
    return {ok ? a : 0, ok ? b - a : 0};
}

// The state slots that sequence s reads and writes: -1 for none (a start from
// zero; a slot outside the pool, whose sequence is left out by the caller).
__device__ __forceinline__ int scan_slot(const int32_t* slots, int s, int pool) {
    const int slot = slots != nullptr ? slots[s] : s;
    return slot >= 0 && slot < pool ? slot : -1;
}

// exp of a log decay.  Below -104 the factor is 0 in fp32 (2^-150); the bound
// keeps running sums of -inf apart from NaN.
__device__ __forceinline__ float scan_log(float g) { return g < -104.0f ? -104.0f : g; }

// Sum over lanes l, l ^ 8, l ^ 16, l ^ 32 (a row rotation by 8, then the swaps
// of lane halves).
__device__ __forceinline__ float sum_over_8(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
    v = butterfly_step16(v);
    return butterfly_step32(v);
}

}  // namespace lrmoe
