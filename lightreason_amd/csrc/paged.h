// Arguments and element helpers of the paged-cache kernels (paged.hip,
// paged_attention.hip) and of the draft verification (verify.hip).
#pragma once

#include "lrmoe_device.h"

namespace lrmoe {

constexpr int kPageMaxRows = LRMOE_PAGE_MAX_ROWS;
constexpr int kPageStatusTokens = LRMOE_PAGE_STATUS_TOKENS;
constexpr int kPageStatusRow = LRMOE_PAGE_STATUS_ROW;
constexpr int kPageStatusPool = LRMOE_PAGE_STATUS_POOL;
constexpr int kPageStatusStale = LRMOE_PAGE_STATUS_STALE;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float f16_to_f(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}
__device__ __forceinline__ uint32_t f_to_f16(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Eight 16-bit floats (bf16, or fp16) of a 16-byte word to and from fp32.
template <bool FP16>
__device__ __forceinline__ void unpack16(uint4 w, float* x) {
    if constexpr (FP16) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = f16_to_f(v[i] & 0xffffu);
            x[2 * i + 1] = f16_to_f(v[i] >> 16);
        }
    } else {
        unpack8(w, x);
    }
}
template <bool FP16>
__device__ __forceinline__ uint32_t pack16_2(float lo, float hi) {
    if constexpr (FP16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, f16x2));
    }
    return pack_bf2(lo, hi);
}
template <bool FP16>
__device__ __forceinline__ uint4 pack16(const float* x) {
    return make_uint4(pack16_2<FP16>(x[0], x[1]), pack16_2<FP16>(x[2], x[3]), pack16_2<FP16>(x[4], x[5]),
                      pack16_2<FP16>(x[6], x[7]));
}
template <bool FP16>
__device__ __forceinline__ float elem16(uint16_t bits) {
    if constexpr (FP16) return f16_to_f(bits);
    return bf2f(bits);
}

// Inclusive sum over the lanes (DPP row shifts, then row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

struct PagePlanArgs {
    int rows, pages, page_shift, max_pages, tokens;
    const int32_t *new_tokens, *lengths, *held, *free_pages;
    int32_t *state, *table, *starts, *kv_lengths, *held_out, *positions, *info;
    int64_t* slots;
};
hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t stream);

struct PageCommitArgs {
    int rows;
    const int32_t *starts, *kv_lengths, *held_new, *info, *accepted, *block_starts;
    int32_t *lengths, *held, *state;
};
hipError_t launch_page_commit(const PageCommitArgs& a, hipStream_t stream);

struct PageReleaseArgs {
    int rows, pages, max_pages;
    const uint8_t* mask;
    const int32_t* table;
    int32_t *lengths, *held, *free_pages, *state;
};
hipError_t launch_page_release(const PageReleaseArgs& a, hipStream_t stream);

struct PagedAppendArgs {
    int tokens, heads, kv_heads, rotary, pages, page_shift, rope_rows, rope_fp32;
    float eps;
    const uint16_t *q, *k, *v, *q_norm, *k_norm;
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    uint16_t *q_out, *k_cache, *v_cache;
    int64_t k_page_stride, k_cache_head_stride, k_row_stride, v_page_stride, v_cache_head_stride, v_row_stride;
    const void *cos, *sin;
    const int32_t* positions;
    const int64_t* slots;
};
hipError_t launch_paged_append(const PagedAppendArgs& a, bool fp16, int dim, hipStream_t stream);

struct PagedAttnArgs {
    int seqs, tokens, heads, kv_heads, group, pages, page_shift, max_pages;
    int group_inverse;  // ceil(2^21 / group)
    float scale;  // of the scores, times log2(e): the softmax runs on powers of two
    const uint16_t *q, *gate, *k_cache, *v_cache;
    int64_t q_token_stride, q_head_stride, gate_token_stride, gate_head_stride;
    int64_t k_page_stride, k_head_stride, k_row_stride, v_page_stride, v_head_stride, v_row_stride;
    const int32_t *table, *starts, *kv_lengths;
    uint16_t* out;
    int64_t out_token_stride, out_head_stride;
};
hipError_t launch_paged_attention(const PagedAttnArgs& a, bool fp16, int dim, int max_new, void* workspace,
                                  hipStream_t stream);
size_t paged_attn_workspace_bytes(int tokens, int seqs, int heads, int kv_heads, int dim, int max_new,
                                  int64_t capacity);

struct VerifyArgs {
    int seqs, rows, vocab;
    const int64_t* tokens;
    const void *target, *draft;
    int64_t target_stride, draft_stride;
    const int32_t* starts;
    const float *uniforms, *samples;
    int32_t* accepted;
    int64_t* next;
    double* sums;  // scratch: a block's outcome, then the chunks' sums
};
hipError_t launch_verify_drafts(const VerifyArgs& a, int type, hipStream_t stream);
size_t verify_workspace_bytes(int seqs, int vocab);

}  // namespace lrmoe
