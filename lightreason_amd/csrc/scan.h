// Arguments and shared pieces of the gated delta rule over packed sequences
// (scan.hip: forward; scan_grad.hip: gradient).
#pragma once

#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {

struct ScanArgs {
    int seqs, tokens, heads, key_heads, group, dim, value_dim, pool;
    int normalize, beta_fp32, clear;
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
};
hipError_t launch_delta_scan(const ScanArgs& a, bool fp16, int max_new, void* workspace, hipStream_t stream);
size_t delta_scan_workspace_bytes(const ScanArgs& a, bool fp16, int max_new);

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
