// Attention of a step's new positions over a paged key/value cache.  Row t of
// sequence b (n_b new positions, kv_b cached ones with them) sees positions
// 0 .. kv_b - n_b + t: out = sum_p softmax(q . k_p scale)_p v_p, times
// sigmoid(gate) when a gate is given.
#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __builtin_exp2f(-1.4426950408889634f * x)); }

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The sequence that holds token t of starts[0 .. seqs], or -1.
__device__ __forceinline__ int sequence_of(const int32_t* starts, int seqs, int t) {
    if (t < starts[0] || t >= starts[seqs]) return -1;
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// One wave per (token, head): a lane per position for the scores (64 at a
// time), a lane per D / 64 elements for the values, softmax statistics and
// accumulators in fp32.  Positions that the row does not see are never read.
template <bool FP16, int D>
__global__ __launch_bounds__(kThreads) void attend_row_kernel(PagedAttnArgs a) {
    constexpr int WAVES = kThreads / kWave;
    constexpr int E = D / kWave;
    __shared__ float qs[WAVES][D];
    __shared__ float ps[WAVES][kWave];
    __shared__ int64_t vs[WAVES][kWave];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * WAVES + wave;
    if (item >= static_cast<int64_t>(a.tokens) * a.heads) return;
    const int t = static_cast<int>(item / a.heads), h = static_cast<int>(item % a.heads);
    const int b = sequence_of(a.starts, a.seqs, t);
    if (b < 0) return;
    const int n = a.starts[b + 1] - a.starts[b];
    const int64_t capacity = static_cast<int64_t>(a.max_pages) << a.page_shift;
    const int64_t kv = min(static_cast<int64_t>(max(a.kv_lengths[b], 0)), capacity);
    const int64_t seen = kv - n + (t - a.starts[b]) + 1;
    const uint16_t* q = a.q + t * a.q_token_stride + h * a.q_head_stride;
    const int64_t kh = static_cast<int64_t>(h / a.group);
    // LDS rows here belong to one wave, whose accesses stay in order; the
    // barriers below only keep the compiler from moving them.
    for (int e = lane; e < D; e += kWave) qs[wave][e] = elem16<FP16>(q[e]) * a.scale;
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.max_pages;
    float m = -__builtin_inff(), l = 0.0f, acc[E] = {};
    bool bad = false;
    wave_lds_fence();
    for (int64_t base = 0; base < seen; base += kWave) {
        const int64_t p = base + lane;
        float s = -__builtin_inff();
        if (p < seen) {
            int64_t block = table[p >> a.page_shift];
            bad |= block < 0 || block >= a.pages;
            block = min(max(block, static_cast<int64_t>(0)), static_cast<int64_t>(a.pages) - 1);
            const int64_t row = p & ((1 << a.page_shift) - 1);
            const uint16_t* k = a.k_cache + block * a.k_page_stride + kh * a.k_head_stride + row * a.k_row_stride;
            vs[wave][lane] = block * a.v_page_stride + kh * a.v_head_stride + row * a.v_row_stride;
            s = 0.0f;
            for (int e = 0; e < D; e += 8) {
                float x[8];
                unpack16<FP16>(ldg16(k + e), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) s = __builtin_fmaf(x[j], qs[wave][e + j], s);
            }
        }
        float top = s;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) {
            const float o = __shfl_xor(top, off);
            top = top != top ? top : (o > top || o != o ? o : top);  // a NaN score stays
        }
        const float mn = top > m || top != top ? top : m;
        const float shift = mn == -__builtin_inff() ? 0.0f : mn;
        const float w = p < seen ? __builtin_exp2f(s - shift) : 0.0f;
        const float fall = __builtin_exp2f(m - shift);
        float sum = w;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) sum += __shfl_xor(sum, off);
        l = l * fall + sum;
        m = mn;
        ps[wave][lane] = w;
        wave_lds_fence();
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] *= fall;
        const int count = static_cast<int>(min(static_cast<int64_t>(kWave), seen - base));
        for (int j = 0; j < count; ++j) {
            const uint16_t* v = a.v_cache + vs[wave][j] + lane * E;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] = __builtin_fmaf(ps[wave][j], elem16<FP16>(v[i]), acc[i]);
        }
        wave_lds_fence();
    }
    const bool nan = __any(bad);
    uint16_t* out = a.out + t * a.out_token_stride + h * a.out_head_stride + lane * E;
    const uint16_t* gate = a.gate + t * a.gate_token_stride + h * a.gate_head_stride + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float o = l == 0.0f ? 0.0f : acc[i] / l;
        if (nan) o = __builtin_nanf("");
        if (a.gate != nullptr) o *= sigmoid(elem16<FP16>(gate[i]));
        out[i] = static_cast<uint16_t>(FP16 ? f_to_f16(o) : f2bf(o));
    }
}

}  // namespace

size_t paged_attn_workspace_bytes(int, int, int, int, int, int) { return 0; }

hipError_t launch_paged_attention(const PagedAttnArgs& a, bool fp16, int dim, int, void*, hipStream_t stream) {
    const int64_t items = static_cast<int64_t>(a.tokens) * a.heads;
    const dim3 grid(static_cast<unsigned>((items + 3) / 4));
#define LR_ROW(F, N) hipLaunchKernelGGL((attend_row_kernel<F, N>), grid, dim3(kThreads), 0, stream, a)
    if (dim == 64) { if (fp16) LR_ROW(true, 64); else LR_ROW(false, 64); }
    else if (dim == 128) { if (fp16) LR_ROW(true, 128); else LR_ROW(false, 128); }
    else { if (fp16) LR_ROW(true, 256); else LR_ROW(false, 256); }
#undef LR_ROW
    return hipGetLastError();
}

}  // namespace lrmoe
