// Verification of drafted tokens.  A block's rows i = 0 .. n - 1 hold the
// target's probabilities p_i of the position after fed token i; the token fed
// at row i + 1 is draft i, drawn from q_i.  Draft i stands while
// u_i q_i(x_i) < p_i(x_i); at the first that fails the next token is drawn
// from max(p_i - q_i, 0), and from p at the last row when all stand.  Drawn by
// inverse distribution: the first token whose running sum of mass passes
// sample * total.
//
// A token of a vocabulary of hundreds of thousands carries about 2^-17 of the
// mass, so running sums in fp32 (2^-24 a step) would move draws by a token
// now and then: sums are held in 64 bits, in one fixed order.  What bounds it
// is reading one probability row per side and block (HBM, or latency for a
// single block): launch one sums chunks of the row over many workgroups,
// launch two finds the chunk and rereads that chunk only.
#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // elements per workgroup of the summing launch

// Element types of the probabilities: 0 fp32, 1 bf16, 2 fp16.
template <int TYPE>
__device__ __forceinline__ float prob_at(const void* base, int64_t i) {
    if constexpr (TYPE == 0) return static_cast<const float*>(base)[i];
    return elem16<TYPE == 2>(static_cast<const uint16_t*>(base)[i]);
}

// A positive finite value, or 0: an entry that is negative, infinite or NaN
// carries no mass.
__device__ __forceinline__ double mass_of(double x) { return x > 0.0 && x <= 3.5e38 ? x : 0.0; }

struct Block {
    int first, n, stop;  // rows first .. first + n - 1; the row whose distribution is drawn from
};

// Drafts of block b tested by all threads, a round of kThreads at a time;
// n = 0 for a block without rows.
template <int TYPE>
__device__ __forceinline__ Block examine(const VerifyArgs& a, int b, int* lds) {
    Block blk;
    blk.first = a.starts[b];
    const int end = a.starts[b + 1];
    blk.n = blk.first >= 0 && end <= a.rows && end > blk.first ? end - blk.first : 0;
    blk.stop = blk.n - 1;
    for (int base = 0; base < blk.n - 1; base += kThreads) {
        if (threadIdx.x == 0) *lds = blk.n;
        __syncthreads();
        const int i = base + threadIdx.x;
        if (i < blk.n - 1) {
            const int64_t row = blk.first + i;
            const int64_t x = a.tokens[row + 1];
            bool ok = false;
            if (x >= 0 && x < a.vocab) {
                const double p = prob_at<TYPE>(a.target, row * a.target_stride + x);
                const double q = a.draft ? prob_at<TYPE>(a.draft, row * a.draft_stride + x) : 1.0;
                ok = static_cast<double>(a.uniforms[row]) * q < p;
            }
            if (!ok) atomicMin(lds, i);
        }
        __syncthreads();
        const int fail = *lds;
        __syncthreads();
        if (fail < blk.n - 1) {
            blk.stop = fail;
            break;
        }
    }
    return blk;
}

// What a token's mass is made of at the row that is drawn from.
struct Row {
    int64_t p, q;    // element offsets of the rows
    int64_t dropped; // the rejected token when there are no draft probabilities, else -1
    bool rejected;
};
__device__ __forceinline__ Row row_of(const VerifyArgs& a, const Block& blk) {
    Row r;
    const int64_t row = blk.first + blk.stop;
    r.rejected = blk.stop < blk.n - 1;
    r.p = row * a.target_stride;
    r.q = row * a.draft_stride;
    r.dropped = r.rejected && a.draft == nullptr ? a.tokens[row + 1] : -1;
    return r;
}
template <int TYPE>
__device__ __forceinline__ void masses(const VerifyArgs& a, const Row& r, int v, double* whole, double* rest) {
    const double p = prob_at<TYPE>(a.target, r.p + v);
    *whole = mass_of(p);
    if (!r.rejected) *rest = *whole;
    else if (a.draft != nullptr) *rest = mass_of(p - static_cast<double>(prob_at<TYPE>(a.draft, r.q + v)));
    else *rest = v == r.dropped ? 0.0 : *whole;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) v += __shfl_xor(v, off);
    if (__lane_id() == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    const double sum = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    __syncthreads();
    return sum;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs a, int chunks) {
    __shared__ int fail;
    __shared__ double sums[kThreads / kWave];
    const int b = blockIdx.y, c = blockIdx.x;
    const Block blk = examine<TYPE>(a, b, &fail);
    if (blk.n == 0) return;
    const Row row = row_of(a, blk);
    double whole = 0.0, rest = 0.0;
    for (int k = 0; k < kChunk / kThreads; ++k) {
        const int64_t v = static_cast<int64_t>(c) * kChunk + k * kThreads + threadIdx.x;
        if (v < a.vocab) {
            double w, r;
            masses<TYPE>(a, row, static_cast<int>(v), &w, &r);
            whole += w;
            rest += r;
        }
    }
    whole = block_sum(whole, sums);
    rest = block_sum(rest, sums);
    if (threadIdx.x == 0) {
        double* out = a.sums + 2 * (static_cast<int64_t>(b) * chunks + c);
        out[0] = rest;
        out[1] = whole;
    }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a, int chunks) {
    __shared__ int fail;
    __shared__ double partial[kThreads];
    __shared__ int picked;
    __shared__ double below;
    const int b = blockIdx.x, tid = threadIdx.x;
    const Block blk = examine<TYPE>(a, b, &fail);
    if (blk.n == 0) {
        if (tid == 0) {
            a.accepted[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    const Row row = row_of(a, blk);
    const double* sums = a.sums + 2 * static_cast<int64_t>(b) * chunks;
    // Which of the two masses, and its total.
    double total = 0.0, all = 0.0;
    for (int c = 0; c < chunks; ++c) {
        total += sums[2 * c];
        all += sums[2 * c + 1];
    }
    const int which = total > 0.0 ? 0 : 1;
    if (which == 1) total = all;
    const float sample = a.samples[b];
    const double border = (sample > 0.0f ? static_cast<double>(sample) : 0.0) * total;
    if (tid == 0) {
        a.accepted[b] = blk.stop;
        // The chunk in which the running sum passes the border, else the last
        // one that has mass.
        int at = -1;
        double run = 0.0, before = 0.0;
        for (int c = 0; c < chunks; ++c) {
            const double s = sums[2 * c + which];
            if (s > 0.0) {
                at = c;
                before = run;
                if (run + s > border) break;
            }
            run += s;
        }
        picked = at;
        below = before;
        if (at < 0) a.next[b] = -1;
    }
    __syncthreads();
    if (picked < 0) return;
    constexpr int PER = kChunk / kThreads;
    const int64_t v0 = static_cast<int64_t>(picked) * kChunk + tid * PER;
    double mine = 0.0;
    for (int k = 0; k < PER && v0 + k < a.vocab; ++k) {
        double w, r;
        masses<TYPE>(a, row, static_cast<int>(v0 + k), &w, &r);
        mine += which ? w : r;
    }
    partial[tid] = mine;
    __syncthreads();
    if (tid == 0) {
        double run = below;
        int at = -1;
        double before = 0.0;
        for (int t = 0; t < kThreads; ++t) {
            if (partial[t] > 0.0) {
                at = t;
                before = run;
                if (run + partial[t] > border) break;
            }
            run += partial[t];
        }
        fail = at;
        below = before;
    }
    __syncthreads();
    if (tid == fail) {
        double run = below;
        int64_t token = -1;
        for (int k = 0; k < PER && v0 + k < a.vocab; ++k) {
            double w, r;
            masses<TYPE>(a, row, static_cast<int>(v0 + k), &w, &r);
            const double m = which ? w : r;
            if (m > 0.0) {
                token = v0 + k;
                run += m;
                if (run > border) break;
            }
        }
        a.next[b] = token;
    }
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

size_t verify_workspace_bytes(int seqs, int vocab) {
    return static_cast<size_t>(seqs) * chunks_of(vocab) * 2 * sizeof(double);
}

hipError_t launch_verify_drafts(const VerifyArgs& a, int type, hipStream_t stream) {
    const int chunks = chunks_of(a.vocab);
    const dim3 grid(chunks, a.seqs);
#define LR_VERIFY(T)                                                                                             \
    do {                                                                                                         \
        hipLaunchKernelGGL((verify_sum_kernel<T>), grid, dim3(kThreads), 0, stream, a, chunks);                  \
        hipLaunchKernelGGL((verify_draw_kernel<T>), dim3(a.seqs), dim3(kThreads), 0, stream, a, chunks);         \
    } while (0)
    if (type == 0) LR_VERIFY(0);
    else if (type == 1) LR_VERIFY(1);
    else LR_VERIFY(2);
#undef LR_VERIFY
    return hipGetLastError();
}

}  // namespace lrmoe
