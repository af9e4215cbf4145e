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
// is reading one probability row per side and block from HBM, and for a few
// blocks the chain of dependent reads (starts, tokens, their probabilities,
// the row).  Launch one tests a block's drafts in every workgroup (a lane per
// draft, no barrier) and sums a chunk of the row that is drawn from; launch
// two finds the chunk from its sums and reads that chunk only.  Rows of
// 151,936 fp32 on both sides: one block of 5 takes 11.1 us, 64 blocks of up to
// 8 take 20.8, the first launch at 6 TB/s.
#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 4096;               // elements per workgroup of the summing launch
constexpr int kPer = kChunk / kThreads;    // 16 per thread

// Element types of the probabilities: 0 fp32, 1 bf16, 2 fp16.
template <int TYPE>
__device__ __forceinline__ float prob_at(const void* base, int64_t i) {
    if constexpr (TYPE == 0) return static_cast<const float*>(base)[i];
    return elem16<TYPE == 2>(static_cast<const uint16_t*>(base)[i]);
}

// N elements from i on (i + n of them within the row, the others 0): by 16
// bytes where the rows are aligned to them, else one by one.
template <int TYPE, bool VEC, int N>
__device__ __forceinline__ void probs_from(const void* base, int64_t i, int n, float (&x)[N]) {
    constexpr int W = TYPE == 0 ? 4 : 8;   // elements of 16 bytes
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < N; k += W) {
            if (k + W <= n) {
                const uint4 v = ldg16(static_cast<const uint8_t*>(base) + (i + k) * (TYPE == 0 ? 4 : 2));
                if constexpr (TYPE == 0) {
                    x[k] = __uint_as_float(v.x);
                    x[k + 1] = __uint_as_float(v.y);
                    x[k + 2] = __uint_as_float(v.z);
                    x[k + 3] = __uint_as_float(v.w);
                } else {
                    unpack16<TYPE == 2>(v, &x[k]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) x[k + j] = k + j < n ? prob_at<TYPE>(base, i + k + j) : 0.0f;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = k < n ? prob_at<TYPE>(base, i + k) : 0.0f;
    }
}

// A positive finite value, or 0: an entry that is negative, infinite or NaN
// carries no mass.
__device__ __forceinline__ double mass_of(double x) { return x > 0.0 && x <= 3.5e38 ? x : 0.0; }

struct Block {
    int first, n, stop;  // rows first .. first + n - 1; of them the one whose distribution is drawn from
};

// The drafts of block b, 64 at a time, by every wave for itself; n = 0 for a
// block without rows.
template <int TYPE>
__device__ __forceinline__ Block examine(const VerifyArgs& a, int b) {
    Block blk;
    blk.first = a.starts[b];
    const int end = a.starts[b + 1];
    blk.n = blk.first >= 0 && end <= a.rows && end > blk.first ? end - blk.first : 0;
    blk.stop = blk.n - 1;
    for (int base = 0; base < blk.n - 1; base += kWave) {
        const int i = base + threadIdx.x % kWave;
        bool fails = false;
        if (i < blk.n - 1) {
            const int64_t row = blk.first + i;
            const int64_t x = a.tokens[row + 1];
            const float u = a.uniforms[row];
            fails = true;
            if (x >= 0 && x < a.vocab) {
                const double p = prob_at<TYPE>(a.target, row * a.target_stride + x);
                const double q = a.draft ? prob_at<TYPE>(a.draft, row * a.draft_stride + x) : 1.0;
                fails = !(static_cast<double>(u) * q < p);
            }
        }
        const uint64_t who = __ballot(fails);
        if (who != 0) {
            blk.stop = base + __builtin_ctzll(who);
            break;
        }
    }
    return blk;
}

// What a token's mass is made of at the row that is drawn from: whole = p,
// rest = what is left of it after a rejection.
struct Row {
    int64_t p, q;     // element offsets of the rows
    int64_t dropped;  // the rejected token when there are no draft probabilities, else -1
    bool both;        // p - q
};
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int first, int n, int stop) {
    Row r;
    const int64_t row = first + stop;
    const bool rejected = stop < n - 1;
    r.p = row * a.target_stride;
    r.q = row * a.draft_stride;
    r.both = rejected && a.draft != nullptr;
    r.dropped = rejected && a.draft == nullptr ? a.tokens[row + 1] : -1;
    return r;
}
__device__ __forceinline__ double rest_of(const Row& r, int64_t v, float p, float q) {
    // (A token that the target gives no mass has none left, whatever q is.)
    if (r.both) return p > 0.0f ? mass_of(static_cast<double>(p) - static_cast<double>(q)) : 0.0;
    return v == r.dropped ? 0.0 : mass_of(p);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) v += __shfl_xor(v, off);
    return v;
}

// What launch one leaves of a block for launch two.
struct Found {
    int first, n, stop, pad;
};

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs a, int chunks) {
    __shared__ double sums[2][kWaves];
    const int b = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const Block blk = examine<TYPE>(a, b);
    if (c == 0 && tid == 0) {
        reinterpret_cast<Found*>(a.sums)[b] = {blk.first, blk.n, blk.stop, 0};
        a.accepted[b] = blk.n > 0 ? blk.stop : 0;
    }
    if (blk.n == 0) return;
    const Row row = row_of(a, blk.first, blk.n, blk.stop);
    constexpr int W = !VEC ? 1 : TYPE == 0 ? 4 : 8;   // elements per load
    double whole = 0.0, rest = 0.0;
    float p[kPer], q[kPer];
    const int64_t base = static_cast<int64_t>(c) * kChunk;
    // Thread t takes pieces t, t + 256, ... of W elements: all loads first.
#pragma unroll
    for (int k = 0; k < kPer / W; ++k) {
        const int64_t v = base + (k * kThreads + tid) * W;
        float x[W];
        probs_from<TYPE, VEC>(a.target, row.p + v, static_cast<int>(min(a.vocab - v, static_cast<int64_t>(W))), x);
#pragma unroll
        for (int j = 0; j < W; ++j) p[k * W + j] = x[j];
    }
    if (row.both) {
#pragma unroll
        for (int k = 0; k < kPer / W; ++k) {
            const int64_t v = base + (k * kThreads + tid) * W;
            float x[W];
            probs_from<TYPE, VEC>(a.draft, row.q + v, static_cast<int>(min(a.vocab - v, static_cast<int64_t>(W))), x);
#pragma unroll
            for (int j = 0; j < W; ++j) q[k * W + j] = x[j];
        }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int64_t v = base + (k / W * kThreads + tid) * W + k % W;
        whole += mass_of(p[k]);
        rest += rest_of(row, v, p[k], row.both ? q[k] : 0.0f);
    }
    whole = wave_sum(whole);
    rest = wave_sum(rest);
    if (tid % kWave == 0) {
        sums[0][tid / kWave] = rest;
        sums[1][tid / kWave] = whole;
    }
    __syncthreads();
    if (tid < 2) {
        const double* s = sums[tid];
        double* out = a.sums + 2 * a.seqs + 2 * (static_cast<int64_t>(b) * chunks + c);
        out[tid] = (s[0] + s[1]) + (s[2] + s[3]);
    }
}

// The first of the wave's lanes whose running sum passes `border`, from
// `*run` on, among those with mass, or, without one, the last lane with mass;
// -1 when no lane has any.  *before: the running sum in front of that lane;
// *run: after all lanes.  `passed` tells whether the border was passed.
__device__ __forceinline__ int first_past(double mass, double border, double* run, double* before, bool* passed) {
    double upto = mass;
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const double up = __shfl_up(upto, off);
        if (static_cast<int>(__lane_id()) >= off) upto += up;
    }
    upto += *run;
    const double front = upto - mass;
    const uint64_t has = __ballot(mass > 0.0), past = __ballot(mass > 0.0 && upto > border);
    *passed = past != 0;
    const int who = past != 0 ? __builtin_ctzll(past) : has != 0 ? 63 - __builtin_clzll(has) : -1;
    *before = __shfl(front, who < 0 ? 0 : who);
    *run = __shfl(upto, kWave - 1);
    return who;
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a, int chunks) {
    __shared__ double wave_mass[kWaves];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const Found f = reinterpret_cast<const Found*>(a.sums)[b];
    if (f.n == 0) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    const Row row = row_of(a, f.first, f.n, f.stop);
    const float sample = a.samples[b];
    // Every wave finds the chunk: totals of the two masses first.
    const double2* sums = reinterpret_cast<const double2*>(a.sums + 2 * a.seqs) + static_cast<int64_t>(b) * chunks;
    double rest = 0.0, whole = 0.0;
    for (int c = lane; c < chunks; c += kWave) {
        rest += sums[c].x;
        whole += sums[c].y;
    }
    rest = wave_sum(rest);
    whole = wave_sum(whole);
    const bool left = rest > 0.0;   // else p itself
    const double border = (sample > 0.0f ? static_cast<double>(sample) : 0.0) * (left ? rest : whole);
    int chunk = -1;
    double run = 0.0, below = 0.0;
    for (int base = 0; base < chunks; base += kWave) {
        const int c = base + lane;
        const double2 s = c < chunks ? sums[c] : make_double2(0.0, 0.0);
        double before;
        bool passed;
        const int who = first_past(left ? s.x : s.y, border, &run, &before, &passed);
        if (who >= 0) {
            chunk = base + who;
            below = before;
        }
        if (passed) break;
    }
    if (chunk < 0) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    // The chunk, 16 elements in order per thread.
    const int64_t v0 = static_cast<int64_t>(chunk) * kChunk + tid * kPer;
    const int n = static_cast<int>(max(min(a.vocab - v0, static_cast<int64_t>(kPer)), static_cast<int64_t>(0)));
    float p[kPer], q[kPer];
    probs_from<TYPE, VEC>(a.target, row.p + v0, n, p);
    const bool both = row.both && left;
    if (both) probs_from<TYPE, VEC>(a.draft, row.q + v0, n, q);
    double mine = 0.0, m[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        m[k] = k >= n ? 0.0 : left ? rest_of(row, v0 + k, p[k], both ? q[k] : 0.0f) : mass_of(p[k]);
        mine += m[k];
    }
    const double sum = wave_sum(mine);
    if (lane == 0) wave_mass[wave] = sum;
    __syncthreads();
    // The wave, then its thread, then its element: each the first past the
    // border, or the last with mass where rounding leaves none past it.
    int pick = -1;
    double front = below, at = below;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const double s = wave_mass[w];
        if (s > 0.0) {
            pick = w;
            front = at;
            if (at + s > border) break;
        }
        at += s;
    }
    if (pick < 0) {   // sums of a chunk with mass have mass again
        if (tid == 0) a.next[b] = -1;
        return;
    }
    if (wave != pick) return;
    double before;
    bool passed;
    run = front;
    const int who = first_past(mine, border, &run, &before, &passed);
    if (lane != who) return;
    int64_t token = -1;
    bool done = false;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        if (done || !(m[k] > 0.0)) continue;
        token = v0 + k;
        before += m[k];
        done = before > border;
    }
    a.next[b] = token;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

size_t verify_workspace_bytes(int seqs, int vocab) {
    return static_cast<size_t>(seqs) * (chunks_of(vocab) + 1) * 2 * sizeof(double);   // a Found and the sums
}

hipError_t launch_verify_drafts(const VerifyArgs& a, int type, hipStream_t stream) {
    const int chunks = chunks_of(a.vocab);
    const dim3 grid(chunks, a.seqs);
    // Rows that start at multiples of 16 bytes are read by 16 bytes.
    const int64_t bytes = type == 0 ? 4 : 2;
    auto aligned = [&](const void* p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0;
    };
    const bool vec = aligned(a.target, a.target_stride) && (a.draft == nullptr || aligned(a.draft, a.draft_stride));
#define LR_VERIFY(T, V)                                                                                          \
    do {                                                                                                         \
        hipLaunchKernelGGL((verify_sum_kernel<T, V>), grid, dim3(kThreads), 0, stream, a, chunks);               \
        hipLaunchKernelGGL((verify_draw_kernel<T, V>), dim3(a.seqs), dim3(kThreads), 0, stream, a, chunks);      \
    } while (0)
    if (type == 0) { if (vec) LR_VERIFY(0, true); else LR_VERIFY(0, false); }
    else if (type == 1) { if (vec) LR_VERIFY(1, true); else LR_VERIFY(1, false); }
    else { if (vec) LR_VERIFY(2, true); else LR_VERIFY(2, false); }
#undef LR_VERIFY
    return hipGetLastError();
}

}  // namespace lrmoe
