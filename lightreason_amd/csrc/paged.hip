// The page plan of a serving step over a paged key/value cache, its commit
// and the release of finished rows, and the append of a step's normed and
// rotated keys and values into their slots.
//
// The plan is integer work on a few kilobytes: what bounds it is latency
// (one launch, two dependent round trips to memory).  Every workgroup scans
// the per-row counts itself (4096 rows are 16 per thread) instead of handing
// the scan on through memory, so one launch does the whole plan and no
// workgroup waits for another.  The plan changes nothing of the pool: it
// writes its own outputs and table entries past the rows' held pages, which
// nobody reads before the commit.
#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;

// Inclusive scan over the wave's lanes.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const int64_t up = __shfl_up(v, off);
        if (static_cast<int>(__lane_id()) >= off) v += up;
    }
    return v;
}

// Exclusive prefix of v over the workgroup's threads; *total gets the sum.
template <int WAVES>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int64_t* total) {
    const int wave = threadIdx.x / kWave;
    const int64_t inc = wave_scan(v);
    if (__lane_id() == kWave - 1) lds[wave] = inc;
    __syncthreads();
    int64_t base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) base += lds[w];
        sum += lds[w];
    }
    __syncthreads();
    *total = sum;
    return base + inc - v;
}

// Largest r with from[r] <= x, for from ascending and from[0] <= x.
__device__ __forceinline__ int last_at_most(const int* from, int n, int x) {
    int lo = 0, hi = n;  // from[lo] <= x; from[hi] > x or hi == n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (from[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void page_plan_kernel(PagePlanArgs a) {
    __shared__ int starts[kPageMaxRows + 1];
    __shared__ int before[kPageMaxRows];
    __shared__ int64_t scratch[kThreads / kWave];
    __shared__ int status;
    const int tid = threadIdx.x;
    const int per = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    const int page = 1 << a.page_shift;
    const int64_t row_limit = static_cast<int64_t>(a.max_pages) << a.page_shift;
    if (tid == 0) status = 0;
    const int count = a.state[0];
    const int epoch = a.state[1];
    int bad = 0;
    int64_t tokens = 0, fresh = 0;
    for (int r = r0; r < r1; ++r) {
        const int64_t n = a.new_tokens[r], len = a.lengths[r], held = a.held[r];
        if (n < 0) bad |= kPageStatusTokens;
        if (len < 0 || held < 0 || held > a.max_pages || len + n > row_limit) bad |= kPageStatusRow;
        const int64_t need = (len + n + page - 1) >> a.page_shift;
        tokens += n;
        fresh += need > held ? need - held : 0;
    }
    __syncthreads();
    if (bad) atomicOr(&status, bad);
    int64_t total_tokens, total_fresh;
    int64_t at = block_scan<kThreads / kWave>(tokens, scratch, &total_tokens);
    int64_t fat = block_scan<kThreads / kWave>(fresh, scratch, &total_fresh);
    // (block_scan's barriers also publish `status`)
    int refuse = status;
    if (total_tokens > a.tokens) refuse |= kPageStatusTokens;
    if (total_fresh > count || count > a.pages) refuse |= kPageStatusPool;
    const bool ok = refuse == 0;
    for (int r = r0; r < r1; ++r) {
        const int n = ok ? a.new_tokens[r] : 0, len = a.lengths[r], held = a.held[r];
        const int need = ok ? static_cast<int>((static_cast<int64_t>(len) + n + page - 1) >> a.page_shift) : 0;
        starts[r] = ok ? static_cast<int>(at) : 0;
        before[r] = ok ? static_cast<int>(fat) : 0;
        at += n;
        fat += need > held ? need - held : 0;
        if (blockIdx.x == 0) {
            a.starts[r] = starts[r];
            a.kv_lengths[r] = len + n;
            a.held_out[r] = need > held ? need : held;
        }
    }
    const int live = ok ? static_cast<int>(total_tokens) : 0;
    const int taken = ok ? static_cast<int>(total_fresh) : 0;
    if (tid == 0) {
        starts[a.rows] = live;
        if (blockIdx.x == 0) {
            a.starts[a.rows] = live;
            a.info[0] = refuse;
            a.info[1] = live;
            a.info[2] = taken;
            a.info[3] = epoch;
        }
    }
    __syncthreads();
    const int first = blockIdx.x * kThreads + tid, step = gridDim.x * kThreads;
    for (int i = first; i < a.tokens; i += step) {
        int position = 0;
        int64_t slot = -1;
        if (i < live) {
            const int r = last_at_most(starts, a.rows, i);
            position = a.lengths[r] + i - starts[r];
            const int p = position >> a.page_shift, held = a.held[r];
            const int entry = p < held ? a.table[static_cast<int64_t>(r) * a.max_pages + p]
                                       : a.free_pages[count - 1 - (before[r] + p - held)];
            slot = (static_cast<int64_t>(entry) << a.page_shift) + (position & (page - 1));
        }
        a.positions[i] = position;
        a.slots[i] = slot;
    }
    for (int j = first; j < taken; j += step) {
        const int r = last_at_most(before, a.rows, j);
        a.table[static_cast<int64_t>(r) * a.max_pages + a.held[r] + j - before[r]] = a.free_pages[count - 1 - j];
    }
}

__global__ __launch_bounds__(kThreads) void page_commit_kernel(PageCommitArgs a) {
    const int refuse = a.info[0] | (a.info[3] != a.state[1] ? kPageStatusStale : 0);
    const int count = a.state[0], epoch = a.state[1], status = a.state[2];
    __syncthreads();  // every thread has read the state that thread 0 changes
    if (refuse == 0) {
        for (int r = threadIdx.x; r < a.rows; r += kThreads) {
            const int n = a.starts[r + 1] - a.starts[r];
            if (a.accepted == nullptr) {
                a.lengths[r] = a.kv_lengths[r];
            } else if (n > 0) {
                a.lengths[r] += min(max(a.accepted[r], 0) + 1, n);
            }
            a.held[r] = a.held_new[r];
        }
    }
    if (threadIdx.x == 0) {
        if (refuse == 0) {
            a.state[0] = count - a.info[2];
            a.state[1] = epoch + 1;
        }
        a.state[2] = status | refuse;
    }
}

__global__ __launch_bounds__(kThreads) void page_release_kernel(PageReleaseArgs a) {
    __shared__ int before[kPageMaxRows];
    __shared__ int64_t scratch[kThreads / kWave];
    const int tid = threadIdx.x;
    const int per = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    const int count = a.state[0];
    int64_t mine = 0, total;
    for (int r = r0; r < r1; ++r) mine += a.mask[r] ? min(max(a.held[r], 0), a.max_pages) : 0;
    int64_t at = block_scan<kThreads / kWave>(mine, scratch, &total);
    const bool ok = count >= 0 && count + total <= a.pages;
    for (int r = r0; r < r1; ++r) {
        before[r] = static_cast<int>(at);
        at += a.mask[r] ? min(max(a.held[r], 0), a.max_pages) : 0;
    }
    __syncthreads();
    if (ok) {
        for (int j = tid; j < total; j += kThreads) {
            const int r = last_at_most(before, a.rows, j);
            a.free_pages[count + j] = a.table[static_cast<int64_t>(r) * a.max_pages + j - before[r]];
        }
        __syncthreads();
        for (int r = r0; r < r1; ++r) {
            if (!a.mask[r]) continue;
            a.held[r] = 0;
            a.lengths[r] = 0;
        }
    }
    if (tid == 0) {
        if (ok) {
            a.state[0] = count + static_cast<int>(total);
            a.state[1] += 1;
        } else {
            a.state[2] |= kPageStatusPool;
        }
    }
}

// ---- append ------------------------------------------------------------------

// One group of D / 8 lanes per head row (query, key or value), 16 bytes per
// lane: y = x / sqrt(mean(x^2) + eps) (1 + w) and the rotation of the first
// `rotary` elements (element e of the first half with e + rotary / 2) in
// fp32, one rounding to the tensor's type at the end.  A pass over the data:
// each row is read once and written once; what bounds it is HBM bandwidth.
template <bool FP16, int D>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int LANES = D / 8;
    const int64_t group = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LANES;
    const int l = threadIdx.x % LANES;
    const int rows = a.heads + 2 * a.kv_heads;
    const int64_t t = group / rows;
    if (t >= a.tokens) return;
    int h = static_cast<int>(group - t * rows);
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= (static_cast<int64_t>(a.pages) << a.page_shift)) return;
    const int64_t block = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    if (h >= a.heads + a.kv_heads) {
        h -= a.heads + a.kv_heads;
        const uint4 v = ldg16(a.v + t * a.v_token_stride + h * a.v_head_stride + 8 * l);
        *reinterpret_cast<uint4*>(a.v_cache + block * a.v_page_stride + h * a.v_cache_head_stride +
                                  row * a.v_row_stride + 8 * l) = v;
        return;
    }
    const uint16_t *src, *weight;
    uint16_t* dst;
    if (h < a.heads) {
        src = a.q + t * a.q_token_stride + h * a.q_head_stride;
        weight = a.q_norm;
        dst = a.q_out + (t * a.heads + h) * D;
    } else {
        h -= a.heads;
        src = a.k + t * a.k_token_stride + h * a.k_head_stride;
        weight = a.k_norm;
        dst = a.k_cache + block * a.k_page_stride + h * a.k_cache_head_stride + row * a.k_row_stride;
    }
    float x[8];
    unpack16<FP16>(ldg16(src + 8 * l), x);
    if (weight != nullptr) {
        float w[8];
        unpack16<FP16>(ldg16(weight + 8 * l), w);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
#pragma unroll
        for (int off = 1; off < LANES; off *= 2) sum += __shfl_xor(sum, off);
        const float scale = 1.0f / __builtin_sqrtf(sum / static_cast<float>(D) + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (x[j] * scale) * (1.0f + w[j]);
    }
    if (a.rotary > 0) {
        const int half = a.rotary / 16;  // lanes per half of the rotated elements
        float other[8];
        const int partner = l < half ? l + half : l - half;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            other[j] = __shfl(x[j], static_cast<int>(__lane_id()) - l + (l < 2 * half ? partner : l));
        if (l < 2 * half) {
            const int64_t p = a.positions != nullptr ? a.positions[t] : t;
            float c[8], s[8];
            if (p < 0 || p >= a.rope_rows) {  // no such row: the rotated elements are NaN
#pragma unroll
                for (int j = 0; j < 8; ++j) c[j] = s[j] = __builtin_nanf("");
            } else if (a.rope_fp32) {
                const float* cr = static_cast<const float*>(a.cos) + p * a.rotary + 8 * l;
                const float* sr = static_cast<const float*>(a.sin) + p * a.rotary + 8 * l;
#pragma unroll
                for (int j = 0; j < 8; ++j) { c[j] = cr[j]; s[j] = sr[j]; }
            } else {
                unpack16<FP16>(ldg16(static_cast<const uint16_t*>(a.cos) + p * a.rotary + 8 * l), c);
                unpack16<FP16>(ldg16(static_cast<const uint16_t*>(a.sin) + p * a.rotary + 8 * l), s);
            }
            const float sign = l < half ? -1.0f : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * c[j] + sign * other[j] * s[j];
        }
    }
    *reinterpret_cast<uint4*>(dst + 8 * l) = pack16<FP16>(x);
}

}  // namespace

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t stream) {
    // One position per thread up to 256 workgroups; at least enough threads
    // that a step of few positions still spreads its rows' fresh pages.
    const int blocks = min(256, max(1, (a.tokens + kThreads - 1) / kThreads));
    hipLaunchKernelGGL(page_plan_kernel, dim3(blocks), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_page_commit(const PageCommitArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(page_commit_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_page_release(const PageReleaseArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, bool fp16, int dim, hipStream_t stream) {
    const int64_t lanes = static_cast<int64_t>(a.tokens) * (a.heads + 2 * a.kv_heads) * (dim / 8);
    const dim3 grid(static_cast<unsigned>((lanes + kThreads - 1) / kThreads));
#define LR_APPEND(F, N) hipLaunchKernelGGL((paged_append_kernel<F, N>), grid, dim3(kThreads), 0, stream, a)
    if (dim == 64) { if (fp16) LR_APPEND(true, 64); else LR_APPEND(false, 64); }
    else if (dim == 128) { if (fp16) LR_APPEND(true, 128); else LR_APPEND(false, 128); }
    else { if (fp16) LR_APPEND(true, 256); else LR_APPEND(false, 256); }
#undef LR_APPEND
    return hipGetLastError();
}

}  // namespace lrmoe
