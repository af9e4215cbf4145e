// The page plan of a serving step over a paged key/value cache, its commit
// and the release of finished rows, and the append of a step's normed and
// rotated keys and values into their slots.
//
// The plan is integer work on a few kilobytes: what bounds it is latency (one
// launch, two dependent round trips to memory: 4-5 us for 4 rows, 6.4 for 1000
// rows of up to 65 new positions).  Every workgroup scans the per-row counts
// itself (4096 rows are 16 per thread) instead of handing the scan on through
// memory, so one launch does the whole plan and no workgroup waits for another.
// The plan changes nothing that rows hold: it writes its own outputs, its
// number, and table entries past the rows' held pages.  Those are read by the
// step's attention and kept by its commit, so only the plan that wrote them
// last can be committed.
//
// Commit and release run in one workgroup: a plan with its commit takes 4.4 us
// for 4 rows, 8 for 1000 and 29 for 4096; a release 2.4 us for 268 pages, 11
// for 4288, 218 for 67,000 (a page per thread at a time; rows end seldom).
#include <algorithm>

#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;

// Exclusive prefixes of two counts over the workgroup's threads, and their
// totals.  The counts may be anything (a caller's numbers): the totals are
// right while they are below 2^30, and `huge` tells when they are not.
struct Prefix {
    int a, b, total_a, total_b;
    bool huge;
};
struct PrefixLds {
    int a[kThreads / kWave], b[kThreads / kWave];
    float size[kThreads / kWave];
};
__device__ __forceinline__ Prefix block_prefix(int a, int b, float size, PrefixLds* lds) {
    const int wave = threadIdx.x / kWave;
    const int upto_a = wave_scan(a), upto_b = wave_scan(b);
    size = wave_butterfly_sum(size);
    if (__lane_id() == kWave - 1) {
        lds->a[wave] = upto_a;
        lds->b[wave] = upto_b;
        lds->size[wave] = size;
    }
    __syncthreads();
    Prefix p = {upto_a - a, upto_b - b, 0, 0, false};
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        if (w < wave) {
            p.a += lds->a[w];
            p.b += lds->b[w];
        }
        p.total_a += lds->a[w];
        p.total_b += lds->b[w];
        all += lds->size[w];
    }
    p.huge = !(all < 1073741824.0f);
    return p;
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

// The number of the made-th plan (from 1 on) between two changes of the pool.
// Two of them are equal only where the epochs' difference times the counts' is
// about 2^31 or more (the factor is 2^32 over the golden ratio, whose multiples
// keep apart).
__device__ __forceinline__ int plan_number(int epoch, int made) {
    return static_cast<int>(static_cast<uint32_t>(epoch) * 0x9e3779b1u + static_cast<uint32_t>(made));
}

__global__ __launch_bounds__(kThreads) void page_plan_kernel(PagePlanArgs a) {
    __shared__ int starts[kPageMaxRows + 1];
    __shared__ int before[kPageMaxRows];
    __shared__ PrefixLds prefix;
    __shared__ int status;
    constexpr int KEEP = 4;   // rows per thread that stay in registers (1024 rows)
    const int tid = threadIdx.x;
    const int per = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    const int page = 1 << a.page_shift;
    const int64_t row_limit = static_cast<int64_t>(a.max_pages) << a.page_shift;
    if (tid == 0) status = 0;
    const int count = a.state[0], epoch = a.state[1];
    // (state[3] is the first workgroup's alone: it changes the word below.)
    const int made = blockIdx.x == 0 && tid == 0 ? a.state[3] : 0;
    struct Row {
        int n, len, held;
    };
    Row kept[KEEP];
    if (per <= KEEP) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            const int r = r0 + k < r1 ? r0 + k : 0;
            kept[k] = {a.new_tokens[r], a.lengths[r], a.held[r]};
        }
    }
    // Runs f(row, values) over the thread's rows.
    auto each = [&](auto&& f) {
        if (per <= KEEP) {
#pragma unroll
            for (int k = 0; k < KEEP; ++k)
                if (r0 + k < r1) f(r0 + k, kept[k]);
        } else {
            for (int r = r0; r < r1; ++r) f(r, Row{a.new_tokens[r], a.lengths[r], a.held[r]});
        }
    };
    auto need_of = [&](const Row& x) {
        return static_cast<int>((static_cast<int64_t>(x.len) + x.n + page - 1) >> a.page_shift);
    };
    int bad = 0, tokens = 0, fresh = 0;
    float size = 0.0f;
    each([&](int, const Row& x) {
        if (x.n < 0) bad |= kPageStatusTokens;
        if (x.len < 0 || x.held < 0 || x.held > a.max_pages || static_cast<int64_t>(x.len) + x.n > row_limit ||
            x.len > static_cast<int64_t>(x.held) << a.page_shift)
            bad |= kPageStatusRow;
        tokens += x.n;
        fresh += max(need_of(x) - x.held, 0);
        size += static_cast<float>(x.n);
    });
    const Prefix pre = block_prefix(tokens, fresh, size, &prefix);
    if (bad) atomicOr(&status, bad);
    __syncthreads();
    int refuse = status;
    // (a row's fresh pages are no more than its new positions where nothing
    // else is wrong: its length lies within the pages that it holds)
    if (pre.huge || pre.total_a > a.tokens) refuse |= kPageStatusTokens;
    if ((refuse == 0 && pre.total_b > count) || count > a.pages) refuse |= kPageStatusPool;
    const bool ok = refuse == 0;
    int at = pre.a, fat = pre.b;
    each([&](int r, const Row& x) {
        const int n = ok ? x.n : 0, need = ok ? need_of(x) : 0;
        starts[r] = ok ? at : 0;
        before[r] = ok ? fat : 0;
        at += n;
        fat += max(need - x.held, 0);
        if (blockIdx.x == 0) {
            a.starts[r] = starts[r];
            a.kv_lengths[r] = x.len + n;
            a.held_out[r] = max(need, x.held);
        }
    });
    const int live = ok ? pre.total_a : 0;
    const int taken = ok ? pre.total_b : 0;
    if (tid == 0) {
        starts[a.rows] = live;
        if (blockIdx.x == 0) {
            a.starts[a.rows] = live;
            a.info[0] = refuse;
            a.info[1] = live;
            a.info[2] = taken;
            // A refused plan writes no table entries and replaces no other.
            const int number = static_cast<int>(static_cast<uint32_t>(made) + (ok ? 1u : 0u));
            a.info[3] = plan_number(epoch, number);
            if (ok) a.state[3] = number;
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
    const int count = a.state[0], epoch = a.state[1], status = a.state[2], made = a.state[3];
    int refuse = a.info[0];
    // Not the last plan made, or none at all since the pool changed.
    if (a.info[3] != plan_number(epoch, made) || (refuse == 0 && made == 0)) refuse |= kPageStatusStale;
    __syncthreads();  // every thread has read the state that thread 0 changes
    if (refuse == 0) {
        for (int r = threadIdx.x; r < a.rows; r += kThreads) {
            const int n = a.starts[r + 1] - a.starts[r];
            if (a.accepted == nullptr) {
                a.lengths[r] = a.kv_lengths[r];
            } else if (n > 0) {
                // The first row of a verified block is no draft, and positions
                // of the step that the block has no row for are none either.
                const int64_t block = a.block_starts == nullptr
                                          ? n
                                          : static_cast<int64_t>(a.block_starts[r + 1]) - a.block_starts[r];
                const int64_t grown = n - max(block, INT64_C(1)) + max(a.accepted[r], 0) + 1;
                a.lengths[r] += static_cast<int>(min(max(grown, INT64_C(1)), static_cast<int64_t>(n)));
            }
            a.held[r] = a.held_new[r];
        }
    }
    if (threadIdx.x == 0) {
        if (refuse == 0) {
            a.state[0] = count - a.info[2];
            a.state[1] = epoch + 1;
            a.state[3] = 0;
        }
        a.state[2] = status | refuse;
    }
}

__global__ __launch_bounds__(kThreads) void page_release_kernel(PageReleaseArgs a) {
    __shared__ int before[kPageMaxRows];
    __shared__ PrefixLds prefix;
    const int tid = threadIdx.x;
    const int per = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    const int count = a.state[0];
    int mine = 0;
    for (int r = r0; r < r1; ++r) mine += a.mask[r] ? min(max(a.held[r], 0), a.max_pages) : 0;
    const Prefix pre = block_prefix(mine, 0, static_cast<float>(mine), &prefix);
    const int total = pre.total_a;
    int at = pre.a;
    const bool ok = !pre.huge && count >= 0 && static_cast<int64_t>(count) + total <= a.pages;
    for (int r = r0; r < r1; ++r) {
        before[r] = at;
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
            a.state[0] = count + total;
            a.state[1] += 1;
            a.state[3] = 0;
        } else {
            a.state[2] |= kPageStatusPool;
        }
    }
}

// ---- rows that take over their parents' positions -----------------------------

// One workgroup: a row r whose parent p is another row, one that keeps its own,
// gets p's length and as many pages as that needs (fresh ones as a plan takes
// them, rows in order).  before[r] is the first of r's pages among all that are
// to be copied, before[rows] their count (0 where the fork is refused).
__global__ __launch_bounds__(kThreads) void page_fork_kernel(PageForkArgs a) {
    __shared__ PrefixLds prefix;
    __shared__ int status;
    const int tid = threadIdx.x;
    const int per = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    const int page = 1 << a.page_shift;
    const int count = a.state[0], epoch = a.state[1], earlier = a.state[2];
    if (tid == 0) status = 0;
    // (pages, fresh pages) of a row, -1 pages for one that is wrong
    auto look = [&](int r, int& length, int& fresh) {
        const int p = a.parents[r];
        fresh = length = 0;
        if (p == r) return 0;
        if (p < 0 || p >= a.rows || a.parents[p] != p) return -1;
        length = a.lengths[p];
        const int held = a.held[r], parent_held = a.held[p];
        if (held < 0 || held > a.max_pages || parent_held < 0 || parent_held > a.max_pages || length < 0 ||
            length > static_cast<int64_t>(parent_held) << a.page_shift)
            return -1;
        const int need = static_cast<int>((static_cast<int64_t>(length) + page - 1) >> a.page_shift);
        fresh = max(need - held, 0);
        return need;
    };
    int bad = 0, pages = 0, fresh = 0;
    float size = 0.0f;
    for (int r = r0; r < r1; ++r) {
        int length, more;
        const int need = look(r, length, more);
        bad |= need < 0;
        pages += max(need, 0);
        fresh += more;
        size += static_cast<float>(max(need, 0));
    }
    const Prefix pre = block_prefix(pages, fresh, size, &prefix);
    if (bad) atomicOr(&status, kPageStatusRow);
    __syncthreads();
    int refuse = status;
    if (pre.huge) refuse |= kPageStatusRow;
    if ((refuse == 0 && pre.total_b > count) || count > a.pages) refuse |= kPageStatusPool;
    const bool ok = refuse == 0;
    int at = pre.a, taken = pre.b;
    for (int r = r0; r < r1; ++r) {
        int length, more;
        const int need = max(look(r, length, more), 0);
        a.before[r] = ok ? at : 0;
        if (!ok || a.parents[r] == r) continue;
        const int held = a.held[r];
        for (int j = 0; j < more; ++j)
            a.table[static_cast<int64_t>(r) * a.max_pages + held + j] = a.free_pages[count - 1 - (taken + j)];
        at += need;
        taken += more;
        // (No row reads these of another: parents keep theirs.)
        a.held[r] = max(held, need);
        a.lengths[r] = length;
    }
    if (tid == 0) {
        a.before[a.rows] = ok ? pre.total_a : 0;
        if (ok) {
            a.state[0] = count - pre.total_b;
            a.state[1] = epoch + 1;
            a.state[3] = 0;
        }
        a.state[2] = earlier | refuse;
    }
}

// The pages' contents: a workgroup has a page and some of its pieces (a head of
// a layer), at least kForkBytes in all, and a wave copies a piece at a time.
// Pages that are read belong to rows that keep theirs, so none is written.
// Bound by HBM (8 prompts to 4 beams each, 1.17 GB read and written: 233 us, 5 TB/s).
constexpr int kForkBytes = 65536;
__global__ __launch_bounds__(kThreads) void page_fork_copy(PageForkArgs a) {
    const int total = a.before[a.rows], lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int parts = (a.pieces + a.share - 1) / a.share;
    const int64_t work = static_cast<int64_t>(total) * parts;
    for (int64_t i = blockIdx.x; i < work; i += gridDim.x) {
        const int unit = static_cast<int>(i / parts), first = static_cast<int>(i - static_cast<int64_t>(unit) * parts) * a.share;
        // (Rows without pages to copy share their place with the next: the last
        // of those is meant.)
        const int r = last_at_most(a.before, a.rows, unit), j = unit - a.before[r], p = a.parents[r];
        const int to = a.table[static_cast<int64_t>(r) * a.max_pages + j];
        const int from = a.table[static_cast<int64_t>(p) * a.max_pages + j];
        if (to < 0 || to >= a.pages || from < 0 || from >= a.pages) continue;
        const int rows = min(a.lengths[r] - (j << a.page_shift), 1 << a.page_shift);
        for (int k = first + wave; k < min(first + a.share, a.pieces); k += kThreads / kWave) {
            int piece = k, c = 0;
            while (piece >= a.cache[c].layers * a.cache[c].heads) {
                piece -= a.cache[c].layers * a.cache[c].heads;
                ++c;
            }
            const ForkCache& cache = a.cache[c];
            uint8_t* base = cache.base + piece / cache.heads * cache.layer_stride + piece % cache.heads * cache.head_stride;
            uint8_t* d = base + to * cache.page_stride;
            const uint8_t* s = base + from * cache.page_stride;
            const int lanes = cache.row_bytes / 16, n = rows * lanes;
            if (cache.row_stride == cache.row_bytes) {
                u32x4* dst = reinterpret_cast<u32x4*>(d);
                const u32x4* src = reinterpret_cast<const u32x4*>(s);
                int x = lane;
                for (; x + 7 * kWave < n; x += 8 * kWave) {
                    u32x4 v[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) v[y] = __builtin_nontemporal_load(src + x + y * kWave);
#pragma unroll
                    for (int y = 0; y < 8; ++y) __builtin_nontemporal_store(v[y], dst + x + y * kWave);
                }
                for (; x < n; x += kWave) dst[x] = src[x];
            } else {
                for (int x = lane; x < n; x += kWave) {
                    const int64_t at = x / lanes * cache.row_stride + x % lanes * 16;
                    *reinterpret_cast<u32x4*>(d + at) = *reinterpret_cast<const u32x4*>(s + at);
                }
            }
        }
    }
}

// ---- append ------------------------------------------------------------------

// A group of D / 8 lanes takes ROWS head rows (query, key or value) of one
// token, 16 bytes per lane and row: y = x / sqrt(mean(x^2) + eps) (1 + w) and
// the rotation of the first `rotary` elements (element e of the first half
// with e + rotary / 2) in fp32, one rounding to the tensor's type at the end.
// A pass over the data: each row is read once and written once.  What bounds
// it is HBM bandwidth (6827 tokens of 20 rows of 256: 30.4 us, 4.7 TB/s read
// and written; a device copy reaches 5.2), and in short steps the chain of
// reads token -> slot and position -> cos and sin (8 tokens: 4.2 us); the rows
// of a group share that chain, and are all requested before the first is used.
template <bool FP16, int D, int ROWS>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int LANES = D / 8;
    const int64_t group = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LANES;
    const int l = threadIdx.x % LANES;
    const int rows = a.heads + 2 * a.kv_heads, pieces = (rows + ROWS - 1) / ROWS;
    const int64_t t = group / pieces;
    if (t >= a.tokens) return;
    const int h0 = static_cast<int>(group - t * pieces) * ROWS;
    const int64_t slot = a.slots[t];
    const int half = a.rotary / 16;   // lanes per half of the rotated elements
    const int64_t p = a.rotary == 0 ? 0 : a.positions != nullptr ? a.positions[t] : t;
    uint4 raw[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int h = min(h0 + i, rows - 1);
        const uint16_t* src = h < a.heads ? a.q + t * a.q_token_stride + h * a.q_head_stride
                              : h < a.heads + a.kv_heads
                                  ? a.k + t * a.k_token_stride + (h - a.heads) * a.k_head_stride
                                  : a.v + t * a.v_token_stride + (h - a.heads - a.kv_heads) * a.v_head_stride;
        raw[i] = ldg16(src + 8 * l);
    }
    if (slot < 0 || slot >= (static_cast<int64_t>(a.pages) << a.page_shift)) return;
    const int64_t block = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    // (The first half takes - sin, the second + sin.)
    float c[8], s[8];
    if (l < 2 * half) {
        if (p < 0 || p >= a.rope_rows) {   // no such row: the rotated elements are NaN
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = s[j] = __builtin_nanf("");
        } else if (a.rope_fp32) {
            const float* cr = static_cast<const float*>(a.cos) + p * a.rotary + 8 * l;
            const float* sr = static_cast<const float*>(a.sin) + p * a.rotary + 8 * l;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(cr + j), y = *reinterpret_cast<const float4*>(sr + j);
                c[j] = x.x; c[j + 1] = x.y; c[j + 2] = x.z; c[j + 3] = x.w;
                s[j] = y.x; s[j + 1] = y.y; s[j + 2] = y.z; s[j + 3] = y.w;
            }
        } else {
            unpack16<FP16>(ldg16(static_cast<const uint16_t*>(a.cos) + p * a.rotary + 8 * l), c);
            unpack16<FP16>(ldg16(static_cast<const uint16_t*>(a.sin) + p * a.rotary + 8 * l), s);
        }
        if (l < half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = -s[j];
        }
    }
    const int partner = static_cast<int>(__lane_id()) + (l < half ? half : l < 2 * half ? -half : 0);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int h = h0 + i;
        if (h >= rows) return;
        if (h >= a.heads + a.kv_heads) {
            *reinterpret_cast<uint4*>(a.v_cache + block * a.v_page_stride +
                                      (h - a.heads - a.kv_heads) * a.v_cache_head_stride + row * a.v_row_stride +
                                      8 * l) = raw[i];
            continue;
        }
        const bool query = h < a.heads;
        const uint16_t* weight = query ? a.q_norm : a.k_norm;
        uint16_t* dst = query ? a.q_out + (t * a.heads + h) * D
                              : a.k_cache + block * a.k_page_stride + (h - a.heads) * a.k_cache_head_stride +
                                    row * a.k_row_stride;
        float x[8];
        unpack16<FP16>(raw[i], x);
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
            float other[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) other[j] = __shfl(x[j], partner);
            if (l < 2 * half) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = x[j] * c[j] + other[j] * s[j];
            }
        }
        *reinterpret_cast<uint4*>(dst + 8 * l) = pack16<FP16>(x);
    }
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

hipError_t launch_page_fork(PageForkArgs a, hipStream_t stream) {
    int64_t bytes = 0;   // of a page in all caches
    for (int c = 0; c < LRMOE_FORK_CACHES; ++c)
        bytes += static_cast<int64_t>(a.cache[c].layers) * a.cache[c].heads * a.cache[c].row_bytes << a.page_shift;
    const int64_t parts = std::max(bytes / kForkBytes, INT64_C(1));
    a.share = static_cast<int>(std::max((a.pieces + parts - 1) / parts, INT64_C(1)));
    page_fork_kernel<<<1, kThreads, 0, stream>>>(a);
    if (a.pieces > 0) page_fork_copy<<<2048, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_page_release(const PageReleaseArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

template <bool FP16, int D>
static void append_rows(const PagedAppendArgs& a, hipStream_t stream) {
    const int64_t rows = a.heads + 2 * a.kv_heads, per = kThreads / (D / 8);   // groups of a workgroup
    // Four rows per group where that still makes three workgroups per CU (20
    // rows of 256: 8192 tokens 32.7 us against 38 with one row, 2048 tokens 12.1
    // against 13.0), else one, where latency counts (1024 tokens 7.9 us against
    // 8.4 with four, 8 tokens 3.4 against 5.7).
    const int64_t pieces = (rows + 3) / 4;
    const bool four = a.tokens * pieces >= per * 768;
    const dim3 grid(static_cast<unsigned>((a.tokens * (four ? pieces : rows) + per - 1) / per));
    if (four) hipLaunchKernelGGL((paged_append_kernel<FP16, D, 4>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<FP16, D, 1>), grid, dim3(kThreads), 0, stream, a);
}

hipError_t launch_paged_append(const PagedAppendArgs& a, bool fp16, int dim, hipStream_t stream) {
    if (dim == 64) fp16 ? append_rows<true, 64>(a, stream) : append_rows<false, 64>(a, stream);
    else if (dim == 128) fp16 ? append_rows<true, 128>(a, stream) : append_rows<false, 128>(a, stream);
    else fp16 ? append_rows<true, 256>(a, stream) : append_rows<false, 256>(a, stream);
    return hipGetLastError();
}

}  // namespace lrmoe
