// Beam search: the choice of a group's best continuations, and the rows of
// states that follow their parents.
//
// A group has W beams, rows of logits x; beam w's continuation by token t has
// the score s_w + x_t - log sum_j exp x_j.  Chosen are the W best of the group's
// W vocab (ties: the lowest w vocab + t).  What bounds it is reading the logits
// once; for a few rows, the chain of two launches.
#include "beam.h"

namespace lrmoe {
namespace {

constexpr int kSlice = 2048;          // logits that a wave takes
constexpr int kPer = kSlice / kWave;  // and a lane
constexpr int kThreads = 256;
constexpr int kJoinThreads = 512;
// Candidates of a row (its slices' W best) that a lane of the join keeps in
// registers, so that each of the W passes over them reads none from memory: up to 10,
// 640 in all.  The join takes, with room for 10, 20 and 40 and always from memory:
// 4 beams of 151936 (300 candidates) 6.1, 7.0, 9.8, 7.6 us; 8 beams (600) 9.6, 11.4,
// 16.8, 19.0; 9 beams (675) 34, 17, 26, 34; 16 beams (1200) 98, 33, 49, 98; 32 beams
// (2400) 713, 709, 196, 713: room that is not used costs searches of few beams as
// much, in proportion, as it would spare those of many.
constexpr int kKeep = 10;

// A finite value and its token as one key: the larger value first, then the
// lower token.  0 stands for no candidate.
__device__ __forceinline__ uint64_t beam_key(float x, int token) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // (-0 becomes +0)
    const uint32_t ordered = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<uint64_t>(ordered) << 32) | (0xffffffffu - static_cast<uint32_t>(token));
}
__device__ __forceinline__ float beam_value(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int beam_token(uint64_t key) {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    const uint32_t hi = wave_max_u32(static_cast<uint32_t>(v >> 32));
    const uint32_t lo = wave_max_u32(static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
// Orders a wave's LDS accesses (it runs in step).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
    if constexpr (TYPE == 0) return static_cast<const float*>(row)[i];
    const uint16_t b = static_cast<const uint16_t*>(row)[i];
    return TYPE == 1 ? bf2f(b) : f16_to_f(b);
}

// 16 bytes of a row, which begins at any element (global loads need no more; 256
// rows of 151935 in bf16: 59.7 us a call with single loads, 36.7 so, as 151936).
typedef __attribute__((address_space(1))) const u32x4 __attribute__((aligned(2))) RowBytes;
__device__ __forceinline__ uint4 load_row(const void* row, int64_t byte) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<RowBytes*>(reinterpret_cast<uintptr_t>(row) + byte));
    return make_uint4(v.x, v.y, v.z, v.w);
}
template <int TYPE, int VEC>
__device__ __forceinline__ void logits_of(uint4 raw, float* x) {
    if constexpr (TYPE == 0) {
        x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y);
        x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
    } else {
        unpack16<TYPE == 2>(raw, x);
    }
}

// A beam takes part with its logits while it is neither finished nor dead (a
// score that is not finite).
__device__ __forceinline__ bool beam_open(const BeamArgs& a, int row) {
    return finite_bits(a.scores[row]) && (a.finished == nullptr || a.finished[row] == 0);
}

// A list that a wave has gathered: at most kWave keys, of which it keeps the W
// best, best first (lane r the r-th): a key's place is the number of larger ones.
constexpr int kGather = kWave;
__device__ __forceinline__ uint64_t gathered_best(const uint64_t* list, uint64_t* best, int n, int W, int lane) {
    const uint64_t key = lane < n ? list[lane] : 0;
    int place = 0;
    for (int i = 0; i < n; ++i) place += list[i] > key;
    if (lane < n && place < W) best[place] = key;
    wave_sync();
    return lane < min(n, W) ? best[lane] : 0;
}

// The W best of a wave's keys, best first, as each lane's own calls to
// each(f) pass them: lane r gets the r-th (0 where there are no more).
template <typename Each>
__device__ __forceinline__ uint64_t wave_best(int W, int lane, Each&& each) {
    uint64_t mine = 0, last = ~UINT64_C(0);
    for (int r = 0; r < W; ++r) {
        uint64_t top = 0;
        each([&](uint64_t key) { top = key < last && key > top ? key : top; });
        last = wave_max_u64(top);
        if (lane == r) mine = last;
        if (last == 0) break;
    }
    return mine;
}

// A wave takes 2048 logits of a row in registers: their maximum and sum of
// exponentials, and the W best. Those are no smaller than the W-th largest of the
// lanes' maxima, so that only what reaches it is gathered and ranked, W numbers
// and a few more; where equal values make them more than a list holds, the
// registers are gone through W times instead.  Bound by the logits where they are
// fp32 (256 rows of 151936, a tenth of them finished: 20.4 us, 6.9 TB/s; with W
// passes for every slice 55 us), by its instructions in 16 bits (256 rows in bf16
// 25 us, 3.1 TB/s); 4 rows in bf16 5.4 us, launch and latency.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void beam_slices(BeamArgs a) {
    __shared__ uint64_t lists[kThreads / kWave][kGather], bests[kThreads / kWave][kBeamMax];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int slices = (a.vocab + kSlice - 1) / kSlice;
    const int slice = blockIdx.x * (kThreads / kWave) + wave;
    const int row = blockIdx.y;
    if (slice >= slices || !beam_open(a, row)) return;
    constexpr int SIZE = TYPE == 0 ? 4 : 2, VEC = 16 / SIZE;
    const void* base = static_cast<const uint8_t*>(a.logits) + row * a.stride * SIZE;
    const int first = slice * kSlice;
    float x[kPer];
    if (first + kSlice <= a.vocab) {
        uint4 raw[kPer / VEC];
#pragma unroll
        for (int i = 0; i < kPer / VEC; ++i)
            raw[i] = load_row(base, static_cast<int64_t>(first + (i * kWave + lane) * VEC) * SIZE);
#pragma unroll
        for (int i = 0; i < kPer / VEC; ++i) logits_of<TYPE, VEC>(raw[i], x + VEC * i);
    } else {
#pragma unroll
        for (int i = 0; i < kPer / VEC; ++i) {
            const int at = first + (i * kWave + lane) * VEC;
            if (at + VEC <= a.vocab) {
                logits_of<TYPE, VEC>(load_row(base, static_cast<int64_t>(at) * SIZE), x + VEC * i);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    x[VEC * i + j] = at + j < a.vocab ? load_logit<TYPE>(base, at + j) : -__builtin_inff();
            }
        }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        x[i] = finite_bits(x[i]) ? x[i] + 0.0f : -__builtin_inff();   // (-0 becomes +0)
        top = __builtin_fmaxf(top, x[i]);
    }
    // The lanes' maxima, largest first, until W of them: the border.
    uint32_t left = finite_bits(top) ? static_cast<uint32_t>(beam_key(top, 0) >> 32) : 0u;
    uint32_t border = 0;
    float m = 0.0f;
    bool some = false;
    for (int r = 0; r < a.beams; ++r) {
        border = wave_max_u32(left);
        if (r == 0) {
            some = border != 0;
            m = some ? beam_value(static_cast<uint64_t>(border) << 32) : 0.0f;
        }
        if (border == 0) break;
        const uint64_t with = __ballot(left == border);
        if (lane == __builtin_ctzll(with)) left = 0;
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += __builtin_amdgcn_exp2f((x[i] - m) * 1.4426950408889634f);
    sum = wave_butterfly_sum(sum);
    const int64_t at = static_cast<int64_t>(row) * slices + slice;
    if (lane == 0) a.sums[at] = make_float2(m, some ? sum : 0.0f);
    // (No border: fewer than W lanes have any.)
    const float least = border ? beam_value(static_cast<uint64_t>(border) << 32) : -__builtin_inff();
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool in = x[i] >= least && finite_bits(x[i]);
        const uint64_t with = __ballot(in);
        if (with == 0) continue;
        const int place = n + __popcll(with & ((UINT64_C(1) << lane) - 1));
        if (in && place < kGather)
            lists[wave][place] = beam_key(x[i], first + (i / VEC * kWave + lane) * VEC + i % VEC);
        n += __popcll(with);
    }
    uint64_t best;
    if (n <= kGather) {
        wave_sync();
        best = gathered_best(lists[wave], bests[wave], n, a.beams, lane);
    } else {
        best = wave_best(a.beams, lane, [&](auto&& f) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (finite_bits(x[i])) f(beam_key(x[i], first + (i / VEC * kWave + lane) * VEC + i % VEC));
        });
    }
    if (lane < a.beams)
        a.best[at * a.beams + lane] = make_uint2(static_cast<uint32_t>(best), static_cast<uint32_t>(best >> 32));
}

// One workgroup per group: each wave joins the slices of a row, then the W W
// candidates are ranked by counting those ahead of each, in 64 bits (distinct
// logits of a row stay distinct).  Bound by its chain of loads and W maxima over a
// wave: 5.6 us for 1 x 4 beams, 9.9 for 32 x 8.
__global__ __launch_bounds__(kJoinThreads) void beam_join(BeamArgs a) {
    __shared__ double score[kBeamMax * kBeamMax];
    __shared__ int token[kBeamMax * kBeamMax];
    __shared__ int chosen[kBeamMax];
    const int W = a.beams, lane = threadIdx.x % kWave;
    const int slices = (a.vocab + kSlice - 1) / kSlice;
    const double none = -__builtin_inf();
    for (int w = threadIdx.x / kWave; w < W; w += kJoinThreads / kWave) {
        const int row = blockIdx.x * W + w;
        const float given = a.scores[row];
        if (!beam_open(a, row)) {
            // A finished beam goes on as it is, a dead one not at all.
            if (lane < W) {
                score[w * W + lane] = lane == 0 && finite_bits(given) ? static_cast<double>(given) : none;
                token[w * W + lane] = -1;
            }
            continue;
        }
        const float2* sums = a.sums + static_cast<int64_t>(row) * slices;
        const uint2* best = a.best + static_cast<int64_t>(row) * slices * W;
        const int n = slices * W;
        // Up to kKeep candidates a lane stay in registers.
        uint64_t keys[kKeep];
        const bool fits = n <= kKeep * kWave;
        if (fits) {
#pragma unroll
            for (int i = 0; i < kKeep; ++i) {
                const int at = i * kWave + lane;
                const uint2 x = best[min(at, n - 1)];
                keys[i] = at < n ? (static_cast<uint64_t>(x.y) << 32) | x.x : 0;
            }
        }
        float m = -__builtin_inff();
        for (int i = lane; i < slices; i += kWave) m = sums[i].y > 0.0f ? __builtin_fmaxf(m, sums[i].x) : m;
        const uint64_t top = wave_max_u64(finite_bits(m) ? beam_key(m, 0) : 0);
        m = top ? beam_value(top) : 0.0f;
        double sum = 0.0;
        for (int i = lane; i < slices; i += kWave)
            if (sums[i].y > 0.0f)
                sum += static_cast<double>(sums[i].y) * __builtin_amdgcn_exp2f((sums[i].x - m) * 1.4426950408889634f);
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) sum += __shfl_xor(sum, off);
        const uint64_t key = wave_best(W, lane, [&](auto&& f) {
            if (fits) {
#pragma unroll
                for (int i = 0; i < kKeep; ++i) f(keys[i]);
            } else {
                for (int i = lane; i < n; i += kWave) f((static_cast<uint64_t>(best[i].y) << 32) | best[i].x);
            }
        });
        if (lane < W) {
            score[w * W + lane] =
                key ? static_cast<double>(given) + (static_cast<double>(beam_value(key)) - m - log(sum)) : none;
            token[w * W + lane] = key ? beam_token(key) : -1;
        }
    }
    if (threadIdx.x < kBeamMax) chosen[threadIdx.x] = -1;
    __syncthreads();
    for (int c = threadIdx.x; c < W * W; c += kJoinThreads) {
        const double mine = score[c];
        if (mine == none) continue;
        // (A row's candidates are in order: those of equal score by token.)
        int ahead = 0;
        for (int o = 0; o < W * W; ++o) ahead += score[o] > mine || (score[o] == mine && o < c);
        if (ahead < W) chosen[ahead] = c;
    }
    __syncthreads();
    // The first of a parent's continuations takes the parent's row, the others
    // in their order the rows left over; then rows without one.
    if (threadIdx.x >= kWave) return;
    const int c = lane < W ? chosen[lane] : -1;
    const int parent = c < 0 ? -1 : c / W;
    uint32_t taken = 0;
    bool stays = c >= 0;
    for (int i = 0; i < W; ++i) {
        const int other = __shfl(parent, i);
        if (other >= 0) taken |= 1u << other;
        if (i < lane && other == parent) stays = false;
    }
    const uint64_t moving = __ballot(c >= 0 && !stays);
    uint32_t spare = ~taken & (W == 32 ? 0xffffffffu : (1u << W) - 1u);
    const int ahead = __popcll(moving & ((UINT64_C(1) << lane) - 1));
    int place = parent;
    if (c >= 0 && !stays) {
        uint32_t left = spare;
        for (int i = 0; i < ahead; ++i) left &= left - 1;
        place = __builtin_ctz(left);
    }
    // (Each row's own entry first, then those that were chosen.)
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * W;
    uint32_t used = taken;
    for (int i = 0; i < __popcll(moving); ++i) {
        used |= spare & (0u - spare);
        spare &= spare - 1;
    }
    if (lane < W && !((used >> lane) & 1u)) {
        a.tokens[row0 + lane] = -1;
        a.parents[row0 + lane] = static_cast<int32_t>(row0 + lane);
        a.scores_out[row0 + lane] = -__builtin_inff();
    }
    if (c >= 0) {
        a.tokens[row0 + place] = token[c];
        a.parents[row0 + place] = static_cast<int32_t>(row0 + parent);
        a.scores_out[row0 + place] = static_cast<float>(score[c]);
    }
}

// ---- rows that follow their parents ------------------------------------------

constexpr int kForkBytes = LRMOE_FORK_BYTES;   // of a row per workgroup

template <typename T>
__device__ __forceinline__ void fork_copy(uint8_t* to, const uint8_t* from, int64_t bytes) {
    T* d = reinterpret_cast<T*>(to);
    const T* s = reinterpret_cast<const T*>(from);
    const int n = static_cast<int>(bytes / sizeof(T));
    int i = threadIdx.x;
    for (; i + 3 * kThreads < n; i += 4 * kThreads) {
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = s[i + j * kThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j) d[i + j * kThreads] = v[j];
    }
    for (; i < n; i += kThreads) d[i] = s[i];
}

// A workgroup copies a piece of a row.  Rows that are read keep their places
// (a row whose parent moves itself is left alone), so nothing that is read is
// written.  Bound by HBM: each byte that moves is read and written once (60 tensors
// of 32 rows' states: 5.3 to 6 TB/s of what moves).
__global__ __launch_bounds__(kThreads) void fork_rows_kernel(ForkRowsArgs a) {
    int i = 0;
    while (i + 1 < a.tensors && static_cast<int>(blockIdx.x) >= a.t[i + 1].first) ++i;
    const ForkTensor& t = a.t[i];
    const int pieces = static_cast<int>((t.bytes + kForkBytes - 1) / kForkBytes);
    const int at = static_cast<int>(blockIdx.x) - t.first;
    const int row = at / pieces;
    const int parent = a.parents[row];
    if (parent == row || parent < 0 || parent >= a.rows || a.parents[parent] != parent) return;
    const int64_t begin = static_cast<int64_t>(at % pieces) * kForkBytes;
    const int64_t bytes = min(t.bytes - begin, static_cast<int64_t>(kForkBytes));
    uint8_t* to = t.base + row * t.stride + begin;
    const uint8_t* from = t.base + parent * t.stride + begin;
    switch (t.width) {
        case 16: fork_copy<u32x4>(to, from, bytes); break;
        case 8: fork_copy<uint2>(to, from, bytes); break;
        case 4: fork_copy<uint32_t>(to, from, bytes); break;
        case 2: fork_copy<uint16_t>(to, from, bytes); break;
        default: fork_copy<uint8_t>(to, from, bytes); break;
    }
}

}  // namespace

size_t beam_workspace_bytes(int groups, int beams, int vocab) {
    const size_t slices = (static_cast<size_t>(vocab) + kSlice - 1) / kSlice;
    return static_cast<size_t>(groups) * beams * slices * (sizeof(float2) + beams * sizeof(uint2));
}

hipError_t launch_beam_select(BeamArgs a, int type, void* workspace, hipStream_t stream) {
    const int slices = (a.vocab + kSlice - 1) / kSlice, per = kThreads / kWave;
    a.sums = static_cast<float2*>(workspace);
    a.best = reinterpret_cast<uint2*>(a.sums + static_cast<size_t>(a.groups) * a.beams * slices);
    const dim3 grid((slices + per - 1) / per, a.groups * a.beams);
    if (type == 0) beam_slices<0><<<grid, kThreads, 0, stream>>>(a);
    else if (type == 1) beam_slices<1><<<grid, kThreads, 0, stream>>>(a);
    else beam_slices<2><<<grid, kThreads, 0, stream>>>(a);
    beam_join<<<a.groups, kJoinThreads, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_fork_rows(ForkRowsArgs a, hipStream_t stream) {
    int64_t blocks = 0;
    for (int i = 0; i < a.tensors; ++i) {
        ForkTensor& t = a.t[i];
        t.first = static_cast<int>(blocks);
        const uintptr_t all = reinterpret_cast<uintptr_t>(t.base) | static_cast<uintptr_t>(t.stride) |
                              static_cast<uintptr_t>(t.bytes);
        t.width = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
        blocks += (t.bytes + kForkBytes - 1) / kForkBytes * a.rows;
    }
    if (blocks == 0) return hipSuccess;
    fork_rows_kernel<<<static_cast<uint32_t>(blocks), kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace lrmoe
