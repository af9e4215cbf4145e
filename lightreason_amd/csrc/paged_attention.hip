// Attention of a step's new positions over a paged key/value cache.  Row t of
// sequence b (n_b new positions, kv_b cached ones with them) sees positions
// 0 .. kv_b - n_b + t: out = sum_p softmax(q . k_p scale)_p v_p, times
// sigmoid(gate) when a gate is given.
//
// The rows that share keys and values (a sequence's new tokens, times the
// query heads of one key/value head) form tiles of 32 or 128; a workgroup
// takes a tile over a range of positions, in one pass: a block of scores
// S^T = K Q^T, a running maximum per row and a point m at or (fp16) 2^7 below
// it (moved, and the sums rescaled, only when the maximum grew by more than
// 2^8: what is summed is relative to m, whatever m is, so the result does not
// depend on it), weights exp2(s - m) as one or two numbers of the tensors' type
// (PARTS), and their product with the values into fp32 sums.  Both
// products are 32x32x16 matrix instructions.  In the transposed form a lane
// holds scores of one row only, so maxima and sums stay in the lane (and its
// partner 32 lanes on), and the weights are the second product's operand as
// they are, once the values are read in the matching order: the transposing
// LDS read gives each lane four positions of one element.
//
// Keys and values go from the pages into LDS without passing registers.  In
// tiles of 128 rows all four waves read what they load together, one tile of
// positions ahead of its use in the other of two buffers; in tiles of 32 a wave
// has one buffer of keys and one of values, each filled again once it is read,
// the keys during the product with the values and those during the next keys'.
// Width 256 needs 192 registers per lane for queries and sums alone; what is
// left of the 256 that two waves per SIMD may have goes to fragments read ahead
// (read_ahead), which is why the LDS places (Place) are chosen for few
// addresses.
//
// What bounds it (16 query over 2 key/value heads of 256, pages of 64): 4096
// new positions over 28003 cached take 1.66 ms, 1.21 PFLOP/s; the matrix units
// are busy in 67 % of the cycles and the card's power limit holds the clock at
// 1.4-1.6 GHz then, LDS reads have no bank conflicts.  2048 positions from an
// empty cache take 74 us, 0.46 PFLOP/s: 60 of attention, whose 376 workgroups
// of 1-34 steps load the CUs unevenly (by the schedule the fullest holds two of
// 62 steps together, the mean is 32.5, a step of two workgroups takes 1.75 us),
// 13 of the merge of 33 MB of partial rows.  One decode position for each of 64
// sequences of 200-16000 takes 203 us, 5.4 TB/s of keys and values, the rate of
// a large copy.  One sequence of 1000 takes 14.3 us, a chain of reads (lengths,
// table, rows, partial rows) in two launches.
#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;

// By the exponential and reciprocal instructions, an ulp each (2^-23 of a
// result that is rounded to 16 bits): the exact division and exponential take
// some 40 instructions, which for the gates of 2048 positions of 16 heads of
// 256 were more than the merge's memory time.
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One row (token t of sequence b, head h) by one wave, reading only the
// positions that the row sees: a lane per position for the scores (64 at a
// time), a lane per D / 64 elements for the values.  The path of rows whose
// tile holds values that are not finite and that some of its rows do not see
// (in a tile's matrix product their zero weights would not hide them).
template <bool FP16, int D>
__device__ void attend_row(const PagedAttnArgs& a, int b, int64_t t, int64_t h, int64_t seen, float* qs, float* ps,
                           int64_t* vs) {
    constexpr int E = D / kWave;
    const int lane = threadIdx.x % kWave;
    const uint16_t* q = a.q + t * a.q_token_stride + h * a.q_head_stride;
    const int64_t kh = h / a.group;
    // LDS rows here belong to one wave, whose accesses stay in order; the
    // fences below only keep the compiler from moving them.
    for (int e = lane; e < D; e += kWave) qs[e] = elem16<FP16>(q[e]) * a.scale;
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
            block = block < 0 || block >= a.pages ? 0 : block;
            const int64_t row = p & ((1 << a.page_shift) - 1);
            const uint16_t* k = a.k_cache + block * a.k_page_stride + kh * a.k_head_stride + row * a.k_row_stride;
            vs[lane] = block * a.v_page_stride + kh * a.v_head_stride + row * a.v_row_stride;
            s = 0.0f;
            for (int e = 0; e < D; e += 8) {
                float x[8];
                unpack16<FP16>(ldg16(k + e), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) s = __builtin_fmaf(x[j], qs[e + j], s);
            }
        }
        float top = s;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, off));
        const float mn = __builtin_fmaxf(m, top);
        const float shift = mn == -__builtin_inff() ? 0.0f : mn;
        const float w = p < seen ? __builtin_exp2f(s - shift) : 0.0f;
        const float fall = __builtin_exp2f(m - shift);
        float sum = w;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) sum += __shfl_xor(sum, off);
        l = l * fall + sum;
        m = mn;
        ps[lane] = w;
        wave_lds_fence();
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] *= fall;
        const int count = static_cast<int>(min(static_cast<int64_t>(kWave), seen - base));
        for (int j = 0; j < count; ++j) {
            const uint16_t* v = a.v_cache + vs[j] + lane * E;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] = __builtin_fmaf(ps[j], elem16<FP16>(v[i]), acc[i]);
        }
        wave_lds_fence();
    }
    const bool nan = __any(bad);
    uint16_t* out = a.out + t * a.out_token_stride + h * a.out_head_stride + lane * E;
    const uint16_t* gate = a.gate + t * a.gate_token_stride + h * a.gate_head_stride + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float o = seen > 0 ? acc[i] / l : 0.0f;
        if (nan) o = __builtin_nanf("");
        if (a.gate != nullptr) o *= sigmoid(elem16<FP16>(gate[i]));
        out[i] = static_cast<uint16_t>(FP16 ? f_to_f16(o) : f2bf(o));
    }
}

// ---- the step's schedule ----------------------------------------------------------
//
// A sequence's rows (token-major, then the heads of one key/value head's
// group) are cut into tiles of BM rows; a tile's positions into splits, so
// that a few long sequences fill the chip.  W is the sum over all tiles of
// their steps and one; c steps, more than W / target, are the most of a split.
// Tiles of 32 rows are all counted as long as their sequence's last, so they
// make at most target splits and one per tile, and fewer than 2 target slots
// for those that are split; longer tiles, counted as the mean of the
// sequence's first and last, up to twice as many.
// Every wave works this out for itself from starts and kv_lengths (a lane per
// sequence, cross-lane sums, no LDS and no barrier): nothing of it depends on
// the host, no launch precedes the attention's, and what it costs is the one
// round trip for the two arrays.

struct Sequence {
    int first, n, kv;  // first token, new tokens, cached positions
};
// Positions that token i of the sequence sees.
__device__ __forceinline__ int seen_by(const Sequence& s, int i) { return max(s.kv - s.n + i + 1, 0); }

struct Split {
    int b, tile, split, splits;
    int slot;       // of the tile's first partial rows, before the head
    int ordinal;    // of the tile among all tiles
    Sequence seq;
};

__device__ __forceinline__ int tiles_of(int n, int group, int bm) { return (n * group + bm - 1) / bm; }
__device__ __forceinline__ int steps_of(int positions, int step) { return max((positions + step - 1) / step, 1); }
// Positions that the tile's last row sees.
__device__ __forceinline__ int tile_end(const Sequence& s, int group, int bm, int tile) {
    const int rows = min((tile + 1) * bm, s.n * group);
    return seen_by(s, (rows - 1) / group);
}
// Tiles (of the sequence's `count`) of at most `splits` splits of c steps: the
// first ones, which see least.
template <int BM, int STEP>
__device__ __forceinline__ int tiles_upto(const Sequence& s, int group, int count, int splits, int c) {
    const int64_t tokens = static_cast<int64_t>(splits) * c * STEP - s.kv + s.n;   // that see no more than that
    return tokens >= s.n ? count : tokens <= 0 ? 0 : static_cast<int>(tokens) * group / BM;
}

// The sequence, tile and split of item `item` (wave-uniform), heavy tiles
// first, and how many tiles there are; false past the last item, and for
// starts that are not ascending within [0, tokens] (such a step is empty).
// HELD: sequences per lane that stay in registers.
template <int BM, int STEP, int HELD>
__device__ __forceinline__ bool find_split(const PagedAttnArgs& a, int item, int target, int least, Split* out,
                                           int* all_tiles) {
    const int lane = threadIdx.x % kWave;
    const int64_t capacity = static_cast<int64_t>(a.max_pages) << a.page_shift;
    Sequence s[HELD];
    bool bad = false;
    auto load = [&](int base) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int b = base + k * kWave + lane;
            const bool in = b < a.seqs;
            const int first = a.starts[in ? b : 0], next = a.starts[in ? b + 1 : 0], kv = a.kv_lengths[in ? b : 0];
            bad |= first < 0 || next < first || next > a.tokens;
            s[k].first = first;
            s[k].n = next - first;   // 0 past the last sequence
            s[k].kv = static_cast<int>(min(static_cast<int64_t>(max(kv, 0)), capacity));
        }
    };
    float work = 0.0f;
    int tiles = 0;
    for (int base = 0; base < a.seqs; base += HELD * kWave) {
        load(base);
#pragma unroll
        for (int k = 0; k < HELD; ++k)
            if (s[k].n > 0) {
                const int count = tiles_of(s[k].n, a.group, BM), last = steps_of(s[k].kv, STEP);
                const int first = BM > 32 ? steps_of(tile_end(s[k], a.group, BM, 0), STEP) : last;
                tiles += count;
                work += static_cast<float>(count) * (0.5f * (first + last) + 1.0f);
            }
    }
    *all_tiles = 0;
    if (__any(bad)) return false;
    *all_tiles = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
    work = wave_butterfly_sum(work) * a.kv_heads;
    // Up to 64 sequences of many tiles are taken longest first, so that none of
    // the long ones starts last (nine prompts of 1-900 tokens over up to 5000
    // cached: 290 us against 306 in their own order).
    int who_is = lane;   // the sequence of this lane's s[0]
    if (BM > 32 && a.seqs > 1 && a.seqs <= kWave) {
        int rank = 0;
        for (int j = 0; j < a.seqs; ++j) {
            const int other = __builtin_amdgcn_readlane(s[0].kv, j);
            rank += other > s[0].kv || (other == s[0].kv && j < lane);
        }
        if (lane >= a.seqs) rank = lane;
        auto to_rank = [&](int v) { return __builtin_amdgcn_ds_permute(rank << 2, v); };
        s[0] = {to_rank(s[0].first), to_rank(s[0].n), to_rank(s[0].kv)};
        who_is = to_rank(lane);
    }
    const float each = work / target;
    const int c = __builtin_amdgcn_readfirstlane(max(each < 1.0e9f ? static_cast<int>(each) + 1 : 1 << 30, least));
    int at = 0, slot = 0, ordinal = 0;
    for (int base = 0; base < a.seqs; base += HELD * kWave) {
        if (a.seqs > HELD * kWave) load(base);
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            if (base + k * kWave >= a.seqs) break;
            // A tile of t splits stands in t - 1 of the sums over all splits
            // but the first of the tiles that have more.
            const int splits = (steps_of(s[k].kv, STEP) + c - 1) / c;
            const int count = tiles_of(s[k].n, a.group, BM);
            int items = count * splits, slots = splits > 1 ? items : 0;
            if (count > 1 && splits > 1) {
                for (int t = (steps_of(tile_end(s[k], a.group, BM, 0), STEP) + c - 1) / c; t < splits; ++t) {
                    const int fewer = tiles_upto<BM, STEP>(s[k], a.group, count, t, c);
                    items -= fewer;
                    slots -= t == 1 ? 2 * fewer : fewer;
                }
            }
            const int upto = wave_scan(items), upto_slots = wave_scan(slots), upto_tiles = wave_scan(count);
            const int all = __builtin_amdgcn_readlane(upto, 63);
            if (item < at + all) {
                const int who = __builtin_ctzll(__ballot(item < at + upto));
                int local = item - at - __builtin_amdgcn_readlane(upto - items, who);
                out->b = base + k * kWave + (k == 0 ? __builtin_amdgcn_readlane(who_is, who) : who);
                out->slot = slot + __builtin_amdgcn_readlane(upto_slots - slots, who) + local;
                out->seq.first = __builtin_amdgcn_readlane(s[k].first, who);
                out->seq.n = __builtin_amdgcn_readlane(s[k].n, who);
                out->seq.kv = __builtin_amdgcn_readlane(s[k].kv, who);
                // Tiles of most splits first, each one's splits together.
                int t = __builtin_amdgcn_readlane(splits, who), upto_t = tiles_of(out->seq.n, a.group, BM);
                for (;; --t) {
                    const int upto_less = t > 1 ? tiles_upto<BM, STEP>(out->seq, a.group, upto_t, t - 1, c) : 0;
                    if (local < (upto_t - upto_less) * t) break;
                    local -= (upto_t - upto_less) * t;
                    upto_t = upto_less;
                }
                const int up = local / t;
                out->splits = t;
                out->tile = upto_t - 1 - up;
                out->split = local - up * t;
                out->slot -= out->split;
                out->ordinal = ordinal + __builtin_amdgcn_readlane(upto_tiles - count, who) + out->tile;
                return true;
            }
            at += all;
            slot += __builtin_amdgcn_readlane(upto_slots, 63);
            ordinal += __builtin_amdgcn_readlane(upto_tiles, 63);
        }
    }
    return false;
}

// What the attention launch leaves for the merge, one per tile and head.
struct Piece {
    int splits;   // 0 past the last tile
    int item;     // workgroup of its first split (its further splits: every kv_heads-th from there)
    int b, tile, slot;
    Sequence seq;
};

// The rows of a tile: row r is that of token i and head j of the key/value
// head's group, i and j the quotient and rest of first + r by the group.  That
// is less than 1024 + 128, so its product with ceil(2^21 / group) holds the
// quotient above bit 21: a division by a variable takes some 30 instructions.
struct TileRows {
    int token, head;   // of the step: those of i = 0 and j = 0
    int first, seen;   // positions that token i = 0 sees (negative ones: none)
};
struct RowAt {
    int64_t token, head;
    int seen;
};
__device__ __forceinline__ TileRows rows_of(const PagedAttnArgs& a, const Sequence& s, int kh, int row_at) {
    const int i = row_at / a.group;
    return {s.first + i, kh * a.group, row_at - i * a.group, s.kv - s.n + i + 1};
}
__device__ __forceinline__ RowAt row_at_of(const PagedAttnArgs& a, const TileRows& t, int r) {
    const uint32_t x = static_cast<uint32_t>(t.first + r);
    const int i = static_cast<int>(__umul24(x, static_cast<uint32_t>(a.group_inverse)) >> 21);
    return {t.token + i, t.head + static_cast<int>(x) - i * a.group, max(t.seen + i, 0)};
}

// Eight gates d .. d + 7 of a row.
__device__ __forceinline__ uint4 gate_of(const PagedAttnArgs& a, const RowAt& r, int d) {
    return ldg16(a.gate + r.token * a.gate_token_stride + r.head * a.gate_head_stride + d);
}
// Eight elements d .. d + 7 of a row's result: x times the gate (when there
// is one), rounded once.
template <bool FP16>
__device__ __forceinline__ void store_gated8(const PagedAttnArgs& a, const RowAt& r, int d, const float* v,
                                             uint4 gate) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = v[k];
    if (a.gate != nullptr) {
        float g[8];
        unpack16<FP16>(gate, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= sigmoid(g[k]);
    }
    *reinterpret_cast<uint4*>(a.out + r.token * a.out_token_stride + r.head * a.out_head_stride + d) =
        pack16<FP16>(x);
}
// The same of sums over l (0 for a row that sees nothing; where every score
// that it sees is -inf, l is 0 and the result NaN, as the softmax is).
template <bool FP16>
__device__ __forceinline__ void store_row8(const PagedAttnArgs& a, const RowAt& r, int d, const float* v, float l) {
    const uint4 gate = a.gate == nullptr ? make_uint4(0u, 0u, 0u, 0u) : gate_of(a, r, d);
    const float inv = r.seen > 0 ? __builtin_amdgcn_rcpf(l) : 0.0f;   // (an ulp, as in sigmoid)
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = v[k] * inv;
    store_gated8<FP16>(a, r, d, x, gate);
}

// ---- the tile kernel --------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) const uint8_t lds_u8;
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;

template <bool FP16>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (FP16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// gfx9 s_waitcnt immediate with expcnt at its maximum.
constexpr int wait_imm(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }
template <int VM, int LGKM>
__device__ __forceinline__ void wait_counts() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_imm(VM, LGKM));
    asm volatile("" ::: "memory");
}

// 16 bytes per lane from global memory straight into LDS (lane i's to lds_at +
// 16 i, lds_at the same in every lane).  Written as assembly because the
// compiler puts a wait for every outstanding one before each LDS read, which
// would end the read-ahead; it has no register output, and the waits are the
// kernel's own (wait_counts before the barrier that publishes a tile).
__device__ __forceinline__ void load_lds16(uint32_t lds_at, const void* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds_at), "v"(offset), "s"(base)
                 : "memory");
}
__device__ __forceinline__ void load_lds16(uint32_t lds_at, const void* address) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds_at), "v"(address)
                 : "memory");
}
// N of them for rows that follow each other in memory: an instruction's offset
// moves both addresses by 1024, the rest of the step in LDS goes through m0.
template <int N, int PAD>
__device__ __forceinline__ void load_lds16_n(uint32_t lds_at, const void* base, uint32_t offset) {
    static_assert(N == 1 || N == 2 || N == 4, "rows of a unit");
    if constexpr (N == 1)
        load_lds16(lds_at, base, offset);
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400"
                     :
                     : "s"(lds_at), "v"(offset), "s"(base), "n"(PAD)
                     : "memory", "scc");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x800\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:0xc00"
                     :
                     : "s"(lds_at), "v"(offset), "s"(base), "n"(PAD)
                     : "memory", "scc");
}

__device__ const uint4 kZeros = {0u, 0u, 0u, 0u};  // what rows past a tile's end read

// The LDS byte address of a __shared__ array.
__device__ __forceinline__ uint32_t lds_address(void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)p));
}

// Where a tile's rows are in LDS.  A load of the wave writes 1024 bytes in
// lane order, PER rows; the loads are PAD bytes apart, and a row's 16-byte
// chunks are moved by an exclusive or that depends on the row's place in its
// load only, so a lane's source offset is the same for every load.  Keys: the
// 16 rows that a read of 64 lanes takes per cycle at one chunk fall on 16
// different chunk places of 256 bytes; values: so do 4 chunks of 4 rows, which
// the transposing read takes.  Few bits are moved, so that the products' reads
// differ by constant offsets: one address for all keys at width 256 (two
// below), two for all values (four at width 128).
template <int D, bool VALUES>
struct Place {
    static constexpr int PER = 512 / D;   // rows per load
    static constexpr int PAD = VALUES ? (D == 256 ? 64 : 0) : (D == 256 ? 32 : 64);
    static constexpr int LOAD = 1024 + PAD;
    static constexpr int MOVED = VALUES ? (D == 256 ? 8 : D == 128 ? 12 : 4) : (D == 256 ? 1 : 3);   // chunk bits
    __device__ static __forceinline__ int swizzle(int row) {   // row within its load
        if constexpr (VALUES) return D == 256 ? 8 * row : D == 128 ? 4 * row : 4 * ((row >> 1) & 1);
        return D == 64 ? (row >> 1) & 3 : row;
    }
    static constexpr int bytes(int rows) { return rows / PER * LOAD; }
};

// 64 pages of a sequence: where each one's rows are in the two caches, lane i
// page first + i (in units of 16 bytes, so 32 bits reach 64 GiB).
struct PageWindow {
    uint32_t k, v;
    int first;
};
struct CacheView {
    const uint8_t* data;  // at the key/value head
    uint32_t pitch;       // bytes from one row to the next
};

// What a lane adds to a load's address: its row and its chunk.
template <int D, bool VALUES>
__device__ __forceinline__ uint32_t lane_offset(int lane, uint32_t pitch) {
    constexpr int CHUNKS = D / 8;
    const int r = lane / CHUNKS;
    return 16 * ((lane % CHUNKS) ^ Place<D, VALUES>::swizzle(r)) + r * pitch;
}

// ROWS rows from position `pos` on to `lds_at`, for the positions before `end`
// (zeros past it).  A page holds at least 8 rows, so one table entry serves
// that many, or all ROWS.  DENSE: the rows of a page follow each other.
template <int D, int ROWS, bool VALUES, bool DENSE>
__device__ __forceinline__ void stage_rows(const PagedAttnArgs& a, const CacheView& c, const PageWindow& win,
                                           uint32_t offset, int pos, int end, uint32_t lds_at) {
    typedef Place<D, VALUES> P;
    constexpr int UNIT = 8, N = UNIT / P::PER;
    const uint32_t pitch = DENSE ? 2 * D : c.pitch;   // bytes
    auto page_of = [&](int p) {
        const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(
            static_cast<int>(VALUES ? win.v : win.k), (p >> a.page_shift) - win.first));
        return c.data + (static_cast<uint64_t>(at) << 4) + static_cast<uint32_t>(p & ((1 << a.page_shift) - 1)) * pitch;
    };
    auto unit = [&](int u, const uint8_t* base) {
        if constexpr (DENSE) {
            load_lds16_n<N, P::PAD>(lds_at + P::bytes(u), base, offset);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                load_lds16(lds_at + P::bytes(u) + i * P::LOAD, base + i * P::PER * pitch, offset);
        }
    };
    if (pos + ROWS <= end) {
        if (ROWS <= 1 << a.page_shift) {
            const uint8_t* base = page_of(pos);
#pragma unroll
            for (int u = 0; u < ROWS; u += UNIT) unit(u, base + u * pitch);
        } else {
#pragma unroll 1
            for (int u = 0; u < ROWS; u += UNIT) unit(u, page_of(pos + u));
        }
    } else {
        int lane = threadIdx.x % kWave;
        asm volatile("" : "+v"(lane));   // nothing of this path stays in registers through the others
        const int lrow = lane / (D / 8);
#pragma unroll 1
        for (int r = 0; r < ROWS; r += P::PER) {
            const uint8_t* base = pos + r < end ? page_of(pos + r) : nullptr;
            load_lds16(lds_at + P::bytes(r), pos + r + lrow < end ? static_cast<const void*>(base + offset)
                                                                  : static_cast<const void*>(&kZeros));
        }
    }
}

// Orders the LDS reads of FRAGS operand fragments (READS instructions each)
// and the products that take them: AHEAD fragments before the first product,
// then one more after each.  Left to itself the compiler reads each fragment
// right before its product, to save registers, and every product waits for
// LDS (4096 positions over 28003 cached at width 256: 2.63 ms; 1.90 with four
// ahead in both products; five or more cost spills or gain nothing).
template <int FRAGS, int READS, int PRODUCTS = 1>
__device__ __forceinline__ void read_ahead() {
    constexpr int AHEAD = 4, PRODUCT = 0x8, LDS_READ = 0x100;
    __builtin_amdgcn_sched_group_barrier(LDS_READ, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < FRAGS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(PRODUCT, PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(LDS_READ, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(PRODUCT, PRODUCTS * AHEAD, 0);
}

// A product that no later operation is fused with.
__device__ __forceinline__ float opaque(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Highest value over the two lanes (q, q + 32) that share a row.
__device__ __forceinline__ float pair_max(float v) {
    const int x = __float_as_int(v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}

struct Partials {
    float* o;       // [slot][BM][D] sums of exp2(s - m) v
    float* ml;      // [slot][BM][2] m, sum of exp2(s - m)
    Piece* pieces;  // [tiles]
    int* dirty;     // [workgroups of the attention launch]: the split holds values that some of its rows must not see
    int tiles, workgroups;
};

constexpr float kLowest = -3.40282347e38f;  // the running maximum before any position: no finite score is below
constexpr float kSlack = 8.0f;              // a maximum may lag by 2^8 before sums are rescaled
// What is summed is relative to a point this far below the maximum (and above
// it by no more than the slack later on).  fp16 weights then are 2^7 to 2^15 at
// the top of its range, and keep all bits from 2^-21 of the highest down to
// where they have none, 2^-32; at 2^0 to 2^8 those were 2^-14 and 2^-25, which
// long rows of small weights add up to.  bf16 has the range of fp32.
template <bool FP16>
constexpr float kBelow = FP16 ? 7.0f : 0.0f;
// From this maximum on, a score's product with the scale is rounded before the
// maximum is taken off it: the exact product (one fused operation, below)
// differs from the maximum, which is a rounded one, by up to 2^-24 of it, and
// weights of 2^that would leave fp16's range.
constexpr float kRounded = 4194304.0f;

// WQ waves of 32 rows each over the same tiles of 32 NB positions, which they
// load together, the next one in flight (eight waves on one tile instead of two
// workgroups of four per CU took 2.03 ms where these took 1.82: their barriers
// keep them in step), or WK waves that share 32 rows and take tiles of their
// own.
template <bool FP16, int D, int WQ, int WK, int NB, bool DENSE>
__global__ __launch_bounds__(kWave * WQ * WK, (WK > 1 && D == 256) ? 1 : 2) void attend_tile_kernel(
    PagedAttnArgs a, Partials part, int target, int least) {
    constexpr int THREADS = kWave * WQ * WK;
    constexpr int KT = 32 * NB;           // positions of a tile
    constexpr int STEP = KT * WK;         // positions per step of the workgroup
    constexpr int BM = 32 * WQ;
    typedef Place<D, false> KP;
    typedef Place<D, true> VP;
    constexpr int KTILE = KP::bytes(KT), VTILE = VP::bytes(KT);   // bytes of a tile of keys, of values
    constexpr int STAGES = WK == 1 ? 2 : 1;
    constexpr int KS = D / 16, DB = D / 32;
    // 16-bit numbers that make up a weight in the second product.  Two for bf16
    // where few rows share keys and values: HBM sets the pace, the further
    // products are nearly free (one sequence of 1000 positions 13.5 -> 13.7 us,
    // 64 of 200-16000 201.8 -> 202.4) and the result is as far from 64 bits as
    // its own rounding is (1.7e-3; 2.1e-3 to 2.3e-3 with one).  fp16 keeps three
    // more bits in one (2.9e-4 against 2.1e-4).  Tiles of 128 rows are bound by
    // the products or by the chain of a step, and round a weight once, as the
    // Transformers forward does (two: 16 verify blocks 37.5 -> 38.9 us, 33.8 ->
    // 38.7 with their keys cached; 2048 positions 68 -> 91 us; 4096 over 28003
    // 1.66 -> 2.38 ms).
    constexpr int PARTS = WK > 1 && !FP16 ? 2 : 1;
    constexpr int ROWS = WK == 1 ? KT / WQ : KT;   // rows that a wave stages
    constexpr int LOADS = ROWS * D / 512;          // of a key or value tile, per wave
    constexpr int LDS = STAGES * WK * (KTILE + VTILE);
    __shared__ __align__(1024) uint8_t lds[LDS];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int hi = lane >> 5, q = lane & 31;
    const int item = blockIdx.x / a.kv_heads, kh = blockIdx.x % a.kv_heads;
    Split sp;
    int all_tiles;
    // (A path of its own for up to 64 sequences where latency counts: one
    // sequence of 1000 positions 14.3 -> 13.9 us; in the kernel of longer tiles
    // it gained nothing.)
    const bool live = WK > 1 && a.seqs <= kWave ? find_split<BM, STEP, 1>(a, item, target, least, &sp, &all_tiles)
                                                : find_split<BM, STEP, 4>(a, item, target, least, &sp, &all_tiles);
    if (threadIdx.x == 0 && item >= all_tiles && static_cast<int>(blockIdx.x) < part.tiles)
        part.pieces[blockIdx.x].splits = 0;
    if (!live) return;
    const int end = tile_end(sp.seq, a.group, BM, sp.tile);
    const int splits = sp.splits;
    const int row_at = sp.tile * BM;
    const int rows = min(BM, sp.seq.n * a.group - row_at);
    const TileRows places = rows_of(a, sp.seq, kh, row_at);
    const int least_seen = max(places.seen, 0);
    const int steps_all = steps_of(end, STEP), share = (steps_all + splits - 1) / splits;
    const int k0 = sp.split * share * STEP;
    const int k1 = min(end, k0 + share * STEP);
    const int steps = k1 > k0 ? (k1 - k0 + STEP - 1) / STEP : 0;
    const int wq = WK == 1 ? wave : 0, wk = WK == 1 ? 0 : wave;
    const int my_row = wq * 32 + q;
    const bool works = wq * 32 < rows;   // a wave without rows only stages

    // The maximum is taken before the scaling, so a negative scale turns the
    // queries' signs instead, and scale 0 is queries of 0 (a hidden score of
    // -inf must not meet a factor of 0).
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale == 0.0f ? 0u : 0xffffffffu;
    const float scale = a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale);
    const CacheView kc = {reinterpret_cast<const uint8_t*>(a.k_cache + kh * a.k_head_stride),
                          static_cast<uint32_t>(2 * a.k_row_stride)};
    const CacheView vc = {reinterpret_cast<const uint8_t*>(a.v_cache + kh * a.v_head_stride),
                          static_cast<uint32_t>(2 * a.v_row_stride)};
    const int32_t* table = a.table + static_cast<int64_t>(sp.b) * a.max_pages;
    const int last_page = max(end - 1, 0) >> a.page_shift;
    const int stage_row = WK == 1 ? wave * ROWS : 0;
    const int mine = k0 + wk * KT + stage_row;   // first position that this wave stages in a step
    bool bad = false, dirty = false;
    auto request_window = [&](int p) {
        return static_cast<uint32_t>(table[min((p >> a.page_shift) + lane, last_page)]);
    };
    auto window_of = [&](int p, uint32_t entry) {
        PageWindow w;
        w.first = p >> a.page_shift;
        bad |= end > 0 && entry >= static_cast<uint32_t>(a.pages);   // (of pages that the tile's rows see)
        entry = entry < static_cast<uint32_t>(a.pages) ? entry : 0;
        w.k = entry * static_cast<uint32_t>(a.k_page_stride >> 3);
        w.v = entry * static_cast<uint32_t>(a.v_page_stride >> 3);
        // waited for here, not (with every staged row) where it is used
        asm volatile("" : "+v"(w.k), "+v"(w.v));
        return w;
    };
    const int window_from = min(mine, max(end - 1, 0));
    PageWindow win = window_of(window_from, request_window(window_from));
    // Moves the window when the ROWS positions from p on are not within it.
    auto slide = [&](int p) {
        if (p < end && (min(p + ROWS, end) - 1) >> a.page_shift >= win.first + kWave)
            win = window_of(p, request_window(p));
    };
    const uint32_t lds0 = lds_address(lds);
    auto k_at = [&](int stage) { return lds0 + (WK == 1 ? stage : wk) * KTILE; };
    auto v_at = [&](int stage) { return lds0 + STAGES * WK * KTILE + (WK == 1 ? stage : wk) * VTILE; };
    const uint32_t k_offset = lane_offset<D, false>(lane, DENSE ? 2 * D : kc.pitch);
    const uint32_t v_offset = lane_offset<D, true>(lane, DENSE ? 2 * D : vc.pitch);
    auto stage_k = [&](int j) {
        stage_rows<D, ROWS, false, DENSE>(a, kc, win, k_offset, mine + j * STEP, k1,
                                          k_at(j & 1) + KP::bytes(stage_row));
    };
    auto stage_v = [&](int j) {
        stage_rows<D, ROWS, true, DENSE>(a, vc, win, v_offset, mine + j * STEP, k1,
                                         v_at(j & 1) + VP::bytes(stage_row));
    };

    f32x16 o[DB] = {};
    float m = kLowest, l = 0.0f;
    // A lane's places in the products' reads: keys row q (chunk 2 ks + hi),
    // values row 4 hi + i / 4 of 8 and chunk 4 db + 2 (lane / 16 % 2) + i % 4 / 2
    // for lane i of 16, 8 bytes each.
    const int v_row = 4 * hi + ((lane & 15) >> 2);
    const int k_off = q / KP::PER * KP::LOAD + q % KP::PER * 2 * D, k_move = KP::swizzle(q % KP::PER);
    const int v_off = v_row / VP::PER * VP::LOAD + v_row % VP::PER * 2 * D +
                      16 * (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    const int v_move = VP::swizzle(v_row % VP::PER);

    if (steps > 0) stage_k(0);
    // Queries: lane (q, hi) holds elements 16 ks + 8 hi .. + 7 of row q.
    uint4 qf[KS];
    int seen;
    {
        const RowAt r = row_at_of(a, places, my_row < rows ? my_row : 0);
        seen = my_row < rows ? r.seen : 0;
        const uint16_t* src = a.q + r.token * a.q_token_stride + r.head * a.q_head_stride;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = ldg16(src + 16 * ks + 8 * hi);
    }
    if (a.scale <= 0.0f) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qf[ks] = make_uint4((qf[ks].x ^ flip) & keep, (qf[ks].y ^ flip) & keep, (qf[ks].z ^ flip) & keep,
                                (qf[ks].w ^ flip) & keep);
    }
    // The queries are waited for here, with the first keys and in front of the
    // first values: the compiler, which does not count the staged rows, would
    // wait for every outstanding load at their first use inside the loop.
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
        asm volatile("" : "+v"(qf[ks].x), "+v"(qf[ks].y), "+v"(qf[ks].z), "+v"(qf[ks].w));
    if (steps > 0) stage_v(0);

    // Scores of the tile's KT positions from base, softmax, and the weights
    // packed for the second product.  S^T = K Q^T, so a lane holds 16 NB
    // positions of its row and the weights are the second product's operand as
    // they are: of a step of 16 positions lane (q, hi) holds 4 hi + {0..3,
    // 8..11}.  The product takes 16-bit operands, so the weights are rounded to
    // the tensors' type, or split into two numbers of it, the second what the
    // first leaves (15 bits and more of each weight); their sum is not rounded.
    auto scores = [&](uint32_t kt, int base, uint4 (&pw)[2 * NB * PARTS]) {
        f32x16 s[NB] = {};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                lds_u8* at = reinterpret_cast<lds_u8*>(kt + k_off + ((((2 * ks & KP::MOVED) + hi) ^ k_move) << 4));
                const u32x4 kv = *reinterpret_cast<lds_u32x4*>(at + nb * KP::bytes(32) + ((2 * ks & ~KP::MOVED) << 4));
                s[nb] = mfma32<FP16>(make_uint4(kv.x, kv.y, kv.z, kv.w), qf[ks], s[nb]);
            }
        read_ahead<NB * KS, 1>();
        if (base + KT > least_seen) {
            asm volatile("" ::: "memory");   // a branch: not selects in every step
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int p = base + 32 * nb + 8 * (i >> 2) + 4 * hi + (i & 3);
                    s[nb][i] = p < seen ? s[nb][i] : -__builtin_inff();
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[nb][i]);
        top = pair_max(top) * scale;
        // (m is kBelow below the maximum of its time; the difference, as a sum
        // with m may be rounded up to top)
        const bool grew = top - m > kSlack + kBelow<FP16>;
        if (__any(grew)) {
            // A row's own step: other rows may see what it does not.
            const float mn = grew ? __builtin_fmaxf(m, top - kBelow<FP16>) : m;
            const float fall = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= fall;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= fall;
        }
        float factor = scale, off = m;
        const bool coarse = __builtin_fabsf(m) > kRounded && m != kLowest;
        if (__any(coarse)) {
            factor = coarse ? 1.0f : scale;
            off = coarse ? 0.0f : m;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float product = s[nb][i] * scale;
                    s[nb][i] = coarse ? opaque(product) - m : s[nb][i];
                }
        }
        float sum = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][8 * k + j], factor, -off));
                    sum += w[j];
                }
                if constexpr (PARTS == 1) {
                    pw[2 * nb + k] = pack16<FP16>(w);
                } else {
                    // The upper half of the weight's bits, and what that leaves,
                    // kept above 0 with the weight: an infinite value's two
                    // products then have one sign, and a weight of 0 has none.
                    uint32_t high[4];
                    float rest[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        rest[j] = __builtin_amdgcn_fmed3f(
                            w[j] - __uint_as_float(__float_as_uint(w[j]) & 0xffff0000u), 1.17549435e-38f, w[j]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        high[j] = __builtin_amdgcn_perm(__float_as_uint(w[2 * j + 1]), __float_as_uint(w[2 * j]),
                                                        0x07060302u);
                    pw[4 * nb + 2 * k] = make_uint4(high[0], high[1], high[2], high[3]);
                    pw[4 * nb + 2 * k + 1] = pack16<false>(rest);
                }
            }
        l += sum;
    };
    auto values = [&](uint32_t vt, const uint4 (&pw)[2 * NB * PARTS]) {
        __builtin_amdgcn_sched_barrier(0);   // the order below is kept within its own region only
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                lds_u8* at = reinterpret_cast<lds_u8*>(vt + v_off + (((4 * db & VP::MOVED) ^ v_move) << 4));
                at += k * VP::bytes(16) + ((4 * db & ~VP::MOVED) << 4);
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
                const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + VP::bytes(8)));
                const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, up);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    o[db] = mfma32<FP16>(make_uint4(x.x, x.y, y.x, y.y), pw[k * PARTS + part], o[db]);
            }
        read_ahead<2 * NB * DB, 2, PARTS>();
    };
    // A value that is not finite among the tile's: all exponent bits set.
    auto look = [&](uint32_t vt) {
        constexpr uint32_t E = FP16 ? 0x7c00u : 0x7f80u;
        for (int i = WK == 1 ? threadIdx.x : lane; i < KT * D / 8; i += WK == 1 ? THREADS : kWave) {
            const u32x4 v = *reinterpret_cast<lds_u32x4*>(vt + i / kWave * VP::LOAD + i % kWave * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) dirty |= (v[j] & E) == E || ((v[j] >> 16) & E) == E;
        }
    };

    uint4 pw[2 * NB * PARTS];
    if constexpr (WK == 1) {
        for (int j = 0; j < steps; ++j) {
            const int base = k0 + j * STEP;
            wait_counts<0, 0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (j + 1 < steps) {
                slide(mine + (j + 1) * STEP);
                stage_k(j + 1);
                stage_v(j + 1);
            }
            if (end > least_seen && base + KT > least_seen) look(v_at(j & 1));
            if (works) {
                scores(k_at(j & 1), base, pw);
                values(v_at(j & 1), pw);
            }
        }
    } else {
        // A wave's tiles are its own: no barrier, and its next keys are on
        // their way during its values' product, the next values during its
        // keys'.
        for (int j = 0; j < steps; ++j) {
            const int base = k0 + j * STEP + wk * KT;
            wait_counts<LOADS, 15>();
            scores(k_at(0), base, pw);
            wait_counts<63, 0>();
            const bool more = j + 1 < steps;
            if (more) {
                slide(mine + (j + 1) * STEP);
                stage_k(j + 1);
                wait_counts<LOADS, 15>();
            } else {
                wait_counts<0, 15>();
            }
            if (end > least_seen && base + KT > least_seen) look(v_at(0));
            values(v_at(0), pw);
            wait_counts<63, 0>();
            if (more) stage_v(j + 1);
        }
    }
    {
        const int x = __float_as_int(l);
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        l = __int_as_float(r[0]) + __int_as_float(r[1]);
    }
    // (__syncthreads_or gives 0 or 1: the two flags one after the other.)
    const bool flags = __syncthreads_or(bad || dirty);
    const bool any_bad = flags && __syncthreads_or(bad);
    const bool any_dirty = flags && __syncthreads_or(dirty);
    if (threadIdx.x == 0) {
        part.dirty[blockIdx.x] = any_dirty && !any_bad;
        if (sp.split == 0)
            part.pieces[sp.ordinal * a.kv_heads + kh] = {splits, static_cast<int>(blockIdx.x), sp.b, sp.tile, sp.slot,
                                                         sp.seq};
    }
    const int64_t slot = static_cast<int64_t>(sp.slot + sp.split) * a.kv_heads + kh;
    if (any_bad) l = __builtin_nanf("");

    if constexpr (WK > 1) {
        // The waves' sums over their own positions, joined in LDS in the
        // waves' order.
        float* ml = reinterpret_cast<float*>(lds);           // [WK][32][2]
        float* acc = ml + WK * 32 * 2;                       // [WK][rows of the tile][D + 4]
        constexpr int PITCH = D + 4;
        constexpr int ROOM = (LDS - WK * 32 * 8) / (4 * WK * PITCH);   // rows that fit at once
        if (hi == 0) {
            ml[(wk * 32 + q) * 2] = m;
            ml[(wk * 32 + q) * 2 + 1] = l;
        }
        __syncthreads();
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = __builtin_fmaxf(top, ml[(w * 32 + q) * 2]);
        const float fall = __builtin_amdgcn_exp2f(m - top);
        for (int r0 = 0; r0 < rows; r0 += ROOM) {
            if (r0 > 0) __syncthreads();
            if (q >= r0 && q < min(rows, r0 + ROOM)) {
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(acc + (wk * ROOM + q - r0) * PITCH + 32 * db + 8 * g + 4 * hi) =
                            make_float4(o[db][4 * g] * fall, o[db][4 * g + 1] * fall, o[db][4 * g + 2] * fall,
                                        o[db][4 * g + 3] * fall);
            }
            __syncthreads();
            const int count = min(rows - r0, ROOM);
            for (int i = threadIdx.x; i < count * (D / 8); i += THREADS) {
                const int r = i / (D / 8), d = i % (D / 8) * 8;
                float v[8] = {};
#pragma unroll
                for (int w = 0; w < WK; ++w)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] += acc[(w * ROOM + r) * PITCH + d + k];
                float rm = kLowest, rl = 0.0f;
#pragma unroll
                for (int w = 0; w < WK; ++w) rm = __builtin_fmaxf(rm, ml[(w * 32 + r0 + r) * 2]);
#pragma unroll
                for (int w = 0; w < WK; ++w)
                    rl += ml[(w * 32 + r0 + r) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * 32 + r0 + r) * 2] - rm);
                if (splits > 1) {
                    const int64_t at = slot * BM + r0 + r;
                    *reinterpret_cast<float4*>(part.o + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(part.o + at * D + d + 4) = make_float4(v[4], v[5], v[6], v[7]);
                    if (d == 0) *reinterpret_cast<float2*>(part.ml + 2 * at) = make_float2(rm, rl);
                } else {
                    store_row8<FP16>(a, row_at_of(a, places, r0 + r), d, v, rl);
                }
            }
        }
    } else if (!works) {
    } else if (splits > 1) {
        // Partial rows as the lanes hold them: 1 KB per store.
        float4* to = reinterpret_cast<float4*>(part.o + (slot * BM + wq * 32) * D) + lane;
        if (hi == 0) *reinterpret_cast<float2*>(part.ml + 2 * (slot * BM + my_row)) = make_float2(m, l);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                to[(4 * db + g) * kWave] =
                    make_float4(o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]);
    } else {
        // Rows through LDS (the wave's own 32 rows, DBC blocks of 32 elements
        // at a time), so that 8 elements of a row leave per lane.
        constexpr int DBC = DB < 4 ? DB : 4;
        constexpr int CHUNKS = 8 * DBC;   // of four floats, per row
        static_assert(32 * 32 * DBC * 4 * WQ <= LDS, "the rows fit");
        float4* mine_at = reinterpret_cast<float4*>(lds) + wave * 32 * CHUNKS;
        const float inv = seen > 0 ? __builtin_amdgcn_rcpf(l) : 0.0f;
        constexpr int PER = kWave / (CHUNKS / 2), ROUNDS = 32 / PER;   // rows at a time
        const int c = lane % (CHUNKS / 2) * 2;
        auto row_of = [&](int i) { return wq * 32 + i * PER + lane / (CHUNKS / 2); };
        // All gates are requested in front of the first store: a load behind
        // stores is waited for only when those have reached memory.  The loop
        // below takes two rounds per pass and moves the rest of them down;
        // unrolled it would take longer to fetch than to run.
        constexpr int GATES = DB / DBC * ROUNDS;
        uint4 gates[GATES] = {};
        if (a.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < ROUNDS; ++i) {
                const RowAt r = row_at_of(a, places, min(row_of(i), rows - 1));
#pragma unroll
                for (int k = 0; k < DB / DBC; ++k) gates[k * ROUNDS + i] = gate_of(a, r, 32 * DBC * k + 4 * c);
            }
        }
#pragma unroll
        for (int k = 0; k < DB / DBC; ++k) {
            wave_lds_fence();
#pragma unroll
            for (int db = 0; db < DBC; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int at = 8 * db + 2 * g + hi;
                    const f32x16& x = o[DBC * k + db];
                    mine_at[q * CHUNKS + (at ^ (q % CHUNKS))] =
                        make_float4(x[4 * g] * inv, x[4 * g + 1] * inv, x[4 * g + 2] * inv, x[4 * g + 3] * inv);
                }
            wave_lds_fence();
#pragma unroll 1
            for (int i = 0; i < ROUNDS; i += 2) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = (i + j) * PER + lane / (CHUNKS / 2);
                    const float4 x = mine_at[r * CHUNKS + (c ^ (r % CHUNKS))];
                    const float4 y = mine_at[r * CHUNKS + ((c + 1) ^ (r % CHUNKS))];
                    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    if (wq * 32 + r < rows)
                        store_gated8<FP16>(a, row_at_of(a, places, wq * 32 + r), 32 * DBC * k + 4 * c, v, gates[j]);
                }
#pragma unroll
                for (int j = 2; j < GATES; ++j) gates[j - 2] = gates[j];
            }
        }
    }
}

// Joins the splits of each tile, in their order, and recomputes the rows of
// dirty tiles one by one.  NATIVE: partial rows as the tile kernel's lanes
// hold them, thread (wave, lane) takes that lane's elements of blocks
// blockIdx.y, ... of 32; else row by row, a row's splits over the four waves,
// then the waves, rows blockIdx.y, ....
template <bool FP16, int D, int BM, bool NATIVE>
__global__ __launch_bounds__(kThreads) void attend_merge_kernel(PagedAttnArgs a, Partials part) {
    constexpr int WAVES = kThreads / kWave;
    __shared__ __align__(16) float qs[WAVES][D];
    __shared__ float ps[WAVES][kWave];
    __shared__ int64_t vs[WAVES][kWave];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const Piece pc = part.pieces[blockIdx.x];
    if (pc.splits == 0) return;
    int dirty = 0;
    for (int s = lane; s < pc.splits; s += kWave) dirty |= part.dirty[pc.item + s * a.kv_heads];
    const bool any_dirty = __any(dirty);
    if (pc.splits == 1 && !any_dirty) return;
    const int kh = blockIdx.x % a.kv_heads, row_at = pc.tile * BM;
    const int rows = min(BM, pc.seq.n * a.group - row_at);
    const TileRows places = rows_of(a, pc.seq, kh, row_at);
    if (any_dirty) {
        for (int r = blockIdx.y * WAVES + wave; r < rows; r += gridDim.y * WAVES) {
            const RowAt at = row_at_of(a, places, r);
            attend_row<FP16, D>(a, pc.b, at.token, at.head, at.seen, qs[wave], ps[wave], vs[wave]);
        }
        return;
    }
    const int64_t slot = static_cast<int64_t>(pc.slot) * a.kv_heads + kh;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * BM;   // rows from one split to the next
    if constexpr (NATIVE) {
        constexpr int GROUPS = BM / 32, DB = D / 32;
        for (int w = wave; w < GROUPS; w += WAVES) {
            if (32 * w >= rows) break;
            const int hi = lane >> 5, r = 32 * w + (lane & 31);
            const float* ml = part.ml + 2 * (slot * BM + r);
            for (int db = blockIdx.y; db < DB; db += gridDim.y) {
                float4 v[4] = {};
                float m = kLowest, l = 0.0f;
                const float4* from = reinterpret_cast<const float4*>(part.o + (slot * BM + 32 * w) * D) +
                                     4 * db * kWave + lane;
                // Four splits at a time, all requested before the first is used.
                for (int s0 = 0; s0 < pc.splits; s0 += 4) {
                    float2 x[4];
                    float4 y[4][4] = {};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        x[k] = make_float2(kLowest, 0.0f);
                        if (s0 + k < pc.splits) {
                            x[k] = *reinterpret_cast<const float2*>(ml + 2 * (s0 + k) * step);
#pragma unroll
                            for (int g = 0; g < 4; ++g) y[k][g] = from[(s0 + k) * step * (D / 4) + g * kWave];
                        }
                    }
                    float top = m;
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = __builtin_fmaxf(top, x[k].x);
                    const float fall = __builtin_amdgcn_exp2f(m - top);
                    l *= fall;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        v[g].x *= fall; v[g].y *= fall; v[g].z *= fall; v[g].w *= fall;
                    }
                    m = top;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float f = __builtin_amdgcn_exp2f(x[k].x - m);
                        l = __builtin_fmaf(f, x[k].y, l);
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            v[g].x = __builtin_fmaf(f, y[k][g].x, v[g].x);
                            v[g].y = __builtin_fmaf(f, y[k][g].y, v[g].y);
                            v[g].z = __builtin_fmaf(f, y[k][g].z, v[g].z);
                            v[g].w = __builtin_fmaf(f, y[k][g].w, v[g].w);
                        }
                    }
                }
                // Lane (q, hi) holds elements 8 g + 4 hi .. + 3: pairs of
                // groups are exchanged so that each lane stores 8 in a row
                // (hi = 0 groups 0 and 2, hi = 1 groups 1 and 3).
#pragma unroll
                for (int g = 0; g < 4; g += 2) {
                    const float4 give = hi ? v[g] : v[g + 1], keep = hi ? v[g + 1] : v[g];
                    const float4 got = make_float4(__shfl_xor(give.x, 32), __shfl_xor(give.y, 32),
                                                   __shfl_xor(give.z, 32), __shfl_xor(give.w, 32));
                    const float4 lo = hi ? got : keep, up = hi ? keep : got;
                    const float x[8] = {lo.x, lo.y, lo.z, lo.w, up.x, up.y, up.z, up.w};
                    if (r < rows) store_row8<FP16>(a, row_at_of(a, places, r), 32 * db + 8 * (g + hi), x, l);
                }
            }
        }
    } else {
        constexpr int E = D / 8;   // lanes that store, eight elements each
        constexpr int F = D / 4;   // lanes that sum, four each
        __shared__ float2 sums[WAVES];
        for (int r = blockIdx.y; r < rows; r += gridDim.y) {
            const int64_t at = slot * BM + r;
            float m = kLowest, l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            // Four splits of the wave at a time, their sums and rows all
            // requested before the first is used.
            for (int s0 = wave; s0 < pc.splits; s0 += 4 * WAVES) {
                float2 x[4];
                float4 y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int s = s0 + k * WAVES;
                    x[k] = make_float2(kLowest, 0.0f);
                    y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (s < pc.splits) {
                        x[k] = *reinterpret_cast<const float2*>(part.ml + 2 * (at + s * step));
                        if (lane < F) y[k] = *reinterpret_cast<const float4*>(part.o + (at + s * step) * D + 4 * lane);
                    }
                }
                float top = m;
#pragma unroll
                for (int k = 0; k < 4; ++k) top = __builtin_fmaxf(top, x[k].x);
                const float fall = __builtin_amdgcn_exp2f(m - top);
                l *= fall;
                v.x *= fall; v.y *= fall; v.z *= fall; v.w *= fall;
                m = top;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float w = __builtin_amdgcn_exp2f(x[k].x - m);
                    l = __builtin_fmaf(w, x[k].y, l);
                    v.x = __builtin_fmaf(w, y[k].x, v.x);
                    v.y = __builtin_fmaf(w, y[k].y, v.y);
                    v.z = __builtin_fmaf(w, y[k].z, v.z);
                    v.w = __builtin_fmaf(w, y[k].w, v.w);
                }
            }
            if (lane < F) *reinterpret_cast<float4*>(&qs[wave][4 * lane]) = v;
            if (lane == 0) sums[wave] = make_float2(m, l);
            __syncthreads();
            if (wave == 0 && lane < E) {
                float top = kLowest;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) top = __builtin_fmaxf(top, sums[w].x);
                l = 0.0f;
                float x[8] = {};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float f = __builtin_amdgcn_exp2f(sums[w].x - top);
                    l = __builtin_fmaf(f, sums[w].y, l);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = __builtin_fmaf(f, qs[w][8 * lane + k], x[k]);
                }
                store_row8<FP16>(a, row_at_of(a, places, r), 8 * lane, x, l);
            }
            __syncthreads();
        }
    }
}

struct Shape {
    int bm, step, target, least;
};
// The kernel of a step.  Where every sequence's rows fit into 32: one tile of
// them, four waves on positions of their own, many splits (64 sequences of
// 200-16000 positions: 204 us with a target of 1024, 227 with 512, 252 with
// 2048; a split may be one step, so that a single sequence spreads).  Else
// tiles of 128 rows, two workgroups per CU: a target of 256, which with a part
// of a split per tile stays within the 512 places (16 verify blocks of 2-9
// positions over 1000-8000: 34.3 us, 35.0 with 320, 36.5 with 400, 37.0 with
// 192; 2048 positions from an empty cache: 73.5, 73.4, 72.4, 78; 128, where
// the latter has no splits: 45.7 and 88), and splits of at least 8 steps,
// whose partial rows cost about as much (the verify blocks: 35.6 us, 39.4 with
// 16).
Shape shape_of(int group, int max_new, int dim) {
    if (static_cast<int64_t>(max_new) * group <= 32) return {32, 128, 1024, 1};
    return {128, dim == 256 ? 32 : 64, 256, 8};
}

struct Layout {
    Partials part;
    size_t bytes;
};
Layout carve(void* base, int tokens, int seqs, int heads, int kv_heads, int dim, int max_new, int64_t capacity) {
    const int group = heads / kv_heads;
    const Shape sh = shape_of(group, max_new, dim);
    const int64_t tiles = static_cast<int64_t>(tokens) * group / sh.bm + (seqs < tokens ? seqs : tokens);
    // A tile has at most one split per `least` steps of what a row can hold;
    // the tiles of a sequence of several count up to twice.
    const int64_t most = (capacity / sh.step + sh.least) / sh.least;
    const int64_t share = (sh.bm == 32 ? 1 : 2) * (sh.target / kv_heads + 1);   // splits beyond one per tile, per head
    const int64_t per_head = tiles * most < share + tiles ? tiles * most : share + tiles;
    const int64_t workgroups = per_head * kv_heads;
    const int64_t splits = 2 * share * kv_heads + 16;   // (16: the work is summed in 24 bits)
    const int64_t slots = splits < workgroups ? splits : workgroups;
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* r = p + at;
        at += (bytes + 255) & ~static_cast<size_t>(255);
        return r;
    };
    Layout l;
    l.part.workgroups = static_cast<int>(workgroups);
    l.part.tiles = static_cast<int>(tiles * kv_heads);
    l.part.pieces = reinterpret_cast<Piece*>(take(l.part.tiles * sizeof(Piece)));
    l.part.dirty = reinterpret_cast<int*>(take(workgroups * 4));
    l.part.ml = reinterpret_cast<float*>(take(slots * sh.bm * 8));
    l.part.o = reinterpret_cast<float*>(take(slots * sh.bm * static_cast<size_t>(dim) * 4));
    l.bytes = at;
    return l;
}

template <bool FP16, int D, int WQ, int WK, int NB>
void launch_shape(const PagedAttnArgs& a, const Shape& sh, const Partials& part, int max_new, hipStream_t stream) {
    const dim3 grid(part.workgroups), block(kWave * WQ * WK);
    if (a.k_row_stride == D && a.v_row_stride == D)
        hipLaunchKernelGGL((attend_tile_kernel<FP16, D, WQ, WK, NB, true>), grid, block, 0, stream, a, part, sh.target,
                           sh.least);
    else
        hipLaunchKernelGGL((attend_tile_kernel<FP16, D, WQ, WK, NB, false>), grid, block, 0, stream, a, part,
                           sh.target, sh.least);
    // Merge workgroups per tile: a row each, or a block of 32 elements each.
    const int64_t rows = static_cast<int64_t>(max_new) * a.group;
    const unsigned each = WK == 1 ? D / 32 : static_cast<unsigned>(rows < 1 ? 1 : rows < 16 ? rows : 16);
    hipLaunchKernelGGL((attend_merge_kernel<FP16, D, 32 * WQ, WK == 1>), dim3(part.tiles, each), dim3(kThreads), 0,
                       stream, a, part);
}

template <bool FP16, int D>
hipError_t launch(const PagedAttnArgs& a, int max_new, const Partials& part, hipStream_t stream) {
    const Shape sh = shape_of(a.group, max_new, D);
    if (sh.bm == 32) launch_shape<FP16, D, 1, 4, 1>(a, sh, part, max_new, stream);
    else launch_shape<FP16, D, 4, 1, (D == 256 ? 1 : 2)>(a, sh, part, max_new, stream);
    return hipGetLastError();
}

}  // namespace

size_t paged_attn_workspace_bytes(int tokens, int seqs, int heads, int kv_heads, int dim, int max_new,
                                  int64_t capacity) {
    return carve(nullptr, tokens, seqs, heads, kv_heads, dim, max_new, capacity).bytes;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, bool fp16, int dim, int max_new, void* workspace,
                                  hipStream_t stream) {
    const Partials part = carve(workspace, a.tokens, a.seqs, a.heads, a.kv_heads, dim, max_new,
                                static_cast<int64_t>(a.max_pages) << a.page_shift).part;
    if (dim == 64) return fp16 ? launch<true, 64>(a, max_new, part, stream) : launch<false, 64>(a, max_new, part, stream);
    if (dim == 128)
        return fp16 ? launch<true, 128>(a, max_new, part, stream) : launch<false, 128>(a, max_new, part, stream);
    return fp16 ? launch<true, 256>(a, max_new, part, stream) : launch<false, 256>(a, max_new, part, stream);
}

}  // namespace lrmoe
