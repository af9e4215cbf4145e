// The gated delta rule in chunks of 64 tokens, as matrix products.  With G the
// running sum of g inside a chunk, S the state before it, k and q already
// normalized, the chunk's tokens i, j give
//     L_ij = e^(G_i - G_j) k_i . k_j   (j < i),   P_ij = scale e^(G_i - G_j) q_i . k_j   (j <= i),
//     R_i = v_i - e^(G_i) S^T k_i,     w = (I + L beta)^-1 R,     u = beta w,
//     out_i = scale e^(G_i) S^T q_i + sum_j P_ij u_j,
//     S <- e^(G_63) S + sum_j e^(G_63 - G_j) k_j u_j^T.
// Launch one computes what does not depend on the state for all chunks at once:
// T = (I + L beta)^-1, P and the factors.  Launch two goes through a
// sequence's chunks one after another, per value head and block of columns.
//
// Products are of bf16 matrix instructions with nothing rounded: q and k are
// bf16 as they come (an fp16 number is two bf16 ones), and an fp32 factor is
// split into three bf16 numbers whose sum it is, so that states, outputs and
// gradients are as good as sums in fp32.  (Two would leave 2^-18 of each factor
// out: of outputs that are rounded to bf16 0.3 % then came out a step off, 0.02 %
// of a recurrence in fp32, and what cancels is off without a bound.)  The raw q
// and k enter the products; their norms are factors of rows.
#include "scan.h"

namespace lrmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kPitch = 68;   // floats of a row of a 64 x 64 matrix in LDS

__device__ __forceinline__ f32x4 mfma_f16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool FP16>
__device__ __forceinline__ f32x4 mfma_raw(uint4 a, uint4 b, f32x4 c) {
    if constexpr (FP16) return mfma_f16(a, b, c);
    return mfma16x16x32(a, b, c);
}

// The sequence whose chunk slots hold slot c (the last one that begins at or
// before it), a wave at a time: 64 of them are looked at in one step.
__device__ __forceinline__ int find_sequence(const ScanArgs& a, int c) {
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + kWave - 1) / kWave;
        const int at = lo + (static_cast<int>(__lane_id()) + 1) * step;
        const bool before = at < hi && scan_first_chunk(a, at) <= c;
        const int n = __popcll(__ballot(before));
        lo += n * step;
        hi = min(lo + step, hi);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// A number of which the compiler knows nothing, least of all that it was there before.
__device__ __forceinline__ int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ uint4 frag16(const uint8_t* p, uint32_t at) { return *reinterpret_cast<const uint4*>(p + at); }

// Orders a wave's LDS accesses (it runs in step).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float power(double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x)); }

__device__ __forceinline__ double wave_scan_f64(double v) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const double below = __shfl_up(v, off);
        if (static_cast<int>(__lane_id()) >= off) v += below;
    }
    return v;
}

// ---- launch one: what does not depend on the state ------------------------------
//
// A workgroup has a chunk and a key head: its rows once, their products with one
// another, then per value head the inverse and the fragments.  Bound by what it
// writes, 37 KB per chunk and value head and 48 KB per chunk and key head of 128
// bf16 (8192 tokens, 16 / 32 heads: 69-73 us, 4.5 TB/s read and written).  38 KB
// of LDS, four workgroups per CU: one's stores hide the next one's substitution.

struct PrepareLds {
    float a[kChunk * kPitch];   // K rows, then L beta, then P
    float t[kChunk * kPitch];   // Q rows, then the inverse
    double sum[4][kChunk];      // of four heads at a time
    float beta[4][kChunk], rk[kChunk], rq[kChunk];
};

// The value of lane L of a lane's row of 16.
template <int L>
__device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + L, 0xf, 0xf, false));
}
// Subtracts row L's multiple from the rows below it.
template <int L>
__device__ __forceinline__ void eliminate(const float (&m)[16], float (&x)[4]) {
    if constexpr (L < 15) {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = __builtin_fmaf(-m[L], row_lane<L>(x[c]), x[c]);
        eliminate<L + 1>(m, x);
    }
}

// t = (I + a)^-1 for the strictly lower triangular a, by blocks of 16: those of
// the diagonal by substitution, a wave per block, lane n of group g with row n
// and columns 4 g .. + 3 (a row is handed to the others by a DPP broadcast);
// below, block column by block column, T_ij = -T_ii sum_k A_ik T_kj with fp32
// matrix instructions, a wave per block column.
__device__ __forceinline__ void invert(PrepareLds& lds, int wave, int lane) {
    const int n = lane % 16, g = lane / 16;
    {
        float m[16], x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(lds.a + (16 * wave + n) * kPitch + 16 * wave + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) m[4 * i + j] = v[j];
            x[i] = n == 4 * g + i ? 1.0f : 0.0f;
        }
        eliminate<0>(m, x);
        *reinterpret_cast<f32x4*>(lds.t + (16 * wave + n) * kPitch + 16 * wave + 4 * g) = (f32x4){x[0], x[1], x[2], x[3]};
    }
    __syncthreads();
    const int j = wave;
    for (int i = j + 1; i < 4; ++i) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = j; k < i; ++k) {
            const f32x4 row = *reinterpret_cast<const f32x4*>(lds.a + (16 * i + n) * kPitch + 16 * k + 4 * g);
            const float* col = lds.t + (16 * k + 4 * g) * kPitch + 16 * j + n;
#pragma unroll
            for (int s = 0; s < 4; ++s)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(row[s], col[s * kPitch], acc, 0, 0, 0);
        }
        f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
        const f32x4 row = *reinterpret_cast<const f32x4*>(lds.t + (16 * i + n) * kPitch + 16 * i + 4 * g);
#pragma unroll
        for (int s = 0; s < 4; ++s) out = __builtin_amdgcn_mfma_f32_16x16x4f32(row[s], acc[s], out, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) lds.t[(16 * i + 4 * g + r) * kPitch + 16 * j + n] = -out[r];
        wave_sync();
    }
    __syncthreads();
}

// Eight floats as the parts of a fragment, to to + part * kFragBytes.
template <int PARTS>
__device__ __forceinline__ void store_parts(uint8_t* to, const float (&x)[8]) {
    Split2 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = split2<PARTS>(x[2 * i], x[2 * i + 1]);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
        *reinterpret_cast<uint4*>(to + p * kFragBytes) =
            make_uint4(s[0].part[p], s[1].part[p], s[2].part[p], s[3].part[p]);
}

template <int D, bool FP16, bool GRAD>
__global__ __launch_bounds__(kThreads, 4) void scan_prepare(ScanArgs a, ScanChunks w) {
    constexpr int RAW = D + 8;   // 16-bit elements of a row in LDS
    constexpr int PARTS = FP16 ? 2 : 1;
    __shared__ PrepareLds lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int slot = blockIdx.x / a.key_heads, kh = blockIdx.x % a.key_heads;
    const int s = find_sequence(a, slot);
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    const int first = (slot - scan_first_chunk(a, s)) * kChunk;
    if (first < 0 || first >= seq.n || seq.n <= a.token_wise) return;
    const int count = min(seq.n - first, kChunk), t0 = seq.a + first;
    // g and beta of the wave's head among four.
    float raw_g;
    uint32_t raw_beta;
    auto load_gates = [&](int hv) {
        const int h = kh * a.group + min(hv + wave, a.group - 1);
        const int64_t t = t0 + min(lane, count - 1);
        raw_g = a.g[t * a.g_token + h];
        if (a.beta_fp32) raw_beta = static_cast<const uint32_t*>(a.beta)[t * a.beta_token + h];
        else raw_beta = static_cast<const uint16_t*>(a.beta)[t * a.beta_token + h];
    };
    load_gates(0);
    uint16_t* raw_k = reinterpret_cast<uint16_t*>(lds.a);
    uint16_t* raw_q = reinterpret_cast<uint16_t*>(lds.t);
    for (int i = tid; i < kChunk * D / 8; i += kThreads) {
        const int r = i / (D / 8), e = i % (D / 8) * 8;
        uint4 k = make_uint4(0u, 0u, 0u, 0u), q = k;
        if (r < count) {
            k = ldg16(a.k + static_cast<int64_t>(t0 + r) * a.k_token + kh * a.k_head + e);
            q = ldg16(a.q + static_cast<int64_t>(t0 + r) * a.q_token + kh * a.q_head + e);
        }
        *reinterpret_cast<uint4*>(raw_k + r * RAW + e) = k;
        *reinterpret_cast<uint4*>(raw_q + r * RAW + e) = q;
    }
    __syncthreads();
    // k_i . k_j and q_i . k_j for the row tile of the wave, and |q_i|^2.
    f32x4 kk[4], qk[4], qq = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 4; ++t) kk[t] = qk[t] = qq;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
        const int e = 32 * ks + 8 * g;
        const uint4 ak = *reinterpret_cast<const uint4*>(raw_k + (16 * wave + n) * RAW + e);
        const uint4 aq = *reinterpret_cast<const uint4*>(raw_q + (16 * wave + n) * RAW + e);
        qq = mfma_raw<FP16>(aq, aq, qq);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const uint4 b = *reinterpret_cast<const uint4*>(raw_k + (16 * t + n) * RAW + e);
            kk[t] = mfma_raw<FP16>(ak, b, kk[t]);
            qk[t] = mfma_raw<FP16>(aq, b, qk[t]);
        }
    }
    if (n / 4 == g) {
        f32x4 own = kk[0];
#pragma unroll
        for (int t = 1; t < 4; ++t) own = t == wave ? kk[t] : own;
        float k2 = own[0], q2 = qq[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            k2 = n % 4 == i ? own[i] : k2;
            q2 = n % 4 == i ? qq[i] : q2;
        }
        lds.rk[16 * wave + n] = a.normalize ? 1.0f / __builtin_sqrtf(k2 + 1e-6f) : 1.0f;
        lds.rq[16 * wave + n] = a.normalize ? 1.0f / __builtin_sqrtf(q2 + 1e-6f) : 1.0f;
    }
    // Fragments of K^T: row m of tile t is element 32 (t / 2) + 8 (m / 4) + 4 (t
    // % 2) + m % 4, so that a lane's rows of two tiles are eight in a row.
    const int64_t by_key = static_cast<int64_t>(slot) * a.key_heads + kh;
    for (int f = wave; f < D / 16 * 2; f += kThreads / kWave) {
        const int t = f / 2, ks = f % 2, d = 32 * (t / 2) + 8 * (n / 4) + 4 * (t % 2) + n % 4;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = elem16<FP16>(raw_k[(32 * ks + 16 * (j / 4) + 4 * g + j % 4) * RAW + d]);
        store_parts<PARTS>(w.kt + ((by_key * (D / 16 * 2) + f) * PARTS) * kFragBytes + lane * 16, x);
        if constexpr (GRAD) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = elem16<FP16>(raw_q[(32 * ks + 16 * (j / 4) + 4 * g + j % 4) * RAW + d]);
            store_parts<PARTS>(w.qt + ((by_key * (D / 16 * 2) + f) * PARTS) * kFragBytes + lane * 16, x);
        }
    }
    if constexpr (GRAD) {
        __syncthreads();   // (the norms)
        if (tid < 2 * kChunk) w.norms[by_key * 2 * kChunk + tid] = tid < kChunk ? lds.rk[tid] : lds.rq[tid - kChunk];
    }
    // Rows of K and Q as fragments: every block of columns reads them, and where a
    // token's row is a view of a longer one (16 KB apart) its lines meet in few of
    // the caches' channels (one prompt of 8192: 12 us more here, 262 -> 238 there).
    for (int ks = 0; ks < D / 32; ++ks) {
        const int from = (16 * wave + n) * RAW + 32 * ks + 8 * g;
        const int64_t at = (((by_key * 4 + wave) * (D / 32) + ks) * PARTS) * kFragBytes + lane * 16;
        auto store_row = [&](uint8_t* to, const uint16_t* raw) {
            const uint4 row = *reinterpret_cast<const uint4*>(raw + from);
            if constexpr (FP16) {
                float x[8];
                unpack16<FP16>(row, x);
                store_parts<PARTS>(to + at, x);
            } else {
                *reinterpret_cast<uint4*>(to + at) = row;
            }
        };
        store_row(w.kf, raw_k);
        if constexpr (!GRAD) store_row(w.qf, raw_q);
    }
    for (int hv = 0; hv < a.group; ++hv) {
        const int h = kh * a.group + hv;
        const int64_t by_head = static_cast<int64_t>(slot) * a.heads + h;
        __syncthreads();   // (rows and the last head's matrices are done with)
        if (hv % 4 == 0) {
            // Running sums (in powers of two) and factors of the next four heads, a
            // wave each.
            const float beta = a.beta_fp32 ? __uint_as_float(raw_beta) : elem16<FP16>(static_cast<uint16_t>(raw_beta));
            const bool in = lane < count;   // (rows past the sequence repeat its last one)
            const double sum = wave_scan_f64(in ? scan_log(raw_g) * 1.4426950408889634 : 0.0);
            lds.sum[wave][lane] = sum;
            lds.beta[wave][lane] = in ? beta : 0.0f;
            if (hv + wave < a.group) {
                if constexpr (GRAD) w.sums[(by_head + wave) * kChunk + lane] = sum;
                const double last = __shfl(sum, kWave - 1);
                const float decay = power(sum), rest = power(last - sum);
                float* vec = w.vec + (by_head + wave) * kVec;
                vec[lane] = in ? decay * lds.rk[lane] : 0.0f;
                vec[64 + lane] = in ? decay * lds.rq[lane] * a.scale : 0.0f;
                vec[128 + lane] = in ? rest * lds.rk[lane] : 0.0f;
                vec[192 + lane] = in ? beta : 0.0f;
                if (lane == kWave - 1) vec[256] = decay;
            }
            load_gates(hv + 4);
            __syncthreads();
        }
        const double* sums = lds.sum[hv % 4];
        const float* betas = lds.beta[hv % 4];
        float fade[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int j = 16 * t + n;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * g + r;
                fade[t][r] = power(sums[i] - sums[j]) * lds.rk[j];
                // (The gradient's T is (I + beta L)^-1: T beta is the same.)
                lds.a[i * kPitch + j] = j < i ? fade[t][r] * lds.rk[i] * betas[GRAD ? i : j] * kk[t][r] : 0.0f;
            }
        }
        __syncthreads();
        invert(lds, wave, lane);
        // A fragment of the wave's rows (for the gradient: of its columns) is eight
        // numbers of a lane.
        const int row = 16 * wave + n;
        auto eight = [&](const float* m, int ks, float (&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int o = 32 * ks + 16 * (j / 4) + 4 * g + j % 4, block = 2 * ks + j / 4;
                const bool in = GRAD ? block >= wave : block <= wave;
                x[j] = in ? m[GRAD ? o * kPitch + row : row * kPitch + o] : 0.0f;
            }
        };
        const int64_t blocks = by_head * kBlocks;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (GRAD ? 2 * ks + 1 < wave : 2 * ks > wave) continue;
            float x[8];
            eight(lds.t, ks, x);
            const int64_t block = blocks + (GRAD ? upper_block(ks, wave) : lower_block(ks, wave));
            store_parts<3>(w.t + block * 3 * kFragBytes + lane * 16, x);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int j = 16 * t + n;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * g + r;
                lds.a[i * kPitch + j] = j <= i ? fade[t][r] * lds.rq[i] * a.scale * qk[t][r] : 0.0f;
            }
        }
        if constexpr (GRAD) __syncthreads();   // (else a wave reads its own rows)
        else wave_sync();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (GRAD ? 2 * ks + 1 < wave : 2 * ks > wave) continue;
            float x[8];
            eight(lds.a, ks, x);
            const int64_t block = blocks + (GRAD ? upper_block(ks, wave) : lower_block(ks, wave));
            store_parts<3>(w.p + block * 3 * kFragBytes + lane * 16, x);
        }
    }
}

// ---- launch two: chunk after chunk -----------------------------------------------

constexpr int kChainThreads = 768;      // the chain, the outputs, the loads
constexpr int kChainGradThreads = 512;

// Four values of a lane as half a B fragment (element 4 half on), in parts.
template <int PARTS, int KS, int NC>
__device__ __forceinline__ void put_parts(uint4 (&to)[PARTS][KS][NC][kWave], int ks, int half, int c, int lane, f32x4 x) {
    const Split2 lo = split2<PARTS>(x[0], x[1]), hi = split2<PARTS>(x[2], x[3]);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
        reinterpret_cast<uint2*>(&to[p][ks][c][lane])[half] = make_uint2(lo.part[p], hi.part[p]);
}

// Four rows of a lane's NC columns of an fp32 matrix [rows][value_dim].
template <int NC>
__device__ __forceinline__ void put_rows(float* to, int value_dim, const f32x4 (&x)[NC]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (NC == 1) to[i * value_dim] = x[0][i];
        else *reinterpret_cast<float2*>(to + i * value_dim) = make_float2(x[0][i], x[1][i]);
    }
}

// The NC 16-bit values of a lane's columns, and one of them.
template <int NC>
__device__ __forceinline__ uint32_t load_cols(const uint8_t* p, uint32_t at) {
    if constexpr (NC == 1) return *reinterpret_cast<const uint16_t*>(p + at);
    return *reinterpret_cast<const uint32_t*>(p + at);
}
template <bool FP16>
__device__ __forceinline__ float col_value(uint32_t v, int c) {
    return elem16<FP16>(static_cast<uint16_t>(c ? v >> 16 : v));
}
template <int NC, bool FP16>
__device__ __forceinline__ uint32_t pack_cols(const f32x4 (&x)[NC], int i) {
    if constexpr (NC == 1) return pack16_2<FP16>(x[0][i], 0.0f);
    return pack16_2<FP16>(x[0][i], x[1][i]);
}
template <int NC>
__device__ __forceinline__ void store_cols(uint16_t* to, uint32_t v) {
    if constexpr (NC == 1) *to = static_cast<uint16_t>(v);
    else *reinterpret_cast<uint32_t*>(to) = v;
}

// A workgroup's part of the work: a sequence, a value head and a block of
// columns. Blocks that share fragments (those of a key head, or of a head where
// those are too few) follow each other on one XCD, whose cache holds them, and
// their groups go round the XCDs, so that each sequence is spread over all; up
// to 64 sequences take their turns from the longest on (one prompt of 1500 tokens
// among five of 300 and more: 225 -> 133 us).
struct ScanItem {
    int s, h, cb;
    bool in;
};
__device__ __forceinline__ int longest_first(const ScanArgs& a, int rank) {
    if (a.seqs > kWave || a.seqs == 1) return rank;
    const int lane = static_cast<int>(__lane_id());
    const int n = lane < a.seqs ? scan_seq(a.starts, lane, a.tokens).n : -1;
    int place = 0;
    for (int i = 0; i < a.seqs; ++i) {
        const int other = __builtin_amdgcn_readlane(n, i);
        place += other > n || (other == n && i < lane);
    }
    return __builtin_ctzll(__ballot(lane < a.seqs && place == rank));
}
__device__ __forceinline__ ScanItem scan_item(const ScanArgs& a, int columns, int share) {
    const int blocks = a.value_dim / columns, total = a.seqs * a.heads * blocks;
    const int xcd = blockIdx.x % 8, i = blockIdx.x / 8;
    const int item = (i / share * 8 + xcd) * share + i % share;
    if (item >= total) return {0, 0, 0, false};
    return {longest_first(a, item / blocks / a.heads), item / blocks % a.heads, item % blocks, true};
}
struct ScanGrid {
    int share;
    uint32_t blocks;
};
ScanGrid scan_grid(const ScanArgs& a, int columns) {
    const int blocks = a.value_dim / columns, total = a.seqs * a.heads * blocks;
    int share = blocks * a.group;
    if (total / share < 16) share = blocks;
    if (total / share < 16) share = 1;
    const int groups = (total + share - 1) / share;
    return {share, static_cast<uint32_t>((groups + 7) / 8 * 8) * share};
}

// Waves 0 to 3 have the state's rows of the tiles w TPW .. + TPW - 1, in the
// accumulators of its own update (column NC n + c of the block in lane n of a
// group and tile c), and the token rows of tile w on the way there; waves 4 to
// 7 the outputs of those rows; waves 8 to 11 read what the chain needs, a chunk
// ahead. The products hand their results on through LDS, as the B fragments of
// the next ones, which the lanes write as they hold them. A step is a chain of
// three products and hand-overs, and the instructions of one wave on each SIMD;
// the other waves' fill the gaps.  That chain bounds a long sequence (8192 tokens,
// 32 heads of 128: 128 steps of 2.1 us, 262-271 us; the chain by itself 145), and
// with a tape HBM joins it (4378 tokens of five sequences: 136 us for 448 MB).
// Loads by the chain's own waves took 9 % longer.
template <int D, int NC, int PARTS>
struct ScanLds {
    uint4 s[3][D / 32][NC][kWave];
    uint4 r[3][2][NC][kWave];
    uint4 u[3][2][NC][kWave];    // for the outputs
    uint4 uk[3][2][NC][kWave];   // times the factors of K^T U
    // What waves 8 to 11 have read for waves 0 to 3.
    uint4 k[4][D / 32 * PARTS][kWave], t[4][6][kWave], kt[4][D / 64 * 2 * PARTS][kWave];
    f32x4 vec[2][4][16];         // the factors, of two chunks
    float decay[2];
    uint32_t v[4][4][kWave];
    int odd[4];                  // whether a wave has met a number that is not finite
};

template <int D, int NC, bool FP16, bool TAPE>
__global__ __launch_bounds__(kChainThreads, 3) void scan_chunks(ScanArgs a, ScanChunks w, int share) {
    constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64, KS = D / 32;
    __shared__ ScanLds<D, NC, PARTS> lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int role = __builtin_amdgcn_readfirstlane(tid / kWave), wave = role % 4;
    const ScanItem item = scan_item(a, 16 * NC, share);
    if (!item.in) return;
    const int s = item.s, h = item.h, kh = h / a.group, col0 = 16 * NC * item.cb, col = col0 + NC * n;
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    if (a.clear && (s == 0 || s == a.seqs - 1)) {
        const int head = min(max(a.starts[0], 0), a.tokens), tail = min(max(a.starts[a.seqs], 0), a.tokens);
        uint16_t* row = a.out + h * a.out_head + col0;
        if (s == 0)
            for (int i = tid; i < head * 16 * NC; i += kChainThreads)
                row[i / (16 * NC) * a.out_token + i % (16 * NC)] = 0;
        if (s == a.seqs - 1)
            for (int i = tid; i < (a.tokens - tail) * 16 * NC; i += kChainThreads)
                row[(tail + i / (16 * NC)) * a.out_token + i % (16 * NC)] = 0;
    }
    if (seq.n <= a.token_wise) return;   // (the next launch's)
    uint32_t* flag = w.flags + (static_cast<int64_t>(s) * a.heads + h) * (a.value_dim / 16) + NC * item.cb;
    const int into = scan_slot(a.into, s, a.pool);
    const bool fresh = a.initial == nullptr || (a.fresh != nullptr && a.fresh[s] != 0);
    const int from = fresh ? 0 : scan_slot(a.from, s, a.pool);
    if (into < 0 || from < 0) {
        if (tid < NC) flag[tid] = 0;
        return;
    }
    const int chunks = (seq.n + kChunk - 1) / kChunk;
    const int64_t slot0 = scan_first_chunk(a, s);
    // Addresses are a scalar base per chunk and offsets of 32 bits; rows past the
    // sequence repeat its last one (their factors are 0, and their u).
    const int r0 = 16 * wave + 4 * g;
    const uint32_t frag = lane * 16;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    auto load_rows = [&](uint4 (&to)[KS][PARTS], const uint8_t* frags, int ch) {
        const uint8_t* at = frags + (((slot0 + ch) * a.key_heads + kh) * 4 + wave) * KS * PARTS * kFragBytes;
#pragma unroll
        for (int i = 0; i < KS * PARTS; ++i) to[i / PARTS][i % PARTS] = frag16(at + i * kFragBytes, frag);
    };
    auto load_blocks = [&](uint4 (&to)[2][3], const uint8_t* blocks, int ch) {
        const uint8_t* at = blocks + ((slot0 + ch) * a.heads + h) * kBlocks * 3 * kFragBytes;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            to[0][p] = frag16(at + (lower_block(0, wave) * 3 + p) * kFragBytes, frag);
            to[1][p] = frag16(at + (lower_block(1, max(wave, 2)) * 3 + p) * kFragBytes, frag);
        }
    };
    if (role >= 8) {
        uint4 k[KS][PARTS], t[2][3], kt[TPW][2][PARTS];
        uint32_t v[4];
        f32x4 vec;
        float decay;
        auto load_kt = [&](int ch) {
            const uint8_t* at = w.kt + (((slot0 + ch) * a.key_heads + kh) * (D / 16) + wave * TPW) * 2 * PARTS * kFragBytes;
#pragma unroll
            for (int i = 0; i < TPW * 2 * PARTS; ++i)
                kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = frag16(at + i * kFragBytes, frag);
        };
        auto load_values = [&](int ch) {
            const float* from = w.vec + ((slot0 + ch) * a.heads + h) * kVec;
            vec = *reinterpret_cast<const f32x4*>(from + 64 * wave + 4 * n);
            decay = from[256];
            const uint8_t* at = reinterpret_cast<const uint8_t*>(a.v + static_cast<int64_t>(seq.a + ch * kChunk) * a.v_token +
                                                                 h * a.v_head + col0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t row = min(r0 + i, seq.n - 1 - ch * kChunk);
                v[i] = load_cols<NC>(at, row * (2 * static_cast<uint32_t>(a.v_token)) + 2 * NC * n);
            }
        };
        auto put_k = [&](int ch) {
#pragma unroll
            for (int i = 0; i < KS * PARTS; ++i) lds.k[wave][i][lane] = k[i / PARTS][i % PARTS];
#pragma unroll
            for (int i = 0; i < 4; ++i) lds.v[wave][i][lane] = v[i];
            if (g == 0) lds.vec[ch % 2][wave][n] = vec;
            if (wave == 3) lds.decay[ch % 2] = decay;
        };
        auto put_t = [&] {
#pragma unroll
            for (int i = 0; i < 6; ++i) lds.t[wave][i][lane] = t[i / 3][i % 3];
        };
        if (chunks > 0) {
            load_rows(k, w.kf, 0);
            load_values(0);
            load_blocks(t, w.t, 0);
            put_k(0);
            put_t();
            // (In the loop's order, so that its waits count the same loads.)
            __builtin_amdgcn_sched_barrier(0);
            load_kt(0);
            __builtin_amdgcn_sched_barrier(0);
            load_rows(k, w.kf, min(1, chunks - 1));
            load_values(min(1, chunks - 1));
            __builtin_amdgcn_sched_barrier(0);
            load_blocks(t, w.t, min(1, chunks - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int ch = 0; ch < chunks; ++ch) {
            const int next = min(ch + 1, chunks - 1), after = min(ch + 2, chunks - 1);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TPW * 2 * PARTS; ++i) lds.kt[wave][i][lane] = kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS];
            __builtin_amdgcn_sched_barrier(0);
            load_kt(next);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            put_k(next);
            __builtin_amdgcn_sched_barrier(0);
            load_rows(k, w.kf, after);
            load_values(after);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            put_t();
            __builtin_amdgcn_sched_barrier(0);
            load_blocks(t, w.t, after);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        return;
    }
    if (role >= 4) {
        __builtin_amdgcn_s_setprio(1);
        uint4 q[KS][PARTS], p[2][3];
        uint32_t packed[4];   // the last chunk's outputs
        auto store = [&](int ch) {
            const int left = seq.n - ch * kChunk;
            uint16_t* to = a.out + static_cast<int64_t>(seq.a + ch * kChunk + r0) * a.out_token + h * a.out_head + col;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + i < left) store_cols<NC>(to + i * a.out_token, packed[i]);
        };
        if (chunks > 0) {
            load_rows(q, w.qf, 0);
            __builtin_amdgcn_sched_barrier(0);
            load_blocks(p, w.p, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int ch = 0; ch < chunks; ++ch) {
            const int next = min(ch + 1, chunks - 1);
            __syncthreads();
            f32x4 o[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) o[c] = zero;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int b = 0; b < 3; ++b)
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const uint4 f = lds.s[b][i][c][lane];
#pragma unroll
                        for (int r = 0; r < PARTS && r + b < 3; ++r) o[c] = mfma16x16x32(q[i][r], f, o[c]);
                    }
            __builtin_amdgcn_sched_barrier(0);
            load_rows(q, w.qf, next);
            __builtin_amdgcn_sched_barrier(0);
            {
                const f32x4 fq = lds.vec[ch % 2][1][4 * wave + g];
#pragma unroll
                for (int c = 0; c < NC; ++c) o[c] *= fq;
            }
            __syncthreads();
            if (ch > 0) store(ch - 1);   // (these waves have nothing else between here)
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (2 * j > wave) continue;
#pragma unroll
                for (int b = 0; b < 3; ++b)
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const uint4 f = lds.u[b][j][c][lane];
#pragma unroll
                        for (int r = 0; r + b < 3; ++r) o[c] = mfma16x16x32(p[j][r], f, o[c]);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_blocks(p, w.p, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) packed[i] = pack_cols<NC, FP16>(o, i);
        }
        if (chunks > 0) store(chunks - 1);
        __syncthreads();
        return;
    }
    const int64_t size = static_cast<int64_t>(D) * a.value_dim;
    // The first of the lane's four rows of tile x.
    auto row_of = [&](int x) {
        const int t = wave * TPW + x;
        return 32 * (t / 2) + 8 * g + 4 * (t % 2);
    };
    f32x4 S[TPW][NC];
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                S[x][c][i] = fresh ? 0.0f
                                   : a.initial[(static_cast<int64_t>(from) * a.heads + h) * size +
                                               static_cast<int64_t>(row_of(x) + i) * a.value_dim + col + c];
    float* tape_s = reinterpret_cast<float*>(a.tape);
    float* tape_w = tape_s + tape_states(w.slots, a.heads, D, a.value_dim);
    __builtin_amdgcn_s_setprio(2);
    if (lane == 0) lds.odd[wave] = 0;
    bool odd = false;   // a number that is not finite, or whose first bf16 part may not be (from 2^127 on)
    for (int ch = 0; ch < chunks; ++ch) {
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                put_parts<3>(lds.s, (wave * TPW + i) / 2, (wave * TPW + i) % 2, c, lane, S[i][c]);
        __syncthreads();
        uint4 k[KS * PARTS];
#pragma unroll
        for (int i = 0; i < KS * PARTS; ++i) k[i] = lds.k[wave][i][lane];
        f32x4 r[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) r[c] = zero;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.s[p][i][c][lane];
#pragma unroll
                    for (int x = 0; x < PARTS && x + p < 3; ++x) r[c] = mfma16x16x32(k[i * PARTS + x], b, r[c]);
                }
        const f32x4 fk = lds.vec[ch % 2][0][4 * wave + g], fu = lds.vec[ch % 2][2][4 * wave + g];
        const f32x4 beta = lds.vec[ch % 2][3][4 * wave + g];
        const float decay = lds.decay[ch % 2];
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lds.v[wave][i][lane];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[c][i] = col_value<FP16>(v[i], c) - fk[i] * r[c][i];
            put_parts<3>(lds.r, wave / 2, wave % 2, c, lane, r[c]);
        }
        if constexpr (TAPE) {
            float* to = tape_s + ((slot0 + ch) * a.heads + h) * size + col;
#pragma unroll
            for (int i = 0; i < TPW; ++i) put_rows<NC>(to + row_of(i) * a.value_dim, a.value_dim, S[i]);
        }
        __syncthreads();
        f32x4 bare[NC];   // w: u before its beta
#pragma unroll
        for (int c = 0; c < NC; ++c) bare[c] = zero;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * i > wave) continue;
            uint4 t[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) t[p] = lds.t[wave][3 * i + p][lane];
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.r[p][i][c][lane];
#pragma unroll
                    for (int x = 0; x + p < 3; ++x) bare[c] = mfma16x16x32(t[x], b, bare[c]);
                }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const f32x4 u = bare[c] * beta;
            put_parts<3>(lds.u, wave / 2, wave % 2, c, lane, u);
            put_parts<3>(lds.uk, wave / 2, wave % 2, c, lane, u * fu);
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (__float_as_uint(u[i]) & 0x7f800000u) >= 0x7f000000u;
        }
        if constexpr (TAPE)
            put_rows<NC>(tape_w + (((slot0 + ch) * a.heads + h) * kChunk + r0) * a.value_dim + col, a.value_dim, bare);
        __syncthreads();
        uint4 kt[TPW * 2 * PARTS];
#pragma unroll
        for (int i = 0; i < TPW * 2 * PARTS; ++i) kt[i] = lds.kt[wave][i][lane];
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) S[i][c] *= decay;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.uk[p][j][c][lane];
#pragma unroll
                    for (int i = 0; i < TPW; ++i)
#pragma unroll
                        for (int x = 0; x < PARTS && x + p < 3; ++x) S[i][c] = mfma16x16x32(kt[(2 * i + j) * PARTS + x], b, S[i][c]);
                }
    }
    // (What u times its factor, or the last update, may have come to.)
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (__float_as_uint(S[x][c][i]) & 0x7f800000u) == 0x7f800000u;
    // Where a value was not finite, a product's zero weights have let it through
    // to earlier tokens: the next launch goes through these columns again.
    if (__ballot(odd) != 0 && lane == 0) lds.odd[wave] = 1;
    __syncthreads();
    if ((lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3]) != 0) {
        if (tid < NC) flag[tid] = 1;
        return;
    }
    if (tid < NC) flag[tid] = 0;
#pragma unroll
    for (int x = 0; x < TPW; ++x)
        put_rows<NC>(a.final + (static_cast<int64_t>(into) * a.heads + h) * size +
                         static_cast<int64_t>(row_of(x)) * a.value_dim + col,
                     a.value_dim, S[x]);
}

// ---- the gradient: chunk after chunk, backwards -----------------------------------

// With dS the gradient of the state after a chunk and do that of its outputs,
//     X_j = sum_i P_ij do_i + e^(G_63 - G_j) dS^T k_j,     du = ((I + beta L)^-1)^T X,     dR = beta du = dv,
//     dS <- e^(G_63) dS + sum_i scale e^(G_i) q_i do_i^T - sum_i e^(G_i) k_i dR_i^T:
// the forward launch with the matrices transposed, for the same columns. Waves 0
// to 3 have the chain; waves 4 to 7 compute the two sums over do, which need no
// dS, a chunk ahead.  Bound as the forward launch is (the same 4378 tokens: 159 us
// for 448 MB).
template <int D, int NC, int PARTS>
struct ScanGradLds {
    uint4 s[3][D / 32][NC][kWave];
    uint4 x[3][2][NC][kWave];
    uint4 rk[3][2][NC][kWave];           // - dR times the factors of k
    uint4 o[PARTS][2][NC][kWave];        // do
    uint4 oq[3][2][NC][kWave];           // do times the factors of q
    f32x4 y[4][NC][kWave];               // sum P do, as the chain's accumulators
    f32x4 z[2][D / 16][NC][kWave];       // sum q do, of two chunks
};

template <int D, bool FP16>
__global__ __launch_bounds__(kChainGradThreads, 2) void scan_chunks_grad(ScanArgs a, ScanGradArgs d, ScanChunks w, int share) {
    constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64, KS = D / 32, NC = 2;
    __shared__ ScanGradLds<D, NC, PARTS> lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int role = __builtin_amdgcn_readfirstlane(tid / kWave), wave = role % 4;
    const ScanItem item = scan_item(a, 16 * NC, share);
    if (!item.in) return;
    const int s = item.s, h = item.h, kh = h / a.group, col0 = 16 * NC * item.cb, col = col0 + NC * n;
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    if (s == 0 || s == a.seqs - 1) {
        // Rows of no sequence have no gradient.
        const int head = min(max(a.starts[0], 0), a.tokens), tail = min(max(a.starts[a.seqs], 0), a.tokens);
        auto clear = [&](int from, int to) {
            const int rows = to - from;
            for (int i = tid; i < rows * 32; i += kChainGradThreads)
                d.dv[(static_cast<int64_t>(from + i / 32) * a.heads + h) * a.value_dim + col0 + i % 32] = 0;
            if (item.cb != 0) return;
            for (int i = tid; i < rows; i += kChainGradThreads) {
                const int64_t at = static_cast<int64_t>(from + i) * a.heads + h;
                d.dg[at] = 0.0f;
                if (a.beta_fp32) static_cast<float*>(d.dbeta)[at] = 0.0f;
                else static_cast<uint16_t*>(d.dbeta)[at] = 0;
            }
            if (h % a.group != 0) return;
            for (int i = tid; i < rows * D; i += kChainGradThreads) {
                const int64_t at = (static_cast<int64_t>(from + i / D) * a.key_heads + kh) * D + i % D;
                d.dq[at] = 0;
                d.dk[at] = 0;
            }
        };
        if (s == 0) clear(0, head);
        if (s == a.seqs - 1) clear(tail, a.tokens);
    }
    const int chunks = (seq.n + kChunk - 1) / kChunk;
    const int64_t slot0 = scan_first_chunk(a, s);
    const int r0 = 16 * wave + 4 * g;
    const uint32_t frag = lane * 16;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    auto load_blocks = [&](uint4 (&to)[2][3], const uint8_t* blocks, int ch) {
        const uint8_t* at = blocks + ((slot0 + ch) * a.heads + h) * kBlocks * 3 * kFragBytes;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            to[0][p] = frag16(at + (upper_block(0, min(wave, 1)) * 3 + p) * kFragBytes, frag);
            to[1][p] = frag16(at + (upper_block(1, wave) * 3 + p) * kFragBytes, frag);
        }
    };
    auto load_transposed = [&](uint4 (&to)[TPW][2][PARTS], const uint8_t* frags, int ch) {
        const uint8_t* at = frags + (((slot0 + ch) * a.key_heads + kh) * (D / 16) + wave * TPW) * 2 * PARTS * kFragBytes;
#pragma unroll
        for (int i = 0; i < TPW * 2 * PARTS; ++i)
            to[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = frag16(at + i * kFragBytes, frag);
    };
    auto factors = [&](int ch, int kind) {
        return *reinterpret_cast<const f32x4*>(w.vec + ((slot0 + ch) * a.heads + h) * kVec + 64 * kind + r0);
    };
    if (role >= 4) {
        if (chunks == 0) return;
        uint32_t o[4];
        uint4 pt[2][3], qt[TPW][2][PARTS];
        f32x4 fq;
        auto load_out = [&](int ch) {
            fq = factors(ch, 1);
            const uint8_t* at = reinterpret_cast<const uint8_t*>(
                d.d_out + static_cast<int64_t>(seq.a + ch * kChunk) * d.d_out_token + h * d.d_out_head + col0);
            const int left = seq.n - ch * kChunk;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t row = min(r0 + i, left - 1);
                o[i] = load_cols<NC>(at, row * (2 * static_cast<uint32_t>(d.d_out_token)) + 2 * NC * n);
            }
        };
        auto put_out = [&](int ch) {
            const int left = seq.n - ch * kChunk;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4 x;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = r0 + i < left ? col_value<FP16>(o[i], c) : 0.0f;
                put_parts<PARTS>(lds.o, wave / 2, wave % 2, c, lane, x);
                put_parts<3>(lds.oq, wave / 2, wave % 2, c, lane, x * fq);
            }
        };
        f32x4 y[NC], z[TPW][NC];
        auto products = [&] {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                y[c] = zero;
#pragma unroll
                for (int i = 0; i < TPW; ++i) z[i][c] = zero;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        const uint4 b = lds.o[p][j][c][lane];
                        if (2 * j + 1 < wave) continue;
#pragma unroll
                        for (int x = 0; x + p < 3; ++x) y[c] = mfma16x16x32(pt[j][x], b, y[c]);
                    }
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const uint4 b = lds.oq[p][j][c][lane];
#pragma unroll
                        for (int i = 0; i < TPW; ++i)
#pragma unroll
                            for (int x = 0; x < PARTS && x + p < 3; ++x) z[i][c] = mfma16x16x32(qt[i][j][x], b, z[i][c]);
                    }
                }
        };
        auto hand_on = [&](int half) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                lds.y[wave][c][lane] = y[c];
#pragma unroll
                for (int i = 0; i < TPW; ++i) lds.z[half][wave * TPW + i][c][lane] = z[i][c];
            }
        };
        load_out(chunks - 1);
        load_blocks(pt, w.p, chunks - 1);
        load_transposed(qt, w.qt, chunks - 1);
        put_out(chunks - 1);
        __syncthreads();
        products();
        hand_on((chunks - 1) % 2);
        load_out(max(chunks - 2, 0));
        __builtin_amdgcn_sched_barrier(0);
        load_blocks(pt, w.p, max(chunks - 2, 0));
        load_transposed(qt, w.qt, max(chunks - 2, 0));
        __builtin_amdgcn_sched_barrier(0);
        for (int ch = chunks - 1; ch >= 0; --ch) {
            const int next = max(ch - 1, 0), after = max(ch - 2, 0);
            __syncthreads();
            put_out(next);
            __builtin_amdgcn_sched_barrier(0);
            load_out(after);
            __syncthreads();
            products();
            __builtin_amdgcn_sched_barrier(0);
            load_blocks(pt, w.p, after);
            load_transposed(qt, w.qt, after);
            __syncthreads();
            hand_on((ch + 1) % 2);
        }
        return;
    }
    const int64_t size = static_cast<int64_t>(D) * a.value_dim;
    auto row_of = [&](int x) {
        const int t = wave * TPW + x;
        return 32 * (t / 2) + 8 * g + 4 * (t % 2);
    };
    auto state_at = [&](int x) {
        return (static_cast<int64_t>(s) * a.heads + h) * size + static_cast<int64_t>(row_of(x)) * a.value_dim + col;
    };
    f32x4 S[TPW][NC];
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                S[x][c][i] = d.d_final != nullptr ? d.d_final[state_at(x) + i * a.value_dim + c] : 0.0f;
    uint4 k[KS][PARTS], tt[2][3], kt[TPW][2][PARTS];
    f32x4 fk, fu, beta;
    float decay = 0.0f;
    auto load_k = [&](int ch) {
        fu = factors(ch, 2);
        const uint8_t* at = w.kf + (((slot0 + ch) * a.key_heads + kh) * 4 + wave) * KS * PARTS * kFragBytes;
#pragma unroll
        for (int i = 0; i < KS * PARTS; ++i) k[i / PARTS][i % PARTS] = frag16(at + i * kFragBytes, frag);
    };
    auto load_t = [&](int ch) {
        fk = factors(ch, 0);
        beta = factors(ch, 3);
        load_blocks(tt, w.t, ch);
    };
    auto load_rest = [&](int ch) {
        decay = w.vec[((slot0 + ch) * a.heads + h) * kVec + 256];
        load_transposed(kt, w.kt, ch);
    };
    if (chunks > 0) {
        load_k(chunks - 1);
        __builtin_amdgcn_sched_barrier(0);
        load_t(chunks - 1);
        __builtin_amdgcn_sched_barrier(0);
        load_rest(chunks - 1);
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
    }
    for (int ch = chunks - 1; ch >= 0; --ch) {
        const int next = max(ch - 1, 0);
        const int64_t by_head = (slot0 + ch) * a.heads + h;
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                put_parts<3>(lds.s, (wave * TPW + i) / 2, (wave * TPW + i) % 2, c, lane, S[i][c]);
        __syncthreads();
        f32x4 x[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) x[c] = zero;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.s[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r < PARTS && r + p < 3; ++r) x[c] = mfma16x16x32(k[i][r], b, x[c]);
                }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            x[c] = x[c] * fu + lds.y[wave][c][lane];
            put_parts<3>(lds.x, wave / 2, wave % 2, c, lane, x[c]);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        {
            float* to = w.ds + by_head * size + col;
#pragma unroll
            for (int i = 0; i < TPW; ++i) put_rows<NC>(to + row_of(i) * a.value_dim, a.value_dim, S[i]);
        }
        __syncthreads();
        f32x4 du[NC], dr[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) du[c] = zero;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * i + 1 < wave) continue;
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.x[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r + p < 3; ++r) du[c] = mfma16x16x32(tt[i][r], b, du[c]);
                }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            dr[c] = du[c] * beta;
            put_parts<3>(lds.rk, wave / 2, wave % 2, c, lane, -(dr[c] * fk));
        }
        __builtin_amdgcn_sched_barrier(0);
        load_t(next);
        __builtin_amdgcn_sched_barrier(0);
        put_rows<NC>(w.du + (by_head * kChunk + r0) * a.value_dim + col, a.value_dim, du);
        {
            const int left = seq.n - ch * kChunk;
            uint16_t* to = d.dv + (static_cast<int64_t>(seq.a + ch * kChunk + r0) * a.heads + h) * a.value_dim + col;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + i < left) store_cols<NC>(to + static_cast<int64_t>(i) * a.heads * a.value_dim, pack_cols<NC, FP16>(dr, i));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) S[i][c] = S[i][c] * decay + lds.z[ch % 2][wave * TPW + i][c][lane];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.rk[p][j][c][lane];
#pragma unroll
                    for (int i = 0; i < TPW; ++i)
#pragma unroll
                        for (int r = 0; r < PARTS && r + p < 3; ++r) S[i][c] = mfma16x16x32(kt[i][j][r], b, S[i][c]);
                }
        __builtin_amdgcn_sched_barrier(0);
        load_rest(next);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (d.d_initial != nullptr) {
#pragma unroll
        for (int x = 0; x < TPW; ++x) put_rows<NC>(d.d_initial + state_at(x), a.value_dim, S[x]);
    }
}

// ---- the gradient: what does not hand on a state ------------------------------------

// With S the state before a chunk, dS the gradient of that after it, and per
// value head B1_ij = e^(G_i - G_j) do_i . u_j (j <= i), B2_ij = e^(G_i - G_j) dR_i . u_j
// (j < i), for the normalized q and k:
//     dq_i = scale (e^(G_i) S do_i + sum_j B1_ij k_j),
//     dk_i = -(e^(G_i) S dR_i + sum_j B2_ij k_j) + e^(G_63 - G_i) dS u_i
//            + sum_j (B1_ji scale q_j - B2_ji k_j).
// dbeta_i = w_i . du_i.  What is read are w and du, so that a beta of 0 has its
// gradient too; u = beta w and dR = beta du are factors of rows.  A decay g_t acts on what passes
// from before t to t or later: its gradient is, with M_ij = scale B1_ij q_i . k_j
// - B2_ij k_i . k_j,
//     sum_(i >= t) e^(G_i) (scale q_i . S do_i - k_i . S dR_i) + sum_(j < t) e^(G_63 - G_j) k_j . dS u_j
//     + e^(G_63) <S, dS> + sum_(i >= t > j) M_ij,
// as a running sum of rows less columns, with the same numbers on both sides, so
// that what lies within either side cancels to fp32's last bits.
//
// A workgroup has a chunk and a key head and goes through its value heads.  Its
// eight waves have two row tiles (of 16 tokens) and a quarter of the columns of
// dq and dk each. What is fp32 (S, dS, w, du) is read once by the workgroup, 32
// columns at a time, split into three bf16 numbers and shared through LDS, the
// next 32 while the products of those before run (training step of 4000 tokens:
// 300 -> 257 us with two parts in the products over tokens, 274-289 with three):
// the decays' gradient is fp32 and as exact as that. Bound by its one workgroup
// per CU: 208 KB of S, dS, w and du per chunk and value head, and with the rest
// 775 MB in all, come and go at 2.7 TB/s.
constexpr int kGradThreads = 512;
template <int D>
struct ScanInputsLds {
    struct Stage {
        uint4 s[D / 16][3][kWave], ds[D / 16][3][kWave], u[4][3][kWave], r[4][3][kWave];
    };
    union {
        Stage stage[2];
        struct {
            float b1[kChunk * kPitch], b2[kChunk * kPitch];   // at first q . k and k . k, in the end dq and dk
            float sum[kChunk * kPitch];         // M
            uint4 frag[4][kBlocks][3][kWave];   // B1 and B2 by rows (lower blocks), by columns (upper ones)
        } m;
    };
    double sum[kChunk];
    float rk[kChunk], rq[kChunk], decay[kChunk], rest[kChunk], beta[kChunk], dbeta[kChunk];
    float dot[4][kChunk], row[4][kChunk], col[4][kChunk], state[8], moved[8];
};

__device__ __forceinline__ float sum_over_16(float v) {
    v = v + __int_as_float(lane_xor<1>(__float_as_int(v)));
    v = v + __int_as_float(lane_xor<2>(__float_as_int(v)));
    v = butterfly_step4(v);
    return butterfly_step8(v);
}

// Eight floats as a fragment of so many parts.
template <int PARTS>
__device__ __forceinline__ void parts_of(uint4 (&to)[PARTS], const float (&f)[8]) {
    Split2 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = split2<PARTS>(f[2 * j], f[2 * j + 1]);
#pragma unroll
    for (int j = 0; j < PARTS; ++j) to[j] = make_uint4(p[0].part[j], p[1].part[j], p[2].part[j], p[3].part[j]);
}

template <int D, bool FP16>
__global__ __launch_bounds__(kGradThreads, 2) void scan_inputs_grad(ScanArgs a, ScanGradArgs d, ScanChunks w) {
    constexpr int PARTS = FP16 ? 2 : 1, TILES = D / 16, TPQ = D / 64, RAW = D + 8;
    __shared__ ScanInputsLds<D> lds;
    const int tid = threadIdx.x;
    int lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), pair = wave % 2, quarter = wave / 2;
    const int slot = blockIdx.x / a.key_heads, kh = blockIdx.x % a.key_heads;
    const int s = find_sequence(a, slot);
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    const int first = (slot - scan_first_chunk(a, s)) * kChunk;
    if (first < 0 || first >= seq.n) return;
    const int count = min(seq.n - first, kChunk), t0 = seq.a + first;
    const int64_t by_key = static_cast<int64_t>(slot) * a.key_heads + kh;
    const int E = a.value_dim;
    if (tid < kChunk) {
        lds.rk[tid] = w.norms[by_key * 2 * kChunk + tid];
        lds.rq[tid] = w.norms[by_key * 2 * kChunk + kChunk + tid];
    }
    // Row i of the lane's of the wave's row tile x, and element of its column in
    // the wave's column tile t.
    auto row_of = [&](int x, int i) { return 32 * pair + 16 * x + 4 * g + i; };
    auto element_of = [&](int tile) { return 32 * (tile / 2) + 8 * (n / 4) + 4 * (tile % 2) + n % 4; };
    auto element = [&](int t) { return element_of(quarter * TPQ + t); };
    uint32_t q[2][TPQ][2], k[2][TPQ][2];   // raw, rows in pairs
#pragma unroll
    for (int t = 0; t < TPQ; ++t) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // (Rows past the sequence repeat its last one: what they meet is 0.)
                uint32_t of_q[2], of_k[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t at = t0 + min(row_of(x, 2 * i + j), count - 1);
                    of_q[j] = a.q[at * a.q_token + kh * a.q_head + element(t)];
                    of_k[j] = a.k[at * a.k_token + kh * a.k_head + element(t)];
                }
                q[x][t][i] = of_q[0] | (of_q[1] << 16);
                k[x][t][i] = of_k[0] | (of_k[1] << 16);
            }
    }
    // q_i . k_j, or in the second two quarters k_i . k_j, of the wave's rows and
    // every other column tile.
    const int odd = quarter % 2;
    {
        f32x4 pairs[2][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) pairs[x][0] = pairs[x][1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        const uint16_t* side = quarter < 2 ? a.q : a.k;
        const int64_t token = quarter < 2 ? a.q_token : a.k_token, head = quarter < 2 ? a.q_head : a.k_head;
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            const int e = 32 * ks + 8 * g;
            uint4 of[2], with[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                of[x] = ldg16(side + (t0 + min(32 * pair + 16 * x + n, count - 1)) * token + kh * head + e);
                with[x] = ldg16(a.k + (t0 + min(16 * (2 * x + odd) + n, count - 1)) * a.k_token + kh * a.k_head + e);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int c = 0; c < 2; ++c) pairs[x][c] = mfma_raw<FP16>(of[x], with[c], pairs[x][c]);
        }
        float* to = quarter < 2 ? lds.m.b1 : lds.m.b2;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) to[row_of(x, i) * kPitch + 16 * (2 * c + odd) + n] = pairs[x][c][i];
    }
    // Each thread's part of them waits in memory for its turn per value head.
    f32x4* my_pairs = w.pairs + by_key * 4 * kGradThreads + tid;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = (16 * (wave / 2) + n) * kPitch + 32 * (wave % 2) + 16 * j + 4 * g;
        my_pairs[j * kGradThreads] = *reinterpret_cast<const f32x4*>(lds.m.b1 + at);
        my_pairs[(2 + j) * kGradThreads] = *reinterpret_cast<const f32x4*>(lds.m.b2 + at);
    }
    __syncthreads();
    auto raw = [&](const uint32_t (&v)[2], int i) { return elem16<FP16>(static_cast<uint16_t>(v[i / 2] >> (16 * (i % 2)))); };
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 dq[2][TPQ], dk[2][TPQ];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int t = 0; t < TPQ; ++t) dq[x][t] = dk[x][t] = zero;
    const int64_t size = static_cast<int64_t>(D) * E, states = tape_states(w.slots, a.heads, D, E);
    const int rows = kChunk * E;
    auto bytes = [](const void* p) { return static_cast<const uint8_t*>(p); };
    for (int hv = 0; hv < a.group; ++hv) {
        // (Addresses are computed where they are used: kept over the loop they
        // would take more registers than there are.)
        lane = opaque(lane);
        n = lane % 16, g = lane / 16;
        const int h = kh * a.group + hv;
        const int64_t by_head = static_cast<int64_t>(slot) * a.heads + h;
        const float* tape = reinterpret_cast<const float*>(d.tape);
        // The wave's share of a step's staging: a tile of S and dS, one of w or du.
        const bool has_tile = wave < TILES;
        const uint32_t tile_at = 4 * (element_of(wave) * E + 8 * g), rows_at = 4 * ((16 * (wave % 4) + n) * E + 8 * g);
        const uint8_t* at_s = bytes(tape + by_head * size);
        const uint8_t* at_ds = bytes(w.ds + by_head * size);
        const uint8_t* at_rows = bytes(wave < 4 ? tape + states + by_head * rows : w.du + by_head * rows);
        const uint16_t* out = d.d_out + static_cast<int64_t>(t0) * d.d_out_token + h * d.d_out_head;
        // S do, S du and dS w of the wave's rows and columns; of do . w (the first
        // two quarters) and du . w the tiles of its rows and every other column.
        f32x4 so[2][TPQ], sr[2][TPQ], su[2][TPQ], xu[2][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int t = 0; t < TPQ; ++t) so[x][t] = sr[x][t] = su[x][t] = zero;
            xu[x][0] = xu[x][1] = zero;
        }
        float both = 0.0f;   // <S, dS>
        uint4 raw_s[2], raw_ds[2], raw_rows[2], o[2][PARTS];
        auto load = [&](int e0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (has_tile) {
                    raw_s[i] = frag16(at_s + 4 * e0 + 16 * i, tile_at);
                    raw_ds[i] = frag16(at_ds + 4 * e0 + 16 * i, tile_at);
                }
                raw_rows[i] = frag16(at_rows + 4 * e0 + 16 * i, rows_at);
            }
        };
        auto floats = [](const uint4 (&v)[2], float (&f)[8]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[4 * i] = __uint_as_float(v[i].x), f[4 * i + 1] = __uint_as_float(v[i].y);
                f[4 * i + 2] = __uint_as_float(v[i].z), f[4 * i + 3] = __uint_as_float(v[i].w);
            }
        };
        auto stage = [&](uint4 (&to)[3][kWave], const float (&f)[8]) {
            Split2 p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = split2<3>(f[2 * j], f[2 * j + 1]);
#pragma unroll
            for (int j = 0; j < 3; ++j) to[j][lane] = make_uint4(p[0].part[j], p[1].part[j], p[2].part[j], p[3].part[j]);
        };
        load(0);
        __builtin_amdgcn_sched_barrier(0);
        // (Used behind the loop: a row's running sum, the last one, raw beta.)
        const double* sums = w.sums + by_head * kChunk;
        const double sum = sums[lane], last = sums[kChunk - 1];
        uint32_t raw_beta;
        {
            const int64_t at = static_cast<int64_t>(t0 + min(lane, count - 1)) * a.beta_token + h;
            if (a.beta_fp32) raw_beta = static_cast<const uint32_t*>(a.beta)[at];
            else raw_beta = static_cast<const uint16_t*>(a.beta)[at];
        }
        __builtin_amdgcn_sched_barrier(0);
        // 32 columns are staged while the products of those before them run.
        auto put = [&](auto& to) {
            float f[8], f1[8];
            if (has_tile) {
                floats(raw_s, f);
                floats(raw_ds, f1);
                stage(to.s[wave], f);
                stage(to.ds[wave], f1);
#pragma unroll
                for (int j = 0; j < 8; ++j) both = __builtin_fmaf(f[j], f1[j], both);
            }
            floats(raw_rows, f);
            if (wave < 4) stage(to.u[wave % 4], f);
            else stage(to.r[wave % 4], f);
        };
        auto load_out = [&](int e0) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t row = min(32 * pair + 16 * x + n, count - 1);
                o[x][0] = frag16(bytes(out), 2 * (row * static_cast<uint32_t>(d.d_out_token) + e0 + 8 * g));
            }
        };
        load_out(0);
        put(lds.stage[0]);
        if (32 < E) load(32);
#pragma unroll 1
        for (int e0 = 0; e0 < E; e0 += 32) {
            auto& now = lds.stage[e0 / 32 % 2];
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (32 * pair + 16 * x + n >= count) o[x][0] = make_uint4(0u, 0u, 0u, 0u);
                if constexpr (FP16) {
                    float f[8];
                    unpack16<true>(o[x][0], f);
                    parts_of(reinterpret_cast<uint4 (&)[2]>(o[x]), f);
                }
            }
            uint4 u[2][3], r[2][3];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    u[x][p] = now.u[2 * pair + x][p][lane];
                    r[x][p] = now.r[2 * pair + x][p][lane];
                }
#pragma unroll
            for (int p = 0; p < 3; ++p) {
#pragma unroll
                for (int t = 0; t < TPQ; ++t) {
                    const uint4 bs = now.s[quarter * TPQ + t][p][lane], bd = now.ds[quarter * TPQ + t][p][lane];
#pragma unroll
                    for (int y = 0; y + p < 3; ++y)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (y < PARTS) so[x][t] = mfma16x16x32(o[x][y], bs, so[x][t]);
                            sr[x][t] = mfma16x16x32(r[x][y], bs, sr[x][t]);
                            su[x][t] = mfma16x16x32(u[x][y], bd, su[x][t]);
                        }
                }
                // (Tiles above the diagonal are computed and not used.)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 bu = now.u[2 * j + odd][p][lane];
                    if (quarter >= 2) {
#pragma unroll
                        for (int y = 0; y + p < 3; ++y)
#pragma unroll
                            for (int x = 0; x < 2; ++x) xu[x][j] = mfma16x16x32(r[x][y], bu, xu[x][j]);
                    } else {
#pragma unroll
                        for (int y = 0; y < PARTS && y + p < 3; ++y)
#pragma unroll
                            for (int x = 0; x < 2; ++x) xu[x][j] = mfma16x16x32(o[x][y], bu, xu[x][j]);
                    }
                }
            }
            if (e0 + 32 < E) {
                load_out(e0 + 32);
                put(lds.stage[e0 / 32 % 2 ^ 1]);
                if (e0 + 64 < E) load(e0 + 64);
            }
        }
        f32x4 of_qk[2], of_kk[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            of_qk[j] = my_pairs[j * kGradThreads];
            of_kk[j] = my_pairs[(2 + j) * kGradThreads];
        }
        both = wave_butterfly_sum(both);
        if (lane == 0) lds.state[wave] = both;
        if (tid < kChunk) {
            lds.sum[tid] = sum;
            lds.decay[tid] = power(sum);
            lds.rest[tid] = power(last - sum);
            const float beta = a.beta_fp32 ? __uint_as_float(raw_beta) : elem16<FP16>(static_cast<uint16_t>(raw_beta));
            lds.beta[tid] = tid < count ? beta : 0.0f;   // (rows past the sequence have a w)
        }
        __syncthreads();   // (the staging is done with)
        {
            float* to = quarter < 2 ? lds.m.b1 : lds.m.b2;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) to[row_of(x, i) * kPitch + 16 * (2 * c + odd) + n] = xu[x][c][i];
        }
        __syncthreads();
        // Of the matrices a thread has row or column `own` and eight of the others,
        // as a fragment has them: B1 and B2 with their decays and M's sum by rows,
        const int tile = wave / 2, half = wave % 2, own = 16 * tile + n;
        const float own_q = lds.rq[own] * a.scale, own_k = lds.rk[own];
        if (2 * half <= tile) {
            const double own_sum = lds.sum[own];
            const float own_beta = lds.beta[own];
            float by_row = 0.0f, x1[8], x2[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int o = 32 * half + 16 * (j / 4) + 4 * g + j % 4, at = own * kPitch + o;
                const float fade = power(own_sum - lds.sum[o]), rk = lds.rk[o], raw2 = lds.m.b2[at];
                if (o == own) lds.dbeta[own] = raw2;
                const float beta = fade * lds.beta[o];
                const float b1 = o <= own ? beta * lds.m.b1[at] : 0.0f, b2 = o < own ? beta * own_beta * raw2 : 0.0f;
                lds.m.b1[at] = b1;
                lds.m.b2[at] = b2;
                const float m = b1 * of_qk[j / 4][j % 4] * (own_q * rk) - b2 * of_kk[j / 4][j % 4] * (own_k * rk);
                lds.m.sum[at] = m;
                by_row += o < own ? m : 0.0f;
                x1[j] = b1 * rk;
                x2[j] = b2 * rk;
            }
            by_row = butterfly_step32(butterfly_step16(by_row));
            if (g == 0) lds.row[half][own] = by_row;
            uint4 parts[3];
            const int block = lower_block(half, tile);
            parts_of(parts, x1);
#pragma unroll
            for (int p = 0; p < 3; ++p) lds.m.frag[0][block][p][lane] = parts[p];
            parts_of(parts, x2);
#pragma unroll
            for (int p = 0; p < 3; ++p) lds.m.frag[1][block][p][lane] = parts[p];
        } else if (g == 0) {
            lds.row[half][own] = 0.0f;
        }
        __syncthreads();
        // and by columns.
        if (2 * half + 1 >= tile) {
            float by_col = 0.0f, x1[8], x2[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int o = 32 * half + 16 * (j / 4) + 4 * g + j % 4, at = o * kPitch + own;
                const bool in = o >= own;
                const float rq = lds.rq[o] * a.scale, rk = lds.rk[o];
                const float b1 = in ? lds.m.b1[at] : 0.0f, b2 = in ? lds.m.b2[at] : 0.0f;
                by_col += o > own ? lds.m.sum[at] : 0.0f;
                x1[j] = b1 * rq;
                x2[j] = -b2 * rk;
            }
            by_col = butterfly_step32(butterfly_step16(by_col));
            if (g == 0) lds.col[half][own] = by_col;
            uint4 parts[3];
            const int block = upper_block(half, tile);
            parts_of(parts, x1);
#pragma unroll
            for (int p = 0; p < 3; ++p) lds.m.frag[2][block][p][lane] = parts[p];
            parts_of(parts, x2);
#pragma unroll
            for (int p = 0; p < 3; ++p) lds.m.frag[3][block][p][lane] = parts[p];
        } else if (g == 0) {
            lds.col[half][own] = 0.0f;
        }
        uint4 kt[TPQ][2][PARTS], qt[TPQ][2][PARTS];
#pragma unroll
        for (int i = 0; i < TPQ * 2 * PARTS; ++i) {
            const int64_t at = ((by_key * TILES + quarter * TPQ) * 2 * PARTS + i) * kFragBytes;
            kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = frag16(w.kt + at, lane * 16);
            qt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = frag16(w.qt + at, lane * 16);
        }
        // The states' parts of the decays' gradient, before the products over
        // tokens join them.
        float moved = 0.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row_of(x, i);
                float of_q = 0.0f, of_k = 0.0f, of_u = 0.0f;
#pragma unroll
                for (int t = 0; t < TPQ; ++t) {
                    so[x][t][i] *= lds.decay[row];
                    sr[x][t][i] *= lds.decay[row] * lds.beta[row];
                    su[x][t][i] *= lds.rest[row] * lds.beta[row];
                    of_q = __builtin_fmaf(raw(q[x][t], i), so[x][t][i], of_q);
                    of_k = __builtin_fmaf(raw(k[x][t], i), sr[x][t][i], of_k);
                    of_u = __builtin_fmaf(raw(k[x][t], i), su[x][t][i], of_u);
                }
                of_u = sum_over_16(of_u * lds.rk[row]);
                const float sum = sum_over_16(of_q * lds.rq[row] * a.scale - of_k * lds.rk[row]) - of_u;
                if (n == 0) lds.dot[quarter][row] = sum;
                moved += of_u;
            }
        moved = butterfly_step32(butterfly_step16(moved));
        if (lane == 0) lds.moved[wave] = moved;
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int tile = 2 * pair + x;
#pragma unroll
                for (int kind = 0; kind < 4; ++kind) {
                    if (kind < 2 ? 2 * ks > tile : 2 * ks + 1 < tile) continue;
                    const int block = kind < 2 ? lower_block(ks, tile) : upper_block(ks, tile);
#pragma unroll
                    for (int y = 0; y < 3; ++y) {
                        const uint4 f = lds.m.frag[kind][block][y][lane];
#pragma unroll
                        for (int t = 0; t < TPQ; ++t)
#pragma unroll
                            for (int p = 0; p < PARTS && p + y < 3; ++p) {
                                if (kind == 0) so[x][t] = mfma16x16x32(f, kt[t][ks][p], so[x][t]);
                                if (kind == 1) sr[x][t] = mfma16x16x32(f, kt[t][ks][p], sr[x][t]);
                                if (kind == 2) su[x][t] = mfma16x16x32(f, qt[t][ks][p], su[x][t]);
                                if (kind == 3) su[x][t] = mfma16x16x32(f, kt[t][ks][p], su[x][t]);
                            }
                    }
                }
            }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int t = 0; t < TPQ; ++t) {
                    dq[x][t][i] += so[x][t][i];
                    dk[x][t][i] += su[x][t][i] - sr[x][t][i];
                }
            }
        __syncthreads();
        if (wave == 0) {
            // From t on: the sum over the rows from there, and the state's.
            float after = 0.0f, before = 0.0f;
#pragma unroll
            for (int i = 0; i < kGradThreads / kWave; ++i) {
                after += lds.moved[i];
                before += lds.state[i];
            }
            after = __builtin_fmaf(before, lds.decay[kChunk - 1], after);
            const int t = kChunk - 1 - lane;
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x += lds.dot[i][t];
            x += (lds.row[0][t] + lds.row[1][t]) - (lds.col[0][t] + lds.col[1][t]);
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const float other = __shfl_up(x, off);
                if (lane >= off) x += other;
            }
            if (t < count) {
                const int64_t at = static_cast<int64_t>(t0 + t) * a.heads + h;
                d.dg[at] = x + after;
                if (a.beta_fp32) static_cast<float*>(d.dbeta)[at] = lds.dbeta[t];
                else static_cast<uint16_t*>(d.dbeta)[at] = static_cast<uint16_t>(pack16_2<FP16>(lds.dbeta[t], 0.0f));
            }
        }
        __syncthreads();
    }
    // Through the norms, and out by rows.
    if (a.normalize) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float of_q = 0.0f, of_k = 0.0f;
#pragma unroll
                for (int t = 0; t < TPQ; ++t) {
                    of_q = __builtin_fmaf(raw(q[x][t], i), dq[x][t][i], of_q);
                    of_k = __builtin_fmaf(raw(k[x][t], i), dk[x][t][i], of_k);
                }
                of_q = sum_over_16(of_q), of_k = sum_over_16(of_k);
                if (n == 0) {
                    lds.row[quarter][row_of(x, i)] = of_q;
                    lds.col[quarter][row_of(x, i)] = of_k;
                }
            }
    }
    __syncthreads();
    uint16_t* rows_q = reinterpret_cast<uint16_t*>(lds.m.b1);
    uint16_t* rows_k = reinterpret_cast<uint16_t*>(lds.m.b2);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = row_of(x, i);
            const float rq = lds.rq[row], rk = lds.rk[row];
            float back_q = 0.0f, back_k = 0.0f;
            if (a.normalize) {
                back_q = rq * rq * ((lds.row[0][row] + lds.row[1][row]) + (lds.row[2][row] + lds.row[3][row]));
                back_k = rk * rk * ((lds.col[0][row] + lds.col[1][row]) + (lds.col[2][row] + lds.col[3][row]));
            }
#pragma unroll
            for (int t = 0; t < TPQ; ++t) {
                const float y = (dq[x][t][i] - raw(q[x][t], i) * back_q) * rq * a.scale;
                const float z = (dk[x][t][i] - raw(k[x][t], i) * back_k) * rk;
                rows_q[row * RAW + element(t)] = static_cast<uint16_t>(pack16_2<FP16>(y, 0.0f));
                rows_k[row * RAW + element(t)] = static_cast<uint16_t>(pack16_2<FP16>(z, 0.0f));
            }
        }
    __syncthreads();
    for (int i = tid; i < kChunk * D / 8; i += kGradThreads) {
        const int r = i / (D / 8), e = i % (D / 8) * 8;
        if (r >= count) continue;
        const int64_t to = (static_cast<int64_t>(t0 + r) * a.key_heads + kh) * D + e;
        *reinterpret_cast<uint4*>(d.dq + to) = *reinterpret_cast<const uint4*>(rows_q + r * RAW + e);
        *reinterpret_cast<uint4*>(d.dk + to) = *reinterpret_cast<const uint4*>(rows_k + r * RAW + e);
    }
}

ScanChunks layout(const ScanArgs& a, bool fp16, bool grad, uint8_t* base, size_t* bytes) {
    ScanChunks w{};
    w.slots = scan_slots(a);
    w.parts = fp16 ? 2 : 1;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return base + here;
    };
    const size_t by_head = static_cast<size_t>(w.slots) * a.heads, by_key = static_cast<size_t>(w.slots) * a.key_heads;
    const size_t transposed = by_key * (a.dim / 16) * 2 * w.parts * kFragBytes;
    w.t = take(by_head * kBlocks * 3 * kFragBytes);
    w.p = take(by_head * kBlocks * 3 * kFragBytes);
    w.vec = reinterpret_cast<float*>(take(by_head * kVec * sizeof(float)));
    w.kt = take(transposed);
    w.kf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
    if (grad) {
        const size_t columns = static_cast<size_t>(a.value_dim) * sizeof(float);
        w.qt = take(transposed);
        w.sums = reinterpret_cast<double*>(take(by_head * kChunk * sizeof(double)));
        w.norms = reinterpret_cast<float*>(take(by_key * 2 * kChunk * sizeof(float)));
        w.ds = reinterpret_cast<float*>(take(by_head * a.dim * columns));
        w.du = reinterpret_cast<float*>(take(by_head * kChunk * columns));
        w.pairs = reinterpret_cast<f32x4*>(take(by_key * 4 * kGradThreads * sizeof(f32x4)));
    } else {
        w.qf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
        w.flags = reinterpret_cast<uint32_t*>(take(static_cast<size_t>(a.seqs) * a.heads * (a.value_dim / 16) * 4));
    }
    *bytes = at;
    return w;
}

// Launches hold fewer than 2^32 threads: tokens / 64 * heads are at most 2^20,
// seqs * heads * value_dim / 32 at most 2^22.
template <int D, bool FP16>
void launch(const ScanArgs& a, const ScanChunks& w, hipStream_t stream) {
    scan_prepare<D, FP16, false><<<static_cast<uint32_t>(w.slots) * a.key_heads, kThreads, 0, stream>>>(a, w);
    // Blocks of 16 columns where those of 32 would leave half of the CUs idle.
    const bool narrow = a.tape == nullptr && a.seqs * a.heads * (a.value_dim / 32) <= 128;
    const ScanGrid grid = scan_grid(a, narrow ? 16 : 32);
    if (a.tape != nullptr) scan_chunks<D, 2, FP16, true><<<grid.blocks, kChainThreads, 0, stream>>>(a, w, grid.share);
    else if (narrow) scan_chunks<D, 1, FP16, false><<<grid.blocks, kChainThreads, 0, stream>>>(a, w, grid.share);
    else scan_chunks<D, 2, FP16, false><<<grid.blocks, kChainThreads, 0, stream>>>(a, w, grid.share);
}

template <int D, bool FP16>
void launch_grad(const ScanArgs& a, const ScanGradArgs& d, const ScanChunks& w, hipStream_t stream) {
    const uint32_t chunks = static_cast<uint32_t>(w.slots) * a.key_heads;
    scan_prepare<D, FP16, true><<<chunks, kThreads, 0, stream>>>(a, w);
    const ScanGrid grid = scan_grid(a, 32);
    scan_chunks_grad<D, FP16><<<grid.blocks, kChainGradThreads, 0, stream>>>(a, d, w, grid.share);
    scan_inputs_grad<D, FP16><<<chunks, kGradThreads, 0, stream>>>(a, d, w);
}

}  // namespace

size_t scan_chunk_bytes(const ScanArgs& a, bool fp16) {
    size_t bytes = 0;
    layout(a, fp16, false, nullptr, &bytes);
    return bytes;
}

hipError_t launch_scan_chunks(const ScanArgs& a, bool fp16, void* workspace, const uint32_t** flags,
                              hipStream_t stream) {
    size_t bytes = 0;
    const ScanChunks w = layout(a, fp16, false, static_cast<uint8_t*>(workspace), &bytes);
    if (a.dim == 64) {
        if (fp16) launch<64, true>(a, w, stream); else launch<64, false>(a, w, stream);
    } else {
        if (fp16) launch<128, true>(a, w, stream); else launch<128, false>(a, w, stream);
    }
    *flags = w.flags;
    return hipGetLastError();
}

size_t delta_scan_tape_bytes(const ScanArgs& a) {
    return static_cast<size_t>(scan_slots(a)) * a.heads * (a.dim + kChunk) * a.value_dim * sizeof(float);
}

size_t delta_scan_grad_workspace_bytes(const ScanArgs& a, bool fp16) {
    size_t bytes = 0;
    layout(a, fp16, true, nullptr, &bytes);
    return bytes;
}

hipError_t launch_delta_scan_grad(const ScanArgs& a, const ScanGradArgs& d, bool fp16, void* workspace,
                                  hipStream_t stream) {
    size_t bytes = 0;
    const ScanChunks w = layout(a, fp16, true, static_cast<uint8_t*>(workspace), &bytes);
    if (a.dim == 64) {
        if (fp16) launch_grad<64, true>(a, d, w, stream); else launch_grad<64, false>(a, d, w, stream);
    } else {
        if (fp16) launch_grad<128, true>(a, d, w, stream); else launch_grad<128, false>(a, d, w, stream);
    }
    return hipGetLastError();
}

}  // namespace lrmoe
