// The gated delta rule in chunks of 64 tokens, as matrix products.  With G the
// running sum of g inside a chunk, S the state before it, k and q already
// normalized, the chunk's tokens i, j give
//     L_ij = e^(G_i - G_j) k_i . k_j   (j < i),   P_ij = scale e^(G_i - G_j) q_i . k_j   (j <= i),
//     R_i = v_i - e^(G_i) S^T k_i,     w = (I + L beta)^-1 R,     u = beta w,
//     out_i = scale e^(G_i) S^T q_i + sum_j P_ij u_j,
//     S <- e^(G_63) S + sum_j e^(G_63 - G_j) k_j u_j^T.
// Launch one computes what does not depend on the state for all chunks at once:
// T = beta (I + L beta)^-1, P and the factors.  Launch two goes through a
// sequence's chunks one after another, per value head and block of columns.
//
// Products are of bf16 matrix instructions with nothing rounded: q and k are
// bf16 as they come (an fp16 number is two bf16 ones), and an fp32 factor is
// split into three bf16 numbers whose sum it is (two for the products that only
// reach the outputs, which are rounded to 16 bits themselves), so that states
// are as good as sums in fp32.  The raw q and k enter the products; their
// norms are factors of rows.
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
__device__ __forceinline__ int find_sequence(const int32_t* starts, int seqs, int c) {
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + kWave - 1) / kWave;
        const int at = lo + (static_cast<int>(__lane_id()) + 1) * step;
        const bool before = at < hi && scan_first_chunk(starts, at) <= c;
        const int n = __popcll(__ballot(before));
        lo += n * step;
        hi = min(lo + step, hi);
    }
    return __builtin_amdgcn_readfirstlane(lo);
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

struct PrepareLds {
    float a[kChunk * kPitch];   // K rows, then I + L beta
    float b[kChunk * kPitch];   // Q rows, then P
    float t[kChunk * kPitch];   // the inverse
    double sum[kChunk];
    float beta[kChunk], rk[kChunk], rq[kChunk];
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
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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
__global__ __launch_bounds__(kThreads, 3) void scan_prepare(ScanArgs a, ScanChunks w) {
    constexpr int RAW = D + 8;   // 16-bit elements of a row in LDS
    constexpr int PARTS = FP16 ? 2 : 1;
    __shared__ PrepareLds lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int slot = blockIdx.x / a.key_heads, kh = blockIdx.x % a.key_heads;
    const int s = find_sequence(a.starts, a.seqs, slot);
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    const int first = (slot - scan_first_chunk(a.starts, s)) * kChunk;
    if (first < 0 || first >= seq.n) return;
    const int count = min(seq.n - first, kChunk), t0 = seq.a + first;
    uint16_t* raw_k = reinterpret_cast<uint16_t*>(lds.a);
    uint16_t* raw_q = reinterpret_cast<uint16_t*>(lds.b);
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
    if constexpr (FP16) {
        for (int ks = 0; ks < D / 32; ++ks) {
            float x[8];
            const int64_t at = (((by_key * 4 + wave) * (D / 32) + ks) * PARTS) * kFragBytes + lane * 16;
            unpack16<FP16>(*reinterpret_cast<const uint4*>(raw_k + (16 * wave + n) * RAW + 32 * ks + 8 * g), x);
            store_parts<PARTS>(w.kf + at, x);
            if constexpr (!GRAD) {
                unpack16<FP16>(*reinterpret_cast<const uint4*>(raw_q + (16 * wave + n) * RAW + 32 * ks + 8 * g), x);
                store_parts<PARTS>(w.qf + at, x);
            }
        }
    }
    for (int hv = 0; hv < a.group; ++hv) {
        const int h = kh * a.group + hv;
        const int64_t by_head = static_cast<int64_t>(slot) * a.heads + h;
        __syncthreads();   // (rows and the last head's matrices are done with)
        if (wave == 0) {
            float gl = 0.0f, b = 0.0f;
            if (lane < count) {
                const int64_t t = t0 + lane;
                gl = scan_log(a.g[t * a.g_token + h]);
                b = a.beta_fp32 ? static_cast<const float*>(a.beta)[t * a.beta_token + h]
                                : elem16<FP16>(static_cast<const uint16_t*>(a.beta)[t * a.beta_token + h]);
            }
            // (In powers of two.)
            const double sum = wave_scan_f64(gl * 1.4426950408889634);
            lds.sum[lane] = sum;
            lds.beta[lane] = lane < count ? scan_beta(b) : 0.0f;
            if constexpr (GRAD) w.sums[by_head * kChunk + lane] = sum;
            const double last = __shfl(sum, kWave - 1);
            const float decay = power(sum), rest = power(last - sum);
            float* vec = w.vec + by_head * 256;
            const bool in = lane < count;   // (rows past the sequence repeat its last one)
            vec[lane] = in ? decay * lds.rk[lane] : 0.0f;
            vec[64 + lane] = in ? decay * lds.rq[lane] * a.scale : 0.0f;
            vec[128 + lane] = in ? rest * lds.rk[lane] : 0.0f;
            if (lane == kWave - 1) vec[192] = decay;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int j = 16 * t + n;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * g + r;
                const float fade = power(lds.sum[i] - lds.sum[j]) * lds.rk[j];
                lds.a[i * kPitch + j] = j < i ? fade * lds.rk[i] * lds.beta[j] * kk[t][r] : 0.0f;
                lds.b[i * kPitch + j] = j <= i ? fade * lds.rq[i] * a.scale * qk[t][r] : 0.0f;
            }
        }
        __syncthreads();
        invert(lds, wave, lane);
        const int row = 16 * wave + n;
        if constexpr (GRAD) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (2 * ks + 1 < wave) continue;
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = 32 * ks + 16 * (j / 4) + 4 * g + j % 4;
                    const bool in = 2 * ks + j / 4 >= wave;
                    x[j] = in ? lds.beta[i] * lds.t[i * kPitch + row] : 0.0f;
                    y[j] = in ? lds.b[i * kPitch + row] : 0.0f;
                }
                const int64_t block = by_head * kBlocks + upper_block(ks, wave);
                store_parts<3>(w.t + block * 3 * kFragBytes + lane * 16, x);
                store_parts<3>(w.p + block * 3 * kFragBytes + lane * 16, y);
            }
            continue;
        }
        const float b = lds.beta[row];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (2 * ks > wave) continue;
            float x[8], y[8];
            const int at = row * kPitch + 32 * ks + 4 * g;
            const bool half = 2 * ks + 1 <= wave;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = b * lds.t[at + j];
                x[4 + j] = half ? b * lds.t[at + 16 + j] : 0.0f;
                y[j] = lds.b[at + j];
                y[4 + j] = half ? lds.b[at + 16 + j] : 0.0f;
            }
            const int64_t block = by_head * kBlocks + lower_block(ks, wave);
            store_parts<3>(w.t + block * 3 * kFragBytes + lane * 16, x);
            store_parts<2>(w.p + block * 2 * kFragBytes + lane * 16, y);
        }
    }
}

// ---- launch two: chunk after chunk -----------------------------------------------

// A workgroup has 16 NC columns of a state; wave w its rows of the tiles w TPW
// .. + TPW - 1, in the accumulators of the state's own update (column NC n + c
// of the block in lane n of a group and tile c).  A step's products hand their
// results on through LDS, as the B fragments of the next ones, which the lanes
// write as they hold them.
template <int D, int NC>
struct ScanLds {
    uint4 s[3][D / 32][NC][kWave];
    uint4 r[3][2][NC][kWave];
    uint4 u[2][2][NC][kWave];    // for the outputs
    uint4 uk[3][2][NC][kWave];   // times the factors of K^T U
};

// Four values of a lane as half a B fragment (element 4 half on), in parts.
template <int PARTS, int KS, int NC>
__device__ __forceinline__ void put_parts(uint4 (&to)[PARTS][KS][NC][kWave], int ks, int half, int c, int lane, f32x4 x) {
    const Split2 lo = split2<PARTS>(x[0], x[1]), hi = split2<PARTS>(x[2], x[3]);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
        reinterpret_cast<uint2*>(&to[p][ks][c][lane])[half] = make_uint2(lo.part[p], hi.part[p]);
}

// Four rows of a lane's columns, from row `row` on, as two bf16 parts of a
// [rows][value_dim] matrix, `apart` elements from part to part.
template <int NC>
__device__ __forceinline__ void put_rows(uint16_t* to, int64_t apart, int value_dim, int row, int col,
                                         const f32x4 (&x)[NC]) {
    static_assert(NC == 2, "pairs of columns");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Split2 s = split2<2>(x[0][i], x[1][i]);
        uint16_t* p = to + static_cast<int64_t>(row + i) * value_dim + col;
        *reinterpret_cast<uint32_t*>(p) = s.part[0];
        *reinterpret_cast<uint32_t*>(p + apart) = s.part[1];
    }
}

template <int D, int NC, bool FP16>
struct ScanLoads {
    static constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64;
    uint4 k[D / 32][PARTS], q[D / 32][PARTS], t[2][3], p[2][2], kt[TPW][2][PARTS];
    uint32_t v[4][NC / 2 + NC % 2];
    f32x4 fk, fq, fu;   // factors of the lane's four tokens
    float decay;
};

template <int NC>
__device__ __forceinline__ void load_cols(uint32_t (&v)[NC / 2 + NC % 2], const uint8_t* p, uint32_t at) {
    if constexpr (NC == 1) v[0] = *reinterpret_cast<const uint16_t*>(p + at);
    if constexpr (NC == 2) v[0] = *reinterpret_cast<const uint32_t*>(p + at);
}
__device__ __forceinline__ uint4 frag16(const uint8_t* p, uint32_t at) { return *reinterpret_cast<const uint4*>(p + at); }
template <int NC, bool FP16>
__device__ __forceinline__ float col_value(const uint32_t (&v)[NC / 2 + NC % 2], int c) {
    return elem16<FP16>(static_cast<uint16_t>(c % 2 ? v[c / 2] >> 16 : v[c / 2]));
}

template <int D, int NC, bool FP16, bool TAPE>
__global__ __launch_bounds__(kThreads, 2) void scan_chunks(ScanArgs a, ScanChunks w) {
    constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64, KS = D / 32;
    __shared__ ScanLds<D, NC> lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    // Blocks of one head, and of one key head, on the same XCD.
    const int blocks = a.value_dim / (16 * NC), per = (gridDim.x + 7) / 8;
    const int item = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (item >= a.seqs * a.heads * blocks) return;
    const int cb = item % blocks, h = item / blocks % a.heads, s = item / blocks / a.heads, kh = h / a.group;
    const int col = 16 * NC * cb + NC * n;
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    if (a.clear && (s == 0 || s == a.seqs - 1)) {
        const int head = min(max(a.starts[0], 0), a.tokens), tail = min(max(a.starts[a.seqs], 0), a.tokens);
        uint16_t* row = a.out + h * a.out_head + 16 * NC * cb;
        if (s == 0)
            for (int i = tid; i < head * 16 * NC; i += kThreads) row[i / (16 * NC) * a.out_token + i % (16 * NC)] = 0;
        if (s == a.seqs - 1)
            for (int i = tid; i < (a.tokens - tail) * 16 * NC; i += kThreads)
                row[(tail + i / (16 * NC)) * a.out_token + i % (16 * NC)] = 0;
    }
    uint32_t* flag = w.flags + (static_cast<int64_t>(s) * a.heads + h) * (a.value_dim / 16) + NC * cb;
    const int into = scan_slot(a.into, s, a.pool);
    const bool fresh = a.initial == nullptr || (a.fresh != nullptr && a.fresh[s] != 0);
    const int from = fresh ? 0 : scan_slot(a.from, s, a.pool);
    if (into < 0 || from < 0) {
        if (tid < NC) flag[tid] = 0;
        return;
    }
    const int64_t size = static_cast<int64_t>(D) * a.value_dim;
    f32x4 S[TPW][NC];
    // Row i of the lane's of tile x.
    auto row_of = [&](int x, int i) {
        const int t = wave * TPW + x;
        return 32 * (t / 2) + 8 * g + 4 * (t % 2) + i;
    };
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                S[x][c][i] = fresh ? 0.0f
                                   : a.initial[(static_cast<int64_t>(from) * a.heads + h) * size +
                                               static_cast<int64_t>(row_of(x, i)) * a.value_dim + col + c];
    const int chunks = (seq.n + kChunk - 1) / kChunk;
    const int64_t slot0 = scan_first_chunk(a.starts, s);
    uint16_t* tape_s = reinterpret_cast<uint16_t*>(a.tape);
    uint16_t* tape_u = tape_s + tape_states(w.slots, a.heads, D, a.value_dim);
    ScanLoads<D, NC, FP16> x;
    // Addresses are a scalar base per chunk and offsets of 32 bits; rows past the
    // sequence repeat its last one (their factors are 0, and their u).
    const int r0 = 16 * wave + 4 * g;
    const uint32_t frag = lane * 16;
    auto load_rows = [&](int ch) {
        if constexpr (FP16) {
            const int64_t at = (((slot0 + ch) * a.key_heads + kh) * 4 + wave) * KS * PARTS * kFragBytes;
#pragma unroll
            for (int i = 0; i < KS * PARTS; ++i) {
                x.k[i / PARTS][i % PARTS] = frag16(w.kf + at + i * kFragBytes, frag);
                x.q[i / PARTS][i % PARTS] = frag16(w.qf + at + i * kFragBytes, frag);
            }
        } else {
            const int64_t t = seq.a + ch * kChunk;
            const uint8_t* k = reinterpret_cast<const uint8_t*>(a.k + t * a.k_token + kh * a.k_head);
            const uint8_t* q = reinterpret_cast<const uint8_t*>(a.q + t * a.q_token + kh * a.q_head);
            const uint32_t row = min(16 * wave + n, seq.n - 1 - ch * kChunk);
            const uint32_t k_at = row * (2 * static_cast<uint32_t>(a.k_token)) + 16 * g;
            const uint32_t q_at = row * (2 * static_cast<uint32_t>(a.q_token)) + 16 * g;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                x.k[i][0] = frag16(k + 64 * i, k_at);
                x.q[i][0] = frag16(q + 64 * i, q_at);
            }
        }
    };
    auto load_values = [&](int ch) {
        const float* vec = w.vec + ((slot0 + ch) * a.heads + h) * 256;
        x.fk = *reinterpret_cast<const f32x4*>(vec + r0);
        const uint8_t* v = reinterpret_cast<const uint8_t*>(a.v + static_cast<int64_t>(seq.a + ch * kChunk) * a.v_token +
                                                            h * a.v_head + 16 * NC * cb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = min(r0 + i, seq.n - 1 - ch * kChunk);
            load_cols<NC>(x.v[i], v, row * (2 * static_cast<uint32_t>(a.v_token)) + 2 * NC * n);
        }
    };
    auto load_t = [&](int ch) {
        const uint8_t* t = w.t + ((slot0 + ch) * a.heads + h) * kBlocks * 3 * kFragBytes;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            x.t[0][p] = frag16(t + (lower_block(0, wave) * 3 + p) * kFragBytes, frag);
            x.t[1][p] = frag16(t + (lower_block(1, max(wave, 2)) * 3 + p) * kFragBytes, frag);
        }
    };
    auto load_factors = [&](int ch) {
        const float* vec = w.vec + ((slot0 + ch) * a.heads + h) * 256;
        x.fq = *reinterpret_cast<const f32x4*>(vec + 64 + r0);
        x.fu = *reinterpret_cast<const f32x4*>(vec + 128 + r0);
        x.decay = vec[192];
    };
    auto load_rest = [&](int ch) {
        const int64_t by_head = (slot0 + ch) * a.heads + h, by_key = (slot0 + ch) * a.key_heads + kh;
        const uint8_t* at = w.p + by_head * kBlocks * 2 * kFragBytes;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            x.p[0][p] = frag16(at + (lower_block(0, wave) * 2 + p) * kFragBytes, frag);
            x.p[1][p] = frag16(at + (lower_block(1, max(wave, 2)) * 2 + p) * kFragBytes, frag);
        }
        const uint8_t* kt = w.kt + ((by_key * (D / 16) + wave * TPW) * 2 * PARTS) * kFragBytes;
#pragma unroll
        for (int i = 0; i < TPW * 2 * PARTS; ++i)
            x.kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = frag16(kt + i * kFragBytes, frag);
    };
    if (chunks > 0) {
        // (In the loop's order, so that its waits count the same loads.)
        load_rows(0);
        __builtin_amdgcn_sched_barrier(0);
        load_values(0);
        __builtin_amdgcn_sched_barrier(0);
        load_t(0);
        load_factors(0);
        __builtin_amdgcn_sched_barrier(0);
        load_rest(0);
        __builtin_amdgcn_sched_barrier(0);
    }
    bool odd = false;   // a number that is not finite
    for (int ch = 0; ch < chunks; ++ch) {
        const int next = min(ch + 1, chunks - 1);
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                put_parts<3>(lds.s, (wave * TPW + i) / 2, (wave * TPW + i) % 2, c, lane, S[i][c]);
        const int64_t taped = (slot0 + ch) * a.heads + h;
        if constexpr (TAPE) {
#pragma unroll
            for (int i = 0; i < TPW; ++i)
                put_rows<NC>(tape_s + taped * 2 * size, size, a.value_dim, row_of(i, 0), col, S[i]);
        }
        __syncthreads();
        f32x4 ks[NC], qs[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) ks[c] = qs[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint4 b = lds.s[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r < PARTS; ++r) {
                        if (r + p < 3) ks[c] = mfma16x16x32(x.k[i][r], b, ks[c]);
                        if (r + p < 2) qs[c] = mfma16x16x32(x.q[i][r], b, qs[c]);
                    }
                }
        __builtin_amdgcn_sched_barrier(0);
        load_rows(next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            f32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = col_value<NC, FP16>(x.v[i], c) - x.fk[i] * ks[c][i];
            put_parts<3>(lds.r, wave / 2, wave % 2, c, lane, r);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_values(next);
        __syncthreads();
        f32x4 u[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (2 * k > wave) continue;
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const uint4 b = lds.r[p][k][c][lane];
#pragma unroll
                    for (int r = 0; r + p < 3; ++r) u[c] = mfma16x16x32(x.t[k][r], b, u[c]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_t(next);
        __builtin_amdgcn_sched_barrier(0);
        const f32x4 fq = x.fq;
        const float decay = x.decay;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (__float_as_uint(u[c][i]) & 0x7f800000u) == 0x7f800000u;
            put_parts<2>(lds.u, wave / 2, wave % 2, c, lane, u[c]);
            put_parts<3>(lds.uk, wave / 2, wave % 2, c, lane, u[c] * x.fu);
        }
        load_factors(next);
        if constexpr (TAPE)
            put_rows<NC>(tape_u + taped * 2 * kChunk * a.value_dim, kChunk * a.value_dim, a.value_dim, 16 * wave + 4 * g,
                         col, u);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                S[i][c] *= decay;
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const uint4 b = lds.uk[p][k][c][lane];
#pragma unroll
                        for (int r = 0; r < PARTS; ++r)
                            if (r + p < 3) S[i][c] = mfma16x16x32(x.kt[i][k][r], b, S[i][c]);
                    }
            }
        f32x4 o[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            o[c] = qs[c] * fq;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (2 * k > wave) continue;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint4 b = lds.u[p][k][c][lane];
#pragma unroll
                    for (int r = 0; r + p < 2; ++r) o[c] = mfma16x16x32(x.p[k][r], b, o[c]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_rest(next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ch * kChunk + 16 * wave + 4 * g + i;
            if (t >= seq.n) continue;
            uint16_t* to = a.out + static_cast<int64_t>(seq.a + t) * a.out_token + h * a.out_head + col;
            if constexpr (NC == 1) {
                *to = static_cast<uint16_t>(pack16_2<FP16>(o[0][i], 0.0f));
            } else {
                *reinterpret_cast<uint32_t*>(to) = pack16_2<FP16>(o[0][i], o[1][i]);
            }
        }
    }
    // Where a value was not finite, a product's zero weights have let it through
    // to earlier tokens: the next launch goes through these columns again.
    if (__syncthreads_or(odd)) {
        if (tid < NC) flag[tid] = 1;
        return;
    }
    if (tid < NC) flag[tid] = 0;
#pragma unroll
    for (int x1 = 0; x1 < TPW; ++x1)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                a.final[(static_cast<int64_t>(into) * a.heads + h) * size +
                        static_cast<int64_t>(row_of(x1, i)) * a.value_dim + col + c] = S[x1][c][i];
}

// ---- the gradient: chunk after chunk, backwards -----------------------------------

// With dS the gradient of the state after a chunk and do that of its outputs,
//     X_j = sum_i P_ij do_i + e^(G_63 - G_j) dS^T k_j,     dR = (beta (I + L beta)^-1)^T X = dv,
//     dS <- e^(G_63) dS + sum_i scale e^(G_i) q_i do_i^T - sum_i e^(G_i) k_i dR_i^T:
// the forward launch with the matrices transposed, for the same columns.
template <int D, int NC, int PARTS>
struct ScanGradLds {
    uint4 s[3][D / 32][NC][kWave];
    uint4 o[PARTS][2][NC][kWave];   // do
    uint4 x[3][2][NC][kWave];
    uint4 oq[3][2][NC][kWave];      // do times the factors of q
    uint4 rk[3][2][NC][kWave];      // - dR times the factors of k
};

template <int D, bool FP16>
__global__ __launch_bounds__(kThreads, 2) void scan_chunks_grad(ScanArgs a, ScanGradArgs d, ScanChunks w) {
    constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64, KS = D / 32, NC = 2;
    __shared__ ScanGradLds<D, NC, PARTS> lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int blocks = a.value_dim / (16 * NC), per = (gridDim.x + 7) / 8;
    const int item = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (item >= a.seqs * a.heads * blocks) return;
    const int cb = item % blocks, h = item / blocks % a.heads, s = item / blocks / a.heads, kh = h / a.group;
    const int col = 16 * NC * cb + NC * n;
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    if (s == 0 || s == a.seqs - 1) {
        // Rows of no sequence have no gradient.
        const int head = min(max(a.starts[0], 0), a.tokens), tail = min(max(a.starts[a.seqs], 0), a.tokens);
        auto clear = [&](int from, int to) {
            const int rows = to - from;
            for (int i = tid; i < rows * 32; i += kThreads)
                d.dv[(static_cast<int64_t>(from + i / 32) * a.heads + h) * a.value_dim + 32 * cb + i % 32] = 0;
            if (cb != 0) return;
            for (int i = tid; i < rows; i += kThreads) {
                const int64_t at = static_cast<int64_t>(from + i) * a.heads + h;
                d.dg[at] = 0.0f;
                if (a.beta_fp32) static_cast<float*>(d.dbeta)[at] = 0.0f;
                else static_cast<uint16_t*>(d.dbeta)[at] = 0;
            }
            if (h % a.group != 0) return;
            for (int i = tid; i < rows * D; i += kThreads) {
                const int64_t at = (static_cast<int64_t>(from + i / D) * a.key_heads + kh) * D + i % D;
                d.dq[at] = 0;
                d.dk[at] = 0;
            }
        };
        if (s == 0) clear(0, head);
        if (s == a.seqs - 1) clear(tail, a.tokens);
    }
    const int64_t size = static_cast<int64_t>(D) * a.value_dim;
    f32x4 S[TPW][NC];
    auto row_of = [&](int x, int i) {
        const int t = wave * TPW + x;
        return 32 * (t / 2) + 8 * g + 4 * (t % 2) + i;
    };
    auto state_at = [&](int x, int i) {
        return (static_cast<int64_t>(s) * a.heads + h) * size + static_cast<int64_t>(row_of(x, i)) * a.value_dim + col;
    };
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) S[x][c][i] = d.d_final != nullptr ? d.d_final[state_at(x, i) + c] : 0.0f;
    const int chunks = (seq.n + kChunk - 1) / kChunk;
    const int64_t slot0 = scan_first_chunk(a.starts, s);
    uint4 k[KS][PARTS], tt[2][3], pt[2][3], kt[TPW][2][PARTS], qt[TPW][2][PARTS];
    uint32_t o[4][1];
    f32x4 fk, fq, fu;
    float decay = 0.0f;
    const int r0 = 16 * wave + 4 * g;
    auto load_k = [&](int ch) {
        if constexpr (FP16) {
            const int64_t at = (((slot0 + ch) * a.key_heads + kh) * 4 + wave) * KS * PARTS * kFragBytes + lane * 16;
#pragma unroll
            for (int i = 0; i < KS * PARTS; ++i) k[i / PARTS][i % PARTS] = ldg16(w.kf + at + i * kFragBytes);
        } else {
            const int t = ch * kChunk + 16 * wave + n;
            const bool in = t < seq.n;
            const int64_t row = seq.a + (in ? t : 0);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                k[i][0] = make_uint4(0u, 0u, 0u, 0u);
                if (in) k[i][0] = ldg16(a.k + row * a.k_token + kh * a.k_head + 32 * i + 8 * g);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ch * kChunk + r0 + i;
            o[i][0] = 0u;
            if (t < seq.n)
                load_cols<NC>(o[i], reinterpret_cast<const uint8_t*>(d.d_out + static_cast<int64_t>(seq.a + t) * d.d_out_token + h * d.d_out_head + col), 0);
        }
        const float* vec = w.vec + ((slot0 + ch) * a.heads + h) * 256;
        fk = *reinterpret_cast<const f32x4*>(vec + r0);
        fq = *reinterpret_cast<const f32x4*>(vec + 64 + r0);
        fu = *reinterpret_cast<const f32x4*>(vec + 128 + r0);
        decay = vec[192];
    };
    auto load_matrices = [&](int ch) {
        const int64_t at = ((slot0 + ch) * a.heads + h) * kBlocks * 3 * kFragBytes + lane * 16;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            if (wave < 2) {
                tt[0][p] = ldg16(w.t + at + (upper_block(0, wave) * 3 + p) * kFragBytes);
                pt[0][p] = ldg16(w.p + at + (upper_block(0, wave) * 3 + p) * kFragBytes);
            }
            tt[1][p] = ldg16(w.t + at + (upper_block(1, wave) * 3 + p) * kFragBytes);
            pt[1][p] = ldg16(w.p + at + (upper_block(1, wave) * 3 + p) * kFragBytes);
        }
    };
    auto load_transposed = [&](int ch) {
        const int64_t by_key = (slot0 + ch) * a.key_heads + kh;
#pragma unroll
        for (int i = 0; i < TPW * 2 * PARTS; ++i) {
            const int64_t at = ((by_key * (D / 16) + wave * TPW) * 2 * PARTS + i) * kFragBytes + lane * 16;
            kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = ldg16(w.kt + at);
            qt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] = ldg16(w.qt + at);
        }
    };
    if (chunks > 0) {
        load_k(chunks - 1);
        load_matrices(chunks - 1);
        load_transposed(chunks - 1);
    }
    for (int ch = chunks - 1; ch >= 0; --ch) {
        const int next = max(ch - 1, 0);
        const int64_t by_head = (slot0 + ch) * a.heads + h;
        f32x4 od[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) od[c][i] = col_value<NC, FP16>(o[i], c);
            put_parts<PARTS>(lds.o, wave / 2, wave % 2, c, lane, od[c]);
        }
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
                put_parts<3>(lds.s, (wave * TPW + i) / 2, (wave * TPW + i) % 2, c, lane, S[i][c]);
            put_rows<NC>(w.ds + by_head * 2 * size, size, a.value_dim, row_of(i, 0), col, S[i]);
        }
        __syncthreads();
        f32x4 x[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            x[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const uint4 b = lds.s[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r < PARTS; ++r)
                        if (r + p < 3) x[c] = mfma16x16x32(k[i][r], b, x[c]);
                }
            x[c] *= fu;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (2 * i + 1 < wave) continue;
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const uint4 b = lds.o[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r + p < 3; ++r) x[c] = mfma16x16x32(pt[i][r], b, x[c]);
                }
            }
            put_parts<3>(lds.x, wave / 2, wave % 2, c, lane, x[c]);
        }
        const f32x4 factor_k = fk, factor_q = fq;
        const float fade = decay;
        load_k(next);
        __syncthreads();
        f32x4 dr[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            dr[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (2 * i + 1 < wave) continue;
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const uint4 b = lds.x[p][i][c][lane];
#pragma unroll
                    for (int r = 0; r + p < 3; ++r) dr[c] = mfma16x16x32(tt[i][r], b, dr[c]);
                }
            }
            put_parts<3>(lds.rk, wave / 2, wave % 2, c, lane, -(dr[c] * factor_k));
            put_parts<3>(lds.oq, wave / 2, wave % 2, c, lane, od[c] * factor_q);
        }
        load_matrices(next);
        put_rows<NC>(w.dr + by_head * 2 * kChunk * a.value_dim, kChunk * a.value_dim, a.value_dim, r0, col, dr);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ch * kChunk + r0 + i;
            if (t < seq.n)
                *reinterpret_cast<uint32_t*>(d.dv + (static_cast<int64_t>(seq.a + t) * a.heads + h) * a.value_dim + col) =
                    pack16_2<FP16>(dr[0][i], dr[1][i]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                S[i][c] *= fade;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const uint4 bq = lds.oq[p][j][c][lane], bk = lds.rk[p][j][c][lane];
#pragma unroll
                        for (int r = 0; r < PARTS; ++r)
                            if (r + p < 3) {
                                S[i][c] = mfma16x16x32(qt[i][j][r], bq, S[i][c]);
                                S[i][c] = mfma16x16x32(kt[i][j][r], bk, S[i][c]);
                            }
                    }
            }
        load_transposed(next);
    }
    if (d.d_initial != nullptr) {
#pragma unroll
        for (int x = 0; x < TPW; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) d.d_initial[state_at(x, i) + c] = S[x][c][i];
    }
}

// ---- the gradient: what does not hand on a state ------------------------------------

// With S the state before a chunk, dS the gradient of that after it, and per
// value head B1_ij = e^(G_i - G_j) do_i . u_j (j <= i), B2_ij = e^(G_i - G_j) dR_i . u_j
// (j < i), for the normalized q and k:
//     dq_i = scale (e^(G_i) S do_i + sum_j B1_ij k_j),
//     dk_i = -(e^(G_i) S dR_i + sum_j B2_ij k_j) + e^(G_63 - G_i) dS u_i
//            + sum_j (B1_ji scale q_j - B2_ji k_j),
// the first bracket by k_i's own row, the rest by its column.  The running sum
// G_i has the gradient q_i . dq_i + k_i . (dk_i by its row) - k_i . (dk_i by its
// column), the last one <state after, dS> as well, and g_t the sum of those from
// t on.  dbeta_i = w_i . du_i = u_i . dR_i / beta_i^2.
//
// A workgroup has a chunk and a key head and goes through its value heads; wave
// w has the token rows of tile w, in the accumulators' layout with the columns
// of the K^T fragments' rows.
struct ScanInputsLds {
    float b1[kChunk * kPitch], b2[kChunk * kPitch];   // then dq and dk, 16 bit
    double sum[kChunk];
    float rk[kChunk], rq[kChunk], row[kChunk], state[4];
};

__device__ __forceinline__ float sum_over_16(float v) {
    v = v + __int_as_float(lane_xor<1>(__float_as_int(v)));
    v = v + __int_as_float(lane_xor<2>(__float_as_int(v)));
    v = butterfly_step4(v);
    return butterfly_step8(v);
}

template <int D, bool FP16>
__global__ __launch_bounds__(kThreads, 1) void scan_inputs_grad(ScanArgs a, ScanGradArgs d, ScanChunks w) {
    constexpr int PARTS = FP16 ? 2 : 1, TILES = D / 16, RAW = D + 8;
    __shared__ ScanInputsLds lds;
    const int tid = threadIdx.x, lane = tid % kWave, n = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int slot = blockIdx.x / a.key_heads, kh = blockIdx.x % a.key_heads;
    const int s = find_sequence(a.starts, a.seqs, slot);
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    const int first = (slot - scan_first_chunk(a.starts, s)) * kChunk;
    if (first < 0 || first >= seq.n) return;
    const int count = min(seq.n - first, kChunk), t0 = seq.a + first;
    const int64_t by_key = static_cast<int64_t>(slot) * a.key_heads + kh;
    const int E = a.value_dim, r0 = 16 * wave + 4 * g;
    if (tid < kChunk) {
        lds.rk[tid] = w.norms[by_key * 2 * kChunk + tid];
        lds.rq[tid] = w.norms[by_key * 2 * kChunk + kChunk + tid];
    }
    // Element of column n of tile t (as the fragments' rows), and the raw q and k there.
    auto element = [&](int t) { return 32 * (t / 2) + 8 * (n / 4) + 4 * (t % 2) + n % 4; };
    uint16_t q[TILES][4], k[TILES][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[t][i] = k[t][i] = 0;
            if (r0 + i < count) {
                q[t][i] = a.q[static_cast<int64_t>(t0 + r0 + i) * a.q_token + kh * a.q_head + element(t)];
                k[t][i] = a.k[static_cast<int64_t>(t0 + r0 + i) * a.k_token + kh * a.k_head + element(t)];
            }
        }
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 dq[TILES], dk[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) dq[t] = dk[t] = zero;
    const int64_t states = tape_states(w.slots, a.heads, D, E);
    for (int hv = 0; hv < a.group; ++hv) {
        const int h = kh * a.group + hv;
        const int64_t by_head = static_cast<int64_t>(slot) * a.heads + h, size = static_cast<int64_t>(D) * E;
        const uint16_t* tape = reinterpret_cast<const uint16_t*>(d.tape);
        const uint16_t* S = tape + by_head * 2 * size;
        const uint16_t* U = tape + states + by_head * 2 * kChunk * E;
        const uint16_t* dS = w.ds + by_head * 2 * size;
        const uint16_t* dR = w.dr + by_head * 2 * kChunk * E;
        if (tid < kChunk) lds.sum[tid] = w.sums[by_head * kChunk + tid];
        f32x4 so[TILES], sr[TILES], su[TILES], ou[4], ru[4];
#pragma unroll
        for (int t = 0; t < TILES; ++t) so[t] = sr[t] = su[t] = zero;
#pragma unroll
        for (int t = 0; t < 4; ++t) ou[t] = ru[t] = zero;
        float both = 0.0f;   // <S, dS>, a quarter of the tiles per wave
        for (int e = 8 * g; e < E; e += 32) {
            const int row = 16 * wave + n;
            uint4 o[PARTS], u[2], r[2];
            {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (row < count) x = ldg16(d.d_out + static_cast<int64_t>(t0 + row) * d.d_out_token + h * d.d_out_head + e);
                if constexpr (FP16) {
                    float f[8];
                    unpack16<true>(x, f);
                    Split2 p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = split2<2>(f[2 * j], f[2 * j + 1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[j] = make_uint4(p[0].part[j], p[1].part[j], p[2].part[j], p[3].part[j]);
                } else {
                    o[0] = x;
                }
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                u[p] = ldg16(U + (p * kChunk + row) * E + e);
                r[p] = ldg16(dR + (p * kChunk + row) * E + e);
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                uint4 bs[2], bd[2];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    bs[p] = ldg16(S + p * size + static_cast<int64_t>(element(t)) * E + e);
                    bd[p] = ldg16(dS + p * size + static_cast<int64_t>(element(t)) * E + e);
                }
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int x = 0; x + p < 2; ++x) {
                        if (x < PARTS) so[t] = mfma16x16x32(o[x], bs[p], so[t]);
                        sr[t] = mfma16x16x32(r[x], bs[p], sr[t]);
                        su[t] = mfma16x16x32(u[x], bd[p], su[t]);
                    }
                if (t % 4 == wave) {
                    float x[8], x1[8], y[8], y1[8];
                    unpack8(bs[0], x), unpack8(bs[1], x1), unpack8(bd[0], y), unpack8(bd[1], y1);
#pragma unroll
                    for (int j = 0; j < 8; ++j) both = __builtin_fmaf(x[j] + x1[j], y[j] + y1[j], both);
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t > wave) continue;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint4 b = ldg16(U + (p * kChunk + 16 * t + n) * E + e);
#pragma unroll
                    for (int x = 0; x + p < 2; ++x) {
                        if (x < PARTS) ou[t] = mfma16x16x32(o[x], b, ou[t]);
                        ru[t] = mfma16x16x32(r[x], b, ru[t]);
                    }
                }
            }
        }
        both = wave_butterfly_sum(both);
        if (lane == 0) lds.state[wave] = both;
        __syncthreads();   // (sums, and the last head's matrices are done with)
        const double last = lds.sum[kChunk - 1];
        f32x4 decay, rest;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            decay[i] = power(lds.sum[r0 + i]);
            rest[i] = power(last - lds.sum[r0 + i]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int j = 16 * t + n;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = r0 + r;
                const float fade = power(lds.sum[i] - lds.sum[j]);
                lds.b1[i * kPitch + j] = j <= i ? fade * ou[t][r] : 0.0f;
                lds.b2[i * kPitch + j] = j < i ? fade * ru[t][r] : 0.0f;
                if (i == j && i < count) {
                    const int64_t at = static_cast<int64_t>(t0 + i) * a.heads + h, from = static_cast<int64_t>(t0 + i) * a.beta_token + h;
                    const float b = scan_beta(a.beta_fp32 ? static_cast<const float*>(a.beta)[from]
                                                          : elem16<FP16>(static_cast<const uint16_t*>(a.beta)[from]));
                    const float db = ru[t][r] / b / b;
                    if (a.beta_fp32) static_cast<float*>(d.dbeta)[at] = db;
                    else static_cast<uint16_t*>(d.dbeta)[at] = static_cast<uint16_t>(pack16_2<FP16>(db, 0.0f));
                }
            }
        }
        __syncthreads();
        // The four products over tokens: rows of B1 and B2, then their columns.
        f32x4 by_q[TILES], by_row[TILES], by_col[TILES];
        f32x4 dot_state = zero;   // k_i . (dS u_i) e^(G_63 - G_i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            by_q[t] = so[t] * decay;
            by_row[t] = sr[t] * decay;
            by_col[t] = su[t] * rest;
#pragma unroll
            for (int i = 0; i < 4; ++i) dot_state[i] = __builtin_fmaf(elem16<FP16>(k[t][i]), by_col[t][i], dot_state[i]);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            uint4 q_row[2], k_row[2], q_col[2], k_col[2];
            const bool rows = 2 * ks <= wave, cols = 2 * ks + 1 >= wave;
            {
                float x[4][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int block = 2 * ks + j / 4, o = 16 * block + 4 * g + j % 4, own = 16 * wave + n;
                    const bool low = block <= wave, high = block >= wave;
                    const float rk = lds.rk[o], rq = lds.rq[o] * a.scale;
                    x[0][j] = low ? lds.b1[own * kPitch + o] * rk : 0.0f;
                    x[1][j] = low ? lds.b2[own * kPitch + o] * rk : 0.0f;
                    x[2][j] = high ? lds.b1[o * kPitch + own] * rq : 0.0f;
                    x[3][j] = high ? -lds.b2[o * kPitch + own] * rk : 0.0f;
                }
                auto parts = [&](uint4 (&to)[2], const float (&f)[8]) {
                    Split2 p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = split2<2>(f[2 * j], f[2 * j + 1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) to[j] = make_uint4(p[0].part[j], p[1].part[j], p[2].part[j], p[3].part[j]);
                };
                parts(q_row, x[0]);
                parts(k_row, x[1]);
                parts(q_col, x[2]);
                parts(k_col, x[3]);
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const int64_t at = ((by_key * TILES * 2 + t * 2 + ks) * PARTS + p) * kFragBytes + lane * 16;
                    const uint4 bk = ldg16(w.kt + at), bq = ldg16(w.qt + at);
#pragma unroll
                    for (int x = 0; x + p < 2; ++x) {
                        if (rows) {
                            by_q[t] = mfma16x16x32(q_row[x], bk, by_q[t]);
                            by_row[t] = mfma16x16x32(k_row[x], bk, by_row[t]);
                        }
                        if (cols) {
                            by_col[t] = mfma16x16x32(q_col[x], bq, by_col[t]);
                            by_col[t] = mfma16x16x32(k_col[x], bk, by_col[t]);
                        }
                    }
                }
        }
        f32x4 dot_q = zero, dot_k = zero;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dot_q[i] = __builtin_fmaf(elem16<FP16>(q[t][i]), by_q[t][i], dot_q[i]);
                dot_k[i] = __builtin_fmaf(elem16<FP16>(k[t][i]), -by_row[t][i] - by_col[t][i], dot_k[i]);
            }
            dq[t] += by_q[t];
            dk[t] += by_col[t] - by_row[t];
        }
        float moved = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float rk = lds.rk[r0 + i];
            const float sum = sum_over_16(dot_q[i] * lds.rq[r0 + i] * a.scale + dot_k[i] * rk);
            moved += sum_over_16(dot_state[i] * rk);
            if (n == 0) lds.row[r0 + i] = sum;
        }
        moved += __shfl_xor(moved, 16);
        moved += __shfl_xor(moved, 32);
        const float before = lds.state[0] + lds.state[1] + lds.state[2] + lds.state[3];
        __syncthreads();
        if (lane == 0) lds.state[wave] = moved;
        __syncthreads();
        if (wave == 0) {
            // From t on: the whole less what lies before.
            const float after = lds.state[0] + lds.state[1] + lds.state[2] + lds.state[3] +
                                before * power(last);
            float x = lds.row[kChunk - 1 - lane];
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const float other = __shfl_up(x, off);
                if (lane >= off) x += other;
            }
            const int t = kChunk - 1 - lane;
            if (t < count) d.dg[static_cast<int64_t>(t0 + t) * a.heads + h] = x + after;
        }
        __syncthreads();
    }
    // Through the norms, and out by rows.
    uint16_t* out = reinterpret_cast<uint16_t*>(lds.b1);
    for (int side = 0; side < 2; ++side) {
        f32x4 factor, back = zero;
#pragma unroll
        for (int i = 0; i < 4; ++i) factor[i] = side ? lds.rk[r0 + i] : lds.rq[r0 + i];
        if (a.normalize) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float dot = 0.0f;
#pragma unroll
                for (int t = 0; t < TILES; ++t)
                    dot = __builtin_fmaf(elem16<FP16>(side ? k[t][i] : q[t][i]), side ? dk[t][i] : dq[t][i], dot);
                back[i] = sum_over_16(dot) * factor[i] * factor[i];
            }
        }
        const float by = side ? 1.0f : a.scale;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = elem16<FP16>(side ? k[t][i] : q[t][i]);
                const float y = (side ? dk[t][i] : dq[t][i]) - x * back[i];
                out[(r0 + i) * RAW + element(t)] = static_cast<uint16_t>(pack16_2<FP16>(y * factor[i] * by, 0.0f));
            }
        __syncthreads();
        uint16_t* to = side ? d.dk : d.dq;
        for (int i = tid; i < kChunk * D / 8; i += kThreads) {
            const int r = i / (D / 8), e = i % (D / 8) * 8;
            if (r < count)
                *reinterpret_cast<uint4*>(to + (static_cast<int64_t>(t0 + r) * a.key_heads + kh) * D + e) =
                    *reinterpret_cast<const uint4*>(out + r * RAW + e);
        }
        __syncthreads();
    }
}

ScanChunks layout(const ScanArgs& a, bool fp16, bool grad, uint8_t* base, size_t* bytes) {
    ScanChunks w{};
    w.slots = scan_slots(a.tokens, a.seqs);
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
    w.p = take(by_head * kBlocks * (grad ? 3 : 2) * kFragBytes);
    w.vec = reinterpret_cast<float*>(take(by_head * 256 * sizeof(float)));
    w.kt = take(transposed);
    if (fp16) w.kf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
    if (grad) {
        const size_t columns = static_cast<size_t>(a.value_dim) * sizeof(uint16_t);
        w.qt = take(transposed);
        w.sums = reinterpret_cast<double*>(take(by_head * kChunk * sizeof(double)));
        w.norms = reinterpret_cast<float*>(take(by_key * 2 * kChunk * sizeof(float)));
        w.ds = reinterpret_cast<uint16_t*>(take(by_head * 2 * a.dim * columns));
        w.dr = reinterpret_cast<uint16_t*>(take(by_head * 2 * kChunk * columns));
    } else {
        if (fp16) w.qf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
        w.flags = reinterpret_cast<uint32_t*>(take(static_cast<size_t>(a.seqs) * a.heads * (a.value_dim / 16) * 4));
    }
    *bytes = at;
    return w;
}

// A launch holds fewer than 2^31 workgroups: slots * key_heads stay below
// (2^14 + 2^16) 2^10.
template <int D, bool FP16>
void launch(const ScanArgs& a, const ScanChunks& w, hipStream_t stream) {
    scan_prepare<D, FP16, false><<<static_cast<uint32_t>(w.slots) * a.key_heads, kThreads, 0, stream>>>(a, w);
    const int items = a.seqs * a.heads * (a.value_dim / 32);
    const int grid = (items + 7) / 8 * 8;
    if (a.tape != nullptr) scan_chunks<D, 2, FP16, true><<<grid, kThreads, 0, stream>>>(a, w);
    else if (items <= 128) scan_chunks<D, 1, FP16, false><<<(2 * items + 7) / 8 * 8, kThreads, 0, stream>>>(a, w);
    else scan_chunks<D, 2, FP16, false><<<grid, kThreads, 0, stream>>>(a, w);
}

template <int D, bool FP16>
void launch_grad(const ScanArgs& a, const ScanGradArgs& d, const ScanChunks& w, hipStream_t stream) {
    const uint32_t chunks = static_cast<uint32_t>(w.slots) * a.key_heads;
    scan_prepare<D, FP16, true><<<chunks, kThreads, 0, stream>>>(a, w);
    const int items = a.seqs * a.heads * (a.value_dim / 32);
    scan_chunks_grad<D, FP16><<<(items + 7) / 8 * 8, kThreads, 0, stream>>>(a, d, w);
    scan_inputs_grad<D, FP16><<<chunks, kThreads, 0, stream>>>(a, d, w);
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
    return static_cast<size_t>(scan_slots(a.tokens, a.seqs)) * a.heads * 2 * (a.dim + kChunk) * a.value_dim *
           sizeof(uint16_t);
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
