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

// t = (I + a)^-1 for the strictly lower triangular a, by blocks of 16: those of
// the diagonal by substitution, a lane per column; below, block column by block
// column, T_ij = -T_ii sum_k A_ik T_kj with fp32 matrix instructions, a wave per
// block column.
__device__ __forceinline__ void invert(PrepareLds& lds, int wave, int lane) {
    const int n = lane % 16, g = lane / 16;
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float acc = r == n ? 1.0f : 0.0f;
        const float* row = lds.a + (16 * wave + r) * kPitch + 16 * wave;
#pragma unroll
        for (int l = 0; l < r; ++l) acc = __builtin_fmaf(-row[l], x[l], acc);
        x[r] = acc;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (r / 4 == g) lds.t[(16 * wave + r) * kPitch + 16 * wave + n] = x[r];
    __syncthreads();
    const int j = wave;
    for (int i = j + 1; i < 4; ++i) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = j; k < i; ++k) {
            const float* row = lds.a + (16 * i + n) * kPitch + 16 * k + 4 * g;
            const float* col = lds.t + (16 * k + 4 * g) * kPitch + 16 * j + n;
#pragma unroll
            for (int s = 0; s < 4; ++s)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(row[s], col[s * kPitch], acc, 0, 0, 0);
        }
        f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
        const float* row = lds.t + (16 * i + n) * kPitch + 16 * i + 4 * g;
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

template <int D, bool FP16>
__global__ __launch_bounds__(kThreads, 3) void scan_prepare(ScanArgs a, ScanChunks w) {
    constexpr int RAW = D + 8;   // 16-bit elements of a row in LDS
    constexpr int PARTS = FP16 ? 2 : 1;
    __shared__ PrepareLds lds;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = lane % 16, g = lane / 16;
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
        lds.rq[16 * wave + n] = a.scale * (a.normalize ? 1.0f / __builtin_sqrtf(q2 + 1e-6f) : 1.0f);
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
    }
    if constexpr (FP16) {
        for (int ks = 0; ks < D / 32; ++ks) {
            float x[8];
            const int64_t at = (((by_key * 4 + wave) * (D / 32) + ks) * PARTS) * kFragBytes + lane * 16;
            unpack16<FP16>(*reinterpret_cast<const uint4*>(raw_k + (16 * wave + n) * RAW + 32 * ks + 8 * g), x);
            store_parts<PARTS>(w.kf + at, x);
            unpack16<FP16>(*reinterpret_cast<const uint4*>(raw_q + (16 * wave + n) * RAW + 32 * ks + 8 * g), x);
            store_parts<PARTS>(w.qf + at, x);
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
            const double sum = wave_scan_f64(gl);
            lds.sum[lane] = sum;
            lds.beta[lane] = b;
            const double last = __shfl(sum, kWave - 1);
            const float decay = expf(static_cast<float>(sum)), rest = expf(static_cast<float>(last - sum));
            float* vec = w.vec + by_head * 256;
            vec[lane] = decay * lds.rk[lane];
            vec[64 + lane] = decay * lds.rq[lane];
            vec[128 + lane] = rest * lds.rk[lane];
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
                const float fade = expf(static_cast<float>(lds.sum[i] - lds.sum[j])) * lds.rk[j];
                lds.a[i * kPitch + j] = j < i ? fade * lds.rk[i] * lds.beta[j] * kk[t][r] : 0.0f;
                lds.b[i * kPitch + j] = j <= i ? fade * lds.rq[i] * qk[t][r] : 0.0f;
            }
        }
        __syncthreads();
        invert(lds, wave, lane);
        const int row = 16 * wave + n;
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

template <int D, int NC, bool FP16>
struct ScanLoads {
    static constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64;
    uint4 k[D / 32][PARTS], q[D / 32][PARTS], t[2][3], p[2][2], kt[TPW][2][PARTS];
    uint32_t v[4][NC / 2 + NC % 2];
    f32x4 fk, fq, fu;   // factors of the lane's four tokens
    float decay;
};

template <int NC>
__device__ __forceinline__ void load_cols(uint32_t (&v)[NC / 2 + NC % 2], const uint16_t* p) {
    if constexpr (NC == 1) v[0] = *p;
    if constexpr (NC == 2) v[0] = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (NC == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v[0] = x.x, v[1] = x.y;
    }
}
template <int NC, bool FP16>
__device__ __forceinline__ float col_value(const uint32_t (&v)[NC / 2 + NC % 2], int c) {
    return elem16<FP16>(static_cast<uint16_t>(c % 2 ? v[c / 2] >> 16 : v[c / 2]));
}

template <int D, int NC, bool FP16>
__global__ __launch_bounds__(kThreads, 2) void scan_chunks(ScanArgs a, ScanChunks w) {
    constexpr int PARTS = FP16 ? 2 : 1, TPW = D / 64, KS = D / 32;
    __shared__ ScanLds<D, NC> lds;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = lane % 16, g = lane / 16;
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
    uint32_t* flag = w.flags + (static_cast<int64_t>(s) * a.heads + h) * (a.value_dim / 32) + 16 * NC * cb / 32;
    const int into = scan_slot(a.into, s, a.pool);
    const bool fresh = a.initial == nullptr || (a.fresh != nullptr && a.fresh[s] != 0);
    const int from = fresh ? 0 : scan_slot(a.from, s, a.pool);
    if (into < 0 || from < 0) {
        if (tid == 0) *flag = 0;
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
    ScanLoads<D, NC, FP16> x;
    auto load_rows = [&](int ch) {
        if constexpr (FP16) {
            const int64_t at = (((slot0 + ch) * a.key_heads + kh) * 4 + wave) * KS * PARTS * kFragBytes + lane * 16;
#pragma unroll
            for (int i = 0; i < KS * PARTS; ++i) {
                x.k[i / PARTS][i % PARTS] = ldg16(w.kf + at + i * kFragBytes);
                x.q[i / PARTS][i % PARTS] = ldg16(w.qf + at + i * kFragBytes);
            }
        } else {
            const int t = ch * kChunk + 16 * wave + n;
            const bool in = t < seq.n;
            const int64_t row = seq.a + (in ? t : 0);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                x.k[i][0] = x.q[i][0] = make_uint4(0u, 0u, 0u, 0u);
                if (in) {
                    x.k[i][0] = ldg16(a.k + row * a.k_token + kh * a.k_head + 32 * i + 8 * g);
                    x.q[i][0] = ldg16(a.q + row * a.q_token + kh * a.q_head + 32 * i + 8 * g);
                }
            }
        }
    };
    auto load_t = [&](int ch) {
        const int64_t at = (((slot0 + ch) * a.heads + h) * kBlocks) * 3 * kFragBytes + lane * 16;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            x.t[0][p] = ldg16(w.t + at + (lower_block(0, wave) * 3 + p) * kFragBytes);
            if (wave >= 2) x.t[1][p] = ldg16(w.t + at + (lower_block(1, wave) * 3 + p) * kFragBytes);
        }
    };
    auto load_rest = [&](int ch) {
        const int64_t by_head = (slot0 + ch) * a.heads + h, by_key = (slot0 + ch) * a.key_heads + kh;
        const int64_t at = by_head * kBlocks * 2 * kFragBytes + lane * 16;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            x.p[0][p] = ldg16(w.p + at + (lower_block(0, wave) * 2 + p) * kFragBytes);
            if (wave >= 2) x.p[1][p] = ldg16(w.p + at + (lower_block(1, wave) * 2 + p) * kFragBytes);
        }
#pragma unroll
        for (int i = 0; i < TPW * 2 * PARTS; ++i)
            x.kt[i / (2 * PARTS)][i / PARTS % 2][i % PARTS] =
                ldg16(w.kt + ((by_key * (D / 16) + wave * TPW) * 2 * PARTS + i) * kFragBytes + lane * 16);
        const float* vec = w.vec + by_head * 256;
        const int r0 = 16 * wave + 4 * g;
        x.fk = *reinterpret_cast<const f32x4*>(vec + r0);
        x.fq = *reinterpret_cast<const f32x4*>(vec + 64 + r0);
        x.fu = *reinterpret_cast<const f32x4*>(vec + 128 + r0);
        x.decay = vec[192];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ch * kChunk + r0 + i;
#pragma unroll
            for (int c = 0; c < NC / 2 + NC % 2; ++c) x.v[i][c] = 0u;
            if (t < seq.n) load_cols<NC>(x.v[i], a.v + static_cast<int64_t>(seq.a + t) * a.v_token + h * a.v_head + col);
        }
    };
    if (chunks > 0) {
        load_rows(0);
        load_t(0);
        load_rest(0);
    }
    bool odd = false;   // a number that is not finite
    for (int ch = 0; ch < chunks; ++ch) {
        const int next = min(ch + 1, chunks - 1);
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                put_parts<3>(lds.s, (wave * TPW + i) / 2, (wave * TPW + i) % 2, c, lane, S[i][c]);
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
        load_rows(next);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            f32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = col_value<NC, FP16>(x.v[i], c) - x.fk[i] * ks[c][i];
            put_parts<3>(lds.r, wave / 2, wave % 2, c, lane, r);
        }
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
        load_t(next);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (__float_as_uint(u[c][i]) & 0x7f800000u) == 0x7f800000u;
            put_parts<2>(lds.u, wave / 2, wave % 2, c, lane, u[c]);
            put_parts<3>(lds.uk, wave / 2, wave % 2, c, lane, u[c] * x.fu);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                S[i][c] *= x.decay;
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
            o[c] = qs[c] * x.fq;
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
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ch * kChunk + 16 * wave + 4 * g + i;
            if (t >= seq.n) continue;
            uint16_t* to = a.out + static_cast<int64_t>(seq.a + t) * a.out_token + h * a.out_head + col;
            if constexpr (NC == 1) {
                *to = static_cast<uint16_t>(pack16_2<FP16>(o[0][i], 0.0f));
            } else if constexpr (NC == 2) {
                *reinterpret_cast<uint32_t*>(to) = pack16_2<FP16>(o[0][i], o[1][i]);
            } else {
                *reinterpret_cast<uint2*>(to) =
                    make_uint2(pack16_2<FP16>(o[0][i], o[1][i]), pack16_2<FP16>(o[NC - 2][i], o[NC - 1][i]));
            }
        }
        load_rest(next);
    }
    // Where a value was not finite, a product's zero weights have let it through
    // to earlier tokens: the next launch goes through these columns again.
    if (__syncthreads_or(odd)) {
        if (tid == 0) *flag = 1;
        return;
    }
    if (tid == 0) *flag = 0;
#pragma unroll
    for (int x1 = 0; x1 < TPW; ++x1)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                a.final[(static_cast<int64_t>(into) * a.heads + h) * size +
                        static_cast<int64_t>(row_of(x1, i)) * a.value_dim + col + c] = S[x1][c][i];
}

ScanChunks layout(const ScanArgs& a, bool fp16, uint8_t* base, size_t* bytes) {
    ScanChunks w{};
    w.slots = a.tokens / kChunk + a.seqs;
    w.parts = fp16 ? 2 : 1;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return base + here;
    };
    const size_t by_head = static_cast<size_t>(w.slots) * a.heads, by_key = static_cast<size_t>(w.slots) * a.key_heads;
    w.t = take(by_head * kBlocks * 3 * kFragBytes);
    w.p = take(by_head * kBlocks * 2 * kFragBytes);
    w.vec = reinterpret_cast<float*>(take(by_head * 256 * sizeof(float)));
    w.kt = take(by_key * (a.dim / 16) * 2 * w.parts * kFragBytes);
    if (fp16) {
        w.kf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
        w.qf = take(by_key * 4 * (a.dim / 32) * w.parts * kFragBytes);
    }
    w.flags = reinterpret_cast<uint32_t*>(take(static_cast<size_t>(a.seqs) * a.heads * (a.value_dim / 32) * 4));
    *bytes = at;
    return w;
}

template <int D, bool FP16>
void launch(const ScanArgs& a, const ScanChunks& w, hipStream_t stream) {
    scan_prepare<D, FP16><<<static_cast<uint32_t>(w.slots) * a.key_heads, kThreads, 0, stream>>>(a, w);
    const int items = a.seqs * a.heads * (a.value_dim / 32);
    scan_chunks<D, 2, FP16><<<(items + 7) / 8 * 8, kThreads, 0, stream>>>(a, w);
}

}  // namespace

size_t scan_chunk_bytes(const ScanArgs& a, bool fp16) {
    size_t bytes = 0;
    layout(a, fp16, nullptr, &bytes);
    return bytes;
}

hipError_t launch_scan_chunks(const ScanArgs& a, bool fp16, void* workspace, const uint32_t** flags,
                              hipStream_t stream) {
    size_t bytes = 0;
    const ScanChunks w = layout(a, fp16, static_cast<uint8_t*>(workspace), &bytes);
    if (a.dim == 64) {
        if (fp16) launch<64, true>(a, w, stream); else launch<64, false>(a, w, stream);
    } else {
        if (fp16) launch<128, true>(a, w, stream); else launch<128, false>(a, w, stream);
    }
    *flags = w.flags;
    return hipGetLastError();
}

}  // namespace lrmoe
