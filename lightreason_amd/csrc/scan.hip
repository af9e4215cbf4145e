// The gated delta rule over packed sequences: per sequence and value head a
// state S [dim][value_dim] in fp32 and, token by token,
//     S <- e^g S,  u = beta (v - S^T k),  S <- S + k u^T,  out = scale S^T q,
// the recurrence of edge35b/delta_decode.py:11-36 with nothing rounded but the
// inputs and the outputs.  A column of S needs no other column, so the work is
// split over sequences, value heads and blocks of columns.
#include "scan.h"

namespace lrmoe {
namespace {

// ---- token by token --------------------------------------------------------------
//
// A wave holds 32 columns of a state: lane l columns 4 (l % 8) .. + 3 of rows
// (D / 8) (l / 8) .. + D / 8 - 1.  One pass over the state per token gives S^T k
// and S^T q of the faded state together (out = e^g S^T q + (q . k) u), so that
// the sums over rows meet once; then S = e^g S + k u^T.  Bound by the states, read
// and written once (256 single tokens of 32 heads of 128 x 128: 198 us, 5.4 TB/s,
// a device copy's rate); one sequence alone by a launch and its loads (5 us).
template <int D, bool FP16>
struct RecurToken {
    static constexpr int ROWS = D / 8;
    uint4 k[ROWS / 8], q[ROWS / 8];
    uint2 v;
    float g, beta;
};

template <int D, bool FP16>
__device__ __forceinline__ void recur_load(const ScanArgs& a, RecurToken<D, FP16>& x, int t, int h, int kh, int rows0,
                                           int col) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        x.k[i] = ldg16(a.k + t * a.k_token + kh * a.k_head + rows0 + 8 * i);
        x.q[i] = ldg16(a.q + t * a.q_token + kh * a.q_head + rows0 + 8 * i);
    }
    x.v = *reinterpret_cast<const uint2*>(a.v + t * a.v_token + h * a.v_head + col);
    x.g = a.g[t * a.g_token + h];
    x.beta = a.beta_fp32 ? static_cast<const float*>(a.beta)[t * a.beta_token + h]
                         : elem16<FP16>(static_cast<const uint16_t*>(a.beta)[t * a.beta_token + h]);
}

// With flags given the chunked form has run: what is left are short sequences and
// the blocks of columns that the flags mark, in which it met a number that is not
// finite.
template <int D, bool FP16>
__global__ __launch_bounds__(256) void scan_recur(ScanArgs a, const uint32_t* flags) {
    constexpr int ROWS = D / 8;
    const int lane = threadIdx.x % kWave;
    const int blocks = a.value_dim / 32;
    const int64_t wave = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kWave;
    if (wave >= static_cast<int64_t>(a.seqs) * a.heads * blocks) return;
    const int cb = static_cast<int>(wave % blocks);
    const int h = static_cast<int>(wave / blocks % a.heads), s = static_cast<int>(wave / blocks / a.heads);
    const int kh = h / a.group;
    const int rows0 = ROWS * (lane / 8), col = 32 * cb + 4 * (lane % 8);
    const ScanSeq seq = scan_seq(a.starts, s, a.tokens);
    bool marked = true;
    if (flags != nullptr && seq.n > a.token_wise) {
        const uint32_t first = flags[2 * wave], last = flags[2 * wave + 1];   // of 16 columns each
        if ((first | last) == 0) return;
        marked = (lane % 8 < 4 ? first : last) != 0;
    }
    // Rows of no sequence.
    if (a.clear && flags == nullptr && (s == 0 || s == a.seqs - 1)) {
        const int64_t row0 = h * a.out_head + col;
        const int head = min(max(a.starts[0], 0), a.tokens), tail = min(max(a.starts[a.seqs], 0), a.tokens);
        if (s == 0)
            for (int t = lane / 8; t < head; t += 8)
                *reinterpret_cast<uint2*>(a.out + t * a.out_token + row0) = make_uint2(0u, 0u);
        if (s == a.seqs - 1)
            for (int t = tail + lane / 8; t < a.tokens; t += 8)
                *reinterpret_cast<uint2*>(a.out + t * a.out_token + row0) = make_uint2(0u, 0u);
    }
    const int into = scan_slot(a.into, s, a.pool);
    const bool fresh = a.initial == nullptr || (a.fresh != nullptr && a.fresh[s] != 0);
    const int from = fresh ? 0 : scan_slot(a.from, s, a.pool);
    if (into < 0 || from < 0) return;
    const int64_t state_size = static_cast<int64_t>(D) * a.value_dim;
    float S[ROWS][4];
    if (fresh) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) S[i][0] = S[i][1] = S[i][2] = S[i][3] = 0.0f;
    } else {
        const float* p = a.initial + (static_cast<int64_t>(from) * a.heads + h) * state_size +
                         static_cast<int64_t>(rows0) * a.value_dim + col;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const uint4 x = ldg16(p + i * a.value_dim);
            S[i][0] = __uint_as_float(x.x), S[i][1] = __uint_as_float(x.y);
            S[i][2] = __uint_as_float(x.z), S[i][3] = __uint_as_float(x.w);
        }
    }
    RecurToken<D, FP16> next;
    if (seq.n > 0) recur_load<D, FP16>(a, next, seq.a, h, kh, rows0, col);
    for (int t = seq.a; t < seq.a + seq.n; ++t) {
        const RecurToken<D, FP16> x = next;
        if (t + 1 < seq.a + seq.n) recur_load<D, FP16>(a, next, t + 1, h, kh, rows0, col);
        float k[ROWS], q[ROWS], v[4];
#pragma unroll
        for (int i = 0; i < ROWS / 8; ++i) {
            unpack16<FP16>(x.k[i], k + 8 * i);
            unpack16<FP16>(x.q[i], q + 8 * i);
        }
        v[0] = elem16<FP16>(static_cast<uint16_t>(x.v.x)), v[1] = elem16<FP16>(static_cast<uint16_t>(x.v.x >> 16));
        v[2] = elem16<FP16>(static_cast<uint16_t>(x.v.y)), v[3] = elem16<FP16>(static_cast<uint16_t>(x.v.y >> 16));
        float sk[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sq[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float kk = 0.0f, qq = 0.0f, qk = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] = __builtin_fmaf(S[i][j], k[i], sk[j]);
                sq[j] = __builtin_fmaf(S[i][j], q[i], sq[j]);
            }
            kk = __builtin_fmaf(k[i], k[i], kk);
            qq = __builtin_fmaf(q[i], q[i], qq);
            qk = __builtin_fmaf(q[i], k[i], qk);
        }
        qk = sum_over_8(qk);
        float rk = 1.0f, rq = a.scale;
        if (a.normalize) {
            rk = 1.0f / __builtin_sqrtf(sum_over_8(kk) + 1e-6f);
            rq *= 1.0f / __builtin_sqrtf(sum_over_8(qq) + 1e-6f);
        }
        const float decay = expf(scan_log(x.g));
        float out[4], u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = x.beta * (v[j] - decay * rk * sum_over_8(sk[j]));
            out[j] = rq * __builtin_fmaf(qk * rk, u[j], decay * sum_over_8(sq[j]));
            u[j] *= rk;
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf(k[i], u[j], decay * S[i][j]);
        if (lane < 8 && marked)
            *reinterpret_cast<uint2*>(a.out + t * a.out_token + h * a.out_head + col) =
                make_uint2(pack16_2<FP16>(out[0], out[1]), pack16_2<FP16>(out[2], out[3]));
    }
    if (!marked) return;
    float* p = a.final + (static_cast<int64_t>(into) * a.heads + h) * state_size +
               static_cast<int64_t>(rows0) * a.value_dim + col;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        *reinterpret_cast<float4*>(p + i * a.value_dim) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
}

}  // namespace

// Tokens up to which a sequence goes token by token: about what the chunked
// form's launches and its chunk of 64 cost. Measured at 20 to 26 tokens where the
// waves are few (1 sequence of 32 heads and 128 columns: 16 tokens 20 us against
// 20, 32 tokens 37 against 23) and 35 to 55 where they fill the card (64 of
// them: 32 tokens 226 against 324, 48 tokens 325 against 340). Sequences of one
// call may go either way. (The tape is the chunked form's.)
static int token_wise(const ScanArgs& a) {
    if (a.tape != nullptr) return 0;
    return static_cast<int64_t>(a.seqs) * a.heads * (a.value_dim / 32) <= 1024 ? 24 : 40;
}

size_t delta_scan_workspace_bytes(ScanArgs a, bool fp16, int max_new) {
    a.token_wise = token_wise(a);
    return max_new <= a.token_wise ? 0 : scan_chunk_bytes(a, fp16);
}

hipError_t launch_delta_scan(ScanArgs a, bool fp16, int max_new, void* workspace, hipStream_t stream) {
    const uint32_t* flags = nullptr;
    a.token_wise = token_wise(a);
    if (max_new > a.token_wise) {
        const hipError_t err = launch_scan_chunks(a, fp16, workspace, &flags, stream);
        if (err != hipSuccess) return err;
    }
    const int64_t waves = static_cast<int64_t>(a.seqs) * a.heads * (a.value_dim / 32);
    const int per = waves < 2048 ? 1 : 4;
    const dim3 grid(static_cast<uint32_t>((waves + per - 1) / per)), block(per * kWave);
    auto run = [&](auto kernel) { kernel<<<grid, block, 0, stream>>>(a, flags); };
    if (a.dim == 64) {
        if (fp16) run(scan_recur<64, true>); else run(scan_recur<64, false>);
    } else {
        if (fp16) run(scan_recur<128, true>); else run(scan_recur<128, false>);
    }
    return hipGetLastError();
}

}  // namespace lrmoe
