// k_ssm.hip -- the state-space mixer's operators: GGML_OP_SSM_CONV (the short
// depthwise causal convolution over the carried and the step's columns) and
// GGML_OP_SSM_SCAN (the selective scan).
#include <type_traits>

#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

// ---------------------------------------------------------------- conv ---

// y[c, t, s] = sum_j w[j, c] sx[t + j, c, s]
__global__ __launch_bounds__(256) void k_ssm_conv(ssm_conv_args a) {
    const int64_t n = a.channels * a.tokens * a.seqs;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) {
        const int64_t c = i % a.channels, t = i / a.channels % a.tokens, s = i / (a.channels * a.tokens);
        const char * row = a.sx + c * a.sx_nb1 + s * a.sx_nb2;
        const float * w = (const float *) (a.w + c * a.w_nb1);
        float y = 0.0f;
        for (int j = 0; j < a.taps; j++) y = fmaf(w[j], *(const float *) (row + (t + j) * a.sx_nb0), y);
        a.out[i] = y;
    }
}

void launch_ssm_conv(const ssm_conv_args & a, hipStream_t s, int n_cu) {
    const int64_t n = a.channels * a.tokens * a.seqs;
    if (n == 0) return;
    const int64_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(k_ssm_conv, dim3((unsigned) (blocks < 16 * n_cu ? blocks : 16 * n_cu)), dim3(256), 0, s, a);
}

// ---------------------------------------------------------------- scan ---

// softplus as the op defines it: the identity past 20
__device__ __forceinline__ float ssm_softplus(float v) { return v <= 20.0f ? log1pf(expf(v)) : v; }

// token by token: W lanes hold one (sequence, head, channel) row's state, R
// elements a lane
template <int W, int R>
__global__ __launch_bounds__(256) void k_ssm_scan_rows(ssm_scan_args a) {
    const int lane = threadIdx.x % W;
    const int64_t row = ((int64_t) blockIdx.x * 256 + threadIdx.x) / W;
    const int64_t rows = (int64_t) a.seqs * a.heads * a.dim;
    if (row >= rows) return;  // whole groups of W lanes
    const int p = (int) (row % a.dim), h = (int) (row / a.dim % a.heads), s = (int) (row / ((int64_t) a.dim * a.heads));
    const int g = h / (a.heads / a.groups);
    const int64_t slot = a.ids[s];
    const bool has = slot >= 0 && slot < a.slots;
    const float * s0 = (const float *) (a.s + (has ? slot : 0) * a.s_nb3) + ((int64_t) h * a.dim + p) * a.n;
    float st[R], av[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int k = lane + W * r;
        st[r] = has && k < a.n ? s0[k] : 0.0f;
        av[r] = k < a.n ? *(const float *) (a.A + h * a.A_nb1 + (a.a_elem ? 4 * k : 0)) : 0.0f;
    }
    for (int64_t t = 0; t < a.tokens; t++) {
        const float dt = ssm_softplus(*(const float *) (a.dt + 4 * h + t * a.dt_nb1 + s * a.dt_nb2));
        const float xv = *(const float *) (a.x + 4 * p + h * a.x_nb1 + t * a.x_nb2 + s * a.x_nb3) * dt;
        const float * b = (const float *) (a.B + g * a.B_nb1 + t * a.B_nb2 + s * a.B_nb3);
        const float * c = (const float *) (a.C + g * a.C_nb1 + t * a.C_nb2 + s * a.C_nb3);
        float y = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int k = lane + W * r;
            const bool ok = k < a.n;
            st[r] = fmaf(st[r], expf(dt * av[r]), ok ? xv * b[k] : 0.0f);
            y = fmaf(st[r], ok ? c[k] : 0.0f, y);
        }
        y = group_sum<W>(y);
        if (lane == 0) a.y[((s * a.tokens + t) * a.heads + h) * a.dim + p] = y;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int k = lane + W * r;
        if (k < a.n) a.out[row * a.n + k] = st[r];
    }
}

// ------------------------------------------------- scan, a decay a head ---
//
// Chunks of 64 tokens as matrix products. With c_t the sum of the log decays
// from the chunk's start to token t, u_j = dt_j x_j and H the state entering:
//   y_t  = exp(c_t) H C_t + sum_{j <= t} (C_t . B_j) exp(c_t - c_j) u_j
//   H'   = exp(c_L) H + sum_j exp(c_L - c_j) u_j B_j^T
// which takes 4 P N + O(64 P) multiply-adds a token on the matrix cores, where
// the token by token form takes 3 P N vector operations and a sum over lanes.
//
// Products of f32 operands on the f16 matrix cores: every row (or column) that
// a sum runs along is scaled by a power of two so that its largest element is
// in [2^13, 2^14), and split into f16 hi + lo (22 bits down to 2^-17 of that
// element, 2^-39 of it below); a product is hi hi + hi lo + lo hi, summed in
// f32: a sum is off by some 2^-22 of its terms' magnitudes and 2^-38 of its
// operands' largest elements' product. Against f32 MFMAs (an
// eighth of the f16 rate after the three products) the sums are as good as
// f32's own roundings; states, decays and sums are f32, the log decays f64
// until they are split into whole and fractional powers of two.
//
// k_ssm_split makes the operands that a group's heads share: C in rows and B
// in columns, split, with their scales, and C_t . B_j. k_ssm_chunks gives a
// workgroup a (sequence, head, 64 channels, segment of chunks): wave w owns
// the state's rows n in its quarter (accumulator layout) and, for y, 16
// tokens. Where there are few heads the sequence is cut into segments: the
// first pass (OUT false) makes each segment's own state from zeros, and the
// second starts from the earlier segments' states, decayed and added.
//
// Non-finite values would spread inside a chunk (0 * inf), and tokens far
// larger than the ones before them would cost those their bits: such a chunk,
// and one whose decays leave the exact range, runs token by token
// (ssm_chunk_slow), where a value reaches what the recurrence takes it to.

typedef float ssm_v4f __attribute__((ext_vector_type(4)));
typedef _Float16 ssm_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 ssm_v4h __attribute__((ext_vector_type(4)));

constexpr int kSsmL = 64;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ ssm_v4f ssm_mfma(ssm_v8h a, ssm_v8h b, ssm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// 2^e, e a whole number in f32's normal range
__device__ __forceinline__ float ssm_pow2(int e) { return __uint_as_float((uint32_t) (e + 127) << 23); }
// the exponent k that brings a largest magnitude (its bits) into [2^13, 2^14);
// 0 for zero, at most 74 (a magnitude under 2^-60 keeps fewer bits)
__device__ __forceinline__ int ssm_scale(uint32_t bits) {
    const int e = (int) (bits >> 23) - 127;  // floor(log2), -127 for zero and subnormals
    return bits == 0 ? 0 : min(13 - e, 74);
}
__device__ __forceinline__ uint32_t ssm_mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
template <int W>
__device__ __forceinline__ uint32_t ssm_group_max(uint32_t v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = max(v, (uint32_t) __shfl_xor((int) v, o, W));
    return v;
}
__device__ __forceinline__ bool ssm_finite(uint32_t mag) { return mag < 0x7F800000u; }

// the operands' places in scratch, for NP = the padded state size
struct ssm_chunk_args {
    ssm_scan_args a;
    _Float16 *c_hi, *c_lo;  // [seq, group][token][NP]
    _Float16 *b_hi, *b_lo;  // [seq, group][chunk][NP][64 tokens]
    float *c_s, *b_s;       // [seq, group][token]: a row's value is its operand times this
    float * cb;             // [seq, group][chunk][64][64]: C_t . B_j for 16-blocks of j up to t's
    int * bad;              // [seq, group][chunk][4]: whether a quarter's rows hold a non-finite value
    float * seg_state;      // [seq, head, channel block][segment][64][NP]
    double * seg_decay;     // [seq, head][segment]: its log2 decay
    int64_t chunks;
    int segs, seg_chunks, pblocks;
};

template <int NP>
__global__ __launch_bounds__(256) void k_ssm_split(ssm_chunk_args q) {
    constexpr int kRow = NP + 4;
    __shared__ float sb[kSsmL][kRow];
    __shared__ float sc[16][kRow];
    const ssm_scan_args & a = q.a;
    const int part = blockIdx.x % 4;
    const int64_t chunk = blockIdx.x / 4 % q.chunks, sg = blockIdx.x / 4 / q.chunks;
    const int s = (int) (sg / a.groups), g = (int) (sg % a.groups);
    const int64_t t0 = chunk * kSsmL;
    const int tid = threadIdx.x;
    const char * B = a.B + g * a.B_nb1 + s * a.B_nb3;
    const char * C = a.C + g * a.C_nb1 + s * a.C_nb3;
    for (int i = tid; i < kSsmL * NP; i += 256) {
        const int t = i / NP, n = i % NP;
        const bool ok = t0 + t < a.tokens && n < a.n;
        sb[t][n] = ok ? ((const float *) (B + (t0 + t) * a.B_nb2))[n] : 0.0f;
    }
    for (int i = tid; i < 16 * NP; i += 256) {
        const int t = 16 * part + i / NP, n = i % NP;
        const bool ok = t0 + t < a.tokens && n < a.n;
        sc[i / NP][n] = ok ? ((const float *) (C + (t0 + t) * a.C_nb2))[n] : 0.0f;
    }
    __syncthreads();
    const int64_t tp = q.chunks * kSsmL;
    // rows: 16 threads each
    const int row = tid / 16, sub = tid % 16;
    uint32_t mb = 0, mc = 0;
    for (int n = sub; n < NP; n += 16) {
        mb = max(mb, ssm_mag(sb[16 * part + row][n]));
        mc = max(mc, ssm_mag(sc[row][n]));
    }
    mb = ssm_group_max<16>(mb);
    mc = ssm_group_max<16>(mc);
    const int kb = ssm_finite(mb) ? ssm_scale(mb) : 0, kc = ssm_finite(mc) ? ssm_scale(mc) : 0;
    const int any = __syncthreads_or(!ssm_finite(mb) || !ssm_finite(mc));
    if (tid == 0) q.bad[(sg * q.chunks + chunk) * 4 + part] = any;
    const int64_t t = t0 + 16 * part + row;
    if (sub == 0) {
        q.b_s[sg * tp + t] = ssm_pow2(-kb);
        q.c_s[sg * tp + t] = ssm_pow2(-kc);
    }
    const float fc = ssm_pow2(kc), fb = ssm_pow2(kb);
    for (int n = 8 * sub; n < NP; n += 128) {
        ssm_v8h hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = sc[row][n + e] * fc;
            hi[e] = (_Float16) v;
            lo[e] = (_Float16) (v - (float) hi[e]);
        }
        *(ssm_v8h *) (q.c_hi + (sg * tp + t) * NP + n) = hi;
        *(ssm_v8h *) (q.c_lo + (sg * tp + t) * NP + n) = lo;
    }
    // C . B: wave w the block of tokens 16 w .. (not past its own), K in an
    // order both operands share
    const int lane = tid & 63, wave = tid >> 6, r = lane & 15, gq = lane >> 4;
    if (wave <= part) {
        ssm_v4f acc = {0, 0, 0, 0};
        for (int n = 4 * gq; n < NP; n += 16) {
            const float4 x = *(const float4 *) &sc[r][n], y = *(const float4 *) &sb[16 * wave + r][n];
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, acc, 0, 0, 0);
        }
        float * cb = q.cb + ((sg * q.chunks + chunk) * kSsmL + 16 * part) * kSsmL + 16 * wave;
#pragma unroll
        for (int i = 0; i < 4; i++) cb[(4 * gq + i) * kSsmL + r] = acc[i];
    }
    // B's columns: the rows scaled in place, then 16 tokens of a column a thread
    __syncthreads();
    for (int n = sub; n < NP; n += 16) sb[16 * part + row][n] *= fb;
    __syncthreads();
    if (tid < NP) {
        _Float16 * oh = q.b_hi + ((sg * q.chunks + chunk) * NP + tid) * kSsmL + 16 * part;
        _Float16 * ol = q.b_lo + ((sg * q.chunks + chunk) * NP + tid) * kSsmL + 16 * part;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            ssm_v8h hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = sb[16 * part + 8 * h + e][tid];
                hi[e] = (_Float16) v;
                lo[e] = (_Float16) (v - (float) hi[e]);
            }
            *(ssm_v8h *) (oh + 8 * h) = hi;
            *(ssm_v8h *) (ol + 8 * h) = lo;
        }
    }
}

constexpr int kSsmXRow = kSsmL + 8;  // halfs of a staged channel's tokens, padded

template <int NP>
struct ssm_lds {
    _Float16 x[4][64][kSsmXRow];  // u for y (hi, lo), u exp(c_L - c_j) b_s for the state (hi, lo): [channel][token]
    _Float16 st[2][64][NP + 8];   // the entering state (hi, lo): [channel][n]
    float whole[kSsmL], frac[kSsmL];  // c_t in powers of two
    uint32_t mag[4][4][64];       // a channel's largest u, u for the state, state, and its first u but 0, by wave
    float red[4][64];
};

// token by token: the chunk's tokens t0 .. t0 + nt over the state rows of
// every wave, for chunks with non-finite values
template <int NP, bool OUT>
__device__ __noinline__ void ssm_chunk_slow(const ssm_scan_args & a, ssm_lds<NP> & L, ssm_v4f (&st)[NP / 64][4], int s,
                                            int h, int p0, int64_t t0, int nt, float dt, float z) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, gq = lane >> 4;
    const int g = h / (a.heads / a.groups);
    for (int t = 0; t < nt; t++) {
        const float d = __shfl(dt, t), ea = __builtin_amdgcn_exp2f(__shfl(z, t));
        const float * b = (const float *) (a.B + g * a.B_nb1 + (t0 + t) * a.B_nb2 + s * a.B_nb3);
        const float * c = (const float *) (a.C + g * a.C_nb1 + (t0 + t) * a.C_nb2 + s * a.C_nb3);
        const float * x = (const float *) (a.x + h * a.x_nb1 + (t0 + t) * a.x_nb2 + s * a.x_nb3);
#pragma unroll
        for (int pt = 0; pt < 4; pt++) {
            const int p = p0 + 16 * pt + r;
            const float u = p < a.dim ? x[p] * d : 0.0f;
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < NP / 64; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = wave * (NP / 4) + 16 * k + 4 * gq + i;
                    if (n < a.n) {
                        st[k][pt][i] = fmaf(st[k][pt][i], ea, u * b[n]);
                        y = fmaf(st[k][pt][i], c[n], y);
                    }
                }
            if constexpr (OUT) {
                y += __shfl_xor(y, 16);
                y += __shfl_xor(y, 32);
                if (gq == 0) L.red[wave][16 * pt + r] = y;
            }
        }
        if constexpr (OUT) {
            __syncthreads();
            const int p = p0 + (int) threadIdx.x;
            if (threadIdx.x < 64 && p < a.dim)
                a.y[((s * a.tokens + t0 + t) * a.heads + h) * a.dim + p] =
                    (L.red[0][threadIdx.x] + L.red[1][threadIdx.x]) + (L.red[2][threadIdx.x] + L.red[3][threadIdx.x]);
            __syncthreads();
        }
    }
}

template <int NP, bool OUT>
__global__ __launch_bounds__(256, 2) void k_ssm_chunks(ssm_chunk_args q) {
    constexpr int NT = NP / 64;  // 16-row tiles of the state a wave owns
    __shared__ __align__(16) ssm_lds<NP> L;
    const ssm_scan_args & a = q.a;
    const int lane = threadIdx.x & 63, r = lane & 15, gq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int unit = blockIdx.x, seg = blockIdx.y;
    const int pb = unit % q.pblocks, h = unit / q.pblocks % a.heads, s = unit / (q.pblocks * a.heads);
    const int g = h / (a.heads / a.groups), p0 = 64 * pb;
    const int64_t sg = (int64_t) s * a.groups + g, tp = q.chunks * kSsmL;
    const float A = *(const float *) (a.A + h * a.A_nb1);
    const int nbase = wave * (NP / 4);

    // the state: rows n = nbase + 16 k + 4 gq + i, channels p0 + 16 pt + r
    ssm_v4f st[NT][4];
    {
        float carry = 1.0f;
        if constexpr (OUT) {
            double d = 0.0;
            for (int m = 0; m < seg; m++) d += q.seg_decay[((int64_t) s * a.heads + h) * q.segs + m];
            carry = __builtin_amdgcn_exp2f((float) d);
        }
        const int64_t slot = a.ids[s];
        const bool has = OUT && slot >= 0 && slot < a.slots;
        const float * s0 = (const float *) (a.s + (has ? slot : 0) * a.s_nb3) + (int64_t) h * a.dim * a.n;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int pt = 0; pt < 4; pt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = nbase + 16 * k + 4 * gq + i, p = p0 + 16 * pt + r;
                    const bool ok = has && n < a.n && p < a.dim;
                    st[k][pt][i] = ok ? s0[(int64_t) p * a.n + n] * carry : 0.0f;
                }
        if constexpr (OUT) {
            for (int m = 0; m < seg; m++) {
                double d = 0.0;
                for (int e = m + 1; e < seg; e++) d += q.seg_decay[((int64_t) s * a.heads + h) * q.segs + e];
                const float f = __builtin_amdgcn_exp2f((float) d);
                const float * o = q.seg_state + ((int64_t) unit * q.segs + m) * 64 * NP;
#pragma unroll
                for (int k = 0; k < NT; k++)
#pragma unroll
                    for (int pt = 0; pt < 4; pt++) {
                        const float4 v = *(const float4 *) (o + (16 * pt + r) * NP + nbase + 16 * k + 4 * gq);
                        st[k][pt][0] = fmaf(v.x, f, st[k][pt][0]);
                        st[k][pt][1] = fmaf(v.y, f, st[k][pt][1]);
                        st[k][pt][2] = fmaf(v.z, f, st[k][pt][2]);
                        st[k][pt][3] = fmaf(v.w, f, st[k][pt][3]);
                    }
            }
        }
    }
    const int64_t c0 = (int64_t) seg * q.seg_chunks, c1 = min(c0 + q.seg_chunks, q.chunks);
    const int px = p0 + lane;  // the channel this lane stages
    auto load_x = [&](int64_t c, float (&x)[16]) {
        const char * xp = a.x + h * a.x_nb1 + s * a.x_nb3 + 4 * (int64_t) (px < a.dim ? px : 0);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int64_t t = c * kSsmL + 16 * wave + i;
            x[i] = *(const float *) (xp + (t < a.tokens ? t : 0) * a.x_nb2);
        }
    };
    auto load_dt = [&](int64_t c) {
        const int64_t t = c * kSsmL + lane;
        return *(const float *) (a.dt + 4 * h + (t < a.tokens ? t : 0) * a.dt_nb1 + s * a.dt_nb2);
    };
    float xn[16], dtn = 0.0f;
    if (c0 < c1) {
        load_x(c0, xn);
        dtn = load_dt(c0);
    }
    double decayed = 0.0;
    for (int64_t c = c0; c < c1; c++) {
        const int64_t t0 = c * kSsmL;
        const int nt = (int) min((int64_t) kSsmL, a.tokens - t0);
        // the decays: lane t's step, the inclusive sums in f64
        const float dt = lane < nt ? ssm_softplus(dtn) : 0.0f;
        const float z = dt * A * kLog2e;
        double cum = (double) dt * (double) A * 1.4426950408889634074;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(cum, o);
            if (lane >= o) cum += v;
        }
        const double total = __shfl(cum, 63);
        const double whole = floor(cum);
        const float left = __builtin_amdgcn_exp2f((float) (total - cum));
        const float wj = dt * left * q.b_s[sg * tp + t0 + lane];
        float u[16], v[16];
        uint32_t mu = 0, mv = 0, first = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int t = 16 * wave + i;
            const float x = px < a.dim && t < nt ? xn[i] : 0.0f;
            u[i] = x * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dt), t));
            v[i] = x * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wj), t));
            mu = max(mu, ssm_mag(u[i]));
            first = first ? first : mu;
            mv = max(mv, ssm_mag(v[i]));
        }
        uint32_t ms = 0;  // of channel 16 gq + r = lane
#pragma unroll
        for (int pt = 0; pt < 4; pt++) {
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) m = max(m, ssm_mag(st[k][pt][i]));
            m = max(m, (uint32_t) __shfl_xor((int) m, 16));
            m = max(m, (uint32_t) __shfl_xor((int) m, 32));
            ms = gq == pt ? m : ms;
        }
        // (past 2^23 the whole powers are no longer exact in f32)
        const bool odd = !(fabs(total) < 8388608.0);
        L.mag[0][wave][lane] = mu;
        L.mag[1][wave][lane] = mv;
        L.mag[2][wave][lane] = ms;
        L.mag[3][wave][lane] = first;
        if (c + 1 < c1) {
            load_x(c + 1, xn);
            dtn = load_dt(c + 1);
        }
        __syncthreads();  // the magnitudes; every wave is done with the chunk before
        auto largest = [&](int kind) {
            return max(max(L.mag[kind][0][lane], L.mag[kind][1][lane]), max(L.mag[kind][2][lane], L.mag[kind][3][lane]));
        };
        mu = largest(0), mv = largest(1), ms = largest(2);
        first = L.mag[3][0][lane] ? L.mag[3][0][lane] : L.mag[3][1][lane] ? L.mag[3][1][lane] : L.mag[3][2][lane] ? L.mag[3][2][lane] : mu;
        // one step of the exponent is 2^23 in a float's bits
        const bool rising = mu > first && (mu >> 23) - (first >> 23) > 24;
        decayed += total;
        {
            const int4 bad = *(const int4 *) (q.bad + (sg * q.chunks + c) * 4);
            // the same for every wave: they see the same magnitudes
            if (odd || __any(rising || !ssm_finite(mu) || !ssm_finite(mv) || !ssm_finite(ms)) || (bad.x | bad.y | bad.z | bad.w)) {
                ssm_chunk_slow<NP, OUT>(a, L, st, s, h, p0, t0, nt, dt, z);
                __syncthreads();
                continue;
            }
        }
        // lane's channel's exponents, then those of the accumulators' columns
        const int ku = ssm_scale(mu), ks = ssm_scale(ms);
        // (terms under 2^-30 of the state need no bits of their own: keeps
        // the state in their units far from f32's ends)
        const int kv = ms ? min(ssm_scale(mv), ks + 30) : ssm_scale(mv);
        int kup[4], ksp[4], kvp[4];
#pragma unroll
        for (int pt = 0; pt < 4; pt++) {
            kup[pt] = __shfl(ku, 16 * pt + r);
            ksp[pt] = __shfl(ks, 16 * pt + r);
            kvp[pt] = __shfl(kv, 16 * pt + r);
        }
        {
            const float fu = ssm_pow2(ku), fv = ssm_pow2(kv);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                ssm_v8h uh, ul, vh, vl;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = u[8 * half + e] * fu, y = v[8 * half + e] * fv;
                    uh[e] = (_Float16) x;
                    ul[e] = (_Float16) (x - (float) uh[e]);
                    vh[e] = (_Float16) y;
                    vl[e] = (_Float16) (y - (float) vh[e]);
                }
                const int at = 16 * wave + 8 * half;
                if constexpr (OUT) {
                    *(ssm_v8h *) &L.x[0][lane][at] = uh;
                    *(ssm_v8h *) &L.x[1][lane][at] = ul;
                }
                *(ssm_v8h *) &L.x[2][lane][at] = vh;
                *(ssm_v8h *) &L.x[3][lane][at] = vl;
            }
            if constexpr (OUT) {
#pragma unroll
                for (int k = 0; k < NT; k++)
#pragma unroll
                    for (int pt = 0; pt < 4; pt++) {
                        const float fs = ssm_pow2(ksp[pt]);
                        ssm_v4h hi, lo;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float x = st[k][pt][i] * fs;
                            hi[i] = (_Float16) x;
                            lo[i] = (_Float16) (x - (float) hi[i]);
                        }
                        const int n = nbase + 16 * k + 4 * gq;
                        *(ssm_v4h *) &L.st[0][16 * pt + r][n] = hi;
                        *(ssm_v4h *) &L.st[1][16 * pt + r][n] = lo;
                    }
                if (wave == 0) {
                    L.whole[lane] = (float) whole;
                    L.frac[lane] = (float) (cum - whole);
                }
            }
        }
        __syncthreads();
        if constexpr (OUT) {
            const int t = 16 * wave + r;  // the token of this lane's operand rows
            ssm_v4f yh[4], yx[4];
#pragma unroll
            for (int pt = 0; pt < 4; pt++) yh[pt] = yx[pt] = ssm_v4f{0, 0, 0, 0};
            // H C_t
            const _Float16 * ch = q.c_hi + (sg * tp + t0 + t) * NP + 8 * gq;
            const _Float16 * cl = q.c_lo + (sg * tp + t0 + t) * NP + 8 * gq;
#pragma unroll
            for (int kk = 0; kk < NP / 32; kk++) {
                const ssm_v8h ah = *(const ssm_v8h *) (ch + 32 * kk), al = *(const ssm_v8h *) (cl + 32 * kk);
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    const ssm_v8h bh = *(const ssm_v8h *) &L.st[0][16 * pt + r][32 * kk + 8 * gq];
                    const ssm_v8h bl = *(const ssm_v8h *) &L.st[1][16 * pt + r][32 * kk + 8 * gq];
                    yh[pt] = ssm_mfma(ah, bh, yh[pt]);
                    yh[pt] = ssm_mfma(ah, bl, yh[pt]);
                    yh[pt] = ssm_mfma(al, bh, yh[pt]);
                }
            }
            // the chunk's own tokens: the decayed C . B of this lane's row
            const float tw = L.whole[t], tf = L.frac[t];
            const float * cb = q.cb + ((sg * q.chunks + c) * kSsmL + t) * kSsmL + 8 * gq;
            float m[2][8];
            uint32_t mm = 0;
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                if (kk == 1 && wave < 2) continue;
                float gv[8], jw[8], jf[8];
                *(float4 *) &gv[0] = *(const float4 *) (cb + 32 * kk);
                *(float4 *) &gv[4] = *(const float4 *) (cb + 32 * kk + 4);
                *(float4 *) &jw[0] = *(const float4 *) &L.whole[32 * kk + 8 * gq];
                *(float4 *) &jw[4] = *(const float4 *) &L.whole[32 * kk + 8 * gq + 4];
                *(float4 *) &jf[0] = *(const float4 *) &L.frac[32 * kk + 8 * gq];
                *(float4 *) &jf[4] = *(const float4 *) &L.frac[32 * kk + 8 * gq + 4];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float dec = __builtin_amdgcn_exp2f((tw - jw[e]) + (tf - jf[e]));
                    m[kk][e] = 32 * kk + 8 * gq + e <= t ? gv[e] * dec : 0.0f;
                    mm = max(mm, ssm_mag(m[kk][e]));
                }
            }
            mm = max(mm, (uint32_t) __shfl_xor((int) mm, 16));
            mm = max(mm, (uint32_t) __shfl_xor((int) mm, 32));
            const int km = ssm_scale(mm);  // of the lane's row
            const float fm = ssm_pow2(km);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                if (kk == 1 && wave < 2) continue;
                ssm_v8h ah, al;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = m[kk][e] * fm;
                    ah[e] = (_Float16) x;
                    al[e] = (_Float16) (x - (float) ah[e]);
                }
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    const ssm_v8h bh = *(const ssm_v8h *) &L.x[0][16 * pt + r][32 * kk + 8 * gq];
                    const ssm_v8h bl = *(const ssm_v8h *) &L.x[1][16 * pt + r][32 * kk + 8 * gq];
                    yx[pt] = ssm_mfma(ah, bh, yx[pt]);
                    yx[pt] = ssm_mfma(ah, bl, yx[pt]);
                    yx[pt] = ssm_mfma(al, bh, yx[pt]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int tr = 16 * wave + 4 * gq + i;  // the token of the accumulators' row i
                const float fx = ssm_pow2(-__shfl(km, 4 * gq + i));
                const float fh = __builtin_amdgcn_exp2f(L.whole[tr] + L.frac[tr]) * q.c_s[sg * tp + t0 + tr];
                if (tr >= nt) continue;
                float * y = a.y + ((s * a.tokens + t0 + tr) * a.heads + h) * a.dim + p0;
#pragma unroll
                for (int pt = 0; pt < 4; pt++)
                    if (p0 + 16 * pt + r < a.dim)
                        y[16 * pt + r] = fmaf(yh[pt][i], fh * ssm_pow2(-ksp[pt]), yx[pt][i] * (fx * ssm_pow2(-kup[pt])));
            }
        }
        // the state after the chunk, in the staged operand's units meanwhile
        {
            const float fd = __builtin_amdgcn_exp2f((float) total);
            const _Float16 * bh = q.b_hi + ((sg * q.chunks + c) * NP + nbase + r) * kSsmL + 8 * gq;
            const _Float16 * bl = q.b_lo + ((sg * q.chunks + c) * NP + nbase + r) * kSsmL + 8 * gq;
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++) st[k][pt] *= fd * ssm_pow2(kvp[pt]);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                ssm_v8h xh[4], xl[4];
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    xh[pt] = *(const ssm_v8h *) &L.x[2][16 * pt + r][32 * kk + 8 * gq];
                    xl[pt] = *(const ssm_v8h *) &L.x[3][16 * pt + r][32 * kk + 8 * gq];
                }
#pragma unroll
                for (int k = 0; k < NT; k++) {
                    const ssm_v8h ah = *(const ssm_v8h *) (bh + 16 * k * kSsmL + 32 * kk);
                    const ssm_v8h al = *(const ssm_v8h *) (bl + 16 * k * kSsmL + 32 * kk);
#pragma unroll
                    for (int pt = 0; pt < 4; pt++) {
                        st[k][pt] = ssm_mfma(ah, xh[pt], st[k][pt]);
                        st[k][pt] = ssm_mfma(ah, xl[pt], st[k][pt]);
                        st[k][pt] = ssm_mfma(al, xh[pt], st[k][pt]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++) st[k][pt] *= ssm_pow2(-kvp[pt]);
        }
    }
    if constexpr (OUT) {
        if (seg != q.segs - 1) return;
        float * o = a.out + ((int64_t) s * a.heads + h) * a.dim * a.n;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int pt = 0; pt < 4; pt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = nbase + 16 * k + 4 * gq + i, p = p0 + 16 * pt + r;
                    if (n < a.n && p < a.dim) o[(int64_t) p * a.n + n] = st[k][pt][i];
                }
    } else {
        if (pb == 0 && threadIdx.x == 0) q.seg_decay[((int64_t) s * a.heads + h) * q.segs + seg] = decayed;
        float * o = q.seg_state + ((int64_t) unit * q.segs + seg) * 64 * NP;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int pt = 0; pt < 4; pt++)
                *(float4 *) (o + (16 * pt + r) * NP + nbase + 16 * k + 4 * gq) =
                    make_float4(st[k][pt][0], st[k][pt][1], st[k][pt][2], st[k][pt][3]);
    }
}

// ------------------------------------------------------------- launches ---

bool ssm_scan_supported(int64_t n) { return n >= 1 && n <= 256; }

static size_t ssm_al(size_t v) { return (v + 255) / 256 * 256; }

// the chunked form takes a decay a head over enough tokens, channels and
// state elements to fill its tiles
static bool ssm_chunked(const ssm_scan_args & a) { return !a.a_elem && a.tokens >= 16 && a.dim >= 16 && a.n >= 16; }

static int ssm_np(const ssm_scan_args & a) { return a.n <= 64 ? 64 : a.n <= 128 ? 128 : 256; }

// segments of a chunked scan: workgroups for every CU where the heads alone
// are too few, each of four chunks at least
static void ssm_segments(const ssm_scan_args & a, int n_cu, ssm_chunk_args & q) {
    q.a = a;
    q.chunks = (a.tokens + kSsmL - 1) / kSsmL;
    q.pblocks = (a.dim + 63) / 64;
    const int64_t units = (int64_t) a.seqs * a.heads * q.pblocks;
    int64_t segs = (2 * n_cu + units - 1) / units;
    segs = segs < 1 ? 1 : segs;
    const int64_t most = (q.chunks + 3) / 4;
    segs = segs < most ? segs : most;
    q.seg_chunks = (int) ((q.chunks + segs - 1) / segs);
    q.segs = (int) ((q.chunks + q.seg_chunks - 1) / q.seg_chunks);
}

// the scratch's parts, in order; base null: their total size only
static size_t ssm_carve(ssm_chunk_args & q, char * base) {
    const ssm_scan_args & a = q.a;
    const size_t np = (size_t) ssm_np(a), sg = (size_t) a.seqs * a.groups, tp = (size_t) q.chunks * kSsmL;
    size_t at = 0;
    auto take = [&](auto *& p, size_t bytes) {
        p = (typename std::remove_reference<decltype(p)>::type) (base + at);
        at += ssm_al(bytes);
    };
    take(q.c_hi, sg * tp * np * 2);
    take(q.c_lo, sg * tp * np * 2);
    take(q.b_hi, sg * tp * np * 2);
    take(q.b_lo, sg * tp * np * 2);
    take(q.c_s, sg * tp * 4);
    take(q.b_s, sg * tp * 4);
    take(q.cb, sg * tp * kSsmL * 4);
    take(q.bad, sg * (size_t) q.chunks * 16);
    const size_t segs = q.segs > 1 ? (size_t) q.segs : 0;
    take(q.seg_state, (size_t) a.seqs * a.heads * q.pblocks * segs * 64 * np * 4);
    take(q.seg_decay, (size_t) a.seqs * a.heads * segs * 8);
    return at;
}

size_t ssm_scan_scratch_bytes(const ssm_scan_args & a, int n_cu) {
    if (!ssm_chunked(a)) return 0;
    ssm_chunk_args q{};
    ssm_segments(a, n_cu, q);
    return ssm_carve(q, nullptr);
}

static void launch_ssm_chunks(const ssm_scan_args & a, void * scratch, hipStream_t s, int n_cu) {
    ssm_chunk_args q{};
    ssm_segments(a, n_cu, q);
    ssm_carve(q, (char *) scratch);
    auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        const unsigned units = (unsigned) (a.seqs * a.heads * q.pblocks);
        hipLaunchKernelGGL(k_ssm_split<NP>, dim3((unsigned) (4 * q.chunks * a.seqs * a.groups)), dim3(256), 0, s, q);
        if (q.segs > 1)
            hipLaunchKernelGGL((k_ssm_chunks<NP, false>), dim3(units, (unsigned) (q.segs - 1)), dim3(256), 0, s, q);
        hipLaunchKernelGGL((k_ssm_chunks<NP, true>), dim3(units, (unsigned) q.segs), dim3(256), 0, s, q);
    };
    const int np = ssm_np(a);
    if (np == 64) go(std::integral_constant<int, 64>{});
    else if (np == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
}

void launch_ssm_scan(const ssm_scan_args & a, void * scratch, hipStream_t s, int n_cu) {
    const int64_t rows = (int64_t) a.seqs * a.heads * a.dim;
    if (rows == 0) return;
    if (ssm_chunked(a)) return launch_ssm_chunks(a, scratch, s, n_cu);
    auto go = [&](auto kernel, int w) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) ((rows * w + 255) / 256)), dim3(256), 0, s, a);
    };
    if (a.n <= 16) go(k_ssm_scan_rows<16, 1>, 16);
    else if (a.n <= 64) go(k_ssm_scan_rows<64, 1>, 64);
    else if (a.n <= 128) go(k_ssm_scan_rows<64, 2>, 64);
    else go(k_ssm_scan_rows<64, 4>, 64);
}

}  // namespace mi355x
