// k_ssm.hip -- the state-space mixer's operators: GGML_OP_SSM_CONV (the short
// depthwise causal convolution over the carried and the step's columns) and
// GGML_OP_SSM_SCAN (the selective scan).
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

typedef float ssm_v4f __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- conv ---

// y[c, t, s] = silu(bias[c] + sum_j w[j, c] col[t + j, c, s]): every column is
// read once and every result written once, so memory bounds it: 2 x 1777
// tokens of 5376 channels (153 MB) in 31 us, a copy's rate (4.9 TB/s). The
// SILU's exponential is f32's, within an ulp: the elementwise operator's one in
// doubles bounded the launch (48 us).
__device__ __forceinline__ float ssm_conv_end(const ssm_conv_args & a, float v, float bias) {
    if (a.bias) v = v + bias;
    return a.silu ? v / (1.0f + expf(-v)) : v;
}

// Channels adjacent: a lane takes NC channels and a run of tokens, the window
// of TAPS - 1 columns in registers, U columns' loads ahead of their products.
// (Runs of 16 tokens with 4 ahead: 31 us; 32 with 8, twice the registers and
// half the waves, 40; 8 with 4, more columns read twice, 32.)
// The lane with a channel's first token alone reads its carried columns, so it
// may write the ones carried on over them.
// PACKED (NC 4): four channels' taps and carried columns come in whole 16-byte
// pieces (one token of 32 streams: 5.3 us, element by element 7.3).
template <int TAPS, int NC, int U, bool PACKED>
__global__ __launch_bounds__(256) void k_ssm_conv_rows(ssm_conv_args a, int run) {
    const int lane = threadIdx.x & 63;
    const int64_t cgroups = (a.channels + 64 * NC - 1) / (64 * NC), runs = (a.tokens + run - 1) / run;
    const int64_t units = cgroups * runs * a.seqs;
    for (int64_t u = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t) gridDim.x * 4) {
        const int64_t c = (u % cgroups * 64 + lane) * NC, s = u / (cgroups * runs);
        const int64_t t0 = u / cgroups % runs * run, t1 = min(t0 + run, a.tokens);
        if (c >= a.channels) continue;
        typedef float vec __attribute__((ext_vector_type(NC)));
        float w[TAPS][NC], bias[NC];
        if constexpr (PACKED) {
            ssm_v4f v[TAPS];
#pragma unroll
            for (int j = 0; j < TAPS; j++) v[j] = ((const ssm_v4f *) (a.w + c * a.w_nb1))[j];
#pragma unroll
            for (int i = 0; i < NC * TAPS; i++) w[i % TAPS][i / TAPS] = v[i / 4][i % 4];
        } else {
#pragma unroll
            for (int e = 0; e < NC; e++)
#pragma unroll
                for (int j = 0; j < TAPS; j++) w[j][e] = ((const float *) (a.w + (c + e) * a.w_nb1))[j];
        }
#pragma unroll
        for (int e = 0; e < NC; e++) bias[e] = a.bias ? a.bias[c + e] : 0.0f;
        const char * x = a.x + c * a.x_nb1 + s * a.x_nb2;
        const char * st = a.st + c * a.st_nb1 + s * a.st_nb2;
        auto column = [&](int64_t i) {  // of x
            vec v;
            if constexpr (NC == 1) v[0] = *(const float *) (x + i * a.x_nb0);
            else v = *(const vec *) (x + i * a.x_nb0);
            return v;
        };
        vec win[TAPS - 1];
        const bool packed = PACKED && a.lead > 0 && t0 == 0;
        if (packed) {
            ssm_v4f v[TAPS - 1];
#pragma unroll
            for (int j = 0; j < TAPS - 1; j++) v[j] = ((const ssm_v4f *) st)[j];
#pragma unroll
            for (int i = 0; i < NC * (TAPS - 1); i++) win[i % (TAPS - 1)][i / (TAPS - 1)] = v[i / 4][i % 4];
        }
#pragma unroll
        for (int j = 0; j < TAPS - 1; j++) {
            const int64_t i = t0 + j;
            if (packed) continue;
            if (i < a.lead) {
#pragma unroll
                for (int e = 0; e < NC; e++) win[j][e] = *(const float *) (st + e * a.st_nb1 + i * a.st_nb0);
            } else win[j] = column(i - a.lead);
        }
        const int64_t in = TAPS - 1 - a.lead;  // token t's newest column is x's t + in
        if (a.carry && t0 == 0) {
            vec on[TAPS - 1];
#pragma unroll
            for (int j = 0; j < TAPS - 1; j++) {
                const int64_t i = a.tokens + j - (TAPS - 1);
                if (i >= 0) on[j] = column(i);
                else
#pragma unroll
                    for (int k = 1; k < TAPS - 1; k++)
                        if (a.tokens + j == k) on[j] = win[k];
            }
            if constexpr (PACKED) {
                ssm_v4f v[TAPS - 1];
#pragma unroll
                for (int i = 0; i < NC * (TAPS - 1); i++) v[i / 4][i % 4] = on[i % (TAPS - 1)][i / (TAPS - 1)];
#pragma unroll
                for (int j = 0; j < TAPS - 1; j++) ((ssm_v4f *) (a.carry + c * a.c_nb1 + s * a.c_nb2))[j] = v[j];
            } else {
#pragma unroll
                for (int j = 0; j < TAPS - 1; j++)
#pragma unroll
                    for (int e = 0; e < NC; e++)
                        *(float *) (a.carry + (c + e) * a.c_nb1 + j * a.c_nb0 + s * a.c_nb2) = on[j][e];
            }
        }
        float * out = a.out + (s * a.tokens) * a.channels + c;
        vec next[U];
#pragma unroll
        for (int k = 0; k < U; k++) next[k] = column(min(t0 + k, t1 - 1) + in);
        for (int64_t t = t0; t < t1; t += U) {
            vec cur[U];
#pragma unroll
            for (int k = 0; k < U; k++) cur[k] = next[k];
            if (U > 1 && t + U < t1) {
#pragma unroll
                for (int k = 0; k < U; k++) next[k] = column(min(t + U + k, t1 - 1) + in);
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (U > 1 && t + k >= t1) break;
                vec y;
#pragma unroll
                for (int e = 0; e < NC; e++) {
                    float v = 0.0f;
#pragma unroll
                    for (int j = 0; j < TAPS - 1; j++) v = fmaf(w[j][e], win[j][e], v);
                    y[e] = ssm_conv_end(a, fmaf(w[TAPS - 1][e], cur[k][e], v), bias[e]);
                }
#pragma unroll
                for (int j = 0; j < TAPS - 2; j++) win[j] = win[j + 1];
                win[TAPS - 2] = cur[k];
                if constexpr (NC == 1) out[(t + k) * a.channels] = y[0];
                else *(vec *) (out + (t + k) * a.channels) = y;
            }
            if (U == 1 && t + 1 < t1) next[0] = column(t + 1 + in);
        }
    }
}

// Columns adjacent, one tensor: 64 channels' columns of 64 tokens through LDS,
// read along the columns and written along the channels, whole lines both
constexpr int kConvTaps = 33;  // the most of this form
__global__ __launch_bounds__(256) void k_ssm_conv_cols(ssm_conv_args a) {
    __shared__ float tile[64][64 + kConvTaps];  // (odd rows: a column's reads on distinct banks)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t cgroups = (a.channels + 63) / 64, tgroups = (a.tokens + 63) / 64, n = cgroups * tgroups * a.seqs;
    for (int64_t u = blockIdx.x; u < n; u += gridDim.x) {
        const int64_t t0 = u % tgroups * 64, c0 = u / tgroups % cgroups * 64, s = u / (tgroups * cgroups);
        const int cols = (int) min((int64_t) 64, a.tokens - t0) + a.taps - 1;
        for (int r = wave; r < 64; r += 4) {
            const char * row = a.x + min(c0 + r, a.channels - 1) * a.x_nb1 + s * a.x_nb2 + t0 * a.x_nb0;
            for (int i = lane; i < cols; i += 64) tile[r][i] = *(const float *) (row + i * a.x_nb0);
        }
        __syncthreads();
        const int64_t c = c0 + lane;
        if (c < a.channels) {
            const float * w = (const float *) (a.w + c * a.w_nb1);
            const float bias = a.bias ? a.bias[c] : 0.0f;
            const int t1 = cols - (a.taps - 1);
            for (int t = 16 * wave; t < min(16 * wave + 16, t1); t++) {
                float v = 0.0f;
                for (int j = 0; j < a.taps; j++) v = fmaf(w[j], tile[lane][t + j], v);
                a.out[(s * a.tokens + t0 + t) * a.channels + c] = ssm_conv_end(a, v, bias);
            }
        }
        __syncthreads();  // the tile is read
    }
}

// any taps and strides
__global__ __launch_bounds__(256) void k_ssm_conv_any(ssm_conv_args a) {
    const int64_t n = a.channels * a.tokens * a.seqs;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) {
        const int64_t c = i % a.channels, t = i / a.channels % a.tokens, s = i / (a.channels * a.tokens);
        const char * row = a.x + c * a.x_nb1 + s * a.x_nb2;
        const float * w = (const float *) (a.w + c * a.w_nb1);
        float y = 0.0f;
        for (int j = 0; j < a.taps; j++) y = fmaf(w[j], *(const float *) (row + (t + j) * a.x_nb0), y);
        a.out[i] = ssm_conv_end(a, y, a.bias ? a.bias[c] : 0.0f);
    }
}

bool ssm_conv_rows(const ssm_conv_args & a) { return a.taps >= 2 && a.taps <= 4 && (a.x_nb1 == 4 || a.tokens == 1); }

template <int TAPS>
static void launch_conv_rows(const ssm_conv_args & a, hipStream_t s) {
    const bool vec = a.channels % 4 == 0 && a.x_nb1 == 4 && a.x_nb0 % 16 == 0 && a.x_nb2 % 16 == 0 &&
                     (((uintptr_t) a.x | (uintptr_t) a.out) & 15) == 0;
    const int nc = vec ? 4 : 1, run = 16;
    const int64_t units = (a.channels + 64 * nc - 1) / (64 * nc) * ((a.tokens + run - 1) / run) * a.seqs;
    const dim3 grid((unsigned) std::min<int64_t>((units + 3) / 4, 1 << 22));
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, s, a, run); };
    auto pieces = [](const char * p, int64_t nb0, int64_t nb1, int64_t nb2, int n) {  // rows of n, one after another
        return p == nullptr || (nb0 == 4 && nb1 == 4 * n && nb2 % 16 == 0 && (uintptr_t) p % 16 == 0);
    };
    const bool packed = vec && pieces(a.w, 4, a.w_nb1, 0, TAPS) && pieces(a.st, a.st_nb0, a.st_nb1, a.st_nb2, TAPS - 1) &&
                        pieces(a.carry, a.c_nb0, a.c_nb1, a.c_nb2, TAPS - 1);
    if (a.tokens < 4) packed ? go(k_ssm_conv_rows<TAPS, 4, 1, true>) : vec ? go(k_ssm_conv_rows<TAPS, 4, 1, false>) : go(k_ssm_conv_rows<TAPS, 1, 1, false>);
    else packed ? go(k_ssm_conv_rows<TAPS, 4, 4, true>) : vec ? go(k_ssm_conv_rows<TAPS, 4, 4, false>) : go(k_ssm_conv_rows<TAPS, 1, 4, false>);
}

void launch_ssm_conv(const ssm_conv_args & a, hipStream_t s) {
    const int64_t n = a.channels * a.tokens * a.seqs;
    if (n == 0) return;
    if (ssm_conv_rows(a)) {
        if (a.taps == 2) launch_conv_rows<2>(a, s);
        else if (a.taps == 3) launch_conv_rows<3>(a, s);
        else launch_conv_rows<4>(a, s);
    } else if (a.x_nb0 == 4 && a.taps <= kConvTaps) {
        const int64_t tiles = (a.channels + 63) / 64 * ((a.tokens + 63) / 64) * a.seqs;
        hipLaunchKernelGGL(k_ssm_conv_cols, dim3((unsigned) std::min<int64_t>(tiles, 1 << 22)), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_ssm_conv_any, dim3((unsigned) std::min<int64_t>((n + 255) / 256, 1 << 22)), dim3(256), 0, s, a);
    }
}

// ---------------------------------------------------------------- scan ---

// softplus as the op defines it, the identity past 20: max(v, 0) + log(1 + z),
// z = exp(-|v|), and log(1 + z) = 2 atanh(s), s = z / (2 + z) <= 1/3, by its
// series. Within 3.7 half steps of the value (the past-20 cut included: there
// z is less than v's last place); log1pf(expf(v)) takes three times the
// instructions.
__device__ __forceinline__ float ssm_softplus(float v) {
    const float z = expf(-fabsf(v)), d = 2.0f + z, r = __builtin_amdgcn_rcpf(d);
    float s = z * r;
    s = fmaf(fmaf(-s, d, z), r, s);
    const float w = s * s;
    float p = 1.0f / 15;
    p = fmaf(p, w, 1.0f / 13);
    p = fmaf(p, w, 1.0f / 11);
    p = fmaf(p, w, 1.0f / 9);
    p = fmaf(p, w, 1.0f / 7);
    p = fmaf(p, w, 1.0f / 5);
    p = fmaf(p, w, 1.0f / 3);
    const float t = s + s;
    return fmaxf(v, 0.0f) + fmaf(t, p * w, t);
}

// token by token: a wave holds one (sequence, head, channel) row's state, R
// elements a lane (any n and alignment)
template <int R>
__global__ __launch_bounds__(256) void k_ssm_scan_rows(ssm_scan_args a) {
    const int lane = threadIdx.x & 63;
    const int64_t rows = (int64_t) a.seqs * a.heads * a.dim;
    for (int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t) gridDim.x * 4) {
        const int p = (int) (row % a.dim), h = (int) (row / a.dim % a.heads), s = (int) (row / ((int64_t) a.dim * a.heads));
        const int g = h / (a.heads / a.groups);
        const int64_t slot = a.ids[s];
        const bool has = slot >= 0 && slot < a.slots;
        const float * s0 = (const float *) (a.s + (has ? slot : 0) * a.s_nb3) + ((int64_t) h * a.dim + p) * a.n;
        float st[R], av[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int k = lane + 64 * r;
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
                const int k = lane + 64 * r;
                const bool ok = k < a.n;
                st[r] = ok ? fmaf(st[r], expf(dt * av[r]), xv * b[k]) : 0.0f;  // (past n nothing, an infinite step neither)
                y = fmaf(st[r], ok ? c[k] : 0.0f, y);
            }
            y = wave_sum(y);
            if (lane == 0) a.y[((s * a.tokens + t) * a.heads + h) * a.dim + p] = y;
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int k = lane + 64 * r;
            if (k < a.n) a.out[row * a.n + k] = st[r];
        }
    }
}

// The same with 16-byte pieces: W lanes hold a row's state, four elements a
// lane, and a wave 64 U / W rows of one head at once. One token reads and
// writes every state once, which bounds it: all rows' loads are in flight
// together, beside the token's operands (48 sequences of 80 x 64 x 128 states,
// 252 MB: 46 us, 5.5 TB/s; an element a lane, 145 us).
template <int W, int U>
__global__ __launch_bounds__(256) void k_ssm_scan_pieces(ssm_scan_args a) {
    constexpr int kRows = 64 / W;  // of one load
    const int lane = threadIdx.x & 63, sub = lane / W, k = lane % W * 4;
    const uint32_t pblocks = (uint32_t) ((a.dim + kRows * U - 1) / (kRows * U));
    const int64_t unit = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= (int64_t) pblocks * a.heads * a.seqs) return;
    const int p0 = (int) (unit % pblocks) * kRows * U + sub, h = (int) (unit / pblocks % a.heads);
    const int s = (int) (unit / ((int64_t) pblocks * a.heads)), g = h / (a.heads / a.groups);
    const bool in = k < a.n;
    const int kc = in ? k : 0;
    const int64_t slot = a.ids[s];
    const bool has = slot >= 0 && slot < a.slots;
    const int64_t row0 = (int64_t) h * a.dim;
    const float * s0 = (const float *) (a.s + (has ? slot : 0) * a.s_nb3) + kc;
    struct token {
        float dt, x[U];
        ssm_v4f b, c;
    };
    auto load = [&](int64_t t, token & v) {
        v.dt = *(const float *) (a.dt + 4 * h + t * a.dt_nb1 + s * a.dt_nb2);
        v.b = *(const ssm_v4f *) (a.B + 4 * kc + g * a.B_nb1 + t * a.B_nb2 + s * a.B_nb3);
        v.c = *(const ssm_v4f *) (a.C + 4 * kc + g * a.C_nb1 + t * a.C_nb2 + s * a.C_nb3);
        const char * x = a.x + h * a.x_nb1 + t * a.x_nb2 + s * a.x_nb3;
#pragma unroll
        for (int u = 0; u < U; u++) v.x[u] = *(const float *) (x + 4 * min(p0 + kRows * u, a.dim - 1));
    };
    ssm_v4f st[U];
    if (a.slots > 0) {
#pragma unroll
        for (int u = 0; u < U; u++) st[u] = *(const ssm_v4f *) (s0 + (row0 + min(p0 + kRows * u, a.dim - 1)) * a.n);
    }
    float av[4];
#pragma unroll
    for (int e = 0; e < 4; e++) av[e] = *(const float *) (a.A + h * a.A_nb1 + (a.a_elem ? 4 * (kc + e) : 0));
    token next;
    if (a.tokens > 0) load(0, next);
#pragma unroll
    for (int u = 0; u < U; u++)
        if (!has) st[u] = ssm_v4f{0, 0, 0, 0};
    for (int64_t t = 0; t < a.tokens; t++) {
        token v = next;
        if (t + 1 < a.tokens) load(t + 1, next);
        const float dt = ssm_softplus(v.dt);
        float d[4];
        d[0] = expf(dt * av[0]);
#pragma unroll
        for (int e = 1; e < 4; e++) d[e] = a.a_elem ? expf(dt * av[e]) : d[0];
        float y[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float xv = v.x[u] * dt;
            y[u] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                st[u][e] = fmaf(st[u][e], d[e], xv * v.b[e]);
                y[u] = fmaf(st[u][e], v.c[e], y[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            y[u] = group_sum<W>(in ? y[u] : 0.0f);  // (past n the state's first elements again)
            if (k == 0 && p0 + kRows * u < a.dim) a.y[(s * a.tokens + t) * a.heads * a.dim + row0 + p0 + kRows * u] = y[u];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (in && p0 + kRows * u < a.dim)
            *(ssm_v4f *) (a.out + ((int64_t) s * a.heads * a.dim + row0 + p0 + kRows * u) * a.n + k) = st[u];
}

// Short states (n <= 16): a lane a row, its state in registers, B and C of the
// wave's group in scalar registers, no sums across lanes. An exponential a
// state and token bounds it, so the tokens are cut into segments until there
// are waves enough: the first pass (OUT false) makes each segment's own state
// from zeros and its sum of steps D, and the second starts from the earlier
// segments' states, each decayed by exp(A D) as a whole. (5120 channels of 16,
// 1000 tokens: 32 + 49 us, of which the 82 M exponentials of a pass are 8 and
// its other instructions 20; a row's 16 states on 16 lanes, unsegmented, 1040.)
struct ssm_lane_args {
    ssm_scan_args a;
    float * part;  // [segment][n states, D][row of (sequence, head, channel)]
    int segs;
    int64_t seg_tokens, blocks;  // blocks: of 64 rows, a group
};
constexpr int kSsmLane = 16;

template <bool FULL, bool OUT>
__global__ __launch_bounds__(256) void k_ssm_scan_lanes(ssm_lane_args q) {
    const ssm_scan_args & a = q.a;
    constexpr int N = kSsmLane;
    constexpr float kLog2 = 1.44269504088896340736f;
    typedef const __attribute__((address_space(4))) float * scalar_ptr;  // read-only here: scalar loads
    const int lane = threadIdx.x & 63, n = FULL ? N : a.n;
    const int64_t w = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t units = q.blocks * a.groups * a.seqs;
    const int seg = (int) (w / units);
    if (seg >= q.segs - (OUT ? 0 : 1)) return;
    const int64_t unit = w % units;
    const int g = (int) (unit / q.blocks % a.groups), s = (int) (unit / (q.blocks * a.groups));
    const int64_t per = (int64_t) a.heads / a.groups * a.dim, in = unit % q.blocks * 64 + lane;
    const bool mine = in < per;
    const int64_t row = g * per + (mine ? in : per - 1), all = (int64_t) a.seqs * a.heads * a.dim, at = s * per * a.groups + row;
    const int64_t h = row / a.dim, p = row % a.dim;
    float A[N], st[N], low = 0.0f, high = 0.0f;  // A log2(e); the least and the largest of them
#pragma unroll
    for (int k = 0; k < N; k++) {
        A[k] = FULL || k < n ? kLog2 * *(const float *) (a.A + h * a.A_nb1 + (a.a_elem ? 4 * k : 0)) : 0.0f;
        low = fminf(low, A[k]);
        high = fmaxf(high, A[k]);
        st[k] = 0.0f;
    }
    if constexpr (OUT) {
        const int64_t slot = a.ids[s];
        if (slot >= 0 && slot < a.slots) {
            const float * s0 = (const float *) (a.s + slot * a.s_nb3) + row * n;
#pragma unroll
            for (int k = 0; k < N; k++)
                if (FULL || k < n) st[k] = s0[k];
        }
        float own[N], D = 0.0f;  // the next segment's own state, a step ahead
        auto fetch = [&](int j) {
            const float * part = q.part + (int64_t) j * (n + 1) * all + at;
#pragma unroll
            for (int k = 0; k < N; k++)
                if (FULL || k < n) own[k] = part[k * all];
            D = part[n * all];
        };
        if (seg > 0) fetch(0);
        for (int j = 0; j < seg; j++) {
            float add[N];
            const float d = D;
#pragma unroll
            for (int k = 0; k < N; k++) add[k] = FULL || k < n ? own[k] : 0.0f;
            fetch(min(j + 1, seg - 1));
            if (__all(d * low >= -126.0f && d * high <= 0.0f)) {
#pragma unroll
                for (int k = 0; k < N; k++) st[k] = fmaf(st[k], __builtin_amdgcn_exp2f(A[k] * d), add[k]);
            } else {  // 2^z in two parts: neither over- nor underflows before the product does
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const float z = fminf(fmaxf(A[k] * d, -1000.0f), 1000.0f), zi = rintf(z);
                    st[k] = ldexpf(st[k] * exp2f(z - zi), (int) zi) + add[k];
                }
            }
        }
    }
    const int64_t t0 = seg * q.seg_tokens, t1 = min(t0 + q.seg_tokens, a.tokens);
    const char * dtp = a.dt + 4 * h + s * a.dt_nb2;
    const char * xp = a.x + 4 * p + h * a.x_nb1 + s * a.x_nb3;
    const char *bp = a.B + g * a.B_nb1 + s * a.B_nb3, *cp = a.C + g * a.C_nb1 + s * a.C_nb3;
    constexpr int U = 4;  // tokens whose dt and x are loaded ahead
    float dtn[U], xn[U];
    auto load = [&](int64_t t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t i = min(t + u, t1 - 1);
            dtn[u] = *(const float *) (dtp + i * a.dt_nb1);
            xn[u] = *(const float *) (xp + i * a.x_nb2);
        }
    };
    // a token's B and C: a step ahead where they are whole
    float B[N], C[N], Bn[N], Cn[N];
    auto fetch = [&](int64_t t) {
        const scalar_ptr b = (scalar_ptr) (uintptr_t) (bp + t * a.B_nb2), c = (scalar_ptr) (uintptr_t) (cp + t * a.C_nb2);
#pragma unroll
        for (int k = 0; k < N; k++) {
            if (!FULL && k >= n) break;
            Bn[k] = b[k];
            if constexpr (OUT) Cn[k] = c[k];
        }
    };
    double D = 0.0;
    if (t0 < t1) {
        load(t0);
        fetch(t0);
    }
    for (int64_t t = t0; t < t1; t += U) {
        float dts[U], xs[U];
#pragma unroll
        for (int u = 0; u < U; u++) dts[u] = ssm_softplus(dtn[u]), xs[u] = xn[u] * dts[u];
        if (t + U < t1) load(t + U);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u >= t1) break;
            const float dt = dts[u], xv = xs[u];
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (!FULL && k >= n) break;
                B[k] = Bn[k];
                if constexpr (OUT) C[k] = Cn[k];
            }
            fetch(min(t + u + 1, t1 - 1));
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!OUT) D += (double) dt;
            float e[N], y = 0.0f;
#pragma unroll
            for (int k = 0; k < N; k++) e[k] = __builtin_amdgcn_exp2f(dt * A[k]);
            if (__any(dt * low < -126.0f || dt * high > 127.0f)) {  // at the ends of the instruction's range
#pragma unroll
                for (int k = 0; k < N; k++) {
                    e[k] = exp2f(dt * A[k]);
                    // (a segment's own zero is none of the state's: it has no growth to be spoilt by)
                    if (!OUT && st[k] == 0.0f) e[k] = 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (!FULL && k >= n) break;
                st[k] = fmaf(st[k], e[k], xv * B[k]);
                if constexpr (OUT) y = fmaf(st[k], C[k], y);
            }
            if constexpr (OUT)
                if (mine) a.y[(s * a.tokens + t + u) * a.heads * a.dim + row] = y;
        }
    }
    if (!mine) return;
    if constexpr (!OUT) {
        float * part = q.part + (int64_t) seg * (n + 1) * all + at;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (FULL || k < n) part[k * all] = st[k];
        part[n * all] = (float) D;
    } else if (seg == q.segs - 1) {
        float * o = a.out + at * n;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (FULL || k < n) o[k] = st[k];
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
// Products of f32 operands on the bf16 matrix cores: an operand is the sum of
// three bf16 (8 bits each: all 24 of an f32, in its range of exponents), and a
// product the six of theirs that f32 can hold (what is left out is 2^-26 of it
// and less), summed in f32. So an element keeps its bits however far it lies
// under its neighbours, over tokens and over n alike, and the error is that of
// f32 sums. The f32 matrix instructions need no parts, but take the vector
// unit's time at 1/16 of the rate (a vector instruction beside one takes its
// own again): 2 x 2048 tokens of 80 heads of 64 x 128 took 151 us, and 68 for
// the first pass, where these take 104 and 46 (and 11 for the shared operands;
// 333 tokens of 24 x 64 x 64: 12 + 7 + 5 us). Bound by reads of LDS (114 KB a
// wave and chunk, 8 waves), the issue of loads after each barrier, and the
// vector instructions around the products (some 800 a wave and chunk).
//
// The log decays are f64 until they are split into whole and fractional powers
// of two; where they are deep, an operand takes its whole power by ldexp, so
// that it underflows only where the product does.
//
// k_ssm_split makes the operands that a group's heads share (the parts of C and
// B, and C_t . B_j) and the heads' decays, in the matrix instructions' order:
// 64 lanes' 16 bytes one after another. A workgroup of k_ssm_chunks takes two
// blocks of (head, 64 channels) of a group, four waves each, and a segment of
// chunks; only the shared operands and the decayed C . B go through LDS. Wave w
// of a block keeps the state of its channels 16 w .. in its accumulators, which
// are the products' operands as they lie: lane (g, r) holds n = 4 g .. 4 g + 3
// of channel r, and K runs in that order for both sides (32 of K: the 4 g .. of
// two blocks of 16). Where there are few heads the sequence is cut into
// segments: the first pass (OUT false) makes each segment's own state from
// zeros, and the second starts from the earlier segments' states, decayed and
// added.
//
// Non-finite values would spread inside a chunk (0 * inf), and the products'
// order could take large ones out of f32's range where the recurrence does not:
// such a wave's chunk, and one whose decays leave the exact range, runs token
// by token (ssm_tokens), where a value reaches what the recurrence takes it to.

typedef uint32_t ssm_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t ssm_u4 __attribute__((ext_vector_type(4)));
typedef int ssm_i4 __attribute__((ext_vector_type(4)));
typedef float ssm_v2f __attribute__((ext_vector_type(2)));
typedef __bf16 ssm_v2b __attribute__((ext_vector_type(2)));
typedef __bf16 ssm_v8b __attribute__((ext_vector_type(8)));

// (what the launch before wrote and all lanes read alike: scalar loads)
#define SSM_UNIFORM const __attribute__((address_space(4)))

constexpr int kSsmL = 64;

// two f32 as the sums of three bf16 each, rounded to nearest
__device__ __forceinline__ void ssm_parts2(float a, float b, uint32_t & h, uint32_t & m, uint32_t & l) {
    auto pack = [](float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(ssm_v2f{x, y}, ssm_v2b)); };
    auto less = [](float & x, float & y, uint32_t p) {
        x -= __uint_as_float(p << 16);
        y -= __uint_as_float(p & 0xFFFF0000u);
    };
    h = pack(a, b);
    less(a, b, h);
    m = pack(a, b);
    less(a, b, m);
    l = pack(a, b);
}
struct ssm_parts {  // a lane's eight elements of K
    ssm_u4 v[3];
};
__device__ __forceinline__ void ssm_parts8(ssm_v4f a, ssm_v4f b, ssm_parts & p) {
    uint32_t h[4], m[4], l[4];
    ssm_parts2(a[0], a[1], h[0], m[0], l[0]);
    ssm_parts2(a[2], a[3], h[1], m[1], l[1]);
    ssm_parts2(b[0], b[1], h[2], m[2], l[2]);
    ssm_parts2(b[2], b[3], h[3], m[3], l[3]);
    p.v[0] = ssm_u4{h[0], h[1], h[2], h[3]};
    p.v[1] = ssm_u4{m[0], m[1], m[2], m[3]};
    p.v[2] = ssm_u4{l[0], l[1], l[2], l[3]};
}
__device__ __forceinline__ ssm_v4f ssm_mfma(ssm_u4 a, ssm_u4 b, ssm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ssm_v8b, a), __builtin_bit_cast(ssm_v8b, b), c, 0, 0, 0);
}
// the i-th of a product's six, the small ones first
__device__ __forceinline__ ssm_v4f ssm_product(int i, const ssm_parts & a, const ssm_parts & b, ssm_v4f c) {
    constexpr int of_a[6] = {2, 0, 1, 1, 0, 0}, of_b[6] = {0, 2, 1, 0, 1, 0};
    return ssm_mfma(a.v[of_a[i]], b.v[of_b[i]], c);
}
// an element at a uniform base and a lane's byte offset
template <typename T>
__device__ __forceinline__ T & ssm_at(const void * base, uint32_t off) {
    return *(T *) ((char *) base + off);
}
// The matrix form's operands are at most 2^30 (u, B and C). A chunk then adds at
// most 2^66 to a state, so one that begins under 2^80 is under 2^87 after 2^20
// chunks, its product with a row of C under 2^125.
constexpr uint32_t kSsmLargest = (127u + 30) << 23, kSsmLargestState = (127u + 80) << 23;
constexpr int64_t kSsmMostTokens = (int64_t) kSsmL << 20;
// whether one of the values is larger, infinite or NaN: the largest of their bits
// as signed numbers (among the positive ones), and as unsigned (the negative)
struct ssm_most {
    int pos = 0;
    uint32_t neg = 0;
    __device__ __forceinline__ void add(float a, float b) {
        pos = max(max(pos, __float_as_int(a)), __float_as_int(b));
        neg = max(max(neg, __float_as_uint(a)), __float_as_uint(b));
    }
    __device__ __forceinline__ bool past(uint32_t limit) const { return pos > (int) limit || neg > (limit | 0x80000000u); }
};
// a power of two of any size: v times the fraction's power, then the whole one
__device__ __forceinline__ float ssm_decayed(float v, float frac_pow2, float whole) { return ldexpf(v * frac_pow2, (int) whole); }
struct ssm_power {
    float frac, whole;
};
__device__ __forceinline__ ssm_power ssm_split_power(double z) {
    const double whole = floor(fmin(fmax(z, -100000.0), 100000.0));
    return {__builtin_amdgcn_exp2f((float) fmin(fmax(z - whole, 0.0), 1.0)), (float) whole};
}

// what a chunk's decays need besides the tokens' own
struct ssm_decay {
    double total;  // its log2 decay
    int kind;      // kSsmOdd: outside what the matrix form takes; kSsmDeep: powers that f32 may not hold
    int pad;
};
constexpr int kSsmOdd = 1, kSsmDeep = 2;

// The operands in scratch: a record a (sequence, group, chunk) and one a
// (sequence, head, chunk), byte offsets of their arrays, NP the padded state
// size. A fragment is 64 lanes' 16 bytes, lane (g, r).
template <int NP>
struct ssm_shared_at {
    static constexpr int KB = NP / 32, NK = NP / 16;
    static constexpr int c = 0;                     // [4 tb][KB][part] bf16: token 16 tb + r, n 4 g .. of two blocks of 16
    static constexpr int b = 12 * KB * 1024;        // [2 jb][NK][part] bf16: n r of 16, tokens 4 g .. of two blocks of 16
    static constexpr int cb = b + 6 * NK * 1024;    // blocks (tb, jb) f32: token t r of 16, tokens j 4 g .. (zeros past t)
    static constexpr int bad = cb + 12 * 1024;      // [4] bytes: a quarter's rows hold a value past 2^30
    static constexpr int size = bad + 256;
};
// The blocks of C . B in turn: two for the first tokens' 16 and the second's,
// four for the others' (pairs of blocks make a fragment)
__device__ __forceinline__ int ssm_block(int tb, int jb) { return (tb < 2 ? 2 * tb : 4 * tb - 4) + jb; }
struct ssm_head_at {  // c_t: the sum of the log2 decays from the chunk's start to token t
    static constexpr int dt = 0;          // [64] f32: the step
    static constexpr int left = 256;      // [64] f32: 2^(c_L - c_t), deep: of its fraction
    static constexpr int left_whole = 512;  // [64] i32: deep: its whole part (else 0)
    static constexpr int in = 768;        // [64] f32: 2^c_t, deep: of its fraction
    static constexpr int whole = 1024;    // c_t's whole part
    static constexpr int frac = 1280;     // c_t's fractional part
    static constexpr int decay = 1536;    // ssm_decay
    static constexpr int size = 1792;
    static constexpr int tokens = 6;      // arrays of 64
};
struct ssm_chunk_args {
    ssm_scan_args a;
    char *shared, *heads;
    float * seg_state;   // [seq, head, channel block][segment][wave][NP / 16 fragments]
    double * seg_decay;  // [seq, head][segment]: its log2 decay
    int64_t chunks;
    int segs, seg_chunks, pblocks;
    int pairs;             // workgroups a group: of two (head, channel block)s
    uint32_t split_blocks;
    int xvec, yvec, svec;  // x, y and the states in 16-byte pieces
};

// the decays of one (sequence, head, chunk): a lane a token, the sums in f64
__device__ __forceinline__ void ssm_decays(const ssm_chunk_args & q, int64_t unit) {
    const ssm_scan_args & a = q.a;
    const int lane = threadIdx.x & 63;
    const int64_t c = unit % q.chunks, sh = unit / q.chunks;
    if (sh >= (int64_t) a.seqs * a.heads) return;
    const int h = (int) (sh % a.heads), s = (int) (sh / a.heads);
    const int64_t t = c * kSsmL + lane;
    char * rec = q.heads + unit * ssm_head_at::size;
    const float A = *(const float *) (a.A + h * a.A_nb1);
    const float dt = t < a.tokens ? ssm_softplus(*(const float *) (a.dt + 4 * h + t * a.dt_nb1 + s * a.dt_nb2)) : 0.0f;
    double cum = (double) dt * (double) A * 1.4426950408889634074;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double v = __shfl_up(cum, o);
        if (lane >= o) cum += v;
    }
    const double total = __shfl(cum, 63);
    ssm_decay d{};
    d.total = total;
    // A positive, decays whose whole parts leave f32's exact range, steps that are not finite
    const bool odd = !(total <= 0.0 && total > -8388608.0) || __any((__float_as_uint(dt) & 0x7FFFFFFFu) >= 0x7F800000u);
    const bool deep = total < -120.0;  // else every power is one factor
    d.kind = (odd ? kSsmOdd : 0) | (deep ? kSsmDeep : 0);
    const ssm_power left = ssm_split_power(total - cum), in = ssm_split_power(cum);
    auto put = [&](int at, float v) { ((float *) (rec + at))[lane] = v; };
    put(ssm_head_at::dt, dt);
    put(ssm_head_at::left, deep ? left.frac : ssm_decayed(1.0f, left.frac, left.whole));
    ((int *) (rec + ssm_head_at::left_whole))[lane] = deep ? (int) left.whole : 0;
    put(ssm_head_at::in, deep ? in.frac : ssm_decayed(1.0f, in.frac, in.whole));
    put(ssm_head_at::whole, (float) floor(cum));
    put(ssm_head_at::frac, (float) (cum - floor(cum)));
    if (lane == 0) *(ssm_decay *) (rec + ssm_head_at::decay) = d;
}

// the first blocks the shared operands, a quarter of a chunk's rows each; the
// others the heads' decays, a wave a chunk
template <int NP>
__global__ __launch_bounds__(256) void k_ssm_split(ssm_chunk_args q) {
    if (blockIdx.x >= q.split_blocks) {
        ssm_decays(q, (int64_t) (blockIdx.x - q.split_blocks) * 4 + (threadIdx.x >> 6));
        return;
    }
    constexpr int kRow = NP + 4;
    __shared__ float sb[kSsmL][kRow];
    __shared__ float sc[16][kRow];
    const ssm_scan_args & a = q.a;
    const int part = blockIdx.x % 4;
    const int64_t chunk = blockIdx.x / 4 % q.chunks, sg = blockIdx.x / 4 / q.chunks;
    const int s = (int) (sg / a.groups), g = (int) (sg % a.groups);
    const int64_t t0 = chunk * kSsmL;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const char * B = a.B + g * a.B_nb1 + s * a.B_nb3;
    const char * C = a.C + g * a.C_nb1 + s * a.C_nb3;
    const int brows = 16 * part + 16;  // the rows of B up to this quarter's last
    ssm_most most;
    const bool vec = a.n % 4 == 0 && (((uintptr_t) B | (uintptr_t) C | (uintptr_t) a.B_nb2 | (uintptr_t) a.C_nb2) & 15) == 0;
    auto mags = [&](float4 v) { most.add(v.x, v.y), most.add(v.z, v.w); };
    if (vec) {
        float4 vb[kSsmL * NP / 1024], vc[16 * NP / 1024];
#pragma unroll
        for (int k = 0; k < kSsmL * NP / 1024; k++) {
            const int i = tid + 256 * k, t = i / (NP / 4), n = i % (NP / 4) * 4;
            const bool ok = t0 + t < a.tokens && n < a.n && t < brows;
            vb[k] = make_float4(0, 0, 0, 0);
            if (ok) vb[k] = *(const float4 *) (B + (t0 + t) * a.B_nb2 + 4 * n);
        }
#pragma unroll
        for (int k = 0; k < 16 * NP / 1024; k++) {
            const int i = tid + 256 * k, t = 16 * part + i / (NP / 4), n = i % (NP / 4) * 4;
            const bool ok = t0 + t < a.tokens && n < a.n;
            vc[k] = make_float4(0, 0, 0, 0);
            if (ok) vc[k] = *(const float4 *) (C + (t0 + t) * a.C_nb2 + 4 * n);
        }
#pragma unroll
        for (int k = 0; k < kSsmL * NP / 1024; k++) {
            const int i = tid + 256 * k;
            *(float4 *) &sb[i / (NP / 4)][i % (NP / 4) * 4] = vb[k];
            mags(vb[k]);
        }
#pragma unroll
        for (int k = 0; k < 16 * NP / 1024; k++) {
            const int i = tid + 256 * k;
            *(float4 *) &sc[i / (NP / 4)][i % (NP / 4) * 4] = vc[k];
            mags(vc[k]);
        }
    } else {
        for (int i = tid; i < brows * NP; i += 256) {
            const int t = i / NP, n = i % NP;
            const bool ok = t0 + t < a.tokens && n < a.n;
            sb[t][n] = ok ? ((const float *) (B + (t0 + t) * a.B_nb2))[n] : 0.0f;
            most.add(sb[t][n], 0.0f);
        }
        for (int i = tid; i < 16 * NP; i += 256) {
            const int t = 16 * part + i / NP, n = i % NP;
            const bool ok = t0 + t < a.tokens && n < a.n;
            sc[i / NP][n] = ok ? ((const float *) (C + (t0 + t) * a.C_nb2))[n] : 0.0f;
            most.add(sc[i / NP][n], 0.0f);
        }
    }
    const int bad = __syncthreads_or(most.past(kSsmLargest));  // (and the rows are staged)
    using at = ssm_shared_at<NP>;
    char * rec = q.shared + (sg * q.chunks + chunk) * at::size;
    if (tid == 0) *(uint8_t *) (rec + at::bad + part) = bad != 0;
    const int r = lane & 15, gq = lane >> 4;
    for (int kb = wave; kb < at::KB; kb += 4) {
        ssm_parts p;
        ssm_parts8(*(const ssm_v4f *) &sc[r][32 * kb + 4 * gq], *(const ssm_v4f *) &sc[r][32 * kb + 16 + 4 * gq], p);
#pragma unroll
        for (int i = 0; i < 3; i++) ((ssm_u4 *) (rec + at::c))[((part * at::KB + kb) * 3 + i) * 64 + lane] = p.v[i];
    }
    for (int k = wave; k < at::NK; k += 4) {  // a half of each fragment: this quarter's tokens
        const float * b = &sb[16 * part + 4 * gq][16 * k + r];
        uint32_t h[2], m[2], l[2];
        ssm_parts2(b[0], b[kRow], h[0], m[0], l[0]);
        ssm_parts2(b[2 * kRow], b[3 * kRow], h[1], m[1], l[1]);
        ssm_u2 * o = (ssm_u2 *) (rec + at::b) + ((part / 2 * at::NK + k) * 3 * 64 + lane) * 2 + part % 2;
        o[0] = ssm_u2{h[0], h[1]}, o[128] = ssm_u2{m[0], m[1]}, o[256] = ssm_u2{l[0], l[1]};
    }
    // C . B: wave w the 16-block of tokens j from 16 w on (rows j, columns t: a
    // lane ends with its elements), K in an order both operands share, in f32
    if (wave > (part | 1)) return;
    ssm_v4f acc = {0, 0, 0, 0}, acc2 = {0, 0, 0, 0};
    if (wave <= part) {
#pragma unroll 4
        for (int k = 0; k < at::NK; k++) {
            const int n = 16 * k + 4 * gq;
            const float4 x = *(const float4 *) &sb[16 * wave + r][n], y = *(const float4 *) &sc[r][n];
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, acc, 0, 0, 0);
            acc2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, acc2, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, acc, 0, 0, 0);
            acc2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, acc2, 0, 0, 0);
        }
        acc += acc2;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (wave == part && 4 * gq + i > r) acc[i] = 0.0f;  // past the row's token: not seen
    }
    ((ssm_v4f *) (rec + at::cb))[ssm_block(part, wave) * 64 + lane] = acc;
}

// token by token: the chunk's nt tokens from t0 on for a wave's 16 channels,
// for chunks the matrix form cannot take. Lane (g, r) holds n = 16 k + 4 g + i
// of channel p, as the matrix form does.
template <int NP, bool OUT>
__device__ __forceinline__ void ssm_tokens(ssm_v4f (&st)[NP / 16], int s, int h, int p, int64_t t0, int nt) {
    // (the kernel's arguments, read here: kept over the caller's loop, they would spill)
    SSM_UNIFORM ssm_scan_args * ap = (SSM_UNIFORM ssm_scan_args *) __builtin_amdgcn_kernarg_segment_ptr();
    static_assert(offsetof(ssm_chunk_args, a) == 0, "the kernel's first argument");
    asm volatile("" : "+s"(ap));
    SSM_UNIFORM ssm_scan_args & a = *ap;
    const float A = *(const float *) (a.A + h * a.A_nb1);
    const int g = h / (a.heads / a.groups);
    const bool mine = p < a.dim;
#pragma unroll 1
    for (int t = 0; t < nt; t++) {
        int gq = (threadIdx.x & 63) >> 4;
        asm volatile("" : "+v"(gq));  // (what follows from the lane is made anew: kept, it would spill)
        const float d = ssm_softplus(*(const float *) (a.dt + 4 * h + (t0 + t) * a.dt_nb1 + s * a.dt_nb2));
        const float ea = expf(d * A);
        const float * b = (const float *) (a.B + g * a.B_nb1 + (t0 + t) * a.B_nb2 + s * a.B_nb3);
        const float * c = (const float *) (a.C + g * a.C_nb1 + (t0 + t) * a.C_nb2 + s * a.C_nb3);
        const float * x = (const float *) (a.x + h * a.x_nb1 + (t0 + t) * a.x_nb2 + s * a.x_nb3);
        const float u = mine ? x[p] * d : 0.0f;
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < NP / 16; k++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = 16 * k + 4 * gq + i, at = min(n, a.n - 1);
                // (a segment's own zero is none of the state's: no growth spoils it)
                const float v = !OUT && st[k][i] == 0.0f ? u * b[at] : fmaf(st[k][i], ea, u * b[at]);
                st[k][i] = mine && n < a.n ? v : 0.0f;
                if constexpr (OUT) y = n < a.n ? fmaf(v, c[at], y) : y;
            }
            __builtin_amdgcn_sched_barrier(0);  // (one tile's loads at a time)
        }
        if constexpr (OUT) {
            y += __shfl_xor(y, 16);
            y += __shfl_xor(y, 32);
            if (gq == 0 && mine) a.y[((s * a.tokens + t0 + t) * a.heads + h) * a.dim + p] = y;
        }
    }
}

// 16 bytes a lane of N KB from a record straight to LDS, wave w of eight its
// share of them. What it writes is there after ssm_staged.
template <int N>
__device__ __forceinline__ void ssm_stage(const char * from, ssm_u4 * lds, int wave, uint32_t lane) {
    static_assert(N % 8 == 0, "as much for every wave");
#pragma unroll
    for (int k = 0; k < N / 8; k++)
        __builtin_amdgcn_global_load_lds(
            (const void __attribute__((address_space(1))) *) &ssm_at<const char>(from, 16 * lane + 1024u * (uint32_t) wave + 8192u * k),
            (void __attribute__((address_space(3))) *) (lds + 64 * (8 * k + wave)), 16, 0, 0);
}
// every wave's requests have arrived, and what they wrote to LDS is seen by all
__device__ __forceinline__ void ssm_staged() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0 (gfx9 encoding), the others as they are
    __syncthreads();
}

// lane q of each four holds v[e] of row q, and is given v[q] of row e: across
// neighbours, then across pairs
__device__ __forceinline__ void ssm_turn(ssm_v4f & v, int lane) {
    auto swap = [&](bool upper, auto ctrl, float & lo, float & hi) {
        const int got = __builtin_amdgcn_update_dpp(0, __float_as_int(upper ? lo : hi), decltype(ctrl)::value, 0xf, 0xf, true);
        if (upper) lo = __int_as_float(got);
        else hi = __int_as_float(got);
    };
    float a = v[0], b = v[1], c = v[2], d = v[3];
    const std::integral_constant<int, 0xB1> next;  // quad_perm 1, 0, 3, 2
    const std::integral_constant<int, 0x4E> pair;  // quad_perm 2, 3, 0, 1
    swap(lane & 1, next, a, b);
    swap(lane & 1, next, c, d);
    swap(lane & 2, pair, a, c);
    swap(lane & 2, pair, b, d);
    v = ssm_v4f{a, b, c, d};
}

// A step's instructions in order: 12 matrix ones with V vector ones under each,
// R reads of LDS after the third. (While requests to LDS are in flight a wait
// for the step before's reads is a wait for all there are: these come after it.)
template <int R, int V>
__device__ __forceinline__ void ssm_interleave() {
#pragma unroll
    for (int i = 0; i < 12; i++) {
        if (i == 3) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <int NP, bool OUT>
__global__ __launch_bounds__(512, 2) void k_ssm_chunks(ssm_chunk_args q) {
    using at = ssm_shared_at<NP>;
    constexpr int NK = at::NK, KB = at::KB;
    // Room for C's fragments and B's (OUT false: B's of two chunks); for states
    // of 256 for one of them at a time.
    constexpr bool kOne = NP > 128;
    __shared__ ssm_u4 s_c[12 * KB * 64];
    __shared__ ssm_u4 s_other[kOne ? 1 : 6 * NK * 64];
    static_assert(12 * KB == 6 * NK, "C and B are of one size");
    __shared__ ssm_u4 s_m[OUT ? 2 * 6 * 3 * 64 : 1];  // a block's C . B times the decays between: [fragment][part]
    __shared__ float s_dec[2][2][ssm_head_at::tokens][kSsmL];
    const ssm_scan_args & a = q.a;
    const int tid = threadIdx.x;
    // eight waves: four a block
    const int first_wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = first_wave >> 2;
    const int seg = blockIdx.y;
    const int g = (int) (blockIdx.x / q.pairs % a.groups), s = (int) (blockIdx.x / q.pairs / a.groups);
    const int per = a.heads / a.groups, blocks = per * q.pblocks;
    const int of_group = 2 * (int) (blockIdx.x % q.pairs) + half, blk = min(of_group, blocks - 1);
    const int h = g * per + blk / q.pblocks, pb = blk % q.pblocks, unit = (s * a.heads + h) * q.pblocks + pb;
    const int first_p = 64 * pb + 16 * (first_wave & 3);
    const bool idle = of_group >= blocks || first_p >= a.dim;  // the wave has no channel: it only stages
    const int64_t sg = (int64_t) s * a.groups + g, sh = (int64_t) s * a.heads + h;

    ssm_v4f st[NK];  // n = 16 k + 4 gq + i, channel p
    {
        const int lane = tid & 63, r = lane & 15, gq = lane >> 4, p = first_p + r;
        ssm_power carry = {1.0f, 0.0f};
        if constexpr (OUT) {
            double d = 0.0;
            for (int m = 0; m < seg; m++) d += q.seg_decay[sh * q.segs + m];
            carry = ssm_split_power(d);
        }
        const int64_t slot = a.ids[s];
        const bool has = OUT && slot >= 0 && slot < a.slots && p < a.dim;
        const float * s0 = (const float *) (a.s + (has ? slot : 0) * a.s_nb3) + ((int64_t) h * a.dim + p) * a.n;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int n = 16 * k + 4 * gq;
            st[k] = ssm_v4f{0, 0, 0, 0};
            if (q.svec) {
                if (has && n < a.n) st[k] = *(const ssm_v4f *) (s0 + n);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (has && n + i < a.n) st[k][i] = s0[n + i];
            }
        }
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) st[k][i] = ssm_decayed(st[k][i], carry.frac, carry.whole);
            for (int m = 0; m < seg; m++) {
                double d = 0.0;
                for (int e = m + 1; e < seg; e++) d += q.seg_decay[sh * q.segs + e];
                const ssm_power f = ssm_split_power(d);
                const ssm_v4f * o = (const ssm_v4f *) q.seg_state + (((int64_t) unit * q.segs + m) * 4 + (first_wave & 3)) * NK * 64 + lane;
#pragma unroll
                for (int k = 0; k < NK; k++) {
                    const ssm_v4f v = o[64 * k];
#pragma unroll
                    for (int i = 0; i < 4; i++) st[k][i] += ssm_decayed(v[i], f.frac, f.whole);
                }
            }
        }
    }
    const int c0 = seg * q.seg_chunks, c1 = (int) min((int64_t) c0 + q.seg_chunks, q.chunks);
    // (a lane's part of an address in 32 bits, the rest uniform)
    const uint32_t yrow = (uint32_t) (a.heads * a.dim);
    char * ybase = (char *) (a.y + ((s * a.tokens + (int64_t) c0 * kSsmL) * a.heads + h) * a.dim);
    const char * const xbase = a.x + h * a.x_nb1 + s * a.x_nb3;
    const char * gp = q.shared + (sg * q.chunks + c0) * at::size;              // the chunk's records
    const char * hp = q.heads + (sh * q.chunks + c0) * ssm_head_at::size;
    // A chunk's C, C . B, x and decays (OUT false: B for C) are in flight under
    // the products before, its B under those of its own C.
    ssm_v4f cbn[OUT ? 3 : 1], xn[4];
    float dn[2];
    int next_kind = 0, next_bad = 0;
    auto load_next = [&](int c, bool more, const char * gp, const char * hp, int tid, int wave, auto to_other) {
        const uint32_t lane = tid & 63, gq = lane >> 4, nb = (uint32_t) a.x_nb2;
        // token 4 gq + r % 4, channels r / 4 * 4 ..: ssm_turn makes u's of them (rows
        // past the last token: that one again)
        const char * row = xbase + (int64_t) c * kSsmL * a.x_nb2;
        const uint32_t last = (uint32_t) min((int64_t) kSsmL, a.tokens - (int64_t) c * kSsmL) - 1;
        const int p = 64 * pb + 16 * (wave & 3) + (tid & 12);
        if (q.xvec) {
#pragma unroll
            for (int b = 0; b < 4; b++)
                xn[b] = ssm_at<const ssm_v4f>(row, 4u * (uint32_t) min(p, a.dim - 4) + min(16u * b + 4 * gq + (tid & 3), last) * nb);
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++)
                xn[k / 4][k % 4] = ssm_at<const float>(row, 4u * (uint32_t) min(p + k % 4, a.dim - 1) +
                                                                min(16u * (k / 4) + 4 * gq + (tid & 3), last) * nb);
        }
        next_kind = *(SSM_UNIFORM int *) (hp + ssm_head_at::decay + offsetof(ssm_decay, kind));
        next_bad = *(SSM_UNIFORM int *) (gp + at::bad);
        dn[0] = ssm_at<const float>(hp, 4u * (uint32_t) (tid & 255));
        dn[1] = ssm_at<const float>(hp + 1024, 4u * (uint32_t) (tid & 127));
        // (behind the others: a wait for those does not wait for it)
        if (!kOne && more) ssm_stage<12 * KB>(gp + (OUT ? at::c : at::b), decltype(to_other)::value ? s_other : s_c, wave, lane);
    };
    auto load_cb = [&](const char * gp, int tid, int wave) {
        const uint32_t lane = tid & 63;
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < 3; k++) cbn[k] = ssm_at<const ssm_v4f>(gp + at::cb, 1024u * (uint32_t) ((wave & 3) + 4 * k) + 16 * lane);
        }
    };
    static_assert(ssm_head_at::tokens * kSsmL == 384 && ssm_head_at::decay == 4 * 384, "the threads' share of the decays");
    enum { kDt, kLeft, kLeftWhole, kIn, kWhole, kFrac };
    // whether the wave's states are past what the matrix form takes: at the
    // start, and after chunks it did not
    auto large_state = [&] {
        ssm_most most;
#pragma unroll
        for (int k = 0; k < NK; k++) most.add(st[k][0], st[k][1]), most.add(st[k][2], st[k][3]);
        return (bool) __any(most.past(kSsmLargestState));
    };
    bool large = large_state();
    if (c0 < c1) {
        load_next(c0, true, gp, hp, tid, first_wave, std::false_type{});
        load_cb(gp, tid, first_wave);
    }
    auto next = [&] { gp += at::size, hp += ssm_head_at::size, ybase += 4 * kSsmL * (int64_t) yrow; };
    // OUT false: odd chunks' B is in the other room (as types: reads of one room
    // do not wait for requests to the other)
    auto chunk = [&](int c, auto odd) {
        constexpr bool kOdd = decltype(odd)::value;
        // The lane and the wave are unknown to the compiler anew in every
        // iteration: what follows from them, kept over the loop, would spill.
        int tid = threadIdx.x, wave = first_wave;
        asm volatile("" : "+v"(tid), "+s"(wave));
        const int lane = tid & 63, r = lane & 15, gq = lane >> 4, w = wave & 3;
        const int64_t t0 = (int64_t) c * kSsmL;
        const int nt = (int) min((int64_t) kSsmL, a.tokens - t0);
        float (&dec)[ssm_head_at::tokens][kSsmL] = s_dec[c & 1][wave >> 2];
        const bool deep = next_kind & kSsmDeep, apart = (next_kind & kSsmOdd) || next_bad;
        (&dec[0][0])[tid & 255] = dn[0];
        if ((tid & 255) < 128) (&dec[0][0])[256 + (tid & 127)] = dn[1];
        if constexpr (kOne) {
            __syncthreads();  // the products of the chunk before have read B
            ssm_stage<12 * KB>(gp + (OUT ? at::c : at::b), s_c, wave, lane);
        }
        ssm_staged();  // C (OUT false: B) and the decays; the products of the chunk before have read B and the decayed C . B
        // u: channel r, tokens 16 b + 4 gq + i. (A token past the last has a step of
        // zero; channels past the last are never stored.)
        ssm_v4f u[4];
        ssm_most most;
#pragma unroll
        for (int b = 0; b < 4; b++) {
            u[b] = xn[b];
            ssm_turn(u[b], lane);
            u[b] *= *(const ssm_v4f *) &dec[kDt][16 * b + 4 * gq];
            most.add(u[b][0], u[b][1]), most.add(u[b][2], u[b][3]);
        }
        const bool by_token = apart || large || __any(most.past(kSsmLargest));
        ssm_v4f y[4];  // token 16 tb + r, channels 16 w + 4 gq + i
        ssm_parts us[2];
        ssm_u4 * const sm = s_m + (OUT ? (wave >> 2) * 6 * 3 * 64 : 0);
        if constexpr (OUT) {
            // (reads of the decays before requests to LDS: behind them they would wait)
            float tw[3], tf[3], e[4];
            ssm_v4f jw[3], jf[3];
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const int tb = k == 0 ? w >> 1 : 1 + k, jb = k == 0 ? w & 1 : w;
                tw[k] = dec[kWhole][16 * tb + r], tf[k] = dec[kFrac][16 * tb + r];
                jw[k] = *(const ssm_v4f *) &dec[kWhole][16 * jb + 4 * gq], jf[k] = *(const ssm_v4f *) &dec[kFrac][16 * jb + 4 * gq];
            }
#pragma unroll
            for (int tb = 0; tb < 4; tb++) e[tb] = dec[kIn][16 * tb + r];
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!kOne) ssm_stage<6 * NK>(gp + at::b, s_other, wave, lane);
            // the decayed C . B: three blocks a wave, half a fragment each
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const int i = w + 4 * k;
#pragma unroll
                for (int v = 0; v < 4; v++) cbn[k][v] = ssm_decayed(cbn[k][v], __builtin_amdgcn_exp2f(tf[k] - jf[k][v]), tw[k] - jw[k][v]);
                uint32_t h[2], m[2], l[2];
                ssm_parts2(cbn[k][0], cbn[k][1], h[0], m[0], l[0]);
                ssm_parts2(cbn[k][2], cbn[k][3], h[1], m[1], l[1]);
                ssm_u2 * o = (ssm_u2 *) sm + ((i / 2) * 3 * 64 + lane) * 2 + i % 2;
                o[0] = ssm_u2{h[0], h[1]}, o[128] = ssm_u2{m[0], m[1]}, o[256] = ssm_u2{l[0], l[1]};
            }
            if (!idle && !by_token) {
                // H C_t: a step takes 32 n and 32 tokens. The next step's fragments
                // are read under its products, with a share of the vector work
                // beside them: the state's next parts, then those of u.
                ssm_parts f[2][2], hs[2];
                auto read = [&](int m, ssm_parts (&v)[2]) {
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int i = 0; i < 3; i++) v[e].v[i] = s_c[(((2 * (m & 1) + e) * KB + m / 2) * 3 + i) * 64 + lane];
                };
#pragma unroll
                for (int tb = 0; tb < 4; tb++) y[tb] = ssm_v4f{0, 0, 0, 0};
                if constexpr (!kOne) read(0, f[0]);
                ssm_parts8(st[0], st[1], hs[0]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int m = 0; m < 2 * KB; m++) {
                    if constexpr (kOne) read(m, f[m & 1]);
                    else if (m + 1 < 2 * KB) read(m + 1, f[(m + 1) & 1]);
                    if ((m & 1) && m + 1 < 2 * KB) ssm_parts8(st[m + 1], st[m + 2], hs[(m / 2 + 1) & 1]);
                    if (m == 2 * KB - 1) ssm_parts8(u[0], u[1], us[0]);
#pragma unroll
                    for (int i = 0; i < 6; i++)
#pragma unroll
                        for (int e = 0; e < 2; e++) y[2 * (m & 1) + e] = ssm_product(i, hs[m / 2 & 1], f[m & 1][e], y[2 * (m & 1) + e]);
                    ssm_interleave<6, 4>();
                }
#pragma unroll
                for (int tb = 0; tb < 4; tb++) y[tb] *= e[tb];
                if (deep)
#pragma unroll
                    for (int tb = 0; tb < 4; tb++)
#pragma unroll
                        for (int i = 0; i < 4; i++) y[tb][i] = ldexpf(y[tb][i], (int) dec[kWhole][16 * tb + r]);
            }
        }
        if constexpr (OUT && kOne) {
            __syncthreads();  // the products have read C
            ssm_stage<6 * NK>(gp + at::b, s_c, wave, lane);
        }
        const ssm_u4 * const s_b = OUT ? (kOne ? s_c : s_other) : (!kOne && kOdd ? s_other : s_c);
        if constexpr (OUT) ssm_staged();  // B and the decayed C . B; the products have read C
        tid = threadIdx.x;  // (anew again: the addresses of the first products would stay)
        asm volatile("" : "+v"(tid));
        const int lane2 = tid & 63, r2 = lane2 & 15, gq2 = lane2 >> 4;
        const float ef = dec[kIn][63];
        __builtin_amdgcn_sched_barrier(0);
        const bool more = c + 1 < c1;
        // (at the end the last chunk's loads again, unused: no branch around what a
        // register waits for. But no request to LDS: none may outlive the kernel.)
        const char *const gn = more ? gp + at::size : gp, *const hn = more ? hp + ssm_head_at::size : hp;
        load_next(more ? c + 1 : c, more, gn, hn, tid, wave, std::integral_constant<bool, !OUT && !kOdd>{});
        if (idle) {
            load_cb(gn, tid, wave);
            return next();
        }
        if (by_token) {
            load_cb(gn, tid, wave);
            ssm_tokens<NP, OUT>(st, s, h, 64 * pb + 16 * w + r2, t0, nt);
            large = large_state();
            return next();
        }
        ssm_parts f[2][2], left_us[2];
        // the parts of 32 tokens' u, decayed to the chunk's end
        ssm_v4f left[2];
        ssm_i4 left_whole[2];
        auto read_left = [&](int m) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                left[e] = *(const ssm_v4f *) &dec[kLeft][32 * m + 16 * e + 4 * gq2];
                left_whole[e] = *(const ssm_i4 *) &dec[kLeftWhole][32 * m + 16 * e + 4 * gq2];
            }
        };
        auto make_left = [&](int m) {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) left[e][i] = ldexpf(u[2 * m + e][i] * left[e][i], left_whole[e][i]);
            ssm_parts8(left[0], left[1], left_us[m]);
        };
        auto read_b = [&](int m, ssm_parts (&v)[2]) {  // step m of the state's: 32 tokens, 32 n
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 3; i++) v[e].v[i] = s_b[((m / KB * NK + 2 * (m % KB) + e) * 3 + i) * 64 + lane2];
        };
        if constexpr (OUT) {
            // the chunk's own tokens: fragments 0 .. 3 of the first 32, 3 and 5 of the others
            auto read_m = [&](int m, ssm_parts (&v)[2]) {
                constexpr int frag[3][2] = {{0, 1}, {2, 4}, {3, 5}};
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int i = 0; i < 3; i++) v[e].v[i] = sm[(frag[m][e] * 3 + i) * 64 + lane2];
            };
            read_m(0, f[0]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < 3; m++) {  // tokens t 0 .. 31, 32 .. of the first 32; 32 .. of the others
                if (m + 1 < 3) read_m(m + 1, f[(m + 1) & 1]);
                else read_b(0, f[(m + 1) & 1]);
                if (m == 0) ssm_parts8(u[2], u[3], us[1]);
                else make_left(m - 1);
                if (m < 2) read_left(m);
#pragma unroll
                for (int i = 0; i < 6; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) y[2 * (m > 0) + e] = ssm_product(i, us[m / 2], f[m & 1][e], y[2 * (m > 0) + e]);
                if (m < 2) ssm_interleave<10, 4>();
                else ssm_interleave<6, 4>();
            }
            const int py = 64 * pb + 16 * w + 4 * gq2;
#pragma unroll
            for (int tb = 0; tb < 4; tb++) {
                const uint32_t at32 = 4u * ((uint32_t) (16 * tb + r2) * yrow + (uint32_t) py);
                if (q.yvec) {
                    if (py < a.dim && 16 * tb + r2 < nt) ssm_at<ssm_v4f>(ybase, at32) = y[tb];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (py + i < a.dim && 16 * tb + r2 < nt) ssm_at<float>(ybase, at32 + 4 * i) = y[tb][i];
                }
            }
        } else {
            read_b(0, f[1]);
#pragma unroll
            for (int m = 0; m < 2; m++) {
                read_left(m);
                make_left(m);
            }
        }
        // the state after the chunk
#pragma unroll
        for (int k = 0; k < NK; k++) st[k] *= ef;
        if (deep) {
            const int ew = (int) dec[kWhole][63];
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) st[k][i] = ldexpf(st[k][i], ew);
        }
        // step m: tokens 32 (m / KB) .., the state's tiles 2 (m % KB) ..
#pragma unroll
        for (int m = 0; m < 2 * KB; m++) {
            if constexpr (kOne) read_b(m, f[(m + 1) & 1]);
            else if (m + 1 < 2 * KB) read_b(m + 1, f[m & 1]);
#pragma unroll
            for (int i = 0; i < 6; i++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    st[2 * (m % KB) + e] = ssm_product(i, f[(m + 1) & 1][e], left_us[m / KB], st[2 * (m % KB) + e]);
            ssm_interleave<6, 4>();
        }
        load_cb(gn, tid, wave);
        next();
    };
    for (int c = c0; c < c1; c++) {
        chunk(c, std::false_type{});
        if (!OUT && !kOne && ++c < c1) chunk(c, std::true_type{});
    }
    if (of_group >= blocks) return;
    const int lane = tid & 63, gq = lane >> 4, p = first_p + (lane & 15);
    if constexpr (OUT) {
        if (seg != q.segs - 1 || p >= a.dim) return;
        float * o = a.out + (sh * a.dim + p) * a.n;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int n = 16 * k + 4 * gq;
            if (q.svec) {
                if (n < a.n) *(ssm_v4f *) (o + n) = st[k];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (n + i < a.n) o[n + i] = st[k][i];
            }
        }
    } else {
        if (pb == 0 && (tid & 255) == 0) {
            double decayed = 0.0;
            hp = q.heads + (sh * q.chunks + c0) * ssm_head_at::size;
            for (int c = c0; c < c1; c++) decayed += ((const ssm_decay *) (hp + (c - c0) * ssm_head_at::size + ssm_head_at::decay))->total;
            q.seg_decay[sh * q.segs + seg] = decayed;
        }
        ssm_v4f * o = (ssm_v4f *) q.seg_state + (((int64_t) unit * q.segs + seg) * 4 + (first_wave & 3)) * NK * 64 + lane;
#pragma unroll
        for (int k = 0; k < NK; k++) o[64 * k] = st[k];
    }
}

// ------------------------------------------------------------- launches ---

bool ssm_scan_supported(int64_t n) { return n >= 1 && n <= 256; }

static size_t ssm_al(size_t v) { return (v + 255) / 256 * 256; }

// The chunked form takes a decay a head over enough tokens, channels and state
// elements to fill its tiles. Chunked / token by token, us: 80 heads of 64 x 128,
// one sequence 8 tokens 19 / 21, 12 19 / 30; 16 sequences 8 51 / 51, 12 51 / 67; 48
// sequences 8 128 / 122, 12 128 / 164; 24 heads of 64 x 32 8 tokens 14 / 13, 12 14 /
// 17, 64 15 / 74; 8 heads of 16 x 20 8 tokens 14 / 13, 12 14 / 17; 4 sequences of 40
// heads of 64 x 256 12 tokens 38 / 36, 24 39 / 64.
static bool ssm_chunked(const ssm_scan_args & a) {
    return !a.a_elem && a.tokens >= 12 && a.dim >= 16 && a.n >= 16 &&
           (int64_t) a.heads * a.dim < 1 << 22 && a.x_nb2 < 1 << 25 &&  // (a lane's rows of y and x in 32-bit offsets)
           a.tokens <= kSsmMostTokens;
}

static int ssm_np(const ssm_scan_args & a) { return a.n <= 64 ? 64 : a.n <= 128 ? 128 : 256; }

// Segments of a chunked scan. A workgroup a CU runs at a time, so n segments
// take the rounds of their workgroups times a segment's chunks and what it
// reads of the segments before it; the first pass, which forms no outputs,
// about half of that for all segments but the last, and a launch. In quarters
// of a chunk's time.
static void ssm_segments(const ssm_scan_args & a, int n_cu, ssm_chunk_args & q) {
    q.a = a;
    q.chunks = (a.tokens + kSsmL - 1) / kSsmL;
    q.pblocks = (a.dim + 63) / 64;
    q.pairs = (a.heads / a.groups * q.pblocks + 1) / 2;
    const int64_t units = (int64_t) a.seqs * a.groups * q.pairs;
    auto rounds = [&](int64_t wgs) { return (wgs + n_cu - 1) / n_cu; };
    int64_t best = 0, best_cost = INT64_MAX;
    for (int64_t n = 1; n <= 32 && n <= q.chunks; n++) {
        const int64_t each = (q.chunks + n - 1) / n, segs = (q.chunks + each - 1) / each;
        const int64_t cost = rounds(units * segs) * (4 * each + segs / 2 + 2) +
                             (segs > 1 ? rounds(units * (segs - 1)) * (2 * each + 2) + 8 : 0);
        if (cost < best_cost) best = each, best_cost = cost;
    }
    q.seg_chunks = (int) best;
    q.segs = (int) ((q.chunks + best - 1) / best);
}

// the scratch's parts, in order; base null: their total size only
static size_t ssm_carve(ssm_chunk_args & q, char * base) {
    const ssm_scan_args & a = q.a;
    const size_t np = (size_t) ssm_np(a);
    size_t at = 0;
    auto take = [&](auto *& p, size_t bytes) {
        p = (typename std::remove_reference<decltype(p)>::type) (base + at);
        at += ssm_al(bytes);
    };
    const size_t rec = (size_t) (np == 64 ? ssm_shared_at<64>::size : np == 128 ? ssm_shared_at<128>::size : ssm_shared_at<256>::size);
    take(q.shared, (size_t) a.seqs * a.groups * q.chunks * rec);
    take(q.heads, (size_t) a.seqs * a.heads * q.chunks * ssm_head_at::size);
    const size_t segs = q.segs > 1 ? (size_t) q.segs : 0;
    take(q.seg_state, (size_t) a.seqs * a.heads * q.pblocks * segs * 64 * np * 4);
    take(q.seg_decay, (size_t) a.seqs * a.heads * segs * 8);
    return at;
}

// Segments of the short states' form: about two waves a SIMD, of 16 tokens or
// more, since each reads the earlier segments' states. At 4 / 8 / 16 waves a CU,
// us, states of 16: 5120 channels, 1000 tokens 105 / 81 / 89, two sequences of
// them 185 / 133 / 120; 4096 channels, 2000 tokens 151 / 123 / 123; 4 x 200 tokens
// of 2048 38 / 43 / 42; 1024 channels, 300 or 1000 tokens alike.
static bool ssm_lanes(const ssm_scan_args & a) { return a.n <= kSsmLane; }
static void ssm_lane_segments(const ssm_scan_args & a, int n_cu, ssm_lane_args & q) {
    q.a = a;
    q.blocks = ((int64_t) a.heads / a.groups * a.dim + 63) / 64;
    const int64_t units = q.blocks * a.groups * a.seqs;
    const int64_t segs = std::max<int64_t>(1, std::min<int64_t>({8 * n_cu / units, a.tokens / 16, 32}));
    q.seg_tokens = (a.tokens + segs - 1) / segs;
    q.segs = q.seg_tokens ? (int) ((a.tokens + q.seg_tokens - 1) / q.seg_tokens) : 1;
}

size_t ssm_scan_scratch_bytes(const ssm_scan_args & a, int n_cu) {
    if ((int64_t) a.seqs * a.heads * a.dim == 0) return 0;
    if (ssm_chunked(a)) {
        ssm_chunk_args q{};
        ssm_segments(a, n_cu, q);
        return ssm_carve(q, nullptr);
    }
    if (!ssm_lanes(a)) return 0;
    ssm_lane_args q{};
    ssm_lane_segments(a, n_cu, q);
    return (size_t) (q.segs - 1) * (a.n + 1) * 4 * a.seqs * a.heads * a.dim;
}

static void launch_ssm_lanes(const ssm_scan_args & a, void * scratch, hipStream_t s, int n_cu) {
    ssm_lane_args q{};
    ssm_lane_segments(a, n_cu, q);
    q.part = (float *) scratch;
    const int64_t units = q.blocks * a.groups * a.seqs;
    auto go = [&](auto k, int64_t segs) {
        hipLaunchKernelGGL(k, dim3((unsigned) ((units * segs + 3) / 4)), dim3(256), 0, s, q);
    };
    const bool full = a.n == kSsmLane;
    if (q.segs > 1) full ? go(k_ssm_scan_lanes<true, false>, q.segs - 1) : go(k_ssm_scan_lanes<false, false>, q.segs - 1);
    full ? go(k_ssm_scan_lanes<true, true>, q.segs) : go(k_ssm_scan_lanes<false, true>, q.segs);
}

// whole 16-byte pieces of the states and the streams
static bool ssm_pieces(const ssm_scan_args & a) {
    const uintptr_t at = (uintptr_t) a.s | (uintptr_t) a.s_nb3 | (uintptr_t) a.B | (uintptr_t) a.C | (uintptr_t) a.out |
                         (uintptr_t) a.B_nb1 | (uintptr_t) a.B_nb2 | (uintptr_t) a.B_nb3 | (uintptr_t) a.C_nb1 |
                         (uintptr_t) a.C_nb2 | (uintptr_t) a.C_nb3;
    return a.n % 4 == 0 && (at & 15) == 0;
}

static void launch_ssm_chunks(const ssm_scan_args & a, void * scratch, hipStream_t s, int n_cu) {
    ssm_chunk_args q{};
    ssm_segments(a, n_cu, q);
    ssm_carve(q, (char *) scratch);
    auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        const unsigned units = (unsigned) (a.seqs * a.groups * q.pairs);
        const auto whole = [](uintptr_t bits) { return (bits & 15) == 0; };
        q.xvec = a.dim % 4 == 0 && whole((uintptr_t) a.x | (uintptr_t) a.x_nb1 | (uintptr_t) a.x_nb2 | (uintptr_t) a.x_nb3);
        q.yvec = a.dim % 4 == 0 && whole((uintptr_t) a.y);
        q.svec = a.n % 4 == 0 && whole((uintptr_t) a.s | (uintptr_t) a.s_nb3 | (uintptr_t) a.out);
        q.split_blocks = (uint32_t) (4 * q.chunks * a.seqs * a.groups);
        const uint32_t decay_blocks = (uint32_t) ((q.chunks * a.seqs * a.heads + 3) / 4);
        hipLaunchKernelGGL(k_ssm_split<NP>, dim3(q.split_blocks + decay_blocks), dim3(256), 0, s, q);
        if (q.segs > 1)
            hipLaunchKernelGGL((k_ssm_chunks<NP, false>), dim3(units, (unsigned) (q.segs - 1)), dim3(512), 0, s, q);
        hipLaunchKernelGGL((k_ssm_chunks<NP, true>), dim3(units, (unsigned) q.segs), dim3(512), 0, s, q);
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
    if (ssm_lanes(a)) return launch_ssm_lanes(a, scratch, s, n_cu);
    const int per = a.n <= 128 ? 16 : 8;  // rows of a head a wave of k_ssm_scan_pieces takes
    const int64_t waves = (a.dim + per - 1) / per * (int64_t) a.heads * a.seqs;
    if (ssm_pieces(a) && waves <= 1 << 25) {  // (the other form's grid may be shorter than its rows)
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned) ((waves + 3) / 4)), dim3(256), 0, s, a); };
        if (a.n <= 64) go(k_ssm_scan_pieces<16, 4>);
        else if (a.n <= 128) go(k_ssm_scan_pieces<32, 8>);
        else go(k_ssm_scan_pieces<64, 8>);
        return;
    }
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) std::min<int64_t>((rows + 3) / 4, 1 << 22)), dim3(256), 0, s, a);
    };
    if (a.n <= 64) go(k_ssm_scan_rows<1>);
    else if (a.n <= 128) go(k_ssm_scan_rows<2>);
    else go(k_ssm_scan_rows<4>);
}

}  // namespace mi355x
