// k_ssm.hip -- the state-space mixer's operators: GGML_OP_SSM_CONV (the short
// depthwise causal convolution over the carried and the step's columns) and
// GGML_OP_SSM_SCAN (the selective scan).
#include <algorithm>
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
                st[r] = fmaf(st[r], expf(dt * av[r]), ok ? xv * b[k] : 0.0f);
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
        if (!has || !in) st[u] = ssm_v4f{0, 0, 0, 0};
    for (int64_t t = 0; t < a.tokens; t++) {
        token v = next;
        if (t + 1 < a.tokens) load(t + 1, next);
        const float dt = ssm_softplus(v.dt);
        float d[4];
        d[0] = expf(dt * av[0]);
#pragma unroll
        for (int e = 1; e < 4; e++) d[e] = a.a_elem ? expf(dt * av[e]) : d[0];
        if (!in) v.b = v.c = ssm_v4f{0, 0, 0, 0};
        float y[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float xv = v.x[u] * dt;
            y[u] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                st[u][e] = fmaf(st[u][e], d[e], in ? xv * v.b[e] : 0.0f);
                y[u] = fmaf(st[u][e], v.c[e], y[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            y[u] = group_sum<W>(y[u]);
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
            if (__any(dt * low < -126.0f)) {  // below the instruction's range
#pragma unroll
                for (int k = 0; k < N; k++) e[k] = exp2f(dt * A[k]);
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
// 2 x 2048 tokens of 80 heads of 64 x 128: 110 us and 41 for the first pass,
// bound by the vector instructions around the products (965 a wave and chunk:
// scales, halves, decays; the products, three for each, are 40 GFLOP: 37 us at
// a large product's rate), and 11 for the shared operands. 333 tokens of 24 x 64 x 64: 14 + 6 + 7 us.
//
// k_ssm_split makes the operands that a group's heads share: C in rows and B
// in columns, split, with their scales, and C_t . B_j. k_ssm_chunks gives a
// workgroup a (sequence, head, 64 channels, segment of chunks): wave w owns
// the state's rows n in its quarter (in accumulators) and, for y, 16 tokens.
// k_ssm_split also sums the heads' log decays. Where there are few heads the sequence is cut into segments: the
// first pass (OUT false) makes each segment's own state from zeros, and the
// second starts from the earlier segments' states, decayed and added.
//
// Non-finite values would spread inside a chunk (0 * inf), and tokens far
// larger than the ones before them would cost those their bits: such a chunk,
// and one whose decays leave the exact range, runs token by token
// (ssm_chunk_slow), where a value reaches what the recurrence takes it to.

typedef float ssm_v2f __attribute__((ext_vector_type(2)));
typedef _Float16 ssm_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 ssm_v4h __attribute__((ext_vector_type(4)));
typedef _Float16 ssm_v2h __attribute__((ext_vector_type(2)));

constexpr int kSsmL = 64;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ ssm_v4f ssm_mfma(ssm_v8h a, ssm_v8h b, ssm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// a b of split halves for four b's: the three products of one accumulator
// apart, since each waits for the one before
__device__ __forceinline__ void ssm_products(ssm_v8h ah, ssm_v8h al, const ssm_v8h (&bh)[4], const ssm_v8h (&bl)[4],
                                             ssm_v4f (&c)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = ssm_mfma(ah, bh[i], c[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = ssm_mfma(ah, bl[i], c[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = ssm_mfma(al, bh[i], c[i]);
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
// an element at a uniform base, a lane's byte offset and a constant one: the
// address form a load takes without 64-bit vector arithmetic
template <typename T>
__device__ __forceinline__ T & ssm_at(const void * base, uint32_t off, int fixed = 0) {
    return *(T *) ((char *) base + off + fixed);
}
template <int W>
__device__ __forceinline__ uint32_t ssm_group_max(uint32_t v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = max(v, (uint32_t) __shfl_xor((int) v, o, W));
    return v;
}
__device__ __forceinline__ bool ssm_finite(uint32_t mag) { return mag < 0x7F800000u; }

// f16 hi + lo of N products x f (the lo part by a fused multiply-add)
template <int N, typename V, typename F>
__device__ __forceinline__ void ssm_halves(const float (&x)[N], F f, V & hi, V & lo) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const ssm_v2f v = {x[e] * f(e), x[e + 1] * f(e + 1)};
        const ssm_v2h h = __builtin_convertvector(v, ssm_v2h);
        const ssm_v2f d = {fmaf(x[e], f(e), -(float) h.x), fmaf(x[e + 1], f(e + 1), -(float) h.y)};
        const ssm_v2h l = __builtin_convertvector(d, ssm_v2h);
        hi[e] = h.x, hi[e + 1] = h.y;
        lo[e] = l.x, lo[e + 1] = l.y;
    }
}

// what a chunk's decays need besides the tokens' own
struct ssm_decay {
    double total;       // its log2 decay
    int e_dt, e_left;   // the exponents of the largest step, and of the largest step times the decay after it
    int odd, pad;       // outside what the matrix form takes
};
struct ssm_flags {
    int bad[4];  // a quarter's rows hold a non-finite value
    int kb;      // B's operand is its value times 2^kb
    int pad[3];
};

// The operands in scratch: a record a (sequence, group, chunk) and one a
// (sequence, head, chunk), byte offsets of their parts, NP the padded state size
template <int NP>
struct ssm_shared_at {
    static constexpr int c_hi = 0;              // [64 tokens][NP] f16, each token's row scaled
    static constexpr int c_lo = 128 * NP;
    static constexpr int b_hi = 256 * NP;       // [NP][64 tokens] f16, scaled
    static constexpr int b_lo = 384 * NP;
    static constexpr int cb = 512 * NP;         // [64][64] f32: C_t . B_j for j <= t (zeros past it), rows scaled
    static constexpr int c_s = cb + 16384;      // [64] f32: a row of C is its operand times this
    static constexpr int cb_s = c_s + 256;      // [64] f32: a row of C . B is its operand times this
    static constexpr int flags = cb_s + 256;    // ssm_flags
    static constexpr int size = flags + 256;
};
struct ssm_head_at {  // c_t: the sum of the log2 decays from the chunk's start to token t
    static constexpr int dt = 0;        // [64] f32: the step over 2^e_dt
    static constexpr int left = 256;    // [64] f32: the step times 2^(c_L - c_t), over 2^e_left
    static constexpr int whole = 512;   // [64] f32: c_t's whole and fractional part
    static constexpr int frac = 768;
    static constexpr int decay = 1024;  // ssm_decay
    static constexpr int size = 1280;
};
struct ssm_chunk_args {
    ssm_scan_args a;
    char *shared, *heads;
    float * seg_state;   // [seq, head, channel block][segment][64][NP]
    double * seg_decay;  // [seq, head][segment]: its log2 decay
    int64_t chunks;
    int segs, seg_chunks, pblocks;
    uint32_t split_blocks;
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
    const double total = __shfl(cum, 63), whole = floor(cum);
    const float left = dt * __builtin_amdgcn_exp2f((float) (total - cum));
    // the largest step's exponents: the operands' scales are bounded by them
    const uint32_t md = ssm_group_max<64>(ssm_mag(dt)), ml = ssm_group_max<64>(ssm_mag(left));
    ssm_decay d{};
    d.total = total;
    d.e_dt = max((int) (md >> 23) - 127, -60);
    d.e_left = max((int) (ml >> 23) - 127, -60);
    // A positive, or decays whose whole parts leave f32's exact range
    d.odd = !(total <= 0.0 && total > -8388608.0) || !ssm_finite(md);
    ((float *) (rec + ssm_head_at::dt))[lane] = dt * ssm_pow2(-d.e_dt);
    ((float *) (rec + ssm_head_at::left))[lane] = left * ssm_pow2(-d.e_left);
    ((float *) (rec + ssm_head_at::whole))[lane] = (float) whole;
    ((float *) (rec + ssm_head_at::frac))[lane] = (float) (cum - whole);
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
    uint32_t mb = 0;
    const bool vec = a.n % 4 == 0 && (((uintptr_t) B | (uintptr_t) C | (uintptr_t) a.B_nb2 | (uintptr_t) a.C_nb2) & 15) == 0;
    if (vec) {
        float4 vb[kSsmL * NP / 1024], vc[16 * NP / 1024];
#pragma unroll
        for (int k = 0; k < kSsmL * NP / 1024; k++) {
            const int i = tid + 256 * k, t = i / (NP / 4), n = i % (NP / 4) * 4;
            const bool ok = t0 + t < a.tokens && n < a.n;
            vb[k] = *(const float4 *) (B + (ok ? t0 + t : 0) * a.B_nb2 + (ok ? 4 * n : 0));
            if (!ok) vb[k] = make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 16 * NP / 1024; k++) {
            const int i = tid + 256 * k, t = 16 * part + i / (NP / 4), n = i % (NP / 4) * 4;
            const bool ok = t0 + t < a.tokens && n < a.n;
            vc[k] = *(const float4 *) (C + (ok ? t0 + t : 0) * a.C_nb2 + (ok ? 4 * n : 0));
            if (!ok) vc[k] = make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kSsmL * NP / 1024; k++) {
            const int i = tid + 256 * k;
            *(float4 *) &sb[i / (NP / 4)][i % (NP / 4) * 4] = vb[k];
            mb = max(max(mb, max(ssm_mag(vb[k].x), ssm_mag(vb[k].y))), max(ssm_mag(vb[k].z), ssm_mag(vb[k].w)));
        }
#pragma unroll
        for (int k = 0; k < 16 * NP / 1024; k++) {
            const int i = tid + 256 * k;
            *(float4 *) &sc[i / (NP / 4)][i % (NP / 4) * 4] = vc[k];
        }
    } else {
        for (int i = tid; i < kSsmL * NP; i += 256) {
            const int t = i / NP, n = i % NP;
            const bool ok = t0 + t < a.tokens && n < a.n;
            sb[t][n] = ok ? ((const float *) (B + (t0 + t) * a.B_nb2))[n] : 0.0f;
            mb = max(mb, ssm_mag(sb[t][n]));
        }
        for (int i = tid; i < 16 * NP; i += 256) {
            const int t = 16 * part + i / NP, n = i % NP;
            const bool ok = t0 + t < a.tokens && n < a.n;
            sc[i / NP][n] = ok ? ((const float *) (C + (t0 + t) * a.C_nb2))[n] : 0.0f;
        }
    }
    __shared__ uint32_t s_mb[4];
    mb = ssm_group_max<64>(mb);
    if (lane == 0) s_mb[wave] = mb;
    __syncthreads();
    mb = max(max(s_mb[0], s_mb[1]), max(s_mb[2], s_mb[3]));
    using at = ssm_shared_at<NP>;
    char * rec = q.shared + (sg * q.chunks + chunk) * at::size;
    // C's rows: 16 threads each
    const int row = tid / 16, sub = tid % 16;
    uint32_t mc = 0;
    for (int n = sub; n < NP; n += 16) mc = max(mc, ssm_mag(sc[row][n]));
    mc = ssm_group_max<16>(mc);
    const int kb = ssm_finite(mb) ? ssm_scale(mb) : 0, kc = ssm_finite(mc) ? ssm_scale(mc) : 0;
    const int any = __syncthreads_or(!ssm_finite(mb) || !ssm_finite(mc));
    if (tid == 0) {
        ssm_flags * fl = (ssm_flags *) (rec + at::flags);
        fl->bad[part] = any;
        if (part == 0) fl->kb = kb;
    }
    const int t = 16 * part + row;
    if (sub == 0) ((float *) (rec + at::c_s))[t] = ssm_pow2(-kc);
    const float fc = ssm_pow2(kc), fb = ssm_pow2(kb);
    for (int n = 8 * sub; n < NP; n += 128) {
        float v[8];
        ssm_v8h hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = sc[row][n + e];
        ssm_halves(v, [&](int) { return fc; }, hi, lo);
        *(ssm_v8h *) (rec + at::c_hi + 2 * (t * NP + n)) = hi;
        *(ssm_v8h *) (rec + at::c_lo + 2 * (t * NP + n)) = lo;
    }
    // B's columns: 16 tokens of one a thread
    if (tid < NP) {
        _Float16 * oh = (_Float16 *) (rec + at::b_hi) + tid * kSsmL + 16 * part;
        _Float16 * ol = (_Float16 *) (rec + at::b_lo) + tid * kSsmL + 16 * part;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float v[8];
            ssm_v8h hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = sb[16 * part + 8 * h + e][tid];
            ssm_halves(v, [&](int) { return fb; }, hi, lo);
            *(ssm_v8h *) (oh + 8 * h) = hi;
            *(ssm_v8h *) (ol + 8 * h) = lo;
        }
    }
    // C . B: wave w the 16-block of tokens j from 16 w on, K in an order both operands share
    const int r = lane & 15, gq = lane >> 4;
    ssm_v4f acc = {0, 0, 0, 0};
    if (wave <= part) {
        ssm_v4f acc2 = {0, 0, 0, 0};
#pragma unroll 4
        for (int n = 4 * gq; n < NP; n += 16) {
            const float4 x = *(const float4 *) &sc[r][n], y = *(const float4 *) &sb[16 * wave + r][n];
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, acc, 0, 0, 0);
            acc2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, acc2, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, acc, 0, 0, 0);
            acc2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, acc2, 0, 0, 0);
        }
        acc += acc2;
    }
    // rows 4 gq + i, column r: what is past the row's token is not seen
    __shared__ uint32_t s_row[4][16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (wave == part && r > 4 * gq + i) acc[i] = 0.0f;
        const uint32_t m = ssm_group_max<16>(ssm_mag(acc[i]));
        if (r == 0) s_row[wave][4 * gq + i] = m;
    }
    __syncthreads();
    float * cb = (float *) (rec + at::cb) + 16 * part * kSsmL + 16 * wave;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int m = 4 * gq + i;
        const int k = ssm_scale(max(max(s_row[0][m], s_row[1][m]), max(s_row[2][m], s_row[3][m])));
        cb[m * kSsmL + r] = acc[i] * ssm_pow2(k);
        if (wave == 0 && r == 0) ((float *) (rec + at::cb_s))[16 * part + m] = ssm_pow2(-k);
    }
}

constexpr int kSsmXRow = kSsmL + 8;  // halfs of a staged channel's tokens, padded

template <int NP>
struct ssm_lds {
    _Float16 x[4][64][kSsmXRow];  // u for y (hi, lo), u 2^(c_L - c_j) for the state (hi, lo): [channel][token]
    _Float16 st[2][64][NP + 8];   // the entering state (hi, lo): [channel][n]
    float whole[kSsmL], frac[kSsmL];  // c_t
    uint32_t mag[3][4][64];       // a channel's largest x, state, and its first x but 0, by wave
    float red[4][64];
    float steps[4][32];           // a wave's tokens' dt, then left (read by their wave only)
};

// token by token: the chunk's nt tokens from t0 on, for chunks the matrix
// form cannot take. The state is in LDS (in the place of its split halves,
// [channel][n]); wave w takes its quarter of n, a lane its channel.
template <int NP, bool OUT>
__device__ __forceinline__ void ssm_chunk_slow(const ssm_scan_args & a, ssm_lds<NP> & L, int s, int h, int p0, int64_t t0,
                                               int nt, float A) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (nothing of this path is kept over the caller's loop)
    const int wave = threadIdx.x >> 6;
    const int g = h / (a.heads / a.groups), p = p0 + lane;
    float * st = (float *) &L.st[0][0][0] + lane * (NP + 8);
    const int n1 = min((wave + 1) * (NP / 4), a.n);
#pragma unroll 1
    for (int t = 0; t < nt; t++) {
        const float d = ssm_softplus(*(const float *) (a.dt + 4 * h + (t0 + t) * a.dt_nb1 + s * a.dt_nb2));
        const float ea = __builtin_amdgcn_exp2f(d * A * kLog2e);
        const float * b = (const float *) (a.B + g * a.B_nb1 + (t0 + t) * a.B_nb2 + s * a.B_nb3);
        const float * c = (const float *) (a.C + g * a.C_nb1 + (t0 + t) * a.C_nb2 + s * a.C_nb3);
        const float * x = (const float *) (a.x + h * a.x_nb1 + (t0 + t) * a.x_nb2 + s * a.x_nb3);
        const float u = p < a.dim ? x[p] * d : 0.0f;
        float y = 0.0f;
#pragma unroll 1
        for (int n = wave * (NP / 4); n < n1; n++) {
            st[n] = fmaf(st[n], ea, u * b[n]);
            y = fmaf(st[n], c[n], y);
        }
        if constexpr (OUT) {
            L.red[wave][lane] = y;
            __syncthreads();
            if (wave == 0 && p < a.dim)
                a.y[((s * a.tokens + t0 + t) * a.heads + h) * a.dim + p] =
                    (L.red[0][lane] + L.red[1][lane]) + (L.red[2][lane] + L.red[3][lane]);
            __syncthreads();
        }
    }
}

// (what the launch before wrote and all lanes read alike: scalar loads)
#define SSM_UNIFORM const __attribute__((address_space(4)))

template <int NP, bool OUT>
__global__ __launch_bounds__(256, NP == 256 ? 1 : 2) void k_ssm_chunks(ssm_chunk_args q) {
    constexpr int NT = NP / 64;  // 16-row tiles of the state a wave owns
    __shared__ __align__(16) ssm_lds<NP> L;
    const ssm_scan_args & a = q.a;
    const int lane = threadIdx.x & 63, r = lane & 15, gq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int unit = blockIdx.x, seg = blockIdx.y;
    const int pb = unit % q.pblocks, h = unit / q.pblocks % a.heads, s = unit / (q.pblocks * a.heads);
    const int g = h / (a.heads / a.groups), p0 = 64 * pb;
    const int64_t sg = (int64_t) s * a.groups + g, sh = (int64_t) s * a.heads + h;
    const float A = *(const float *) (a.A + h * a.A_nb1);
    const int nbase = wave * (NP / 4);

    // the state: rows n = nbase + 16 k + 4 gq + i, channels 16 pt + r; its
    // value times 2^ks[pt] (channel lane: 2^kst)
    ssm_v4f st[NT][4];
    int ks[4] = {0, 0, 0, 0}, kst = 0;
    {
        float carry = 1.0f;
        if constexpr (OUT) {
            double d = 0.0;
            for (int m = 0; m < seg; m++) d += q.seg_decay[sh * q.segs + m];
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
                    st[k][pt][i] = has && n < a.n && p < a.dim ? s0[(int64_t) p * a.n + n] * carry : 0.0f;
                }
        if constexpr (OUT) {
            for (int m = 0; m < seg; m++) {
                double d = 0.0;
                for (int e = m + 1; e < seg; e++) d += q.seg_decay[sh * q.segs + e];
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
    const int64_t yrow = (int64_t) a.heads * a.dim;
    const char * const xbase = a.x + h * a.x_nb1 + s * a.x_nb3;
    using at = ssm_shared_at<NP>;
    const char * gp = q.shared + (sg * q.chunks + c0) * at::size;              // the chunk's records
    const char * hp = q.heads + (sh * q.chunks + c0) * ssm_head_at::size;
    // the next chunk's x and c_t, in flight under this one's products
    float xn[16], stepn = 0.0f, wholen = 0.0f, fracn = 0.0f;
    // (a lane's part of an address in 32 bits, the rest uniform)
    auto load_next = [&](int64_t c, const char * hp, int lane) {
        const uint32_t xo = 4u * (uint32_t) (p0 + lane < a.dim ? p0 + lane : 0), lo4 = 4u * (uint32_t) lane;
        // lanes 0 .. 15 the wave's dt, 16 .. 31 its left
        stepn = ssm_at<const float>(hp + 64 * wave, 4u * (uint32_t) ((lane & 15) + 4 * (lane & 16)));
        if (OUT && wave == 0) {
            wholen = ssm_at<const float>(hp, lo4, ssm_head_at::whole);
            fracn = ssm_at<const float>(hp, lo4, ssm_head_at::frac);
        }
        // rows from the wave's first token on, the last token's again past it
        const int64_t t = min(c * kSsmL + 16 * wave, a.tokens - 1);
        const char * row = xbase + t * a.x_nb2;
        const int left = (int) min((int64_t) 16, a.tokens - 1 - t);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            xn[i] = ssm_at<const float>(row, xo);
            row += i < left ? a.x_nb2 : 0;
        }
    };
    if (c0 < c1) load_next(c0, hp, lane);
    double decayed = 0.0;
    for (int64_t c = c0; c < c1; c++, gp += at::size, hp += ssm_head_at::size) {
        // The lane is unknown to the compiler anew in every iteration: the
        // addresses that follow from it, kept over the loop, would spill, and
        // a spill's reload waits for every load in flight.
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int r = lane & 15, gq = lane >> 4, px = p0 + lane;  // px: the channel this lane stages
        const uint32_t co = 2u * (uint32_t) ((16 * wave + r) * NP + 8 * gq);
        const uint32_t bo = 2u * (uint32_t) ((nbase + r) * kSsmL + 8 * gq);
        const uint32_t cbo = 4u * (uint32_t) ((16 * wave + r) * kSsmL + 8 * gq), cso = 4u * (uint32_t) (16 * wave + 4 * gq);
        const uint32_t yo = 4u * ((uint32_t) (16 * wave + 4 * gq) * (uint32_t) yrow + (uint32_t) r);
        const int64_t t0 = c * kSsmL;
        const int nt = (int) min((int64_t) kSsmL, a.tokens - t0);
        const bool inside = nt == kSsmL && p0 + 64 <= a.dim;
        SSM_UNIFORM ssm_decay * dec = (SSM_UNIFORM ssm_decay *) (hp + ssm_head_at::decay);
        SSM_UNIFORM ssm_flags * fl = (SSM_UNIFORM ssm_flags *) (gp + at::flags);
        static_assert(ssm_head_at::left == 256 && ssm_head_at::dt == 0, "the lanes' offsets of dt and left");
        if (lane < 32) L.steps[wave][lane] = stepn;
        const double total = dec->total;
        const int e_dt = dec->e_dt, e_left = dec->e_left, odd = dec->odd;
        const int bad = fl->bad[0] | fl->bad[1] | fl->bad[2] | fl->bad[3], kb = fl->kb;
        const float whole = wholen, frac = fracn;
        float x[16];
        uint32_t mx = 0, first = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = xn[i];
        if (!inside) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = px < a.dim && 16 * wave + i < nt ? x[i] : 0.0f;
        }
        if (!OUT && c + 1 < c1) load_next(c + 1, hp + ssm_head_at::size, lane);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            mx = max(mx, ssm_mag(x[i]));
            first = first ? first : mx;
        }
#pragma unroll
        for (int pt = 0; pt < 4; pt++) {
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) m = max(m, ssm_mag(st[k][pt][i]));
            m = max(m, (uint32_t) __shfl_xor((int) m, 16));
            m = max(m, (uint32_t) __shfl_xor((int) m, 32));
            if (gq == 0) L.mag[1][wave][16 * pt + r] = m;
        }
        L.mag[0][wave][lane] = mx;
        L.mag[2][wave][lane] = first;
        __syncthreads();  // the magnitudes; every wave is done with the chunk before
        // The chunk's operands, requested where the arithmetic up to their use
        // covers their latency, and ahead of the next chunk's x: loads return
        // in order, and x comes from HBM.
        ssm_v8h ch[OUT ? NP / 32 : 1], cl[OUT ? NP / 32 : 1];
        float cbv[2][8], cs[4], cbs[4];
        if constexpr (OUT) {
#pragma unroll
            for (int kk = 0; kk < NP / 32; kk++) {
                ch[kk] = ssm_at<const ssm_v8h>(gp + at::c_hi, co, 64 * kk);
                cl[kk] = ssm_at<const ssm_v8h>(gp + at::c_lo, co, 64 * kk);
            }
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                *(float4 *) &cbv[kk][0] = ssm_at<const float4>(gp + at::cb, cbo, 128 * kk);
                *(float4 *) &cbv[kk][4] = ssm_at<const float4>(gp + at::cb, cbo, 128 * kk + 16);
            }
            *(float4 *) cs = ssm_at<const float4>(gp + at::c_s, cso);
            *(float4 *) cbs = ssm_at<const float4>(gp + at::cb_s, cso);
        }
        mx = max(max(L.mag[0][0][lane], L.mag[0][1][lane]), max(L.mag[0][2][lane], L.mag[0][3][lane]));
        const uint32_t ms = max(max(L.mag[1][0][lane], L.mag[1][1][lane]), max(L.mag[1][2][lane], L.mag[1][3][lane]));
        first = L.mag[2][0][lane] ? L.mag[2][0][lane] : L.mag[2][1][lane] ? L.mag[2][1][lane]
                : L.mag[2][2][lane] ? L.mag[2][2][lane] : L.mag[2][3][lane];
        // one step of the exponent is 2^23 in a float's bits
        const bool rising = (mx >> 23) > (first >> 23) + 24;
        decayed += total;
        // the same for every wave: they see the same magnitudes
        if (bad || odd || __any(rising || !ssm_finite(mx) || !ssm_finite(ms))) {
            float * sl = (float *) &L.st[0][0][0];
            static_assert(sizeof(L.st) == sizeof(float) * 64 * (NP + 8), "the state fits in place of its halves");
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++)
                    *(ssm_v4f *) (sl + (16 * pt + r) * (NP + 8) + nbase + 16 * k + 4 * gq) = st[k][pt] * ldexpf(1.0f, -ks[pt]);
            __syncthreads();
            ssm_chunk_slow<NP, OUT>(a, L, s, h, p0, t0, nt, A);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++)
                    st[k][pt] = *(const ssm_v4f *) (sl + (16 * pt + r) * (NP + 8) + nbase + 16 * k + 4 * gq);
#pragma unroll
            for (int pt = 0; pt < 4; pt++) ks[pt] = 0;
            kst = 0;
            __syncthreads();
            if (OUT && c + 1 < c1) load_next(c + 1, hp + ssm_head_at::size, lane);
            continue;
        }
        // Channel lane's exponents: x 2^kx below 2^14, so u below 2^15 over the
        // steps' exponent; the state, in its units, 2^km below 2^14. The
        // state's next units are those its new terms are staged in, 2^kv (at
        // most 2^30 finer than it needs: far from f32's ends).
        const int kx = ssm_scale(mx), km = ssm_scale(ms);
        int kv = min(kx - e_left + kb, 120);
        if (ms) kv = min(kv, kst + km + 30);
        int kxp[4], kmp[4], kvp[4];  // of the accumulators' channels
#pragma unroll
        for (int pt = 0; pt < 4; pt++) {
            kxp[pt] = __shfl(kx, 16 * pt + r);
            kmp[pt] = __shfl(km, 16 * pt + r);
            kvp[pt] = __shfl(kv, 16 * pt + r);
        }
        kst = kv;
        {
            const float fx = ssm_pow2(kx), fv = ldexpf(1.0f, kv + e_left - kb);
            const float *dts = L.steps[wave], *lefts = L.steps[wave] + 16;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float xs[8];
                ssm_v8h hi, lo;
                const int to = 16 * wave + 8 * half;
                if constexpr (OUT) {
#pragma unroll
                    for (int e = 0; e < 8; e++) xs[e] = x[8 * half + e] * fx;
                    ssm_halves(xs, [&](int e) { return dts[8 * half + e]; }, hi, lo);
                    *(ssm_v8h *) &L.x[0][lane][to] = hi;
                    *(ssm_v8h *) &L.x[1][lane][to] = lo;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) xs[e] = x[8 * half + e] * fv;
                ssm_halves(xs, [&](int e) { return lefts[8 * half + e]; }, hi, lo);
                *(ssm_v8h *) &L.x[2][lane][to] = hi;
                *(ssm_v8h *) &L.x[3][lane][to] = lo;
            }
        }
        if (OUT && c + 1 < c1) load_next(c + 1, hp + ssm_head_at::size, lane);
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    const float fs = ssm_pow2(kmp[pt]);
                    float v[4];
                    ssm_v4h hi, lo;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = st[k][pt][i];
                    ssm_halves(v, [&](int) { return fs; }, hi, lo);
                    const int n = nbase + 16 * k + 4 * gq;
                    *(ssm_v4h *) &L.st[0][16 * pt + r][n] = hi;
                    *(ssm_v4h *) &L.st[1][16 * pt + r][n] = lo;
                }
            if (wave == 0) {
                L.whole[lane] = whole;
                L.frac[lane] = frac;
            }
        }
        ssm_v8h bh[2][NT], bl[2][NT];
        auto load_b = [&] {
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
                for (int k = 0; k < NT; k++) {
                    bh[kk][k] = ssm_at<const ssm_v8h>(gp + at::b_hi, bo, 32 * k * kSsmL + 64 * kk);
                    bl[kk][k] = ssm_at<const ssm_v8h>(gp + at::b_lo, bo, 32 * k * kSsmL + 64 * kk);
                }
        };
        if constexpr (!OUT) load_b();
        __syncthreads();
        if constexpr (OUT) {
            ssm_v4f yh[4], yx[4];
#pragma unroll
            for (int pt = 0; pt < 4; pt++) yh[pt] = yx[pt] = ssm_v4f{0, 0, 0, 0};
            ssm_v8h oh[4], ol[4];
            // H C_t
#pragma unroll
            for (int kk = 0; kk < NP / 32; kk++) {
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    oh[pt] = *(const ssm_v8h *) &L.st[0][16 * pt + r][32 * kk + 8 * gq];
                    ol[pt] = *(const ssm_v8h *) &L.st[1][16 * pt + r][32 * kk + 8 * gq];
                }
                ssm_products(ch[kk], cl[kk], oh, ol, yh);
                // (one K step's operands at a time: more in flight spill)
                __builtin_amdgcn_sched_barrier(0);
            }
            load_b();  // (in the registers that held C)
            __builtin_amdgcn_sched_barrier(0);
            // the chunk's own tokens: the decayed C . B of this lane's row (the
            // 16-blocks past the wave's tokens are zeros; a decay is at most one)
            const float tw = L.whole[16 * wave + r], tf = L.frac[16 * wave + r];
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                if (kk == 1 && wave < 2) continue;
                float jw[8], jf[8], m[8];
                *(float4 *) &jw[0] = *(const float4 *) &L.whole[32 * kk + 8 * gq];
                *(float4 *) &jw[4] = *(const float4 *) &L.whole[32 * kk + 8 * gq + 4];
                *(float4 *) &jf[0] = *(const float4 *) &L.frac[32 * kk + 8 * gq];
                *(float4 *) &jf[4] = *(const float4 *) &L.frac[32 * kk + 8 * gq + 4];
#pragma unroll
                for (int e = 0; e < 8; e++)
                    m[e] = __builtin_amdgcn_exp2f(fminf((tw - jw[e]) + (tf - jf[e]), 0.0f));
                ssm_v8h ah, al;
                ssm_halves(m, [&](int e) { return cbv[kk][e]; }, ah, al);
#pragma unroll
                for (int pt = 0; pt < 4; pt++) {
                    oh[pt] = *(const ssm_v8h *) &L.x[0][16 * pt + r][32 * kk + 8 * gq];
                    ol[pt] = *(const ssm_v8h *) &L.x[1][16 * pt + r][32 * kk + 8 * gq];
                }
                ssm_products(ah, al, oh, ol, yx);
                __builtin_amdgcn_sched_barrier(0);
            }
            float fh[4], fxr[4], fk[4], fu[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {  // rows: the tokens 16 wave + 4 gq + i
                const int tr = 16 * wave + 4 * gq + i;
                fh[i] = __builtin_amdgcn_exp2f(L.whole[tr] + L.frac[tr]) * cs[i];
                fxr[i] = cbs[i] * ssm_pow2(e_dt);
            }
#pragma unroll
            for (int pt = 0; pt < 4; pt++) {
                fk[pt] = ldexpf(1.0f, -ks[pt] - kmp[pt]);
                fu[pt] = ssm_pow2(-kxp[pt]);
            }
            float * yp = a.y + (((s * a.tokens + t0) * a.heads + h) * a.dim + p0);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int pt = 0; pt < 4; pt++)
                    yh[pt][i] = fmaf(yh[pt][i], fk[pt] * fh[i], yx[pt][i] * (fu[pt] * fxr[i]));
            if (inside) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int pt = 0; pt < 4; pt++) ssm_at<float>(yp + i * yrow, yo, 64 * pt) = yh[pt][i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int pt = 0; pt < 4; pt++)
                        if (16 * wave + 4 * gq + i < nt && p0 + 16 * pt + r < a.dim)
                            ssm_at<float>(yp + i * yrow, yo, 64 * pt) = yh[pt][i];
            }
        }
        // the state after the chunk
        {
            const float fd = __builtin_amdgcn_exp2f((float) total);
#pragma unroll
            for (int pt = 0; pt < 4; pt++) {
                const float f = fd * ssm_pow2(max(min(kvp[pt] - ks[pt], 126), -126));
#pragma unroll
                for (int k = 0; k < NT; k++) st[k][pt] *= f;
                ks[pt] = kvp[pt];
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            ssm_v8h xh[4], xl[4];
#pragma unroll
            for (int pt = 0; pt < 4; pt++) {
                xh[pt] = *(const ssm_v8h *) &L.x[2][16 * pt + r][32 * kk + 8 * gq];
                xl[pt] = *(const ssm_v8h *) &L.x[3][16 * pt + r][32 * kk + 8 * gq];
            }
#pragma unroll
            for (int k = 0; k < NT; k++) ssm_products(bh[kk][k], bl[kk][k], xh, xl, st[k]);
        }
    }
    float back[4];
#pragma unroll
    for (int pt = 0; pt < 4; pt++) back[pt] = ldexpf(1.0f, -ks[pt]);
    if constexpr (OUT) {
        if (seg != q.segs - 1) return;
        float * o = a.out + sh * a.dim * a.n;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int pt = 0; pt < 4; pt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = nbase + 16 * k + 4 * gq + i, p = p0 + 16 * pt + r;
                    if (n < a.n && p < a.dim) o[(int64_t) p * a.n + n] = st[k][pt][i] * back[pt];
                }
    } else {
        if (pb == 0 && threadIdx.x == 0) q.seg_decay[sh * q.segs + seg] = decayed;
        float * o = q.seg_state + ((int64_t) unit * q.segs + seg) * 64 * NP;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int pt = 0; pt < 4; pt++)
                *(float4 *) (o + (16 * pt + r) * NP + nbase + 16 * k + 4 * gq) =
                    make_float4(st[k][pt][0] * back[pt], st[k][pt][1] * back[pt], st[k][pt][2] * back[pt],
                                st[k][pt][3] * back[pt]);
    }
}

// ------------------------------------------------------------- launches ---

bool ssm_scan_supported(int64_t n) { return n >= 1 && n <= 256; }

static size_t ssm_al(size_t v) { return (v + 255) / 256 * 256; }

// The chunked form takes a decay a head over enough tokens, channels and state
// elements to fill its tiles. 80 heads of 64 x 128, with the call, chunked /
// token by token: one sequence 8 tokens 33 / 31 us, 12 33 / 40, 64 32 / 147;
// 16 sequences 12 tokens 83 / 79 us, 16 83 / 97, 64 83 / 309.
static bool ssm_chunked(const ssm_scan_args & a) {
    return !a.a_elem && a.tokens >= 12 && a.dim >= 16 && a.n >= 16 &&
           (int64_t) a.heads * a.dim < 1 << 22;  // (a chunk's rows of y in 32-bit offsets)
}

static int ssm_np(const ssm_scan_args & a) { return a.n <= 64 ? 64 : a.n <= 128 ? 128 : 256; }

// Segments of a chunked scan. Two workgroups a CU run at a time, so n segments
// take the rounds of their workgroups times a segment's chunks and what it
// reads of the segments before it; the first pass, which forms no outputs,
// about half of that for all segments but the last, and a launch. In quarters
// of a chunk's time.
static void ssm_segments(const ssm_scan_args & a, int n_cu, ssm_chunk_args & q) {
    q.a = a;
    q.chunks = (a.tokens + kSsmL - 1) / kSsmL;
    q.pblocks = (a.dim + 63) / 64;
    const int64_t units = (int64_t) a.seqs * a.heads * q.pblocks;
    auto rounds = [&](int64_t wgs) { return (wgs + 2 * n_cu - 1) / (2 * n_cu); };
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
// more, since each reads the earlier segments' states (5120 channels, 1000
// tokens, both passes: 8 waves a CU 83 us, 4 107, 6 97, 12 89, 16 100).
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
    if (a.seqs == 0) return 0;
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
        const unsigned units = (unsigned) (a.seqs * a.heads * q.pblocks);
        q.split_blocks = (uint32_t) (4 * q.chunks * a.seqs * a.groups);
        const uint32_t decay_blocks = (uint32_t) ((q.chunks * a.seqs * a.heads + 3) / 4);
        hipLaunchKernelGGL(k_ssm_split<NP>, dim3(q.split_blocks + decay_blocks), dim3(256), 0, s, q);
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
