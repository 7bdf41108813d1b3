// k_ssm.hip -- the state-space mixer's operators: GGML_OP_SSM_CONV (the short
// depthwise causal convolution over the carried and the step's columns) and
// GGML_OP_SSM_SCAN (the selective scan).
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

bool ssm_scan_supported(int64_t n) { return n >= 1 && n <= 256; }

void launch_ssm_scan(const ssm_scan_args & a, hipStream_t s) {
    const int64_t rows = (int64_t) a.seqs * a.heads * a.dim;
    if (rows == 0) return;
    auto go = [&](auto kernel, int w) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) ((rows * w + 255) / 256)), dim3(256), 0, s, a);
    };
    if (a.n <= 16) go(k_ssm_scan_rows<16, 1>, 16);
    else if (a.n <= 64) go(k_ssm_scan_rows<64, 1>, 64);
    else if (a.n <= 128) go(k_ssm_scan_rows<64, 2>, 64);
    else go(k_ssm_scan_rows<64, 4>, 64);
}

}  // namespace mi355x
