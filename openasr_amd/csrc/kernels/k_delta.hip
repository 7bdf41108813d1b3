// k_delta.hip -- the gated delta rule (GGML_OP_GATED_DELTA_NET), a linear
// attention layer's recurrence, and L2_NORM, which its queries and keys go
// through. A head's state S [K, V] takes a token by
//     S <- e^g S,   d = beta (v - S^T k),   S <- S + k d^T,   y = S^T q / sqrt(K)
// with S held as V rows of K elements.
#include <algorithm>
#include <type_traits>

#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

typedef float dl_v4f __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------- l2 norm ---

// a wave a row, the sum of squares in f64; memory bounds it
__global__ __launch_bounds__(256) void k_l2_norm(tview d, tview a, float eps, int64_t rows) {
    const int lane = threadIdx.x & 63;
    const int64_t n = a.ne[0];
    for (int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t) gridDim.x * 4) {
        const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
        const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
        float * y = (float *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]);
        double sum = 0.0;
        for (int64_t i = lane; i < n; i += 64) sum += (double) x[i] * (double) x[i];
        const float inv = 1.0f / fmaxf(sqrtf((float) wave_sum_d(sum)), eps);
        for (int64_t i = lane; i < n; i += 64) y[i] = x[i] * inv;
    }
}

void launch_l2_norm(const tview & d, const tview & a, float eps, hipStream_t s) {
    const int64_t rows = a.ne[1] * a.ne[2] * a.ne[3];
    if (rows == 0 || a.ne[0] == 0) return;
    hipLaunchKernelGGL(k_l2_norm, dim3((unsigned) std::min<int64_t>((rows + 3) / 4, 1 << 20)), dim3(256), 0, s, d, a, eps, rows);
    note_hip_error(hipGetLastError());
}

// -------------------------------------------------------- token by token ---

// the sum over the 16 lanes of a row, in every lane
__device__ __forceinline__ float dl_sum16(float v) {
    auto add = [&](auto ctrl) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    add(std::integral_constant<int, 0x128>{});  // row_ror:8, 4, 2, 1
    add(std::integral_constant<int, 0x124>{});
    add(std::integral_constant<int, 0x122>{});
    add(std::integral_constant<int, 0x121>{});
    return v;
}

// 16 lanes hold a state row, P pieces of four elements a lane (4 (l + 16 p) ..),
// a wave 4 U rows of one head; the next tokens' operands are loaded ahead. VEC:
// every row in whole 16-byte pieces.
template <int P, int U, int AHEAD, bool VEC, bool ELEM>
__global__ __launch_bounds__(256) void k_delta_rows(delta_args a) {
    const int lane = threadIdx.x & 63, l = lane & 15, sub = lane >> 4;
    const uint32_t blocks = (uint32_t) ((a.V + 4 * U - 1) / (4 * U));
    const int64_t unit = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= (int64_t) blocks * a.heads * a.seqs) return;
    const int j0 = (int) (unit % blocks) * 4 * U + sub, h = (int) (unit / blocks % a.heads);
    const int s = (int) (unit / ((int64_t) blocks * a.heads)), hk = h % a.key_heads;
    auto piece = [&](const char * row, int p) {
        const int i = 4 * (l + 16 * p);
        dl_v4f v = {0, 0, 0, 0};
        if constexpr (VEC) {
            if (i < a.K) v = *(const dl_v4f *) (row + 4 * i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + e < a.K) v[e] = ((const float *) row)[i + e];
        }
        return v;
    };
    const char *q = a.q + hk * a.q_nb1 + s * a.q_nb3, *k = a.k + hk * a.k_nb1 + s * a.k_nb3;
    const char *v = a.v + h * a.v_nb1 + s * a.v_nb3, *g = a.g + h * a.g_nb1 + s * a.g_nb3, *b = a.beta + h * a.b_nb1 + s * a.b_nb3;
    struct token {
        dl_v4f q[P], k[P], g[ELEM ? P : 1];
        float beta, v[U];
    };
    auto load = [&](int64_t t, token & x) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            x.q[p] = piece(q + t * a.q_nb2, p);
            x.k[p] = piece(k + t * a.k_nb2, p);
            if constexpr (ELEM) x.g[p] = piece(g + t * a.g_nb2, p);
        }
        if constexpr (!ELEM) x.g[0][0] = *(const float *) (g + t * a.g_nb2);
        x.beta = *(const float *) (b + t * a.b_nb2);
#pragma unroll
        for (int u = 0; u < U; u++) x.v[u] = ((const float *) (v + t * a.v_nb2))[min(j0 + 4 * u, a.V - 1)];
    };
    token next[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; n++)
        if (a.tokens > 0) load(min((int64_t) n, a.tokens - 1), next[n]);
    dl_v4f st[U][P];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const char * row = a.s + s * a.s_nb3 + 4 * ((int64_t) h * a.V + min(j0 + 4 * u, a.V - 1)) * a.K;
#pragma unroll
        for (int p = 0; p < P; p++) st[u][p] = piece(row, p);
    }
    auto length = [&](const dl_v4f (&x)[P], float eps) {  // what a row is multiplied by
        if (eps < 0.0f) return 1.0f;
        float sum = 0.0f;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum = fmaf(x[p][e], x[p][e], sum);
        return 1.0f / fmaxf(sqrtf(dl_sum16(sum)), eps);
    };
    for (int64_t t0 = 0; t0 < a.tokens; t0 += AHEAD) {
#pragma unroll
        for (int n = 0; n < AHEAD; n++) {
            const int64_t t = t0 + n;
            if (t >= a.tokens) break;
            token x = next[n];
            if (t + AHEAD < a.tokens) load(t + AHEAD, next[n]);
            const float kl = length(x.k, a.k_eps), ql = length(x.q, a.q_eps) * a.scale;
            dl_v4f eg[ELEM ? P : 1];
#pragma unroll
            for (int p = 0; p < P; p++) {
                x.k[p] *= kl, x.q[p] *= ql;
                if constexpr (ELEM) {
#pragma unroll
                    for (int e = 0; e < 4; e++) eg[p][e] = expf(x.g[p][e]);
                }
            }
            if constexpr (!ELEM) {
                const float d = expf(x.g[0][0]);
                eg[0] = dl_v4f{d, d, d, d};
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float dot = 0.0f, y = 0.0f;
#pragma unroll
                for (int p = 0; p < P; p++) {
                    st[u][p] *= eg[ELEM ? p : 0];
#pragma unroll
                    for (int e = 0; e < 4; e++) dot = fmaf(st[u][p][e], x.k[p][e], dot);
                }
                const float d = x.beta * (x.v[u] - dl_sum16(dot));
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        st[u][p][e] = fmaf(x.k[p][e], d, st[u][p][e]);
                        y = fmaf(st[u][p][e], x.q[p][e], y);
                    }
                y = dl_sum16(y);
                if (l == 0 && j0 + 4 * u < a.V) a.y[((s * a.tokens + t) * a.heads + h) * a.V + j0 + 4 * u] = y;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (j0 + 4 * u >= a.V) continue;
        float * row = (float *) (a.out + s * a.out_nb3) + ((int64_t) h * a.V + j0 + 4 * u) * a.K;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int i = 4 * (l + 16 * p);
            if constexpr (VEC) {
                if (i < a.K) *(dl_v4f *) (row + i) = st[u][p];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < a.K) row[i + e] = st[u][p][e];
            }
        }
    }
}

// ------------------------------------------------------------- launches ---

bool delta_supported(int64_t K) { return K >= 1 && K <= 256; }

size_t delta_scratch_bytes(const delta_args & a, int n_cu) {
    (void) a, (void) n_cu;
    return 0;
}

template <int P, int U, int AHEAD>
static void launch_delta_rows(const delta_args & a, bool vec, hipStream_t s) {
    const int64_t units = (int64_t) ((a.V + 4 * U - 1) / (4 * U)) * a.heads * a.seqs;
    const dim3 grid((unsigned) ((units + 3) / 4));
    if (a.g_elem) {
        if (vec) hipLaunchKernelGGL((k_delta_rows<P, U, AHEAD, true, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_delta_rows<P, U, AHEAD, false, true>), grid, dim3(256), 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((k_delta_rows<P, U, AHEAD, true, false>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_delta_rows<P, U, AHEAD, false, false>), grid, dim3(256), 0, s, a);
    }
    note_hip_error(hipGetLastError());
}

void launch_delta(const delta_args & a, void * scratch, hipStream_t s, int n_cu) {
    (void) scratch, (void) n_cu;
    if (a.seqs == 0 || a.heads == 0 || a.V == 0) return;
    const uintptr_t al = (uintptr_t) a.q | (uintptr_t) a.k | (uintptr_t) a.s | (uintptr_t) a.out | (uintptr_t) a.q_nb1 |
                         (uintptr_t) a.q_nb2 | (uintptr_t) a.q_nb3 | (uintptr_t) a.k_nb1 | (uintptr_t) a.k_nb2 |
                         (uintptr_t) a.k_nb3 | (uintptr_t) a.s_nb3 | (uintptr_t) a.out_nb3 | (uintptr_t) (4 * a.K) |
                         (a.g_elem ? (uintptr_t) a.g | (uintptr_t) a.g_nb1 | (uintptr_t) a.g_nb2 | (uintptr_t) a.g_nb3 : 0);
    const bool vec = al % 16 == 0;
    if (a.K <= 64) launch_delta_rows<1, 2, 2>(a, vec, s);
    else if (a.K <= 128) launch_delta_rows<2, 2, 2>(a, vec, s);
    else launch_delta_rows<4, 2, 2>(a, vec, s);
}

}  // namespace mi355x
