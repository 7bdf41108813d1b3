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
typedef uint32_t dl_u2 __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------- l2 norm ---

// a wave a row, the sum of squares and its root in f64 (f32's squares end at rows of
// 1e-19 and 1e19). 131072 rows of 128 50 us, 2.7 TB/s, and of 256 3.8: the row's
// reduction bounds it
__global__ __launch_bounds__(256) void k_l2_norm(tview d, tview a, float eps, int64_t rows) {
    const int lane = threadIdx.x & 63;
    const int64_t n = a.ne[0];
    for (int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t) gridDim.x * 4) {
        const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
        const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
        float * y = (float *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]);
        double sum = 0.0;
        for (int64_t i = lane; i < n; i += 64) sum += (double) x[i] * (double) x[i];
        const float inv = 1.0f / fmaxf((float) sqrt(wave_sum_d(sum)), eps);
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

// e^x: the product's rounding error put back, so within an ulp or two at any x
__device__ __forceinline__ float dl_exp(float x) {
    const float z = x * 1.4426950408889634f, r = fmaf(x, 1.4426950408889634f, -z) + x * 1.925963e-8f;
    const float p = __builtin_amdgcn_exp2f(z);
    return x > -200.0f ? fmaf(p, r * 0.6931471805599453f, p) : p;  // (no infinity less itself)
}

// the largest of lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float dl_max4(float x) {
    // (the swaps' results as values: a bit cast of a vector's element takes its first)
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const uint32_t m = __float_as_uint(fmaxf(__uint_as_float(a0), __uint_as_float(a1)));
    const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return fmaxf(__uint_as_float(b0), __uint_as_float(b1));
}

// a row's sum of squares past this (an infinity) is made again of the row times 2^-64
constexpr float kDlSquares = 0x1.fffffep127f;

// 16 lanes hold a state row, P pieces of four elements a lane (4 (l + 16 p) ..),
// a wave 4 U rows of one head; the next token's operands are loaded ahead (four
// tokens' measured the same: 500 tokens of 16 heads of 12 x 128 255 us for 252). VEC:
// every row in whole 16-byte pieces.
template <int P, int U, bool VEC, bool ELEM>
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
    token next;
    if (a.tokens > 0) load(0, next);
    dl_v4f st[U][P];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const char * row = a.s + s * a.s_nb3 + 4 * ((int64_t) h * a.V + min(j0 + 4 * u, a.V - 1)) * a.K;
#pragma unroll
        for (int p = 0; p < P; p++) st[u][p] = piece(row, p);
    }
    // what a row is multiplied by: 1 / max(its length, eps), by v_rsq_f32, an ulp off (the
    // other forms take a root and a quotient)
    const float k_most = 1.0f / a.k_eps, q_most = 1.0f / a.q_eps;
    auto dot = [](const dl_v4f (&x)[P], const dl_v4f (&y)[P]) {
        dl_v4f v = x[0] * y[0];
#pragma unroll
        for (int p = 1; p < P; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = fmaf(x[p][e], y[p][e], v[e]);
        return (v[0] + v[1]) + (v[2] + v[3]);
    };
    auto squares = [&](const dl_v4f (&x)[P], float eps) { return eps < 0.0f ? 1.0f : dl_sum16(dot(x, x)); };
    auto by_small = [&](const dl_v4f (&x)[P]) {
        dl_v4f z[P];
#pragma unroll
        for (int p = 0; p < P; p++) z[p] = x[p] * 0x1p-64f;
        return __builtin_amdgcn_rsqf(dl_sum16(dot(z, z))) * 0x1p-64f;
    };
    for (int64_t t = 0; t < a.tokens; t++) {
        token x = next;
        if (t + 1 < a.tokens) load(t + 1, next);
        const float kk = squares(x.k, a.k_eps), qq = squares(x.q, a.q_eps);
        const float kl = a.k_eps < 0.0f ? 1.0f : fminf(__builtin_amdgcn_rsqf(kk), k_most);
        const float ql = (a.q_eps < 0.0f ? 1.0f : fminf(__builtin_amdgcn_rsqf(qq), q_most)) * a.scale;
        dl_v4f eg[ELEM ? P : 1];
        if constexpr (ELEM) {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) eg[p][e] = dl_exp(x.g[p][e]);
        } else {
            const float d = dl_exp(x.g[0][0]);
            eg[0] = dl_v4f{d, d, d, d};
        }
        float y[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int p = 0; p < P; p++) st[u][p] *= eg[ELEM ? p : 0];
            const float d = x.beta * (x.v[u] - kl * dl_sum16(dot(st[u], x.k))) * kl;
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) st[u][p][e] = fmaf(x.k[p][e], d, st[u][p][e]);
            y[u] = ql * dl_sum16(dot(st[u], x.q));
        }
        if (fmaxf(kk, qq) > kDlSquares) {
            // Squares past f32: kl, or ql, came out as 0, and the state is only decayed. The
            // token again (asked here, where nothing waits for the sums: before, 10 % of a token)
            const bool anew = kk > kDlSquares;
            const float kn = anew ? fminf(by_small(x.k), k_most) : kl, qn = qq > kDlSquares ? fminf(by_small(x.q), q_most) * a.scale : ql;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float d = anew ? x.beta * (x.v[u] - kn * dl_sum16(dot(st[u], x.k))) * kn : 0.0f;
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int e = 0; e < 4; e++) st[u][p][e] = fmaf(x.k[p][e], d, st[u][p][e]);
                y[u] = qn * dl_sum16(dot(st[u], x.q));
            }
        }
        float * to = a.y + ((s * a.tokens + t) * a.heads + h) * a.V + j0;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (l == 0 && j0 + 4 * u < a.V) to[4 * u] = y[u];
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

// Gates an element, many tokens. What every wave of a head would make again of a
// token's operands is made once: q's and k's rows brought to length (q's times the
// scale) and the decays, in rows of 64 P elements (zeros past K) [sequence][token][q of
// the key heads, k of them, decays of the heads]. 16 lanes a row.
template <int P>
__global__ __launch_bounds__(256) void k_delta_ready(delta_args a, float * out) {
    const int l = threadIdx.x & 15, rows = 2 * a.key_heads + a.heads;
    const int64_t unit = (int64_t) blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t u = min(unit, a.tokens * rows * a.seqs - 1);
    const int r = (int) (u % rows);
    const int64_t t = u / rows % a.tokens, s = u / rows / a.tokens;
    const bool q = r < a.key_heads, k = !q && r < 2 * a.key_heads;
    const char * x = q   ? a.q + r * a.q_nb1 + t * a.q_nb2 + s * a.q_nb3
                     : k ? a.k + (r - a.key_heads) * a.k_nb1 + t * a.k_nb2 + s * a.k_nb3
                         : a.g + (r - 2 * a.key_heads) * a.g_nb1 + t * a.g_nb2 + s * a.g_nb3;
    dl_v4f v[P];
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = 4 * (l + 16 * p);
        v[p] = dl_v4f{0, 0, 0, 0};
        if (i < a.K) v[p] = *(const dl_v4f *) (x + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) sum = fmaf(v[p][e], v[p][e], sum);
    }
    const float eps = q ? a.q_eps : a.k_eps;
    sum = dl_sum16(sum);
    float len = sqrtf(sum);
    if (sum > kDlSquares) {  // (all 16 lanes alike)
        sum = 0.0f;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum = fmaf(v[p][e] * 0x1p-64f, v[p][e] * 0x1p-64f, sum);
        len = sqrtf(dl_sum16(sum)) * 0x1p64f;
    }
    const float by = (eps < 0.0f ? 1.0f : 1.0f / fmaxf(len, eps)) * (q ? a.scale : 1.0f);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = 4 * (l + 16 * p);
#pragma unroll
        for (int e = 0; e < 4; e++) v[p][e] = q || k ? v[p][e] * by : i < a.K ? dl_exp(v[p][e]) : 0.0f;
        if (unit == u) *(dl_v4f *) &out[u * 64 * P + i] = v[p];
    }
}

// k_delta_rows on those rows: 16 lanes a state row, 4 U rows a wave, AHEAD tokens'
// operands loaded ahead and no branch between them. 500 tokens of 16 heads of 128 x
// 128: 107 us (and 8 for the rows; k_delta_rows 342), 0.21 a token, of it 190 cycles the
// CU's two waves' loads. Waves four a workgroup, on half of the CUs: 137
template <int P, int U>
__global__ __launch_bounds__(64) void k_delta_steps(delta_args a, const float * ready) {
    constexpr int AHEAD = P == 4 ? 4 : 8;
    const int l = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const uint32_t blocks = (uint32_t) ((a.V + 4 * U - 1) / (4 * U));
    const int64_t unit = blockIdx.x;
    const int j0 = (int) (unit % blocks) * 4 * U + sub, h = (int) (unit / blocks % a.heads);
    const int s = (int) (unit / ((int64_t) blocks * a.heads)), hk = h % a.key_heads, rows = 2 * a.key_heads + a.heads;
    const int64_t step = (int64_t) rows * 64 * P;
    const float * at = ready + s * a.tokens * step;
    const char *v = a.v + h * a.v_nb1 + s * a.v_nb3, *b = a.beta + h * a.b_nb1 + s * a.b_nb3;
    const int of[3] = {hk * 64 * P + 4 * l, (a.key_heads + hk) * 64 * P + 4 * l, (2 * a.key_heads + h) * 64 * P + 4 * l};
    int v_of[U];
#pragma unroll
    for (int u = 0; u < U; u++) v_of[u] = min(j0 + 4 * u, a.V - 1);
    struct token {
        dl_v4f q[P], k[P], g[P];
        float beta, v[U];
    };
    int64_t loaded = 0;
    auto load = [&](token & x) {  // the next token, or the last one again
#pragma unroll
        for (int p = 0; p < P; p++) {
            x.q[p] = *(const dl_v4f *) (at + of[0] + 64 * p);
            x.k[p] = *(const dl_v4f *) (at + of[1] + 64 * p);
            x.g[p] = *(const dl_v4f *) (at + of[2] + 64 * p);
        }
        x.beta = *(const float *) b;
#pragma unroll
        for (int u = 0; u < U; u++) x.v[u] = ((const float *) v)[v_of[u]];
        const bool more = ++loaded < a.tokens;
        at += more ? step : 0, v += more ? a.v_nb2 : 0, b += more ? a.b_nb2 : 0;
    };
    token next[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; n++) load(next[n]);
    dl_v4f st[U][P];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const char * row = a.s + s * a.s_nb3 + 4 * ((int64_t) h * a.V + v_of[u]) * a.K;
#pragma unroll
        for (int p = 0; p < P; p++) {
            st[u][p] = dl_v4f{0, 0, 0, 0};
            if (4 * (l + 16 * p) < a.K) st[u][p] = *(const dl_v4f *) (row + 16 * (l + 16 * p));
        }
    }
    auto dot = [](const dl_v4f (&x)[P], const dl_v4f (&y)[P]) {
        dl_v4f v = x[0] * y[0];
#pragma unroll
        for (int p = 1; p < P; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = fmaf(x[p][e], y[p][e], v[e]);
        return (v[0] + v[1]) + (v[2] + v[3]);
    };
    const int64_t y_step = (int64_t) a.heads * a.V;
    float * y = a.y + ((int64_t) s * a.y_tokens * a.heads + h) * a.V + j0 + l * y_step;
    float mine[U];  // y of token l of the AHEAD
    auto take = [&](const token & x, int n) {
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int p = 0; p < P; p++) st[u][p] *= x.g[p];
            const float d = x.beta * (x.v[u] - dl_sum16(dot(st[u], x.k)));
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) st[u][p][e] = fmaf(x.k[p][e], d, st[u][p][e]);
            const float r = dl_sum16(dot(st[u], x.q));
            mine[u] = l == n ? r : mine[u];
        }
    };
    // (a store a token waited for would hold back the loads that follow it)
    auto put = [&](int n) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (l < n && j0 + 4 * u < a.V) y[4 * u] = mine[u];
        y += AHEAD * y_step;
    };
#pragma unroll
    for (int u = 0; u < U; u++) mine[u] = 0.0f;
    int64_t t = 0;
    for (; t + AHEAD <= a.tokens; t += AHEAD) {
#pragma unroll
        for (int n = 0; n < AHEAD; n++) {
            take(next[n], n);
            load(next[n]);
        }
        put(AHEAD);
    }
#pragma unroll
    for (int n = 0; n < AHEAD; n++)
        if (t + n < a.tokens) take(next[n], n);
    put((int) (a.tokens - t));
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (j0 + 4 * u >= a.V) continue;
        float * row = (float *) (a.out + s * a.out_nb3) + ((int64_t) h * a.V + j0 + 4 * u) * a.K;
#pragma unroll
        for (int p = 0; p < P; p++)
            if (4 * (l + 16 * p) < a.K) *(dl_v4f *) (row + 4 * (l + 16 * p)) = st[u][p];
    }
}

// ---------------------------------------------------------------- chunks ---
//
// Chunks of C = 64 tokens as matrix products. With a_t the sum of the chunk's g
// up to t, L_ts = e^(a_t - a_s) and
//     A = strictly lower (beta_t k_t . k_s L_ts),   T = (1 + A)^-1
// a chunk turns the state S0 it meets into
//     D = T (beta V - beta e^a K S0),   Y = (e^a Q S0 + lower(Q K^T L) D) / sqrt(K)
//     S1 = e^(a_C) S0 + (e^(a_C - a) K)^T D
// k_delta_solve makes T, lower(Q K^T L) and the decays of every chunk at once
// (forward substitution by blocks of 16 tokens, whose diagonal blocks are
// inverted column by column: as stable as the recurrence), k_delta_chunks goes
// through the chunks, a workgroup a head and 16 or 32 columns of the state.
//
// k_delta_solve's products are f32's, on v_mfma_f32_16x16x4f32: A lane l = row l
// % 16, k l / 16; B lane l = column l % 16, the same k; result lane l = rows 4 (l
// / 16) .. + 3, column l % 16. Step i of four takes k = 4 (l / 16) + i, so that
// a result's four elements are the next product's B operand as they are, and A's
// rows come in 16-byte pieces.
//
// k_delta_chunks, whose chain of products is the time, makes them on the f16
// matrix cores: an operand is the sum of two f16 (22 bits), a product three of
// theirs, 24 cycles for 16 k where f32's take 128 (three bf16 parts and six
// products, 48, and their making in the chain took more time than they). The low
// parts are kept 2^10 times as large, and the two products with them summed apart:
// so an operand's error is 2^-22 of its own or 2^-34 of one, whichever is more.
// Rows of Q, K, T and lower(Q K^T L) are split by k_delta_solve, each row scaled to
// 2^13 by a power of two that the row's factor takes back; the state, T's operand
// and D are split as they are made, each of the state's columns in a scale of its
// own: a power of two from the largest value that the column of the state and of v
// has at the chunk's start. Columns, which the rule keeps apart, so never share an
// error, and a column's steps are 2^-40 of its largest value in the chunk (one scale a
// workgroup, and low parts as they are, had columns of 1e-5 of the largest 4e-4 off).
// The state itself is split before that value is known, in the scale of a chunk before
// (steps of 2^-33 of the largest at worst), and again where that is further off. A lane's
// eight k of 32 are four of one block of 16 and four of the next, so that results are
// operands here too.
//
// A chunk whose values are not finite or past 2^40, whose g are above zero, or whose scaled
// values would leave f16's range, runs token by token, 120 us a chunk: 2048 tokens of 32
// heads of 128 x 128 with keys of length 1e-3 3860 us, of length one 139 (and those short
// ones by k_delta_rows 923).

constexpr int kDlC = 64;
constexpr int kDlReady = 32;
// what the products take: q's and k's rows as they come, and (the largest element of a
// row) brought to length (the state of keys much shorter than one lies far under v, in
// whose scale it is split: with low parts as they are, keys of 1e-4 were 2e-3 off); beta; a row of |T| (1 to 3 for
// keys of length one and beta up to one; tokens of one key with a beta of 2, which turn
// the state over and over, come to 127, and were 4e-4 off); scaled values. The state
// and v: up to 2^40
constexpr int kDlLeastKExp = -7;
constexpr float kDlRaw = 0x1p50f, kDlRow = 0x1p10f, kDlLeastQ = 0x1p-20f, kDlLeastK = 0x1p-7f, kDlBeta = 16.0f, kDlRowSum = 64.0f, kDlHalf = 60000.0f;

struct dl_chunk_args {
    delta_args a;
    char * rec;          // records [sequence][head][chunk of the slab]
    char * krec;         // K^T [sequence][key head][chunk]: blocks (16 dims, 16 tokens), lane = row d l % 16, t 4 (l / 16) ..
    const char * s_in;   // the states the slab starts from
    int64_t s_in_nb3;
    int64_t c0, chunks;  // the slab's first chunk and its chunks
    int cols;            // column blocks of the state: 16 or 32 columns
};
// byte offsets in a record of a head's chunk
struct dl_rec {
    // [64] f32 each, what a row is multiplied by: of Q S0 (e^a, 1 / sqrt(K) and
    // what takes the scales back, times that of p's row), of Y (takes p's back), of
    // K S0 (beta, e^a), of V (beta), of T's product, of D for the state (e^(a_C - a)
    // over the largest of these)
    static constexpr int in = 0, y = 256, ks = 512, beta = 768, t_row = 1024, left = 1280;
    static constexpr int end = 1536;  // e^(a_C); what left was divided by; whether the chunk goes token by token
    // [4 token blocks][2 steps of 32 tokens][2 parts][lane] of lower(Q K^T L) / sqrt(K), and of T
    static constexpr int p = 2048, t = p + 16 * 1024;
    static constexpr int size = t + 16 * 1024;
};
// of a key head's: rows of Q and of K [4 token blocks][steps of 32 dims][2 parts][lane], K^T [dim blocks][2 steps of 32 tokens][2 parts][lane]
template <int NP>
struct dl_krec {
    static constexpr int q = 0, k = 4 * kDlC * NP, kt = 2 * k, size = 3 * k;
};
__device__ __forceinline__ int dl_pair(int tb, int sb) { return tb * (tb + 1) / 2 + sb; }

__device__ __forceinline__ dl_v4f dl_mfma(dl_v4f a, dl_v4f b, dl_v4f c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ bool dl_past(float v, float limit) { return !(fabsf(v) <= limit); }

typedef uint32_t dl_u4 __attribute__((ext_vector_type(4)));
typedef _Float16 dl_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 dl_h8 __attribute__((ext_vector_type(8)));
// two f32 as the sums of two f16 each, the low one times 2^10: so the smallest step is
// 2^-34 (f16's own is 2^-24)
constexpr float kDlLow = 0x1p10f;
__device__ __forceinline__ void dl_split2(float a, float b, uint32_t & hi, uint32_t & lo) {
    const dl_h2 h = __builtin_bit_cast(dl_h2, __builtin_amdgcn_cvt_pkrtz(a, b));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float) h[0], -kDlLow, a * kDlLow), fmaf((float) h[1], -kDlLow, b * kDlLow)));
}
struct dl_split {  // a lane's eight elements of k
    dl_u4 v[2];
};
__device__ __forceinline__ dl_split dl_split8(dl_v4f a, dl_v4f b) {
    uint32_t h[4], l[4];
    dl_split2(a[0], a[1], h[0], l[0]);
    dl_split2(a[2], a[3], h[1], l[1]);
    dl_split2(b[0], b[1], h[2], l[2]);
    dl_split2(b[2], b[3], h[3], l[3]);
    return {{dl_u4{h[0], h[1], h[2], h[3]}, dl_u4{l[0], l[1], l[2], l[3]}}};
}
// a sum of products: of the high parts, and of a high and a low one (times 2^10)
struct dl_sum {
    dl_v4f hi, lo;
};
// the i-th of a product's three
__device__ __forceinline__ void dl_product(int i, const dl_split & a, const dl_split & b, dl_sum & c) {
    dl_v4f & to = i < 2 ? c.lo : c.hi;
    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(dl_h8, a.v[i == 0]), __builtin_bit_cast(dl_h8, b.v[i == 1]), to, 0, 0, 0);
}
__device__ __forceinline__ dl_v4f dl_whole(const dl_sum & c) {
    dl_v4f v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = fmaf(c.lo[e], 1.0f / kDlLow, c.hi[e]);
    return v;
}
// 2^e, and the exponent of the power of two at or under |v| (within what f32's powers and their inverses hold)
__device__ __forceinline__ float dl_pow2(int e) { return __uint_as_float((uint32_t) (e + 127) << 23); }
__device__ __forceinline__ int dl_exponent(float v) { return min(max((int) ((__float_as_uint(v) >> 23) & 255) - 127, -100), 100); }

template <int NP>
__global__ __launch_bounds__(256, 2) void k_delta_solve(dl_chunk_args q) {
    constexpr int kRow = NP + 4, KB = NP / 16, kLoads = kDlC * NP / 1024;
    __shared__ __align__(16) float s_k[kDlC][kRow];
    __shared__ __align__(16) float s_kexp[kDlC], s_qexp[kDlC], s_beta[kDlC];  // s_kexp, s_qexp: a row's scale, to 2^13
    __shared__ double s_cum[kDlC];
    // A's blocks, lane = row t l % 16, s 4 (l / 16) ..; then T's rows
    __shared__ __align__(16) float s_at[kDlC * (kDlC + 4)];
    __shared__ __align__(16) float s_d[4][16][20];  // the diagonal blocks, then their inverses, row by row
    dl_v4f(&s_a)[10][64] = *(dl_v4f(*)[10][64]) s_at;
    float(&s_t)[kDlC][kDlC + 4] = *(float(*)[kDlC][kDlC + 4]) s_at;
    const delta_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
    const int64_t c = blockIdx.x % q.chunks;
    const int hk = (int) (blockIdx.x / q.chunks % a.key_heads), s = (int) (blockIdx.x / q.chunks / a.key_heads);
    const int64_t t0 = (q.c0 + c) * kDlC;
    const int nt = (int) min((int64_t) kDlC, a.tokens - t0);
    const char * kb = a.k + hk * a.k_nb1 + t0 * a.k_nb2 + s * a.k_nb3;
    const char * qb = a.q + hk * a.q_nb1 + t0 * a.q_nb2 + s * a.q_nb3;
    char * const krec = q.krec + (((int64_t) s * a.key_heads + hk) * q.chunks + c) * dl_krec<NP>::size;
    bool bad = false;
    // k's rows, and the wave's 16 rows of q as a B operand, all loads in flight
    dl_v4f kv[kLoads], qr[KB];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int e = tid + 256 * i, t = e / (NP / 4), n = e % (NP / 4) * 4;
        kv[i] = *(const dl_v4f *) (kb + min(t, nt - 1) * a.k_nb2 + 4 * min(n, a.K - 4));
    }
    const int tq = 16 * wave + l16;
#pragma unroll
    for (int k = 0; k < KB; k++) qr[k] = *(const dl_v4f *) (qb + min(tq, nt - 1) * a.q_nb2 + 4 * min(16 * k + 4 * lg, a.K - 4));
    // a head's gates and betas, a token a lane
    const int tg = min(lane, nt - 1);
    auto gate = [&](int h) { return *(const float *) (a.g + h * a.g_nb1 + (t0 + tg) * a.g_nb2 + s * a.g_nb3); };
    auto beta = [&](int h) { return *(const float *) (a.beta + h * a.b_nb1 + (t0 + tg) * a.b_nb2 + s * a.b_nb3); };
    float next_g = gate(hk), next_b = beta(hk);
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int e = tid + 256 * i, t = e / (NP / 4), n = e % (NP / 4) * 4;
        if (t >= nt || n >= a.K) kv[i] = dl_v4f{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; j++) bad |= dl_past(kv[i][j], kDlRaw);
        *(dl_v4f *) &s_k[t][n] = kv[i];
    }
    {
        float sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int k = 0; k < KB; k++) {
            if (tq >= nt || 16 * k + 4 * lg >= a.K) qr[k] = dl_v4f{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) bad |= dl_past(qr[k][j], kDlRaw), sum = fmaf(qr[k][j], qr[k][j], sum), most = fmaxf(most, fabsf(qr[k][j]));
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        const float f = a.q_eps < 0.0f ? 1.0f : 1.0f / fmaxf(sqrtf(sum), a.q_eps);
        most *= f;
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        bad |= dl_past(most, kDlRow) || (most > 0.0f && most < kDlLeastQ);
        const float sc = dl_pow2(13 - dl_exponent(most));
        dl_u4 * o = (dl_u4 *) (krec + dl_krec<NP>::q) + wave * (KB / 2) * 128 + lane;
#pragma unroll
        for (int k = 0; k < KB; k += 2) {
            qr[k] *= f, qr[k + 1] *= f;
            const dl_split x = dl_split8(qr[k] * sc, qr[k + 1] * sc);
            o[64 * k] = x.v[0], o[64 * k + 64] = x.v[1];
        }
        if (lg == 0) s_qexp[tq] = sc;
    }
    __syncthreads();
    {
        // k's lengths: four threads a row
        const int t = tid >> 2, n0 = (tid & 3) * (NP / 4);
        float sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int n = 0; n < NP / 4; n += 4) {
            const dl_v4f v = *(const dl_v4f *) &s_k[t][n0 + n];
#pragma unroll
            for (int e = 0; e < 4; e++) sum = fmaf(v[e], v[e], sum), most = fmaxf(most, fabsf(v[e]));
        }
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        const float f = a.k_eps < 0.0f ? 1.0f : 1.0f / fmaxf(sqrtf(sum), a.k_eps);
#pragma unroll
        for (int n = 0; n < NP / 4; n += 4) {
            dl_v4f v = *(const dl_v4f *) &s_k[t][n0 + n];
            v *= f;
            *(dl_v4f *) &s_k[t][n0 + n] = v;
        }
        most *= f;
        most = fmaxf(most, __shfl_xor(most, 1));
        most = fmaxf(most, __shfl_xor(most, 2));
        bad |= dl_past(most, kDlRow) || (most > 0.0f && most < kDlLeastK);
        // (a row of zeros is scaled as the shortest keys are: `left` of a chunk of such rows
        // alone has its largest element in a divisor of k_delta_chunks)
        if ((tid & 3) == 0) s_kexp[t] = dl_pow2(13 - max(dl_exponent(most), kDlLeastKExp));
    }
    bad = __syncthreads_or(bad);
    {
        // K's rows and K^T
        const float sc = s_kexp[tq];
        dl_u4 * o = (dl_u4 *) (krec + dl_krec<NP>::k) + wave * (KB / 2) * 128 + lane;
#pragma unroll
        for (int k = 0; k < KB; k += 2) {
            const dl_split x = dl_split8(*(const dl_v4f *) &s_k[tq][16 * k + 4 * lg] * sc, *(const dl_v4f *) &s_k[tq][16 * k + 16 + 4 * lg] * sc);
            o[64 * k] = x.v[0], o[64 * k + 64] = x.v[1];
        }
        o = (dl_u4 *) (krec + dl_krec<NP>::kt) + lane;
#pragma unroll 2
        for (int i = wave; i < 2 * KB; i += 4) {
            const int t = 32 * (i & 1) + 4 * lg;
            const float * x = &s_k[t][16 * (i >> 1) + l16];
            const dl_v4f s0 = *(const dl_v4f *) &s_kexp[t], s1 = *(const dl_v4f *) &s_kexp[t + 16];
            const dl_split z = dl_split8(dl_v4f{x[0], x[kRow], x[2 * kRow], x[3 * kRow]} * s0,
                                         dl_v4f{x[16 * kRow], x[17 * kRow], x[18 * kRow], x[19 * kRow]} * s1);
            o[128 * i] = z.v[0], o[128 * i + 64] = z.v[1];
        }
    }
    // k_s . q_t for the wave's t, k_s . k_t for those of wave 3 - w: rows s, columns t, five blocks a wave
    const int tk = 3 - wave;
    dl_v4f kq[4], kk[4];
#pragma unroll
    for (int sb = 0; sb < 4; sb++) {
        kq[sb] = kk[sb] = dl_v4f{0, 0, 0, 0};
        if (sb <= wave) {
#pragma unroll
            for (int k = 0; k < KB; k++) kq[sb] = dl_mfma(*(const dl_v4f *) &s_k[16 * sb + l16][16 * k + 4 * lg], qr[k], kq[sb]);
        }
        if (sb <= tk) {
#pragma unroll
            for (int k = 0; k < KB; k++)
                kk[sb] = dl_mfma(*(const dl_v4f *) &s_k[16 * sb + l16][16 * k + 4 * lg], *(const dl_v4f *) &s_k[16 * tk + l16][16 * k + 4 * lg], kk[sb]);
        }
    }
    // the wave's rows of a matrix over the chunk's tokens, split
    auto put_rows = [&](dl_u4 * o, const dl_v4f (&v)[4], float sc) {
#pragma unroll
        for (int m = 0; m < 2; m++) {
            if (2 * m > wave) continue;
            const dl_split x = dl_split8(v[2 * m] * sc, v[2 * m + 1] * sc);
            o[(2 * wave + m) * 128 + lane] = x.v[0], o[(2 * wave + m) * 128 + 64 + lane] = x.v[1];
        }
    };
    for (int h = hk; h < a.heads; h += a.key_heads) {
        char * rec = q.rec + (((int64_t) s * a.heads + h) * q.chunks + c) * dl_rec::size;
        bool own_bad = bad;
        const float g = lane < nt ? next_g : 0.0f, b = lane < nt ? next_b : 0.0f;
        const int more = min(h + a.key_heads, a.heads - 1);
        next_g = gate(more), next_b = beta(more);
        if (wave == 0) {
            // the decays: their base 2 logarithms summed in f64 (from -1000 on a power is zero)
            own_bad |= !(g <= 0.0f) || dl_past(b, kDlBeta);
            double cum = fmax((double) g, -1000.0) * 1.4426950408889634074;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double v = __shfl_up(cum, o);
                if (lane >= o) cum += v;
            }
            const double all = __shfl(cum, 63);
            const float e = __builtin_amdgcn_exp2f((float) cum);
            const float kinv = 1.0f / s_kexp[lane];
            float most = kinv;  // (the last token's decay is one)
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
            s_cum[lane] = cum;
            s_beta[lane] = b;
            ((float *) (rec + dl_rec::ks))[lane] = b * e * kinv;
            ((float *) (rec + dl_rec::beta))[lane] = b;
            ((float *) (rec + dl_rec::left))[lane] = __builtin_amdgcn_exp2f((float) (all - cum)) * (kinv / most);
            if (lane == 0) ((float *) (rec + dl_rec::end))[0] = __builtin_amdgcn_exp2f((float) all), ((float *) (rec + dl_rec::end))[1] = most;
        }
        __syncthreads();
        {
            const int t = 16 * wave + l16, u = 16 * tk + l16;
            const double ct = s_cum[t], cu = s_cum[u];
            const float bu = s_beta[u];
            dl_v4f v[4];
            float most = 0.0f;
#pragma unroll
            for (int sb = 0; sb < 4; sb++) {
                dl_v4f w;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int ss = 16 * sb + 4 * lg + e;
                    const double cs = s_cum[ss];
                    v[sb][e] = ss <= t ? kq[sb][e] * a.scale * __builtin_amdgcn_exp2f((float) (ct - cs)) : 0.0f;
                    w[e] = ss < u ? kk[sb][e] * bu * __builtin_amdgcn_exp2f((float) (cu - cs)) : 0.0f;
                    most = fmaxf(most, fabsf(v[sb][e]));
                }
                if (sb <= tk) s_a[dl_pair(tk, sb)][lane] = w;
                if (sb == tk) *(dl_v4f *) &s_d[tk][l16][4 * lg] = w;
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float sc = dl_pow2(13 - max(dl_exponent(most), -60));  // (Y is made in this scale: no larger one)
            put_rows((dl_u4 *) (rec + dl_rec::p), v, sc);
            if (lg == 0) {
                ((float *) (rec + dl_rec::in))[t] = __builtin_amdgcn_exp2f((float) ct) * a.scale * (sc / s_qexp[t]);
                ((float *) (rec + dl_rec::y))[t] = 1.0f / sc;
            }
        }
        __syncthreads();
        if (wave == 0) {
            // column l16 of the inverse of diagonal block lg
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                dl_v4f v = {i == l16 ? 1.0f : 0.0f, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < i; j += 4) {
                    const dl_v4f r = *(const dl_v4f *) &s_d[lg][i][j];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (j + e < i) v[e] = fmaf(-r[e], x[j + e], v[e]);
                }
                x[i] = (v[0] + v[1]) + (v[2] + v[3]);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) s_d[lg][i][l16] = x[i];  // (every read of the block came before: one wave)
        }
        __syncthreads();
        // T's columns of the wave's token block: x_b = inv_b (1 - A_b. x)
        dl_v4f inv[4], off[6], x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) inv[i] = *(const dl_v4f *) &s_d[i][l16][4 * lg];
#pragma unroll
        for (int i = 1; i < 4; i++)
#pragma unroll
            for (int e = 0; e < i; e++) off[i * (i - 1) / 2 + e] = -s_a[dl_pair(i, e)][lane];
        __syncthreads();  // (s_t lies over s_a)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = dl_v4f{0, 0, 0, 0};
            if (i < wave) continue;
            dl_v4f r;
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = i == wave && 4 * lg + e == l16 ? 1.0f : 0.0f;
#pragma unroll
            for (int e = 0; e < i; e++)
                if (e >= wave) r = dl_mfma(off[i * (i - 1) / 2 + e], x[e], r);
            x[i] = dl_mfma(inv[i], r, dl_v4f{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s_t[16 * i + 4 * lg + e][16 * wave + l16] = x[i][e];
            }
        }
        __syncthreads();
        {
            dl_v4f v[4];
            float most = 0.0f, sum = 0.0f;
#pragma unroll
            for (int sb = 0; sb < 4; sb++) {
                v[sb] = dl_v4f{0, 0, 0, 0};
                if (sb <= wave) v[sb] = *(const dl_v4f *) &s_t[16 * wave + l16][16 * sb + 4 * lg];
#pragma unroll
                for (int e = 0; e < 4; e++) most = fmaxf(most, fabsf(v[sb][e])), sum += fabsf(v[sb][e]);
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            own_bad |= dl_past(sum, kDlRowSum);
            const float sc = dl_pow2(13 - dl_exponent(most));
            put_rows((dl_u4 *) (rec + dl_rec::t), v, sc);
            if (lg == 0) ((float *) (rec + dl_rec::t_row))[16 * wave + l16] = 1.0f / sc;
        }
        own_bad = __syncthreads_or(own_bad);  // (and the next head's A lies over it)
        if (tid == 0) ((int *) (rec + dl_rec::end))[2] = own_bad;
    }
}

// Eight waves. Wave w < 4 makes the token block w's rows of K S0 and so of beta V
// - beta e^a K S0, the others those of Q S0; all make D's (token block w % 4, for
// a half of the columns where there are two), then wave w the state's rows 16 w
// .. (and 16 (w + 8) .. for keys past 128), and the last four Y.
template <int NP, int NC>
__global__ __launch_bounds__(512, 2) void k_delta_chunks(dl_chunk_args q) {
    constexpr int KB = NP / 16, KS = NP / 32, NS = (KB + 7) / 8;
    __shared__ dl_u4 s_s[KS][2][NC][64], s_r[2][2][NC][64], s_d[2][2][NC][64], s_ds[2][2][NC][64];  // S0, T's operand, D, D for the state
    __shared__ float s_red[2][8][16];
    __shared__ uint32_t s_most[2][NC][16];  // a column's largest |value| of the state and of v at a chunk's start (its bits)
    __shared__ int s_past[2], s_late[2];  // a chunk whose S0, or whose D, leaves f16's range
    const delta_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
    // workgroups of one head on one XCD: they read the same records
    const int n_blk = (int) gridDim.x;
    int b = (int) blockIdx.x;
    if (n_blk % 8 == 0) b = (b % 8) * (n_blk / 8) + b / 8;
    const int vb = b % q.cols, h = b / q.cols % a.heads, s = b / q.cols / a.heads, hk = h % a.key_heads;
    const int col0 = 16 * NC * vb + l16, tb = wave & 3;
    const bool keys = wave < 4;
    const char * rec0 = q.rec + ((int64_t) s * a.heads + h) * q.chunks * dl_rec::size;
    const char * krec0 = q.krec + ((int64_t) s * a.key_heads + hk) * q.chunks * dl_krec<NP>::size;
    const char * kp = a.k + hk * a.k_nb1 + s * a.k_nb3;
    const char * qp = a.q + hk * a.q_nb1 + s * a.q_nb3;
    const char * vp = a.v + h * a.v_nb1 + s * a.v_nb3;

    dl_v4f st[NS][NC];  // rows 16 (w + 8 n) + 4 lg .., column 16 cb + l16
#pragma unroll
    for (int n = 0; n < NS; n++)
#pragma unroll
        for (int cb = 0; cb < NC; cb++) {
            const int d = 16 * (wave + 8 * n) + 4 * lg, col = col0 + 16 * cb;
            st[n][cb] = dl_v4f{0, 0, 0, 0};
            if (col < a.V && d < a.K) st[n][cb] = *(const dl_v4f *) (q.s_in + s * q.s_in_nb3 + 4 * (((int64_t) h * a.V + col) * a.K + d));
        }
    if (tid < 2) s_past[tid] = s_late[tid] = 0;
    if (tid < 2 * NC * 16) (&s_most[0][0][0])[tid] = 0;

    // A chunk's operands. Each is loaded for the next chunk as soon as its
    // registers are free (two sets would spill), and by all waves alike: a
    // branch's loads would be waited for.
    dl_split rows[KS], t[2], kt[NS][2], p[2];
    dl_v4f f, beta, v[NC], t_row, left, y_row;
    float end, left_most;
    int bad;
    // (a lane's byte offsets in v, of its four tokens and its columns: 32 bits, the rest uniform)
    uint32_t v_tok[4], v_col[NC];
#pragma unroll
    for (int cb = 0; cb < NC; cb++) v_col[cb] = 4u * (uint32_t) min(col0 + 16 * cb, a.V - 1);
    auto v_tokens = [&](int last) {
#pragma unroll
        for (int e = 0; e < 4; e++) v_tok[e] = (uint32_t) min(16 * tb + 4 * lg + e, last) * (uint32_t) a.v_nb2;
    };
    v_tokens(kDlC - 1);
    auto load_rows = [&](int64_t c) {
        const char * rec = rec0 + c * dl_rec::size;
        const int64_t t0 = (q.c0 + c) * kDlC;
        if (t0 + kDlC > a.tokens) v_tokens((int) (a.tokens - t0) - 1);
        const dl_u4 * row = (const dl_u4 *) (krec0 + c * dl_krec<NP>::size + (keys ? dl_krec<NP>::k : dl_krec<NP>::q)) + tb * KS * 128 + lane;
#pragma unroll
        for (int k = 0; k < KS; k++) rows[k].v[0] = row[128 * k], rows[k].v[1] = row[128 * k + 64];
        const char * of_rows = rec + 4 * (16 * tb + 4 * lg);
        f = *(const dl_v4f *) (of_rows + (keys ? dl_rec::ks : dl_rec::in));
        beta = *(const dl_v4f *) (of_rows + dl_rec::beta);
        const char * vt = vp + t0 * a.v_nb2;
#pragma unroll
        for (int cb = 0; cb < NC; cb++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[cb][e] = *(const float *) (vt + (v_tok[e] + v_col[cb]));
        // (by vector loads: a wait for LDS would wait for scalar ones)
        bad = ((const int *) (rec + dl_rec::end))[2 + (lane >> 6)];
    };
    auto load_t = [&](int64_t c) {
        const char * rec = rec0 + c * dl_rec::size;
        const dl_u4 * x = (const dl_u4 *) (rec + dl_rec::t) + tb * 256 + lane;
#pragma unroll
        for (int m = 0; m < 2; m++) t[m].v[0] = x[128 * min(m, tb / 2)], t[m].v[1] = x[128 * min(m, tb / 2) + 64];
        t_row = *(const dl_v4f *) (rec + 4 * (16 * tb + 4 * lg) + dl_rec::t_row);
        left = *(const dl_v4f *) (rec + 4 * (16 * tb + 4 * lg) + dl_rec::left);
    };
    auto load_kt = [&](int64_t c) {
        const char * rec = rec0 + c * dl_rec::size;
        const dl_u4 * k = (const dl_u4 *) (krec0 + c * dl_krec<NP>::size + dl_krec<NP>::kt) + lane;
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int m = 0; m < 2; m++) {
                const int at = 128 * (2 * min(wave + 8 * n, KB - 1) + m);
                kt[n][m].v[0] = k[at], kt[n][m].v[1] = k[at + 64];
            }
        const dl_u4 * x = (const dl_u4 *) (rec + dl_rec::p) + tb * 256 + lane;
#pragma unroll
        for (int m = 0; m < 2; m++) p[m].v[0] = x[128 * min(m, tb / 2)], p[m].v[1] = x[128 * min(m, tb / 2) + 64];
        y_row = *(const dl_v4f *) (rec + 4 * (16 * tb + 4 * lg) + dl_rec::y);
        end = ((const float *) (rec + dl_rec::end))[lane >> 6];
        left_most = ((const float *) (rec + dl_rec::end))[1 + (lane >> 6)];
    };
    // a result's four rows as the half of a lane's eight k
    auto put = [&](dl_u4 (&to)[2][NC][64], int cb, int half, dl_v4f v) {
        uint32_t x[2], y[2];
        dl_split2(v[0], v[1], x[0], y[0]);
        dl_split2(v[2], v[3], x[1], y[1]);
        ((dl_u2 *) &to[0][cb][lane])[half] = dl_u2{x[0], x[1]};
        ((dl_u2 *) &to[1][cb][lane])[half] = dl_u2{y[0], y[1]};
    };
    auto get = [&](const dl_u4 (&from)[2][NC][64], int cb) { return dl_split{{from[0][cb][lane], from[1][cb][lane]}}; };
    // whether a scaled result might leave f16's range (or is not finite)
    auto past = [](dl_v4f v, float limit) { return dl_past((fabsf(v[0]) + fabsf(v[1])) + (fabsf(v[2]) + fabsf(v[3])), limit); };
    auto put_most = [&](int slot) {
#pragma unroll
        for (int cb = 0; cb < NC; cb++) {
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                m = fmaxf(m, fabsf(v[cb][e]));
#pragma unroll
                for (int n = 0; n < NS; n++)
                    if (wave + 8 * n < KB) m = fmaxf(m, fabsf(st[n][cb][e]));
            }
            m = dl_max4(m);
            if (lg == 0) atomicMax(&s_most[slot][cb][l16], __float_as_uint(m));
        }
    };
    // token by token, for chunks the products cannot take
    auto tokens = [&](int64_t t0) {
        const int nt = (int) min((int64_t) kDlC, a.tokens - t0);
        for (int t = 0; t < nt; t++) {
            const int64_t tt = t0 + t;
            const float * k = (const float *) (kp + tt * a.k_nb2);
            const float * qr = (const float *) (qp + tt * a.q_nb2);
            auto length = [&](const float * x, float eps) {
                if (eps < 0.0f) return 1.0f;
                double sum = 0.0;
                for (int i = lane; i < a.K; i += 64) sum += (double) x[i] * (double) x[i];
                return 1.0f / fmaxf((float) sqrt(wave_sum_d(sum)), eps);
            };
            const float kl = length(k, a.k_eps), ql = length(qr, a.q_eps) * a.scale;
            const float eg = expf(*(const float *) (a.g + h * a.g_nb1 + tt * a.g_nb2 + s * a.g_nb3));
            const float bt = *(const float *) (a.beta + h * a.b_nb1 + tt * a.b_nb2 + s * a.b_nb3);
#pragma unroll
            for (int cb = 0; cb < NC; cb++) {
                const int col = col0 + 16 * cb;
                const float vt = col < a.V ? ((const float *) (vp + tt * a.v_nb2))[col] : 0.0f;
                float dot = 0.0f, y = 0.0f;
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int d = 16 * (wave + 8 * n) + 4 * lg + e;
                        st[n][cb][e] = d < a.K ? st[n][cb][e] * eg : 0.0f;
                        if (d < a.K) dot = fmaf(st[n][cb][e], k[d] * kl, dot);
                    }
                dot += __shfl_xor(dot, 16);
                dot += __shfl_xor(dot, 32);
                if (lg == 0) s_red[0][wave][l16] = dot;
                __syncthreads();
                dot = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; w++) dot += s_red[0][w][l16];
                const float d = bt * (vt - dot);
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = 16 * (wave + 8 * n) + 4 * lg + e;
                        if (i < a.K) {
                            st[n][cb][e] = fmaf(k[i] * kl, d, st[n][cb][e]);
                            y = fmaf(st[n][cb][e], qr[i] * ql, y);
                        }
                    }
                y += __shfl_xor(y, 16);
                y += __shfl_xor(y, 32);
                if (lg == 0) s_red[1][wave][l16] = y;
                __syncthreads();
                if (tid < 16 && col < a.V) {
                    y = 0.0f;
#pragma unroll
                    for (int w = 0; w < 8; w++) y += s_red[1][w][l16];
                    a.y[((s * a.tokens + tt) * a.heads + h) * a.V + col] = y;
                }
                __syncthreads();
            }
        }
    };
    if (q.chunks > 0) load_rows(0), load_t(0), load_kt(0);
    __syncthreads();
    int size[NC], now[NC];  // log2 of a column's largest of the state and v: a chunk before, and in this one
#pragma unroll
    for (int cb = 0; cb < NC; cb++) size[cb] = 0;
    auto put_state = [&]() {  // S0, in its columns' scales; whether all of it is finite
        bool odd = false;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const int kb = wave + 8 * n;
            if (kb < KB) {
#pragma unroll
                for (int cb = 0; cb < NC; cb++) {
                    put(s_s[kb >> 1], cb, kb & 1, st[n][cb] * dl_pow2(5 - size[cb]));
                    odd |= past(st[n][cb], 0x1p120f);
                }
            }
        }
        return !odd;
    };
    for (int64_t c = 0; c < q.chunks; c++) {
        const int64_t t0 = (q.c0 + c) * kDlC, more = min(c + 1, q.chunks - 1);
        put_most(c & 1);
        if (!put_state()) s_past[c & 1] = 1;
        __syncthreads();
        // (the reads of LDS ahead of the products, half of them where there are many)
        constexpr int kReads = KS * NC > 8 ? 2 : KS > 4 ? KS / 2 : KS;
        dl_split x[kReads][NC];
        auto read_state = [&](int k0) {
#pragma unroll
            for (int k = 0; k < kReads; k++)
#pragma unroll
                for (int cb = 0; cb < NC; cb++) x[k][cb] = get(s_s[k0 + k], cb);
            __builtin_amdgcn_sched_barrier(0);
        };
        read_state(0);
        bool other = false, large = false;
#pragma unroll
        for (int cb = 0; cb < NC; cb++) {
            now[cb] = dl_exponent(__uint_as_float(s_most[c & 1][cb][l16]));
            other |= now[cb] > size[cb] + 9 || now[cb] < size[cb] - 6, large |= now[cb] > 40;
        }
        const bool by_token = __builtin_amdgcn_readfirstlane(bad) || s_past[c & 1] || __any(large);
        if (tid == 0) s_past[(c + 1) & 1] = s_late[(c + 1) & 1] = 0;
        if (tid < NC * 16) (&s_most[(c + 1) & 1][0][0])[tid] = 0;
        dl_sum sum[NC];
        dl_v4f acc[NC];
        if (by_token) goto one_by_one;
        if (__any(other)) {  // (every wave holds all columns: they agree)
            __syncthreads();
#pragma unroll
            for (int cb = 0; cb < NC; cb++) size[cb] = now[cb];
            put_state();
            __syncthreads();
            read_state(0);
        }
#pragma unroll
        for (int cb = 0; cb < NC; cb++) sum[cb].hi = sum[cb].lo = dl_v4f{0, 0, 0, 0};
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += kReads) {
            if (k0 > 0) read_state(k0);
#pragma unroll
            for (int k = 0; k < kReads; k++)
#pragma unroll
                for (int i = 0; i < 3; i++)
#pragma unroll
                    for (int cb = 0; cb < NC; cb++) dl_product(i, rows[k0 + k], x[k][cb], sum[cb]);
        }
#pragma unroll
        for (int cb = 0; cb < NC; cb++) {
            acc[cb] = dl_whole(sum[cb]) * (f * dl_pow2(size[cb] - 5));
            size[cb] = now[cb];
            if (keys) {
                const dl_v4f x = (v[cb] * beta - acc[cb]) * dl_pow2(8 - size[cb]);
                put(s_r[tb >> 1], cb, tb & 1, x);
                large |= past(x, kDlHalf);
            }
        }
        if (large) s_late[c & 1] = 1;
        load_rows(more);
        __syncthreads();
        {
            // D, in the scale 2^(6 - size): a token block, half of the columns (one column block: the first waves)
            const int half = NC == 2 ? wave >> 2 : 0;
            if (NC == 2 || keys) {
                dl_sum z = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    if (2 * m > tb) continue;
                    const dl_split x = get(s_r[m], half);
#pragma unroll
                    for (int i = 0; i < 3; i++) dl_product(i, t[m], x, z);
                }
                const dl_v4f d = dl_whole(z) * (t_row * 0.25f);
                put(s_d[tb >> 1], half, tb & 1, d);
                put(s_ds[tb >> 1], half, tb & 1, d * left);
                if (past(d, kDlHalf)) s_late[c & 1] = 1;
            }
        }
        load_t(more);
        __syncthreads();
        if (s_late[c & 1]) goto one_by_one;
        {
            dl_split z[2][NC];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int cb = 0; cb < NC; cb++) z[m][cb] = get(s_ds[m], cb);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NS; n++) {
                // the state in D's scale, and back (left_most is 2^-20 to 2^-3: the factor of end 2^-37 to 2^126)
#pragma unroll
                for (int cb = 0; cb < NC; cb++) sum[cb].hi = st[n][cb] * (end * (dl_pow2(6 - size[cb]) / left_most)), sum[cb].lo = dl_v4f{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < 2; m++) {
#pragma unroll
                    for (int i = 0; i < 3; i++)
#pragma unroll
                        for (int cb = 0; cb < NC; cb++) dl_product(i, kt[n][m], z[m][cb], sum[cb]);
                }
#pragma unroll
                for (int cb = 0; cb < NC; cb++) st[n][cb] = dl_whole(sum[cb]) * (left_most * dl_pow2(size[cb] - 6));
            }
            if (!keys) {
#pragma unroll
                for (int cb = 0; cb < NC; cb++) sum[cb].hi = acc[cb] * dl_pow2(6 - size[cb]), sum[cb].lo = dl_v4f{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    if (2 * m > tb) continue;
                    dl_split x[NC];
#pragma unroll
                    for (int cb = 0; cb < NC; cb++) x[cb] = get(s_d[m], cb);
#pragma unroll
                    for (int i = 0; i < 3; i++)
#pragma unroll
                        for (int cb = 0; cb < NC; cb++) dl_product(i, p[m], x[cb], sum[cb]);
                }
                // (in two steps: y_row's inverse may be 2^73, the state's scale 2^106)
#pragma unroll
                for (int cb = 0; cb < NC; cb++) acc[cb] = dl_whole(sum[cb]) * dl_pow2(size[cb] - 6);
                char * y = (char *) (a.y + ((s * a.tokens + t0) * a.heads + h) * a.V);
                const uint32_t y_nb = 4u * (uint32_t) a.heads * (uint32_t) a.V, at = (uint32_t) (16 * tb + 4 * lg) * y_nb + 4u * (uint32_t) col0;
                const int left_over = (int) min((int64_t) kDlC, a.tokens - t0) - 16 * tb - 4 * lg;
#pragma unroll
                for (int cb = 0; cb < NC; cb++) {
                    if (col0 + 16 * cb >= a.V) continue;
                    if (left_over >= 4) {
#pragma unroll
                        for (int e = 0; e < 4; e++) *(float *) (y + (int64_t) e * y_nb + (at + 64 * cb)) = acc[cb][e] * y_row[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 3; e++)
                            if (e < left_over) *(float *) (y + (int64_t) e * y_nb + (at + 64 * cb)) = acc[cb][e] * y_row[e];
                    }
                }
            }
            load_kt(more);
            continue;
        }
    one_by_one:
        tokens(t0);
        load_rows(more), load_t(more), load_kt(more);
    }
#pragma unroll
    for (int n = 0; n < NS; n++)
#pragma unroll
        for (int cb = 0; cb < NC; cb++) {
            const int d = 16 * (wave + 8 * n) + 4 * lg, col = col0 + 16 * cb;
            if (col < a.V && d < a.K) *(dl_v4f *) (a.out + s * a.out_nb3 + 4 * (((int64_t) h * a.V + col) * a.K + d)) = st[n][cb];
        }
}

// ------------------------------------------------------------- launches ---

bool delta_supported(int64_t K) { return K >= 1 && K <= 256; }

static int dl_np(const delta_args & a) { return a.K <= 64 ? 64 : a.K <= 96 ? 96 : a.K <= 128 ? 128 : 256; }
// of the records of one chunk of all heads
static int64_t dl_chunk_size(const delta_args & a) {
    return ((int64_t) dl_rec::size * a.heads + 12 * kDlC * (int64_t) dl_np(a) * a.key_heads) * a.seqs;
}
// Chunks of one slab, whose records lie in scratch: the two launches take turns.
// 4096 tokens of 32 heads of 128 x 128 (2.7 MB a chunk), us of the launches by MB of
// scratch: 40 350, 60 312, 96 290, 200 298.
static int64_t dl_slab(const delta_args & a) {
    const int64_t chunks = (a.tokens + kDlC - 1) / kDlC, one = dl_chunk_size(a);
    const int64_t fit = std::max<int64_t>(1, a.scratch_bytes / one), slabs = (chunks + fit - 1) / fit;
    return (chunks + slabs - 1) / slabs;
}
static bool dl_vec(const delta_args & a) {
    const uintptr_t al = (uintptr_t) a.q | (uintptr_t) a.k | (uintptr_t) a.s | (uintptr_t) a.out | (uintptr_t) a.q_nb1 |
                         (uintptr_t) a.q_nb2 | (uintptr_t) a.q_nb3 | (uintptr_t) a.k_nb1 | (uintptr_t) a.k_nb2 |
                         (uintptr_t) a.k_nb3 | (uintptr_t) a.s_nb3 | (uintptr_t) a.out_nb3 | (uintptr_t) (4 * a.K) |
                         (a.g_elem ? (uintptr_t) a.g | (uintptr_t) a.g_nb1 | (uintptr_t) a.g_nb2 | (uintptr_t) a.g_nb3 : 0);
    return al % 16 == 0;
}
// chunks: a gate a head, and tokens enough for the products to pay. us of rows and of
// chunks, which take the same from 24 to 64 tokens: 32 heads of 128, one sequence, 24
// tokens 19.5 / 29.9, 40 29.0 / 30.0, 64 43 / 30; 16 of them, 24 63 / 90, 40 97 / 93, 64
// 150 / 96; three of 12 heads of 64 x 96, 24 15.6 / 19.6, 32 20.8 / 19.7: they meet at 30
// to 40 tokens, above this border
static bool dl_chunked(const delta_args & a) {
    return !a.g_elem && a.tokens >= 24 && a.K >= 16 && dl_vec(a) &&
           a.v_nb2 >= 0 && a.v_nb2 < 1 << 25 && (int64_t) a.heads * a.V < 1 << 23;  // (a lane's rows of v and y in 32-bit offsets)
}

// k_delta_ready's tokens a slab; 0: it is not worth its launch, or has no room. us without
// and with it, heads of 128: one sequence of 16 heads, 8 tokens 10.0 / 10.2, 16 16.5 / 11.8,
// 31 28.4 / 14.6; eight of 32 heads, 24 tokens 48.6 / 52.0, 31 60.3 / 58.6
static int dl_pieces(const delta_args & a) { return a.K <= 64 ? 1 : a.K <= 128 ? 2 : 4; }  // of 64 elements a row
static int64_t dl_ready_bytes(const delta_args & a) { return 256ll * dl_pieces(a) * (2 * a.key_heads + a.heads) * a.seqs; }
static int64_t dl_ready_slab(const delta_args & a) {
    if (!a.g_elem || a.tokens < kDlReady) return 0;
    const int64_t room = std::min(kDeltaScratch, a.scratch_bytes) / dl_ready_bytes(a);
    return room < kDlReady ? 0 : std::min(room, a.tokens);
}

size_t delta_scratch_bytes(const delta_args & a, int n_cu) {
    (void) n_cu;
    if (a.seqs == 0 || a.heads == 0 || a.V == 0) return 0;
    // (a graph planned before it is allocated: the addresses may still allow chunks)
    if (a.g_elem) return (size_t) (dl_ready_slab(a) * dl_ready_bytes(a));
    if (a.tokens < 24 || a.K < 16) return 0;
    return (size_t) (dl_slab(a) * dl_chunk_size(a));
}

template <int NP>
static void launch_delta_chunks(const delta_args & a, void * scratch, hipStream_t s, int n_cu) {
    dl_chunk_args q{};
    q.a = a;
    q.rec = (char *) scratch;
    // 32 columns a workgroup halve what is read of the records, but a chunk takes
    // longer: where these fill the CUs. us of 16 / 32 columns, 1000 tokens of 32 heads
    // of 128 x 128 82 / 96, of 64 143 / 108. (Where 32 columns do not fill the CUs and 16
    // take two rounds of workgroups, these are the better too, 40 heads 138 / 104, and not taken)
    const bool wide = (int64_t) ((a.V + 31) / 32) * a.heads * a.seqs >= n_cu;
    q.cols = wide ? (a.V + 31) / 32 : (a.V + 15) / 16;
    q.s_in = a.s, q.s_in_nb3 = a.s_nb3;
    const int64_t chunks = (a.tokens + kDlC - 1) / kDlC, slab = dl_slab(a);
    q.krec = q.rec + slab * dl_rec::size * a.heads * a.seqs;
    for (q.c0 = 0; q.c0 < chunks; q.c0 += slab) {
        q.chunks = std::min(slab, chunks - q.c0);
        hipLaunchKernelGGL(k_delta_solve<NP>, dim3((unsigned) (q.chunks * a.key_heads * a.seqs)), dim3(256), 0, s, q);
        note_hip_error(hipGetLastError());
        const dim3 grid((unsigned) ((int64_t) q.cols * a.heads * a.seqs));
        if (wide) hipLaunchKernelGGL((k_delta_chunks<NP, 2>), grid, dim3(512), 0, s, q);
        else hipLaunchKernelGGL((k_delta_chunks<NP, 1>), grid, dim3(512), 0, s, q);
        note_hip_error(hipGetLastError());
        q.s_in = a.out, q.s_in_nb3 = a.out_nb3;
    }
}

template <int P, int U, bool VEC>
static void launch_delta_rows(const delta_args & a, hipStream_t s) {
    const int64_t units = (int64_t) ((a.V + 4 * U - 1) / (4 * U)) * a.heads * a.seqs;
    const dim3 grid((unsigned) ((units + 3) / 4));
    if (a.g_elem) hipLaunchKernelGGL((k_delta_rows<P, U, VEC, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_delta_rows<P, U, VEC, false>), grid, dim3(256), 0, s, a);
    note_hip_error(hipGetLastError());
}

// gates an element, many tokens: slabs of k_delta_ready's rows, the state handed on.
// us of U = 1 / 2, 500 tokens of 16 heads of 128 x 128: one sequence 113 / 145, two 146 /
// 156, four 218 / 164, eight 428 / 325
template <int P, int U>
static void launch_delta_ready(const delta_args & a, void * scratch, hipStream_t s) {
    const int64_t slab = dl_ready_slab(a);
    delta_args b = a;
    for (int64_t t0 = 0; t0 < a.tokens; t0 += slab) {
        b.q = a.q + t0 * a.q_nb2, b.k = a.k + t0 * a.k_nb2, b.g = a.g + t0 * a.g_nb2;
        b.tokens = std::min(slab, a.tokens - t0);
        const int64_t rows = b.tokens * (2 * a.key_heads + a.heads) * a.seqs;
        hipLaunchKernelGGL(k_delta_ready<P>, dim3((unsigned) ((rows + 15) / 16)), dim3(256), 0, s, b, (float *) scratch);
        note_hip_error(hipGetLastError());
        b.v = a.v + t0 * a.v_nb2, b.beta = a.beta + t0 * a.b_nb2, b.y = a.y + t0 * a.heads * a.V;
        const int64_t units = (int64_t) ((a.V + 4 * U - 1) / (4 * U)) * a.heads * a.seqs;
        hipLaunchKernelGGL((k_delta_steps<P, U>), dim3((unsigned) units), dim3(64), 0, s, b, (const float *) scratch);
        note_hip_error(hipGetLastError());
        b.s = a.out, b.s_nb3 = a.out_nb3;
    }
}

// A wave takes 4 U rows: few where that leaves waves a SIMD, many where there
// are enough anyhow (the token's work beside the rows is shared). 32 heads of 128
// x 128, us, U = 1 / 2 / 4: 8 tokens of one sequence 7.9 / 8.7 / 11.5, of 16 37 /
// 30 / 30; one token of 48 34 / 35 / 34.
template <int P>
static void launch_delta_tokens(const delta_args & a, void * scratch, hipStream_t s, int n_cu) {
    const int64_t rows = (int64_t) a.V * a.heads * a.seqs, enough = 16 * (int64_t) n_cu;  // four waves a CU, of 4 rows
    if (dl_vec(a) && dl_ready_slab(a) > 0) {
        if (rows >= 2 * enough) launch_delta_ready<P, 2>(a, scratch, s);
        else launch_delta_ready<P, 1>(a, scratch, s);
    } else if (!dl_vec(a)) launch_delta_rows<P, 2, false>(a, s);
    else if (rows >= 4 * enough) launch_delta_rows<P, 4, true>(a, s);
    else if (rows >= 2 * enough) launch_delta_rows<P, 2, true>(a, s);
    else launch_delta_rows<P, 1, true>(a, s);
}

void launch_delta(const delta_args & args, void * scratch, hipStream_t s, int n_cu) {
    delta_args a = args;
    a.y_tokens = a.tokens;
    if (a.seqs == 0 || a.heads == 0 || a.V == 0) return;
    if (dl_chunked(a)) {
        switch (dl_np(a)) {
            case 64: launch_delta_chunks<64>(a, scratch, s, n_cu); break;
            case 96: launch_delta_chunks<96>(a, scratch, s, n_cu); break;
            case 128: launch_delta_chunks<128>(a, scratch, s, n_cu); break;
            default: launch_delta_chunks<256>(a, scratch, s, n_cu); break;
        }
        return;
    }
    if (a.K <= 64) launch_delta_tokens<1>(a, scratch, s, n_cu);
    else if (a.K <= 128) launch_delta_tokens<2>(a, scratch, s, n_cu);
    else launch_delta_tokens<4>(a, scratch, s, n_cu);
}

}  // namespace mi355x
