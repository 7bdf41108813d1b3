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

// ---------------------------------------------------------------- chunks ---
//
// Chunks of C = 64 tokens as matrix products. With a_t the sum of the chunk's g
// up to t, L_ts = e^(a_t - a_s) and
//     A = strictly lower (beta_t k_t . k_s L_ts),   (1 + A) U = beta V,   (1 + A) W = beta e^a K
// a chunk turns the state S0 it meets into
//     D = U - W S0,   Y = (e^a Q S0 + lower(Q K^T L) D) / sqrt(K),   S1 = e^(a_C) S0 + (e^(a_C - a) K)^T D
// k_delta_solve makes W, U, lower(Q K^T L) and the decays of every chunk at once
// (forward substitution by blocks of 16 tokens, whose diagonal blocks are
// inverted column by column: as stable as the recurrence), k_delta_chunks goes
// through the chunks, a workgroup a head and 16 columns of the state.
// All products are f32's, on v_mfma_f32_16x16x4f32: A lane l = row l % 16, k l /
// 16; B lane l = column l % 16, the same k; result lane l = rows 4 (l / 16) ..
// + 3, column l % 16. Step i of four takes k = 4 (l / 16) + i, so that a result's
// four elements are the next product's B operand as they are, and A's rows come
// in 16-byte pieces.
//
// A chunk whose values are not finite, whose g are above zero, or whose sizes
// could leave f32's range in the products' order, runs token by token: the
// normalised rows of q and k are at most 2^10, W 2^20, U and the state 2^60, so
// D is under 2^88, a state after under 2^113, y under 2^122.

typedef uint32_t dl_u4 __attribute__((ext_vector_type(4)));

constexpr int kDlC = 64;
constexpr float kDlRow = 0x1p10f, kDlRaw = 0x1p50f, kDlW = 0x1p20f, kDlU = 0x1p60f;

struct dl_chunk_args {
    delta_args a;
    char * rec;          // records [sequence][head][chunk of the slab]
    const char * s_in;   // the states the slab starts from
    int64_t s_in_nb3;
    int64_t c0, chunks;  // the slab's first chunk and its chunks
    int vblocks;         // 16-column blocks of the state
    int rec_size;
};
// byte offsets in a record
struct dl_rec {
    // [64] f32 each: what a row of Q S0 is multiplied by (e^a, q's length and
    // 1 / sqrt(K)); what a row of D is for the state (e^(a_C - a) and k's length)
    static constexpr int in = 0, left = 256;
    static constexpr int end = 512;   // e^(a_C); whether the chunk goes token by token
    static constexpr int bad = 516;
    static constexpr int p = 1024;    // lower(Q K^T L) / sqrt(K): blocks (tb, sb <= tb), lane = row t l % 16, s 4 (l / 16) ..
    static constexpr int w = p + 10 * 1024;  // -W [64][NP]
    // then U: [column block][token block][lane] of results
};
__device__ __forceinline__ int dl_pair(int tb, int sb) { return tb * (tb + 1) / 2 + sb; }

__device__ __forceinline__ dl_v4f dl_mfma(dl_v4f a, dl_v4f b, dl_v4f c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ bool dl_past(float v, float limit) { return !(fabsf(v) <= limit); }

template <int NP>
__global__ __launch_bounds__(256) void k_delta_solve(dl_chunk_args q) {
    constexpr int kRow = NP + 4, KB = NP / 16;
    __shared__ __align__(16) float s_k[kDlC][kRow], s_q[kDlC][kRow];
    __shared__ float s_klen[kDlC], s_qlen[kDlC], s_beta[kDlC];
    __shared__ double s_cum[kDlC];
    __shared__ dl_v4f s_a[10][64];                    // A's blocks, lane = row t l % 16, s 4 (l / 16) ..
    __shared__ __align__(16) float s_d[4][16][20];    // the diagonal ones, then their inverses, row by row
    const delta_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, lg = lane >> 4;
    const int64_t c = blockIdx.x % q.chunks;
    const int hk = (int) (blockIdx.x / q.chunks % a.key_heads), s = (int) (blockIdx.x / q.chunks / a.key_heads);
    const int64_t t0 = (q.c0 + c) * kDlC;
    const int nt = (int) min((int64_t) kDlC, a.tokens - t0);
    const char * kb = a.k + hk * a.k_nb1 + t0 * a.k_nb2 + s * a.k_nb3;
    const char * qb = a.q + hk * a.q_nb1 + t0 * a.q_nb2 + s * a.q_nb3;
    bool bad = false;
    for (int i = tid; i < kDlC * NP / 4; i += 256) {
        const int t = i / (NP / 4), n = i % (NP / 4) * 4;
        dl_v4f kv = {0, 0, 0, 0}, qv = {0, 0, 0, 0};
        if (t < nt && n < a.K) {
            kv = *(const dl_v4f *) (kb + t * a.k_nb2 + 4 * n);
            qv = *(const dl_v4f *) (qb + t * a.q_nb2 + 4 * n);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) bad |= dl_past(kv[e], kDlRaw) || dl_past(qv[e], kDlRaw);
        *(dl_v4f *) &s_k[t][n] = kv;
        *(dl_v4f *) &s_q[t][n] = qv;
    }
    __syncthreads();
    {
        // the rows' lengths: four threads a row
        const int t = tid >> 2, n0 = (tid & 3) * (NP / 4);
        auto scale = [&](float (&rows)[kDlC][kRow], float eps) {
            float sum = 0.0f, most = 0.0f;
#pragma unroll
            for (int n = 0; n < NP / 4; n += 4) {
                const dl_v4f v = *(const dl_v4f *) &rows[t][n0 + n];
#pragma unroll
                for (int e = 0; e < 4; e++) sum = fmaf(v[e], v[e], sum), most = fmaxf(most, fabsf(v[e]));
            }
            sum += __shfl_xor(sum, 1);
            sum += __shfl_xor(sum, 2);
            const float f = eps < 0.0f ? 1.0f : 1.0f / fmaxf(sqrtf(sum), eps);
            bad |= dl_past(most * f, kDlRow);
#pragma unroll
            for (int n = 0; n < NP / 4; n += 4) {
                dl_v4f v = *(const dl_v4f *) &rows[t][n0 + n];
                v *= f;
                *(dl_v4f *) &rows[t][n0 + n] = v;
            }
            return f;
        };
        const float kl = scale(s_k, a.k_eps), ql = scale(s_q, a.q_eps);
        if ((tid & 3) == 0) s_klen[t] = t < nt ? kl : 0.0f, s_qlen[t] = t < nt ? ql : 0.0f;
    }
    bad = __syncthreads_or(bad);
    // k_s . k_t and k_s . q_t: rows s, columns t, twenty blocks over the waves
    dl_v4f dots[5];
#pragma unroll
    for (int n = 0; n < 5; n++) {
        const int i = wave + 4 * n, pr = i < 10 ? i : i - 10;
        const int tb = pr < 1 ? 0 : pr < 3 ? 1 : pr < 6 ? 2 : 3, sb = pr - tb * (tb + 1) / 2;
        const float(&x)[kDlC][kRow] = i < 10 ? s_k : s_q;
        dots[n] = dl_v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KB; k++)
            dots[n] = dl_mfma(*(const dl_v4f *) &s_k[16 * sb + l16][16 * k + 4 * lg], *(const dl_v4f *) &x[16 * tb + l16][16 * k + 4 * lg], dots[n]);
    }
    for (int h = hk; h < a.heads; h += a.key_heads) {
        char * rec = q.rec + (((int64_t) s * a.heads + h) * q.chunks + c) * q.rec_size;
        bool own_bad = bad;
        if (wave == 0) {
            // the decays: their logarithms summed in f64 (from -1000 on a power is zero)
            const bool in = lane < nt;
            const float g = in ? *(const float *) (a.g + h * a.g_nb1 + (t0 + lane) * a.g_nb2 + s * a.g_nb3) : 0.0f;
            const float b = in ? *(const float *) (a.beta + h * a.b_nb1 + (t0 + lane) * a.b_nb2 + s * a.b_nb3) : 0.0f;
            own_bad |= !(g <= 0.0f) || dl_past(b, kDlRow);
            double cum = fmax((double) g, -1000.0);
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double v = __shfl_up(cum, o);
                if (lane >= o) cum += v;
            }
            const double all = __shfl(cum, 63);
            s_cum[lane] = cum;
            s_beta[lane] = b;
            ((float *) (rec + dl_rec::in))[lane] = expf((float) cum) * s_qlen[lane] * a.scale;
            ((float *) (rec + dl_rec::left))[lane] = expf((float) (all - cum)) * s_klen[lane];
            if (lane == 0) *(float *) (rec + dl_rec::end) = expf((float) all);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < 5; n++) {
            const int i = wave + 4 * n, pr = i < 10 ? i : i - 10;
            const int tb = pr < 1 ? 0 : pr < 3 ? 1 : pr < 6 ? 2 : 3, sb = pr - tb * (tb + 1) / 2;
            const int t = 16 * tb + l16;
            const double ct = s_cum[t];
            const float f = i < 10 ? s_beta[t] : a.scale;
            dl_v4f v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int ss = 16 * sb + 4 * lg + e;
                const bool in = i < 10 ? ss < t : ss <= t;
                v[e] = in ? dots[n][e] * f * expf((float) (ct - s_cum[ss])) : 0.0f;
            }
            if (i < 10) {
                s_a[pr][lane] = v;
                if (tb == sb) *(dl_v4f *) &s_d[tb][l16][4 * lg] = v;
            } else {
                ((dl_v4f *) (rec + dl_rec::p))[pr * 64 + lane] = v;
            }
        }
        __syncthreads();
        if (wave == 0) {
            // column l16 of the inverse of diagonal block lg
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v = i == l16 ? 1.0f : 0.0f;
#pragma unroll
                for (int j = 0; j < i; j += 4) {
                    const dl_v4f r = *(const dl_v4f *) &s_d[lg][i][j];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (j + e < i) v = fmaf(-r[e], x[j + e], v);
                }
                x[i] = v;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) s_d[lg][i][l16] = x[i];  // (every read of the block came before: one wave)
        }
        __syncthreads();
        dl_v4f inv[4], off[6];
#pragma unroll
        for (int b = 0; b < 4; b++) inv[b] = *(const dl_v4f *) &s_d[b][l16][4 * lg];
#pragma unroll
        for (int b = 1; b < 4; b++)
#pragma unroll
            for (int e = 0; e < b; e++) off[b * (b - 1) / 2 + e] = -s_a[dl_pair(b, e)][lane];
        const char * vb = a.v + h * a.v_nb1 + t0 * a.v_nb2 + s * a.v_nb3;
        for (int ct = wave; ct < q.vblocks + KB; ct += 4) {
            const bool is_u = ct < q.vblocks;
            const int col = 16 * (is_u ? ct : ct - q.vblocks) + l16;
            dl_v4f x[4];
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int t = 16 * b + 4 * lg + e;
                    if (is_u) {
                        const float v = t < nt && col < a.V ? ((const float *) (vb + t * a.v_nb2))[col] : 0.0f;
                        x[b][e] = v * s_beta[t];
                        own_bad |= dl_past(v, kDlU);
                    } else {
                        x[b][e] = -s_k[t][col] * s_beta[t] * expf((float) s_cum[t]);
                    }
                }
#pragma unroll
            for (int b = 0; b < 4; b++) {
                dl_v4f r = x[b];
#pragma unroll
                for (int e = 0; e < b; e++) r = dl_mfma(off[b * (b - 1) / 2 + e], x[e], r);
                x[b] = dl_mfma(inv[b], r, dl_v4f{0, 0, 0, 0});
#pragma unroll
                for (int e = 0; e < 4; e++) own_bad |= dl_past(x[b][e], is_u ? kDlU : kDlW);
            }
            if (is_u) {
                dl_v4f * u = (dl_v4f *) (rec + dl_rec::w + 4 * kDlC * NP) + (int64_t) ct * 256 + lane;
#pragma unroll
                for (int b = 0; b < 4; b++) u[64 * b] = x[b];
            } else {
                float * w = (float *) (rec + dl_rec::w) + col;
#pragma unroll
                for (int b = 0; b < 4; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++) w[(16 * b + 4 * lg + e) * NP] = x[b][e];
            }
        }
        own_bad = __syncthreads_or(own_bad);  // (and LDS has been read)
        if (tid == 0) *(int *) (rec + dl_rec::bad) = own_bad;
    }
}

// Eight waves: the first four make D's token blocks, the others Y's, and wave w
// holds the state's rows 16 w .. (and 16 (w + 8) .. for keys past 128) of the
// workgroup's 16 columns.
template <int NP>
__global__ __launch_bounds__(512, 2) void k_delta_chunks(dl_chunk_args q) {
    constexpr int KB = NP / 16, NS = (KB + 7) / 8;
    __shared__ dl_v4f s_s[KB][64], s_dy[4][64], s_ds[4][64];  // S0, D, and D for the state, as B operands
    __shared__ float s_red[2][8][16];
    __shared__ int s_large[2];
    const delta_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
    // workgroups of one head on one XCD: they read the same records
    const int n_blk = (int) gridDim.x;
    int b = (int) blockIdx.x;
    if (n_blk % 8 == 0) b = (b % 8) * (n_blk / 8) + b / 8;
    const int vb = b % q.vblocks, h = b / q.vblocks % a.heads, s = b / q.vblocks / a.heads, hk = h % a.key_heads;
    const int col = 16 * vb + l16, tb = wave & 3;
    const bool makes_d = wave < 4;
    const char * rec0 = q.rec + ((int64_t) s * a.heads + h) * q.chunks * q.rec_size;
    const char * kp = a.k + hk * a.k_nb1 + s * a.k_nb3;
    const char * qp = a.q + hk * a.q_nb1 + s * a.q_nb3;

    dl_v4f st[NS];  // rows 16 (w + 8 n) + 4 lg .., column l16
#pragma unroll
    for (int n = 0; n < NS; n++) {
        const int d = 16 * (wave + 8 * n) + 4 * lg;
        st[n] = dl_v4f{0, 0, 0, 0};
        if (col < a.V && d < a.K) st[n] = *(const dl_v4f *) (q.s_in + s * q.s_in_nb3 + 4 * (((int64_t) h * a.V + col) * a.K + d));
    }
    if (tid < 2) s_large[tid] = 0;
    __syncthreads();

    // a chunk's operands: rows of -W or of Q; K^T; U; lower(Q K^T L)
    dl_v4f a1[KB], kt[NS][4], u, p[4], in, left;
    float end;
    int bad;
    auto load_1 = [&](int64_t c) {
        const char * rec = rec0 + c * q.rec_size;
        const int64_t t0 = (q.c0 + c) * kDlC;
        if (makes_d) {
            const float * w = (const float *) (rec + dl_rec::w) + (16 * tb + l16) * NP + 4 * lg;
#pragma unroll
            for (int k = 0; k < KB; k++) a1[k] = *(const dl_v4f *) (w + 16 * k);
            u = ((const dl_v4f *) (rec + dl_rec::w + 4 * kDlC * NP))[(int64_t) vb * 256 + 64 * tb + lane];
            left = *(const dl_v4f *) (rec + dl_rec::left + 4 * (16 * tb + 4 * lg));
        } else {
            const char * row = qp + min(t0 + 16 * tb + l16, a.tokens - 1) * a.q_nb2;
#pragma unroll
            for (int k = 0; k < KB; k++) a1[k] = *(const dl_v4f *) (row + 4 * min(16 * k + 4 * lg, a.K - 4));
            in = *(const dl_v4f *) (rec + dl_rec::in + 4 * (16 * tb + 4 * lg));
        }
        end = *(const float *) (rec + dl_rec::end);
        bad = *(const int *) (rec + dl_rec::bad);
    };
    auto load_2 = [&](int64_t c) {
        const char * rec = rec0 + c * q.rec_size;
        const int64_t t0 = (q.c0 + c) * kDlC;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const int d = 16 * (wave + 8 * n) + l16;
#pragma unroll
            for (int sb = 0; sb < 4; sb++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = *(const float *) (kp + min(t0 + 16 * sb + 4 * lg + e, a.tokens - 1) * a.k_nb2 + 4 * min(d, a.K - 1));
                    kt[n][sb][e] = d < a.K ? v : 0.0f;  // (rows past K stay zero)
                }
        }
        if (!makes_d) {
#pragma unroll
            for (int sb = 0; sb < 4; sb++)
                if (sb <= tb) p[sb] = ((const dl_v4f *) (rec + dl_rec::p))[dl_pair(tb, sb) * 64 + lane];
        }
    };
    if (q.chunks > 0) {
        load_1(0);
        load_2(0);
    }
    for (int64_t c = 0; c < q.chunks; c++) {
        const int64_t t0 = (q.c0 + c) * kDlC, more = min(c + 1, q.chunks - 1);
        bool large = false;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            if (wave + 8 * n < KB) s_s[wave + 8 * n][lane] = st[n];
#pragma unroll
            for (int e = 0; e < 4; e++) large |= dl_past(st[n][e], kDlU);
        }
        if (large) s_large[c & 1] = 1;
        __syncthreads();
        const bool by_token = bad || s_large[c & 1];
        if (tid == 0) s_large[(c + 1) & 1] = 0;
        if (by_token) {
            const int nt = (int) min((int64_t) kDlC, a.tokens - t0);
            for (int t = 0; t < nt; t++) {
                const int64_t tt = t0 + t;
                const float * k = (const float *) (kp + tt * a.k_nb2);
                const float * qr = (const float *) (qp + tt * a.q_nb2);
                auto length = [&](const float * x, float eps) {
                    if (eps < 0.0f) return 1.0f;
                    float sum = 0.0f;
                    for (int i = lane; i < a.K; i += 64) sum = fmaf(x[i], x[i], sum);
                    return 1.0f / fmaxf(sqrtf(wave_sum(sum)), eps);
                };
                const float kl = length(k, a.k_eps), ql = length(qr, a.q_eps) * a.scale;
                const float eg = expf(*(const float *) (a.g + h * a.g_nb1 + tt * a.g_nb2 + s * a.g_nb3));
                const float beta = *(const float *) (a.beta + h * a.b_nb1 + tt * a.b_nb2 + s * a.b_nb3);
                const float v = col < a.V ? ((const float *) (a.v + h * a.v_nb1 + tt * a.v_nb2 + s * a.v_nb3))[col] : 0.0f;
                float kv[NS][4], dot = 0.0f, y = 0.0f;
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int d = 16 * (wave + 8 * n) + 4 * lg + e;
                        kv[n][e] = d < a.K ? k[d] * kl : 0.0f;
                        st[n][e] = d < a.K ? st[n][e] * eg : 0.0f;
                        if (d < a.K) dot = fmaf(st[n][e], kv[n][e], dot);
                    }
                dot += __shfl_xor(dot, 16);
                dot += __shfl_xor(dot, 32);
                if (lg == 0) s_red[0][wave][l16] = dot;
                __syncthreads();
                dot = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; w++) dot += s_red[0][w][l16];
                const float d = beta * (v - dot);
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = 16 * (wave + 8 * n) + 4 * lg + e;
                        if (i < a.K) {
                            st[n][e] = fmaf(kv[n][e], d, st[n][e]);
                            y = fmaf(st[n][e], qr[i] * ql, y);
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
            }
            load_1(more);
            load_2(more);
            __syncthreads();
            continue;
        }
        dl_v4f acc = makes_d ? u : dl_v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KB; k++) acc = dl_mfma(a1[k], s_s[k][lane], acc);
        if (makes_d) {
            s_dy[tb][lane] = acc;
            s_ds[tb][lane] = acc * left;
        } else {
            acc *= in;
        }
        const float e_end = end;
        load_1(more);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NS; n++) {
            st[n] *= e_end;
#pragma unroll
            for (int sb = 0; sb < 4; sb++) st[n] = dl_mfma(kt[n][sb], s_ds[sb][lane], st[n]);
        }
        if (!makes_d) {
#pragma unroll
            for (int sb = 0; sb < 4; sb++)
                if (sb <= tb) acc = dl_mfma(p[sb], s_dy[sb][lane], acc);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int64_t t = t0 + 16 * tb + 4 * lg + e;
                if (t < a.tokens && col < a.V) a.y[((s * a.tokens + t) * a.heads + h) * a.V + col] = acc[e];
            }
        }
        load_2(more);
    }
#pragma unroll
    for (int n = 0; n < NS; n++) {
        const int d = 16 * (wave + 8 * n) + 4 * lg;
        if (col < a.V && d < a.K) *(dl_v4f *) (a.out + s * a.out_nb3 + 4 * (((int64_t) h * a.V + col) * a.K + d)) = st[n];
    }
}

// ------------------------------------------------------------- launches ---

bool delta_supported(int64_t K) { return K >= 1 && K <= 256; }

static int dl_np(const delta_args & a) { return a.K <= 64 ? 64 : a.K <= 96 ? 96 : a.K <= 128 ? 128 : 256; }
static int64_t dl_rec_size(const delta_args & a) {
    return dl_rec::w + 4 * kDlC * (int64_t) dl_np(a) + 4 * kDlC * 16 * (int64_t) ((a.V + 15) / 16);
}
// chunks of one slab: the records of more would not stay in the caches
constexpr int64_t kDlSlab = 40 << 20;
static int64_t dl_slab(const delta_args & a) {
    const int64_t chunks = (a.tokens + kDlC - 1) / kDlC, one = dl_rec_size(a) * a.heads * a.seqs;
    const int64_t fit = std::max<int64_t>(1, kDlSlab / one), slabs = (chunks + fit - 1) / fit;
    return (chunks + slabs - 1) / slabs;
}
static bool dl_vec(const delta_args & a) {
    const uintptr_t al = (uintptr_t) a.q | (uintptr_t) a.k | (uintptr_t) a.s | (uintptr_t) a.out | (uintptr_t) a.q_nb1 |
                         (uintptr_t) a.q_nb2 | (uintptr_t) a.q_nb3 | (uintptr_t) a.k_nb1 | (uintptr_t) a.k_nb2 |
                         (uintptr_t) a.k_nb3 | (uintptr_t) a.s_nb3 | (uintptr_t) a.out_nb3 | (uintptr_t) (4 * a.K) |
                         (a.g_elem ? (uintptr_t) a.g | (uintptr_t) a.g_nb1 | (uintptr_t) a.g_nb2 | (uintptr_t) a.g_nb3 : 0);
    return al % 16 == 0;
}
// chunks: a gate a head, and tokens enough for the products to pay
static bool dl_chunked(const delta_args & a) { return !a.g_elem && a.tokens >= 24 && a.K >= 16 && dl_vec(a); }

size_t delta_scratch_bytes(const delta_args & a, int n_cu) {
    (void) n_cu;
    // (a graph planned before it is allocated: the addresses may still allow chunks)
    if (a.g_elem || a.tokens < 24 || a.K < 16) return 0;
    return (size_t) (dl_slab(a) * dl_rec_size(a) * a.heads * a.seqs);
}

template <int NP>
static void launch_delta_chunks(const delta_args & a, void * scratch, hipStream_t s) {
    dl_chunk_args q{};
    q.a = a;
    q.rec = (char *) scratch;
    q.rec_size = (int) dl_rec_size(a);
    q.vblocks = (a.V + 15) / 16;
    q.s_in = a.s, q.s_in_nb3 = a.s_nb3;
    const int64_t chunks = (a.tokens + kDlC - 1) / kDlC, slab = dl_slab(a);
    for (q.c0 = 0; q.c0 < chunks; q.c0 += slab) {
        q.chunks = std::min(slab, chunks - q.c0);
        hipLaunchKernelGGL(k_delta_solve<NP>, dim3((unsigned) (q.chunks * a.key_heads * a.seqs)), dim3(256), 0, s, q);
        note_hip_error(hipGetLastError());
        hipLaunchKernelGGL(k_delta_chunks<NP>, dim3((unsigned) ((int64_t) q.vblocks * a.heads * a.seqs)), dim3(512), 0, s, q);
        note_hip_error(hipGetLastError());
        q.s_in = a.out, q.s_in_nb3 = a.out_nb3;
    }
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
    (void) n_cu;
    if (a.seqs == 0 || a.heads == 0 || a.V == 0) return;
    if (dl_chunked(a)) {
        switch (dl_np(a)) {
            case 64: launch_delta_chunks<64>(a, scratch, s); break;
            case 96: launch_delta_chunks<96>(a, scratch, s); break;
            case 128: launch_delta_chunks<128>(a, scratch, s); break;
            default: launch_delta_chunks<256>(a, scratch, s); break;
        }
        return;
    }
    const bool vec = dl_vec(a);
    if (a.K <= 64) launch_delta_rows<1, 2, 2>(a, vec, s);
    else if (a.K <= 128) launch_delta_rows<2, 2, 2>(a, vec, s);
    else launch_delta_rows<4, 2, 2>(a, vec, s);
}

}  // namespace mi355x
