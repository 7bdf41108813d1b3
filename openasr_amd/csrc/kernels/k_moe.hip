// k_moe.hip -- the mixture-of-experts operators: GGML_OP_MUL_MAT_ID (each
// column by the matrix of its own expert) and the router's GGML_OP_ARGSORT
// and GGML_OP_SUM_ROWS.
#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

// ----------------------------------------------------------- MUL_MAT_ID ---

// one wave a (row, column): the dot product over the row's blocks
template <int WT>
__global__ __launch_bounds__(256) void k_mul_mat_id_rows(mul_mat_id_args a) {
    const int lane = threadIdx.x & 63;
    const int64_t m = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= a.M) return;
    for (int64_t col = blockIdx.y; col < a.pairs; col += gridDim.y) {
        const int64_t slot = col % a.used, tok = col / a.used;
        const int64_t e = *(const int32_t *) (a.ids + slot * a.ids_nb0 + tok * a.ids_nb1);
        double sum = 0.0;
        if (e >= 0 && e < a.experts) {
            const char * w = a.W + e * a.W_nb2 + m * a.W_nb1;
            const int64_t bcol = tok * a.b_ne1 + slot % a.b_ne1;
            if constexpr (WT == GGML_TYPE_Q8_0) {
                const int64_t nb = a.K / 32;
                const int * aq = (const int *) (a.act.q + bcol * a.K);
                const uint16_t * ds = (const uint16_t *) (w + a.K);
                for (int64_t b = lane; b < nb; b += 64) {
                    int is = 0;
                    for (int j = 0; j < 8; j++) is = dot4_i8(((const int *) w)[8 * b + j], aq[8 * b + j], is);
                    sum += (double) is * (double) (half_bits_to_float(ds[b]) * a.act.d[bcol * nb + b]);
                }
            } else if constexpr (WT == GGML_TYPE_Q4_K) {
                const int64_t nb = a.K / 32;
                const int * aq = (const int *) (a.act.q + bcol * a.K);
                for (int64_t b = lane; b < nb; b += 64) {
                    const uint8_t * blk = (const uint8_t *) w + (b / 8) * 144;
                    const int j = (int) (b % 8);
                    const uint8_t * sc = blk + 4;
                    const int scale = j < 4 ? sc[j] & 63 : (sc[j + 4] & 15) | ((sc[j - 4] >> 6) << 4);
                    const int mn = j < 4 ? sc[j + 4] & 63 : (sc[j + 4] >> 4) | ((sc[j] >> 6) << 4);
                    const int * q = (const int *) (blk + 16 + 32 * (j / 2));
                    int is = 0;
                    for (int k = 0; k < 8; k++) is = dot4_i8((q[k] >> (4 * (j & 1))) & 0x0F0F0F0F, aq[8 * b + k], is);
                    const uint16_t * dd = (const uint16_t *) blk;
                    const double da = (double) a.act.d[bcol * (a.K / 256) + b / 8];
                    sum += (double) half_bits_to_float(dd[0]) * da * (double) (scale * is) -
                           (double) half_bits_to_float(dd[1]) * da * (double) (mn * a.act.ssum[bcol * nb + b]);
                }
            } else {
                const float * x = (const float *) (a.b + (slot % a.b_ne1) * a.b_nb1 + tok * a.b_nb2);
                for (int64_t k = lane; k < a.K; k += 64)
                    sum += WT == GGML_TYPE_F16 ? (double) (half_bits_to_float(((const uint16_t *) w)[k]) * round_to_half(x[k]))
                                               : (double) ((const float *) w)[k] * (double) x[k];
            }
        }
        sum = wave_sum_d(sum);
        if (lane == 0) a.out[col * a.M + m] = (float) sum;
    }
}

void launch_mul_mat_id(int wtype, const mul_mat_id_args & a, hipStream_t s) {
    if (a.M == 0 || a.pairs == 0) return;
    const dim3 grid((unsigned) ((a.M + 3) / 4), (unsigned) (a.pairs < 32768 ? a.pairs : 32768));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (wtype == GGML_TYPE_Q8_0) go(k_mul_mat_id_rows<GGML_TYPE_Q8_0>);
    else if (wtype == GGML_TYPE_Q4_K) go(k_mul_mat_id_rows<GGML_TYPE_Q4_K>);
    else if (wtype == GGML_TYPE_F16) go(k_mul_mat_id_rows<GGML_TYPE_F16>);
    else go(k_mul_mat_id_rows<GGML_TYPE_F32>);
}

// -------------------------------------------------------------- ARGSORT ---

// order-preserving bits of a float: equal floats (both zeros) have equal
// keys, NaN the largest
__device__ __forceinline__ uint32_t sort_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 -> +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// one wave a row: an element's place is the number of elements before it
__global__ __launch_bounds__(256) void k_argsort_rank(tview d, tview a, int desc, int64_t rows) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
    const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
    int32_t * o = (int32_t *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]);
    const int n = (int) a.ne[0];
    for (int i = lane; i < n; i += 64) {
        const uint32_t k = sort_key(x[i]);
        int at = 0;
        for (int j = 0; j < n; j++) {
            const uint32_t q = sort_key(x[j]);
            at += (desc ? q > k : q < k) || (q == k && j < i);
        }
        o[at] = i;
    }
}

bool argsort_supported(int64_t n) { return n >= 0 && n <= 8192; }

void launch_argsort(const tview & d, const tview & a, int desc, hipStream_t s) {
    const int64_t rows = a.ne[1] * a.ne[2] * a.ne[3];
    if (rows == 0 || a.ne[0] == 0) return;
    hipLaunchKernelGGL(k_argsort_rank, dim3((unsigned) ((rows + 3) / 4)), dim3(256), 0, s, d, a, desc, rows);
}

// one wave a row, the sum held in double
__global__ __launch_bounds__(256) void k_sum_rows(tview d, tview a, int64_t rows) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
    const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
    double sum = 0.0;
    for (int64_t i = lane; i < a.ne[0]; i += 64) sum += (double) x[i];
    sum = wave_sum_d(sum);
    if (lane == 0) *(float *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]) = (float) sum;
}

void launch_sum_rows(const tview & d, const tview & a, hipStream_t s) {
    const int64_t rows = a.ne[1] * a.ne[2] * a.ne[3];
    if (rows == 0) return;
    hipLaunchKernelGGL(k_sum_rows, dim3((unsigned) ((rows + 3) / 4)), dim3(256), 0, s, d, a, rows);
}

}  // namespace mi355x
