// k_moe.hip -- the mixture-of-experts operators: GGML_OP_MUL_MAT_ID (each
// column by the matrix of its own expert) and the router's GGML_OP_ARGSORT
// and GGML_OP_SUM_ROWS.
#include <algorithm>
#include <type_traits>

#include "../mfma_units.h"
#include "../mi355x_common.h"
#include "../ops.h"
#include "../quant_dev.h"

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

// ------------------------------------------------- few columns: streaming ---
//
// A workgroup takes 16 rows of one expert (PAIR: of both its matrices, whose
// SwiGLU it stores) and the columns routed to it, 16 at a time; its waves
// split K, their sums added through LDS in order. Bound by the weights'
// stream: each wave reads its own, straight into the matrix cores' operand
// layout (activations A, weights B: lane l ends with weight row l % 16). The routing is done in place: workgroup y serves
// the expert of pair y if no earlier pair has it. Q4_K, 8 tokens of 8 (40
// experts of 2 x 768 x 2048, 71 MB): 35 us, most of it the loads' way from
// memory after the ids' own; f16, one token of 4 (17 MB): 7 us.
constexpr int kMoeFew = 256;  // pairs a workgroup's threads hold

typedef _Float16 moe_v8h __attribute__((ext_vector_type(8)));
typedef float moe_v4f __attribute__((ext_vector_type(4)));

// eight f32 values at p as f16 (rounded to nearest even)
__device__ __forceinline__ moe_v8h moe_round8(const float * p) {
    const float4 a = *(const float4 *) p, b = *(const float4 *) (p + 4);
    return moe_v8h{(_Float16) a.x, (_Float16) a.y, (_Float16) a.z, (_Float16) a.w,
                   (_Float16) b.x, (_Float16) b.y, (_Float16) b.z, (_Float16) b.w};
}

// pair p's token and slot, without a division (p < 2^26: the product's high
// half is the quotient or one less)
__device__ __forceinline__ void moe_pair(const mul_mat_id_args & a, int p, int & token, int & slot) {
    const int used = (int) a.used;
    token = (int) __umulhi((uint32_t) p, a.used_inv);
    slot = p - token * used;
    if (slot >= used) token++, slot -= used;
}
// its token, and which of the token's columns of b it takes
__device__ __forceinline__ void moe_column(const mul_mat_id_args & a, int p, int & token, int & of) {
    moe_pair(a, p, token, of);
    const int per = (int) a.b_ne1;
    if (per == 1) of = 0;
    else if (per != (int) a.used) of %= per;
}

// The 16 x 16 sums of NM matrices' rows and 16 columns over wave w's share of
// K. The operand's row r holds column r / 4 + 4 (r % 4), so that lane group g
// ends with the columns g + 4 i, and few columns need the first i only (NCL of
// them: with 4 always, the scaling of absent columns was most of the
// instructions). bcol: the lane's operand column in b's order, bc4: the
// columns g + 4 i.
template <int WT, int NM>
struct moe_tile;

template <int NM>
struct moe_tile<GGML_TYPE_F16, NM> {
    template <int NCL>
    static __device__ __forceinline__ void run(const mul_mat_id_args & a, const char * const (&wrow)[NM], const char * xcol, int64_t bcol,
                                               const int (&)[4], int wave, int waves, int g, double (&out)[NM][4]) {
        const float * x = (const float *) xcol;
        const int64_t steps = (a.K + 31) / 32;
        moe_v4f acc[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) acc[m] = moe_v4f{0, 0, 0, 0};
        constexpr int U = 4;  // steps in flight
        for (int64_t s0 = wave; s0 < steps; s0 += (int64_t) U * waves) {
            uint4 w[NM][U];
            moe_v8h xv[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t k = (s0 + (int64_t) u * waves) * 32 + 8 * g;
                const bool ok = k < a.K;  // K % 8 == 0: eight at a time
#pragma unroll
                for (int m = 0; m < NM; m++) w[m][u] = *(const uint4 *) (wrow[m] + 2 * (ok ? k : 0));
                xv[u] = moe_round8(x + (ok ? k : 0));
                if (!ok) {
#pragma unroll
                    for (int m = 0; m < NM; m++) w[m][u] = make_uint4(0, 0, 0, 0);
                    xv[u] = moe_v8h{0, 0, 0, 0, 0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int m = 0; m < NM; m++)
                    acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xv[u], __builtin_bit_cast(moe_v8h, w[m][u]), acc[m], 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < NM; m++)
#pragma unroll
            for (int i = 0; i < NCL; i++) out[m][i] = acc[m][i];
    }
};

template <int NM>
struct moe_tile<GGML_TYPE_Q8_0, NM> {
    template <int NCL>
    static __device__ __forceinline__ void run(const mul_mat_id_args & a, const char * const (&wrow)[NM], const char * xcol, int64_t bcol,
                                               const int (&bc4)[4], int wave, int waves, int g, double (&out)[NM][4]) {
        const int64_t nblk = a.K / 32;
        const int8_t * aq = a.act.q + bcol * a.K;
        constexpr int U = 4;
        for (int64_t b0 = wave; b0 < nblk; b0 += (int64_t) U * waves) {
            long q[NM][U], af[U];
            uint16_t d[NM][U];
            float da[U][4];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t b = min(b0 + (int64_t) u * waves, nblk - 1);
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    q[m][u] = *(const long *) (wrow[m] + 32 * b + 8 * g);
                    d[m][u] = *(const uint16_t *) (wrow[m] + a.K + 2 * b);
                }
                af[u] = *(const long *) (aq + 32 * b + 8 * g);
#pragma unroll
                for (int i = 0; i < NCL; i++) da[u][i] = a.act.d[bc4[i] * nblk + b];
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (b0 + (int64_t) u * waves < nblk)
#pragma unroll
                    for (int m = 0; m < NM; m++) q8_0_block<NCL>(af[u], q[m][u], d[m][u], da[u], out[m]);
        }
    }
};

template <int NM>
struct moe_tile<GGML_TYPE_Q4_K, NM> {
    template <int NCL>
    static __device__ __forceinline__ void run(const mul_mat_id_args & a, const char * const (&wrow)[NM], const char * xcol, int64_t bcol,
                                               const int (&bc4)[4], int wave, int waves, int g, double (&out)[NM][4]) {
        const int64_t nsb = a.K / 256;
        const int8_t * aq = a.act.q + bcol * a.K;
        const int16_t * ass = a.act.ssum + bcol * (a.K / 32);
        struct block {
            uint4 hdr[NM];
            long q[NM][4], af[8];
            float ad[4], ssa[2];
        };
        auto load = [&](int64_t b, block & v) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const char * blk = wrow[m] + b * 144;
                v.hdr[m] = *(const uint4 *) blk;
#pragma unroll
                for (int c = 0; c < 4; c++) v.q[m][c] = *(const long *) (blk + 16 + 32 * c + 8 * g);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) v.af[j] = *(const long *) (aq + 256 * b + 32 * j + 8 * g);
#pragma unroll
            for (int i = 0; i < NCL; i++) v.ad[i] = a.act.d[bc4[i] * nsb + b];
            q4k_ssum_operand(ass + 8 * b, true, g, v.ssa);
        };
        if (wave >= nsb) return;
        block cur, next;  // a block ahead
        load(wave, cur);
        for (int64_t b = wave; b < nsb; b += waves) {
            load(min(b + waves, nsb - 1), next);
#pragma unroll
            for (int m = 0; m < NM; m++) q4k_unit<NCL>(cur.hdr[m], cur.q[m], cur.af, cur.ad, cur.ssa, out[m]);
            cur = next;
        }
    }
};

__device__ __forceinline__ float moe_swiglu(float g, float u) { return (g / (1.0f + expf_det(-g))) * u; }

template <int WT, bool PAIR>
__global__ __launch_bounds__(256) void k_moe_few(mul_mat_id_args a) {
    __shared__ int s_id[kMoeFew];
    __shared__ int s_list[kMoeFew];
    __shared__ int s_n[4];
    __shared__ double s_acc[2][3][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int me = blockIdx.y;
    const int64_t m0 = (int64_t) blockIdx.x * 16;
    int id = -1;
    if (tid < a.pairs) {
        int token, slot;
        moe_pair(a, tid, token, slot);
        id = *(const int32_t *) (a.ids + slot * a.ids_nb0 + token * a.ids_nb1);
    }
    s_id[tid] = id;
    __syncthreads();
    const int e = s_id[me];
    if (e < 0 || e >= a.experts) {  // no expert: the pair's column is zero
        if (tid < 16 && m0 + tid < a.M) a.out[(int64_t) me * a.M + m0 + tid] = 0.0f;
        return;
    }
    const bool mine = tid < a.pairs && id == e;
    const uint64_t have = __ballot(mine);
    if (lane == 0) s_n[wave] = __popcll(have);
    if (__syncthreads_or(mine && tid < me)) return;  // an earlier pair's workgroup serves this expert
    int at = 0, n = 0;
    for (int w = 0; w < 4; w++) {
        at += w < wave ? s_n[w] : 0;
        n += s_n[w];
    }
    if (mine) s_list[at + __popcll(have & ((1ull << lane) - 1))] = tid;
    __syncthreads();
    const int64_t row = min(m0 + r, a.M - 1);
    constexpr int NM = PAIR ? 2 : 1;
    const char * wrow[NM];
    wrow[0] = a.W + e * a.W_nb2 + row * a.W_nb1;
    if constexpr (PAIR) wrow[1] = a.W2 + e * a.W_nb2 + row * a.W_nb1;
    for (int c0 = 0; c0 < n; c0 += 16) {
        int token, of, bc4[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            moe_column(a, s_list[min(c0 + g + 4 * i, n - 1)], token, of);
            bc4[i] = token * (int) a.b_ne1 + of;
        }
        moe_column(a, s_list[min(c0 + (r >> 2) + 4 * (r & 3), n - 1)], token, of);
        const int64_t bcol = token * a.b_ne1 + of;
        const char * xcol = a.b + token * a.b_nb2 + of * a.b_nb1;
        double acc[NM][4] = {};
        using tile = moe_tile<WT, NM>;
        if (n - c0 <= 4) tile::template run<1>(a, wrow, xcol, bcol, bc4, wave, 4, g, acc);
        else if (n - c0 <= 8) tile::template run<2>(a, wrow, xcol, bcol, bc4, wave, 4, g, acc);
        else tile::template run<4>(a, wrow, xcol, bcol, bc4, wave, 4, g, acc);
        if (wave > 0) {
#pragma unroll
            for (int m = 0; m < NM; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) s_acc[m][wave - 1][i][lane] = acc[m][i];
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int m = 0; m < NM; m++)
#pragma unroll
                    for (int w = 0; w < 3; w++) acc[m][i] += s_acc[m][w][i][lane];
                const int c = c0 + g + 4 * i;
                if (c < n && m0 + r < a.M)
                    a.out[(int64_t) s_list[c] * a.M + m0 + r] =
                        PAIR ? moe_swiglu((float) acc[0][i], (float) acc[1][i]) : (float) acc[0][i];
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------ many columns: tile GEMM ---
//
// k_moe_prepare sorts the pairs by expert (a counting sort of one workgroup,
// each expert's pairs in their order) and cuts every expert's run into tiles
// of BN columns; its other workgroups make the columns' f16 operands: the
// rounded values of F16 weights, the whole numbers of the quantized blocks
// otherwise (with their scales beside them). k_moe_gemm takes 128 weight rows
// (PAIR: 64 of each matrix) by BN columns of one expert, K in steps of 64
// through LDS (16-byte pieces swizzled by row), the next steps' loads in
// flight.
//
// F16 (1501 tokens of 4, 32 experts of 2 x 1024 x 2048): 108 us, 460 TFLOP/s
// of the columns there are. Loads, LDS stores and barriers alone take 105, the
// rest without loads 89: bound by 1.07 GB through the L2s (268 MB of weights
// twice, columns for each row tile) with the matrix cores waiting. Q8_0 (700
// tokens of 8, 64 experts of 2048 x 768): 84 us, most of it waiting (35 % of the
// waves' cycles on memory and barriers, 25 % on issue); 38 % of the cycles issue
// vector instructions (8 for the scales of each product of 16 x 16 x 32, 7 others),
// the matrix cores are busy 10 %, and the tiles' last round leaves CUs idle.
//
// Quantized weights are staged as the whole numbers of their blocks too:
// a block's sum of 32 products is exact on the f16 matrix cores, and a block
// then costs a multiply and a fused multiply-add an output for its scales
// (Q4_K's minimum: another). The sums are f32: within the roundings of K / 32
// terms of the exact block sums.
constexpr int kMoeK = 64;
constexpr int kMoeRows = 128;

struct moe_wide_args {
    mul_mat_id_args a;
    int * head;     // [0]: the number of tiles
    int4 * tiles;   // the expert (-1: none), its first place, its columns, its first tile
    int * sorted;   // place -> pair
    _Float16 * x;   // [b column][Kp]
    float * xd;     // quantized: the blocks' scales, [b column][Kp / 32 or Kp / 256]
    float * xs;     // Q4_K: scale times sum of 32 elements, [b column][Kp / 32]
    int64_t kp, bcols, row_tiles;
    int bn, max_tiles;
};

__device__ __forceinline__ void moe_route(const moe_wide_args & q) {
    extern __shared__ int s_hist[];  // [16][bins], bins = experts + 1 (no expert)
    const mul_mat_id_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bins = (int) a.experts + 1, pairs = (int) a.pairs;
    for (int i = tid; i < 16 * bins; i += 1024) s_hist[i] = 0;
    __syncthreads();
    // wave w's share: consecutive groups of 64 pairs
    const int groups = (pairs + 63) / 64, per = (groups + 15) / 16;
    auto expert_of = [&](int p) {
        int token, slot;
        moe_pair(a, p, token, slot);
        const int e = *(const int32_t *) (a.ids + slot * a.ids_nb0 + token * a.ids_nb1);
        return e < 0 || e >= a.experts ? (int) a.experts : e;
    };
    // a batch of groups' ids in flight at once (one by one, each waits for its load)
    constexpr int kBatch = 8;
    int e[kBatch];
    auto load = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int p = (wave * per + k0 + k) * 64 + lane, v = expert_of(min(p, pairs - 1));
            e[k] = k0 + k < per && p < pairs ? v : -1;
        }
    };
    for (int k0 = 0; k0 < per; k0 += kBatch) {
        load(k0);
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (e[k] >= 0) atomicAdd(&s_hist[wave * bins + e[k]], 1);
    }
    __syncthreads();
    // the bins' totals, their exclusive sums (places and tiles) over bins in order
    __shared__ int s_sum[2][16];
    int base = 0, tbase = 0;
    for (int b0 = 0; b0 < bins; b0 += 1024) {
        const int b = b0 + tid;
        int total = 0;
        if (b < bins)
            for (int w = 0; w < 16; w++) total += s_hist[w * bins + b];
        const int nt = (total + q.bn - 1) / q.bn;
        int sum = total, tsum = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o), tv = __shfl_up(tsum, o);
            if (lane >= o) sum += v, tsum += tv;
        }
        if (lane == 63) s_sum[0][wave] = sum, s_sum[1][wave] = tsum;
        __syncthreads();
        int before = base, tbefore = tbase;
        for (int w = 0; w < 16; w++) {
            before += w < wave ? s_sum[0][w] : 0;
            tbefore += w < wave ? s_sum[1][w] : 0;
            base += s_sum[0][w];
            tbase += s_sum[1][w];
        }
        if (b < bins) {
            int at = before + sum - total;
            const int t0 = tbefore + tsum - nt;
            for (int t = 0; t < nt; t++) q.tiles[t0 + t] = make_int4(b < a.experts ? b : -1, at, total, t0);
            int count[16];  // the waves' first places
#pragma unroll
            for (int w = 0; w < 16; w++) count[w] = s_hist[w * bins + b];
#pragma unroll
            for (int w = 0; w < 16; w++) {
                s_hist[w * bins + b] = at;
                at += count[w];
            }
        }
        __syncthreads();
    }
    if (tid == 0) q.head[0] = tbase;
    // places: within a group of 64, pairs of one expert in lane order
    for (int k0 = 0; k0 < per; k0 += kBatch) {
        if (per > kBatch) load(k0);
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (k0 + k >= per) break;
            const bool ok = e[k] >= 0;
            uint64_t same = __ballot(ok);
            for (int bit = 1; bit < bins; bit <<= 1) {
                const uint64_t set = __ballot(ok && (e[k] & bit));
                same &= (e[k] & bit) ? set : ~set;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            if (ok) q.sorted[s_hist[wave * bins + e[k]] + rank] = (wave * per + k0 + k) * 64 + lane;
            __builtin_amdgcn_wave_barrier();
            if (ok && rank == 0) s_hist[wave * bins + e[k]] += __popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// the first workgroup sorts, the others make the operands, one wave 256
// elements of a column
template <int WT>
__global__ __launch_bounds__(1024) void k_moe_prepare(moe_wide_args q) {
    if (blockIdx.x == 0) {
        moe_route(q);
        return;
    }
    const mul_mat_id_args & a = q.a;
    const int lane = threadIdx.x & 63;
    // (the wave's place in scalars of 32 bits: bcols * kp < 2^31)
    const uint32_t chunks = (uint32_t) ((q.kp + 255) / 256);
    const uint32_t w = (blockIdx.x - 1) * 16 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wcol = w / chunks, per = (uint32_t) a.b_ne1, btoken = wcol / per;
    const int64_t col = wcol, k = (int64_t) (w - wcol * chunks) * 256 + 4 * lane;
    if (col >= q.bcols) return;
    const float * x = (const float *) (a.b + (int64_t) (wcol - btoken * per) * a.b_nb1 + btoken * a.b_nb2);
    float4 v = make_float4(0, 0, 0, 0);
    if (k < a.K) v = *(const float4 *) (x + k);  // K % 4 == 0
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    v4h o = {(_Float16) v.x, (_Float16) v.y, (_Float16) v.z, (_Float16) v.w};
    if constexpr (WT == GGML_TYPE_Q8_0) {
        const q8_0_lane l = quantize_q8_0_group(v);
        o = v4h{(_Float16) (float) l.q.x, (_Float16) (float) l.q.y, (_Float16) (float) l.q.z, (_Float16) (float) l.q.w};
        if ((lane & 7) == 0 && k < q.kp) q.xd[col * (q.kp / 32) + k / 32] = l.d;
    } else if constexpr (WT == GGML_TYPE_Q4_K) {
        const q8_K_lane l = quantize_q8_K_wave(v, lane);
        o = v4h{(_Float16) (float) l.q.x, (_Float16) (float) l.q.y, (_Float16) (float) l.q.z, (_Float16) (float) l.q.w};
        if ((lane & 7) == 0) q.xs[col * (q.kp / 32) + k / 32] = l.d * (float) l.ssum;
        if (lane == 0) q.xd[col * (q.kp / 256) + k / 256] = l.d;
    }
    if (k < q.kp) *(v4h *) (q.x + col * q.kp + k) = o;
}

// the staged row's 16-byte piece p at slot p ^ (row % 8): fragment reads (16
// rows, one piece each) spread over the banks
__device__ __forceinline__ uint4 * moe_slot(_Float16 (*s)[kMoeK], int row, int piece) {
    return (uint4 *) &s[row][8 * (piece ^ (row & 7))];
}

// eight bytes' values as f16, less `bias`: the byte in the mantissa under the
// exponent of 1024
__device__ __forceinline__ uint4 moe_bytes(uint32_t w0, uint32_t w1, float bias) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 k = {(_Float16) (1024.0f + bias), (_Float16) (1024.0f + bias)};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) - k;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) - k;
    const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) - k;
    const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) - k;
    return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                      __builtin_bit_cast(uint32_t, d));
}

// a thread's share of a step's weights: row t / 2, 32 of its 64 elements
// (Q4_K: 16 elements of each of the step's two blocks)
template <int WT>
struct moe_w;
typedef uint32_t moe_u4 __attribute__((ext_vector_type(4)));  // (an array of uint4 stayed in memory)
template <>
struct moe_w<GGML_TYPE_F16> {
    moe_u4 v[4];
};
template <>
struct moe_w<GGML_TYPE_Q8_0> {
    moe_u4 v[2];
};
template <>
struct moe_w<GGML_TYPE_Q4_K> {
    moe_u4 v;
};

// and of the scales of four steps: a row's of four blocks (Q4_K: its
// super-block's header), a column's of four
template <int WT>
struct moe_scales {
    moe_u4 hdr;
    float d, s[4];
};
template <>
struct moe_scales<GGML_TYPE_Q8_0> {
    uint16_t w[4];
    float2 x[2];
};

// and of its columns, 16-byte pieces
template <int XP>
struct moe_x {
    moe_u4 v[XP];
};

template <int C, int XP>
__device__ __forceinline__ void moe_x_load(moe_x<C> & x, const _Float16 * base, const uint32_t (&at)[XP]) {
#pragma unroll
    for (int u = 0; u < C; u++) x.v[u] = *(const moe_u4 *) ((const char *) base + at[u]);
}
template <int C>
__device__ __forceinline__ void moe_x_store(const moe_x<C> & x, _Float16 (*s)[kMoeK], int tid) {
#pragma unroll
    for (int u = 0; u < C; u++) *(moe_u4 *) moe_slot(s, (tid + 256 * u) / 8, tid % 8) = x.v[u];
}

template <int WT, int BN, int NB>
struct moe_lds {
    static constexpr int kS = WT == GGML_TYPE_F16 ? 1 : 8, kM = WT == GGML_TYPE_Q4_K ? 8 : 1;
    _Float16 w[NB][kMoeRows][kMoeK];
    _Float16 x[NB][BN][kMoeK];
    float wd[NB][kS][kMoeRows];  // a block's scale by [buffer][block of four steps][row]
    float wm[NB][kM][kMoeRows];  // Q4_K: its minimum
    float xd[NB][kS][BN];        // the columns' scales (Q4_K: one)
    float xs[NB][kM][BN];        // Q4_K: scale times sum
    int col[BN];               // the columns' places in b
    int pair[BN];              // and in the result
};

template <int WT, bool PAIR, int BN>
__global__ __launch_bounds__(256, 2) void k_moe_gemm(moe_wide_args q) {
    constexpr int kQ = WT != GGML_TYPE_F16, NB = kQ && BN == 128 ? 1 : 2;
    constexpr int NR = 4, NC = BN / 32;  // a wave's 16-tiles of rows and columns: 64 rows, BN / 2 columns
    __shared__ __align__(16) moe_lds<WT, BN, NB> L;
    const mul_mat_id_args & a = q.a;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave & 1, wc = wave >> 1;
    // Workgroup i is on XCD i % 8. Each expert's row tiles go to the XCDs in
    // turn, so that a much used expert's work is spread; a row tile's column
    // tiles are adjacent: they read the same weights at the same time, once
    // beyond their XCD's L2.
    const uint32_t rows = (uint32_t) q.row_tiles, each = (rows + 7) / 8, t = blockIdx.x / 8;
    if (t >= (uint32_t) q.head[0] * each) return;
    const int4 of = q.tiles[t / each];  // its expert's columns and first tile
    const uint32_t in = t - (uint32_t) of.w * each, run = (uint32_t) (of.z + BN - 1) / BN, nth = in / run, ct = in - nth * run;
    const uint32_t rt = 8 * nth + (blockIdx.x + (uint32_t) of.w) % 8;
    if (rt >= rows) return;
    const int64_t m0 = (int64_t) rt * (PAIR ? 64 : 128);
    const int n = __builtin_amdgcn_readfirstlane(min(BN, of.z - (int) ct * BN)), at = of.y + (int) ct * BN;
    if (tid < BN) {
        const int p = q.sorted[at + min(tid, n - 1)];
        L.pair[tid] = p;
        int token, of;
        moe_column(a, p, token, of);
        L.col[tid] = token * (int) a.b_ne1 + of;
    }
    __syncthreads();
    if (of.x < 0) {  // no expert: zeros
        const int rows = (int) min((int64_t) (PAIR ? 64 : 128), a.M - m0);
        for (int i = tid; i < n * rows; i += 256) a.out[(int64_t) L.pair[i / rows] * a.M + m0 + i % rows] = 0.0f;
        return;
    }
    // staging: thread t row t / 2 of the tile, half t % 2; PAIR: rows 0 .. 63 of
    // W, then the same of W2
    const int srow = tid >> 1, half = tid & 1;
    const int64_t mrow = min(PAIR ? m0 + (srow & 63) : m0 + srow, a.M - 1);
    const char * wrow = (PAIR && srow >= 64 ? a.W2 : a.W) + of.x * a.W_nb2 + mrow * a.W_nb1;
    // (F16: pieces t % 8 of the rows t / 8 + 32 u, whole lines a load)
    const char * wp[WT == GGML_TYPE_F16 ? 4 : 1];
    if constexpr (WT == GGML_TYPE_F16) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t m = min(m0 + (PAIR ? (tid / 8 + 32 * u) & 63 : tid / 8 + 32 * u), a.M - 1);
            wp[u] = (PAIR && u >= 2 ? a.W2 : a.W) + of.x * a.W_nb2 + m * a.W_nb1 + 16 * (tid % 8);
        }
    }
    const int64_t steps = (a.K + kMoeK - 1) / kMoeK;
    uint32_t xat[NC];  // the columns' pieces (byte offsets in 32 bits: mul_mat_id_wide)
#pragma unroll
    for (int u = 0; u < NC; u++) xat[u] = 2 * ((uint32_t) L.col[(tid + 256 * u) / 8] * (uint32_t) q.kp + 8 * (tid % 8));
    // wave (wr, wc): the 16-column tiles wc, wc + 2, ..; rows 64 wr .., or 32 wr .. of
    // both matrices. Tiles past the last column are neither staged nor multiplied.
    auto tile_col = [&](int j) { return 32 * j + 16 * wc; };
    auto tile_row = [&](int i) { return PAIR ? 64 * (i >> 1) + 32 * wr + 16 * (i & 1) : 64 * wr + 16 * i; };
    moe_v4f acc[NR][NC];
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
        for (int j = 0; j < NC; j++) acc[i][j] = moe_v4f{0, 0, 0, 0};
    const moe_v4f zero = {0, 0, 0, 0};
    // C: the tile's 32-column groups that hold columns (the workgroup's one value)
    auto products_of = [&](auto groups) {
        constexpr int C = decltype(groups)::value;
        // (the values of the lane made anew for each C: shared ones were kept and spilled)
        int tid = (int) threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, r = lane & 15, g = lane >> 4, srow = tid >> 1, half = tid & 1;
        const int scol = tid % BN, sblk = tid / BN;  // the scale this thread stages (sblk < 2)
        struct stage {
            moe_w<WT> w;
            moe_x<C> x;
        };
        // The scales are fetched and staged for four steps at once: a load a
        // step touched a line of its own for each row and column, as much
        // again as the weights.
        auto load_scales = [&](int64_t s, moe_scales<WT> & sc) {
            const int64_t c = L.col[scol];
            if constexpr (WT == GGML_TYPE_Q8_0) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int64_t blk = 2 * s + 4 * half + i;
                    sc.w[i] = *(const uint16_t *) (wrow + a.K + 2 * (32 * blk < a.K ? blk : 0));
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
                    sc.x[i] = *(const float2 *) (q.xd + c * (q.kp / 32) + 2 * min(s + 2 * (sblk & 1) + i, steps - 1));
            } else if constexpr (WT == GGML_TYPE_Q4_K) {
                sc.hdr = *(const moe_u4 *) (wrow + s / 4 * 144);
                sc.d = q.xd[c * (q.kp / 256) + s / 4];
                *(float4 *) sc.s = *(const float4 *) (q.xs + c * (q.kp / 32) + 2 * s + 4 * (sblk & 1));
            }
        };
        auto store_scales = [&](int b, const moe_scales<WT> & sc) {
            if constexpr (WT == GGML_TYPE_Q8_0) {
#pragma unroll
                for (int i = 0; i < 4; i++) L.wd[b][4 * half + i][srow] = half_bits_to_float(sc.w[i]);
                if (sblk < 2) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        L.xd[b][4 * sblk + 2 * i][scol] = sc.x[i].x, L.xd[b][4 * sblk + 2 * i + 1][scol] = sc.x[i].y;
                }
            } else if constexpr (WT == GGML_TYPE_Q4_K) {
                // block j's 6-bit scale and minimum of the packed 12 bytes
                const float d = half_bits_to_float((uint16_t) sc.hdr.x), m = -half_bits_to_float((uint16_t) (sc.hdr.x >> 16));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t s6 = half ? (sc.hdr.w >> (8 * i) & 15) | (sc.hdr.y >> (8 * i + 6) & 3) << 4 : sc.hdr.y >> (8 * i) & 63;
                    const uint32_t m6 = half ? (sc.hdr.w >> (8 * i + 4) & 15) | (sc.hdr.z >> (8 * i + 6) & 3) << 4 : sc.hdr.z >> (8 * i) & 63;
                    L.wd[b][4 * half + i][srow] = d * (float) s6;
                    L.wm[b][4 * half + i][srow] = m * (float) m6;
                }
                if (sblk < 2) {
#pragma unroll
                    for (int i = 0; i < 4; i++) L.xs[b][4 * sblk + i][scol] = sc.s[i];
                    if (sblk == 0) L.xd[b][0][scol] = sc.d;
                }
            }
        };
        auto load = [&](int64_t s, stage & st) {
            moe_w<WT> & w = st.w;
            const int64_t k0 = s * kMoeK;
            if constexpr (WT == GGML_TYPE_F16) {
                if (k0 + kMoeK <= a.K) {
#pragma unroll
                    for (int u = 0; u < 4; u++) w.v[u] = *(const moe_u4 *) (wp[u] + 2 * k0);
                } else {  // past K: the row's first piece, masked when stored
#pragma unroll
                    for (int u = 0; u < 4; u++) w.v[u] = *(const moe_u4 *) (wp[u] + (k0 + 8 * (tid % 8) < a.K ? 2 * k0 : -16 * (tid % 8)));
                }
            } else if constexpr (WT == GGML_TYPE_Q8_0) {
                const int64_t b = 2 * s + half;
                const int64_t bc = 32 * b < a.K ? b : 0;  // past K: the columns' scale is zero
                const moe_u4 * p = (const moe_u4 *) (wrow + 32 * bc);
                w.v[0] = p[0];
                w.v[1] = p[1];
            } else {
                w.v = *(const moe_u4 *) (wrow + s / 4 * 144 + 16 + 32 * (s % 4) + 16 * half);
            }
            moe_x_load<C>(st.x, q.x + k0, xat);
        };
        auto store = [&](int b, int64_t s, const stage & st) {
            const moe_w<WT> & w = st.w;
            if constexpr (WT == GGML_TYPE_F16) {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint32_t in = s * kMoeK + 8 * (tid % 8) < a.K ? 0xFFFFFFFFu : 0u;
                    *(moe_u4 *) moe_slot(L.w[b], tid / 8 + 32 * u, tid % 8) = w.v[u] & in;
                }
            } else if constexpr (WT == GGML_TYPE_Q8_0) {
                const uint32_t z = 0x80808080u;
                const uint32_t v[8] = {w.v[0].x, w.v[0].y, w.v[0].z, w.v[0].w, w.v[1].x, w.v[1].y, w.v[1].z, w.v[1].w};
#pragma unroll
                for (int u = 0; u < 4; u++) *moe_slot(L.w[b], srow, 4 * half + u) = moe_bytes(v[2 * u] ^ z, v[2 * u + 1] ^ z, 128.0f);
            } else {
                const uint32_t lo = 0x0F0F0F0Fu;
                const uint32_t v[4] = {w.v.x, w.v.y, w.v.z, w.v.w};
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    *moe_slot(L.w[b], srow, 2 * half + u) = moe_bytes(v[2 * u] & lo, v[2 * u + 1] & lo, 0.0f);
                    *moe_slot(L.w[b], srow, 4 + 2 * half + u) = moe_bytes(v[2 * u] >> 4 & lo, v[2 * u + 1] >> 4 & lo, 0.0f);
                }
            }
            moe_x_store<C>(st.x, L.x[b], tid);
        };
        auto multiply = [&](int b, int64_t s) {
            const int gb = NB == 2 ? (int) (s / 4 & 1) : 0;  // the scales' buffer
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                __builtin_amdgcn_sched_barrier(0);  // (one block's operands at a time: more in flight spill)
                moe_v8h wf[NR], xf[C];
#pragma unroll
                for (int i = 0; i < NR; i++)
                    wf[i] = __builtin_bit_cast(moe_v8h, *moe_slot(L.w[b], tile_row(i) + r, 4 * kk + g));
#pragma unroll
                for (int j = 0; j < C; j++)
                    xf[j] = __builtin_bit_cast(moe_v8h, *moe_slot(L.x[b], tile_col(j) + r, 4 * kk + g));
                if constexpr (kQ) {
                    float dw[NR], mw[NR];
#pragma unroll
                    for (int i = 0; i < NR; i++) {
                        dw[i] = L.wd[gb][2 * (s % 4) + kk][tile_row(i) + r];
                        if constexpr (WT == GGML_TYPE_Q4_K) mw[i] = L.wm[gb][2 * (s % 4) + kk][tile_row(i) + r];
                    }
#pragma unroll
                    for (int j = 0; j < C; j++) {
                        const float4 dx = *(const float4 *) &L.xd[gb][WT == GGML_TYPE_Q4_K ? 0 : 2 * (s % 4) + kk][tile_col(j) + 4 * g];
                        const float d4[4] = {dx.x, dx.y, dx.z, dx.w};
                        float s4[4];
                        if constexpr (WT == GGML_TYPE_Q4_K) *(float4 *) s4 = *(const float4 *) &L.xs[gb][2 * (s % 4) + kk][tile_col(j) + 4 * g];
#pragma unroll
                        for (int i = 0; i < NR; i++) {
                            const moe_v4f p = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[j], wf[i], zero, 0, 0, 0);
#pragma unroll
                            for (int v = 0; v < 4; v++) {
                                acc[i][j][v] = fmaf(p[v], dw[i] * d4[v], acc[i][j][v]);
                                if constexpr (WT == GGML_TYPE_Q4_K) acc[i][j][v] = fmaf(mw[i], s4[v], acc[i][j][v]);
                            }
                        }
                    }
                }
            }
        };
        // Two steps in flight: a step's products take a fraction of a load's way.
        // (The loads past the last step are the last step's again: one that may
        // not have been made would be waited for with all later ones. Quantized
        // weights at 128 columns have the registers for one: a second one spilled 34
        // of them for Q4_K, 46 for Q8_0.)
        constexpr int kAhead = kQ && BN == 128 ? 1 : 2;
        stage s0, s1;
        load(0, s0);
        if constexpr (kAhead == 2) load(min((int64_t) 1, steps - 1), s1);
        if constexpr (!kQ) {
            // A half step's operands are read under the products of the one
            // before: the second half's at the step's start, the next step's first
            // half's after the barrier in its middle, by which that step is staged.
            struct half_step {
                moe_v8h w[NR], x[C];
            };
            auto read = [&](int b, int kk, half_step & f) {
#pragma unroll
                for (int j = 0; j < C; j++)
                    f.x[j] = __builtin_bit_cast(moe_v8h, *moe_slot(L.x[b], tile_col(j) + r, 4 * kk + g));
#pragma unroll
                for (int i = 0; i < NR; i++)
                    f.w[i] = __builtin_bit_cast(moe_v8h, *moe_slot(L.w[b], tile_row(i) + r, 4 * kk + g));
            };
            auto products = [&](const half_step & f) {
#pragma unroll
                for (int i = 0; i < NR; i++)
#pragma unroll
                    for (int j = 0; j < C; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.x[j], f.w[i], acc[i][j], 0, 0, 0);
            };
            half_step f0, f1;
            store(0, 0, s0);
            __syncthreads();
            load(min((int64_t) 2, steps - 1), s0);
            read(0, 0, f0);
            // step s of buffer b; `next` holds step s + 1
            auto step = [&](int64_t s, int b, stage & next) {
                read(b, 1, f1);
                store(b ^ 1, min(s + 1, steps - 1), next);
                products(f0);
                __syncthreads();
                load(min(s + 3, steps - 1), next);
                read(b ^ 1, 0, f0);
                products(f1);
            };
            for (int64_t s = 0;;) {
                step(s, 0, s1);
                if (++s >= steps) break;
                step(s, 1, s0);
                if (++s >= steps) break;
            }
        } else {
            moe_scales<WT> sc;
            load_scales(0, sc);
            // step s: its scales first, where four begin; the next four's loads
            // then have four steps
            auto scales = [&](int64_t s) {
                if (s % 4 != 0) return;
                store_scales(NB == 2 ? (int) (s / 4 & 1) : 0, sc);
                load_scales(s + 4 < steps ? s + 4 : 0, sc);
            };
            if constexpr (kAhead == 1) {
                for (int64_t s = 0; s < steps; s++) {
                    scales(s);
                    store(0, s, s0);
                    __syncthreads();
                    load(min(s + 1, steps - 1), s0);
                    multiply(0, s);
                    __syncthreads();  // the step's operands are read
                }
            } else {
                for (int64_t s = 0;;) {
                    scales(s);
                    store(0, s, s0);
                    __syncthreads();  // the step is staged; the buffer of the step before is free
                    load(min(s + 2, steps - 1), s0);
                    multiply(0, s);
                    if (++s >= steps) break;
                    store(1, s, s1);
                    __syncthreads();
                    load(min(s + 2, steps - 1), s1);
                    multiply(1, s);
                    if (++s >= steps) break;
                }
            }
        }
    };
    switch (kQ ? (n + 31) / 32 : NC) {
        case 1: products_of(std::integral_constant<int, 1>{}); break;
        case 2: products_of(std::integral_constant<int, NC < 2 ? NC : 2>{}); break;
        case 3: products_of(std::integral_constant<int, NC < 3 ? NC : 3>{}); break;
        default: products_of(std::integral_constant<int, NC>{}); break;
    }
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int c = tile_col(j) + 4 * g + v;
            if (c >= n) continue;
            float * o = a.out + (int64_t) L.pair[c] * a.M;
            if constexpr (PAIR) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int64_t m = m0 + 32 * wr + 16 * i + r;
                    if (m < a.M) o[m] = moe_swiglu(acc[i][j][v], acc[i + 2][j][v]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    const int64_t m = m0 + 64 * wr + 16 * i + r;
                    if (m < a.M) o[m] = acc[i][j][v];
                }
            }
        }
}

// ------------------------------------------------------ the slots' sum ---

// out[m, t] = sum over a token's slots, in order, of w[slot, t] y[m, slot, t];
// four rows a thread, four slots' loads in flight (700 tokens of 8 x 2048: 8.7 us,
// 5.9 TB/s)
template <bool VEC>
__global__ __launch_bounds__(256) void k_moe_sum(moe_sum_args a) {
    const int64_t m = ((int64_t) blockIdx.x * 256 + threadIdx.x) * 4;
    if (m >= a.M) return;
    const int left = (int) min((int64_t) 4, a.M - m);
    for (int64_t t = blockIdx.y; t < a.tokens; t += gridDim.y) {
        const float * y = a.y + t * a.used * a.M + m;
        const char * wp = a.w + t * a.w_nb2;
        float s[4] = {0, 0, 0, 0};
        for (int64_t k0 = 0; k0 < a.used; k0 += 4) {
            float v[4][4], w[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int64_t k = k0 + u < a.used ? k0 + u : k0;
                w[u] = a.w ? *(const float *) (wp + k * a.w_nb1) : 1.0f;
                if constexpr (VEC) *(float4 *) v[u] = *(const float4 *) (y + k * a.M);
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) v[u][e] = y[k * a.M + min(e, left - 1)];
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (k0 + u < a.used)  // (the first slot's product as it is: 0 + -0 would be 0)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[e] = k0 + u == 0 ? v[u][e] * w[u] : s[e] + v[u][e] * w[u];
        }
        float * o = a.out + t * a.M + m;
        if constexpr (VEC) *(float4 *) o = *(const float4 *) s;
        else
            for (int e = 0; e < left; e++) o[e] = s[e];
    }
}

void launch_moe_sum(const moe_sum_args & a, hipStream_t s) {
    if (a.M == 0 || a.tokens == 0) return;
    const bool vec = a.M % 4 == 0 && (((uintptr_t) a.y | (uintptr_t) a.out) & 15) == 0;
    const dim3 grid((unsigned) ((a.M + 1023) / 1024), (unsigned) (a.tokens < 65535 ? a.tokens : 65535));
    if (vec) hipLaunchKernelGGL(k_moe_sum<true>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_moe_sum<false>, grid, dim3(256), 0, s, a);
}

// ------------------------------------------------------------- launches ---

// whether the matrix-core forms read these operands: 16-byte pieces of rows
static bool moe_aligned(int wtype, const mul_mat_id_args & a) {
    const uintptr_t w = (uintptr_t) a.W | (uintptr_t) a.W2 | (uintptr_t) a.W_nb2;
    if (((uintptr_t) a.b | (uintptr_t) a.b_nb1 | (uintptr_t) a.b_nb2) & 15) return false;
    if (wtype == GGML_TYPE_F16) return a.K % 8 == 0 && ((w | (uintptr_t) a.W_nb1) & 15) == 0;
    return wtype == GGML_TYPE_Q8_0 || (wtype == GGML_TYPE_Q4_K && (w & 15) == 0);
}

// Up to how many pairs the streaming form is the faster one. 64 experts, 768 x
// 1024 weights, SwiGLU pairs, with the call, streaming / wide: f16 128 pairs
// 48 / 52 us, 256 55 / 54; Q4_K 32 pairs 26 / 38, 256 52 / 63; Q8_0 (whose
// blocks' scales it applies one by one) 32 pairs 38 / 38, 48 41 / 39, 128 65 / 57.
static int moe_few_pairs(int wtype) { return wtype == GGML_TYPE_Q8_0 ? 32 : kMoeFew; }

bool mul_mat_id_wide(int wtype, const mul_mat_id_args & a) {
    return moe_aligned(wtype, a) && a.pairs > moe_few_pairs(wtype) && a.experts <= 960 && a.pairs < 1 << 26 &&
           (a.K + 63) / 64 * 64 * a.b_ne1 * (a.pairs / a.used) < 1ll << 31;
}

static bool moe_few(int wtype, const mul_mat_id_args & a) {
    return moe_aligned(wtype, a) && a.pairs <= kMoeFew && !mul_mat_id_wide(wtype, a);
}

bool mul_mat_id_pairs(int wtype, const mul_mat_id_args & a) { return moe_few(wtype, a) || mul_mat_id_wide(wtype, a); }

static size_t moe_carve(int wtype, const mul_mat_id_args & a, moe_wide_args & q, char * base) {
    q.a = a;
    // (32 experts, 768 x 1024, pairs an expert: f16 16 28 / 32 us with 32 / 128
    // columns; 32 of all types 1 or 2 us for 32; 48 Q4_K 56 / 50, the others even)
    q.bn = a.pairs >= 40 * a.experts ? 128 : 32;
    q.kp = (a.K + 63) / 64 * 64;
    q.bcols = a.b_ne1 * (a.pairs / a.used);
    q.row_tiles = (a.M + (a.W2 ? 64 : 128) - 1) / (a.W2 ? 64 : 128);
    const int64_t runs = a.experts + 1 < a.pairs ? a.experts + 1 : a.pairs;
    q.max_tiles = (int) (a.pairs / q.bn + runs);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char * p = base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    q.head = (int *) take(256);
    q.tiles = (int4 *) take((size_t) q.max_tiles * 16);
    q.sorted = (int *) take((size_t) a.pairs * 4);
    q.x = (_Float16 *) take((size_t) (q.bcols * q.kp) * 2);
    if (wtype == GGML_TYPE_Q8_0) q.xd = (float *) take((size_t) (q.bcols * (q.kp / 32)) * 4);
    if (wtype == GGML_TYPE_Q4_K) {
        q.xd = (float *) take((size_t) (q.bcols * (q.kp / 256)) * 4);
        q.xs = (float *) take((size_t) (q.bcols * (q.kp / 32)) * 4);
    }
    return at;
}

size_t mul_mat_id_scratch_bytes(int wtype, const mul_mat_id_args & a) {
    moe_wide_args q{};
    return mul_mat_id_wide(wtype, a) ? moe_carve(wtype, a, q, nullptr) : 0;
}

template <int WT>
static void launch_moe_wide(const mul_mat_id_args & a, char * scratch, hipStream_t s) {
    moe_wide_args q{};
    moe_carve(WT, a, q, scratch);
    const int64_t waves = (q.kp + 255) / 256 * q.bcols;
    hipLaunchKernelGGL(k_moe_prepare<WT>, dim3((unsigned) ((waves + 15) / 16 + 1)), dim3(1024),
                       (size_t) (16 * (a.experts + 1)) * 4, s, q);
    const unsigned grid = (unsigned) (q.max_tiles * ((q.row_tiles + 7) / 8 * 8));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, q); };
    if (q.bn == 128) a.W2 ? go(k_moe_gemm<WT, true, 128>) : go(k_moe_gemm<WT, false, 128>);
    else a.W2 ? go(k_moe_gemm<WT, true, 32>) : go(k_moe_gemm<WT, false, 32>);
}

void launch_mul_mat_id(int wtype, const mul_mat_id_args & args, void * scratch, hipStream_t s) {
    mul_mat_id_args a = args;
    if (a.M == 0 || a.pairs == 0) return;
    a.used_inv = a.used == 1 ? 0xFFFFFFFFu : (uint32_t) ((1ull << 32) / (uint64_t) a.used);
    if (mul_mat_id_wide(wtype, a)) {
        if (wtype == GGML_TYPE_Q8_0) launch_moe_wide<GGML_TYPE_Q8_0>(a, (char *) scratch, s);
        else if (wtype == GGML_TYPE_Q4_K) launch_moe_wide<GGML_TYPE_Q4_K>(a, (char *) scratch, s);
        else launch_moe_wide<GGML_TYPE_F16>(a, (char *) scratch, s);
        return;
    }
    if (moe_few(wtype, a)) {
        const dim3 grid((unsigned) ((a.M + 15) / 16), (unsigned) a.pairs);
        auto go = [&](auto one, auto pair) {
            if (a.W2) hipLaunchKernelGGL(pair, grid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL(one, grid, dim3(256), 0, s, a);
        };
        if (wtype == GGML_TYPE_Q8_0) go(k_moe_few<GGML_TYPE_Q8_0, false>, k_moe_few<GGML_TYPE_Q8_0, true>);
        else if (wtype == GGML_TYPE_Q4_K) go(k_moe_few<GGML_TYPE_Q4_K, false>, k_moe_few<GGML_TYPE_Q4_K, true>);
        else go(k_moe_few<GGML_TYPE_F16, false>, k_moe_few<GGML_TYPE_F16, true>);
        return;
    }
    // F32 weights, and rows without 16-byte pieces
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

// Sorted ascending by (key, index), descending turns the keys' bits: a
// workgroup a row, a bitonic sort of 64-bit (key, index) in LDS. 4096 rows of
// 128 take 10 us; counting each element's predecessors from LDS instead, a wave a
// row, took 13 us there and 38 us for rows of 256 (here 18 us).
constexpr int kArgsortMost = 8192;
__global__ __launch_bounds__(1024) void k_argsort(tview d, tview a, uint32_t flip, int size, int64_t rows) {
    extern __shared__ uint64_t k[];  // [size]
    const int threads = (int) blockDim.x;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
        const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
        int32_t * o = (int32_t *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]);
        const int n = (int) a.ne[0], tid = threadIdx.x;
        for (int i = tid; i < size; i += threads) k[i] = i < n ? (uint64_t) (sort_key(x[i]) ^ flip) << 32 | (uint32_t) i : ~0ull;
        for (int run = 2; run <= size; run *= 2) {
            for (int step = run / 2; step > 0; step /= 2) {
                __syncthreads();
                for (int i = tid; i < size / 2; i += threads) {
                    const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                    const uint64_t u = k[lo], v = k[hi];
                    if ((u > v) == ((lo & run) == 0)) k[lo] = v, k[hi] = u;
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < n; i += threads) o[i] = (int32_t) (uint32_t) k[i];
        __syncthreads();
    }
}

// workgroups of four rows, each in turn where there are more
static unsigned row_blocks(int64_t rows) { return (unsigned) std::min<int64_t>((rows + 3) / 4, 1 << 22); }

bool argsort_supported(int64_t n) { return n >= 0 && n <= kArgsortMost; }

void launch_argsort(const tview & d, const tview & a, int desc, hipStream_t s) {
    const int64_t rows = a.ne[1] * a.ne[2] * a.ne[3];
    if (rows == 0 || a.ne[0] == 0) return;
    const uint32_t flip = desc ? 0xFFFFFFFFu : 0;
    int size = 2;
    while (size < a.ne[0]) size *= 2;
    hipLaunchKernelGGL(k_argsort, dim3((unsigned) std::min<int64_t>(rows, 1 << 20)), dim3(std::min(1024, std::max(64, size / 2))),
                       (size_t) size * 8, s, d, a, flip, size, rows);
}

// ------------------------------------------------------------ a router ---

// the largest of the wave's values, by adjacent lanes, rows of 16 and halves
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto with = [&](int got) { v = max(v, (uint32_t) got); };
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x112, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x114, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x118, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
    with(__builtin_amdgcn_update_dpp(0, (int) v, 0x143, 0xc, 0xf, false));
    return (uint32_t) __builtin_amdgcn_readlane((int) v, 63);
}

// The first k places of a descending ARGSORT and what a router does with
// them: the k values, their softmax, or their shares of their sum. A wave a
// row, V adjacent values a lane: k times the largest key left, of the lowest
// lane that holds it; then lane j has the j-th. The epilogues are SOFT_MAX's
// and SUM_ROWS' and DIV's operations in their order. 4096 rows of 128, 8 of
// each: 6 us (the sort, GET_ROWS and SOFT_MAX: 10 + 5 + 4); a row: 3 us. With
// the call, 4096 rows of 1024: 27 us for 8, 46 for 32, the sort 97; a row: 17,
// 26 and 25.
template <int V>
__global__ __launch_bounds__(256) void k_top_k(top_k_args a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t row = (int64_t) blockIdx.x * 4 + wave; row < a.rows; row += (int64_t) gridDim.x * 4) {
        const float * x = (const float *) (a.x + row * a.x_nb1);
        uint32_t key[V], most = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = lane * V + v;
            key[v] = i < a.n ? sort_key(x[i]) : 0;  // (no value has the key 0)
            most = max(most, key[v]);
        }
        int mine = 0;
        for (int j = 0; j < a.k; j++) {
            const uint32_t top = wave_max_u32(most);
            const int from = __ffsll((unsigned long long) __ballot(most == top)) - 1;
            int at = 0;
            if (lane == from) {
                most = 0;
                bool taken = false;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    if (!taken && key[v] == top) {
                        taken = true;
                        at = v;
                        key[v] = 0;
                    }
                    most = max(most, key[v]);
                }
            }
            at = __builtin_amdgcn_readlane(at, from);
            if (lane == j) mine = from * V + at;
        }
        if (lane < a.k) *(int32_t *) (a.ids + row * a.ids_nb1 + 4 * lane) = mine;
        if (!a.out) continue;
        const float w = lane < a.k ? x[mine] : 0.0f;
        float y = w;
        if (a.mode == kTopKSoftMax) {
            const float z = w * a.scale + 0.0f, mx = wave_max(lane < a.k ? z : -INFINITY);
            const float e = lane < a.k ? expf_det(z - mx) : 0.0f;
            y = e * (float) (1.0 / wave_sum_d((double) e));
        } else if (a.mode == kTopKShares) {
            y = w / (float) wave_sum_d((double) w);
        }
        if (lane < a.k) a.out[row * a.k + lane] = y;
    }
}

bool top_k_supported(int64_t n, int64_t k) { return n >= 1 && n <= 1024 && k >= 1 && k <= 32 && k <= n; }

void launch_top_k(const top_k_args & a, hipStream_t s) {
    if (a.rows == 0) return;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(row_blocks(a.rows)), dim3(256), 0, s, a);
    };
    if (a.n <= 64) go(k_top_k<1>);
    else if (a.n <= 128) go(k_top_k<2>);
    else if (a.n <= 256) go(k_top_k<4>);
    else if (a.n <= 512) go(k_top_k<8>);
    else go(k_top_k<16>);
}

// one wave a row, the sum held in double
__global__ __launch_bounds__(256) void k_sum_rows(tview d, tview a, int64_t rows) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t) gridDim.x * 4) {
        const int64_t i1 = row % a.ne[1], i2 = row / a.ne[1] % a.ne[2], i3 = row / (a.ne[1] * a.ne[2]);
        const float * x = (const float *) (a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3]);
        double sum = 0.0;
        for (int64_t i = lane; i < a.ne[0]; i += 64) sum += (double) x[i];
        sum = wave_sum_d(sum);
        if (lane == 0) *(float *) (d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3]) = (float) sum;
    }
}

void launch_sum_rows(const tview & d, const tview & a, hipStream_t s) {
    const int64_t rows = a.ne[1] * a.ne[2] * a.ne[3];
    if (rows == 0) return;
    hipLaunchKernelGGL(k_sum_rows, dim3(row_blocks(rows)), dim3(256), 0, s, d, a, rows);
}

}  // namespace mi355x
