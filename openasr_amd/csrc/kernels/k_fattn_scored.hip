// k_fattn_scored.hip -- GGML_OP_FLASH_ATTN_EXT whose scores are more than a
// product and a mask: capped by a tanh (logit_softcap), biased by distance
// (max_bias: the mask times a slope a head), masked a head each; and any
// attention with heads of 256 or other group sizes than the kernels before
// take. One definition at either precision:
//     s = (f16(q) . k) scale;  s <- cap tanh(s / cap);  s <- s + slope mask
//     p = exp(s - max s),  out = sum p v / sum p  (0 where nothing is seen)
// in f32, products of f16 (exact in f32), p as the sum of two f16 (22 bits: a
// single one would leave the result 11).
//
// Work: a workgroup of four waves owns R = 64 RW rows -- R / g queries times
// the g query heads of a kv head -- and walks the open 64-position tiles of its
// split of the span; wave w owns rows 16 RW w .. of them, RW = 2 reading every
// K and V fragment once for 32 rows (16 rows a wave read 98 of the 128 bytes a
// cycle that LDS gives). MFMA 16x16x32 layouts: A lane l = row l % 16, k 8 (l /
// 16) .. + 7; B lane l = column l % 16, the same k; result lane l = rows 4 (l /
// 16) .. + 3, column l % 16. Scores are made transposed (rows = positions), so
// a lane holds 16 positions of a row and its p are the P V product's own B
// operand, V^T read in the same order of positions.
//
// A first launch looks at the mask once for all heads: which tiles a block of
// queries sees at all, which of them have no masked or no nonzero entry, and
// which positions some query sees.
//
// What bounds it: a score takes about 16 vector instructions beside its MFMA
// time (the cap 7: a polynomial of (s / cap)^2; 1 mask, 2 maximum and
// subtraction, a quarter-rate exponential, 2 for the halves of p).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../fattn_scored_dev.h"
#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

namespace {

constexpr int kFsTile = 64;
constexpr int kFsThreads = 256;
// p is scaled by 2^12: its low half stays a normal f16 down to 2^-15 of the maximum
constexpr float kFsUp = 12.0f;

typedef _Float16 fs_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 fs_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 fs_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t fs_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t fs_u2 __attribute__((ext_vector_type(2)));

// a tile of a query block: nothing seen; seen, and all entries zero; seen, no
// entry -inf; seen, some entry -inf (or past the span)
enum : uint8_t { kFsClosed = 0, kFsPlain = 1, kFsAdds = 2, kFsMixed = 3 };

struct fs_args {
    fattn_args a;
    fs_score score;
    int g, qpw;       // query heads a kv head, queries a workgroup
    int q_blocks, n_tiles, split, per;
    int heads_mask;   // the mask differs by head: rows of it by query and head
    uint64_t * seen;  // [mask sequence][kv head or one][query block][tile]
    uint8_t * cls;
    float * part;
    float * out;
};

// eight mask entries at pos of a row, -inf past the span
template <bool V16>
__device__ __forceinline__ fs_u4 fs_mask8(const uint16_t * row, int pos, int n_kv) {
    fs_u4 m;
    if constexpr (V16) {
        m = *(const fs_u4 *) (row + min(pos, (n_kv - 1) & ~7));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            m[j] = (uint32_t) row[min(pos + 2 * j, n_kv - 1)] | ((uint32_t) row[min(pos + 2 * j + 1, n_kv - 1)] << 16);
    }
    if (pos + 8 > n_kv) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (pos + 2 * j >= n_kv) m[j] = (m[j] & 0xFFFF0000u) | kFsNegInf;
            if (pos + 2 * j + 1 >= n_kv) m[j] = (m[j] & 0xFFFFu) | (kFsNegInf << 16);
        }
    }
    return m;
}

__device__ __forceinline__ const char * fs_mask_of(const fattn_args & a, int seq, int head) {
    return a.mask + (int64_t) (seq % a.m_ne3) * a.m_nb3 + (int64_t) (head % a.m_ne2) * a.m_nb2;
}

// one wave a tile of a query block: lane = 8-position piece l % 8 of rows l / 8, + 8 ..
template <bool V16>
__global__ __launch_bounds__(256) void k_fattn_tiles(fs_args f, int64_t units) {
    const fattn_args & a = f.a;
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const int tile = (int) (u % f.n_tiles), qb = (int) (u / f.n_tiles % f.q_blocks);
    const int64_t hs = u / ((int64_t) f.n_tiles * f.q_blocks);
    const int kinds = f.heads_mask ? a.hkv : 1, kvh = (int) (hs % kinds), ms = (int) (hs / kinds);
    const int q0 = qb * f.qpw, nq = min(f.qpw, a.n_q - q0), heads = f.heads_mask ? f.g : 1, rows = nq * heads;
    const int c = lane & 7, pos = tile * kFsTile + 8 * c;
    uint32_t open = 0, closed = 0, adds = 0;
    for (int r0 = lane >> 3; r0 < rows; r0 += 32) {
        fs_u4 m[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int r = min(r0 + 8 * k, rows - 1);
            m[k] = fs_mask8<V16>((const uint16_t *) (fs_mask_of(a, ms, kvh * f.g + r % heads) + (int64_t) (q0 + r / heads) * a.m_nb1), pos, a.n_kv);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool lo = (m[k][j] & 0xFFFFu) == kFsNegInf, hi = (m[k][j] >> 16) == kFsNegInf;
                open |= (lo ? 0u : 1u << (2 * j)) | (hi ? 0u : 2u << (2 * j));
                closed |= lo || hi;
                adds |= m[k][j] & 0x7FFF7FFFu;  // (-0 adds as 0)
            }
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) open |= __shfl_xor(open, o);
    uint64_t seen = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) seen |= (uint64_t) (uint32_t) __shfl(open, k) << (8 * k);
    const bool any_closed = __any(closed != 0), any_adds = __any(adds != 0);
    if (lane == 0) {
        f.seen[u] = seen;
        f.cls[u] = !seen ? kFsClosed : any_closed ? kFsMixed : any_adds ? kFsAdds : kFsPlain;
    }
}

// whether one of eight f16 is infinite or NaN
__device__ __forceinline__ bool fs_odd(fs_u4 v) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; j++) odd |= (v[j] & 0x7C00u) == 0x7C00u || (v[j] & 0x7C000000u) == 0x7C000000u;
    return odd;
}

__device__ __forceinline__ fs_f4 fs_mfma(fs_h8 a, fs_h8 b, fs_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// MM: 0 no mask, 1 rows of 16-byte pieces, 2 other rows
template <int D, int RW, bool CAP, int MM>
__global__ __launch_bounds__(kFsThreads, D == 256 ? 1 : 2) void k_fattn_scored(fs_args f) {
    constexpr int R = 64 * RW;                            // rows of a workgroup
    constexpr int KS = D / 32, NT = D / 16;
    constexpr int KP = D + 8, VP = kFsTile + 8, MP = kFsTile + 8;
    constexpr int PC = D / 8;                             // 16-byte pieces of a K / V row
    constexpr int KLD = kFsTile * PC / kFsThreads, VLD = KLD / 2;
    constexpr int MLD = MM ? R * 8 / kFsThreads : 1;
    __shared__ __align__(16) _Float16 s_k[kFsTile][KP];
    __shared__ __align__(16) _Float16 s_vt[D][VP];
    __shared__ __align__(16) uint16_t s_m[MM ? R : 1][MP];
    __shared__ unsigned long long s_bad;                  // positions of the tile whose V is not finite
    const fattn_args & a = f.a;
    const int tid = (int) threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, lg = lane >> 4;
    // Workgroup b runs on XCD b % 8: an XCD takes a contiguous run of (split,
    // query block, kv head, sequence), so that those which read the same K and
    // V share an L2; the last query blocks, whose causal span is the longest, first
    const int n_blk = (int) gridDim.x;
    int b = (int) blockIdx.x;
    if (n_blk % 8 == 0) b = (b % 8) * (n_blk / 8) + b / 8;
    const int z = b % f.split;
    const int qb = f.q_blocks - 1 - b / f.split % f.q_blocks, hs = b / f.split / f.q_blocks;
    const int kvh = hs % a.hkv, seq = hs / a.hkv, kv_seq = seq / a.rk3;
    const int q0 = qb * f.qpw, nq = min(f.qpw, a.n_q - q0);
    const int mheads = f.heads_mask ? f.g : 1, mrows = nq * mheads;
    const char * kbase = a.k + (int64_t) kvh * a.k_nb2 + (int64_t) kv_seq * a.k_nb3;
    const char * vbase = a.v + (int64_t) kvh * a.v_nb2 + (int64_t) kv_seq * a.v_nb3;
    const int t_begin = z * f.per, t_end = min(f.n_tiles, t_begin + f.per);
    const int64_t tile0 = MM ? ((int64_t) ((seq % a.m_ne3) * (f.heads_mask ? a.hkv : 1) + (f.heads_mask ? kvh : 0)) * f.q_blocks + qb) * f.n_tiles : 0;
    auto class_of = [&](int t) -> int {
        if constexpr (MM != 0) return f.cls[tile0 + t];
        else return (t + 1) * kFsTile <= a.n_kv ? kFsPlain : kFsMixed;
    };
    auto next_open = [&](int t) {
        if constexpr (MM != 0) {
            while (t < t_end && f.cls[tile0 + t] == kFsClosed) t++;
        }
        return t;
    };

    fs_u4 kr[KLD], vr[VLD][2], mr[MLD];
    auto issue = [&](int tile, int cls) {
        const int p0 = tile * kFsTile;
#pragma unroll
        for (int i = 0; i < KLD; i++) {
            const int e = tid + i * kFsThreads, p = e / PC, piece = e % PC;
            kr[i] = *(const fs_u4 *) (kbase + (int64_t) min(p0 + p, a.n_kv - 1) * a.k_nb1 + 16 * piece);
        }
#pragma unroll
        for (int i = 0; i < VLD; i++) {
            const int e = tid + i * kFsThreads, pair = e % (kFsTile / 2), piece = e / (kFsTile / 2);
#pragma unroll
            for (int h = 0; h < 2; h++)
                vr[i][h] = *(const fs_u4 *) (vbase + (int64_t) min(p0 + 2 * pair + h, a.n_kv - 1) * a.v_nb1 + 16 * piece);
        }
        if constexpr (MM != 0) {
            if (cls >= kFsAdds) {
#pragma unroll
                for (int i = 0; i < MLD; i++) {
                    const int e = tid + i * kFsThreads, r = min(e >> 3, mrows - 1), c = e & 7;
                    mr[i] = fs_mask8<MM == 1>((const uint16_t *) (fs_mask_of(a, seq, kvh * f.g + r % mheads) + (int64_t) (q0 + r / mheads) * a.m_nb1),
                                              p0 + 8 * c, a.n_kv);
                }
            }
        }
    };
    int tile = next_open(t_begin), cls = tile < t_end ? class_of(tile) : kFsClosed;
    if (tile < t_end) issue(tile, cls);

    // this lane's query rows (the score product's B operand), rounded to f16
    fs_h8 qa[RW][KS];
    float slope[RW];
    int mrow[RW];
#pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = 16 * (RW * wave + w) + l16, ql = min(r / f.g, nq - 1), head = kvh * f.g + r % f.g;
        const char * qp = a.q + (int64_t) (q0 + ql) * a.q_nb1 + (int64_t) head * a.q_nb2 + (int64_t) seq * a.q_nb3;
#pragma unroll
        for (int kk = 0; kk < KS; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) qa[w][kk][j] = (_Float16) ((const float *) qp)[32 * kk + 8 * lg + j];
        slope[w] = fs_slope(f.score, a.max_bias, head);
        mrow[w] = f.heads_mask ? min(ql * f.g + r % f.g, mrows - 1) : ql;
    }
    if (tid == 0) s_bad = 0;

    float m[RW], l[RW];
    fs_f4 o[RW][NT];
#pragma unroll
    for (int w = 0; w < RW; w++) {
        m[w] = -INFINITY, l[w] = 0.0f;
#pragma unroll
        for (int ct = 0; ct < NT; ct++) o[w][ct] = fs_f4{0, 0, 0, 0};
    }

    while (tile < t_end) {
        __syncthreads();  // the tile before has been read
#pragma unroll
        for (int i = 0; i < KLD; i++) {
            const int e = tid + i * kFsThreads;
            *(fs_u4 *) &s_k[e / PC][8 * (e % PC)] = kr[i];
        }
        uint64_t seen = ~0ull;
        if (cls == kFsMixed) {
            if constexpr (MM != 0) seen = f.seen[tile0 + tile];
            else seen = ~0ull >> ((tile + 1) * kFsTile - a.n_kv);
        }
#pragma unroll
        for (int i = 0; i < VLD; i++) {
            const int e = tid + i * kFsThreads, pair = e % (kFsTile / 2), piece = e / (kFsTile / 2);
            if (cls == kFsMixed) {
                // V rows that no query sees are zeros (0 times anything), and
                // pieces of rows that are not finite are added query by query
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const bool odd = fs_odd(vr[i][h]);
                    const bool in = (seen >> (2 * pair + h)) & 1;
                    if (in && odd) atomicOr(&s_bad, 1ull << (2 * pair + h));
                    if (!in || odd) vr[i][h] = fs_u4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                *(uint32_t *) &s_vt[8 * piece + 2 * j][2 * pair] = __builtin_amdgcn_perm(vr[i][1][j], vr[i][0][j], 0x05040100u);
                *(uint32_t *) &s_vt[8 * piece + 2 * j + 1][2 * pair] = __builtin_amdgcn_perm(vr[i][1][j], vr[i][0][j], 0x07060302u);
            }
        }
        if constexpr (MM != 0) {
            if (cls >= kFsAdds) {
#pragma unroll
                for (int i = 0; i < MLD; i++) {
                    const int e = tid + i * kFsThreads;
                    if ((e >> 3) < mrows) *(fs_u4 *) &s_m[e >> 3][8 * (e & 7)] = mr[i];
                }
            }
        }
        __syncthreads();
        const int nxt = next_open(tile + 1), nxt_cls = nxt < t_end ? class_of(nxt) : kFsClosed;
        if (nxt < t_end) issue(nxt, nxt_cls);

        // S^T = K Q^T: lane (lg, l16) gets positions 16 t + 4 lg + i of row l16
        fs_f4 sc[RW][4];
#pragma unroll
        for (int w = 0; w < RW; w++)
#pragma unroll
            for (int t = 0; t < 4; t++) sc[w][t] = fs_f4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
            fs_h8 kb[4];
#pragma unroll
            for (int t = 0; t < 4; t++) kb[t] = *(const fs_h8 *) &s_k[16 * t + l16][32 * kk + 8 * lg];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int w = 0; w < RW; w++) sc[w][t] = fs_mfma(kb[t], qa[w][kk], sc[w][t]);
        }
        fs_h8 hi[RW][2], lo[RW][2];  // p's halves, k slot 8 lg + j of step kk: position 32 kk + 16 (j / 4) + 4 lg + j % 4
        const bool odd_rows = cls == kFsMixed && s_bad != 0;
        fs_f4 pv[RW][4];
#pragma unroll
        for (int w = 0; w < RW; w++) {
            float z[4][4];
            if constexpr (CAP) {
                float most = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(sc[w][t][i]));
                if (__any(!(most * f.score.in < kFsPolyEnd))) {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) z[t][i] = fs_cap_any(f.score, sc[w][t][i] * f.score.in);
                } else {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) z[t][i] = fs_cap_small(f.score, sc[w][t][i] * f.score.in);
                }
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) z[t][i] = sc[w][t][i] * f.score.in;
            }
            if constexpr (MM != 0) {
                if (cls >= kFsAdds) {
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const fs_h4 mk = *(const fs_h4 *) &s_m[mrow[w]][16 * t + 4 * lg];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float v = (float) mk[i];
                            z[t][i] = v == -INFINITY ? -INFINITY : fmaf(v, slope[w], z[t][i]);
                        }
                    }
                }
            } else if (cls == kFsMixed) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (tile * kFsTile + 16 * t + 4 * lg + i >= a.n_kv) z[t][i] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, z[t][i]);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m[w], mx);
            const float base = mn == -INFINITY ? 0.0f : kFsUp - mn;  // a row with nothing open yet
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[w] - mn);
            m[w] = mn;
#pragma unroll
            for (int t = 0; t < 4; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) z[t][i] = __builtin_amdgcn_exp2f(z[t][i] + base);
                pv[w][t] = fs_f4{z[t][0], z[t][1], z[t][2], z[t][3]};
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const fs_h2 h = __builtin_bit_cast(fs_h2, __builtin_amdgcn_cvt_pkrtz(z[t][i], z[t][i + 1]));
                    const fs_h2 r = __builtin_bit_cast(fs_h2, __builtin_amdgcn_cvt_pkrtz(z[t][i] - (float) h[0], z[t][i + 1] - (float) h[1]));
                    hi[w][t >> 1][4 * (t & 1) + i] = h[0], hi[w][t >> 1][4 * (t & 1) + i + 1] = h[1];
                    lo[w][t >> 1][4 * (t & 1) + i] = r[0], lo[w][t >> 1][4 * (t & 1) + i + 1] = r[1];
                }
            }
            // the row's sum: a product with ones, every lane of the row's column gets it
            const fs_h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
            fs_f4 ps = {0, 0, 0, 0};
#pragma unroll
            for (int kk = 0; kk < 2; kk++) ps = fs_mfma(ones, hi[w][kk], fs_mfma(ones, lo[w][kk], ps));
            l[w] = l[w] * alpha + ps[0];
            if (__any(alpha != 1.0f)) {
#pragma unroll
                for (int ct = 0; ct < NT; ct++) o[w][ct] *= alpha;
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int ct = 0; ct < NT; ct++) {
                const _Float16 * vrow = &s_vt[16 * ct + l16][32 * kk + 4 * lg];
                const fs_h4 v0 = *(const fs_h4 *) vrow, v1 = *(const fs_h4 *) (vrow + 16);
                const fs_h8 va = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
                for (int w = 0; w < RW; w++) o[w][ct] = fs_mfma(va, hi[w][kk], fs_mfma(va, lo[w][kk], o[w][ct]));
            }
        if (odd_rows) {
            // V rows that are not finite: for the rows that see them alone
            const uint64_t bad = s_bad;
            for (int p = 0; p < kFsTile; p++) {
                if (!((bad >> p) & 1)) continue;
#pragma unroll
                for (int w = 0; w < RW; w++) {
                    float mine = 0.0f;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (t == p >> 4 && i == (p & 3)) mine = pv[w][t][i];
                    const float pp = __shfl(mine, 16 * ((p & 15) >> 2) + l16);
                    bool sees = true;
                    if constexpr (MM != 0) sees = s_m[mrow[w]][p] != kFsNegInf;
                    if (!sees) continue;
                    const char * vrow = vbase + (int64_t) (tile * kFsTile + p) * a.v_nb1;
#pragma unroll
                    for (int ct = 0; ct < NT; ct++) {
                        const fs_h8 v8 = *(const fs_h8 *) (vrow + 2 * (16 * ct + 8 * (lg >> 1)));
                        if (!fs_odd(__builtin_bit_cast(fs_u4, v8))) continue;  // it is in s_vt
#pragma unroll
                        for (int i = 0; i < 4; i++) o[w][ct][i] = fmaf(pp, (float) (lg & 1 ? v8[4 + i] : v8[i]), o[w][ct][i]);
                    }
                }
            }
            __syncthreads();
            if (tid == 0) s_bad = 0;
        }
        tile = nxt;
        cls = nxt_cls;
    }

#pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = 16 * (RW * wave + w) + l16;
        if (f.split > 1) {
            // partials of split z: O unnormalised, then (m, l), a workgroup row
            const int64_t rows = (int64_t) n_blk * R;
            const int64_t pr = (((int64_t) hs * f.q_blocks + qb) * f.split + z) * R + r;
#pragma unroll
            for (int ct = 0; ct < NT; ct++) *(fs_f4 *) &f.part[pr * D + 16 * ct + 4 * lg] = o[w][ct];
            if (lg == 0) *(float2 *) &f.part[rows * D + 2 * pr] = make_float2(m[w], l[w]);
        } else if (r / f.g < nq) {
            float * op = f.out + (((int64_t) seq * a.n_q + q0 + r / f.g) * a.hq + kvh * f.g + r % f.g) * D;
#pragma unroll
            for (int ct = 0; ct < NT; ct++) *(fs_f4 *) &op[16 * ct + 4 * lg] = l[w] != 0.0f ? o[w][ct] / l[w] : fs_f4{0, 0, 0, 0};
        }
    }
}

// A row's splits joined: LN lanes of D / 4 threads take every LN-th split, a
// thread four dims, their sums added through LDS. (A lane a row went through 78
// splits one after the other: 37 us for 80 rows of 64.)
template <int D, int LN>
__global__ __launch_bounds__(256) void k_fattn_join(fs_join f) {
    constexpr int T = D / 4 * LN, RW = 256 / T;  // threads a row, rows a workgroup
    __shared__ fs_f4 s_acc[256];
    __shared__ float2 s_ml[256];
    const int tid = (int) threadIdx.x, t = tid % T, ln = t / (D / 4), d = t % (D / 4) * 4;
    const int64_t row = (int64_t) blockIdx.x * RW + tid / T, rc = min(row, f.rows - 1);  // of (sequence, query, head)
    const int head = (int) (rc % f.hq), q = (int) (rc / f.hq % f.n_q), seq = (int) (rc / ((int64_t) f.hq * f.n_q));
    const int64_t blk = ((int64_t) seq * (f.hq / f.g) + head / f.g) * f.q_blocks + q / f.qpw;
    const int64_t p0 = blk * f.split * f.R + (q % f.qpw) * f.g + head % f.g;
    const float * ml = f.part + f.partials * D;
    float M = -INFINITY, L = 0.0f;
    fs_f4 acc = {0, 0, 0, 0};
    for (int z0 = ln; z0 < f.split; z0 += 4 * LN) {
        float2 v[4];
        fs_f4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t p = p0 + (int64_t) min(z0 + k * LN, f.split - 1) * f.R;
            v[k] = *(const float2 *) &ml[2 * p];
            x[k] = *(const fs_f4 *) &f.part[p * D + d];
        }
        float most = M;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (z0 + k * LN >= f.split) v[k] = make_float2(-INFINITY, 0.0f);
            most = fmaxf(most, v[k].x);
        }
        const float w0 = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - most);
        L *= w0, acc *= w0, M = most;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (v[k].x == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(v[k].x - most);
            L = fmaf(w, v[k].y, L);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(w, x[k][i], acc[i]);
        }
    }
    if constexpr (LN > 1) {
        s_acc[tid] = acc;
        s_ml[tid] = make_float2(M, L);
        __syncthreads();
        if (ln != 0) return;
        float most = -INFINITY;
#pragma unroll
        for (int k = 0; k < LN; k++) most = fmaxf(most, s_ml[tid + k * (D / 4)].x);
        acc = fs_f4{0, 0, 0, 0}, L = 0.0f;
#pragma unroll
        for (int k = 0; k < LN; k++) {
            const float2 v = s_ml[tid + k * (D / 4)];
            if (v.x == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(v.x - most);
            L = fmaf(w, v.y, L);
            const fs_f4 x = s_acc[tid + k * (D / 4)];
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(w, x[i], acc[i]);
        }
    }
    if (row < f.rows) *(fs_f4 *) &f.out[row * D + d] = L != 0.0f ? acc / L : fs_f4{0, 0, 0, 0};
}

size_t fs_al(size_t v) { return (v + 255) & ~(size_t) 255; }

int fs_rw(const fattn_args & a) {
    // rows of a workgroup: 128, where a kv head has more than 64
    return a.d != 256 && (int64_t) a.n_q * (a.hq / a.hkv) > 64 ? 2 : 1;
}

// the launch's shape, and its scratch: the tiles' classes, then the splits' partials
size_t fs_plan(const fattn_args & a, fs_args & f) {
    f = fs_args{};
    f.a = a;
    const int R = 64 * fs_rw(a);
    f.g = a.hq / a.hkv;
    f.qpw = std::min(R / f.g, a.n_q);
    f.q_blocks = (a.n_q + f.qpw - 1) / f.qpw;
    f.n_tiles = (a.n_kv + kFsTile - 1) / kFsTile;
    f.split = std::max(1, a.scored_split);
    f.per = (f.n_tiles + f.split - 1) / f.split;
    f.split = (f.n_tiles + f.per - 1) / f.per;
    f.heads_mask = a.mask && a.m_ne2 > 1;
    f.score = fs_score_of(a);
    size_t need = 0;
    if (a.mask) {
        const size_t n = (size_t) a.m_ne3 * (f.heads_mask ? a.hkv : 1) * f.q_blocks * f.n_tiles;
        need = fs_al(8 * n) + fs_al(n);
    }
    if (f.split > 1) need += sizeof(float) * (size_t) a.n_seq * a.hkv * f.q_blocks * f.split * R * (a.d + 2);
    return need;
}

}  // namespace

bool fattn_scored_supported(const fattn_args & a) {
    const int g = a.hkv > 0 ? a.hq / a.hkv : 0;
    const bool aligned = (a.k_nb1 | a.k_nb2 | a.k_nb3 | a.v_nb1 | a.v_nb2 | a.v_nb3) % 16 == 0;
    return (a.d == 64 || a.d == 128 || a.d == 256) && g >= 1 && g <= 64 && a.n_kv > 0 && aligned;
}

void fattn_scored_plan(fattn_args & a, int n_cu) {
    if (fattn_scored_dec_supported(a)) return fattn_scored_dec_plan(a, n_cu);
    // splits of the span while one sequence's query blocks leave CUs idle: two
    // workgroups a CU, at least four tiles a split. By one sequence's shape, so
    // that its rows get the same bits alone or in a batch
    const int R = 64 * fs_rw(a), g = a.hq / a.hkv, qpw = std::min(R / g, std::max(1, a.n_q));
    const int64_t base = (int64_t) ((a.n_q + qpw - 1) / qpw) * a.hkv;
    const int n_tiles = (a.n_kv + kFsTile - 1) / kFsTile;
    a.scored = 1;
    a.scored_split = (int) std::max<int64_t>(1, std::min<int64_t>((2 * n_cu + base - 1) / std::max<int64_t>(1, base), n_tiles / 4));
}

size_t fattn_scored_scratch_bytes(const fattn_args & a) {
    if (fattn_scored_dec_supported(a)) return fattn_scored_dec_scratch_bytes(a);
    fs_args f;
    return fs_plan(a, f);
}

void launch_fattn_scored(const fattn_args & a, void * scratch, float * out, hipStream_t s) {
    if (a.n_q == 0 || a.n_seq == 0) return;
    if (fattn_scored_dec_supported(a)) return launch_fattn_scored_dec(a, scratch, out, s);
    fs_args f;
    fs_plan(a, f);
    f.out = out;
    char * p = (char *) scratch;
    const bool v16 = (((uintptr_t) a.mask | (uintptr_t) a.m_nb1 | (uintptr_t) a.m_nb2 | (uintptr_t) a.m_nb3) & 15) == 0;
    if (a.mask) {
        const int64_t n = (int64_t) a.m_ne3 * (f.heads_mask ? a.hkv : 1) * f.q_blocks * f.n_tiles;
        f.seen = (uint64_t *) p;
        f.cls = (uint8_t *) (p + fs_al(8 * (size_t) n));
        p += fs_al(8 * (size_t) n) + fs_al((size_t) n);
        const dim3 grid((unsigned) ((n + 3) / 4));
        if (v16) hipLaunchKernelGGL(k_fattn_tiles<true>, grid, dim3(256), 0, s, f, n);
        else hipLaunchKernelGGL(k_fattn_tiles<false>, grid, dim3(256), 0, s, f, n);
        note_hip_error(hipGetLastError());
    }
    f.part = (float *) p;
    const int rw = fs_rw(a);
    const dim3 grid((unsigned) ((int64_t) f.q_blocks * a.hkv * a.n_seq * f.split));
    auto go = [&](auto d, auto w, auto cap) {
        constexpr int D = decltype(d)::value, RW = decltype(w)::value;
        constexpr bool CAP = decltype(cap)::value;
        if (!a.mask) hipLaunchKernelGGL((k_fattn_scored<D, RW, CAP, 0>), grid, dim3(kFsThreads), 0, s, f);
        else if (v16) hipLaunchKernelGGL((k_fattn_scored<D, RW, CAP, 1>), grid, dim3(kFsThreads), 0, s, f);
        else hipLaunchKernelGGL((k_fattn_scored<D, RW, CAP, 2>), grid, dim3(kFsThreads), 0, s, f);
    };
    auto rows = [&](auto d, auto w) {
        if (a.softcap > 0.0f) go(d, w, std::true_type{});
        else go(d, w, std::false_type{});
    };
    using one = std::integral_constant<int, 1>;
    using two = std::integral_constant<int, 2>;
    if (a.d == 256) rows(std::integral_constant<int, 256>{}, one{});
    else if (a.d == 128 && rw == 2) rows(std::integral_constant<int, 128>{}, two{});
    else if (a.d == 128) rows(std::integral_constant<int, 128>{}, one{});
    else if (rw == 2) rows(std::integral_constant<int, 64>{}, two{});
    else rows(std::integral_constant<int, 64>{}, one{});
    note_hip_error(hipGetLastError());
    if (f.split > 1) {
        fs_join j{};
        j.part = f.part, j.out = out, j.rows = (int64_t) a.n_seq * a.n_q * a.hq;
        j.partials = (int64_t) a.n_seq * a.hkv * f.q_blocks * f.split * 64 * rw;
        j.split = f.split, j.d = a.d, j.hq = a.hq, j.n_q = a.n_q, j.g = f.g, j.qpw = f.qpw, j.q_blocks = f.q_blocks, j.R = 64 * rw;
        launch_fattn_join(j, s);
    }
}

void launch_fattn_join(const fs_join & j, hipStream_t s) {
    auto go = [&](auto d, auto ln) {
        constexpr int D = decltype(d)::value, LN = decltype(ln)::value, RW = 256 / (D / 4 * LN);
        hipLaunchKernelGGL((k_fattn_join<D, LN>), dim3((unsigned) ((j.rows + RW - 1) / RW)), dim3(256), 0, s, j);
    };
    auto lanes = [&](auto d) {
        if (j.split > 8) go(d, std::integral_constant<int, 4>{});
        else go(d, std::integral_constant<int, 1>{});
    };
    if (j.d == 64) lanes(std::integral_constant<int, 64>{});
    else if (j.d == 128) lanes(std::integral_constant<int, 128>{});
    else lanes(std::integral_constant<int, 256>{});
    note_hip_error(hipGetLastError());
}

}  // namespace mi355x
