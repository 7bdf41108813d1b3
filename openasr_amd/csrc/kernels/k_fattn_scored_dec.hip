// k_fattn_scored_dec.hip -- GGML_OP_FLASH_ATTN_EXT with one query position and
// capped or biased scores, masks a head, heads of 256 or any group size: the
// decode step of k_fattn_scored.hip's attention, in its arithmetic (f16 products
// in f32, the cap's polynomial, base 2 exponents, p and p V in f32).
//
// Work: a workgroup of eight waves per (sequence, kv head, up to eight of its
// query heads, KV split); wave w takes the split's tiles w, w + 8 .. of TP
// positions. A tile: K rows are the A operand straight from memory (MFMA
// 16x16x32: A lane l = row l % 16, k 8 (l / 16) .. + 7, one 16-byte load), the
// query heads the B operand's columns; the scores go through a wave's own LDS so
// that a lane has a position and G heads of it; V rows lie across lanes, D / 8 a
// row, and p is read back in their order. The waves' states are merged in LDS;
// several splits leave partials that a launch joins.
//
// K and V are read once, which bounds it.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../fattn_scored_dev.h"
#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

namespace {

constexpr int kFcWaves = 8;

typedef _Float16 fc_h8 __attribute__((ext_vector_type(8)));

struct fc_args {
    fattn_args a;
    fs_score score;
    int g, gs, groups;   // query heads a kv head, of a workgroup, workgroups a kv head
    int n_tiles, split, per;
    float * part;
    float * out;
};

__device__ __forceinline__ void fc_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// the wave's maximum and sum, in every lane: 16 lanes by DPP, then across rows
template <typename F>
__device__ __forceinline__ float fc_reduce(float v, F op) {
    auto step = [&](auto ctrl) {
        v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true)));
    };
    step(std::integral_constant<int, 0x128>{});  // row_ror:8, 4, 2, 1
    step(std::integral_constant<int, 0x124>{});
    step(std::integral_constant<int, 0x122>{});
    step(std::integral_constant<int, 0x121>{});
    v = op(v, __shfl_xor(v, 16));
    return op(v, __shfl_xor(v, 32));
}

// a wave's value that all lanes hold alike, in a scalar register
__device__ __forceinline__ float fc_uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }

// positions a tile, whose K and V rows lie in a wave's registers beside the heads' sums
constexpr int fc_tile(int d, int g) { return d == 64 ? 64 : d == 128 ? (g == 8 ? 32 : 64) : g >= 4 ? 16 : 32; }

// HM: the mask differs by head
template <int D, int G, bool HM>
__global__ __launch_bounds__(64 * kFcWaves) void k_fattn_scored_dec(fc_args f) {
    constexpr int TP = fc_tile(D, G);                    // positions a tile
    constexpr int KS = D / 32, NB = TP / 16;
    constexpr int LPR = D / 8, RPI = 64 / LPR, NV = TP / RPI;  // lanes a V row, rows a load, loads a tile
    __shared__ __align__(16) float s_sc[kFcWaves][G][TP];
    __shared__ __align__(16) float s_p[kFcWaves][G][TP];
    __shared__ __align__(16) float s_acc[kFcWaves][G][D];
    __shared__ float s_m[kFcWaves][G], s_l[kFcWaves][G];
    const fattn_args & a = f.a;
    const int lane = (int) threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), l16 = lane & 15, lg = lane >> 4;
    const int z = (int) blockIdx.x % f.split, unit = (int) blockIdx.x / f.split;
    const int hg = unit % f.groups, kvh = unit / f.groups % a.hkv, seq = unit / f.groups / a.hkv;
    const int h0 = kvh * f.g + hg * f.gs, heads = min(f.gs, f.g - hg * f.gs);
    const char * kb = a.k + (int64_t) kvh * a.k_nb2 + (int64_t) (seq / a.rk3) * a.k_nb3;
    const char * vb = a.v + (int64_t) kvh * a.v_nb2 + (int64_t) (seq / a.rk3) * a.v_nb3;
    const int t_end = min(f.n_tiles, (z + 1) * f.per);
    int tile = z * f.per + w;

    // a tile's mask entries (lane = position), as f16 bits; -inf past the span
    uint32_t mk[HM ? G : 1];
    auto load_mask = [&](int t, uint32_t (&to)[HM ? G : 1]) {
        const int pos = t * TP + (lane & (TP - 1));
        const bool in = t < t_end && pos < a.n_kv && lane < TP;
#pragma unroll
        for (int h = 0; h < (HM ? G : 1); h++) {
            uint32_t v = 0;
            if (a.mask) {
                const char * row = a.mask + (int64_t) (seq % a.m_ne3) * a.m_nb3 + (int64_t) ((h0 + min(h, heads - 1)) % a.m_ne2) * a.m_nb2;
                v = ((const uint16_t *) row)[min(pos, a.n_kv - 1)];
            }
            to[h] = in ? v : kFsNegInf;
        }
    };
    auto open_of = [&](const uint32_t (&m)[HM ? G : 1]) {
        bool open = false;
#pragma unroll
        for (int h = 0; h < (HM ? G : 1); h++) open |= m[h] != kFsNegInf;
        return __ballot(open);
    };
    uint4 kr[NB][KS], vr[NV];
    auto load_k = [&](int t) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const char * row = kb + (int64_t) min(t * TP + 16 * b + l16, a.n_kv - 1) * a.k_nb1 + 16 * lg;
#pragma unroll
            for (int s = 0; s < KS; s++) kr[b][s] = *(const uint4 *) (row + 64 * s);
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int u = 0; u < NV; u++)
            vr[u] = *(const uint4 *) (vb + (int64_t) min(t * TP + u * RPI + lane / LPR, a.n_kv - 1) * a.v_nb1 + 16 * (lane % LPR));
    };
    load_mask(tile, mk);
    const bool any = tile < t_end;
    if (any) load_k(tile), load_v(tile);  // the first tile before its mask arrives

    // the query heads as the B operand's columns, rounded to f16
    fc_h8 qb[KS];
    {
        const float * q = (const float *) (a.q + (int64_t) (h0 + min(l16, heads - 1)) * a.q_nb2 + (int64_t) seq * a.q_nb3);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) qb[s][j] = (_Float16) q[32 * s + 8 * lg + j];
    }
    float slope[G], m[G], l[G], acc[G][8];
#pragma unroll
    for (int h = 0; h < G; h++) {
        slope[h] = fc_uniform(fs_slope(f.score, a.max_bias, h0 + min(h, heads - 1)));
        m[h] = -INFINITY, l[h] = 0.0f;  // l: the lane's own positions
#pragma unroll
        for (int i = 0; i < 8; i++) acc[h][i] = 0.0f;
    }
    const bool cap = a.softcap > 0.0f;
    uint64_t open = any ? open_of(mk) : 0;
    while (tile < t_end) {
        const int nxt = tile + kFcWaves;
        uint32_t nk[HM ? G : 1];
        load_mask(nxt, nk);
        if (open) {
            // S^T = K q^T: lane (lg, l16) has positions 16 b + 4 lg + i of head l16
#pragma unroll
            for (int b = 0; b < NB; b++) {
                fs_f4 sc = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; s++)
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fc_h8, kr[b][s]), qb[s], sc, 0, 0, 0);
                if (l16 < G) *(fs_f4 *) &s_sc[w][l16 < G ? l16 : 0][16 * b + 4 * lg] = sc;
            }
        }
        const uint64_t nxt_open = open_of(nk);
        if (nxt_open) load_k(nxt);  // (K's registers are free)
        if (open) {
            fc_wave_sync();
            float p[G], alpha[G];
#pragma unroll
            for (int h = 0; h < G; h++) {
                const float x = s_sc[w][h][lane & (TP - 1)] * f.score.in;
                const float bias = half_bits_to_float((uint16_t) mk[HM ? h : 0]);
                float t = x;
                if (cap) t = __any(!(fabsf(x) < kFsPolyEnd)) ? fs_cap_any(f.score, x) : fs_cap_small(f.score, x);
                t = mk[HM ? h : 0] == kFsNegInf ? -INFINITY : fmaf(bias, slope[h], t);
                const float most = fmaxf(m[h], fc_uniform(fc_reduce(t, [](float u, float v) { return fmaxf(u, v); })));
                alpha[h] = most == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[h] - most);
                m[h] = most;
                // (below zero: not seen by this head alone)
                p[h] = __builtin_amdgcn_exp2f(t - (most == -INFINITY ? 0.0f : most));
                l[h] = fmaf(l[h], alpha[h], p[h]);
                if constexpr (HM) p[h] = mk[h] == kFsNegInf ? -1.0f : p[h];
                if (TP == 64 || lane < TP) s_p[w][h][(lane % RPI) * NV + lane / RPI] = p[h];
            }
            if (open != (TP == 64 ? ~0ull : (1ull << TP) - 1)) {
                // V rows that no head sees are zeros (0 times anything)
#pragma unroll
                for (int u = 0; u < NV; u++)
                    if (!((open >> (u * RPI + lane / LPR)) & 1)) vr[u] = make_uint4(0, 0, 0, 0);
            }
            fc_wave_sync();
#pragma unroll
            for (int h = 0; h < G; h++) {
#pragma unroll
                for (int i = 0; i < 8; i++) acc[h][i] *= alpha[h];
                const float * ph = &s_p[w][h][lane / LPR * NV];
#pragma unroll
                for (int u0 = 0; u0 < NV; u0 += 4) {
                    const fs_f4 pp = *(const fs_f4 *) (ph + u0);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t x[4] = {vr[u0 + j].x, vr[u0 + j].y, vr[u0 + j].z, vr[u0 + j].w};
                        float pj = pp[j];
                        if constexpr (HM) {
                            const uint32_t sees = pj < 0.0f ? 0u : ~0u;
                            pj = fmaxf(pj, 0.0f);
#pragma unroll
                            for (int i = 0; i < 4; i++) x[i] &= sees;
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            acc[h][2 * i] = fmaf(pj, half_bits_to_float((uint16_t) (x[i] & 0xFFFF)), acc[h][2 * i]);
                            acc[h][2 * i + 1] = fmaf(pj, half_bits_to_float((uint16_t) (x[i] >> 16)), acc[h][2 * i + 1]);
                        }
                    }
                }
            }
        }
        if (nxt_open) load_v(nxt);
        tile = nxt;
        open = nxt_open;
#pragma unroll
        for (int h = 0; h < (HM ? G : 1); h++) mk[h] = nk[h];
    }
    // the row groups' sums of each dim, then the wave's state into LDS
#pragma unroll
    for (int h = 0; h < G; h++) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int off = LPR; off < 64; off <<= 1) acc[h][i] += __shfl_xor(acc[h][i], off);
        l[h] = fc_reduce(l[h], [](float u, float v) { return u + v; });
    }
    if (lane < LPR) {
#pragma unroll
        for (int h = 0; h < G; h++) {
            *(fs_f4 *) &s_acc[w][h][8 * lane] = fs_f4{acc[h][0], acc[h][1], acc[h][2], acc[h][3]};
            *(fs_f4 *) &s_acc[w][h][8 * lane + 4] = fs_f4{acc[h][4], acc[h][5], acc[h][6], acc[h][7]};
        }
    }
    if (lane == 0) {
#pragma unroll
        for (int h = 0; h < G; h++) s_m[w][h] = m[h], s_l[w][h] = l[h];
    }
    __syncthreads();
    for (int e = (int) threadIdx.x; e < heads * (D / 4); e += 64 * kFcWaves) {
        const int h = e / (D / 4), d = e % (D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int v = 0; v < kFcWaves; v++) M = fmaxf(M, s_m[v][h]);
        fs_f4 o = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < kFcWaves; v++) {
            // (a sum of 0: the wave saw nothing. Its maximum is not asked: it is -inf, too, where
            // every score is a NaN, and the sum is one then)
            if (s_l[v][h] == 0.0f) continue;
            const float c = __builtin_amdgcn_exp2f(s_m[v][h] - M);
            L = fmaf(c, s_l[v][h], L);
            const fs_f4 x = *(const fs_f4 *) &s_acc[v][h][d];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = fmaf(c, x[i], o[i]);
        }
        const int64_t row = (int64_t) seq * a.hq + h0 + h;
        if (f.split == 1) {
            *(fs_f4 *) &f.out[row * D + d] = L != 0.0f ? o / L : fs_f4{0, 0, 0, 0};
        } else {
            const int64_t pr = (row / f.g * f.split + z) * f.g + row % f.g, partials = (int64_t) a.n_seq * a.hq * f.split;
            *(fs_f4 *) &f.part[pr * D + d] = o;
            if (d == 0) *(float2 *) &f.part[partials * D + 2 * pr] = make_float2(M, L);
        }
    }
}

// the kernel's G: heads of a workgroup, up to a power of two
int fc_heads(int gs) { return gs <= 2 ? gs : gs <= 4 ? 4 : 8; }

}  // namespace

bool fattn_scored_dec_supported(const fattn_args & a) { return a.n_q == 1; }

void fattn_scored_dec_plan(fattn_args & a, int n_cu) {
    const int g = a.hq / a.hkv, groups = (g + 7) / 8;
    const int tp = fc_tile(a.d, fc_heads((g + groups - 1) / groups)), n_tiles = (a.n_kv + tp - 1) / tp;
    const int64_t units = (int64_t) a.n_seq * a.hkv * groups;
    a.scored = 1;
    a.scored_split = 1;
    // The splits by a model of the time, in units of 0.55 us: a workgroup (one a
    // CU) takes 11 and one for each 32 KB of its K and V, the joining launch 6.
    // us of splits 1 / 2 / 4 / 8 / 16: heads of 128, 8 kv heads, 1024 positions
    // 14.8 / 13.3 / 10.7 / 10.2 / 9.4; 8 sequences of 4096 50 / 34 / 27 / 35 / -;
    // 12 of them, of 2 / 3 / 4 38 / 43 / 44; heads of 64, 500 of 2 sequences of 16 kv
    // heads 6.9 / 8.5 / 7.8 / 8.4; four of 20000, 4 kv heads of 5 query heads, of
    // 10 / 14 / 16 / 20 33 / 30 / 27 / 43.
    double best = 1e30;
    for (int split = 1; split <= std::min(n_tiles, n_cu); split++) {
        const int per = (n_tiles + split - 1) / split;
        const double rounds = std::ceil((double) units * ((n_tiles + per - 1) / per) / n_cu);
        const double t = rounds * (11.0 + per * (double) (tp * a.d) / 8192) + (per < n_tiles ? 6.0 : 0.0);
        if (t < best) best = t, a.scored_split = split;
    }
}

static void fc_plan(const fattn_args & a, fc_args & f) {
    f = fc_args{};
    f.a = a;
    f.score = fs_score_of(a);
    f.g = a.hq / a.hkv;
    f.groups = (f.g + 7) / 8;
    f.gs = (f.g + f.groups - 1) / f.groups;
    const int tp = fc_tile(a.d, fc_heads(f.gs));
    f.n_tiles = (a.n_kv + tp - 1) / tp;
    f.per = (f.n_tiles + std::max(1, a.scored_split) - 1) / std::max(1, a.scored_split);
    f.split = (f.n_tiles + f.per - 1) / f.per;
}

size_t fattn_scored_dec_scratch_bytes(const fattn_args & a) {
    fc_args f;
    fc_plan(a, f);
    return f.split > 1 ? sizeof(float) * (size_t) a.n_seq * a.hq * f.split * (a.d + 2) : 0;
}

void launch_fattn_scored_dec(const fattn_args & a, void * scratch, float * out, hipStream_t s) {
    fc_args f;
    fc_plan(a, f);
    f.part = (float *) scratch;
    f.out = out;
    const dim3 grid((unsigned) ((int64_t) a.n_seq * a.hkv * f.groups * f.split));
    auto go = [&](auto d, auto g) {
        constexpr int D = decltype(d)::value, G = decltype(g)::value;
        if (a.mask && a.m_ne2 > 1) hipLaunchKernelGGL((k_fattn_scored_dec<D, G, true>), grid, dim3(64 * kFcWaves), 0, s, f);
        else hipLaunchKernelGGL((k_fattn_scored_dec<D, G, false>), grid, dim3(64 * kFcWaves), 0, s, f);
    };
    auto heads = [&](auto d) {
        const int G = fc_heads(f.gs);
        if (G == 1) go(d, std::integral_constant<int, 1>{});
        else if (G == 2) go(d, std::integral_constant<int, 2>{});
        else if (G == 4) go(d, std::integral_constant<int, 4>{});
        else go(d, std::integral_constant<int, 8>{});
    };
    if (a.d == 64) heads(std::integral_constant<int, 64>{});
    else if (a.d == 128) heads(std::integral_constant<int, 128>{});
    else heads(std::integral_constant<int, 256>{});
    note_hip_error(hipGetLastError());
    if (f.split > 1) {
        fs_join j{};
        j.part = f.part, j.out = out, j.rows = (int64_t) a.n_seq * a.hq, j.partials = j.rows * f.split;
        j.split = f.split, j.d = a.d, j.hq = a.hq, j.n_q = 1, j.g = f.g, j.qpw = 1, j.q_blocks = 1, j.R = f.g;
        launch_fattn_join(j, s);
    }
}

}  // namespace mi355x
