// fattn_scored_dev.h -- what the two forms of attention with capped or biased
// scores share (k_fattn_scored.hip, many queries; k_fattn_scored_dec.hip, one):
// the cap, the heads' slopes, and the joining of a row's KV splits.
#pragma once

#include <cmath>

#include "mi355x_common.h"
#include "ops.h"

namespace mi355x {

typedef float fs_f4 __attribute__((ext_vector_type(4)));

constexpr float kFsLog2e = 1.4426950408889634f;
constexpr uint32_t kFsNegInf = 0xFC00u;
// tanh(x) / x as a polynomial of x^2 up to |x| = 0.625, interpolated at
// Chebyshev nodes: 4e-9 off
constexpr float kFsPolyEnd = 0.625f;
constexpr double kFsPoly[6] = {0.9999999960227207,   -0.3333325986294283,  0.13331114055632276,
                               -0.05372010765402796, 0.02058819145009359, -0.005657135182291668};

// the same up to |x| = 0.25: 2.5e-9 off
constexpr float kFsLowEnd = 0.25f;
constexpr double kFsLow[4] = {0.9999999975205603, -0.33333206285536215, 0.13323126058728388, -0.051327005164006706};

// scores in base 2 exponent units: cap log2(e) tanh(scale / cap product), or scale log2(e) product
struct fs_score {
    float poly[6];  // tanh(x) / x times cap log2(e), of x = s / cap
    float low[4];   // the shorter one as a polynomial of the product itself, for products below low_end
    float low_end;
    float in;       // what a product is multiplied by: scale / cap, or scale log2(e)
    float cap2;     // cap log2(e)
    double m0, m1;  // the slopes' bases (log2)
    int n_low;
};

inline fs_score fs_score_of(const fattn_args & a) {
    fs_score f{};
    const double log2e = 1.4426950408889634074;
    if (a.softcap > 0.0f) {
        f.in = (float) ((double) a.scale / a.softcap);
        f.cap2 = (float) (a.softcap * log2e);
        for (int k = 0; k < 6; k++) f.poly[k] = (float) (kFsPoly[k] * a.softcap * log2e);
        const double in = (double) a.scale / a.softcap;
        bool normal = true;  // (the coefficients, up to in^7)
        for (int k = 0; k < 4; k++) {
            const double c = kFsLow[k] * a.softcap * log2e * std::pow(in, 2 * k + 1);
            normal = normal && std::fabs(c) >= 1e-37 && std::fabs(c) <= 1e38;
            f.low[k] = (float) c;
        }
        f.low_end = normal ? (float) (kFsLowEnd / std::fabs(in)) : 0.0f;
    } else {
        f.in = (float) (a.scale * log2e);
    }
    f.n_low = 1;
    while (2 * f.n_low <= a.hq) f.n_low *= 2;
    f.m0 = -(double) a.max_bias / f.n_low;
    f.m1 = 0.5 * f.m0;
    return f;
}

// what a head's mask is multiplied by: its slope times log2(e)
__device__ __forceinline__ float fs_slope(const fs_score & f, float max_bias, int head) {
    if (!(max_bias > 0.0f)) return kFsLog2e;
    return (float) (exp2(head < f.n_low ? f.m0 * (head + 1) : f.m1 * (2 * (head - f.n_low) + 1)) * 1.4426950408889634074);
}

// the cap where |x| < kFsPolyEnd
__device__ __forceinline__ float fs_cap_small(const fs_score & f, float x) {
    const float y = x * x;
    float p = f.poly[5];
#pragma unroll
    for (int k = 4; k >= 0; k--) p = fmaf(p, y, f.poly[k]);
    return x * p;
}

// the cap of a product below low_end in size, plus base
__device__ __forceinline__ float fs_cap_low(const fs_score & f, float s, float base) {
    const float y = s * s;
    return fmaf(s, fmaf(fmaf(fmaf(f.low[3], y, f.low[2]), y, f.low[1]), y, f.low[0]), base);
}

// for any x: 1 - 2 / (e^2x + 1), from the polynomial where that cancels
__device__ __forceinline__ float fs_cap_any(const fs_score & f, float x) {
    const float e = __builtin_amdgcn_exp2f(2.0f * kFsLog2e * fabsf(x));  // +inf from |x| = 45 on: the quotient is 0
    const float t = copysignf(fmaf(-2.0f * f.cap2, __builtin_amdgcn_rcpf(e + 1.0f), f.cap2), x);
    return fabsf(x) < kFsPolyEnd ? fs_cap_small(f, x) : t;
}

// The decode form (k_fattn_scored_dec.hip). Partials of `split` splits a row in
// part: D values, unnormalised, a (row, split), then (maximum, sum) of each
bool fattn_scored_dec_supported(const fattn_args & a);
void fattn_scored_dec_plan(fattn_args & a, int n_cu);
size_t fattn_scored_dec_scratch_bytes(const fattn_args & a);
void launch_fattn_scored_dec(const fattn_args & a, void * scratch, float * out, hipStream_t s);

// joins the partials of rows (sequence, query, head); row r's are at at(r) + z
// of `partials` in all
struct fs_join {
    const float * part;
    const int2 * pieces;  // of a (sequence, kv head, query block): how many partials, and the first one's place; null: `split` each, in order
    float * out;
    int64_t rows, partials;
    int split, d;
    // partial of row (seq, q, head): ((seq hkv + head / g) q_blocks + q / qpw) split R + z R + (q % qpw) g + head % g
    int hq, n_q, g, qpw, q_blocks, R;
};
void launch_fattn_join(const fs_join & j, hipStream_t s);

}  // namespace mi355x
