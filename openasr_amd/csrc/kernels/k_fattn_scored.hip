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
// Work: a workgroup of eight waves owns R = 128 RW rows -- R / g queries times the g
// query heads of a kv head -- and walks its piece of the open 64-position tiles of
// the span; wave w owns rows 16 RW w .. of them, RW = 2 reading every K and V
// fragment once for 32 rows. MFMA 16x16x32 layouts: A lane l = row l % 16, k 8 (l /
// 16) .. + 7; B lane l = column l % 16, the same k; result lane l = rows 4 (l /
// 16) .. + 3, column l % 16. Scores are made transposed (rows = positions), so
// a lane holds 16 positions of a row and its p are the P V product's own B
// operand, V^T read in the same order of positions (by the transposing LDS reads).
//
// A first launch looks at the mask once for all heads: which tiles a block of
// queries sees at all, which of them have no masked or no nonzero entry, and
// which positions some query sees. From its counts every workgroup finds the same
// pieces of the same length, and a third launch joins a row's where there are several.
//
// What bounds it: 256 rows of 128 by a tile take 8300 cycles of a CU, its 832 matrix
// instructions 3328 of each SIMD's and its exponentials 4000 to 4900 of the vector
// units' (9 vector instructions a score with a cap -- a polynomial of the product
// five, p's halves two -- and a quarter-rate exponential); the two overlap, a
// request for 1 KB of K or V holds its wave for 100 to 300 cycles of it. us of the
// call without a barrier between the two kinds of work (four waves a workgroup, two
// workgroups a CU, which fell into step) and with it: two sequences of 4096 causal
// queries, 16 heads of 128 over 8, capped 264 / 251, not capped 240 / 227; one of
// 1777 in three documents, 8 heads of 256 59 / 52.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../fattn_pieces.h"
#include "../fattn_scored_dev.h"
#include "../mi355x_common.h"
#include "../ops.h"

namespace mi355x {

namespace {

constexpr int kFsTile = 64;
// p is scaled by 2^12: its low half stays a normal f16 down to 2^-15 of the maximum
constexpr float kFsUp = 12.0f;
constexpr float kFsOver = 3.0f;  // (and stays below f16's 2^16)
constexpr float kFsBase = 64.0f;

typedef _Float16 fs_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 fs_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 fs_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t fs_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t fs_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t fs_u2h __attribute__((ext_vector_type(2), aligned(2)));  // (the mask's rows have two-byte alignment)
typedef float fs_f4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t fs_u4h __attribute__((ext_vector_type(4), aligned(2)));

// a tile of a query block: nothing seen; seen, and all entries zero; seen, no
// entry -inf; seen, some entry -inf (or past the span)
constexpr int kFsUnits = 512;  // query blocks, and masks, of a launch in pieces, at most
enum : uint8_t { kFsClosed = 0, kFsPlain = 1, kFsAdds = 2, kFsMixed = 3 };

struct fs_args {
    fattn_args a;
    fs_score score;
    int g, qpw;       // query heads a kv head, queries a workgroup
    int q_blocks, n_tiles;
    int split, slots;  // the most pieces of a query block's open tiles; workgroups that the card holds at once
    int heads_mask;   // the mask differs by head: rows of it by query and head
    uint64_t * seen;  // [mask sequence][kv head or one][query block][tile]
    uint8_t * cls;    // [n_cls], the same order
    int64_t n_cls;
    int2 * pieces;    // [sequence][kv head][query block]: how many, and the first one's place in part
    int64_t partials; // rows of part
    float * part;
    float * out;
};

// eight mask entries at pos of a row, -inf past the span
__device__ __forceinline__ fs_u4 fs_mask8(const uint16_t * row, int pos, int n_kv) {
    if (pos + 8 <= n_kv) return *(const fs_u4h *) (row + pos);
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = pos + j < n_kv ? (uint32_t) row[pos + j] : kFsNegInf;
    return fs_u4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
}

__device__ __forceinline__ const char * fs_mask_of(const fattn_args & a, int seq, int head) {
    return a.mask + (int64_t) (seq % a.m_ne3) * a.m_nb3 + (int64_t) (head % a.m_ne2) * a.m_nb2;
}

// One workgroup a tile of a query block: thread = 8-position piece t % 8 of rows t / 8, + 32 ..
__global__ __launch_bounds__(256) void k_fattn_tiles(fs_args f) {
    __shared__ uint32_t s_bits[4][2];
    __shared__ uint64_t s_seen[4];
    const fattn_args & a = f.a;
    const int tid = (int) threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t u = blockIdx.x;
    const int tile = (int) (u % f.n_tiles), qb = (int) (u / f.n_tiles % f.q_blocks);
    const int64_t hs = u / ((int64_t) f.n_tiles * f.q_blocks);
    const int kinds = f.heads_mask ? a.hkv : 1, kvh = (int) (hs % kinds), ms = (int) (hs / kinds);
    const int q0 = qb * f.qpw, nq = min(f.qpw, a.n_q - q0), heads = f.heads_mask ? f.g : 1, rows = nq * heads;
    const int pos = tile * kFsTile + 8 * (tid & 7);
    fs_u4 m[8];  // (at most 256 rows)
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int r = (tid >> 3) + 32 * k;
        m[k] = fs_u4{};
        if (r < rows) m[k] = fs_mask8((const uint16_t *) (fs_mask_of(a, ms, kvh * f.g + r % heads) + (int64_t) (q0 + r / heads) * a.m_nb1), pos, a.n_kv);
    }
    uint32_t open = 0, closed = 0, adds = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if ((tid >> 3) + 32 * k >= rows) continue;
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
    if (lane == 0) s_seen[wave] = seen, s_bits[wave][0] = any_closed, s_bits[wave][1] = any_adds;
    __syncthreads();
    if (tid != 0) return;
    bool c = false, d = false;
    seen = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) seen |= s_seen[w], c |= s_bits[w][0] != 0, d |= s_bits[w][1] != 0;
    if (u == f.n_cls - 1)
        for (int64_t i = f.n_cls; i & 15; i++) f.cls[i] = kFsClosed;  // (counted 16 at a time)
    f.seen[u] = seen;
    f.cls[u] = !seen ? kFsClosed : c ? kFsMixed : d ? kFsAdds : kFsPlain;
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

// LDS holds a tile's K and V rows as they lie, 16-byte piece p of row r in slot p
// ^ 2 fs_turn(r): K's fragments (rows of 16 lanes, a piece each) and V's (two
// pieces of four rows a group of 16 lanes) then reach all 64 banks
template <int D>
__device__ __forceinline__ int fs_turn(int row) {
    return D == 64 ? (row >> 1) & 3 : row & 7;
}

typedef short fs_s4 __attribute__((ext_vector_type(4)));
// column l % 16 of the four rows of 16 halves that the lane's group of 16 reads, four halves a lane
__device__ __forceinline__ fs_h4 fs_read_turned(const char * p) {
    return __builtin_bit_cast(fs_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) fs_s4 *) p));
}

// the largest of lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float fs_max4(float x) {
    // (the swaps' results as values: a bit cast of a vector's element takes its first)
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const uint32_t v = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// z less the low, high half of h: one instruction (the compiler takes two)
__device__ __forceinline__ float fs_less_low(float z, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(z));
    return r;
}
__device__ __forceinline__ float fs_less_high(float z, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(z));
    return r;
}

// Sixteen bytes a lane from memory to LDS: lane l's at lds + 16 l. Not by the
// builtin, after which the compiler waits for all such loads before any read of
// LDS: here they are waited for by hand, two phases later
__device__ __forceinline__ void fs_to_lds(const char * src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}

// The phases' boundary: LDS reads are done; loads to LDS stay in flight
__device__ __forceinline__ void fs_phase_end() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int D, int RW, bool CAP, bool MASK>
__global__ __launch_bounds__(512, 2) void k_fattn_scored(fs_args f) {
    constexpr int NW = 8, NTH = 64 * NW, R = 16 * RW * NW;  // waves, threads, rows of a workgroup
    constexpr int KS = D / 32, NT = D / 16;
    constexpr int PC = D / 8;                       // 16-byte pieces of a K / V row
    constexpr int LTH = NTH / 2, KLD = kFsTile * PC / LTH;  // threads that load, and pieces of K, or V, of each
    constexpr int TB = kFsTile * 2 * D;             // bytes of a tile's K, or V
    __shared__ __align__(16) char s_kv[2][2][TB];   // [K, V][parity of the tile]
    __shared__ unsigned long long s_bad[2];         // positions of the tile whose V is not finite
    const fattn_args & a = f.a;
    const int tid = (int) threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
    // Workgroup b runs on XCD b % 8. Where the (sequence, kv head) pairs of a mask
    // divide by eight an XCD takes its share of them, whose K and V its L2 then holds;
    // the last query blocks, whose causal span is longest, first.
    const int units = a.hkv * a.n_seq * f.q_blocks, kinds = (f.heads_mask ? a.hkv : 1) * (MASK ? a.m_ne3 : 1);
    const int like = units / f.q_blocks / kinds;  // pairs that read the same mask
    int b = (int) blockIdx.x, inst = b % like, r = b / like;
    if (like % 8 == 0) inst = b % 8 * (like / 8) + b / 8 % (like / 8), r = b / 8 / (like / 8);
    int pieces = 1, z = 0, at_piece = 0;
    if (f.split == 1) {
    } else if constexpr (MASK) {
        // The open tiles of a query block in equal pieces of at most `len` tiles: the
        // least len from four on with which all blocks' pieces have a place on the card
        // at once, since a second round costs as much as the first. Workgroup b is
        // the b-th of those pieces, and every one counts them for itself. us of the
        // call with a length from the sum of the open tiles alone, and so: 2048 causal
        // queries 95 / 79, two sequences of 1500 90 / 81, three documents 63 / 61
        __shared__ int s_open[kFsUnits], s_of[NW];
        const int n_units = kinds * f.q_blocks;
        for (int i = tid; i < kFsUnits; i += NTH) s_open[i] = 0;
        __syncthreads();
        for (int i = 16 * tid; i < (int) f.n_cls; i += 16 * NTH) {
            const fs_u4 c = *(const fs_u4 *) &f.cls[i];
            uint32_t open = 0;  // a bit a tile
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t x = (c[j] | (c[j] >> 1)) & 0x01010101u;
                open |= ((x | x >> 7 | x >> 14 | x >> 21) & 15u) << (4 * j);
            }
            for (int e = 0; e < 16;) {
                const int u = (i + e) / f.n_tiles, n = min(16 - e, (u + 1) * f.n_tiles - i - e);
                if (u < n_units) atomicAdd(&s_open[(f.q_blocks - 1 - u % f.q_blocks) * kinds + u / f.q_blocks], __popc((open >> e) & ((1u << n) - 1)));
                e += n;
            }
        }
        __syncthreads();
        static_assert(NTH == kFsLengths, "a thread a length");
        const int mine_len = fs_length(tid, f.n_tiles);
        int total = 0;
        for (int u = 0; u < n_units; u++) total += like * fs_pieces(s_open[u], mine_len, f.split);
        const uint64_t fits = __ballot(total <= f.slots);
        if (lane == 0) s_of[wave] = fits ? 64 * wave + __builtin_ctzll(fits) : NTH - 1;
        __syncthreads();
        int first = NTH - 1;
#pragma unroll
        for (int w = 0; w < NW; w++) first = min(first, s_of[w]);
        const int len = fs_length(first, f.n_tiles);
        // the block that piece r of a pair is of: units 64 at a time
        int before = 0, u = -1;
        for (int u0 = 0; u0 < n_units; u0 += 64) {
            const int mine = u0 + lane < n_units ? fs_pieces(s_open[u0 + lane], len, f.split) : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(sum, o);
                if (lane >= o) sum += x;
            }
            const uint64_t past = __ballot(before + sum > r);
            if (u < 0 && past) {
                const int l0 = __builtin_ctzll(past);
                u = u0 + l0, pieces = __shfl(mine, l0), z = r - (before + __shfl(sum, l0) - pieces);
            }
            before += __shfl(sum, 63);
        }
        if (u < 0) return;  // (r is past the last piece)
        at_piece = __builtin_amdgcn_readfirstlane(inst * before + r);
        pieces = __builtin_amdgcn_readfirstlane(pieces), z = __builtin_amdgcn_readfirstlane(z), r = __builtin_amdgcn_readfirstlane(u);
    } else {
        pieces = f.split, z = r % f.split, r /= f.split;
        at_piece = (inst * f.q_blocks + r) * pieces + z;
    }
    const int qb = f.q_blocks - 1 - r / kinds, kind = r % kinds;
    const int hs = f.heads_mask ? (kind / a.hkv + a.m_ne3 * inst) * a.hkv + kind % a.hkv
                                : (kind + kinds * (inst / a.hkv)) * a.hkv + inst % a.hkv;
    if (f.split > 1 && z == 0 && tid == 0) f.pieces[hs * f.q_blocks + qb] = int2{pieces, at_piece};
    const int kvh = hs % a.hkv, seq = hs / a.hkv, kv_seq = seq / a.rk3;
    const int q0 = qb * f.qpw, nq = min(f.qpw, a.n_q - q0);
    const char * kbase = a.k + (int64_t) kvh * a.k_nb2 + (int64_t) kv_seq * a.k_nb3;
    const char * vbase = a.v + (int64_t) kvh * a.v_nb2 + (int64_t) kv_seq * a.v_nb3;
    const int64_t tile0 = MASK ? ((int64_t) ((seq % a.m_ne3) * (f.heads_mask ? a.hkv : 1) + (f.heads_mask ? kvh : 0)) * f.q_blocks + qb) * f.n_tiles : 0;

    // the rows' queries are on their way while the tiles are looked at
    fs_f4 qraw[RW][KS][2];
    float slope[RW];
    const char * mrow[RW];
#pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = 16 * (RW * wave + w) + l16, ql = min(r / f.g, nq - 1), head = kvh * f.g + r % f.g;
        const char * qp = a.q + (int64_t) (q0 + ql) * a.q_nb1 + (int64_t) head * a.q_nb2 + (int64_t) seq * a.q_nb3;
#pragma unroll
        for (int kk = 0; kk < KS; kk++)
#pragma unroll
            for (int h = 0; h < 2; h++) qraw[w][kk][h] = *(const fs_f4a *) (qp + 4 * (32 * kk + 8 * lg + 4 * h));
        slope[w] = fs_slope(f.score, a.max_bias, head);
        mrow[w] = MASK ? fs_mask_of(a, seq, head) + (int64_t) (q0 + ql) * a.m_nb1 : nullptr;
    }

    // The classes of 64 tiles from w_base on, a bit a tile
    int w_base = 0;
    uint64_t w_open, w_adds, w_mixed;
    auto window = [&]() {
        const int t = w_base + lane;
        int c = kFsClosed;
        if constexpr (MASK) {
            if (t < f.n_tiles) c = f.cls[tile0 + t];
        } else {
            if (t < f.n_tiles) c = (t + 1) * kFsTile <= a.n_kv ? kFsPlain : kFsMixed;
        }
        w_open = __ballot(c != kFsClosed), w_adds = __ballot(c >= kFsAdds), w_mixed = __ballot(c == kFsMixed);
    };
    int n_open = 0, skip = 0;
    if (MASK) {
        for (w_base = 0; w_base < f.n_tiles; w_base += 64) {
            window();
            n_open += __popcll(w_open);
        }
    } else {
        n_open = f.n_tiles;
    }
    if (pieces > 1) {
        const int each = n_open / pieces, more = n_open % pieces;
        skip = z * each + min(z, more);
        n_open = each + (z < more ? 1 : 0);
    }
    w_base = 0;
    window();
    auto next_open = [&]() {  // the first open tile of the window or after it, taken out of it
        while (w_open == 0) w_base += 64, window();
        const int t = __builtin_ctzll(w_open);
        w_open &= w_open - 1;
        return w_base + t;
    };
    auto class_of = [&](int t) { return (w_mixed >> (t & 63)) & 1 ? kFsMixed : (w_adds >> (t & 63)) & 1 ? kFsAdds : kFsPlain; };
    if (n_open > 0) {
        while (skip >= __popcll(w_open)) skip -= __popcll(w_open), w_base += 64, window();
        for (; skip > 0; skip--) w_open &= w_open - 1;
    }

    // this lane's query rows (the score product's B operand), rounded to f16
    fs_h8 qa[RW][KS];
#pragma unroll
    for (int w = 0; w < RW; w++)
#pragma unroll
        for (int kk = 0; kk < KS; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) qa[w][kk][j] = (_Float16) qraw[w][kk][j >> 2][j & 3];
    if (tid < 2) s_bad[tid] = 0;

    // A tile's K and V go to LDS by themselves, 16 bytes a lane, LTH / PC rows a step
    // (a multiple of what fs_turn repeats after). Group 0 (below) requests V, group 1 K
    const int st_row = tid % LTH / PC, st_piece = (tid % PC) ^ (2 * fs_turn<D>(st_row));
    const char * const st[2] = {kbase + st_row * a.k_nb1 + 16 * st_piece, vbase + st_row * a.v_nb1 + 16 * st_piece};
    const uint32_t lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) char *) &s_kv[0][0][0] + 1024 * (wave & 3);
    auto issue_one = [&](int h, int i, int tile, int par) {  // h: 0 K, 1 V
        const int64_t nb1 = h ? a.v_nb1 : a.k_nb1;
        const int row = tile * kFsTile + i * (LTH / PC);
        const char * p = st[h] + row * nb1;
        if ((tile + 1) * kFsTile > a.n_kv) p += (min(row + st_row, a.n_kv - 1) - (row + st_row)) * nb1;
        fs_to_lds(p, lds0 + (2 * h + par) * TB + i * LTH * 16);
    };
    auto issue = [&](int h, int tile, int par) {
#pragma unroll
        for (int i = 0; i < KLD; i++) issue_one(h, i, tile, par);
    };
    // Group 0, at the tile's arrival. Where not every query sees everything,
    // positions of V that no query sees become zeros (0 times anything), and pieces
    // that are not finite too: those are added query by query. (Where every query does,
    // an infinite value comes out infinite, or as a NaN from a p whose low part is zero)
    auto landed = [&](int tile, int cls, int par) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        asm volatile("" ::: "memory");
        if (cls != kFsMixed) return;
        uint64_t seen;
        if constexpr (MASK) seen = f.seen[tile0 + tile];
        else seen = ~0ull >> ((tile + 1) * kFsTile - a.n_kv);
#pragma unroll
        for (int i = 0; i < KLD; i++) {
            const int row = st_row + i * (LTH / PC);
            fs_u4 * p = (fs_u4 *) &s_kv[1][par][(i * LTH + tid) * 16];
            const bool in = (seen >> row) & 1, odd = fs_odd(*p);
            if (in && odd) atomicOr(&s_bad[par], 1ull << row);
            if (!in || odd) *p = fs_u4{0, 0, 0, 0};
        }
    };
    // this lane's entries (positions 16 t + 4 lg + i) of its rows' mask, if the tile needs them
    fs_u2 mr[RW][4];
    auto issue_mask = [&](int tile, int cls) {
        if constexpr (MASK) {
            const int p0 = tile * kFsTile;
            if (cls >= kFsAdds && p0 + kFsTile <= a.n_kv) {
#pragma unroll
                for (int w = 0; w < RW; w++)
#pragma unroll
                    for (int t = 0; t < 4; t++) mr[w][t] = *(const fs_u2h *) (mrow[w] + 2 * (p0 + 16 * t + 4 * lg));
            } else if (cls >= kFsAdds) {
#pragma unroll
                for (int w = 0; w < RW; w++)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        uint32_t e[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int pos = p0 + 16 * t + 4 * lg + i;
                            e[i] = ((const uint16_t *) mrow[w])[min(pos, a.n_kv - 1)];
                            if (pos >= a.n_kv) e[i] = kFsNegInf;
                        }
                        mr[w][t] = fs_u2{e[0] | e[1] << 16, e[2] | e[3] << 16};
                    }
            }
        }
    };

    // A row's exponents are its scores plus base, which puts its maximum at kFsUp
    // when it is set; it is set anew where a score goes past that by more than
    // kFsOver, not with every new maximum. A score is made as a sum with base only up to
    // kFsBase, half a step of which is 2^-18: a row whose tiles so far hold a mask's large
    // finite values has a base of 2^16, which would round the scores that follow to 2^-8
    float base[RW], l[RW];
    fs_f4 o[RW][NT];
#pragma unroll
    for (int w = 0; w < RW; w++) {
        base[w] = 0.0f, l[w] = 0.0f;
#pragma unroll
        for (int ct = 0; ct < NT; ct++) o[w][ct] = fs_f4{0, 0, 0, 0};
    }

    // Two groups of four waves, one of each a SIMD, take turns: while one makes
    // P V of a tile and K Q of the next on the matrix cores, the other makes its
    // exponentials on the vector units. A phase ends with a barrier; group 1 is a
    // phase behind:
    //     group 0   Q K 0 | softmax 0 | P V 0, Q K 1 | softmax 1 | ...
    //     group 1         | Q K 0     | softmax 0    | P V 0, Q K 1 | ...
    // In even phase 2 s group 0 requests V s between its products and group 1 K s + 1,
    // over V s - 2 and K s - 1,
    // which nobody reads any more; they wait for them at the end of phase 2 s + 1.
    const int grp = wave >> 2;
    fs_f4 sc[RW][4];
    fs_h8 hi[RW][2], lo[RW][2];  // p's halves, k slot 8 lg + j of step kk: position 32 kk + 16 (j / 4) + 4 lg + j % 4
    // Steps of the products, each of one fragment from LDS, read DIST steps ahead:
    // O^T += V^T P^T (two steps of 32 positions for each 16 dims), then S^T = K Q^T of
    // the next tile (lane (lg, l16) gets positions 16 t + 4 lg + i of row l16)
    constexpr int PV = 2 * NT, QK = 4 * KS, DIST = 4, EVERY = 4;
    static_assert(1 + EVERY * (KLD - 1) < PV + QK, "a step for each request");
    auto products = [&](const char * sv, const char * sk, auto from, auto loads, int tile, int par) {
        constexpr int FROM = decltype(from)::value;
        constexpr bool LOADS = decltype(loads)::value;  // V of a tile, between the steps
        fs_h8 ring[DIST + 1];
        // the rows' sums: products with ones, every lane of a row's column gets it
        const fs_h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
        fs_f4 sum[RW];
#pragma unroll
        for (int w = 0; w < RW; w++) sum[w] = fs_f4{0, 0, 0, 0};
        const int lrow = 4 * lg + (l16 >> 2), vturn = 2 * fs_turn<D>(lrow), kturn = 2 * fs_turn<D>(l16);  // (16 rows on: the same turn)
        auto read = [&](int i) {
            if (i < PV) {
                const int ct = i % NT, kk = i / NT;
                const char * p = &sv[(32 * kk + lrow) * 2 * D + (((2 * ct + ((l16 >> 1) & 1)) ^ vturn) * 16) + 8 * (l16 & 1)];
                const fs_h4 v0 = fs_read_turned(p), v1 = fs_read_turned(p + 16 * 2 * D);
                ring[i % (DIST + 1)] = fs_h8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
            } else {
                const int t = (i - PV) % 4, kk = (i - PV) / 4;
                ring[i % (DIST + 1)] = *(const fs_h8 *) &sk[(16 * t + l16) * 2 * D + (((4 * kk + lg) ^ kturn) * 16)];
            }
        };
#pragma unroll
        for (int i = FROM; i < FROM + DIST; i++) read(i);
#pragma unroll
        for (int i = FROM; i < PV + QK; i++) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + DIST < PV + QK) read(i + DIST);
            if (LOADS && i % EVERY == 1 && i / EVERY < KLD) issue_one(1, i / EVERY, tile, par);
            const fs_h8 x = ring[i % (DIST + 1)];
            if (i < PV) {
                const int ct = i % NT, kk = i / NT;
#pragma unroll
                for (int w = 0; w < RW; w++) o[w][ct] = fs_mfma(x, lo[w][kk], o[w][ct]);
#pragma unroll
                for (int w = 0; w < RW; w++) o[w][ct] = fs_mfma(x, hi[w][kk], o[w][ct]);
                if (ct < 2) {
#pragma unroll
                    for (int w = 0; w < RW; w++) sum[w] = fs_mfma(ones, ct ? hi[w][kk] : lo[w][kk], sum[w]);
                }
                if (i == PV - 1) {
#pragma unroll
                    for (int w = 0; w < RW; w++) l[w] += sum[w][0];
                }
            } else {
                const int t = (i - PV) % 4, kk = (i - PV) / 4;
#pragma unroll
                for (int w = 0; w < RW; w++) sc[w][t] = fs_mfma(x, qa[w][kk], kk == 0 ? fs_f4{0, 0, 0, 0} : sc[w][t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    int tile[3] = {0, 0, 0}, cls[3] = {kFsClosed, kFsClosed, kFsClosed}, par = 0;  // of tiles t, t + 1, t + 2
    auto take = [&](int k, int left) {
        if (left > 0) tile[k] = next_open(), cls[k] = class_of(tile[k]);
        else tile[k] = tile[k - 1];
    };
    auto run = [&](auto group) {
        constexpr int GRP = decltype(group)::value;
        tile[0] = next_open(), cls[0] = class_of(tile[0]), take(1, n_open - 1);
        if constexpr (GRP == 1) {
            issue(0, tile[0], 0);
            __builtin_amdgcn_s_waitcnt(0x0F70);
        }
        issue_mask(tile[0], cls[0]);
        fs_phase_end();
        if constexpr (GRP == 0) {
            issue(1, tile[0], 0);
        } else {
            issue(0, tile[1], 1);
            fs_phase_end();
        }
        products(s_kv[1][0], s_kv[0][0], std::integral_constant<int, PV>{}, std::false_type{}, 0, 0);
        if constexpr (GRP == 1) __builtin_amdgcn_s_waitcnt(0x0F70);
        fs_phase_end();
        for (; n_open > 0; n_open--, par ^= 1) {
            take(2, n_open - 2);
#pragma unroll
            for (int w = 0; w < RW; w++) {
                if constexpr (GRP == 1) {
#pragma unroll
                    for (int i = w * KLD / RW; i < (w + 1) * KLD / RW; i++) issue_one(0, i, tile[2], par);
                }
                float z[4][4];  // with b0
                const float b0 = fabsf(base[w]) <= kFsBase ? base[w] : 0.0f, off = base[w] - b0;
                if constexpr (CAP) {
                    float most = 0.0f;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(sc[w][t][i]));
                    if (!__any(!(most < f.score.low_end))) {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) z[t][i] = fs_cap_low(f.score, sc[w][t][i], b0);
                    } else {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) z[t][i] = fs_cap_any(f.score, sc[w][t][i] * f.score.in) + b0;
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) z[t][i] = fmaf(sc[w][t][i], f.score.in, b0);
                }
                if constexpr (MASK) {
                    if (cls[0] >= kFsAdds) {
                        if (cls[0] == kFsAdds) {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) z[t][i] = fmaf((float) __builtin_bit_cast(fs_h4, mr[w][t])[i], slope[w], z[t][i]);
                        } else {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float v = (float) __builtin_bit_cast(fs_h4, mr[w][t])[i];
                                z[t][i] = v == -INFINITY ? -INFINITY : fmaf(v, slope[w], z[t][i]);
                            }
                        }
                    }
                } else if (cls[0] == kFsMixed) {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (tile[0] * kFsTile + 16 * t + 4 * lg + i >= a.n_kv) z[t][i] = -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) mx = fmaxf(mx, z[t][i]);
                // (a sum of 0: no score yet. The first one's exponential is 2^kFsUp)
                if (__any(mx + off > kFsUp + kFsOver || (l[w] == 0.0f && mx != -INFINITY) || off != 0.0f)) {
                    const float most = fs_max4(mx);
                    const bool first = l[w] == 0.0f;
                    const bool anew = (first && most != -INFINITY) || most + off > kFsUp + kFsOver;
                    const float to = anew ? b0 + (kFsUp - most) : base[w];
                    if (__any(anew && !first)) {
                        const float alpha = first ? 1.0f : __builtin_amdgcn_exp2f(to - base[w]);
                        l[w] *= alpha;
#pragma unroll
                        for (int ct = 0; ct < NT; ct++) o[w][ct] *= alpha;
                    }
                    base[w] = to;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) z[t][i] += to - b0;
                }
#pragma unroll
                for (int t = 0; t < 4; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) z[t][i] = __builtin_amdgcn_exp2f(z[t][i]);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(z[t][i], z[t][i + 1]));
                        const fs_h2 hh = __builtin_bit_cast(fs_h2, h);
                        const fs_h2 r = __builtin_bit_cast(fs_h2, __builtin_amdgcn_cvt_pkrtz(fs_less_low(z[t][i], h), fs_less_high(z[t][i + 1], h)));
                        hi[w][t >> 1][4 * (t & 1) + i] = hh[0], hi[w][t >> 1][4 * (t & 1) + i + 1] = hh[1];
                        lo[w][t >> 1][4 * (t & 1) + i] = r[0], lo[w][t >> 1][4 * (t & 1) + i + 1] = r[1];
                    }
                }
            }
            if constexpr (GRP == 0) landed(tile[0], cls[0], par);
            fs_phase_end();
            if (n_open > 1) issue_mask(tile[1], cls[1]);
            if (cls[0] == kFsMixed && s_bad[par] != 0) {
                // V rows that are not finite: for the rows that see them alone
                const uint64_t bad = s_bad[par];
                for (int p = 0; p < kFsTile; p++) {
                    if (!((bad >> p) & 1)) continue;
#pragma unroll
                    for (int w = 0; w < RW; w++) {
                        float mine = 0.0f;
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (t == p >> 4 && i == (p & 3)) mine = (float) hi[w][t >> 1][4 * (t & 1) + i] + (float) lo[w][t >> 1][4 * (t & 1) + i];
                        const float pp = __shfl(mine, 16 * ((p & 15) >> 2) + l16);
                        if constexpr (MASK) {
                            if (((const uint16_t *) mrow[w])[tile[0] * kFsTile + p] == kFsNegInf) continue;
                        }
                        const char * vrow = vbase + (int64_t) (tile[0] * kFsTile + p) * a.v_nb1;
#pragma unroll
                        for (int ct = 0; ct < NT; ct++) {
                            const fs_h8 v8 = *(const fs_h8 *) (vrow + 2 * (16 * ct + 8 * (lg >> 1)));
                            if (!fs_odd(__builtin_bit_cast(fs_u4, v8))) continue;  // it is in LDS
#pragma unroll
                            for (int i = 0; i < 4; i++) o[w][ct][i] = fmaf(pp, (float) (lg & 1 ? v8[4 + i] : v8[i]), o[w][ct][i]);
                        }
                    }
                }
            }
            if (tid == 0) s_bad[par ^ 1] = 0;  // read to the end, and not yet of tile t + 1
            // (behind the last tile V of the last but one is requested again, and K of none read)
            products(s_kv[1][par], s_kv[0][par ^ 1], std::integral_constant<int, 0>{}, std::integral_constant<bool, GRP == 0>{}, tile[1], par ^ 1);
            if constexpr (GRP == 1) __builtin_amdgcn_s_waitcnt(0x0F70);  // K of tile t + 2
            if (GRP == 0 || n_open > 1) fs_phase_end();
            tile[0] = tile[1], cls[0] = cls[1], tile[1] = tile[2], cls[1] = cls[2];
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (the last requests, before the workgroup's LDS is given back)
    };
    if (n_open > 0) {
        if (grp == 0) run(std::integral_constant<int, 0>{});
        else run(std::integral_constant<int, 1>{});
    }

#pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = 16 * (RW * wave + w) + l16;
        if (pieces > 1) {
            // partials of piece z: O unnormalised, then (m, l), a workgroup row
            const int64_t rows = f.partials;
            const int64_t pr = (int64_t) at_piece * R + r;
#pragma unroll
            for (int ct = 0; ct < NT; ct++) *(fs_f4 *) &f.part[pr * D + 16 * ct + 4 * lg] = o[w][ct];
            if (lg == 0) *(float2 *) &f.part[rows * D + 2 * pr] = make_float2(l[w] == 0.0f ? -INFINITY : kFsUp - base[w], l[w]);
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
    const int2 piece = f.pieces ? f.pieces[blk] : int2{f.split, (int) blk * f.split};
    const int64_t p0 = (int64_t) piece.y * f.R + (q % f.qpw) * f.g + head % f.g;
    const int split = piece.x;
    const bool whole = f.pieces && split == 1;  // written by its one piece
    if (LN == 1 && whole) return;
    const float * ml = f.part + f.partials * D;
    float M = -INFINITY, L = 0.0f;
    fs_f4 acc = {0, 0, 0, 0};
    for (int z0 = ln; z0 < split; z0 += 4 * LN) {
        float2 v[4];
        fs_f4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t p = p0 + (int64_t) min(z0 + k * LN, split - 1) * f.R;
            v[k] = *(const float2 *) &ml[2 * p];
            x[k] = *(const fs_f4 *) &f.part[p * D + d];
        }
        float most = M;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (z0 + k * LN >= split) v[k] = make_float2(-INFINITY, 0.0f);
            most = fmaxf(most, v[k].x);
        }
        const float w0 = L == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(M - most);
        L *= w0, acc *= w0, M = most;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (v[k].y == 0.0f) continue;  // nothing seen (a NaN is a sum too)
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
            if (v.y == 0.0f) continue;
            const float w = __builtin_amdgcn_exp2f(v.x - most);
            L = fmaf(w, v.y, L);
            const fs_f4 x = s_acc[tid + k * (D / 4)];
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(w, x[i], acc[i]);
        }
    }
    if (row < f.rows && !whole) *(fs_f4 *) &f.out[row * D + d] = L != 0.0f ? acc / L : fs_f4{0, 0, 0, 0};
}

size_t fs_al(size_t v) { return (v + 255) & ~(size_t) 255; }

// Rows of a workgroup: 16 a wave, or 32 (each fragment of K and V read once for
// them) where a kv head has more than 128; for heads of 256 the outputs of 32
// would take half of the registers
int fs_rows(const fattn_args & a) { return a.d != 256 && (int64_t) a.n_q * (a.hq / a.hkv) > 128 ? 256 : 128; }

// the launch's shape, and its scratch: the tiles' classes, then the splits' partials
size_t fs_plan(const fattn_args & a, fs_args & f) {
    f = fs_args{};
    f.a = a;
    const int R = fs_rows(a);
    f.g = a.hq / a.hkv;
    f.qpw = std::min(R / f.g, a.n_q);
    f.q_blocks = (a.n_q + f.qpw - 1) / f.qpw;
    f.n_tiles = (a.n_kv + kFsTile - 1) / kFsTile;
    f.split = std::max(1, a.scored_split);
    f.slots = a.scored_slots;
    f.heads_mask = a.mask && a.m_ne2 > 1;
    f.score = fs_score_of(a);
    size_t need = 0;
    if (a.mask) {
        f.n_cls = (int64_t) a.m_ne3 * (f.heads_mask ? a.hkv : 1) * f.q_blocks * f.n_tiles;
        need = fs_al(8 * f.n_cls) + fs_al(f.n_cls);
    }
    // (with a mask at most `slots` pieces in all)
    const int64_t units = (int64_t) a.n_seq * a.hkv * f.q_blocks;
    f.partials = (a.mask ? std::min<int64_t>(f.slots, units * f.split) : units * f.split) * R;
    if (f.split > 1) need += fs_al(sizeof(int2) * (size_t) units) + sizeof(float) * (size_t) f.partials * (a.d + 2);
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
    // Pieces of a query block's open tiles where query blocks leave CUs idle, of at
    // least four tiles. How many a block gets under a mask is for the launch to say
    const int R = fs_rows(a), g = a.hq / a.hkv, qpw = std::min(R / g, std::max(1, a.n_q));
    const int64_t units = std::max<int64_t>(1, (int64_t) ((a.n_q + qpw - 1) / qpw) * a.hkv * a.n_seq);
    const int n_tiles = (a.n_kv + kFsTile - 1) / kFsTile;
    a.scored = 1;
    a.scored_slots = n_cu;
    const int64_t most = a.mask ? a.scored_slots : a.scored_slots / units;
    a.scored_split = units >= a.scored_slots || units > kFsUnits ? 1 : (int) std::max<int64_t>(1, std::min<int64_t>(most, n_tiles / 4));
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
    if (a.mask) {
        const int64_t n = f.n_cls;
        f.seen = (uint64_t *) p;
        f.cls = (uint8_t *) (p + fs_al(8 * (size_t) n));
        p += fs_al(8 * (size_t) n) + fs_al((size_t) n);
        hipLaunchKernelGGL(k_fattn_tiles, dim3((unsigned) n), dim3(256), 0, s, f);
        note_hip_error(hipGetLastError());
    }
    f.pieces = (int2 *) p;
    if (f.split > 1) p += fs_al(sizeof(int2) * (size_t) a.n_seq * a.hkv * f.q_blocks);
    f.part = (float *) p;
    const int rows = fs_rows(a);
    const dim3 grid((unsigned) (f.split > 1 ? f.partials / rows : (int64_t) f.q_blocks * a.hkv * a.n_seq));
    auto go = [&](auto d, auto rw) {
        constexpr int D = decltype(d)::value, RW = decltype(rw)::value;
        if (a.softcap > 0.0f) {
            if (a.mask) hipLaunchKernelGGL((k_fattn_scored<D, RW, true, true>), grid, dim3(512), 0, s, f);
            else hipLaunchKernelGGL((k_fattn_scored<D, RW, true, false>), grid, dim3(512), 0, s, f);
        } else {
            if (a.mask) hipLaunchKernelGGL((k_fattn_scored<D, RW, false, true>), grid, dim3(512), 0, s, f);
            else hipLaunchKernelGGL((k_fattn_scored<D, RW, false, false>), grid, dim3(512), 0, s, f);
        }
    };
    auto width = [&](auto d) {
        constexpr int wide = decltype(d)::value == 256 ? 1 : 2;
        if (rows == 256) go(d, std::integral_constant<int, wide>{});
        else go(d, std::integral_constant<int, 1>{});
    };
    if (a.d == 256) width(std::integral_constant<int, 256>{});
    else if (a.d == 128) width(std::integral_constant<int, 128>{});
    else width(std::integral_constant<int, 64>{});
    note_hip_error(hipGetLastError());
    if (f.split > 1) {
        fs_join j{};
        j.part = f.part, j.pieces = f.pieces, j.out = out, j.rows = (int64_t) a.n_seq * a.n_q * a.hq;
        j.partials = f.partials;
        j.split = f.split, j.d = a.d, j.hq = a.hq, j.n_q = a.n_q, j.g = f.g, j.qpw = f.qpw, j.q_blocks = f.q_blocks, j.R = rows;
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
