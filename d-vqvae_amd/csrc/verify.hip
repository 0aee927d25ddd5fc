// Verification of drafted codes against the prior's distribution (gfx950).
//
// A cheap model drafts codes x_0 .. x_{n-1} with distributions q_g, the prior gives its own distributions p_g for the
// same history in one pass.  Code x_g is kept while  u_g q_g(x_g) < p_g(x_g)  (a draw that is right with probability
// min(1, p/q)); at the first one that is not, the row's next code is drawn from max(p_g - q_g, 0) / mass, and behind the
// last kept one from p_n.  The codes that come out are distributed as if the prior had drawn them one by one.
//
// The outputs are whole numbers, so comparison and draw have to come out as in 64 bits: next to a border 32 bits decide
// differently for another order of summation.  The work is split accordingly.
//   Tests: one pass over the row in 32-bit exponentials, the sums of few of them collected in 64 bits.  Their error is
//     bounded (kVerifyMargin); a test that clears the bound is decided, one within it -- one in ten thousand -- has its
//     sums taken again in 64 bits.
//   Draw: one position per row, 64-bit exponentials, in one pass although the weights e_p - k e_q (k = S_p / S_q) need the
//     pass's own sums: k is known to kVerifyMargin from the test, which settles the sign of all weights but those next to
//     zero, and with the signs settled a tile's mass follows k through the sum of e_q over its positive codes.  Tiles that hold a code
//     next to zero are done again once k is known.  A tile is 512 codes, one wave; the tiles' masses find the tile, a scan
//     inside it the code.
// Three forms: rows of up to 1024 codes stay in the registers of one wave per position; longer rows have a workgroup per
// row that stops at the first rejection; few very long rows, and long rows whose codes do not lie side by side, are cut among
// workgroups (three launches).
// Times below are of whole calls one after the other, or of a kernel where that is said.
#include "common.h"

namespace dvq {

// Residual mass below this is rounding (p and q equal up to 64-bit noise): the draw is then from p itself.
constexpr double kVerifyNoMass = 9.094947017729282e-13;   // 2^-40
constexpr int kTile = 512;                                // codes of a tile: 8 per lane
// Relative error of u q / p from sums taken in 32 bits, in units of e = 2^-23.  A term exp2((x - r) log2 e) carries |x - r| 1.5 e from
// its argument (difference, constant and product rounded) and e from the exponential; eight of them are added in 32 bits
// (1.5 e), the eights in 64.  When the lane's reference r moves up by D > kVerifySlack, what is summed takes a factor with an
// error of D 1.5 e + e: at most (R - r) 1.625 e over all moves up to the last reference R (at most (R - r) / 8 of them).  A term
// lies at most kVerifySlack above the reference it was summed with, so it carries at most (R - x) 1.625 e where x <= r, and
// (R - x + 8) 1.625 e + 8 * 1.5 e where x > r: (R - x) 1.625 e + 25 e + e in all cases.  Joining lanes, waves and workgroups
// moves sums to larger references, counted in R, at e + 3.5 e for the exponential and seven roundings each of three times.
// R is at most the largest logit, from which the mean distance under the distribution is at most ln V <= 13.9: a sum is off by
// less than (22.6 + 26 + 1.5 + 13.5) e = 7.6e-6, the quotient of two by less than 1.6e-5.  Two and a half times that:
constexpr double kVerifyMargin = 4e-5;
constexpr float kVerifySlack = 8.f;

struct VerifyArgs {
    const void* logits; int64_t lb, lp, lv;
    const void* draft; int64_t db, dg, dv;
    const int64_t* tokens; int64_t tb, tg;
    const double* u; int64_t ub, ug;
    const double* r; int64_t rb;
    const int64_t* lengths; int64_t nb;
    int64_t* accepted; int64_t* next;
    int64_t B; int G, P, V;
    bool unit;                                            // codes of target and draft lie side by side
};

__device__ __forceinline__ float verify_load(const float* p) { return *p; }
__device__ __forceinline__ float verify_load(const unsigned short* p) { return bf16_bits_to_f32(*p); }

// The wave's number, known to be the same in every lane (addresses that follow from it are scalar).
__device__ __forceinline__ int verify_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// One step of a wave reduction: the value of the lane that the DPP control names, `none` where there is no such lane.
template <int CTRL>
__device__ __forceinline__ float verify_dpp(float v, float none) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double verify_dpp(double v) {
    const long long b = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ double verify_lane(double v, int lane) {
    const long long b = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
// Sums of the lanes up to each: inside rows of 16 lanes (shifts by 1, 2, 4, 8), then the row before (0x142), then the lower
// half (0x143) into the rows behind.
__device__ __forceinline__ double wave_scan(double v) {
    v += verify_dpp<0x111>(v);
    v += verify_dpp<0x112>(v);
    v += verify_dpp<0x114>(v);
    v += verify_dpp<0x118>(v);
    const int row = (threadIdx.x & 63) >> 4;
    const double t = verify_dpp<0x142>(v);
    if (row & 1) v += t;
    const double h = verify_dpp<0x143>(v);
    if (row & 2) v += h;
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    v += verify_dpp<0x111>(v, 0.f);
    v += verify_dpp<0x112>(v, 0.f);
    v += verify_dpp<0x114>(v, 0.f);
    v += verify_dpp<0x118>(v, 0.f);
    v += verify_dpp<0x142>(v, 0.f);
    v += verify_dpp<0x143>(v, 0.f);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ double wave_sum(double v) {            // (only lane 63 has to be right: no row is spared)
    v += verify_dpp<0x111>(v);
    v += verify_dpp<0x112>(v);
    v += verify_dpp<0x114>(v);
    v += verify_dpp<0x118>(v);
    v += verify_dpp<0x142>(v);
    v += verify_dpp<0x143>(v);
    return verify_lane(v, 63);
}
__device__ __forceinline__ float wave_max(float v) {
    const float none = -__builtin_inff();
    v = fmaxf(v, verify_dpp<0x111>(v, none));
    v = fmaxf(v, verify_dpp<0x112>(v, none));
    v = fmaxf(v, verify_dpp<0x114>(v, none));
    v = fmaxf(v, verify_dpp<0x118>(v, none));
    v = fmaxf(v, verify_dpp<0x142>(v, none));
    v = fmaxf(v, verify_dpp<0x143>(v, none));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// exp(d), d <= 700 and not NaN, in 64 bits: with y = 32 d / ln 2 and k the whole number next to it, 2^(k / 32) -- 32nds of an
// octave from a table in LDS (32 entries of 8 bytes: a half wave's reads are in banks of their own or shared) -- times the
// Taylor polynomial of exp((y - k) ln 2 / 32), whose rest after degree 5 is below (ln 2 / 64)^6 / 6! = 2.3e-15.  Adding
// 1.5 * 2^52 leaves k in the low bits.  Below -746 the result is 0 (-inf among it).
__device__ __constant__ const double kVerify32nds[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
struct Exp {
    const double* tab;
    __device__ __forceinline__ double operator()(double d) const {
        d = fmax(d, -750.0);
        const double t = __builtin_fma(d, 46.16624130844683, 6755399441055744.0);       // 32 / ln 2
        const int k = (int)__builtin_bit_cast(long long, t);
        const double f = __builtin_fma(d, 46.16624130844683, 6755399441055744.0 - t);
        double s = __builtin_fma(f, 3.973709984549416e-11, 9.172562701824643e-09);
        s = __builtin_fma(s, f, 1.693850972437182e-06);
        s = __builtin_fma(s, f, 0.0002345961982022468);
        s = __builtin_fma(s, f, 0.02166084939249829);
        s = __builtin_fma(s, f, 1.0);
        return __builtin_ldexp(s * tab[k & 31], k >> 5);
    }
};
// The table in LDS; every thread of the workgroup calls it once.
__device__ __forceinline__ Exp verify_table(double* lds) {
    if (threadIdx.x < 32) lds[threadIdx.x] = kVerify32nds[threadIdx.x];
    __syncthreads();
    return Exp{lds};
}

// Eight codes side by side as they lie in memory (16-byte loads at any alignment).
template <typename T> struct Raw;
template <> struct Raw<float> {
    f32x4 w[2];
    __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(&w[0], p, 16); __builtin_memcpy(&w[1], p + 4, 16); }
    __device__ __forceinline__ float operator[](int j) const { return w[j >> 2][j & 3]; }
};
template <> struct Raw<unsigned short> {
    u16x8 w;
    __device__ __forceinline__ void load(const unsigned short* p) { __builtin_memcpy(&w, p, 16); }
    __device__ __forceinline__ float operator[](int j) const { return bf16_bits_to_f32(w[j]); }
};

// First code that verify_tile reads for the tile at v0: with unit stride the last tile of a row is read from 512 codes before
// the row's end (whole 16-byte loads, no lane by itself), and those that belong to the tile in front of it are dropped.
__device__ __forceinline__ int verify_base(bool unit, int v0, int V) { return unit && V >= kTile && v0 + kTile > V ? V - kTile : v0; }

// This lane's eight codes of the tile at v0, `fill` for codes that are not in it or not in the row.  Where target and draft
// both have unit stride: codes base + 8 lane + j, otherwise v0 + 64 j + lane for both.
template <typename T>
__device__ __forceinline__ void verify_tile(const T* row, int64_t sv, bool unit, int v0, int V, int lane, float fill, float (&x)[8]) {
    if (unit && V >= kTile) {
        const int base = verify_base(unit, v0, V), skip = v0 - base - 8 * lane;
        Raw<T> r;
        r.load(row + base + 8 * lane);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = r[j];
        if (base != v0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = j < skip ? fill : x[j];
        }
    } else if (v0 + kTile <= V) {
        const T* at = row + (v0 + lane) * sv;
#pragma unroll
        for (int j = 0; j < 8; ++j, at += 64 * sv) x[j] = verify_load(at);
    } else {
        const int first = unit ? v0 + 8 * lane : v0 + lane, step = unit ? 1 : 64;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = first + step * j;
            x[j] = v < V ? verify_load(row + v * sv) : fill;
        }
    }
}

// Reference point and sum of exp(x - ref) of logits seen so far; no distribution: ref = -inf, or s not a number (a NaN or
// +inf among the logits makes it one).
struct Sum { float ref, at; double s; };                          // at: ref, or 0 where ref is -inf
__device__ __forceinline__ bool sum_ok(const Sum& a) { return a.ref > -__builtin_inff() && a.ref < __builtin_inff() && a.s == a.s; }
__device__ __forceinline__ double sum_moved(const Exp& ex, const Sum& a, float ref) {        // a.s for reference point ref >= a.ref
    return a.ref > -__builtin_inff() && a.ref < ref ? a.s * ex((double)a.ref - (double)ref) : a.s;
}

// The reference moves up only where the next eight codes of some lane exceed it by more than kVerifySlack.  What the lane has summed
// may be most of its mass then (many codes just within the slack): the factor's error counts in kVerifyMargin.
__device__ __forceinline__ void sum_add(Sum& a, const float (&x)[8]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
    const bool up = m > a.ref + kVerifySlack;
    if (__any(up)) {
        if (up) {
            a.s *= (double)__builtin_amdgcn_exp2f((a.ref - m) * 1.44269504f);
            a.ref = m;
        }
        a.at = a.ref > -__builtin_inff() ? a.ref : 0.f;              // (nothing but -inf and NaN so far: any point will do)
    }
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f((x[j] - a.at) * 1.44269504f);
    a.s += (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
}
// Sums of several lanes or parts as one, moved to the largest reference point and added in 32 bits; the same in every lane.
__device__ __forceinline__ Sum sum_join(float ref, double s) {
    const float top = wave_max(ref);
    const float f = ref < top ? (float)s * __builtin_amdgcn_exp2f((ref - top) * 1.44269504f) : (float)s;
    return Sum{top, top, (double)wave_sum(ref > -__builtin_inff() ? f : s == s ? 0.f : __builtin_nanf(""))};
}
__device__ __forceinline__ Sum sum_wave(const Sum& a) { return sum_join(a.ref, a.s); }
__device__ __forceinline__ Sum sum_parts(const Sum* parts, int n) {                // every wave for itself, all the same
    const int lane = threadIdx.x & 63;
    const Sum t = lane < n ? parts[lane] : Sum{-__builtin_inff(), 0.f, 0.0};
    return sum_join(t.ref, t.s);
}

// The test sum of a row that a wave holds: its largest logit is at hand, and the lanes' sums are added in 32 bits (ten
// roundings; with |x - ref| <= ln 1024 in the mean still well inside kVerifyMargin).
template <int TILES>
__device__ __forceinline__ Sum sum_held(const float (&x)[TILES][8]) {
    float m = x[0][0];
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[i][j]);
    m = wave_max(m);
    const float at = m > -__builtin_inff() ? m : 0.f;                // (nothing but -inf and NaN: any point will do, and a NaN stays)
    float f = 0.f;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f((x[i][j] - at) * 1.44269504f);
        f += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    }
    return Sum{m, m, (double)wave_sum(f)};
}

enum { VERIFY_KEEP = 0, VERIFY_REJECT = 1, VERIFY_BAD = 2, VERIFY_UNSURE = 3 };

// What the tests of a row's drafted codes read beside the sums: lane l holds that of position g0 + l, so that it is asked for
// once, in front of everything else (the row's length among it: positions behind it are read in vain).  A code outside the
// table reads the table's end.
template <typename T, typename D>
struct Drafted {
    float t, d; double u; int inside;
    __device__ __forceinline__ void fetch(const VerifyArgs& a, int64_t b, int g0, int lane) {
        if (g0 >= a.G) return;
        const int g = g0 + lane < a.G ? g0 + lane : a.G - 1;
        const int64_t x = a.tokens[b * a.tb + g * a.tg], at = x < 0 ? 0 : x < a.V ? x : a.V - 1;
        inside = x == at;
        u = a.u[b * a.ub + g * a.ug];
        t = verify_load(reinterpret_cast<const T*>(a.logits) + b * a.lb + g * a.lp + at * a.lv);
        d = verify_load(reinterpret_cast<const D*>(a.draft) + b * a.db + g * a.dg + at * a.dv);
    }
    __device__ __forceinline__ Drafted of(int l) const {             // lane l's, in every lane
        Drafted f;
        f.t = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, t), l));
        f.d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), l));
        f.u = verify_lane(u, l);
        f.inside = __builtin_amdgcn_readlane(inside, l);
        return f;
    }
};

// p, q: sums of the position's logits (q unused with PROBS).  `exact`: the sums were taken in 64 bits.
template <bool PROBS, typename T, typename D>
__device__ __forceinline__ int verify_test(const Exp& ex, const Drafted<T, D>& f, const Sum& p, const Sum& q, bool exact) {
    if (!sum_ok(p) || (!PROBS && !sum_ok(q))) return VERIFY_BAD;
    if (!f.inside) return VERIFY_REJECT;
    if (PROBS && !(f.d >= 0.f && f.d < __builtin_inff())) return VERIFY_BAD;
    // u q < p, both sides times the two sums; u last, so that equal distributions keep every u below 1
    const double px = PROBS ? ex((double)f.t - (double)p.ref) : ex((double)f.t - (double)p.ref) * q.s;
    const double lhs = f.u * ((PROBS ? (double)f.d : ex((double)f.d - (double)q.ref)) * p.s);
    if (!exact && px > 0.0 && lhs > 0.0 && !(fabs(lhs - px) > kVerifyMargin * px)) return VERIFY_UNSURE;
    return lhs < px ? VERIFY_KEEP : VERIFY_REJECT;
}

__device__ __forceinline__ int verify_length(const VerifyArgs& a, int64_t b) {
    if (!a.lengths) return a.G;
    const int64_t n = a.lengths[b * a.nb];
    return n < 0 ? 0 : n > a.G ? a.G : (int)n;
}

// Weights of a position's codes: e_p - k e_q where positive (residual), else e_p, with e_p = exp(t - p_ref) and e_q = exp(q -
// q_ref), or q itself where probabilities are given (k = S_p then).
struct Weights { double p_ref, q_ref, k; bool residual; };

// e_p and e_q of this lane's eight codes of a tile; a given probability that is none makes its e_q NaN.
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ void verify_terms(const Exp& ex, const VerifyArgs& a, const T* lr, const D* dr, const Weights& w, bool unit, int v0,
                                             int lane, double (&ep)[8], double (&eq)[8]) {
    float t[8], q[8];
    verify_tile(lr, a.lv, unit, v0, a.V, lane, -__builtin_inff(), t);
    if (w.residual) verify_tile(dr, a.dv, unit, v0, a.V, lane, PROBS ? 0.f : -__builtin_inff(), q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        ep[j] = ex((double)t[j] - w.p_ref);
        eq[j] = 0.0;
        if (w.residual) eq[j] = !PROBS ? ex((double)q[j] - w.q_ref) : (q[j] >= 0.f && q[j] < __builtin_inff()) ? (double)q[j] : __builtin_nan("");
        if (j & 1) __builtin_amdgcn_sched_barrier(0);            // (all eight at once do not fit the registers of four waves)
    }
}
__device__ __forceinline__ double verify_weight(const Weights& w, double ep, double eq) {
    if (!w.residual) return ep;
    const double d = __builtin_fma(-w.k, eq, ep);
    return d > 0.0 || d != d ? d : 0.0;
}
__device__ __forceinline__ double verify_sum8(const double (&w)[8]) {
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
}

// What the one pass leaves: this lane's sums of e_p and e_q, and of a tile (the same in every lane) the mass with the k that
// is known so far, the sum of e_q over its positive codes (the mass falls by it times what k lacks), and whether it holds
// a code whose sign that k does not settle.
struct Tile { double mass, c; bool near; };

// One wave.  w.k is within kVerifyMargin / 2 of the true one.
template <bool PROBS, typename T, typename D>
__device__ __forceinline__ Tile verify_pass(const Exp& ex, const Weights& w, const T& t, const D& q, double& sp, double& sq) {
    double mass[2] = {0.0, 0.0}, c[2] = {0.0, 0.0}, p2[2] = {0.0, 0.0}, q2[2] = {0.0, 0.0};
    bool near = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double ep = ex((double)t[j] - w.p_ref);
        p2[j & 1] += ep;
        if (w.residual) {
            const float v = q[j];
            const double eq = !PROBS ? ex((double)v - w.q_ref) : (v >= 0.f && v < __builtin_inff()) ? (double)v : __builtin_nan("");
            const double kq = w.k * eq, d = ep - kq;
            q2[j & 1] += eq;
            mass[j & 1] += fmax(d, 0.0);
            c[j & 1] += d > 0.0 ? eq : 0.0;
            near |= fabs(d) < kVerifyMargin * kq;
        }
        if (j & 1) __builtin_amdgcn_sched_barrier(0);            // (all eight at once do not fit the registers of four waves)
    }
    sp += p2[0] + p2[1];
    sq += q2[0] + q2[1];
    Tile r = {0.0, 0.0, false};
    if (w.residual) {
        r.mass = wave_sum(mass[0] + mass[1]);
        r.c = wave_sum(c[0] + c[1]);
        r.near = __any(near);
    } else r.mass = wave_sum(p2[0] + p2[1]);
    return r;
}
// Mass of a tile with the weights known exactly; one wave.
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ double verify_tile_mass(const Exp& ex, const VerifyArgs& a, const T* lr, const D* dr, const Weights& w, bool unit, int v0, int lane) {
    double ep[8], eq[8];
    verify_terms<T, D, PROBS>(ex, a, lr, dr, w, unit, v0, lane, ep, eq);
#pragma unroll
    for (int j = 0; j < 8; ++j) ep[j] = verify_weight(w, ep[j], eq[j]);
    return wave_sum(verify_sum8(ep));
}

// One wave: the first code of the tile at v0 whose cumulated weight (with `before` in front of it) exceeds thr, the last code
// with weight if none does (the tile's own sum was taken in another order) or if `over`.  w: the weights as verify_tile
// lays them out; lds: 576 doubles.
__device__ __forceinline__ int verify_locate(const double (&w)[8], bool unit, int v0, int V, double before, double thr, bool over, double* lds) {
    const int lane = threadIdx.x & 63;
    double c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = w[j];
    if (!unit) {                                                 // from 64 j + lane to 8 lane + j
#pragma unroll
        for (int j = 0; j < 8; ++j) { const int at = 64 * j + lane; lds[at + (at >> 3)] = w[j]; }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = lds[9 * lane + j];
    }
    double own = 0.0;
    int last = -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) { own += c[j]; if (c[j] > 0.0) last = j; }
    const double incl = wave_scan(own);
    const unsigned long long some = __ballot(last >= 0), hit = __ballot(!over && last >= 0 && before + incl > thr);
    const int l = hit ? __ffsll(hit) - 1 : some ? 63 - __clzll(some) : 0;
    int at = last;
    if (hit) {
        double cum = before + (incl - own);
        bool found = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cum += c[j];
            if (!found && c[j] > 0.0 && cum > thr) { found = true; at = j; }
        }
    }
    return verify_base(unit, v0, V) + 8 * l + __builtin_amdgcn_readlane(at, l);
}

// The tile that holds the draw, from the masses of all tiles (one wave): returns its number, `before` = mass in front of it;
// over: rounding leaves none, the last tile with mass.
__device__ __forceinline__ int verify_pick(const double* mass, int tiles, double thr, double& before, bool& over) {
    const int lane = threadIdx.x & 63;
    before = 0.0;
    int last = 0;
    for (int base = 0; base < tiles; base += 64) {
        const double m = base + lane < tiles ? mass[base + lane] : 0.0;
        const double incl = wave_scan(m);
        const unsigned long long some = __ballot(m > 0.0), hit = __ballot(m > 0.0 && before + incl > thr);
        if (hit) {
            const int l = __ffsll(hit) - 1;
            before += verify_lane(incl - m, l);
            over = false;
            return base + l;
        }
        if (some) last = base + 63 - __clzll(some);
        before += verify_lane(incl, 63);
    }
    over = true;
    return last;
}
// Sum of n values in the order that verify_pick takes (one wave).
__device__ __forceinline__ double verify_total(const double* v, int n) {
    const int lane = threadIdx.x & 63;
    double total = 0.0;
    for (int base = 0; base < n; base += 64) total += wave_sum(base + lane < n ? v[base + lane] : 0.0);
    return total;
}

// Sum of exp(x - ref) of a whole row in 64 bits by the whole workgroup, for the tests too near to tell.
template <typename T>
static __device__ __noinline__ double verify_row_sum64(Exp ex, const T* row, int64_t sv, bool unit, int V, double ref, double* parts) {
    const int wave = verify_wave(), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    double s = 0.0;
    for (int v0 = wave * kTile; v0 < V; v0 += waves * kTile) {
        float x[8];
        verify_tile(row, sv, unit, v0, V, lane, -__builtin_inff(), x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s += ex((double)x[j] - ref);
            if (j & 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) parts[wave] = s;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < waves; ++w) all += parts[w];
    return all;
}

// Copies elements that lie side by side into LDS; the whole workgroup.  Four loads of a thread are under way at a time (one
// behind the end reads the last 16 bytes once more: left out, it would make the others wait).
template <typename T>
__device__ __forceinline__ void verify_copy(const T* from, int total, T* to) {
    constexpr int N = 16 / sizeof(T), U = 4;
    const int step = blockDim.x * N, whole = total / N * N;
    for (int i0 = 0; i0 < whole; i0 += U * step) {
        u32x4 v[U];
        int at[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            at[k] = i0 + k * step + (int)threadIdx.x * N;
            __builtin_memcpy(&v[k], from + (at[k] < whole ? at[k] : whole - N), 16);
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (at[k] < whole) *reinterpret_cast<u32x4*>(to + at[k]) = v[k];
    }
    for (int i = whole + (int)threadIdx.x; i < total; i += blockDim.x) to[i] = from[i];
}

// ------------------------------------------------------------------------------------------------ rows of up to 1024 codes
// One workgroup per row, one wave per position: `blockDim / 64` positions at a time until the first that stops the row.
// Its wave holds the position's logits in registers and draws from them.
//
// STAGED: the prior's forward hands its logits over as [B, V, cells], all positions of a code side by side.  Read position
// by position, every position fetches every cache line of the row again (from L2: 4096 grids of 9 x 512 took 38 us, bound
// by that); the row's block is copied into LDS once instead: 25 us a call, 16 of them the memory's.  One grid takes 4.0 us of kernel
// over one set of operands, 5.2 over three in turns (medians of traced launches).
template <int TILES, bool STAGED, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(TILES == 1 && PROBS ? 8 : 4))) void verify_short_kernel(VerifyArgs a) {
    extern __shared__ __align__(16) char block[];                // the staged block, later room for verify_locate
    __shared__ int state[16];
    __shared__ double table[32];
    double* const lds = reinterpret_cast<double*>(block);
    const int64_t b = blockIdx.x;
    const int wave = verify_wave(), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int V = a.V;
    const int n = verify_length(a, b);
    const double at_draw = a.r[b * a.rb];
    Drafted<T, D> drafted;
    drafted.fetch(a, b, 0, lane);
    const float none = -__builtin_inff();
    T* const staged = reinterpret_cast<T*>(block);
    if (STAGED) {
        const T* from = reinterpret_cast<const T*>(a.logits) + b * a.lb;
        verify_copy(from, V * a.P, staged);
    }
    const Exp ex = verify_table(table);
    int held = 0;                                                // first of the 64 drafted codes at hand
    for (int base = 0;; base += waves) {
        const int g = base + wave;                               // n: the position behind all drafts
        float t[TILES][8], q[TILES][8];
        if (g - held >= 64) {
            held = g / 64 * 64;
            drafted.fetch(a, b, held, lane);
        }
        const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)g * a.lp;
        const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)g * a.dg;
        Sum p = {none, 0.f, 0.0}, s = {none, 0.f, 0.0};
        int st = g == n ? VERIFY_REJECT : VERIFY_KEEP;           // (behind n: not looked at)
        if (g <= n && g < a.P) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                if (STAGED) verify_tile(staged + g, (int64_t)a.P, false, i * kTile, V, lane, none, t[i]);
                else verify_tile(lr, a.lv, a.unit, i * kTile, V, lane, none, t[i]);
            }
            if (!PROBS && g < n)
#pragma unroll
                for (int i = 0; i < TILES; ++i) verify_tile(dr, a.dv, a.unit, i * kTile, V, lane, none, q[i]);
            p = sum_held(t);
            if (g < n) {
                const Drafted<T, D> f = drafted.of(g & 63);
                if (!PROBS) s = sum_held(q);
                st = verify_test<PROBS>(ex, f, p, s, false);
                if (st == VERIFY_UNSURE) {
                    double e = 0.0;
#pragma unroll
                    for (int i = 0; i < TILES; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) e += ex((double)t[i][j] - (double)p.ref);
                    p.s = wave_sum(e);
                    if (!PROBS) {
                        e = 0.0;
#pragma unroll
                        for (int i = 0; i < TILES; ++i)
#pragma unroll
                            for (int j = 0; j < 8; ++j) e += ex((double)q[i][j] - (double)s.ref);
                        s.s = wave_sum(e);
                    }
                    st = verify_test<PROBS>(ex, f, p, s, true);
                }
            } else if (!sum_ok(p)) st = VERIFY_BAD;
        }
        int stop = st == VERIFY_KEEP ? waves : 0;                // first wave of these whose position stops the row
        if (waves > 1) {
            __syncthreads();
            if (lane == 0) state[wave] = st;
            __syncthreads();
            for (stop = 0; stop < waves && state[stop] == VERIFY_KEEP; ++stop) {}
        }
        if (stop == waves) continue;                             // (position n always stops: the loop ends)
        if (wave != stop) return;
        if (lane == 0) a.accepted[b] = g;
        if (st == VERIFY_BAD || g >= a.P) {
            if (lane == 0) a.next[b] = -1;
            return;
        }
        const bool residual = g < n;
        if (PROBS && residual)
#pragma unroll
            for (int i = 0; i < TILES; ++i) verify_tile(dr, a.dv, a.unit, i * kTile, V, lane, 0.f, q[i]);
        // all terms stay in registers: sums first, weights from them
        double w[TILES][8], eq[TILES][8], mass[TILES], sp = 0.0, sq = 0.0, total = 0.0;
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[i][j] = ex((double)t[i][j] - (double)p.ref);
                eq[i][j] = 0.0;
                if (residual) {
                    const float v = q[i][j];
                    eq[i][j] = !PROBS ? ex((double)v - (double)s.ref) : (v >= 0.f && v < __builtin_inff()) ? (double)v : __builtin_nan("");
                }
                sp += w[i][j];
                sq += eq[i][j];
                if (j & 1) __builtin_amdgcn_sched_barrier(0);
            }
        sp = wave_sum(sp);
        if (!PROBS && residual) sq = wave_sum(sq);
        Weights k = {(double)p.ref, (double)s.ref, PROBS ? sp : sp / sq, residual};
        if (residual) {
            double d[TILES];
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                double x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = verify_weight(k, w[i][j], eq[i][j]);
                total += d[i] = wave_sum(verify_sum8(x));
            }
            k.residual = !(total <= kVerifyNoMass * sp);         // nothing left over: from p
        }
        total = 0.0;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[i][j] = verify_weight(k, w[i][j], eq[i][j]);
            total += mass[i] = wave_sum(verify_sum8(w[i]));
        }
        if (total != total) {
            if (lane == 0) a.next[b] = -1;
            return;
        }
        const double thr = at_draw * total;
        int at = 0;
        if (TILES == 1) at = verify_locate(w[0], a.unit, 0, V, 0.0, thr, !(total > thr), lds);
        else {
            const bool second = mass[0] > thr ? false : (mass[TILES - 1] > 0.0 || !(mass[0] > 0.0));
            at = second ? verify_locate(w[TILES - 1], a.unit, kTile, V, mass[0], thr, !(total > thr), lds)
                        : verify_locate(w[0], a.unit, 0, V, 0.0, thr, !(mass[0] > thr), lds);
        }
        if (lane == 0) a.next[b] = at;
        return;
    }
}

// --------------------------------------------------------------------------------- longer rows, one workgroup per row
// The draw of a row whose tiles have been passed over: mass, c and near of every tile in LDS, sp and sq the sums of e_p and e_q.
// Every wave calls it.
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ void verify_finish(const Exp& ex, const VerifyArgs& args, int64_t b, double at_draw, const T* lr, const D* dr,
                                              Weights w, bool unit, double sp, double sq, double* a, const double* c,
                                              const unsigned char* near, int tiles, double* lds) {
    const int wave = verify_wave(), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    double total = 0.0;
    if (w.residual) {
        const double k = PROBS ? sp : sp / sq;
        for (int i = threadIdx.x; i < tiles; i += blockDim.x)
            if (!near[i]) a[i] = __builtin_fma(w.k - k, c[i], a[i]);
        w.k = k;
        int turn = 0;                                            // tiles to do again are dealt to the waves one by one
        for (int base = 0; base < tiles; base += 64)
            for (unsigned long long m = __ballot(base + lane < tiles && near[base + lane]); m; m &= m - 1) {
                if (turn == wave) {
                    const int i = base + __ffsll(m) - 1;
                    const double mass = verify_tile_mass<T, D, PROBS>(ex, args, lr, dr, w, unit, i * kTile, lane);
                    if (lane == 0) a[i] = mass;
                }
                turn = turn + 1 == waves ? 0 : turn + 1;
            }
        __syncthreads();
        total = verify_total(a, tiles);                          // every wave for itself, in one order
        if (total <= kVerifyNoMass * sp) {                       // nothing left over: from p
            __syncthreads();
            w.residual = false;
            for (int i = wave; i < tiles; i += waves) {
                const double m = verify_tile_mass<T, D, PROBS>(ex, args, lr, dr, w, unit, i * kTile, lane);
                if (lane == 0) a[i] = m;
            }
            __syncthreads();
            total = verify_total(a, tiles);
        }
    } else total = verify_total(a, tiles);
    if (wave != 0) return;
    if (total != total || sq != sq) {                            // (sq: a given probability that is none)
        if (lane == 0) args.next[b] = -1;
        return;
    }
    const double thr = at_draw * total;
    double before, ep[8], eq[8];
    bool over;
    const int i = verify_pick(a, tiles, thr, before, over);
    verify_terms<T, D, PROBS>(ex, args, lr, dr, w, unit, i * kTile, lane, ep, eq);
#pragma unroll
    for (int j = 0; j < 8; ++j) ep[j] = verify_weight(w, ep[j], eq[j]);
    const int at = verify_locate(ep, unit, i * kTile, args.V, before, thr, over, lds);
    if (lane == 0) args.next[b] = at;
}

// Adds eight codes of a row to a lane's sum; those before `skip` are left out.
template <typename T>
__device__ __forceinline__ void sum_raw(Sum& a, const Raw<T>& x) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[j];
    sum_add(a, v);
}
template <typename T>
__device__ __forceinline__ void sum_raw(Sum& a, const Raw<T>& x, int skip) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < skip ? -__builtin_inff() : x[j];
    sum_add(a, v);
}

// Tiles of a row and (Q) of its draft's on their way into registers, a ring of N: while one is worked on, the others are in
// flight, and behind a position's last tiles the next position's first ones -- asked for before it is known whether the
// row gets there, N tiles in vain once a row against a memory latency in every position.  No load is left out (one that
// may be makes the compiler wait for all): where there is nothing to load it is a line that is at hand.
template <typename T, typename D, bool Q>
struct Ring {
    static constexpr int N = sizeof(T) == 2 ? 4 : 2;
    Raw<T> x[N], tx;                                             // tx, ty: the last 512 codes, for those behind the whole tiles
    Raw<D> y[N], ty;
};
// A wave's tiles of whole rows: wave, wave + step, .. < full; t counts them.
struct Share {
    int wave, step, full, cnt, rounds;
    __device__ __forceinline__ Share(int w, int s, int V, int n)
        : wave(w), step(s), full(V / kTile), cnt((V / kTile - w + s - 1) / s), rounds(0) {
        cnt = cnt > 0 ? cnt : 0;
        rounds = cnt > n ? (cnt + n - 1) / n * n : n;
    }
    __device__ __forceinline__ int at(int t, int lane) const {
        const int tile = wave + t * step;
        return (tile < full ? tile : full - 1) * kTile + 8 * lane;
    }
};
template <typename T, typename D, bool Q>
__device__ __forceinline__ void verify_start(Ring<T, D, Q>& ring, const Share& w, const T* lr, const D* dr, bool both, int V, int lane) {
    ring.tx.load(lr + V - kTile + 8 * lane);
    if (Q) ring.ty.load(dr + (both ? V - kTile + 8 * lane : 8 * lane));
#pragma unroll
    for (int s = 0; s < Ring<T, D, Q>::N; ++s) {
        ring.x[s].load(lr + w.at(s, lane));
        if (Q) ring.y[s].load(dr + (both ? w.at(s, lane) : 8 * lane));
    }
}
// This wave's share of the test sums of one position, whose first tiles the ring holds; nl, nd, nboth: the next position's.
template <typename T, typename D, bool Q>
__device__ __forceinline__ void verify_sums(Ring<T, D, Q>& ring, const Share& w, const T* lr, const D* dr, bool both, const T* nl, const D* nd, bool nboth,
                                            int V, int lane, Sum& p, Sum& q) {
    constexpr int N = Ring<T, D, Q>::N;
    for (int i = 0; i < w.rounds; i += N) {
#pragma unroll
        for (int s = 0; s < N; ++s) {
            if (i + s < w.cnt) {
                sum_raw(p, ring.x[s]);
                if (Q && both) sum_raw(q, ring.y[s]);
            }
            const int t = i + s + N;
            const bool own = t < w.rounds;
            const int at = w.at(own ? t : t - w.rounds, lane);
            ring.x[s].load((own ? lr : nl) + at);
            if (Q) ring.y[s].load((own ? dr : nd) + ((own ? both : nboth) ? at : 8 * lane));
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (w.full * kTile < V && w.full % w.step == w.wave) {
        const int skip = w.full * kTile - (V - kTile) - 8 * lane;
        sum_raw(p, ring.tx, skip);
        if (Q && both) sum_raw(q, ring.ty, skip);
    }
    ring.tx.load(nl + V - kTile + 8 * lane);
    if (Q) ring.ty.load(nd + (nboth ? V - kTile + 8 * lane : 8 * lane));
}

// Codes side by side (a.unit).  The tests run at 86 % of a copy's rate (1024 rows x 16381 bf16, all drafts kept, no draw: 60 us for 268 MB);
// the draw, 64-bit exponentials of the whole row once more, takes 45 us where every row ends in one, 24 without a residual.  With rows
// that stop at different positions 86 us over three sets of operands in turns, 78 over one that fits the last cache (41 of memory); 1000 of
// up to 5 x 8192 46 to 48 us (14), where a draw in 32 bits saved 1 to 3: what holds it is that rows of 0 to 5 positions end apart.
template <int WAVES, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(4))) void verify_row_kernel(VerifyArgs a) {
    extern __shared__ double tile_a[];                           // per tile of the row: a, c, near
    __shared__ Sum parts[2][2][WAVES];
    __shared__ double parts64[2][WAVES], lds[kTile + kTile / 8], table[32];
    const Exp ex = verify_table(table);
    const int64_t b = blockIdx.x;
    const int wave = verify_wave(), lane = threadIdx.x & 63;
    const int V = a.V, tiles = (V + kTile - 1) / kTile;
    double* tile_c = tile_a + tiles;
    unsigned char* tile_near = reinterpret_cast<unsigned char*>(tile_c + tiles);
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db;
    Sum p = {0.f, 0.f, 1.0}, q = {0.f, 0.f, 1.0};
    int g = 0, st = VERIFY_KEEP;
    const int n = verify_length(a, b);
    const double at_draw = a.r[b * a.rb];
    Drafted<T, D> drafted;
    drafted.fetch(a, b, 0, lane);
    const Share share(wave, WAVES, V, Ring<T, D, !PROBS>::N);
    Ring<T, D, !PROBS> ring;
    if (a.G == 0) dr = reinterpret_cast<const D*>(lr);           // (read in vain, and 512 codes of either type fit a row)
    verify_start(ring, share, lr, dr, n > 0, V, lane);
    for (; g < a.P && g <= n; ++g) {
        const bool both = !PROBS && g < n, more = g + 1 < a.P && g + 1 <= n, nboth = !PROBS && g + 1 < n;
        const T* nl = more ? lr + a.lp : lr;
        const D* nd = g + 1 < n ? dr + a.dg : dr;
        if (g > 0 && g % 64 == 0) drafted.fetch(a, b, g, lane);
        p = q = Sum{-__builtin_inff(), 0.f, 0.0};
        verify_sums(ring, share, lr, dr, both, nl, nd, nboth, V, lane, p, q);
        __builtin_amdgcn_sched_barrier(0);
        p = sum_wave(p);
        if (both) q = sum_wave(q);
        Sum (*at)[WAVES] = parts[g & 1];                         // (in turns: one barrier a position)
        if (lane == 0) { at[0][wave] = p; at[1][wave] = q; }
        __syncthreads();
        p = sum_parts(at[0], WAVES);
        if (both) q = sum_parts(at[1], WAVES);
        if (g == n) {                                            // every draft kept: one more code
            st = sum_ok(p) ? VERIFY_REJECT : VERIFY_BAD;
            break;
        }
        const Drafted<T, D> f = drafted.of(g & 63);
        st = verify_test<PROBS>(ex, f, p, q, false);             // (the same for every thread: one code's values)
        if (st == VERIFY_UNSURE) {
            p.s = verify_row_sum64(ex, lr, 1, true, V, (double)p.ref, parts64[0]);
            if (!PROBS) q.s = verify_row_sum64(ex, dr, 1, true, V, (double)q.ref, parts64[1]);
            st = verify_test<PROBS>(ex, f, p, q, true);
        }
        if (st != VERIFY_KEEP) break;
        lr = nl;
        dr = nd;
    }
    if (threadIdx.x == 0) a.accepted[b] = g;
    if (st != VERIFY_REJECT) {
        if (threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    const Weights w = {(double)p.ref, (double)q.ref, PROBS ? p.s : p.s / q.s, g < n};
    double sp = 0.0, sq = 0.0;
    const float none = -__builtin_inff();
    // two tiles in turns, as in verify_sums
    Raw<T> t[2];
    Raw<D> d[2];
    const auto load = [&](int k, int i) {
        i = i < tiles ? i : tiles - 1;
        const int at = verify_base(true, i * kTile, V) + 8 * lane;
        t[k].load(lr + at);
        d[k].load(dr + (w.residual ? at : 8 * lane));
    };
    const auto pass = [&](int k, int i) {
        const int skip = i * kTile - verify_base(true, i * kTile, V) - 8 * lane;
        float x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = j < skip ? none : t[k][j];
            y[j] = j < skip ? (PROBS ? 0.f : none) : d[k][j];
        }
        const Tile r = verify_pass<PROBS>(ex, w, x, y, sp, sq);
        if (lane == 0) { tile_a[i] = r.mass; tile_c[i] = r.c; tile_near[i] = r.near; }
    };
    load(0, wave);
    for (int i = wave; i < tiles; i += 2 * WAVES) {
        load(1, i + WAVES);
        __builtin_amdgcn_sched_barrier(0);
        pass(0, i);
        load(0, i + 2 * WAVES);
        __builtin_amdgcn_sched_barrier(0);
        if (i + WAVES < tiles) pass(1, i + WAVES);
    }
    sp = wave_sum(sp);
    sq = wave_sum(sq);
    __syncthreads();
    if (lane == 0) { parts64[0][wave] = sp; parts64[1][wave] = sq; }
    __syncthreads();
    sp = sq = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) { sp += parts64[0][i]; sq += parts64[1][i]; }
    verify_finish<T, D, PROBS>(ex, a, b, at_draw, lr, dr, w, true, sp, sq, tile_a, tile_c, tile_near, tiles, lds);
}

// ------------------------------------------------------------- long rows cut among workgroups: three launches
constexpr int kSplitWaves = 4;
constexpr int kChunk = 8;                                        // tiles whose test sums one workgroup takes
// Workspace of one row: test sums of every position's chunks (target, then draft), the decision, what the pass leaves of
// every tile.
struct Decision { double k; float p_ref, q_ref; int g, st; };
struct SplitRow {
    Sum* p; Sum* q; Decision* d;
    double *sp, *sq, *a, *c; unsigned char* near;
};
// Test sums of a position: one per chunk, one per tile where codes do not lie side by side.
__host__ __device__ inline int64_t split_parts(int V, bool unit) {
    const int64_t tiles = (V + kTile - 1) / kTile;
    return unit ? (tiles + kChunk - 1) / kChunk : tiles;
}
__host__ __device__ inline int64_t split_bytes(int P, int G, int V, bool unit) {
    const int64_t tiles = (V + kTile - 1) / kTile, chunks = split_parts(V, unit);
    return (P + G) * chunks * (int64_t)sizeof(Sum) + (int64_t)sizeof(Decision) + 4 * tiles * 8 + (tiles + 15) / 16 * 16 + 8;
}
__device__ __forceinline__ SplitRow split_row(char* ws, const VerifyArgs& a, int64_t b) {
    const int64_t tiles = (a.V + kTile - 1) / kTile, chunks = split_parts(a.V, a.unit);
    char* at = ws + b * ((split_bytes(a.P, a.G, a.V, a.unit) + 15) / 16 * 16);
    SplitRow r;
    r.p = reinterpret_cast<Sum*>(at);
    r.q = r.p + a.P * chunks;
    r.d = reinterpret_cast<Decision*>(r.q + a.G * chunks);
    r.sp = reinterpret_cast<double*>(r.d + 1);
    r.sq = r.sp + tiles;
    r.a = r.sq + tiles;
    r.c = r.a + tiles;
    r.near = reinterpret_cast<unsigned char*>(r.c + tiles);
    return r;
}

// Test sums of one chunk of one position.  All positions are summed: which ones the row needs is not known yet.  8 rows of 4 drafts x
// 65536 fp32: 7.1 us here, 7.0 in the pass, 8.0 in the draw, each bound by its chain of loads and joins.
template <typename T, typename D, bool PROBS>
__global__ __launch_bounds__(kSplitWaves * 64) void verify_stats_kernel(VerifyArgs a, char* ws, int chunks) {
    __shared__ Sum parts[2][kSplitWaves];
    const int wave = verify_wave(), lane = threadIdx.x & 63;
    const int64_t id = blockIdx.x;
    const int chunk = (int)(id % chunks), g = (int)(id / chunks % a.P);
    const int64_t b = id / chunks / a.P;
    const int n = verify_length(a, b);
    if (g > n) return;
    const SplitRow row = split_row(ws, a, b);
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)g * a.lp;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)g * a.dg;
    const bool both = !PROBS && g < n;
    Sum p = {-__builtin_inff(), 0.f, 0.0}, q = p;
    const int tiles = (a.V + kTile - 1) / kTile, last = (chunk + 1) * kChunk < tiles ? (chunk + 1) * kChunk : tiles;
    constexpr int N = kChunk / kSplitWaves;                      // this wave's tiles, all asked for at once
    Raw<T> x[N];
    Raw<D> y[N];
    int at[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = chunk * kChunk + wave + k * kSplitWaves;
        at[k] = verify_base(true, (i < tiles ? i : tiles - 1) * kTile, a.V) + 8 * lane;
        x[k].load(lr + at[k]);
    }
    if (both)
#pragma unroll
        for (int k = 0; k < N; ++k) y[k].load(dr + at[k]);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = chunk * kChunk + wave + k * kSplitWaves;
        if (i >= last) continue;
        sum_raw(p, x[k], i * kTile - at[k]);
        if (both) sum_raw(q, y[k], i * kTile - at[k]);
    }
    p = sum_wave(p);
    if (both) q = sum_wave(q);
    if (lane == 0) { parts[0][wave] = p; parts[1][wave] = q; }
    __syncthreads();
    if (wave == 0) {
        p = sum_parts(parts[0], kSplitWaves);
        q = sum_parts(parts[1], kSplitWaves);
        if (lane == 0) {
            row.p[g * chunks + chunk] = p;
            if (both) row.q[g * chunks + chunk] = q;
        }
    }
}

// Codes that do not lie side by side: the test sums of `per` tiles of all positions, one wave per tile and position in turns.  The
// positions of a code share cache lines; where they are all that lies between a code and the next (the prior's forward), the
// tile of all positions is one piece of memory and is copied into LDS (TS, DS: target, draft) instead of fetched anew by every
// position.
// 59 rows of 9 x 31730 fp32 (135 MB) 32 us, 4.3 TB/s; 79 of 12 x 15825 bf16 (60 MB) 26 us, bound by the exponentials and the joins.
constexpr int kCellWaves = 8;
template <bool STAGED, typename T>
__device__ __forceinline__ Sum verify_cell_sum(const T* row, int64_t sv, const T* staged, int cells, int codes, int lane) {
    float x[1][8];
    if (STAGED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = 64 * j + lane;
            const float f = verify_load(staged + (v < codes ? v : codes - 1) * cells);
            x[0][j] = v < codes ? f : -__builtin_inff();
        }
    } else verify_tile(row, sv, false, 0, codes, lane, -__builtin_inff(), x[0]);
    return sum_held(x);
}
template <bool TS, bool DS, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(kCellWaves * 64) void verify_cells_kernel(VerifyArgs a, char* ws, int per, int groups) {
    extern __shared__ __align__(16) char block[];
    const int wave = verify_wave(), lane = threadIdx.x & 63;
    const int tiles = (a.V + kTile - 1) / kTile, first = (int)((int64_t)blockIdx.x % groups) * per;
    const int64_t b = (int64_t)blockIdx.x / groups;
    const int codes = a.V - first * kTile < per * kTile ? a.V - first * kTile : per * kTile;
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)first * kTile * a.lv;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)first * kTile * a.dv;
    T* const t = reinterpret_cast<T*>(block);
    D* const d = reinterpret_cast<D*>(block + (TS ? per * kTile * a.P * sizeof(T) : 0));
    if (TS) verify_copy(lr, codes * a.P, t);
    if (DS) verify_copy(dr, codes * a.G, d);
    const int n = verify_length(a, b);
    const SplitRow row = split_row(ws, a, b);
    __syncthreads();
    const int rows = PROBS ? a.P : a.P + a.G;
    for (int i = wave; i < per * rows; i += kCellWaves) {
        const int k = i / rows, g = i % rows, off = k * kTile, rest = codes - off < kTile ? codes - off : kTile;
        if (rest <= 0) break;
        if (g < a.P) {
            if (g > n) continue;
            const Sum p = verify_cell_sum<TS>(lr + (int64_t)g * a.lp + off * a.lv, a.lv, t + (off * a.P + g), a.P, rest, lane);
            if (lane == 0) row.p[(int64_t)g * tiles + first + k] = p;
        } else if (!PROBS && g - a.P < n) {
            const int m = g - a.P;
            const Sum q = verify_cell_sum<DS>(dr + (int64_t)m * a.dg + off * a.dv, a.dv, d + (off * a.G + m), a.G, rest, lane);
            if (lane == 0) row.q[(int64_t)m * tiles + first + k] = q;
        }
    }
}

// The chunks' sums as one (one wave); `a`: this lane's first part.
__device__ __forceinline__ Sum split_join(const Exp& ex, Sum a, const Sum* parts, int chunks, int lane) {
    if (lane >= chunks) a = Sum{-__builtin_inff(), 0.f, 0.0};
    for (int i = lane + 64; i < chunks; i += 64) {
        const Sum t = parts[i];
        const float top = fmaxf(a.ref, t.ref);
        a.s = sum_moved(ex, a, top) + sum_moved(ex, t, top);
        a.ref = top;
    }
    return sum_wave(a);
}

// One tile per wave of the position that stops the row.  Every workgroup finds that position for itself from the chunks' sums,
// one wave per position; the first of a row writes it down.
template <typename T, typename D, bool PROBS>
__global__ __launch_bounds__(kSplitWaves * 64) void verify_pass_kernel(VerifyArgs a, char* ws, int chunks, int groups) {
    __shared__ Sum sums[2][kSplitWaves];
    __shared__ int state[kSplitWaves];
    __shared__ double parts64[kSplitWaves], table[32];
    const Exp ex = verify_table(table);
    const int wave = verify_wave(), lane = threadIdx.x & 63;
    const int64_t b = (int64_t)blockIdx.x / groups;
    const int first = (int)((int64_t)blockIdx.x % groups);
    const int n = verify_length(a, b);
    const SplitRow row = split_row(ws, a, b);
    Sum p = {0.f, 0.f, 1.0}, q = {0.f, 0.f, 1.0};
    int st = VERIFY_KEEP, g = 0;
    Sum pp, qq;                                            // this lane's part of the wave's position
    const auto ask = [&](int mine) {                             // (a position that is not there: the last one)
        const int at = lane < chunks ? lane : chunks - 1;
        pp = row.p[(mine < a.P ? mine : a.P - 1) * chunks + at];
        if (!PROBS && a.G > 0) qq = row.q[(mine < a.G ? mine : a.G - 1) * chunks + at];
    };
    ask(wave);
    Drafted<T, D> drafted;
    drafted.fetch(a, b, 0, lane);
    for (int base = 0; st == VERIFY_KEEP; base += kSplitWaves) {
        if (base > 0) ask(base + wave);
        const int mine = base + wave;
        int s = mine == n ? (n < a.P ? VERIFY_REJECT : VERIFY_BAD) : VERIFY_KEEP;
        // (every wave, also one whose own position is not there: all of them read position g's if its test is unsure)
        if (base > 0 && base % 64 == 0) drafted.fetch(a, b, base, lane);
        if (mine <= n && mine < a.P) {
            p = split_join(ex, pp, row.p + mine * chunks, chunks, lane);
            if (mine < n) {
                if (!PROBS) q = split_join(ex, qq, row.q + mine * chunks, chunks, lane);
                s = verify_test<PROBS>(ex, drafted.of(mine & 63), p, q, false);
            } else if (!sum_ok(p)) s = VERIFY_BAD;
        }
        __syncthreads();
        if (lane == 0) {
            sums[0][wave] = p;
            if (!PROBS) sums[1][wave] = q;
            state[wave] = s;
        }
        __syncthreads();
        for (int i = 0; i < kSplitWaves && st == VERIFY_KEEP; ++i) {     // (position n always stops: the loop ends)
            st = state[i];
            g = base + i;
            if (st == VERIFY_KEEP) continue;
            p = sums[0][i];
            if (!PROBS) q = sums[1][i];
            if (st == VERIFY_UNSURE) {
                const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)g * a.lp;
                const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)g * a.dg;
                p.s = verify_row_sum64(ex, lr, a.lv, a.unit, a.V, (double)p.ref, parts64);
                if (!PROBS) q.s = verify_row_sum64(ex, dr, a.dv, a.unit, a.V, (double)q.ref, parts64);
                st = verify_test<PROBS>(ex, drafted.of(g & 63), p, q, true);
            }
        }
    }
    const Weights w = {(double)p.ref, (double)q.ref, PROBS ? p.s : p.s / q.s, g < n};
    if (first == 0 && threadIdx.x == 0) {
        a.accepted[b] = g;
        *row.d = Decision{w.k, p.ref, q.ref, g, st};
        if (st != VERIFY_REJECT) a.next[b] = -1;
    }
    const int i = first * kSplitWaves + wave;
    if (st != VERIFY_REJECT || i * kTile >= a.V) return;
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)g * a.lp;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)g * a.dg;
    float t[8], d[8];
    verify_tile(lr, a.lv, a.unit, i * kTile, a.V, lane, -__builtin_inff(), t);
    if (w.residual) verify_tile(dr, a.dv, a.unit, i * kTile, a.V, lane, PROBS ? 0.f : -__builtin_inff(), d);
    double sp = 0.0, sq = 0.0;
    const Tile r = verify_pass<PROBS>(ex, w, t, d, sp, sq);
    sp = wave_sum(sp);
    sq = wave_sum(sq);
    if (lane == 0) {
        row.sp[i] = sp;
        row.sq[i] = sq;
        row.a[i] = r.mass;
        row.c[i] = r.c;
        row.near[i] = r.near;
    }
}

// One workgroup per row: the draw.
template <typename T, typename D, bool PROBS>
__global__ __launch_bounds__(kSplitWaves * 64) void verify_draw_kernel(VerifyArgs a, char* ws) {
    extern __shared__ double tile_a[];                           // per tile of the row: a, c, near
    __shared__ double parts64[2][kSplitWaves], lds[kTile + kTile / 8], table[32];
    const int wave = verify_wave(), lane = threadIdx.x & 63;
    const int64_t b = blockIdx.x;
    const SplitRow row = split_row(ws, a, b);
    const int tiles = (a.V + kTile - 1) / kTile, n = verify_length(a, b);
    const Decision d = *row.d;
    const double at_draw = a.r[b * a.rb];
    double* tile_c = tile_a + tiles;
    unsigned char* tile_near = reinterpret_cast<unsigned char*>(tile_c + tiles);
    double sp = 0.0, sq = 0.0;
    for (int i = threadIdx.x; i < tiles; i += kSplitWaves * 64) {      // (not written where the row draws nothing, and not used there)
        sp += row.sp[i];
        sq += row.sq[i];
        tile_a[i] = row.a[i];
        tile_c[i] = row.c[i];
        tile_near[i] = row.near[i];
    }
    const Exp ex = verify_table(table);
    if (d.st != VERIFY_REJECT) return;
    sp = wave_sum(sp);
    sq = wave_sum(sq);
    if (lane == 0) { parts64[0][wave] = sp; parts64[1][wave] = sq; }
    __syncthreads();
    sp = sq = 0.0;
#pragma unroll
    for (int i = 0; i < kSplitWaves; ++i) { sp += parts64[0][i]; sq += parts64[1][i]; }
    const Weights w = {(double)d.p_ref, (double)d.q_ref, d.k, d.g < n};
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)d.g * a.lp;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)d.g * a.dg;
    verify_finish<T, D, PROBS>(ex, a, b, at_draw, lr, dr, w, a.unit, sp, sq, tile_a, tile_c, tile_near, tiles, lds);
}

// Long rows whose codes lie side by side have a workgroup each, and are cut among workgroups -- three launches -- only where they
// are few and long.  us of a call, cut / one workgroup of 8 waves, 4 drafts, fp32 logits: 8 rows x 4096 20 / 17, x 8192 20 / 21, x 40000 21 /
// 50; 64 rows x 8192 22 / 21, x 16384 25 / 29; 128 x 16384 36 / 31, x 40000 63 / 66; 190 x 16384 42 / 33, x 40000 85 / 72.
constexpr int kRowsMin = 128, kRowsTo = 8192;
// Its waves: eight for long rows as long as there is a CU for each, two for many rows of a few tiles, else four: more leave more of
// the card idle when a row stops.  us of eight / four / two, 4 drafts, fp32 logits: 256 rows x 30000 62 / 71 / -, x 8192 25.0 / 25.5 / -,
// x 4096 20 / 19 / -; 500 rows x 8192 40 / 37 / -, x 1100 22 / 18 / 21; 700 x 4096 - / 31.4 / 31.5; 1000 x 4096 - / 40 / 37, x 8192
// - / 65 / 66; 4096 x 1100 - / 84 / 61, x 4096 - / 121 / 114, x 8192 - / 197 / 204.
constexpr int kRows8 = 256, kRows2 = 512, kRowsShort = 4096;
// Short rows, positions at a time: all at once for few rows, so that the call takes one position's time; with more rows a wave
// behind the first rejection is work in vain.  So many waves in all (us with 1024 / 2048 / 4096 / 16384, logits side by side: 1050 rows of
// 8 x 223 bf16 21 / 16 / 15 / 20, 719 of 13 x 1005 fp32 19 / 18 / 20 / 31, 300 of 12 x 300 14 / 14 / 17 / 17, 4096 of 9 x 512 26 / 26 / 27 / 35), and
// of a row whose block is staged one for so many bytes at least (2000 rows of 7 x 1000, codes of all positions side by side: 4608 /
// 6144 / 20000 bytes 65 / 44 / 49; 4096 of 9 x 512 39 / 35 / 43).
constexpr int kShortWaves = 2048;
constexpr int kShortStage = 6144;
constexpr size_t kCellBytes = 65536;                         // LDS of a tile of all positions
static bool verify_split(int64_t B, int V, bool unit) { return V > 2 * kTile && (!unit || (B < kRowsMin && V > kRowsTo)); }
// Short rows: whether the row's block of `size`-byte logits is staged, and the waves of a workgroup.
static bool verify_staged(int V, int P, int64_t lp, int64_t lv, size_t size) { return P > 1 && lp == 1 && lv == P && (size_t)V * P * size <= 32768; }
static int verify_short_waves(int64_t B, int V, int G, int P, bool staged, size_t size) {
    int64_t waves = (kShortWaves + B - 1) / B;
    const int64_t least = staged ? (int64_t)((size_t)V * P * size / kShortStage) : 0;
    if (waves < least) waves = least;
    if (waves > G + 1) waves = G + 1;
    if (waves > 16) waves = 16;
    return waves < 1 ? 1 : (int)waves;
}

template <typename T, typename D, bool PROBS>
static int verify_launch(const VerifyArgs& a, char* ws, hipStream_t st) {
    const dim3 grid((unsigned)a.B);
    if (a.V <= 2 * kTile) {
        const size_t block = (size_t)a.V * a.P * sizeof(T), room = (kTile + kTile / 8) * sizeof(double);
        const bool staged = verify_staged(a.V, a.P, a.lp, a.lv, sizeof(T));
        const dim3 blk((unsigned)verify_short_waves(a.B, a.V, a.G, a.P, staged, sizeof(T)) * 64);
        const size_t lds = staged && block > room ? block : room;
        if (a.V <= kTile) {
            if (staged) hipLaunchKernelGGL((verify_short_kernel<1, true, T, D, PROBS>), grid, blk, lds, st, a);
            else hipLaunchKernelGGL((verify_short_kernel<1, false, T, D, PROBS>), grid, blk, lds, st, a);
        } else {
            if (staged) hipLaunchKernelGGL((verify_short_kernel<2, true, T, D, PROBS>), grid, blk, lds, st, a);
            else hipLaunchKernelGGL((verify_short_kernel<2, false, T, D, PROBS>), grid, blk, lds, st, a);
        }
        return check_launch("prior_verify");
    }
    const int tiles = (a.V + kTile - 1) / kTile;
    if (verify_split(a.B, a.V, a.unit)) {
        const int chunks = (int)split_parts(a.V, a.unit), per = (tiles + kSplitWaves - 1) / kSplitWaves;
        const dim3 blk(kSplitWaves * 64);
        if (a.unit) hipLaunchKernelGGL((verify_stats_kernel<T, D, PROBS>), dim3((unsigned)(a.B * a.P * chunks)), blk, 0, st, a, ws, chunks);
        else {
            const int rows = PROBS ? a.P : a.P + a.G, each = rows < kCellWaves ? kCellWaves / rows : 1, groups = (tiles + each - 1) / each;
            size_t lds = 0;
            const size_t t_bytes = each * kTile * sizeof(T) * a.P, d_bytes = each * kTile * sizeof(D) * a.G;
            const bool t_staged = a.P > 1 && a.lp == 1 && a.lv == a.P && t_bytes <= kCellBytes;
            if (t_staged) lds += t_bytes;
            const bool d_staged = !PROBS && a.G > 1 && a.dg == 1 && a.dv == a.G && lds + d_bytes <= kCellBytes;
            if (d_staged) lds += d_bytes;
            const dim3 cgrid((unsigned)(a.B * groups)), cblk(kCellWaves * 64);
            if (t_staged && d_staged) hipLaunchKernelGGL((verify_cells_kernel<true, !PROBS, T, D, PROBS>), cgrid, cblk, lds, st, a, ws, each, groups);
            else if (t_staged) hipLaunchKernelGGL((verify_cells_kernel<true, false, T, D, PROBS>), cgrid, cblk, lds, st, a, ws, each, groups);
            else if (d_staged) hipLaunchKernelGGL((verify_cells_kernel<false, !PROBS, T, D, PROBS>), cgrid, cblk, lds, st, a, ws, each, groups);
            else hipLaunchKernelGGL((verify_cells_kernel<false, false, T, D, PROBS>), cgrid, cblk, lds, st, a, ws, each, groups);
        }
        hipLaunchKernelGGL((verify_pass_kernel<T, D, PROBS>), dim3((unsigned)(a.B * per)), blk, 0, st, a, ws, chunks, per);
        hipLaunchKernelGGL((verify_draw_kernel<T, D, PROBS>), grid, blk, (size_t)tiles * 17, st, a, ws);
        return check_launch("prior_verify");
    }
    const size_t lds = (size_t)tiles * 17;
    if (a.B <= kRows8 && a.V > kRowsShort) hipLaunchKernelGGL((verify_row_kernel<8, T, D, PROBS>), grid, dim3(512), lds, st, a);
    else if (a.B > kRows2 && a.V <= kRowsShort) hipLaunchKernelGGL((verify_row_kernel<2, T, D, PROBS>), grid, dim3(128), lds, st, a);
    else hipLaunchKernelGGL((verify_row_kernel<4, T, D, PROBS>), grid, dim3(256), lds, st, a);
    return check_launch("prior_verify");
}

}  // namespace dvq

using namespace dvq;

extern "C" size_t dvq_prior_verify_workspace_bytes(const DvqPriorVerify* v) {
    if (!v || v->B < 1 || v->V < 1 || v->P < 1 || v->G < 0) return 0;
    const bool unit = v->logits_v == 1 && (v->draft_v == 1 || v->G == 0);
    if (!verify_split(v->B, v->V, unit)) return 0;
    return (size_t)v->B * (size_t)((split_bytes(v->P, v->G, v->V, unit) + 15) / 16 * 16);
}

extern "C" int dvq_prior_verify(const DvqPriorVerify* v, void* workspace, size_t workspace_bytes, void* stream) {
    if (!v) return fail(DVQ_EINVAL, "prior_verify: null arguments");
    if (v->B < 0 || v->B > 0x7FFFFFFF || v->V < 1 || v->V > (1 << 20)) return fail(DVQ_EINVAL, "prior_verify: 0 <= B < 2^31, 1 <= V <= 2^20");
    if (v->G < 0 || v->G > 65535 || (v->P != v->G && v->P != v->G + 1) || v->P < 1)
        return fail(DVQ_EINVAL, "prior_verify: P positions of logits for G drafted codes: P = G or G + 1 (got P = %d, G = %d)", v->P, v->G);
    if ((v->logits_dtype != DVQ_F32 && v->logits_dtype != DVQ_BF16) || (v->draft_dtype != DVQ_F32 && v->draft_dtype != DVQ_BF16))
        return fail(DVQ_EINVAL, "prior_verify: dtypes must be DVQ_F32 or DVQ_BF16");
    if (v->B == 0) return DVQ_OK;
    if (!v->logits || !v->u_draw || !v->accepted || !v->next || (v->G > 0 && (!v->draft || !v->tokens || !v->u_accept)))
        return fail(DVQ_EINVAL, "prior_verify: null pointer");
    // (threads of the largest launch: the waves of a short row, a workgroup per row, or per row and part of it)
    const bool unit = v->logits_v == 1 && (v->draft_v == 1 || v->G == 0);
    const bool short_rows = v->V <= 2 * kTile, split = verify_split(v->B, v->V, unit);
    const int64_t parts = split_parts(v->V, unit) * (unit ? v->P : 1), per = (v->V + kTile * kSplitWaves - 1) / (kTile * kSplitWaves);
    const int64_t groups = !split ? 1 : parts > per ? parts : per;
    const size_t size = v->logits_dtype == DVQ_F32 ? 4 : 2;
    const int short_waves = verify_short_waves(v->B, v->V, v->G, v->P, verify_staged(v->V, v->P, v->logits_p, v->logits_v, size), size);
    if (!launch_fits(v->B * groups, (short_rows ? short_waves : kCellWaves) * 64)) return fail(DVQ_EINVAL, "prior_verify: B x P x V too large");
    const size_t need = dvq_prior_verify_workspace_bytes(v);
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return fail(DVQ_EINVAL, "prior_verify: needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : 0);
    VerifyArgs a;
    a.logits = v->logits; a.lb = v->logits_b; a.lp = v->logits_p; a.lv = v->logits_v;
    a.draft = v->draft; a.db = v->draft_b; a.dg = v->draft_g; a.dv = v->draft_v;
    a.tokens = v->tokens; a.tb = v->tokens_b; a.tg = v->tokens_g;
    a.u = v->u_accept; a.ub = v->u_accept_b; a.ug = v->u_accept_g;
    a.r = v->u_draw; a.rb = v->u_draw_b;
    a.lengths = v->lengths; a.nb = v->lengths_b;
    a.accepted = v->accepted; a.next = v->next;
    a.B = v->B; a.G = v->G; a.P = v->P; a.V = v->V;
    a.unit = a.lv == 1 && (a.dv == 1 || a.G == 0);
    char* ws = reinterpret_cast<char*>(workspace);
    hipStream_t st = as_stream(stream);
    const bool tf = v->logits_dtype == DVQ_F32, df = v->draft_dtype == DVQ_F32;
    typedef unsigned short u16;
    if (v->draft_probs) {
        if (tf) return df ? verify_launch<float, float, true>(a, ws, st) : verify_launch<float, u16, true>(a, ws, st);
        return df ? verify_launch<u16, float, true>(a, ws, st) : verify_launch<u16, u16, true>(a, ws, st);
    }
    if (tf) return df ? verify_launch<float, float, false>(a, ws, st) : verify_launch<float, u16, false>(a, ws, st);
    return df ? verify_launch<u16, float, false>(a, ws, st) : verify_launch<u16, u16, false>(a, ws, st);
}
