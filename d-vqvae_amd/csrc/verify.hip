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
//   Draw: one position per row, 64-bit exponentials.  The row is cut into tiles of 512 codes, one wave each; the masses
//     of the tiles find the tile, a scan inside it the code.
// Three forms: rows of up to 1024 codes stay in the registers of one wave per position; longer rows have a workgroup per
// row that stops at the first rejection; few long rows, and long rows whose positions lie interleaved in memory, are cut
// among workgroups (three launches).
#include "common.h"

namespace dvq {

// Residual mass below this is rounding (p and q equal up to 64-bit noise): the draw is then from p itself.
constexpr double kVerifyNoMass = 9.094947017729282e-13;   // 2^-40
constexpr int kTile = 512;                                // codes of a tile: 8 per lane
// Relative error of u q / p from sums taken in 32 bits.  A term exp2((x - ref) log2 e) carries |x - ref| 1.5 * 2^-23 from its
// argument (difference, constant and product rounded) and 2^-23 from the exponential; eight of them are added in 32 bits
// (7 * 2^-24), everything after that in 64.  ref lies at most kVerifySlack below the largest logit and the mean of
// |x - ref| under the distribution is at most kVerifySlack + ln V <= 8 + 13.9, so a sum is off by less than
// 22 * 1.5 * 2^-23 + 2^-23 + 7 * 2^-24 = 4.5e-6 relative, the quotient of two by less than 1e-5.  Four times that:
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

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// exp(d) in 64 bits: d = k ln 2 + f with |f| <= ln 2 / 2 (ln 2 in two parts), the Taylor polynomial of degree 13 (its rest
// is below f^14 / 14! = 4e-18), scaled by 2^k.  NaN stays NaN, below -746 the result is 0.
__device__ __forceinline__ double verify_exp(double d) {
    const double k = rint(d * 1.4426950408889634);
    double f = __builtin_fma(-k, 0.6931471805599453, d);
    f = __builtin_fma(-k, 2.3190468138462996e-17, f);
    double s = 1.0 / 6227020800.0;
    s = __builtin_fma(s, f, 1.0 / 479001600.0);
    s = __builtin_fma(s, f, 1.0 / 39916800.0);
    s = __builtin_fma(s, f, 1.0 / 3628800.0);
    s = __builtin_fma(s, f, 1.0 / 362880.0);
    s = __builtin_fma(s, f, 1.0 / 40320.0);
    s = __builtin_fma(s, f, 1.0 / 5040.0);
    s = __builtin_fma(s, f, 1.0 / 720.0);
    s = __builtin_fma(s, f, 1.0 / 120.0);
    s = __builtin_fma(s, f, 1.0 / 24.0);
    s = __builtin_fma(s, f, 1.0 / 6.0);
    s = __builtin_fma(s, f, 0.5);
    s = __builtin_fma(s, f, 1.0);
    s = __builtin_fma(s, f, 1.0);
    return d < -746.0 ? 0.0 : __builtin_ldexp(s, (int)k);
}

// exp(x - ref) in 32 bits for the tests.
__device__ __forceinline__ float verify_exp32(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }

// This lane's eight codes of the tile that starts at code v0, `fill` behind the row's end.  Where target and draft both
// have unit stride: codes v0 + 8 lane + j (16-byte loads at any alignment), otherwise v0 + 64 j + lane for both.
template <typename T>
__device__ __forceinline__ void verify_tile(const T* row, int64_t sv, bool unit, int v0, int V, int lane, float fill, float (&x)[8]) {
    if (unit) {
        const int v = v0 + 8 * lane;
        if (v + 8 <= V) {
            if constexpr (sizeof(T) == 2) {
                u16x8 w;
                __builtin_memcpy(&w, row + v, 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = bf16_bits_to_f32(w[j]);
            } else {
                f32x4 w[2];
                __builtin_memcpy(&w[0], row + v, 16);
                __builtin_memcpy(&w[1], row + v + 4, 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = w[j >> 2][j & 3];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = v + j < V ? verify_load(row + v + j) : fill;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = v0 + 64 * j + lane;
            x[j] = v < V ? verify_load(row + v * sv) : fill;
        }
    }
}

// Reference point and sum of exp(x - ref) of logits seen so far; no distribution: ref = -inf, or s not a number (a NaN or
// +inf among the logits makes it one).
struct Sum { float ref; double s; };
__device__ __forceinline__ bool sum_ok(const Sum& a) { return a.ref > -__builtin_inff() && a.s == a.s; }

// The reference moves up only where the next eight exceed it by more than kVerifySlack, and then exactly.
__device__ __forceinline__ void sum_add(Sum& a, const float (&x)[8]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
    if (m > a.ref + kVerifySlack) {
        a.s *= verify_exp((double)a.ref - (double)m);
        a.ref = m;
    }
    const float ref = a.ref > -__builtin_inff() ? a.ref : 0.f;       // (nothing but -inf and NaN so far)
    float f = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f += verify_exp32(x[j] - ref);
    a.s += (double)f;
}
__device__ __forceinline__ Sum sum_wave(Sum a) {
    const float top = wave_max(a.ref);
    a.s = wave_sum(a.ref > -__builtin_inff() ? a.s * verify_exp((double)a.ref - (double)top) : a.s);
    a.ref = top;
    return a;
}
template <int N>
__device__ __forceinline__ Sum sum_join(const Sum* parts) {         // the same for every thread that calls it
    Sum a = parts[0];
#pragma unroll
    for (int i = 1; i < N; ++i) a.ref = fmaxf(a.ref, parts[i].ref);
    a.s = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) a.s += parts[i].ref > -__builtin_inff() ? parts[i].s * verify_exp((double)parts[i].ref - (double)a.ref) : parts[i].s;
    return a;
}

enum { VERIFY_KEEP = 0, VERIFY_REJECT = 1, VERIFY_BAD = 2, VERIFY_UNSURE = 3 };

// The test of one drafted code; p, q: sums of the position's logits (q unused with PROBS).  `exact`: the sums were taken
// in 64 bits.
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ int verify_test(const VerifyArgs& a, int64_t b, int g, const Sum& p, const Sum& q, bool exact) {
    if (!sum_ok(p) || (!PROBS && !sum_ok(q))) return VERIFY_BAD;
    const int64_t x = a.tokens[b * a.tb + g * a.tg];
    if (x < 0 || x >= a.V) return VERIFY_REJECT;
    const float t = verify_load(reinterpret_cast<const T*>(a.logits) + b * a.lb + g * a.lp + x * a.lv);
    const float d = verify_load(reinterpret_cast<const D*>(a.draft) + b * a.db + g * a.dg + x * a.dv);
    if (PROBS && !(d >= 0.f && d < __builtin_inff())) return VERIFY_BAD;
    const double px = verify_exp((double)t - (double)p.ref) / p.s;
    const double lhs = a.u[b * a.ub + g * a.ug] * (PROBS ? (double)d : verify_exp((double)d - (double)q.ref) / q.s);
    if (!exact && px > 0.0 && lhs > 0.0 && !(fabs(lhs - px) > kVerifyMargin * px)) return VERIFY_UNSURE;
    return lhs < px ? VERIFY_KEEP : VERIFY_REJECT;
}

__device__ __forceinline__ int verify_length(const VerifyArgs& a, int64_t b) {
    if (!a.lengths) return a.G;
    const int64_t n = a.lengths[b * a.nb];
    return n < 0 ? 0 : n > a.G ? a.G : (int)n;
}

// What the draw needs: reference points and reciprocal sums (64 bits) of p and q, and whether q is taken off.
struct Draw { double p_ref, p_inv, q_ref, q_inv; bool residual; };

// Mass of this lane's eight codes of a tile; a given probability that is none makes it NaN.
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ void verify_mass(const Draw& d, const float (&t)[8], const float (&q)[8], double (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = verify_exp((double)t[j] - d.p_ref) * d.p_inv;
        if (d.residual) {
            const double e = PROBS ? (double)q[j] : verify_exp((double)q[j] - d.q_ref) * d.q_inv;
            const bool bad = PROBS && !(q[j] >= 0.f && q[j] < __builtin_inff());
            w[j] = bad ? __builtin_nan("") : fmax(w[j] - e, 0.0);
        }
    }
}
template <typename T, typename D, bool PROBS>
__device__ __forceinline__ void verify_tile_mass(const VerifyArgs& a, const T* lr, const D* dr, const Draw& d, int v0, int lane, double (&w)[8]) {
    float t[8], q[8];
    verify_tile(lr, a.lv, a.unit, v0, a.V, lane, -__builtin_inff(), t);
    if (d.residual) verify_tile(dr, a.dv, a.unit, v0, a.V, lane, PROBS ? 0.f : -__builtin_inff(), q);
    verify_mass<T, D, PROBS>(d, t, q, w);
}
__device__ __forceinline__ double verify_sum8(const double (&w)[8]) {
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
}

// One wave: the first code of the tile at v0 whose cumulated mass (with `before` in front of it) exceeds thr, the last code
// with mass if none does (the tile's own sum was taken in another order) or if `over`.  w: the masses as verify_tile lays
// them out; lds: 8 x 72 doubles of this wave's own.
__device__ __forceinline__ int verify_locate(const double (&w)[8], bool unit, int v0, double before, double thr, bool over, double* lds) {
    const int lane = threadIdx.x & 63;
    double c[8];
    if (unit) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = w[j];
    } else {
        // from 64 j + lane to 8 lane + j
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
    double incl = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(incl, o, 64);
        if (lane >= o) incl += t;
    }
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
    return v0 + 8 * l + __shfl(at, l, 64);
}

// The tile that holds the draw, from the masses of all tiles (one wave): returns its number, `before` = mass in front of it;
// over: rounding leaves none, the last tile with mass.
__device__ __forceinline__ int verify_pick(const double* mass, int tiles, double thr, double& before, bool& over) {
    const int lane = threadIdx.x & 63;
    before = 0.0;
    int last = 0;
    for (int base = 0; base < tiles; base += 64) {
        const double m = base + lane < tiles ? mass[base + lane] : 0.0;
        double incl = m;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double t = __shfl_up(incl, o, 64);
            if (lane >= o) incl += t;
        }
        const unsigned long long some = __ballot(m > 0.0), hit = __ballot(m > 0.0 && before + incl > thr);
        if (hit) {
            const int l = __ffsll(hit) - 1;
            before += __shfl(incl - m, l, 64);
            over = false;
            return base + l;
        }
        if (some) last = base + 63 - __clzll(some);
        before += __shfl(incl, 63, 64);
    }
    over = true;
    return last;
}
// Sum of the masses of all tiles in the order that verify_pick takes (one wave).
__device__ __forceinline__ double verify_total(const double* mass, int tiles) {
    const int lane = threadIdx.x & 63;
    double total = 0.0;
    for (int base = 0; base < tiles; base += 64) total += wave_sum(base + lane < tiles ? mass[base + lane] : 0.0);
    return total;
}

// Sum of exp(x - ref) of a whole row in 64 bits, codes dealt to `waves` waves tile by tile; this wave's share.
template <typename T>
__device__ __forceinline__ double verify_sum64(const T* row, int64_t sv, bool unit, int V, double ref, int first, int step, int lane) {
    double s = 0.0;
    for (int v0 = first * kTile; v0 < V; v0 += step * kTile) {
        float x[8];
        verify_tile(row, sv, unit, v0, V, lane, -__builtin_inff(), x);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += verify_exp((double)x[j] - ref);
    }
    return wave_sum(s);
}

// ------------------------------------------------------------------------------------------------ rows of up to 1024 codes
// One workgroup per row, one wave per position: `blockDim / 64` positions at a time until the first that stops the row.
// Its wave holds the position's logits in registers and draws from them.
template <int TILES, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(1024) void verify_short_kernel(VerifyArgs a) {
    __shared__ int state[16];
    __shared__ double lds[kTile + kTile / 8];
    const int64_t b = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int V = a.V;
    const int n = verify_length(a, b);
    const float none = -__builtin_inff();
    for (int base = 0;; base += waves) {
        const int g = base + wave;                               // n: the position behind all drafts
        float t[TILES][8], q[TILES][8];
        const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb + (int64_t)g * a.lp;
        const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db + (int64_t)g * a.dg;
        Sum p = {none, 0.0}, s = {none, 0.0};
        int st = g > n ? VERIFY_KEEP : g == n ? VERIFY_REJECT : VERIFY_KEEP;
        if (g <= n && g < a.P) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) verify_tile(lr, a.lv, a.unit, i * kTile, V, lane, none, t[i]);
            if (!PROBS && g < n)
#pragma unroll
                for (int i = 0; i < TILES; ++i) verify_tile(dr, a.dv, a.unit, i * kTile, V, lane, none, q[i]);
#pragma unroll
            for (int i = 0; i < TILES; ++i) sum_add(p, t[i]);
            p = sum_wave(p);
            if (g < n) {
                if (!PROBS) {
#pragma unroll
                    for (int i = 0; i < TILES; ++i) sum_add(s, q[i]);
                    s = sum_wave(s);
                }
                st = verify_test<T, D, PROBS>(a, b, g, p, s, false);
            } else if (!sum_ok(p)) st = VERIFY_BAD;
        }
        // sums in 64 bits: of the position that may stop the row, and of one too near to tell
        if (st == VERIFY_REJECT || st == VERIFY_UNSURE) {
            if (g < a.P && sum_ok(p)) {
                double e = 0.0;
#pragma unroll
                for (int i = 0; i < TILES; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) e += verify_exp((double)t[i][j] - (double)p.ref);
                p.s = wave_sum(e);
            }
            if (!PROBS && g < n) {
                double e = 0.0;
#pragma unroll
                for (int i = 0; i < TILES; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) e += verify_exp((double)q[i][j] - (double)s.ref);
                s.s = wave_sum(e);
            }
            if (st == VERIFY_UNSURE) st = verify_test<T, D, PROBS>(a, b, g, p, s, true);
        }
        int stop = st == VERIFY_KEEP ? waves : 0;                // first wave of this round whose position stops the row
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
        Draw d = {(double)p.ref, 1.0 / p.s, (double)s.ref, 1.0 / s.s, g < n};
        if (PROBS && g < n)
#pragma unroll
            for (int i = 0; i < TILES; ++i) verify_tile(dr, a.dv, a.unit, i * kTile, V, lane, 0.f, q[i]);
        double w[TILES][8], mass[TILES], total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            total = 0.0;
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                verify_mass<T, D, PROBS>(d, t[i], q[i], w[i]);
                total += mass[i] = wave_sum(verify_sum8(w[i]));
            }
            if (!d.residual || !(total <= kVerifyNoMass)) break;
            d.residual = false;                                  // nothing left over: from p
        }
        if (total != total) {
            if (lane == 0) a.next[b] = -1;
            return;
        }
        const double thr = a.r[b * a.rb] * total;
        int at = 0;
        if (TILES == 1) at = verify_locate(w[0], a.unit, 0, 0.0, thr, !(total > thr), lds);
        else {
            const bool second = mass[0] > thr ? false : (mass[TILES - 1] > 0.0 || !(mass[0] > 0.0));
            at = second ? verify_locate(w[TILES - 1], a.unit, kTile, mass[0], thr, !(total > thr), lds)
                        : verify_locate(w[0], a.unit, 0, 0.0, thr, !(mass[0] > thr), lds);
        }
        if (lane == 0) a.next[b] = at;
        return;
    }
}

// --------------------------------------------------------------------------------- longer rows, one workgroup per row
template <int WAVES, typename T>
__device__ __forceinline__ Sum verify_row_sum(const T* row, int64_t sv, bool unit, int V, Sum* parts) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    Sum a = {-__builtin_inff(), 0.0};
#pragma unroll 4
    for (int v0 = wave * kTile; v0 < V; v0 += WAVES * kTile) {
        float x[8];
        verify_tile(row, sv, unit, v0, V, lane, -__builtin_inff(), x);
        sum_add(a, x);
    }
    a = sum_wave(a);
    __syncthreads();
    if (lane == 0) parts[wave] = a;
    __syncthreads();
    return sum_join<WAVES>(parts);
}
template <int WAVES, typename T>
__device__ __forceinline__ double verify_row_sum64(const T* row, int64_t sv, bool unit, int V, double ref, double* parts) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const double s = verify_sum64(row, sv, unit, V, ref, wave, WAVES, lane);
    __syncthreads();
    if (lane == 0) parts[wave] = s;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += parts[w];
    return all;
}

template <int WAVES, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(WAVES * 64) void verify_row_kernel(VerifyArgs a) {
    extern __shared__ double mass[];                             // one per tile of the row
    __shared__ Sum parts[WAVES];
    __shared__ double parts64[WAVES];
    __shared__ double lds[kTile + kTile / 8];
    const int64_t b = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int V = a.V, tiles = (V + kTile - 1) / kTile;
    const int n = verify_length(a, b);
    const T* lr = reinterpret_cast<const T*>(a.logits) + b * a.lb;
    const D* dr = reinterpret_cast<const D*>(a.draft) + b * a.db;
    Sum p = {0.f, 1.0}, q = {0.f, 1.0};
    int g = 0, st = VERIFY_KEEP;
    bool exact = false;
    for (; g < n; ++g, lr += a.lp, dr += a.dg) {
        p = verify_row_sum<WAVES>(lr, a.lv, a.unit, V, parts);
        if (!PROBS) q = verify_row_sum<WAVES>(dr, a.dv, a.unit, V, parts);
        st = verify_test<T, D, PROBS>(a, b, g, p, q, false);     // (the same for every thread: one code's values)
        exact = false;
        if (st == VERIFY_UNSURE) {
            p.s = verify_row_sum64<WAVES>(lr, a.lv, a.unit, V, (double)p.ref, parts64);
            if (!PROBS) q.s = verify_row_sum64<WAVES>(dr, a.dv, a.unit, V, (double)q.ref, parts64);
            st = verify_test<T, D, PROBS>(a, b, g, p, q, true);
            exact = true;
        }
        if (st != VERIFY_KEEP) break;
    }
    if (threadIdx.x == 0) a.accepted[b] = g;
    if (st == VERIFY_KEEP && g < a.P) {                          // every draft kept: one more code
        p = verify_row_sum<WAVES>(lr, a.lv, a.unit, V, parts);
        st = sum_ok(p) ? VERIFY_REJECT : VERIFY_BAD;
        exact = false;
    }
    if (st != VERIFY_REJECT) {
        if (threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    const bool residual = g < n;
    if (!exact) {
        p.s = verify_row_sum64<WAVES>(lr, a.lv, a.unit, V, (double)p.ref, parts64);
        if (!PROBS && residual) q.s = verify_row_sum64<WAVES>(dr, a.dv, a.unit, V, (double)q.ref, parts64);
    }
    // (a code outside the table is rejected before its draft's sums are needed: they are there all the same)
    Draw d = {(double)p.ref, 1.0 / p.s, (double)q.ref, 1.0 / q.s, residual};
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int i = wave; i < tiles; i += WAVES) {
            double w[8];
            verify_tile_mass<T, D, PROBS>(a, lr, dr, d, i * kTile, lane, w);
            const double m = wave_sum(verify_sum8(w));
            if (lane == 0) mass[i] = m;
        }
        __syncthreads();
        total = verify_total(mass, tiles);                       // every wave for itself, in one order
        if (!d.residual || !(total <= kVerifyNoMass)) break;
        d.residual = false;                                      // nothing left over: from p
        __syncthreads();
    }
    if (wave != 0) return;
    if (total != total) {
        if (lane == 0) a.next[b] = -1;
        return;
    }
    const double thr = a.r[b * a.rb] * total;
    double before, w[8];
    bool over;
    const int i = verify_pick(mass, tiles, thr, before, over);
    verify_tile_mass<T, D, PROBS>(a, lr, dr, d, i * kTile, lane, w);
    const int at = verify_locate(w, a.unit, i * kTile, before, thr, over, lds);
    if (lane == 0) a.next[b] = at;
}

template <typename T, typename D, bool PROBS>
static int verify_launch(const VerifyArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)a.B);
    if (a.V <= 2 * kTile) {
        // positions at a time: all at once for few rows, one after the other where the rows alone fill the card
        int64_t waves = 8192 / (a.B > 0 ? a.B : 1);
        if (waves > a.G + 1) waves = a.G + 1;
        if (waves > 16) waves = 16;
        if (waves < 1) waves = 1;
        const dim3 blk((unsigned)waves * 64);
        if (a.V <= kTile) hipLaunchKernelGGL((verify_short_kernel<1, T, D, PROBS>), grid, blk, 0, st, a);
        else hipLaunchKernelGGL((verify_short_kernel<2, T, D, PROBS>), grid, blk, 0, st, a);
        return check_launch("prior_verify");
    }
    const size_t lds = (size_t)((a.V + kTile - 1) / kTile) * sizeof(double);
    if (a.B >= 768) hipLaunchKernelGGL((verify_row_kernel<4, T, D, PROBS>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((verify_row_kernel<8, T, D, PROBS>), grid, dim3(512), lds, st, a);
    return check_launch("prior_verify");
}

}  // namespace dvq

using namespace dvq;

extern "C" int dvq_prior_verify(const DvqPriorVerify* v, void* stream) {
    if (!v) return fail(DVQ_EINVAL, "prior_verify: null arguments");
    if (v->B < 0 || v->B > 0x7FFFFFFF || v->V < 1 || v->V > (1 << 20)) return fail(DVQ_EINVAL, "prior_verify: 0 <= B < 2^31, 1 <= V <= 2^20");
    if (v->G < 0 || v->G > 65535 || (v->P != v->G && v->P != v->G + 1) || v->P < 1)
        return fail(DVQ_EINVAL, "prior_verify: P positions of logits for G drafted codes: P = G or G + 1 (got P = %d, G = %d)", v->P, v->G);
    if ((v->logits_dtype != DVQ_F32 && v->logits_dtype != DVQ_BF16) || (v->draft_dtype != DVQ_F32 && v->draft_dtype != DVQ_BF16))
        return fail(DVQ_EINVAL, "prior_verify: dtypes must be DVQ_F32 or DVQ_BF16");
    if (v->B == 0) return DVQ_OK;
    if (!v->logits || !v->u_draw || !v->accepted || !v->next || (v->G > 0 && (!v->draft || !v->tokens || !v->u_accept)))
        return fail(DVQ_EINVAL, "prior_verify: null pointer");
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
    hipStream_t st = as_stream(stream);
    const bool tf = v->logits_dtype == DVQ_F32, df = v->draft_dtype == DVQ_F32;
    typedef unsigned short u16;
    if (v->draft_probs) {
        if (tf) return df ? verify_launch<float, float, true>(a, st) : verify_launch<float, u16, true>(a, st);
        return df ? verify_launch<u16, float, true>(a, st) : verify_launch<u16, u16, true>(a, st);
    }
    if (tf) return df ? verify_launch<float, float, false>(a, st) : verify_launch<float, u16, false>(a, st);
    return df ? verify_launch<u16, float, false>(a, st) : verify_launch<u16, u16, false>(a, st);
}
