// Verification of drafted codes against the prior's distribution (gfx950).
//
// A cheap model drafts codes x_0 .. x_{n-1} with distributions q_g, the prior gives its own distributions p_g for the
// same history in one pass.  Code x_g is kept while  u_g q_g(x_g) < p_g(x_g)  (a draw that is right with probability
// min(1, p/q)); at the first one that is not, the row's next code is drawn from max(p_g - q_g, 0) / mass, and behind the
// last kept one from p_n.  The codes that come out are distributed as if the prior had drawn them one by one.
//
// The outputs are whole numbers, so the comparison and the draw are made in 64 bits: next to a border 32 bits decide
// differently for another order of summation.
#include "common.h"

namespace dvq {

// Residual mass below this is rounding (p and q equal up to 64-bit noise): the draw is then from p itself.
constexpr double kVerifyNoMass = 9.094947017729282e-13;   // 2^-40

struct VerifyArgs {
    const void* logits; int64_t lb, lp, lv;
    const void* draft; int64_t db, dg, dv;
    const int64_t* tokens; int64_t tb, tg;
    const double* u; int64_t ub, ug;
    const double* r; int64_t rb;
    const int64_t* lengths; int64_t nb;
    int64_t* accepted; int64_t* next;
    int64_t B; int G, P, V;
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

// Maximum and sum of exponentials of one row of logits; ok = false where the row has no distribution (nothing above
// -inf, a NaN or +inf).
struct RowStats { float m; double s; bool ok; };

template <int WAVES, typename T>
__device__ RowStats verify_stats(const T* row, int64_t sv, int V, double* sh) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    float m = -__builtin_inff();
    bool bad = false;
    for (int v = tid; v < V; v += WAVES * 64) {
        const float x = verify_load(row + v * sv);
        bad |= !(x < __builtin_inff());
        m = fmaxf(m, x);
    }
    m = wave_max(m);
    bad = __any(bad);
    __syncthreads();
    if (lane == 0) { sh[wave] = (double)m; sh[WAVES + wave] = bad ? 1.0 : 0.0; }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) { m = fmaxf(m, (float)sh[w]); bad |= sh[WAVES + w] != 0.0; }
    RowStats st;
    st.m = m;
    st.ok = !bad && m > -__builtin_inff();
    st.s = 1.0;
    if (!st.ok) return st;                      // (the same for every thread of the workgroup)
    double s = 0.0;
    for (int v = tid; v < V; v += WAVES * 64) s += exp((double)verify_load(row + v * sv) - (double)m);
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) sh[wave] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < WAVES; ++w) s += sh[w];
    st.s = s;
    return st;
}

// One workgroup per row, position after position until the first rejection.
template <int WAVES, typename T, typename D, bool PROBS>
__global__ __launch_bounds__(WAVES * 64) void verify_row_kernel(VerifyArgs a) {
    __shared__ double sh[2 * WAVES];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int V = a.V;
    const T* lrow = reinterpret_cast<const T*>(a.logits) + b * a.lb;
    const D* drow = reinterpret_cast<const D*>(a.draft) + b * a.db;
    int n = a.G;
    if (a.lengths) {
        const int64_t given = a.lengths[b * a.nb];
        n = given < 0 ? 0 : given > a.G ? a.G : (int)given;
    }
    RowStats tp, tq;
    tq.m = 0.f; tq.s = 1.0; tq.ok = true;
    int g = 0;
    bool rejected = false, ok = true;
    for (; g < n; ++g) {
        tp = verify_stats<WAVES>(lrow + g * a.lp, a.lv, V, sh);
        if (!PROBS) tq = verify_stats<WAVES>(drow + g * a.dg, a.dv, V, sh);
        if (!tp.ok || !tq.ok) { ok = false; break; }
        const int64_t x = a.tokens[b * a.tb + g * a.tg];
        double px = 0.0, qx = 0.0;
        if (x >= 0 && x < V) {
            px = exp((double)verify_load(lrow + g * a.lp + x * a.lv) - (double)tp.m) / tp.s;
            const double d = (double)verify_load(drow + g * a.dg + x * a.dv);
            qx = PROBS ? d : exp(d - (double)tq.m) / tq.s;
            if (PROBS && !(d >= 0.0 && d < (double)__builtin_inff())) { ok = false; break; }
        }
        if (!(a.u[b * a.ub + g * a.ug] * qx < px)) { rejected = true; break; }
    }
    if (tid == 0) a.accepted[b] = g;
    if (ok && !rejected) {                      // every draft kept: one more code where the prior has looked that far
        if (g >= a.P) ok = false;
        else { tp = verify_stats<WAVES>(lrow + g * a.lp, a.lv, V, sh); ok = tp.ok; }
    }
    if (!ok) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    // The row's codes cut into one run of codes per wave: mass of each run, then the run that holds the draw.
    const T* lr = lrow + g * a.lp;
    const D* dr = drow + g * a.dg;
    bool bad = false;
    const int run = ((V + WAVES - 1) / WAVES + 63) / 64 * 64;
    auto mass = [&](int v, bool residual) -> double {
        const double p = exp((double)verify_load(lr + v * a.lv) - (double)tp.m) / tp.s;
        if (!residual) return p;
        const double d = (double)verify_load(dr + v * a.dv);
        if (PROBS && !(d >= 0.0 && d < (double)__builtin_inff())) bad = true;
        const double w = p - (PROBS ? d : exp(d - (double)tq.m) / tq.s);
        return w > 0.0 ? w : 0.0;
    };
    double total = 0.0;
    bool residual = rejected;
    for (int pass = 0; pass < 2; ++pass) {
        double s = 0.0;
        for (int v = wave * run + lane; v < V && v < (wave + 1) * run; v += 64) s += mass(v, residual);
        s = wave_sum(s);
        bad = __any(bad);
        __syncthreads();
        if (lane == 0) { sh[wave] = s; sh[WAVES + wave] = bad ? 1.0 : 0.0; }
        __syncthreads();
        total = 0.0;
        for (int w = 0; w < WAVES; ++w) { total += sh[w]; bad |= sh[WAVES + w] != 0.0; }
        if (!residual || bad || total > kVerifyNoMass) break;
        residual = false;                       // nothing left over: from p
    }
    if (bad) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    // First code whose cumulated mass exceeds the threshold; if rounding leaves none, the last code with mass.
    const double thr = a.r[b * a.rb] * total;
    double before = 0.0;
    int w = 0, last = 0;
    for (; w < WAVES; ++w) {
        if (sh[w] > 0.0) last = w;
        if (before + sh[w] > thr) break;
        before += sh[w];
    }
    const bool over = w == WAVES;
    if (over) { w = last; before = -1.0; }
    if (wave != w) return;
    int found = -1;
    for (int base = w * run; base < V && base < (w + 1) * run && found < 0; base += 64) {
        const int v = base + lane;
        const double x = (v < V && v < (w + 1) * run) ? mass(v, residual) : 0.0;
        double incl = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double t = __shfl_up(incl, o, 64);
            if (lane >= o) incl += t;
        }
        const unsigned long long hit = __ballot(!over && before + incl > thr && x > 0.0);
        if (hit) found = base + __ffsll(hit) - 1;
        before += __shfl(incl, 63, 64);
    }
    if (found < 0)                              // (the run's own sum was taken in another order)
        for (int base = w * run; base < V && base < (w + 1) * run; base += 64) {
            const int v = base + lane;
            const unsigned long long some = __ballot(v < V && v < (w + 1) * run && mass(v, residual) > 0.0);
            if (some) found = base + 63 - __clzll(some);
        }
    if (lane == 0) a.next[b] = found;
}

template <typename T, typename D, bool PROBS>
static int verify_launch(const VerifyArgs& a, hipStream_t st) {
    if (a.V <= 4096) hipLaunchKernelGGL((verify_row_kernel<4, T, D, PROBS>), dim3((unsigned)a.B), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((verify_row_kernel<16, T, D, PROBS>), dim3((unsigned)a.B), dim3(1024), 0, st, a);
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
