// Matrix product in 8-bit integers with a scale per row of x and per row of W (gfx950).
//
//   codes  c[m,k] = round(127 x[m,k] / a_m),  a_m = max_k |x[m,k]|,  s_m = a_m / 127
//   y[m,n] = act( (sum_k c[m,k] w[n,k]) s_m t_n + b_n )
//
// The sum is taken by the i8 matrix instructions in 32-bit integers and is exact (K < 2^17), so no tiling or split of k
// changes a result.  Both operands are k-contiguous ([M,K], [N,K]).
#include "common.h"

namespace dvq {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kInt8MaxBatch = 8;
struct QuantBatch {
    const void* x[kInt8MaxBatch];
    int8_t* codes[kInt8MaxBatch];
    float* scale[kInt8MaxBatch];
};
struct Int8Batch {
    const int8_t* x[kInt8MaxBatch];
    const float* xs[kInt8MaxBatch];
    const int8_t* W[kInt8MaxBatch];
    const float* ws[kInt8MaxBatch];
    const float* b[kInt8MaxBatch];
    void* y[kInt8MaxBatch];
};

__device__ __forceinline__ float int8_load(const float* p) { return *p; }
__device__ __forceinline__ float int8_load(const unsigned short* p) { return bf16_bits_to_f32(*p); }

// Code of x in a row whose factor is inv = 127 / a in 64 bits: the nearest whole number to the EXACT quotient 127 x / a,
// ties to even.  x * inv is off by at most 2^-46 (|quotient| <= 127).  A quotient that is not a half differs from every
// half by at least 2^-34 (x and a have 24-bit significands, and near a half at most 8 binary places lie between them),
// so rounding to multiples of 2^-40 first (adding and taking away 1.5 * 2^12 does that) makes a true tie exact and
// moves nothing else across one.
__device__ __forceinline__ int int8_code(float x, double inv) {
    const double t = ((double)x * inv + 6144.0) - 6144.0;
    return (int)rint(t);
}

// One workgroup per row: |x| as bit patterns orders like the values and puts infinities and NaN on top.
template <typename T>
__global__ __launch_bounds__(256) void int8_quantize_kernel(QuantBatch p, int64_t ldx, int K, int64_t ldc) {
    __shared__ unsigned top[4];
    const int64_t m = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(p.x[blockIdx.y]) + m * ldx;
    int8_t* c = p.codes[blockIdx.y] + m * ldc;
    unsigned a = 0;
    for (int k = tid; k < K; k += 256) {
        const unsigned bits = __builtin_bit_cast(unsigned, int8_load(x + k)) & 0x7FFFFFFFu;
        a = bits > a ? bits : a;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned other = __shfl_xor(a, o, 64);
        a = other > a ? other : a;
    }
    if ((tid & 63) == 0) top[tid >> 6] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) a = top[w] > a ? top[w] : a;
    const bool finite = a < 0x7F800000u;
    const double amax = (double)__builtin_bit_cast(float, a);
    const double inv = finite && a > 0 ? 127.0 / amax : 0.0;
    for (int k = tid; k < ldc; k += 256) c[k] = (k < K && inv > 0.0) ? (int8_t)int8_code(int8_load(x + k), inv) : (int8_t)0;
    if (tid == 0) p.scale[blockIdx.y][m] = finite ? (float)(amax / 127.0) : __builtin_nanf("");
}

// 16 bytes of a row from byte k on, zeros behind the row's end; never reads outside the row.
__device__ __forceinline__ i32x4 int8_chunk(const int8_t* row, int k, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) __builtin_memcpy(&v, row + k, 16);
    else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (k + j < K) v[j >> 2] |= (int)(unsigned char)row[k + j] << (8 * (j & 3));
    }
    return v;
}

// Scaled in 64 bits, rounded once: no intermediate leaves the range of 32 bits where the result does not (s is up to 2^121,
// the sum up to 2^31), at four 64-bit instructions per output.
__device__ __forceinline__ float int8_scale(int acc, float s, float t, float b, int relu) {
    const float v = (float)__builtin_fma((double)acc, (double)s * (double)t, (double)b);
    return relu && v < 0.f ? 0.f : v;
}
__device__ __forceinline__ void int8_store(float* y, float v) { *y = v; }
__device__ __forceinline__ void int8_store(unsigned short* y, float v) { *y = f32_to_bf16_bits(v); }

// Any strides and alignments: 64 x 64 outputs per workgroup, 64 k per step, operands through registers into LDS.
template <typename Y>
__global__ __launch_bounds__(256) void int8_any_kernel(Int8Batch p, int64_t ldx, int64_t ldw, int M, int K, int N, int relu,
                                                       int64_t ldy) {
    constexpr int LD = 80;                       // bytes per LDS row: 64 + 16, so that rows start 20 banks apart
    __shared__ __align__(16) int8_t sa[64 * LD], sb[64 * LD];
    const int bz = blockIdx.y;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int nt = (N + 63) / 64;
    const int m0 = (int)(blockIdx.x / nt) * 64, n0 = (int)(blockIdx.x % nt) * 64;
    const int row = tid >> 2, ch = (tid & 3) * 16;
    const int ma = m0 + row < M ? m0 + row : M - 1, nb = n0 + row < N ? n0 + row : N - 1;
    const int8_t* pa = p.x[bz] + (int64_t)ma * ldx;
    const int8_t* pb = p.W[bz] + (int64_t)nb * ldw;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    const int r = lane & 31, h = lane >> 5;
    i32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0;
    for (int k0 = 0; k0 < K; k0 += 64) {
        const i32x4 va = int8_chunk(pa, k0 + ch, K), vb = int8_chunk(pb, k0 + ch, K);
        __syncthreads();
        *reinterpret_cast<i32x4*>(sa + row * LD + ch) = va;
        *reinterpret_cast<i32x4*>(sb + row * LD + ch) = vb;
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 64; kk += 32) {
            const i32x4 fa = *reinterpret_cast<const i32x4*>(sa + (wm + r) * LD + kk + 16 * h);
            const i32x4 fb = *reinterpret_cast<const i32x4*>(sb + (wn + r) * LD + kk + 16 * h);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa, fb, acc, 0, 0, 0);
        }
    }
    const int n = n0 + wn + r;
    if (n >= N) return;
    const float t = p.ws[bz][n], bias = p.b[bz] ? p.b[bz][n] : 0.f;
    Y* y = reinterpret_cast<Y*>(p.y[bz]);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int m = m0 + wm + (e & 3) + 8 * (e >> 2) + 4 * h;
        if (m < M) int8_store(y + (int64_t)m * ldy + n, int8_scale(acc[e], p.xs[bz][m], t, bias, relu));
    }
}

}  // namespace dvq

using namespace dvq;

extern "C" int dvq_int8_quantize_rows(int n_batch, const void* const* x, int dtype, int64_t ldx, int M, int K, void* const* codes,
                                      int64_t ldc, float* const* scale, void* stream) {
    if (n_batch < 1 || n_batch > kInt8MaxBatch) return fail(DVQ_EINVAL, "int8_quantize_rows: 1..%d matrices per launch", kInt8MaxBatch);
    if (dtype != DVQ_F32 && dtype != DVQ_BF16) return fail(DVQ_EINVAL, "int8_quantize_rows: dtype must be DVQ_F32 or DVQ_BF16");
    if (M < 0 || K < 1 || K >= (1 << 17) || ldx < 0 || ldc < K || (ldc % 16) != 0)
        return fail(DVQ_EINVAL, "int8_quantize_rows: M >= 0, 1 <= K < 2^17, ldc >= K a multiple of 16 (got M = %d, K = %d, ldc = %lld)", M, K, (long long)ldc);
    if (M == 0) return DVQ_OK;
    if (!x || !codes || !scale) return fail(DVQ_EINVAL, "int8_quantize_rows: null pointer");
    QuantBatch p;
    for (int i = 0; i < n_batch; ++i) {
        if (!x[i] || !codes[i] || !scale[i]) return fail(DVQ_EINVAL, "int8_quantize_rows: null pointer");
        p.x[i] = x[i]; p.codes[i] = reinterpret_cast<int8_t*>(codes[i]); p.scale[i] = scale[i];
    }
    const dim3 grid((unsigned)M, (unsigned)n_batch);
    if (dtype == DVQ_F32) hipLaunchKernelGGL(int8_quantize_kernel<float>, grid, dim3(256), 0, as_stream(stream), p, ldx, K, ldc);
    else hipLaunchKernelGGL(int8_quantize_kernel<unsigned short>, grid, dim3(256), 0, as_stream(stream), p, ldx, K, ldc);
    return check_launch("int8_quantize_rows");
}

extern "C" int dvq_linear_int8(int n_batch, const void* const* x, const float* const* xs, int64_t ldx, const void* const* W,
                               const float* const* ws, int64_t ldw, const float* const* b, int M, int K, int N, int relu,
                               void* const* y, int y_dtype, int64_t ldy, void* stream) {
    if (n_batch < 1 || n_batch > kInt8MaxBatch) return fail(DVQ_EINVAL, "linear_int8: 1..%d products per launch", kInt8MaxBatch);
    if (y_dtype != DVQ_F32 && y_dtype != DVQ_BF16) return fail(DVQ_EINVAL, "linear_int8: y_dtype must be DVQ_F32 or DVQ_BF16");
    if (M < 0 || N < 1 || K < 1 || K >= (1 << 17)) return fail(DVQ_EINVAL, "linear_int8: M >= 0, N >= 1, 1 <= K < 2^17 (got M = %d, N = %d, K = %d)", M, N, K);
    if (ldx < 0 || ldw < 0 || ldy < N) return fail(DVQ_EINVAL, "linear_int8: bad row stride");
    if (M == 0) return DVQ_OK;
    if (!x || !xs || !W || !ws || !y) return fail(DVQ_EINVAL, "linear_int8: null pointer");
    Int8Batch p;
    for (int i = 0; i < n_batch; ++i) {
        if (!x[i] || !xs[i] || !W[i] || !ws[i] || !y[i]) return fail(DVQ_EINVAL, "linear_int8: null pointer");
        p.x[i] = reinterpret_cast<const int8_t*>(x[i]); p.xs[i] = xs[i];
        p.W[i] = reinterpret_cast<const int8_t*>(W[i]); p.ws[i] = ws[i];
        p.b[i] = b ? b[i] : nullptr;
        p.y[i] = y[i];
    }
    const int64_t tiles = (int64_t)((M + 63) / 64) * ((N + 63) / 64);
    if (tiles > 0x7FFFFFFF) return fail(DVQ_EINVAL, "linear_int8: M x N too large");
    const dim3 grid((unsigned)tiles, (unsigned)n_batch);
    if (y_dtype == DVQ_F32) hipLaunchKernelGGL(int8_any_kernel<float>, grid, dim3(256), 0, as_stream(stream), p, ldx, ldw, M, K, N, relu, ldy);
    else hipLaunchKernelGGL(int8_any_kernel<unsigned short>, grid, dim3(256), 0, as_stream(stream), p, ldx, ldw, M, K, N, relu, ldy);
    return check_launch("linear_int8");
}
