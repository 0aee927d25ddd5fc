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
// Up to so many 64 x 64 tiles the kernel that splits k runs: its workgroups (four to a tile) then fit the CUs in one round.
// Tiles against split, int8 operands in place: 64 tiles (128 x 2048 x 2048) 9.1 / 8.4 us, 32 (100 x 1000 x 512) 6.0 / 4.9;
// 80 tiles (128 x 2560 x 1024) 6.8 / 8.7, 96 (200 x 1536 x 4096) 13.8 / 21.5.
constexpr int kInt8SplitTo = 64;
// Floats are quantised by every workgroup of 16 x 16 outputs for itself -- one launch, no workspace, the rows read once per 16
// channels -- as long as the workgroups fit the chip in a round: two launches / one, us of a call, fp32: 64 x 4096 -> 1024 (256 workgroups)
// 22 / 15, 128 x 2560 -> 1024 (512) 17 / 17, 256 x 2560 -> 1024 (1024) 17 / 29; up to 1024 features, where four fit a CU, 256 x 1024 ->
// 1024 16 / 14.
constexpr int kInt8OneLaunch = 256, kInt8OneLaunchShort = 1024;
struct Int8Prepare {
    const void* x[kInt8MaxBatch];
    const int8_t* W[kInt8MaxBatch];
    int8_t* codes[kInt8MaxBatch];
    int8_t* w_codes[kInt8MaxBatch];
    float* scale[kInt8MaxBatch];
};
struct Int8Batch {
    const void* x[kInt8MaxBatch];
    const float* xs[kInt8MaxBatch];
    const int8_t* W[kInt8MaxBatch];
    const float* ws[kInt8MaxBatch];
    const float* b[kInt8MaxBatch];
    void* y[kInt8MaxBatch];
};

// Code of x in a row whose factor is inv = 127 / a in 64 bits, in the low 8 bits: the nearest whole number to the EXACT quotient
// 127 x / a, ties to even.  The first sum rounds x * inv to a multiple of 2^-40 (6144 = 1.5 * 2^12): the product is off by
// 2^-46 at most, and a quotient that is not a half differs from every half by at least 2^-34 (x and a have 24-bit
// significands, and near a half at most 8 binary places lie between them), so a true tie becomes exact and nothing else
// moves across one.  The second rounds to the whole number and leaves it in the low bits.
__device__ __forceinline__ unsigned int8_code(float x, double inv) {
    const double t = __builtin_fma((double)x, inv, 6144.0) + (6755399441055744.0 - 6144.0);
    return (unsigned)__builtin_bit_cast(unsigned long long, t);
}

// 16 bytes of a row from byte k on, zeros behind the row's end; any alignment, never reads outside the row.
__device__ __forceinline__ i32x4 int8_chunk(const int8_t* row, int k, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) __builtin_memcpy(&v, row + k, 16);
    else if (K >= 16) {                                      // the row's last 16 bytes, moved down
        unsigned __int128 u = 0;
        if (k < K) {
            __builtin_memcpy(&u, row + K - 16, 16);
            u >>= 8 * (16 - (K - k));
        }
        __builtin_memcpy(&v, &u, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (k + j < K) v[j >> 2] |= (int)(unsigned char)row[k + j] << (8 * (j & 3));
    }
    return v;
}

// Four elements of a row from element k on (k % 4 == 0), zeros behind the row's end.  `wide`: rows start at multiples of
// four elements' bytes.
__device__ __forceinline__ f32x4 int8_load4(const float* x, int k, int K, bool wide) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (wide && k + 4 <= K) return *reinterpret_cast<const f32x4*>(x + k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (k + j < K) v[j] = x[k + j];
    return v;
}
__device__ __forceinline__ f32x4 int8_load4(const unsigned short* x, int k, int K, bool wide) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (wide && k + 4 <= K) {
        const uint2 u = *reinterpret_cast<const uint2*>(x + k);
        v[0] = __builtin_bit_cast(float, u.x << 16); v[1] = __builtin_bit_cast(float, u.x & 0xFFFF0000u);
        v[2] = __builtin_bit_cast(float, u.y << 16); v[3] = __builtin_bit_cast(float, u.y & 0xFFFF0000u);
        return v;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (k + j < K) v[j] = bf16_bits_to_f32(x[k + j]);
    return v;
}

// |x| as bit patterns orders like the values and puts infinities and NaN on top.
__device__ __forceinline__ unsigned int8_top(unsigned a, f32x4 v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float f = v[j];                   // (a bit cast of the vector's element itself reads element 0)
        const unsigned bits = __builtin_bit_cast(unsigned, f) & 0x7FFFFFFFu;
        a = bits > a ? bits : a;
    }
    return a;
}
__device__ __forceinline__ unsigned wave_top(unsigned a) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned other = __shfl_xor(a, o, 64);
        a = other > a ? other : a;
    }
    return a;
}
// Factor of the codes and scale of a row whose largest |x| has the bit pattern `top`.
__device__ __forceinline__ double int8_inv(unsigned top, float& scale) {
    const bool finite = top < 0x7F800000u;
    const double amax = (double)__builtin_bit_cast(float, top);
    scale = finite ? (float)(amax / 127.0) : __builtin_nanf("");
    return finite && top > 0 ? 127.0 / amax : 0.0;
}
__device__ __forceinline__ unsigned int8_codes4(f32x4 v, double inv) {
    unsigned c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = int8_code(v[j], inv);
    const unsigned lo = __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000C0Cu);
    return inv > 0.0 ? lo | hi : 0u;
}

// One wave per row; rows of up to kInt8Held features are read once and stay in registers between the maximum and the codes.
constexpr int kInt8Held = 4096;
template <typename T>
__device__ __forceinline__ void int8_quantize_row(const T* x, int K, bool wide, int8_t* c, int ldc, float* scale) {
    const int lane = threadIdx.x & 63;
    f32x4 v[kInt8Held / 256];
    unsigned a = 0;
    if (K <= kInt8Held) {
#pragma unroll
        for (int i = 0; i < kInt8Held / 256; ++i)
            if (i * 256 < K) { v[i] = int8_load4(x, i * 256 + lane * 4, K, wide); }
#pragma unroll
        for (int i = 0; i < kInt8Held / 256; ++i)
            if (i * 256 < K) a = int8_top(a, v[i]);
    } else {
#pragma unroll 4
        for (int k = lane * 4; k < K; k += 256) a = int8_top(a, int8_load4(x, k, K, wide));
    }
    float s;
    const double inv = int8_inv(wave_top(a), s);
    if (K <= kInt8Held) {
#pragma unroll
        for (int i = 0; i < kInt8Held / 256; ++i) {
            const int k = i * 256 + lane * 4;
            if (i * 256 < K && k < ldc) *reinterpret_cast<unsigned*>(c + k) = int8_codes4(v[i], inv);
        }
        for (int k = (K + 255) / 256 * 256 + lane * 4; k < ldc; k += 256) *reinterpret_cast<unsigned*>(c + k) = 0;
    } else {
#pragma unroll 4
        for (int k = lane * 4; k < ldc; k += 256) *reinterpret_cast<unsigned*>(c + k) = int8_codes4(int8_load4(x, k, K, wide), inv);
    }
    if (lane == 0) *scale = s;
}

// Rows 0 .. M-1 of every matrix of the batch are quantised; T = int8_t: copied to rows that start at multiples of 16 bytes.
// The N rows behind them (if any) are weights, copied alike.  One wave per row: the maximum needs no barrier, and a row's 16-byte
// loads are all under way at once.  Bound by memory: 4096 x 2560 fp32 (42 MB read, 10.5 written) 12.6 us, 4.2 TB/s -- four fifths of a
// copy's rate (median of traced launches over three sets of operands, as all times of kernels here; 12.0 over one).
template <typename T>
__global__ __launch_bounds__(64) void int8_prepare_kernel(Int8Prepare p, int64_t ldx, int64_t ldw, int M, int K, int64_t ldc) {
    const int bz = blockIdx.y;
    const bool weight = (int)blockIdx.x >= M;
    const int64_t m = weight ? (int)blockIdx.x - M : (int)blockIdx.x;
    if (weight || sizeof(T) == 1) {
        const int8_t* from = weight ? p.W[bz] + m * ldw : reinterpret_cast<const int8_t*>(p.x[bz]) + m * ldx;
        int8_t* to = (weight ? p.w_codes[bz] : p.codes[bz]) + m * ldc;
        for (int k = (int)threadIdx.x * 16; k < ldc; k += 1024) *reinterpret_cast<i32x4*>(to + k) = int8_chunk(from, k, K);
        return;
    }
    if constexpr (sizeof(T) != 1) {
        const T* x = reinterpret_cast<const T*>(p.x[bz]) + m * ldx;
        const bool wide = (reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T))) == 0;
        int8_quantize_row<T>(x, K, wide, p.codes[bz] + m * ldc, (int)ldc, p.scale[bz] + m);
    }
}

// Scaled in 64 bits: no intermediate leaves the range of 32 bits where the result does not (s is up to 2^121, the sum up to
// 2^31), at four 64-bit instructions per output, seven for 16 bits.  Stored with one rounding to the output's type: on its way
// to 16 bits through 32, a value next to the border of two 16-bit values would be rounded onto the border and then to the
// even side.
__device__ __forceinline__ double int8_scale(int acc, double s, double t, double b, int relu) {
    const double v = __builtin_fma((double)acc, s * t, b);
    return relu && v < 0.0 ? 0.0 : v;
}
__device__ __forceinline__ unsigned short int8_to_bf16(double v) { return __builtin_bit_cast(unsigned short, static_cast<__bf16>(v)); }
__device__ __forceinline__ void int8_store(float* y, double v) { *y = (float)v; }
__device__ __forceinline__ void int8_store(unsigned short* y, double v) { *y = int8_to_bf16(v); }
__device__ __forceinline__ void int8_store4(float* y, const double (&v)[4]) {
    *reinterpret_cast<f32x4*>(y) = f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
__device__ __forceinline__ void int8_store4(unsigned short* y, const double (&v)[4]) {
    uint2 o;
    o.x = int8_to_bf16(v[0]) | (unsigned)int8_to_bf16(v[1]) << 16;
    o.y = int8_to_bf16(v[2]) | (unsigned)int8_to_bf16(v[3]) << 16;
    *reinterpret_cast<uint2*>(y) = o;
}

// 16 elements of a row from element k on (k % 16 == 0), zeros behind the row's end.
template <typename T>
__device__ __forceinline__ void int8_load16(const T* x, int k, int K, bool wide, f32x4 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = int8_load4(x, k + 4 * j, K, wide);
}

// Few rows: a workgroup takes 16 output channels of up to 16 rows over the whole of k, cut among its eight waves, and adds
// the waves' sums in LDS; the rows are quantised by every workgroup for itself, so that the layer is one launch.  A wave
// reads weights and activations of its own share of k straight in the operand layout of the 16x16x64 instruction (lane l: 16
// consecutive k of row l % 16) and quantises in registers; all that the waves exchange before the products is the rows'
// maxima.  STEPS: blocks of 64 k per wave; K <= 512 STEPS.  Bound by latency (loads, maxima, codes, products, sums one after the
// other): 1 x 2560 -> 1024 fp32 6.9 us, 16 x 2048 -> 1024 bf16 9.2 us for 2.6 MB, where two launches took 26.  2048 features run
// the instance of up to 2560: a fifth of its loads and products there is for nothing.
template <int STEPS, typename T, typename Y>
__global__ __launch_bounds__(512) void int8_rows16_kernel(Int8Batch p, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy) {
    __shared__ unsigned tops[8][16];
    __shared__ float sc[16];
    __shared__ __align__(16) int red[8 * 256];
    const int bz = blockIdx.y, n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.z * 16;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int r = lane & 15, kl = 64 * wave + 16 * (lane >> 4);
    const int wr = n0 + r < N ? n0 + r : N - 1;
    const int8_t* w = p.W[bz] + (int64_t)wr * ldw;
    const T* x = reinterpret_cast<const T*>(p.x[bz]) + (int64_t)(m0 + r < M ? m0 + r : M - 1) * ldx;
    const bool wide = (reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T))) == 0;
    i32x4 wf[STEPS];
    f32x4 v[STEPS][4];
    unsigned a = 0;
    if (K % 16 == 0 && __all(wide)) {
        // whole pieces: a lane behind the row's end reads its last piece, and its weights are zeros
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int k = kl + 512 * i, at = k < K ? k : K - 16;
            __builtin_memcpy(&wf[i], w + at, 16);
            int8_load16(x, at, K, true, v[i]);
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (kl + 512 * i >= K) wf[i] = i32x4{0, 0, 0, 0};
        }
    } else {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            wf[i] = int8_chunk(w, kl + 512 * i, K);
            int8_load16(x, kl + 512 * i, K, wide, v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) a = int8_top(a, v[i][j]);
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
        const unsigned other = __shfl_xor(a, o, 64);
        a = other > a ? other : a;
    }
    if (lane < 16) tops[wave][lane] = a;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 8; ++g) a = tops[g][r] > a ? tops[g][r] : a;
    float s;
    const double inv = int8_inv(a, s);
    if (tid < 16) sc[tid] = s;
    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        i32x4 xf;
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[j] = (int)int8_codes4(v[i][j], inv);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], xf, acc, 0, 0, 0);
    }
    *reinterpret_cast<i32x4*>(red + wave * 256 + lane * 4) = acc;
    __syncthreads();
    if (tid >= 256) return;
    const int m = tid >> 4, n = tid & 15;
    if (m0 + m >= M || n0 + n >= N) return;
    int sum = 0;
#pragma unroll
    for (int g = 0; g < 8; ++g) sum += red[g * 256 + (m + 16 * (n >> 2)) * 4 + (n & 3)];
    int8_store(reinterpret_cast<Y*>(p.y[bz]) + (int64_t)(m0 + m) * ldy + n0 + n,
               int8_scale(sum, sc[m], p.ws[bz][n0 + n], p.b[bz] ? p.b[bz][n0 + n] : 0.f, relu));
}
template <typename T, typename Y>
static int int8_rows16(const Int8Batch& p, int n_batch, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy, hipStream_t st) {
    const dim3 grid((unsigned)((N + 15) / 16), (unsigned)n_batch, (unsigned)((M + 15) / 16)), blk(512);
    if (K <= 1024) hipLaunchKernelGGL((int8_rows16_kernel<2, T, Y>), grid, blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
    else if (K <= 2560) hipLaunchKernelGGL((int8_rows16_kernel<5, T, Y>), grid, blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
    else hipLaunchKernelGGL((int8_rows16_kernel<8, T, Y>), grid, blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
    return check_launch("linear_int8");
}

// Rows quantised before, few tiles: 16 channels x 16 RM rows per workgroup over the whole of k, split among eight waves; both
// operands go from memory (rows: L2) straight into operand registers.  Any strides and alignments.  Bound by the latency of its
// two or three steps of k: 333 x 1037 -> 501 7.6 us (11.4 while a row's last bytes were read one by one).
template <int RM, typename Y>
__global__ __launch_bounds__(512) void int8_split_kernel(Int8Batch p, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy) {
    __shared__ __align__(16) int red[8 * RM * 256];
    const int bz = blockIdx.z, n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * RM;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int wr = n0 + (lane & 15) < N ? n0 + (lane & 15) : N - 1;
    const int8_t* w = p.W[bz] + (int64_t)wr * ldw;
    const int8_t* x[RM];
    i32x4 acc[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int m = m0 + 16 * i + (lane & 15) < M ? m0 + 16 * i + (lane & 15) : M - 1;
        x[i] = reinterpret_cast<const int8_t*>(p.x[bz]) + (int64_t)m * ldx;
        acc[i] = i32x4{0, 0, 0, 0};
    }
#pragma unroll 4
    for (int k = 64 * wave + 16 * (lane >> 4); k - 16 * (lane >> 4) < K; k += 512) {
        const i32x4 wf = int8_chunk(w, k, K);
#pragma unroll
        for (int i = 0; i < RM; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, int8_chunk(x[i], k, K), acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) *reinterpret_cast<i32x4*>(red + (wave * RM + i) * 256 + lane * 4) = acc[i];
    __syncthreads();
    for (int o = tid; o < RM * 256; o += 512) {
        const int i = o >> 8, m = (o >> 4) & 15, n = o & 15;
        const int row = m0 + 16 * i + m;
        if (row >= M || n0 + n >= N) continue;
        int sum = 0;
#pragma unroll
        for (int g = 0; g < 8; ++g) sum += red[(g * RM + i) * 256 + (m + 16 * (n >> 2)) * 4 + (n & 3)];
        int8_store(reinterpret_cast<Y*>(p.y[bz]) + (int64_t)row * ldy + n0 + n,
                   int8_scale(sum, p.xs[bz][row], p.ws[bz][n0 + n], p.b[bz] ? p.b[bz][n0 + n] : 0.f, relu));
    }
}

__device__ __forceinline__ void int8_glds16(const void* gsrc_lane, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc_lane,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

// Waits until at most VM vector memory operations are under way and every LDS read has arrived.  (The builtin: the compiler
// counts on from it, where it takes inline assembly for nothing and waits for everything again.)
template <int VM>
__device__ __forceinline__ void int8_wait() {
    static_assert(VM >= 0 && VM < 64, "six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}

__device__ __attribute__((aligned(16))) const int int8_zeros[4] = {0, 0, 0, 0};

// Tiles of BM x BN outputs, WVM x WVN waves, k in stages of BK bytes through a ring of R buffers in LDS: the copies of R
// stages go straight from memory into LDS while the products of the stage in front of them run, one barrier a stage.  Rows
// of both operands start at multiples of 16 bytes and K is a multiple of 16 (zeros behind the features); stages behind K
// are copied from a line of zeros, so that every stage is the same number of loads.
// LDS serves 16 lanes of a 16-byte read at a time from 64 banks (256 bytes): with rows of 128 (64) bytes those are 16 rows, of
// which every second (fourth) falls on the same banks.  16-byte piece c of a row lies at place c ^ (row / 2 % 8) (c ^ (row / 4
// % 4)), which spreads them over all banks; the copies stay linear in LDS, each lane picks its source.
// 256 x 256: 8192 x 4096 x 4096 149 us, 1.85 POP/s; the matrix pipes are busy 54 % of the cycles (131 k of 243 k per SIMD, at
// 1.85 GHz), 29 % of the waves' cycles are waits, in 43 % an instruction is held back.  128 x 128: 4096 x 2560 -> 1024 19.4 us; matrix
// pipes 30 %, waits 45 %: one tile a CU, so that neither the ring's filling and emptying nor the 168 MB from L2 into LDS
// (8.7 TB/s) run behind another tile; the two were not measured apart.  64 x 64: six of 512 x 1024 -> 512 9.8 us.  No fence keeps
// the fragments' reads in front of the products (170 us with one: the scheduler interleaves them better).
template <int BM, int BN, int WVM, int WVN, int BK, int R, typename Y>
__global__ __launch_bounds__(WVM * WVN * 64) void int8_tile_kernel(Int8Batch p, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy) {
    constexpr int WV = WVM * WVN, TM = BM / WVM / 32, TN = BN / WVN / 32;
    constexpr int PR = BK / 16, RU = 64 / PR, LOG = BK == 128 ? 1 : 2;      // pieces of a row, rows of a 1-KiB unit
    constexpr int UA = BM / RU, UB = BN / RU, PER = (UA + UB) / WV;
    constexpr int STAGE = (BM + BN) * BK;
    static_assert((BK == 64 || BK == 128) && TM >= 1 && TN >= 1 && UA % WV == 0 && UB % WV == 0, "tile");
    extern __shared__ __align__(16) int8_t smem[];
    __shared__ __align__(16) double tb[2 * BN];              // scales and biases of the tile's channels
    const int bz = blockIdx.y;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int nx = (N + BN - 1) / BN, ny = (M + BM - 1) / BM;
    int tx, ty;
    xcd_tile((int)blockIdx.x, nx, ny, tx, ty);
    const int m0 = ty * BM, n0 = tx * BN;
    for (int n = tid; n < BN; n += WV * 64) {
        const int at = n0 + n < N ? n0 + n : N - 1;
        tb[n] = p.ws[bz][at];
        tb[BN + n] = p.b[bz] ? p.b[bz][at] : 0.;
    }

    const int8_t* src[PER];
    static_assert(WV * RU % (PR << LOG) == 0, "a wave's units are alike");
    const int urow = lane / PR, piece = (lane % PR) ^ (((wave * RU + urow) >> LOG) & (PR - 1));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int u = (i < UA / WV ? i : i - UA / WV) * WV + wave;
        const int row = (i < UA / WV ? m0 : n0) + u * RU + urow;
        src[i] = i < UA / WV ? reinterpret_cast<const int8_t*>(p.x[bz]) + (int64_t)(row < M ? row : M - 1) * ldx + piece * 16
                             : p.W[bz] + (int64_t)(row < N ? row : N - 1) * ldw + piece * 16;
    }
    uintptr_t zeros = reinterpret_cast<uintptr_t>(int8_zeros);
    asm("" : "+s"(zeros));                                   // (known to be another object it becomes a load of its own, with half of the lanes)
    int put = 0, k_put = 0;
    auto issue = [&]() {
        int8_t* dst = smem + put * STAGE + wave * 1024;
        const bool in = k_put + piece * 16 < K;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uintptr_t at = in ? reinterpret_cast<uintptr_t>(src[i] + k_put) : zeros;
            int8_glds16(reinterpret_cast<const void*>(at), dst + (i < UA / WV ? i : i - UA / WV) * WV * 1024 + (i < UA / WV ? 0 : BM * BK));
        }
        put = put + 1 == R ? 0 : put + 1;
        k_put += BK;
    };

    const int wm = (wave / WVN) * (BM / WVM), wn = (wave % WVN) * (BN / WVN);
    const int r = lane & 31, h = lane >> 5, f = (r >> LOG) & (PR - 1);
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    // The fragments of a step of 32 k are read during the products of the step in front of it, also across stages: the wait
    // for the next stage and its barrier lie in front of a stage's last products.  At that barrier everyone holds the last
    // fragments of this stage in registers, so that its buffer can be filled again.
    constexpr int KK = BK / 32;
    static_assert(KK % 2 == 0, "two sets of fragments in turns");
    i32x4 fa[2][TM], fb[2][TN];
    int get = 0;
    auto read = [&](int kk, int set) {
        const int8_t* sa = smem + get * STAGE + (wm + r) * BK;
        const int8_t* sb = smem + get * STAGE + BM * BK + (wn + r) * BK;
        const int at = ((2 * kk + h) ^ f) << 4;
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[set][i] = *reinterpret_cast<const i32x4*>(sa + i * 32 * BK + at);
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[set][j] = *reinterpret_cast<const i32x4*>(sb + j * 32 * BK + at);
    };
    const int stages = (K + BK - 1) / BK;
#pragma unroll
    for (int i = 0; i < R; ++i) issue();
    int8_wait<(R - 1) * PER>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0);
    for (int st = 0; st < stages; ++st) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            if (kk + 1 < KK) read(kk + 1, (kk + 1) & 1);
            else {
                // own copies of the next stage have landed (R - 2 younger stages are under way), own reads of this one are done
                int8_wait<(R - 2) * PER>();
                __builtin_amdgcn_s_barrier();                // so have everyone's
                asm volatile("" ::: "memory");
                get = get + 1 == R ? 0 : get + 1;
                read(0, 0);
                issue();
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[kk & 1][j], fa[kk & 1][i], acc[i][j], 0, 0, 0);
        }
    }
    int8_wait<0>();                                          // (the copies behind the last stage)
    __syncthreads();                                         // nobody reads the ring any more
    // A lane holds 4 x 4 channels of one row: 32 rows at a time they go through LDS, so that the stores are whole lines of
    // consecutive channels (stored as they lie, 64 bytes of two rows per instruction, the outputs cost 50 of 190 us at 8192 x
    // 4096 x 4096 in 16 bits and 10 of 30 us at 4096 x 2560 x 1024).
    constexpr int COLS = TN * 32, RS = COLS * (int)sizeof(Y) + 16, PV = 16 / (int)sizeof(Y), LPR = COLS / PV;
    static_assert(WV * 32 * RS <= R * STAGE, "the outputs fit the ring");
    int8_t* slab = smem + wave * 32 * RS;
    Y* y = reinterpret_cast<Y*>(p.y[bz]);
    const int nw = n0 + wn;
    const bool vec = nw + COLS <= N && ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * (int64_t)sizeof(Y))) % 16) == 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int mw = m0 + wm + 32 * i, m = mw + r;
        const double s = (double)p.xs[bz][m < M ? m : M - 1];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = 32 * j + 8 * q + 4 * h;
                const double* t = tb + wn + n;
                double v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = int8_scale(acc[i][j][4 * q + e], s, t[e], t[BN + e], relu);
                int8_store4(reinterpret_cast<Y*>(slab + r * RS) + n, v);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (vec) {
#pragma unroll
            for (int c = 0; c < 32 * LPR / 64; ++c) {
                const int row = (c * 64 + lane) / LPR, col = (c * 64 + lane) % LPR * PV;
                const u32x4 v = *reinterpret_cast<const u32x4*>(slab + row * RS + col * (int)sizeof(Y));
                if (mw + row < M) *reinterpret_cast<u32x4*>(y + (int64_t)(mw + row) * ldy + nw + col) = v;
            }
        } else {
            for (int c = lane; c < 32 * COLS; c += 64) {
                const int row = c / COLS, col = c % COLS;
                if (mw + row < M && nw + col < N) y[(int64_t)(mw + row) * ldy + nw + col] = *(reinterpret_cast<const Y*>(slab + row * RS) + col);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int WVM, int WVN, int BK, int R, typename Y>
static int int8_tiles(const Int8Batch& p, int n_batch, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy, hipStream_t st) {
    auto kern = int8_tile_kernel<BM, BN, WVM, WVN, BK, R, Y>;
    const size_t lds = (size_t)R * (BM + BN) * BK;
    if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), lds, "linear_int8")) return rc;
    const int64_t tiles = (int64_t)((M + BM - 1) / BM) * ((N + BN - 1) / BN);
    if (!launch_fits(tiles, WVM * WVN * 64)) return fail(DVQ_EINVAL, "linear_int8: M x N too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (unsigned)n_batch), dim3(WVM * WVN * 64), lds, st, p, ldx, ldw, M, K, N, relu, ldy);
    return check_launch("linear_int8");
}

static inline int64_t tile_count(int M, int N, int b, int n_batch) { return (int64_t)((M + b - 1) / b) * ((N + b - 1) / b) * n_batch; }

// The product of rows that are codes already (p.x).  `tiles`: rows of both operands start at multiples of 16 bytes, K % 16 == 0.
template <typename Y>
static int int8_product(const Int8Batch& p, int n_batch, int64_t ldx, int64_t ldw, int M, int K, int N, int relu, int64_t ldy, bool tiles,
                        hipStream_t st) {
    if (!tiles) {
        const dim3 blk(512);
        const unsigned gx = (unsigned)((N + 15) / 16);
        if (M <= 16) hipLaunchKernelGGL((int8_split_kernel<1, Y>), dim3(gx, 1, n_batch), blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
        else if (M <= 32) hipLaunchKernelGGL((int8_split_kernel<2, Y>), dim3(gx, 1, n_batch), blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
        else hipLaunchKernelGGL((int8_split_kernel<4, Y>), dim3(gx, (M + 63) / 64, n_batch), blk, 0, st, p, ldx, ldw, M, K, N, relu, ldy);
        return check_launch("linear_int8");
    }
    // A larger tile reads its operands less often, a smaller one leaves fewer CUs idle.  Tiles of 256 / 128 / 64, us: 4096 x
    // 2560 x 1024 (160 / 640 / 2560 tiles) 25 / 31 / 38, 2048 x 4096 x 4096 (128 / 512 / 2048) 58 / 60 / 85, 2048 x 2560 x 1024
    // (80 / 320 / 1280) 24 / 20 / 20, 1024 x 2560 x 1024 (40 / 160 / 640) 23 / 12 / 14, 1024 x 2048 x 2048 (32 / 128 / 512) 31 /
    // 15 / 13: the smallest as long as its tiles fit the chip in one round, two to a CU.
    if (tile_count(M, N, 256, n_batch) >= 128) return int8_tiles<256, 256, 2, 4, 64, 4, Y>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st);
    if (tile_count(M, N, 64, n_batch) > 512) return int8_tiles<128, 128, 2, 4, 128, 4, Y>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st);
    return int8_tiles<64, 64, 2, 2, 128, 4, Y>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st);
}

static bool aligned16(const void* const* ptrs, int n, int64_t ld) {
    if (ld % 16) return false;
    for (int i = 0; i < n; ++i)
        if (reinterpret_cast<uintptr_t>(ptrs[i]) % 16) return false;
    return true;
}

static inline int64_t int8_ld(int K) { return (K + 63) / 64 * 64; }
static inline int64_t int8_each(int rows, int K) { return rows * int8_ld(K) + (rows * (int64_t)4 + 15) / 16 * 16; }

}  // namespace dvq

using namespace dvq;

// Rows of a float matrix quantised by each workgroup for itself: no workspace, one launch.
static bool int8_one_launch(int n_batch, int M, int K, int N) {
    return K <= kInt8Held && (M <= 16 || tile_count(M, N, 16, n_batch) <= (K <= 1024 ? kInt8OneLaunchShort : kInt8OneLaunch));
}

extern "C" size_t dvq_linear_int8_workspace_bytes(int n_batch, int M, int K, int N) {
    if (n_batch < 1 || M < 1 || K < 1 || N < 1) return 0;
    return (size_t)n_batch * (size_t)(int8_each(M, K) + (int64_t)N * int8_ld(K));
}

extern "C" int dvq_int8_quantize_rows(const void* x, int dtype, int64_t ldx, int M, int K, void* codes, int64_t ldc, float* scale, void* stream) {
    if (dtype != DVQ_F32 && dtype != DVQ_BF16) return fail(DVQ_EINVAL, "int8_quantize_rows: dtype must be DVQ_F32 or DVQ_BF16");
    if (M < 0 || K < 1 || K >= (1 << 17) || ldx < 0 || ldc < K || (ldc % 16) != 0 || ldc > (1 << 30))
        return fail(DVQ_EINVAL, "int8_quantize_rows: M >= 0, 1 <= K < 2^17, ldc >= K a multiple of 16 (got M = %d, K = %d, ldc = %lld)", M, K, (long long)ldc);
    if (!launch_fits(M, 64)) return fail(DVQ_EINVAL, "int8_quantize_rows: M must stay below 2^26");
    if (M == 0) return DVQ_OK;
    if (!x || !codes || !scale || reinterpret_cast<uintptr_t>(codes) % 16) return fail(DVQ_EINVAL, "int8_quantize_rows: null or unaligned pointer");
    Int8Prepare p = {};
    p.x[0] = x; p.codes[0] = reinterpret_cast<int8_t*>(codes); p.scale[0] = scale;
    if (dtype == DVQ_F32) hipLaunchKernelGGL(int8_prepare_kernel<float>, dim3((unsigned)M, 1), dim3(64), 0, as_stream(stream), p, ldx, 0, M, K, ldc);
    else hipLaunchKernelGGL(int8_prepare_kernel<unsigned short>, dim3((unsigned)M, 1), dim3(64), 0, as_stream(stream), p, ldx, 0, M, K, ldc);
    return check_launch("int8_quantize_rows");
}

extern "C" int dvq_linear_int8_batched(int n_batch, const void* const* x, int x_dtype, const float* const* xs, int64_t ldx, const void* const* W,
                               const float* const* ws, int64_t ldw, const float* const* b, int M, int K, int N, int relu,
                               void* const* y, int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    if (n_batch < 1 || n_batch > kInt8MaxBatch) return fail(DVQ_EINVAL, "linear_int8: 1..%d products per launch", kInt8MaxBatch);
    if (x_dtype != DVQ_F32 && x_dtype != DVQ_BF16 && x_dtype != DVQ_I8) return fail(DVQ_EINVAL, "linear_int8: x_dtype must be DVQ_F32, DVQ_BF16 or DVQ_I8");
    if (y_dtype != DVQ_F32 && y_dtype != DVQ_BF16) return fail(DVQ_EINVAL, "linear_int8: y_dtype must be DVQ_F32 or DVQ_BF16");
    if (M < 0 || N < 1 || K < 1 || K >= (1 << 17)) return fail(DVQ_EINVAL, "linear_int8: M >= 0, N >= 1, 1 <= K < 2^17 (got M = %d, N = %d, K = %d)", M, N, K);
    if (ldx < 0 || ldw < 0 || ldy < N) return fail(DVQ_EINVAL, "linear_int8: bad row stride");
    if (M > (1 << 30) || N > (1 << 30)) return fail(DVQ_EINVAL, "linear_int8: M and N up to 2^30");
    if (M == 0) return DVQ_OK;
    const bool codes = x_dtype == DVQ_I8;
    if (!x || !W || !ws || !y || (codes && !xs)) return fail(DVQ_EINVAL, "linear_int8: null pointer");
    for (int i = 0; i < n_batch; ++i)
        if (!x[i] || !W[i] || !ws[i] || !y[i] || (codes && !xs[i])) return fail(DVQ_EINVAL, "linear_int8: null pointer");
    Int8Batch p = {};
    for (int i = 0; i < n_batch; ++i) {
        p.x[i] = x[i]; p.xs[i] = codes ? xs[i] : nullptr;
        p.W[i] = reinterpret_cast<const int8_t*>(W[i]); p.ws[i] = ws[i];
        p.b[i] = b ? b[i] : nullptr;
        p.y[i] = y[i];
    }
    hipStream_t st = as_stream(stream);
    const bool f32 = y_dtype == DVQ_F32;
    if (!codes && int8_one_launch(n_batch, M, K, N)) {
        if (!launch_fits((N + 15) / 16, 512)) return fail(DVQ_EINVAL, "linear_int8: N too large");
        typedef unsigned short u16;
        if (x_dtype == DVQ_F32)
            return f32 ? int8_rows16<float, float>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st)
                       : int8_rows16<float, u16>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st);
        return f32 ? int8_rows16<u16, float>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st)
                   : int8_rows16<u16, u16>(p, n_batch, ldx, ldw, M, K, N, relu, ldy, st);
    }
    // What the tiles cannot read in place -- features to quantise, rows that do not start at multiples of 16 bytes -- is
    // laid out in the workspace by one launch.
    const bool tiles = tile_count(M, N, 64, n_batch) > kInt8SplitTo;
    const bool wide = K % 16 == 0;
    const bool copy_w = tiles && !(wide && aligned16(W, n_batch, ldw));
    const bool copy_x = !codes || (tiles && !(wide && aligned16(x, n_batch, ldx)));
    int Kt = K;
    if (copy_w || copy_x) {
        const size_t need = dvq_linear_int8_workspace_bytes(n_batch, M, K, N);
        if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
            return fail(DVQ_EINVAL, "linear_int8: needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : 0);
        Int8Prepare q = {};
        int8_t* base = reinterpret_cast<int8_t*>(workspace);
        const int64_t ldc = int8_ld(K);
        for (int i = 0; i < n_batch; ++i) {
            q.x[i] = p.x[i]; q.W[i] = p.W[i];
            q.codes[i] = base; q.scale[i] = reinterpret_cast<float*>(base + M * ldc);
            base += int8_each(M, K);
            q.w_codes[i] = base;
            base += N * ldc;
            if (copy_x) { p.x[i] = q.codes[i]; if (!codes) p.xs[i] = q.scale[i]; }
            if (copy_w) p.W[i] = q.w_codes[i];
        }
        const int rows = copy_x ? M : 0;
        if (!launch_fits((int64_t)rows + (copy_w ? N : 0), 64)) return fail(DVQ_EINVAL, "linear_int8: too many rows to quantise or lay out (2^26)");
        const dim3 grid((unsigned)(rows + (copy_w ? N : 0)), (unsigned)n_batch);
        if (x_dtype == DVQ_F32) hipLaunchKernelGGL(int8_prepare_kernel<float>, grid, dim3(64), 0, st, q, ldx, ldw, rows, K, ldc);
        else if (x_dtype == DVQ_BF16) hipLaunchKernelGGL(int8_prepare_kernel<unsigned short>, grid, dim3(64), 0, st, q, ldx, ldw, rows, K, ldc);
        else hipLaunchKernelGGL(int8_prepare_kernel<int8_t>, grid, dim3(64), 0, st, q, ldx, ldw, rows, K, ldc);
        if (int rc = check_launch("linear_int8")) return rc;
        if (copy_x) ldx = ldc;
        if (copy_w) ldw = ldc;
        if (tiles) Kt = (K + 15) / 16 * 16;             // (zeros behind the features)
    }
    return f32 ? int8_product<float>(p, n_batch, ldx, ldw, M, Kt, N, relu, ldy, tiles, st)
               : int8_product<unsigned short>(p, n_batch, ldx, ldw, M, Kt, N, relu, ldy, tiles, st);
}

extern "C" int dvq_linear_int8(const void* x, int x_dtype, const float* xs, int64_t ldx, const void* W, const float* ws, int64_t ldw, const float* b,
                               int M, int K, int N, int relu, void* y, int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    return dvq_linear_int8_batched(1, &x, x_dtype, &xs, ldx, &W, &ws, ldw, &b, M, K, N, relu, &y, y_dtype, ldy, workspace, workspace_bytes, stream);
}
