// Products with a matrix of 128 x 128 blocks in 8-bit floating point, one power-of-two scale per block:
// y = A x, dx = A^T dy, the gradient of the stored blocks, and vectors to 8 bits and back.

#include "internal.h"
#include "device_utils.h"

#include <algorithm>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

namespace spmv {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned piece __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes of a vector, wherever they lie
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kB = 128;                       // block edge, and length of a vector's group
constexpr int kBlockBytes = kB * kB;

// Place of (row, column) inside a block's 16 KB: 16 x 16 subtiles of 256 bytes, so that one 16-byte load per lane
// is a contiguous 1 KB piece of a matrix-instruction operand (16 rows of one strip, 64 columns).  A strip holds the rows
// {4 i + s} of one 64-row half (s = strip in the half, i = 0..15): with the rows along the lanes of a result, 4 strips'
// results in a lane are 4 consecutive rows of y, and those of 16 lanes 64.
__host__ __device__ __forceinline__ int block8_offset(int row, int col)
{
    const int strip = (row >> 6) * 4 + (row & 3), i = (row >> 2) & 15;
    return ((strip * 8 + (col >> 4)) * 16 + i) * 16 + (col & 15);
}

__device__ __forceinline__ float scale_value(int b) { return __int_as_float(b << 23); }      // 2^(b-127)
// 2^(b-128), b >= 1, for the scaled conversions alone: they read the exponent's byte, and 0 there stands for 2^-127
__device__ __forceinline__ float scale_half(int b) { return __int_as_float((b - 1) << 23); }

// scale byte of a group whose largest finite magnitude is `amax`: the least e >= -126 with amax <= 448 * 2^e =
// 1.75 * 2^(e+8), from the bits -- adding 0x1fffff to a float carries into its exponent where the mantissa is above 1.75
__device__ __forceinline__ int scale_byte(float amax)
{
    if (amax == 0.0f) return 127;
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;      // exponent byte of the scale
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ void unpack4(unsigned w, float scale, _Float16 *out)      // exact where fp16 holds the results
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
    const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    out[0] = lo[0]; out[1] = lo[1]; out[2] = hi[0]; out[3] = hi[1];
}
// Four e4m3 bytes times a power of two -> four bf16.  The products widen by half the scale (scale_half) and double their
// sums: the largest fp32 numbers round to 256 * 2^120, which bf16 has no number for, but half of it.  Exact for scale
// bytes 4 to 247; below, where half a value can lie under bf16's smallest step, off by at most 2^-134 (2^-133 of the value).
__device__ __forceinline__ void unpack4(unsigned w, float scale, __bf16 *out)
{
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
    out[0] = lo[0]; out[1] = lo[1]; out[2] = hi[0]; out[3] = hi[1];
}

template <int V> using ic = std::integral_constant<int, V>;

template <int DT> struct elem;
template <> struct elem<SPMV_HIP_F32> { typedef float type; };
template <> struct elem<SPMV_HIP_BF16> { typedef __bf16 type; };
template <> struct elem<SPMV_HIP_F16> { typedef _Float16 type; };

static size_t elem_size(int dtype) { return dtype == SPMV_HIP_F32 ? 4 : dtype == SPMV_HIP_E4M3 ? 1 : 2; }
static bool wide_dtype(int dtype) { return dtype == SPMV_HIP_F32 || dtype == SPMV_HIP_BF16 || dtype == SPMV_HIP_F16; }

// calls f with the element type of `dtype`
template <typename F> static void with_elem(int dtype, F f)
{
    if (dtype == SPMV_HIP_F32) f(float());
    else if (dtype == SPMV_HIP_BF16) f(__bf16());
    else f(_Float16());
}

// K entries of a vector as they lie in memory (any alignment), zero from `left` on
template <typename T, int K> struct Raw {
    T v[K];
    __device__ __forceinline__ void load(const T *p, int left)
    {
        if (left >= K) __builtin_memcpy(v, p, sizeof v);
        else
#pragma unroll
            for (int k = 0; k < K; k++) v[k] = k < left ? p[k] : (T)0.0f;
    }
    // the largest magnitude's bits, of numbers that are not finite too
    __device__ __forceinline__ unsigned top() const
    {
        unsigned m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < K; k++) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
            return m;
        } else {
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            u16x2 w[K / 2], t = {0, 0};
            __builtin_memcpy(w, v, sizeof v);
#pragma unroll
            for (int k = 0; k < K / 2; k++) t = __builtin_elementwise_max(t, (u16x2)(w[k] & (unsigned short)0x7fff));
            return max((unsigned)t[0], (unsigned)t[1]);
        }
    }
    // K / 4 words of e4m3 of v / scale, scale a power of two; infinities and NaN give NaN
    __device__ __forceinline__ void pack(float scale, unsigned *w) const
    {
        typedef short i16x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int k = 0; k < K; k += 4) {
            i16x2 o = {0, 0};
            if constexpr (std::is_same<T, float>::value) {
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, v[k], v[k + 1], scale, false);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, v[k + 2], v[k + 3], scale, true);
            } else if constexpr (std::is_same<T, __bf16>::value) {
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, bf16x2{v[k], v[k + 1]}, scale, false);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, bf16x2{v[k + 2], v[k + 3]}, scale, true);
            } else {
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, f16x2{v[k], v[k + 1]}, scale, false);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, f16x2{v[k + 2], v[k + 3]}, scale, true);
            }
            __builtin_memcpy(&w[k / 4], &o, 4);
        }
    }
};

// the largest finite magnitude of a lane's entries
template <typename T, int K> __device__ __forceinline__ float finite_top(const Raw<T, K> &r)
{
    constexpr unsigned inf = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
    unsigned m = r.top();
    if (m >= inf) {                                          // rare: leave out what is not finite
        m = 0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            Raw<T, 2> one{{r.v[k], (T)0.0f}};
            const unsigned t = one.top();
            m = t < inf ? max(m, t) : m;
        }
    }
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    else {
        const unsigned short h = (unsigned short)m;
        T v;
        __builtin_memcpy(&v, &h, 2);
        return (float)v;
    }
}

// ---- to 8 bits and back ---------------------------------------------------------------------------------------

// Bound by memory.  A wave takes 4 neighbouring groups of R vectors, 16 lanes a group, a lane one 16-byte piece (of fp32 two, 64
// entries apart): whole lines at every load and store.  Neighbouring workgroups take neighbouring columns.  16384 x 8192 of
// bf16: to 8 bits 69 us (5.8 TB/s; 100 us with a wave on 16 vectors and neighbouring workgroups on neighbouring vectors),
// back 57 us (117 us).
constexpr int kQuantGroups = 4, kQuantWaves = kBlock / kWave;

// The scale bytes meet in LDS, because those of one group lie vector by vector.
template <typename T, int R>
__global__ __launch_bounds__(kBlock) void quantize8_kernel(int n, int groups, int columns, const T *__restrict__ x, int64_t ldx,
                                                           uint8_t *__restrict__ x8, int64_t ldx8, uint8_t *__restrict__ scale,
                                                           int64_t lds)
{
    constexpr int K = 16 / sizeof(T), H = 8 / K, TV = R * kQuantWaves;
    __shared__ uint8_t bytes[kQuantGroups][TV];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, gq = lane >> 4;
    const unsigned gtiles = (groups + kQuantGroups - 1) / kQuantGroups;
    const int g0 = blockIdx.x % gtiles * kQuantGroups, c = (g0 + gq) * kB + (lane & 15) * K;
    const int64_t v0 = (int64_t)(blockIdx.x / gtiles) * TV;
    Raw<T, K> a[R][H];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int64_t v = v0 + wave * R + r;
#pragma unroll
        for (int h = 0; h < H; h++) a[r][h].load(x + (v < n ? v : n - 1) * ldx + c + h * 16 * K, columns - c - h * 16 * K);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int64_t v = v0 + wave * R + r;
        float top = finite_top(a[r][0]);
        if constexpr (H == 2) top = fmaxf(top, finite_top(a[r][1]));
#pragma unroll
        for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        const int b = scale_byte(top);
#pragma unroll
        for (int h = 0; h < H; h++) {
            unsigned w[2];
            a[r][h].pack(scale_value(b), w);
            if (v < n && g0 + gq < groups) __builtin_memcpy(__builtin_assume_aligned(x8 + v * ldx8 + c + h * 16 * K, K), w, K);
        }
        if ((lane & 15) == 0) bytes[gq][wave * R + r] = (uint8_t)b;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < kQuantGroups * TV; t += kBlock) {
        const int g = g0 + t / TV;
        const int64_t v = v0 + t % TV;
        if (g < groups && v < n) scale[(int64_t)g * lds + v] = bytes[t / TV][t % TV];
    }
}

template <typename T> __device__ __forceinline__ float largest_finite();
template <> __device__ __forceinline__ float largest_finite<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float largest_finite<__bf16>() { return 3.38953139e38f; }
template <> __device__ __forceinline__ float largest_finite<_Float16>() { return 65504.0f; }

// ONCE: the result goes past the caches
template <typename T, int R, bool ONCE>
__global__ __launch_bounds__(kBlock) void restore8_kernel(int n, int groups, int columns, const uint8_t *__restrict__ x8,
                                                          int64_t ldx8, const uint8_t *__restrict__ scale, int64_t lds,
                                                          T *__restrict__ x, int64_t ldx)
{
    constexpr int K = 16 / sizeof(T), H = 8 / K;             // entries of a 16-byte store; stores a vector takes
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const unsigned gtiles = (groups + kQuantGroups - 1) / kQuantGroups;
    const int g = blockIdx.x % gtiles * kQuantGroups + (lane >> 4), c0 = g * kB + (lane & 15) * K;
    if (g >= groups) return;
    const int64_t v0 = ((int64_t)(blockIdx.x / gtiles) * kQuantWaves + wave) * R;
    const float top = largest_finite<T>();
    unsigned w[R][2];
    int b[R];
#pragma unroll
    for (int u = 0; u < R; u++) {
        const int64_t v = v0 + u < n ? v0 + u : n - 1;
#pragma unroll
        for (int h = 0; h < H; h++) __builtin_memcpy(&w[u][h], __builtin_assume_aligned(x8 + v * ldx8 + c0 + h * 16 * K, K), K);
        b[u] = scale[(int64_t)g * lds + v];
    }
#pragma unroll
    for (int u = 0; u < R; u++) {
        if (v0 + u >= n) continue;
        const float s = scale_value(b[u]);
#pragma unroll
        for (int h = 0; h < H; h++) {
            T y[K];
#pragma unroll
            for (int k = 0; k < K; k++) {
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                const unsigned d = w[u][h + k / 4];
                const f32x2 p = (k & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8(d, true) : __builtin_amdgcn_cvt_pk_f32_fp8(d, false);
                const float f = p[k & 1] * s;
                y[k] = (T)(f > top ? top : f < -top ? -top : f);             // NaN stays
            }
            const int c = c0 + h * 16 * K;
            T *o = x + (v0 + u) * ldx + c;
            if (columns - c >= K) {
                piece v;
                __builtin_memcpy(&v, y, 16);
                if (ONCE) __builtin_nontemporal_store(v, (piece *)o);
                else *(piece *)o = v;
            } else
                for (int k = 0; k < K; k++)
                    if (k < columns - c) o[k] = y[k];
        }
    }
}

// One workgroup per block, its 16384 values in registers; the 8-bit block is put in the handle's order in LDS.
template <typename T>
__global__ __launch_bounds__(kBlock) void set_values_kernel(int rows, int columns, const int *__restrict__ block_row,
                                                            const int *__restrict__ block_col, const T *__restrict__ values,
                                                            uint8_t *__restrict__ val8, const int *__restrict__ bt_at,
                                                            int *__restrict__ scale8, int *__restrict__ bt_scale8)
{
    __shared__ float part[kBlock / kWave];
    __shared__ uint8_t out[kBlockBytes];
    const int64_t k = blockIdx.x;
    const int r0 = threadIdx.x >> 4, c = (threadIdx.x & 15) * 8;
    const int rows_in = rows - block_row[k] * kB, cols_in = columns - block_col[k] * kB;
    Raw<T, 8> a[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int r = j * 16 + r0;
        a[j].load(values + k * kBlockBytes + r * kB + c, r < rows_in ? cols_in - c : 0);
    }
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) top = fmaxf(top, finite_top(a[j]));
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = top;
    __syncthreads();
    const int b = scale_byte(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
#pragma unroll
    for (int j = 0; j < 8; j++) {
        unsigned w[2];
        a[j].pack(scale_value(b), w);
        *(uint2 *)&out[block8_offset(j * 16 + r0, c)] = uint2{w[0], w[1]};
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int at = (j * kBlock + threadIdx.x) * 16;
        *(u32x4 *)(val8 + k * kBlockBytes + at) = *(const u32x4 *)&out[at];
    }
    if (threadIdx.x == 0) { scale8[k] = b; bt_scale8[bt_at[k]] = b; }
}

__device__ __forceinline__ u32x4 load16(const void *p)       // any alignment
{
    u32x4 w;
    __builtin_memcpy(&w, p, 16);
    return w;
}

// row-major 8-bit blocks into the handle's order and back
__global__ __launch_bounds__(kBlock) void load8_kernel(int rows, int columns, const int *__restrict__ block_row,
                                                       const int *__restrict__ block_col, const uint8_t *__restrict__ values8,
                                                       const uint8_t *__restrict__ scale, uint8_t *__restrict__ val8,
                                                       const int *__restrict__ bt_at, int *__restrict__ scale8,
                                                       int *__restrict__ bt_scale8)
{
    const int64_t k = blockIdx.x;
    for (int p = threadIdx.x; p < kBlockBytes / 16; p += kBlock) {
        const int r = p >> 3, c = (p & 7) * 16;
        const int left = block_row[k] * kB + r < rows ? columns - block_col[k] * kB - c : 0;      // bytes inside the matrix
        u32x4 w = load16(values8 + k * kBlockBytes + p * 16);
#pragma unroll
        for (int d = 0; d < 4; d++) {
            const int keep = left - 4 * d;
            if (keep < 4) w[d] &= keep <= 0 ? 0u : (1u << (8 * keep)) - 1;
        }
        *(u32x4 *)(val8 + k * kBlockBytes + block8_offset(r, c)) = w;
    }
    if (threadIdx.x == 0) { scale8[k] = scale[k]; bt_scale8[bt_at[k]] = scale[k]; }
}

__global__ __launch_bounds__(kBlock) void store8_kernel(const uint8_t *__restrict__ val8, const int *__restrict__ scale8,
                                                        uint8_t *__restrict__ values8, uint8_t *__restrict__ scale)
{
    const int64_t k = blockIdx.x;
    for (int p = threadIdx.x; p < kBlockBytes / 16; p += kBlock) {
        const u32x4 w = *(const u32x4 *)(val8 + k * kBlockBytes + block8_offset(p >> 3, (p & 7) * 16));
        __builtin_memcpy(values8 + k * kBlockBytes + p * 16, &w, 16);
    }
    if (threadIdx.x == 0) scale[k] = (uint8_t)scale8[k];
}

// p[k] for a wave-uniform k, of a table no kernel writes while it runs: a scalar load.  Left to the compiler it becomes a
// vector load behind the memory barriers, and waiting for it waits for every load of the stage before.
__device__ __forceinline__ int table(const int *p, int k)
{
    return ((const __attribute__((address_space(4))) int *)p)[__builtin_amdgcn_readfirstlane(k)];
}

// ---- few vectors ----------------------------------------------------------------------------------------------

// One workgroup per S strips of 16 rows and NT tiles of 16 vectors; its W waves take the strips' blocks in turn and add
// their results in LDS.  Bound by reading the matrix once (8192 x 8192, up to 16 vectors in 8 bits: 12.5 us, 5.4 TB/s),
// for small matrices by latency -- a wave's next block is on its way while it works on one -- and with more vectors by
// widening x, which every strip's workgroup does again: two strips share it.  XT: uint8_t (x in 8 bits) or a wide type,
// rounded to 8 bits here: lane (i, q) holds the 32 entries of vector i that it multiplies, 4 lanes a group of 128.
// Operands are widened to bf16 (unpack4), sums are 32 bits.
template <typename XT, int NT, int W, int S>
__global__ __launch_bounds__(W *kWave) void few_vectors_kernel(int n, int rows, int columns, const int *__restrict__ block_ptr,
                                                               const int *__restrict__ block_col, const uint8_t *__restrict__ val8,
                                                               const int *__restrict__ scale8, const XT *__restrict__ x,
                                                               int64_t ldx, const uint8_t *__restrict__ xscale, int64_t lds,
                                                               void *__restrict__ y, int y_dtype, int64_t ldy)
{
    constexpr bool kEight = std::is_same<XT, uint8_t>::value;
    __shared__ f32x4 part[W][NT][kWave];
    const int brow = blockIdx.x / (8 / S), strip0 = blockIdx.x % (8 / S) * S;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), i = lane & 15, q = lane >> 4;
    f32x4 acc[S][NT];
#pragma unroll
    for (int k = 0; k < S; k++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[k][t] = f32x4{0, 0, 0, 0};
    const int v0 = blockIdx.y * 16 * NT;
    // vectors past the last read the last: a column of the result that is not stored
    int64_t vec[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) vec[t] = min(v0 + t * 16 + i, n - 1);

    constexpr bool AHEAD = NT * sizeof(XT) <= 4;             // x ahead too, in up to 32 registers
    struct Vector {
        Raw<XT, 16> h[2];
        int scale;
    };
    struct Stage {
        u32x4 a[S][2];
        int scale, group;
        Vector x[AHEAD ? NT : 1];
    };
    auto load_x = [&](int t, int group) {
        Vector r;
        const int c = group * kB + 16 * q;
        const XT *p = x + vec[t] * ldx + c;
        if constexpr (kEight) {
            r.h[0].load(p, 16);
            r.h[1].load(p + 64, 16);
            r.scale = xscale[(int64_t)group * lds + vec[t]];
        } else {
            r.h[0].load(p, columns - c);
            r.h[1].load(p + 64, columns - c - 64);
        }
        return r;
    };
    auto load = [&](int b) {
        Stage s;
        const uint8_t *block = val8 + (int64_t)b * kBlockBytes + (strip0 * 2 * kWave + lane) * 16;
#pragma unroll
        for (int k = 0; k < 2 * S; k++) s.a[k >> 1][k & 1] = *(const u32x4 *)(block + k * kWave * 16);
        s.scale = table(scale8, b);
        s.group = table(block_col, b);
        if constexpr (AHEAD)
#pragma unroll
            for (int t = 0; t < NT; t++) s.x[t] = load_x(t, s.group);
        return s;
    };
    auto use = [&](const Stage &s) {
        const float sa = scale_half(s.scale);
        bf16x8 a[S][4];
#pragma unroll
        for (int d = 0; d < 8 * S; d++) unpack4(s.a[d >> 3][d >> 2 & 1][d & 3], sa, (__bf16 *)&a[d >> 3][d >> 1 & 3] + 4 * (d & 1));
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const Vector v = AHEAD ? s.x[AHEAD ? t : 0] : load_x(t, s.group);
            unsigned w8[8];
            int bx;
            if constexpr (kEight) {
                __builtin_memcpy(w8, v.h, 32);
                bx = v.scale;
            } else {
                float top = fmaxf(finite_top(v.h[0]), finite_top(v.h[1]));
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                bx = scale_byte(top);
                v.h[0].pack(scale_value(bx), w8);
                v.h[1].pack(scale_value(bx), w8 + 4);
            }
            const float sx = scale_half(bx);
#pragma unroll
            for (int p = 0; p < 4; p++) {
                bf16x8 b;
                unpack4(w8[2 * p], sx, (__bf16 *)&b);
                unpack4(w8[2 * p + 1], sx, (__bf16 *)&b + 4);
#pragma unroll
                for (int k = 0; k < S; k++) acc[k][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k][p], b, acc[k][t], 0, 0, 0);
            }
        }
    };
    const int first = table(block_ptr, brow) + wave, last = table(block_ptr, brow + 1);
    if (first < last) {
        Stage now = load(first);
        for (int b = first; b < last; b += W) {
            const Stage next = load(b + W < last ? b + W : b);
            use(now);
            now = next;
        }
    }
#pragma unroll
    for (int k = 0; k < S; k++) {
        const int strip = strip0 + k;
        if (k) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) part[wave][t][lane] = acc[k][t];
        __syncthreads();
        for (int id = threadIdx.x; id < NT * kWave; id += W * kWave) {
            const int t = id / kWave, l = id & (kWave - 1), v = v0 + t * 16 + (l & 15);
            f32x4 s = part[0][t][l];
#pragma unroll
            for (int w = 1; w < W; w++) s += part[w][t][l];
            s *= 4.0f;                                       // both operands were halves
            const int r0 = brow * kB + (strip >> 2) * 64 + 16 * (l >> 4) + (strip & 3);
            if (v >= n) continue;
            for (int e = 0; e < 4; e++) {
                if (r0 + 4 * e >= rows) break;
                const int64_t at = (int64_t)v * ldy + r0 + 4 * e;
                if (y_dtype == SPMV_HIP_F32) ((float *)y)[at] = s[e];
                else if (y_dtype == SPMV_HIP_BF16) ((__bf16 *)y)[at] = (__bf16)s[e];
                else ((_Float16 *)y)[at] = (_Float16)s[e];
            }
        }
    }
}

// ---- many vectors ---------------------------------------------------------------------------------------------

// One workgroup: 128 rows (or columns, of one block row or column) x 32 NU vectors; a wave has half the rows and half the
// vectors, 64 x 16 NU.  What comes from LDS is read as 16 bytes a lane where the layout allows: such a read takes the LDS 7
// cycles a wave, an 8-byte read as long, a 16-byte write from registers 13.  R stages are in flight or in use; a stage's
// loads are issued R - 1 steps ahead: one step where two workgroups of 256 vectors share a CU and cover each other's waits,
// three where there are few workgroups and a step is short.


// Keeps a scalar load where it is written: the compiler would move it down to its use in the next step, and wait there
__device__ __forceinline__ void here(int &a) { asm volatile("" : "+s"(a)); }

// Wait until at most N of the wave's loads are outstanding and its LDS reads are done, then meet the others.  What the
// compiler does not see, it does not move: the asm statements order the memory accesses around them.
template <int N> __device__ __forceinline__ void stage_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b)
{
    return (i32x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// `records` bytes at a wave-uniform address (a raw buffer descriptor); loads past them bring zeros
__device__ __forceinline__ u32x4 buffer(const void *base, unsigned records)
{
    const uint64_t at = (uint64_t)base;
    return u32x4{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, records, 0x00027000u};
}
// 64 lanes x 16 bytes into LDS, lane l to lds + 16 l (lds is the wave's), from its own offset into the buffer.
// ASM: behind the builtin the compiler makes LDS reads that it cannot tell apart from these stores wait for all of them; in
// assembly it does not see them, and the wait is stage_barrier's alone (transposed product of 8192 vectors, full 8192 x
// 8192: 890 -> 824 us).  But neither does it move anything past the assembly (the product: 430 -> 490 us), so it is for
// the kernel that needs it.  The load has no register results; m0 needs a cycle before it is used, and a descriptor that
// a vector instruction made (readfirstlane) five.
template <bool ASM> __device__ __forceinline__ void load_to_lds(u32x4 r, unsigned offset, uint8_t *lds)
{
    const auto to = (__attribute__((address_space(3))) uint8_t *)lds;
    if constexpr (ASM)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                     ::"v"(offset), "s"(r), "s"(__builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)to)) : "memory", "m0");
    else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)r[1] << 32 | r[0]), 0, (int)r[2], (int)r[3]),
            (__attribute__((address_space(3))) void *)to, 16, (int)offset, 0, 0, 0);
}

// step(slot, k, behind) for k = first .. last - 1, slot = (k - first) % R as a constant: whole rounds, then what is left (exits
// from inside a round would cost the accumulators copies).  `behind`: how many stages have been issued behind stage k when
// the step begins, so that its wait may leave their loads outstanding.  A step of a whole round issues stage k + R - 1;
// the last ones, `behind` = TAIL + that number, issue nothing: all stages are under way, and loads that nothing uses any more
// would be dropped by the compiler while the wait went on counting them.
constexpr int TAIL = 100;
template <int R, typename F> __device__ __forceinline__ void ring(int first, int last, F step)
{
    int k = first;
    for (; k + R <= last; k += R) {
        step(ic<0>(), k, ic<R - 2>());
        step(ic<1>(), k + 1, ic<R - 2>());
        if constexpr (R > 2) step(ic<2>(), k + 2, ic<R - 2>());
        if constexpr (R > 3) step(ic<3>(), k + 3, ic<R - 2>());
    }
    if (k < last) step(ic<0>(), k, ic<TAIL + R - 2>());
    if constexpr (R > 2) if (k + 1 < last) step(ic<1>(), k + 1, ic<TAIL + R - 3>());
    if constexpr (R > 3) if (k + 2 < last) step(ic<2>(), k + 2, ic<TAIL + R - 4>());
}
// Keeps the memory accesses before it before those behind it: a wait counts the loads of whole stages, in their order
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// G = 2 groups of four waves share a tile whose workgroup has a CU to itself, each with half of the sum and its own stages: one
// group's loads and LDS reads run beside the other's matrix instructions.  Every barrier is the whole workgroup's, so
// both pass as many; `rounds`, the steps of the first, is the larger number.
template <int G> __device__ __forceinline__ int half_of(int group, int *first, int *last)
{
    if (G == 1) return *last - *first;
    const int rounds = (*last - *first + 1) / 2;
    if (group) *first += rounds;
    else *last = *first + rounds;
    return rounds;
}
// adds the second group's sums to the first's, through LDS that nothing else uses any more; true in the first
template <int G, int NU> __device__ __forceinline__ bool joined(int group, int tid, f32x4 *lds, f32x4 (&acc)[NU][4])
{
    if constexpr (G > 1) {
        if (group)
#pragma unroll
            for (int k = 0; k < 4 * NU; k++) lds[k * kBlock + tid] = acc[k >> 2][k & 3];
        __syncthreads();
        if (group) return false;
#pragma unroll
        for (int k = 0; k < 4 * NU; k++) acc[k >> 2][k & 3] += lds[k * kBlock + tid];
    }
    return true;
}

// logical tile of a workgroup: every XCD walks its own eighth of the tiles, in it `side` block rows (columns) side by side
// and then the next vectors, so that the blocks and the vectors of the workgroups that run together stay in its L2
__device__ __forceinline__ void tile_of_block(unsigned bid, int majors, int vtiles, unsigned side, int *major, int *vtile)
{
    const unsigned id = xcd_contiguous_block(bid, (unsigned)majors * vtiles);
    const unsigned per = side * vtiles, group = id / per, in = id % per;
    const unsigned wide = (unsigned)majors - group * side < side ? (unsigned)majors - group * side : side;
    *major = (int)(group * side + in % wide);
    *vtile = (int)(in / wide);
}

// results m .. m + 4 COUNT - 1 of one vector, as many as there are below `limit`
template <typename OT, int COUNT>
__device__ __forceinline__ void store_row(OT *o, int left, const f32x4 *a)
{
    if (left >= 4 * COUNT) {
        OT v[4 * COUNT];
#pragma unroll
        for (int k = 0; k < 4 * COUNT; k++) v[k] = (OT)a[k >> 2][k & 3];
        __builtin_memcpy(o, v, sizeof v);
    } else {
        for (int k = 0; k < 4 * COUNT; k++)
            if (k < left) o[k] = (OT)a[k >> 2][k & 3];
    }
}

struct ProductArgs {
    int n, rows, brows, vtiles;
    const int *ptr, *col, *scale8;
    const uint8_t *val8, *x8, *xscale;
    int64_t ldx8, lds, ldy;
};

// y = A x, a block a step.  The vectors go to LDS by direct loads, rows of 128 bytes, their 16-byte pieces exchanged by
// XOR so that the 8 lanes of a read cycle meet 8 different pieces; the blocks, whose layout is the operand's, go straight
// to the registers of the two waves that need each half.  Vector NU i + u belongs to lane i of tile u: a lane's scale
// bytes are neighbours.
// EXACT: operands widened to bf16 in registers (unpack4), 32-bit sums.  Otherwise the 8-bit matrix instruction, which applies
// both scales and runs at twice the rate, but aligns 8 products at a time and drops what lies 13 bits below the largest:
// good to about 16 bits, for bf16 results only.
// 8192 vectors, full 8192 x 8192, bf16: 422 us at the least, 489 in the median of a kernel trace, 2.6 and 2.25 PFLOP/s (a library
// product of plain 8-bit matrices of that size reaches 3.2); the matrix pipes are busy 64 % of the cycles at the 1.9 GHz that
// the power allows.  Widened: 830 us in calls one after the other, where bf16 takes 415-430.  LDS reads that
// meet twice as many banks (vectors exchanged in pairs too) changed nothing.  Few workgroups are bound by the chain of a
// step -- LDS, widening, products -- which two groups of waves overlap.
template <bool EXACT, int NU, int G, typename OT>
__global__ __launch_bounds__(G *kBlock, 2) void product_kernel(ProductArgs g, OT *__restrict__ y)
{
    constexpr int R = NU == 8 ? 2 : NU == 4 ? 3 : 4, TOK = 32 * NU;
    __shared__ uint8_t all_x[G][R][TOK * kB];
    const int group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock), tid = G == 1 ? threadIdx.x : threadIdx.x % kBlock;
    auto &X = all_x[group];
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), i = lane & 15, q = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    int major, vtile;
    tile_of_block(blockIdx.x, g.brows, g.vtiles, 8, &major, &vtile);
    const int t0 = vtile * TOK, v0 = t0 + wn * 16 * NU + NU * i;             // the tile's and the lane's first vector
    int first = table(g.ptr, major), last = table(g.ptr, major + 1);
    const int rounds = half_of<G>(group, &first, &last);
    f32x4 acc[NU][4];
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int s = 0; s < 4; s++) acc[u][s] = f32x4{0, 0, 0, 0};

    // piece j of a thread: 16 bytes of vector 32 j + t.  The 16-byte pieces of vector v are exchanged by v / NU, which
    // for 256 vectors differs between even and odd j.  Past the last vector zeros.
    const int t = wave * 8 + (lane >> 3);
    const unsigned at = (unsigned)t * (unsigned)g.ldx8 + (((lane & 7) ^ ((t / NU) & 7)) << 4);
    const uint8_t *xbase = g.x8 + (int64_t)t0 * g.ldx8;
    const unsigned ldx8 = (unsigned)g.ldx8, records = (unsigned)min(g.n - t0, TOK) * ldx8;
    const u32x4 xs = buffer(xbase, records);
    const int back = max(v0 - g.n + NU, 0);                  // n > NU, so the load of scale bytes can move back from the end

    i32x8 a[R][4];
    uint64_t sx[R];
    int sa[R], c = 0, scale = 0;                             // c, scale: of the block issued next, loaded a step before
    auto look_up = [&](int b) { c = table(g.col, b); scale = table(g.scale8, b); };
    auto issue = [&](auto slot, int b) {
        constexpr int S = decltype(slot)::value;
#pragma unroll
        for (int j = 0; j < NU; j++) {
            const unsigned skip = j * 32 * ldx8 + c * kB;
            uint8_t *to = &X[S][(j * 32 + wave * 8) * kB];
            if constexpr (NU < 8) load_to_lds<false>(xs, at + skip, to);
            else {                                           // 8 offsets more are too many registers: the buffer moves
                const unsigned gone = min(skip, records);
                load_to_lds<false>(buffer(xbase + gone, records - gone), j & 1 ? at ^ 64 : at, to);
            }
        }
        const uint8_t *half = g.val8 + (int64_t)b * kBlockBytes + wm * (kBlockBytes / 2);
#pragma unroll
        for (int s = 0; s < 4; s++) a[S][s] = join(*(const u32x4 *)(half + (lane * 16u + s * 2048)), *(const u32x4 *)(half + (lane * 16u + s * 2048 + 1024)));
        sa[S] = EXACT ? scale - 1 : scale;                   // of half the scale, for widening (unpack4)
        sx[S] = 0;
        __builtin_memcpy(&sx[S], g.xscale + (int64_t)c * g.lds + (v0 - back), NU);
        look_up(min(b + 1, last - 1));
    };
    auto step = [&](auto slot, int b, auto behind) {
        constexpr int S = decltype(slot)::value, BEHIND = decltype(behind)::value;
        constexpr bool MORE = BEHIND < TAIL;
        here(c);
        here(scale);
        stage_barrier<BEHIND % TAIL * (NU + 8)>();
        auto operand = [&](int u) {
            const uint8_t *row = &X[S][(wn * 16 * NU + NU * i + u) * kB];
            return join(*(const u32x4 *)(row + ((q ^ (i & 7)) << 4)), *(const u32x4 *)(row + (((q + 4) ^ (i & 7)) << 4)));
        };
        // The first reads before the next stage's loads, which take a while to issue.  With few tiles all of them; with 8
        // one tile ahead and no more: left alone, the compiler reads all of them first and runs out of registers.
        constexpr int AHEAD = NU == 8 || EXACT ? 1 : NU;
        i32x8 w[NU];
        if constexpr (MORE && NU == 8) issue(ic<(S + R - 1) % R>(), min(b + R - 1, last - 1));
#pragma unroll
        for (int u = 0; u < AHEAD; u++) w[u] = operand(u);
        if constexpr (MORE && NU < 8) issue(ic<(S + R - 1) % R>(), min(b + R - 1, last - 1));
        // for widening those of half the scales; past the last vector, in the upper bytes, whatever it is
        const uint64_t bytes = (sx[S] >> (8 * min(back, 7))) - (EXACT ? 0x0101010101010101u : 0);
        bf16x8 aw[4][EXACT ? 4 : 1];
        if constexpr (EXACT) {
            const float fa = scale_value(sa[S]);
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int d = 0; d < 8; d++) unpack4((unsigned)a[S][s][d], fa, (__bf16 *)&aw[s][d >> 1] + 4 * (d & 1));
        }
#pragma unroll
        for (int u = 0; u < NU; u++) {
            if (u + AHEAD < NU) w[u + AHEAD] = operand(u + AHEAD);
            const int su = (int)(bytes >> (8 * u)) & 255;
            if constexpr (EXACT) {
                const float fx = scale_value(su);
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    bf16x8 xw;
                    unpack4((unsigned)w[u][2 * p], fx, (__bf16 *)&xw);
                    unpack4((unsigned)w[u][2 * p + 1], fx, (__bf16 *)&xw + 4);
#pragma unroll
                    for (int s = 0; s < 4; s++) acc[u][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xw, aw[s][p], acc[u][s], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int s = 0; s < 4; s++)
                    acc[u][s] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[u], a[S][s], acc[u][s], 0, 0, 0, su, 0, sa[S]);
            }
            if (NU == 8) __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (first < last) {
        look_up(first);
        issue(ic<0>(), first);
        in_order();
        if constexpr (R > 2) issue(ic<1>(), min(first + 1, last - 1));
        in_order();
        if constexpr (R > 3) issue(ic<2>(), min(first + 2, last - 1));
        ring<R>(first, last, step);
    }
    for (int k = last - first; k < rounds; k++) stage_barrier<0>();      // as many as the other group
    stage_barrier<0>();                                      // no load to LDS outlives the workgroup
    if (!joined<G, NU>(group, tid, (f32x4 *)&all_x[0][0][0], acc)) return;
    // result k of tile (u, s) is vector NU (4 q + k) + u, row 4 i + s of the wave's 64: 16 lanes write 64 neighbours.
    const int r = major * kB + wm * 64 + 4 * i, v1 = t0 + wn * 16 * NU + NU * 4 * q;
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int u = 0; u < NU; u++) {
            f32x4 f = {acc[u][0][k], acc[u][1][k], acc[u][2][k], acc[u][3][k]};
            if (EXACT) f *= 4.0f;                            // both operands were halves
            const int v = v1 + NU * k + u;
            if (v < g.n && r < g.rows) store_row<OT, 1>(y + (int64_t)v * g.ldy + r, g.rows - r, &f);
        }
}

// dy is used as it is: as PARTS bf16 numbers that add up to it exactly (1 for bf16, 2 for fp16, 3 for fp32: each holds 8
// bits of the mantissa), one matrix instruction each.  Of fp32 entries below 2^-110 what lies under bf16's smallest step,
// 2^-133, is lost.
template <typename DT> struct parts_of { static constexpr int value = 1; };
template <> struct parts_of<_Float16> { static constexpr int value = 2; };
template <> struct parts_of<float> { static constexpr int value = 3; };

static int parts(int dtype) { return dtype == SPMV_HIP_BF16 ? 1 : dtype == SPMV_HIP_F16 ? 2 : 3; }

// dy into its parts, `plane` entries apart, vectors `ld` apart (a multiple of 128), zero past `length`; 8 entries a
// thread.  Before the products rather than in them: there the splitting stood between loads and matrix instructions of
// every step (fp32, 333 vectors, 264 blocks: 41 us, now 5 + 20).
template <typename T>
__global__ __launch_bounds__(kBlock) void split_kernel(int n, int length, int ld, const T *__restrict__ dy, int64_t lddy,
                                                       __bf16 *__restrict__ out, int64_t plane)
{
    constexpr int PARTS = parts_of<T>::value;
    const int64_t at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 8;
    if (at >= plane) return;
    const int64_t v = at / ld;
    const int c = (int)(at % ld);
    Raw<T, 8> r;
    r.load(dy + v * lddy + c, length - c);
    bf16x8 part[PARTS];
    if constexpr (PARTS == 1) __builtin_memcpy(&part[0], r.v, 16);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // each part the upper half of what is left, cut off, not rounded: the largest numbers would round to infinity
            float f = (float)r.v[e];
            const bool finite = fabsf(f) < __builtin_inff(); // infinities and NaN: all in the first
#pragma unroll
            for (int p = 0; p < PARTS; p++) {
                const float top = finite ? __uint_as_float(__float_as_uint(f) & 0xffff0000u) : f;
                part[p][e] = (__bf16)top;
                f = finite ? f - top : 0.0f;
            }
        }
#pragma unroll
    for (int p = 0; p < PARTS; p++) *(bf16x8 *)(out + p * plane + at) = part[p];
}

template <typename E> using vec8 = E __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct TransposedArgs {
    int n, rows, columns, bcols, vtiles;
    unsigned side;                 // block columns side by side
    const int *ptr, *row, *id, *scale;               // lists by block column, their blocks' scales
    const uint8_t *val8;
    const void *dy;
    int64_t lddy, plane, lddx, slice;    // plane: from one part of dy to the next; slice: of dx, where the sum is cut
};

// dx = A^T dy, half a block (64 rows) a step, blocks and vectors through LDS.  ds_read_b64_tr_b8 hands every lane one
// column of 8 rows of the block, widened to bf16 (unpack4) on the way to the matrix instruction.  8 rows of dy are 2 rows in
// each of four strips of the block (block8_offset); in LDS the 4-row pieces of a 16 x 16 subtile are exchanged by XOR
// with the strip, which puts the four on different banks.  The blocks of a last block row that is not whole come last in
// every list: they are taken after the others, one by one, with the entries past the end masked (dy in parts is padded
// and has no such rows).  fp16 dy multiplies blocks widened without their scale, which is put on the sums of half a block.
// 8192 vectors, full 8192 x 8192, bf16: 816 us at the least, 886 in the median of a kernel trace, 1.35 and 1.24 PFLOP/s (a
// library product of plain bf16 matrices 1.45); the matrix
// pipes are busy 64 % of the cycles at 2 GHz.
template <typename E, int PARTS, int NU, int G, typename OT>
__global__ __launch_bounds__(G *kBlock, 2) void transposed_kernel(TransposedArgs g, OT *__restrict__ dx)
{
    constexpr bool HALF = std::is_same<E, _Float16>::value;
    typedef vec8<E> e8;
    constexpr int R = PARTS * NU >= 6 ? 2 : PARTS * NU == 4 ? 3 : 4, TOK = 32 * NU;
    __shared__ uint8_t all_y[G][R][PARTS][TOK * 128];
    __shared__ uint8_t all_a[G][R][kBlockBytes / 2];
    const int group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock), tid = G == 1 ? threadIdx.x : threadIdx.x % kBlock;
    auto &Y = all_y[group];
    auto &A = all_a[group];
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), i = lane & 15, q = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    int major, vtile;
    tile_of_block(blockIdx.x, g.bcols, g.vtiles, g.side, &major, &vtile);
    const int t0 = vtile * TOK;
    const int begin = table(g.ptr, major), end = table(g.ptr, major + 1);
    int whole = end;
    if (PARTS == 1 && g.rows % kB)
        while (whole > begin && table(g.row, whole - 1) == g.rows / kB) whole--;
    int first = 2 * begin, last = 2 * whole, edge = last;    // half blocks of this slice; those with masked entries
    if (gridDim.y > 1) {
        const int per = (last - first + (int)gridDim.y - 1) / (int)gridDim.y;
        first = min(first + (int)blockIdx.y * per, last);
        last = min(first + per, last);
        if (blockIdx.y + 1 < gridDim.y) edge = 2 * end;
        dx += blockIdx.y * g.slice;
    }
    const int rounds = half_of<G>(group, &first, &last);
    f32x4 acc[NU][4];
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int s = 0; s < 4; s++) acc[u][s] = f32x4{0, 0, 0, 0};

    // piece j of a thread: 8 entries of vector 32 j + 8 wave + lane / 8, in place lane % 8 of its row in LDS; a
    // row's pieces are exchanged by XOR.  Past the last vector the loads bring zeros, and the result is not stored.
    const E *ybase = (const E *)g.dy + (int64_t)t0 * g.lddy;
    const int row_of_lane = wave * 8 + (lane >> 3), piece = (lane & 7) ^ ((row_of_lane >> 1) & 7);
    const unsigned lddy = (unsigned)g.lddy, near = row_of_lane * lddy + 8 * piece;
    u32x4 ys[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; p++) ys[p] = buffer(ybase + p * g.plane, (unsigned)min(g.n - t0, TOK) * lddy * 2);

    int sa[R], id = 0, row = 0, scale = 0;                   // id, row, scale: of the half block issued next, loaded a step before
    auto look_up = [&](int k) {
        id = table(g.id, k >> 1);
        row = table(g.row, k >> 1);
        scale = table(g.scale, k >> 1);
    };
    auto issue_block = [&](auto slot, int k) {
        constexpr int S = decltype(slot)::value;
        const u32x4 half = buffer(g.val8 + (int64_t)id * kBlockBytes + (k & 1) * (kBlockBytes / 2), kBlockBytes / 2);
        sa[S] = scale;
        // wave w brings strip w: 2 x 4 subtiles of 256 bytes
        const int from = wave * 2048 + q * 256 + ((i ^ (wave << 2)) << 4);
        load_to_lds<true>(half, from, &A[S][wave * 2048]);
        load_to_lds<true>(half, from + 1024, &A[S][wave * 2048 + 1024]);
    };
    auto issue = [&](auto slot, int k) {
        constexpr int S = decltype(slot)::value;
        issue_block(slot, k);
        const unsigned r = row * kB + (k & 1) * 64;
#pragma unroll
        for (int p = 0; p < PARTS; p++)
#pragma unroll
            for (int j = 0; j < NU; j++) load_to_lds<true>(ys[p], near * 2 + (j * 32 * lddy + r) * 2, &Y[S][p][(j * 32 + wave * 8) * 128]);
        look_up(min(k + 1, last - 1));
    };
    // `between` runs after the first reads from LDS: the next stage's loads, which take a while to issue.  All reads of the block
    // come before it -- the compiler cannot tell what a transposing read touches, and one behind the direct loads would wait
    // for them -- and with few tiles those of dy; with many, one tile ahead and no more.
    auto compute = [&](auto slot, auto between) {
        constexpr int S = decltype(slot)::value;
        constexpr bool ALL = PARTS * NU <= 4;
        auto read_a = [&](int h, int s) {
            // row 32 h + 8 q + w, w = i >> 1, columns 8 (i & 1) .. + 7 of a subtile
            const int strip = (i >> 1) & 3, in = 8 * h + 2 * q + (i >> 3);
            const uint8_t *p = &A[S][strip * 2048 + wm * 1024 + ((in ^ (strip << 2)) << 4) + (i & 1) * 8];
            return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2 *)(p + s * 256));
        };
        auto read_b = [&](int h, int part, int u) {
            const int t = wn * 16 * NU + 16 * u + i;
            return *(const e8 *)&Y[S][part][t * 128 + (((4 * h + q) ^ ((t >> 1) & 7)) << 4)];
        };
        i32x2 w[2][4];
        e8 b[2][PARTS][NU];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int s = 0; s < 4; s++) w[h][s] = read_a(h, s);
            if (ALL || h == 0)
#pragma unroll
                for (int part = 0; part < PARTS; part++)
#pragma unroll
                    for (int u = 0; u < (ALL ? NU : 1); u++) b[h][part][u] = read_b(h, part, u);
        }
        const float fa = HALF ? scale_value(sa[S]) : scale_half(sa[S]);
        between();
        e8 a[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if constexpr (!ALL && !HALF)
                if (h == 1) {
#pragma unroll
                    for (int part = 0; part < PARTS; part++) b[1][part][0] = read_b(1, part, 0);
                }
            if constexpr (HALF) {
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int d = 0; d < 2; d++) unpack4((unsigned)w[h][s][d], 1.0f, (E *)&a[h][s] + 4 * d);
                continue;
            }
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int d = 0; d < 2; d++) unpack4((unsigned)w[h][s][d], fa, (E *)&a[h][s] + 4 * d);
#pragma unroll
            for (int part = 0; part < PARTS; part++)
#pragma unroll
                for (int u = 0; u < NU; u++) {
                    if constexpr (!ALL) if (u + 1 < NU) b[h][part][u + 1] = read_b(h, part, u + 1);
#pragma unroll
                    for (int s = 0; s < 4; s++) acc[u][s] = mfma(a[h][s], b[h][part][u], acc[u][s]);
                    if (NU == 8 && (u & 1)) __builtin_amdgcn_sched_barrier(0);
                }
        }
        if constexpr (HALF) {
#pragma unroll
            for (int u = 0; u < NU; u++) {
                if (!ALL && u) {
                    b[0][0][u] = read_b(0, 0, u);
                    b[1][0][u] = read_b(1, 0, u);
                } else if (!ALL) b[1][0][0] = read_b(1, 0, 0);
                f32x4 t[4];
#pragma unroll
                for (int s = 0; s < 4; s++) t[s] = mfma(a[0][s], b[0][0][u], f32x4{0, 0, 0, 0});
#pragma unroll
                for (int s = 0; s < 4; s++) t[s] = mfma(a[1][s], b[1][0][u], t[s]);
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[u][s][r] = __builtin_fmaf(t[s][r], fa, acc[u][s][r]);
                if (NU == 8) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    auto step = [&](auto slot, int k, auto behind) {
        constexpr int S = decltype(slot)::value, BEHIND = decltype(behind)::value;
        here(id);
        here(row);
        here(scale);
        stage_barrier<BEHIND % TAIL * (2 + PARTS * NU)>();
        compute(slot, [&] { if constexpr (BEHIND < TAIL) issue(ic<(S + R - 1) % R>(), min(k + R - 1, last - 1)); });
    };
    if (first < last) {
        look_up(first);
        issue(ic<0>(), first);
        if constexpr (R > 2) issue(ic<1>(), min(first + 1, last - 1));
        if constexpr (R > 3) issue(ic<2>(), min(first + 2, last - 1));
        ring<R>(first, last, step);
    }
    for (int k = last - first; k < rounds; k++) stage_barrier<0>();      // as many as the other group
    stage_barrier<0>();                                      // no load to LDS outlives the workgroup, or meets the next
    for (int k = edge; k < 2 * end; k++) {
        look_up(k);
        issue_block(ic<0>(), k);
        const int r = row * kB + (k & 1) * 64;
        for (int j = 0; j < NU; j++) {
            Raw<E, 8> one;
            one.load(ybase + r + (unsigned)min(j * 32 + row_of_lane, g.n - 1 - t0) * lddy + 8 * piece, g.rows - (r + 8 * piece));
            __builtin_memcpy(&Y[0][0][(j * 32 + wave * 8) * 128 + lane * 16], one.v, 16);
        }
        stage_barrier<0>();
        if (group == 0) compute(ic<0>(), [] {});
        stage_barrier<0>();
    }
    if (!joined<G, NU>(group, tid, (f32x4 *)&all_y[0][0][0][0], acc)) return;
#pragma unroll
    for (int u = 0; u < NU; u++) {
        const int v = t0 + wn * 16 * NU + 16 * u + i;
        if (v >= g.n) continue;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const int c = major * kB + wm * 64 + 16 * s + 4 * q;
            if (!HALF) acc[u][s] *= 2.0f;                    // the blocks were halves
            if (c < g.columns) store_row<OT, 1>(dx + (int64_t)v * g.lddx + c, g.columns - c, &acc[u][s]);
        }
    }
}

struct GradientArgs {
    int n, rows, edge, columns, accumulate;      // rows of dy, and the matrix's; dy in parts is padded with zeros
    const int *list;               // NB blocks of one block row per workgroup, -1 = none
    const int *block_row, *block_col;
    const uint8_t *x8, *xscale;
    const __bf16 *dy;
    int64_t ldx8, lds, lddy, plane, slice;       // slice: of dv, where the sum is cut
};

// dA = dy^T x at the stored blocks, 32 vectors a step.  With NB = 2 a workgroup has two blocks of one block row, a wave
// 128 rows x 64 columns; with NB = 1 one block, a wave 64 x 64.  Both operands lie vector by vector, along the sum,
// and have to be turned.  dy, which all waves share, comes into LDS by direct loads and is turned by ds_read_b64_tr_b16 (a
// lane gets one row of 4 vectors); a vector's 16-byte pieces are exchanged by XOR so that the 8 vectors of a read cycle
// lie on different banks.  x goes straight into the registers of the wave that needs it, 4 columns of 8 vectors a lane:
// widened there with the vectors' scales (unpack4; pairs of columns, which share a scale), then the pairs are turned.  Lane
// i's columns are 4 i + s.
// 8192 vectors, full 8192 x 8192, bf16: 892 us at the least, 933 in the median of a kernel trace, 1.23 and 1.18 PFLOP/s; the
// matrix pipes are busy 59 % of the cycles at 2 GHz.  x
// through LDS as well, a third of the loads, left that as it is and made fp32's slower (fewer stages fit).
template <int PARTS, int NB, int G, typename OT>
__global__ __launch_bounds__(G *kBlock, 2) void gradient_kernel(GradientArgs g, OT *__restrict__ dv)
{
    constexpr int STEP = 32, NU = 4 * NB, R = NB == 2 ? (PARTS == 1 ? 3 : 2) : PARTS == 3 ? 3 : 4;
    __shared__ uint8_t all_y[G][R][PARTS][STEP * kB * 2];
    const int group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock), tid = G == 1 ? threadIdx.x : threadIdx.x % kBlock;
    auto &Y = all_y[group];
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), i = lane & 15, q = lane >> 4;
    const int wg = (int)xcd_contiguous_block(blockIdx.x, gridDim.x);
    const int which = NB == 2 ? wave >> 1 : 0;               // the wave's block, its columns and rows in it
    const int id0 = table(g.list, NB * wg), id = table(g.list, NB * wg + which);
    const int col = table(g.block_col, id < 0 ? id0 : id), c0 = (wave & 1) * 64, n0 = NB == 2 ? 0 : (wave >> 1) * 64;
    const int row0 = table(g.block_row, id0) * kB;
    f32x4 acc[NU][4];
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int s = 0; s < 4; s++) acc[u][s] = f32x4{0, 0, 0, 0};

    unsigned xr[R][8];
    uint64_t sx[R];
    const unsigned xat = 8 * (unsigned)q * (unsigned)g.ldx8 + 4 * i;
    // a thread's pieces of dy: 8 rows from `prow` on, of vectors 8 wave + q and 4 further
    const int prow = row0 + 8 * (i ^ (q << 1 | (wave & 1) << 3));
    const unsigned lddy = (unsigned)g.lddy, near = ((8 * wave + q) * lddy + prow) * 2;
    // The bound of the loads: the last vector's rows up to a whole 16 bytes.  A piece that the bound cuts loses the word it cuts
    // (odd `rows`); what lies past the rows is inside the piece's own 16 aligned bytes and reaches only rows that are not stored.
    const unsigned records = ((STEP - 1) * lddy + (((unsigned)g.rows + 7) & ~7u)) * 2;
    auto issue = [&](auto slot, int k) {                     // 32 whole vectors
        constexpr int S = decltype(slot)::value;
        const int t0 = k * STEP;
        const uint8_t *xp = g.x8 + (int64_t)t0 * g.ldx8 + col * kB + c0;
#pragma unroll
        for (int w = 0; w < 8; w++) xr[S][w] = *(const unsigned *)(xp + w * g.ldx8 + xat);
        __builtin_memcpy(&sx[S], g.xscale + (int64_t)col * g.lds + t0 + 8 * q, 8);
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const u32x4 y = buffer(g.dy + p * g.plane + (int64_t)t0 * g.lddy, records);
#pragma unroll
            for (int j = 0; j < 2; j++) load_to_lds<true>(y, near + j * 8 * lddy, &Y[S][p][(8 * wave + 4 * j) * 256]);
        }
    };
    // the vectors after the last whole 32; past the last dy is zero, and x the last one's, so that nothing new that is not
    // finite comes in
    auto bring_rest = [&](int t0) {
        const uint8_t *xp = g.x8 + (int64_t)t0 * g.ldx8 + col * kB + c0 + 4 * i;
        const uint8_t *sp = g.xscale + (int64_t)col * g.lds + t0;
        const int top = g.n - 1 - t0;
        sx[0] = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) {
            const int tx = min(8 * q + w, top);
            xr[0][w] = *(const unsigned *)(xp + (int64_t)tx * g.ldx8);
            sx[0] |= (uint64_t)sp[tx] << (8 * w);
        }
#pragma unroll
        for (int p = 0; p < PARTS; p++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int ty = 8 * wave + 4 * j + q;
                Raw<__bf16, 8> one;
                one.load(g.dy + p * g.plane + (int64_t)(t0 + min(ty, top)) * g.lddy + prow, ty <= top ? g.rows - prow : 0);
                __builtin_memcpy(&Y[0][p][(8 * wave + 4 * j) * 256 + lane * 16], one.v, 16);
            }
    };
    auto compute = [&](auto slot, auto between) {
        constexpr int S = decltype(slot)::value, AHEAD = PARTS * NU <= 8 ? PARTS * NU : 4;
        auto read_b = [&](int k) {
            typedef short i16x4 __attribute__((ext_vector_type(4)));
            // lane i: 4 rows of vector 8 q + i / 4, then of the one 4 further; it gets row i of those vectors
            const int v = 8 * q + (i >> 2), piece = n0 / 8 + 2 * (k % NU) + ((i >> 1) & 1);
            const uint8_t *at = &Y[S][k / NU][v * 256 + ((piece ^ ((v & 3) << 1 | (q & 1) << 3)) << 4) + (i & 1) * 8];
            union { i16x4 h[2]; bf16x8 v; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)at);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(at + 4 * 256));
            return u.v;
        };
        bf16x8 b[PARTS * NU];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) b[k] = read_b(k);
        bf16x8 a[4];
        {
            unsigned pair[8][2];                             // columns (0, 1) and (2, 3) of 8 vectors
            const uint64_t halves = sx[S] - 0x0101010101010101u;
#pragma unroll
            for (int w = 0; w < 8; w++) {
                const float f = scale_value((int)((unsigned)(halves >> (8 * w)) & 255));
                __bf16 u[4];
                unpack4(xr[S][w], f, u);
                __builtin_memcpy(pair[w], u, 8);
            }
#pragma unroll
            for (int s = 0; s < 4; s++) {
                unsigned v[4];
#pragma unroll
                for (int w = 0; w < 4; w++) v[w] = __builtin_amdgcn_perm(pair[2 * w + 1][s >> 1], pair[2 * w][s >> 1], s & 1 ? 0x07060302 : 0x05040100);
                __builtin_memcpy(&a[s], v, 16);
            }
        }
        // the loads of a later stage, which take a while to issue; with three parts halfway, or registers spill (2048 vectors,
        // 2048 blocks: 312 us, 400 before the products)
        constexpr int THEN = PARTS == 3 ? PARTS * NU / 2 : 0;
#pragma unroll
        for (int k = 0; k < PARTS * NU; k++) {
            if (k == THEN) between();
            if (k + AHEAD < PARTS * NU) b[k + AHEAD] = read_b(k + AHEAD);
#pragma unroll
            for (int s = 0; s < 4; s++) acc[k % NU][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[k], a[s], acc[k % NU][s], 0, 0, 0);
        }
    };
    const int whole = g.n / STEP;
    int first = 0, last = whole, rest = whole * STEP;
    if (gridDim.y > 1) {                                     // this slice of the sum
        const int per = (whole + (int)gridDim.y - 1) / (int)gridDim.y;
        first = min((int)blockIdx.y * per, whole);
        last = min(first + per, whole);
        if (blockIdx.y + 1 < gridDim.y) rest = g.n;
        dv += blockIdx.y * g.slice;
    }
    const int rounds = half_of<G>(group, &first, &last);
    if (first < last) {
        issue(ic<0>(), first);
        if constexpr (R > 2) issue(ic<1>(), min(first + 1, last - 1));
        if constexpr (R > 3) issue(ic<2>(), min(first + 2, last - 1));
        ring<R>(first, last, [&](auto slot, int k, auto behind) {
            constexpr int S = decltype(slot)::value, BEHIND = decltype(behind)::value;
            stage_barrier<BEHIND % TAIL * (9 + 2 * PARTS)>();
            compute(slot, [&] { if constexpr (BEHIND < TAIL) issue(ic<(S + R - 1) % R>(), min(k + R - 1, last - 1)); });
        });
    }
    for (int k = last - first; k < rounds; k++) stage_barrier<0>();      // as many as the other group
    stage_barrier<0>();                                      // no load to LDS outlives the workgroup, or meets the next
    if (rest < g.n) {
        bring_rest(rest);
        stage_barrier<0>();
        if (group == 0) compute(ic<0>(), [] {});
        if (G > 1) stage_barrier<0>();
    }
    if (!joined<G, NU>(group, tid, (f32x4 *)&all_y[0][0][0][0], acc)) return;
    if (id < 0) return;
    // result r of tile (u, s) is row 16 u + 4 q + r, column 4 i + s: 16 lanes write 64 neighbours of a row.  (With the
    // operands the other way round a lane had 16 neighbours, and a store 64 pieces of 16 bytes: 50 us more for 8192 vectors.)
    const int c = c0 + 4 * i, left = g.columns - (col * kB + c);
    OT *o = dv + (int64_t)id * kBlockBytes + (n0 + 4 * q) * kB + c;
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 16 * u + r;
            // beyond the edge x is zero, but for 8-bit vectors that were not made by quantize8
            const int here = row0 + n0 + 4 * q + row < g.edge ? left : 0;
            f32x4 v;
#pragma unroll
            for (int s = 0; s < 4; s++) v[s] = s < here ? 2.0f * acc[u][s][r] : 0.0f;      // x was halved
            if (g.accumulate) {
                Raw<OT, 4> old;
                old.load(o + row * kB, 4);
#pragma unroll
                for (int s = 0; s < 4; s++) v[s] += (float)old.v[s];
            }
            store_row<OT, 1>(o + row * kB, 4, &v);
        }
}

// out (+)= the slices of a cut sum, added in their order; rows of `ldin` entries (a multiple of 4), 4 a thread
template <typename OT>
__global__ __launch_bounds__(kBlock) void join_kernel(int64_t count, int columns, int slices, const float *__restrict__ in, int64_t ldin,
                                                      int64_t slice, OT *__restrict__ out, int64_t ldout, int accumulate)
{
    const int64_t at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 4;
    if (at >= count) return;
    const int64_t r = at / ldin;
    const int c = (int)(at % ldin), left = columns - c;
    if (left <= 0) return;
    OT *o = out + r * ldout + c;
    f32x4 sum = *(const f32x4 *)(in + at);
    for (int z = 1; z < slices; z++) sum += *(const f32x4 *)(in + z * slice + at);
    if (accumulate) {
        Raw<OT, 4> old;
        old.load(o, left);
#pragma unroll
        for (int k = 0; k < 4; k++) sum[k] += (float)old.v[k];
    }
    store_row<OT, 1>(o, left, &sum);
}

// ---- launches -------------------------------------------------------------------------------------------------

static int launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return 1;
}

// groups of `per` vectors; n may be the largest int
static int tiles_of(int n, int per) { return (int)(((int64_t)n + per - 1) / per); }
static int groups_of(int length) { return length / kB + (length % kB != 0); }

// a launch has fewer than 2^32 threads along x
static int check_launch(const char *what, int64_t workgroups, int threads)
{
    if (workgroups <= 0xffffffffll / threads) return 0;
    set_error("%s: %lld workgroups of %d threads are more than one launch takes", what, (long long)workgroups, threads);
    return 1;
}

static int launch_few(const spmv_hip_matrix *m, int n, const void *x, int x_dtype, int64_t ldx, const uint8_t *xscale,
                      int64_t lds, void *y, int y_dtype, int64_t ldy, hipStream_t st)
{
    // 16 waves a workgroup where every one of them gets a block, else 4; two strips a workgroup where that leaves workgroups
    // for two CUs in three (8 bits, 64 vectors: 8192 x 8192 37.7 us with one, 22.3 with two; 4096 x 4096 11.1 and 12.4)
    const bool many_waves = m->nblocks >= 16 * (int64_t)m->brows, pairs = m->brows * (int64_t)6 >= m->cus;
    if (check_launch("block8_mult", m->brows * (int64_t)(pairs ? 4 : 8), (many_waves ? 16 : 4) * kWave)) return 1;
    auto go = [&](auto t) {
        typedef decltype(t) XT;
        auto launch = [&](auto kernel, int waves, int strips) {
            hipLaunchKernelGGL(kernel, dim3(m->brows * (8 / strips), tiles_of(n, 64)), dim3(waves * kWave), 0, st, n, m->rows, m->columns, m->d_block_ptr,
                               m->d_block_col, m->d_val8, m->d_scale8, (const XT *)x, ldx, xscale, lds, y, y_dtype, ldy);
        };
        auto tiles = [&](auto w, auto two) {
            constexpr int W = decltype(w)::value, S = decltype(two)::value;
            if (n <= 16) launch(few_vectors_kernel<XT, 1, W, S>, W, S);
            else if (n <= 32) launch(few_vectors_kernel<XT, 2, W, S>, W, S);
            else launch(few_vectors_kernel<XT, 4, W, S>, W, S);
        };
        if (many_waves && pairs) tiles(ic<16>(), ic<2>());
        else if (many_waves) tiles(ic<16>(), ic<1>());
        else if (pairs) tiles(ic<4>(), ic<2>());
        else tiles(ic<4>(), ic<1>());
    };
    if (x_dtype == SPMV_HIP_E4M3) go(uint8_t());
    else with_elem(x_dtype, go);
    return launched("block8_mult");
}

int launch_block8_f32(const spmv_hip_matrix *m, int n, const float *d_x, int64_t ldx, float *d_y, int64_t ldy,
                      hipStream_t stream)
{
    if (m->rows == 0) return 0;
    for (int64_t v = 0; v < n; v += SPMV_HIP_BLOCK8_MAX_WIDE) {
        const int k = (int)std::min(n - v, (int64_t)SPMV_HIP_BLOCK8_MAX_WIDE);
        if (launch_few(m, k, d_x + v * ldx, SPMV_HIP_F32, ldx, nullptr, 0, d_y + v * ldy, SPMV_HIP_F32, ldy, stream)) return 1;
    }
    return 0;
}

static int bad_dtype(const char *what, int dtype)
{
    set_error("%s: element type %d must be F32, BF16 or F16", what, dtype);
    return 1;
}
static int check_vectors(const char *what, int n, const void *p, int64_t ld, int length)
{
    if (n < 0) { set_error("%s: negative vector count %d", what, n); return 1; }
    if (n > 0 && length > 0 && !p) { set_error("%s: NULL vector block", what); return 1; }
    if (n > 1 && ld < length) { set_error("%s: vectors %lld apart are shorter than their length %d", what, (long long)ld, length); return 1; }
    return 0;
}
static int check_eight(const char *what, int n, int columns, const void *x8, int64_t ldx8, const void *scale, int64_t lds)
{
    if (n < 0) { set_error("%s: negative vector count %d", what, n); return 1; }
    if (n == 0 || columns == 0) return 0;
    if (!x8 || !scale) { set_error("%s: NULL 8-bit vectors or scales", what); return 1; }
    if (ldx8 % kB || ldx8 < (int64_t)groups_of(columns) * kB) {
        set_error("%s: 8-bit vectors %lld apart, need a multiple of 128 of at least %lld", what, (long long)ldx8, (long long)groups_of(columns) * kB);
        return 1;
    }
    if ((uintptr_t)x8 % 16) { set_error("%s: 8-bit vectors are not 16-byte aligned", what); return 1; }
    if (ldx8 >= (int64_t)1 << 24) {          // 256 of them stay inside 32-bit offsets
        set_error("%s: 8-bit vectors %lld apart, at most 2^24 - 128", what, (long long)ldx8);
        return 1;
    }
    if (lds < n) { set_error("%s: %lld scales per group for %d vectors", what, (long long)lds, n); return 1; }
    return 0;
}
static int check_block8(const char *what, const spmv_hip_matrix *m)
{
    if (!m) { set_error("NULL handle"); return 1; }
    if (m->format != SPMV_HIP_BLOCK8) { set_error("%s needs a handle of 8-bit blocks (format %d)", what, m->format); return 1; }
    return 0;
}
// workgroups of quantize8 / restore8; R vectors a wave
static bool many_groups(int n, int groups) { return (int64_t)(n / 16) * ((groups + kQuantGroups - 1) / kQuantGroups) >= 512; }
static int64_t group_grid(int n, int groups, int r)
{
    return (int64_t)tiles_of(n, kQuantWaves * r) * ((groups + kQuantGroups - 1) / kQuantGroups);
}

// Tiles of 16 vectors a wave takes: `most` where that still makes `least` workgroups, else half, down to 2; 4 are enough with
// `four` workgroups
static int vector_tiles(int majors, int n, int most, int least, int four)
{
    int nu = most;
    while (nu > 2 && (int64_t)majors * tiles_of(n, 32 * nu) < (nu == 4 ? four : least)) nu /= 2;
    return nu;
}

// How a backward call runs; `work` in bytes: the parts of dy, its copy for dx, then the slices of a cut sum
struct BackwardPlan {
    int dx_parts, dv_parts;        // bf16 numbers an entry of dy is taken as
    bool pairs;                    // two blocks of a block row a workgroup
    bool dx_halves, dv_halves;     // a workgroup is two groups of waves
    int tiles, dx_slices, dv_slices;
    int64_t dx_slice, dv_slice, parts_bytes, copy_bytes, work;
};

// Slices to cut sums of `steps` steps into, whose `tiles` workgroups leave CUs idle: as many as take the least time by
// what was measured -- `step` us for two steps in a CU's two groups of waves; the slices, `bytes` each, written and
// read again at 4 TB/s, and 5 us for the launch that adds them.
static int slices(int64_t tiles, int64_t steps, int cus, float step, int64_t bytes)
{
    int best = 1;
    float least = (steps + 1) / 2 * step;
    for (int64_t k = 2; k * tiles <= cus && k <= steps; k += k / 2) {
        const float us = (steps + 2 * k - 1) / (2 * k) * step + 5.0f + k * bytes * 0.5e-6f;
        if (us < least) { least = us; best = (int)k; }
    }
    return best;
}

static BackwardPlan backward_plan(const spmv_hip_matrix *m, int n, const void *d_dy, int dtype, int64_t lddy, bool with_dx, bool with_dv)
{
    BackwardPlan p{};
    p.dx_slices = p.dv_slices = 1;
    if (n <= 0) return p;
    // Into the products dy goes in bf16 parts (fp32: 3; fp16: 2, for dvalues), or as it lies (bf16; fp16, for dx), from 16-byte
    // aligned vectors: others are copied first.
    const bool lies = (uintptr_t)d_dy % 16 == 0 && (n == 1 || lddy % 8 == 0);
    p.dv_parts = parts(dtype);
    p.dx_parts = dtype == SPMV_HIP_F32 ? 3 : 1;
    if (m->rows > 0) {
        const int64_t plane = (int64_t)n * m->brows * kB * 2;
        if (dtype == SPMV_HIP_F32 ? with_dx || with_dv : dtype == SPMV_HIP_F16 ? with_dv : !lies) p.parts_bytes = p.dv_parts * plane;
        if (dtype == SPMV_HIP_F16 && with_dx && !lies) p.copy_bytes = plane;
    }
    if (with_dx && m->bcols) {
        // dy in parts: 2, so that two workgroups fit a CU (fp32, 3000 vectors, 440 blocks: 157 us, 189 with 4).  bf16: more
        // only with 1 1/2 workgroups a CU left (777 vectors: 30 us, 42 with 4; 3000: 66 us with 8, 77 with 2)
        p.tiles = p.dx_parts > 1 ? 2 : vector_tiles(m->bcols, n, 8, m->cus * 3 / 2, m->cus * 3 / 2);
        p.dx_slice = (int64_t)n * m->bcols * kB;
        const int64_t tiles = (int64_t)m->bcols * tiles_of(n, 32 * p.tiles), steps = 2 * (int64_t)m->longest;
        p.dx_slices = slices(tiles, steps, m->cus, 0.2f + 0.3f * p.dx_parts, p.dx_slice * 4);
        p.dx_halves = p.tiles == 2 && tiles * p.dx_slices <= m->cus && steps >= 4 * p.dx_slices;
    }
    if (with_dv && m->nblocks) {
        // two blocks a workgroup once they fill the GPU (512 blocks, 2000 vectors of bf16: 44 us, 56 with one), and not where
        // many pairs lack their second block
        p.pairs = m->npairs >= m->cus && m->nblocks * (int64_t)4 >= m->npairs * (int64_t)7;
        p.dv_slice = (int64_t)m->nblocks * kBlockBytes;
        p.dv_slices = slices(p.pairs ? m->npairs : m->nblocks, n / 32, m->cus, 0.2f + 0.25f * p.dv_parts, p.dv_slice * 4);
        p.dv_halves = !p.pairs && (int64_t)m->nblocks * p.dv_slices <= m->cus && n / 32 >= 4 * p.dv_slices;
    }
    p.work = p.parts_bytes + p.copy_bytes + 4 * std::max(p.dx_slices > 1 ? p.dx_slices * p.dx_slice : 0, p.dv_slices > 1 ? p.dv_slices * p.dv_slice : 0);
    return p;
}

template <typename O>
static void launch_join(int64_t rows, int64_t ldin, int columns, int slices, const float *in, O *out, int64_t ldout, int accumulate, hipStream_t st)
{
    const int64_t count = rows * ldin;
    hipLaunchKernelGGL(join_kernel<O>, dim3((unsigned)((count / 4 + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, count, columns, slices, in, ldin,
                       count, out, ldout, accumulate);
}

} // namespace spmv

using namespace spmv;

extern "C" {

spmv_hip_matrix *spmv_hip_create_block8(int rows, int columns, int nblocks, const int *block_ptr, const int *block_col)
{
    clear_error();
    if (rows < 0 || columns < 0 || nblocks < 0) { set_error("negative dimension"); return nullptr; }
    if (!block_ptr || (nblocks > 0 && !block_col)) { set_error("NULL block array"); return nullptr; }
    const int brows = groups_of(rows), bcols = groups_of(columns);
    if (block_ptr[0] != 0 || block_ptr[brows] != nblocks) {
        set_error("block_ptr[0] must be 0 and block_ptr[%d] must equal nblocks", brows);
        return nullptr;
    }
    for (int r = 0; r < brows; r++)
        if (block_ptr[r + 1] < block_ptr[r]) { set_error("block_ptr decreases at block row %d", r); return nullptr; }
    for (int k = 0; k < nblocks; k++)
        if (block_col[k] < 0 || block_col[k] >= bcols) { set_error("block column %d out of range at block %d", block_col[k], k); return nullptr; }
    spmv_hip_matrix *m = new (std::nothrow) spmv_hip_matrix();
    if (!m) { set_error("out of host memory"); return nullptr; }
    m->format = SPMV_HIP_BLOCK8; m->dtype = SPMV_HIP_F32; m->rows = rows; m->columns = columns;
    m->nblocks = nblocks; m->brows = brows; m->bcols = bcols;
    m->stored = (int64_t)nblocks * kBlockBytes;
    if (hipGetDevice(&m->device) != hipSuccess) { set_error("no HIP device available"); delete m; return nullptr; }
    if (hipDeviceGetAttribute(&m->cus, hipDeviceAttributeMultiprocessorCount, m->device) != hipSuccess) m->cus = 0;
    (void)hipGetLastError();
    bool ok = false;
    try {
        // the blocks once more, by block column; inside one in ascending block row
        std::vector<int> row((size_t)nblocks), tptr((size_t)bcols + 1, 0), trow((size_t)nblocks), tid((size_t)nblocks),
            tat((size_t)nblocks);
        for (int r = 0; r < brows; r++)
            for (int k = block_ptr[r]; k < block_ptr[r + 1]; k++) {
                row[(size_t)k] = r;
                tptr[(size_t)block_col[k] + 1]++;
                m->nnz += (int64_t)(rows - r * kB < kB ? rows - r * kB : kB) *
                          (columns - block_col[k] * kB < kB ? columns - block_col[k] * kB : kB);
            }
        for (int c = 0; c < bcols; c++) {
            m->longest = std::max(m->longest, tptr[(size_t)c + 1]);
            tptr[(size_t)c + 1] += tptr[(size_t)c];
        }
        std::vector<int> at(tptr.begin(), tptr.end());
        for (int k = 0; k < nblocks; k++) {
            const int w = at[(size_t)block_col[k]]++;
            trow[(size_t)w] = row[(size_t)k];
            tid[(size_t)w] = k;
            tat[(size_t)k] = w;
        }
        // For the gradient: the blocks, and two neighbours of a block row each, in an order in which those that run together
        // share what they read -- 8 block rows and 16 block columns at a time.
        std::vector<int> order((size_t)nblocks), pair;
        std::vector<std::pair<int, int>> two;
        for (int k = 0; k < nblocks; k++) order[(size_t)k] = k;
        for (int r = 0; r < brows; r++)
            for (int k = block_ptr[r]; k < block_ptr[r + 1]; k += 2) two.emplace_back(k, k + 1 < block_ptr[r + 1] ? k + 1 : -1);
        auto before = [&](int a, int b) {
            const int ra = row[(size_t)a], rb = row[(size_t)b], ca = block_col[a] / 16, cb = block_col[b] / 16;
            if (ra / 8 != rb / 8) return ra / 8 < rb / 8;
            if (ca != cb) return ca < cb;
            return ra != rb ? ra < rb : a < b;
        };
        std::sort(order.begin(), order.end(), before);
        std::sort(two.begin(), two.end(), [&](const std::pair<int, int> &a, const std::pair<int, int> &b) { return before(a.first, b.first); });
        for (const auto &t : two) { pair.push_back(t.first); pair.push_back(t.second); }
        m->npairs = (int)two.size();
        const std::vector<int> scale((size_t)nblocks, 127);
        auto up = [&](int **d, const int *h, size_t count) {
            if (dev_alloc(m, d, count)) return false;
            if (count) SPMV_HIP_TRY(hipMemcpy(*d, h, count * sizeof(int), hipMemcpyHostToDevice), return false);
            return true;
        };
        ok = up(&m->d_block_ptr, block_ptr, (size_t)brows + 1) && up(&m->d_block_col, block_col, (size_t)nblocks) &&
             up(&m->d_block_row, row.data(), (size_t)nblocks) && up(&m->d_bt_ptr, tptr.data(), (size_t)bcols + 1) &&
             up(&m->d_bt_row, trow.data(), (size_t)nblocks) && up(&m->d_bt_id, tid.data(), (size_t)nblocks) &&
             up(&m->d_order, order.data(), order.size()) && up(&m->d_pair, pair.data(), pair.size()) && up(&m->d_bt_at, tat.data(), (size_t)nblocks) && up(&m->d_scale8, scale.data(), (size_t)nblocks) &&
             up(&m->d_bt_scale8, scale.data(), (size_t)nblocks) && dev_alloc(m, &m->d_val8, (size_t)nblocks * kBlockBytes) == 0;
        if (ok && nblocks) {
            ok = hipMemset(m->d_val8, 0, (size_t)nblocks * kBlockBytes) == hipSuccess && hipDeviceSynchronize() == hipSuccess;
            if (!ok) set_error("clearing the blocks failed");
        }
    } catch (const std::bad_alloc &) { set_error("out of host memory"); ok = false; }
    if (!ok) { spmv_hip_free(m); return nullptr; }
    return m;
}

int spmv_hip_block8_set_values_dev(spmv_hip_matrix *m, const void *d_values, int dtype, void *stream)
{
    if (check_block8("block8_set_values", m)) return 1;
    if (!wide_dtype(dtype)) return bad_dtype("block8_set_values", dtype);
    if (m->nblocks == 0) return 0;
    if (!d_values) { set_error("block8_set_values: NULL values"); return 1; }
    DeviceGuard on(m->device);
    if (!on.ok) return 1;
    with_elem(dtype, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((set_values_kernel<T>), dim3(m->nblocks), dim3(kBlock), 0, (hipStream_t)stream, m->rows, m->columns,
                           m->d_block_row, m->d_block_col, (const T *)d_values, m->d_val8, m->d_bt_at, m->d_scale8, m->d_bt_scale8);
    });
    return launched("block8_set_values");
}

int spmv_hip_block8_load_dev(spmv_hip_matrix *m, const uint8_t *d_values8, const uint8_t *d_scale, void *stream)
{
    if (check_block8("block8_load", m)) return 1;
    if (m->nblocks == 0) return 0;
    if (!d_values8 || !d_scale) { set_error("block8_load: NULL argument"); return 1; }
    DeviceGuard on(m->device);
    if (!on.ok) return 1;
    hipLaunchKernelGGL(load8_kernel, dim3(m->nblocks), dim3(kBlock), 0, (hipStream_t)stream, m->rows, m->columns, m->d_block_row,
                       m->d_block_col, d_values8, d_scale, m->d_val8, m->d_bt_at, m->d_scale8, m->d_bt_scale8);
    return launched("block8_load");
}

int spmv_hip_block8_store_dev(const spmv_hip_matrix *m, uint8_t *d_values8, uint8_t *d_scale, void *stream)
{
    if (check_block8("block8_store", m)) return 1;
    if (m->nblocks == 0) return 0;
    if (!d_values8 || !d_scale) { set_error("block8_store: NULL argument"); return 1; }
    DeviceGuard on(m->device);
    if (!on.ok) return 1;
    hipLaunchKernelGGL(store8_kernel, dim3(m->nblocks), dim3(kBlock), 0, (hipStream_t)stream, m->d_val8, m->d_scale8, d_values8, d_scale);
    return launched("block8_store");
}

int spmv_hip_quantize8_dev(int n, int columns, const void *d_x, int dtype, int64_t ldx, uint8_t *d_x8, int64_t ldx8,
                           uint8_t *d_scale, int64_t lds, void *stream)
{
    if (!wide_dtype(dtype)) return bad_dtype("quantize8", dtype);
    if (columns < 0) { set_error("quantize8: negative length %d", columns); return 1; }
    if (check_vectors("quantize8", n, d_x, ldx, columns) || check_eight("quantize8", n, columns, d_x8, ldx8, d_scale, lds)) return 1;
    const int groups = groups_of(columns);
    if (n == 0 || groups == 0) return 0;
    const bool many = many_groups(n, groups);
    const int64_t grid = group_grid(n, groups, many ? 4 : 1);
    if (check_launch("quantize8", grid, kBlock)) return 1;
    with_elem(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kBlock), 0, (hipStream_t)stream, n, groups, columns, (const T *)d_x, ldx, d_x8, ldx8, d_scale, lds);
        };
        if (many) go(quantize8_kernel<T, 4>);
        else go(quantize8_kernel<T, 1>);
    });
    return launched("quantize8");
}

int spmv_hip_restore8_dev(int n, int columns, const uint8_t *d_x8, int64_t ldx8, const uint8_t *d_scale, int64_t lds,
                          void *d_x, int dtype, int64_t ldx, void *stream)
{
    if (!wide_dtype(dtype)) return bad_dtype("restore8", dtype);
    if (columns < 0) { set_error("restore8: negative length %d", columns); return 1; }
    if (check_vectors("restore8", n, d_x, ldx, columns) || check_eight("restore8", n, columns, d_x8, ldx8, d_scale, lds)) return 1;
    const int groups = groups_of(columns);
    if (n == 0 || groups == 0) return 0;
    const int64_t grid = group_grid(n, groups, 2);
    if (check_launch("restore8", grid, kBlock)) return 1;
    with_elem(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kBlock), 0, (hipStream_t)stream, n, groups, columns, d_x8, ldx8, d_scale, lds, (T *)d_x, ldx);
        };
        // Past the caches where the 256 MB of the last one would not hold both sides (16384 x 8192 of bf16: 57 us, 67 through
        // them), but not below (30000 x 1000 of fp32: 36 us, 24 through them)
        if ((int64_t)n * columns * (int64_t)(sizeof(T) + 1) > (int64_t)192 << 20) go(restore8_kernel<T, 2, true>);
        else go(restore8_kernel<T, 2, false>);
    });
    return launched("restore8");
}

int spmv_hip_block8_mult_dev(const spmv_hip_matrix *m, int n, const void *d_x, int x_dtype, int64_t ldx,
                             const uint8_t *d_scale, int64_t lds, void *d_y, int y_dtype, int64_t ldy, void *stream)
{
    const char *what = "block8_mult";
    if (check_block8(what, m)) return 1;
    if (!wide_dtype(y_dtype)) return bad_dtype(what, y_dtype);
    if (x_dtype == SPMV_HIP_E4M3) {
        if (check_eight(what, n, m->columns, d_x, ldx, d_scale, lds)) return 1;
    } else {
        if (!wide_dtype(x_dtype)) { set_error("%s: element type %d must be F32, BF16, F16 or E4M3", what, x_dtype); return 1; }
        if (check_vectors(what, n, d_x, ldx, m->columns)) return 1;
        if (d_scale) { set_error("%s: scales belong to vectors in 8 bits", what); return 1; }
        if (n > SPMV_HIP_BLOCK8_MAX_WIDE) {
            set_error("%s: %d wide vectors, at most %d are rounded inside the product (quantize8 first)", what, n, (int)SPMV_HIP_BLOCK8_MAX_WIDE);
            return 1;
        }
    }
    if (check_vectors(what, n, d_y, ldy, m->rows)) return 1;
    if (n == 0 || m->rows == 0) return 0;
    DeviceGuard on(m->device);
    if (!on.ok) return 1;
    // few vectors, or few tiles of many: there the strips, eight times as many, give the GPU more to do (fp32, 8192 x 1024, 128
    // vectors: 11 us, 21 in tiles; 32 tiles of 64 vectors 12 and 21 us, 64 tiles 22 and 22)
    if (x_dtype != SPMV_HIP_E4M3 || n <= 64 || (int64_t)m->brows * tiles_of(n, 64) * 8 <= m->cus)
        return launch_few(m, n, d_x, x_dtype, ldx, d_scale, lds, d_y, y_dtype, ldy, (hipStream_t)stream);
    ProductArgs a{};
    a.n = n; a.rows = m->rows; a.brows = m->brows;
    a.ptr = m->d_block_ptr; a.col = m->d_block_col; a.val8 = m->d_val8; a.scale8 = m->d_scale8;
    a.x8 = (const uint8_t *)d_x; a.xscale = d_scale; a.ldx8 = ldx; a.lds = lds; a.ldy = ldy;
    // With 4 tiles of vectors a wave, workgroups for every second CU are enough: they are two groups of waves then.
    const int nu = vector_tiles(m->brows, n, y_dtype == SPMV_HIP_BF16 ? 8 : 4, m->cus, m->cus / 2);
    a.vtiles = tiles_of(n, 32 * nu);
    const bool halves = nu < 8 && (int64_t)m->brows * a.vtiles <= m->cus && m->nblocks >= (int64_t)4 * m->brows;
    if (check_launch(what, (int64_t)m->brows * a.vtiles, (halves ? 2 : 1) * kBlock)) return 1;
    with_elem(y_dtype, [&](auto t) {
        typedef decltype(t) T;
        constexpr bool exact = !std::is_same<T, __bf16>::value;
        auto go = [&](auto kernel, int groups) {
            hipLaunchKernelGGL(kernel, dim3(m->brows * a.vtiles), dim3(groups * kBlock), 0, (hipStream_t)stream, a, (T *)d_y);
        };
        if constexpr (!exact) if (nu == 8) { go(product_kernel<exact, 8, 1, T>, 1); return; }
        if (nu == 4 && halves) go(product_kernel<exact, 4, 2, T>, 2);
        else if (nu == 4) go(product_kernel<exact, 4, 1, T>, 1);
        else if (halves) go(product_kernel<exact, 2, 2, T>, 2);
        else go(product_kernel<exact, 2, 1, T>, 1);
    });
    return launched(what);
}

int64_t spmv_hip_block8_backward_work(const spmv_hip_matrix *m, int n, const void *d_dy, int dy_dtype, int64_t lddy, int with_dx, int with_dvalues)
{
    if (!m || m->format != SPMV_HIP_BLOCK8 || !wide_dtype(dy_dtype)) return 0;
    return backward_plan(m, n, d_dy, dy_dtype, lddy, with_dx != 0, with_dvalues != 0).work;
}

int spmv_hip_block8_backward_dev(const spmv_hip_matrix *m, int n, const void *d_dy, int dy_dtype, int64_t lddy,
                                 const uint8_t *d_x8, int64_t ldx8, const uint8_t *d_scale, int64_t lds, void *d_dx, int dx_dtype,
                                 int64_t lddx, void *d_dvalues, int dv_dtype, int accumulate, void *d_work, void *stream)
{
    const char *what = "block8_backward";
    if (check_block8(what, m)) return 1;
    if (!wide_dtype(dy_dtype)) return bad_dtype(what, dy_dtype);
    if (check_vectors(what, n, d_dy, lddy, m->rows)) return 1;
    if (n > 1 && lddy >= (int64_t)1 << 23) {                  // 256 of them stay inside 32-bit offsets
        set_error("%s: vectors %lld apart, at most 2^23 - 1", what, (long long)lddy);
        return 1;
    }
    if (d_dx) {
        if (!wide_dtype(dx_dtype)) return bad_dtype(what, dx_dtype);
        if (check_vectors(what, n, d_dx, lddx, m->columns)) return 1;
    }
    if (d_dvalues) {
        if (!wide_dtype(dv_dtype)) return bad_dtype(what, dv_dtype);
        if (check_eight(what, n, m->columns, d_x8, ldx8, d_scale, lds)) return 1;
    }
    const BackwardPlan plan = backward_plan(m, n, d_dy, dy_dtype, lddy, d_dx != nullptr, d_dvalues != nullptr);
    if (plan.work && !d_work) {
        set_error("%s: NULL workspace, %lld bytes needed", what, (long long)plan.work);
        return 1;
    }
    if (plan.work && (uintptr_t)d_work % 16) { set_error("%s: workspace is not 16-byte aligned", what); return 1; }
    if (!d_dx && !d_dvalues) return 0;
    if (n == 1) lddy = m->rows;                               // bounds the loads; the caller's says nothing
    DeviceGuard on(m->device);
    if (!on.ok) return 1;
    const hipStream_t st = (hipStream_t)stream;
    // dy and the distance of its vectors for either product; bf16 parts are padded with zeros to whole blocks
    const void *dx_dy = d_dy, *dv_dy = d_dy;
    int64_t dx_ld = lddy, dv_ld = lddy, plane = 0;
    int dx_rows = m->rows, dv_rows = m->rows;
    if (plan.parts_bytes || plan.copy_bytes) {
        const int64_t wide = m->brows * (int64_t)kB;
        const int padded = (int)wide;
        plane = n * wide;
        if (wide >= 1 << 23 || (plane / 8 + kBlock - 1) / kBlock > 0xffffffffll / kBlock) { set_error("%s: %d vectors of %d are more than one launch takes", what, n, m->rows); return 1; }
        auto go = [&](auto kernel, auto *from, void *to) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((plane / 8 + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, n, m->rows, padded, from, lddy, (__bf16 *)to, plane);
        };
        if (plan.parts_bytes) {
            with_elem(dy_dtype, [&](auto t) {
                typedef decltype(t) T;
                go(split_kernel<T>, (const T *)d_dy, d_work);
            });
            dv_dy = d_work;
            dv_ld = dv_rows = padded;
            if (dy_dtype != SPMV_HIP_F16) { dx_dy = d_work; dx_ld = dx_rows = padded; }
        }
        if (plan.copy_bytes) {                                // 16 bits as they are
            void *to = (char *)d_work + plan.parts_bytes;
            go(split_kernel<__bf16>, (const __bf16 *)d_dy, to);
            dx_dy = to;
            dx_ld = dx_rows = padded;
        }
    }
    float *cut = (float *)((char *)d_work + plan.parts_bytes + plan.copy_bytes);     // slices of dx, then of dvalues
    auto with_parts = [&](auto f) {
        if (plan.dv_parts == 1) f(ic<1>());
        else if (plan.dv_parts == 2) f(ic<2>());
        else f(ic<3>());
    };
    if (d_dx && n > 0 && m->columns > 0) {
        TransposedArgs a{};
        a.n = n; a.rows = dx_rows; a.columns = m->columns; a.bcols = m->bcols;
        // In a full matrix all columns read the same of dy at the same time; in a pruned one, uneven, more of them keep each
        // other company (4096 vectors, 8192 x 8192, a quarter stored: 164 us with 8, 143 with 64; full 812 and 832)
        a.side = (int64_t)m->nblocks * 4 >= (int64_t)m->brows * m->bcols * 3 ? 8 : 64;
        a.ptr = m->d_bt_ptr; a.row = m->d_bt_row; a.id = m->d_bt_id; a.val8 = m->d_val8; a.scale = m->d_bt_scale8;
        a.dy = dx_dy; a.lddy = dx_ld; a.plane = plane; a.slice = plan.dx_slice;
        const int nu = plan.tiles;
        a.vtiles = tiles_of(n, 32 * nu);
        if (check_launch(what, (int64_t)m->bcols * a.vtiles, (plan.dx_halves ? 2 : 1) * kBlock)) return 1;
        auto into = [&](auto *to, int64_t ld) {
            typedef std::remove_pointer_t<decltype(to)> O;
            a.lddx = ld;
            auto go = [&](auto kernel, int groups) {
                hipLaunchKernelGGL(kernel, dim3(m->bcols * a.vtiles, plan.dx_slices), dim3(groups * kBlock), 0, st, a, to);
            };
            auto tiles = [&](auto e) {
                typedef decltype(e) E;
                if (nu == 8) go(transposed_kernel<E, 1, 8, 1, O>, 1);
                else if (nu == 4) go(transposed_kernel<E, 1, 4, 1, O>, 1);
                else if (plan.dx_halves) go(transposed_kernel<E, 1, 2, 2, O>, 2);
                else go(transposed_kernel<E, 1, 2, 1, O>, 1);
            };
            if (dy_dtype == SPMV_HIP_F16) tiles(_Float16());
            else if (dy_dtype == SPMV_HIP_BF16) tiles(__bf16());
            else if (plan.dx_halves) go(transposed_kernel<__bf16, 3, 2, 2, O>, 2);
            else go(transposed_kernel<__bf16, 3, 2, 1, O>, 1);
        };
        with_elem(dx_dtype, [&](auto o) {
            typedef decltype(o) O;
            if (plan.dx_slices == 1) { into((O *)d_dx, lddx); return; }
            into(cut, m->bcols * (int64_t)kB);
            launch_join(n, m->bcols * (int64_t)kB, m->columns, plan.dx_slices, cut, (O *)d_dx, lddx, 0, st);
        });
    }
    if (d_dvalues && m->nblocks > 0) {
        GradientArgs a{};
        a.n = n; a.rows = dv_rows; a.edge = m->rows; a.columns = m->columns;
        a.block_row = m->d_block_row; a.block_col = m->d_block_col;
        a.x8 = d_x8; a.xscale = d_scale; a.ldx8 = ldx8; a.lds = lds; a.dy = (const __bf16 *)dv_dy; a.lddy = dv_ld; a.plane = plane; a.slice = plan.dv_slice;
        a.list = plan.pairs ? m->d_pair : m->d_order;
        auto into = [&](auto *to, int add) {
            typedef std::remove_pointer_t<decltype(to)> O;
            a.accumulate = add;
            with_parts([&](auto p) {
                constexpr int P = decltype(p)::value;
                auto go = [&](auto kernel, int wgs, int groups) {
                    hipLaunchKernelGGL(kernel, dim3(wgs, plan.dv_slices), dim3(groups * kBlock), 0, st, a, to);
                };
                if (plan.pairs) go(gradient_kernel<P, 2, 1, O>, m->npairs, 1);
                else if (plan.dv_halves) go(gradient_kernel<P, 1, 2, O>, m->nblocks, 2);
                else go(gradient_kernel<P, 1, 1, O>, m->nblocks, 1);
            });
        };
        with_elem(dv_dtype, [&](auto o) {
            typedef decltype(o) O;
            if (plan.dv_slices == 1) { into((O *)d_dvalues, accumulate); return; }
            into(cut, 0);
            launch_join(m->nblocks, (int64_t)kBlockBytes, kBlockBytes, plan.dv_slices, cut, (O *)d_dvalues, (int64_t)kBlockBytes, accumulate, st);
        });
    }
    return launched(what);
}

} // extern "C"
