// int8 operators with a scale for each token and channel.
//
//   quantise     a = max(max_k |x_k|, 2^-100), s = fl(a / 127), r = fl(127 / a), q = rint(x r)
//   product      y_ij = relu(fma(fl(fl(sum_k q_ik w_jk) s_i), t_j, b_j)), rounded to its type
//   requantise   the product's rows in 32 bits, quantised as above or by one given scale
//
// Sums of products are whole numbers below 2^31 (k <= 131,071) and exact in int32, so a result
// does not depend on the kernel, the tile or the split of K that computed it; the roundings
// after the sum are fixed above.  A decoder that works token by token therefore reproduces what
// an encoder computed in batches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "sc_internal.h"
#include "sc_int8.h"
#include "sc_tc.cuh"

namespace sc {
namespace {

// ---- launches that overlap the end of the one before ------------------------------------------
// Every kernel here is launched so that it may start while the kernel before it in the stream ends.  All
// its threads wait for that kernel's results before they touch global memory, so the set-up alone
// overlaps, and no kernel ends before the one before it has.
__device__ __forceinline__ void previous_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- element types ---------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- a row's scale ---------------------------------------------------------------------------
// Magnitudes are compared as bit patterns: for floats without their sign the order of the bits is
// the order of the values, infinity and NaN above all others, so one whole-number maximum also
// tells whether the row holds a value that cannot be quantised.
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr uint32_t kSmallestBits = 0x0d800000u;      // 2^-100: 127 / a stays finite

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
    float s, r;          // scale and reciprocal; both zero when the row cannot be quantised
    bool finite;
};

__device__ __forceinline__ RowScale row_scale(uint32_t top)
{
    RowScale o;
    o.finite = top < kInfBits;
    const float a = __uint_as_float(max(top, kSmallestBits));
    o.s = __fdiv_rn(a, 127.0f);
    o.r = __fdiv_rn(127.0f, a);
    return o;
}

// rint(v r) in the low byte.  The sum with 1.5 * 2^23 has a unit in the last place of one, so the
// fused multiply-add rounds the exact product to a whole number, ties to even, in one rounding.
// |v r| <= 127 (1 + 2^-24), so nothing saturates.
constexpr float kMagic = 12582912.0f;
__device__ __forceinline__ uint32_t quantise_bits(float v, float r) { return __float_as_uint(__fmaf_rn(v, r, kMagic)); }

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// A vector of 16 bytes of a row, kept as it was read: the row is converted where it is used, which
// halves the registers of 16-bit types and takes their magnitudes two at a time.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ uint32_t top(const uint4 &r, uint32_t m)
    {
        return max(max(m, max(r.x & 0x7fffffffu, r.y & 0x7fffffffu)), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
    }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return m; }
    static __device__ __forceinline__ void quantise(const uint4 &v, float r, uint32_t (&o)[1])
    {
        o[0] = pack4(quantise_bits(__uint_as_float(v.x), r), quantise_bits(__uint_as_float(v.y), r),
                     quantise_bits(__uint_as_float(v.z), r), quantise_bits(__uint_as_float(v.w), r));
    }
};
template <typename T> struct Vec16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint32_t top(const uint4 &r, uint32_t m)
    {
        m = __vmaxu2(m, __vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu));
        return __vmaxu2(m, __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
    }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t m)
    {
        const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
        return __float_as_uint(to_f32<T>(*reinterpret_cast<const T *>(&h)));
    }
    static __device__ __forceinline__ void quantise(const uint4 &v, float r, uint32_t (&o)[2])
    {
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            o[i] = pack4(quantise_bits(to_f32<T>(e[4 * i]), r), quantise_bits(to_f32<T>(e[4 * i + 1]), r),
                         quantise_bits(to_f32<T>(e[4 * i + 2]), r), quantise_bits(to_f32<T>(e[4 * i + 3]), r));
    }
};
template <> struct Vec<__half> : Vec16<__half> {};
template <> struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16> {};

// 16 bytes from byte `at` (0 to 15, a multiple of E) of 32
template <int E>
__device__ __forceinline__ uint4 shifted16(const uint4 &a, const uint4 &b, uint32_t at)
{
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = at & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = at & 4 ? w[i + 1] : w[i];
    if (E == 4) return make_uint4(w[0], w[1], w[2], w[3]);
    const uint32_t bits = (at & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// 16 bytes if `in`, else zeros: a predicated load and no branch, so that several are in flight
__device__ __forceinline__ uint4 load_if(bool in, const void *at)
{
    uint4 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at), "r"((int)in) : "memory");
    return v;
}

// Element by element what lies within low .. high, zeros in place of the rest
template <typename T>
__device__ __forceinline__ uint4 load_elements(const T *at, const T *low, const T *high)
{
    uint4 raw = make_uint4(0, 0, 0, 0);
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
        if (at + i >= low && at + i < high) e[i] = at[i];
    return raw;
}

// the first `bytes` of 16, zeros behind them
__device__ __forceinline__ uint4 first_bytes(uint4 v, int bytes)
{
    auto keep = [&](uint32_t w, int from) {
        const int n = bytes - from;
        return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
    };
    return make_uint4(keep(v.x, 0), keep(v.y, 4), keep(v.z, 8), keep(v.w, 12));
}

// ---- quantise --------------------------------------------------------------------------------
// A row is read once: THREADS threads (a part of a warp, a warp or more) hold its 16-byte vectors in registers through
// the maximum, R rows at a time where rows are short, so that enough loads are in flight.  Bound by HBM
// (e + 1 bytes per element): 262,144 x 512 fp16 in 61 us, 6.6 TB/s; 20,480 x 8,192 bf16 in 74 us, 6.8 TB/s.  Rows of 511
// at any address: 112 us, bound by the instructions that shift them.
template <typename T, int THREADS, int HELD, int R, bool ALIGNED>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
k_quantize(const T *__restrict__ x, int64_t rows, int cols, int64_t x_stride, int8_t *__restrict__ q, int64_t q_stride,
           float *__restrict__ scales, int q_vec)
{
    constexpr int N = Vec<T>::N;
    constexpr int GROUPS = THREADS < 256 ? 256 / THREADS : 1;      // of THREADS threads, R rows each
    __shared__ uint32_t tops[R][32];
    const int t = threadIdx.x % THREADS, grp = threadIdx.x / THREADS;
    const int64_t row0 = ((int64_t)blockIdx.x * GROUPS + grp) * R;
    const T *end = x + (rows - 1) * x_stride + cols;
    next_may_start();
    previous_done();
    // Aligned vectors are requested first, all of them; where rows do not start on 16 bytes (ALIGNED false) a thread has
    // the one that holds its first column and gets the next from its neighbour, and the last thread of a warp
    // or part reads that too.  Only addresses within x are read: at its ends element by element.
    constexpr int LANES = THREADS < 32 ? THREADS : 32;
    const bool last = (threadIdx.x & (LANES - 1)) == LANES - 1;
    uint4 v[R][HELD], w[ALIGNED ? 1 : R][ALIGNED ? 1 : HELD];
    uint32_t top[R], at[R];
    const T *from[R];
    int low[R], high[R];                                           // the vectors of a row that lie in x: low to high - 1
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const T *row = x + min(row0 + i, rows - 1) * x_stride;
        at[i] = ALIGNED ? 0 : (uint32_t)(uintptr_t)row & 15u;
        from[i] = reinterpret_cast<const T *>(reinterpret_cast<const char *>(row) - at[i]) + t * N;
        const int live = row0 + i < rows ? cols : -2 * N;          // behind the last row: a row of no columns
        if (!ALIGNED) {
            low[i] = from[i] - t * N < x;
            high[i] = (int)min((int64_t)INT_MAX, (int64_t)(end - (from[i] - t * N)) / N);
        }
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int g = h * THREADS + t, c = g * N;
            v[i][h] = load_if(ALIGNED ? c + N <= live : g >= low[i] && g < high[i] && c < live + N, from[i] + h * THREADS * N);
            if (!ALIGNED) w[i][h] = load_if(last && g + 1 < high[i] && c < live, from[i] + (h * THREADS + 1) * N);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int live = row0 + i < rows ? cols : -2 * N;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int g = h * THREADS + t, c = g * N;
            const T *p = from[i] + h * THREADS * N;
            if (ALIGNED) {
                if (c < live && c + N > live) v[i][h] = load_elements(p, p, p + (live - c));
            } else {
                if ((g < low[i] || g >= high[i]) && c < live + N) v[i][h] = load_elements(p, x, end);
                if (last && g + 1 >= high[i] && c < live) w[i][h] = load_elements(p + N, x, end);
                const uint4 o = v[i][h];
                uint4 next = make_uint4(__shfl_down_sync(0xffffffffu, o.x, 1, LANES), __shfl_down_sync(0xffffffffu, o.y, 1, LANES),
                                        __shfl_down_sync(0xffffffffu, o.z, 1, LANES), __shfl_down_sync(0xffffffffu, o.w, 1, LANES));
                if (last) next = w[i][h];
                v[i][h] = shifted16<sizeof(T)>(o, next, at[i]);
                if (c + N > live) v[i][h] = first_bytes(v[i][h], (live - c) * (int)sizeof(T));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h) m = Vec<T>::top(v[i][h], m);
        m = Vec<T>::top_bits(m);
        if (THREADS >= 32) {
            top[i] = __reduce_max_sync(0xffffffffu, m);
            if (THREADS > 32 && (threadIdx.x & 31) == 0) tops[i][threadIdx.x >> 5] = top[i];
        } else {
#pragma unroll
            for (int d = 1; d < THREADS; d *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
            top[i] = m;
        }
    }
    if (THREADS > 32) {
        __syncthreads();
        const int w = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < R; ++i)
            top[i] = __reduce_max_sync(0xffffffffu, w < THREADS / 32 ? tops[i][grp * (THREADS / 32) + w] : 0u);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (row0 + i >= rows) break;
        const RowScale rs = row_scale(top[i]);
        if (t == 0) scales[row0 + i] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
        int8_t *qr = q + (row0 + i) * q_stride;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int c = (h * THREADS + t) * N;
            uint32_t o[N / 4];
            Vec<T>::quantise(v[i][h], rs.r, o);
            if (!rs.finite)
#pragma unroll
                for (int j = 0; j < N / 4; ++j) o[j] = 0;
            if (q_vec && c + N <= cols) {
                if constexpr (N == 8) *reinterpret_cast<uint2 *>(qr + c) = make_uint2(o[0], o[1]);
                else *reinterpret_cast<uint32_t *>(qr + c) = o[0];
            } else if (q_vec) {                                    // the row's last bytes: four, two and one of them
                int n = cols - c;
                if (n >= 4) {
                    *reinterpret_cast<uint32_t *>(qr + c) = o[0];
                    o[0] = o[N / 4 - 1];
                }
                if (n > 0 && n & 2) {
                    *reinterpret_cast<uint16_t *>(qr + c + (n & 4)) = (uint16_t)o[0];
                    o[0] >>= 16;
                }
                if (n > 0 && n & 1) qr[c + (n & 6)] = (int8_t)o[0];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (c + j < cols) qr[c + j] = (int8_t)(o[j / 4] >> (8 * (j % 4)));
            }
        }
    }
}

// Rows longer than a block holds: read twice, the second time mostly from L2.
template <typename T>
__global__ void __launch_bounds__(1024)
k_quantize_long(const T *__restrict__ x, int cols, int64_t x_stride, int8_t *__restrict__ q, int64_t q_stride,
                float *__restrict__ scales)
{
    __shared__ uint32_t tops[32];
    const T *xr = x + (int64_t)blockIdx.x * x_stride;
    next_may_start();
    previous_done();
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) top = max(top, magnitude(to_f32<T>(xr[c])));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[threadIdx.x & 31]);
    const RowScale rs = row_scale(top);
    if (threadIdx.x == 0) scales[blockIdx.x] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
    int8_t *qr = q + (int64_t)blockIdx.x * q_stride;
    for (int64_t c = threadIdx.x; c < cols; c += 1024)
        qr[c] = rs.finite ? (int8_t)quantise_bits(to_f32<T>(xr[c]), rs.r) : 0;
}

// ---- dequantise ------------------------------------------------------------------------------
// 16 bytes of results a thread and row, four rows in flight: a block's 256 threads are 2^log_lanes
// vectors wide.  Bound by HBM (1 + e bytes per element): 262,144 x 512 to fp16 in 62 us, 6.5 TB/s.  Where y's rows do not start on 16 bytes (ALIGNED false), a
// row's vectors are those of the addresses, so the first one and the last may be parts, and their bytes
// of q are read as the three words around them.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256)
k_dequantize(const int8_t *__restrict__ q, int64_t q_stride, const float *__restrict__ scales, float scale, int64_t rows,
             int cols, T *__restrict__ y, int64_t y_stride, int log_lanes, int q_words)
{
    constexpr int N = Vec<T>::N, U = 4;
    const int deep = 256 >> log_lanes;                             // rows of one pass
    const int64_t row0 = (int64_t)blockIdx.x * deep * U + (threadIdx.x >> log_lanes);
    const int lane = threadIdx.x & ((1 << log_lanes) - 1);
    next_may_start();
    previous_done();
    for (int64_t c64 = ((int64_t)blockIdx.y << log_lanes) * N; c64 < cols + (ALIGNED ? 0 : N - 1);
         c64 += ((int64_t)gridDim.y << log_lanes) * N) {
        int c[U];
        uint32_t raw[U][N / 4];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row0 + u * deep;
            c[u] = (int)c64 + lane * N;
            if (r >= rows) continue;
            const int8_t *qr = q + r * q_stride;
            s[u] = scales ? scales[r] : scale;
            if (!ALIGNED) c[u] -= (int)(((uintptr_t)(y + r * y_stride) & 15) / sizeof(T));
            const bool whole = c[u] >= 0 && c[u] + N <= cols;
            if (ALIGNED && whole) {
                if constexpr (N == 8) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(qr + c[u]);
                    raw[u][0] = v.x, raw[u][N / 4 - 1] = v.y;
                } else raw[u][0] = *reinterpret_cast<const uint32_t *>(qr + c[u]);
            } else if (!ALIGNED && q_words && whole && (r + 1 < rows || c[u] + N + 4 <= cols)) {
                // the words may reach four bytes behind the vector, which lie in q but at its very end
                const uint32_t *at = reinterpret_cast<const uint32_t *>(qr + (c[u] & ~3));
                uint32_t w[N / 4 + 1];
#pragma unroll
                for (int i = 0; i <= N / 4; ++i) w[i] = at[i];
#pragma unroll
                for (int i = 0; i < N / 4; ++i) raw[u][i] = __funnelshift_r(w[i], w[i + 1], (c[u] & 3) * 8);
            } else {
                uint32_t b[N];
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = c[u] + i >= 0 && c[u] + i < cols ? (uint32_t)(uint8_t)qr[c[u] + i] : 0;
#pragma unroll
                for (int i = 0; i < N / 4; ++i) raw[u][i] = pack4(b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row0 + u * deep;
            if (r >= rows) continue;
            T *yr = y + r * y_stride;
            __align__(16) T out[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                out[i] = from_f32<T>(__fmul_rn((float)(int8_t)(raw[u][i / 4] >> (8 * (i % 4))), s[u]));
            if (c[u] >= 0 && c[u] + N <= cols) {
                *reinterpret_cast<uint4 *>(yr + c[u]) = *reinterpret_cast<const uint4 *>(out);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (c[u] + i >= 0 && c[u] + i < cols) yr[c[u] + i] = out[i];
            }
        }
    }
}

// ---- product ---------------------------------------------------------------------------------
// Roundings of one result, see the head of this file.  max.NaN keeps a NaN that the scale carries.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ float affine(int32_t acc, float s, float t, float b, int relu)
{
    const float y = __fmaf_rn(__fmul_rn(__int2float_rn(acc), s), t, b);
    return relu ? max_nan(y, 0.0f) : y;
}

// sat(rint(y / scale)) in the low byte; a NaN becomes 0
__device__ __forceinline__ uint32_t static_bits(float y, float scale)
{
    int32_t o;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(o) : "f"(__fdiv_rn(y, scale)));
    return (uint32_t)o & 0xffu;
}

__device__ __forceinline__ uint32_t static_bits(uint32_t y, float least, float scale)
{
    const float v = __uint_as_float(y);
    return static_bits(least == 0.0f ? max_nan(v, 0.0f) : v, scale);
}

// The same for 32 results, after ReLU where `least` is 0 and not -128: y times the rounded reciprocal is within 2.3e-5 of
// y / scale below 128, so only a product that close to a half, or one that is no number, needs the division
// (about one of 17,000), and then all 32 are divided.  usual: whether the reciprocal is that near.
__device__ __forceinline__ void static32(const uint32_t (&y)[32], float scale, float inv, bool usual, float least,
                                         uint32_t (&o)[8])
{
    bool exact = usual;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = __fmul_rn(__uint_as_float(y[4 * i + j]), inv);
            float c;
            asm("max.NaN.f32 %0, %1, %2;\n\tmin.NaN.f32 %0, %0, 0f42FE0000;" : "=&f"(c) : "f"(t), "f"(least));     // 127
            const float v = __fadd_rn(c, kMagic), d = __fsub_rn(c, __fsub_rn(v, kMagic));
            exact = exact && fabsf(d) <= 0.49997f;
            b[j] = __float_as_uint(v);
        }
        o[i] = pack4(b[0], b[1], b[2], b[3]);
    }
    if (!exact) {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            uint32_t w = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k == i)
                    w = pack4(static_bits(y[4 * k], least, scale), static_bits(y[4 * k + 1], least, scale),
                              static_bits(y[4 * k + 2], least, scale), static_bits(y[4 * k + 3], least, scale));
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k == i) o[k] = w;
        }
    }
}

}  // namespace
}  // namespace sc

#include "sc_int8_mm.cuh"
#include "sc_int8_token.cuh"

namespace sc {
namespace {

// ---- host side -------------------------------------------------------------------------------

// Rows copied to a multiple of 16 bytes apart, for arrays that TMA cannot read as they lie.  Bytes behind
// a row's end stay as they are: the tensor map ends with the row.
__global__ void __launch_bounds__(256)
k_spread(const int8_t *__restrict__ x, int64_t rows, int cols, int64_t x_stride, int8_t *__restrict__ y, int64_t y_stride)
{
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    next_may_start();
    previous_done();
    if (row >= rows) return;
    const int8_t *xr = x + row * x_stride;
    for (int c = (threadIdx.x & 31) * 4; c < cols; c += 128) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) v |= (uint32_t)(uint8_t)xr[c + i] << (8 * i);
        *reinterpret_cast<uint32_t *>(y + row * y_stride + c) = v;
    }
}

bool aligned(const void *p, int64_t stride_bytes, int a)
{
    return ((uintptr_t)p % a) == 0 && stride_bytes % a == 0;
}

unsigned grid_x(int64_t blocks)
{
    if (blocks > INT_MAX) throw CudaError{cudaErrorInvalidValue, "too many rows for one launch"};
    return (unsigned)blocks;
}

template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, unsigned cluster, A... args)
{
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    SC_CUDA(cudaLaunchKernelEx(&cfg, kernel, (P)args...));
    count_launch();
}

// SMs that plans count on (a B200's), so that a plan and its workspace do not depend on the current device.
constexpr int kSms = 148;

int sm_count()
{
    static std::atomic<int> counts[64];
    int dev = 0, n = 0;
    SC_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && (n = counts[dev].load(std::memory_order_relaxed)) > 0) return n;
    SC_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) counts[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <typename T, int THREADS, int HELD, int R>
void launch_quantize(const T *x, int64_t rows, int cols, int64_t xs, int8_t *q, int64_t qs, float *scales, cudaStream_t s)
{
    constexpr int PER_BLOCK = (THREADS < 256 ? 256 / THREADS : 1) * R;
    const unsigned g = grid_x((rows + PER_BLOCK - 1) / PER_BLOCK), b = THREADS < 256 ? 256 : THREADS;
    const int q_vec = aligned(q, qs, Vec<T>::N);
    if (aligned(x, xs * (int64_t)sizeof(T), 16))
        launch(k_quantize<T, THREADS, HELD, R, true>, g, b, 0, s, 1, x, rows, cols, xs, q, qs, scales, q_vec);
    else
        launch(k_quantize<T, THREADS, HELD, R, false>, g, b, 0, s, 1, x, rows, cols, xs, q, qs, scales, q_vec);
}

template <typename T>
void quantize(const T *x, int64_t rows, int cols, int64_t xs, int8_t *q, int64_t qs, float *scales, cudaStream_t s)
{
    const int vecs = (cols + Vec<T>::N - 1) / Vec<T>::N;
    // few rows: one vector a thread, so that a row's latency is one load's
    const bool few = rows <= 2 * kSms;
    if (vecs <= 1) launch_quantize<T, 1, 1, 4>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 4) launch_quantize<T, 4, 1, 4>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 8) launch_quantize<T, 8, 1, 4>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 16) launch_quantize<T, 16, 1, 4>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 32) launch_quantize<T, 32, 1, 4>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 64 && !few) launch_quantize<T, 32, 2, 2>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 128 && !few) launch_quantize<T, 32, 4, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 128) launch_quantize<T, 128, 1, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 256 && !few) launch_quantize<T, 128, 2, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 512 && !few) launch_quantize<T, 128, 4, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 256 && few) launch_quantize<T, 256, 1, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 1024 && few) launch_quantize<T, 1024, 1, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 1024) launch_quantize<T, 256, 4, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 2048) launch_quantize<T, 512, 4, 1>(x, rows, cols, xs, q, qs, scales, s);
    else if (vecs <= 4096) launch_quantize<T, 1024, 4, 1>(x, rows, cols, xs, q, qs, scales, s);
    else launch(k_quantize_long<T>, grid_x(rows), 1024, 0, s, 1, x, cols, xs, q, qs, scales);
}

template <typename T>
void dequantize(const int8_t *q, int64_t qs, const float *scales, float scale, int64_t rows, int cols, T *y, int64_t ys,
                cudaStream_t s)
{
    constexpr int N = Vec<T>::N;
    const bool al = aligned(q, qs, N) && aligned(y, ys * (int64_t)sizeof(T), 16);
    const int wide_cols = al ? cols : cols + N - 1;             // a row's vectors may begin before it
    // as wide as a row, or of the widths from a warp's up the one that leaves the fewest lanes behind its end
    int log_lanes = 0;
    while (log_lanes < 8 && (N << log_lanes) < wide_cols) ++log_lanes;
    auto behind = [&](int l) { return ((int64_t)wide_cols + (N << l) - 1) / (N << l) * (N << l); };
    for (int l = log_lanes - 1; l >= 5; --l)
        if (behind(l) < behind(log_lanes)) log_lanes = l;
    const int64_t deep = (256 >> log_lanes) * 4, wide = (int64_t)N << log_lanes;
    const dim3 g(grid_x((rows + deep - 1) / deep), (unsigned)std::min<int64_t>((wide_cols + wide - 1) / wide, 65535));
    if (al) launch(k_dequantize<T, true>, g, 256, 0, s, 1, q, qs, scales, scale, rows, cols, y, ys, log_lanes, 1);
    else
        launch(k_dequantize<T, false>, g, 256, 0, s, 1, q, qs, scales, scale, rows, cols, y, ys, log_lanes,
               (int)(aligned(q, qs, 4) && qs >= cols));
}

struct Rows8 {
    const int8_t *p;
    int64_t stride;
};

// The kernel's shared memory limit (and clusters of 16), set once per device.
template <typename F>
void allow_smem(F *kernel, int bytes, std::atomic<uint64_t> &done, bool wide_cluster = false)
{
    int dev = 0;
    SC_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
    SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (wide_cluster) SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename T> constexpr CUtensorMapDataType map_type();
template <> constexpr CUtensorMapDataType map_type<float>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT32; }
template <> constexpr CUtensorMapDataType map_type<__half>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }
template <> constexpr CUtensorMapDataType map_type<__nv_bfloat16>() { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }
template <> constexpr CUtensorMapDataType map_type<int8_t>() { return CU_TENSOR_MAP_DATA_TYPE_UINT8; }

// y (T; int8: requantised with a scale for each row, at most 512 channels) of int8 rows, on SM pairs
template <typename T, int MODE>
void product_pairs(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, T *y, int64_t y_stride, cudaStream_t s,
                   uint32_t *tops = nullptr)
{
    static std::atomic<uint64_t> ready{0};
    allow_smem(k_pair<T, MODE>, P_SMEM, ready);
    PairParams a;
    a.x = tensor_map(x.p, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.k, p.rows, x.stride, PK, PM);
    a.w = tensor_map(w.p, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.k, p.n, w.stride, PK, PN / 2);
    a.y_tma = aligned(y, y_stride * (int64_t)sizeof(T), 16);
    if (a.y_tma) a.y = tensor_map(y, map_type<T>(), p.n, p.rows, y_stride * sizeof(T), 128 / sizeof(T), 32);
    a.xs = xs;
    a.ws = p.w_scales;
    a.bias = p.bias;
    a.rows = p.rows;
    a.n = (int)p.n;
    a.k = (int)p.k;
    a.relu = p.relu;
    a.yp = y;
    a.y_stride = y_stride;
    a.y_scales = p.y_scales;
    a.output_scale = p.output_scale;
    a.tops = tops;
    const int64_t tiles = (p.rows + 2 * PM - 1) / (2 * PM), units = (p.n + PN - 1) / PN;
    const int64_t work = MODE == ROWS ? tiles : tiles * units;
    const unsigned pairs = (unsigned)std::min<int64_t>(work, sm_count() / 2);
    launch(k_pair<T, MODE>, 2 * pairs, P_THREADS, P_SMEM, s, 2, a);
}

// y of few int8 rows: float types, int8 by one scale, or (ROWS_OUT) int8 with a scale for each row; BT tokens per
// tile, K split over `split` CTAs
template <int BT, bool ROWS_OUT, typename T>
void launch_few(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, T *y, int64_t y_stride, int split, cudaStream_t s)
{
    using C = FewCfg<BT>;
    static std::atomic<uint64_t> ready{0};
    allow_smem(k_few<BT, T, ROWS_OUT>, C::SMEM, ready, ROWS_OUT);
    FewParams a;
    a.w = tensor_map(w.p, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.k, p.n, w.stride, PK, 128);
    a.x = tensor_map(x.p, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.k, p.rows, x.stride, PK, BT);
    a.xs = xs;
    a.ws = p.w_scales;
    a.bias = p.bias;
    a.rows = p.rows;
    a.n = (int)p.n;
    a.k = (int)p.k;
    a.relu = p.relu;
    a.y = y;
    a.y_stride = y_stride;
    a.y_vec = aligned(y, y_stride * (int64_t)sizeof(T), 4 * sizeof(T));
    a.output_scale = p.output_scale;
    a.y_scales = p.y_scales;
    a.split = split;
    const unsigned tiles = (unsigned)((p.n + 127) / 128), deep = (unsigned)((p.rows + BT - 1) / BT);
    const unsigned cluster = ROWS_OUT ? tiles * split : split;
    launch(k_few<BT, T, ROWS_OUT>, dim3(cluster, ROWS_OUT ? 1 : tiles, deep), C::THREADS, C::SMEM, s, cluster, a);
}

template <int BT>
void product_few(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, void *y, int y_type, int64_t y_stride, int split,
                 cudaStream_t s)
{
    if (y_type == SC_TYPE_F32) launch_few<BT, false>(p, x, xs, w, (float *)y, y_stride, split, s);
    else if (y_type == SC_TYPE_F16) launch_few<BT, false>(p, x, xs, w, (__half *)y, y_stride, split, s);
    else if (y_type == SC_TYPE_BF16) launch_few<BT, false>(p, x, xs, w, (__nv_bfloat16 *)y, y_stride, split, s);
    else launch_few<BT, false>(p, x, xs, w, (int8_t *)y, y_stride, split, s);
}

// How one or two rows run on k_token; per_cta = 0 where they do not.
struct TokenPlan {
    int per_cta, log_s, ctas;
};

TokenPlan token_plan(int64_t rows, int64_t n, int64_t k)
{
    TokenPlan t{0, 0, 0};
    if (rows > 2) return t;
    const int target = 2 * kSms;
    // a warp for four channels, or several, down to one 512-byte step of K each, while warps are few
    while (t.log_s < 3 && (n << t.log_s) < (int64_t)target * TK_WARPS * TK_CH && (512 << t.log_s) < k) ++t.log_s;
    const int abreast = (TK_WARPS >> t.log_s) * TK_CH;
    const int64_t per = ((n + target - 1) / target + abreast - 1) / abreast * abreast;
    // two CTAs to an SM
    if (per > 4096 || token_smem((int)rows, (int)k, (int)per, t.log_s) > TK_SMEM) return t;
    t.per_cta = (int)per;
    t.ctas = (int)((n + per - 1) / per);
    return t;
}

template <typename X, int MT>
void launch_token(const TokenParams &a, const TokenPlan &t, cudaStream_t s)
{
    static std::atomic<uint64_t> ready{0};
    allow_smem(k_token<X, MT>, TK_SMEM, ready);
    launch(k_token<X, MT>, (unsigned)t.ctas, TK_THREADS, (size_t)token_smem(MT, a.k, t.per_cta, t.log_s), s, 1, a);
}

template <typename X>
void product_token(const TokenParams &a, const TokenPlan &t, cudaStream_t s)
{
    if (a.rows == 1) launch_token<X, 1>(a, t, s);
    else launch_token<X, 2>(a, t, s);
}

// Clusters of k_few, one CTA to an SM, that fit a B200 at once (cudaOccupancyMaxActiveClusters; a cluster lies
// within a group of 14 to 20 SMs).
int cluster_room(int ctas)
{
    return ctas == 1 ? 148 : ctas == 2 ? 74 : ctas == 3 ? 45 : ctas == 4 ? 33 : ctas == 5 ? 26 : ctas == 6 ? 22
           : ctas <= 9 ? 15 : ctas == 10 ? 11 : 7;
}

// What multiplies a number of rows: the kernel, its tile and split, whether the rows are quantised by a launch of
// their own, and the time in microseconds that it is expected to take.
struct Way {
    enum { TOKEN = SC_INT8_TOKEN, FEW = SC_INT8_FEW, FEW_ROWS = SC_INT8_FEW_ROWS, PAIRS = SC_INT8_PAIRS,
           PAIRS_ROWS = SC_INT8_PAIRS_ROWS, PAIRS_TWICE = SC_INT8_PAIRS_TWICE } kernel;
    int bt, split;
    TokenPlan t;
    bool requant;
    double time;
};

// The way that is expected to take least.  The times are so many waves of CTAs, each of them a start and an end plus
// its K blocks, and about 2 us for a launch that quantises rows; fitted to measurements.  At 1 to 20,480 rows of
// seven layers (512 x 256 to 4,096 x 4,096) calls take 0.74 to 1.40 times what is expected, 1.02 in the median.  Among
// them, k_few against k_pair:
//   K = 512, N = 512:     16 rows 3.4 / 5.9,  1,000 rows 4.5 / 6.5,  3,000 rows 7.9 / 6.2
//   K = 8,192, N = 512:   16 rows 5.2 / 22,  1,000 rows 12.1 / 23,  3,000 rows 24.1 / 22.8
//   K = 4,096, N = 4,096: 16 rows 6.0 / 13.8,  400 rows 15.8 / 14.4,  1,000 rows 29.9 / 15.3
// and, requantised, one launch against two: 16 rows of 512 x 512 3.8 / 5.9, of 8,192 x 512 9.1 / 6.3.
Way choose(int64_t rows, int64_t n, int64_t k, bool rows_out)
{
    const int64_t nkb = (k + PK - 1) / PK, pairs = kSms / 2;
    const int64_t tiles = (rows + 2 * PM - 1) / (2 * PM), blocks = (n + PN - 1) / PN, channels = (n + 127) / 128;
    auto waves = [](int64_t count, int64_t room) { return (double)((count + room - 1) / room); };
    // a product in 32 bits is written, read and quantised
    const double extra = rows_out ? 2.0 + (double)rows * (double)n * 9.0 / 5e6 : 0.0;
    const TokenPlan t = token_plan(rows, n, k);
    Way best{Way::PAIRS, 0, 1, t, rows_out, 4.2 + waves(tiles * blocks, pairs) * (0.3 * (double)nkb + 0.5) + extra};
    auto offer = [&](decltype(best.kernel) kernel, int bt, int split, bool requant, double time) {
        if (time < best.time) best = {kernel, bt, split, t, requant, time};
    };
    // k_token reads about 6 MB of weights a microsecond
    if (t.per_cta > 0) offer(Way::TOKEN, 0, 1, rows_out, 3.0 + (double)n * (double)k / 6e6 + extra);
    const struct { int bt; double fixed, block; } sizes[] = {{16, 2.9, 0.24}, {32, 3.4, 0.25}, {64, 4.3, 0.27}, {128, 6.1, 0.33}};
    for (const auto &z : sizes) {
        const int64_t count = (rows + z.bt - 1) / z.bt * channels;
        if (count > 4 * kSms || t.per_cta > 0 || (z.bt > 16 && rows <= z.bt / 2)) continue;
        for (int split = 1; split <= F_MAX_SPLIT && split <= nkb; split *= 2)
            offer(Way::FEW, z.bt, split, rows_out,
                  waves(count, cluster_room(split)) * (z.fixed + z.block * (double)((nkb + split - 1) / split)) + extra);
    }
    if (rows_out) {
        const int64_t deep = (rows + 15) / 16;
        for (int split = 1; split <= F_MAX_SPLIT && split <= nkb && split * channels <= F_MAX_CLUSTER; split *= 2)
            if (deep <= cluster_room((int)(split * channels)))
                offer(Way::FEW_ROWS, 16, split, false, 3.2 + 0.24 * (double)((nkb + split - 1) / split));
        if (blocks <= 2)
            offer(Way::PAIRS_ROWS, 0, 1, false, 4.2 + waves(tiles, pairs) * ((double)blocks * 0.3 * (double)nkb + 2.9));
        // both launches multiply; nothing in 32 bits leaves the chip (28,467 rows of 128 x 4,650: 181 us against 282,
        // 20,480 of 1,024 x 1,024: 43 against 46)
        offer(Way::PAIRS_TWICE, 0, 1, false,
              10.0 + waves(tiles * blocks, pairs) * (2 * std::max(0.3 * (double)nkb, 0.2) + 2.6));
    }
    return best;
}

// The rows of a call, cut in two where the pair kernel's last wave would leave most SMs idle for the time that its
// K takes: 20,480 rows of 8,192 x 512 requantised, 97 us in two waves, 82 us as one wave and 1,536 rows apart.
struct Ways {
    int64_t cut;                 // rows of the first way; the others take the second
    Way way[2];
};

Ways cut_rows(int64_t rows, int64_t n, int64_t k, bool rows_out)
{
    Ways o{rows, {choose(rows, n, k, rows_out), {}}};
    const Way &all = o.way[0];
    if (all.kernel != Way::PAIRS && all.kernel != Way::PAIRS_ROWS) return o;
    const int64_t tiles = (rows + 2 * PM - 1) / (2 * PM), blocks = (n + PN - 1) / PN, pairs = kSms / 2;
    const int64_t per_tile = all.kernel == Way::PAIRS_ROWS ? 1 : blocks;
    const int64_t full = tiles * per_tile / pairs * pairs / per_tile * 2 * PM;      // rows of the full waves
    if (full <= 0 || full >= rows) return o;
    const Way main = choose(full, n, k, rows_out), rest = choose(rows - full, n, k, rows_out);
    if (main.time + rest.time < all.time) o = {full, {main, rest}};
    return o;
}

}  // namespace

void quantize_tokens(const void *x, int type, int64_t rows, int64_t cols, int64_t x_stride, int8_t *q, int64_t q_stride,
                     float *scales, cudaStream_t s)
{
    if (type == SC_TYPE_F32) quantize((const float *)x, rows, (int)cols, x_stride, q, q_stride, scales, s);
    else if (type == SC_TYPE_F16) quantize((const __half *)x, rows, (int)cols, x_stride, q, q_stride, scales, s);
    else quantize((const __nv_bfloat16 *)x, rows, (int)cols, x_stride, q, q_stride, scales, s);
}

void dequantize_tokens(const int8_t *q, int64_t q_stride, const float *scales, float scale, int64_t rows, int64_t cols,
                       void *y, int type, int64_t y_stride, cudaStream_t s)
{
    if (type == SC_TYPE_F32) dequantize(q, q_stride, scales, scale, rows, (int)cols, (float *)y, y_stride, s);
    else if (type == SC_TYPE_F16) dequantize(q, q_stride, scales, scale, rows, (int)cols, (__half *)y, y_stride, s);
    else dequantize(q, q_stride, scales, scale, rows, (int)cols, (__nv_bfloat16 *)y, y_stride, s);
}

static int64_t pad(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// What a call consists of.  Its workspace holds, in this order and where they are there: the scales and the
// rows of a float x held in 8 bits, x and w spread where TMA cannot read them, and the product's rows
// in 32 bits where a launch of their own quantises them.
struct Plan {
    Ways ways;
    bool quantise, spread_x, spread_w;
    int64_t wide;                // bytes of the product in 32 bits, or of the rows' largest magnitudes
    int64_t bytes;
};

static Plan plan(const Int8Linear &p)
{
    Plan o{};
    o.ways = cut_rows(p.rows, p.n, p.k, p.y_type == SC_TYPE_I8 && p.y_scales);
    const Way *w = o.ways.way;
    const bool token = w[0].kernel == Way::TOKEN;
    o.quantise = p.x_type != SC_TYPE_I8 && !token;
    o.spread_x = p.x_type == SC_TYPE_I8 && !token && !p.x_packed;
    o.spread_w = !p.w_packed;
    auto wide = [&](const Way &way, int64_t rows) {
        return way.requant ? rows * pad(p.n, 4) * 4 : way.kernel == Way::PAIRS_TWICE ? rows * 4 : 0;
    };
    o.wide = wide(w[0], o.ways.cut);
    if (o.ways.cut < p.rows) o.wide = std::max(o.wide, wide(w[1], p.rows - o.ways.cut));
    if (o.quantise) o.bytes += pad(p.rows * 4, 256);
    if (o.quantise || o.spread_x) o.bytes += pad(p.rows * pad(p.k, 16), 256);
    if (o.spread_w) o.bytes += pad(p.n * pad(p.k, 16), 256);
    o.bytes += pad(o.wide, 256);
    return o;
}

int64_t int8_linear_workspace(const Int8Linear &p) { return plan(p).bytes; }

int int8_linear_ways(int64_t rows, int64_t n, int64_t k, bool rows_out, int64_t *out)
{
    const Ways o = cut_rows(rows, n, k, rows_out);
    const int parts = o.cut < rows ? 2 : 1;
    for (int i = 0; i < parts; ++i) {
        const Way &w = o.way[i];
        const int64_t values[5] = {i == 0 ? o.cut : rows - o.cut, w.kernel, w.kernel == Way::FEW ? w.bt : 0, w.split,
                                   (int64_t)(w.time * 1e3)};
        std::copy(values, values + 5, out + 5 * i);
    }
    return parts;
}

// p's rows, x and w being int8 rows that TMA can read (k_token: as they are); `wide` takes a product in 32 bits
static void multiply(const Int8Linear &p, const Way &way, Rows8 x, const float *xs, Rows8 w, float *wide, cudaStream_t s)
{
    void *y = way.requant ? wide : p.y;
    const int y_type = way.requant ? SC_TYPE_F32 : p.y_type;
    const int64_t ys = way.requant ? pad(p.n, 4) : p.y_stride;     // rows on 16 bytes, for TMA
    switch (way.kernel) {
    case Way::TOKEN: {
        const TokenParams a{p.x, p.x_stride, xs, w.p, w.stride, p.w_scales, p.bias, p.rows, (int)p.n, (int)p.k, p.relu,
                            y_type, y, ys, p.output_scale, way.t.per_cta, way.t.log_s};
        if (p.x_type == SC_TYPE_I8) product_token<int8_t>(a, way.t, s);
        else if (p.x_type == SC_TYPE_F32) product_token<float>(a, way.t, s);
        else if (p.x_type == SC_TYPE_F16) product_token<__half>(a, way.t, s);
        else product_token<__nv_bfloat16>(a, way.t, s);
        break;
    }
    case Way::FEW:
        if (way.bt == 16) product_few<16>(p, x, xs, w, y, y_type, ys, way.split, s);
        else if (way.bt == 32) product_few<32>(p, x, xs, w, y, y_type, ys, way.split, s);
        else if (way.bt == 64) product_few<64>(p, x, xs, w, y, y_type, ys, way.split, s);
        else product_few<128>(p, x, xs, w, y, y_type, ys, way.split, s);
        break;
    case Way::FEW_ROWS: launch_few<16, true>(p, x, xs, w, (int8_t *)y, ys, way.split, s); break;
    case Way::PAIRS_ROWS: product_pairs<int8_t, ROWS>(p, x, xs, w, (int8_t *)y, ys, s); break;
    case Way::PAIRS_TWICE: {
        uint32_t *tops = (uint32_t *)wide;
        SC_CUDA(cudaMemsetAsync(tops, 0, (size_t)p.rows * 4, s));
        product_pairs<int8_t, TOPS>(p, x, xs, w, (int8_t *)y, ys, s, tops);
        product_pairs<int8_t, BY_TOPS>(p, x, xs, w, (int8_t *)y, ys, s, tops);
        break;
    }
    case Way::PAIRS:
        if (y_type == SC_TYPE_I8) product_pairs<int8_t, STATIC>(p, x, xs, w, (int8_t *)y, ys, s);
        else if (y_type == SC_TYPE_F32) product_pairs<float, PLAIN>(p, x, xs, w, (float *)y, ys, s);
        else if (y_type == SC_TYPE_F16) product_pairs<__half, PLAIN>(p, x, xs, w, (__half *)y, ys, s);
        else product_pairs<__nv_bfloat16, PLAIN>(p, x, xs, w, (__nv_bfloat16 *)y, ys, s);
        break;
    }
    if (way.requant) quantize((const float *)y, p.rows, (int)p.n, ys, (int8_t *)p.y, p.y_stride, p.y_scales, s);
}

void int8_linear(const Int8Linear &p, cudaStream_t s)
{
    const Plan o = plan(p);
    uint8_t *ws = (uint8_t *)p.workspace;
    auto take = [&](int64_t bytes) {
        uint8_t *at = ws;
        ws += pad(bytes, 256);
        return at;
    };
    auto spread = [&](const int8_t *from, int64_t rows, int64_t stride) {
        int8_t *to = (int8_t *)take(rows * pad(p.k, 16));
        launch(k_spread, grid_x((rows + 7) / 8), 256, 0, s, 1, from, rows, p.k, stride, to, pad(p.k, 16));
        return Rows8{to, pad(p.k, 16)};
    };
    Rows8 x{(const int8_t *)p.x, p.x_stride}, w{p.w, p.w_stride};
    const float *xs = p.x_scales;
    if (o.quantise) {
        float *sc = (float *)take(p.rows * 4);
        int8_t *q = (int8_t *)take(p.rows * pad(p.k, 16));
        quantize_tokens(p.x, p.x_type, p.rows, p.k, p.x_stride, q, pad(p.k, 16), sc, s);
        x = {q, pad(p.k, 16)};
        xs = sc;
    } else if (o.spread_x) {
        x = spread(x.p, p.rows, x.stride);
    }
    if (o.spread_w) w = spread(p.w, p.n, p.w_stride);
    float *wide = (float *)ws;
    // rows r .. r + count on their way
    auto rows_of = [&](int64_t r, int64_t count, const Way &way) {
        Int8Linear part = p;
        part.rows = count;
        part.y = (uint8_t *)p.y + r * p.y_stride * (p.y_type == SC_TYPE_F32 ? 4 : p.y_type == SC_TYPE_I8 ? 1 : 2);
        part.y_scales = p.y_scales ? p.y_scales + r : nullptr;
        if (r > 0) {            // x is int8 here: k_token takes a float x whole
            part.x = x.p + r * x.stride;
            part.x_type = SC_TYPE_I8;
            part.x_stride = x.stride;
        }
        multiply(part, way, {x.p + r * x.stride, x.stride}, xs ? xs + r : nullptr, w, wide, s);
    };
    rows_of(0, o.ways.cut, o.ways.way[0]);
    if (o.ways.cut < p.rows) rows_of(o.ways.cut, p.rows - o.ways.cut, o.ways.way[1]);
}

namespace {

// A wait that nothing ends: gives up after its time limit, is counted, and the kernel ends.
__global__ void __launch_bounds__(32) k_int8_wait_selftest()
{
    __shared__ __align__(8) uint64_t bar;
    next_may_start();
    previous_done();
    if (threadIdx.x == 0) {
        tc::mbar_init(&bar, 1);
        tc::fence_mbar_init();
    }
    __syncwarp();
    if (threadIdx.x == 0) tc::mbar_wait(&bar, 0);
}

}  // namespace

void int8_wait_selftest(cudaStream_t s) { launch(k_int8_wait_selftest, 1, 32, 0, s, 1); }

int int8_waits_given_up(cudaStream_t s)
{
    int v = 0;
    SC_CUDA(cudaMemcpyFromSymbolAsync(&v, tc::g_device_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    SC_CUDA(cudaStreamSynchronize(s));
    return v;
}

}  // namespace sc
