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

#include "sc_internal.h"
#include "sc_int8.h"
#include "sc_tc.cuh"

namespace sc {
namespace {

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
__device__ __forceinline__ uint32_t quantise_bits(float v, float r) { return __float_as_uint(__fmaf_rn(v, r, 12582912.0f)); }

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// ---- quantise --------------------------------------------------------------------------------
// A row is read once: T threads hold its 16-byte vectors in registers through the maximum.
// Bound by HBM (e + 1 bytes per element).
template <typename T, int THREADS, int HELD, bool ALIGNED>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
k_quantize(const T *__restrict__ x, int64_t rows, int cols, int64_t x_stride, int8_t *__restrict__ q, int64_t q_stride,
           float *__restrict__ scales)
{
    constexpr int V = 16 / sizeof(T);
    constexpr int PER_BLOCK = THREADS < 256 ? 256 / THREADS : 1;
    __shared__ uint32_t tops[32];
    const int t = threadIdx.x % THREADS;
    const int64_t row = (int64_t)blockIdx.x * PER_BLOCK + threadIdx.x / THREADS;
    if (THREADS <= 32 && row >= rows) return;        // whole warps: THREADS divides 32's multiples
    const T *xr = x + row * x_stride;
    float v[HELD][V];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int c = (h * THREADS + t) * V;
        if (ALIGNED && c + V <= cols) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(xr + c);
            const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int i = 0; i < V; ++i) v[h][i] = to_f32<T>(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[h][i] = c + i < cols ? to_f32<T>(xr[c + i]) : 0.0f;
        }
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, magnitude(v[h][i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (THREADS > 32) {
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
        const int w = threadIdx.x & 31;
        top = __reduce_max_sync(0xffffffffu, w < THREADS / 32 ? tops[w] : 0u);
    }
    const RowScale rs = row_scale(top);
    if (t == 0) scales[row] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
    int8_t *qr = q + row * q_stride;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int c = (h * THREADS + t) * V;
        uint32_t p[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            p[i] = rs.finite ? pack4(quantise_bits(v[h][4 * i], rs.r), quantise_bits(v[h][4 * i + 1], rs.r),
                                     quantise_bits(v[h][4 * i + 2], rs.r), quantise_bits(v[h][4 * i + 3], rs.r))
                             : 0u;
        if (ALIGNED && c + V <= cols) {
            if (V == 8) *reinterpret_cast<uint2 *>(qr + c) = make_uint2(p[0], p[V / 4 - 1]);
            else *reinterpret_cast<uint32_t *>(qr + c) = p[0];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < cols) qr[c + i] = (int8_t)(p[i / 4] >> (8 * (i % 4)));
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
    uint32_t top = 0;
    for (int c = threadIdx.x; c < cols; c += 1024) top = max(top, magnitude(to_f32<T>(xr[c])));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[threadIdx.x & 31]);
    const RowScale rs = row_scale(top);
    if (threadIdx.x == 0) scales[blockIdx.x] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
    int8_t *qr = q + (int64_t)blockIdx.x * q_stride;
    for (int c = threadIdx.x; c < cols; c += 1024)
        qr[c] = rs.finite ? (int8_t)quantise_bits(to_f32<T>(xr[c]), rs.r) : 0;
}

// ---- dequantise ------------------------------------------------------------------------------
// One warp per 512 columns of a row, 16 values a thread.  Bound by HBM (1 + e bytes per element).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256)
k_dequantize(const int8_t *__restrict__ q, int64_t q_stride, const float *__restrict__ scales, float scale, int64_t rows,
             int cols, T *__restrict__ y, int64_t y_stride)
{
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const float s = scales ? scales[row] : scale;
    const int8_t *qr = q + row * q_stride;
    T *yr = y + row * y_stride;
    for (int64_t c0 = (int64_t)blockIdx.y * 512; c0 < cols; c0 += (int64_t)gridDim.y * 512) {
        const int c = (int)c0 + (threadIdx.x & 31) * 16;
        if (ALIGNED && c + 16 <= cols) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(qr + c);
            const int8_t *e = reinterpret_cast<const int8_t *>(&raw);
            __align__(16) T out[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) out[i] = from_f32<T>(__fmul_rn((float)e[i], s));
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i)
                reinterpret_cast<uint4 *>(yr + c)[i] = reinterpret_cast<const uint4 *>(out)[i];
        } else {
            for (int i = 0; i < 16 && c + i < cols; ++i) yr[c + i] = from_f32<T>(__fmul_rn((float)qr[c + i], s));
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

// Any sizes, strides and alignment: 64 x 64 results a block, K in blocks of 64, CUDA cores.
template <typename T>
__global__ void __launch_bounds__(256)
k_product_any(const int8_t *__restrict__ x, int64_t x_stride, const float *__restrict__ xs, const int8_t *__restrict__ w,
              int64_t w_stride, const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int n, int k,
              int relu, T *__restrict__ y, int64_t y_stride)
{
    __shared__ int32_t a[64][17], b[64][17];
    const int64_t m0 = (int64_t)blockIdx.x * 64;
    const int n0 = blockIdx.y * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int32_t acc[4][4] = {};
    for (int k0 = 0; k0 < k; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = i >> 6, c = i & 63;
            const bool in = k0 + c < k;
            reinterpret_cast<int8_t *>(a[r])[c] = in && m0 + r < rows ? x[(m0 + r) * x_stride + k0 + c] : 0;
            reinterpret_cast<int8_t *>(b[r])[c] = in && n0 + r < n ? w[(int64_t)(n0 + r) * w_stride + k0 + c] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[ty + 16 * i][c], b[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = m0 + ty + 16 * i;
            const int c = n0 + tx + 16 * j;
            if (r < rows && c < n)
                y[r * y_stride + c] = from_f32<T>(affine(acc[i][j], xs[r], ws[c], bias ? bias[c] : 0.0f, relu));
        }
}

// sat(rint(y / scale)) in the low byte; a NaN becomes 0
__device__ __forceinline__ uint32_t static_bits(float y, float scale)
{
    int32_t o;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(o) : "f"(__fdiv_rn(y, scale)));
    return (uint32_t)o & 0xffu;
}

}  // namespace
}  // namespace sc

#include "sc_int8_mm.cuh"

namespace sc {
namespace {

// ---- host side -------------------------------------------------------------------------------

// Rows copied to a multiple of 16 bytes apart, for arrays that TMA cannot read as they lie.  Bytes behind
// a row's end stay as they are: the tensor map ends with the row.
__global__ void __launch_bounds__(256)
k_spread(const int8_t *__restrict__ x, int64_t rows, int cols, int64_t x_stride, int8_t *__restrict__ y, int64_t y_stride)
{
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
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

template <typename T>
void quantize(const T *x, int64_t rows, int cols, int64_t xs, int8_t *q, int64_t qs, float *scales, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool al = aligned(x, xs * (int64_t)sizeof(T), 16) && aligned(q, qs, V);
#define SC_Q(THREADS, HELD)                                                                                        \
    do {                                                                                                           \
        const unsigned g = grid_x(THREADS < 256 ? (rows + 256 / THREADS - 1) / (256 / THREADS) : rows);            \
        if (al) k_quantize<T, THREADS, HELD, true><<<g, THREADS < 256 ? 256 : THREADS, 0, s>>>(x, rows, cols, xs, q, qs, scales); \
        else k_quantize<T, THREADS, HELD, false><<<g, THREADS < 256 ? 256 : THREADS, 0, s>>>(x, rows, cols, xs, q, qs, scales);   \
    } while (0)
    if (cols <= 32 * V) SC_Q(32, 1);
    else if (cols <= 64 * V) SC_Q(32, 2);
    else if (cols <= 128 * V) SC_Q(32, 4);
    else if (cols <= 256 * V) SC_Q(256, 1);
    else if (cols <= 512 * V) SC_Q(256, 2);
    else if (cols <= 1024 * V) SC_Q(1024, 1);
    else if (cols <= 4096 * V) SC_Q(1024, 4);
    else k_quantize_long<T><<<grid_x(rows), 1024, 0, s>>>(x, cols, xs, q, qs, scales);
#undef SC_Q
    SC_LAUNCH_CHECK();
    count_launch();
}

template <typename T>
void dequantize(const int8_t *q, int64_t qs, const float *scales, float scale, int64_t rows, int cols, T *y, int64_t ys,
                cudaStream_t s)
{
    const dim3 g(grid_x((rows + 7) / 8), (unsigned)std::min((cols + 511) / 512, 65535));
    if (aligned(q, qs, 16) && aligned(y, ys * (int64_t)sizeof(T), 16))
        k_dequantize<T, true><<<g, 256, 0, s>>>(q, qs, scales, scale, rows, cols, y, ys);
    else
        k_dequantize<T, false><<<g, 256, 0, s>>>(q, qs, scales, scale, rows, cols, y, ys);
    SC_LAUNCH_CHECK();
    count_launch();
}

struct Rows8 {
    const int8_t *p;
    int64_t stride;
};

int sm_count()
{
    static int counts[64];
    int dev = 0;
    SC_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && counts[dev] > 0) return counts[dev];
    int n = 0;
    SC_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) counts[dev] = n;
    return n;
}

// The kernel's shared memory limit, set once per device.
template <typename F>
void allow_smem(F *kernel, int bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    SC_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
    SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename T> constexpr CUtensorMapDataType map_type();
template <> constexpr CUtensorMapDataType map_type<float>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT32; }
template <> constexpr CUtensorMapDataType map_type<__half>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }
template <> constexpr CUtensorMapDataType map_type<__nv_bfloat16>() { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }
template <> constexpr CUtensorMapDataType map_type<int8_t>() { return CU_TENSOR_MAP_DATA_TYPE_UINT8; }

// y (T; int8: requantised with a scale for each row, at most 512 channels) of int8 rows, on SM pairs
template <typename T, int MODE>
void product_pairs(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, T *y, int64_t y_stride, cudaStream_t s)
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
    const int64_t tiles = (p.rows + 2 * PM - 1) / (2 * PM), units = (p.n + PN - 1) / PN;
    const int64_t work = MODE == ROWS ? tiles : tiles * units;
    const unsigned pairs = (unsigned)std::min<int64_t>(work, sm_count() / 2);
    k_pair<T, MODE><<<2 * pairs, P_THREADS, P_SMEM, s>>>(a);
    SC_LAUNCH_CHECK();
    count_launch();
}

// y (float types, or int8 by one scale) of few int8 rows; `bt` tokens per tile, K split over `split` CTAs
template <int BT>
void product_few(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, void *y, int y_type, int64_t y_stride, int split,
                 cudaStream_t s)
{
    using C = FewCfg<BT>;
    static std::atomic<uint64_t> ready{0};
    allow_smem(k_few<BT>, C::SMEM, ready);
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
    a.y_type = y_type;
    a.y = y;
    a.y_stride = y_stride;
    a.output_scale = p.output_scale;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)split, (unsigned)((p.n + 127) / 128), (unsigned)((p.rows + BT - 1) / BT));
    cfg.blockDim = dim3(F_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    SC_CUDA(cudaLaunchKernelEx(&cfg, k_few<BT>, a));
    count_launch();
}

// Whether the pair kernel's units leave SM pairs without work.
bool few(int64_t rows, int64_t n) { return (rows + 2 * PM - 1) / (2 * PM) * ((n + PN - 1) / PN) < 64; }

int64_t pad(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

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

// Workspace: the rows of a float x held in 8 bits and their scales, x and w spread where TMA cannot read
// them, and the product's rows in 32 bits where they come back quantised by a launch of their own.
static bool own_requant(const Int8Linear &p)
{
    return p.y_type == SC_TYPE_I8 && p.y_scales && (p.n > 2 * PN || few(p.rows, p.n));
}

static void product(const Int8Linear &p, Rows8 x, const float *xs, Rows8 w, void *y, int y_type, int64_t y_stride,
                    cudaStream_t s)
{
    const bool rows = y_type == SC_TYPE_I8 && p.y_scales;
    if (!rows && few(p.rows, p.n)) {
        const int64_t nkb = (p.k + PK - 1) / PK;
        const int bt = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : 64;
        const int64_t tiles = (p.rows + bt - 1) / bt * ((p.n + 127) / 128);
        int split = 1;
        while (split < F_MAX_SPLIT && 2 * split <= nkb && 2 * split * tiles <= sm_count()) split *= 2;
        if (bt == 16) product_few<16>(p, x, xs, w, y, y_type, y_stride, split, s);
        else if (bt == 32) product_few<32>(p, x, xs, w, y, y_type, y_stride, split, s);
        else product_few<64>(p, x, xs, w, y, y_type, y_stride, split, s);
    } else if (rows) product_pairs<int8_t, ROWS>(p, x, xs, w, (int8_t *)y, y_stride, s);
    else if (y_type == SC_TYPE_I8) product_pairs<int8_t, STATIC>(p, x, xs, w, (int8_t *)y, y_stride, s);
    else if (y_type == SC_TYPE_F32) product_pairs<float, PLAIN>(p, x, xs, w, (float *)y, y_stride, s);
    else if (y_type == SC_TYPE_F16) product_pairs<__half, PLAIN>(p, x, xs, w, (__half *)y, y_stride, s);
    else product_pairs<__nv_bfloat16, PLAIN>(p, x, xs, w, (__nv_bfloat16 *)y, y_stride, s);
}

int64_t int8_linear_workspace(const Int8Linear &p)
{
    int64_t b = 0;
    if (p.x_type != SC_TYPE_I8) b += pad(p.rows * 4, 256);
    if (p.x_type != SC_TYPE_I8 || !p.x_packed) b += pad(p.rows * pad(p.k, 16), 256);
    if (!p.w_packed) b += pad(p.n * pad(p.k, 16), 256);
    if (own_requant(p)) b += pad(p.rows * p.n * 4, 256);
    return b;
}

void int8_linear(const Int8Linear &p, cudaStream_t s)
{
    uint8_t *ws = (uint8_t *)p.workspace;
    auto take = [&](int64_t bytes) {
        uint8_t *at = ws;
        ws += pad(bytes, 256);
        return at;
    };
    auto spread = [&](const int8_t *from, int64_t rows, int64_t stride) {
        int8_t *to = (int8_t *)take(rows * pad(p.k, 16));
        k_spread<<<grid_x((rows + 7) / 8), 256, 0, s>>>(from, rows, (int)p.k, stride, to, pad(p.k, 16));
        SC_LAUNCH_CHECK();
        count_launch();
        return Rows8{to, pad(p.k, 16)};
    };
    Rows8 x{(const int8_t *)p.x, p.x_stride}, w{p.w, p.w_stride};
    const float *xs = p.x_scales;
    if (p.x_type != SC_TYPE_I8) {
        float *sc = (float *)take(p.rows * 4);
        int8_t *q = (int8_t *)take(p.rows * pad(p.k, 16));
        quantize_tokens(p.x, p.x_type, p.rows, p.k, p.x_stride, q, pad(p.k, 16), sc, s);
        x = {q, pad(p.k, 16)};
        xs = sc;
    } else if (!p.x_packed) {
        x = spread(x.p, p.rows, x.stride);
    }
    if (!p.w_packed) w = spread(p.w, p.n, p.w_stride);
    if (own_requant(p)) {
        float *y = (float *)take(p.rows * p.n * 4);
        product(p, x, xs, w, y, SC_TYPE_F32, p.n, s);
        quantize(y, p.rows, (int)p.n, p.n, (int8_t *)p.y, p.y_stride, p.y_scales, s);
    } else {
        product(p, x, xs, w, p.y, p.y_type, p.y_stride, s);
    }
}

int int8_device_error()
{
    int v = 0, z = 0;
    SC_CUDA(cudaMemcpyFromSymbol(&v, tc::g_device_error, sizeof(int)));
    if (v) SC_CUDA(cudaMemcpyToSymbol(tc::g_device_error, &z, sizeof(int)));
    return v;
}

}  // namespace sc
