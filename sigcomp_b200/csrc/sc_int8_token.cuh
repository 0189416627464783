// Products of single tokens and a few of them on CUDA cores.  Included by sc_int8.cu.
#pragma once

namespace sc {
namespace {

// With one or two rows a layer costs one reading of its weights, and no tile fills a tensor core, so
// what counts is how soon every byte of them is in flight and how little comes before and after:
// no tensor memory, no barriers in memory, one launch, little code.  A warp takes four channels at a time
// and walks their rows (or one of S parts of them, where the channels alone would leave SMs idle) in
// 512-byte steps, two steps ahead, multiplying with dp4a against the tokens in shared memory; a token's
// vector is read once for the four channels.  The first steps are requested before the tokens are there.
// Float tokens are quantised on the way to shared memory by every CTA for itself, which costs a
// reading of the token from L2 and saves a launch.  One token: 3.1 us for 512 x 512, 3.7 for 8,192 x 512 (4.9 from bf16),
// 4.6 for 4,096 x 4,096 (3.6 TB/s); k_few takes 3.3, 5.1 and 5.9.
struct TokenParams {
    const void *x;
    int64_t x_stride;
    const float *xs;                 // of int8 tokens
    const int8_t *w;
    int64_t w_stride;
    const float *ws, *bias;
    int64_t rows;                    // the kernel's MT
    int n, k, relu, y_type;
    void *y;
    int64_t y_stride;
    float output_scale;
    int per_cta;                     // channels of a CTA, a multiple of 4 * (8 >> log_s)
    int log_s;                       // 2^log_s warps share a channel
};

constexpr int TK_WARPS = 8, TK_THREADS = 32 * TK_WARPS;
constexpr int TK_SMEM = 100 * 1024;   // two CTAs to an SM
constexpr int TK_CH = 4;             // channels a warp takes at a time

__host__ __device__ inline int token_smem(int mt, int k, int per_cta, int log_s)
{
    return mt * ((k + 15) / 16 * 16) + mt * 4 + (per_cta << log_s) * mt * 4 + TK_WARPS * 4;
}

// 16 bytes of an int8 row that ends within them; what lies behind its end counts as zero
__device__ __noinline__ uint4 last_vec(const int8_t *row, int at, int k)
{
    uint32_t v[4] = {};
    for (int i = 0; i < 16; ++i)
        if (at + i < k) {
            const uint32_t b = (uint32_t)(uint8_t)row[at + i] << (8 * (i & 3));
            if (i < 4) v[0] |= b;
            else if (i < 8) v[1] |= b;
            else if (i < 12) v[2] |= b;
            else v[3] |= b;
        }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename X, int MT>
__global__ void __launch_bounds__(TK_THREADS, 2) k_token(const TokenParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const int kpad = (p.k + 15) / 16 * 16, S = 1 << p.log_s;
    int8_t *xq = reinterpret_cast<int8_t *>(smem);                         // [MT][kpad]
    float *xs = reinterpret_cast<float *>(smem + MT * kpad);               // [MT]
    int32_t *red = reinterpret_cast<int32_t *>(xs + MT);                   // [per_cta][S][MT]
    uint32_t *tops = reinterpret_cast<uint32_t *>(red + (p.per_cta << p.log_s) * MT);   // [warps]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = blockIdx.x * p.per_cta;

    // this warp's channel group and part of K; steps of 32 vectors
    const int slot = warp >> p.log_s, seg = warp & (S - 1);
    const int kv = kpad / 16, v0 = (int)((int64_t)kv * seg >> p.log_s), v1 = (int)((int64_t)kv * (seg + 1) >> p.log_s);
    const int steps = (v1 - v0 + 31) / 32;
    auto load = [&](uint4(&w)[TK_CH], int c, int v) {
#pragma unroll
        for (int i = 0; i < TK_CH; ++i) {
            w[i] = make_uint4(0, 0, 0, 0);
            const int8_t *row = p.w + (int64_t)(c + i) * p.w_stride;
            if (c + i < p.n && v < v1) {
                // a vector may reach behind its row's end, into the next row, where the tokens are zero
                if (v * 16 + 16 <= p.k || c + i + 1 < p.n)
                    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "l"(row + v * 16));
                else w[i] = last_vec(row, v * 16, p.k);
            }
        }
    };
    next_may_start();
    previous_done();
    int c = c0 + slot * TK_CH;                                             // the group's first channel
    uint4 wa[TK_CH], wb[TK_CH];
    load(wa, c, v0 + lane);
    load(wb, c, v0 + 32 + lane);
    // scale and bias of this thread's first result
    const int first = c0 + threadIdx.x % p.per_cta;
    const float ws0 = first < p.n ? p.ws[first] : 0.0f, bias0 = first < p.n && p.bias ? p.bias[first] : 0.0f;

    // the tokens
    if (sizeof(X) == 1) {
        const int8_t *x = reinterpret_cast<const int8_t *>(p.x);
        const bool packed = ((uintptr_t)x & 15) == 0 && (p.x_stride & 15) == 0;
#pragma unroll 1
        for (int t = 0; t < MT; ++t) {
            const int8_t *row = x + (int64_t)t * p.x_stride;
            for (int v = threadIdx.x; v < kv; v += TK_THREADS)
                *reinterpret_cast<uint4 *>(xq + t * kpad + v * 16) =
                    packed && v * 16 + 16 <= p.k ? *reinterpret_cast<const uint4 *>(row + v * 16) : last_vec(row, v * 16, p.k);
        }
        if (threadIdx.x < MT) xs[threadIdx.x] = p.xs[threadIdx.x];
    } else {
        using V = Vec<typename std::conditional<sizeof(X) == 1, float, X>::type>;
        using E = typename std::conditional<sizeof(X) == 1, float, X>::type;
        constexpr int PER = TK_WARPS / MT;                                 // warps of a token
        const int t = warp / PER, th = (warp % PER) * 32 + lane;
        const E *row = reinterpret_cast<const E *>(p.x) + (int64_t)t * p.x_stride;
        const bool packed = ((uintptr_t)p.x & 15) == 0 && (p.x_stride * sizeof(E) & 15) == 0;
        uint32_t m = 0;
        for (int c = th * V::N; c < p.k; c += PER * 32 * V::N)
            m = V::top(packed && c + V::N <= p.k ? *reinterpret_cast<const uint4 *>(row + c) : load_elements<E>(row + c, row, row + p.k), m);
        m = __reduce_max_sync(0xffffffffu, V::top_bits(m));
        if (lane == 0) tops[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) m = max(m, tops[t * PER + i]);
        const RowScale rs = row_scale(m);
        if (th == 0) xs[t] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
        for (int c = th * V::N; c < kpad; c += PER * 32 * V::N) {
            uint32_t o[V::N / 4] = {};
            if (rs.finite && c < p.k)
                V::quantise(packed && c + V::N <= p.k ? *reinterpret_cast<const uint4 *>(row + c) : load_elements<E>(row + c, row, row + p.k), rs.r, o);
#pragma unroll
            for (int i = 0; i < V::N / 4; ++i) *reinterpret_cast<uint32_t *>(xq + t * kpad + c + 4 * i) = o[i];
        }
    }
    __syncthreads();

    // the sums
    for (int g = slot; g * TK_CH < p.per_cta; g += TK_WARPS >> p.log_s) {
        int32_t acc[TK_CH][MT] = {};
        auto multiply = [&](const uint4(&w)[TK_CH], int v) {
            const int at = v < v1 ? v * 16 : 0;                            // behind the part's end w is zero
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint4 a = *reinterpret_cast<const uint4 *>(xq + t * kpad + at);
#pragma unroll
                for (int i = 0; i < TK_CH; ++i) {
                    acc[i][t] = __dp4a((int)a.x, (int)w[i].x, acc[i][t]);
                    acc[i][t] = __dp4a((int)a.y, (int)w[i].y, acc[i][t]);
                    acc[i][t] = __dp4a((int)a.z, (int)w[i].z, acc[i][t]);
                    acc[i][t] = __dp4a((int)a.w, (int)w[i].w, acc[i][t]);
                }
            }
        };
        const int next = c + TK_CH * (TK_WARPS >> p.log_s);                // first channel of the next group
        const bool more = (g + (TK_WARPS >> p.log_s)) * TK_CH < p.per_cta;
#pragma unroll 1
        for (int j = 0; j < steps; j += 2) {
            const int v = v0 + j * 32 + lane;
            multiply(wa, v);
            if (j + 2 < steps) load(wa, c, v + 64);
            else if (more) load(wa, next, v0 + lane);
            multiply(wb, v + 32);
            if (j + 2 < steps) load(wb, c, v + 96);
            else if (more) load(wb, next, v0 + 32 + lane);
        }
#pragma unroll
        for (int i = 0; i < TK_CH; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int32_t sum = __reduce_add_sync(0xffffffffu, acc[i][t]);
                if (lane == 0) red[(((g * TK_CH + i) << p.log_s) + seg) * MT + t] = sum;
            }
        c = next;
    }
    __syncthreads();

    // the results, neighbouring threads on neighbouring channels
    for (int i = threadIdx.x; i < MT * p.per_cta; i += TK_THREADS) {
        const int t = i / p.per_cta, ch = i % p.per_cta, c = c0 + ch;
        if (c >= p.n) continue;
        int32_t sum = 0;
        for (int g = 0; g < S; ++g) sum += red[((ch << p.log_s) + g) * MT + t];
        const bool is_first = i == (int)threadIdx.x;
        const float y = affine(sum, xs[t], is_first ? ws0 : p.ws[c], is_first ? bias0 : p.bias ? p.bias[c] : 0.0f, p.relu);
        store_one(p.y, p.y_type, (int64_t)t * p.y_stride + c, y, p.output_scale);
    }
}

}  // namespace
}  // namespace sc
