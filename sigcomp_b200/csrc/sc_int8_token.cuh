// Products of single tokens and a few of them on CUDA cores.  Included by sc_int8.cu.
#pragma once

namespace sc {
namespace {

// With one to eight rows a layer costs one reading of its weights, and no tile fills a tensor core, so
// what counts is how soon every byte of them is in flight and how little comes before and after:
// no tensor memory, no barriers in memory, one launch.  A warp reads a channel's row (or one of S parts of
// it, where the channels alone would leave SMs idle) in 512-byte steps and multiplies it with dp4a against
// the tokens, which lie in shared memory; the first U steps are requested before the tokens are there.
// Float tokens are quantised on the way to shared memory by every CTA for itself, which costs a
// reading of the token from L2 and saves a launch.
//
// Requantised rows (ROWS_OUT): the CTAs along x are one cluster and have all channels between them; they
// exchange their rows' maxima through shared memory.
struct TokenParams {
    const void *x;
    int64_t x_stride;
    const float *xs;                 // of int8 tokens
    const int8_t *w;
    int64_t w_stride;
    const float *ws, *bias;
    int64_t rows;
    int n, k, relu, y_type;
    void *y;
    int64_t y_stride;
    float output_scale;
    float *y_scales;
    int per_cta;                     // channels of a CTA, a multiple of 8 >> log_s
    int log_s;                       // 2^log_s warps share a channel
};

constexpr int TK_WARPS = 8, TK_THREADS = 32 * TK_WARPS;
constexpr int TK_CLUSTER = 16;       // CTAs that share a row's maximum, at most

__host__ __device__ inline int token_smem(int mt, int k, int per_cta, int log_s, bool rows_out)
{
    return mt * ((k + 15) / 16 * 16) + mt * 4 + (per_cta << log_s) * mt * 4 +
           (rows_out ? per_cta * mt * 4 + (TK_CLUSTER + 1) * mt * 4 : 0) + TK_WARPS * 4;
}

// 16 bytes of a weight row; what lies behind its end counts as zero
__device__ __forceinline__ uint4 weight_vec(const int8_t *row, int at, int k)
{
    uint4 v = make_uint4(0, 0, 0, 0);
    if (at + 16 <= k) {
        asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
            : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + at));
    } else {
        int8_t *e = reinterpret_cast<int8_t *>(&v);
        for (int i = 0; at + i < k; ++i) e[i] = row[at + i];
    }
    return v;
}

template <typename X, int MT, bool ROWS_OUT>
__global__ void __launch_bounds__(TK_THREADS) k_token(const TokenParams p)
{
    constexpr int U = 8;
    extern __shared__ __align__(16) uint8_t smem[];
    const int kpad = (p.k + 15) / 16 * 16, S = 1 << p.log_s;
    int8_t *xq = reinterpret_cast<int8_t *>(smem);                         // [MT][kpad]
    float *xs = reinterpret_cast<float *>(smem + MT * kpad);               // [MT]
    int32_t *red = reinterpret_cast<int32_t *>(xs + MT);                   // [per_cta][S][MT]
    uint32_t *tops = reinterpret_cast<uint32_t *>(red + (p.per_cta << p.log_s) * MT);   // [warps]
    uint32_t *local = tops + TK_WARPS;                                     // [MT] this CTA's maxima
    uint32_t *mx = local + MT;                                             // [cluster][MT]
    float *yb = reinterpret_cast<float *>(mx + TK_CLUSTER * MT);           // [MT][per_cta]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = blockIdx.x * p.per_cta;
    const int64_t t0 = (int64_t)blockIdx.y * MT;

    // this warp's steps: channels slot, slot + abreast, ... of the CTA, in each the vectors of its part
    const int abreast = TK_WARPS >> p.log_s, slot = warp >> p.log_s, seg = warp & (S - 1);
    const int kv = kpad / 16, v0 = (int)((int64_t)kv * seg >> p.log_s), v1 = (int)((int64_t)kv * (seg + 1) >> p.log_s);
    const int per_channel = (((kv + S - 1) >> p.log_s) + 31) / 32;
    const int items = p.per_cta / abreast * per_channel;
    int li = 0, lj = 0;                                                    // next step to load
    auto load = [&]() {
        const int c = c0 + slot + li * abreast, v = v0 + lj * 32 + lane;
        const uint4 r = li * per_channel < items && c < p.n && v < v1
                            ? weight_vec(p.w + (int64_t)c * p.w_stride, v * 16, p.k) : make_uint4(0, 0, 0, 0);
        if (++lj == per_channel) { lj = 0; ++li; }
        return r;
    };
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load();

    // the tokens
    if (sizeof(X) == 1) {
        const int8_t *x = reinterpret_cast<const int8_t *>(p.x);
        const bool packed = ((uintptr_t)x & 15) == 0 && (p.x_stride & 15) == 0;
        for (int i = threadIdx.x; i < MT * kv; i += TK_THREADS) {
            const int t = i / kv, at = i % kv * 16;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (t0 + t < p.rows) {
                const int8_t *row = x + (t0 + t) * p.x_stride;
                if (packed && at + 16 <= p.k) {
                    v = *reinterpret_cast<const uint4 *>(row + at);
                } else {
                    int8_t *e = reinterpret_cast<int8_t *>(&v);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (at + j < p.k) e[j] = row[at + j];
                }
            }
            *reinterpret_cast<uint4 *>(xq + t * kpad + at) = v;
        }
        if (threadIdx.x < MT) xs[threadIdx.x] = t0 + threadIdx.x < p.rows ? p.xs[t0 + threadIdx.x] : 0.0f;
    } else {
        using V = Vec<typename std::conditional<sizeof(X) == 1, float, X>::type>;
        using E = typename std::conditional<sizeof(X) == 1, float, X>::type;
        constexpr int PER = TK_WARPS / MT;                                 // warps of a token
        const int t = warp / PER, th = (warp % PER) * 32 + lane;
        const E *row = reinterpret_cast<const E *>(p.x) + (t0 + t) * p.x_stride;
        const bool live = t0 + t < p.rows;
        const bool packed = ((uintptr_t)p.x & 15) == 0 && (p.x_stride * sizeof(E) & 15) == 0;
        uint32_t m = 0;
        if (live)
            for (int c = th * V::N; c < p.k; c += PER * 32 * V::N)
                m = V::top(packed ? load_vec<E, true>(row, c, p.k) : load_vec<E, false>(row, c, p.k), m);
        m = __reduce_max_sync(0xffffffffu, V::top_bits(m));
        if (lane == 0) tops[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) m = max(m, tops[t * PER + i]);
        const RowScale rs = row_scale(m);
        if (th == 0) xs[t] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
        for (int c = th * V::N; c < kpad; c += PER * 32 * V::N) {
            uint32_t o[V::N / 4] = {};
            if (live && rs.finite && c < p.k)
                V::quantise(packed ? load_vec<E, true>(row, c, p.k) : load_vec<E, false>(row, c, p.k), rs.r, o);
#pragma unroll
            for (int i = 0; i < V::N / 4; ++i) *reinterpret_cast<uint32_t *>(xq + t * kpad + c + 4 * i) = o[i];
        }
    }
    if (ROWS_OUT && threadIdx.x < MT) local[threadIdx.x] = 0;
    __syncthreads();
    if (ROWS_OUT) cluster_arrive();                                        // this CTA runs: its memory may be written

    // the sums
    int32_t acc[MT] = {};
    int ci = 0, cj = 0;
    for (int it = 0; it < items; it += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (it + u >= items) break;
            const int v = v0 + cj * 32 + lane;
            const int at = v < v1 ? v * 16 : 0;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint4 a = *reinterpret_cast<const uint4 *>(xq + t * kpad + at);
                acc[t] = __dp4a((int)a.x, (int)w[u].x, acc[t]);
                acc[t] = __dp4a((int)a.y, (int)w[u].y, acc[t]);
                acc[t] = __dp4a((int)a.z, (int)w[u].z, acc[t]);
                acc[t] = __dp4a((int)a.w, (int)w[u].w, acc[t]);
            }
            w[u] = load();
            if (++cj == per_channel) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int32_t sum = __reduce_add_sync(0xffffffffu, acc[t]);
                    if (lane == 0) red[(((slot + ci * abreast) << p.log_s) + seg) * MT + t] = sum;
                    acc[t] = 0;
                }
                cj = 0;
                ++ci;
            }
        }
    }
    __syncthreads();

    // the results, neighbouring threads on neighbouring channels
    for (int i = threadIdx.x; i < MT * p.per_cta; i += TK_THREADS) {
        const int t = i / p.per_cta, ch = i % p.per_cta, c = c0 + ch;
        if (c >= p.n || t0 + t >= p.rows) continue;
        int32_t sum = 0;
        for (int g = 0; g < S; ++g) sum += red[((ch << p.log_s) + g) * MT + t];
        const float y = affine(sum, xs[t], p.ws[c], p.bias ? p.bias[c] : 0.0f, p.relu);
        if constexpr (ROWS_OUT) {
            yb[i] = y;
            atomicMax(&local[t], magnitude(y));
        } else {
            store_one(p.y, p.y_type, (t0 + t) * p.y_stride + c, y, p.output_scale);
        }
    }
    if constexpr (ROWS_OUT) {
        __syncthreads();
        cluster_wait();
        const uint32_t rank = cluster_ctarank();
        for (int i = threadIdx.x; i < (int)gridDim.x * MT; i += TK_THREADS) {
            const uint32_t at = map_to_rank(&mx[rank * MT + i % MT], i / MT);
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(local[i % MT]) : "memory");
        }
        cluster_sync();
        for (int i = threadIdx.x; i < MT * p.per_cta; i += TK_THREADS) {
            const int t = i / p.per_cta, c = c0 + i % p.per_cta;
            if (c >= p.n || t0 + t >= p.rows) continue;
            uint32_t top = 0;
            for (int r = 0; r < (int)gridDim.x; ++r) top = max(top, mx[r * MT + t]);
            const RowScale rs = row_scale(top);
            reinterpret_cast<int8_t *>(p.y)[(t0 + t) * p.y_stride + c] = rs.finite ? (int8_t)quantise_bits(yb[i], rs.r) : 0;
            if (c == 0) p.y_scales[t0 + t] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
        }
    }
}

}  // namespace
}  // namespace sc
