// Tensor-core products of the int8 operators.  Included by sc_int8.cu (one translation unit with its
// device error flag).
#pragma once

namespace sc {
namespace {

using namespace tc;

// ---- products on SM pairs ----------------------------------------------------------------------
//
// A unit is 256 rows x 256 channels: one tcgen05.mma (cta_group::2, M = 256, N = 256) per 32 bytes of
// K over a pair of SMs, each holding its 128 rows of x and half of the weight rows of every K block
// (128 bytes) in a ring of 32 KB stages that TMA fills.  Two accumulators of 256 TMEM columns let the
// epilogue of one unit run under the products of the next.  Units go channel block by channel block
// over the same rows, so that x comes from L2 after its first block.
//
// Warps: 0 TMA producer, 1 MMA issuer (leader CTA), 2-9 epilogue (two for each TMEM lane quarter, half
// of a unit's columns each).  Every warp of the epilogue keeps its own scales and bias and writes
// its results through a 4 KB tile of its own, 32 rows of 128 bytes in the 128-byte swizzle, from which
// TMA stores them: no warp waits for another, but for the row maximum of requantised rows.
//
// Requantised rows (REQUANT): a tile is 256 rows x all channels, at most the two accumulators' 512.
// The first pass over a half turns its sums into results in 32 bits, puts them back into TMEM and takes
// the row's maximum; the second, once both halves' maximum is known, scales and packs them.  The first
// pass over half 0 runs under the products of half 1, the second over half 1 under those of the next
// tile's half 0.
//
// Rows of more channels are quantised by two launches that both multiply: the first keeps the rows' largest magnitudes
// (TOPS), the second quantises by them (BY_TOPS).  Those and rows quantised by one scale (STATIC) go unit by unit through
// the same two passes, without a maximum, so that a row's bytes are staged sixteen at a time.
//
// Every wait is bounded; a warp that gives up ends, and the others end on their own limits.
//
// Measured: 65,536 x 8,192 -> 512 bf16 in 171 us (3.2 P operations a second, tensor pipe 89 % active; 214 us in a long
// loop, where the 1 kW cap holds the clock at 1.18 GHz), 4,096 cubed in 47 to 56 us, 262,144 x 512 -> 512 bf16 in
// 77 us and requantised in 75 to 87 us, where the epilogue bounds it (ALU 40 %, its passes wait for the products).
constexpr int PM = 128;                        // rows per CTA
constexpr int PN = 256;                        // channels per unit
constexpr int PK = 128;                        // bytes of K per stage
constexpr int P_STAGES = 5;
constexpr int P_A = PM * PK, P_B = (PN / 2) * PK, P_STAGE = P_A + P_B;
constexpr int P_EPI = 8;
constexpr int P_THREADS = 32 * (2 + P_EPI);
constexpr int P_OFF_OUT = P_STAGES * P_STAGE;                      // staging: 4 KB per epilogue warp
constexpr int P_OFF_TB = P_OFF_OUT + P_EPI * 4096;                 // {scale, bias} per warp and column
constexpr int P_TB = 2 * (PN / 2) * 8;                             // two halves when requantising
constexpr int P_OFF_MAX = P_OFF_TB + P_EPI * P_TB;                 // [2 parities][2 groups][128] row maxima
constexpr int P_OFF_BAR = P_OFF_MAX + 2 * 2 * PM * 4;
constexpr int P_NBAR = 2 * P_STAGES + 4 + 1;
constexpr int P_OFF_CNT = P_OFF_BAR + P_NBAR * 8;                  // [8] row-maximum counters
constexpr int P_OFF_TMEM = P_OFF_CNT + P_EPI * 4;
constexpr int P_SMEM = P_OFF_TMEM + 16 + 1024;                     // + alignment slack
static_assert(P_SMEM <= 232448, "shared memory per CTA");

// What becomes of the results in 32 bits: rounded to T; quantised row by row; by one scale; only their rows' largest
// magnitudes kept; quantised by those.
enum { PLAIN, ROWS, STATIC, TOPS, BY_TOPS };

struct PairParams {
    CUtensorMap x, w;                          // box 128 rows x 128 bytes
    CUtensorMap y;                             // box 32 rows x 128 bytes
    const float *xs, *ws, *bias;
    int64_t rows;
    int n, k, relu;
    int y_tma;                                 // y is stored by TMA (16-byte aligned rows)
    void *yp;
    int64_t y_stride;
    float *y_scales;
    float output_scale;
    uint32_t *tops;                            // TOPS, BY_TOPS: bits of the rows' largest magnitudes
};

// One lane of a converged warp, the same each time.  The loops around TMA and MMA are run by whole warps
// and only the instructions themselves by this lane: under a branch on the lane's number the compiler
// has to take their operands through a loop over the lanes, which costs over 100 clocks each.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_store_2d(const void *tmap, const void *smem, int32_t x, int32_t y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(tmap), "r"(smem_u32(smem)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 16 TMEM lanes x 32 columns, four lanes of the warp sharing a row: register 4 j + 2 i + e of lane l is row
// 8 i + l / 4, column 8 j + 2 (l % 4) + e.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// shared memory of this CTA -> shared memory of another one of the cluster, signalled on its barrier
__device__ __forceinline__ void bulk_copy_to(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "r"(smem_u32(src)), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Two floats at a time: one instruction on Blackwell, each half rounded by itself.
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b)
{
    F2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    F2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// 32 rows x 32 columns of sums (two halves of 16 rows) -> results before ReLU, in place.  tb: {scale, scale, bias,
// bias} of the columns' pairs; s: the scales of the thread's four rows.  Four rows share what is read of
// shared memory: with a row to each thread, reading tb alone took as long as the products of K = 512.
__device__ __forceinline__ void affine_16x32(uint32_t (&v)[2][16], const float4 *tb, const float (&s)[4])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 c = tb[4 * j];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t &a = v[h][4 * j + 2 * i], &b = v[h][4 * j + 2 * i + 1];
                const F2 f = {__int2float_rn((int32_t)a), __int2float_rn((int32_t)b)};
                const F2 y = fma2(mul2(f, {s[2 * h + i], s[2 * h + i]}), {c.x, c.y}, {c.z, c.w});
                a = __float_as_uint(y.x);
                b = __float_as_uint(y.y);
            }
    }
}

// largest of three, and of three magnitudes; a NaN stays
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c)
{
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// This warp's 32 rows of 128 bytes from its staging tile to y: by TMA, which drops what lies beyond
// the last row or column.  Where y's rows are not 16-byte aligned, eight lanes have a row: they store the 16-byte
// vectors that its addresses have whole, shifted together from two of the tile's, and then the elements
// before and after them.
template <typename T>
__device__ __forceinline__ void store_tile(const PairParams &p, const uint8_t *tile, int64_t row0, int col0, int lane)
{
    if (p.y_tma) {
        fence_proxy_async_smem();
        __syncwarp();
        if (row0 < p.rows && col0 < p.n && elect_one()) {
            tma_store_2d(&p.y, tile, col0, (int32_t)row0);
            bulk_commit();
        }
    } else {
        constexpr int E = 16 / sizeof(T);
        __syncwarp();
        const int live = (int)min((int64_t)32, p.rows - row0), wide = min(8 * E, p.n - col0);
        for (int r = lane >> 3; r < live; r += 4) {
            T *yr = reinterpret_cast<T *>(p.yp) + (row0 + r) * p.y_stride + col0;
            const int head = (int)((16 - ((uintptr_t)yr & 15)) & 15) / (int)sizeof(T);     // elements before the first vector
            const int whole = head < wide ? (wide - head) / E : 0;                         // vectors
            const int j = lane & 7;
            if (j < whole) {
                const uint4 a = *reinterpret_cast<const uint4 *>(tile + sw128_offset(r, j));
                const uint4 b = *reinterpret_cast<const uint4 *>(tile + sw128_offset(r, j < 7 ? j + 1 : 7));
                *reinterpret_cast<uint4 *>(yr + head + j * E) = shifted16<sizeof(T)>(a, b, head * (uint32_t)sizeof(T));
            }
            for (int e = j; e < wide - whole * E; e += 8) {
                const uint32_t c = e < head ? e : e + whole * E, off = c * (uint32_t)sizeof(T);
                yr[c] = *reinterpret_cast<const T *>(tile + sw128_offset(r, off >> 4) + (off & 15));
            }
        }
        __syncwarp();
    }
}

// the staging tile may be written again
__device__ __forceinline__ void staging_free(const PairParams &p, int lane)
{
    if (p.y_tma && elect_one()) bulk_wait_read();
    __syncwarp();
}

// The (row tile, channel block) pairs of one SM pair, `tile_step` tiles and `block_step` blocks further each time.
struct PairWalk {
    int tile, block, tile_step, block_step, blocks;
    __device__ __forceinline__ void next()
    {
        tile += tile_step;
        block += block_step;
        if (block >= blocks) {
            block -= blocks;
            ++tile;
        }
    }
};

template <typename T, int MODE>
__global__ void __launch_bounds__(P_THREADS, 1) k_pair(const __grid_constant__ PairParams p)
{
    constexpr bool REQUANT = MODE == ROWS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = (uint64_t *)(smem + P_OFF_BAR), *empty = full + P_STAGES;
    uint64_t *acc_full = empty + P_STAGES, *acc_empty = acc_full + 2, *drain = acc_empty + 2;
    uint32_t *max_cnt = (uint32_t *)(smem + P_OFF_CNT);
    uint32_t *tmem_slot = (uint32_t *)(smem + P_OFF_TMEM);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int nu = (p.n + PN - 1) / PN;                        // units per row tile
    const int tiles = (int)((p.rows + 2 * PM - 1) / (2 * PM));
    // this pair's units: every pairs-th, or, requantising, those of every pairs-th row tile
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const PairWalk first = REQUANT ? PairWalk{pair, 0, pairs, 0, nu} : PairWalk{pair / nu, pair % nu, pairs / nu, pairs % nu, nu};
    const int per_step = REQUANT ? nu : 1;                     // units of a step of the walk
    const int nkb = (p.k + PK - 1) / PK;
    const int last_k32 = (p.k - (nkb - 1) * PK + 31) / 32;     // 32-byte steps of the last K block

    if (threadIdx.x == 0) {
        for (int s = 0; s < P_STAGES; ++s) {
            mbar_init(&full[s], 1);                            // leader's producer (+ both CTAs' bytes)
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * P_EPI);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < P_EPI; ++i) max_cnt[i] = 0;
        fence_mbar_init();
        prefetch_tmap(&p.x);
        prefetch_tmap(&p.w);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2 * PN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                            // both CTAs' barriers exist
    tc_fence_after();
    next_may_start();
    previous_done();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (PairWalk g = first; g.tile < tiles && ok; g.next())
            for (int h = 0; h < per_step && ok; ++h) {
                const int row0 = g.tile * 2 * PM + (int)rank * PM;
                const int col0 = (g.block + h) * PN + (int)rank * (PN / 2);
                for (int kb = 0; kb < nkb; ++kb, ++it) {
                    const int s = it % P_STAGES;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(&empty[s], ((it / P_STAGES) & 1) ^ 1)))) break;
                    if (elect_one()) {
                        uint8_t *st = smem + s * P_STAGE;
                        const uint32_t fb = map_to_rank(&full[s], 0);
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * P_STAGE);
                        tma_load_2d_pair(st, &p.x, fb, kb * PK, row0);
                        tma_load_2d_pair(st + P_A, &p.w, fb, kb * PK, col0);
                    }
                    __syncwarp();
                }
            }
        if (!ok) {
            // gave up: loads issued into this CTA may still land, see the fused kernels' abort path
            for (uint32_t i = it > (uint32_t)P_STAGES ? it - P_STAGES : 0; i < it; ++i)
                mbar_wait_cluster_drain(rank == 0 ? &full[i % P_STAGES] : &empty[i % P_STAGES], (i / P_STAGES) & 1);
            spin_ns(100000);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = idesc_i8(2 * PM, PN);
            uint32_t it = 0, uu = 0;
            bool ok = true;
            for (PairWalk g = first; g.tile < tiles && ok; g.next())
                for (int h = 0; h < per_step && ok; ++h, ++uu) {
                    const int ab = uu & 1;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[ab], ((uu >> 1) & 1) ^ 1)))) break;
                    tc_fence_after();
                    const uint32_t d = tmem_base + ab * PN;
                    for (int kb = 0; kb < nkb; ++kb, ++it) {
                        const int s = it % P_STAGES;
                        if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full[s], (it / P_STAGES) & 1)))) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t a = smem_desc_sw128(smem_u32(smem + s * P_STAGE));
                            const uint64_t b = smem_desc_sw128(smem_u32(smem + s * P_STAGE + P_A));
                            const int steps = kb == nkb - 1 ? last_k32 : PK / 32;
#pragma unroll
                            for (int i = 0; i < PK / 32; ++i)          // 32 bytes further: 2 in the descriptor's units
                                if (i < steps) mma_i8_pair(d, a + 2 * i, b + 2 * i, idesc, (kb | i) ? 1u : 0u);
                            mma_commit_pair(&empty[s], 0x3);
                            if (kb == nkb - 1) mma_commit_pair(&acc_full[ab], 0x3);
                        }
                        __syncwarp();
                    }
                }
            if (elect_one()) mma_commit_pair(drain, 0x3);              // completes after every MMA and commit above
        }
        __syncwarp();
    } else {
        const int q = warp & 3, grp = (warp - 2) >> 2;
        uint8_t *tile = smem + P_OFF_OUT + (warp - 2) * 4096;
        float *tb = (float *)(smem + P_OFF_TB + (warp - 2) * P_TB);
        float *row_max = (float *)(smem + P_OFF_MAX);
        const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16) + grp * (PN / 2);
        uint32_t uu = 0, step = 0;
        int have = -1;                                         // the channel block whose scales and bias are in tb
        bool ok = true;
        // this thread's rows of the warp's 32: rl, rl + 8, rl + 16, rl + 24; their scales are read a step ahead
        const int rl = lane >> 2, cl = lane & 3;
        float s_next[4];
        auto read_scales = [&](const PairWalk &w) {
            const int64_t r = (int64_t)w.tile * 2 * PM + rank * PM + q * 32 + rl;
#pragma unroll
            for (int i = 0; i < 4; ++i) s_next[i] = r + 8 * i < p.rows ? p.xs[r + 8 * i] : 0.0f;
        };
        read_scales(first);
        for (PairWalk g = first; g.tile < tiles && ok; ++step) {
            const int64_t row0 = (int64_t)g.tile * 2 * PM + rank * PM + q * 32;
            const int block = g.block;
            const float s[4] = {s_next[0], s_next[1], s_next[2], s_next[3]};
            g.next();
            if (g.tile < tiles) read_scales(g);
            if (block != have) {                               // (requantising, once)
                have = block;
                __syncwarp();
                for (int h = 0; h < (REQUANT ? nu : 1); ++h) {
                    const int c0 = (block + h) * PN + grp * (PN / 2);
#pragma unroll
                    for (int i = 0; i < PN / 2; i += 32) {
                        const int c = c0 + i + lane;
                        float *to = tb + h * PN + (i + lane) / 2 * 4 + (lane & 1);
                        to[0] = c < p.n ? p.ws[c] : 0.0f;
                        to[2] = c < p.n && p.bias ? p.bias[c] : 0.0f;
                    }
                }
                __syncwarp();
            }
            if constexpr (MODE == PLAIN) {
                const int ab = uu & 1;
                const int col0 = block * PN + grp * (PN / 2);
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_full[ab], (uu >> 1) & 1)))) break;
                ++uu;
                tc_fence_after();
                constexpr int COLS = 128 / sizeof(T);          // columns of a staging tile
                auto release = [&]() {                         // the accumulator's last columns are read
                    tc_fence_before();
                    __syncwarp();
                    if (elect_one()) mbar_arrive_cluster_relaxed(map_to_rank(&acc_empty[ab], 0));
                };
                if (col0 >= p.n) release();
#pragma unroll 1
                for (int c = 0; c < PN / 2 && col0 + c < p.n; c += COLS) {
                    staging_free(p, lane);
#pragma unroll 1
                    for (int h = 0; h < COLS; h += 32) {
                        uint32_t v[2][16];
                        tmem_ld_16x32(lane_base + ab * PN + c + h, v[0]);
                        tmem_ld_16x32(lane_base + (16u << 16) + ab * PN + c + h, v[1]);
                        tmem_ld_wait();
                        affine_16x32(v, reinterpret_cast<const float4 *>(tb) + (c + h) / 2 + cl, s);
                        if (p.relu) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                v[i / 16][i % 16] = __float_as_uint(max_nan(__uint_as_float(v[i / 16][i % 16]), 0.0f));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float y0 = __uint_as_float(v[i / 2][4 * j + 2 * (i % 2)]);
                                const float y1 = __uint_as_float(v[i / 2][4 * j + 2 * (i % 2) + 1]);
                                const uint32_t r = rl + 8 * i, at = (h + 8 * j + 2 * cl) * (uint32_t)sizeof(T);
                                uint8_t *to = tile + sw128_offset(r, at >> 4) + (at & 15);
                                if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(to) = make_float2(y0, y1);
                                else *reinterpret_cast<uint32_t *>(to) = pack2(y0, y1, T());
                            }
                    }
                    if (c + COLS >= PN / 2 || col0 + c + COLS >= p.n) release();
                    store_tile<T>(p, tile, row0, col0 + c, lane);
                }
            } else {
                // with ReLU the row's largest result, or 0, is its largest magnitude; the results themselves
                // stay as they are until they are scaled
                float top[4] = {};
                const int halves = REQUANT ? nu : 1, first_block = REQUANT ? 0 : block;
                for (int h = 0; h < halves && ok; ++h) {
                    const int ab = (uu + h) & 1;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_full[ab], ((uu + h) >> 1) & 1)))) break;
                    tc_fence_after();
                    const int live = p.n - (first_block + h) * PN - grp * (PN / 2);            // channels of this warp's half
#pragma unroll 1
                    for (int c = 0; c < PN / 2 && c < live; c += 32) {
                        uint32_t v[2][16];
                        tmem_ld_16x32(lane_base + ab * PN + c, v[0]);
                        tmem_ld_16x32(lane_base + (16u << 16) + ab * PN + c, v[1]);
                        tmem_ld_wait();
                        affine_16x32(v, reinterpret_cast<const float4 *>(tb + h * PN) + c / 2 + cl, s);
                        // columns behind the last channel are no results: sums of zero, which an infinite scale of the
                        // row makes NaN, stay out of its maximum
                        if ((MODE == ROWS || MODE == TOPS) && c + 32 > live) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (c + i / 8 * 8 + 2 * cl + i % 2 >= live) v[i / 4 % 2][i / 8 * 4 + i / 2 % 2 * 2 + i % 2] = 0;
                        }
                        if (MODE != TOPS) {
                            tmem_st_16x32(lane_base + ab * PN + c, v[0]);
                            tmem_st_16x32(lane_base + (16u << 16) + ab * PN + c, v[1]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int i = 0; i < 4 && MODE != BY_TOPS && MODE != STATIC; ++i) {
                                const float y0 = __uint_as_float(v[i / 2][4 * j + 2 * (i % 2)]);
                                const float y1 = __uint_as_float(v[i / 2][4 * j + 2 * (i % 2) + 1]);
                                top[i] = p.relu ? max3_nan(top[i], y0, y1) : max3_abs_nan(top[i], y0, y1);
                            }
                    }
                    if (MODE != TOPS) tmem_st_wait();
                }
                if (!ok) break;
                if constexpr (MODE == TOPS) {
                    tc_fence_before();
                    __syncwarp();
                    if (elect_one()) mbar_arrive_cluster_relaxed(map_to_rank(&acc_empty[uu & 1], 0));
                    ++uu;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                        // magnitudes' bits are in their order, whichever comes first
                        const int64_t row = row0 + rl + 8 * i;
                        if (cl == i && row < p.rows) atomicMax(p.tops + row, magnitude(top[i]));
                    }
                    continue;
                }
                const int mine = q * 32 + lane;
                uint32_t largest = 0;
                if constexpr (MODE == BY_TOPS) {
                    if (row0 + lane < p.rows) largest = p.tops[row0 + lane];
                } else if constexpr (MODE == ROWS) {
                    // the row's other half of the columns is with the other warp of this quarter, which
                    // cannot be more than one tile ahead: two parities of the buffer are enough
                    float *mx = row_max + (step & 1) * 2 * PM;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                        if (cl == i) mx[grp * PM + q * 32 + rl + 8 * i] = top[i];
                    }
                    __syncwarp();
                    if (elect_one()) counter_add_release(&max_cnt[grp * 4 + q], 1);
                    if (!(ok = __all_sync(0xffffffffu, counter_wait(&max_cnt[(grp ^ 1) * 4 + q], step + 1)))) break;
                    largest = magnitude(max_nan(mx[mine], mx[PM + mine]));
                }
                // from here on a thread has a row of its own: its results lie in 16 bytes at a time
                const RowScale rs = row_scale(largest);
                if (MODE != STATIC && grp == 0 && first_block == 0 && row0 + lane < p.rows) p.y_scales[row0 + lane] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
                const bool all_finite = __all_sync(0xffffffffu, rs.finite);
                const float least = MODE == STATIC ? (p.relu ? 0.0f : -128.0f) : p.relu ? kMagic : -INFINITY;
                const float inv = __fdiv_rn(1.0f, p.output_scale);                       // STATIC
                const bool usual = p.output_scale >= 0x1p-100f && p.output_scale <= 0x1p100f;
                for (int h = 0; h < halves; ++h) {
                    const int ab = (uu + h) & 1;
                    const int live = p.n - (first_block + h) * PN - grp * (PN / 2);
                    staging_free(p, lane);
                    auto scale32 = [&](const uint32_t(&now)[32], int c) {
                        uint32_t o[8];
                        if constexpr (MODE == STATIC) static32(now, p.output_scale, inv, usual, least, o);
#pragma unroll
                        for (int i = 0; i < 8 && MODE != STATIC; ++i) {
                            F2 z[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const F2 y = {__uint_as_float(now[4 * i + 2 * j]), __uint_as_float(now[4 * i + 2 * j + 1])};
                                z[j] = fma2(y, {rs.r, rs.r}, {kMagic, kMagic});
                                // ReLU after the multiply-add: results below zero, however far, become 0
                                z[j] = {fmaxf(z[j].x, least), fmaxf(z[j].y, least)};
                            }
                            o[i] = pack4(__float_as_uint(z[0].x), __float_as_uint(z[0].y), __float_as_uint(z[1].x),
                                         __float_as_uint(z[1].y));
                        }
                        if (MODE != STATIC && !all_finite && !rs.finite) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = 0;
                        }
                        *reinterpret_cast<uint4 *>(tile + sw128_offset(lane, c / 16)) = make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4 *>(tile + sw128_offset(lane, c / 16 + 1)) =
                            make_uint4(o[4], o[5], o[6], o[7]);
                    };
                    if (live >= PN / 2) {
                        uint32_t v[2][32];                     // the next columns are on their way meanwhile
                        tmem_ld32(lane_base + ab * PN, v[0]);
#pragma unroll
                        for (int c = 0; c < PN / 2; c += 32) {
                            tmem_ld_wait();
                            if (c + 32 < PN / 2) tmem_ld32(lane_base + ab * PN + c + 32, v[(c / 32 + 1) % 2]);
                            scale32(v[c / 32 % 2], c);
                        }
                    } else {
#pragma unroll 1
                        for (int c = 0; c < live; c += 32) {
                            uint32_t v[32];
                            tmem_ld32(lane_base + ab * PN + c, v);
                            tmem_ld_wait();
                            scale32(v, c);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (elect_one()) mbar_arrive_cluster_relaxed(map_to_rank(&acc_empty[ab], 0));
                    store_tile<int8_t>(p, tile, row0, (first_block + h) * PN + grp * (PN / 2), lane);
                }
                uu += halves;
            }
        }
        if (p.y_tma && elect_one()) bulk_wait_all();
        __syncwarp();
    }
    if (warp == 1) mbar_wait_cluster_drain(drain, 0);
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                            // no CTA leaves while its peer may signal it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 2 * PN);
    }
}

// ---- products of a few tokens, K split over a cluster -------------------------------------------
//
// With few rows the weights are what has to be read, so they take the side of the MMA that is always
// full: a CTA computes 128 channels (M) x BT tokens (N = 16, 32, 64 or 128), and where such tiles are fewer
// than the SMs a cluster of up to eight CTAs splits the tile's K.  Each CTA then owns BT / S of the tokens:
// the others send it their whole sums for them, one bulk copy into its shared memory each, and the owner adds
// the S parts (whole numbers: any order) and writes the results, a warp writing a token's 128 channels at
// once.  No workspace, no counters, one launch.  (Stores to the owner's memory by each thread, and a cluster
// barrier, took 10,500 clocks for 64 tokens.)
//
// Bound by the latency of its chain (set-up, load, MMA, exchange, store), then by what a few CTAs read of L2: 16 rows of
// 512 x 512 in 3.4 us, of 8,192 x 512 in 5.1, of 4,096 x 4,096 in 5.9 (2.8 TB/s of weights).
//
// Requantised rows (ROWS_OUT): the cluster holds all channels of its tokens, C = n / 128 CTAs with S parts of K
// each, at most sixteen CTAs; those that own the same tokens exchange their rows' maxima.
//
// Warps: 0 TMA producer, 1 MMA issuer, then the epilogue: four warps, or from 64 tokens on eight, two for each TMEM lane
// quarter with half of the tokens each (1,000 rows of 1,024 x 1,024: 6.9 us with four, 6.1 with eight; with 16
// tokens eight are slower, 3.55 against 3.4).
struct FewParams {
    CUtensorMap w, x;                          // boxes 128 and BT rows x 128 bytes
    const float *xs, *ws, *bias;
    int64_t rows;
    int n, k, relu, y_vec;                     // y_vec: four results of y lie on a multiple of their size
    void *y;
    int64_t y_stride;
    float output_scale;
    float *y_scales;
    int split;                                 // S, a power of two, at most BT / 2
};

__device__ __forceinline__ void store_one(void *y, int type, int64_t at, float v, float output_scale)
{
    if (type == SC_TYPE_F32) reinterpret_cast<float *>(y)[at] = v;
    else if (type == SC_TYPE_F16) reinterpret_cast<__half *>(y)[at] = __float2half_rn(v);
    else if (type == SC_TYPE_BF16) reinterpret_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<int8_t *>(y)[at] = (int8_t)static_bits(v, output_scale);
}

constexpr int F_MAX_SPLIT = 8;                 // CTAs that split a tile's K
constexpr int F_MAX_CLUSTER = 16;              // CTAs with the same tokens, requantising

template <int BT>
struct FewCfg {
    static constexpr int EPI = BT >= 64 ? 8 : 4;                       // epilogue warps
    static constexpr int GROUPS = EPI / 4, COLS = BT / GROUPS;         // tokens of each group of four
    static constexpr int THREADS = 32 * (2 + EPI);
    static constexpr int STAGES = BT <= 32 ? 9 : BT == 64 ? 7 : 4;
    static constexpr int STAGE = 128 * PK + BT * PK;
    static constexpr int OFF_RECV = STAGES * STAGE;                    // [S - 1][BT / S][128] sums from the other CTAs
    static constexpr int OFF_BAR = OFF_RECV + BT * 128 * 4;
    static constexpr int OFF_TMEM = OFF_BAR + (2 * STAGES + 2) * 8;
    static constexpr int OFF_XS = OFF_TMEM + 16;                       // the tokens' scales
    static constexpr int OFF_MAX = OFF_XS + BT * 4;                    // [C][BT] row maxima
    static constexpr int SMEM = OFF_MAX + F_MAX_CLUSTER * BT * 4 + 1024;
    static constexpr int TMEM = BT < 32 ? 32 : BT;
    static_assert(SMEM <= 232448 && BT * 128 * 4 <= STAGES * STAGE, "shared memory per CTA");
};

// a barrier of the epilogue's threads, which all reach it
template <int THREADS>
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }

template <typename T>
__device__ __forceinline__ T result(float y, float output_scale)
{
    if constexpr (sizeof(T) == 1) return (T)static_bits(y, output_scale);
    else return from_f32<T>(y);
}

template <int BT, typename T, bool ROWS_OUT>
__global__ void __launch_bounds__(FewCfg<BT>::THREADS, 1) k_few(const __grid_constant__ FewParams p)
{
    using C = FewCfg<BT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = (uint64_t *)(smem + C::OFF_BAR), *empty = full + C::STAGES, *done = empty + C::STAGES;
    uint64_t *got = done + 1;                                          // the other CTAs' sums
    uint32_t *tmem_slot = (uint32_t *)(smem + C::OFF_TMEM);
    int32_t *recv = (int32_t *)(smem + C::OFF_RECV);
    float *xs = (float *)(smem + C::OFF_XS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = p.split, own = BT / S;
    // the cluster is the grid's x: the parts of K, and requantising those of every channel tile
    const int part = blockIdx.x & (S - 1), tile0 = blockIdx.x - part;
    const int c0 = (ROWS_OUT ? tile0 / S : blockIdx.y) * 128;
    const bool alone = gridDim.x == 1;
    const int64_t t0 = (int64_t)blockIdx.z * BT;
    const int nkb_all = (p.k + PK - 1) / PK;
    const int kb0 = (int)((int64_t)nkb_all * part / S), kb1 = (int)((int64_t)nkb_all * (part + 1) / S);
    const int last_k32 = (p.k - (nkb_all - 1) * PK + 31) / 32;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        mbar_init(got, 1);
        fence_mbar_init();
        if (S > 1) mbar_arrive_expect_tx(got, (uint32_t)((S - 1) * own * 128 * 4));
        prefetch_tmap(&p.w);
        prefetch_tmap(&p.x);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (!alone) cluster_arrive();                                      // this CTA runs: its memory may be written
    const uint32_t tmem = *tmem_slot;
    next_may_start();
    previous_done();

    if (warp == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % C::STAGES;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1)))) break;
            if (elect_one()) {
                uint8_t *st = smem + s * C::STAGE;
                mbar_arrive_expect_tx(&full[s], C::STAGE);
                tma_load_2d(st, &p.w, &full[s], kb * PK, c0);
                tma_load_2d(st + 128 * PK, &p.x, &full[s], kb * PK, (int)t0);
            }
            __syncwarp();
        }
        if (!ok) {                                                     // loads still landing, then end
            for (uint32_t i = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; i < it; ++i)
                mbar_wait_cluster_drain(&full[i % C::STAGES], (i / C::STAGES) & 1);
            spin_ns(100000);
        }
        __syncwarp();
        if (!alone) cluster_wait();
        if (ROWS_OUT && !alone) cluster_sync();                            // the rows' maxima
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_i8(128, BT);
        uint32_t it = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % C::STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (it / C::STAGES) & 1))) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t a = smem_desc_sw128(smem_u32(smem + s * C::STAGE));
                const uint64_t b = smem_desc_sw128(smem_u32(smem + s * C::STAGE + 128 * PK));
                const int steps = kb == nkb_all - 1 ? last_k32 : PK / 32;
#pragma unroll
                for (int i = 0; i < PK / 32; ++i)
                    if (i < steps) mma_i8(tmem, a + 2 * i, b + 2 * i, idesc, (it | i) ? 1u : 0u);
                mma_commit(&empty[s]);
            }
            __syncwarp();
        }
        if (elect_one()) mma_commit(done);                             // after every MMA above, given up or not
        __syncwarp();
        if (!alone) cluster_wait();
        if (ROWS_OUT && !alone) cluster_sync();                            // the rows' maxima
    } else {
        // a channel is a lane of TMEM; tokens are the columns
        const int q = warp & 3, grp = (warp - 2) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
        for (int i = threadIdx.x - 64; i < BT; i += 32 * C::EPI) xs[i] = t0 + i < p.rows ? p.xs[t0 + i] : 0.0f;
        if (!ROWS_OUT && S == 1) {
            const int ch = c0 + q * 32 + lane;
            const float t = ch < p.n ? p.ws[ch] : 0.0f, b = ch < p.n && p.bias ? p.bias[ch] : 0.0f;
            epilogue_sync<32 * C::EPI>();                              // the scales are there; no warp has left
            mbar_wait(done, 0);
            __syncwarp();
            tc_fence_after();
            T *to = reinterpret_cast<T *>(p.y) + (t0 + grp * C::COLS) * p.y_stride + ch;
#pragma unroll 1
            for (int j0 = grp * C::COLS; j0 < (grp + 1) * C::COLS && t0 + j0 < p.rows; j0 += 16) {
                uint32_t v[16];
                tmem_ld16(taddr + j0, v);
                tmem_ld_wait();
                const int live = (int)min((int64_t)16, p.rows - t0 - j0);
                if (ch < p.n) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j < live)
                            to[j * p.y_stride] = result<T>(affine((int32_t)v[j], xs[j0 + j], t, b, p.relu), p.output_scale);
                }
                to += 16 * p.y_stride;
                __syncwarp();
            }
            tc_fence_before();
        } else {
            float t[4] = {}, b[4] = {};                                // of this lane's four channels
            const int ch = c0 + 4 * lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ch + i < p.n) {
                    t[i] = p.ws[ch + i];
                    b[i] = p.bias ? p.bias[ch + i] : 0.0f;
                }
            mbar_wait(done, 0);
            __syncwarp();
            tc_fence_after();
            // the stages are read: their memory takes the sums, token by token
            int32_t *sums = (int32_t *)smem + q * 32 + lane;
#pragma unroll 1
            for (int j0 = grp * C::COLS; j0 < (grp + 1) * C::COLS; j0 += 16) {
                uint32_t v[16];
                tmem_ld16(taddr + j0, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[(j0 + j) * 128] = (int32_t)v[j];
            }
            tc_fence_before();
            fence_proxy_async_smem();
            epilogue_sync<32 * C::EPI>();                              // no warp has left
            if (!alone) cluster_wait();                                // every CTA of the cluster runs
            if (S > 1) {
                if (warp == 2 && elect_one()) {
                    for (int r = 1; r < S; ++r) {                      // to each owner, a different one first
                        const int to = (part + r) & (S - 1);
                        bulk_copy_to(map_to_rank(recv + (part < to ? part : part - 1) * own * 128, (uint32_t)(tile0 + to)),
                                     (int32_t *)smem + to * own * 128, (uint32_t)(own * 128 * 4),
                                     map_to_rank(got, (uint32_t)(tile0 + to)));
                    }
                }
                __syncwarp();
                mbar_wait_cluster(got, 0);
                __syncwarp();
            }
            auto results = [&](int j, float(&y)[4]) {
                int4 sum = *reinterpret_cast<const int4 *>((const int32_t *)smem + (part * own + j) * 128 + 4 * lane);
                for (int i = 0; i < S - 1; ++i) {
                    const int4 o = *reinterpret_cast<const int4 *>(recv + (i * own + j) * 128 + 4 * lane);
                    sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
                }
                const float s = xs[part * own + j];
                y[0] = affine(sum.x, s, t[0], b[0], p.relu);
                y[1] = affine(sum.y, s, t[1], b[1], p.relu);
                y[2] = affine(sum.z, s, t[2], b[2], p.relu);
                y[3] = affine(sum.w, s, t[3], b[3], p.relu);
            };
            auto store4 = [&](int64_t r, const T(&o)[4]) {
                T *to = reinterpret_cast<T *>(p.y) + r * p.y_stride + ch;
                if (p.y_vec && ch + 4 <= p.n) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(o);
                    else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(o);
                    else *reinterpret_cast<uint32_t *>(to) = *reinterpret_cast<const uint32_t *>(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (ch + i < p.n) to[i] = o[i];
                }
            };
            const int64_t first = t0 + part * own;                     // the CTA's first own token
            if constexpr (!ROWS_OUT) {
#pragma unroll 2
                for (int j = warp - 2; j < own; j += C::EPI) {
                    float y[4];
                    results(j, y);
                    if (first + j >= p.rows) continue;
                    __align__(16) T o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = result<T>(y[i], p.output_scale);
                    store4(first + j, o);
                }
            } else {
                float y[BT / C::EPI][4];
                uint32_t *mx = (uint32_t *)(smem + C::OFF_MAX);
                const int tiles = gridDim.x / S;
#pragma unroll
                for (int u = 0; u < BT / C::EPI; ++u) {
                    const int j = warp - 2 + C::EPI * u;
                    if (j >= own) break;
                    results(j, y[u]);
                    // channels behind the last one are sums of zero, which an infinite scale of the row makes NaN
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (ch + i < p.n) top = max(top, magnitude(y[u][i]));
                    top = __reduce_max_sync(0xffffffffu, top);
                    if (lane < tiles) {
                        const uint32_t at = map_to_rank(mx + tile0 / S * BT + j, (uint32_t)(lane * S + part));
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(top) : "memory");
                    }
                }
                if (!alone) cluster_sync();
                else __syncwarp();
#pragma unroll
                for (int u = 0; u < BT / C::EPI; ++u) {
                    const int j = warp - 2 + C::EPI * u;
                    if (j >= own || first + j >= p.rows) break;
                    uint32_t top = 0;
                    for (int i = 0; i < tiles; ++i) top = max(top, mx[i * BT + j]);
                    const RowScale rs = row_scale(top);
                    __align__(4) T o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = rs.finite ? (T)quantise_bits(y[u][i], rs.r) : (T)0;
                    store4(first + j, o);
                    if (tile0 == 0 && lane == 0) p.y_scales[first + j] = rs.finite ? rs.s : __uint_as_float(0x7fc00000u);
                }
            }
        }
    }
    __syncthreads();
    if (!ROWS_OUT && !alone) cluster_sync();                           // what this CTA sent has been received
    if (warp == 1) {
        mbar_wait_cluster_drain(done, 0);
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

}  // namespace
}  // namespace sc
