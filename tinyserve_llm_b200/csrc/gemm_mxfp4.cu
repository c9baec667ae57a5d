// Products y = x . W^T on the fifth-generation tensor cores with W in microscaled 4-bit floating point (mxfp4.cuh), for any number of
// rows of x.  Two forms of the same kernel:
//
//   rows in bfloat16: eight warps read W's codes and scales from global memory, make bfloat16 numbers of them (exactly) and lay them into
//   shared memory in the 128-byte swizzle that TMA would give them, where tcgen05.mma kind::f16 reads them; x comes by TMA.
//   rows in four bits too: codes of both sides come by TMA as they are, 256 numbers a row of 128 bytes, and tcgen05.mma kind::mxf4 multiplies
//   them, four times as many a cycle.  The scales it reads from tensor memory: two warps gather a stage's bytes into shared memory, 16 bytes
//   for lane l of which bytes 4 j .. 4 j + 3 belong to row 32 j + l, and tcgen05.cp hands them to all four quarters of the lanes.
//
// W's rows are the M of the MMA, 128 a tile, and x's rows its N (BN: 32 to 256), so that a few rows of x cost an MMA of few columns and
// not one of 128 rows: accumulator lane = row of W, column = row of x.  A stage of the ring is 128 bytes of a row on either side.
//
// Gated (y = act(x Wgate^T, x Wup^T), W = [gate rows | up rows]): a tile holds 16 gate rows, the 16 up rows that belong to them, and so
// on, so that a gate lies 16 lanes before its up in the same warp's quarter of tensor memory and one shuffle brings them together.
//
// Many tiles: persistent, one CTA an SM, two accumulators, so that a tile's epilogue runs under the next one's MMAs.  Few tiles: a cluster
// of `splits` CTAs takes a tile, each its share of K, and leaves its sums in its own shared memory; each CTA then adds up a share of the
// columns from all of them, in the order of their ranks.  Nothing of that needs a workspace in global memory, and the order is fixed.
//
// Every wait on an mbarrier gives up after about two seconds, records where in an error word the host can read, and the CTA goes on to
// free its tensor memory and return.
#include "mxfp4.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int BM = 128, ROW = 128;                    // rows of W a tile; bytes of a row a stage holds
constexpr int EPI_WARPS = 8, SPREAD_WARPS = 8, SCALE_WARPS = 2;
constexpr int A_BYTES = BM * ROW;
constexpr int AHEAD = 4;                               // stages whose codes a spreading thread has on their way

struct MxParams {
    const uint8_t* w_codes;
    const uint8_t* w_scales;
    long long w_ld_codes, w_ld_scales;
    const uint8_t* x_scales;                           // rows in four bits
    long long x_ld_scales;
    void* y;
    long long ldy;
    int M, N, K, blocks;                               // rows of x, rows of W, columns, blocks of 32 of them
    int inter;                                         // gated: rows of W per half
    int out_f32, act;
    float act_limit, act_alpha;
    int splits;
    int* error;
};

__device__ __forceinline__ void umma_bf16(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void umma_mxf4(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(leader) : "memory");
}
// 32 rows of 16 bytes of shared memory into four columns of tensor memory, the same for each quarter of the lanes.
__device__ __forceinline__ void copy_scales(uint32_t leader, uint32_t tmem, uint64_t desc) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}"
                 ::"r"(tmem), "l"(desc), "r"(leader) : "memory");
}
// Descriptor of 32 rows of 16 bytes that lie one behind the other: groups of eight rows 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t scale_desc(const void* at) {
    return (uint64_t)((smem_u32(at) & 0x3FFFF) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// bfloat16 x bfloat16 -> float32, both K-major.
__device__ __forceinline__ uint32_t desc_bf16(int n) { return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(BM >> 4) << 24; }
// e2m1 x e2m1 -> float32 with scales of power-of-two bytes, two a row and MMA; `pair`: which two of the four bytes of a column.
__device__ __forceinline__ uint32_t desc_mxf4(int n, int pair) {
    return (uint32_t)(2 * pair) << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(BM >> 7) << 27 | (uint32_t)(2 * pair) << 29;
}

template <int COLS>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[COLS]);
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
}

__device__ __forceinline__ float gated_value(const MxParams& p, float g, float u) {
    if (p.act == TS_ACT_SILU) return __fdividef(g, 1.f + __expf(-g)) * u;
    return ts_gated_activation(p.act, g, u, p.act_limit, p.act_alpha);
}

// The row of W in lane l of a tile whose first output column is f0.
template <bool GATED>
__device__ __forceinline__ int row_of(const MxParams& p, int f0, int l) {
    if (!GATED) return f0 + l;
    return f0 + (l >> 5) * 16 + (l & 15) + ((l & 16) ? p.inter : 0);
}

template <bool BOTH>
__host__ __device__ constexpr int threads_of() { return 64 + 32 * (EPI_WARPS + (BOTH ? SCALE_WARPS : SPREAD_WARPS)); }
template <bool BOTH, int BN>
__host__ __device__ constexpr int scale_columns() { return BOTH ? 8 + 8 * ((BN + 127) / 128) : 0; }       // of tensor memory, a stage
template <bool BOTH, int BN>
__host__ __device__ constexpr int stage_bytes() { return A_BYTES + BN * ROW + 128 * scale_columns<BOTH, BN>(); }
__host__ __device__ constexpr int power_of_two(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

template <bool BOTH, bool GATED, int BN, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(threads_of<BOTH>(), 1)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, MxParams p) {
    constexpr int BK = BOTH ? 256 : 64;                               // columns of K a stage holds
    constexpr int B_BYTES = BN * ROW, SCALE_COLS = scale_columns<BOTH, BN>(), SCALE_BYTES = SCALE_COLS * 128;
    constexpr int ACCUMULATORS = SPLIT ? 1 : 2, OUTS = GATED ? BM / 2 : BM;
    constexpr int TMEM_USED = ACCUMULATORS * BN + STAGES * SCALE_COLS, TMEM_COLS = power_of_two(TMEM_USED);
    static_assert(TMEM_USED <= 512, "tensor memory has 512 columns");
    static_assert(!SPLIT || BM * BN * 4 <= STAGES * (A_BYTES + B_BYTES), "a split tile's sums go where the ring was");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int failed;

    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* scale_ring = stages + STAGES * (A_BYTES + B_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outs = GATED ? p.inter : p.N;
    const int x_tiles = (p.M + BN - 1) / BN, num_tiles = x_tiles * ((outs + OUTS - 1) / OUTS);
    const int all_kblocks = (p.blocks * MX_BLOCK + BK - 1) / BK;
    const int rank = SPLIT ? (int)pair_rank() : 0;
    const int first_tile = SPLIT ? (int)blockIdx.x / p.splits : (int)blockIdx.x, tile_step = SPLIT ? num_tiles : (int)gridDim.x;
    const int kb0 = SPLIT ? (int)((long long)all_kblocks * rank / p.splits) : 0;
    const int kb1 = SPLIT ? (int)((long long)all_kblocks * (rank + 1) / p.splits) : all_kblocks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1 + (BOTH ? SCALE_WARPS : SPREAD_WARPS));   // the producer's bytes, and the warps that write shared memory
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tmem_full_bar[b], 1);
            mbar_init(&tmem_empty_bar[b], EPI_WARPS);
        }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_base_slot;

    chain_wait();                                    // x, or the weights themselves, may come from a kernel ahead on the stream
    chain_release();

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0) {
            int kg = 0;                              // stages filled so far, over all tiles
            for (int tile = first_tile; tile < num_tiles && !failed; tile += tile_step) {
                const int t0 = (tile % x_tiles) * BN, f0 = (tile / x_tiles) * OUTS;
                for (int kb = kb0; kb < kb1; ++kb, ++kg) {
                    const int s = kg % STAGES;
                    if (!mbar_wait(&empty_bar[s], ((kg / STAGES) & 1) ^ 1, p.error, 41)) { failed = 1; break; }
                    unsigned char* a_tile = stages + s * (A_BYTES + B_BYTES);
                    mbar_expect_tx(&full_bar[s], (BOTH ? A_BYTES : 0) + B_BYTES);
                    if (BOTH) {
                        if (GATED) {
#pragma unroll
                            for (int g = 0; g < BM / 16; ++g)                       // 16 gate rows, their up rows, ...
                                tma_load_2d(a_tile + g * 16 * ROW, &map_w, &full_bar[s], kb * ROW, row_of<true>(p, f0, g * 16));
                        } else {
                            tma_load_2d(a_tile, &map_w, &full_bar[s], kb * ROW, f0);
                        }
                    }
                    tma_load_2d(a_tile + A_BYTES, &map_x, &full_bar[s], BOTH ? kb * ROW : kb * BK, t0);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint32_t leader = elect_one();
        const uint32_t tmem_scales = tmem_base + ACCUMULATORS * BN;
        bool ok = true;                              // the same in all lanes
        int kg = 0, iter = 0;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++iter) {
            const int buf = SPLIT ? 0 : iter & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&tmem_empty_bar[buf], ((iter >> 1) & 1) ^ 1, p.error, 44) && !failed);
            if (!ok) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + buf * BN;
            for (int kb = kb0; kb < kb1; ++kb, ++kg) {
                const int s = kg % STAGES;
                ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[s], (kg / STAGES) & 1, p.error, 42));
                if (!ok) { failed = 1; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t a_desc = smem_desc(stages + s * (A_BYTES + B_BYTES));
                const uint64_t b_desc = smem_desc(stages + s * (A_BYTES + B_BYTES) + A_BYTES);
                if (BOTH) {
                    // a stage's scales have columns of their own: they are free when the stage is, once the MMAs that read them have retired
                    constexpr int X_SETS = (BN + 127) / 128;
                    const uint32_t sa = tmem_scales + s * SCALE_COLS, sb = sa + 8;
                    const unsigned char* from = scale_ring + s * SCALE_BYTES;
#pragma unroll
                    for (int i = 0; i < 2 + 2 * X_SETS; ++i) copy_scales(leader, sa + 4 * i, scale_desc(from + 512 * i));
#pragma unroll
                    for (int k = 0; k < 4; ++k)      // 64 columns of K are 32 bytes and two scales a row
                        umma_mxf4(leader, tmem_d, a_desc + 2 * k, b_desc + 2 * k, desc_mxf4(BN, k & 1), sa + (k >> 1) * 4,
                                  sb + (k >> 1) * 4 * X_SETS, (kb > kb0) | (k != 0));
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(leader, tmem_d, a_desc + 2 * k, b_desc + 2 * k, desc_bf16(BN), (kb > kb0) | (k != 0));
                }
                if (leader) umma_commit(&empty_bar[s]);
            }
            if (leader) umma_commit(&tmem_full_bar[buf]);
        }
    } else if (warp < 2 + EPI_WARPS) {
        // ---------------------------------------------------------------- epilogue
        const int quarter = warp & 3, side = (warp - 2) >> 2;         // the 32 lanes this warp may read; which half of the columns
        int iter = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++iter) {
            const int buf = SPLIT ? 0 : iter & 1;
            const int t0 = (tile % x_tiles) * BN, f0 = (tile / x_tiles) * OUTS;
            if (!mbar_wait(&tmem_full_bar[buf], (iter >> 1) & 1, p.error, 43) || failed) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t lane_addr = tmem_base + buf * BN + side * (BN / 2) + ((uint32_t)(quarter * 32) << 16);
            const int f = GATED ? f0 + quarter * 16 + (lane & 15) : f0 + quarter * 32 + lane;
#pragma unroll 1
            for (int c0 = 0; c0 < BN / 2; c0 += 16) {
                uint32_t acc[16];
                __syncwarp();
                tmem_ld<16>(lane_addr + c0, acc);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (!SPLIT && c0 + 16 == BN / 2) {                    // the last of it: the accumulator goes back before the stores
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tmem_empty_bar[buf]);
                }
                const int c = side * (BN / 2) + c0, t = t0 + c;
                if (SPLIT) {
                    float* sums = reinterpret_cast<float*>(stages);   // [column][lane]
#pragma unroll
                    for (int j = 0; j < 16; ++j) sums[(c + j) * BM + quarter * 32 + lane] = __uint_as_float(acc[j]);
                } else if (GATED) {
                    __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)t * p.ldy + f;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {                 // the lower half of the lanes finishes column j, the upper one j + 1
                        const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(lane < 16 ? acc[j + 1] : acc[j]), 16);
                        const float mine = __uint_as_float(lane < 16 ? acc[j] : acc[j + 1]);
                        const float v = lane < 16 ? gated_value(p, mine, other) : gated_value(p, other, mine);
                        const int jj = j + (lane >> 4);
                        if (t + jj < p.M && f < outs) out[(long long)jj * p.ldy] = __float2bfloat16_rn(v);
                    }
                } else if (f < outs) {
                    if (p.out_f32) {
                        float* out = (float*)p.y + (long long)t * p.ldy + f;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (t + j < p.M) out[(long long)j * p.ldy] = __uint_as_float(acc[j]);
                    } else {
                        __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)t * p.ldy + f;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (t + j < p.M) out[(long long)j * p.ldy] = __float2bfloat16_rn(__uint_as_float(acc[j]));
                    }
                }
            }
        }
    } else if (BOTH) {
        // ---------------------------------------------------------------- scales: one warp for W's, one for x's
        const bool of_x = warp == 3 + EPI_WARPS;
        const uint8_t* base = of_x ? p.x_scales : p.w_scales;
        const long long ld = of_x ? p.x_ld_scales : p.w_ld_scales;
        constexpr int X_SETS = (BN + 127) / 128, ROWS = 4 * X_SETS;   // rows a lane gathers (W: the first four)
        const int sets = of_x ? X_SETS : 1;
        bool ok = true;
        int kg = 0;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            const int t0 = (tile % x_tiles) * BN, f0 = (tile / x_tiles) * OUTS;
            const uint8_t* row[ROWS];
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
                const int l = j * 32 + lane;
                int r = of_x ? min(t0 + min(l, BN - 1), p.M - 1) : min(row_of<GATED>(p, f0, min(l, BM - 1)), p.N - 1);
                row[j] = base + (long long)r * ld;
            }
            auto load = [&](int kb, uint2 (&v)[ROWS]) {               // the stage's eight scales of each row; behind the last block: 1
#pragma unroll
                for (int j = 0; j < ROWS; ++j) {
                    if (j >= 4 * sets) continue;
                    const int b = kb * 8;
                    if (b + 8 <= p.blocks) {
                        v[j] = *reinterpret_cast<const uint2*>(row[j] + b);
                    } else {
                        uint32_t half[2] = {0x7f7f7f7fu, 0x7f7f7f7fu};
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (b + i < p.blocks) half[i >> 2] = (half[i >> 2] & ~(0xffu << (8 * (i & 3)))) | (uint32_t)row[j][b + i] << (8 * (i & 3));
                        v[j] = make_uint2(half[0], half[1]);
                    }
                }
            };
            uint2 now[ROWS], next[ROWS];
            load(kb0, now);
            for (int kb = kb0; kb < kb1; ++kb, ++kg) {
                const int s = kg % STAGES;
                if (kb + 1 < kb1) load(kb + 1, next);
                ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[s], ((kg / STAGES) & 1) ^ 1, p.error, 45) && !failed);
                if (!ok) { failed = 1; break; }
                unsigned char* to = scale_ring + s * SCALE_BYTES + (of_x ? 1024 : 0);
#pragma unroll
                for (int b = 0; b < X_SETS; ++b) {
                    if (b >= sets) continue;
                    *reinterpret_cast<uint4*>(to + b * 512 + lane * 16) = make_uint4(now[4 * b].x, now[4 * b + 1].x, now[4 * b + 2].x, now[4 * b + 3].x);
                    *reinterpret_cast<uint4*>(to + (sets + b) * 512 + lane * 16) =
                        make_uint4(now[4 * b].y, now[4 * b + 1].y, now[4 * b + 2].y, now[4 * b + 3].y);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full_bar[s]);
#pragma unroll
                for (int j = 0; j < ROWS; ++j) now[j] = next[j];
            }
        }
    } else {
        // ---------------------------------------------------------------- codes to bfloat16 numbers
        const int id = threadIdx.x - 32 * (2 + EPI_WARPS), l = id >> 1, part = id & 1;       // a row of the tile, one of a stage's two blocks
        bool ok = true;
        int kg = 0;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            const int f0 = (tile / x_tiles) * OUTS, row = min(row_of<GATED>(p, f0, l), p.N - 1);
            const uint8_t* codes = p.w_codes + (long long)row * p.w_ld_codes;
            const uint8_t* scales = p.w_scales + (long long)row * p.w_ld_scales;
            uint4 code[AHEAD];
            uint32_t scale[AHEAD];
            auto load = [&](int kb, int u) {
                const int b = kb * 2 + part;
                const bool there = kb < kb1 && b < p.blocks;
                code[u] = make_uint4(0, 0, 0, 0);
                scale[u] = 0;
                if (there) {
                    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(code[u].x), "=r"(code[u].y), "=r"(code[u].z), "=r"(code[u].w) : "l"(codes + (long long)b * 16));
                    scale[u] = __ldg(scales + b);
                }
            };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) load(kb0 + u, u);
            for (int kbs = kb0; kbs < kb1 && ok; kbs += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    if (kbs + u >= kb1 || !ok) break;
                    const int s = kg % STAGES;
                    const uint32_t w[4] = {code[u].x, code[u].y, code[u].z, code[u].w}, sc = scale[u];
                    load(kbs + u + AHEAD, u);
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[s], ((kg / STAGES) & 1) ^ 1, p.error, 46) && !failed);
                    if (!ok) { failed = 1; break; }
                    unsigned char* to = stages + s * (A_BYTES + B_BYTES) + l * ROW;
                    const MxFactor factor = mx_factor_large(sc);
                    const bool large = __any_sync(0xffffffffu, mx_large(sc));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {                      // eight numbers, a 16-byte piece of the row
                        uint32_t q[4];
                        mx_spread(w[j], q);
#pragma unroll
                        for (int i = 0; i < 4; ++i) q[i] = mx_mul(q[i], factor.first);
                        if (large) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) q[i] = mx_mul(q[i], factor.more);
                        }
                        const uint4 v = make_uint4(__byte_perm(q[0], q[1], 0x5410), __byte_perm(q[2], q[3], 0x5410),
                                                   __byte_perm(q[0], q[1], 0x7632), __byte_perm(q[2], q[3], 0x7632));
                        *reinterpret_cast<uint4*>(to + (((part * 4 + j) ^ (l & 7)) << 4)) = v;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full_bar[s]);
                    ++kg;
                }
            }
        }
    }
    __syncwarp();
    if (SPLIT) {
        pair_sync();                                 // every CTA's sums are in its shared memory
        if (warp >= 2 && warp < 2 + EPI_WARPS) {
            const int id = threadIdx.x - 64, tile = first_tile;
            const int t0 = (tile % x_tiles) * BN, f0 = (tile / x_tiles) * OUTS, columns = min(BN, p.M - t0);
            const uint32_t sums = smem_u32(stages);
            auto total = [&](int column, int l) {
                float v = 0.f;
                for (int r = 0; r < p.splits; ++r) {
                    uint32_t remote;
                    float part;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(sums + (uint32_t)(column * BM + l) * 4), "r"(r));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(remote));
                    v += part;
                }
                return v;
            };
            const int f = GATED ? id & 63 : id & 127;
            if (f0 + f < outs) {
                for (int c = rank + p.splits * (id / OUTS); c < columns; c += p.splits * (32 * EPI_WARPS / OUTS)) {
                    const long long at = (long long)(t0 + c) * p.ldy + f0 + f;
                    if (GATED) {
                        const int l = (f >> 4) * 32 + (f & 15);
                        ((__nv_bfloat16*)p.y)[at] = __float2bfloat16_rn(gated_value(p, total(c, l), total(c, l + 16)));
                    } else if (p.out_f32) {
                        ((float*)p.y)[at] = total(c, f);
                    } else {
                        ((__nv_bfloat16*)p.y)[at] = __float2bfloat16_rn(total(c, f));
                    }
                }
            }
        }
        __syncwarp();
        pair_sync();                                 // nobody reads another CTA's sums any more
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (failed) {                                    // copies and MMAs still under way get some half a millisecond before the CTA goes
        const long long start = clock64();
        while (clock64() - start < 1000000) {}
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

template <bool BOTH, bool GATED, int BN, int STAGES, bool SPLIT>
int launch(const CUtensorMap& map_w, const void* x, long long ldx, MxParams& p, int sms, cudaStream_t stream) {
    CUtensorMap map_x;
    if (BOTH) {
        if (make_tile_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, p.M, (long long)p.blocks * 16, ldx, BN, "gemm_mxfp4")) return 1;
    } else {
        if (make_tile_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, p.M, p.K, ldx, BN, "gemm_mxfp4")) return 1;
    }
    auto kernel = gemm_mxfp4_kernel<BOTH, GATED, BN, STAGES, SPLIT>;
    const size_t smem = (size_t)STAGES * stage_bytes<BOTH, BN>() + 1024;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return ts_fail("gemm_mxfp4: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    const long long outs = GATED ? p.inter : p.N, per = GATED ? BM / 2 : BM;
    const long long tiles = ((p.M + BN - 1) / BN) * ((outs + per - 1) / per);
    TS_REQUIRE(tiles * (SPLIT ? p.splits : 1) <= 0x7fffffffll, "gemm_mxfp4: too many tiles");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(SPLIT ? tiles * p.splits : (tiles < sms ? tiles : sms)));
    cfg.blockDim = dim3(threads_of<BOTH>());
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT ? p.splits : 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ts_chaining_enabled() ? 2 : 1;
    TS_CHAINED_CHECK("gemm_mxfp4", cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p));
    return 0;
}

template <bool BOTH, bool GATED>
int dispatch(const CUtensorMap& map_w, const void* x, long long ldx, MxParams& p, cudaStream_t stream) {
    int sms = 148, device = 0;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    constexpr int WIDE = BOTH ? 192 : 256;
    const long long outs = GATED ? p.inter : p.N, per = GATED ? BM / 2 : BM, w_tiles = (outs + per - 1) / per;
    const int kblocks = (p.blocks * MX_BLOCK + (BOTH ? 255 : 63)) / (BOTH ? 256 : 64);
    if (p.M > 128 && w_tiles * ((p.M + WIDE - 1) / WIDE) * 4 >= 3ll * sms)
        return launch<BOTH, GATED, WIDE, BOTH ? 5 : 4, false>(map_w, x, ldx, p, sms, stream);
    const int bn = p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
    const long long tiles = w_tiles * ((p.M + bn - 1) / bn);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= kblocks) splits *= 2;
    p.splits = splits;
    if (bn == 32) return launch<BOTH, GATED, 32, 8, true>(map_w, x, ldx, p, sms, stream);
    if (bn == 64) return launch<BOTH, GATED, 64, 8, true>(map_w, x, ldx, p, sms, stream);
    return launch<BOTH, GATED, 128, 6, true>(map_w, x, ldx, p, sms, stream);
}

}  // namespace

// y = x . W^T (gated 0; y [M, N], bfloat16 or float32) or y = act(x Wgate^T, x Wup^T) with W = [gate rows | up rows] (gated 1; y [M, N / 2],
// bfloat16; TS_ACT_* of common.cuh).  x: bfloat16 [M, K], rows ldx elements apart, if x_scales is null; else codes, rows ldx bytes apart,
// and scales.  K a multiple of 8; rows of codes and of scales start 16-byte aligned, and so do x and its rows.
TS_API int ts_gemm_mxfp4(const void* w_codes, const void* w_scales, long long w_ld_codes, long long w_ld_scales, const void* x, long long ldx,
                         const void* x_scales, long long x_ld_scales, void* y, int M, int N, int K, long long ldy, int gated, int act,
                         float limit, float alpha, int out_dtype, int* error, cudaStream_t stream) {
    TS_REQUIRE(M >= 0 && N > 0 && K > 0 && K <= 0x3fffffff, "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
    TS_REQUIRE(out_dtype == TS_BF16 || (out_dtype == TS_F32 && !gated), "gemm_mxfp4: unsupported output dtype %d", out_dtype);
    TS_REQUIRE(!gated || (N % 2 == 0 && act >= TS_ACT_SILU && act <= TS_ACT_LAST), "gemm_mxfp4: N=%d, activation %d", N, act);
    TS_REQUIRE(x_scales || K % 8 == 0, "gemm_mxfp4: K=%d is not a multiple of 8", K);
    TS_REQUIRE(error != nullptr, "gemm_mxfp4: an error word is needed");
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    TS_REQUIRE((uintptr_t)w_codes % 16 == 0 && w_ld_codes % 16 == 0 && w_ld_codes >= (long long)blocks * 16 && (uintptr_t)w_scales % 16 == 0 &&
                   w_ld_scales % 16 == 0 && w_ld_scales >= blocks,
               "gemm_mxfp4: rows of W's codes and scales must start 16-byte aligned (%lld and %lld bytes apart)", w_ld_codes, w_ld_scales);
    TS_REQUIRE((uintptr_t)x % 16 == 0 && (x_scales ? ldx % 16 == 0 && ldx >= (long long)blocks * 16 : ldx % 8 == 0 && ldx >= K),
               "gemm_mxfp4: rows of x must start 16-byte aligned (stride %lld)", ldx);
    TS_REQUIRE(!x_scales || ((uintptr_t)x_scales % 16 == 0 && x_ld_scales % 16 == 0 && x_ld_scales >= blocks),
               "gemm_mxfp4: rows of x's scales must start 16-byte aligned (%lld bytes apart)", x_ld_scales);
    if (M == 0) return 0;
    MxParams p{(const uint8_t*)w_codes, (const uint8_t*)w_scales, w_ld_codes, w_ld_scales, (const uint8_t*)x_scales, x_ld_scales, y, ldy,
               M, N, K, blocks, N / 2, out_dtype == TS_F32 ? 1 : 0, act, limit, alpha, 1, error};
    CUtensorMap map_w{};
    if (x_scales && make_tile_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w_codes, N, (long long)blocks * 16, w_ld_codes, gated ? 16 : BM, "gemm_mxfp4"))
        return 1;
    if (x_scales) return gated ? dispatch<true, true>(map_w, x, ldx, p, stream) : dispatch<true, false>(map_w, x, ldx, p, stream);
    return gated ? dispatch<false, true>(map_w, x, ldx, p, stream) : dispatch<false, false>(map_w, x, ldx, p, stream);
}
