// Products over microscaled 4-bit weights on tcgen05, rows of x in four bits too.
//
// Codes of both sides come by TMA, 256 numbers a row of 128 bytes, and tcgen05.mma kind::mxf4 multiplies them, four times as many a cycle
// as bfloat16 numbers.  The scales it reads from tensor memory: four warps gather their bytes from global memory, 16 scales of a row at a
// time, two stages' (at one stage's eight bytes the loads of 384 rows, a sector each, took longer than the MMAs, and so did a barrier a
// stage), and put them into a ring of their own in shared memory, of a stage's 16 bytes for lane l bytes 4 j .. 4 j + 3 of row 32 j + l;
// tcgen05.cp hands them to all four quarters of the lanes.
//
// A few rows of bfloat16 numbers take the same way (KIND 8): each row becomes two rows of 8-bit floating point (e4m3, blocks of 32 under a
// scale of a power of two), the number rounded to four bits and what that left, and tcgen05.mma kind::mxf8f6f4 multiplies them with W's
// codes as they are; the two products are added up.  Four bits and four make a bfloat16's eight: only of numbers 2^13 times smaller than
// their block's largest something is lost, less than 2^-21 of that largest.  An MMA of some columns costs next to nothing beside the stream of
// W, where spreading W's codes to bfloat16, for tensor memory or in registers, takes longer than bringing them (28,672 rows of 4,096, eight
// rows of x: 41 us).  A block of x with a NaN is NaN.  Infinities have no place in these blocks: one that holds some, and no NaN, is zeros and
// then NaN, and results whose second piece alone is NaN are worked out again, number by number.
#include <cuda_fp16.h>

#include "gemm_mxfp4.cuh"

namespace {

// Warps: producer, issuer, eight of the epilogue, four that gather scales.
constexpr int EPI_WARPS = 8, GATHER = 4, THREADS = 32 * (2 + EPI_WARPS + GATHER);

__device__ __forceinline__ void umma(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
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
__device__ __forceinline__ void umma8(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                      uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(leader) : "memory");
}
// e2m1 x e2m1 -> float32 (KIND 4) with two scales a row and MMA, or e2m1 x e4m3 (KIND 8) with one; scales are power-of-two bytes, `byte`: the
// first of an MMA's in the four bytes of a column.
template <int KIND>
__device__ __forceinline__ uint32_t instr_desc(int n, int byte) {
    return (uint32_t)byte << 4 | (KIND == 4 ? 1u << 7 | 1u << 10 : 5u << 7) | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(BM >> 7) << 27 |
           (uint32_t)byte << 29;
}

template <int BN>
__host__ __device__ constexpr int x_sets() { return (BN + 127) / 128; }                    // of 128 rows of x's scales
template <int KIND, int BN>
__host__ __device__ constexpr int scale_columns() { return (KIND == 4 ? 8 : 4) * (1 + x_sets<BN>()); }        // of tensor memory, a stage

constexpr int PIECES8 = 2;                             // rows of e4m3 numbers a row of bfloat16 ones becomes

// One product of a row of W with a bfloat16 row of x, number by number.
__device__ __noinline__ float plain_dot(const uint8_t* codes, const uint8_t* scales, const __nv_bfloat16* x, int K) {
    float sum = 0.f;
    for (int i = 0; i < K; ++i) {
        const uint32_t byte = codes[i >> 1];
        sum = fmaf(mx_code_value(i & 1 ? byte >> 4 : byte & 15) * mx_scale(scales[i / MX_BLOCK]), to_float(x[i]), sum);
    }
    return sum;
}
__device__ __forceinline__ float plain_dot(const MxParams& p, int row, int t) {
    return plain_dot(p.w_codes + row * p.w_ld_codes, p.w_scales + row * p.w_ld_scales, p.x16 + t * p.x16_ld, p.K);
}

// A result from its two pieces' products; infinite (whatever its sign) stands for one that has to be worked out again.
__device__ __forceinline__ float added(float first, float second) {
    return second != second && first == first ? __int_as_float(0x7f800000) : first + second;
}

// The columns of a tile whose x came in two pieces a row: an epilogue warp's share, 16 columns, eight rows of x, at a time.
template <bool GATED, int SHARE>
__device__ __forceinline__ void finish_pieces(const MxParams& p, uint32_t tmem, int first, int t0, int f0, int outs, int quarter, int lane,
                                              float* sums) {
    const uint32_t addr = tmem + first + ((uint32_t)(quarter * 32) << 16);
    const int f = GATED ? f0 + quarter * 16 + (lane & 15) : f0 + quarter * 32 + lane;
#pragma unroll 1
    for (int c0 = 0; c0 < SHARE; c0 += 16) {
        uint32_t acc[16];
        __syncwarp();
        tmem_ld16(addr + c0, acc);
        tmem_wait16(acc);
        const int column = (first + c0) / PIECES8, t = t0 + column;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = added(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1]));
        if (p.splits > 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[(column + j) * BM + quarter * 32 + lane] = v[j];
            continue;
        }
        if (t >= p.M) continue;
        const int row = row_of<GATED>(p, f0, quarter * 32 + lane);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (isinf(v[j]) && t + j < p.M && row < p.N) v[j] = plain_dot(p, row, t + j);
        __syncwarp();
        if (GATED) {                                                  // the lower half of the lanes finishes even rows of x, the upper one odd ones
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[j + 1] : v[j], 16);
                const float y = lane < 16 ? gate_one(p, v[j], other) : gate_one(p, other, v[j + 1]);
                const int at = t + j + (lane >> 4);
                if (at < p.M && f < outs) ((__nv_bfloat16*)p.y)[(long long)at * p.ldy + f] = __float2bfloat16_rn(y);
            }
        } else if (f < outs) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (t + j >= p.M) break;
                if (p.out_f32) ((float*)p.y)[(long long)(t + j) * p.ldy + f] = v[j];
                else ((__nv_bfloat16*)p.y)[(long long)(t + j) * p.ldy + f] = __float2bfloat16_rn(v[j]);
            }
        }
    }
}

// Scales come in groups of 16 a row, which last two stages (KIND 8: four), and a ring of a few groups.
template <int KIND>
__host__ __device__ constexpr int group_bits() { return KIND == 4 ? 1 : 2; }
template <int KIND>
__host__ __device__ constexpr int groups_held() { return KIND == 4 ? 3 : 2; }
template <int KIND, int BN, int STAGES>
__host__ __device__ constexpr int ring_bytes() {
    return STAGES * (A_BYTES + BN * ROW) + (groups_held<KIND>() << group_bits<KIND>()) * 128 * scale_columns<KIND, BN>();
}

// Small rings leave room for two CTAs an SM, so that one's beginning and end run beside the other's stream of W.
template <int KIND, bool GATED, int BN, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(THREADS, ring_bytes<KIND, BN, STAGES>() <= 113 * 1024 ? 2 : 1)
rows4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, MxParams p) {
    constexpr int PIECES = KIND == 4 ? 1 : PIECES8, CHUNK = KIND == 4 ? 256 : 128;      // columns of K in the 128 bytes of a row and stage
    constexpr int SETS = KIND == 4 ? 2 : 1;          // of four scales a row and stage
    constexpr int GROUP_BITS = group_bits<KIND>(), PER_GROUP = 1 << GROUP_BITS, GROUPS_HELD = groups_held<KIND>();
    constexpr int B_BYTES = BN * ROW, SCALE_COLS = scale_columns<KIND, BN>(), SCALE_BYTES = SCALE_COLS * 128, X_SETS = x_sets<BN>();
    constexpr int ACCUMULATORS = SPLIT ? 1 : 2, OUTS = GATED ? BM / 2 : BM, SHARE = BN / (EPI_WARPS / 4);
    constexpr int TMEM_USED = ACCUMULATORS * BN + STAGES * SCALE_COLS, TMEM_COLS = power_of_two(TMEM_USED);
    static_assert(TMEM_USED <= 512, "tensor memory has 512 columns");
    static_assert(PIECES == 1 || SPLIT, "pieces are added up by tiles");
    static_assert(!SPLIT || BM * BN / PIECES * 4 <= STAGES * (A_BYTES + B_BYTES), "a split tile's sums go where the ring was");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ __align__(8) uint64_t scales_full[GROUPS_HELD], scales_empty[GROUPS_HELD];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int failed;

    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* scale_ring = stages + STAGES * (A_BYTES + B_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outs = GATED ? p.inter : p.N;
    const int x_tiles = (p.M * PIECES + BN - 1) / BN, num_tiles = x_tiles * ((outs + OUTS - 1) / OUTS);
    const int all_chunks = (p.blocks * MX_BLOCK + CHUNK - 1) / CHUNK;
    const int rank = SPLIT && p.splits > 1 ? (int)pair_rank() : 0;
    const int first_tile = SPLIT ? (int)blockIdx.x / p.splits : (int)blockIdx.x, tile_step = SPLIT ? num_tiles : (int)gridDim.x;
    const int chunk0 = SPLIT ? (int)((long long)all_chunks * rank / p.splits) : 0;
    const int chunk1 = SPLIT ? (int)((long long)all_chunks * (rank + 1) / p.splits) : all_chunks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < GROUPS_HELD; ++b) {
            mbar_init(&scales_full[b], GATHER);
            mbar_init(&scales_empty[b], 1);
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
            Ring<STAGES> r;
            for (int tile = first_tile; tile < num_tiles && !failed; tile += tile_step) {
                const int t0 = (tile % x_tiles) * (BN / PIECES), f0 = (tile / x_tiles) * OUTS;
                for (int chunk = chunk0; chunk < chunk1; ++chunk, r.next()) {
                    const int s = r.at;
                    if (!wait_for(&empty_bar[s], r.parity ^ 1, p.error, 41)) { failed = 1; break; }
                    unsigned char* tile_at = stages + s * (A_BYTES + B_BYTES);
                    mbar_expect_tx(&full_bar[s], (KIND == 4 ? A_BYTES : A_BYTES / 2) + B_BYTES);      // spaced codes count without the space
                    load_codes<GATED>(tile_at, &map_w, &full_bar[s], p, chunk * ROW, f0);
                    tma_load_2d(tile_at + A_BYTES, &map_x, &full_bar[s], chunk * ROW, t0 * PIECES);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint32_t leader = elect_one();
        const uint32_t tmem_scales = tmem_base + ACCUMULATORS * BN;
        bool ok = true;                              // the same in all lanes
        Ring<STAGES> r;
        Ring<GROUPS_HELD> g;
        const uint64_t a_first = smem_desc(stages), b_first = smem_desc(stages + A_BYTES), scales_first = scale_desc(scale_ring);
        int iter = 0;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++iter) {
            const int buf = SPLIT ? 0 : iter & 1;
            ok = __all_sync(0xffffffffu, wait_for(&tmem_empty_bar[buf], ((iter >> 1) & 1) ^ 1, p.error, 44) && !failed);
            if (!ok) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + buf * BN;
            uint32_t add = 0;                        // the tile's first MMA starts its sums
            for (int chunk = chunk0; chunk < chunk1; ++chunk, r.next()) {
                ok = __all_sync(0xffffffffu, wait_for(&full_bar[r.at], r.parity, p.error, 42));
                if (chunk == chunk0 || (chunk & (PER_GROUP - 1)) == 0)
                    ok = __all_sync(0xffffffffu, ok && wait_for(&scales_full[g.at], g.parity, p.error, 49));
                if (!ok) { failed = 1; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t a_desc = a_first + r.at * ((A_BYTES + B_BYTES) / 16), b_desc = b_first + r.at * ((A_BYTES + B_BYTES) / 16);
                const uint64_t from = scales_first + (g.at * PER_GROUP + (chunk & (PER_GROUP - 1))) * (SCALE_BYTES / 16);
                // a stage's scales have columns of their own: they are free when the stage is, once the MMAs that read them have retired
                const uint32_t sa = tmem_scales + r.at * SCALE_COLS, sb = sa + 4 * SETS;
#pragma unroll
                for (int i = 0; i < SETS * (1 + X_SETS); ++i) copy_scales(leader, sa + 4 * i, from + 32 * i);
#pragma unroll
                for (int k = 0; k < 4; ++k, add = 1) {                // an MMA takes 32 bytes of a row: 64 columns of K or (KIND 8) 32
                    if (KIND == 4)
                        umma(leader, tmem_d, a_desc + 2 * k, b_desc + 2 * k, instr_desc<4>(BN, 2 * (k & 1)), sa + (k >> 1) * 4,
                             sb + (k >> 1) * 4 * X_SETS, add);
                    else
                        umma8(leader, tmem_d, a_desc + 2 * k, b_desc + 2 * k, instr_desc<8>(BN, k), sa, sb, add);
                }
                if (leader) umma_commit(&empty_bar[r.at]);
                if (chunk + 1 == chunk1 || (chunk & (PER_GROUP - 1)) == PER_GROUP - 1) {
                    if (leader) umma_commit(&scales_empty[g.at]);
                    g.next();
                }
            }
            if (leader) umma_commit(&tmem_full_bar[buf]);
        }
    } else if (warp < 2 + EPI_WARPS) {
        // ---------------------------------------------------------------- epilogue
        const int quarter = warp & 3, first = ((warp - 2) >> 2) * SHARE;      // the 32 lanes this warp may read; its share of the columns
        const bool paired = (p.ldy & 1) == 0 && ((uintptr_t)p.y & 3) == 0;
        int iter = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++iter) {
            const int buf = SPLIT ? 0 : iter & 1;
            const int t0 = (tile % x_tiles) * (BN / PIECES), f0 = (tile / x_tiles) * OUTS;
            const bool ok = wait_for(&tmem_full_bar[buf], (iter >> 1) & 1, p.error, 43) && !failed;
            if (!__all_sync(0xffffffffu, ok)) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (PIECES > 1)
                finish_pieces<GATED, SHARE>(p, tmem_base, first, t0, f0, outs, quarter, lane, reinterpret_cast<float*>(stages));
            else
                finish_tile<GATED, SHARE, SPLIT>(p, tmem_base + buf * BN, first, t0, f0, outs, paired, quarter, lane, reinterpret_cast<float*>(stages),
                                                 &tmem_empty_bar[buf]);
        }
    } else {
        // ---------------------------------------------------------------- scales
        // Groups of 32 rows, a row a lane: 0 to 3 of W, from 4 on of x; a warp has every fourth.  What a group leaves out of its 512 bytes
        // (fewer than 128 rows of x) belongs to columns that no MMA reads.
        constexpr int GROUPS = 4 + BN / 32, MINE = (GROUPS + GATHER - 1) / GATHER;
        const int w = warp - 2 - EPI_WARPS;
        bool ok = true;
        Ring<GROUPS_HELD> r;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            const int t0 = (tile % x_tiles) * (BN / PIECES), f0 = (tile / x_tiles) * OUTS;
            const uint8_t* row[MINE];
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int g = w + i * GATHER;
                row[i] = g < 4 ? p.w_scales + (long long)min(row_of<GATED>(p, f0, g * 32 + lane), p.N - 1) * p.w_ld_scales
                               : p.x_scales + (long long)min(t0 * PIECES + (g - 4) * 32 + lane, p.M * PIECES - 1) * p.x_ld_scales;
            }
            auto load = [&](int group, uint4 (&v)[MINE]) {            // 16 scales of each row; behind the last block 1
                const int b = group * 16;
#pragma unroll
                for (int i = 0; i < MINE; ++i) {
                    if (w + i * GATHER >= GROUPS) continue;
                    if (b + 16 <= p.blocks) {
                        v[i] = __ldg(reinterpret_cast<const uint4*>(row[i] + b));
                    } else {
                        uint32_t q[4] = {0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (b + j < p.blocks) q[j >> 2] = (q[j >> 2] & ~(0xffu << (8 * (j & 3)))) | (uint32_t)row[i][b + j] << (8 * (j & 3));
                        v[i] = make_uint4(q[0], q[1], q[2], q[3]);
                    }
                }
            };
            uint4 now[MINE], next[MINE];
            const int last = (chunk1 - 1) >> GROUP_BITS;
            load(chunk0 >> GROUP_BITS, now);
            for (int group = chunk0 >> GROUP_BITS; group <= last; ++group, r.next()) {
                if (group < last) load(group + 1, next);
                ok = __all_sync(0xffffffffu, wait_for(&scales_empty[r.at], r.parity ^ 1, p.error, 45));
                if (!ok || failed) { failed = 1; break; }
#pragma unroll
                for (int i = 0; i < MINE; ++i) {
                    const int g = w + i * GATHER;
                    if (g >= GROUPS) continue;
                    // word j of the row: stage j / SETS of the group, set j % SETS
                    const int of_x = g < 4 ? 0 : SETS * 512 + ((g - 4) >> 2) * 512;
                    unsigned char* to = scale_ring + r.at * PER_GROUP * SCALE_BYTES + of_x + lane * 16 + (g & 3) * 4;
                    const int set = g < 4 ? 512 : X_SETS * 512;
                    *reinterpret_cast<uint32_t*>(to) = now[i].x;
                    *reinterpret_cast<uint32_t*>(to + (SETS == 2 ? set : SCALE_BYTES)) = now[i].y;
                    *reinterpret_cast<uint32_t*>(to + (SETS == 2 ? SCALE_BYTES : 2 * SCALE_BYTES)) = now[i].z;
                    *reinterpret_cast<uint32_t*>(to + (SETS == 2 ? SCALE_BYTES + set : 3 * SCALE_BYTES)) = now[i].w;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&scales_full[r.at]);
#pragma unroll
                for (int i = 0; i < MINE; ++i) now[i] = next[i];
            }
        }
    }
    __syncwarp();
    if (SPLIT && p.splits > 1) {
        pair_sync();                                 // every CTA's sums are in its shared memory
        const int t0 = (first_tile % x_tiles) * (BN / PIECES), f0 = (first_tile / x_tiles) * OUTS;
        const auto again = [&](int l, int t, float v) { return PIECES > 1 && isinf(v) ? plain_dot(p, min(row_of<GATED>(p, f0, l), p.N - 1), t) : v; };
        join_splits<GATED>(p, smem_u32(stages), rank, min(BN / PIECES, p.M - t0), t0, f0, outs, threadIdx.x, THREADS, again);
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

// bfloat16 rows as two rows of e4m3 numbers each, m * 2 and m * 2 + 1.  Four lanes a block, eight numbers a lane.
__global__ void __launch_bounds__(256) pieces_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, uint2* __restrict__ numbers,
                                                     uint8_t* __restrict__ scales, int M, int K, int blocks, int ld_scales) {
    chain_wait();
    chain_release();
    const int lanes = blocks * 4;
    const long long total = (long long)M * lanes, first = (long long)blockIdx.x * 256 + (threadIdx.x & ~31), at = first + (threadIdx.x & 31);
    if (first >= total) return;                                       // a whole warp
    const bool mine = at < total;
    const int m = mine ? (int)(at / lanes) : 0, part = mine ? (int)(at - (long long)m * lanes) : 0;
    float v[8];
    if (mine && part * 8 < K) {                                       // K is a multiple of 8
        const uint4 q = *reinterpret_cast<const uint4*>(x + (long long)m * ldx + part * 8);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < PIECES8; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);       // what is not finite is largest
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest becomes a number from 128 to 256, of 448 that there is room for
        const int exponent = (int)(top >> 23);
        int s = exponent == 255 ? 255 : max(exponent - 7, 0);
        uint2 packed = make_uint2(0, 0);
        if (exponent != 255) {
            const float inverse = __uint_as_float((uint32_t)(254 - s) << 23), scale = mx_scale(s);
            uint32_t two[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint16_t codes;
                uint32_t halves;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(codes) : "f"(v[2 * e + 1] * inverse), "f"(v[2 * e] * inverse));
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(codes));
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&halves));
                v[2 * e] -= back.x * scale;                           // exact: a bfloat16 less its leading bits
                v[2 * e + 1] -= back.y * scale;
                two[e] = codes;
            }
            packed = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
        } else {
            if (i == 0 && top == 0x7f800000u) {
                s = 0;                                                // infinities and no NaN: the second piece is NaN
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.f;
            }
        }
        if (mine) {
            numbers[((long long)m * PIECES8 + i) * lanes + part] = packed;
            if ((part & 3) == 0) scales[((long long)m * PIECES8 + i) * ld_scales + (part >> 2)] = (uint8_t)s;
        }
    }
}

template <int KIND, bool GATED, int BN, int STAGES, bool SPLIT>
int run(const void* x, long long ldx, MxParams& p, long long tiles, int sms, int device, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (make_codes_map<GATED>(&map_w, p, KIND == 8)) return 1;
    const long long rows = (long long)p.M * (KIND == 4 ? 1 : PIECES8), bytes = (long long)p.blocks * (KIND == 4 ? 16 : 32);
    if (make_tile_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, rows, bytes, ldx, BN, "gemm_mxfp4")) return 1;
    static unsigned long long allowed = 0;
    return launch_mxfp4(rows4_kernel<KIND, GATED, BN, STAGES, SPLIT>, allowed, THREADS, (size_t)ring_bytes<KIND, BN, STAGES>() + 1024, SPLIT, tiles, sms,
                        device, map_w, map_x, p, stream);
}

template <bool GATED>
int dispatch(const void* x, long long ldx, MxParams& p, cudaStream_t stream) {
    int sms = 148, device = 0;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return cut_mxfp4<GATED, 192>(p, p.M, sms, [&](int bn, bool split, long long tiles) {
        if (bn == 256) return run<4, GATED, 256, 4, true>(x, ldx, p, tiles, sms, device, stream);
        if (bn == 192) return run<4, GATED, 192, 5, false>(x, ldx, p, tiles, sms, device, stream);
        if (bn == 128) return split ? run<4, GATED, 128, 3, true>(x, ldx, p, tiles, sms, device, stream)
                                    : run<4, GATED, 128, 6, false>(x, ldx, p, tiles, sms, device, stream);
        if (bn == 64) return run<4, GATED, 64, 4, true>(x, ldx, p, tiles, sms, device, stream);
        return run<4, GATED, 32, 4, true>(x, ldx, p, tiles, sms, device, stream);
    });
}

template <bool GATED>
int dispatch_pieces(const void* numbers, MxParams& p, cudaStream_t stream) {
    int sms = 148, device = 0;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    const int rows = p.M * PIECES8, bn = rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    const long long ldx = (long long)p.blocks * 32;
    const long long outs = GATED ? p.inter : p.N, per = GATED ? BM / 2 : BM, tiles = (outs + per - 1) / per * ((rows + bn - 1) / bn);
    p.splits = splits_of(p, tiles, sms);
    if (bn == 32) return run<8, GATED, 32, 5, true>(numbers, ldx, p, tiles, sms, device, stream);
    if (bn == 64) return run<8, GATED, 64, 4, true>(numbers, ldx, p, tiles, sms, device, stream);
    if (bn == 128) return run<8, GATED, 128, 3, true>(numbers, ldx, p, tiles, sms, device, stream);
    return run<8, GATED, 256, 4, true>(numbers, ldx, p, tiles, sms, device, stream);
}

}  // namespace

int mxfp4_rows4(const void* x, long long ldx, MxParams& p, int gated, cudaStream_t stream) {
    return gated ? dispatch<true>(x, ldx, p, stream) : dispatch<false>(x, ldx, p, stream);
}

bool mxfp4_takes_pieces(const void* w_codes, long long w_ld_codes, int K) {
    return K % 128 == 0 && w_ld_codes % 32 == 0 && (uintptr_t)w_codes % 32 == 0;      // what TMA asks of 4-bit numbers that it spaces out
}

long long mxfp4_pieces_bytes(int M, int blocks) { return (long long)M * PIECES8 * (blocks * 32 + (blocks + 15) / 16 * 16); }

int mxfp4_pieces(const void* x, long long ldx, void* scratch, MxParams& p, int gated, cudaStream_t stream) {
    uint8_t* numbers = (uint8_t*)scratch;
    uint8_t* scales = numbers + (long long)p.M * PIECES8 * p.blocks * 32;
    p.x_scales = scales;
    p.x_ld_scales = (p.blocks + 15) / 16 * 16;
    p.x16 = (const __nv_bfloat16*)x;
    p.x16_ld = ldx;
    const dim3 grid((unsigned)(((long long)p.M * p.blocks * 4 + 255) / 256));
    TS_CHAINED_CHECK("gemm_mxfp4", launch_chained(pieces_kernel, grid, dim3(256), 0, stream, (const __nv_bfloat16*)x, ldx, (uint2*)numbers, scales,
                                                  p.M, p.K, p.blocks, (int)p.x_ld_scales));
    return gated ? dispatch_pieces<true>(numbers, p, stream) : dispatch_pieces<false>(numbers, p, stream);
}
