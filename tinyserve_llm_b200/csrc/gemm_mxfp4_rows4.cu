// Products over microscaled 4-bit weights on tcgen05, rows of x in four bits too.
//
// Codes of both sides come by TMA, 256 numbers a row of 128 bytes, and tcgen05.mma kind::mxf4 multiplies them, four times as many a cycle
// as bfloat16 numbers.  The scales it reads from tensor memory: four warps gather their bytes from global memory, 16 scales of a row at a
// time, two stages' (at one stage's eight bytes the loads of 384 rows, a sector each, took longer than the MMAs, and so did a barrier a
// stage), and put them into a ring of their own in shared memory, of a stage's 16 bytes for lane l bytes 4 j .. 4 j + 3 of row 32 j + l;
// tcgen05.cp hands them to all four quarters of the lanes.
//
// A few rows of bfloat16 numbers take the same way (KIND 8): each row becomes three rows of 8-bit floating point (e5m2, blocks of 32 under a
// scale of a power of two), the number rounded to three bits, what that left, and what that left again, and tcgen05.mma kind::mxf8f6f4
// multiplies them with W's codes as they are; the three products are added up.  Three bits, their signs and a third piece make a bfloat16's
// eight, exactly, of numbers down to some 2^31 times smaller than their block's largest.  (Two pieces of e4m3 have the bits, but not the
// range: they lose some of numbers 2^14 times smaller, and of a norm's output one number in 5,000 is.)  A block with numbers smaller still
// that are not zero, with infinities or NaNs is zeros in the pieces, under a scale of its own, and multiplied number by number: right, but slow
// where most blocks are such (exponents drawn evenly from -60 to 60: eight rows of 28,672 by 4,096 1.05 ms).
//
// An MMA of some columns costs next to nothing beside the stream of W, where spreading W's codes to bfloat16, for tensor memory or in
// registers, takes longer than bringing them (28,672 rows of 4,096, eight rows of x: 41 us).
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
// e2m1 x e2m1 -> float32 (KIND 4) with two scales a row and MMA, or e2m1 x e5m2 (KIND 8) with one; scales are power-of-two bytes, `byte`: the
// first of an MMA's in the four bytes of a column.
template <int KIND>
__device__ __forceinline__ uint32_t instr_desc(int n, int byte) {
    return (uint32_t)byte << 4 | (KIND == 4 ? 1u : 5u) << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(BM >> 7) << 27 |
           (uint32_t)byte << 29;
}

template <int BN>
__host__ __device__ constexpr int x_sets() { return (BN + 127) / 128; }                    // of 128 rows of x's scales
template <int KIND, int BN>
__host__ __device__ constexpr int scale_columns() { return (KIND == 4 ? 8 : 4) * (1 + x_sets<BN>()); }        // of tensor memory, a stage

constexpr int PIECES8 = 3;                             // rows of e5m2 numbers a row of bfloat16 ones becomes
constexpr uint32_t BY_HAND = 254;                      // scale of a block that is not in the pieces: no other block has it
// Rows of x in a tile whose MMAs have BN columns: its first pieces, then the second, then the third.  (32 columns: 24 and eight nobody reads.)
template <int KIND, int BN>
__host__ __device__ constexpr int tile_rows() { return KIND == 4 ? BN : BN == 32 ? 8 : BN / PIECES8; }

__device__ __forceinline__ void tma_load_3d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait8(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}

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

// What the blocks that are not in the pieces, from `block0` to `block1` (multiples of four), add to the product of a lane's row of W with a row of
// x, whose first pieces' scales are `x_scales`.
__device__ __noinline__ float by_hand(const uint8_t* codes, const uint8_t* scales, const __nv_bfloat16* x, const uint8_t* x_scales, int block0,
                                      int block1, int lane) {
    float sum = 0.f;
    for (int b0 = block0; b0 < block1; b0 += 128) {                   // a lane looks at four blocks' scales
        const int four = b0 + lane * 4;
        const uint32_t word = four < block1 ? __ldg(reinterpret_cast<const uint32_t*>(x_scales + four)) : 0;
        const uint32_t mine = __vcmpeq4(word, BY_HAND * 0x01010101u);
        for (uint32_t who = __ballot_sync(0xffffffffu, mine != 0); who; who &= who - 1) {
            const int l = __ffs(who) - 1;
            for (uint32_t left = __shfl_sync(0xffffffffu, mine, l) & 0x01010101u; left; left &= left - 1) {
                const int block = b0 + l * 4 + (__ffs(left) - 1) / 8;
                const uint4 code = __ldg(reinterpret_cast<const uint4*>(codes + block * 16ll));
                const float scale = mx_scale(__ldg(scales + block));
                const float number = to_float(x[block * 32ll + lane]);
                const uint32_t words[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    sum = fmaf(mx_code_value(words[e >> 3] >> (4 * (e & 7)) & 15) * scale, __shfl_sync(0xffffffffu, number, e), sum);
            }
        }
    }
    return sum;
}

// The columns of a tile whose x came in pieces, eight rows of x at a time: an epilogue warp takes every other eight (`half`).  `marked`: a bit
// for each of the tile's rows that has blocks, of its CTA's, to be multiplied by hand.
template <bool GATED, int ROWS>
__device__ __forceinline__ void finish_pieces(const MxParams& p, uint32_t tmem, int half, int t0, int f0, int outs, int quarter, int lane, float* sums,
                                              const uint32_t* marked, int block0, int block1) {
    const uint32_t addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const int f = GATED ? f0 + quarter * 16 + (lane & 15) : f0 + quarter * 32 + lane;
    const int row = min(row_of<GATED>(p, f0, quarter * 32 + lane), p.N - 1);
#pragma unroll 1
    for (int r = half * 8; r < ROWS; r += 16) {
        const int t = t0 + r;
        if (t >= p.M) break;
        uint32_t acc[PIECES8][8];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PIECES8; ++i) tmem_ld8(addr + i * ROWS + r, acc[i]);
#pragma unroll
        for (int i = 0; i < PIECES8; ++i) tmem_wait8(acc[i]);
        float v[8];
        uint32_t past = 0;                                            // the first pieces, rounded up, may leave float32's range alone
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = __uint_as_float(acc[0][j]) + (__uint_as_float(acc[1][j]) + __uint_as_float(acc[2][j]));
            past |= (isinf(v[j]) ? 1u : 0u) << j;
        }
        const uint32_t some = marked[r >> 5] >> (r & 31) & 0xff;
        if (some) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((some >> j & 1) && t + j < p.M)
                    v[j] += by_hand(p.w_codes + row * p.w_ld_codes, p.w_scales + row * p.w_ld_scales, p.x16 + (t + j) * p.x16_ld,
                                    p.x_scales + (t + j) * p.x_ld_scales, block0, block1, lane);
        }
        if (p.splits > 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[(r + j) * BM + quarter * 32 + lane] = v[j];
            continue;
        }
        if (past) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((past >> j & 1) && t + j < p.M) v[j] = plain_dot(p, row, t + j);
        }
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
    constexpr int ROWS = tile_rows<KIND, BN>(), CHUNK = KIND == 4 ? 256 : 128;      // columns of K in the 128 bytes of a row and stage
    constexpr int SETS = KIND == 4 ? 2 : 1;          // of four scales a row and stage
    constexpr int GROUP_BITS = group_bits<KIND>(), PER_GROUP = 1 << GROUP_BITS, GROUPS_HELD = groups_held<KIND>();
    constexpr int B_BYTES = BN * ROW, SCALE_COLS = scale_columns<KIND, BN>(), SCALE_BYTES = SCALE_COLS * 128, X_SETS = x_sets<BN>();
    constexpr int ACCUMULATORS = SPLIT ? 1 : 2, OUTS = GATED ? BM / 2 : BM, SHARE = BN / (EPI_WARPS / 4);
    constexpr int TMEM_USED = ACCUMULATORS * BN + STAGES * SCALE_COLS, TMEM_COLS = power_of_two(TMEM_USED);
    static_assert(TMEM_USED <= 512, "tensor memory has 512 columns");
    static_assert(KIND == 4 || SPLIT, "pieces are added up by tiles");
    static_assert(KIND == 4 || (ROWS % 8 == 0 && ROWS <= 64 && ROWS * PIECES8 <= BN), "eights of rows, a bit each in two words");
    static_assert(!SPLIT || BM * ROWS * 4 <= STAGES * (A_BYTES + B_BYTES), "a split tile's sums go where the ring was");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ __align__(8) uint64_t scales_full[GROUPS_HELD], scales_empty[GROUPS_HELD];
    __shared__ uint32_t tmem_base_slot, marked[2];
    __shared__ int failed;

    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* scale_ring = stages + STAGES * (A_BYTES + B_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outs = GATED ? p.inter : p.N;
    const int x_tiles = (p.M + ROWS - 1) / ROWS, num_tiles = x_tiles * ((outs + OUTS - 1) / OUTS);
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
        marked[0] = marked[1] = 0;
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
                const int t0 = (tile % x_tiles) * ROWS, f0 = (tile / x_tiles) * OUTS;
                for (int chunk = chunk0; chunk < chunk1; ++chunk, r.next()) {
                    const int s = r.at;
                    if (!wait_for(&empty_bar[s], r.parity ^ 1, p.error, 41)) { failed = 1; break; }
                    unsigned char* tile_at = stages + s * (A_BYTES + B_BYTES);
                    // spaced codes count without the space
                    mbar_expect_tx(&full_bar[s], KIND == 4 ? A_BYTES + B_BYTES : A_BYTES / 2 + ROWS * PIECES8 * ROW);
                    load_codes<GATED>(tile_at, &map_w, &full_bar[s], p, chunk * ROW, f0);
                    if (KIND == 4) tma_load_2d(tile_at + A_BYTES, &map_x, &full_bar[s], chunk * ROW, t0);
                    else tma_load_3d(tile_at + A_BYTES, &map_x, &full_bar[s], chunk * ROW, t0, 0);
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
            const int t0 = (tile % x_tiles) * ROWS, f0 = (tile / x_tiles) * OUTS;
            const bool ok = wait_for(&tmem_full_bar[buf], (iter >> 1) & 1, p.error, 43) && !failed;
            if (!__all_sync(0xffffffffu, ok)) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if constexpr (KIND == 8) {
                // what the warps of the scales have marked is there when they have handed on their last ones
                const int last = ((chunk1 - 1) >> GROUP_BITS) - (chunk0 >> GROUP_BITS);
                const bool all = wait_for(&scales_full[last % GROUPS_HELD], (last / GROUPS_HELD) & 1, p.error, 43);
                if (!__all_sync(0xffffffffu, all)) { failed = 1; break; }
                finish_pieces<GATED, ROWS>(p, tmem_base, (warp - 2) >> 2, t0, f0, outs, quarter, lane, reinterpret_cast<float*>(stages),
                                                           marked, chunk0 * 4, chunk1 * 4);
            } else {
                finish_tile<GATED, SHARE, SPLIT>(p, tmem_base + buf * BN, first, t0, f0, outs, paired, quarter, lane, reinterpret_cast<float*>(stages),
                                                 &tmem_empty_bar[buf]);
            }
        }
    } else {
        // ---------------------------------------------------------------- scales
        // Groups of 32 rows, a row a lane: 0 to 3 of W, from 4 on of x; a warp has every fourth.  What a group leaves out of its 512 bytes
        // (fewer than 128 rows of x) belongs to columns that no MMA reads.
        constexpr int GROUPS = 4 + (BN + 31) / 32, MINE = (GROUPS + GATHER - 1) / GATHER;
        const int w = warp - 2 - EPI_WARPS;
        auto x_row = [&](int t0, int n) -> long long {                // of the matrix of x's scales, for row n of a tile
            if (KIND == 4) return min(t0 + n, p.M - 1);
            return (long long)min(n / ROWS, PIECES8 - 1) * p.M + min(t0 + n % ROWS, p.M - 1);
        };
        bool ok = true;
        Ring<GROUPS_HELD> r;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            const int t0 = (tile % x_tiles) * ROWS, f0 = (tile / x_tiles) * OUTS;
            const uint8_t* row[MINE];
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int g = w + i * GATHER;
                row[i] = g < 4 ? p.w_scales + (long long)min(row_of<GATED>(p, f0, g * 32 + lane), p.N - 1) * p.w_ld_scales
                               : p.x_scales + x_row(t0, (g - 4) * 32 + lane) * p.x_ld_scales;
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
                    if (KIND == 8 && g >= 4 && (g - 4) * 32 < ROWS) {             // the tile's rows, a lane each: which are to be multiplied by hand
                        const uint32_t hand = BY_HAND * 0x01010101u;
                        if (__vcmpeq4(now[i].x, hand) | __vcmpeq4(now[i].y, hand) | __vcmpeq4(now[i].z, hand) | __vcmpeq4(now[i].w, hand))
                            if ((g - 4) * 32 + lane < ROWS) atomicOr(&marked[(g - 4) & 1], 1u << lane);
                    }
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
        const int t0 = (first_tile % x_tiles) * ROWS, f0 = (first_tile / x_tiles) * OUTS;
        const auto again = [&](int l, int t, float v) {
            return KIND == 8 && isinf(v) ? plain_dot(p, min(row_of<GATED>(p, f0, l), p.N - 1), t) : v;
        };
        join_splits<GATED>(p, smem_u32(stages), rank, min(ROWS, p.M - t0), t0, f0, outs, threadIdx.x, THREADS, again);
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

// bfloat16 rows as three rows of e5m2 numbers each: all first pieces, all second ones, all third ones.  Four lanes a block, eight numbers a lane.
__global__ void __launch_bounds__(256) pieces_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, uint2* __restrict__ numbers,
                                                     uint8_t* __restrict__ scales, int M, int blocks, int ld_scales) {
    chain_wait();
    chain_release();
    const int lanes = blocks * 4;
    const long long total = (long long)M * lanes, first = (long long)blockIdx.x * 256 + (threadIdx.x & ~31), at = first + (threadIdx.x & 31);
    if (first >= total) return;                                       // a whole warp
    const bool mine = at < total;
    const int m = mine ? (int)(at / lanes) : 0, part = mine ? (int)(at - (long long)m * lanes) : 0;
    float v[8];
    const uint4 q = mine ? *reinterpret_cast<const uint4*>(x + (long long)m * ldx + part * 8) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    uint2 packed[PIECES8];
    int scale_byte[PIECES8];
    bool hand = false;                                                // not finite, or something is left of it
#pragma unroll
    for (int i = 0; i < PIECES8; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);       // what is not finite is largest
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (i == 0) hand = top >= 0x7f800000u;
        // the largest becomes a number from 2^14 to 2^15, of 1.75 2^15 that there is room for
        const int s = max((int)(top >> 23) - 14, 0);
        const float inverse = __uint_as_float((uint32_t)(254 - s) << 23), scale = mx_scale(s);
        uint32_t two[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint16_t codes;
            uint32_t halves;
            asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(codes) : "f"(v[2 * e + 1] * inverse), "f"(v[2 * e] * inverse));
            asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(halves) : "h"(codes));
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&halves));
            v[2 * e] -= back.x * scale;                               // exact: a bfloat16 less its leading bits
            v[2 * e + 1] -= back.y * scale;
            two[e] = codes;
        }
        packed[i] = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
        scale_byte[i] = s;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) hand |= v[e] != 0.f;
    const uint32_t block_lanes = 0xfu << (threadIdx.x & 28);
    hand = (__ballot_sync(0xffffffffu, hand) & block_lanes) != 0;     // any of the block's
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < PIECES8; ++i) {
        const long long row = (long long)i * M + m;
        numbers[row * lanes + part] = hand ? make_uint2(0, 0) : packed[i];
        if ((part & 3) == 0) scales[row * ld_scales + (part >> 2)] = (uint8_t)(hand ? BY_HAND : scale_byte[i]);
    }
}

template <int KIND, bool GATED, int BN, int STAGES, bool SPLIT>
int run(const void* x, long long ldx, MxParams& p, long long tiles, int sms, int device, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (make_codes_map<GATED>(&map_w, p, KIND == 8)) return 1;
    if (KIND == 4) {
        if (make_tile_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, p.M, p.blocks * 16ll, ldx, BN, "gemm_mxfp4")) return 1;
    } else {                                         // bytes, rows, pieces
        const cuuint64_t dims[3] = {(cuuint64_t)ldx, (cuuint64_t)p.M, PIECES8}, strides[2] = {(cuuint64_t)ldx, (cuuint64_t)ldx * p.M};
        const cuuint32_t box[3] = {ROW, (cuuint32_t)tile_rows<KIND, BN>(), PIECES8}, elem[3] = {1, 1, 1};
        const CUresult r = encode_tiled()(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(x), dims, strides, box, elem,
                                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return ts_fail("gemm_mxfp4: cuTensorMapEncodeTiled failed with %d", (int)r);
    }
    static unsigned long long allowed = 0;
    return launch_mxfp4(rows4_kernel<KIND, GATED, BN, STAGES, SPLIT>, allowed, THREADS, (size_t)ring_bytes<KIND, BN, STAGES>() + 1024, SPLIT,
                        tiles, sms, device, map_w, map_x, p, stream);
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
    const long long ldx = (long long)p.blocks * 32;
    const long long outs = GATED ? p.inter : p.N, per = GATED ? BM / 2 : BM, tiles = (outs + per - 1) / per;
    p.splits = splits_of(p, tiles, sms);
    if (p.M <= 8) return run<8, GATED, 32, 5, true>(numbers, ldx, p, tiles, sms, device, stream);
    if (p.M <= 16) return run<8, GATED, 48, 4, true>(numbers, ldx, p, tiles, sms, device, stream);
    if (p.M <= 32) return run<8, GATED, 96, 3, true>(numbers, ldx, p, tiles, sms, device, stream);
    // more tiles than SMs: two CTAs an SM, with what is left of a ring each (28,672 by 4,096 gated, 64 rows 34.7 us, 40.8 one behind the other);
    // else one (6,144 by 4,096 14.1 and 18.7)
    if (tiles > sms) return run<8, GATED, 192, 2, true>(numbers, ldx, p, tiles, sms, device, stream);
    return run<8, GATED, 192, 4, true>(numbers, ldx, p, tiles, sms, device, stream);
}

}  // namespace

int mxfp4_rows4(const void* x, long long ldx, MxParams& p, int gated, cudaStream_t stream) {
    return gated ? dispatch<true>(x, ldx, p, stream) : dispatch<false>(x, ldx, p, stream);
}

long long mxfp4_pieces_bytes(int M, int blocks) { return (long long)M * PIECES8 * (blocks * 32ll + (blocks + 15) / 16 * 16); }

int mxfp4_pieces(const void* x, long long ldx, void* scratch, MxParams& p, int gated, cudaStream_t stream) {
    uint8_t* numbers = (uint8_t*)scratch;
    uint8_t* scales = numbers + (long long)p.M * PIECES8 * p.blocks * 32;
    p.x_scales = scales;
    p.x_ld_scales = (p.blocks + 15) / 16 * 16;
    p.x16 = (const __nv_bfloat16*)x;
    p.x16_ld = ldx;
    const dim3 grid((unsigned)(((long long)p.M * p.blocks * 4 + 255) / 256));
    TS_CHAINED_CHECK("gemm_mxfp4", launch_chained(pieces_kernel, grid, dim3(256), 0, stream, (const __nv_bfloat16*)x, ldx, (uint2*)numbers, scales,
                                                  p.M, p.blocks, (int)p.x_ld_scales));
    return gated ? dispatch_pieces<true>(numbers, p, stream) : dispatch_pieces<false>(numbers, p, stream);
}
