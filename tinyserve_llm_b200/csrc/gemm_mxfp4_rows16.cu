// Products over microscaled 4-bit weights on tcgen05, rows of x in bfloat16.
//
// W's codes come into shared memory by TMA as they are, 128 rows of a chunk at a time; sixteen warps make bfloat16 numbers of them (exactly)
// and store them into tensor memory, where tcgen05.mma kind::f16 takes its first operand from; x comes by TMA, 64 numbers a row and stage, and
// is the second.  Shared memory's 128 bytes a cycle would bound the other way: with the numbers laid there too, 16 KB more are written and read
// per 64 columns of K, beside 32 KB of x written and read, against 512 cycles of MMAs of 256 columns (2,048 rows, 8,192 by 2,048: 58 us; 49 now).
//
// Bound by instructions: some 1,900 of a warp for 64 columns of K and a tile, half of them the codes' (27 for a warp's 8 x 32 codes), at 0.64 of the
// issue slots, tensor cores 0.67 busy.  So tiles are as wide as tensor memory lets them be, 256 rows of x on one accumulator: codes once spread
// serve 256 columns, and a tile's epilogue costs less than it would save to hide it.  Device times in a graph: gated, 2,048 rows over 2 x 8,192
// by 2,048, 115 us with 192 rows and two accumulators, 104 to 106 with 256 and one (1.30 PFLOP/s; a call from Python takes 125); 2,048 rows
// through an 8B model's gate and up projections 376 and 344 (1.40).
#include "gemm_mxfp4.cuh"

namespace {

// Warps: producer of x, issuer, four of the epilogue (eight where a tile's epilogue is not under the next one's MMAs), one that brings codes,
// teams of four that spread them: four teams, or two where tiles are small and two CTAs share an SM, one's beginning and end beside the other's
// stream of W.
constexpr int TEAM = 4;
__host__ __device__ constexpr int epilogue_warps(int bn) { return bn == 256 ? 8 : 4; }
__host__ __device__ constexpr int threads_of(int bn, int teams) { return 32 * (3 + epilogue_warps(bn) + teams * TEAM); }
constexpr int BK = 64, PER_CHUNK = CHUNK / BK, STAGE_COLS = BK / 2;    // a stage's columns of K; of tensor memory

__device__ __forceinline__ void umma(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
// bfloat16 x bfloat16 -> float32, the second operand K-major.
__device__ __forceinline__ uint32_t instr_desc(int n) { return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(BM >> 4) << 24; }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// BN: rows of x a tile.  STAGES: x's ring.  PACKED: chunks of codes in shared memory.  MADE: stages of numbers in tensor memory.
template <bool GATED, int BN, int STAGES, int PACKED, bool SPLIT, int TEAMS>
__global__ void __launch_bounds__(threads_of(BN, TEAMS), TEAMS == 2 ? 2 : 1)
rows16_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, MxParams p) {
    constexpr int EPI_WARPS = epilogue_warps(BN), THREADS = threads_of(BN, TEAMS);
    constexpr int B_BYTES = BN * ROW, ACCUMULATORS = SPLIT || BN == 256 ? 1 : 2, OUTS = GATED ? BM / 2 : BM, SHARE = BN / (EPI_WARPS / 4);
    constexpr int ROOM = (512 - ACCUMULATORS * BN) / STAGE_COLS;
    constexpr int MADE = TEAMS == 2 ? 4 : STAGES < 8 ? (STAGES < ROOM ? STAGES : ROOM) : ROOM < 8 ? 4 : 8;
    constexpr int TMEM_COLS = power_of_two(ACCUMULATORS * BN + MADE * STAGE_COLS);
    static_assert(TMEM_COLS * (TEAMS == 2 ? 2 : 1) <= 512 && ACCUMULATORS * BN + MADE * STAGE_COLS <= TMEM_COLS, "tensor memory has 512 columns");
    static_assert(STAGES >= MADE, "a stage's barriers go round once more only after its place in tensor memory has been waited for");
    static_assert(!SPLIT || BM * BN * 4 <= STAGES * B_BYTES, "a split tile's sums go where the ring was");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ __align__(8) uint64_t packed_full[PACKED], packed_empty[PACKED];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int failed;

    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* packed_ring = stages + STAGES * B_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outs = GATED ? p.inter : p.N;
    const int x_tiles = (p.M + BN - 1) / BN, num_tiles = x_tiles * ((outs + OUTS - 1) / OUTS);
    const int all_chunks = (p.blocks * MX_BLOCK + CHUNK - 1) / CHUNK;
    const int rank = SPLIT && p.splits > 1 ? (int)pair_rank() : 0;
    const int first_tile = SPLIT ? (int)blockIdx.x / p.splits : (int)blockIdx.x, tile_step = SPLIT ? num_tiles : (int)gridDim.x;
    const int chunk0 = SPLIT ? (int)((long long)all_chunks * rank / p.splits) : 0;
    const int chunk1 = SPLIT ? (int)((long long)all_chunks * (rank + 1) / p.splits) : all_chunks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1 + TEAM);       // x's bytes, and the warps that made W's numbers
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tmem_full_bar[b], 1);
            mbar_init(&tmem_empty_bar[b], EPI_WARPS);
        }
        for (int b = 0; b < PACKED; ++b) {
            mbar_init(&packed_full[b], 1);
            mbar_init(&packed_empty[b], TEAM * TEAMS);
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
    const uint32_t tmem_made = tmem_base + ACCUMULATORS * BN;

    // x, or the weights themselves, may come from a kernel ahead on the stream: everyone waits for those, but for the warp that brings
    // codes written long ago
    const bool codes_first = p.settled && warp == 2 + EPI_WARPS;
    if (!codes_first) {
        chain_wait();
        chain_release();
    }

    if (warp == 0) {
        // ---------------------------------------------------------------- x
        if (lane == 0) {
            Ring<STAGES> r;
            for (int tile = first_tile; tile < num_tiles && !failed; tile += tile_step) {
                const int t0 = (tile % x_tiles) * BN;
                for (int kb = chunk0 * PER_CHUNK; kb < chunk1 * PER_CHUNK; ++kb, r.next()) {
                    if (!wait_for(&empty_bar[r.at], r.parity ^ 1, p.error, 41)) { failed = 1; break; }
                    mbar_expect_tx(&full_bar[r.at], B_BYTES);
                    tma_load_2d(stages + r.at * B_BYTES, &map_x, &full_bar[r.at], kb * BK, t0);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint32_t leader = elect_one();
        bool ok = true;                              // the same in all lanes
        Ring<STAGES> r;
        Ring<MADE> m;
        const uint64_t b_first = smem_desc(stages);
        int iter = 0;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++iter) {
            const int buf = ACCUMULATORS == 1 ? 0 : iter & 1, round = ACCUMULATORS == 1 ? iter : iter >> 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&tmem_empty_bar[buf], (round & 1) ^ 1, p.error, 44) && !failed);
            if (!ok) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + buf * BN;
            uint32_t add = 0;                        // the tile's first MMA starts its sums
            for (int left = (chunk1 - chunk0) * PER_CHUNK; left > 0; --left, r.next(), m.next()) {
                ok = __all_sync(0xffffffffu, wait_for(&full_bar[r.at], r.parity, p.error, 42));
                if (!ok) { failed = 1; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t b_desc = b_first + r.at * (B_BYTES / 16);
                const uint32_t a = tmem_made + m.at * STAGE_COLS;
#pragma unroll
                for (int k = 0; k < 4; ++k, add = 1) umma(leader, tmem_d, a + 8 * k, b_desc + 2 * k, instr_desc(BN), add);
                if (leader) umma_commit(&empty_bar[r.at]);
            }
            if (leader) umma_commit(&tmem_full_bar[buf]);
        }
    } else if (warp < 2 + EPI_WARPS) {
        // ---------------------------------------------------------------- epilogue
        const int quarter = warp & 3, first = ((warp - 2) >> 2) * SHARE;      // the 32 lanes this warp may read; its share of the columns
        const bool paired = (p.ldy & 1) == 0 && ((uintptr_t)p.y & 3) == 0;
        int iter = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++iter) {
            const int buf = ACCUMULATORS == 1 ? 0 : iter & 1, round = ACCUMULATORS == 1 ? iter : iter >> 1;
            const int t0 = (tile % x_tiles) * BN, f0 = (tile / x_tiles) * OUTS;
            const bool ok = mbar_wait(&tmem_full_bar[buf], round & 1, p.error, 43) && !failed;
            if (!__all_sync(0xffffffffu, ok)) { failed = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            finish_tile<GATED, SHARE, SPLIT>(p, tmem_base + buf * BN, first, t0, f0, outs, paired, quarter, lane, reinterpret_cast<float*>(stages),
                                             &tmem_empty_bar[buf]);
        }
    } else if (warp == 2 + EPI_WARPS) {
        // ---------------------------------------------------------------- codes of W, a chunk at a time
        if (lane == 0) {
            Ring<PACKED> b;
            for (int tile = first_tile; tile < num_tiles && !failed; tile += tile_step) {
                const int f0 = (tile / x_tiles) * OUTS;
                for (int chunk = chunk0; chunk < chunk1; ++chunk, b.next()) {
                    if (!wait_for(&packed_empty[b.at], b.parity ^ 1, p.error, 47)) { failed = 1; break; }
                    mbar_expect_tx(&packed_full[b.at], A_BYTES);
                    load_codes<GATED>(packed_ring + b.at * A_BYTES, &map_w, &packed_full[b.at], p, chunk * ROW, f0);
                }
            }
        }
        __syncwarp();
        if (codes_first) chain_wait();
    } else {
        // ---------------------------------------------------------------- codes to bfloat16 numbers
        // Team j makes quarter j of every chunk (of two teams each makes two), one stage, so that as many stages are in the making at a time; a
        // thread takes the row of its lane of tensor memory and both blocks of its quarter.  Eight lanes that read shared memory together have
        // eight neighbouring rows, whose 16-byte pieces the swizzle puts into different banks.
        const int team = (warp - 3 - EPI_WARPS) / TEAM, l = (warp & 3) * 32 + lane;
        const uint32_t to = tmem_made + ((uint32_t)((warp & 3) * 32) << 16);
        bool ok = true;
        Ring<PACKED> b;
        int kg = team;                               // the stage to make, counted over all tiles; its place in tensor memory is free when the
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {          // MMAs of stage kg - MADE have retired
            const int f0 = (tile / x_tiles) * OUTS;
            const uint8_t* scales = p.w_scales + (long long)min(row_of<GATED>(p, f0, l), p.N - 1) * p.w_ld_scales;
            auto load_scales = [&](int two) -> uint4 {                // the sixteen scales of two chunks; behind the last block 0
                const int b = two * 16;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (b + 16 <= p.blocks) {
                    v = __ldg(reinterpret_cast<const uint4*>(scales + b));
                } else if (b < p.blocks) {
                    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (b + i < p.blocks) w[i >> 2] |= (uint32_t)scales[b + i] << (8 * (i & 3));
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
                return v;
            };
            uint4 now = load_scales(chunk0 >> 1), next = make_uint4(0, 0, 0, 0);
            for (int chunk = chunk0; chunk < chunk1 && ok; ++chunk, b.next()) {
                if (!(chunk & 1) || chunk == chunk0) next = load_scales((chunk >> 1) + 1);
                ok = __all_sync(0xffffffffu, wait_for(&packed_full[b.at], b.parity, p.error, 48) && !failed);
                if (!ok) { failed = 1; break; }
#pragma unroll
                for (int quarter = team; quarter < PER_CHUNK; quarter += TEAMS, kg += TEAMS) {
                    const int m = kg % MADE;
                    uint4 code[2];
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        code[part] = *reinterpret_cast<const uint4*>(packed_ring + b.at * A_BYTES + l * ROW + (((quarter * 2 + part) ^ (l & 7)) << 4));
                    if (quarter + TEAMS >= PER_CHUNK) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&packed_empty[b.at]);
                    }
                    const uint32_t four = chunk & 1 ? (quarter & 2 ? now.w : now.z) : (quarter & 2 ? now.y : now.x);
                    const uint32_t sc = quarter & 1 ? four >> 16 : four & 0xffff;
                    const bool large = __any_sync(0xffffffffu, max(sc & 255, sc >> 8) > 128);
                    if (kg >= MADE) {
                        const int before = kg - MADE;
                        ok = __all_sync(0xffffffffu, wait_for(&empty_bar[before % STAGES], (before / STAGES) & 1, p.error, 46) && !failed);
                        if (!ok) { failed = 1; break; }
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        const uint32_t w[4] = {code[part].x, code[part].y, code[part].z, code[part].w};
                        const uint32_t scale = part ? sc >> 8 : sc & 255;
                        uint32_t q[16];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t four_of[4];
                            mx_spread_neighbours(w[j], four_of);
#pragma unroll
                            for (int e = 0; e < 4; ++e) q[4 * j + e] = four_of[e];
                        }
                        if (!large) {
                            const uint32_t factor = mx_factor(scale);
#pragma unroll
                            for (int e = 0; e < 16; ++e) q[e] = mx_mul(q[e], factor);
                        } else {
                            const MxFactor two = mx_factor_large(scale);
#pragma unroll
                            for (int e = 0; e < 16; ++e) q[e] = mx_mul(mx_mul(q[e], two.first), two.more);
                        }
                        tmem_st16(to + m * STAGE_COLS + part * 16, q);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full_bar[kg % STAGES]);
                }
                if (chunk & 1) now = next;
            }
        }
    }
    __syncwarp();
    if (SPLIT && p.splits > 1) {
        pair_sync();                                 // every CTA's sums are in its shared memory
        const int t0 = (first_tile % x_tiles) * BN, f0 = (first_tile / x_tiles) * OUTS;
        join_splits<GATED>(p, smem_u32(stages), rank, min(BN, p.M - t0), t0, f0, outs, threadIdx.x, THREADS,
                           [](int, int, float v) { return v; });
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

template <bool GATED, int BN, int STAGES, int PACKED, bool SPLIT, int TEAMS>
int run(const void* x, long long ldx, MxParams& p, long long tiles, int sms, int device, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (make_codes_map<GATED>(&map_w, p)) return 1;
    if (make_tile_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, p.M, p.K, ldx, BN, "gemm_mxfp4")) return 1;
    static unsigned long long allowed = 0;
    return launch_mxfp4(rows16_kernel<GATED, BN, STAGES, PACKED, SPLIT, TEAMS>, allowed, threads_of(BN, TEAMS),
                        (size_t)STAGES * BN * ROW + PACKED * A_BYTES + 1024, SPLIT, tiles, sms, device, map_w, map_x, p, stream);
}

template <bool GATED>
int dispatch(const void* x, long long ldx, MxParams& p, cudaStream_t stream) {
    int sms = 148, device = 0;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return cut_mxfp4<GATED, 256>(p, p.M, sms, [&](int bn, bool split, long long tiles) {
        if (bn == 256) return run<GATED, 256, 5, 3, false, 4>(x, ldx, p, tiles, sms, device, stream);
        if (bn == 128) return split ? run<GATED, 128, 4, 2, true, 2>(x, ldx, p, tiles, sms, device, stream)
                                    : run<GATED, 128, 8, 4, false, 4>(x, ldx, p, tiles, sms, device, stream);
        if (bn == 64) return run<GATED, 64, 6, 3, true, 2>(x, ldx, p, tiles, sms, device, stream);
        return run<GATED, 32, 8, 4, true, 2>(x, ldx, p, tiles, sms, device, stream);
    });
}

}  // namespace

int mxfp4_rows16(const void* x, long long ldx, MxParams& p, int gated, cudaStream_t stream) {
    return gated ? dispatch<true>(x, ldx, p, stream) : dispatch<false>(x, ldx, p, stream);
}
