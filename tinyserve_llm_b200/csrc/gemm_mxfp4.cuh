// What the products y = x . W^T with W in microscaled 4-bit floating point (mxfp4.cuh) share on the fifth-generation tensor cores:
// gemm_mxfp4_rows16.cu takes rows of x in bfloat16, gemm_mxfp4_rows4.cu rows in four bits too.
//
// W's rows are the M of the MMA, 128 a tile, and x's rows its N (BN: 32 to 256), so that a few rows of x cost an MMA of few columns and
// not one of 128 rows: accumulator lane = row of W, column = row of x.  K goes by chunks of 256 numbers, 128 bytes of codes a row.
//
// Gated (y = act(x Wgate^T, x Wup^T), W = [gate rows | up rows]): a tile holds 16 gate rows, the 16 up rows that belong to them, and so
// on, so that a gate lies 16 lanes before its up in the same warp's quarter of tensor memory and one shuffle brings them together.
//
// Many tiles: persistent, one CTA an SM, with two accumulators, so that a tile's epilogue runs under the next one's MMAs, or one of 256 columns,
// beside whose epilogue the next tile's operands are made.  Few tiles: a cluster of `splits` CTAs takes a tile, each its share of K, and leaves
// its sums in its own shared memory; each CTA then adds up a share of the columns from all of them, in the order of their ranks.  Nothing of
// that needs a workspace in global memory, and the order is fixed.
//
// Every wait on an mbarrier gives up after about two seconds, records where in an error word the host can read, and the CTA goes on to
// free its tensor memory and return.
#pragma once

#include "mxfp4.cuh"
#include "tcgen05.cuh"

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
    int one_box;                                       // gated: a tile's codes are one box of a map of four dimensions
    const __nv_bfloat16* x16;                          // rows in bfloat16 that came in pieces: themselves
    long long x16_ld;
    int settled;                                       // W may be read before the kernels ahead on the stream have finished
    int splits;
    int* error;
};

// Either form's products: the launcher's checks have been made.
int mxfp4_rows16(const void* x, long long ldx, MxParams& p, int gated, cudaStream_t stream);
int mxfp4_rows4(const void* x, long long ldx, MxParams& p, int gated, cudaStream_t stream);
// A few rows in bfloat16, 64 at most, as three pieces of eight bits, which take `scratch`.
long long mxfp4_pieces_bytes(int M, int blocks);
int mxfp4_pieces(const void* x, long long ldx, void* scratch, MxParams& p, int gated, cudaStream_t stream);

namespace {

constexpr int BM = 128, ROW = 128, CHUNK = 256;       // rows of W a tile; bytes of a row of codes (or of a stage); numbers they hold
constexpr int A_BYTES = BM * ROW;

// A bounded wait whose first look costs no clock: between MMAs of few columns the issuer's own instructions are what takes the time.  (A hint
// how long to sleep before a look fails made waits end later: 77 rows of 4,096 by 4,096 12.0 -> 14.4 us.)
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* error, int code) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done ? true : mbar_wait(bar, parity, error, code);
}
// A place in a ring of SIZE barriers and the parity of its round.
template <int SIZE>
struct Ring {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == SIZE) at = 0, parity ^= 1;
    }
};

__device__ __forceinline__ void tma_load_4d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(smem)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
}

// What tmem_ld16 reads is there; named, so that nothing that uses it comes before.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// The activation is chosen once for many values, so that what runs is one short loop and not four activations in a row.
template <int ACT>
__device__ __forceinline__ float gated_value(const MxParams& p, float g, float u) {
    if (ACT == TS_ACT_SILU) return __fdividef(g, 1.f + __expf(-g)) * u;
    return ts_gated_activation(ACT, g, u, p.act_limit, p.act_alpha);
}
template <int ACT>
__device__ __forceinline__ void gate_eight(const MxParams& p, float (&v)[8], const float (&u)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gated_value<ACT>(p, v[j], u[j]);
}
__device__ __forceinline__ float gate_one(const MxParams& p, float g, float u) {
    if (p.act == TS_ACT_SILU) return gated_value<TS_ACT_SILU>(p, g, u);
    return ts_gated_activation(p.act, g, u, p.act_limit, p.act_alpha);
}

// The row of W in lane l of a tile whose first output column is f0.
template <bool GATED>
__device__ __forceinline__ int row_of(const MxParams& p, int f0, int l) {
    if (!GATED) return f0 + l;
    return f0 + (l >> 5) * 16 + (l & 15) + ((l & 16) ? p.inter : 0);
}

__host__ __device__ constexpr int power_of_two(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

// Sixteen columns of a warp's quarter: column c of the accumulator is row t + c of x.  `f`: this lane's output column.  `whole`: all rows and
// columns are there and neighbours in a row start 4-byte aligned, which is most of a large product: no comparisons, and a lane swaps with its
// neighbour so that it stores two outputs at once.
template <bool GATED>
__device__ __forceinline__ void store_sixteen(const MxParams& p, const uint32_t (&acc)[16], int t, int f, int outs, bool whole, int lane) {
    const int odd = lane & 1;
    if (GATED) {
        float v[8], u[8];                            // the lower half of the lanes finishes columns 0, 2, ..., the upper one 1, 3, ...
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = __uint_as_float(acc[2 * j]), b = __uint_as_float(acc[2 * j + 1]);
            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? b : a, 16);
            v[j] = lane < 16 ? a : other;
            u[j] = lane < 16 ? other : b;
        }
        if (p.act == TS_ACT_SILU) gate_eight<TS_ACT_SILU>(p, v, u);
        else if (p.act == TS_ACT_RELU) gate_eight<TS_ACT_RELU>(p, v, u);
        else if (p.act == TS_ACT_CLAMPED_SWISH) gate_eight<TS_ACT_CLAMPED_SWISH>(p, v, u);
        else gate_eight<TS_ACT_GELU_TANH>(p, v, u);
        t += lane >> 4;
        const long long two_rows = 2 * p.ldy;
        if (whole) {                                 // an even lane stores both outputs of one row, an odd one of the row two further on
            __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)(t + 2 * odd) * p.ldy + f - odd;
#pragma unroll
            for (int j = 0; j < 8; j += 2, out += 2 * two_rows) {
                const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
                *reinterpret_cast<__nv_bfloat162*>(out) = odd ? __floats2bfloat162_rn(other, v[j + 1]) : __floats2bfloat162_rn(v[j], other);
            }
        } else if (f < outs) {
            __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)t * p.ldy + f;
#pragma unroll
            for (int j = 0; j < 8; ++j, out += two_rows)
                if (t + 2 * j < p.M) *out = __float2bfloat16_rn(v[j]);
        }
    } else if (p.out_f32) {
        float* out = (float*)p.y + (long long)t * p.ldy + f;
#pragma unroll
        for (int j = 0; j < 16; ++j, out += p.ldy)
            if (t + j < p.M && f < outs) *out = __uint_as_float(acc[j]);
    } else if (whole) {
        __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)(t + odd) * p.ldy + f - odd;
        const long long two_rows = 2 * p.ldy;
#pragma unroll
        for (int j = 0; j < 16; j += 2, out += two_rows) {
            const float a = __uint_as_float(acc[j]), b = __uint_as_float(acc[j + 1]);
            const float other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
            *reinterpret_cast<__nv_bfloat162*>(out) = odd ? __floats2bfloat162_rn(other, b) : __floats2bfloat162_rn(a, other);
        }
    } else if (f < outs) {
        __nv_bfloat16* out = (__nv_bfloat16*)p.y + (long long)t * p.ldy + f;
#pragma unroll
        for (int j = 0; j < 16; ++j, out += p.ldy)
            if (t + j < p.M) *out = __float2bfloat16_rn(__uint_as_float(acc[j]));
    }
}

// W's codes of a chunk, 128 rows of 128 bytes; gated 16 gate rows, their up rows, and so on, which a map of four dimensions (bytes, 16
// rows, halves, groups of 16 rows) brings in that order in one box.  Its groups have to be whole: else a box for every 16 rows.
template <bool GATED>
__device__ __forceinline__ void load_codes(unsigned char* to, const CUtensorMap* map, uint64_t* bar, const MxParams& p, int column, int f0) {
    if (!GATED) {
        tma_load_2d(to, map, bar, column, f0);
    } else if (p.one_box) {
        tma_load_4d(to, map, bar, column, 0, 0, f0 / 16);
    } else {
#pragma unroll
        for (int g = 0; g < BM / 16; ++g) tma_load_2d(to + g * 16 * ROW, map, bar, column, row_of<true>(p, f0, g * 16));
    }
}
// `spaced`: codes as elements of four bits, which TMA leaves 16 bytes for 16 of in shared memory, eight of them codes, as kind::mxf8f6f4 reads
// them; else as they are, two in a byte.  Either way a box has 128 elements, and 128 bytes of shared memory, a row.
template <bool GATED>
int make_codes_map(CUtensorMap* map, MxParams& p, bool spaced = false) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return ts_fail("gemm_mxfp4: the driver does not export cuTensorMapEncodeTiled");
    const CUtensorMapDataType type = spaced ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const cuuint64_t elements = (cuuint64_t)p.blocks * (spaced ? 32 : 16), ld = (cuuint64_t)p.w_ld_codes;
    p.one_box = GATED && p.inter % 16 == 0 && p.inter / 16 >= 4;
    const cuuint64_t dims[4] = {elements, p.one_box ? 16ull : (cuuint64_t)p.N, 2, (cuuint64_t)p.inter / 16};
    const cuuint64_t strides[3] = {ld, ld * p.inter, ld * 16};
    const cuuint32_t box[4] = {128, GATED ? 16u : (cuuint32_t)BM, 2, 4}, elem[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, type, p.one_box ? 4 : 2, const_cast<uint8_t*>(p.w_codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return ts_fail("gemm_mxfp4: cuTensorMapEncodeTiled failed with %d", (int)r);
    return 0;
}

// An epilogue warp's share of a tile: columns `first` to `first + SHARE` of the accumulator at `tmem`.  `sums`: where a split tile's go, by column
// and lane.
template <bool GATED, int SHARE, bool SPLIT>
__device__ __forceinline__ void finish_tile(const MxParams& p, uint32_t tmem, int first, int t0, int f0, int outs, bool paired, int quarter, int lane,
                                            float* sums, uint64_t* drained) {
    const uint32_t addr = tmem + first + ((uint32_t)(quarter * 32) << 16);
    const int f = GATED ? f0 + quarter * 16 + (lane & 15) : f0 + quarter * 32 + lane;
#pragma unroll 1
    for (int c0 = 0; c0 < SHARE; c0 += 16) {
        uint32_t acc[16];
        __syncwarp();
        tmem_ld16(addr + c0, acc);
        tmem_wait16(acc);
        if (!SPLIT && c0 + 16 == SHARE) {                             // the last of it: the accumulator goes back before the stores
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(drained);
        }
        if (SPLIT && p.splits > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(first + c0 + j) * BM + quarter * 32 + lane] = __uint_as_float(acc[j]);
        } else if (t0 + first + c0 < p.M) {
            store_sixteen<GATED>(p, acc, t0 + first + c0, f, outs, paired && t0 + first + c0 + 16 <= p.M && f0 + (GATED ? BM / 2 : BM) <= outs, lane);
        }
    }
}

// A split tile's share of columns, added up over the cluster's CTAs, four neighbouring lanes a thread: `id` of `threads` this one.
// `again` gets each sum and may put another in its place.
template <bool GATED, typename Again>
__device__ __forceinline__ void join_splits(const MxParams& p, uint32_t sums, int rank, int columns, int t0, int f0, int outs, int id, int threads,
                                            const Again& again) {
    constexpr int QUADS = (GATED ? BM / 2 : BM) / 4;
    auto total = [&](int column, int l, float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = 0.f;
        for (int r0 = 0; r0 < p.splits; r0 += 4) {                    // four asked for before the first is added
            float part[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (r0 + r >= p.splits) break;
                uint32_t remote;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(sums + (uint32_t)(column * BM + l) * 4), "r"(r0 + r));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(part[r][0]), "=f"(part[r][1]), "=f"(part[r][2]), "=f"(part[r][3]) : "r"(remote));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (r0 + r >= p.splits) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += part[r][e];
            }
        }
    };
    const int f = (id % QUADS) * 4;
    for (int c = rank + p.splits * (id / QUADS); c < columns && id / QUADS < threads / QUADS; c += p.splits * (threads / QUADS)) {
        const long long at = (long long)(t0 + c) * p.ldy + f0 + f;
        float v[4];
        if (GATED) {
            const int l = (f >> 4) * 32 + (f & 15);
            float u[4];
            total(c, l, v);
            total(c, l + 16, u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (f0 + f + e >= outs) break;
                v[e] = gate_one(p, again(l + e, t0 + c, v[e]), again(l + 16 + e, t0 + c, u[e]));
            }
        } else {
            total(c, f, v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (f0 + f + e < outs) v[e] = again(f + e, t0 + c, v[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (f0 + f + e >= outs) break;
            if (!GATED && p.out_f32) ((float*)p.y)[at + e] = v[e];
            else ((__nv_bfloat16*)p.y)[at + e] = __float2bfloat16_rn(v[e]);
        }
    }
}

// Launches `kernel` over the tiles: persistent on `sms` SMs, or (`split`) a cluster of p.splits CTAs a tile.
template <typename Kernel>
int launch_mxfp4(Kernel kernel, unsigned long long& allowed, int threads, size_t smem, bool split, long long tiles, int sms, int device,
                 const CUtensorMap& map_w, const CUtensorMap& map_x, const MxParams& p, cudaStream_t stream) {
    if (device >= 64 || !(allowed >> device & 1)) {                   // a bit a device: what the kernel may ask for is set once on each
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ts_fail("gemm_mxfp4: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
        if (device < 64) allowed |= 1ull << device;
    }
    TS_REQUIRE(tiles * p.splits <= 0x7fffffffll, "gemm_mxfp4: too many tiles");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(split ? tiles * p.splits : (tiles < sms ? tiles : sms)));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int attrs = 0;
    if (ts_chaining_enabled()) {
        attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[attrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.splits > 1) {
        attr[attrs].id = cudaLaunchAttributeClusterDimension;
        attr[attrs].val.clusterDim.x = p.splits;
        attr[attrs].val.clusterDim.y = 1;
        attr[attrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = attrs;
    TS_CHAINED_CHECK("gemm_mxfp4", cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p));
    return 0;
}

// CTAs a tile: as many as there are SMs for, up to a cluster's eight and the chunks of K.
inline int splits_of(const MxParams& p, long long tiles, int sms) {
    const int chunks = (p.blocks * MX_BLOCK + CHUNK - 1) / CHUNK;
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= chunks) splits *= 2;
    return splits;
}

// How a product is cut.  run(bn, split, tiles) launches tiles of bn rows of x (WIDE, 256, 128, 64, 32).
template <bool GATED, int WIDE, typename Run>
int cut_mxfp4(MxParams& p, int rows, int sms, const Run& run) {
    const long long outs = GATED ? p.inter : p.N, per = GATED ? BM / 2 : BM, w_tiles = (outs + per - 1) / per;
    auto tiles_of = [&](int bn) { return w_tiles * ((rows + bn - 1) / bn); };
    p.splits = 1;
    if (rows > 128) {
        if (tiles_of(256) <= sms && tiles_of(256) * 4 >= 3ll * sms) return run(256, true, tiles_of(256));
        // wide tiles or narrow ones, by the rounds they take and what a tile costs beside its columns
        auto cost = [&](int bn) { return (tiles_of(bn) + sms - 1) / sms * (bn + 128); };
        if (tiles_of(WIDE) > sms && cost(WIDE) <= cost(128)) return run(WIDE, false, tiles_of(WIDE));
    }
    const int bn = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const long long tiles = tiles_of(bn);
    if (tiles > sms) return run(bn, false, tiles);
    p.splits = splits_of(p, tiles, sms);
    return run(bn, true, tiles);
}

}  // namespace
