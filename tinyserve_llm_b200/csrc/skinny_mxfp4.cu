// y = x . W^T for a handful of rows of x (decode steps) with W in microscaled 4-bit floating point (mxfp4.cuh): float32 sums on tensor
// cores (mma.sync m16n8k16), rows of x in bfloat16 or in four bits.  W is the tall operand: a CTA takes 16 of its rows (gated: 8 gate rows
// and their 8 up rows), its warps split K between them in units of 128 numbers, four blocks, one for each of the four threads that share a
// row: a thread streams its block's 16 bytes of codes of two rows, spreads them to bfloat16 in registers and multiplies.  The k indices inside
// a unit are permuted the same way on both sides, so nothing is shuffled: codes i and i + 4 of a word share a register (mx_spread), and x's
// numbers are paired the same way.
//
// Every thread owns a ring of slots in shared memory for its own blocks, filled by cp.async, so the copies in flight are bounded by shared
// memory and there is no barrier.  Weights written long ago (`settled`) are asked for before the wait for the kernel ahead on the stream.
//
// Not bound by memory: a unit's 1,088 bytes of W take 330 instructions of a warp, 200 of them to spread its codes, where HBM brings them in the
// time of 190, and x's loads, 16 bytes a thread of 64-byte pieces, keep L1 busy (2,048 by 8,192, eight rows: 9.0 us, 7.5 where W was written
// long ago; L1 0.64 busy, a third of the issue slots, DRAM 0.09).  What it has is the least between launch and end: 2,048 by 2,048, one row,
// 3.0 us (2.4).
//
// The split of K depends on N and K only, so among the calls that come here a row's result does not depend on the rows beside it.  Which kernel a
// call takes does depend on their number (gemm_mxfp4.cu: it changes behind 8, 16, 32 and 64 rows), and another kernel adds in another order.
#include "mxfp4.cuh"
#include "skinny_mxfp4.h"

namespace {

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool there) {              // not there: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async4(void* smem, const void* gmem, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(there ? 4 : 0)
                 : "memory");
}

// A block's numbers, eight at a time, paired as mx_spread pairs them.
__device__ __forceinline__ void block_numbers(uint32_t word, uint32_t scale, bool large, uint32_t (&q)[4]) {
    mx_spread(word, q);
    if (!large) {
        const uint32_t factor = mx_factor(scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = mx_mul(q[i], factor);
    } else {
        const MxFactor two = mx_factor_large(scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = mx_mul(mx_mul(q[i], two.first), two.more);
    }
}

// MT: tiles of 8 rows of x; WARPS: the split of K; MINB: CTAs an SM the registers are held to; PJ: slots of a thread's ring.
template <int MT, int WARPS, bool GATED, bool X4, typename OUT, int MINB, int PJ>
__global__ void __launch_bounds__(WARPS * 32, MINB) skinny_mxfp4_kernel(SkinnyMx p) {
    constexpr int THREADS = WARPS * 32;
    __shared__ float partial[WARPS][MT][32][4];
    extern __shared__ uint4 ring[];                                   // codes [PJ][low, high][thread], then scales, four bytes a thread
    uint32_t* scale_ring = reinterpret_cast<uint32_t*>(ring + PJ * 2 * THREADS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    long long row_low, row_high;
    int rows_valid;
    if (GATED) {
        const int base = blockIdx.x * 8, inter = p.N / 2;
        rows_valid = min(8, inter - base);
        row_low = base + min(r, rows_valid - 1);
        row_high = (long long)inter + row_low;
    } else {
        const int base = blockIdx.x * 16;
        rows_valid = min(16, p.N - base);
        row_low = base + min(r, rows_valid - 1);
        row_high = base + min(r + 8, rows_valid - 1);
    }
    const uint8_t* codes_low = p.w_codes + row_low * p.w_ld_codes;
    const uint8_t* codes_high = p.w_codes + row_high * p.w_ld_codes;
    const uint8_t* scales_low = p.w_scales + row_low * p.w_ld_scales;
    const uint8_t* scales_high = p.w_scales + row_high * p.w_ld_scales;
    const int units = (p.blocks + 3) / 4, steps = warp < units ? (units - warp + WARPS - 1) / WARPS : 0;
    auto fill = [&](int j) {                                          // unit j of this warp into its slot; behind the last block zeros
        if (j < steps) {
            const int u = j * WARPS + warp, block = u * 4 + c, slot = j % PJ;
            const bool there = block < p.blocks;
            const long long at = there ? block * 16 : 0;
            cp_async16(&ring[(slot * 2 + 0) * THREADS + threadIdx.x], codes_low + at, there);
            cp_async16(&ring[(slot * 2 + 1) * THREADS + threadIdx.x], codes_high + at, there);
            // the four scales of the unit, of which this thread's is byte c (a row of scales starts 16-byte aligned)
            cp_async4(&scale_ring[(slot * 2 + 0) * THREADS + threadIdx.x], scales_low + u * 4, true);
            cp_async4(&scale_ring[(slot * 2 + 1) * THREADS + threadIdx.x], scales_high + u * 4, true);
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    if (!p.settled) chain_wait();
#pragma unroll
    for (int j = 0; j < PJ; ++j) fill(j);
    if (p.settled) chain_wait();
    chain_release();

    // x: the thread's block of a unit, of row t * 8 + r: 32 numbers
    struct Rows {
        uint4 v[MT][X4 ? 1 : 4];
        uint32_t scale[MT];
    };
    auto load_x = [&](int j, Rows& x) {
        const int block = (j * WARPS + warp) * 4 + c;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int token = t * 8 + r;
            if (X4) {
                const bool there = token < p.M && block < p.blocks;
                x.v[t][0] = there ? *reinterpret_cast<const uint4*>((const uint8_t*)p.x + token * p.ldx + block * 16) : make_uint4(0, 0, 0, 0);
                x.scale[t] = there ? p.x_scales[token * p.x_ld_scales + block] : 0;
            } else {
                const __nv_bfloat16* at = (const __nv_bfloat16*)p.x + token * p.ldx + block * 32;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x.v[t][i] = token < p.M && block * 32 + i * 8 < p.K ? *reinterpret_cast<const uint4*>(at + i * 8) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    float acc[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    Rows x, next;
    if (steps > 0) load_x(0, x);
    for (int j = 0; j < steps; ++j) {
        if (j + 1 < steps) load_x(j + 1, next);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(PJ - 1) : "memory");       // this step's copies have landed
        const int slot = j % PJ;
        const uint4 low = ring[(slot * 2 + 0) * THREADS + threadIdx.x], high = ring[(slot * 2 + 1) * THREADS + threadIdx.x];
        const bool there = (j * WARPS + warp) * 4 + c < p.blocks;
        const uint32_t s_low = there ? __byte_perm(scale_ring[(slot * 2 + 0) * THREADS + threadIdx.x], 0, 0x4440 | c) : 0;
        const uint32_t s_high = there ? __byte_perm(scale_ring[(slot * 2 + 1) * THREADS + threadIdx.x], 0, 0x4440 | c) : 0;
        uint32_t most = max(s_low, s_high);
        if (X4) {
#pragma unroll
            for (int t = 0; t < MT; ++t) most = max(most, x.scale[t]);
        }
        const bool large = __any_sync(0xffffffffu, mx_large(most));
        const uint32_t wl[4] = {low.x, low.y, low.z, low.w}, wh[4] = {high.x, high.y, high.z, high.w};
        auto multiply = [&](const bool large_) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t a[4], b[4];
                block_numbers(wl[i], s_low, large_, a);
                block_numbers(wh[i], s_high, large_, b);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    uint32_t v[4];
                    if (X4) {
                        const uint32_t word = i == 0 ? x.v[t][0].x : i == 1 ? x.v[t][0].y : i == 2 ? x.v[t][0].z : x.v[t][0].w;
                        block_numbers(word, x.scale[t], large_, v);
                    } else {
                        const uint4 e = x.v[t][i % (X4 ? 1 : 4)];
                        v[0] = __byte_perm(e.x, e.z, 0x5410), v[1] = __byte_perm(e.x, e.z, 0x7632);
                        v[2] = __byte_perm(e.y, e.w, 0x5410), v[3] = __byte_perm(e.y, e.w, 0x7632);
                    }
                    mma_bf16(acc[t], a[0], b[0], a[1], b[1], v[0], v[1]);
                    mma_bf16(acc[t], a[2], b[2], a[3], b[3], v[2], v[3]);
                }
            }
        };
        if (large) multiply(true);
        else multiply(false);
        fill(j + PJ);                                                 // the slot's values sit in registers
        x = next;
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) partial[warp][t][lane][e] = acc[t][e];
    __syncthreads();
    // the warps' sums in their order; [t][lane][e]: row lane / 4 (+ 8 for e >= 2), token t * 8 + (lane % 4) * 2 + e % 2
    constexpr int PER = GATED ? 2 : 4;
    for (int i = threadIdx.x; i < MT * 32 * PER; i += THREADS) {
        // neighbouring threads take neighbouring rows of W, whose outputs lie together
        const int row8 = i % 8, rest = i / 8, half = GATED ? 0 : rest % 2, token = GATED ? rest : rest / 2;
        const int t = token / 8, l = row8 * 4 + (token % 8) / 2, e = token % 2 + 2 * half;
        float v = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            v += partial[w][t][l][e];
            if (GATED) u += partial[w][t][l][e + 2];
        }
        const int row = row8 + 8 * half;
        if (row >= rows_valid || token >= p.M) continue;
        if (GATED) v = p.act == TS_ACT_SILU ? __fdividef(v, 1.f + __expf(-v)) * u : ts_gated_activation(p.act, v, u, p.act_limit, p.act_alpha);
        ((OUT*)p.y)[token * p.ldy + blockIdx.x * (GATED ? 8 : 16) + row] = from_float<OUT>(v);
    }
}

template <int MT, int WARPS, bool GATED, bool X4, typename OUT, int MINB, int PJ>
int launch(const SkinnyMx& p, cudaStream_t stream) {
    const int tiles = GATED ? (p.N / 2 + 7) / 8 : (p.N + 15) / 16;
    const size_t smem = (size_t)PJ * 2 * WARPS * 32 * (16 + 4);
    auto kernel = skinny_mxfp4_kernel<MT, WARPS, GATED, X4, OUT, MINB, PJ>;
    static unsigned long long allowed = 0;             // a bit a device
    int device = 0;
    if (smem + sizeof(float) * WARPS * MT * 128 > 48 * 1024 && cudaGetDevice(&device) == cudaSuccess && (device >= 64 || !(allowed >> device & 1))) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ts_fail("skinny_mxfp4: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
        if (device < 64) allowed |= 1ull << device;
    }
    TS_CHAINED_CHECK("skinny_mxfp4", launch_chained(kernel, dim3(tiles), dim3(WARPS * 32), smem, stream, p));
    return 0;
}

// How a product is cut into CTAs, from N and K only: many tiles of rows of W, four warps a tile and six CTAs an SM; 149 to 296 tiles, eight
// warps, two CTAs; fewer, sixteen warps.
template <int MT, bool GATED, bool X4, typename OUT>
int dispatch_warps(const SkinnyMx& p, cudaStream_t stream) {
    const int tiles = GATED ? (p.N / 2 + 7) / 8 : (p.N + 15) / 16;
    if (tiles > 296 || p.blocks < 32) return launch<MT, 4, GATED, X4, OUT, MT == 1 ? 6 : 4, 4>(p, stream);
    if (tiles > 148) return launch<MT, 8, GATED, X4, OUT, 2, 4>(p, stream);
    return launch<MT, 16, GATED, X4, OUT, 1, 4>(p, stream);
}
template <int MT, bool X4>
int dispatch_out(const SkinnyMx& p, int gated, int out_f32, cudaStream_t stream) {
    if (gated) return dispatch_warps<MT, true, X4, __nv_bfloat16>(p, stream);
    return out_f32 ? dispatch_warps<MT, false, X4, float>(p, stream) : dispatch_warps<MT, false, X4, __nv_bfloat16>(p, stream);
}

}  // namespace

int skinny_mxfp4(const SkinnyMx& p, int gated, int out_f32, cudaStream_t stream) {
    if (p.M <= 8) return p.x_scales ? dispatch_out<1, true>(p, gated, out_f32, stream) : dispatch_out<1, false>(p, gated, out_f32, stream);
    return p.x_scales ? dispatch_out<2, true>(p, gated, out_f32, stream) : dispatch_out<2, false>(p, gated, out_f32, stream);
}
