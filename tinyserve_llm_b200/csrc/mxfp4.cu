// Numbers to microscaled 4-bit floating point and back (mxfp4.cuh says how it is laid out).
//
// Quantisation: with a the largest magnitude of a block, s = floor(log2 a) - 2 + 127, at least 0; the codes are the nearest to
// x / 2^(s - 127), ties to the even code, magnitudes over 6 to 6.  floor(log2 a) of a normal float32 is its exponent field; a subnormal
// a gives s = 0 either way.  A block that holds an infinity or a NaN gets s = 255 and codes 0.  The division is a product with a power
// of two, exact but for results below 2^-126, which are codes 0 whatever they round to, so the only rounding is the one to four bits.
//
// Every number is read once, every byte written once.  Two lanes take a block, sixteen numbers a lane, by 32-byte loads (and stores, the
// other way) where rows are aligned to them; one shuffle joins the maximum, which is found among the numbers' bits, where what is not finite is
// largest.  With eight numbers a lane the index arithmetic and two shuffles were as much work again: 28,672 by 4,096 bfloat16 numbers 87 us there
// and 77 back.  Columns that end inside a block are zeros there.
#include "mxfp4.cuh"

namespace {

constexpr int THREADS = 256, EACH = 16;                // numbers a lane

struct Eight {
    uint32_t w[8];
};
__device__ __forceinline__ Eight load32(const void* p) {
    Eight v;
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7]) : "l"(p));
    return v;
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// A lane's place: row, and which sixteen numbers of it.  32 bits do for matrices of up to 2^31 sixteens.
__device__ __forceinline__ void place(long long at, int sixteens, long long total, long long& row, int& part) {
    row = total <= 0x7fffffffll ? (long long)((uint32_t)at / (uint32_t)sixteens) : at / sixteens;
    part = (int)(at - row * sixteens);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_mxfp4_kernel(const T* __restrict__ x, uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                 long long rows, int cols, long long ldx, int sixteens, long long ld_codes,
                                                                 long long ld_scales, int wide) {
    chain_wait();
    chain_release();
    const long long total = rows * sixteens, first = (long long)blockIdx.x * THREADS + (threadIdx.x & ~31), at = first + (threadIdx.x & 31);
    if (first >= total) return;                                    // a whole warp: a block's two lanes are there or not as one
    const bool mine = at < total;
    long long row = 0;
    int part = 0;
    if (mine) place(at, sixteens, total, row, part);
    const int valid = mine ? cols - part * EACH : 0;
    const T* from = x + row * ldx + part * EACH;
    float v[EACH];
    uint32_t top = 0;
    if (wide && valid >= EACH) {
        if (sizeof(T) == 2) {
            const Eight q = load32(from);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[2 * i] = __uint_as_float(q.w[i] << 16);
                v[2 * i + 1] = __uint_as_float(q.w[i] & 0xffff0000u);
            }
        } else {
            const Eight q = load32(from), r = load32(from + 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(q.w[i]), v[8 + i] = __uint_as_float(r.w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = i < valid ? to_float<T>(from[i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const int exponent = (int)(top >> 23), s = exponent == 255 ? 255 : max(exponent - 2, 0);
    uint2 packed = make_uint2(0, 0);
    if (exponent != 255) {
        const float inverse = __uint_as_float((uint32_t)(254 - s) << 23);       // 2^(127 - s): the exponent field is at least 2 (s <= 252)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            packed.x |= mx_codes_of_two(v[2 * i] * inverse, v[2 * i + 1] * inverse) << (8 * i);
            packed.y |= mx_codes_of_two(v[8 + 2 * i] * inverse, v[9 + 2 * i] * inverse) << (8 * i);
        }
    }
    if (mine) {
        codes[row * ld_codes + part] = packed;
        if ((part & 1) == 0) scales[row * ld_scales + (part >> 1)] = (uint8_t)s;
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) dequantize_mxfp4_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                   T* __restrict__ y, long long rows, int cols, int sixteens,
                                                                   long long ld_codes, long long ld_scales, int wide) {
    chain_wait();
    chain_release();
    const long long total = rows * sixteens, at = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (at >= total) return;
    long long row;
    int part;
    place(at, sixteens, total, row, part);
    const int valid = cols - part * EACH;
    if (valid <= 0) return;
    const uint2 w = codes[row * ld_codes + part];
    const float scale = mx_scale(scales[row * ld_scales + (part >> 1)]);
    float v[EACH];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t p[4];
        mx_spread(h ? w.y : w.x, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                              // times 2^126: the code's value; a float32 holds both factors' product
            v[8 * h + i] = __uint_as_float(p[i] << 16) * 0x1p126f * scale;
            v[8 * h + i + 4] = __uint_as_float(p[i] & 0xffff0000u) * 0x1p126f * scale;
        }
    }
    T* out = y + row * cols + part * EACH;
    if (wide && valid >= EACH) {
        if (sizeof(T) == 2) {
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                q[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            store32(out, q);
        } else {
            store32(out, reinterpret_cast<const uint32_t*>(v));
            store32(out + 8, reinterpret_cast<const uint32_t*>(v) + 8);
        }
    } else {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (i < valid) out[i] = from_float<T>(v[i]);
    }
}

}  // namespace

// codes: rows of 16 bytes a block; scales: rows of one byte a block, ld_scales apart.
TS_API int ts_quantize_mxfp4(const void* x, void* codes, void* scales, long long rows, int cols, long long ldx, long long ld_codes,
                             long long ld_scales, int dtype, cudaStream_t stream) {
    TS_REQUIRE(rows >= 0 && cols > 0 && cols <= MX_MOST, "quantize_mxfp4: bad sizes: %lld rows of %d", rows, cols);
    TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "quantize_mxfp4: unknown dtype %d", dtype);
    const int blocks = (cols + MX_BLOCK - 1) / MX_BLOCK, size = dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ld_codes >= (long long)blocks * 16 && ld_codes % 8 == 0 && (uintptr_t)codes % 8 == 0 && ld_scales >= blocks,
               "quantize_mxfp4: rows of %lld bytes of codes and %lld scales for %d blocks", ld_codes, ld_scales, blocks);
    if (rows == 0) return 0;
    const int wide = (uintptr_t)x % 32 == 0 && (ldx * size) % 32 == 0;
    TS_REQUIRE(rows * blocks * 2 / THREADS < 0x7fffffffll, "mxfp4: %lld rows of %d blocks", rows, blocks);
    const dim3 grid((unsigned)((rows * blocks * 2 + THREADS - 1) / THREADS)), threads(THREADS);
    if (dtype == TS_F32)
        TS_CHAINED_CHECK("quantize_mxfp4", launch_chained(quantize_mxfp4_kernel<float>, grid, threads, 0, stream, (const float*)x, (uint2*)codes,
                                                          (uint8_t*)scales, rows, cols, ldx, blocks * 2, ld_codes / 8, ld_scales, wide));
    else
        TS_CHAINED_CHECK("quantize_mxfp4", launch_chained(quantize_mxfp4_kernel<__nv_bfloat16>, grid, threads, 0, stream, (const __nv_bfloat16*)x,
                                                          (uint2*)codes, (uint8_t*)scales, rows, cols, ldx, blocks * 2, ld_codes / 8,
                                                          ld_scales, wide));
    return 0;
}

TS_API int ts_dequantize_mxfp4(const void* codes, const void* scales, void* y, long long rows, int cols, long long ld_codes,
                               long long ld_scales, int dtype, cudaStream_t stream) {
    TS_REQUIRE(rows >= 0 && cols > 0 && cols <= MX_MOST, "dequantize_mxfp4: bad sizes: %lld rows of %d", rows, cols);
    TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "dequantize_mxfp4: unknown dtype %d", dtype);
    const int blocks = (cols + MX_BLOCK - 1) / MX_BLOCK, size = dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ld_codes >= (long long)blocks * 16 && ld_codes % 8 == 0 && (uintptr_t)codes % 8 == 0 && ld_scales >= blocks,
               "dequantize_mxfp4: rows of %lld bytes of codes and %lld scales for %d blocks", ld_codes, ld_scales, blocks);
    if (rows == 0) return 0;
    const int wide = (uintptr_t)y % 32 == 0 && ((long long)cols * size) % 32 == 0;
    TS_REQUIRE(rows * blocks * 2 / THREADS < 0x7fffffffll, "mxfp4: %lld rows of %d blocks", rows, blocks);
    const dim3 grid((unsigned)((rows * blocks * 2 + THREADS - 1) / THREADS)), threads(THREADS);
    if (dtype == TS_F32)
        TS_CHAINED_CHECK("dequantize_mxfp4", launch_chained(dequantize_mxfp4_kernel<float>, grid, threads, 0, stream, (const uint2*)codes,
                                                            (const uint8_t*)scales, (float*)y, rows, cols, blocks * 2, ld_codes / 8, ld_scales, wide));
    else
        TS_CHAINED_CHECK("dequantize_mxfp4", launch_chained(dequantize_mxfp4_kernel<__nv_bfloat16>, grid, threads, 0, stream, (const uint2*)codes,
                                                            (const uint8_t*)scales, (__nv_bfloat16*)y, rows, cols, blocks * 2, ld_codes / 8, ld_scales,
                                                            wide));
    return 0;
}
