// Numbers to microscaled 4-bit floating point and back (mxfp4.cuh says how it is laid out).
//
// Quantisation: with a the largest magnitude of a block, s = floor(log2 a) - 2 + 127, at least 0; the codes are the nearest to
// x / 2^(s - 127), ties to the even code, magnitudes over 6 to 6.  floor(log2 a) of a normal float32 is its exponent field; a subnormal
// a gives s = 0 either way.  A block that holds an infinity or a NaN gets s = 255 and codes 0.  The division is a product with a power
// of two, exact but for results below 2^-126, which are codes 0 whatever they round to, so the only rounding is the one to four bits.
//
// Bound by memory: every number is read once, every byte written once.  Four lanes take a block, eight numbers a lane: one or two
// 16-byte loads, two shuffles for the maximum, four bytes of codes a lane, so that a warp reads 256 numbers and writes 128 bytes that lie
// one behind the other.  Columns that end inside a block are zeros there.
#include "mxfp4.cuh"

namespace {

constexpr int THREADS = 256;

template <typename T>
__device__ __forceinline__ void load_eight(const T* p, int valid, bool wide, float (&v)[8]) {
    if (wide && valid >= 8) {
        if (sizeof(T) == 2) {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_float<T>(p[i]) : 0.f;
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_mxfp4_kernel(const T* __restrict__ x, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                 long long rows, int cols, long long ldx, int eighths, long long ld_codes,
                                                                 long long ld_scales, int wide) {
    chain_wait();
    chain_release();
    const long long total = rows * eighths;                       // eighths: lanes of a row, a multiple of four
    // the warp's lanes run together: a block's four lanes are in it or out of it as one, but all of them take part in the shuffles
    for (long long first = (long long)blockIdx.x * THREADS + (threadIdx.x & ~31); first < total; first += (long long)gridDim.x * THREADS) {
        const long long at = first + (threadIdx.x & 31);
        const bool mine = at < total;
        const long long row = total <= 0x7fffffffll ? (long long)((uint32_t)at / (uint32_t)eighths) : at / eighths;
        const int part = (int)(at - row * eighths);
        float v[8];
        load_eight<T>(x + (mine ? row * ldx + part * 8 : 0), mine ? cols - part * 8 : 0, wide, v);
        float top = 0.f;
        bool odd = false;                                          // an infinity or a NaN
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = fmaxf(top, fabsf(v[i]));
            odd |= !(fabsf(v[i]) <= 3.402823466e38f);
        }
        uint32_t bits = odd ? 0x7f800000u : __float_as_uint(top);  // magnitudes order as their bits do
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
        const int exponent = (int)(bits >> 23);
        const int s = exponent == 255 ? 255 : max(exponent - 2, 0);
        // 2^(127 - s): exponent field 254 - s, which is at least 2 (s <= 252)
        const float inverse = exponent == 255 ? 0.f : __uint_as_float((uint32_t)(254 - s) << 23);
        uint32_t packed = 0;
        if (exponent != 255) {
#pragma unroll
            for (int i = 0; i < 4; ++i) packed |= mx_codes_of_two(v[2 * i] * inverse, v[2 * i + 1] * inverse) << (8 * i);
        }
        if (mine) {
            codes[row * ld_codes + part] = packed;
            if ((part & 3) == 0) scales[row * ld_scales + (part >> 2)] = (uint8_t)s;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) dequantize_mxfp4_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                   T* __restrict__ y, long long rows, int cols, int eighths,
                                                                   long long ld_codes, long long ld_scales, int wide) {
    chain_wait();
    chain_release();
    const long long total = rows * eighths;
    for (long long at = (long long)blockIdx.x * THREADS + threadIdx.x; at < total; at += (long long)gridDim.x * THREADS) {
        const long long row = total <= 0x7fffffffll ? (long long)((uint32_t)at / (uint32_t)eighths) : at / eighths;
        const int part = (int)(at - row * eighths), valid = cols - part * 8;
        if (valid <= 0) continue;
        const uint32_t w = codes[row * ld_codes + part];
        const float scale = mx_scale(scales[row * ld_scales + (part >> 2)]);
        float v[8];
        uint32_t p[4];
        mx_spread(w, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                              // times 2^126: the code's value; a float32 holds both factors' product
            v[i] = __uint_as_float(p[i] << 16) * 0x1p126f * scale;
            v[i + 4] = __uint_as_float(p[i] & 0xffff0000u) * 0x1p126f * scale;
        }
        T* out = y + row * cols + part * 8;
        if (wide && valid >= 8) {
            if (sizeof(T) == 2) {
                uint4 q;
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                *reinterpret_cast<uint4*>(out) = q;
            } else {
                reinterpret_cast<float4*>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) out[i] = from_float<T>(v[i]);
        }
    }
}

int blocks_for(long long lanes) {
    const long long blocks = (lanes + THREADS - 1) / THREADS, most = 148 * 8 * 4;
    return (int)(blocks < most ? blocks : most);
}

}  // namespace

// codes: rows of 16 bytes a block; scales: rows of one byte a block, ld_scales apart.
TS_API int ts_quantize_mxfp4(const void* x, void* codes, void* scales, long long rows, int cols, long long ldx, long long ld_codes,
                             long long ld_scales, int dtype, cudaStream_t stream) {
    TS_REQUIRE(rows >= 0 && cols > 0, "quantize_mxfp4: bad sizes: %lld rows of %d", rows, cols);
    TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "quantize_mxfp4: unknown dtype %d", dtype);
    const int blocks = (cols + MX_BLOCK - 1) / MX_BLOCK, size = dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ld_codes >= (long long)blocks * 16 && ld_codes % 4 == 0 && (uintptr_t)codes % 4 == 0 && ld_scales >= blocks,
               "quantize_mxfp4: rows of %lld bytes of codes and %lld scales for %d blocks", ld_codes, ld_scales, blocks);
    if (rows == 0) return 0;
    const int wide = (uintptr_t)x % 16 == 0 && (ldx * size) % 16 == 0;
    const dim3 grid(blocks_for(rows * blocks * 4)), threads(THREADS);
    if (dtype == TS_F32)
        TS_CHAINED_CHECK("quantize_mxfp4", launch_chained(quantize_mxfp4_kernel<float>, grid, threads, 0, stream, (const float*)x, (uint32_t*)codes,
                                                          (uint8_t*)scales, rows, cols, ldx, blocks * 4, ld_codes / 4, ld_scales, wide));
    else
        TS_CHAINED_CHECK("quantize_mxfp4", launch_chained(quantize_mxfp4_kernel<__nv_bfloat16>, grid, threads, 0, stream, (const __nv_bfloat16*)x,
                                                          (uint32_t*)codes, (uint8_t*)scales, rows, cols, ldx, blocks * 4, ld_codes / 4,
                                                          ld_scales, wide));
    return 0;
}

TS_API int ts_dequantize_mxfp4(const void* codes, const void* scales, void* y, long long rows, int cols, long long ld_codes,
                               long long ld_scales, int dtype, cudaStream_t stream) {
    TS_REQUIRE(rows >= 0 && cols > 0, "dequantize_mxfp4: bad sizes: %lld rows of %d", rows, cols);
    TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "dequantize_mxfp4: unknown dtype %d", dtype);
    const int blocks = (cols + MX_BLOCK - 1) / MX_BLOCK, size = dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ld_codes >= (long long)blocks * 16 && ld_codes % 4 == 0 && (uintptr_t)codes % 4 == 0 && ld_scales >= blocks,
               "dequantize_mxfp4: rows of %lld bytes of codes and %lld scales for %d blocks", ld_codes, ld_scales, blocks);
    if (rows == 0) return 0;
    const int wide = (uintptr_t)y % 16 == 0 && ((long long)cols * size) % 16 == 0;
    const dim3 grid(blocks_for(rows * blocks * 4)), threads(THREADS);
    if (dtype == TS_F32)
        TS_CHAINED_CHECK("dequantize_mxfp4", launch_chained(dequantize_mxfp4_kernel<float>, grid, threads, 0, stream, (const uint32_t*)codes,
                                                            (const uint8_t*)scales, (float*)y, rows, cols, blocks * 4, ld_codes / 4, ld_scales, wide));
    else
        TS_CHAINED_CHECK("dequantize_mxfp4", launch_chained(dequantize_mxfp4_kernel<__nv_bfloat16>, grid, threads, 0, stream, (const uint32_t*)codes,
                                                            (const uint8_t*)scales, (__nv_bfloat16*)y, rows, cols, blocks * 4, ld_codes / 4, ld_scales,
                                                            wide));
    return 0;
}
