// The launcher of the products over microscaled 4-bit weights (gemm_mxfp4.cuh): checks of the arguments.
#include "gemm_mxfp4.cuh"
#include "skinny_mxfp4.h"

// Whether a few rows go by the kernel that spreads codes in registers: no kernel has less between its launch and its end, but it takes a
// cycle for every 13 numbers of W and SM.  Device times on a B200 (graphs of different weights): 2,048 by 2,048, 1 to 16 rows in bfloat16 2.9
// to 4.2 us (in pieces 7.4 to 8.1), in four bits 3.1 to 3.7 (tcgen05 4.4 to 5.1); 2,048 by 8,192, 1 to 8 rows in bfloat16 8.1 to 9.0 (9.9 to
// 10.3), 16 rows 11.7 (11.0); 4,096 by 4,096 7.9 to 8.8 (8.4 to 8.9), 16 rows 11.2 (9.3); 6,144 by 4,096 10.6 to 11.7 (10.3 to 10.7); 16,384 by
// 2,048 11.1 to 13.2 (10.6 to 10.8).
static bool few_in_registers(int M, int N, int K, bool both) {
    const long long numbers = (long long)N * K;
    return (M <= SKINNY_MX_ROWS && numbers <= 5ll << 20) || (!both && M <= 8 && numbers <= 1ll << 24);
}

// Whether rows in bfloat16 are multiplied as three rows of 8-bit numbers each, with W's codes as they are, and not with W's codes spread to
// bfloat16.  Device times on a B200, other weights each time, in pieces (spread): up to 16 rows always, 28,672 by 4,096 gated, 8 and 16 rows
// 18.8 and 20.1 us (40.7, 38.5), 4,096 by 14,336 14.7 and 17.2 (23.3), 4,096 by 4,096, 16 rows 9.3 (9.5).  Up to 32 rows where there is enough
// of W or K is long: 28,672 by 4,096 22.7 (39.1), 2,048 by 8,192 12.6 (13.3), but 4,096 by 4,096 10.6 (9.6).  Up to 64 where K is long, N splits in
// enough tiles that clusters of eight CTAs are not needed, which one CTA an SM leaves no room for, and there is enough of W: 28,672 by 4,096
// 34.7 (40.2), 4,096 by 14,336 21.3 (24.9), 6,144 by 4,096 14.1 (15.7), but 16,384 by 2,048 16.6 (14.9), 2,048 by 8,192 20.2 (14.4), 4,096 by
// 4,096 13.4 (10.7).  Beyond, three bytes of x a number are more to bring than spreading costs: 512 rows, 2,048 by 8,192 31.6 (28.3), 4,096 by
// 4,096 33.1 (26.2).
static bool in_pieces(int M, int N, int K) {
    const long long numbers = (long long)N * K;
    if (K % 128 || numbers <= 5ll << 20) return false;
    if (M <= 16) return true;
    if (M <= 32) return K > 4096 || numbers > 1ll << 24;
    return M <= 64 && K >= 4096 && N > 2304 && numbers > 5ll << 22;
}

// Bytes of scratch a product needs (16-byte aligned), 0 if its rows do not go in pieces.  `spaced`: W's rows of codes start 32-byte aligned, as
// TMA asks of 4-bit numbers that it spaces out.
TS_API long long ts_gemm_mxfp4_scratch_bytes(int M, int N, int K, int both, int spaced) {
    if (both || !spaced || M <= 0 || N <= 0 || K <= 0 || few_in_registers(M, N, K, false) || !in_pieces(M, N, K)) return 0;
    return mxfp4_pieces_bytes(M, (K + MX_BLOCK - 1) / MX_BLOCK);
}

// y = x . W^T (gated 0; y [M, N], bfloat16 or float32) or y = act(x Wgate^T, x Wup^T) with W = [gate rows | up rows] (gated 1; y [M, N / 2],
// bfloat16; TS_ACT_* of common.cuh).  x: bfloat16 [M, K], rows ldx elements apart, if x_scales is null; else codes, rows ldx bytes apart,
// and scales.  settled: nothing that may still run ahead on the stream writes W.  K a multiple of 8 (rows in bfloat16); rows of codes and of
// scales start 16-byte aligned, and so do x and its rows.
TS_API int ts_gemm_mxfp4(const void* w_codes, const void* w_scales, long long w_ld_codes, long long w_ld_scales, const void* x, long long ldx,
                         const void* x_scales, long long x_ld_scales, void* y, int M, int N, int K, long long ldy, int gated, int act,
                         float limit, float alpha, int settled, void* scratch, int out_dtype, int* error, cudaStream_t stream) {
    TS_REQUIRE(M >= 0 && M <= MX_MOST && N > 0 && N <= MX_MOST && K > 0 && K <= MX_MOST, "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
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
               M, N, K, blocks, N / 2, out_dtype == TS_F32 ? 1 : 0, act, limit, alpha, 0, nullptr, 0, settled, 1, error};
    const int spaced = (uintptr_t)w_codes % 32 == 0 && w_ld_codes % 32 == 0;
    const long long pieces = ts_gemm_mxfp4_scratch_bytes(M, N, K, x_scales != nullptr, spaced);
    if (pieces) {
        TS_REQUIRE(scratch && (uintptr_t)scratch % 16 == 0, "gemm_mxfp4: %lld bytes of scratch are needed", pieces);
        return mxfp4_pieces(x, ldx, scratch, p, gated, stream);
    }
    if (few_in_registers(M, N, K, x_scales != nullptr)) {
        const SkinnyMx few{(const uint8_t*)w_codes, (const uint8_t*)w_scales, w_ld_codes, w_ld_scales, x, ldx, (const uint8_t*)x_scales, x_ld_scales, y,
                           ldy, M, N, K, blocks, act, limit, alpha, settled};
        return skinny_mxfp4(few, gated, out_dtype == TS_F32, stream);
    }
    return x_scales ? mxfp4_rows4(x, ldx, p, gated, stream) : mxfp4_rows16(x, ldx, p, gated, stream);
}
