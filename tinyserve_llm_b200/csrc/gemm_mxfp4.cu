// The launcher of the products over microscaled 4-bit weights (gemm_mxfp4.cuh): checks of the arguments.
#include "gemm_mxfp4.cuh"
#include "skinny_mxfp4.h"
#include <cstdlib>

// Whether a few rows go by the kernel that spreads codes in registers.
static bool few_in_registers(int M, int N, int K, bool both) {
    if (getenv("MX_FEW")) return M <= atoi(getenv("MX_FEW"));
    return M <= SKINNY_MX_ROWS;
}

// Bytes of scratch a product needs (16-byte aligned; 0: none): rows in bfloat16 that are worked on in pieces.
TS_API long long ts_gemm_mxfp4_scratch_bytes(int M, int N, int K, int both) {
    if (both || M <= 0 || N <= 0 || K <= 0) return 0;
    if (few_in_registers(M, N, K, both)) return 0;
    if (K % 128) return 0;
    if (M > (getenv("MX_PIECES") ? atoi(getenv("MX_PIECES")) : 32)) return 0;
    return mxfp4_pieces_bytes(M, (K + MX_BLOCK - 1) / MX_BLOCK);
}

// y = x . W^T (gated 0; y [M, N], bfloat16 or float32) or y = act(x Wgate^T, x Wup^T) with W = [gate rows | up rows] (gated 1; y [M, N / 2],
// bfloat16; TS_ACT_* of common.cuh).  x: bfloat16 [M, K], rows ldx elements apart, if x_scales is null; else codes, rows ldx bytes apart,
// and scales.  settled: nothing that may still run ahead on the stream writes W.  K a multiple of 8 (rows in bfloat16); rows of codes and of scales start 16-byte aligned, and so do x and its rows.
TS_API int ts_gemm_mxfp4(const void* w_codes, const void* w_scales, long long w_ld_codes, long long w_ld_scales, const void* x, long long ldx,
                         const void* x_scales, long long x_ld_scales, void* y, int M, int N, int K, long long ldy, int gated, int act,
                         float limit, float alpha, int settled, void* scratch, int out_dtype, int* error, cudaStream_t stream) {
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
               M, N, K, blocks, N / 2, out_dtype == TS_F32 ? 1 : 0, act, limit, alpha, 0, nullptr, 0, settled, 1, error};
    const long long pieces = ts_gemm_mxfp4_scratch_bytes(M, N, K, x_scales != nullptr);
    if (pieces && mxfp4_takes_pieces(w_codes, w_ld_codes, K)) {
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
