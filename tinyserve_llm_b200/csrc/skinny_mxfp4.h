// The product of a handful of rows of x with 4-bit weights (skinny_mxfp4.cu).
#pragma once

#include "common.cuh"

struct SkinnyMx {
    const uint8_t* w_codes;
    const uint8_t* w_scales;
    long long w_ld_codes, w_ld_scales;
    const void* x;                                     // bfloat16, rows ldx elements apart; or codes, ldx bytes apart
    long long ldx;
    const uint8_t* x_scales;                           // null: bfloat16
    long long x_ld_scales;
    void* y;
    long long ldy;
    int M, N, K, blocks;
    int act;
    float act_limit, act_alpha;
    int settled;
};

constexpr int SKINNY_MX_ROWS = 16;                     // the most rows of x

int skinny_mxfp4(const SkinnyMx& p, int gated, int out_f32, cudaStream_t stream);
