// ifr_mxfp4.h -- launch interface of the 4-bit microscaled catalogue (ifr_mxfp4.hip) used by ifr_api.hip.
//
// A matrix [n][k] is held as blocks of 32 consecutive columns (kb = ceil(k / 32) blocks a row, zeros behind column k):
//   codes  [n][kb * 16] bytes: element 2j of a row in the low half of byte j, E2M1 (0 .5 1 1.5 2 3 4 6 and their negatives)
//   scales [n][kb] bytes:      exponent + 127 of the block's power of two, 255 = the block holds a NaN or an infinity
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ifr {

struct MxMatrix {
    const uint8_t *codes, *scales;
    int64_t n;
};

struct MxScoreParams {
    MxMatrix x, v;               // queries and catalogue
    int k;
    const float *ubase, *ibase;  // null = none
    void *out;                   // [x.n][ld] fp32 or bf16
    int64_t ld;
    int out_bf16;
};

int launch_mx_quantize(const void *X, int bf16, int64_t n, int64_t k, int64_t ld, uint8_t *codes, uint8_t *scales, hipStream_t s);
int launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, float *out, int64_t ld, hipStream_t s);
int launch_mx_scores(const MxScoreParams &p, hipStream_t s);

}  // namespace ifr
