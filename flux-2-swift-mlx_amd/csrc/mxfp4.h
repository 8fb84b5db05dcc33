// mxfp4.h — launchers of the MXFP4 kernels and of the residual norm.  Every launcher enqueues on `stream` and returns 0 on success
// (1 = bad argument, 2 = launch error).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// ---------------------------------------------------------------- microscaled 4-bit floating point (mxfp4.hip, mxfp4_gemm.hip)
// An MXFP4 matrix [rows, cols]: codes u8 [rows][mxfp4_padded(cols) / 2], two e2m1 codes per byte (the even column in the low half), and
// scale bytes u8 [rows][mxfp4_padded(cols) / 32], one e8m0 byte (2^(byte - 127), 255 = NaN) per 32 columns; the padding is zero codes
// and zero bytes.  codes 16-byte aligned, scales 4-byte aligned.
static inline int mxfp4_padded(int cols) { return (cols + 127) / 128 * 128; }
// dtype: 0 f32, 1 bf16, 2 f16 (flux2mi_dtype); rows of ldx elements
int launch_quantize_mxfp4(hipStream_t stream, const void* x, int dtype, int64_t ldx, int64_t rows, int cols, uint8_t* codes, uint8_t* scales);
int launch_dequantize_mxfp4(hipStream_t stream, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* y, int dtype, int64_t ldy);
// out [M, N] = resid + gate * (A W^T + bias)
struct Mxfp4Gemm {
    const void* a;             // MXFP4 codes [M, K] with a_scales, or bf16 [M, K] of row stride lda with a_scales == nullptr
    const uint8_t* a_scales;
    int64_t lda;
    const uint8_t* w;          // MXFP4 [N, K]
    const uint8_t* w_scales;
    const float* bias;         // f32 [N] or nullptr
    const float* gate;         // f32 [N] or nullptr (1)
    const float* resid;        // f32 [M, N] of row stride ld_resid, or nullptr (0); may be `out`
    int64_t ld_resid;
    void* out;                 // f32 or bf16, row stride ld_out
    int64_t ld_out;
    int out_bf16;
    int M, N, K;
    int steps;                 // mxfp4_padded(K) / 128
};
int launch_mxfp4_gemm(hipStream_t stream, const Mxfp4Gemm& p);

// ---------------------------------------------------------------- norms behind and in front of a block (residual_norm.hip)
enum { RESIDUAL_NORM_NONE = 0, RESIDUAL_NORM_RMS = 1, RESIDUAL_NORM_LAYER = 2 };
constexpr int RESIDUAL_NORM_MAX_DIM = 16384;   // a row lives in a workgroup's registers
struct ResidualNorm {
    const float* x;            // f32 [rows, dim], row stride ldx
    int64_t ldx;
    const void* y;             // bf16 / f32 [rows, dim], row stride ldy, or nullptr
    int64_t ldy;
    int y_bf16;
    float* x_out;              // f32 [rows, dim], row stride ldx_out, or nullptr; may be x
    int64_t ldx_out;
    void* out;                 // bf16 / f32 [rows, dim], row stride ldo, or nullptr
    int64_t ldo;
    int out_bf16;
    int rows, dim, split;      // rows < split take vectors 0 of gate / scale / shift
    int post, pre;             // norm of y, norm of x'
    float post_eps, eps, resid_scale;
    const uint16_t* post_w;    // bf16 [dim] or nullptr (1)
    const uint16_t* w;
    const float* gate[2];      // f32 [dim] or nullptr (1)
    const float* scale[2];     // f32 [dim] or nullptr (0)
    const float* shift[2];
};
int launch_residual_norm(hipStream_t stream, const ResidualNorm& p);
