// residual_norm.hip — the norms behind and in front of a block, fused with the block's gate and the residual's scale (gfx950).
//
//   u    = norm_post(y) * w_post          y: what the block returns; norm_post: none, RMS or LayerNorm
//   x'   = resid_scale * x + gate * u     the residual stream, f32
//   out  = norm(x') * w * (1 + scale) + shift    the next block's operand
// gate, scale and shift are per column, one set for rows < split (text) and one for the others (image), as in layernorm_modulate.
//
// Measured: 4608 x 4096 (y, out bf16) 52 us = 4.4 TB/s, 1031 x 5119 f32 23 us = 3.6 TB/s, with y and out in bf16 27 us = 2.3 TB/s (odd rows go value by
// value), 4608 x 12000 191 us, one row of 2560 4.2 us (a launch and two sums).
// Bound by HBM: x and y are read once, x' and out written once; a row lives in the registers of the threads that own it, its statistics
// are f32 sums over those registers (the variance around the mean of the row, in a second sum over registers, not E[x^2] - mean^2).  What hides
// the sums' and the vectors' latency is other rows' workgroups, so few registers count for more than early loads or vectors kept over several rows (both
// measured: 5 to 40 % slower).
// Rows may start at any element; f32 is moved 16 bytes at any dword, bf16 8 bytes at any dword and value by value where a row starts in the middle of one.
#include "dev.h"
#include "mxfp4.h"

namespace {

// sum over the TPR threads of a row; red: one float per wave of the workgroup
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        __syncthreads();   // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}

typedef f32x4 __attribute__((aligned(4))) f32x4_dword;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 __attribute__((aligned(4))) u32x2_dword;

// value number k of thread t: column
template <int TPR>
__device__ __forceinline__ int col_of(int k, int t) { return ((k >> 2) * TPR + t) * 4 + (k & 3); }

// 4 NV values of a row of f32 / bf16 into registers (columns >= dim: 0)
template <int TPR, int NV>
__device__ __forceinline__ void load_row(const void* p, bool bf16, int dim, int t, float* v) {
    const bool odd = reinterpret_cast<uintptr_t>(p) & 2;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * 4;
        f32x4 f = {0.f, 0.f, 0.f, 0.f};
        if (bf16) {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + c;
            if (c + 4 <= dim && !odd) {
                const u32x2 u = *reinterpret_cast<const u32x2_dword*>(q);
                f = f32x4{lo_bf16(u[0]), hi_bf16(u[0]), lo_bf16(u[1]), hi_bf16(u[1])};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (c + j < dim) f[j] = bf16_bits_to_f32(q[j]);
            }
        } else {
            const float* q = reinterpret_cast<const float*>(p) + c;
            if (c + 4 <= dim) f = *reinterpret_cast<const f32x4_dword*>(q);
            else {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c + j < dim) f[j] = q[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = f[j];
    }
}
template <int TPR, int NV>
__device__ __forceinline__ void store_row(void* p, bool bf16, int dim, int t, const float* v) {
    const bool odd = reinterpret_cast<uintptr_t>(p) & 2;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * 4;
        if (bf16) {
            uint16_t* q = reinterpret_cast<uint16_t*>(p) + c;
            if (c + 4 <= dim && !odd) *reinterpret_cast<u32x2_dword*>(q) = u32x2{pack_bf16x2(v[4 * i], v[4 * i + 1]), pack_bf16x2(v[4 * i + 2], v[4 * i + 3])};
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (c + j < dim) q[j] = f32_to_bf16_bits(v[4 * i + j]);
            }
        } else {
            float* q = reinterpret_cast<float*>(p) + c;
            if (c + 4 <= dim) *reinterpret_cast<f32x4_dword*>(q) = f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            else {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c + j < dim) q[j] = v[4 * i + j];
            }
        }
    }
}

// v <- (v - mean) / sqrt(mean square + eps); mean 0 for the RMS form
template <int TPR, int NV>
__device__ __forceinline__ void normalize(float* v, int kind, float eps, int dim, int t, float* red) {
    if (kind == RESIDUAL_NORM_NONE) return;
    if (kind == RESIDUAL_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) s += v[k];
        const float mean = row_sum<TPR>(s, red) / (float)dim;
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k)
            if (col_of<TPR>(k, t) < dim) v[k] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) q += v[k] * v[k];
    const float r = rsqrtf(row_sum<TPR>(q, red) / (float)dim + eps);
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) v[k] *= r;
}

// TPR threads per row, a row (TPR = 64: four) per workgroup; a thread owns 4 NV values of its row
template <int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_kernel(ResidualNorm p) {
    __shared__ float red[TPR / 64];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, row = TPR == 64 ? group * 4 + threadIdx.x / 64 : group;
    if (row >= p.rows) return;   // whole rows: TPR 64 has no barrier, the others' workgroups return as one
    const int dim = p.dim, set = row < p.split ? 0 : 1;
    float x[4 * NV], v[4 * NV];
    load_row<TPR, NV>(p.x + row * p.ldx, false, dim, t, x);
    if (p.y) {
        load_row<TPR, NV>(p.y_bf16 ? (const void*)(reinterpret_cast<const uint16_t*>(p.y) + row * p.ldy)
                                        : (const void*)(reinterpret_cast<const float*>(p.y) + row * p.ldy), p.y_bf16, dim, t, v);
        normalize<TPR, NV>(v, p.post, p.post_eps, dim, t, red);
        if (p.post_w) {
            float w[4 * NV];
            load_row<TPR, NV>(p.post_w, true, dim, t, w);
#pragma unroll
            for (int k = 0; k < 4 * NV; ++k) v[k] *= w[k];
        }
        if (p.gate[set]) {
            float g[4 * NV];
            load_row<TPR, NV>(p.gate[set], false, dim, t, g);
#pragma unroll
            for (int k = 0; k < 4 * NV; ++k) v[k] *= g[k];
        }
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] = p.resid_scale * x[k] + v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= p.resid_scale;
    }
    if (p.x_out) store_row<TPR, NV>(p.x_out + row * p.ldx_out, false, dim, t, x);
    if (!p.out) return;
    normalize<TPR, NV>(x, p.pre, p.eps, dim, t, red);
    if (p.w) {
        load_row<TPR, NV>(p.w, true, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= v[k];
    }
    if (p.scale[set]) {
        load_row<TPR, NV>(p.scale[set], false, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= 1.f + v[k];
    }
    if (p.shift[set]) {
        load_row<TPR, NV>(p.shift[set], false, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] += v[k];
    }
    store_row<TPR, NV>(p.out_bf16 ? (void*)(reinterpret_cast<uint16_t*>(p.out) + row * p.ldo) : (void*)(reinterpret_cast<float*>(p.out) + row * p.ldo),
                            p.out_bf16, dim, t, x);
}

template <int TPR, int NV>
int launch_form(hipStream_t stream, const ResidualNorm& p) {
    constexpr int RPW = TPR == 64 ? 4 : 1;
    const unsigned groups = (unsigned)((p.rows + RPW - 1) / RPW), most = 1u << 22;   // x 512 threads: below the 2^32 of one grid dimension
    residual_norm_kernel<TPR, NV><<<dim3(groups < most ? groups : most, (groups + most - 1) / most), dim3(TPR * RPW), 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // namespace

int launch_residual_norm(hipStream_t stream, const ResidualNorm& p) {
    // 4608 x 4096: 53 us with 512 threads a row, 52 with 256, 65 with 1024; one row of 2560: 4.2, 5.3, 4.2.  4608 x 12000: 176 us with 512 threads of 32
    // values, 212 with 1024 of 16, 235 with 256 of 64.
    if (p.dim <= 256) return launch_form<64, 1>(stream, p);
    if (p.dim <= 512) return launch_form<64, 2>(stream, p);
    if (p.dim <= 1024) return launch_form<256, 1>(stream, p);
    if (p.dim <= 2048) return launch_form<256, 2>(stream, p);
    if (p.dim <= 4096) return launch_form<512, 2>(stream, p);
    if (p.dim <= 8192) return launch_form<512, 4>(stream, p);
    if (p.dim <= RESIDUAL_NORM_MAX_DIM) return launch_form<512, 8>(stream, p);
    return 1;
}
