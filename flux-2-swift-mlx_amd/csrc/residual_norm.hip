// residual_norm.hip — the norms behind and in front of a block, fused with the block's gate and the residual's scale (gfx950).
//
//   u    = norm_post(y) * w_post          y: what the block returns; norm_post: none, RMS or LayerNorm
//   x'   = resid_scale * x + gate * u     the residual stream, f32
//   out  = norm(x') * w * (1 + scale) + shift    the next block's operand
// gate, scale and shift are per column, one set for rows < split (text) and one for the others (image), as in layernorm_modulate.
//
// Bound by HBM: x and y are read once, x' and out written once; a row lives in the registers of the threads that own it, its statistics
// are f32 sums over those registers (the variance around the mean of the row, in a second sum over registers, not E[x^2] - mean^2).
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

__device__ __forceinline__ float4 bf16x4(uint2 u) { return make_float4(lo_bf16(u.x), hi_bf16(u.x), lo_bf16(u.y), hi_bf16(u.y)); }

// value number k of this thread: column
template <int TPR, bool VEC>
__device__ __forceinline__ int col_of(int k, int t) {
    return VEC ? ((k >> 2) * TPR + t) * 4 + (k & 3) : k * TPR + t;
}

// n values of a row of f32 / bf16 into registers (columns >= dim: 0)
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void load_row(const void* p, bool bf16, int dim, int t, float* v) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            const int c = i * TPR + t;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c * 4 < dim) f = bf16 ? bf16x4(reinterpret_cast<const uint2*>(p)[c]) : reinterpret_cast<const float4*>(p)[c];
            v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (4 * i + j) * TPR + t;
                v[4 * i + j] = c >= dim ? 0.f : bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[c]) : reinterpret_cast<const float*>(p)[c];
            }
        }
    }
}
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void store_row(void* p, bool bf16, int dim, int t, const float* v) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            const int c = i * TPR + t;
            if (c * 4 < dim) {
                if (bf16) reinterpret_cast<uint2*>(p)[c] = make_uint2(pack_bf16x2(v[4 * i], v[4 * i + 1]), pack_bf16x2(v[4 * i + 2], v[4 * i + 3]));
                else reinterpret_cast<float4*>(p)[c] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (4 * i + j) * TPR + t;
                if (c < dim) {
                    if (bf16) reinterpret_cast<uint16_t*>(p)[c] = f32_to_bf16_bits(v[4 * i + j]);
                    else reinterpret_cast<float*>(p)[c] = v[4 * i + j];
                }
            }
        }
    }
}

// v <- (v - mean) / sqrt(mean square + eps); mean 0 for the RMS form
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void normalize(float* v, int kind, float eps, int dim, int t, float* red) {
    if (kind == RESIDUAL_NORM_NONE) return;
    if (kind == RESIDUAL_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) s += v[k];
        const float mean = row_sum<TPR>(s, red) / (float)dim;
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k)
            if (col_of<TPR, VEC>(k, t) < dim) v[k] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) q += v[k] * v[k];
    const float r = rsqrtf(row_sum<TPR>(q, red) / (float)dim + eps);
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) v[k] *= r;
}

// TPR threads per row, 256 / TPR rows per workgroup; a thread owns 4 NV values of its row
template <int TPR, int NV, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_kernel(ResidualNorm p) {
    __shared__ float red[4];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (TPR <= 64 && row >= p.rows) return;   // whole waves; with TPR = 256 the grid is the rows
    const int dim = p.dim, set = row < p.split ? 0 : 1;
    float x[4 * NV], v[4 * NV];
    load_row<TPR, NV, VEC>(p.x + row * p.ldx, false, dim, t, x);
    if (p.y) {
        load_row<TPR, NV, VEC>(p.y_bf16 ? (const void*)(reinterpret_cast<const uint16_t*>(p.y) + row * p.ldy)
                                        : (const void*)(reinterpret_cast<const float*>(p.y) + row * p.ldy), p.y_bf16, dim, t, v);
        normalize<TPR, NV, VEC>(v, p.post, p.post_eps, dim, t, red);
        if (p.post_w) {
            float w[4 * NV];
            load_row<TPR, NV, VEC>(p.post_w, true, dim, t, w);
#pragma unroll
            for (int k = 0; k < 4 * NV; ++k) v[k] *= w[k];
        }
        if (p.gate[set]) {
            float g[4 * NV];
            load_row<TPR, NV, VEC>(p.gate[set], false, dim, t, g);
#pragma unroll
            for (int k = 0; k < 4 * NV; ++k) v[k] *= g[k];
        }
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] = p.resid_scale * x[k] + v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= p.resid_scale;
    }
    if (p.x_out) store_row<TPR, NV, VEC>(p.x_out + row * p.ldx_out, false, dim, t, x);
    if (!p.out) return;
    normalize<TPR, NV, VEC>(x, p.pre, p.eps, dim, t, red);
    if (p.w) {
        load_row<TPR, NV, VEC>(p.w, true, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= v[k];
    }
    if (p.scale[set]) {
        load_row<TPR, NV, VEC>(p.scale[set], false, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] *= 1.f + v[k];
    }
    if (p.shift[set]) {
        load_row<TPR, NV, VEC>(p.shift[set], false, dim, t, v);
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) x[k] += v[k];
    }
    store_row<TPR, NV, VEC>(p.out_bf16 ? (void*)(reinterpret_cast<uint16_t*>(p.out) + row * p.ldo) : (void*)(reinterpret_cast<float*>(p.out) + row * p.ldo),
                            p.out_bf16, dim, t, x);
}

// every row pointer that the kernel forms is aligned for 4-value accesses
bool rows_of_four(const ResidualNorm& p) {
    auto ok = [](const void* q, int64_t ld, int esz) { return !q || (reinterpret_cast<uintptr_t>(q) % (4 * esz) == 0 && ld % 4 == 0); };
    bool r = p.dim % 4 == 0 && ok(p.x, p.ldx, 4) && ok(p.y, p.ldy, p.y_bf16 ? 2 : 4) && ok(p.x_out, p.ldx_out, 4) && ok(p.out, p.ldo, p.out_bf16 ? 2 : 4) &&
             ok(p.post_w, 0, 2) && ok(p.w, 0, 2);
    for (int i = 0; i < 2; ++i) r = r && ok(p.gate[i], 0, 4) && ok(p.scale[i], 0, 4) && ok(p.shift[i], 0, 4);
    return r;
}

template <int TPR, int NV>
int launch_form(hipStream_t stream, const ResidualNorm& p) {
    const dim3 g((unsigned)((p.rows + 256 / TPR - 1) / (256 / TPR))), b(256);
    if (rows_of_four(p)) residual_norm_kernel<TPR, NV, true><<<g, b, 0, stream>>>(p);
    else residual_norm_kernel<TPR, NV, false><<<g, b, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // namespace

int launch_residual_norm(hipStream_t stream, const ResidualNorm& p) {
    if (p.dim <= 256) return launch_form<64, 1>(stream, p);
    if (p.dim <= 512) return launch_form<64, 2>(stream, p);
    if (p.dim <= 1024) return launch_form<256, 1>(stream, p);
    if (p.dim <= 2048) return launch_form<256, 2>(stream, p);
    if (p.dim <= 4096) return launch_form<256, 4>(stream, p);
    if (p.dim <= 8192) return launch_form<256, 8>(stream, p);
    if (p.dim <= RESIDUAL_NORM_MAX_DIM) return launch_form<256, 16>(stream, p);
    return 1;
}
