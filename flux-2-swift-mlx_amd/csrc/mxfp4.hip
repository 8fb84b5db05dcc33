// mxfp4.hip — microscaled 4-bit floating point (MXFP4): quantisation and reading back (gfx950).
//
// A row is cut into blocks of 32 values with one power of two per block.  a = max |x| of the block, E = its biased float exponent
// (floor(log2 a) + 127 for normal a): scale byte = max(E - 2, 0), value of the scale = 2^(byte - 127), so that a / scale lies in [4, 8) and
// the block's largest values reach the top binade of e2m1 (4, 6).  code = x / scale rounded to the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6},
// ties to the even code, |x| / scale > 6 to +-6.  A block that holds a NaN or an infinity gets byte 255 (= NaN for its consumers) and zero codes.
// All of it is exact: the division is by a power of two and v_cvt_scalef32_pk_fp4_f32 rounds once (subnormal inputs and scales included).
//
// Both kernels are bound by HBM; one pass, 8 values per lane (a quad of lanes = one block, its maximum by two DPP steps, no LDS).
#include "dev.h"
#include "mxfp4.h"

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

template <int DT>
__device__ __forceinline__ float load_one(const void* p, int64_t i) {
    if constexpr (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == DT_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    else return (float)reinterpret_cast<const _Float16*>(p)[i];
}

// 8 consecutive values; VEC: the row's start is 16-byte aligned and the 8 lie inside the row
template <int DT>
__device__ __forceinline__ void load_eight(const void* p, int64_t i, float* v) {
    if constexpr (DT == DT_F32) {
        const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        const float4 a = q[0], b = q[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const u32x4 u = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == DT_BF16) { v[2 * j] = lo_bf16(u[j]); v[2 * j + 1] = hi_bf16(u[j]); }
            else {
                typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
                const uint32_t w = u[j];   // a value of its own: __builtin_bit_cast of a vector's element reads element 0
                const half2_t h = __builtin_bit_cast(half2_t, w);
                v[2 * j] = (float)h.x; v[2 * j + 1] = (float)h.y;
            }
        }
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
    return v > o ? v : o;
}

// `lanes` = 1 << lanes_log2 lanes walk one row, 256 / lanes rows per workgroup at a time
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int cols, int chunks,
                                                             uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int lanes_log2) {
    const int lanes = 1 << lanes_log2, per_wg = 256 >> lanes_log2;
    for (int64_t row = (int64_t)blockIdx.x * per_wg + (threadIdx.x >> lanes_log2); row < rows; row += (int64_t)gridDim.x * per_wg) {
        const int64_t base = row * ldx;
        uint32_t* crow = reinterpret_cast<uint32_t*>(codes) + row * chunks;
        uint8_t* srow = scales + row * (chunks >> 2);
        for (int c = threadIdx.x & (lanes - 1); c < chunks; c += lanes) {   // chunks % 16 == 0: a quad is never split
            float v[8];
            if (VEC && c * 8 + 8 <= cols) load_eight<DT>(x, base + c * 8, v);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = c * 8 + j < cols ? load_one<DT>(x, base + c * 8 + j) : 0.f;
            }
            uint32_t top = 0;   // |x| as bits: ordered like the values, infinities and NaN above all finite ones
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
            top = quad_max<0xB1>(top);   // lane ^ 1
            top = quad_max<0x4E>(top);   // lane ^ 2
            const bool finite = top < 0x7f800000u;
            const int e = (int)(top >> 23) - 2;
            const uint32_t byte = finite ? (uint32_t)(e > 0 ? e : 0) : 255u;
            const float s = __builtin_bit_cast(float, byte << 23);   // the conversion reads the exponent field alone: 0 is 2^-127
            uint32_t q = 0;
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
            crow[c] = finite ? q : 0u;
            if ((c & 3) == 0) srow[c >> 2] = (uint8_t)byte;
        }
    }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                                               int cols, int chunks, void* __restrict__ y, int64_t ldy, int lanes_log2) {
    const int lanes = 1 << lanes_log2, per_wg = 256 >> lanes_log2;
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    for (int64_t row = (int64_t)blockIdx.x * per_wg + (threadIdx.x >> lanes_log2); row < rows; row += (int64_t)gridDim.x * per_wg) {
        const uint32_t* crow = reinterpret_cast<const uint32_t*>(codes) + row * chunks;
        const uint8_t* srow = scales + row * (chunks >> 2);
        for (int c = threadIdx.x & (lanes - 1); c * 8 < cols; c += lanes) {
            const uint32_t q = crow[c];
            const float s = __builtin_bit_cast(float, (uint32_t)srow[c >> 2] << 23);
            float v[8];
            f32x2 p;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0); v[0] = p.x; v[1] = p.y;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1); v[2] = p.x; v[3] = p.y;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2); v[4] = p.x; v[5] = p.y;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3); v[6] = p.x; v[7] = p.y;
            const int64_t at = row * ldy + c * 8;
            const bool whole = VEC && c * 8 + 8 <= cols;
            if constexpr (DT == DT_F32) {
                float* o = reinterpret_cast<float*>(y) + at;
                if (whole) {
                    reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (c * 8 + j < cols) o[j] = v[j];
                }
            } else {
                u32x4 u;   // bf16 holds every value exactly; f16 rounds once (to infinity above 65504, to its subnormals below)
                typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    u[j] = DT == DT_BF16 ? pack_bf16x2(v[2 * j], v[2 * j + 1])
                                         : __builtin_bit_cast(uint32_t, half2_t{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
                uint16_t* o = reinterpret_cast<uint16_t*>(y) + at;
                if (whole) *reinterpret_cast<u32x4*>(o) = u;
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (c * 8 + j < cols) o[j] = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
    }
}

// lanes per row: the power of two that covers the row's 8-value chunks, at most a workgroup
int row_lanes_log2(int chunks) {
    int l = 4;
    while ((1 << l) < chunks && l < 8) ++l;
    return l;
}
unsigned row_grid(int64_t rows, int lanes_log2) {
    const int64_t per_wg = 256 >> lanes_log2, n = (rows + per_wg - 1) / per_wg;
    return (unsigned)(n < (1 << 20) ? n : (1 << 20));   // beyond, a workgroup walks several row groups
}
bool aligned16(const void* p, int64_t ld, int esz) { return (reinterpret_cast<uintptr_t>(p) % 16 == 0) && (ld * esz % 16 == 0); }

}  // namespace

int launch_quantize_mxfp4(hipStream_t stream, const void* x, int dtype, int64_t ldx, int64_t rows, int cols, uint8_t* codes, uint8_t* scales) {
    const int chunks = mxfp4_padded(cols) / 8, l = row_lanes_log2(chunks);
    const dim3 g(row_grid(rows, l)), b(256);
    const bool vec = aligned16(x, ldx, dtype == DT_F32 ? 4 : 2);
#define QUANT(DT) \
    if (vec) quantize_mxfp4_kernel<DT, true><<<g, b, 0, stream>>>(x, ldx, rows, cols, chunks, codes, scales, l); \
    else quantize_mxfp4_kernel<DT, false><<<g, b, 0, stream>>>(x, ldx, rows, cols, chunks, codes, scales, l)
    if (dtype == DT_F32) { QUANT(DT_F32); }
    else if (dtype == DT_BF16) { QUANT(DT_BF16); }
    else if (dtype == DT_F16) { QUANT(DT_F16); }
    else return 1;
#undef QUANT
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

int launch_dequantize_mxfp4(hipStream_t stream, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* y, int dtype, int64_t ldy) {
    const int chunks = mxfp4_padded(cols) / 8, l = row_lanes_log2(chunks);
    const dim3 g(row_grid(rows, l)), b(256);
    const bool vec = aligned16(y, ldy, dtype == DT_F32 ? 4 : 2);
#define DEQUANT(DT) \
    if (vec) dequantize_mxfp4_kernel<DT, true><<<g, b, 0, stream>>>(codes, scales, rows, cols, chunks, y, ldy, l); \
    else dequantize_mxfp4_kernel<DT, false><<<g, b, 0, stream>>>(codes, scales, rows, cols, chunks, y, ldy, l)
    if (dtype == DT_F32) { DEQUANT(DT_F32); }
    else if (dtype == DT_BF16) { DEQUANT(DT_BF16); }
    else if (dtype == DT_F16) { DEQUANT(DT_F16); }
    else return 1;
#undef DEQUANT
    return hipGetLastError() == hipSuccess ? 0 : 2;
}
