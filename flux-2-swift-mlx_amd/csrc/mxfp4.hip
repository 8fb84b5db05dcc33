// mxfp4.hip — microscaled 4-bit floating point (MXFP4): quantisation and reading back (gfx950).
//
// A row is cut into blocks of 32 values with one power of two per block.  a = max |x| of the block, E = its biased float exponent
// (floor(log2 a) + 127 for normal a): scale byte = max(E - 2, 0), value of the scale = 2^(byte - 127), so that a / scale lies in [4, 8) and
// the block's largest values reach the top binade of e2m1 (4, 6).  code = x / scale rounded to the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6},
// ties to the even code, |x| / scale > 6 to +-6.  A block that holds a NaN or an infinity gets byte 255 (= NaN for its consumers) and zero codes.
// All of it is exact: the division is by a power of two and v_cvt_scalef32_pk_fp4_f32 rounds once (subnormal inputs and scales included).
//
// Both kernels are bound by HBM: 36864 x 4096 f32 quantised in 123 us (5.6 TB/s; 158 right behind a pass that wrote 600 MB), read back in 120 to
// 132, bf16 66 and 69 us; 20000 x 5119 bf16 (every other row starts in the middle of a dword) 50 and 79 us; 512 x 2560 bf16 3 us each, a launch's latency.  One pass, 8 values per lane (a quad of lanes = one block, its maximum by two DPP steps, no LDS).
// Rows may start at any element: whole dwords are moved all the same (a row of 2-byte values that starts in the middle of one is shifted in registers).
#include "dev.h"
#include "mxfp4.h"

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 __attribute__((aligned(4))) u32x4_dword;   // 16 bytes at any dword
typedef f32x4 __attribute__((aligned(4))) f32x4_dword;

template <int DT>
__device__ __forceinline__ float load_one(const void* p, int64_t i) {
    if constexpr (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == DT_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    else return (float)reinterpret_cast<const _Float16*>(p)[i];
}

// values i ... i + 7; VEC: at a multiple of 16 bytes
template <int DT, bool VEC>
__device__ __forceinline__ void load_eight(const void* p, int64_t i, float* v) {
    if constexpr (DT == DT_F32) {
        const f32x4_dword* q = reinterpret_cast<const f32x4_dword*>(reinterpret_cast<const float*>(p) + i);
        const f32x4 a = q[0], b = q[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
        u32x4 u;
        if constexpr (VEC) u = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + i);
        else {
            const uintptr_t at = reinterpret_cast<uintptr_t>(reinterpret_cast<const uint16_t*>(p) + i);
            u = *reinterpret_cast<const u32x4_dword*>(at & ~(uintptr_t)3);
            if (at & 2) {   // (every dword read holds one of the eight)
                const uint32_t e = *reinterpret_cast<const uint32_t*>((at & ~(uintptr_t)3) + 16);
                u = u32x4{__builtin_amdgcn_alignbit(u[1], u[0], 16), __builtin_amdgcn_alignbit(u[2], u[1], 16), __builtin_amdgcn_alignbit(u[3], u[2], 16),
                          __builtin_amdgcn_alignbit(e, u[3], 16)};
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = u[j];   // a value of its own: __builtin_bit_cast of a vector's element reads element 0
            if constexpr (DT == DT_BF16) { v[2 * j] = lo_bf16(w); v[2 * j + 1] = hi_bf16(w); }
            else {
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
            if (c * 8 + 8 <= cols) load_eight<DT, VEC>(x, base + c * 8, v);
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

// f32: 4 values per lane, so that the lanes of a store are one piece of memory (8 per lane, two stores 32 bytes apart each: 4.1 TB/s instead of 5.6)
__global__ __launch_bounds__(256) void dequantize_mxfp4_f32_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int cols,
                                                                   int chunks, float* __restrict__ y, int64_t ldy, int lanes_log2) {
    const int lanes = 1 << lanes_log2, per_wg = 256 >> lanes_log2;
    for (int64_t row = (int64_t)blockIdx.x * per_wg + (threadIdx.x >> lanes_log2); row < rows; row += (int64_t)gridDim.x * per_wg) {
        const uint16_t* crow = reinterpret_cast<const uint16_t*>(codes) + row * chunks * 2;
        const uint8_t* srow = scales + row * (chunks >> 2);
        for (int c = threadIdx.x & (lanes - 1); c * 4 < cols; c += lanes) {
            const uint32_t q = crow[c];
            const float s = __builtin_bit_cast(float, (uint32_t)srow[c >> 3] << 23);
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1);
            float* o = y + row * ldy + c * 4;
            const f32x4 v = {a.x, a.y, b.x, b.y};
            if (c * 4 + 4 <= cols) *reinterpret_cast<f32x4_dword*>(o) = v;
            else {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c * 4 + j < cols) o[j] = v[j];
            }
        }
    }
}

// 2-byte types: 8 values per lane.  A row that starts in the middle of a dword is written from its second value on, 8 columns a lane (codes and,
// for the eighth value, the scale of the next 8), so that whole dwords are stored; its first value goes alone.
template <int DT>
__device__ __forceinline__ uint32_t pack_two(float a, float b) {   // bf16 holds every value exactly; f16 rounds once (to infinity above 65504)
    if constexpr (DT == DT_BF16) return pack_bf16x2(a, b);
    else return __builtin_bit_cast(uint32_t, half2_t{(_Float16)a, (_Float16)b});
}
template <int DT>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                                               int cols, int chunks, uint16_t* __restrict__ y, int64_t ldy, int lanes_log2) {
    const int lanes = 1 << lanes_log2, per_wg = 256 >> lanes_log2;
    for (int64_t row = (int64_t)blockIdx.x * per_wg + (threadIdx.x >> lanes_log2); row < rows; row += (int64_t)gridDim.x * per_wg) {
        const uint32_t* crow = reinterpret_cast<const uint32_t*>(codes) + row * chunks;
        const uint8_t* srow = scales + row * (chunks >> 2);
        uint16_t* yrow = y + row * ldy;
        const int odd = (int)(reinterpret_cast<uintptr_t>(yrow) >> 1 & 1);
        for (int c = threadIdx.x & (lanes - 1); c * 8 + odd < cols || c == 0; c += lanes) {
            uint32_t q = crow[c];
            const float s = __builtin_bit_cast(float, (uint32_t)srow[c >> 2] << 23);
            float s7 = s;
            if (odd) {
                if (c == 0) yrow[0] = (uint16_t)pack_two<DT>(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0)[0], 0.f);
                const int next = c + 1 < chunks ? c + 1 : c;   // (its values lie behind the row then)
                q = q >> 4 | crow[next] << 28;
                s7 = __builtin_bit_cast(float, (uint32_t)srow[next >> 2] << 23);
            }
            u32x4 u;
            f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0);
            u[0] = pack_two<DT>(v.x, v.y);
            v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1);
            u[1] = pack_two<DT>(v.x, v.y);
            v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2);
            u[2] = pack_two<DT>(v.x, v.y);
            v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3);
            if (odd) v.y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s7, 3)[1];
            u[3] = pack_two<DT>(v.x, v.y);
            const int first = c * 8 + odd;
            uint16_t* o = yrow + first;
            if (first + 8 <= cols) *reinterpret_cast<u32x4_dword*>(o) = u;
            else {
#pragma unroll
                for (int j = 0; j < 7; ++j) if (first + j < cols) o[j] = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
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
}  // namespace

int launch_quantize_mxfp4(hipStream_t stream, const void* x, int dtype, int64_t ldx, int64_t rows, int cols, uint8_t* codes, uint8_t* scales) {
    const int chunks = mxfp4_padded(cols) / 8, l = row_lanes_log2(chunks);
    const dim3 g(row_grid(rows, l)), b(256);
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
#define QUANT(DT) \
    if (vec) quantize_mxfp4_kernel<DT, true><<<g, b, 0, stream>>>(x, ldx, rows, cols, chunks, codes, scales, l); \
    else quantize_mxfp4_kernel<DT, false><<<g, b, 0, stream>>>(x, ldx, rows, cols, chunks, codes, scales, l)
    if (dtype == DT_F32) quantize_mxfp4_kernel<DT_F32, true><<<g, b, 0, stream>>>(x, ldx, rows, cols, chunks, codes, scales, l);   // (any dword will do)
    else if (dtype == DT_BF16) { QUANT(DT_BF16); }
    else if (dtype == DT_F16) { QUANT(DT_F16); }
    else return 1;
#undef QUANT
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

int launch_dequantize_mxfp4(hipStream_t stream, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* y, int dtype, int64_t ldy) {
    const int chunks = mxfp4_padded(cols) / 8, l = row_lanes_log2(dtype == DT_F32 ? 2 * chunks : chunks);
    const dim3 g(row_grid(rows, l)), b(256);
    if (dtype == DT_F32) dequantize_mxfp4_f32_kernel<<<g, b, 0, stream>>>(codes, scales, rows, cols, chunks, reinterpret_cast<float*>(y), ldy, l);
    else if (dtype == DT_BF16) dequantize_mxfp4_kernel<DT_BF16><<<g, b, 0, stream>>>(codes, scales, rows, cols, chunks, reinterpret_cast<uint16_t*>(y), ldy, l);
    else if (dtype == DT_F16) dequantize_mxfp4_kernel<DT_F16><<<g, b, 0, stream>>>(codes, scales, rows, cols, chunks, reinterpret_cast<uint16_t*>(y), ldy, l);
    else return 1;
    return hipGetLastError() == hipSuccess ? 0 : 2;
}
