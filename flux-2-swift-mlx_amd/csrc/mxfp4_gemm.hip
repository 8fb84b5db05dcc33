// mxfp4_gemm.hip — products with MXFP4 weights (gfx950):  out = resid + gate * (A W^T + bias)
//   A in MXFP4 (block scales ride in v_mfma_scale_f32_16x16x128_f8f6f4's scale operands) or in bf16 (W's codes become bf16 exactly, in
//   registers: e2m1 x 2^e has 2 significant bits, then v_mfma_f32_16x16x32_bf16).
// Every product of two code values is exact, sums are f32.
//
// Operand layout (both forms): lane l of a wave holds row l % 16 of its 16-row block and the 32 values 32 (l / 16) ... of a 128-value step:
// 16 bytes of codes = one MXFP4 block, so a lane needs one 16-byte load and one scale byte per step.  W is the MFMA's first operand: the
// accumulator then holds 4 consecutive columns of one output row per lane (16-byte f32 / 8-byte bf16 stores).
#include "dev.h"
#include "mxfp4.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// one 16 x 16 x 128 product of MXFP4 operands; sw, sa: the lanes' scale bytes (low byte)
__device__ __forceinline__ f32x4 mfma_fp4(u32x4 w, u32x4 a, f32x4 c, uint32_t sw, uint32_t sa) {
    const i32x8 wv = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0}, av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, av, c, 4, 4, 0, (int)sw, 0, (int)sa);
}
// 8 codes -> 8 bf16, exactly (the scale's exponent field alone is read: byte 0 is 2^-127, 255 NaN)
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t q, float s) {
    u32x4 u;
    u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0));
    u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1));
    u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2));
    u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3));
    return __builtin_bit_cast(bf16x8, u);
}

// 4 consecutive output columns n ... n + 3 of row m.  VEC: N % 4 == 0 and every pointer / stride takes 4-value accesses
template <bool VEC>
__device__ __forceinline__ void store4(const Mxfp4Gemm& p, int m, int n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
    if constexpr (VEC) {
        if (p.bias) v += *reinterpret_cast<const f32x4*>(p.bias + n);
        if (p.gate) v *= *reinterpret_cast<const f32x4*>(p.gate + n);
        if (p.resid) v += *reinterpret_cast<const f32x4*>(p.resid + m * p.ld_resid + n);
        if (p.out_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + m * p.ld_out + n) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + m * p.ld_out + n) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n + i >= p.N) break;
            float f = v[i];
            if (p.bias) f += p.bias[n + i];
            if (p.gate) f *= p.gate[n + i];
            if (p.resid) f += p.resid[m * p.ld_resid + n + i];
            if (p.out_bf16) reinterpret_cast<uint16_t*>(p.out)[m * p.ld_out + n + i] = f32_to_bf16_bits(f);
            else reinterpret_cast<float*>(p.out)[m * p.ld_out + n + i] = f;
        }
    }
}

// 8 values of a bf16 row from column k on; columns >= K (the padding of W's last step) are zero
template <bool AVEC>
__device__ __forceinline__ bf16x8 load_a8(const uint16_t* row, int k, int K) {
    if (AVEC && k + 8 <= K) return *reinterpret_cast<const bf16x8*>(row + k);
    u32x4 u = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k + j < K) u[j >> 1] |= (uint32_t)row[k + j] << (16 * (j & 1));
    return __builtin_bit_cast(bf16x8, u);
}

// ---------------------------------------------------------------------------------------------- a tile per workgroup, K split over its waves
// 16 MT rows x 16 NT columns; the four waves take the 128-value steps in turn and their sums are added in wave order through LDS.
template <bool A4, bool AVEC, bool VEC, int MT, int NT>
__global__ __launch_bounds__(256) void mxfp4_gemm_rows_kernel(Mxfp4Gemm p, int tiles_n) {
    __shared__ f32x4 part[4][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = (int)(blockIdx.x % tiles_n) * 16 * NT, m0 = (int)(blockIdx.x / tiles_n) * 16 * MT;
    const int64_t row_bytes = (int64_t)p.steps * 64, row_scales = (int64_t)p.steps * 4;
    const uint8_t *wq[NT], *ws[NT], *aq[MT], *as[MT];
    const uint16_t* ab[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {   // rows behind the last one: its copy, never stored
        const int64_t n = n0 + 16 * j + r < p.N ? n0 + 16 * j + r : p.N - 1;
        wq[j] = p.w + n * row_bytes + g * 16;
        ws[j] = p.w_scales + n * row_scales + g;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + 16 * i + r < p.M ? m0 + 16 * i + r : p.M - 1;
        if constexpr (A4) {
            aq[i] = reinterpret_cast<const uint8_t*>(p.a) + m * row_bytes + g * 16;
            as[i] = p.a_scales + m * row_scales + g;
        } else ab[i] = reinterpret_cast<const uint16_t*>(p.a) + m * p.lda;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = wave; s < p.steps; s += 4) {
        u32x4 w[NT];
        uint32_t sw[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            w[j] = *reinterpret_cast<const u32x4*>(wq[j] + (int64_t)s * 64);
            sw[j] = ws[j][(int64_t)s * 4];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (A4) {
                const u32x4 a = *reinterpret_cast<const u32x4*>(aq[i] + (int64_t)s * 64);
                const uint32_t sa = as[i][(int64_t)s * 4];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][i] = mfma_fp4(w[j], a, acc[j][i], sw[j], sa);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bf16x8 a = load_a8<AVEC>(ab[i], s * 128 + g * 32 + q * 8, p.K);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_to_bf16(w[j][q], __builtin_bit_cast(float, sw[j] << 23)), a, acc[j][i], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) part[wave][j * MT + i][lane] = acc[j][i];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += 4) {
        const f32x4 v = part[0][t][lane] + part[1][t][lane] + part[2][t][lane] + part[3][t][lane];
        store4<VEC>(p, m0 + 16 * (t % MT) + r, n0 + 16 * (t / MT) + 4 * g, v);
    }
}

bool four_columns(const Mxfp4Gemm& p) {
    auto ok = [](const void* q, int64_t ld, int esz) { return !q || (reinterpret_cast<uintptr_t>(q) % (4 * esz) == 0 && ld % 4 == 0); };
    return p.N % 4 == 0 && ok(p.out, p.ld_out, p.out_bf16 ? 2 : 4) && ok(p.resid, p.ld_resid, 4) && ok(p.bias, 0, 4) && ok(p.gate, 0, 4);
}

template <bool A4, bool AVEC, int MT, int NT>
int launch_rows(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t tn = (p.N + 16 * NT - 1) / (16 * NT), tm = (p.M + 16 * MT - 1) / (16 * MT);
    if (tn * tm >= (1 << 24)) return 1;
    const dim3 grid((unsigned)(tn * tm)), block(256);
    if (four_columns(p)) mxfp4_gemm_rows_kernel<A4, AVEC, true, MT, NT><<<grid, block, 0, stream>>>(p, (int)tn);
    else mxfp4_gemm_rows_kernel<A4, AVEC, false, MT, NT><<<grid, block, 0, stream>>>(p, (int)tn);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // namespace

int launch_mxfp4_gemm(hipStream_t stream, const Mxfp4Gemm& p) {
    if (p.a_scales) return launch_rows<true, false, 2, 2>(stream, p);
    const bool avec = reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && p.lda % 8 == 0;
    return avec ? launch_rows<false, true, 2, 2>(stream, p) : launch_rows<false, false, 2, 2>(stream, p);
}
