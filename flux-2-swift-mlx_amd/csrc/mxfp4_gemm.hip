// mxfp4_gemm.hip — products with MXFP4 weights (gfx950):  out = resid + gate * (A W^T + bias)
//   A in MXFP4 (block scales ride in v_mfma_scale_f32_16x16x128_f8f6f4's scale operands) or in bf16 (W's codes become bf16 exactly, in
//   registers: e2m1 x 2^e has 2 significant bits, down to the subnormal 2^-128; scale bytes 253 and 254, which the quantiser never writes, reach
//   2^128 = infinity; then v_mfma_f32_16x16x32_bf16, which takes subnormals).
// Every product of two code values is exact, sums are f32.
//
// Operand layout (both forms): lane l of a wave holds row l % 16 of its 16-row block and the 32 values 32 (l / 16) ... of a 128-value step:
// 16 bytes of codes = one MXFP4 block, so a lane needs one 16-byte load and one scale byte per step.  W is the MFMA's first operand: the
// accumulator then holds 4 consecutive columns of one output row per lane (16-byte f32 / 8-byte bf16 stores).
#include <algorithm>
#include <cmath>
#include <utility>

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
// 8 codes -> 8 bf16, exactly below 2^128 (the scale's exponent field alone is read: byte 0 is 2^-127, 255 NaN)
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t q, float s) {
    u32x4 u;
    u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0));
    u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1));
    u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2));
    u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3));
    return __builtin_bit_cast(bf16x8, u);
}

__device__ __forceinline__ void store1(const Mxfp4Gemm& p, int m, int n, float f) {
    if (m >= p.M || n >= p.N) return;
    if (p.bias) f += p.bias[n];
    if (p.gate) f *= p.gate[n];
    if (p.resid) f += p.resid[m * p.ld_resid + n];
    if (p.out_bf16) reinterpret_cast<uint16_t*>(p.out)[m * p.ld_out + n] = f32_to_bf16_bits(f);
    else reinterpret_cast<float*>(p.out)[m * p.ld_out + n] = f;
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
        for (int i = 0; i < 4; ++i) store1(p, m, n + i, v[i]);
    }
}

// 8 values of a bf16 row from column k on; columns >= K (the padding of W's last step) are zero.  AVEC: 16-byte aligned; otherwise the row may start
// anywhere: the 8 values' dwords, shifted by half a dword where they are odd (no dword without one of the values is read).
template <bool AVEC>
__device__ __forceinline__ bf16x8 load_a8(const uint16_t* row, int k, int K) {
    typedef u32x4 __attribute__((aligned(4))) u32x4_dword;
    u32x4 u = {0, 0, 0, 0};
    if (k + 8 <= K) {
        if constexpr (AVEC) return *reinterpret_cast<const bf16x8*>(row + k);
        const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
        const uint32_t shift = (at & 2) * 8;
        const u32x4 d = *reinterpret_cast<const u32x4_dword*>(at & ~(uintptr_t)3);
        const uint32_t e = *reinterpret_cast<const uint32_t*>((at & ~(uintptr_t)3) + (shift ? 16 : 12));
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_alignbit(j < 3 ? d[j < 3 ? j + 1 : 3] : e, d[j], shift);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < K) u[j >> 1] |= (uint32_t)row[k + j] << (16 * (j & 1));
    }
    return __builtin_bit_cast(bf16x8, u);
}

// ---------------------------------------------------------------------------------------------- few rows: K split over the waves of a workgroup
// 16 rows x 16 columns per workgroup; its waves take the 128-value steps in turn (so that together they read whole lines of W) and
// their sums are added in wave order through LDS.  Bound by latency (8 x 2560 x 2560: 3.6 us with W in the caches, 4.2 from HBM) and, with more columns, by reading W: operands go straight
// from memory to registers, U steps of a wave at a time, and the next U are requested before the current ones are used.
constexpr int ROWS_WAVES = 4;
template <bool VEC>
__global__ __launch_bounds__(64 * ROWS_WAVES) void mxfp4_gemm_rows_kernel(Mxfp4Gemm p, int tiles_n) {
    constexpr int U = 4, WAVES = ROWS_WAVES;
    __shared__ f32x4 part[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = (int)(blockIdx.x % tiles_n) * 16, m0 = (int)(blockIdx.x / tiles_n) * 16, steps = p.steps;
    const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1, m = m0 + r < p.M ? m0 + r : p.M - 1;   // rows behind the last one: its copy, never stored
    const uint8_t *wq = p.w + n * steps * 64 + g * 16, *ws = p.w_scales + n * steps * 4 + g;
    const uint8_t *aq = reinterpret_cast<const uint8_t*>(p.a) + m * steps * 64 + g * 16, *as = p.a_scales + m * steps * 4 + g;
    struct Step { u32x4 w, a; uint32_t sw, sa; };
    auto load = [&](int s, Step& x) {
        if (s >= steps) return;
        x.w = *reinterpret_cast<const u32x4*>(wq + (int64_t)s * 64);
        x.a = *reinterpret_cast<const u32x4*>(aq + (int64_t)s * 64);
        x.sw = ws[(int64_t)s * 4];
        x.sa = as[(int64_t)s * 4];
    };
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    Step cur[U], next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(wave + u * WAVES, cur[u]);
    for (int s = wave; s < steps; s += U * WAVES) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(s + (U + u) * WAVES, next[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u * WAVES < steps) acc = mfma_fp4(cur[u].w, cur[u].a, acc, cur[u].sw, cur[u].sa);
#pragma unroll
        for (int u = 0; u < U; ++u) cur[u] = next[u];
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) acc += part[w][lane];
    store4<VEC>(p, m0 + r, n0 + 4 * g, acc);
}

// ---------------------------------------------------------------------------------------------- tiles staged through LDS (MXFP4 x MXFP4)
// BM x BN outputs per workgroup of four waves (2 x 2), each BM/2 x BN/2.  A stage is 256 k = 128 bytes of every row; a group is two stages =
// four 128-k steps = 16 scale bytes of every row.  The codes come by LDS-DMA: pieces of 8 rows x 128 bytes (the 16-byte chunk c of row r lies at
// chunk c ^ (r & 7), so that the eight rows a fragment read touches at once sit in different banks).
//
// The loop body is one group in four phases, one MFMA step each.  While a phase multiplies the fragments of one register set it reads the next
// step's into the other:
//   P0: mfma F0 (step 0), read F1 <- buffer 0 in its first part, buffer 0 is free in its middle;  buffer 1 has landed at its end
//   P1: mfma F1 (step 1), read F0 <- buffer 1
//   P2: mfma F0 (step 2), read F1 <- buffer 1 in its first part, buffer 1 is free in its middle;  buffer 0 has landed at its end
//   P3: mfma F1 (step 3), read F0 <- buffer 0
// A buffer's next stage is requested from the moment it is free on, evenly, over one and a half phases; the other buffer's is then still in flight
// and stays so over the hand-over.  (Requests in P1 and P3 alone, with nothing left in flight at a hand-over: 2 x 64 KB take 5100 cycles even
// without an MFMA, against 2900 for a stream that is never drained and 4100 of the MFMAs.)
// With one wave per SIMD every instruction takes an issue slot of ~5 cycles and an MFMA 16, so the side work goes between single MFMAs ("slots"),
// about one instruction at a time (measured: what an instruction costs beyond that is 4 cycles each).
// A lane's four scale bytes of a group (one per step) are one register, the byte is chosen by the MFMA's op_sel.
// Measured: 4608 x 36864 x 4096 351 us = 4.0 PF, 4608 x 16384 x 16384 529 us = 4.7 PF.  Bound by the matrix pipe's power and by the delivery L2 -> LDS
// together: a group takes 3.5 us, without its requests 2.5, without its LDS reads 3.4, without either 2.4 (7.3 PF, the clock down to 1.8 GHz; the same
// loop on zero operands: 2.8, 1.9 without requests).  A tile's prologue and its output take 8 us.
// Steps behind K: addresses stay inside the row and both scale bytes are 0, 2^-254 times finite codes, which is below f32: exactly 0.
//
// The MFMA is asm with the accumulator pinned to AGPRs: left to itself the register allocator of a one-wave-per-SIMD kernel moves accumulators
// and fragments between the two files (492 copies per 256 MFMAs).  What the compiler then does not see are wait states: fragments come from LDS
// (behind waits that the compiler sees), so do the scale registers, an accumulator is used again 16 or more MFMAs later and read behind drain().
#define MFMA_FP4(SEL) "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL " cbsz:4 blgp:4"
#define SEL0 "op_sel_hi:[0,0,0]"
#define SEL1 "op_sel:[1,1,0] op_sel_hi:[0,0,0]"
#define SEL2 "op_sel_hi:[1,1,0]"
#define SEL3 "op_sel:[1,1,0] op_sel_hi:[1,1,0]"
template <int OP>
__device__ __forceinline__ void mfma_fp4_step(u32x4 w, u32x4 a, f32x4& c, uint32_t sw, uint32_t sa) {
    if constexpr (OP == 0) asm volatile(MFMA_FP4(SEL0) : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 1) asm volatile(MFMA_FP4(SEL1) : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 2) asm volatile(MFMA_FP4(SEL2) : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 3) asm volatile(MFMA_FP4(SEL3) : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
}
// The same with a DMA piece around it: 1 KB per wave instruction, lane l's 16 bytes at base + voff + 1024 PIECE go to LDS at m0 + 1024 PIECE + 16 l.
// M0 is set with the first of four pieces, in front of the MFMA (which is the wait state between the two), and kept for the others: nothing else in
// the loop touches it.  As asm the DMA is not drained by the compiler in front of every LDS read; it has no register result, and the hand-overs wait for it.
template <int OP, int PIECE>
__device__ __forceinline__ void mfma_fp4_dma(u32x4 w, u32x4 a, f32x4& c, uint32_t sw, uint32_t sa, uint32_t voff, const void* base, uint32_t lds) {
#define WITH_DMA(SEL)                                                                                                                       \
    if constexpr (PIECE == 0) asm volatile("s_mov_b32 m0, %7\n\t" MFMA_FP4(SEL) "\n\tglobal_load_lds_dwordx4 %5, %6" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa), "v"(voff), "s"(base), "s"(lds) : "memory"); \
    else asm volatile(MFMA_FP4(SEL) "\n\tglobal_load_lds_dwordx4 %5, %6 offset:%7" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa), "v"(voff), "s"(base), "i"(PIECE * 1024) : "memory")
    if constexpr (OP == 0) { WITH_DMA(SEL0); }
    if constexpr (OP == 1) { WITH_DMA(SEL1); }
    if constexpr (OP == 2) { WITH_DMA(SEL2); }
    if constexpr (OP == 3) { WITH_DMA(SEL3); }
#undef WITH_DMA
}
__device__ __forceinline__ void dma16(uint32_t voff, const void* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
}
// not issued unless `wanted` (uniform): the branch is hidden in the asm, where it costs the compiler's schedule nothing
__device__ __forceinline__ void dma16_if(bool wanted, uint32_t voff, const void* base, uint32_t lds) {
    asm volatile("s_cmp_eq_u32 %3, 0\n\ts_cbranch_scc1 skip%=\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\nskip%=:" ::"v"(voff), "s"(base), "s"(lds),
                 "s"((int)wanted) : "memory", "scc");
}
__device__ __forceinline__ void dma4(uint32_t voff, const void* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
}
// every LDS read has returned (a builtin: the compiler then adds no waits of its own in front of the uses)
__device__ __forceinline__ void lds_returned() { __builtin_amdgcn_s_waitcnt(0xc07f); }
// every piece but the FLYING youngest has landed, and every wave's LDS accesses are done
template <int FLYING>
__device__ __forceinline__ void hand_over() {
    static_assert(FLYING < 64, "vmcnt");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (FLYING & 15) | (FLYING >> 4 << 14));   // vmcnt FLYING, lgkmcnt 0
    asm volatile("s_barrier" ::: "memory");
}
template <int MT, int NT>
__device__ __forceinline__ void settle_acc(f32x4 (&acc)[NT][MT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) asm volatile("" : "+a"(acc[j][i]));
    asm volatile("s_nop 7" ::: "memory");
}
// every MFMA has written its accumulator
template <int MT, int NT>
__device__ __forceinline__ void drain(f32x4 (&acc)[NT][MT]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) asm volatile("" : "+a"(acc[j][i]));
}

template <class F, int... S>
__device__ __forceinline__ void each_slot(F&& f, std::integer_sequence<int, S...>) {
    (f(std::integral_constant<int, S>{}), ...);
}

// The tiles of one XCD (workgroups b, b + 8, ...) are neighbours: consecutive numbers within the XCD, walked in bands of `band` row tiles, so that
// the A and W panels its workgroups share stay in its L2.
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int band, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, x = b & 7, q = total >> 3, rem = total & 7;
    const int id = x * q + (x < rem ? x : rem) + (b >> 3);
    const int per = band * tiles_n, first = id / per * band, rows = tiles_m - first < band ? tiles_m - first : band, in = id % per;
    tm = first + in % rows;
    tn = in / rows;
}

// A wave's 16 MT x 16 NT accumulators -> memory, 16 rows at a time through the wave's own LDS (two slots of 16 rows, so that a block is written
// while the previous one is read): the accumulator layout has one row per lane, and stored straight, every 8 or 16 bytes would be an access of
// their own; through LDS the lanes of an instruction cover whole row pieces.  bf16 is rounded in front of LDS (half the traffic).
// The fields the loop uses are copied to opaque scalars: hipcc otherwise reads them from the kernel's arguments again at every use.
template <int MT, int NT, bool BF16>
constexpr int store_slot_bytes() { return 16 * (16 * NT * (BF16 ? 2 : 4) + (BF16 ? 32 : 16)); }   // row pitches that spread 16 rows over the banks

template <int MT, int NT, bool BF16, bool VEC, bool AFFINE>
__device__ __forceinline__ void store_tile(const Mxfp4Gemm& p, const f32x4 (&acc)[NT][MT], uint8_t* lds, int m0, int n0, int lane) {
    constexpr int COLS = 16 * NT, SLOT = store_slot_bytes<MT, NT, BF16>(), PITCH = SLOT / 16, ESZ = BF16 ? 2 : 4;
    const int r = lane & 15, g = lane >> 4;
    // bias and gate: bf16 takes them in front of its rounding, for the lane's accumulator columns; f32 behind LDS, where a lane keeps its columns
    f32x4 bias[NT], gate[NT];
    if constexpr (AFFINE && BF16) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = n0 + 16 * j + 4 * g;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                bias[j][e] = p.bias && n + e < p.N ? p.bias[n + e] : 0.f;
                gate[j][e] = p.gate && n + e < p.N ? p.gate[n + e] : 1.f;
            }
        }
    }
    auto put = [&](int i) {
        uint8_t* at = lds + (i & 1) * SLOT + r * PITCH + 4 * g * ESZ;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            f32x4 v = acc[j][i];
            if constexpr (AFFINE && BF16) v = (v + bias[j]) * gate[j];
            if constexpr (BF16) *reinterpret_cast<uint2*>(at + 32 * j) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            else *reinterpret_cast<f32x4*>(at + 64 * j) = v;
        }
    };
    auto ordered = [] {   // LDS executes a wave's accesses in order: only the compiler must keep them so
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    uint64_t ld = (uint64_t)p.ld_out * ESZ, ldr = (uint64_t)p.ld_resid * 4;
    const uint8_t* resid = reinterpret_cast<const uint8_t*>(p.resid);
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out);
    asm volatile("" : "+s"(ld), "+s"(ldr), "+s"(resid), "+s"(out));
    put(0);
    if constexpr (VEC) {
        constexpr int CPL = 16 / ESZ, LPR = COLS / CPL, RPI = 64 / LPR, Q = 16 / RPI;   // columns per lane, lanes per row, rows per instruction
        const int c = (lane % LPR) * CPL, n = n0 + c, row = lane / LPR;
        const int rows_left = n < p.N ? p.M - m0 - row : 0;   // N % CPL == 0
        uint8_t* o = out + (uint64_t)(m0 + row) * ld + (uint64_t)n * ESZ;
        const uint8_t* x = resid + (uint64_t)(m0 + row) * ldr + (uint64_t)n * 4;
        f32x4 b4 = {0.f, 0.f, 0.f, 0.f}, g4 = {1.f, 1.f, 1.f, 1.f};
        if constexpr (AFFINE && !BF16) {
            if (p.bias && n < p.N) b4 = *reinterpret_cast<const f32x4*>(p.bias + n);
            if (p.gate && n < p.N) g4 = *reinterpret_cast<const f32x4*>(p.gate + n);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (i + 1 < MT) put(i + 1);
            ordered();
            u32x4 v[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) v[q] = *reinterpret_cast<const u32x4*>(lds + (i & 1) * SLOT + (q * RPI + row) * PITCH + c * ESZ);
            f32x4 res[Q];
            if (!BF16 && resid) {
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (16 * i + q * RPI < rows_left) res[q] = *reinterpret_cast<const f32x4*>(x + (uint64_t)(16 * i + q * RPI) * ldr);
            }
            ordered();
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                if constexpr (AFFINE && !BF16) v[q] = __builtin_bit_cast(u32x4, (__builtin_bit_cast(f32x4, v[q]) + b4) * g4);
                if (!BF16 && resid) v[q] = __builtin_bit_cast(u32x4, __builtin_bit_cast(f32x4, v[q]) + res[q]);
                if (16 * i + q * RPI < rows_left) *reinterpret_cast<u32x4*>(o + (uint64_t)(16 * i + q * RPI) * ld) = v[q];
            }
        }
    } else {   // one column per lane
        const int rows_left = p.M - m0;
        float b1[COLS / 64], g1[COLS / 64];
        if constexpr (AFFINE && !BF16) {
#pragma unroll
            for (int h = 0; h < COLS / 64; ++h) {
                const int n = n0 + 64 * h + lane;
                b1[h] = p.bias && n < p.N ? p.bias[n] : 0.f;
                g1[h] = p.gate && n < p.N ? p.gate[n] : 1.f;
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (i + 1 < MT) put(i + 1);
            ordered();
#pragma unroll 4
            for (int q = 0; q < 16 * COLS / 64; ++q) {
                const int row = q * 64 / COLS, c = q * 64 % COLS + lane, n = n0 + c;
                static_assert(COLS % 64 == 0, "a row piece is whole lanes");
                const uint8_t* at = lds + (i & 1) * SLOT + row * PITCH + c * ESZ;
                if (16 * i + row < rows_left && n < p.N) {
                    uint8_t* o = out + (uint64_t)(m0 + 16 * i + row) * ld + (uint64_t)n * ESZ;
                    if constexpr (BF16) *reinterpret_cast<uint16_t*>(o) = *reinterpret_cast<const uint16_t*>(at);
                    else {
                        float f = *reinterpret_cast<const float*>(at);
                        if constexpr (AFFINE) f = (f + b1[q % (COLS / 64)]) * g1[q % (COLS / 64)];
                        if (resid) f += *reinterpret_cast<const float*>(resid + (uint64_t)(m0 + 16 * i + row) * ldr + (uint64_t)n * 4);
                        *reinterpret_cast<float*>(o) = f;
                    }
                }
            }
            ordered();
        }
    }
}

// CUT: whether the last group is cut; if not, DMA addresses need no per-lane arithmetic in the loop
enum { CUT_NONE = 0, CUT_TAIL = 1, CUT_SHORT = 2 };   // steps % 4 == 0, steps >= 4, steps < 4
template <int BM, int BN, bool BF16, bool VEC, int CUT, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void mxfp4_gemm_tile_kernel(Mxfp4Gemm p, int tiles_m, int tiles_n, int band) {
    constexpr int MT = BM / 32, NT = BN / 32, SLOTS = MT * NT;   // 16-row blocks per wave; MFMAs per phase
    constexpr int ROWS = BM + BN;                          // LDS rows of a stage: W's, then A's
    constexpr int STAGE = ROWS * 128, SCALES = ROWS * 16;
    constexpr int PW = BN / 32, PA = BM / 32, NP = PW + PA; // code pieces per wave and stage
    // slot of P0 (P2) in which the buffer is free; piece k of its next stage goes with slot FREE + 1 + k EVERY, counted on into P1 (P3)
    constexpr int FREE = SLOTS / 2, EVERY = SLOTS * 3 / 2 / NP, FIRST = (SLOTS - FREE - 2) / EVERY + 1;   // FIRST: pieces requested in P0 (P2)
    static_assert(FREE + 1 + (NP - 1) * EVERY < 2 * SLOTS, "the last piece lies in the second phase");
    constexpr int SR = ROWS / 256;                         // scale rows per thread
    extern __shared__ __align__(1024) uint8_t smem[];      // [2][STAGE] codes, [2][SCALES] scales, [2 SCALES] two groups' scales as they came
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, band, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const uint32_t row_bytes = (uint32_t)p.steps * 64, row_scales = (uint32_t)p.steps * 4;
    const uint8_t* wbase = p.w + (int64_t)n0 * row_bytes;
    const uint8_t* abase = reinterpret_cast<const uint8_t*>(p.a) + (int64_t)m0 * row_bytes;
    const int last_w = p.N - 1 - n0, last_a = p.M - 1 - m0;   // rows behind the last one: its copy, never stored
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const int steps = p.steps, groups = (steps + 3) >> 2, last_stage = (steps - 1) >> 1;

    // DMA sources relative to the stage's column: lane l fetches chunk (l % 8) ^ (row % 8) of row l / 8 of its piece.  Four pieces share one M0: the
    // instruction's offset goes to both addresses, so piece k of them starts 1024 k further in LDS and its source offset carries -1024 k (+ LOWER so
    // that it stays unsigned; the scalar base is LOWER lower).
    constexpr uint32_t LOWER = 3 * 1024;
    uint32_t vw[PW], va[PA];
    const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int k = 0; k < PW; ++k) { const int row = (wave * PW + k) * 8 + (lane >> 3); vw[k] = (uint32_t)(row < last_w ? row : last_w) * row_bytes + chunk + LOWER - (k & 3) * 1024; }
#pragma unroll
    for (int k = 0; k < PA; ++k) { const int row = (wave * PA + k) * 8 + (lane >> 3); va[k] = (uint32_t)(row < last_a ? row : last_a) * row_bytes + chunk + LOWER - (k & 3) * 1024; }
    wbase -= LOWER;
    abase -= LOWER;
    // the second step of the last stage may lie behind the row: its chunks are then fetched from the first step (their scales are 0)
    auto back_of = [&](int stage) { return CUT != CUT_NONE && stage == last_stage && (steps & 1) && chunk >= 64 ? 64u : 0u; };
    auto code_lds = [&](int k, int buf) { return lds0 + buf * STAGE + (k < PW ? (wave * PW + (k & ~3)) * 1024 : BN * 128 + (wave * PA + ((k - PW) & ~3)) * 1024); };

    // Scales: the 16 bytes [step][block] of a row and group come to LDS by DMA as they are, two groups at a time (what counts is the lines touched, a
    // third of them if every group's scales came alone: 4608 x 36864 x 4096 369 us, this way 356; 333 x 6144 x 18432 47.8, 44.2); the thread of the row transposes a group's to
    // one register per block with the steps as its bytes and writes [row / 64][block][row % 16][row / 16 % 4]: a fragment lane then reads the
    // registers of four row blocks at once.  (Loaded into registers instead, their use makes the compiler wait for every younger DMA piece too:
    // 388 us against 360 when that was tried.)
    uint32_t vs[2 * SR];
    const uint8_t* sbase[SR];
#pragma unroll
    for (int h = 0; h < SR; ++h) {   // piece 2 h + e: rows wave 64 + 256 h + 32 e ..., two lanes each; CUT_SHORT: piece 2 h, one lane per row
        const int first = wave * 64 + 256 * h, row0 = first < BN ? first : first - BN, last = first < BN ? last_w : last_a;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = CUT == CUT_SHORT ? row0 + lane : row0 + 32 * e + (lane >> 1);
            vs[2 * h + e] = (uint32_t)(row < last ? row : last) * row_scales;
        }
        sbase[h] = first < BN ? p.w_scales + (int64_t)n0 * row_scales : p.a_scales + (int64_t)m0 * row_scales;
    }
    constexpr int RAW = 2 * STAGE + 2 * SCALES;
    // groups `group` and group + 1; a group that K cuts, or that lies behind it, comes as the row's last 16 bytes.  Rows of fewer than four steps: dword by dword
    auto fetch_scales = [&](int i, int group, bool wanted) {
        const int h = i >> 1;
        if constexpr (CUT == CUT_SHORT) {   // LDS: [step][row]
            if (i & 1) return;
#pragma unroll
            for (int s = 0; s < 4; ++s) dma4(vs[i] + (s < steps ? s : steps - 1) * 4, sbase[h], lds0 + RAW + h * 4096 + s * 1024 + wave * 256);
        } else {   // LDS: [row][group][step]
            const uint32_t at = (uint32_t)group * 16 + (lane & 1) * 16, last = row_scales - 16;
            dma16_if(wanted, vs[i] + (at < last ? at : last), sbase[h], lds0 + RAW + (h * 256 + wave * 64) * 32 + (i & 1) * 1024);
        }
    };
    auto take_scales = [&](int h, int group) {   // steps behind K: 0
        u32x4 d;
        if constexpr (CUT == CUT_SHORT) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(smem + RAW + h * 4096 + s * 1024 + threadIdx.x * 4);
                d[s] = s < steps ? v : 0u;
            }
        } else {
            d = *reinterpret_cast<const u32x4*>(smem + RAW + (h * 256 + threadIdx.x) * 32 + (group & 1) * 16);
            if constexpr (CUT == CUT_TAIL) {   // a cut group's bytes lie `skip` steps further on
                const int skip = group * 4 + 4 > steps ? group * 4 + 4 - steps : 0;
                if (skip & 1) d = u32x4{d[1], d[2], d[3], 0u};
                if (skip & 2) d = u32x4{d[2], d[3], 0u, 0u};
            }
        }
        return d;
    };
    auto write_scales = [&](int h, u32x4 d, int buf) {
        const int row = threadIdx.x + 256 * h;
        uint32_t* at = reinterpret_cast<uint32_t*>(smem + 2 * STAGE + buf * SCALES + (row >> 6) * 1024 + (row & 15) * 16 + (row >> 4 & 3) * 4);
        const uint32_t t0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), t1 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
        const uint32_t t2 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), t3 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
        at[0] = __builtin_amdgcn_perm(t2, t0, 0x05040100u);
        at[64] = __builtin_amdgcn_perm(t2, t0, 0x07060302u);
        at[128] = __builtin_amdgcn_perm(t3, t1, 0x05040100u);
        at[192] = __builtin_amdgcn_perm(t3, t1, 0x07060302u);
    };
    // four row blocks of this wave, W's first
    auto read_scales = [&](int t, int buf) {
        const int quad = t < NT / 4 ? wn * (NT / 4) + t : BN / 64 + wm * (MT / 4) + t - NT / 4;
        return *reinterpret_cast<const u32x4*>(smem + 2 * STAGE + buf * SCALES + quad * 1024 + g * 256 + r * 16);
    };

    // fragment reads: LDS bytes of this lane's chunk, per stage buffer and step (opaque, or hipcc recomputes them at every read)
    typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
    uint32_t fbw[2][2], fba[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const uint32_t c = ((4 * ks + g) ^ (r & 7)) * 16;
            fbw[b][ks] = lds0 + b * STAGE + (wn * NT * 16 + r) * 128 + c;
            fba[b][ks] = lds0 + b * STAGE + (BN + wm * MT * 16 + r) * 128 + c;
            asm volatile("" : "+v"(fbw[b][ks]), "+v"(fba[b][ks]));
        }
    auto frag_w = [&](int j, int buf, int ks) { return *reinterpret_cast<lds_u32x4*>((uintptr_t)(fbw[buf][ks] + j * 2048)); };
    auto frag_a = [&](int i, int buf, int ks) { return *reinterpret_cast<lds_u32x4*>((uintptr_t)(fba[buf][ks] + i * 2048)); };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 fw[2][NT], fa[2][MT];
    u32x4 sc[(NT + MT) / 4];   // scale registers of the current group
    auto sw = [&](int j) { return sc[j / 4][j % 4]; };
    auto sa = [&](int i) { return sc[NT / 4 + i / 4][i % 4]; };

    // one latency for the scales of two groups and two stages of codes; the second stage is still in flight when the loop begins
#pragma unroll
    for (int i = 0; i < 2 * SR; ++i) fetch_scales(i, 0, true);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int stage = b < last_stage ? b : last_stage;
#pragma unroll
        for (int k = 0; k < NP; ++k)
            dma16((k < PW ? vw[k] : va[k - PW]) - back_of(stage), (k < PW ? wbase : abase) + stage * 128 + (k & 3) * 1024, code_lds(k, b) + (k & 3) * 1024);
    }
    hand_over<NP>();
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int h = 0; h < SR; ++h) write_scales(h, take_scales(h, b), b);
    lds_returned();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int t = 0; t < (NT + MT) / 4; ++t) sc[t] = read_scales(t, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) fw[0][j] = frag_w(j, 0, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[0][i] = frag_a(i, 0, 0);
    settle_acc<MT, NT>(acc);

    // One loop body without a branch: behind the last group the requests repeat that group's.
    for (int q = 0; q < groups; ++q) {
        const int qn = q + 1 < groups ? q + 1 : q;
        const int s0 = 2 * qn, s1 = 2 * qn + 1 < last_stage ? 2 * qn + 1 : last_stage;
        const uint8_t *w0 = wbase + s0 * 128, *a0 = abase + s0 * 128, *w1 = wbase + s1 * 128, *a1 = abase + s1 * 128;
        const uint32_t back0 = back_of(s0), back1 = back_of(s1);
        // the scales of groups q + 2 and q + 3 (q even) are requested in P1 and have landed at the hand-over behind P2; P3 transposes those of group q + 2
        // and reads those of group q + 1
        u32x4 raw[SR], next[(NT + MT) / 4];
#pragma unroll
        for (int t = 0; t < (NT + MT) / 4; ++t) asm volatile("" : "+v"(sc[t]));
        asm volatile("s_nop 7" ::: "memory");   // the copies of `next` into the scale registers have settled
        auto phase = [&](auto op) {
            constexpr int OP = decltype(op)::value, CUR = OP & 1, NBUF = OP == 1 || OP == 2 ? 1 : 0, NKS = OP & 1 ? 0 : 1;
            constexpr int READS = MT + NT, RSPAN = OP & 1 ? SLOTS / 2 : SLOTS * 3 / 8;
            each_slot([&](auto slot) {
                constexpr int S = decltype(slot)::value, i = S / NT, j = S % NT;
#pragma unroll
                for (int t = 0; t < READS; ++t)
                    if (t * RSPAN / READS == S) {
                        if (t < NT) fw[1 - CUR][t] = frag_w(t, NBUF, NKS);
                        else fa[1 - CUR][t - NT] = frag_a(t - NT, NBUF, NKS);
                    }
                if constexpr (OP == 1) {   // in front of a piece that sets M0
#pragma unroll
                    for (int i = 0; i < 2 * SR; ++i)
                        if (S == FREE + 1 + NP / 2 * EVERY - SLOTS - 1 - i) fetch_scales(i, q + 2, !(q & 1));
                }
                if constexpr (OP == 3) {
#pragma unroll
                    for (int h = 0; h < SR; ++h)
                        if (S == SLOTS / 4 + h) raw[h] = take_scales(h, q + 2);
#pragma unroll
                    for (int h = 0; h < SR; ++h)
                        if (S == SLOTS / 2 + 8 * h) write_scales(h, raw[h], q & 1);
#pragma unroll
                    for (int t = 0; t < (NT + MT) / 4; ++t)
                        if (S == SLOTS / 2 + 1 + 2 * t) next[t] = read_scales(t, (q + 1) & 1);
                }
                if constexpr (!(OP & 1) && S == FREE) {   // everybody has read its last fragments of the buffer
                    lds_returned();
                    asm volatile("s_barrier" ::: "memory");
                }
                constexpr int since = (OP & 1 ? SLOTS : 0) + S - FREE - 1, k = since >= 0 && since % EVERY == 0 ? since / EVERY : NP;
                if constexpr (k < NP) {
                    mfma_fp4_dma<OP, k & 3>(fw[CUR][j], fa[CUR][i], acc[j][i], sw(j), sa(i), (k < PW ? vw[k < PW ? k : 0] : va[k < PW ? 0 : k - PW]) - (OP < 2 ? back0 : back1),
                                            OP < 2 ? (k < PW ? w0 : a0) : (k < PW ? w1 : a1), code_lds(k, OP < 2 ? 0 : 1));
                } else mfma_fp4_step<OP>(fw[CUR][j], fa[CUR][i], acc[j][i], sw(j), sa(i));
                __builtin_amdgcn_sched_barrier(0);
            }, std::make_integer_sequence<int, SLOTS>{});
        };
        phase(std::integral_constant<int, 0>{});
        hand_over<FIRST>();
        phase(std::integral_constant<int, 1>{});
        lds_returned();
        phase(std::integral_constant<int, 2>{});
        hand_over<FIRST>();
        phase(std::integral_constant<int, 3>{});
        lds_returned();
#pragma unroll
        for (int t = 0; t < (NT + MT) / 4; ++t) sc[t] = next[t];
    }
    drain<MT, NT>(acc);
    hand_over<0>();   // everybody has left the stages: their LDS becomes the epilogue's
    uint8_t* mine = smem + wave * 2 * store_slot_bytes<MT, NT, BF16>();
    if (p.bias || p.gate) store_tile<MT, NT, BF16, VEC, true>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
    else store_tile<MT, NT, BF16, VEC, false>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
}

// ---------------------------------------------------------------------------------------------- small tiles, k split over groups of waves
// BM x BN outputs per workgroup of KG WM x WN waves: group kg of the waves takes the 128-k steps KG t + kg, and the groups' sums are added through LDS at
// the end.  With few tiles a CU holds one, and a stage of it takes ~1200 cycles whatever its size (wait, barrier, LDS reads, MFMAs, requests: one wave per
// SIMD issues them in turn), so what counts is how many k a stage holds: 64 x 4096 x 4096 with 64 x 64 tiles and two groups 11.3 us, four 9.4, four and 32 x 64
// tiles 7.4 (the 128 x 128 tiles above 11.9).  Bound by that latency: 16 x 36864 x 4096 17.6 us = 4.6 TB/s of W, 16 x 12288 x 4096 7.2
// (W from HBM: 19.3, 8.2).  A stage is KG / 2 pairs of steps, a pair 128 bytes of every row (pieces and swizzle as above), in a ring of STAGES buffers,
// STAGES - 1 of them requested ahead with a counted wait.  The scales of 16 steps come at once, one dword per row and step, ahead of the first of them;
// slot c of a row holds step c ^ (row / 4) % 4 of the 16, so that the 16 rows a fragment reads lie in different banks.
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool BF16, bool VEC>
__global__ __launch_bounds__(64 * WM * WN * KG) void mxfp4_gemm_ring_kernel(Mxfp4Gemm p, int tiles_m, int tiles_n, int band) {
    constexpr int WAVES = KG * WM * WN, MT = BM / (16 * WM), NT = BN / (16 * WN), ROWS = BM + BN;   // LDS rows of a stage: W's, then A's
    constexpr int HALF = ROWS * 128, STAGE = KG / 2 * HALF, SCALES = ROWS * 64, CNT = KG * ROWS / 16 / WAVES, TPG = 16 / KG, NS = ROWS / 4 / WAVES;   // code pieces per wave and stage; scale pieces per wave and 16 steps
    static_assert(CNT * 16 * WAVES == ROWS * KG && NS * 4 * WAVES == ROWS && BN % 8 == 0 && STAGES <= TPG / 2 + 2, "whole pieces; scales land in front of their use");
    extern __shared__ __align__(1024) uint8_t smem[];   // [STAGES][STAGE] codes, [2][SCALES] scales
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % WM, wn = wave / WM % WN;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, band, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN, steps = p.steps, pairs = (steps + 1) >> 1, stages = (steps + KG - 1) / KG;
    const uint32_t row_bytes = (uint32_t)steps * 64, row_scales = (uint32_t)steps * 4;
    const uint8_t* wbase = p.w + (int64_t)n0 * row_bytes;
    const uint8_t* abase = reinterpret_cast<const uint8_t*>(p.a) + (int64_t)m0 * row_bytes;
    const uint8_t* wsbase = p.w_scales + (int64_t)n0 * row_scales;
    const uint8_t* asbase = p.a_scales + (int64_t)m0 * row_scales;
    const int last_w = p.N - 1 - n0, last_a = p.M - 1 - m0;   // rows behind the last one: its copy, never stored
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    auto clamped = [&](int row) { return (uint32_t)(row < BN ? (row < last_w ? row : last_w) : (row - BN < last_a ? row - BN : last_a)); };

    const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    uint32_t vc[CNT];
#pragma unroll
    for (int k = 0; k < CNT; ++k) vc[k] = clamped((wave * CNT + k) % (ROWS / 8) * 8 + (lane >> 3)) * row_bytes + chunk;
    auto issue = [&](int t, int buf) {   // stage t; behind the end the last one again, so that every stage counts alike
        // the second step of the last pair may lie behind the row: its chunks are then fetched from the first step, and not used
        const uint32_t cut = (steps & 1) && chunk >= 64 ? 64u : 0u;
#pragma unroll
        for (int k = 0; k < CNT; ++k) {
            const int piece = wave * CNT + k, want = t * (KG / 2) + piece / (ROWS / 8), pair = want < pairs ? want : pairs - 1;
            dma16(vc[k] - (pair == pairs - 1 ? cut : 0u), (piece % (ROWS / 8) * 8 < BN ? wbase : abase) + (int64_t)pair * 128, lds0 + buf * STAGE + piece * 1024);
        }
    };
    auto issue_scales = [&](int group, int j) {
        const int piece = wave * NS + j, row = piece * 4 + (lane >> 4), s = group * 16 + ((lane & 15) ^ (piece & 3)), step = s < steps ? s : steps - 1;
        dma4(clamped(row) * row_scales + (uint32_t)step * 4, piece * 4 < BN ? wsbase : asbase, lds0 + STAGES * STAGE + (group & 1) * SCALES + piece * 256);
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int s, int buf) {
        const uint8_t* c = smem + buf * STAGE + kg / 2 * HALF + (((kg & 1) * 4 + g) ^ (r & 7)) * 16;
        const uint8_t* sc = smem + STAGES * STAGE + (s >> 4 & 1) * SCALES + ((s & 15) ^ (r >> 2)) * 4 + g;
        const int wrow = wn * NT * 16 + r, arow = BN + wm * MT * 16 + r;
        u32x4 w[NT], a[MT];
        uint32_t sw[NT], sa[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            w[j] = *reinterpret_cast<const u32x4*>(c + (wrow + 16 * j) * 128);
            sw[j] = sc[(wrow + 16 * j) * 64];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            a[i] = *reinterpret_cast<const u32x4*>(c + (arow + 16 * i) * 128);
            sa[i] = sc[(arow + 16 * i) * 64];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j][i] = mfma_fp4(w[j], a[i], acc[j][i], sw[j], sa[i]);
    };
#pragma unroll
    for (int j = 0; j < NS; ++j) issue_scales(0, j);
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) issue(t, t);
    int buf = 0, before = STAGES - 1;   // t % STAGES, (t - 1) % STAGES
    for (int t = 0; t < stages; ++t) {
        hand_over<(STAGES - 2) * CNT>();   // stage t has landed (scale pieces in flight come on top: it then waits for that much more, never for less)
        const int turn = t % TPG;
        if (turn < TPG / 2) {              // the next 16 steps' scales, into the buffer that the previous 16 have left
            constexpr int EACH = (NS + TPG / 2 - 1) / (TPG / 2);
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (turn * EACH + j < NS) issue_scales(t / TPG + 1, turn * EACH + j);
        }
        issue(t + STAGES - 1, before);     // into the buffer of stage t - 1, which everybody has left
        if (KG * t + kg < steps) compute(KG * t + kg, buf);
        before = buf;
        buf = buf + 1 < STAGES ? buf + 1 : 0;
    }
    hand_over<0>();
    f32x4* part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int half = KG / 2; half >= 1; half /= 2) {   // the k groups' sums, the upper half's added to the lower's
        if (kg >= half && kg < 2 * half) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) part[((wave - half * WM * WN) * NT * MT + j * MT + i) * 64 + lane] = acc[j][i];
        }
        __syncthreads();
        if (kg < half) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[j][i] += part[(wave * NT * MT + j * MT + i) * 64 + lane];
        }
        __syncthreads();
    }
    if (kg > 0) return;
    uint8_t* mine = smem + wave * 2 * store_slot_bytes<MT, NT, BF16>();
    if (p.bias || p.gate) store_tile<MT, NT, BF16, VEC, true>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
    else store_tile<MT, NT, BF16, VEC, false>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
}

// rows of out and resid take 16-byte accesses of the columns a lane of store_tile owns (8 of bf16, 4 of f32)
bool wide_rows(const Mxfp4Gemm& p) {
    auto ok = [](const void* q, int64_t ld, int cols) { return !q || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % cols == 0); };
    const int cols = p.out_bf16 ? 8 : 4;
    return p.N % cols == 0 && ok(p.out, p.ld_out, cols) && ok(p.resid, p.ld_resid, 4) && ok(p.bias, 0, 4) && ok(p.gate, 0, 4);
}
// ---------------------------------------------------------------------------------------------- the same with A in bf16
// A is shared by every wave of a workgroup and comes once per workgroup through LDS, `chunk` steps of all its rows at a time (a multiple of the waves' U steps, so
// that a wave's steps wave, wave + WAVES, ... fall into the chunks alike); W and its scales stream through registers across the chunks.
// Read by every wave for itself, A costs four loads per step against one of W: the vector-memory path, not HBM, is then the bound.
// Measured: 1 x 19456 x 2560 9.3 us = 2.8 TB/s of W from HBM; bound by the latency of staging A and of a wave's first loads.
constexpr int BF16_ROWS_U = 2, BF16_ROWS_WAVES = 8;
template <bool AVEC, bool VEC>
__global__ __launch_bounds__(64 * BF16_ROWS_WAVES) void bf16_mxfp4_gemm_rows_kernel(Mxfp4Gemm p, int tiles_n, int chunk) {
    constexpr int U = BF16_ROWS_U, WAVES = BF16_ROWS_WAVES;
    extern __shared__ __align__(16) uint8_t smem[];   // A: [rows][chunk * 256 + 16] bytes; then the partial sums [WAVES][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = (int)(blockIdx.x % tiles_n) * 16, m0 = (int)(blockIdx.x / tiles_n) * 16;
    const int steps = p.steps, rows = p.M - m0 < 16 ? p.M - m0 : 16, pitch = chunk * 256 + 16;
    const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;   // rows behind the last one: its copy, never stored
    const uint8_t *wq = p.w + n * steps * 64 + g * 16, *ws = p.w_scales + n * steps * 4 + g;
    struct Step { u32x4 w; uint32_t s; };
    auto load = [&](int s, Step& x) {
        if (s >= steps) return;
        x.w = *reinterpret_cast<const u32x4*>(wq + (int64_t)s * 64);
        x.s = ws[(int64_t)s * 4];
    };
    const uint16_t* a = reinterpret_cast<const uint16_t*>(p.a);
    auto stage = [&](int first) {   // steps first ... first + chunk - 1 of A; columns >= K are zero
        const int pieces = chunk * 16;   // of a row, 8 values each
        for (int at = threadIdx.x; at < rows * pieces; at += 64 * WAVES) {
            const int row = at / pieces, c = at - row * pieces, k = first * 128 + c * 8;
            if (k < steps * 128) *reinterpret_cast<bf16x8*>(smem + row * pitch + c * 16) = load_a8<AVEC>(a + (int64_t)(m0 + row) * p.lda, k, p.K);
        }
    };
    const uint8_t* arow = smem + (r < rows ? r : rows - 1) * pitch + g * 64;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto use = [&](int s, int first, const Step& x) {
        if (s >= steps) return;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bf16x8 b = *reinterpret_cast<const bf16x8*>(arow + (s - first) * 256 + q * 16);
            const uint32_t code = x.w[q];
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_to_bf16(code, __builtin_bit_cast(float, x.s << 23)), b, acc, 0, 0, 0);
        }
    };
    Step cur[U], next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(wave + u * WAVES, cur[u]);
    for (int first = 0; first < steps; first += chunk) {
        if (first) __syncthreads();   // the previous chunk has been read
        stage(first);
        __syncthreads();
        const int end = first + chunk < steps ? first + chunk : steps;
        for (int s = first + wave; s < end; s += U * WAVES) {   // (a wave without a step left in the chunk has none later either)
#pragma unroll
            for (int u = 0; u < U; ++u) load(s + (U + u) * WAVES, next[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) use(s + u * WAVES, first, cur[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) cur[u] = next[u];
        }
    }
    __syncthreads();
    f32x4* part = reinterpret_cast<f32x4*>(smem);
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) acc += part[w * 64 + lane];
    store4<VEC>(p, m0 + r, n0 + 4 * g, acc);
}

// ---------------------------------------------------------------------------------------------- tiles staged through LDS (bf16 x MXFP4)
// BM x BN outputs per workgroup of WM x WN waves.  A stage is one 128-k step: 256 bytes of every A row, 64 bytes of codes and 4 scale bytes of every
// W row, all by LDS-DMA into a ring of STAGES buffers; STAGES - 1 of them are requested ahead and the wait is counted, so the stream is never drained.
// W's codes become bf16 in registers (4 conversions per 8 values, used by MT MFMAs), a lane's scale is one byte of the row's four.
// Chunks of 16 bytes are swizzled (A: within each 128-byte half by row & 7; W: the same where the codes of two steps come as one 128-byte line, else
// the 64 bytes by (row / 2) & 3) so that fragment reads meet no bank conflicts.
// Measured (W from HBM): 23 x 5121 x 5120 11.9 us, 512 x 4096 x 12288 57 us = 0.90 PF (53 with W in the 256 MB cache), 4608 x 12288 x 4096 370 us =
// 1.25 PF.  With few rows bound by the latency of a stage.  What the larger ones spend, us at 512 x 4096 x 12288 / 4608 x 12288 x 4096 in one run: all 58 / 393,
// without the requests 46 / 319, without A's LDS reads 54 / 367, without the conversions 56 / 389, without A's reads and the conversions 51 / 347, without any
// of the three 39 / 286: first the delivery into LDS, then A's fragments, which every wave of a k group reads for itself (72 KB of LDS reads per 128 k of a
// 64 x 128 tile, 576 clocks beside 512 of MFMAs), the conversions last.
// A by DMA needs rows of whole dwords (AVEC: even K and row stride); other rows pass through registers, a stage ahead (512 x 4096 x 4095: 38 to 46 us, x 4096 21).  Columns >= K are zeroed where
// the last stage is read or staged.
__device__ __forceinline__ bf16x8 zero_from(bf16x8 v, int keep) {   // values [keep, 8) become zero
    u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t w = u[d];
        u[d] = keep >= 2 * d + 2 ? w : keep == 2 * d + 1 ? w & 0xffffu : 0u;
    }
    return __builtin_bit_cast(bf16x8, u);
}

template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool AVEC, bool BF16, bool VEC>
__global__ __launch_bounds__(64 * WM * WN * KG) void bf16_mxfp4_gemm_tile_kernel(Mxfp4Gemm p, int tiles_m, int tiles_n, int band) {
    constexpr int WAVES = WM * WN * KG, MT = BM / (16 * WM), NT = BN / (16 * WN);
    constexpr int A_BYTES = BM * 256, W_BYTES = BN * 64, STAGE = KG * (A_BYTES + W_BYTES);
    constexpr bool PAIR = KG % 2 == 0;   // W's codes of two steps together: whole 128-byte lines
    constexpr int PA = BM / 4, PW = BN / 16, CNT_A = KG * PA / WAVES, CNT_W = KG * PW / WAVES, CNT = (AVEC ? CNT_A : 0) + CNT_W;   // pieces of a step; per wave and stage
    static_assert(CNT_A * WAVES == KG * PA && CNT_W * WAVES == KG * PW, "whole pieces");
    constexpr int TPG = 4 / KG, AHEAD = (STAGES - 1 + TPG - 1) / TPG, SBUF = AHEAD + 1;   // stages per scale group; groups requested ahead; their buffers
    extern __shared__ __align__(1024) uint8_t smem[];   // [STAGES]{[KG] A, [KG] W}, [SBUF][BN][16] scales
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % WM, wn = wave / WM % WN;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, band, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN, steps = p.steps, stages = (steps + KG - 1) / KG, whole = (steps - 1) / KG;   // stages in front of `whole` lie inside K
    const uint32_t row_bytes = (uint32_t)steps * 64, row_scales = (uint32_t)steps * 4, a_bytes = (uint32_t)p.lda * 2;
    const uint8_t* abase = reinterpret_cast<const uint8_t*>(p.a) + (int64_t)m0 * p.lda * 2;
    const uint8_t* wbase = p.w + (int64_t)n0 * row_bytes;
    const uint8_t* sbase = p.w_scales + (int64_t)n0 * row_scales;
    const int last_w = p.N - 1 - n0, last_a = p.M - 1 - m0;   // rows behind the last one: its copy, never stored
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;

    // piece k of this wave's A (W) pieces of a stage: step `first + k` / PA (PW) of the stage
    auto a_row = [&](int k) { const int row = (wave * CNT_A + k) % PA * 4 + (lane >> 4); return row; };
    auto a_chunk = [&](int k) { return (lane & 8) | ((lane & 7) ^ (a_row(k) & 7)); };
    uint32_t va[CNT_A], vw[CNT_W], vs[(PW + WAVES - 1) / WAVES];
#pragma unroll
    for (int k = 0; k < CNT_A; ++k) {
        const int row = a_row(k), step = (wave * CNT_A + k) / PA;
        va[k] = (uint32_t)(row < last_a ? row : last_a) * a_bytes + a_chunk(k) * 16 + step * 256;
    }
    // W: pieces of 16 rows x one step, or 8 rows x two
    auto w_row = [&](int k) { const int i = wave * CNT_W + k; return PAIR ? i % (BN / 8) * 8 + (lane >> 3) : i % PW * 16 + (lane >> 2); };
    auto w_chunk = [&](int k) { return PAIR ? (lane & 7) ^ (w_row(k) & 7) : (lane & 3) ^ (w_row(k) >> 1 & 3); };
    auto w_step = [&](int k) { const int i = wave * CNT_W + k; return PAIR ? i / (BN / 8) * 2 + (w_chunk(k) >> 2) : i / PW; };
#pragma unroll
    for (int k = 0; k < CNT_W; ++k) vw[k] = (uint32_t)(w_row(k) < last_w ? w_row(k) : last_w) * row_bytes + w_step(k) * 64 + (w_chunk(k) & 3) * 16;
#pragma unroll
    for (int k = 0; k < (PW + WAVES - 1) / WAVES; ++k) {
        const int row = (wave + WAVES * k) * 16 + (lane >> 2);
        vs[k] = (uint32_t)(row < last_w ? row : last_w) * row_scales;
    }
    // Four steps' scales at a time (what the vector-memory path counts is lines, and a row's line is touched once for them).
    auto issue_scales = [&](int group) {
        const int t = group * 4 + (lane & 3), step = t < steps ? t : steps - 1;
#pragma unroll
        for (int k = 0; k < (PW + WAVES - 1) / WAVES; ++k)
            if (wave + WAVES * k < PW) dma4(vs[k] + step * 4, sbase, lds0 + STAGES * STAGE + (uint32_t)(group % SBUF) * (BN * 16) + (wave + WAVES * k) * 256);
    };
    auto issue = [&](int t, int buf) {   // stage t; behind the end the last one again, so that every stage counts alike
        const uint32_t at = lds0 + (uint32_t)buf * STAGE;
        auto a_lds = [&](int k) { const int i = wave * CNT_A + k; return at + i * 1024; };
        auto w_lds = [&](int k) { const int i = wave * CNT_W + k; return at + KG * A_BYTES + i * 1024; };
        if (t < whole) {
            if constexpr (AVEC) {
#pragma unroll
                for (int k = 0; k < CNT_A; ++k) dma16(va[k], abase + (int64_t)t * (KG * 256), a_lds(k));
            }
#pragma unroll
            for (int k = 0; k < CNT_W; ++k) dma16(vw[k], wbase + (int64_t)t * (KG * 64), w_lds(k));
        } else {   // steps and chunks behind K are fetched from the last ones: a row's last 16 bytes, also for a chunk that K cuts
            const int last = steps - 1, first = whole * KG;
            const uint32_t end = (uint32_t)p.K * 2 - 16;
            if constexpr (AVEC) {
#pragma unroll
                for (int k = 0; k < CNT_A; ++k) {
                    const int s = (wave * CNT_A + k) / PA, step = first + s < last ? first + s : last, row = a_row(k);
                    const uint32_t col = (uint32_t)step * 256 + a_chunk(k) * 16;
                    dma16((uint32_t)(row < last_a ? row : last_a) * a_bytes + (col < end ? col : end), abase, a_lds(k));
                }
            }
#pragma unroll
            for (int k = 0; k < CNT_W; ++k) {
                const int s = w_step(k), step = first + s < last ? first + s : last;
                dma16(vw[k] + (uint32_t)(step - s) * 64, wbase, w_lds(k));
            }
        }
    };
    // AVEC false: A through registers, chunk `tid + 64 WAVES c` of the stage's KG BM rows of 16
    constexpr int AC = KG * BM * 16 / (64 * WAVES);
    static_assert(AC * 64 * WAVES == KG * BM * 16, "whole chunks");
    u32x4 areg[AVEC ? 1 : AC];
    auto fetch_a = [&](int t) {
        if constexpr (!AVEC) {
#pragma unroll
            for (int c = 0; c < AC; ++c) {
                const int at = threadIdx.x + 64 * WAVES * c, row = (at >> 4) % BM, step = t * KG + (at >> 4) / BM, k = step * 128 + (at & 15) * 8;
                areg[c] = u32x4{0, 0, 0, 0};
                if (k < p.K) areg[c] = __builtin_bit_cast(u32x4, load_a8<false>(reinterpret_cast<const uint16_t*>(abase + (int64_t)(row < last_a ? row : last_a) * a_bytes), k, p.K));
            }
        }
    };
    auto put_a = [&](int buf) {
        if constexpr (!AVEC) {
#pragma unroll
            for (int c = 0; c < AC; ++c) {
                const int at = threadIdx.x + 64 * WAVES * c, row = (at >> 4) % BM, s = (at >> 4) / BM, ch = at & 15;
                *reinterpret_cast<u32x4*>(smem + buf * STAGE + s * A_BYTES + row * 256 + ((ch & 8) | ((ch & 7) ^ (row & 7))) * 16) = areg[c];
            }
        }
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int s, int buf, auto last) {   // step s, this wave's of the stage in `buf`
        const uint8_t* arow = smem + buf * STAGE + kg * A_BYTES + (wm * MT * 16 + r) * 256;
        const uint8_t* wrow = smem + buf * STAGE + KG * A_BYTES + (PAIR ? kg / 2 * (BN * 128) + (wn * NT * 16 + r) * 128 + (((kg & 1) * 4 + g) ^ (r & 7)) * 16
                                                                       : kg * W_BYTES + (wn * NT * 16 + r) * 64 + (g ^ (r >> 1 & 3)) * 16);
        const uint8_t* srow = smem + STAGES * STAGE + (s >> 2) % SBUF * (BN * 16) + (wn * NT * 16 + r) * 16 + (s & 3) * 4 + g;
        u32x4 w[NT];
        float sc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            w[j] = *reinterpret_cast<const u32x4*>(wrow + j * (PAIR ? 2048 : 1024));
            sc[j] = __builtin_bit_cast(float, (uint32_t)srow[j * 256] << 23);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            bf16x8 a[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int c = 4 * g + q;   // (row & 7 = r & 7 in every 16-row block)
                a[i] = *reinterpret_cast<const bf16x8*>(arow + i * 4096 + ((c & 8) | ((c & 7) ^ (r & 7))) * 16);
                if constexpr (AVEC && decltype(last)::value) {
                    const int keep = p.K - s * 128 - c * 8;   // (even)
                    if (keep > 0 && keep < 8) {               // fetched 8 - keep values early
                        const u32x4 u = __builtin_bit_cast(u32x4, a[i]);
                        a[i] = __builtin_bit_cast(bf16x8, keep == 6 ? u32x4{u[1], u[2], u[3], 0} : keep == 4 ? u32x4{u[2], u[3], 0, 0} : u32x4{u[3], 0, 0, 0});
                    }
                    a[i] = zero_from(a[i], keep);
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint32_t code = w[j][q];
                const bf16x8 b = codes_to_bf16(code, sc[j]);
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a[i], acc[j][i], 0, 0, 0);
            }
        }
    };
    fetch_a(0);
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) issue_scales(q);
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) issue(t, t);
    put_a(0);
    fetch_a(1);
    int buf = 0, before = STAGES - 1;   // t % STAGES, (t - 1) % STAGES
    auto turn = [&](int t, auto last) {
        constexpr int FLY = (STAGES - 2) * CNT;   // (a wave's scale pieces come on top: it then waits for that much more, never for less)
        static_assert(FLY < 64, "vmcnt");
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (FLY & 15) | (FLY >> 4 << 14));   // stage t has landed; lgkmcnt 0
        asm volatile("s_barrier" ::: "memory");
        const int after = buf + 1 < STAGES ? buf + 1 : 0;
        put_a(after);                    // (in front of the requests: its registers' wait would take them along)
        if (t % TPG == 0) issue_scales(t / TPG + AHEAD);
        issue(t + STAGES - 1, before);   // into the buffer of stage t - 1, which everybody has left
        fetch_a(t + 2);
        if constexpr (decltype(last)::value) {
            if (t * KG + kg < steps - 1) compute(t * KG + kg, buf, std::false_type{});
            else if (t * KG + kg == steps - 1) compute(steps - 1, buf, std::true_type{});
        } else compute(t * KG + kg, buf, std::false_type{});
        before = buf;
        buf = after;
    };
    for (int t = 0; t + 1 < stages; ++t) turn(t, std::false_type{});
    turn(stages - 1, std::true_type{});
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (KG > 1) {   // the k groups' sums, added in their order
        f32x4* part = reinterpret_cast<f32x4*>(smem);
        if (kg > 0) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) part[((wave - WM * WN) * NT * MT + j * MT + i) * 64 + lane] = acc[j][i];
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int h = 0; h < KG - 1; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[j][i] += part[((wave + h * WM * WN) * NT * MT + j * MT + i) * 64 + lane];
        }
        __syncthreads();
        if (kg > 0) return;
    }
    if constexpr (NT >= 4) {
        uint8_t* mine = smem + wave * 2 * store_slot_bytes<MT, NT, BF16>();
        if (p.bias || p.gate) store_tile<MT, NT, BF16, VEC, true>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
        else store_tile<MT, NT, BF16, VEC, false>(p, acc, mine, m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
    } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) store4<VEC>(p, m0 + (wm * MT + i) * 16 + r, n0 + (wn * NT + j) * 16 + 4 * g, acc[j][i]);
    }
}

bool four_columns(const Mxfp4Gemm& p) {
    auto ok = [](const void* q, int64_t ld, int esz) { return !q || (reinterpret_cast<uintptr_t>(q) % (4 * esz) == 0 && ld % 4 == 0); };
    return p.N % 4 == 0 && ok(p.out, p.ld_out, p.out_bf16 ? 2 : 4) && ok(p.resid, p.ld_resid, 4) && ok(p.bias, 0, 4) && ok(p.gate, 0, 4);
}

int launch_rows(hipStream_t stream, const Mxfp4Gemm& p) {
    const int tn = (p.N + 15) / 16, tm = (p.M + 15) / 16;
    const dim3 grid((unsigned)(tn * (int64_t)tm)), block(64 * ROWS_WAVES);
    if (four_columns(p)) mxfp4_gemm_rows_kernel<true><<<grid, block, 0, stream>>>(p, tn);
    else mxfp4_gemm_rows_kernel<false><<<grid, block, 0, stream>>>(p, tn);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

template <bool AVEC>
int launch_bf16_rows(hipStream_t stream, const Mxfp4Gemm& p) {
    constexpr int unit = BF16_ROWS_WAVES * BF16_ROWS_U;
    const int64_t tn = (p.N + 15) / 16, tm = (p.M + 15) / 16;
    const int rows = p.M < 16 ? p.M : 16;
    int chunk = 65536 / (rows * 256) / unit * unit;                    // A's part of LDS: 64 KB (at least one unit: 16 rows x 16 steps)
    const int all = (p.steps + unit - 1) / unit * unit;
    if (chunk > all) chunk = all;
    const int lds_a = rows * (chunk * 256 + 16), lds_sums = BF16_ROWS_WAVES * 1024, lds = lds_a > lds_sums ? lds_a : lds_sums;
    const dim3 grid((unsigned)(tn * tm)), block(64 * BF16_ROWS_WAVES);
    const auto fn = four_columns(p) ? bf16_mxfp4_gemm_rows_kernel<AVEC, true> : bf16_mxfp4_gemm_rows_kernel<AVEC, false>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return 2;
    fn<<<grid, block, lds, stream>>>(p, (int)tn, chunk);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

template <int BM, int BN, int PER_CU, bool BF16, bool VEC, int CUT>
int launch_tile_form(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    constexpr int LDS = (BM + BN) * (2 * 128 + 4 * 16);
    const auto fn = mxfp4_gemm_tile_kernel<BM, BN, BF16, VEC, CUT, PER_CU>;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return 2;
    fn<<<dim3((unsigned)(tn * tm)), dim3(256), LDS, stream>>>(p, (int)tm, (int)tn, 6);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}
template <int BM, int BN, int PER_CU, bool BF16, bool VEC>
int launch_tile_cut(hipStream_t stream, const Mxfp4Gemm& p) {
    if (p.steps < 4) return launch_tile_form<BM, BN, PER_CU, BF16, VEC, CUT_SHORT>(stream, p);
    if (p.steps % 4) return launch_tile_form<BM, BN, PER_CU, BF16, VEC, CUT_TAIL>(stream, p);
    return launch_tile_form<BM, BN, PER_CU, BF16, VEC, CUT_NONE>(stream, p);
}
template <int BM, int BN, int PER_CU>
int launch_tile(hipStream_t stream, const Mxfp4Gemm& p) {
    const bool vec = wide_rows(p);
    if (p.out_bf16) return vec ? launch_tile_cut<BM, BN, PER_CU, true, true>(stream, p) : launch_tile_cut<BM, BN, PER_CU, true, false>(stream, p);
    return vec ? launch_tile_cut<BM, BN, PER_CU, false, true>(stream, p) : launch_tile_cut<BM, BN, PER_CU, false, false>(stream, p);
}

template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool BF16, bool VEC>
int launch_ring_form(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    constexpr int NT = BN / (16 * WN), MT = BM / (16 * WM), RING = (BM + BN) * (STAGES * KG * 64 + 2 * 64);
    constexpr int EPI = WM * WN * 2 * store_slot_bytes<MT, NT, BF16>(), SUMS = KG / 2 * WM * WN * NT * MT * 1024, LDS = RING > EPI ? (RING > SUMS ? RING : SUMS) : (EPI > SUMS ? EPI : SUMS);
    static_assert(LDS <= 163840, "160 KB");
    const auto fn = mxfp4_gemm_ring_kernel<BM, BN, WM, WN, KG, STAGES, BF16, VEC>;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return 2;
    fn<<<dim3((unsigned)(tn * tm)), dim3(64 * WM * WN * KG), LDS, stream>>>(p, (int)tm, (int)tn, 6);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}
template <int BM, int BN, int WM, int WN, int KG, int STAGES>
int launch_ring(hipStream_t stream, const Mxfp4Gemm& p) {
    const bool vec = wide_rows(p);
    if (p.out_bf16) return vec ? launch_ring_form<BM, BN, WM, WN, KG, STAGES, true, true>(stream, p) : launch_ring_form<BM, BN, WM, WN, KG, STAGES, true, false>(stream, p);
    return vec ? launch_ring_form<BM, BN, WM, WN, KG, STAGES, false, true>(stream, p) : launch_ring_form<BM, BN, WM, WN, KG, STAGES, false, false>(stream, p);
}

template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool AVEC, bool BF16, bool VEC>
int launch_bf16_tile_form(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    constexpr int NT = BN / (16 * WN), MT = BM / (16 * WM), TPG = 4 / KG, SBUF = (STAGES - 1 + TPG - 1) / TPG + 1;
    constexpr int RING = STAGES * KG * (BM * 256 + BN * 64) + SBUF * BN * 16, EPI = NT >= 4 ? WM * WN * 2 * store_slot_bytes<MT, NT, BF16>() : 0;
    constexpr int SUMS = (KG - 1) * WM * WN * NT * MT * 1024, LDS = RING > EPI ? (RING > SUMS ? RING : SUMS) : (EPI > SUMS ? EPI : SUMS);
    static_assert(LDS <= 163840, "160 KB");
    const auto fn = bf16_mxfp4_gemm_tile_kernel<BM, BN, WM, WN, KG, STAGES, AVEC, BF16, VEC>;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return 2;
    fn<<<dim3((unsigned)(tn * tm)), dim3(64 * WM * WN * KG), LDS, stream>>>(p, (int)tm, (int)tn, 6);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool AVEC>
int launch_bf16_tile(hipStream_t stream, const Mxfp4Gemm& p) {
    const bool vec = BN / WN >= 64 ? wide_rows(p) : four_columns(p);
    if (p.out_bf16) return vec ? launch_bf16_tile_form<BM, BN, WM, WN, KG, STAGES, AVEC, true, true>(stream, p) : launch_bf16_tile_form<BM, BN, WM, WN, KG, STAGES, AVEC, true, false>(stream, p);
    return vec ? launch_bf16_tile_form<BM, BN, WM, WN, KG, STAGES, AVEC, false, true>(stream, p) : launch_bf16_tile_form<BM, BN, WM, WN, KG, STAGES, AVEC, false, false>(stream, p);
}

// Tile of A in bf16: rounds of 256 tiles (a CU each; 16-row tiles have two workgroups per CU) x a fixed part and one per 128-k step, us, fitted to 16 ... 512
// rows x 2560 ... 19456 outputs x 2560 ... 9728 k and to 4608 rows.  With few tiles more k groups count (what a stage takes is latency), with many the
// products per byte.  What the choice gives, us: 64 x 4096 x 4096 8.6 (16 x 32), 9.7 (32 x 64), 12.2 (32 x 128); 128 x 4096 x 4096 15.3, 10.2, 12.6;
// 256 x 4096 x 4096 26.2, 18.9, 13.6; 128 x 12288 x 4096 38, 27, 24 and 20.0 (64 x 128).
enum Bf16Tile { BF16_16x32, BF16_16x64, BF16_32x64, BF16_32x128, BF16_64x128, BF16_64x256, BF16_128x256 };
Bf16Tile pick_bf16_tile(const Mxfp4Gemm& p) {
    auto tiles = [&](int bm, int bn) { return (double)(((p.M + bm - 1) / bm) * (int64_t)((p.N + bn - 1) / bn)); };
    auto two = [](double n) { return n <= 256 ? 1.0 : n <= 512 ? 1.36 : 0.7 + 0.51 * n / 256; };
    const double s = p.steps;
    const double us[] = {(3.35 + 0.08 * s) * two(tiles(16, 32)), (3.2 + 0.163 * s) * two(tiles(16, 64)), (4.05 + 0.172 * s) * std::ceil(tiles(32, 64) / 256),
                         (4.3 + 0.24 * s) * std::ceil(tiles(32, 128) / 256), (4.0 + 0.5 * s) * std::ceil(tiles(64, 128) / 256),
                         (4.0 + 0.86 * s) * std::ceil(tiles(64, 256) / 256), (4.0 + 1.72 * s) * std::ceil(tiles(128, 256) / 256)};
    return (Bf16Tile)(std::min_element(us, us + 7) - us);
}

// columns [0, n) and [n, N) of a product; rows [0, m) and [m, M)
void cut_columns(const Mxfp4Gemm& p, int n, Mxfp4Gemm& a, Mxfp4Gemm& b) {
    a = b = p;
    a.N = n;
    b.N = p.N - n;
    b.w += (int64_t)n * p.steps * 64;
    b.w_scales += (int64_t)n * p.steps * 4;
    if (p.bias) b.bias += n;
    if (p.gate) b.gate += n;
    if (p.resid) b.resid += n;
    b.out = reinterpret_cast<uint8_t*>(p.out) + (int64_t)n * (p.out_bf16 ? 2 : 4);
}
void cut_rows(const Mxfp4Gemm& p, int m, Mxfp4Gemm& a, Mxfp4Gemm& b) {
    a = b = p;
    a.M = m;
    b.M = p.M - m;
    b.a = reinterpret_cast<const uint8_t*>(p.a) + m * (p.a_scales ? (int64_t)p.steps * 64 : p.lda * 2);
    if (p.a_scales) b.a_scales += (int64_t)m * p.steps * 4;
    if (p.resid) b.resid += m * p.ld_resid;
    b.out = reinterpret_cast<uint8_t*>(p.out) + m * p.ld_out * (p.out_bf16 ? 2 : 4);
}

// MXFP4 x MXFP4 tiles.  Measured, us for a group of 512 k: a round of 256 large tiles (256 x 256, one per CU) 4.4, a round of 512 small ones (128 x 128,
// two per CU) 2.7, of up to 256 of them 1.5; a second launch costs 3 us once.  Large tiles read half as much per product; where they leave most of their
// last round empty, the columns of that round go to small ones (4608 x 4096 x 12288, 1.1 rounds: 146 -> 128 us; 4608 x 12288 x 4096, 3.4: 131 -> 129;
// 4608 x 36864 x 4096, 10.1: 384 -> 389, hence the 6 %).
double large_us(int64_t tiles) { return (double)((tiles + 255) / 256) * 4.4; }
double small_us(int64_t tiles) {
    const int64_t rest = tiles % 512;
    return (double)(tiles / 512) * 2.7 + (rest == 0 ? 0.0 : rest <= 256 ? 1.5 : 2.7);
}
int launch_mxfp4_tiles(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t m2 = (p.M + 255) / 256, n2 = (p.N + 255) / 256, m1 = (p.M + 127) / 128, n1 = (p.N + 127) / 128;
    const int64_t whole = m2 * n2 / 256 * 256 / m2;   // columns of large tiles in whole rounds
    const double large = large_us(m2 * n2), small = small_us(m1 * n1);
    const double both = whole > 0 && whole < n2 ? large_us(m2 * whole) + small_us(m1 * (n1 - 2 * whole)) + 3.0 * 4 / p.steps : 1e30;
    if (both < 0.94 * large && both < small) {
        Mxfp4Gemm a, b;
        cut_columns(p, (int)whole * 256, a, b);
        const int r = launch_tile<256, 256, 1>(stream, a);
        return r ? r : launch_tile<128, 128, 2>(stream, b);
    }
    return large < small ? launch_tile<256, 256, 1>(stream, p) : launch_tile<128, 128, 2>(stream, p);
}

// Small tiles or those above: a fixed part and one per 512 k, us, for as many tiles as there are CUs, fitted to 1 ... 512 rows x 2560 ... 36864 outputs x
// 1024 ... 16384 k.  16 x 64 tiles have two workgroups per CU.  What the choice gives, us: 64 x 4096 x 4096 6.5 / 7.6 / 8.6 (16 x 64 / 32 x 64 / 32 x 128)
// and 11.9 (128 x 128), 128 x 4096 x 4096 8.6 / 7.8 / 8.9 and 12.4, 256 x 4096 x 4096 15.3 / 14.3 / 9.4 and 13.1, 384 x 4096 x 4096 21.7 / 20.4 / 16.7 and 13.4.
enum Ring { RING_NONE, RING_16, RING_32, RING_32_WIDE };
Ring pick_ring(const Mxfp4Gemm& p) {
    auto tiles = [&](int bm, int bn) { return (double)(((p.M + bm - 1) / bm) * (int64_t)((p.N + bn - 1) / bn)); };
    const double groups = p.steps / 4.0, n16 = tiles(16, 64), n128 = tiles(128, 128);
    if (n128 > 512) return RING_NONE;
    const double us[] = {3.0 + (n128 <= 256 ? 1.1 : 2.2) * groups, (2.9 + 0.41 * groups) * (n16 <= 256 ? 1.0 : n16 <= 512 ? 1.35 : 0.55 + 0.42 * n16 / 256),
                         (3.9 + 0.44 * groups) * std::ceil(tiles(32, 64) / 256), (4.1 + 0.56 * groups) * std::ceil(tiles(32, 128) / 256)};
    return (Ring)(std::min_element(us, us + 4) - us);
}

}  // namespace

int launch_mxfp4_gemm(hipStream_t stream, const Mxfp4Gemm& p) {
    // A grid dimension holds 2^32 threads, a workgroup has at most 512 and covers at least 16 x 16 outputs: beyond 2^22 of those the longer side is halved
    // (by then each half fills the chip many times over).
    if (((int64_t)p.M + 15) / 16 * (((int64_t)p.N + 15) / 16) > 1 << 22) {
        Mxfp4Gemm a, b;
        if (p.N > p.M) cut_columns(p, p.N / 512 * 256, a, b);
        else cut_rows(p, p.M / 512 * 256, a, b);
        const int r = launch_mxfp4_gemm(stream, a);
        return r ? r : launch_mxfp4_gemm(stream, b);
    }
    const bool offsets32 = p.K < (1 << 24) && p.lda < (1 << 24);   // row offsets inside a tile fit 32 bits
    if (p.a_scales) {
        // Up to 16 rows of at most 4096 outputs (a 16-column workgroup per CU): 8 x 2560 x 2560 3.6 us, 16 x 64 tiles 5.2; 8 x 12288 x 4096 11.0, 7.0.
        // Up to 4 rows also of more outputs while k is short: 1 x 19456 x 2560 7.3 us, 8.2; 1 x 12288 x 4096 8.6, 6.9.
        if ((p.M <= 16 && p.N <= 4096) || (p.M <= 4 && p.steps <= 24) || !offsets32) return launch_rows(stream, p);
        switch (pick_ring(p)) {
            case RING_16: return launch_ring<16, 64, 1, 1, 4, 3>(stream, p);
            case RING_32: return launch_ring<32, 64, 1, 1, 4, 3>(stream, p);
            case RING_32_WIDE: return launch_ring<32, 128, 1, 2, 4, 3>(stream, p);
            case RING_NONE: break;
        }
        return launch_mxfp4_tiles(stream, p);
    }
    const bool aligned = reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && p.lda % 8 == 0;
    // few rows: A whole in LDS (1 x 19456 x 2560 8.5 us, 16-row tiles 11; at 16 rows 23.7 against 8.7)
    if (p.M <= 4 || !offsets32) return aligned ? launch_bf16_rows<true>(stream, p) : launch_bf16_rows<false>(stream, p);
    const bool dma = reinterpret_cast<uintptr_t>(p.a) % 4 == 0 && p.lda % 2 == 0 && p.K % 2 == 0 && p.K >= 8;   // A by DMA, or through registers
    const Bf16Tile tile = pick_bf16_tile(p);
    if (!dma) {
        // A's way through registers bounds these, and it is the shorter the more threads share a tile: 32 x 128 (1024 threads) in place of the middle sizes
        // (256 x 4096 x 4095: 22 us, 64 x 128 tiles of 512 threads 48; 24 x 12288 x 4097: 16 x 64 17, 32 x 64 25)
        if (tile == BF16_128x256) return launch_bf16_tile<128, 256, 2, 4, 1, 3, false>(stream, p);
        if (tile == BF16_16x32) return launch_bf16_tile<16, 32, 1, 2, 4, 3, false>(stream, p);
        if (tile == BF16_16x64 || (tile == BF16_32x64 && p.M <= 32)) return launch_bf16_tile<16, 64, 1, 4, 2, 3, false>(stream, p);
        return launch_bf16_tile<32, 128, 1, 4, 4, 2, false>(stream, p);
    }
    switch (tile) {
        case BF16_16x32: return launch_bf16_tile<16, 32, 1, 2, 4, 3, true>(stream, p);
        case BF16_16x64: return launch_bf16_tile<16, 64, 1, 4, 2, 3, true>(stream, p);
        case BF16_32x64: return launch_bf16_tile<32, 64, 1, 2, 4, 3, true>(stream, p);
        case BF16_32x128: return launch_bf16_tile<32, 128, 1, 4, 4, 2, true>(stream, p);
        case BF16_64x128: return launch_bf16_tile<64, 128, 1, 4, 2, 3, true>(stream, p);
        case BF16_64x256: return launch_bf16_tile<64, 256, 1, 4, 2, 2, true>(stream, p);
        case BF16_128x256: break;
    }
    return launch_bf16_tile<128, 256, 2, 4, 1, 3, true>(stream, p);
}
