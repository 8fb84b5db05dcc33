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

// ---------------------------------------------------------------------------------------------- tiles staged through LDS (MXFP4 x MXFP4)
// BM x BN outputs per workgroup of four waves (2 x 2), each BM/2 x BN/2.  A stage is 256 k = 128 bytes of every row; a group is two stages =
// four 128-k steps = 16 scale bytes of every row.  Both come by LDS-DMA: code pieces of 8 rows x 128 bytes (the 16-byte chunk c of row r lies at
// chunk c ^ (r & 7), so that the eight rows a fragment read touches at once sit in different banks), scale pieces of 16 rows x 16 bytes.
//
// The loop body is one group in four phases, one MFMA step each.  While a phase multiplies the fragments of one register set it reads the next
// step's into the other; the hand-over of a stage (its DMA has landed, everybody has left the previous stage) lies between two phases, so a
// stage's DMA has two whole phases to arrive:
//   P0: mfma F0 (step 0), read F1 <- buffer 0     | hand-over: buffer 1 landed, buffer 0 free
//   P1: mfma F1 (step 1), read F0 <- buffer 1,  DMA of the next group's stage 0 -> buffer 0
//   P2: mfma F0 (step 2), read F1 <- buffer 1     | hand-over: buffer 0 landed, buffer 1 free
//   P3: mfma F1 (step 3), read F0 <- buffer 0,  DMA of the next group's stage 1 -> buffer 1, scales of the next group
// A lane's four scale bytes of a group (one per step) are gathered into one register, the byte is chosen by the MFMA's op_sel.
// Steps behind K: addresses are clamped into the row and both scale bytes are 0, 2^-254 times finite codes, which is below f32: exactly 0.
//
// The MFMA is asm with the accumulator pinned to AGPRs: left to itself the register allocator of a one-wave-per-SIMD kernel moves accumulators
// and fragments between the two files (492 copies per 256 MFMAs).  What the compiler then does not see are wait states: fragments come from LDS
// (behind the compiler's own waits), scale registers pass through settle(), an accumulator is used again 16 or more MFMAs later and read behind drain().
template <int OP>
__device__ __forceinline__ void mfma_fp4_step(u32x4 w, u32x4 a, f32x4& c, uint32_t sw, uint32_t sa) {
    if constexpr (OP == 0) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 1) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 2) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
    if constexpr (OP == 3) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4" : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
}
// wait states between the VALU instructions that made these registers and the asm MFMAs that read them
template <int N>
__device__ __forceinline__ void settle(uint32_t (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(s[i]));
    asm volatile("s_nop 7" ::: "memory");
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

// 1 KB per wave instruction: lane l's 16 (4) bytes at base + voff go to LDS at m0 + 16 (4) l.  Written as asm so that the compiler does not drain
// the DMA in front of every LDS read; it has no register result, and the hand-overs below wait for it.
__device__ __forceinline__ void dma16(uint32_t voff, const void* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma4(uint32_t voff, const void* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void hand_over() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The tiles of one XCD (workgroups b, b + 8, ...) are neighbours: consecutive numbers within the XCD, walked in bands of `band` row tiles, so that
// the A and W panels its workgroups share stay in its L2.
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int band, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, x = b & 7, q = total >> 3, rem = total & 7;
    const int id = x * q + (x < rem ? x : rem) + (b >> 3);
    const int per = band * tiles_n, first = id / per * band, rows = tiles_m - first < band ? tiles_m - first : band, in = id % per;
    tm = first + in % rows;
    tn = in / rows;
}

// A wave's 16 MT x 16 NT accumulators -> memory, 16 rows at a time through the wave's own LDS (the accumulator layout has one row per lane: stored
// straight, every 8 or 16 bytes would be an access of their own; through LDS the lanes of an instruction cover whole row pieces).
template <int MT, int NT, bool VEC>
__device__ __forceinline__ void store_tile(const Mxfp4Gemm& p, const f32x4 (&acc)[NT][MT], float* lds, int m0, int n0, int lane) {
    constexpr int COLS = 16 * NT, PITCH = COLS + 4;
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4*>(lds + r * PITCH + 16 * j + 4 * g) = acc[j][i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if constexpr (VEC) {
            constexpr int LPR = COLS / 8, ROWS = 64 / LPR;   // lanes per row, 8 columns each; rows per instruction
            const int c = (lane % LPR) * 8, n = n0 + c;
#pragma unroll
            for (int q = 0; q < 16 / ROWS; ++q) {
                const int row = q * ROWS + lane / LPR, m = m0 + 16 * i + row;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(lds + row * PITCH + c), hi = *reinterpret_cast<const f32x4*>(lds + row * PITCH + c + 4);
                if (p.out_bf16 && n + 8 <= p.N && !p.resid && p.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0) {
                    if (m < p.M) {
                        f32x4 a = lo, b = hi;
                        if (p.bias) { a += *reinterpret_cast<const f32x4*>(p.bias + n); b += *reinterpret_cast<const f32x4*>(p.bias + n + 4); }
                        if (p.gate) { a *= *reinterpret_cast<const f32x4*>(p.gate + n); b *= *reinterpret_cast<const f32x4*>(p.gate + n + 4); }
                        const u32x4 u = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
                        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p.out) + m * p.ld_out + n) = u;
                    }
                } else {
                    store4<true>(p, m, n, lo);
                    store4<true>(p, m, n + 4, hi);
                }
            }
        } else {
#pragma unroll 4
            for (int q = 0; q < 16 * COLS / 64; ++q) {
                const int at = q * 64 + lane, row = at / COLS, c = at % COLS;
                store1(p, m0 + 16 * i + row, n0 + c, lds[row * PITCH + c]);
            }
        }
    }
}

template <int BM, int BN, bool VEC, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void mxfp4_gemm_tile_kernel(Mxfp4Gemm p, int tiles_m, int tiles_n, int band) {
    constexpr int MT = BM / 32, NT = BN / 32;              // 16-row blocks per wave
    constexpr int ROWS = BM + BN;                          // LDS rows of a stage: W's, then A's
    constexpr int STAGE = ROWS * 128, SCALES = ROWS * 16;
    constexpr int PW = BN / 32, PA = BM / 32;              // code pieces per wave and stage
    constexpr int QW = BN / 64, QA = BM / 64;              // scale pieces per wave and group
    extern __shared__ __align__(1024) uint8_t smem[];      // [2][STAGE] codes, [2][SCALES] scales
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, band, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const uint32_t row_bytes = (uint32_t)p.steps * 64, row_scales = (uint32_t)p.steps * 4;
    const uint8_t* wbase = p.w + (int64_t)n0 * row_bytes;
    const uint8_t* abase = reinterpret_cast<const uint8_t*>(p.a) + (int64_t)m0 * row_bytes;
    const uint8_t* wsbase = p.w_scales + (int64_t)n0 * row_scales;
    const uint8_t* asbase = p.a_scales + (int64_t)m0 * row_scales;
    const int last_w = p.N - 1 - n0, last_a = p.M - 1 - m0;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;

    // DMA sources: lane l fetches chunk (l % 8) ^ (row % 8) of row l / 8 of its piece
    uint32_t vw[PW], va[PA], vsw[QW], vsa[QA];
    const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int k = 0; k < PW; ++k) { const int row = (wave * PW + k) * 8 + (lane >> 3); vw[k] = (uint32_t)(row < last_w ? row : last_w) * row_bytes; }
#pragma unroll
    for (int k = 0; k < PA; ++k) { const int row = (wave * PA + k) * 8 + (lane >> 3); va[k] = (uint32_t)(row < last_a ? row : last_a) * row_bytes; }
#pragma unroll
    for (int k = 0; k < QW; ++k) { const int row = (wave * QW + k) * 16 + (lane >> 2); vsw[k] = (uint32_t)(row < last_w ? row : last_w) * row_scales; }
#pragma unroll
    for (int k = 0; k < QA; ++k) { const int row = (wave * QA + k) * 16 + (lane >> 2); vsa[k] = (uint32_t)(row < last_a ? row : last_a) * row_scales; }

    const int groups = (p.steps + 3) >> 2;
    // piece k of a stage (W's first); `cap`: the chunk's offset inside the row, clamped to its last one
    auto dma_code = [&](int k, int stage, int buf, uint32_t live) {
        uint32_t off = (uint32_t)stage * 128 + chunk;
        off = off < row_bytes ? off : row_bytes - 16;
        if (k < PW) dma16((vw[k] + off) & live, wbase, lds0 + buf * STAGE + (wave * PW + k) * 1024);
        else dma16((va[k - PW] + off) & live, abase, lds0 + buf * STAGE + BN * 128 + (wave * PA + k - PW) * 1024);
    };
    auto dma_scale = [&](int k, int group, uint32_t live) {
        int step = group * 4 + (lane & 3);
        step = step < p.steps ? step : p.steps - 1;
        const uint32_t at = lds0 + 2 * STAGE + (group & 1) * SCALES;
        if (k < QW) dma4((vsw[k] + step * 4) & live, wsbase, at + (wave * QW + k) * 256);
        else dma4((vsa[k - QW] + step * 4) & live, asbase, at + BN * 16 + (wave * QA + k - QW) * 256);
    };
    // fragment reads
    const uint8_t* wrow = smem + (wn * NT * 16 + r) * 128;
    const uint8_t* arow = smem + (BN + wm * MT * 16 + r) * 128;
    const int c0 = (g ^ (r & 7)) * 16, c1 = ((4 + g) ^ (r & 7)) * 16;
    auto frag_w = [&](int j, int buf, int ks) { return *reinterpret_cast<const u32x4*>(wrow + buf * STAGE + j * 2048 + (ks ? c1 : c0)); };
    auto frag_a = [&](int i, int buf, int ks) { return *reinterpret_cast<const u32x4*>(arow + buf * STAGE + i * 2048 + (ks ? c1 : c0)); };
    const uint32_t pick = (uint32_t)g | (uint32_t)(4 + g) << 8;
    auto gather = [&](int row, int group) {   // byte s = scale of step s, block g; zero behind the last step
        const u32x4 d = *reinterpret_cast<const u32x4*>(smem + 2 * STAGE + (group & 1) * SCALES + row * 16);
        const uint32_t lo = __builtin_amdgcn_perm(d[1], d[0], pick), hi = __builtin_amdgcn_perm(d[3], d[2], pick);
        const int left = p.steps - group * 4;
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u) & (left >= 4 ? 0xffffffffu : left > 0 ? (1u << (8 * left)) - 1 : 0u);
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 fw[2][NT], fa[2][MT];
    uint32_t sw[NT], sa[MT];

#pragma unroll
    for (int k = 0; k < QW + QA; ++k) dma_scale(k, 0, ~0u);
#pragma unroll
    for (int k = 0; k < PW + PA; ++k) dma_code(k, 0, 0, ~0u);
#pragma unroll
    for (int k = 0; k < PW + PA; ++k) dma_code(k, 1, 1, ~0u);
    hand_over();
#pragma unroll
    for (int j = 0; j < NT; ++j) { sw[j] = gather(wn * NT * 16 + 16 * j + r, 0); fw[0][j] = frag_w(j, 0, 0); }
#pragma unroll
    for (int i = 0; i < MT; ++i) { sa[i] = gather(BN + wm * MT * 16 + 16 * i + r, 0); fa[0][i] = frag_a(i, 0, 0); }
    settle(sw);
    settle(sa);
    settle_acc<MT, NT>(acc);

    // one phase: MT row groups of NT MFMAs; the reads of the next step in the first half of them, DMA pieces spread over all
#define PHASE(OP, CUR, NBUF, NKS, DMA)                                                                                         \
    _Pragma("unroll") for (int i = 0; i < MT; ++i) {                                                                           \
        if (i < MT / 2) {                                                                                                      \
            _Pragma("unroll") for (int t = i * (MT + NT) / (MT / 2); t < (i + 1) * (MT + NT) / (MT / 2); ++t) {                \
                if (t < NT) fw[1 - CUR][t] = frag_w(t, NBUF, NKS);                                                             \
                else fa[1 - CUR][t - NT] = frag_a(t - NT, NBUF, NKS);                                                          \
            }                                                                                                                  \
        }                                                                                                                      \
        DMA;                                                                                                                   \
        _Pragma("unroll") for (int j = 0; j < NT; ++j) mfma_fp4_step<OP>(fw[CUR][j], fa[CUR][i], acc[j][i], sw[j], sa[i]); \
        __builtin_amdgcn_sched_barrier(0);                                                                                     \
    }
#define CODES(STAGE_, BUF) _Pragma("unroll") for (int k = i * (PW + PA) / MT; k < (i + 1) * (PW + PA) / MT; ++k) dma_code(k, STAGE_, BUF, live);
#define SCALE _Pragma("unroll") for (int k = i * (QW + QA) / MT; k < (i + 1) * (QW + QA) / MT; ++k) dma_scale(k, q + 1, live);
    for (int q = 0; q < groups; ++q) {   // one body without a branch: behind the last group the requests all go to the operands' first bytes
        const uint32_t live = q + 1 < groups ? 0xffffffffu : 0u;
        PHASE(0, 0, 0, 1, )
        hand_over();
        PHASE(1, 1, 1, 0, CODES(2 * q + 2, 0) SCALE)
        PHASE(2, 0, 1, 1, )
        hand_over();
        PHASE(3, 1, 0, 0, CODES(2 * q + 3, 1))
#pragma unroll
        for (int j = 0; j < NT; ++j) sw[j] = gather(wn * NT * 16 + 16 * j + r, q + 1);
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = gather(BN + wm * MT * 16 + 16 * i + r, q + 1);
        settle(sw);
        settle(sa);
    }
#undef PHASE
#undef CODES
#undef SCALE
    drain<MT, NT>(acc);
    hand_over();   // everybody has left the stages: their LDS becomes the epilogue's
    store_tile<MT, NT, VEC>(p, acc, reinterpret_cast<float*>(smem) + wave * (16 * (NT * 16 + 4)), m0 + wm * MT * 16, n0 + wn * NT * 16, lane);
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

template <int BM, int BN, int PER_CU>
int launch_tile(hipStream_t stream, const Mxfp4Gemm& p) {
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    if (tn * tm >= (1 << 24)) return 1;
    constexpr int LDS = 2 * (BM + BN) * (128 + 16);
    const dim3 grid((unsigned)(tn * tm)), block(256);
    const bool vec = four_columns(p);
    const void* fn = vec ? (const void*)mxfp4_gemm_tile_kernel<BM, BN, true, PER_CU> : (const void*)mxfp4_gemm_tile_kernel<BM, BN, false, PER_CU>;
    if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return 2;
    if (vec) mxfp4_gemm_tile_kernel<BM, BN, true, PER_CU><<<grid, block, LDS, stream>>>(p, (int)tm, (int)tn, 6);
    else mxfp4_gemm_tile_kernel<BM, BN, false, PER_CU><<<grid, block, LDS, stream>>>(p, (int)tm, (int)tn, 6);
    return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // namespace

int launch_mxfp4_gemm(hipStream_t stream, const Mxfp4Gemm& p) {
    if (p.a_scales && p.K < (1 << 24)) {
        if (p.M > 128 && (int64_t)p.M * p.N >= (int64_t)256 * 256 * 200) return launch_tile<256, 256, 1>(stream, p);
        if (p.M > 32) return launch_tile<128, 128, 2>(stream, p);
    }
    if (p.a_scales) return launch_rows<true, false, 2, 2>(stream, p);
    const bool avec = reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && p.lda % 8 == 0;
    return avec ? launch_rows<false, true, 2, 2>(stream, p) : launch_rows<false, false, 2, 2>(stream, p);
}
