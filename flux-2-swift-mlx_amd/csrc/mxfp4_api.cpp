// mxfp4_api.cpp — C ABI of the MXFP4 operators and of the residual norm: argument checks, then one launch on the context's stream.
// None of them allocates, synchronises or keeps anything between calls.
#include <stdint.h>

#include "common.h"
#include "mxfp4.h"

namespace {

constexpr int64_t MAX_COLS = (int64_t)1 << 30;
constexpr int64_t MAX_ROWS = (int64_t)1 << 40;

// The launches go to the context's GPU whatever the thread's current device is, which is as it was when the call returns.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

bool is_aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int elem_bytes(int dtype) { return dtype == FLUX2MI_F32 ? 4 : dtype == FLUX2MI_BF16 || dtype == FLUX2MI_F16 ? 2 : 0; }

// the memory of a [rows, cols] matrix of row stride ld (elements of esz bytes)
struct Range { uintptr_t lo, hi, pitch, width; };
Range range_of(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t esz) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    if (!p || rows <= 0 || cols <= 0) return Range{lo, lo, 0, 0};
    uintptr_t hi;   // (no sizes wrap around: such a matrix reaches to the end of memory)
    if (__builtin_mul_overflow((uintptr_t)(rows - 1), (uintptr_t)ld, &hi) || __builtin_add_overflow(hi, (uintptr_t)cols, &hi) ||
        __builtin_mul_overflow(hi, (uintptr_t)esz, &hi) || __builtin_add_overflow(lo, hi, &hi))
        hi = UINTPTR_MAX;
    return Range{lo, hi, (uintptr_t)ld * (uintptr_t)esz, (uintptr_t)cols * (uintptr_t)esz};
}
// Column slices of one buffer (equal pitch) reach into each other's range without sharing an element.
bool overlap(const Range& a, const Range& b) {
    if (a.lo >= b.hi || b.lo >= a.hi) return false;
    if (a.pitch != b.pitch || a.width > a.pitch || b.width > a.pitch) return true;
    const uintptr_t d = b.lo > a.lo ? (b.lo - a.lo) % a.pitch : (a.pitch - (a.lo - b.lo) % a.pitch) % a.pitch;   // b's first column in a's rows
    return d < a.width || d + b.width > a.pitch;
}
Range codes_of(const void* p, int64_t rows, int64_t cols) { const int64_t row = mxfp4_padded((int)cols) / 2; return range_of(p, rows, row, row, 1); }
Range scales_of(const void* p, int64_t rows, int64_t cols) { const int64_t row = mxfp4_padded((int)cols) / 32; return range_of(p, rows, row, row, 1); }
// rows * (padded columns / values_per_byte), 0 for sizes that are none or do not fit 63 bits
int64_t matrix_bytes(int64_t rows, int64_t cols, int values_per_byte) {
    int64_t bytes;
    if (rows < 0 || rows > MAX_ROWS || cols < 1 || cols > MAX_COLS || __builtin_mul_overflow(rows, (int64_t)(mxfp4_padded((int)cols) / values_per_byte), &bytes)) return 0;
    return bytes;
}

int check_matrix(const char* who, const char* name, const uint8_t* codes, const uint8_t* scales) {
    F2_REQUIRE(codes && scales, FLUX2MI_ERR_INVALID_ARG, "%s: %s is NULL", who, name);
    F2_REQUIRE(is_aligned(codes, 16) && is_aligned(scales, 4), FLUX2MI_ERR_INVALID_ARG, "%s: %s: codes must be 16-byte, scales 4-byte aligned", who, name);
    return FLUX2MI_OK;
}

int run_gemm(const char* who, flux2mi_ctx* ctx, Mxfp4Gemm p, int out_dtype) {
    F2_REQUIRE(ctx, FLUX2MI_ERR_INVALID_ARG, "%s: NULL ctx", who);
    F2_REQUIRE(p.M >= 0 && p.N >= 0 && p.K >= 1 && p.K <= MAX_COLS, FLUX2MI_ERR_SHAPE, "%s: M %d, N %d, K %d", who, p.M, p.N, p.K);
    F2_REQUIRE(out_dtype == FLUX2MI_F32 || out_dtype == FLUX2MI_BF16, FLUX2MI_ERR_INVALID_ARG, "%s: out_dtype %d (f32 or bf16)", who, out_dtype);
    F2_REQUIRE(!p.resid || out_dtype == FLUX2MI_F32, FLUX2MI_ERR_INVALID_ARG, "%s: a residual needs an f32 output", who);
    if (p.M == 0 || p.N == 0) return FLUX2MI_OK;
    F2_REQUIRE(p.a && p.out, FLUX2MI_ERR_INVALID_ARG, "%s: NULL operand", who);
    F2_TRY(check_matrix(who, "W", p.w, p.w_scales));
    p.out_bf16 = out_dtype == FLUX2MI_BF16;
    const int oe = p.out_bf16 ? 2 : 4;
    F2_REQUIRE(p.ld_out >= p.N && (!p.resid || p.ld_resid >= p.N), FLUX2MI_ERR_SHAPE, "%s: row stride %lld of out / %lld of resid, N %d", who,
               (long long)p.ld_out, (long long)p.ld_resid, p.N);
    F2_REQUIRE(is_aligned(p.out, oe) && is_aligned(p.bias, 4) && is_aligned(p.gate, 4) && is_aligned(p.resid, 4), FLUX2MI_ERR_INVALID_ARG,
               "%s: a pointer is not aligned to its element", who);
    const Range out = range_of(p.out, p.M, p.N, p.ld_out, oe);
    const Range in[] = {p.a_scales ? codes_of(p.a, p.M, p.K) : range_of(p.a, p.M, p.K, p.lda, 2), scales_of(p.a_scales, p.a_scales ? p.M : 0, p.K),
                        codes_of(p.w, p.N, p.K), scales_of(p.w_scales, p.N, p.K), range_of(p.bias, 1, p.N, 0, 4), range_of(p.gate, 1, p.N, 0, 4)};
    for (const Range& r : in) F2_REQUIRE(!overlap(out, r), FLUX2MI_ERR_INVALID_ARG, "%s: out overlaps an operand", who);
    const bool in_place = p.resid == p.out && p.ld_resid == p.ld_out;   // each element is read and written by one lane
    F2_REQUIRE(in_place || !overlap(out, range_of(p.resid, p.M, p.N, p.ld_resid, 4)), FLUX2MI_ERR_INVALID_ARG,
               "%s: out overlaps resid without being the same matrix", who);
    p.steps = mxfp4_padded(p.K) / 128;
    DeviceScope scope(ctx->device);
    F2_CHECK_HIP(scope.err);
    prof_before(ctx, PROF_DIT_GEMM);
    const int r = launch_mxfp4_gemm(ctx->stream, p);
    prof_after(ctx, PROF_DIT_GEMM, 2.0 * p.M * (double)p.N * p.K);
    F2_LAUNCH(r, who);
    return FLUX2MI_OK;
}

}  // namespace

extern "C" int64_t flux2mi_mxfp4_code_bytes(int64_t rows, int64_t cols) { return matrix_bytes(rows, cols, 2); }
extern "C" int64_t flux2mi_mxfp4_scale_bytes(int64_t rows, int64_t cols) { return matrix_bytes(rows, cols, 32); }

extern "C" int flux2mi_op_quantize_mxfp4(flux2mi_ctx* ctx, const void* x, int dtype, int64_t ldx, int64_t rows, int64_t cols, uint8_t* codes,
                                         uint8_t* scales) {
    const int esz = elem_bytes(dtype);
    F2_REQUIRE(ctx, FLUX2MI_ERR_INVALID_ARG, "op_quantize_mxfp4: NULL ctx");
    F2_REQUIRE(esz, FLUX2MI_ERR_INVALID_ARG, "op_quantize_mxfp4: dtype %d", dtype);
    F2_REQUIRE(rows >= 0 && rows <= MAX_ROWS && cols >= 1 && cols <= MAX_COLS && ldx >= cols, FLUX2MI_ERR_SHAPE,
               "op_quantize_mxfp4: rows %lld, cols %lld, row stride %lld", (long long)rows, (long long)cols, (long long)ldx);
    if (rows == 0) return FLUX2MI_OK;
    F2_REQUIRE(x && is_aligned(x, esz), FLUX2MI_ERR_INVALID_ARG, "op_quantize_mxfp4: x is NULL or not aligned to its element");
    F2_TRY(check_matrix("op_quantize_mxfp4", "the result", codes, scales));
    const Range in = range_of(x, rows, cols, ldx, esz), c = codes_of(codes, rows, cols), s = scales_of(scales, rows, cols);
    F2_REQUIRE(!overlap(in, c) && !overlap(in, s) && !overlap(c, s), FLUX2MI_ERR_INVALID_ARG, "op_quantize_mxfp4: buffers overlap");
    DeviceScope scope(ctx->device);
    F2_CHECK_HIP(scope.err);
    F2_LAUNCH(launch_quantize_mxfp4(ctx->stream, x, dtype, ldx, rows, (int)cols, codes, scales), "op_quantize_mxfp4");
    return FLUX2MI_OK;
}

extern "C" int flux2mi_op_dequantize_mxfp4(flux2mi_ctx* ctx, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* y,
                                           int dtype, int64_t ldy) {
    const int esz = elem_bytes(dtype);
    F2_REQUIRE(ctx, FLUX2MI_ERR_INVALID_ARG, "op_dequantize_mxfp4: NULL ctx");
    F2_REQUIRE(esz, FLUX2MI_ERR_INVALID_ARG, "op_dequantize_mxfp4: dtype %d", dtype);
    F2_REQUIRE(rows >= 0 && rows <= MAX_ROWS && cols >= 1 && cols <= MAX_COLS && ldy >= cols, FLUX2MI_ERR_SHAPE,
               "op_dequantize_mxfp4: rows %lld, cols %lld, row stride %lld", (long long)rows, (long long)cols, (long long)ldy);
    if (rows == 0) return FLUX2MI_OK;
    F2_REQUIRE(y && is_aligned(y, esz), FLUX2MI_ERR_INVALID_ARG, "op_dequantize_mxfp4: y is NULL or not aligned to its element");
    F2_TRY(check_matrix("op_dequantize_mxfp4", "the matrix", codes, scales));
    const Range out = range_of(y, rows, cols, ldy, esz);
    F2_REQUIRE(!overlap(out, codes_of(codes, rows, cols)) && !overlap(out, scales_of(scales, rows, cols)), FLUX2MI_ERR_INVALID_ARG,
               "op_dequantize_mxfp4: buffers overlap");
    DeviceScope scope(ctx->device);
    F2_CHECK_HIP(scope.err);
    F2_LAUNCH(launch_dequantize_mxfp4(ctx->stream, codes, scales, rows, (int)cols, y, dtype, ldy), "op_dequantize_mxfp4");
    return FLUX2MI_OK;
}

extern "C" int flux2mi_op_gemm_mxfp4(flux2mi_ctx* ctx, const uint8_t* a, const uint8_t* a_scales, const uint8_t* w, const uint8_t* w_scales,
                                     const float* bias, const float* gate, const float* resid, int64_t ld_resid, void* out, int out_dtype,
                                     int64_t ld_out, int M, int N, int K) {
    if (M > 0 && N > 0) F2_TRY(check_matrix("op_gemm_mxfp4", "A", a, a_scales));
    Mxfp4Gemm p{a, a_scales, 0, w, w_scales, bias, gate, resid, ld_resid, out, ld_out, 0, M, N, K, 0};
    return run_gemm("op_gemm_mxfp4", ctx, p, out_dtype);
}

extern "C" int flux2mi_op_gemm_bf16_mxfp4(flux2mi_ctx* ctx, const void* a, int64_t lda, const uint8_t* w, const uint8_t* w_scales,
                                          const float* bias, const float* gate, const float* resid, int64_t ld_resid, void* out,
                                          int out_dtype, int64_t ld_out, int M, int N, int K) {
    F2_REQUIRE(M <= 0 || lda >= K, FLUX2MI_ERR_SHAPE, "op_gemm_bf16_mxfp4: row stride %lld of A, K %d", (long long)lda, K);
    F2_REQUIRE(is_aligned(a, 2), FLUX2MI_ERR_INVALID_ARG, "op_gemm_bf16_mxfp4: A is not aligned to its element");
    Mxfp4Gemm p{a, nullptr, lda, w, w_scales, bias, gate, resid, ld_resid, out, ld_out, 0, M, N, K, 0};
    return run_gemm("op_gemm_bf16_mxfp4", ctx, p, out_dtype);
}

extern "C" int flux2mi_op_residual_norm(flux2mi_ctx* ctx, const flux2mi_residual_norm* q) {
    const char* who = "op_residual_norm";
    F2_REQUIRE(ctx && q, FLUX2MI_ERR_INVALID_ARG, "%s: NULL argument", who);
    F2_REQUIRE(q->rows >= 0 && q->rows < (1 << 24) && q->dim >= 1 && q->dim <= RESIDUAL_NORM_MAX_DIM, FLUX2MI_ERR_SHAPE,
               "%s: rows %d (< 2^24), dim %d (<= %d)", who, q->rows, q->dim, RESIDUAL_NORM_MAX_DIM);
    auto kind_ok = [](int k) { return k == FLUX2MI_NORM_NONE || k == FLUX2MI_NORM_RMS || k == FLUX2MI_NORM_LAYER; };
    F2_REQUIRE(kind_ok(q->post_norm) && kind_ok(q->norm), FLUX2MI_ERR_INVALID_ARG, "%s: norm kinds %d, %d", who, q->post_norm, q->norm);
    F2_REQUIRE((q->y_dtype == FLUX2MI_F32 || q->y_dtype == FLUX2MI_BF16) && (q->out_dtype == FLUX2MI_F32 || q->out_dtype == FLUX2MI_BF16),
               FLUX2MI_ERR_INVALID_ARG, "%s: y_dtype %d, out_dtype %d (f32 or bf16)", who, q->y_dtype, q->out_dtype);
    F2_REQUIRE(q->post_eps >= 0.f && q->eps >= 0.f, FLUX2MI_ERR_INVALID_ARG, "%s: negative or NaN eps", who);
    if (q->rows == 0) return FLUX2MI_OK;
    F2_REQUIRE(q->y || (q->post_norm == FLUX2MI_NORM_NONE && !q->post_weight && !q->gate[0] && !q->gate[1]), FLUX2MI_ERR_INVALID_ARG,
               "%s: a norm, weight or gate of y without y", who);
    F2_REQUIRE(q->out || (q->norm == FLUX2MI_NORM_NONE && !q->weight && !q->scale[0] && !q->scale[1] && !q->shift[0] && !q->shift[1]),
               FLUX2MI_ERR_INVALID_ARG, "%s: a norm, weight or modulation of out without out", who);
    F2_REQUIRE(q->x && (q->x_out || q->out), FLUX2MI_ERR_INVALID_ARG, "%s: x, or both x_out and out, are NULL", who);
    const int ye = elem_bytes(q->y_dtype), oe = elem_bytes(q->out_dtype);
    F2_REQUIRE(q->ldx >= q->dim && (!q->y || q->ldy >= q->dim) && (!q->x_out || q->ldx_out >= q->dim) && (!q->out || q->ldo >= q->dim), FLUX2MI_ERR_SHAPE,
               "%s: a row stride is below dim %d", who, q->dim);
    bool al = is_aligned(q->x, 4) && is_aligned(q->y, ye) && is_aligned(q->x_out, 4) && is_aligned(q->out, oe) && is_aligned(q->post_weight, 2) &&
              is_aligned(q->weight, 2);
    for (int i = 0; i < 2; ++i) al = al && is_aligned(q->gate[i], 4) && is_aligned(q->scale[i], 4) && is_aligned(q->shift[i], 4);
    F2_REQUIRE(al, FLUX2MI_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element", who);
    // a row is read whole before it is written, by one workgroup: x_out may be x itself; any other overlap would cross rows
    const Range x = range_of(q->x, q->rows, q->dim, q->ldx, 4), y = range_of(q->y, q->rows, q->dim, q->ldy, ye);
    const Range xo = range_of(q->x_out, q->rows, q->dim, q->ldx_out, 4), o = range_of(q->out, q->rows, q->dim, q->ldo, oe);
    F2_REQUIRE((q->x_out == q->x && q->ldx_out == q->ldx) || !overlap(xo, x), FLUX2MI_ERR_INVALID_ARG, "%s: x_out overlaps x without being x", who);
    bool over = overlap(xo, y) || overlap(xo, o) || overlap(o, x) || overlap(o, y);
    const void* vec[] = {q->gate[0], q->gate[1], q->scale[0], q->scale[1], q->shift[0], q->shift[1]};
    for (const void* v : vec) over = over || overlap(xo, range_of(v, 1, q->dim, 0, 4)) || overlap(o, range_of(v, 1, q->dim, 0, 4));
    const void* wts[] = {q->post_weight, q->weight};
    for (const void* v : wts) over = over || overlap(xo, range_of(v, 1, q->dim, 0, 2)) || overlap(o, range_of(v, 1, q->dim, 0, 2));
    F2_REQUIRE(!over, FLUX2MI_ERR_INVALID_ARG, "%s: an output overlaps another buffer", who);
    ResidualNorm p{};
    p.x = q->x; p.ldx = q->ldx; p.y = q->y; p.ldy = q->ldy; p.y_bf16 = q->y_dtype == FLUX2MI_BF16;
    p.x_out = q->x_out; p.ldx_out = q->ldx_out; p.out = q->out; p.ldo = q->ldo; p.out_bf16 = q->out_dtype == FLUX2MI_BF16;
    p.rows = q->rows; p.dim = q->dim; p.split = q->split;
    p.post = q->post_norm; p.pre = q->norm; p.post_eps = q->post_eps; p.eps = q->eps; p.resid_scale = q->resid_scale;
    p.post_w = reinterpret_cast<const uint16_t*>(q->post_weight);
    p.w = reinterpret_cast<const uint16_t*>(q->weight);
    for (int i = 0; i < 2; ++i) { p.gate[i] = q->gate[i]; p.scale[i] = q->scale[i]; p.shift[i] = q->shift[i]; }
    DeviceScope scope(ctx->device);
    F2_CHECK_HIP(scope.err);
    F2_LAUNCH(launch_residual_norm(ctx->stream, p), who);
    return FLUX2MI_OK;
}
