// rows_api.hip -- host layer of the rows operators (include/speech_hip.h, speech_rows_*): argument checks and launches.
// Every check is made before a device is touched, so that a refused call does nothing.
#include "rows_internal.hpp"
#include <cmath>

namespace speech {
namespace {

#define HIP_TRY(fn, expr)                                                                         \
    do {                                                                                          \
        hipError_t e_ = (expr);                                                                   \
        if (e_ != hipSuccess) { return fail(fn, "HIP call failed: %s (%s)", #expr, hipGetErrorString(e_)); } \
    } while (0)

// the caller's device, back in place when the call returns
struct OnDevice {
    int prev; bool ok;
    explicit OnDevice(int dev) : prev(-1), ok(true)
    {
        int cur = -1;
        if (hipGetDevice(&cur) == hipSuccess && cur == dev) { return; }
        ok = hipSetDevice(dev) == hipSuccess;
        if (ok) { prev = cur; }
    }
    ~OnDevice() { if (prev >= 0) { (void)hipSetDevice(prev); } }
};

const size_t MAX_COLS = (size_t)1 << 30, MAX_ROWS = (size_t)1 << 40, MAX_GRID = ((size_t)1 << 31) - 1;

size_t elem_of(int dtype) { return dtype == SPEECH_F64 ? 8u : dtype == SPEECH_F32 ? 4u : 2u; }
bool is_type(int dtype) { return dtype == SPEECH_F32 || dtype == SPEECH_BF16 || dtype == SPEECH_F16; }

int check_sizes(const char *fn, size_t rows, size_t cols)
{
    if (cols > MAX_COLS) { return fail(fn, "%zu columns: at most 2^30 are supported", cols); }
    if (rows > MAX_ROWS) { return fail(fn, "%zu rows: at most 2^40 are supported", rows); }
    return 0;
}

// a matrix argument: its row stride, its alignment to its elements
int check_rows(const char *fn, const char *what, const void *p, size_t ld, size_t cols, size_t elem)
{
    if (!p) { return fail(fn, "null device pointer %s", what); }
    if (ld < cols) { return fail(fn, "row stride of %s is %zu, below its %zu columns", what, ld, cols); }
    if (ld > MAX_ROWS) { return fail(fn, "row stride of %s is too large", what); }
    if ((uintptr_t)p % elem) { return fail(fn, "%s is not aligned to its elements", what); }
    return 0;
}

int check_held(const char *fn, const char *what, const void *q, size_t ldq, const void *s, size_t lds, size_t cols)
{
    const size_t nb = (cols + ROWS_BLOCK - 1) / ROWS_BLOCK;
    if (!q || !s) { return fail(fn, "null device pointer %s", what); }
    if (ldq < cols || ldq > MAX_ROWS || ldq % 16 || (uintptr_t)q % 16) { return fail(fn, "8-bit rows of %s must start on 16 bytes, %zu columns apart at least", what, cols); }
    if (lds < nb || lds > MAX_ROWS || lds % 4 || (uintptr_t)s % 4) { return fail(fn, "rows of scales of %s must start on 4 bytes, %zu scales apart at least", what, nb); }
    return 0;
}

int check_drop(const char *fn, const speech_drop *d, DropParams *out)
{
    *out = DropParams{0, 0u, 1.0, 0ull, nullptr, nullptr};
    if (!d) { return 0; }
    if (!(d->p >= 0.0 && d->p < 1.0)) { return fail(fn, "p (probability of dropping) must be in [0 1)"); }
    if (d->p == 0.0) { return 0; }
    out->on = 1;
    out->thresh = (uint32_t)std::floor(d->p * 4294967296.0);
    out->scale = 1.0 / (1.0 - d->p);
    out->seed = d->seed; out->step = d->step; out->keys = d->keys;
    return 0;
}

// an output that may be this input: the very same matrix, or no byte in common
bool overlaps(const void *a, size_t lda, size_t ea, const void *b, size_t ldb, size_t eb, size_t rows, size_t cols)
{
    if (!a || !b || rows == 0) { return false; }
    const uintptr_t a0 = (uintptr_t)a, a1 = a0 + ((rows - 1) * lda + cols) * ea, b0 = (uintptr_t)b, b1 = b0 + ((rows - 1) * ldb + cols) * eb;
    return a0 < b1 && b0 < a1;
}
// Matrices of one allocation may interleave (column ranges of a wider matrix): with one row stride that is no overlap when neither
// reaches into the other's columns.
bool clash(const void *a, size_t lda, const void *b, size_t ldb, size_t elem, size_t rows, size_t cols, bool same_is_fine)
{
    if (!overlaps(a, lda, elem, b, ldb, elem, rows, cols)) { return false; }
    if (a == b && (lda == ldb || rows == 1)) { return !same_is_fine; }
    if (lda != ldb) { return true; }
    const size_t d = ((uintptr_t)a > (uintptr_t)b ? (uintptr_t)a - (uintptr_t)b : (uintptr_t)b - (uintptr_t)a), pitch = lda * elem;
    const size_t r = d % pitch;
    return r < cols * elem || pitch - r < cols * elem;
}

}  // namespace
}  // namespace speech

using namespace speech;

extern "C" {

int speech_rows_dropout(int device, int dtype, size_t rows, size_t cols, const void *X, size_t ldx, void *Y, size_t ldy,
                        const speech_drop *drop, void *stream)
{
    const char *fn = "speech_rows_dropout";
    DropParams d;
    if (!is_type(dtype) && dtype != SPEECH_F64) { return fail(fn, "unknown dtype %d", dtype); }
    if (!drop) { return fail(fn, "null drop"); }
    if (check_sizes(fn, rows, cols) || check_drop(fn, drop, &d)) { return 1; }
    if (rows == 0 || cols == 0) { return 0; }
    const size_t e = elem_of(dtype);
    if (check_rows(fn, "X", X, ldx, cols, e) || check_rows(fn, "Y", Y, ldy, cols, e)) { return 1; }
    if (clash(Y, ldy, X, ldx, e, rows, cols, true)) { return fail(fn, "Y overlaps X without being X"); }
    OnDevice g(device);
    if (!g.ok) { return fail(fn, "cannot select device %d", device); }
    HIP_TRY(fn, launch_rows_dropout(dtype, rows, (int)cols, X, ldx, Y, ldy, d, (hipStream_t)stream));
    return 0;
}

int speech_rows_rms_norm(int device, const speech_norm *a, void *stream)
{
    const char *fn = "speech_rows_rms_norm";
    if (!a) { return fail(fn, "null args"); }
    if (!is_type(a->dtype)) { return fail(fn, "unknown dtype %d", a->dtype); }
    if (a->cols < 1) { return fail(fn, "cols must be positive"); }
    if (!(a->eps > 0.0 && (float)a->eps > 0.0f && std::isfinite(a->eps))) { return fail(fn, "eps must be positive"); }
    if (!a->Y && !a->Q) { return fail(fn, "no output: neither Y nor Q"); }
    NormParams p;
    if (check_sizes(fn, a->rows, a->cols) || check_drop(fn, a->drop, &p.drop)) { return 1; }
    if (a->rows == 0) { return 0; }
    const size_t e = elem_of(a->dtype), R = a->rows, C = a->cols;
    if (check_rows(fn, "X", a->X, a->ldx, C, e)) { return 1; }
    if (a->R && check_rows(fn, "R", a->R, a->ldr, C, e)) { return 1; }
    if (a->H && check_rows(fn, "H", a->H, a->ldh, C, e)) { return 1; }
    if (a->Y && check_rows(fn, "Y", a->Y, a->ldy, C, e)) { return 1; }
    if (a->Q && check_held(fn, "Q", a->Q, a->ldq, a->S, a->lds, C)) { return 1; }
    if ((uintptr_t)a->weight % (a->weight_f32 ? 4u : e)) { return fail(fn, "weight is not aligned to its elements"); }
    if (clash(a->H, a->ldh, a->X, a->ldx, e, R, C, true) || clash(a->H, a->ldh, a->R, a->ldr, e, R, C, true)) { return fail(fn, "H overlaps X or R without being it"); }
    if (clash(a->Y, a->ldy, a->X, a->ldx, e, R, C, true) || clash(a->Y, a->ldy, a->R, a->ldr, e, R, C, true)) { return fail(fn, "Y overlaps X or R without being it"); }
    if (clash(a->Y, a->ldy, a->H, a->ldh, e, R, C, false)) { return fail(fn, "Y overlaps H"); }
    OnDevice g(device);
    if (!g.ok) { return fail(fn, "cannot select device %d", device); }
    p.rows = R; p.cols = (int)C; p.weight_f32 = a->weight_f32; p.eps = (float)a->eps;
    p.X = a->X; p.R = a->R; p.weight = a->weight; p.H = a->H; p.Y = a->Y;
    p.ldx = a->ldx; p.ldr = a->ldr; p.ldh = a->ldh; p.ldy = a->ldy;
    p.Q = a->Q; p.S = a->S; p.ldq = a->ldq; p.lds = a->lds; p.rstd = a->rstd;
    HIP_TRY(fn, launch_rows_norm(a->dtype, p, (hipStream_t)stream));
    return 0;
}

int speech_rows_rms_norm_work(size_t rows, size_t cols, size_t *bytes)
{
    const char *fn = "speech_rows_rms_norm_work";
    if (!bytes) { return fail(fn, "null pointer"); }
    if (check_sizes(fn, rows, cols)) { return 1; }
    *bytes = (rows < (size_t)ROWS_GRAD_MAX_WG ? rows : (size_t)ROWS_GRAD_MAX_WG) * cols * sizeof(float);
    return 0;
}

int speech_rows_rms_norm_backward(int device, const speech_norm_grad *a, void *stream)
{
    const char *fn = "speech_rows_rms_norm_backward";
    if (!a) { return fail(fn, "null args"); }
    if (!is_type(a->dtype)) { return fail(fn, "unknown dtype %d", a->dtype); }
    if (a->cols < 1) { return fail(fn, "cols must be positive"); }
    if (!a->dH && !a->dX && !a->dW) { return fail(fn, "no output: neither dH nor dX nor dW"); }
    NormGradParams p;
    if (check_sizes(fn, a->rows, a->cols) || check_drop(fn, a->drop, &p.drop)) { return 1; }
    const size_t e = elem_of(a->dtype), R = a->rows, C = a->cols;
    if (R > 0)
    {
        size_t need = 0;
        if (check_rows(fn, "dY", a->dY, a->lddy, C, e) || check_rows(fn, "H", a->H, a->ldh, C, e)) { return 1; }
        if (!a->rstd) { return fail(fn, "null device pointer rstd"); }
        if (a->dR && check_rows(fn, "dR", a->dR, a->lddr, C, e)) { return 1; }
        if (a->dH && check_rows(fn, "dH", a->dH, a->lddh, C, e)) { return 1; }
        if (a->dX && check_rows(fn, "dX", a->dX, a->lddx, C, e)) { return 1; }
        if ((uintptr_t)a->weight % (a->weight_f32 ? 4u : e)) { return fail(fn, "weight is not aligned to its elements"); }
        if (speech_rows_rms_norm_work(R, C, &need)) { return 1; }
        if (a->dW && (!a->work || a->work_bytes < need || (uintptr_t)a->work % 16)) { return fail(fn, "dW needs a work array of %zu bytes on 16 bytes", need); }
        if (clash(a->dH, a->lddh, a->dY, a->lddy, e, R, C, true) || clash(a->dH, a->lddh, a->dR, a->lddr, e, R, C, true)) { return fail(fn, "dH overlaps dY or dR without being it"); }
        if (clash(a->dX, a->lddx, a->dY, a->lddy, e, R, C, true) || clash(a->dX, a->lddx, a->dR, a->lddr, e, R, C, true)) { return fail(fn, "dX overlaps dY or dR without being it"); }
        if (clash(a->dX, a->lddx, a->dH, a->lddh, e, R, C, false)) { return fail(fn, "dX overlaps dH"); }
        if (clash(a->dX, a->lddx, a->H, a->ldh, e, R, C, false) || clash(a->dH, a->lddh, a->H, a->ldh, e, R, C, false)) { return fail(fn, "dH or dX overlaps H"); }
    }
    else if (!a->dW) { return 0; }
    OnDevice g(device);
    if (!g.ok) { return fail(fn, "cannot select device %d", device); }
    p.rows = R; p.cols = (int)C; p.weight_f32 = a->weight_f32;
    p.dY = a->dY; p.H = a->H; p.dR = a->dR; p.weight = a->weight; p.rstd = a->rstd; p.dH = a->dH; p.dX = a->dX;
    p.lddy = a->lddy; p.ldh = a->ldh; p.lddr = a->lddr; p.lddh = a->lddh; p.lddx = a->lddx;
    p.dW = a->dW; p.work = (float *)a->work;
    HIP_TRY(fn, launch_rows_norm_grad(a->dtype, p, (hipStream_t)stream));
    return 0;
}

int speech_rows_quantize(int device, int dtype, size_t rows, size_t cols, const void *X, size_t ldx, unsigned char *Q, size_t ldq,
                         unsigned char *S, size_t lds, int transpose, void *stream)
{
    const char *fn = "speech_rows_quantize";
    if (!is_type(dtype)) { return fail(fn, "unknown dtype %d", dtype); }
    if (check_sizes(fn, rows, cols)) { return 1; }
    if (rows == 0 || cols == 0) { return 0; }
    if (transpose && rows > MAX_COLS) { return fail(fn, "%zu rows to transpose: at most 2^30 are supported", rows); }
    if (check_rows(fn, "X", X, ldx, cols, elem_of(dtype)) || check_held(fn, "Q", Q, ldq, S, lds, transpose ? rows : cols)) { return 1; }
    if (transpose && ((rows + ROWS_BLOCK - 1) / ROWS_BLOCK) * ((cols + 31) / 32) > MAX_GRID) { return fail(fn, "matrix too large"); }
    OnDevice g(device);
    if (!g.ok) { return fail(fn, "cannot select device %d", device); }
    HIP_TRY(fn, launch_rows_quantize(dtype, rows, cols, X, ldx, Q, ldq, S, lds, transpose, (hipStream_t)stream));
    return 0;
}

int speech_rows_product_work(size_t rows, size_t cols, size_t k, size_t *bytes)
{
    const char *fn = "speech_rows_product_work";
    if (!bytes) { return fail(fn, "null pointer bytes"); }
    if (check_sizes(fn, rows, cols) || check_sizes(fn, rows, k)) { return 1; }
    *bytes = rows && cols ? rows_product_work(rows, cols, k) : 0;
    return 0;
}

int speech_rows_product(int device, int dtype, size_t rows, size_t cols, size_t k, const unsigned char *A, size_t lda,
                        const unsigned char *SA, size_t ldsa, const unsigned char *B, size_t ldb, const unsigned char *SB, size_t ldsb,
                        const float *bias, void *Y, size_t ldy, void *work, size_t work_bytes, void *stream)
{
    const char *fn = "speech_rows_product";
    if (dtype != SPEECH_BF16 && dtype != SPEECH_F16) { return fail(fn, "dtype %d: the result has 16 bits (bf16 or f16)", dtype); }
    if (check_sizes(fn, rows, cols) || check_sizes(fn, rows, k)) { return 1; }
    if (rows == 0 || cols == 0) { return 0; }
    if (k > 0 && (check_held(fn, "A", A, lda, SA, ldsa, k) || check_held(fn, "B", B, ldb, SB, ldsb, k))) { return 1; }
    if (check_rows(fn, "Y", Y, ldy, cols, elem_of(dtype))) { return 1; }
    if ((uintptr_t)bias % 4u) { return fail(fn, "bias is not aligned to its elements"); }
    if (((rows + 15) / 16) * ((cols + 15) / 16) > MAX_GRID) { return fail(fn, "matrix too large"); }
    if ((uintptr_t)work % 16u) { return fail(fn, "work must start on 16 bytes"); }
    OnDevice g(device);
    if (!g.ok) { return fail(fn, "cannot select device %d", device); }
    const ProductParams p{rows, cols, k, A, SA, B, SB, lda, ldsa, ldb, ldsb, bias, Y, ldy, (float *)work, work ? work_bytes : 0, 0};
    HIP_TRY(fn, launch_rows_product(dtype, p, (hipStream_t)stream));
    return 0;
}

}  // extern "C"
