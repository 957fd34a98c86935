// 8-bit linear layer: rows to int8 with a scale each, the integer product with token and channel scales, and the
// straight-through gradients.
//
//   q[r][k] = nearest(127 x[r][k] / a_r), s_r = a_r / 127, a_r = max_k |x[r][k]|
//   y[m][n] = (sum_k qa[m][k] qb[n][k]) sa[m] sb[n] + bias[n]            sum exact in int32
//   dx[m][k] = sum_n (g[m][n] sb[n]) qb[n][k]     dw[n][k] = sum_m (g[m][n] sa[m]) qa[m][k]     db[n] = sum_m g[m][n]
//
// The gradients run on the bfloat16 matrix instructions: an int8 value is exact in bfloat16, and the float32 factor
// g * s is split into bfloat16 pieces whose sum it is (8 bits each: three pieces hold all 24 bits and serve float32
// results, two hold 16 and serve 16-bit results, whose own rounding is far coarser), so nothing but the float32
// accumulation is rounded.  Pieces and transposed operands are laid out in the workspace first, which makes both
// gradients the same product of two row-major operands as the forward pass.
#include <stdlib.h>

#include "few_rows.h"
#include "profile.h"
#include "quant8.h"
#include "tile_product.h"

namespace rexsc {
namespace {

constexpr int MAX_K = 131071; // 128 * 128 * K < 2^31

// ---- rows to 8 bits ------------------------------------------------------------------------------
// Bound by memory: x is read once.  A row lives in the registers of TPR threads (a wave, or a block of 256 or 1024), 16
// elements a thread at most, all its loads in flight together; rows longer than 16384 are read twice.
constexpr int Q_EPT = 16;

struct QuantArgs {
    const void *x;
    int8_t *q;
    float *scale;
    size_t rows, x_stride, q_stride;
    int cols;
};

// Largest magnitude of a row over its TPR threads.
template <int TPR>
__device__ __forceinline__ unsigned row_top(unsigned t, unsigned (&lds)[16])
{
    t = wave_max(t);
    if constexpr (TPR > 64) {
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = t;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 64; i++) t = max(t, lds[i]);
    }
    return t;
}

template <typename T, int V, int TPR>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void quantize_rows_kernel(QuantArgs p)
{
    constexpr int NV = Q_EPT / V;
    typedef typename VecOf<T, V>::type vec;
    __shared__ unsigned lds[16];
    const int tid = TPR == 64 ? threadIdx.x % 64 : threadIdx.x;
    const size_t row = TPR == 64 ? (size_t)blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
    if (row >= p.rows) return; // TPR 64 only: a whole wave
    const T *src = (const T *)p.x + row * p.x_stride;
    vec v[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * TPR + tid) * V;
        v[i] = c < p.cols ? *(const vec *)(src + c) : vec{};
    }
    float x[NV][V];
    unsigned t = 0;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            if constexpr (V == 1) x[i][j] = (float)v[i];
            else x[i][j] = (float)v[i][j];
            t = max(t, mag_bits(x[i][j]));
        }
    const RowScale rs = row_scale(row_top<TPR>(t, lds));
    int8_t *dst = p.q + row * p.q_stride;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * TPR + tid) * V;
        if (c < p.cols) {
            typename VecOf<int8_t, V>::type q;
            if constexpr (V == 1) q = (int8_t)quant8(x[i][0], rs);
            else
#pragma unroll
                for (int j = 0; j < V; j++) q[j] = (int8_t)quant8(x[i][j], rs);
            *(typename VecOf<int8_t, V>::type *)(dst + c) = q;
        }
    }
    for (size_t c = (size_t)p.cols + tid; c < p.q_stride; c += TPR) dst[c] = 0;
    if (tid == 0) p.scale[row] = rs.scale;
}

template <typename T>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(QuantArgs p)
{
    __shared__ unsigned lds[16];
    const T *src = (const T *)p.x + blockIdx.x * p.x_stride;
    unsigned t = 0;
    for (int c = threadIdx.x; c < p.cols; c += 1024) t = max(t, mag_bits((float)src[c]));
    const RowScale rs = row_scale(row_top<1024>(t, lds));
    int8_t *dst = p.q + blockIdx.x * p.q_stride;
    for (size_t c = threadIdx.x; c < p.q_stride; c += 1024) dst[c] = c < (size_t)p.cols ? (int8_t)quant8((float)src[c], rs) : (int8_t)0;
    if (threadIdx.x == 0) p.scale[blockIdx.x] = rs.scale;
}

template <typename T, int V>
void launch_quantize_v(const QuantArgs &p, hipStream_t s)
{
    const unsigned rows = (unsigned)p.rows;
    if (p.cols <= 64 * Q_EPT) hipLaunchKernelGGL((quantize_rows_kernel<T, V, 64>), dim3((rows + 3) / 4), dim3(256), 0, s, p);
    else if (p.cols <= 256 * Q_EPT) hipLaunchKernelGGL((quantize_rows_kernel<T, V, 256>), dim3(rows), dim3(256), 0, s, p);
    else if (p.cols <= 1024 * Q_EPT) hipLaunchKernelGGL((quantize_rows_kernel<T, V, 1024>), dim3(rows), dim3(1024), 0, s, p);
    else hipLaunchKernelGGL(quantize_long_rows_kernel<T>, dim3(rows), dim3(1024), 0, s, p);
}

// Vectors of 16 bytes where every row of x starts on one (and its int8 row, a multiple of 16 bytes, on V).
template <typename T>
void launch_quantize_t(const QuantArgs &p, hipStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool aligned = (uintptr_t)p.x % 16 == 0 && p.cols % V == 0 && (p.x_stride % V == 0 || p.rows == 1);
    if (aligned) launch_quantize_v<T, V>(p, s);
    else launch_quantize_v<T, 1>(p, s);
}

// ---- operands of the gradients ---------------------------------------------------------------------
// v = sum of `pieces` bfloat16 values.  Each but the last keeps the leading 8 bits (truncated, so that nothing
// overflows), the last is rounded.  Of an infinity or NaN the first piece is all.
__device__ __forceinline__ void split(float v, int pieces, bf16_t (&out)[3])
{
    const bool finite = mag_bits(v) < 0x7f800000u;
#pragma unroll
    for (int i = 0; i < 3; i++) {
        if (i >= pieces) break;
        if (!finite) { out[i] = i == 0 ? (bf16_t)v : (bf16_t)0.f; continue; }
        if (i + 1 == pieces) { out[i] = (bf16_t)v; break; }
        const float head = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
        out[i] = (bf16_t)head;
        v -= head;
    }
}

// g [rows][cols] -> out [pieces][rows][ld], elements times scale[column], columns from cols to ld zero.
template <typename T>
__global__ __launch_bounds__(256) void split_rows_kernel(const T *g, const float *scale, int cols, int ld, int pieces, bf16_t *out)
{
    const size_t row = blockIdx.x, rows = gridDim.x;
    for (int c = threadIdx.x; c < ld; c += 256) {
        bf16_t q[3];
        split(c < cols ? (float)g[row * cols + c] * scale[c] : 0.f, pieces, q);
        for (int i = 0; i < pieces; i++) out[(i * rows + row) * ld + c] = q[i];
    }
}

// g [rows][cols] -> out [pieces][cols][ld], elements times scale[row], positions from rows to ld zero; and the sums of
// g's columns over this block's 64 rows to part[row block][cols].  out NULL: only the sums.
template <typename T>
__global__ __launch_bounds__(256) void split_transposed_kernel(const T *g, const float *scale, int rows, int cols, int ld,
                                                               int pieces, bf16_t *out, float *part)
{
    __shared__ float tile[64][65];
    const int row_blocks = ld / 64;
    const int r0 = (int)(blockIdx.x % row_blocks) * 64, c0 = (int)(blockIdx.x / row_blocks) * 64;
    const int tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    for (int i = ty; i < 64; i += 4) {
        const int r = r0 + i, c = c0 + tx;
        tile[i][tx] = r < rows && c < cols ? (float)g[(size_t)r * cols + c] : 0.f;
    }
    __syncthreads();
    if (part && ty == 0 && c0 + tx < cols) {
        float s = 0.f;
        for (int i = 0; i < 64; i++) s += tile[i][tx];
        part[(size_t)(r0 / 64) * cols + c0 + tx] = s;
    }
    if (!out) return;
    const float sc = r0 + tx < rows ? scale[r0 + tx] : 0.f;
    for (int i = ty; i < 64; i += 4) {
        if (c0 + i >= cols) break;
        bf16_t q[3];
        split(r0 + tx < rows ? tile[tx][i] * sc : 0.f, pieces, q);
        for (int j = 0; j < pieces; j++) out[((size_t)j * cols + c0 + i) * ld + r0 + tx] = q[j];
    }
}

// q [rows][cols] int8 -> out [cols][ld] bfloat16, positions from rows to ld zero.
__global__ __launch_bounds__(256) void transpose_i8_kernel(const int8_t *q, size_t stride, int rows, int cols, int ld, bf16_t *out)
{
    __shared__ int8_t tile[64][68];
    const int row_blocks = ld / 64;
    const int r0 = (int)(blockIdx.x % row_blocks) * 64, c0 = (int)(blockIdx.x / row_blocks) * 64;
    const int tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    for (int i = ty; i < 64; i += 4) {
        const int r = r0 + i, c = c0 + tx;
        tile[i][tx] = r < rows && c < cols ? q[(size_t)r * stride + c] : (int8_t)0;
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        if (c0 + i >= cols) break;
        out[(size_t)(c0 + i) * ld + r0 + tx] = (bf16_t)(float)tile[tx][i];
    }
}

// ---- host ------------------------------------------------------------------------------------------
int check_int8(const rexsc_int8_desc *d)
{
    REXSC_CHECK_DESC(d, rexsc_int8_desc);
    REXSC_CHECK_ARG(d->M >= 0 && d->N >= 0, "int8 linear: M %d, N %d", d->M, d->N);
    REXSC_CHECK_ARG(d->K >= 1 && d->K <= MAX_K, "int8 linear: K must be 1..%d, so that the int32 sum cannot overflow (got %d)",
                    MAX_K, d->K);
    REXSC_CHECK_ARG(dtype_ok(d->dtype) && dtype_ok(d->bias_dtype) && dtype_ok(d->weight_dtype),
                    "int8 linear: dtypes %d, %d, %d: each must be float32, float16 or bfloat16", d->dtype, d->bias_dtype,
                    d->weight_dtype);
    REXSC_CHECK_ARG(d->reserved == 0, "int8 linear: reserved field is %d, not 0", d->reserved);
    return REXSC_OK;
}

int check_rows8(const char *what, const void *q, int64_t stride, int K)
{
    REXSC_CHECK_ARG(q != nullptr, "null pointer");
    REXSC_CHECK_ARG((uintptr_t)q % 16 == 0 && stride % 16 == 0 && stride >= K,
                    "int8 linear: the %s' int8 rows must be 16-byte aligned at a distance that is a multiple of 16 and at least "
                    "K = %d (distance %lld)", what, K, (long long)stride);
    return REXSC_OK;
}

inline int64_t pad64(int64_t n) { return (n + 63) / 64 * 64; }
inline int pieces_of(int dtype) { return dtype == REXSC_F32 ? 3 : 2; }

struct Space { size_t tokens, scales, pieces, transposed, part, product, total; };

Space space(const rexsc_int8_desc *d, int what)
{
    Space s{};
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at = align_up(at + bytes, 256); return o; };
    const size_t M = d->M, N = d->N, K = d->K;
    if (what == REXSC_INT8_PRODUCT) {
        s.product = take(tile_product_workspace(d->M, d->N, d->K, 1));
    } else if (what == REXSC_INT8_LINEAR) {
        s.product = take(tile_product_workspace(d->M, d->N, d->K, 1));
        s.tokens = take(M * align_up(K, 128));
        s.scales = take(M * 4);
    } else if (what == REXSC_INT8_GRAD_INPUT) {
        const size_t ld = pad64(N);
        s.product = take(tile_product_workspace(d->M, d->K, (int)ld * 2, pieces_of(d->dtype)));
        s.pieces = take(M * ld * pieces_of(d->dtype) * 2);
        s.transposed = take(K * ld * 2);
    } else if (what == REXSC_INT8_GRAD_WEIGHT) {
        const size_t ld = pad64(M);
        s.product = take(tile_product_workspace(d->N, d->K, (int)ld * 2, pieces_of(d->weight_dtype)));
        s.pieces = take(N * ld * pieces_of(d->weight_dtype) * 2);
        s.transposed = take(K * ld * 2);
        s.part = take(ld / 64 * N * 4);
    }
    s.total = at;
    return s;
}

int check_space(const Space &s, const void *workspace, size_t bytes)
{
    if (s.total && (!workspace || bytes < s.total)) {
        set_error("int8 linear: workspace of %zu bytes needed, %zu given", s.total, workspace ? bytes : (size_t)0);
        return REXSC_ERR_WORKSPACE;
    }
    REXSC_CHECK_ARG((uintptr_t)workspace % 16 == 0, "int8 linear: the workspace must be 16-byte aligned");
    return REXSC_OK;
}

int product(const rexsc_int8_desc *d, const int8_t *a, int64_t a_stride, const float *a_scale, const int8_t *b,
            const float *b_scale, const void *bias, void *y, void *space, hipStream_t stream)
{
    const TileArgs p{(const char *)a, (const char *)b, (size_t)a_stride, (size_t)d->b_stride, d->M, d->N, d->K, 1, 0,
                     a_scale, b_scale, bias, d->bias_dtype, y};
    if (few_rows_takes(d->M, d->N) && !getenv("REXSC_TUNE_INT8_TILE")) return launch_few_rows(p, d->dtype, stream);
    return launch_tile_product(p, false, d->dtype, space, "int8_product", stream);
}

int launch_quantize(const void *x, int dtype, size_t rows, size_t cols, size_t x_stride, int8_t *q, size_t q_stride,
                    float *scale, hipStream_t stream)
{
    ProfScope prof("quantize_rows", (double)rows * cols * (dtype_size(dtype) + 1), stream);
    const QuantArgs p{x, q, scale, rows, x_stride, q_stride, (int)cols};
    REXSC_DTYPE_SWITCH(dtype, launch_quantize_t<T>(p, stream));
    REXSC_CHECK_HIP(hipGetLastError());
    return REXSC_OK;
}

} // namespace
} // namespace rexsc

using namespace rexsc;

extern "C" int rexsc_quantize_rows(const void *x, int dtype, size_t rows, size_t cols, size_t x_stride, int8_t *q,
                                   size_t q_stride, float *scale, rexsc_stream_t stream)
{
    REXSC_CHECK_ARG(dtype_ok(dtype), "quantize_rows: dtype %d is not one of float32, float16, bfloat16", dtype);
    REXSC_CHECK_ARG(cols >= 1 && cols < (1u << 30) && rows < (1ull << 31), "quantize_rows: %zu rows of %zu elements", rows, cols);
    if (rows == 0) return REXSC_OK;
    REXSC_CHECK_ARG(x && q && scale, "null pointer");
    REXSC_CHECK_ARG((uintptr_t)x % dtype_size(dtype) == 0, "quantize_rows: x is not aligned to its element");
    REXSC_CHECK_ARG((uintptr_t)q % 16 == 0 && q_stride % 16 == 0 && q_stride >= cols,
                    "quantize_rows: the int8 rows must be 16-byte aligned at a distance that is a multiple of 16 and at least "
                    "%zu (distance %zu)", cols, q_stride);
    return launch_quantize(x, dtype, rows, cols, x_stride, q, q_stride, scale, (hipStream_t)stream);
}

extern "C" size_t rexsc_int8_workspace_bytes(const rexsc_int8_desc *d, int what)
{
    if (check_int8(d)) return (size_t)-1;
    if (what < REXSC_INT8_PRODUCT || what > REXSC_INT8_GRAD_WEIGHT) {
        set_error("int8 linear: no call has the number %d", what);
        return (size_t)-1;
    }
    return space(d, what).total;
}

extern "C" int rexsc_int8_product(const rexsc_int8_desc *d, const int8_t *a, const float *a_scale, const int8_t *b,
                                  const float *b_scale, const void *bias, void *y, void *workspace, size_t workspace_bytes,
                                  rexsc_stream_t stream)
{
    if (int rc = check_int8(d)) return rc;
    if (d->M == 0 || d->N == 0) return REXSC_OK;
    if (int rc = check_rows8("tokens", a, d->a_stride, d->K)) return rc;
    if (int rc = check_rows8("channels", b, d->b_stride, d->K)) return rc;
    REXSC_CHECK_ARG(a_scale && b_scale && y, "null pointer");
    const Space s = space(d, REXSC_INT8_PRODUCT);
    if (int rc = check_space(s, workspace, workspace_bytes)) return rc;
    return product(d, a, d->a_stride, a_scale, b, b_scale, bias, y, (char *)workspace + s.product, (hipStream_t)stream);
}

extern "C" int rexsc_int8_linear(const rexsc_int8_desc *d, const void *x, const int8_t *b, const float *b_scale,
                                 const void *bias, void *y, void *workspace, size_t workspace_bytes, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_int8(d)) return rc;
    if (d->M == 0 || d->N == 0) return REXSC_OK;
    if (int rc = check_rows8("channels", b, d->b_stride, d->K)) return rc;
    REXSC_CHECK_ARG(x && b_scale && y, "null pointer");
    REXSC_CHECK_ARG((uintptr_t)x % dtype_size(d->dtype) == 0 && (d->x_stride >= d->K || d->M == 1),
                    "int8 linear: x is not aligned to its element, or its rows overlap (distance %lld)", (long long)d->x_stride);
    const Space s = space(d, REXSC_INT8_LINEAR);
    if (int rc = check_space(s, workspace, workspace_bytes)) return rc;
    if (few_rows_fuses(d->M, d->K, x, (size_t)d->x_stride, d->dtype)) {
        const TileArgs p{nullptr, (const char *)b, 0, (size_t)d->b_stride, d->M, d->N, d->K, 1, 0, nullptr, b_scale, bias,
                         d->bias_dtype, y};
        return launch_few_rows_fused(p, x, (size_t)d->x_stride, d->dtype, stream);
    }
    int8_t *q = (int8_t *)workspace + s.tokens;
    float *scale = (float *)((char *)workspace + s.scales);
    const size_t stride = align_up(d->K, 128);
    if (int rc = launch_quantize(x, d->dtype, d->M, d->K, d->x_stride, q, stride, scale, stream)) return rc;
    return product(d, q, (int64_t)stride, scale, b, b_scale, bias, y, (char *)workspace + s.product, stream);
}

extern "C" int rexsc_int8_grad_input(const rexsc_int8_desc *d, const void *g, const int8_t *b, const float *b_scale, void *dx,
                                     void *workspace, size_t workspace_bytes, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_int8(d)) return rc;
    if (d->M == 0) return REXSC_OK;
    REXSC_CHECK_ARG(d->N >= 1, "int8 linear: a gradient needs at least one output channel");
    if (int rc = check_rows8("channels", b, d->b_stride, d->K)) return rc;
    REXSC_CHECK_ARG(g && b_scale && dx, "null pointer");
    const Space s = space(d, REXSC_INT8_GRAD_INPUT);
    if (int rc = check_space(s, workspace, workspace_bytes)) return rc;
    bf16_t *pieces = (bf16_t *)((char *)workspace + s.pieces), *bt = (bf16_t *)((char *)workspace + s.transposed);
    const int P = pieces_of(d->dtype), ld = (int)pad64(d->N);
    {
        ProfScope prof("int8_grad_operands", (double)d->M * d->N * (dtype_size(d->dtype) + 2.0 * P), stream);
        REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(split_rows_kernel<T>, dim3((unsigned)d->M), dim3(256), 0, stream,
                                                        (const T *)g, b_scale, d->N, ld, P, pieces));
        REXSC_CHECK_HIP(hipGetLastError());
    }
    {
        ProfScope prof("int8_grad_operands", 3.0 * d->N * d->K, stream);
        hipLaunchKernelGGL(transpose_i8_kernel, dim3((unsigned)((ld / 64) * ((d->K + 63) / 64))), dim3(256), 0, stream, b,
                           (size_t)d->b_stride, d->N, d->K, ld, bt);
        REXSC_CHECK_HIP(hipGetLastError());
    }
    const TileArgs p{(const char *)pieces, (const char *)bt, (size_t)ld * 2, (size_t)ld * 2, d->M, d->K, ld * 2, P,
                     (size_t)d->M * ld * 2, nullptr, nullptr, nullptr, REXSC_F32, dx};
    return launch_tile_product(p, true, d->dtype, (char *)workspace + s.product, "int8_grad_input", stream);
}

extern "C" int rexsc_int8_grad_weight(const rexsc_int8_desc *d, const void *g, const int8_t *a, const float *a_scale, void *dw,
                                      void *db, void *workspace, size_t workspace_bytes, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_int8(d)) return rc;
    if (d->N == 0 || (!dw && !db)) return REXSC_OK;
    const Space s = space(d, REXSC_INT8_GRAD_WEIGHT);
    if (d->M > 0) {
        if (dw)
            if (int rc = check_rows8("tokens", a, d->a_stride, d->K)) return rc;
        REXSC_CHECK_ARG(g && (a_scale || !dw), "null pointer");
        if (int rc = check_space(s, workspace, workspace_bytes)) return rc;
    }
    bf16_t *pieces = (bf16_t *)((char *)workspace + s.pieces), *at = (bf16_t *)((char *)workspace + s.transposed);
    float *part = (float *)((char *)workspace + s.part);
    const int P = pieces_of(d->weight_dtype), ld = (int)pad64(d->M);
    if (d->M > 0) {
        ProfScope prof("int8_grad_operands", (double)d->M * d->N * (dtype_size(d->dtype) + (dw ? 2.0 * P : 0)), stream);
        REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(split_transposed_kernel<T>,
                                                        dim3((unsigned)((ld / 64) * ((d->N + 63) / 64))), dim3(256), 0, stream,
                                                        (const T *)g, a_scale, d->M, d->N, ld, P, dw ? pieces : nullptr,
                                                        db ? part : nullptr));
        REXSC_CHECK_HIP(hipGetLastError());
    }
    if (db)
        if (int rc = launch_column_sums(part, (size_t)ld / 64, d->N, d->N, db, d->bias_dtype, stream)) return rc;
    if (!dw) return REXSC_OK;
    if (d->M > 0) {
        ProfScope prof("int8_grad_operands", 3.0 * d->M * d->K, stream);
        hipLaunchKernelGGL(transpose_i8_kernel, dim3((unsigned)((ld / 64) * ((d->K + 63) / 64))), dim3(256), 0, stream, a,
                           (size_t)d->a_stride, d->M, d->K, ld, at);
        REXSC_CHECK_HIP(hipGetLastError());
    }
    // without tokens the reduction is empty and the kernel writes zeros
    const TileArgs p{(const char *)pieces, (const char *)at, (size_t)ld * 2, (size_t)ld * 2, d->N, d->K, ld * 2, P,
                     (size_t)d->N * ld * 2, nullptr, nullptr, nullptr, REXSC_F32, dw};
    return launch_tile_product(p, true, d->weight_dtype, (char *)workspace + s.product, "int8_grad_weight", stream);
}
