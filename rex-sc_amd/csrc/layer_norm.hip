// Layer norm, forward and backward, and the column sums of partial weight gradients.
//
//   y  = (x - mu) r w + b,     mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = r (gw - mean(gw) - h mean(gw h)),  gw = g w, h = (x - mu) r;   dw = sum_rows g h;   db = sum_rows g
//
// Bound by memory: forward reads x and writes y, backward reads x and g and writes dx, each once.  A row lives in the
// registers of TPR threads (16 lanes, a wave, or a block of 128 to 1024), so the variance is taken around the true mean
// without a second read.  Blocks are persistent over rows: w and b (forward), w and the two gradient sums (backward)
// stay in registers from row to row, since re-reading float32 w and b from L2 for every 16-bit row would move more bytes
// than the row itself.  The next row is loaded before the current one is reduced (where registers allow).
// Rows longer than 16384 elements take the streaming kernels, which read the row again for each pass (from L2).
// Measured: 16384 x 8192 bfloat16 forward 99 us (5.4 TB/s), backward 184 + 8 us for the sums (4.4 TB/s of x, g and dx);
// 524288 x 128 forward 50 us (5.4), backward 88 us; a copy of 1 GiB reaches 5.1 TB/s.
#include "lowp.h"
#include "profile.h"

namespace rexsc {
namespace {

constexpr int LONGEST = 1024 * 16;  // row that is held in registers
constexpr int STREAM_THREADS = 1024;

struct NormParams {
    const void *x, *w, *b, *g;
    void *y, *dx;
    float *mean, *rstd, *part;      // part: [blocks][2][cols]
    size_t rows, x_stride;
    int cols, w_dtype;
    float eps;
};

// Sum over the TPR threads of a row, the result in all of them.  `slot` alternates between calls (0, 1), so that one
// barrier per call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*lds)[TPR / 64 + 1][N], int slot)
{
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int s = (TPR < 64 ? TPR : 64) / 2; s; s >>= 1) v[i] += __shfl_xor(v[i], s, 64);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int i = 0; i < N; i++) lds[slot][wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < TPR / 64; k++) s += lds[slot][k][i];
            v[i] = s;
        }
    }
}

template <typename T, int V, int NV, int TPR>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void norm_forward_kernel(NormParams p)
{
    constexpr int RPB = TPR <= 64 ? 256 / TPR : 1; // rows a block holds at once
    typedef typename VecOf<T, V>::type vec;
    __shared__ float lds[2][TPR / 64 + 1][1];
    const int tid = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
    const int sub = TPR <= 64 ? threadIdx.x / TPR : 0;
    const float inv = 1.0f / (float)p.cols;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int c = (i * TPR + tid) * V + j;
            w[i][j] = p.w && c < p.cols ? load_any(p.w, p.w_dtype, c) : 1.f;
            b[i][j] = p.b && c < p.cols ? load_any(p.b, p.w_dtype, c) : 0.f;
        }
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + sub;
    vec cur[NV];
    auto fetch = [&](size_t r) {
        const T *src = (const T *)p.x + r * p.x_stride;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + tid) * V;
            cur[i] = c < p.cols ? *(const vec *)(src + c) : vec{};
        }
    };
    if (row < p.rows) fetch(row);
    for (; row < p.rows; row += step) {
        float x[NV][V];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if constexpr (V == 1) x[i][0] = (float)cur[i];
            else
#pragma unroll
                for (int j = 0; j < V; j++) x[i][j] = (float)cur[i][j];
        }
        if (row + step < p.rows) fetch(row + step);
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < V; j++) s[0] += x[i][j];
        row_sum<TPR, 1>(s, lds, 0);
        const float mu = s[0] * inv;
        float q[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                x[i][j] = (i * TPR + tid) * V < p.cols ? x[i][j] - mu : 0.f;
                q[0] = fmaf(x[i][j], x[i][j], q[0]);
            }
        row_sum<TPR, 1>(q, lds, 1);
        const float r = 1.0f / sqrtf(fmaf(q[0], inv, p.eps));
        T *dst = (T *)p.y + row * (size_t)p.cols;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + tid) * V;
            if (c < p.cols) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; j++) o[j] = fmaf(x[i][j] * r, w[i][j], b[i][j]);
                store_vec<V>(dst + c, o);
            }
        }
        if (tid == 0 && p.mean) {
            p.mean[row] = mu;
            p.rstd[row] = r;
        }
    }
}

// RAGGED: rows begin anywhere and end inside a vector.
template <typename T, int V, int NV, int TPR, bool RAGGED = false>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void norm_backward_kernel(NormParams p)
{
    constexpr int RPB = TPR <= 64 ? 256 / TPR : 1; // rows a block holds at once
    typedef typename VecOf<T, V>::type vec;
    __shared__ float lds[2][TPR / 64 + 1][2];
    const int tid = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
    const int sub = TPR <= 64 ? threadIdx.x / TPR : 0;
    const float inv = 1.0f / (float)p.cols;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int c = (i * TPR + tid) * V + j;
            w[i][j] = p.w && c < p.cols ? load_any(p.w, p.w_dtype, c) : 1.f;
            dw[i][j] = db[i][j] = 0.f;
        }
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + sub;
    vec cx[NV], cg[NV];
    auto fetch = [&](size_t r) {
        const T *sx = (const T *)p.x + r * p.x_stride, *sg = (const T *)p.g + r * (size_t)p.cols;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + tid) * V;
            // the vector that the row's end cuts: one shifted load where there are registers for it (5591 x 12001 bfloat16:
            // 140 us against 152 by elements; with 32 elements a thread 181 against 160, in float32 97 against 93)
            if constexpr (RAGGED && sizeof(T) == 2 && NV * V <= 24) {
                cx[i] = load_some<T, V>(sx + c, p.cols - c, c);
                cg[i] = load_some<T, V>(sg + c, p.cols - c, c);
            } else if constexpr (RAGGED) {
                cx[i] = load_some<T, V>(sx + c, p.cols - c);
                cg[i] = load_some<T, V>(sg + c, p.cols - c);
            } else {
                cx[i] = c < p.cols ? *(const vec *)(sx + c) : vec{};
                cg[i] = c < p.cols ? *(const vec *)(sg + c) : vec{};
            }
        }
    };
    constexpr bool AHEAD = NV * V * (int)sizeof(T) <= 64; // registers for a row in flight beside the current one
    if (AHEAD && row < p.rows) fetch(row);
    int slot = 0;
    for (; row < p.rows; row += step) {
        if (!AHEAD) fetch(row);
        const float mu = p.mean[row], r = p.rstd[row];
        float h[NV][V], gw[NV][V], s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                float xv, gv;
                if constexpr (V == 1) { xv = (float)cx[i]; gv = (float)cg[i]; }
                else { xv = (float)cx[i][j]; gv = (float)cg[i][j]; }
                // beyond the row: g is 0, h must be finite
                h[i][j] = (i * TPR + tid) * V + (RAGGED ? j : 0) < p.cols ? (xv - mu) * r : 0.f;
                dw[i][j] = fmaf(gv, h[i][j], dw[i][j]);
                db[i][j] += gv;
                gw[i][j] = gv * w[i][j];
                s[0] += gw[i][j];
                s[1] = fmaf(gw[i][j], h[i][j], s[1]);
            }
        if (AHEAD && row + step < p.rows) fetch(row + step);
        if (p.dx) {
            row_sum<TPR, 2>(s, lds, slot);
            slot ^= 1;
            const float m0 = s[0] * inv, m1 = s[1] * inv;
            T *dst = (T *)p.dx + row * (size_t)p.cols;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * TPR + tid) * V;
                if (c < p.cols) {
                    float o[V];
#pragma unroll
                    for (int j = 0; j < V; j++) o[j] = r * (gw[i][j] - m0 - h[i][j] * m1);
                    if constexpr (RAGGED) {
                        vec t;
#pragma unroll
                        for (int j = 0; j < V; j++) t[j] = (T)o[j];
                        store_some<T, V>(dst + c, t, p.cols - c);
                    } else {
                        store_vec<V>(dst + c, o);
                    }
                }
            }
        }
    }
    if (!p.part) return;
    float *out = p.part + (size_t)blockIdx.x * 2 * p.cols;
    if constexpr (RPB > 1) {
        // the block's rows hold as many sums of the same columns: joined in their order
        __shared__ float join[RPB - 1][2][TPR * NV * V];
        if (sub > 0)
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    join[sub - 1][0][(i * V + j) * TPR + tid] = dw[i][j];
                    join[sub - 1][1][(i * V + j) * TPR + tid] = db[i][j];
                }
        __syncthreads();
        if (sub > 0) return;
#pragma nounroll
        for (int k = 0; k < RPB - 1; k++)
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    dw[i][j] += join[k][0][(i * V + j) * TPR + tid];
                    db[i][j] += join[k][1][(i * V + j) * TPR + tid];
                }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * TPR + tid) * V;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (c + (RAGGED ? j : 0) < p.cols) {
                out[c + j] = dw[i][j];
                out[p.cols + c + j] = db[i][j];
            }
    }
}

// ---- few short rows ------------------------------------------------------------------------------
// The whole backward pass in one launch: a wave per row for dx, and blocks of 16 columns that take dw and db over all
// rows, 16 groups of them joined in order.  x and g are read three times, but from L2, and a launch, an allocation and the
// partial sums are saved, which is what such a call's time goes to.
constexpr int SMALL_ROWS = 512, SMALL_COLS = 2048;
template <typename T>
__global__ __launch_bounds__(256) void norm_backward_small_kernel(NormParams p, void *dw_out, void *db_out, unsigned row_blocks)
{
    __shared__ float lds[2][16][17];
    const T *const x = (const T *)p.x, *const g = (const T *)p.g;
    if (blockIdx.x < row_blocks) {
        const size_t row = (size_t)blockIdx.x * 4 + threadIdx.x / 64;
        if (row >= p.rows) return;
        const int lane = threadIdx.x % 64;
        const T *sx = x + row * p.x_stride, *sg = g + row * (size_t)p.cols;
        const float mu = p.mean[row], r = p.rstd[row], inv = 1.0f / (float)p.cols;
        float s[2] = {0.f, 0.f};
#pragma unroll 4
        for (int c = lane; c < p.cols; c += 64) {
            const float gw = (float)sg[c] * (p.w ? load_any(p.w, p.w_dtype, c) : 1.f);
            s[0] += gw;
            s[1] = fmaf(gw, ((float)sx[c] - mu) * r, s[1]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int o = 32; o; o >>= 1) s[i] += __shfl_xor(s[i], o, 64);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T *dst = (T *)p.dx + row * (size_t)p.cols;
#pragma unroll 4
        for (int c = lane; c < p.cols; c += 64) {
            const float gw = (float)sg[c] * (p.w ? load_any(p.w, p.w_dtype, c) : 1.f);
            dst[c] = (T)(r * (gw - m0 - ((float)sx[c] - mu) * r * m1));
        }
        return;
    }
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, c = (int)(blockIdx.x - row_blocks) * 16 + tx;
    float dw = 0.f, db = 0.f;
    if (c < p.cols)
#pragma unroll 4
        for (size_t row = ty; row < p.rows; row += 16) {
            const float gv = (float)g[row * (size_t)p.cols + c];
            dw = fmaf(gv, ((float)x[row * p.x_stride + c] - p.mean[row]) * p.rstd[row], dw);
            db += gv;
        }
    lds[0][ty][tx] = dw;
    lds[1][ty][tx] = db;
    __syncthreads();
    if (ty > 1 || c >= p.cols) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) sum += lds[ty][i][tx];
    void *const out = ty ? db_out : dw_out;
    if (out) store_any(out, p.w_dtype, c, sum);
}

// ---- rows of any length --------------------------------------------------------------------------
// By single elements, three reads of x forward and two of x and g backward, with another two for the weight's gradients:
// 4096 x 28672 bfloat16 forward 448 us (1.05 TB/s of x and y once each), backward 959 us (0.73 of x, g and dx); float32
// 554 us (1.7) and 1185 us (1.2).
template <typename T>
__global__ __launch_bounds__(STREAM_THREADS) void norm_forward_stream_kernel(NormParams p)
{
    __shared__ float lds[2][STREAM_THREADS / 64 + 1][1];
    const float inv = 1.0f / (float)p.cols;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *src = (const T *)p.x + row * p.x_stride;
        float s[1] = {0.f};
        for (int c = threadIdx.x; c < p.cols; c += STREAM_THREADS) s[0] += (float)src[c];
        row_sum<STREAM_THREADS, 1>(s, lds, 0);
        const float mu = s[0] * inv;
        float q[1] = {0.f};
        for (int c = threadIdx.x; c < p.cols; c += STREAM_THREADS) {
            const float d = (float)src[c] - mu;
            q[0] = fmaf(d, d, q[0]);
        }
        row_sum<STREAM_THREADS, 1>(q, lds, 1);
        const float r = 1.0f / sqrtf(fmaf(q[0], inv, p.eps));
        T *dst = (T *)p.y + row * (size_t)p.cols;
        for (int c = threadIdx.x; c < p.cols; c += STREAM_THREADS) {
            const float w = p.w ? load_any(p.w, p.w_dtype, c) : 1.f, b = p.b ? load_any(p.b, p.w_dtype, c) : 0.f;
            dst[c] = (T)fmaf(((float)src[c] - mu) * r, w, b);
        }
        if (threadIdx.x == 0 && p.mean) {
            p.mean[row] = mu;
            p.rstd[row] = r;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(STREAM_THREADS) void norm_dx_stream_kernel(NormParams p)
{
    __shared__ float lds[2][STREAM_THREADS / 64 + 1][2];
    const float inv = 1.0f / (float)p.cols;
    int slot = 0;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *sx = (const T *)p.x + row * p.x_stride, *sg = (const T *)p.g + row * (size_t)p.cols;
        const float mu = p.mean[row], r = p.rstd[row];
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < p.cols; c += STREAM_THREADS) {
            const float gw = (float)sg[c] * (p.w ? load_any(p.w, p.w_dtype, c) : 1.f);
            s[0] += gw;
            s[1] = fmaf(gw, ((float)sx[c] - mu) * r, s[1]);
        }
        row_sum<STREAM_THREADS, 2>(s, lds, slot);
        slot ^= 1;
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T *dst = (T *)p.dx + row * (size_t)p.cols;
        for (int c = threadIdx.x; c < p.cols; c += STREAM_THREADS) {
            const float gw = (float)sg[c] * (p.w ? load_any(p.w, p.w_dtype, c) : 1.f);
            dst[c] = (T)(r * (gw - m0 - ((float)sx[c] - mu) * r * m1));
        }
    }
}

// dw and db of 256 columns over a share of the rows: grid (column blocks, row shares).
template <typename T>
__global__ __launch_bounds__(256) void norm_dw_stream_kernel(NormParams p)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.cols) return;
    float dw = 0.f, db = 0.f;
    for (size_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float g = (float)((const T *)p.g)[row * (size_t)p.cols + c];
        const float x = (float)((const T *)p.x)[row * p.x_stride + c];
        dw = fmaf(g, (x - p.mean[row]) * p.rstd[row], dw);
        db += g;
    }
    float *out = p.part + (size_t)blockIdx.y * 2 * p.cols;
    out[c] = dw;
    out[p.cols + c] = db;
}

// ---- column sums -----------------------------------------------------------------------------------
// A block sums 16 columns: 64 row groups, each its rows in turn with eight loads in flight, joined in order.  Columns
// from `cols` on (up to twice as many) go to out2.
constexpr int CS_COLS = 16, CS_GROUPS = 64;
__global__ __launch_bounds__(CS_COLS * CS_GROUPS) void column_sums_kernel(const float *part, size_t rows, size_t cols, size_t ld,
                                                                          void *out, void *out2, int out_dtype)
{
    __shared__ float lds[CS_GROUPS][CS_COLS + 1];
    const int tx = threadIdx.x % CS_COLS, ty = threadIdx.x / CS_COLS;
    void *const dst = blockIdx.y ? out2 : out;
    if (!dst) return;
    for (size_t c0 = (size_t)blockIdx.x * CS_COLS; c0 < cols; c0 += (size_t)gridDim.x * CS_COLS) {
        const size_t c = c0 + tx;
        const float *src = part + (blockIdx.y ? cols : 0) + c;
        float s = 0.f;
        if (c < cols) {
#pragma unroll 8
            for (size_t r = ty; r < rows; r += CS_GROUPS) s += src[r * ld];
        }
        lds[ty][tx] = s;
        __syncthreads();
        for (int half = CS_GROUPS / 2; half > 0; half /= 2) {
            if (ty < half) lds[ty][tx] += lds[ty + half][tx];
            __syncthreads();
        }
        if (ty == 0 && c < cols) store_any(dst, out_dtype, c, lds[0][tx]);
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------
// Waves per CU of the persistent grids.  16384 x 8192 bfloat16: forward 110 us at 16, 142 at 8 and 126 at 32; backward
// with its column sums 186 us at 8, 200 at 16, 229 at 32: more blocks, more partial sums to write and add.
constexpr int FWD_WAVES = 16, BWD_WAVES = 8;

struct NormPlan { int V, NV, TPR, grid; }; // TPR 0: streaming kernels

int check_norm(const rexsc_norm_desc *d)
{
    REXSC_CHECK_DESC(d, rexsc_norm_desc);
    REXSC_CHECK_ARG(dtype_ok(d->dtype), "layer norm: dtype %d is not one of float32, float16, bfloat16", d->dtype);
    REXSC_CHECK_ARG(d->weight_dtype == REXSC_F32 || d->weight_dtype == d->dtype,
                    "layer norm: weight and bias must be float32 or of x's type (codes %d, %d)", d->weight_dtype, d->dtype);
    REXSC_CHECK_ARG(d->rows >= 0 && d->cols >= 1 && d->cols < (1 << 30), "layer norm: %lld rows of %lld elements",
                    (long long)d->rows, (long long)d->cols);
    REXSC_CHECK_ARG(d->x_stride >= d->cols || d->rows <= 1, "layer norm: rows of %lld elements at distance %lld",
                    (long long)d->cols, (long long)d->x_stride);
    REXSC_CHECK_ARG(d->eps >= 0.f, "layer norm: eps must not be negative (got %g)", (double)d->eps);
    return REXSC_OK;
}

// Vectors of 16 bytes where every row starts on one, else single elements (vectors that lie anywhere are slower in 16
// bits: 16388 x 4095 bfloat16 forward 101 us against 60, backward 203 against 102; in float32 the two are alike).
//
// A row is held by the fewest threads that have it at 20 elements each (forward in 16 bits 24): rows of a wave need no
// barrier, and 128 or 256 threads of which a part has nothing still wait for each other.  At 16 elements, bfloat16, the
// width that has just outgrown a wave took twice as long: 64527 x 1040 backward 175 us against 86, 60952 x 1101 214
// against 90, 33537 x 2001 137 against 96, 7281 x 9216 forward 80 against 61.  In float32, with half the elements for
// the same bytes, that gains for a wave only (32263 x 1040 backward 102 us against 85; 16768 x 2001 in 128 threads 89
// against 86 in 256, 6553 x 5120 forward 54 in 256 against 50 in 512), and forward rows of 8193 to 10240 (3727 x 9001
// 60 us in 1024 threads, 53 in 512).
//
// The backward pass holds a row of more than 8192 in 512 threads at 24 or 32 elements: with its five values per element,
// 1024 threads have too few registers (8192 x 16384 bfloat16: 640 us with them spilled, against 178; 5591 x 12001 at 12
// elements 162 against 140).  There single elements need too many as well, and vectors that lie anywhere are taken
// (5591 x 12001 bfloat16: 459 us by single elements).
NormPlan norm_plan(const rexsc_norm_desc *d, bool aligned, bool backward)
{
    NormPlan pl{};
    const bool f32 = d->dtype == REXSC_F32;
    const int VMAX = f32 ? 4 : 8, most = f32 || backward ? 20 : 24;
    pl.V = aligned && d->cols % VMAX == 0 && (d->x_stride % VMAX == 0 || d->rows <= 1) ? VMAX : 1;
    pl.TPR = d->cols <= 16 * 16                        ? 16
             : d->cols <= 64 * most                    ? 64
             : d->cols <= 128 * most && !f32           ? 128
             : d->cols <= 256 * (f32 ? 16 : most)      ? 256
             : d->cols <= 512 * (backward ? 16 : most) ? 512
             : d->cols <= LONGEST                      ? 1024
                                                       : 0;
    const int64_t rpb = pl.TPR && pl.TPR <= 64 ? 256 / pl.TPR : 1;
    const int threads = pl.TPR == 0 ? STREAM_THREADS : pl.TPR <= 64 ? 256 : pl.TPR == 1024 && backward ? 512 : pl.TPR;
    const int64_t full = 256 * (int64_t)(backward ? BWD_WAVES : FWD_WAVES) * 64 / threads, want = (d->rows + rpb - 1) / rpb;
    pl.grid = (int)(want < full ? want : full);
    if (pl.TPR) {
        const int ept = (int)((d->cols + pl.TPR - 1) / pl.TPR);
        pl.NV = pl.V > 1 ? (ept + pl.V - 1) / pl.V : (ept + 3) / 4 * 4;
    }
    return pl;
}

// The numbers of threads per row that come with room for EPT elements in each, see norm_plan.
constexpr bool takes(int tpr, int ept, bool f32)
{
    return tpr == 16     ? ept <= 16
           : tpr == 64   ? ept > 4
           : tpr == 128  ? ept > 8 && !f32
           : tpr == 256  ? ept > 4 && (ept <= 16 || !f32)
           : tpr == 512  ? ept > 8
                         : ept > 8 && ept <= 16;
}
template <typename T, int V, int NV, int TPR>
bool launch_fwd_if(const NormPlan &pl, const NormParams &p, hipStream_t s)
{
    if constexpr (takes(TPR, V * NV, sizeof(T) == 4)) {
        if (pl.TPR != TPR) return false;
        hipLaunchKernelGGL((norm_forward_kernel<T, V, NV, TPR>), dim3(pl.grid), dim3(TPR <= 64 ? 256 : TPR), 0, s, p);
        return true;
    }
    return false;
}
template <typename T, int V, int NV, int TPR>
bool launch_bwd_if(const NormPlan &pl, const NormParams &p, hipStream_t s)
{
    if constexpr (takes(TPR, V * NV, sizeof(T) == 4) && (TPR < 512 || V * NV <= 16)) {
        if (pl.TPR != TPR) return false;
        hipLaunchKernelGGL((norm_backward_kernel<T, V, NV, TPR>), dim3(pl.grid), dim3(TPR <= 64 ? 256 : TPR), 0, s, p);
        return true;
    }
    return false;
}
template <typename T, int V, int NV>
bool launch_fwd_tpr(const NormPlan &pl, const NormParams &p, hipStream_t s)
{
    return launch_fwd_if<T, V, NV, 16>(pl, p, s) || launch_fwd_if<T, V, NV, 64>(pl, p, s) || launch_fwd_if<T, V, NV, 128>(pl, p, s) ||
           launch_fwd_if<T, V, NV, 256>(pl, p, s) || launch_fwd_if<T, V, NV, 512>(pl, p, s) || launch_fwd_if<T, V, NV, 1024>(pl, p, s);
}
template <typename T, int V, int NV>
bool launch_bwd_tpr(const NormPlan &pl, const NormParams &p, hipStream_t s)
{
    return launch_bwd_if<T, V, NV, 16>(pl, p, s) || launch_bwd_if<T, V, NV, 64>(pl, p, s) || launch_bwd_if<T, V, NV, 128>(pl, p, s) ||
           launch_bwd_if<T, V, NV, 256>(pl, p, s) || launch_bwd_if<T, V, NV, 512>(pl, p, s);
}
#define NORM_NV(FN)                                                                         \
    do {                                                                                    \
        if constexpr (sizeof(T) == 4) {                                                     \
            if (pl.V == 4 && pl.NV == 1) return FN<T, 4, 1>(pl, p, s);                      \
            if (pl.V == 4 && pl.NV == 2) return FN<T, 4, 2>(pl, p, s);                      \
            if (pl.V == 4 && pl.NV == 3) return FN<T, 4, 3>(pl, p, s);                      \
            if (pl.V == 4 && pl.NV == 4) return FN<T, 4, 4>(pl, p, s);                      \
            if (pl.V == 4) return FN<T, 4, 5>(pl, p, s);                                    \
        } else {                                                                            \
            if (pl.V == 8 && pl.NV == 1) return FN<T, 8, 1>(pl, p, s);                      \
            if (pl.V == 8 && pl.NV == 2) return FN<T, 8, 2>(pl, p, s);                      \
            if (pl.V == 8) return FN<T, 8, 3>(pl, p, s);                                    \
            if (pl.NV == 24) return FN<T, 1, 24>(pl, p, s);                                 \
        }                                                                                   \
        if (pl.NV == 4) return FN<T, 1, 4>(pl, p, s);                                       \
        if (pl.NV == 8) return FN<T, 1, 8>(pl, p, s);                                       \
        if (pl.NV == 12) return FN<T, 1, 12>(pl, p, s);                                     \
        if (pl.NV == 16) return FN<T, 1, 16>(pl, p, s);                                     \
        return FN<T, 1, 20>(pl, p, s);                                                      \
    } while (0)
template <typename T> bool launch_fwd(const NormPlan &pl, const NormParams &p, hipStream_t s) { NORM_NV(launch_fwd_tpr); }
template <typename T> bool launch_bwd(const NormPlan &pl, const NormParams &p, hipStream_t s)
{
    constexpr int W = 16 / sizeof(T);
    if (pl.TPR < 1024) NORM_NV(launch_bwd_tpr);
    const bool shorter = p.cols <= 512 * 24;
    if (pl.V > 1 && shorter) hipLaunchKernelGGL((norm_backward_kernel<T, W, 24 / W, 512>), dim3(pl.grid), dim3(512), 0, s, p);
    else if (pl.V > 1) hipLaunchKernelGGL((norm_backward_kernel<T, W, 32 / W, 512>), dim3(pl.grid), dim3(512), 0, s, p);
    else if (shorter) hipLaunchKernelGGL((norm_backward_kernel<T, W, 24 / W, 512, true>), dim3(pl.grid), dim3(512), 0, s, p);
    else hipLaunchKernelGGL((norm_backward_kernel<T, W, 32 / W, 512, true>), dim3(pl.grid), dim3(512), 0, s, p);
    return true;
}

bool small_backward(const rexsc_norm_desc *d) { return d->rows <= SMALL_ROWS && d->cols <= SMALL_COLS; }

int bwd_blocks(const rexsc_norm_desc *d)
{
    if (d->cols <= LONGEST) return norm_plan(d, false, true).grid;
    int64_t shares = d->rows < 64 ? d->rows : 64;
    while ((d->cols + 255) / 256 * shares >= 1 << 23) shares /= 2; // a launch has fewer than 2^32 threads
    return (int)shares;
}

bool aligned16(const void *a, const void *b, const void *c)
{
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

} // namespace

int launch_column_sums(const float *part, size_t rows, size_t cols, size_t ld, void *out, void *out2, int out_dtype,
                       hipStream_t stream)
{
    ProfScope prof("column_sums", 4.0 * rows * cols * (out && out2 ? 2 : 1), stream);
    constexpr size_t MOST = 1u << 20; // blocks; a launch has fewer than 2^32 threads
    const size_t blocks = (cols + CS_COLS - 1) / CS_COLS;
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)(blocks < MOST ? blocks : MOST), out2 ? 2 : 1), dim3(CS_COLS * CS_GROUPS), 0,
                       stream, part, rows, cols, ld, out, out2, out_dtype);
    REXSC_CHECK_HIP(hipGetLastError());
    return REXSC_OK;
}

} // namespace rexsc

using namespace rexsc;

extern "C" int rexsc_layer_norm_forward(const rexsc_norm_desc *d, const void *x, const void *weight, const void *bias,
                                        void *y, float *mean, float *rstd, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_norm(d)) return rc;
    if (d->rows == 0) return REXSC_OK;
    REXSC_CHECK_ARG(x && y, "null pointer");
    REXSC_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "layer norm: mean and rstd are given together or not at all");
    const size_t es = dtype_size(d->dtype);
    REXSC_CHECK_ARG((((uintptr_t)x | (uintptr_t)y) % es) == 0, "layer norm: a tensor is not aligned to its element");
    const NormPlan pl = norm_plan(d, aligned16(x, y, nullptr), false);
    const NormParams p{x, weight, bias, nullptr, y, nullptr, mean, rstd, nullptr, (size_t)d->rows, (size_t)d->x_stride,
                       (int)d->cols, d->weight_dtype, d->eps};
    ProfScope prof("layer_norm_forward", 2.0 * es * d->rows * d->cols, stream);
    if (pl.TPR == 0)
        REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(norm_forward_stream_kernel<T>, dim3(pl.grid), dim3(STREAM_THREADS), 0,
                                                        stream, p));
    else
        REXSC_DTYPE_SWITCH(d->dtype, REXSC_CHECK_ARG(launch_fwd<T>(pl, p, stream), "layer norm: no kernel for rows of %d", p.cols));
    REXSC_CHECK_HIP(hipGetLastError());
    return REXSC_OK;
}

extern "C" size_t rexsc_layer_norm_backward_workspace_bytes(const rexsc_norm_desc *d)
{
    if (check_norm(d)) return (size_t)-1;
    if (small_backward(d)) return 0;
    return (size_t)bwd_blocks(d) * 2 * (size_t)d->cols * sizeof(float);
}

extern "C" int rexsc_layer_norm_backward(const rexsc_norm_desc *d, const void *grad_out, const void *x, const void *weight,
                                         const float *mean, const float *rstd, void *dx, void *dw, void *db,
                                         void *workspace, size_t workspace_bytes, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_norm(d)) return rc;
    const size_t es = dtype_size(d->dtype), cols = (size_t)d->cols;
    const bool sums = dw || db;
    if (!dx && !sums) return REXSC_OK;
    if (d->rows == 0) // sums over no rows
        return sums ? launch_column_sums(nullptr, 0, cols, cols, dw, db, d->weight_dtype, stream) : REXSC_OK;
    REXSC_CHECK_ARG(grad_out && x && mean && rstd, "null pointer");
    REXSC_CHECK_ARG((((uintptr_t)x | (uintptr_t)grad_out | (uintptr_t)dx) % es) == 0,
                    "layer norm: a tensor is not aligned to its element");
    if (small_backward(d)) {
        const NormParams p{x, weight, nullptr, grad_out, nullptr, dx, const_cast<float *>(mean), const_cast<float *>(rstd), nullptr,
                           (size_t)d->rows, (size_t)d->x_stride, (int)d->cols, d->weight_dtype, d->eps};
        const unsigned row_blocks = dx ? (unsigned)((d->rows + 3) / 4) : 0, col_blocks = sums ? (unsigned)((cols + 15) / 16) : 0;
        ProfScope prof("layer_norm_backward", (dx ? 3.0 : 2.0) * es * d->rows * d->cols, stream);
        REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(norm_backward_small_kernel<T>, dim3(row_blocks + col_blocks), dim3(256), 0, stream,
                                                        p, dw, db, row_blocks));
        REXSC_CHECK_HIP(hipGetLastError());
        return REXSC_OK;
    }
    const size_t need = rexsc_layer_norm_backward_workspace_bytes(d);
    if (sums && (!workspace || workspace_bytes < need)) {
        set_error("layer norm: workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
        return REXSC_ERR_WORKSPACE;
    }
    const NormPlan pl = norm_plan(d, aligned16(x, grad_out, dx), true);
    const NormParams p{x, weight, nullptr, grad_out, nullptr, dx, const_cast<float *>(mean), const_cast<float *>(rstd),
                       sums ? (float *)workspace : nullptr, (size_t)d->rows, (size_t)d->x_stride, (int)d->cols,
                       d->weight_dtype, d->eps};
    const int blocks = bwd_blocks(d);
    {
        ProfScope prof("layer_norm_backward", (dx ? 3.0 : 2.0) * es * d->rows * d->cols, stream);
        if (pl.TPR == 0) {
            if (dx)
                REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(norm_dx_stream_kernel<T>, dim3(pl.grid), dim3(STREAM_THREADS),
                                                                0, stream, p));
            if (sums)
                REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(norm_dw_stream_kernel<T>,
                                                                dim3((unsigned)((cols + 255) / 256), blocks), dim3(256), 0,
                                                                stream, p));
        } else {
            REXSC_DTYPE_SWITCH(d->dtype, REXSC_CHECK_ARG(launch_bwd<T>(pl, p, stream), "layer norm: no kernel for rows of %d", p.cols));
        }
        REXSC_CHECK_HIP(hipGetLastError());
    }
    return sums ? launch_column_sums((const float *)workspace, blocks, cols, 2 * cols, dw, db, d->weight_dtype, stream) : REXSC_OK;
}
