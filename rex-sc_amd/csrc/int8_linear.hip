// 8-bit linear layer: rows to int8 with a scale each, the integer product with token and channel scales, and the
// straight-through gradients.
//
//   q[r][k] = nearest(127 x[r][k] / a_r), s_r = a_r / 127, a_r = max_k |x[r][k]|
//   y[m][n] = (sum_k qa[m][k] qb[n][k]) sa[m] sb[n] + bias[n]            sum exact in int32
//   dx[m][k] = sum_n (g[m][n] sb[n]) qb[n][k]     dw[n][k] = sum_m (g[m][n] sa[m]) qa[m][k]     db[n] = sum_m g[m][n]
//
// The gradients run on the binary16 matrix instructions: an int8 value is exact in binary16, and the float32 factor
// g * s is taken apart into binary16 pieces.  Pieces and transposed operands are laid out in the workspace first, which
// makes both gradients the same product of two row-major operands as the forward pass.
#include <stdlib.h>

#include <type_traits>

#include "few_rows.h"
#include "profile.h"
#include "quant8.h"
#include "tile_product.h"

namespace rexsc {
namespace {

constexpr int MAX_K = 131071; // 128 * 128 * K < 2^31
constexpr int MAX_ROWS = 2147483647 - 255; // tokens or channels: a tile's rows behind the last one still have numbers

// ---- rows to 8 bits ------------------------------------------------------------------------------
// Bound by memory: x is read once, in vectors of 16 bytes wherever they lie (RAGGED: rows that begin anywhere and end
// inside one).  A row lives in the registers of TPR threads, all its loads in flight together; rows longer than 16384 are
// read twice.  8192 x 4096 bfloat16: 24 us (4.2 TB/s of reads and writes); one row of 4096: 3 us, the launch and one round
// trip to memory.  Single elements take longer where rows are not aligned, most of it for storing single bytes (bfloat16
// 16376 x 4098 193 us against 46, float32 72 against 28).  TPR is the smallest number with at most 24 elements a thread:
// with more threads, of which a part has nothing, all wait for each other (at 16 elements: 43690 x 1536 bfloat16 55 us
// against 35, 13107 x 5120 71 against 34; 65536 x 100 in a wave each 22, in 16 lanes 11).
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
    if constexpr (TPR < 64) {
#pragma unroll
        for (int s = TPR / 2; s; s >>= 1) t = max(t, (unsigned)__shfl_xor((int)t, s, 64));
    } else {
        t = wave_max(t);
    }
    if constexpr (TPR > 64) {
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = t;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 64; i++) t = max(t, lds[i]);
    }
    return t;
}

template <typename T, int NV, int TPR, bool RAGGED>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void quantize_rows_kernel(QuantArgs p)
{
    constexpr int V = 16 / sizeof(T), RPB = TPR <= 64 ? 256 / TPR : 1;
    typedef typename VecOf<T, V>::type vec;
    __shared__ unsigned lds[2][16];
    const int tid = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
    int slot = 0;
    for (size_t row = (size_t)blockIdx.x * RPB + (TPR <= 64 ? threadIdx.x / TPR : 0); row < p.rows; row += (size_t)gridDim.x * RPB) {
        const T *src = (const T *)p.x + row * p.x_stride;
        vec v[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + tid) * V;
            if constexpr (RAGGED) v[i] = load_some<T, V>(src + c, p.cols - c, c);
            else v[i] = c < p.cols ? *(const vec *)(src + c) : vec{};
        }
        float x[NV][V];
        unsigned t = 0;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                x[i][j] = (float)v[i][j];
                t = max(t, mag_bits(x[i][j]));
            }
        const RowScale rs = row_scale(row_top<TPR>(t, lds[slot]));
        slot ^= 1; // one barrier a row
        int8_t *dst = p.q + row * p.q_stride;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + tid) * V;
            if (c < p.cols) {
                typename VecOf<int8_t, V>::type q; // zeros behind the row's end, within its padding
#pragma unroll
                for (int j = 0; j < V; j++) q[j] = (int8_t)quant8(x[i][j], rs);
                *(typename VecOf<int8_t, V>::type *)(dst + c) = q;
            }
        }
        for (size_t c = (size_t)p.cols + tid; c < p.q_stride; c += TPR) dst[c] = 0;
        if (tid == 0) p.scale[row] = rs.scale;
    }
}

// Rows of any length, by single elements: 8192 x 28672 bfloat16 458 us (1.5 TB/s of reading once and writing), float32
// 487 us (2.4); 64 x 131072 bfloat16 55 us, in which 64 blocks are all there are.
template <typename T>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(QuantArgs p)
{
    __shared__ unsigned lds[2][16];
    int slot = 0;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *src = (const T *)p.x + row * p.x_stride;
        unsigned t = 0;
        for (int c = threadIdx.x; c < p.cols; c += 1024) t = max(t, mag_bits((float)src[c]));
        const RowScale rs = row_scale(row_top<1024>(t, lds[slot]));
        slot ^= 1;
        int8_t *dst = p.q + row * p.q_stride;
        for (size_t c = threadIdx.x; c < p.q_stride; c += 1024) dst[c] = c < (size_t)p.cols ? (int8_t)quant8((float)src[c], rs) : (int8_t)0;
        if (threadIdx.x == 0) p.scale[row] = rs.scale;
    }
}

template <typename T, int NV, bool RAGGED>
void launch_quantize_nv(const QuantArgs &p, int tpr, hipStream_t s)
{
    constexpr int EPT = NV * (16 / sizeof(T));
    constexpr size_t MOST = 1u << 21; // blocks; a launch has fewer than 2^32 threads
    const size_t rpb = tpr <= 64 ? 256 / tpr : 1, want = (p.rows + rpb - 1) / rpb;
    const dim3 blocks((unsigned)(want < MOST ? want : MOST));
    if (tpr == 64) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 64, RAGGED>), blocks, dim3(256), 0, s, p);
    if constexpr (EPT <= 16) {
        if (tpr == 16) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 16, RAGGED>), blocks, dim3(256), 0, s, p);
    }
    if constexpr (EPT > 8) {
        if (tpr == 128) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 128, RAGGED>), blocks, dim3(128), 0, s, p);
        if (tpr == 256) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 256, RAGGED>), blocks, dim3(256), 0, s, p);
        if (tpr == 512) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 512, RAGGED>), blocks, dim3(512), 0, s, p);
    }
    if constexpr (EPT == 16) {
        if (tpr == 1024) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, 1024, RAGGED>), blocks, dim3(1024), 0, s, p);
    }
}

template <typename T>
void launch_quantize_t(const QuantArgs &p, hipStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    if (p.cols > 1024 * 16) {
        constexpr size_t MOST = 1u << 21;
        hipLaunchKernelGGL(quantize_long_rows_kernel<T>, dim3((unsigned)(p.rows < MOST ? p.rows : MOST)), dim3(1024), 0, s, p);
        return;
    }
    const int tpr = p.cols <= 16 * 16    ? 16
                    : p.cols <= 64 * 24  ? 64
                    : p.cols <= 128 * 24 ? 128
                    : p.cols <= 256 * 24 ? 256
                    : p.cols <= 512 * 24 ? 512
                                         : 1024;
    const int ept = (p.cols + tpr - 1) / tpr;
    auto launch = [&](auto nv) {
        constexpr int NV = nv;
        if ((uintptr_t)p.x % 16 == 0 && p.cols % V == 0 && (p.x_stride % V == 0 || p.rows == 1)) launch_quantize_nv<T, NV, false>(p, tpr, s);
        else launch_quantize_nv<T, NV, true>(p, tpr, s);
    };
    if (ept <= 8) launch(std::integral_constant<int, 8 / V>{});
    else if (ept <= 16) launch(std::integral_constant<int, 16 / V>{});
    else launch(std::integral_constant<int, 24 / V>{});
}

// ---- operands of the gradients ---------------------------------------------------------------------
// Both gradients sum (gradient * scale) * int8.  An int8 value is exact in binary16, and the float32 factor v = g * s is
// taken apart into binary16 pieces, each rounded to nearest: v = h + l to 2^-22 of v, or to 2^-39 of the row's
// largest |v| where that is more (v below 2^-17 of it).  The latter comes from binary16's smallest spacing, 2^-24, and the
// power of two per row of the result that brings the row's largest |v| to between 2^14 and 2^15; it is multiplied back in
// the epilogue, exactly.
// That is less of an error than the float32 additions of a few terms make.  Results in bfloat16 take both pieces too: one
// would be off by 2^-12 of each term, which shows where terms cancel (8192 x 4096 x 4096 with bfloat16 dx: a training
// step's call of 865 us with one piece of it, 1062 with both).
constexpr int PIECES = 2;
struct OperandArgs {
    const void *g;                  // [M][N] dense
    int M, N, K;
    const float *a_scale, *b_scale;
    const int8_t *a, *b;            // tokens [M][K], channels [N][K]
    size_t a_stride, b_stride;
    // for dx: pieces of g * b_scale, [PIECES][M][ldn], with the rows' powers of two, and b transposed, [K][ldn]
    f16_t *g_rows, *b_t;
    float *g_rows_scale;
    int ldn;
    // for dw: pieces of (g * a_scale) transposed, [PIECES][N][ldm], likewise, and a transposed, [K][ldm]
    f16_t *g_cols, *a_t;
    float *g_cols_scale;
    int ldm;
    // statistics of g's columns over each of `shares` runs of `share_rows` rows: sum of g and largest finite |g * a_scale|
    float *sums;
    unsigned *tops;
    int shares, share_rows;
    void *db;
    int db_dtype;
    // blocks of the first launch: rows of g, then tiles of b, then tiles of a, then the statistics
    unsigned row_blocks, b_blocks, a_blocks, stat_blocks;
};

// Magnitude as mag_bits has it, 0 for an infinity or a NaN: a row's power of two comes from its finite values.
__device__ __forceinline__ unsigned finite_bits(float x)
{
    const unsigned b = mag_bits(x);
    return b < 0x7f800000u ? b : 0u;
}
// Exponent e with top * 2^-e in [2^14, 2^15), or below where 2^e would not be a normal number; 0 for an empty row.
__device__ __forceinline__ int piece_exponent(unsigned top)
{
    return top == 0 ? 0 : max(ilogbf(__uint_as_float(top)) - 14, -126);
}
// An infinity or a NaN is its own first piece, so the products are what they are in float32: infinities, or NaN.
__device__ __forceinline__ void split(float v, int e, f16_t &high, f16_t &low)
{
    const float t = ldexpf(v, -e);
    high = (f16_t)t;
    low = mag_bits(t) < 0x7f800000u ? (f16_t)(t - (float)high) : (f16_t)0.f;
}

// The first n of V = 16 / sizeof(T) elements of a row from its element c on, zeros behind them.  RAGGED: they lie
// anywhere, and n may be less than V; else n is at least V or at most 0.
template <bool RAGGED, typename T, int V>
__device__ __forceinline__ void load_row(float (&v)[V], const T *row, int c, int n)
{
    typename VecOf<T, V>::type u{};
    if constexpr (RAGGED) u = load_some<T, V>(row + c, n, c);
    else if (n > 0) u = *(const typename VecOf<T, V>::type *)(row + c);
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = (float)u[j];
}
// The same of a row of g times their channels' scales.
template <bool RAGGED, typename T, int V>
__device__ __forceinline__ void load_scaled(float (&v)[V], const T *g, const float *scale, int c, int n)
{
    load_row<RAGGED>(v, g, c, n);
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        float s[4];
        load_row<RAGGED>(s, scale, c + i, n - i);
#pragma unroll
        for (int j = 0; j < 4; j++) v[i + j] *= s[j];
    }
}

template <typename T, bool RAGGED>
__device__ void split_row(const OperandArgs &p, size_t row, unsigned (&lds)[16])
{
    constexpr int V = 16 / sizeof(T);
    const T *g = (const T *)p.g + row * (size_t)p.N;
    unsigned t = 0;
#pragma unroll 2
    for (int c = threadIdx.x * V; c < p.N; c += 256 * V) {
        float v[V];
        load_scaled<RAGGED>(v, g, p.b_scale, c, p.N - c);
#pragma unroll
        for (int j = 0; j < V; j++) t = max(t, finite_bits(v[j]));
    }
    t = row_top<256>(t, lds);
    const int e = piece_exponent(t);
    f16_t *high = p.g_rows + row * (size_t)p.ldn, *low = high + (size_t)p.M * p.ldn;
    for (int c = threadIdx.x * V; c < p.ldn; c += 256 * V) { // ldn is a multiple of 64: whole vectors
        float v[V];
        load_scaled<RAGGED>(v, g, p.b_scale, c, p.N - c);
        typename VecOf<f16_t, V>::type h, l;
        f16_t *hp = (f16_t *)&h, *lp = (f16_t *)&l;
#pragma unroll
        for (int j = 0; j < V; j++) split(v[j], e, hp[j], lp[j]);
        *(typename VecOf<f16_t, V>::type *)(high + c) = h;
        *(typename VecOf<f16_t, V>::type *)(low + c) = l;
    }
    if (threadIdx.x == 0) p.g_rows_scale[row] = ldexpf(1.f, e);
}

// q [rows][cols] int8 -> out [cols][ld] binary16, positions from rows to ld zero; a 64 x 64 tile.  q's rows are 16-byte
// aligned and readable to the next multiple of 16.
__device__ void transpose_tile(const int8_t *q, size_t stride, int rows, int cols, int ld, f16_t *out, unsigned tile, int8_t (&lds)[64][68])
{
    const int across = ld / 64, r0 = (int)(tile % across) * 64, c0 = (int)(tile / across) * 64;
    const int r = threadIdx.x / 4, c = threadIdx.x % 4 * 16;
    int v[4] = {0, 0, 0, 0};
    if (r0 + r < rows && c0 + c < cols) {
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        const i32x4 u = *(const i32x4 *)(q + (size_t)(r0 + r) * stride + c0 + c);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = u[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) *(int *)&lds[r][c + 4 * i] = v[i];
    __syncthreads();
    const int oc = threadIdx.x / 4, orow = threadIdx.x % 4 * 16;
    if (c0 + oc >= cols) return;
    f16_t *dst = out + (size_t)(c0 + oc) * ld + r0 + orow;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        typename VecOf<f16_t, 8>::type w;
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (f16_t)(float)lds[orow + 8 * h + i][oc];
        *(typename VecOf<f16_t, 8>::type *)(dst + 8 * h) = w;
    }
}

// Sum of g and largest finite |g * a_scale| of 64 columns over one share of the rows: 64 / V threads across, the rest down.
template <typename T, bool RAGGED>
__device__ void column_stats(const OperandArgs &p, unsigned block, float (&ls)[32][64], unsigned (&lt)[32][64])
{
    constexpr int V = 16 / sizeof(T), ACROSS = 64 / V, DOWN = 256 / ACROSS; // 16 or 32 rows at once
    const int share = (int)(block % p.shares), x = threadIdx.x % ACROSS * V, c = (int)(block / p.shares) * 64 + x;
    const int y = threadIdx.x / ACROSS, begin = share * p.share_rows;
    const int end = begin + min(p.share_rows, p.M - begin);
    float s[V] = {};
    unsigned t[V] = {};
    if (c < p.N)
#pragma unroll 4
        for (int m = begin + y; m < end; m += DOWN) {
            float g[V];
            load_row<RAGGED>(g, (const T *)p.g + (size_t)m * p.N, c, p.N - c);
            const float scale = p.a_scale ? p.a_scale[m] : 0.f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                s[j] += g[j];
                t[j] = max(t[j], finite_bits(g[j] * scale));
            }
        }
#pragma unroll
    for (int j = 0; j < V; j++) {
        ls[y][x + j] = s[j];
        lt[y][x + j] = t[j];
    }
    __syncthreads();
    const int n = (int)(block / p.shares) * 64 + threadIdx.x;
    if (threadIdx.x < 64 && n < p.N) {
        float sum = 0.f;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < DOWN; i++) {
            sum += ls[i][threadIdx.x];
            top = max(top, lt[i][threadIdx.x]);
        }
        p.sums[(size_t)share * p.N + n] = sum;
        p.tops[(size_t)share * p.N + n] = top;
    }
}

// All that the gradients' operands need of each other's results is the columns' statistics, so everything else is one
// launch, told apart by the block's number.  Bound by memory: g twice, int8 in and binary16 out for both transposes, g's
// rows out; 8192 x 4096 x 4096 with bfloat16 g: 419 MB in 84-88 us (4.8-5 TB/s), the second launch 201 MB in 37 us (5.4).
template <typename T, bool RAGGED>
__global__ __launch_bounds__(256) void operands_kernel(OperandArgs p)
{
    __shared__ union {
        unsigned top[16];
        int8_t tile[64][68];
        struct { float s[32][64]; unsigned t[32][64]; } stats;
    } lds;
    unsigned b = blockIdx.x;
    if (b < p.row_blocks) return split_row<T, RAGGED>(p, b, lds.top);
    b -= p.row_blocks;
    if (b < p.b_blocks) return transpose_tile(p.b, p.b_stride, p.N, p.K, p.ldn, p.b_t, b, lds.tile);
    b -= p.b_blocks;
    if (b < p.a_blocks) return transpose_tile(p.a, p.a_stride, p.M, p.K, p.ldm, p.a_t, b, lds.tile);
    b -= p.a_blocks;
    column_stats<T, RAGGED>(p, b, lds.stats.s, lds.stats.t);
}

// The second launch: pieces of (g * a_scale) transposed, a 64 x 64 tile per block, and db from the shares' sums.
template <typename T, bool RAGGED>
__global__ __launch_bounds__(256) void transposed_pieces_kernel(OperandArgs p)
{
    constexpr int V = 16 / sizeof(T), ACROSS = 64 / V, DOWN = 256 / ACROSS;
    __shared__ float tile[64][65];
    __shared__ unsigned tops[4][64];
    __shared__ float sums[4][64];
    const int across = p.ldm / 64, m0 = (int)(blockIdx.x % across) * 64, n0 = (int)(blockIdx.x / across) * 64;
#pragma unroll
    for (int i = 0; i < 64; i += DOWN) {
        const int r = i + threadIdx.x / ACROSS, m = m0 + r, c = threadIdx.x % ACROSS * V;
        float v[V];
        load_row<RAGGED>(v, (const T *)p.g + (size_t)m * p.N, n0 + c, m < p.M ? p.N - n0 - c : 0);
        const float scale = m < p.M ? p.a_scale[m] : 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) tile[r][c + j] = v[j] * scale;
    }
    {
        const int x = threadIdx.x % 64, y = threadIdx.x / 64, n = n0 + x;
        unsigned t = 0;
        float s = 0.f;
        if (n < p.N)
#pragma unroll 4
            for (int i = y; i < p.shares; i += 4) {
                t = max(t, p.tops[(size_t)i * p.N + n]);
                s += p.sums[(size_t)i * p.N + n];
            }
        tops[y][x] = t;
        sums[y][x] = s;
    }
    __syncthreads();
    auto top_of = [&](int x) { return max(max(tops[0][x], tops[1][x]), max(tops[2][x], tops[3][x])); };
    if (m0 == 0 && threadIdx.x < 64 && n0 + threadIdx.x < p.N) {
        const int x = threadIdx.x;
        p.g_cols_scale[n0 + x] = ldexpf(1.f, piece_exponent(top_of(x)));
        if (p.db) store_any(p.db, p.db_dtype, n0 + x, ((sums[0][x] + sums[1][x]) + sums[2][x]) + sums[3][x]);
    }
    const int on = threadIdx.x / 4, om = threadIdx.x % 4 * 16;
    if (n0 + on >= p.N) return;
    const int e = piece_exponent(top_of(on));
    f16_t *high = p.g_cols + (size_t)(n0 + on) * p.ldm + m0 + om, *low = high + (size_t)p.N * p.ldm;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        typename VecOf<f16_t, 8>::type hv, lv;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f16_t a, b;
            split(tile[om + 8 * h + i][on], e, a, b);
            hv[i] = a;
            lv[i] = b;
        }
        *(typename VecOf<f16_t, 8>::type *)(high + 8 * h) = hv;
        *(typename VecOf<f16_t, 8>::type *)(low + 8 * h) = lv;
    }
}

// ---- host ------------------------------------------------------------------------------------------
int check_int8(const rexsc_int8_desc *d)
{
    REXSC_CHECK_DESC(d, rexsc_int8_desc);
    REXSC_CHECK_ARG(d->M >= 0 && d->N >= 0 && d->M <= MAX_ROWS && d->N <= MAX_ROWS, "int8 linear: M %d, N %d", d->M, d->N);
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

struct Space { size_t tokens, scales, g_rows, g_rows_scale, b_t, g_cols, g_cols_scale, a_t, sums, tops, product, total; };

constexpr int MAX_SHARES = 32, SHARE_ROWS = 512; // runs of g's rows whose column statistics are taken apart
int share_rows(int M) { return max(SHARE_ROWS, (M + MAX_SHARES - 1) / MAX_SHARES); }
int shares(int M) { return (M - 1) / share_rows(M) + 1; }

constexpr int ALL = REXSC_INT8_DX | REXSC_INT8_DW | REXSC_INT8_DB;

// Whether the launches of the wanted gradients hold d's sizes.
int check_backward(const rexsc_int8_desc *d, int wanted)
{
    if (d->M == 0 || d->N == 0) return REXSC_OK;
    const bool dx = wanted & REXSC_INT8_DX, dw = wanted & REXSC_INT8_DW, stats = wanted & (REXSC_INT8_DW | REXSC_INT8_DB);
    const uint64_t tiles_k = (uint64_t)((d->K + 63) / 64), tiles_n = (uint64_t)pad64(d->N) / 64, tiles_m = (uint64_t)pad64(d->M) / 64;
    // a launch has fewer than 2^32 threads
    REXSC_CHECK_ARG((dx ? d->M + tiles_n * tiles_k : 0) + (dw ? tiles_m * tiles_k : 0) + (stats ? tiles_n * MAX_SHARES : 0) < (1ull << 24) &&
                        (!dw || tiles_m * tiles_n < (1ull << 24)),
                    "int8 linear: gradients of %d x %d x %d are more than a launch holds", d->M, d->N, d->K);
    REXSC_CHECK_ARG((!dx || tiles_n * 128 < MAX_ROW_BYTES) && (!dw || tiles_m * 128 < MAX_ROW_BYTES),
                    "int8 linear: sums over at most %zu tokens (weight's gradient) or channels (input's gradient)", MAX_ROW_BYTES / 2 - 64);
    return REXSC_OK;
}

// wanted: the gradients that a workspace for them is to hold.
Space space(const rexsc_int8_desc *d, int what, int wanted = ALL)
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
    } else if (M > 0 && N > 0) {
        // dx and dw follow each other on the stream, so their partial results share a place
        const size_t ldn = pad64(N), ldm = pad64(M);
        const bool dx = wanted & REXSC_INT8_DX, dw = wanted & REXSC_INT8_DW;
        s.product = take(max(dx ? tile_product_workspace(d->M, d->K, (int)ldn * 2, PIECES) : 0,
                             dw ? tile_product_workspace(d->N, d->K, (int)ldm * 2, PIECES) : 0));
        if (dx) {
            s.g_rows = take(M * ldn * PIECES * 2);
            s.g_rows_scale = take(M * 4);
            s.b_t = take(K * ldn * 2);
        }
        if (dw) {
            s.g_cols = take(N * ldm * PIECES * 2);
            s.g_cols_scale = take(N * 4);
            s.a_t = take(K * ldm * 2);
        }
        if (wanted & (REXSC_INT8_DW | REXSC_INT8_DB)) {
            s.sums = take((size_t)shares(d->M) * N * 4);
            s.tops = take((size_t)shares(d->M) * N * 4);
        }
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
    if (what < REXSC_INT8_PRODUCT || what > REXSC_INT8_BACKWARD) {
        set_error("int8 linear: no call has the number %d", what);
        return (size_t)-1;
    }
    return what == REXSC_INT8_BACKWARD ? rexsc_int8_backward_workspace_bytes(d, ALL) : space(d, what).total;
}

extern "C" size_t rexsc_int8_backward_workspace_bytes(const rexsc_int8_desc *d, int wanted)
{
    if (check_int8(d)) return (size_t)-1;
    if (wanted & ~ALL) {
        set_error("int8 linear: no gradients have the flags %d", wanted);
        return (size_t)-1;
    }
    return check_backward(d, wanted) ? (size_t)-1 : space(d, REXSC_INT8_BACKWARD, wanted).total;
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
    if (few_rows_fuses(d->M, d->N, d->K, x, (size_t)d->x_stride, d->dtype)) {
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

extern "C" int rexsc_int8_backward(const rexsc_int8_desc *d, const void *g, const int8_t *a, const float *a_scale,
                                   const int8_t *b, const float *b_scale, void *dx, void *dw, void *db, void *workspace,
                                   size_t workspace_bytes, rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = check_int8(d)) return rc;
    if (!dx && !dw && !db) return REXSC_OK;
    if (d->M == 0 || d->N == 0) { // sums over nothing: zeros, from the same kernels
        auto zeros = [&](int rows, void *y, int dtype) {
            const TileArgs t{nullptr, nullptr, 0, 0, rows, d->K, 0, 1, 0, nullptr, nullptr, nullptr, REXSC_F32, y};
            return launch_tile_product(t, true, dtype, nullptr, "int8_backward_empty", stream);
        };
        if (dx && d->M > 0)
            if (int rc = zeros(d->M, dx, d->dtype)) return rc;
        if (dw && d->N > 0)
            if (int rc = zeros(d->N, dw, d->weight_dtype)) return rc;
        if (db && d->N > 0) return launch_column_sums(nullptr, 0, d->N, d->N, db, nullptr, d->bias_dtype, stream);
        return REXSC_OK;
    }
    REXSC_CHECK_ARG(g && (!dx || b_scale) && (!dw || a_scale), "null pointer");
    REXSC_CHECK_ARG((uintptr_t)g % dtype_size(d->dtype) == 0, "int8 linear: the gradient is not aligned to its element");
    if (dx)
        if (int rc = check_rows8("channels", b, d->b_stride, d->K)) return rc;
    if (dw)
        if (int rc = check_rows8("tokens", a, d->a_stride, d->K)) return rc;
    const int wanted = (dx ? REXSC_INT8_DX : 0) | (dw ? REXSC_INT8_DW : 0) | (db ? REXSC_INT8_DB : 0);
    if (int rc = check_backward(d, wanted)) return rc;
    const Space s = space(d, REXSC_INT8_BACKWARD, wanted);
    if (int rc = check_space(s, workspace, workspace_bytes)) return rc;
    auto at = [&](size_t o) { return (char *)workspace + o; };

    OperandArgs p{};
    p.g = g;
    p.M = d->M; p.N = d->N; p.K = d->K;
    p.a_scale = dw ? a_scale : nullptr;
    p.b_scale = b_scale;
    p.a = a; p.b = b;
    p.a_stride = (size_t)d->a_stride; p.b_stride = (size_t)d->b_stride;
    p.g_rows = (f16_t *)at(s.g_rows); p.b_t = (f16_t *)at(s.b_t); p.g_rows_scale = (float *)at(s.g_rows_scale);
    p.g_cols = (f16_t *)at(s.g_cols); p.a_t = (f16_t *)at(s.a_t); p.g_cols_scale = (float *)at(s.g_cols_scale);
    p.ldn = (int)pad64(d->N); p.ldm = (int)pad64(d->M);
    p.sums = (float *)at(s.sums); p.tops = (unsigned *)at(s.tops);
    p.shares = shares(d->M); p.share_rows = share_rows(d->M);
    p.db = db; p.db_dtype = d->bias_dtype;
    const uint64_t tiles_k = (uint64_t)((d->K + 63) / 64), tiles_n = (uint64_t)p.ldn / 64, tiles_m = (uint64_t)p.ldm / 64;
    p.row_blocks = dx ? (unsigned)d->M : 0;
    p.b_blocks = dx ? (unsigned)(tiles_n * tiles_k) : 0;
    p.a_blocks = dw ? (unsigned)(tiles_m * tiles_k) : 0;
    p.stat_blocks = dw || db ? (unsigned)(p.shares * tiles_n) : 0;
    // whether every row of g starts on a vector of 16 bytes, and the channels' scales (8192 tokens, 4095 channels, bfloat16, by single
    // elements: 99 and 62 us for both launches, in vectors wherever they lie 89 and 40)
    const bool wide = d->N % (d->dtype == REXSC_F32 ? 4 : 8) == 0 && ((uintptr_t)g | (uintptr_t)b_scale) % 16 == 0;
    {
        const double es = (double)dtype_size(d->dtype), mn = (double)d->M * d->N, k = (double)d->K;
        ProfScope prof("int8_backward_operands", (dx ? mn * (es + 2.0 * PIECES) + 3.0 * k * d->N : 0.0) + (dw || db ? mn * es : 0.0) +
                       (dw ? 3.0 * k * d->M : 0.0), stream);
        const dim3 grid(p.row_blocks + p.b_blocks + p.a_blocks + p.stat_blocks);
        if (wide)
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL((operands_kernel<T, false>), grid, dim3(256), 0, stream, p));
        else
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL((operands_kernel<T, true>), grid, dim3(256), 0, stream, p));
        REXSC_CHECK_HIP(hipGetLastError());
    }
    if (dw) {
        ProfScope prof("int8_backward_pieces", (double)d->M * d->N * (dtype_size(d->dtype) + 2.0 * PIECES), stream);
        const dim3 grid((unsigned)(tiles_m * tiles_n));
        if (wide)
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL((transposed_pieces_kernel<T, false>), grid, dim3(256), 0, stream, p));
        else
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL((transposed_pieces_kernel<T, true>), grid, dim3(256), 0, stream, p));
        REXSC_CHECK_HIP(hipGetLastError());
    } else if (db) {
        if (int rc = launch_column_sums(p.sums, p.shares, d->N, d->N, db, nullptr, d->bias_dtype, stream)) return rc;
    }
    if (dx) {
        const TileArgs t{(const char *)p.g_rows, (const char *)p.b_t, (size_t)p.ldn * 2, (size_t)p.ldn * 2, d->M, d->K, p.ldn * 2,
                         PIECES, (size_t)d->M * p.ldn * 2, p.g_rows_scale, nullptr, nullptr, REXSC_F32, dx};
        if (int rc = launch_tile_product(t, true, d->dtype, at(s.product), "int8_grad_input", stream)) return rc;
    }
    if (dw) {
        const TileArgs t{(const char *)p.g_cols, (const char *)p.a_t, (size_t)p.ldm * 2, (size_t)p.ldm * 2, d->N, d->K, p.ldm * 2,
                         PIECES, (size_t)d->N * p.ldm * 2, p.g_cols_scale, nullptr, nullptr, REXSC_F32, dw};
        if (int rc = launch_tile_product(t, true, d->weight_dtype, at(s.product), "int8_grad_weight", stream)) return rc;
    }
    return REXSC_OK;
}
