// The 8-bit product for up to 48 tokens.
//
// The weights are read once, straight into the matrix instruction's first operand: a load takes 64 bytes of 16 weight
// rows, two loads of a wave a cache line of each, and the eight waves of a block take neighbouring lines of the same
// rows, so a row is read in runs of 1024 bytes.  There is nothing to share in LDS (each weight is used by one wave), and
// nothing to wait for but memory: a wave has UNROLL loads in flight before the first is used.  The waves' int32 sums,
// exact in any order, are joined through LDS.  With few tokens the block takes them to 8 bits itself, while
// its first weights are on their way: a launch of its own would cost more than every block's reading the few kilobytes
// again.
// Measured with weights from memory: 1 x 4096 x 4096 5.9 us from int8 tokens, 8.0 us from float ones (with the rows'
// own launch 9.0); 1 x 16384 x 4096 14.4 us (4.7 TB/s of weights).
#include <stdlib.h>

#include <type_traits>

#include "few_rows.h"
#include "profile.h"
#include "quant8.h"

namespace rexsc {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 8, THREADS = WAVES * 64;
constexpr int LOADS = 8;                   // of 64 bytes of 16 rows that a wave has in flight, at most
constexpr int UNIT = WAVES * 64;           // bytes of a row that the block's waves take with one load each
constexpr int FUSED_ROWS = 16;             // tokens that a block takes to 8 bits by itself, at most

__device__ __forceinline__ i32x4 keep_before(i32x4 v, int n) // the first n bytes (n may be anything)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int l = n - 4 * i;
        v[i] = l >= 4 ? v[i] : l <= 0 ? 0 : v[i] & (int)((1u << (8 * l)) - 1u);
    }
    return v;
}

struct FewArgs {
    TileArgs p;
    const void *x;       // float tokens (fused)
    size_t x_stride;
};

// A block makes 16 channels.  FM: fragments of 16 tokens; U0: loads per wave of the first round; X: type of the tokens, or
// int8_t: already in 8 bits; ELEMS: float elements that the block has room for.
template <int FM, int U0, typename T, typename X, int ELEMS>
__global__ __launch_bounds__(THREADS) void few_rows_kernel(FewArgs g)
{
    constexpr bool FUSED = ELEMS > 0;
    const TileArgs &p = g.p;
    __shared__ __attribute__((aligned(16))) int8_t tokens[FUSED ? ELEMS + FUSED_ROWS * 80 : 16];
    __shared__ int sums[WAVES][FM][256];
    __shared__ unsigned top[FUSED ? FUSED_ROWS : 1];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int n0 = blockIdx.x * 16, K = p.kbytes;
    const int at = wave * 128 + lane / 16 * 16; // this lane's 16 bytes; a wave takes 128 neighbouring bytes of its rows

    const int row = n0 + lane % 16;
    const char *const w = p.b + (size_t)(row < p.N ? row : p.N - 1) * p.b_stride;
    // offset of load u in the round that begins at k0; behind the row's end the row's first chunk is read instead (the
    // tokens are 0 there)
    auto place = [&](int k0, int u) __attribute__((always_inline)) { return k0 + u / 2 * (WAVES * 128) + u % 2 * 64 + at; };
    i32x4 wq[LOADS];
    auto load_w = [&](int k0, auto loads) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < loads; u++) {
            const int k = place(k0, u);
            wq[u] = *(const i32x4 *)(w + (k < K ? k : 0));
        }
    };
    load_w(0, std::integral_constant<int, U0>{});

    const int pitch = (K + 63) / 64 * 64 + 16; // of a token in LDS
    if constexpr (FUSED) {
        // M K <= ELEMS elements in vectors of 16 bytes, SLOTS per thread; rows begin on one
        constexpr int V = 16 / sizeof(X), SLOTS = ELEMS / V / THREADS;
        typedef typename VecOf<X, V>::type vec;
        const int per = K / V, all = p.M * per;
        vec v[SLOTS];
        int row[SLOTS], col[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; s++) {
            const int f = s * THREADS + threadIdx.x, c = f < all ? f : 0;
            row[s] = c / per;
            col[s] = (c - row[s] * per) * V;
            v[s] = *(const vec *)((const X *)g.x + (size_t)row[s] * g.x_stride + col[s]);
        }
        if (threadIdx.x < FUSED_ROWS) top[threadIdx.x] = 0;
        const int behind = pitch - K; // bytes behind a token, zeroed
        for (int i = threadIdx.x; i < p.M * behind; i += THREADS) tokens[i / behind * pitch + K + i % behind] = 0;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < SLOTS; s++) {
            unsigned t = 0;
#pragma unroll
            for (int e = 0; e < V; e++) t = max(t, mag_bits((float)v[s][e]));
            if (p.M == 1) {
                t = wave_max(t);
                if (lane == 0) atomicMax(&top[0], t);
            } else {
                atomicMax(&top[row[s]], t); // a maximum of integers: any order gives the same
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < SLOTS; s++) {
            const RowScale rs = row_scale(top[row[s]]);
            typename VecOf<int8_t, V>::type q;
#pragma unroll
            for (int e = 0; e < V; e++) q[e] = (int8_t)quant8((float)v[s][e], rs);
            *(typename VecOf<int8_t, V>::type *)(tokens + row[s] * pitch + col[s]) = q;
        }
        __syncthreads();
    }

    const char *a[FM];
#pragma unroll
    for (int i = 0; i < FM; i++) {
        const int m = i * 16 + lane % 16, r = m < p.M ? m : p.M - 1;
        a[i] = FUSED ? (const char *)tokens + r * pitch : p.a + (size_t)r * p.a_stride;
    }
    i32x4 acc[FM] = {};
    auto multiply = [&](int k0, auto loads) __attribute__((always_inline)) {
        i32x4 xq[loads][FM];
#pragma unroll
        for (int u = 0; u < loads; u++) {
            const int k = place(k0, u), o = k < K ? k : 0;
#pragma unroll
            for (int i = 0; i < FM; i++) xq[u][i] = *(const i32x4 *)(a[i] + o);
        }
        if (k0 + loads * UNIT > K) { // the row ends in this round
#pragma unroll
            for (int u = 0; u < loads; u++)
#pragma unroll
                for (int i = 0; i < FM; i++) xq[u][i] = keep_before(xq[u][i], K - place(k0, u));
        }
#pragma unroll
        for (int u = 0; u < loads; u++)
#pragma unroll
            for (int i = 0; i < FM; i++) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wq[u], xq[u][i], acc[i], 0, 0, 0);
    };
    multiply(0, std::integral_constant<int, U0>{});
    if constexpr (U0 == LOADS) {
        int k0 = U0 * UNIT;
        for (; K - k0 > 4 * UNIT; k0 += LOADS * UNIT) {
            load_w(k0, std::integral_constant<int, LOADS>{});
            multiply(k0, std::integral_constant<int, LOADS>{});
        }
        for (; k0 < K; k0 += 2 * UNIT) { // what is left: at most two short rounds
            load_w(k0, std::integral_constant<int, 2>{});
            multiply(k0, std::integral_constant<int, 2>{});
        }
    }

    // a lane holds channels 4 (lane / 16) + e of token lane % 16
#pragma unroll
    for (int i = 0; i < FM; i++) *(i32x4 *)&sums[wave][i][lane % 16 * 16 + lane / 16 * 4] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < FM * 256; o += THREADS) {
        const int f = o / 256, m = o / 16, n = n0 + o % 16;
        if (m >= p.M || n >= p.N) continue;
        int s = 0;
#pragma unroll
        for (int v = 0; v < WAVES; v++) s += sums[v][f][o % 256];
        float sa;
        if constexpr (FUSED) sa = row_scale(top[m]).scale;
        else sa = p.a_scale[m];
        const float y = fmaf((float)s * sa, p.b_scale[n], p.bias ? load_any(p.bias, p.bias_dtype, n) : 0.f);
        ((T *)p.y)[(size_t)m * p.N + n] = (T)y;
    }
}

template <int FM, typename T, typename X, int ELEMS>
int launch_u(const FewArgs &g, hipStream_t stream)
{
    REXSC_CHECK_ARG(g.p.N < (1 << 26), "int8 linear: %d output channels are more than a launch holds", g.p.N);
    const dim3 grid((unsigned)((g.p.N + 15) / 16));
    // a round that is longer than the row would load its first chunk over and over
    if (g.p.kbytes > 4 * UNIT) hipLaunchKernelGGL((few_rows_kernel<FM, 8, T, X, ELEMS>), grid, dim3(THREADS), 0, stream, g);
    else if (g.p.kbytes > 2 * UNIT) hipLaunchKernelGGL((few_rows_kernel<FM, 4, T, X, ELEMS>), grid, dim3(THREADS), 0, stream, g);
    else hipLaunchKernelGGL((few_rows_kernel<FM, 2, T, X, ELEMS>), grid, dim3(THREADS), 0, stream, g);
    REXSC_CHECK_HIP(hipGetLastError());
    return REXSC_OK;
}

template <typename T>
int launch_fm(const FewArgs &g, hipStream_t stream)
{
    if (g.p.M <= 16) return launch_u<1, T, int8_t, 0>(g, stream);
    if (g.p.M <= 32) return launch_u<2, T, int8_t, 0>(g, stream);
    return launch_u<3, T, int8_t, 0>(g, stream);
}

double work(const TileArgs &p) { return 2.0 * p.M * p.N * p.kbytes; }

} // namespace

int launch_few_rows(const TileArgs &p, int out_dtype, hipStream_t stream)
{
    ProfScope prof("int8_product_few", work(p), stream);
    const FewArgs g{p, nullptr, 0};
    REXSC_DTYPE_SWITCH(out_dtype, return launch_fm<T>(g, stream));
}

// Up to 8 tokens; up to 48 where the 64 x 64 tiles would leave half of the CUs without one.  Beyond, each block's reading
// all tokens again costs more than the tiles' sharing them in LDS: 32 tokens x 4096 x 4096 9 us here and 12 in tiles,
// but 37 x 11003 x 4099 27 us here and 15 in tiles, 16 x 16384 x 4096 19 and 17.5.
bool few_rows_takes(int M, int N) { return M <= 8 || (M <= FEW_ROWS && N < 64 * 128); }

// Every block of 16 channels takes the tokens to 8 bits again, which hides behind the weights and saves a launch while a
// CU has few blocks: 13.7 us a call against 16 from 1 x 2048 x 1000 to 1 x 4096 x 16384 in 16 bits; 4 x 4096 x 4096, with
// twice the elements, 13.9 against 16.0.  With more blocks or longer rows it costs more than it saves (float32 1 x 4096 x
// 32768 35 us against 32 and 2 x 2048 x 32768 33 against 18; 1 x 16384 x 4096 27 against 23.5).
bool few_rows_fuses(int M, int N, int K, const void *x, size_t x_stride, int dtype)
{
    const size_t es = dtype_size(dtype), elems = (size_t)M * K, out = (size_t)N * es;
    const bool pays = elems <= 8192 ? out <= 32768 : elems <= 16384 && K <= 8192 && out <= 16384;
    return M <= FUSED_ROWS && pays && (size_t)K * es % 16 == 0 && (uintptr_t)x % 16 == 0 && (M == 1 || x_stride * es % 16 == 0);
}

int launch_few_rows_fused(const TileArgs &p, const void *x, size_t x_stride, int dtype, hipStream_t stream)
{
    ProfScope prof("int8_linear_few", work(p), stream);
    const FewArgs g{p, x, x_stride};
    if (p.M * p.kbytes <= 8192) REXSC_DTYPE_SWITCH(dtype, return (launch_u<1, T, T, 8192>(g, stream)));
    REXSC_DTYPE_SWITCH(dtype, return (launch_u<1, T, T, 16384>(g, stream)));
}

} // namespace rexsc
