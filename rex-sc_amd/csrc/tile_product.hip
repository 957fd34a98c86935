// Product of two row-major operands: c[m][n] = sum_k a[m][k] b[n][k].
//
// Bound by the matrix pipe where the result is large, by reading b where it is not.  A tile's operands go to LDS by
// direct loads, whole steps ahead, and from there to registers half a step ahead of the matrix instruction.  256 x 256
// outputs per block of eight waves is the largest tile whose accumulators (128 a lane) leave room for two sets of
// fragments, and a step of 128 bytes the longest of which two fit LDS; it reads 64 KB from L2 for 8.4 M products.
// Measured, int8: 8192^3 398-404 us (2.7 POP/s), 8192 x 16384 x 4096 450-484 us (2.3-2.4), 8192 x 4096 x 4096 108-113 us;
// the library's int8 product reaches 2.24 POP/s at 8192^3 and 1.85 at 8192 x 16384 x 4096.  binary16, 4096 x 4096 x 8192
// in two pieces: 394-407 us (1.35-1.4 PFLOP/s).  The matrix pipe is busy 0.71 of the cycles, at 1.7-1.9 GHz.
#include <stdlib.h>

#include <type_traits>

#include "profile.h"
#include "tile_product.h"

namespace rexsc {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

struct OpI8 { typedef i32x4 acc; };
struct OpF16 { typedef f32x4 acc; };
__device__ __forceinline__ i32x4 mma(OpI8, i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(OpF16, i32x4 a, i32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Waits until at most N of this wave's loads into LDS are still on their way (they land in order), and until its reads
// of LDS are done: what a barrier needs that lets the other waves read the one and overwrite the other.  Nothing may be
// moved across either by the compiler.
template <int N>
__device__ __forceinline__ void loads_left()
{
    static_assert(N < 64, "the counter has six bits");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14); // vmcnt(N), no wait for the other counters
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void reads_done()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void meet()
{
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory"); // the barrier alone does not keep the compiler from reading memory before it
}

// Bytes of a 16-byte chunk at offset k that lie before `end`; the rest become 0.
__device__ __forceinline__ i32x4 keep_before(i32x4 v, int k, int end)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int n = end - k - 4 * i;
        v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & (int)((1u << (8 * n)) - 1u);
    }
    return v;
}

// The same value, which the compiler takes for a new one: what is computed from it is not kept in registers from
// before.
__device__ __forceinline__ int again(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;

// 16 bytes per lane from base + offset to LDS, at dst + 16 * lane; zeros where the offset is not below `bytes`.
__device__ __forceinline__ void load_to_lds(const char *base, unsigned bytes, unsigned offset, char *dst)
{
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, (int)bytes, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)dst, 16, offset, 0, 0, 0);
}

constexpr int KSTEP = 128;          // bytes of the reduction per step
constexpr int CHUNKS = KSTEP / 16;  // 16-byte chunks of a tile row

// Where chunk c of tile row r lies in that row's 128 bytes of LDS.  A fragment read takes the same chunk of 16
// consecutive rows: with the rows' pairs shifted against each other they fall on all 64 banks once.
__device__ __forceinline__ int swizzle(int r, int c) { return c ^ ((r >> 1) & (CHUNKS - 1)); }

// Tile of a block.  Workgroups go to the eight XCDs in turn, each with an L2 of its own: an XCD gets a contiguous run
// of the tile order, and the order walks groups of GROUP_M tile rows column by column, so that the tiles an XCD has in
// flight at once form a patch that shares operand rows.
constexpr int XCDS = 8, GROUP_M = 4;
__device__ __forceinline__ void tile_of(unsigned bid, int tiles_m, int tiles_n, int &tm, int &tn)
{
    const unsigned total = (unsigned)tiles_m * (unsigned)tiles_n, per = total / XCDS, extra = total % XCDS;
    const unsigned x = bid % XCDS, i = bid / XCDS;
    const unsigned t = x * per + (x < extra ? x : extra) + i;
    const unsigned group = (unsigned)(GROUP_M * tiles_n), g = t / group, r = t % group;
    const int left = tiles_m - (int)g * GROUP_M, rows = left < GROUP_M ? left : GROUP_M;
    tm = __builtin_amdgcn_readfirstlane((int)g * GROUP_M + (int)(r % rows)); // (divided in vector registers)
    tn = __builtin_amdgcn_readfirstlane((int)(r / rows));
}

// The tiles first ... end - 1 of the order.
// SPLIT: the grid holds `splits` times the tiles, and a block sums only its share of the steps, into a partial result
// of the accumulator's type (T), a tile of its own, that join_kernel finishes.
// STREAM: the grid holds a block per CU, and a block takes every gridDim.x-th tile.  Its steps are one stream over all
// its tiles: the next tile's first steps are fetched while the last one's are multiplied and while the finished tile is
// stored, from LDS of its own.  Against a block per tile, in turn: 8192 x 16384 x 4096 468 -> 451 us, 8192 x 4096 x 4096
// 114 -> 109, 8192 x 16384 x 1024 165 -> 146-153.
template <typename Op, typename T, int BM, int BN, int WM, int WN, int STAGES, bool SPLIT, bool STREAM>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(TileArgs p, int splits, unsigned first, unsigned end)
{
    static_assert(!(SPLIT && STREAM), "a split tile is one of its own");
    constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES; // loads of 8 rows x 128 bytes per wave and step
    static_assert(LA * WAVES * 8 == BM && LB * WAVES * 8 == BN, "tile rows must divide among the waves");
    constexpr int BUF = (BM + BN) * KSTEP;
    // the tile on its way out: COLS x CR elements per wave, behind the buffers (STREAM) or in their place
    constexpr int COLS = BN / WN, ROWS = BM / WM, RB = COLS * (int)sizeof(T), PART = STREAM ? 16 : sizeof(T) == 4 ? 32 : 64;
    constexpr int CR = ROWS < PART ? ROWS : PART, SHARE = CR * RB;
    static_assert(WAVES * SHARE <= STAGES * BUF, "the waves' shares fit the buffers");
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * BUF + (STREAM ? WAVES * SHARE : 0)];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    const int share = SPLIT ? (int)(blockIdx.x % splits) : 0;
    unsigned tile = first + (SPLIT ? blockIdx.x / splits : blockIdx.x);

    // A wave's loads are 8 * WAVES rows apart, so that a lane takes the same chunk in all of them (the LDS side of a load
    // is fixed: 16 bytes per lane in lane order).  Rows behind the operand's last lie behind the descriptor's range.
    static_assert(WAVES % 2 == 0, "loads of one wave must be 16 rows apart");
    const char *base_a, *base_b;
    unsigned bytes_a, bytes_b;
    auto seek = [&](unsigned t) __attribute__((always_inline)) {
        int tm, tn;
        tile_of(t, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * BM, n0 = tn * BN;
        base_a = p.a + (size_t)m0 * p.a_stride;
        base_b = p.b + (size_t)n0 * p.b_stride;
        bytes_a = (unsigned)(p.M - m0 < BM ? p.M - m0 : BM) * (unsigned)p.a_stride;
        bytes_b = (unsigned)(p.N - n0 < BN ? p.N - n0 : BN) * (unsigned)p.b_stride;
    };
    seek(tile);
    const unsigned chunk = (unsigned)swizzle(wave * 8 + lane / 8, lane % 8) * 16;
    unsigned offa[LA], offb[LB]; // this lane's chunk in each load
#pragma unroll
    for (int i = 0; i < LA; i++) offa[i] = (unsigned)((i * WAVES + wave) * 8 + lane / 8) * (unsigned)p.a_stride + chunk;
#pragma unroll
    for (int i = 0; i < LB; i++) offb[i] = (unsigned)((i * WAVES + wave) * 8 + lane / 8) * (unsigned)p.b_stride + chunk;
    const int steps = p.kbytes > KSTEP ? (p.kbytes + KSTEP - 1) / KSTEP : 1; // (an empty sum: a step of zeros)
    const int every = steps * p.pieces;
    const int begin = SPLIT ? (int)((int64_t)every * share / splits) : 0;
    const int total = (SPLIT ? (int)((int64_t)every * (share + 1) / splits) : every) - begin;
    if constexpr (SPLIT) base_a += (size_t)(begin / steps) * p.piece_stride;

    // what is fetched next: the byte offset in the row, the tile, and the steps that this tile still has
    unsigned k = SPLIT ? (unsigned)(begin % steps) * KSTEP : 0, ahead = tile;
    int left = total;
    auto fetch = [&](char *buf) __attribute__((always_inline)) {
        if (left == 0) return;
        auto load = [&](unsigned beyond) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < LA; i++) load_to_lds(base_a + k, bytes_a - k, offa[i] | beyond, buf + (i * WAVES + wave) * 1024);
#pragma unroll
            for (int i = 0; i < LB; i++)
                load_to_lds(base_b + k, bytes_b - k, offb[i] | beyond, buf + BM * KSTEP + (i * WAVES + wave) * 1024);
        };
        // a chunk behind the row's end is put outside of the descriptor's range and arrives as zeros
        if (k + KSTEP <= (unsigned)p.kbytes) load(0);
        else load(k + chunk < (unsigned)p.kbytes ? 0 : 0x80000000u);
        k += KSTEP;
        if (k >= (unsigned)p.kbytes) { k = 0; base_a += p.piece_stride; }
        left--;
        if (STREAM && left == 0) {
            ahead += gridDim.x;
            if (ahead < end) { left = total; seek(ahead); }
        }
    };
    // int8 rows whose last chunk is not full: what stands behind the row may be anything, and becomes 0 in a's tile
    const int tail = begin + total == every ? p.kbytes % 16 : 0;
    const int clear_at = !tail ? -1 : total == 1 ? 0 : total - 2; // the step before the one with that chunk
    auto clear_tail = [&](lds_char *buf) __attribute__((always_inline)) {
        const int c = p.kbytes % KSTEP / 16;
        for (int r = wave * 64 + again(lane); r < BM; r += WAVES * 64) {
            lds_i32x4 *at = (lds_i32x4 *)(buf + r * KSTEP + swizzle(r, c) * 16);
            *at = keep_before(*at, 0, tail);
        }
        __syncthreads();
    };

    const int wm = wave / WN * ROWS, wn = wave % WN * COLS;
    typename Op::acc acc[FM][FN] = {};
    i32x4 fa[2][FM], fb[2][FN]; // fragments of the half step that is multiplied and of the next one
    // Rows 16 apart lie at the same place of the swizzle, and the second half's chunks 64 bytes across it, so a
    // fragment's address is one of two lane offsets plus a constant.
    const int q = lane % 16 * KSTEP + swizzle(lane % 16, lane / 16) * 16;
    lds_char *const base = (lds_char *)lds;
    const int at_a[2] = {wm * KSTEP + q, wm * KSTEP + (q ^ 64)}, at_b[2] = {(BM + wn) * KSTEP + q, (BM + wn) * KSTEP + (q ^ 64)};
    // Multiplies the fragments of `half` while the next half's are read from `buf`: a row of a's fragment is replaced as
    // soon as its products are issued, so the second set costs no more registers than b's.
    auto multiply = [&](auto half_, const lds_char *buf) __attribute__((always_inline)) {
        constexpr int half = half_, next = half ^ 1;
        const lds_char *const ra = buf + at_a[next], *const rb = buf + at_b[next];
#pragma unroll
        for (int i = 0; i < FM; i++) {
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = mma(Op{}, fb[half][j], fa[half][i], acc[i][j]);
            fa[next][i] = *(const lds_i32x4 *)(ra + i * 16 * KSTEP);
#pragma unroll
            for (int j = i * FN / FM; j < (i + 1) * FN / FM; j++) fb[next][j] = *(const lds_i32x4 *)(rb + j * 16 * KSTEP);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The factors of the wave's rows and columns, one of each per lane, on their way while the tile is multiplied.  What
    // lies behind the last row or column, and a vector that is not there, reads 0.
    constexpr int SA = (ROWS + 63) / 64;
    const bool wide_bias = p.bias_dtype == REXSC_F32;
    int sa_lane[SA] = {}, sb_lane = 0, bias_lane = 0;
    short bias16_lane = 0;
    auto load_factors = [&](int m, int n) __attribute__((always_inline)) {
        if constexpr (SPLIT) return;
        const int l = again(lane);
        const int rows = m < p.M ? (p.M - m < ROWS ? p.M - m : ROWS) : 0, cols = n < p.N ? (p.N - n < COLS ? p.N - n : COLS) : 0;
        auto part = [](const void *v, int first, int count, int size) __attribute__((always_inline)) {
            return __builtin_amdgcn_make_buffer_rsrc((char *)const_cast<void *>(v) + (size_t)first * size, 0, v ? count * size : 0,
                                                     0x00027000);
        };
#pragma unroll
        for (int i = 0; i < SA; i++)
            sa_lane[i] = __builtin_amdgcn_raw_buffer_load_b32(part(p.a_scale, m, rows, 4), (i * 64 + l) * 4, 0, 0);
        sb_lane = __builtin_amdgcn_raw_buffer_load_b32(part(p.b_scale, n, cols, 4), l * 4, 0, 0);
        bias_lane = __builtin_amdgcn_raw_buffer_load_b32(part(wide_bias ? p.bias : nullptr, n, cols, 4), l * 4, 0, 0);
        bias16_lane = __builtin_amdgcn_raw_buffer_load_b16(part(wide_bias ? nullptr : p.bias, n, cols, 2), l * 2, 0, 0);
    };

    // STAGES buffers in a ring.  A step's second half is read while its first is multiplied; then, with every wave's
    // fragments of this buffer in registers and the next buffer filled, one barrier, behind which this buffer is filled
    // anew, STAGES steps ahead, and the first half of the next is read while the second half is multiplied.  (Behind
    // the last step that reads what is not used.)
#pragma unroll
    for (int i = 0; i < STAGES; i++) fetch(lds + i * BUF);
    if (!STREAM && total >= STAGES) loads_left<(STAGES - 1) * (LA + LB)>();
    else loads_left<0>();
    meet();
    if (tail && total == 1) clear_tail(base);
    const int height = SPLIT ? BM : p.M, width = SPLIT ? BN : p.N;
    T *const y = (T *)p.y + (SPLIT ? ((size_t)share * (end - first) + (tile - first)) * (BM * BN) : 0);
    const size_t pitch = (size_t)width * sizeof(T);
    const bool wide = pitch % 16 == 0 && (uintptr_t)y % 16 == 0 && pitch < 0x80000000u / CR;
    lds_char *const mine = base + (STREAM ? STAGES * BUF : 0) + wave * SHARE;
    int cur = 0;
    do {
        int tm, tn;
        tile_of(tile, tiles_m, tiles_n, tm, tn);
        const int first_m = tm * BM + wm, first_n = tn * BN + wn;
        load_factors(first_m, first_n);
#pragma unroll
        for (int i = 0; i < FM; i++) fa[0][i] = *(const lds_i32x4 *)(base + cur + at_a[0] + i * 16 * KSTEP);
#pragma unroll
        for (int j = 0; j < FN; j++) fb[0][j] = *(const lds_i32x4 *)(base + cur + at_b[0] + j * 16 * KSTEP);
        int s = 0;
        do {
            multiply(std::integral_constant<int, 0>{}, base + cur);
            // the loads of steps s + 2 ... s + STAGES - 1 may still be on their way (towards the end there are fewer)
            if (STAGES > 2 && s + STAGES - 1 < total) loads_left<(STAGES - 2) * (LA + LB)>();
            else loads_left<0>();
            reads_done();
            meet();
            const int next = cur + BUF < STAGES * BUF ? cur + BUF : 0;
            if (s == clear_at) clear_tail(base + next);
            fetch(lds + cur);
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
            multiply(std::integral_constant<int, 1>{}, base + cur);
        } while (++s < total);

        // Epilogue.  b was the first operand, so a lane holds four neighbouring columns n of one row m: written like
        // that, a store would touch 16 rows with 8 bytes each.  The wave turns its part of the tile round in LDS (its own
        // share) and stores 16 bytes per lane along the rows.  The 16-byte chunks of a row are permuted by its number,
        // which spreads the 16 rows of a write over all banks.
        const int l = again(lane);
        auto place = [&](int r, int byte) { return r * RB + ((byte / 16 ^ r * RB / 256) & (RB / 16 - 1)) * 16 + byte % 16; };
        const float bias_f = wide_bias ? __builtin_bit_cast(float, bias_lane)
                             : p.bias_dtype == REXSC_F16 ? (float)__builtin_bit_cast(f16_t, bias16_lane)
                                                         : __builtin_bit_cast(float, (int)bias16_lane << 16);
        const float sb_f = p.b_scale ? __builtin_bit_cast(float, sb_lane) : 1.f;
        float sa_f[SA], sb[FN][4], bias[FN][4];
#pragma unroll
        for (int i = 0; i < SA; i++) sa_f[i] = p.a_scale ? __builtin_bit_cast(float, sa_lane[i]) : 1.f;
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = j * 16 + l / 16 * 4 + e;
                sb[j][e] = __shfl(sb_f, c, 64);
                bias[j][e] = __shfl(bias_f, c, 64);
            }
        if (!STREAM) __syncthreads(); // the buffers are the waves' shares from here on
        const int row0 = SPLIT ? wm : first_m, col0 = SPLIT ? wn : first_n;
#pragma unroll
        for (int r0 = 0; r0 < ROWS; r0 += CR) {
#pragma unroll
            for (int i = 0; i < CR / 16; i++) {
                const float sa = __shfl(sa_f[(r0 + i * 16) / 64], (r0 + i * 16) % 64 + l % 16, 64);
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    typename VecOf<T, 4>::type v;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (SPLIT) v[e] = acc[r0 / 16 + i][j][e];
                        else v[e] = (T)fmaf((float)acc[r0 / 16 + i][j][e] * sa, sb[j][e], bias[j][e]);
                    }
                    const int to = place(i * 16 + l % 16, (j * 16 + l / 16 * 4) * (int)sizeof(T));
                    *(__attribute__((address_space(3))) typename VecOf<T, 4>::type *)(mine + to) = v;
                }
            }
            const int rows = height - (row0 + r0) < CR ? height - (row0 + r0) : CR; // of this part, that exist
            T *out = y + (size_t)(row0 + r0) * width + col0;
            if (wide) {
                // rows that do not exist lie behind the descriptor's range, and so do a lane's columns if they do not exist
                constexpr int LANES = RB / 16; // that store a row
                const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
                    out, 0, rows > 0 && col0 < width ? (int)((rows - 1) * pitch + (size_t)(width - col0) * sizeof(T)) : 0, 0x00027000);
                unsigned to = (unsigned)(l / LANES) * (unsigned)pitch + (unsigned)(l % LANES) * 16;
                if (col0 + l % LANES * 16 / (int)sizeof(T) >= width) to = 0x80000000u;
#pragma unroll
                for (int t = 0; t < SHARE / 1024; t++) {
                    const i32x4 v = *(const lds_i32x4 *)(mine + place(t * (64 / LANES) + l / LANES, l % LANES * 16));
                    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, to + (unsigned)(t * (64 / LANES)) * (unsigned)pitch, 0, 0);
                }
            } else {
                // the same wherever the rows begin; the vector that a row's end cuts is stored by elements
                constexpr int LANES = RB / 16, VEC = 16 / sizeof(T);
                const int left = width - col0 - l % LANES * VEC;
#pragma nounroll
                for (int t = 0; t < SHARE / 1024; t++) {
                    const int r = t * (64 / LANES) + l / LANES;
                    const i32x4 v = *(const lds_i32x4 *)(mine + place(r, l % LANES * 16));
                    if (r < rows) store_some<T, VEC>(out + (size_t)r * width + l % LANES * VEC, __builtin_bit_cast(typename VecOf<T, VEC>::type, v), left);
                }
            }
        }
        if (!STREAM) break;
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = typename Op::acc{};
        tile += gridDim.x;
    } while (tile < end);
}

// y = (sum of the partial results, in order) * scales + bias of `count` tiles from `first` on; ACC: int or float.  Four
// elements of a row per thread.
template <typename ACC, typename T>
__global__ __launch_bounds__(256) void join_kernel(TileArgs p, const ACC *part, int splits, unsigned first, unsigned count, int bm, int bn)
{
    const unsigned per = (unsigned)(bm * bn) / 1024, local = blockIdx.x / per;
    const int at = (int)(blockIdx.x % per * 1024 + threadIdx.x * 4);
    int tm, tn;
    tile_of(first + local, (p.M + bm - 1) / bm, (p.N + bn - 1) / bn, tm, tn);
    const int m = tm * bm + at / bn, n = tn * bn + at % bn;
    if (m >= p.M || n >= p.N) return;
    ACC s[4] = {};
    for (int z = 0; z < splits; z++) {
        const typename VecOf<ACC, 4>::type v = *(const typename VecOf<ACC, 4>::type *)(part + ((size_t)z * count + local) * (bm * bn) + at);
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] += v[e];
    }
    const float sa = p.a_scale ? p.a_scale[m] : 1.f;
    T *out = (T *)p.y + (size_t)m * p.N + n;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < p.N) {
            const float sb = p.b_scale ? p.b_scale[n + e] : 1.f, bias = p.bias ? load_any(p.bias, p.bias_dtype, n + e) : 0.f;
            out[e] = (T)fmaf((float)s[e] * sa, sb, bias); // as in the unsplit kernel
        }
}

// ---- host ------------------------------------------------------------------------------------------
constexpr int CUS = 256, MAX_SPLITS = 16;
constexpr double REST_US = 16, REST_TILE_US = 0.12; // of splitting the last tiles, and of each partial result; see tile_plan

struct TilePlan {
    int size;        // 256, 128, 64 (squares) or 32 (64 x 32)
    int splits;      // shares of the reduction
    bool alone;      // no CU gets two 128 x 128 tiles
    int rest_splits; // 256: shares for the tiles behind the last full round, 0 where they are a round like the others
};

int tune(const char *name)
{
    const char *v = getenv(name);
    return v ? atoi(v) : 0;
}

// Tile size by what a launch takes when its busiest CU gets n tiles, in units of one 256 x 256 tile (measured at
// K = 4096 int8, 57 us each): one block of 256 x 256 per CU, n; two of 128 x 128 side by side 0.61, a single one 0.44, or
// 0.37 where no CU gets two and it may take eight waves and four buffers (1024 x 4096: 21 us against 26);
// 64 x 64, up to five side by side, 0.08 + 0.11 n.  E.g. 2048 x 4096: 37 us in 128s against 52 in 256s and 58 in 64s;
// 4096 x 4096: 59 in 256s against 69 in 128s; 512 x 4096: 19 in 64s against 26 in 128s.
// The reduction is split over blocks only where the result has tiles for at most a quarter of the CUs and each share
// keeps 8 steps of 48 at least: the partial results cost a second launch (256 x 10 x 4096, 32 steps: 9.0 us in one
// share, 7.8 in four, less than the launch's host time).  300 x 300 x 16384: 16 us in 8 shares against 37 in one;
// with more tiles, splitting lost in each case measured (128 x 4096 x 4096: 14 us against 16 in two shares).
// 256 x 256 tiles behind the last full round of the CUs would leave most of them idle for a round: where the time says
// so, these are split over up to eight shares.  That costs two launches and the partial results, 256 KB each that are
// written and read (REST_US, REST_TILE_US).  In turn: 4200 x 4200 x 16384 294 -> 247 us, 8192 x 4098 x 4096 153 -> 143,
// the training form of the latter 1143 -> 981; 8192 x 4400 x 4096, 32 steps for 64 tiles, stays as it is at 146.
TilePlan tile_plan(int M, int N, int kbytes, int pieces)
{
    const int steps = (kbytes + KSTEP - 1) / KSTEP * pieces;
    auto tiles = [&](int b) { return (int64_t)((M + b - 1) / b) * ((N + b - 1) / b); };
    auto busiest = [&](int b) { return (tiles(b) + CUS - 1) / CUS; };
    const int64_t n256 = busiest(256), n128 = busiest(128), n64 = busiest(64);
    const int64_t rest = tiles(256) % CUS;
    int rest_splits = 0;
    double t256 = (double)n256;
    if (n256 > 1 && rest > 0)
        for (int n = 2; n <= 8 && n * rest <= CUS && steps / n >= 8; n++) {
            const double t = (double)(n256 - 1) + 1.0 / n + (REST_US + REST_TILE_US * (double)(n * rest)) / (57.0 / 32 * steps);
            if (t < t256) { t256 = t; rest_splits = n; }
        }
    const double t128 = n128 == 1 ? 0.37 : 0.61 * (double)(n128 / 2) + 0.44 * (double)(n128 % 2), t64 = 0.08 + 0.11 * (double)n64;
    TilePlan pl{t256 <= t128 && t256 <= t64 ? 256 : t128 <= t64 ? 128 : 64, 1, n128 == 1, 0};
    // 64 x 32 where that still leaves no CU two tiles: the weights are then read by twice as many (from cold weights
    // 64 x 4096 x 4096: 11.4 us against 13.0; 256 x 4096 x 4096, two tiles for a CU: 15.8 against 13.5)
    const int64_t halves = (int64_t)((M + 63) / 64) * ((N + 31) / 32);
    if (pl.size == 64 && halves <= CUS) pl.size = 32;
    if (const int t = tune("REXSC_TUNE_INT8_TILE")) pl.size = t == 256 || t == 128 || t == 32 ? t : 64;
    const int64_t n = pl.size == 32 ? halves : tiles(pl.size);
    if (n > 0 && 4 * n <= CUS && steps >= 48) {
        const int64_t fill = CUS / n, keep = steps / 8;
        pl.splits = (int)(fill < keep ? fill : keep);
    }
    if (const int t = tune("REXSC_TUNE_INT8_SPLITS")) pl.splits = t;
    else if (pl.size == 256 && pl.splits == 1) pl.rest_splits = rest_splits;
    pl.splits = pl.splits > steps ? steps : pl.splits > MAX_SPLITS ? MAX_SPLITS : pl.splits;
    if (pl.splits < 1) pl.splits = 1;
    return pl;
}

template <typename Op, typename T, int BM, int BN, int WM, int WN, int STAGES>
int launch_one(const TileArgs &p, const TilePlan &pl, void *workspace, hipStream_t stream)
{
    typedef std::conditional_t<std::is_same_v<Op, OpI8>, int, float> ACC;
    const unsigned tiles = (unsigned)(((p.M + BM - 1) / BM) * (int64_t)((p.N + BN - 1) / BN));
    constexpr bool STREAM = BM == 256; // of the smaller ones a CU holds several, which hide each other's ends
    unsigned whole = pl.splits > 1 ? 0 : tiles;
    if (STREAM && pl.rest_splits > 1) whole = tiles / CUS * CUS;
    if (whole > 0) {
        const unsigned blocks = STREAM && whole > CUS ? CUS : whole;
        hipLaunchKernelGGL((tile_kernel<Op, T, BM, BN, WM, WN, STAGES, false, STREAM>), dim3(blocks), dim3(WM * WN * 64), 0, stream, p, 1,
                           0u, whole);
        REXSC_CHECK_HIP(hipGetLastError());
    }
    if (whole == tiles) return REXSC_OK;
    const unsigned count = tiles - whole;
    const int splits = whole > 0 ? pl.rest_splits : pl.splits;
    TileArgs q = p;
    q.y = workspace;
    hipLaunchKernelGGL((tile_kernel<Op, ACC, BM, BN, WM, WN, STAGES, true, false>), dim3(count * splits), dim3(WM * WN * 64), 0, stream, q,
                       splits, whole, tiles);
    REXSC_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL((join_kernel<ACC, T>), dim3(count * (BM * BN / 1024)), dim3(256), 0, stream, p, (const ACC *)workspace, splits,
                       whole, count, BM, BN);
    REXSC_CHECK_HIP(hipGetLastError());
    return REXSC_OK;
}

template <typename Op, typename T>
int launch_size(const TileArgs &p, const TilePlan &pl, void *workspace, hipStream_t stream)
{
    if (pl.size == 256) return launch_one<Op, T, 256, 256, 2, 4, 2>(p, pl, workspace, stream);
    if (pl.size == 128 && pl.alone) return launch_one<Op, T, 128, 128, 2, 4, 4>(p, pl, workspace, stream);
    if (pl.size == 128) return launch_one<Op, T, 128, 128, 2, 2, 2>(p, pl, workspace, stream);
    if (pl.size == 32) return launch_one<Op, T, 64, 32, 2, 2, 4>(p, pl, workspace, stream);
    return launch_one<Op, T, 64, 64, 2, 2, 4>(p, pl, workspace, stream);
}

} // namespace

size_t tile_product_workspace(int M, int N, int kbytes, int pieces)
{
    if (M == 0 || N == 0) return 0;
    const TilePlan pl = tile_plan(M, N, kbytes, pieces);
    const int64_t bm = pl.size == 32 ? 64 : pl.size, tiles = ((M + bm - 1) / bm) * (((int64_t)N + pl.size - 1) / pl.size);
    const int64_t parts = pl.splits > 1 ? tiles * pl.splits : tiles % CUS * pl.rest_splits; // tiles of partial results
    return (size_t)(parts * bm * pl.size) * 4;
}

int launch_tile_product(const TileArgs &p, bool f16, int out_dtype, void *workspace, const char *name, hipStream_t stream)
{
    REXSC_CHECK_ARG(p.a_stride < MAX_ROW_BYTES && p.b_stride < MAX_ROW_BYTES,
                    "int8 linear: operand rows of %zu and %zu bytes, at most %zu are supported", p.a_stride, p.b_stride,
                    MAX_ROW_BYTES - 1);
    const TilePlan pl = tile_plan(p.M, p.N, p.kbytes, p.pieces);
    // tiles are counted in 32 bits, and a launch has fewer than 2^32 threads (256 x 256 tiles, unsplit: 256 blocks)
    const int64_t rows = pl.size == 32 ? 64 : pl.size, tiles = ((p.M + rows - 1) / rows) * (((int64_t)p.N + pl.size - 1) / pl.size);
    REXSC_CHECK_ARG(tiles * pl.splits < (pl.size == 256 && pl.splits == 1 ? 1ll << 31 : 1ll << 23),
                    "int8 linear: a result of %d x %d is more than a launch holds", p.M, p.N);
    ProfScope prof(name, 2.0 * p.M * p.N * (f16 ? p.kbytes / 2 : p.kbytes) * p.pieces, stream);
    if (f16) REXSC_DTYPE_SWITCH(out_dtype, return (launch_size<OpF16, T>(p, pl, workspace, stream)));
    else REXSC_DTYPE_SWITCH(out_dtype, return (launch_size<OpI8, T>(p, pl, workspace, stream)));
}

} // namespace rexsc
