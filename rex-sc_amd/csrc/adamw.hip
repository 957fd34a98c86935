// AdamW step over many tensors at once, with 32-bit or 8-bit states.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = clamp(p (1 - lr wd) - lr/(1 - b1^t) m / (sqrt(v)/sqrt(1 - b2^t) + eps))
//
// Bound by memory: p, m, v are read and written and g is read, once each: 28 bytes per element with float32 tensors and
// 32-bit states, 16 with 8-bit states, 10 with bfloat16 tensors and 8-bit states.  One launch takes a table of tensors
// in its kernel arguments (nothing is copied to the device first, and a captured launch keeps its table), and a
// workgroup finds the tensor its chunk belongs to by bisection over the chunks' running count.
// Measured: 11.7 M float32 values in 62 tensors, 32-bit states, 59-70 us (5.6-4.7 TB/s, part of them still in the
// memory-side cache); 268 M bfloat16 values, 8-bit states, 515 us (5.2 TB/s); a copy of 1 GiB reaches 5.1 TB/s.
//
// 8-bit states: a wave holds two blocks of the 256 elements that share a scale, eight elements per lane, so a block's
// maximum is a reduction over 32 lanes and the conversion to and from e4m3 is the hardware's, two values an instruction.
// At 10 bytes an element the arithmetic counts as well: the update's quotient and root are the hardware's approximations,
// good to one step of float32, where correctly rounded ones would be some 20 instructions an element more.  What is stored
// in 8 bits is decided as the definition has it all the same (store8).  With 32-bit states memory hides correctly rounded
// ones (11.7 M values 78 us a call with either).
#include <math.h>

#include "lowp.h"
#include "profile.h"

namespace rexsc {
namespace {

constexpr int THREADS = 256;
constexpr int BLOCK = 256;                  // elements that share a scale
constexpr int CHUNK = 4096;                 // elements a workgroup takes
constexpr float E4M3_MAX = 448.f;
constexpr float E4M3_MIN = 0.001953125f;    // 2^-9, the smallest positive value
constexpr float TINY = 7.888609052210118e-31f; // 2^-100: a block below it is stored as zeros (1 / scale stays finite)
constexpr float EPS = 9.5367431640625e-07f;    // 2^-20, see store8

struct Coef { float step_size, inv_root_bc2, inv_grad_scale, skip; };

struct Hyper {
    float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, lo, hi; // decay = 1 - lr wd; lo = -inf, hi = inf: no clamp
    Coef coef;                              // where the step number is the host's
    const Coef *coef_dev;                   // else
};

// 96 x 40 and 64 x 56 bytes: the table and the rest of the arguments stay below 4 KB.
constexpr int MAX32 = 96, MAX8 = 64;
struct Table32 {
    void *p[MAX32];
    const void *g[MAX32];
    float *m[MAX32], *v[MAX32];
    unsigned n[MAX32], first[MAX32];        // elements, first chunk
    int count;
};
struct Table8 {
    void *p[MAX8];
    const void *g[MAX8];
    uint8_t *m[MAX8], *v[MAX8];
    float *ms[MAX8], *vs[MAX8];
    unsigned n[MAX8], first[MAX8];
    int count;
};

// The tensor that chunk c belongs to: the last one whose first chunk is not behind it.  Every entry has a chunk.
template <typename Table>
__device__ __forceinline__ int find(const Table &t, unsigned c)
{
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Square root to one step, below the smallest normal number too (8-bit states; where they are stored, store8 decides).
__device__ __forceinline__ float root(float v)
{
    const bool tiny = v < 7.888609052210118e-31f; // 2^-100
    return __builtin_amdgcn_sqrtf(tiny ? v * 1.8446744073709552e19f : v) * (tiny ? 2.3283064365386963e-10f : 1.f); // 2^64, 2^-32
}

// m / den to two steps.
__device__ __forceinline__ float quotient(float m, float den)
{
    // the reciprocal of a den above 2^126 would be lost, that of one below 2^-126 infinite
    const bool far = den > 1e37f, near = den < 1e-37f;
    den = far ? den * 9.313225746154785e-10f : near ? den * 1073741824.f : den; // 2^-30, 2^30
    float q = m * __builtin_amdgcn_rcpf(den);
    return far ? q * 9.313225746154785e-10f : near ? q * 1073741824.f : q;
}

// EXACT: the quotient correctly rounded.
template <bool EXACT>
__device__ __forceinline__ float move(float p, float m, float root_v, const Hyper &h, const Coef &c)
{
    const float den = fmaf(root_v, c.inv_root_bc2, h.eps), q = EXACT ? m / den : quotient(m, den);
    p = fmaf(p, h.decay, -c.step_size * q);
    // a NaN stays one: both comparisons are false
    p = p < h.lo ? h.lo : p;
    return p > h.hi ? h.hi : p;
}

template <typename T, int V>
__device__ __forceinline__ void step32(T *p, const T *g, float *m, float *v, const Hyper &h, const Coef &c)
{
    float pf[V], gf[V], mf[V], vf[V];
    load_vec<V>(pf, p);
    load_vec<V>(gf, g);
    load_vec<V>(mf, m);
    load_vec<V>(vf, v);
#pragma unroll
    for (int j = 0; j < V; j++) {
        const float gj = gf[j] * c.inv_grad_scale;
        mf[j] = fmaf(h.beta1, mf[j], h.one_minus_beta1 * gj);
        vf[j] = fmaf(h.beta2, vf[j], h.one_minus_beta2 * gj * gj);
        pf[j] = move<true>(pf[j], mf[j], sqrtf(vf[j]), h, c);
    }
    store_vec<V>(p, pf);
    store_vec<V>(m, mf);
    store_vec<V>(v, vf);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void adamw32_kernel(Table32 t, Hyper h)
{
    const Coef c = h.coef_dev ? *h.coef_dev : h.coef;
    if (c.skip != 0.f) return;
    const int k = find(t, blockIdx.x);
    const unsigned at = (blockIdx.x - t.first[k]) * (unsigned)CHUNK, left = t.n[k] - at;
    T *p = (T *)t.p[k] + at;
    const T *g = (const T *)t.g[k] + at;
    float *m = t.m[k] + at, *v = t.v[k] + at;
    const bool aligned = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)m | (uintptr_t)v) % 16) == 0;
    if (left >= CHUNK && aligned) {
#pragma unroll
        for (int i = 0; i < CHUNK / (4 * THREADS); i++) {
            const int e = (i * THREADS + threadIdx.x) * 4;
            step32<T, 4>(p + e, g + e, m + e, v + e, h, c);
        }
    } else {
        for (unsigned e = threadIdx.x; e < CHUNK && e < left; e += THREADS) step32<T, 1>(p + e, g + e, m + e, v + e, h, c);
    }
}

// Values to e4m3 and back, four to a word.
template <int V>
__device__ __forceinline__ void to_e4m3(unsigned (&q)[V / 4], const float (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
        q[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], lo, true);
    }
}
template <int V>
__device__ __forceinline__ void from_e4m3(float (&v)[V], const unsigned (&q)[V / 4])
{
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], true);
        v[4 * i] = a[0];
        v[4 * i + 1] = a[1];
        v[4 * i + 2] = b[0];
        v[4 * i + 3] = b[1];
    }
}

// A block's scale, from the bits of its largest magnitude, and its reciprocal from below and from above, see store8.  A
// block with a NaN or an infinity gets scale NaN, which its elements then become.
struct BlockScale { float scale, low, high; };
__device__ __forceinline__ BlockScale block_scale(unsigned top_bits)
{
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) return BlockScale{__uint_as_float(0x7fc00000u), 0.f, 0.f};
    if (top < TINY) return BlockScale{0.f, 0.f, 0.f};
    const float scale = top * (1.0f / E4M3_MAX), inv = 1.0f / scale;
    return BlockScale{scale, inv * (1.0f - EPS), inv * (1.0f + EPS)};
}

constexpr int EPL = 8, LANES = BLOCK / EPL; // elements of a lane, lanes of a block

__device__ __forceinline__ unsigned block_max(unsigned v)
{
#pragma unroll
    for (int s = LANES / 2; s; s >>= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)v, s, 64);
        v = v > o ? v : o;
    }
    return v;
}

struct State8 { float p[EPL], g[EPL]; unsigned m[EPL / 4], v[EPL / 4]; float ms, vs; };

// The e4m3 numbers nearest to the float32 quotients t / scale.  They are what a quotient of t and the reciprocal is
// rounded to unless a midpoint of the e4m3 grid lies within the approximations' error, so it is taken from below and from
// above, a step of 2^-20 apart that covers them (root 2^-23; reciprocal, product, and the definition's own quotient and
// root, 2^-24 each), and only a lane whose values come out differently divides (one in a few hundred).  The largest
// quotient is 448 but for that step, which rounds to 448.  ROOT: t is the square, `approx` its root, and a root that is
// not 0 is stored as 2^-9 at least.
template <bool ROOT>
__device__ __forceinline__ void store8(unsigned (&q)[EPL / 4], const float (&t)[EPL], const float (&approx)[EPL], const BlockScale &s)
{
    float low[EPL], high[EPL];
#pragma unroll
    for (int j = 0; j < EPL; j++) {
        low[j] = approx[j] * s.low;
        high[j] = approx[j] * s.high;
        if constexpr (ROOT) {
            low[j] = t[j] == 0.f ? 0.f : fmaxf(low[j], E4M3_MIN);
            high[j] = t[j] == 0.f ? 0.f : fmaxf(high[j], E4M3_MIN);
        }
    }
    unsigned other[EPL / 4], differ = s.scale != s.scale;
    to_e4m3<EPL>(q, low);
    to_e4m3<EPL>(other, high);
#pragma unroll
    for (int i = 0; i < EPL / 4; i++) differ |= q[i] ^ other[i];
    if (differ) {
#pragma unroll
        for (int j = 0; j < EPL; j++) {
            float v = (ROOT ? sqrtf(t[j]) : t[j]) / s.scale;
            if constexpr (ROOT) v = t[j] == 0.f ? 0.f : fmaxf(v, E4M3_MIN);
            // of a lost block every element is 0 (times scale NaN)
            low[j] = s.scale != s.scale ? 0.f : fminf(fmaxf(v, -E4M3_MAX), E4M3_MAX);
        }
        to_e4m3<EPL>(q, low);
    }
}

// The step of the eight elements of a lane, whose block its 32 lanes hold; afterwards x is what is to be stored.
__device__ __forceinline__ void step8(State8 &x, const Hyper &h, const Coef &c)
{
    float m[EPL], v[EPL], r[EPL];
    from_e4m3<EPL>(m, x.m);
    from_e4m3<EPL>(v, x.v);
    unsigned mt = 0, vt = 0;
#pragma unroll
    for (int j = 0; j < EPL; j++) {
        const float g = x.g[j] * c.inv_grad_scale, u = v[j] * x.vs;
        m[j] = m[j] * x.ms * h.beta1 + g * h.one_minus_beta1;
        v[j] = u * u * h.beta2 + g * g * h.one_minus_beta2;
        r[j] = root(v[j]);
        x.p[j] = move<false>(x.p[j], m[j], r[j], h, c);
        mt = max(mt, mag_bits(m[j]));
        vt = max(vt, mag_bits(v[j]));
    }
    const BlockScale ms = block_scale(block_max(mt)), vs = block_scale(mag_bits(sqrtf(__uint_as_float(block_max(vt)))));
    x.ms = ms.scale;
    x.vs = vs.scale;
    store8<false>(x.m, m, m, ms);
    store8<true>(x.v, v, r, vs);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void adamw8_kernel(Table8 t, Hyper h)
{
    constexpr int ROUNDS = CHUNK / (THREADS * EPL);
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const Coef c = h.coef_dev ? *h.coef_dev : h.coef;
    if (c.skip != 0.f) return;
    const int k = find(t, blockIdx.x);
    const unsigned at = (blockIdx.x - t.first[k]) * (unsigned)CHUNK, n = t.n[k];
    T *p = (T *)t.p[k];
    const T *g = (const T *)t.g[k];
    uint8_t *m = t.m[k], *v = t.v[k];
    float *ms = t.ms[k], *vs = t.vs[k];
    const bool aligned = (((uintptr_t)p | (uintptr_t)g) % 16 | ((uintptr_t)m | (uintptr_t)v) % 8) == 0;
    State8 x[ROUNDS];
    if (aligned && at + CHUNK <= n) { // the whole chunk is loaded before the first element is stepped
#pragma unroll
        for (int i = 0; i < ROUNDS; i++) {
            const unsigned e = at + (i * THREADS + threadIdx.x) * EPL;
            load_vec<EPL>(x[i].p, p + e);
            load_vec<EPL>(x[i].g, g + e);
            const u32x2 a = *(const u32x2 *)(m + e), b = *(const u32x2 *)(v + e);
            x[i].m[0] = a[0];
            x[i].m[1] = a[1];
            x[i].v[0] = b[0];
            x[i].v[1] = b[1];
            x[i].ms = ms[e / BLOCK];
            x[i].vs = vs[e / BLOCK];
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; i++) {
            const unsigned e = at + (i * THREADS + threadIdx.x) * EPL;
            step8(x[i], h, c);
            store_vec<EPL>(p + e, x[i].p);
            *(u32x2 *)(m + e) = u32x2{x[i].m[0], x[i].m[1]};
            *(u32x2 *)(v + e) = u32x2{x[i].v[0], x[i].v[1]};
            if (threadIdx.x % LANES == 0) {
                ms[e / BLOCK] = x[i].ms;
                vs[e / BLOCK] = x[i].vs;
            }
        }
        return;
    }
    for (int i = 0; i < ROUNDS; i++) {
        const unsigned e = at + (i * THREADS + threadIdx.x) * EPL, block = e / BLOCK;
        if (block * BLOCK >= n) continue; // all 32 lanes of a block
        State8 &y = x[0];
        y.m[0] = y.m[1] = y.v[0] = y.v[1] = 0;
#pragma unroll
        for (int j = 0; j < EPL; j++) { // elements behind the tensor are zeros, which change nothing in the block
            const bool in = e + j < n;
            y.p[j] = in ? (float)p[e + j] : 0.f;
            y.g[j] = in ? (float)g[e + j] : 0.f;
            y.m[j / 4] |= in ? (unsigned)m[e + j] << (8 * (j % 4)) : 0u;
            y.v[j / 4] |= in ? (unsigned)v[e + j] << (8 * (j % 4)) : 0u;
        }
        y.ms = ms[block];
        y.vs = vs[block];
        step8(y, h, c);
#pragma unroll
        for (int j = 0; j < EPL; j++)
            if (e + j < n) {
                p[e + j] = (T)y.p[j];
                m[e + j] = (uint8_t)(y.m[j / 4] >> (8 * (j % 4)));
                v[e + j] = (uint8_t)(y.v[j / 4] >> (8 * (j % 4)));
            }
        if (threadIdx.x % LANES == 0) {
            ms[block] = y.ms;
            vs[block] = y.vs;
        }
    }
}

// x^n in 64 bits by squaring: no call into a math library, exact to a few roundings.
__host__ __device__ inline double int_pow(double x, int64_t n)
{
    double r = 1.0;
    for (; n > 0; n >>= 1, x *= x)
        if (n & 1) r *= x;
    return r;
}

__host__ __device__ inline Coef coef_of(double lr, double beta1, double beta2, int64_t t)
{
    Coef c;
    c.step_size = (float)(lr / (1.0 - int_pow(beta1, t)));
    c.inv_root_bc2 = (float)(1.0 / sqrt(1.0 - int_pow(beta2, t)));
    c.inv_grad_scale = 1.f;
    c.skip = 0.f;
    return c;
}

// One thread: counts the step and leaves the numbers that depend on it for the launches behind it.
__global__ void adamw_prepare_kernel(int64_t *step, const float *grad_scale, const float *found_inf, double lr, double beta1,
                                     double beta2, Coef *out)
{
    const bool skip = found_inf && *found_inf != 0.f;
    const int64_t t = *step + (skip ? 0 : 1);
    Coef c = coef_of(lr, beta1, beta2, t < 1 ? 1 : t);
    if (grad_scale) c.inv_grad_scale = 1.0f / *grad_scale;
    c.skip = skip ? 1.f : 0.f;
    *step = t;
    *out = c;
}

} // namespace
} // namespace rexsc

using namespace rexsc;

extern "C" int rexsc_adamw_step(const rexsc_adamw_desc *d, const rexsc_adamw_tensor *tensors, size_t n_tensors,
                                int64_t *step_dev, const float *grad_scale, const float *found_inf, void *coef,
                                rexsc_stream_t stream_)
{
    hipStream_t stream = (hipStream_t)stream_;
    REXSC_CHECK_DESC(d, rexsc_adamw_desc);
    REXSC_CHECK_ARG(dtype_ok(d->dtype), "adamw: dtype %d is not one of float32, float16, bfloat16", d->dtype);
    REXSC_CHECK_ARG(d->state_bits == 32 || d->state_bits == 8, "adamw: states have 32 or 8 bits (got %d)", d->state_bits);
    REXSC_CHECK_ARG(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1, "adamw: betas must be in [0, 1) (got %g, %g)",
                    d->beta1, d->beta2);
    REXSC_CHECK_ARG(d->lr >= 0 && d->eps >= 0 && d->weight_decay >= 0, "adamw: lr, eps and weight_decay must not be negative "
                    "(got %g, %g, %g)", d->lr, d->eps, d->weight_decay);
    REXSC_CHECK_ARG(!d->use_clamp || d->clamp_lo <= d->clamp_hi, "adamw: clamp to [%g, %g]", d->clamp_lo, d->clamp_hi);
    REXSC_CHECK_ARG(step_dev ? coef != nullptr : d->step >= 1, "adamw: the step number counts from 1 (got %lld), or is held on "
                    "the device together with a workspace", (long long)d->step);
    REXSC_CHECK_ARG(step_dev || (!grad_scale && !found_inf), "adamw: grad_scale and found_inf need the step number on the device");
    REXSC_CHECK_ARG(tensors || n_tensors == 0, "null pointer");
    const bool eight = d->state_bits == 8;
    const size_t es = dtype_size(d->dtype);
    for (size_t i = 0; i < n_tensors; i++) {
        const rexsc_adamw_tensor &t = tensors[i];
        REXSC_CHECK_ARG(t.numel >= 0, "adamw: tensor %zu has %lld elements", i, (long long)t.numel);
        if (t.numel == 0) continue;
        REXSC_CHECK_ARG(t.param && t.grad && t.exp_avg && t.exp_avg_sq, "adamw: null pointer in tensor %zu", i);
        REXSC_CHECK_ARG(!eight || (t.exp_avg_scale && t.exp_avg_sq_scale), "adamw: 8-bit states without scales in tensor %zu", i);
        REXSC_CHECK_ARG(((uintptr_t)t.param | (uintptr_t)t.grad) % es == 0 &&
                        (eight || ((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) % 4 == 0),
                        "adamw: tensor %zu is not aligned to its element", i);
    }

    Hyper h{};
    h.beta1 = (float)d->beta1;
    h.one_minus_beta1 = (float)(1.0 - d->beta1);
    h.beta2 = (float)d->beta2;
    h.one_minus_beta2 = (float)(1.0 - d->beta2);
    h.eps = (float)d->eps;
    h.decay = (float)(1.0 - d->lr * d->weight_decay);
    h.lo = d->use_clamp ? (float)d->clamp_lo : -INFINITY;
    h.hi = d->use_clamp ? (float)d->clamp_hi : INFINITY;
    if (step_dev) {
        h.coef_dev = (const Coef *)coef;
        ProfScope prof("adamw_prepare", 64.0, stream);
        hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(1), 0, stream, step_dev, grad_scale, found_inf, d->lr,
                           d->beta1, d->beta2, (Coef *)coef);
        REXSC_CHECK_HIP(hipGetLastError());
    } else {
        h.coef = coef_of(d->lr, d->beta1, d->beta2, d->step);
    }

    Table32 t32;
    Table8 t8;
    int count = 0;
    uint64_t chunks = 0;
    double elems = 0;
    auto flush = [&]() -> int {
        if (count == 0) return REXSC_OK;
        ProfScope prof(eight ? "adamw_8bit" : "adamw", elems * (3.0 * es + (eight ? 4.0 + 16.0 / BLOCK : 16.0)), stream);
        const dim3 grid((unsigned)chunks), block(THREADS);
        if (eight) {
            t8.count = count;
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(adamw8_kernel<T>, grid, block, 0, stream, t8, h));
        } else {
            t32.count = count;
            REXSC_DTYPE_SWITCH(d->dtype, hipLaunchKernelGGL(adamw32_kernel<T>, grid, block, 0, stream, t32, h));
        }
        REXSC_CHECK_HIP(hipGetLastError());
        count = 0;
        chunks = 0;
        elems = 0;
        return REXSC_OK;
    };
    constexpr int64_t PART = (int64_t)1 << 30;     // a longer tensor becomes several entries (32-bit offsets in the kernel)
    constexpr uint64_t MAX_CHUNKS = 1u << 23;      // blocks of a launch, which has fewer than 2^32 threads
    for (size_t i = 0; i < n_tensors; i++) {
        const rexsc_adamw_tensor &t = tensors[i];
        for (int64_t at = 0; at < t.numel; at += PART) {
            const int64_t n = t.numel - at < PART ? t.numel - at : PART;
            const uint64_t c = (uint64_t)((n + CHUNK - 1) / CHUNK);
            if (count == (eight ? MAX8 : MAX32) || chunks + c > MAX_CHUNKS)
                if (int rc = flush()) return rc;
            if (eight) {
                t8.p[count] = (char *)t.param + at * es;
                t8.g[count] = (const char *)t.grad + at * es;
                t8.m[count] = (uint8_t *)t.exp_avg + at;
                t8.v[count] = (uint8_t *)t.exp_avg_sq + at;
                t8.ms[count] = t.exp_avg_scale + at / BLOCK;
                t8.vs[count] = t.exp_avg_sq_scale + at / BLOCK;
                t8.n[count] = (unsigned)n;
                t8.first[count] = (unsigned)chunks;
            } else {
                t32.p[count] = (char *)t.param + at * es;
                t32.g[count] = (const char *)t.grad + at * es;
                t32.m[count] = (float *)t.exp_avg + at;
                t32.v[count] = (float *)t.exp_avg_sq + at;
                t32.n[count] = (unsigned)n;
                t32.first[count] = (unsigned)chunks;
            }
            chunks += c;
            elems += (double)n;
            count++;
        }
    }
    return flush();
}
