// AdamW step over many tensors at once, with 32-bit or 8-bit states.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = clamp(p (1 - lr wd) - lr/(1 - b1^t) m / (sqrt(v)/sqrt(1 - b2^t) + eps))
//
// Bound by memory: p, m, v are read and written and g is read, once each: 28 bytes per element with float32 tensors and
// 32-bit states, 16 with 8-bit states, 10 with bfloat16 tensors and 8-bit states.  One launch takes a table of tensors
// in its kernel arguments (nothing is copied to the device first, and a captured launch keeps its table), and a
// workgroup finds the tensor its chunk belongs to by bisection over the chunks' running count.
//
// 8-bit states: a wave holds the 256 elements that share a scale, four per lane, so the block's maximum is a reduction
// over the lanes and the conversion to and from e4m3 is the hardware's, two values an instruction.
#include <math.h>

#include "lowp.h"
#include "profile.h"

namespace rexsc {
namespace {

constexpr int THREADS = 256;
constexpr int BLOCK = 256;                  // elements that share a scale
constexpr int CHUNK = 4096;                 // elements a workgroup takes: four vectors of four per thread
constexpr float E4M3_MAX = 448.f;
constexpr float E4M3_MIN = 0.001953125f;    // 2^-9, the smallest positive value
constexpr float TINY = 7.888609052210118e-31f; // 2^-100: a block below it is stored as zeros (1 / scale stays finite)

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

__device__ __forceinline__ float move(float p, float m, float root_v, const Hyper &h, const Coef &c)
{
    const float den = fmaf(root_v, c.inv_root_bc2, h.eps);
    p = p * h.decay - c.step_size * (m / den);
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
        pf[j] = move(pf[j], mf[j], sqrtf(vf[j]), h, c);
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

// Four values to e4m3 and back.
__device__ __forceinline__ unsigned to_e4m3(const float (&v)[4])
{
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
}
__device__ __forceinline__ void from_e4m3(float (&v)[4], unsigned q)
{
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
}

// Scale of a block whose largest magnitude has these bits, and what its elements are multiplied by.  A block with a
// NaN or an infinity gets scale NaN, which its elements then become.
__device__ __forceinline__ void block_scale(unsigned top_bits, float &scale, float &inv)
{
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) { scale = __uint_as_float(0x7fc00000u); inv = 0.f; }
    else if (top < TINY) { scale = 0.f; inv = 0.f; }
    else { scale = top / E4M3_MAX; inv = E4M3_MAX / top; }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void adamw8_kernel(Table8 t, Hyper h)
{
    const Coef c = h.coef_dev ? *h.coef_dev : h.coef;
    if (c.skip != 0.f) return;
    const int k = find(t, blockIdx.x);
    const unsigned at = (blockIdx.x - t.first[k]) * (unsigned)CHUNK, n = t.n[k];
    T *p = (T *)t.p[k];
    const T *g = (const T *)t.g[k];
    uint8_t *m = t.m[k], *v = t.v[k];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const bool aligned = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)m | (uintptr_t)v) % 4) == 0;
#pragma unroll
    for (int i = 0; i < CHUNK / BLOCK / (THREADS / 64); i++) {
        const unsigned b0 = at + (unsigned)(i * (THREADS / 64) + wave) * BLOCK;
        if (b0 >= n) continue; // wave-uniform
        const unsigned e = b0 + lane * 4, block = b0 / BLOCK;
        float pf[4], gf[4], mf[4], vf[4];
        const bool whole = aligned && b0 + BLOCK <= n;
        if (whole) {
            load_vec<4>(pf, p + e);
            load_vec<4>(gf, g + e);
            from_e4m3(mf, *(const unsigned *)(m + e));
            from_e4m3(vf, *(const unsigned *)(v + e));
        } else {
            unsigned mq = 0, vq = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool in = e + j < n;
                pf[j] = in ? (float)p[e + j] : 0.f;
                gf[j] = in ? (float)g[e + j] : 0.f;
                mq |= in ? (unsigned)m[e + j] << (8 * j) : 0u;
                vq |= in ? (unsigned)v[e + j] << (8 * j) : 0u;
            }
            from_e4m3(mf, mq);
            from_e4m3(vf, vq);
        }
        const float ms = t.ms[k][block], vs = t.vs[k][block];
        float root[4];
        unsigned mt = 0, vt = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float gj = gf[j] * c.inv_grad_scale, u = vf[j] * vs;
            mf[j] = fmaf(h.beta1, mf[j] * ms, h.one_minus_beta1 * gj);
            root[j] = sqrtf(fmaf(h.beta2, u * u, h.one_minus_beta2 * gj * gj));
            pf[j] = move(pf[j], mf[j], root[j], h, c);
            mt = max(mt, mag_bits(mf[j]));
            vt = max(vt, mag_bits(root[j]));
        }
        float ms_new, mi, vs_new, vi;
        block_scale(wave_max(mt), ms_new, mi);
        block_scale(wave_max(vt), vs_new, vi);
        float mq[4], vq[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // 448 / top * top may end one rounding above 448; of a lost block every element is 0 (times scale NaN)
            mq[j] = mi == 0.f ? 0.f : fminf(fmaxf(mf[j] * mi, -E4M3_MAX), E4M3_MAX);
            vq[j] = vi == 0.f || root[j] == 0.f ? 0.f : fminf(fmaxf(root[j] * vi, E4M3_MIN), E4M3_MAX);
        }
        const unsigned mw = to_e4m3(mq), vw = to_e4m3(vq);
        if (whole) {
            store_vec<4>(p + e, pf);
            *(unsigned *)(m + e) = mw;
            *(unsigned *)(v + e) = vw;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (e + j < n) {
                    p[e + j] = (T)pf[j];
                    m[e + j] = (uint8_t)(mw >> (8 * j));
                    v[e + j] = (uint8_t)(vw >> (8 * j));
                }
        }
        if (lane == 0) {
            t.ms[k][block] = ms_new;
            t.vs[k][block] = vs_new;
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
    constexpr uint64_t MAX_CHUNKS = 1u << 30;      // blocks of a launch
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
