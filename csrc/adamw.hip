// sodkit — AdamW over many tensors at once, with the moments in 32 or in 8
// bits.  One launch sweeps every parameter, whatever its type.
//
// The step, t counting the steps from one, every operation in float32 and
// rounded by itself in this order (no contraction: the step gives the same
// bits as the same operations one at a time on the CPU, and so on every rank):
//
//   g = float(grad) * (grad_scale * scale)
//   m = b1*m + (1-b1)*g              v = b2*v + ((1-b2)*g)*g
//   w = w*(1-lr*wd) - (lr/(1-b1^t)) * (m / (sqrt(v)*(1/sqrt(1-b2^t)) + eps))
//
// The scalars are computed in float64 and rounded once.  A parameter of 16
// bits has a float32 master w and is its rounding; a float32 parameter is
// its own w.
//
// It is bound by memory: 28 bytes an element, 16 with moments in 8 bits.  What
// moves once a step passes the caches by (non-temporal), in whole lines:
//   24.5M bfloat16 parameters   32 bits 110 us, 6.3 TB/s   8 bits 62 us, 6.3
//   391M, float32 / bfloat16            1.72 ms, 6.4               1.00 ms, 6.3
// where a large copy reaches 5.1 to 5.5 TB/s and a fill 6.9.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"

#pragma clang fp contract(off)

namespace sodkit {
namespace aw {

constexpr int CHUNK32 = 1024;   // elements of a workgroup, moments in 32 bits
constexpr int CHUNK8 = 2048;    // and in 8
constexpr int BLOCK = 256;      // elements of an 8-bit block; tensors start at
//                                 multiples of it in the states
constexpr int ROWS = 160;       // table rows in one kernel's arguments

// what stays of a tensor, and what may move from step to step
struct Info {
    long numel;
    long state;                 // its first element in the moments
    long master;                // and in the masters, -1: float32, its own
    double wd;
    long dtype;                 // 0 float32, 1 bfloat16, 2 float16
};
struct Row {
    void *param;
    const void *grad;           // null: no gradient, the tensor is left alone
    long grad_dtype;
    bool operator==(const Row &o) const {
        return param == o.param && grad == o.grad && grad_dtype == o.grad_dtype;
    }
};
struct Rows { Row row[ROWS]; };

// Table rows travel as kernel arguments: no staging buffer to keep alive, and
// a captured graph replays its own.
__global__ void write_rows_kernel(const Rows rows, Row *__restrict__ out, int n) {
    if ((int)threadIdx.x < n) out[threadIdx.x] = rows.row[threadIdx.x];
}

struct Args {
    const Info *info;
    const Row *rows;
    const int2 *chunks;         // tensor, chunk of it
    int *steps;                 // of every chunk: a workgroup counts its own,
    //                             which spares a launch that counts for all
    float *master;
    const float *scale;         // null: 1; 0: skip
    const float *lr_t;          // null: lr
    double lr, b1, b2;
    float fb1, fc1, fb2, fc2;   // b1, 1-b1, b2, 1-b2
    float gscale, eps;
    unsigned seed;
};

// Addresses out of a table: said to be global memory, else they are loaded
// through the flat path, which takes the LDS counter too.
#define SOD_GLOBAL __attribute__((address_space(1)))
template <typename T>
SOD_DEVINL SOD_GLOBAL T *global_ptr(const void *p) {
    return (SOD_GLOBAL T *)(unsigned long)p;
}

template <typename T> struct Vec4;  // 4 elements at any element's address
template <> struct Vec4<float> {
    typedef float elem;
    typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Vec4<__hip_bfloat16> {
    typedef short elem;
    typedef short type __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct Vec4<__half> {
    typedef short elem;
    typedef short type __attribute__((ext_vector_type(4), aligned(2)));
};

// A quad of a parameter or gradient.  NT: past the caches.  FULL: all four lie
// in the tensor, and the load is the only thing that happens (converted where
// it is used, so that nothing waits for it between this and the next load).
template <typename T, bool FULL, bool NT = false>
SOD_DEVINL typename Vec4<T>::type load4(const SOD_GLOBAL T *p, long n) {
    using V = typename Vec4<T>::type;
    if (FULL || n >= 4) {
        const SOD_GLOBAL V *q = (const SOD_GLOBAL V *)p;
        return NT ? __builtin_nontemporal_load(q) : *q;
    }
    V r = {};
    for (int e = 0; e < 3; ++e)
        if (e < n) r[e] = ((const SOD_GLOBAL typename Vec4<T>::elem *)p)[e];
    return r;
}
SOD_DEVINL f32x4 to_f32(Vec4<float>::type v, float) { return v; }
template <typename T>
SOD_DEVINL f32x4 to_f32(typename Vec4<T>::type v, T) {
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = s16_as_f32<T>(v[e]);
    return r;
}

template <typename T, bool FULL>
SOD_DEVINL void store4(SOD_GLOBAL T *p, long n, f32x4 r) {
    using V = typename Vec4<T>::type;
    V v;
    if constexpr (sizeof(T) == 4) v = r;
    else v = pack4<T>(r);
    if (FULL || n >= 4) __builtin_nontemporal_store(v, (SOD_GLOBAL V *)p);
    else
        for (int e = 0; e < 3; ++e)
            if (e < n) ((SOD_GLOBAL typename Vec4<T>::elem *)p)[e] = v[e];
}

// The scalars of a step, equal over a workgroup.
struct Scalars { float rate, rbc2, keep; unsigned key; };

// The finalizer of MurmurHash3 (Appleby, public domain).
SOD_DEVINL unsigned mix32(unsigned h) {
    h ^= h >> 16;
    h *= 0x85EBCA6Bu;
    h ^= h >> 13;
    h *= 0xC2B2AE35u;
    return h ^ (h >> 16);
}

// One wave works them out for its workgroup, another one from workgroup to
// workgroup, as its SIMD has the time to give; its lanes 0 and 1 go through the
// same float64 operations with b1 and b2: the power by squaring, root and
// quotient.  A squaring doubles the relative error that it gets, so the power's
// grows with t, under t * 2^-53 (2^-33 after a million steps, where a float32
// has 2^-24).  That can still decide a rounding to float32: the CPU's path
// goes through the same products (reference._power).
SOD_DEVINL Scalars step_scalars(const Args &a, double wd, int tensor, long off) {
    __shared__ Scalars sh;
    if ((threadIdx.x >> 6) == (blockIdx.x & 3)) {
        const bool second = threadIdx.x & 1;
        unsigned t = (unsigned)a.steps[blockIdx.x] + 1u;
        double lr = a.lr_t ? (double)*a.lr_t : a.lr;
        double b = second ? a.b2 : a.b1, p = 1.0;
        for (unsigned k = t; k; k >>= 1) {
            if (k & 1) p *= b;
            b *= b;
        }
        double bc = 1.0 - p;
        float q = (float)((second ? 1.0 : lr) / (second ? sqrt(bc) : bc));
        if ((threadIdx.x & 63) == 1) sh.rbc2 = q;
        if ((threadIdx.x & 63) == 0) {
            a.steps[blockIdx.x] = (int)t;
            sh.rate = q;
            sh.keep = (float)(1.0 - lr * wd);
            unsigned k = mix32(a.seed + t * 0x9E3779B9u);
            k = mix32(k + (unsigned)tensor);
            sh.key = mix32(k + (unsigned)(off >> 32));
        }
    }
    __syncthreads();
    return sh;
}

SOD_DEVINL float moved(float w, float m, float r, float eps, const Scalars &s) {
    float den = r * s.rbc2 + eps;
    return w * s.keep - s.rate * (m / den);
}

// -------------------------------------------------------------- 32 bits
//
// A thread has one quad, so that a CU has as many workgroups as it can and
// their loads overlap: 116 us for 24.5M bfloat16 parameters, 120 with two or
// four quads, 132 through the caches.  The parameter is written non-temporally
// too (116 -> 110), and read so where it is its own master (391M float32,
// 3 % less); gradients are not, the backward pass has just left them.  The
// scalars go first: with the loads in front of their barrier tensors at odd
// addresses took 8 % more, the others 1 % less.

template <typename P, typename G, bool FULL>
SOD_DEVINL void step32(const Args &a, const Info &I, const Row &R, int tensor,
                       long off, float *m_, float *v_, float gs) {
    Scalars s = step_scalars(a, I.wd, tensor, off);
    long i = off + threadIdx.x * 4, n = I.numel - i;
    SOD_GLOBAL P *p = global_ptr<P>(R.param) + i;
    const SOD_GLOBAL G *g_ = global_ptr<G>(R.grad) + i;
    f32x4 *mp = reinterpret_cast<f32x4 *>(m_ + I.state + i);
    f32x4 *vp = reinterpret_cast<f32x4 *>(v_ + I.state + i);
    f32x4 *wp = reinterpret_cast<f32x4 *>(a.master + I.master + i);
    typename Vec4<G>::type gq;
    f32x4 m, v, w;
    if (FULL || n > 0) {
        gq = load4<G, FULL>(g_, n);
        m = __builtin_nontemporal_load(mp);
        v = __builtin_nontemporal_load(vp);
        if constexpr (sizeof(P) == 4) w = load4<P, FULL, true>(p, n);
        else w = __builtin_nontemporal_load(wp);
    }
    if (!FULL && n <= 0) return;
    f32x4 g = to_f32(gq, G());
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = g[e] * gs;
        m[e] = a.fb1 * m[e] + a.fc1 * x;
        v[e] = a.fb2 * v[e] + (a.fc2 * x) * x;
        w[e] = moved(w[e], m[e], sqrtf(v[e]), a.eps, s);
    }
    // the gap behind a tensor's end read gradients of 0 and stays 0
    __builtin_nontemporal_store(m, mp);
    __builtin_nontemporal_store(v, vp);
    if constexpr (sizeof(P) != 4) __builtin_nontemporal_store(w, wp);
    store4<P, FULL>(p, n, w);
}

// call f with a tag of the parameter's and of the gradient's type
struct F32 { using type = float; };
struct BF16 { using type = __hip_bfloat16; };
struct F16 { using type = __half; };
template <typename P, typename F>
SOD_DEVINL void by_grad(long g, F f) {
    if (g == 0) f(P(), F32());
    else if (g == 1) f(P(), BF16());
    else f(P(), F16());
}
template <typename F>
SOD_DEVINL void by_types(long p, long g, F f) {
    if (p == 0) by_grad<F32>(g, f);
    else if (p == 1) by_grad<BF16>(g, f);
    else by_grad<F16>(g, f);
}

// false: nothing to do here
SOD_DEVINL bool scaled(const Args &a, float &gs) {
    gs = a.gscale;
    if (a.scale != nullptr) {
        // 0: the gradients overflowed.  Nothing moves, the step's count neither
        float s = *a.scale;
        if (s == 0.f) return false;
        gs = gs * s;
    }
    return true;
}

__global__ void __launch_bounds__(256)
adamw32_kernel(const Args a, float *__restrict__ m, float *__restrict__ v) {
    float gs;
    int2 c = a.chunks[blockIdx.x];
    Info I = a.info[c.x];
    Row R = a.rows[c.x];
    if (R.grad == nullptr || !scaled(a, gs)) return;
    by_types(I.dtype, R.grad_dtype, [&](auto p, auto g) {
        using P = typename decltype(p)::type;
        using G = typename decltype(g)::type;
        long off = (long)c.y * CHUNK32;
        if (off + CHUNK32 <= I.numel)
            step32<P, G, true>(a, I, R, c.x, off, m, v, gs);
        else
            step32<P, G, false>(a, I, R, c.x, off, m, v, gs);
    });
}

// --------------------------------------------------------------- 8 bits
//
// A block of 256 elements, in the order of the tensor's storage, has two
// float32 scales: its largest |m| and its largest r = sqrt(v).
//   m  sign and 7 bits c: 0 is 0, else the float with the bits (c+889) << 20,
//      8 steps an octave over 15.9 octaves, 127 standing for 1
//   r  8 bits c: 0 is 0, else the float with the bits (c+1777) << 19, 16 steps
//      an octave over 15.9 octaves, 255 standing for 1
// times the scale.  Both are the top bits of a float32, so a code is a shift
// away from its value and stochastic rounding is an addition of random bits
// below the cut.
//
// Rounded to nearest, r would hardly ever move: with b2 = 0.999 a step changes
// it by 0.05 %, and half a code step is 1.6 to 3.1 %.  The random bits are a
// hash of seed, step, tensor and element.
//
// r is stored and not v: its codes then span 31.9 octaves of v, the next
// step's sqrt(v) needs no second root, and it never rounds to zero unless it
// is zero, which would leave m / eps.  A gradient that is not finite makes
// its block's scales, and so its states, not finite; so does one whose square
// is not, and the codes of such a block say nothing.
//
// Done plainly this is bound by its arithmetic, some 160 operations an element
// where memory leaves time for 115: 99 us for 24.5M bfloat16 parameters.  With
// the table, the root and the coding below it is 68, and 62 with the codes past
// the caches (and the loads in front of the scalars' barrier; behind it 1 %
// slower).  194M float32 parameters, their own masters, take 516 us read past
// the caches, 564 through them.  Quotients stay the compiler's, exact ones.

template <int BIAS, int SHIFT>
SOD_DEVINL float grid(unsigned c) {
    return c ? __uint_as_float((c + BIAS) << SHIFT) : 0.f;
}

// The values of all codes, in LDS: a lookup where shifting, adding and the
// exception for 0 take five operations and the sign two more.
struct Tables { float m[256], r[256]; };

// the largest bits over 32 lanes (floats >= 0 compare like their bits, and
// NaN above all); the exchanges stay in the vector registers
SOD_DEVINL unsigned max32lanes(unsigned v) {
#define SOD_MAX_DPP(ctrl)                                                     \
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF,    \
                                                     0xF, true))
    SOD_MAX_DPP(0xB1);      // lanes 1 apart (quad permutation 1 0 3 2)
    SOD_MAX_DPP(0x4E);      // 2 apart (2 3 0 1)
    SOD_MAX_DPP(0x141);     // the other 4 of 8 (mirrored)
    SOD_MAX_DPP(0x140);     // the other 8 of 16 (mirrored)
#undef SOD_MAX_DPP
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((unsigned)r[0], (unsigned)r[1]);
}

SOD_DEVINL unsigned sub_sat(unsigned a, unsigned b) {
    return __builtin_elementwise_sub_sat(a, b);
}

// the top bytes of four words
SOD_DEVINL unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0703u);
    unsigned hi = __builtin_amdgcn_perm(d, c, 0x0c0c0703u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

template <typename P, typename G, bool FULL>
SOD_DEVINL void step8(const Args &a, const Info &I, const Row &R, int tensor,
                      long off, unsigned char *cm_, unsigned char *cr_,
                      float2 *sc_, Tables &tab, float gs) {
    // 32 lanes have a block; lanes past the tensor's end take part with zeros.
    // A lane has 4 elements of either half: every load and store of the 32 is
    // one stretch, without which the non-temporal ones write lines in parts.
    const long first = off + (threadIdx.x >> 5) * BLOCK;    // of the block
    const bool mine = FULL || first < I.numel;
    const long i = first + (threadIdx.x & 31) * 4, n = I.numel - i;
    const long blk = (I.state + first) / BLOCK;
    SOD_GLOBAL P *p = global_ptr<P>(R.param) + i;
    const SOD_GLOBAL G *g_ = global_ptr<G>(R.grad) + i;
    unsigned *cmp = reinterpret_cast<unsigned *>(cm_ + I.state + i);
    unsigned *crp = reinterpret_cast<unsigned *>(cr_ + I.state + i);
    f32x4 *wp = reinterpret_cast<f32x4 *>(a.master + I.master + i);
    typename Vec4<G>::type g[2];
    f32x4 w[2] = {};
    unsigned cm[2] = {}, cr[2] = {};
    float2 sc = make_float2(0.f, 0.f);
#pragma unroll
    for (int h = 0; h < 2; ++h)
        g[h] = load4<G, FULL>(g_ + 128 * h, n - 128 * h);
    if (mine) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            cm[h] = __builtin_nontemporal_load(cmp + 32 * h);
            cr[h] = __builtin_nontemporal_load(crp + 32 * h);
        }
        sc = sc_[blk];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (sizeof(P) == 4)
            w[h] = load4<P, FULL, true>(p + 128 * h, n - 128 * h);
        else if (mine) w[h] = __builtin_nontemporal_load(wp + 32 * h);
    }
    {
        unsigned c = threadIdx.x;
        float x = grid<889, 20>(c & 127u);
        tab.m[c] = c & 128u ? -x : x;
        tab.r[c] = grid<1777, 19>(c);
    }
    const Scalars s = step_scalars(a, I.wd, tensor, off);

    f32x4 gf[2] = {to_f32(g[0], G()), to_f32(g[1], G())};
    float m[8], r[8], v[8];
    float mm = 0.f;
    unsigned mr = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        unsigned c = (cm[e >> 2] >> (8 * (e & 3))) & 255u;
        unsigned d = (cr[e >> 2] >> (8 * (e & 3))) & 255u;
        float m0 = tab.m[c] * sc.x, r0 = tab.r[d] * sc.y;
        float x = gf[e >> 2][e & 3] * gs;
        m[e] = a.fb1 * m0 + a.fc1 * x;
        v[e] = a.fb2 * (r0 * r0) + (a.fc2 * x) * x;
        r[e] = root_f32(v[e]);
        mm = fmaxf(mm, fabsf(m[e]));
        mr = max(mr, __float_as_uint(r[e]));
    }
    mr = max32lanes(mr);
    if (__any(mr >= 0x4F000000u)) {     // r of 2^31 or more, or not finite
        mr = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            r[e] = sqrtf(v[e]);
            mr = max(mr, __float_as_uint(fabsf(r[e])));
        }
        mr = max32lanes(mr);
    }
    float sr = __uint_as_float(mr);
    float sm = __uint_as_float(max32lanes(__float_as_uint(mm)));
    if (!(sr < INFINITY)) sm = sr;      // a NaN passes fmaxf by
    float im = 1.f / fmaxf(sm, 0x1p-100f), ir = 1.f / fmaxf(sr, 0x1p-100f);
    unsigned bm[8], br[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        unsigned h = mix32((unsigned)i + (e >> 2) * 128 + (e & 3) + s.key);
        // 1 * scale ends up at 127 << 20 and 255 << 19; the code is what is
        // left above the random bits, moved into the top byte
        unsigned u = sub_sat(__float_as_uint(fabsf(m[e]) * im), 889u << 20);
        u = ((h >> 16) << 4) + u;
        bm[e] = ((u << 4) & 0x7FFFFFFFu) | (__float_as_uint(m[e]) & 0x80000000u);
        unsigned d = sub_sat(__float_as_uint(r[e] * ir), 1777u << 19);
        d = ((h & 0xFFFFu) << 3) + d;
        // the middle one of the code, 1 and r's bits: at least 1, unless r is 0
        // (and d noise below 1); the bits of any other r are above every code
        d = max(min(d, 1u << 19), min(max(d, 1u << 19), __float_as_uint(r[e])));
        br[e] = d << 5;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        w[e >> 2][e & 3] = moved(w[e >> 2][e & 3], m[e], r[e], a.eps, s);
    if (mine) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned *x = bm + 4 * h, *y = br + 4 * h;
            __builtin_nontemporal_store(top_bytes(x[0], x[1], x[2], x[3]), cmp + 32 * h);
            __builtin_nontemporal_store(top_bytes(y[0], y[1], y[2], y[3]), crp + 32 * h);
        }
        if ((threadIdx.x & 31) == 0) sc_[blk] = make_float2(sm, sr);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (sizeof(P) != 4)
            if (mine) __builtin_nontemporal_store(w[h], wp + 32 * h);
        store4<P, FULL>(p + 128 * h, n - 128 * h, w[h]);
    }
}

__global__ void __launch_bounds__(256)
adamw8_kernel(const Args a, unsigned char *__restrict__ cm,
              unsigned char *__restrict__ cr, float2 *__restrict__ sc) {
    __shared__ Tables tab;
    float gs;
    int2 c = a.chunks[blockIdx.x];
    Info I = a.info[c.x];
    Row R = a.rows[c.x];
    if (R.grad == nullptr || !scaled(a, gs)) return;
    by_types(I.dtype, R.grad_dtype, [&](auto p, auto g) {
        using P = typename decltype(p)::type;
        using G = typename decltype(g)::type;
        long off = (long)c.y * CHUNK8;
        if (off + CHUNK8 <= I.numel)
            step8<P, G, true>(a, I, R, c.x, off, cm, cr, sc, tab, gs);
        else
            step8<P, G, false>(a, I, R, c.x, off, cm, cr, sc, tab, gs);
    });
}

// The values that the codes stand for, rounded once to bfloat16: 6 bytes an
// element, 6.0 to 6.5 TB/s.
__global__ void __launch_bounds__(256)
adamw8_decode_kernel(const unsigned char *__restrict__ cm,
                     const unsigned char *__restrict__ cr,
                     const float2 *__restrict__ sc,
                     __hip_bfloat16 *__restrict__ m,
                     __hip_bfloat16 *__restrict__ v, long places) {
    long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= places) return;
    uint2 c2 = *reinterpret_cast<const uint2 *>(cm + i);
    uint2 d2 = *reinterpret_cast<const uint2 *>(cr + i);
    float2 s = sc[i / BLOCK];
    f32x4 mo[2], vo[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        unsigned c = ((e < 4 ? c2.x : c2.y) >> (8 * (e & 3))) & 255u;
        unsigned d = ((e < 4 ? d2.x : d2.y) >> (8 * (e & 3))) & 255u;
        float x = grid<889, 20>(c & 127u) * s.x;
        float r = grid<1777, 19>(d) * s.y;
        mo[e >> 2][e & 3] = c & 128u ? -x : x;
        vo[e >> 2][e & 3] = r * r;
    }
    s16x4 a = pack4<__hip_bfloat16>(mo[0]), b = pack4<__hip_bfloat16>(mo[1]);
    s16x4 c = pack4<__hip_bfloat16>(vo[0]), d = pack4<__hip_bfloat16>(vo[1]);
    s16x8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    s16x8 y = __builtin_shufflevector(c, d, 0, 1, 2, 3, 4, 5, 6, 7);
    __builtin_nontemporal_store(x, reinterpret_cast<s16x8 *>(m + i));
    __builtin_nontemporal_store(y, reinterpret_cast<s16x8 *>(v + i));
}

// ---------------------------------------------------------------- plan

int type_code(const torch::Tensor &t, const char *what) {
    auto s = t.scalar_type();
    TORCH_CHECK(s == torch::kFloat32 || s == torch::kBFloat16 ||
                s == torch::kFloat16, "adamw: a ", what,
                " must be float32, bfloat16 or float16, got ", s);
    return s == torch::kFloat32 ? 0 : s == torch::kBFloat16 ? 1 : 2;
}

}  // namespace aw
}  // namespace sodkit

// The tables of one optimizer.  Addresses of parameters and gradients are
// looked up on every step, on the host: a gradient that moved (autograd made
// a new one) is seen, and its table written anew in front of the launch.
class AdamWPlan {
    using Row = sodkit::aw::Row;

  public:
    AdamWPlan(std::vector<torch::Tensor> params, std::vector<double> wd,
              std::vector<int64_t> state, std::vector<int64_t> master,
              torch::Tensor masters, std::vector<torch::Tensor> moments)
        : params_(std::move(params)), masters_(masters),
          moments_(std::move(moments)) {
        using namespace sodkit::aw;
        TORCH_CHECK(!params_.empty() && params_[0].is_cuda());
        dev_ = params_[0].device();
        c10::DeviceGuard guard(dev_);
        home_ = at::hip::getCurrentHIPStream();
        size_t T = params_.size();
        TORCH_CHECK(wd.size() == T && state.size() == T && master.size() == T);
        std::vector<int> chunks;
        long places = 0, mplaces = 0;
        const long chunk = moments_.size() == 2 ? CHUNK32 : CHUNK8;
        for (size_t i = 0; i < T; ++i) {
            auto &p = params_[i];
            TORCH_CHECK(p.device() == dev_,
                        "adamw: parameters must be on one device");
            Info I;
            I.numel = p.numel();
            I.state = state[i];
            I.master = master[i];
            I.wd = wd[i];
            I.dtype = type_code(p, "parameter");
            layouts_.push_back({p.scalar_type(), {}, {}});
            if (!p.is_contiguous()) {
                layouts_.back().sizes = p.sizes().vec();
                layouts_.back().strides = p.strides().vec();
            }
            long pad = (I.numel + BLOCK - 1) / BLOCK * BLOCK;
            TORCH_CHECK(I.state % BLOCK == 0 && I.state == places);
            places += pad;
            if (I.dtype != 0) {
                TORCH_CHECK(I.master == mplaces);
                mplaces += pad;
            }
            first_.push_back((int64_t)chunks.size() / 2);
            for (long off = 0; off < I.numel; off += chunk) {
                chunks.push_back((int)i);
                chunks.push_back((int)(off / chunk));
            }
            infos_.push_back(I);
        }
        n_chunks_ = (int64_t)chunks.size() / 2;
        // a launch counts its threads in 32 bits
        TORCH_CHECK(n_chunks_ < (1L << 24), "adamw: too many elements");
        TORCH_CHECK(masters_.numel() == mplaces &&
                    (moments_.size() == 2 || moments_.size() == 3));
        for (int k = 0; k < 2; ++k)
            TORCH_CHECK(moments_[k].numel() == places &&
                        moments_[k].is_contiguous() &&
                        moments_[k].device() == dev_);
        if (moments_.size() == 3)
            TORCH_CHECK(moments_[2].numel() == places / BLOCK * 2 &&
                        moments_[2].is_contiguous());
        auto i32 = torch::TensorOptions().dtype(torch::kInt32);
        info_ = torch::empty({(long)(T * sizeof(Info))},
                             i32.dtype(torch::kUInt8).device(dev_));
        write_info();
        chunks_ = torch::from_blob(chunks.data(), {(long)chunks.size()}, i32)
                      .to(dev_);
        steps_ = torch::zeros({n_chunks_}, i32.device(dev_));
        grads_.resize(T);
    }

    // Decay and step counts are set in place: a captured step reads them.  They
    // come from host memory, which a capture cannot read.
    void set_decay(std::vector<double> wd) {
        c10::DeviceGuard guard(dev_);
        TORCH_CHECK(!capturing(), "adamw: the weight decay has changed, which "
                    "cannot be captured: call update_decay() before the capture");
        TORCH_CHECK(wd.size() == infos_.size());
        for (size_t i = 0; i < wd.size(); ++i) infos_[i].wd = wd[i];
        write_info();
    }

    // where a gradient is read instead of the parameter's .grad (undefined
    // or empty: there)
    void set_grads(std::vector<torch::Tensor> grads) {
        TORCH_CHECK(grads.size() == params_.size());
        grads_ = std::move(grads);
    }

    // steps taken of every tensor; synchronizes
    std::vector<int64_t> get_steps() const {
        c10::DeviceGuard guard(dev_);
        TORCH_CHECK(!capturing(), "adamw: step counts cannot be read in a capture");
        auto s = steps_.cpu();
        std::vector<int64_t> out;
        for (size_t i = 0; i < params_.size(); ++i)
            out.push_back(infos_[i].numel ? s.data_ptr<int>()[first_[i]] : 0);
        return out;
    }

    void set_steps(std::vector<int64_t> steps) {
        c10::DeviceGuard guard(dev_);
        TORCH_CHECK(!capturing(), "adamw: step counts cannot be set in a capture");
        TORCH_CHECK(steps.size() == params_.size());
        auto s = torch::empty({n_chunks_}, torch::kInt32);
        for (size_t i = 0; i < params_.size(); ++i) {
            int64_t end = i + 1 < params_.size() ? first_[i + 1] : n_chunks_;
            for (int64_t c = first_[i]; c < end; ++c)
                s.data_ptr<int>()[c] = (int)steps[i];
        }
        steps_.copy_(s);
    }

    void step(double lr, torch::Tensor lr_t, double b1, double b2, double eps,
              double gscale, torch::Tensor scale, int64_t seed) {
        using namespace sodkit::aw;
        if (n_chunks_ == 0) return;
        at::NoGradGuard no_grad;
        c10::DeviceGuard guard(dev_);
        auto stream = at::hip::getCurrentHIPStream();
        Args a;
        a.lr_t = scalar(lr_t, "lr");
        a.scale = scalar(scale, "scale_t");
        std::vector<torch::Tensor> copies;      // until the launch is queued
        torch::Tensor rows = table(stream, copies);
        if (stream != home_ && !capturing()) {
            // whoever frees these waits for this stream too
            c10::Stream here(c10::Stream::UNSAFE, dev_, stream.id());
            for (auto *t : {&info_, &chunks_, &steps_, &masters_})
                t->record_stream(here);
            for (auto &t : moments_) t.record_stream(here);
        }
        a.info = reinterpret_cast<const Info *>(info_.data_ptr());
        a.rows = reinterpret_cast<const Row *>(rows.data_ptr());
        a.chunks = reinterpret_cast<const int2 *>(chunks_.data_ptr());
        a.steps = steps_.data_ptr<int>();
        a.master = masters_.numel() ? masters_.data_ptr<float>() : nullptr;
        a.lr = lr;
        a.b1 = b1;
        a.b2 = b2;
        a.fb1 = (float)b1;
        a.fc1 = (float)(1.0 - b1);
        a.fb2 = (float)b2;
        a.fc2 = (float)(1.0 - b2);
        a.eps = (float)eps;
        a.gscale = (float)gscale;
        a.seed = (unsigned)seed;
        if (moments_.size() == 2)
            hipLaunchKernelGGL(adamw32_kernel, dim3(n_chunks_), dim3(256), 0,
                               stream.stream(), a, moments_[0].data_ptr<float>(),
                               moments_[1].data_ptr<float>());
        else
            hipLaunchKernelGGL(adamw8_kernel, dim3(n_chunks_), dim3(256), 0,
                               stream.stream(), a,
                               moments_[0].data_ptr<unsigned char>(),
                               moments_[1].data_ptr<unsigned char>(),
                               reinterpret_cast<float2 *>(
                                   moments_[2].data_ptr<float>()));
    }

  private:
    void write_info() {
        info_.copy_(torch::from_blob(infos_.data(), {info_.numel()},
                                     torch::kUInt8));
    }

    const float *scalar(const torch::Tensor &t, const char *what) const {
        if (!t.defined() || t.numel() == 0) return nullptr;
        TORCH_CHECK(t.device() == dev_ && t.numel() == 1 &&
                    t.scalar_type() == torch::kFloat32, "adamw: ", what,
                    " must be a float32 scalar on the parameters' device");
        return t.data_ptr<float>();
    }

    torch::Tensor table(const c10::hip::HIPStream &stream,
                        std::vector<torch::Tensor> &copies) {
        using namespace sodkit::aw;
        size_t T = params_.size();
        now_.resize(T);
        auto &now = now_;
        for (size_t i = 0; i < T; ++i) {
            const auto &p = params_[i];
            const auto &l = layouts_[i];
            TORCH_CHECK(p.numel() == infos_[i].numel && p.device() == dev_ &&
                        p.scalar_type() == l.dtype &&
                        (l.strides.empty() ? p.is_contiguous()
                                           : p.sizes() == l.sizes &&
                                             same_order(p, l.strides)),
                        "adamw: parameter ", i, " has changed its size, type, "
                        "device or layout since the optimizer was made");
            const auto &g = gradient(i);
            TORCH_CHECK(!p.is_neg(), "adamw: parameter ", i, " is a negated view");
            now[i] = {p.data_ptr(), nullptr, 0};
            if (!g.defined()) continue;
            TORCH_CHECK(g.layout() == torch::kStrided && g.device() == dev_ &&
                        g.sizes() == p.sizes(), "adamw: the gradient of "
                        "parameter ", i, " must be dense, of its size and on "
                        "its device");
            now[i].grad_dtype = type_code(g, "gradient");
            bool same = (l.strides.empty() && g.is_contiguous()) ||
                        same_order(g, p.strides());
            if (!same || g.is_neg()) {
                TORCH_CHECK(g.numel() == 0 || g.storage().nbytes() != 0,
                            "adamw: the gradient of parameter ", i,
                            " has no memory");
                // elements are paired by their place in storage, and a view
                // that stands for its negation is read without the sign
                copies.push_back(torch::empty_strided(p.sizes(), p.strides(),
                                                      g.options()).copy_(g));
                now[i].grad = copies.back().data_ptr();
            } else
                now[i].grad = g.data_ptr();
        }
        if (rows_.defined() && now == host_) {
            if (capturing()) kept_ = true;
            else if (stream != made_on_)
                rows_.record_stream(c10::Stream(c10::Stream::UNSAFE, dev_,
                                                stream.id()));
            return rows_;
        }
        check_memory(now);
        check_apart(now);
        // A table that a graph reads is never written again, and one that is
        // made in a capture belongs to the graph alone.
        auto rows = torch::empty(
            {(long)(T * sizeof(Row))},
            torch::TensorOptions().dtype(torch::kUInt8).device(dev_));
        for (size_t at = 0; at < T; at += ROWS) {
            Rows r;
            int n = (int)std::min<size_t>(ROWS, T - at);
            std::copy(now.begin() + at, now.begin() + at + n, r.row);
            hipLaunchKernelGGL(write_rows_kernel, dim3(1), dim3(256), 0,
                               stream.stream(), r,
                               reinterpret_cast<Row *>(rows.data_ptr()) + at, n);
        }
        if (!capturing()) {
            if (kept_) graphs_.push_back(rows_);
            kept_ = false;
            rows_ = rows;
            host_ = now;
            made_on_ = stream;
        }
        return rows;
    }

    // Two workgroups may not step the same memory.  Looked at where parameters
    // moved since the last look.
    void check_apart(const std::vector<Row> &now) {
        bool moved = apart_.size() != now.size();
        for (size_t i = 0; !moved && i < now.size(); ++i)
            moved = apart_[i] != now[i].param;
        if (!moved) return;
        std::vector<std::pair<const char *, const char *>> spans;
        for (size_t i = 0; i < now.size(); ++i) {
            auto *p = static_cast<const char *>(now[i].param);
            size_t n = params_[i].numel() * params_[i].element_size();
            if (n) spans.push_back({p, p + n});
        }
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            TORCH_CHECK(spans[i - 1].second <= spans[i].first,
                        "adamw: parameters overlap in memory");
        apart_.resize(now.size());
        for (size_t i = 0; i < now.size(); ++i) apart_[i] = now[i].param;
    }

    // Storages may have been resized, or never been there.  An address that
    // was looked at before is good: another size has another.
    void check_memory(const std::vector<Row> &now) const {
        auto held = [](const torch::Tensor &t) {
            return t.numel() == 0 ||
                   t.storage().nbytes() >= (size_t)((t.storage_offset() + t.numel()) *
                                                    t.element_size());
        };
        for (size_t i = 0; i < now.size(); ++i) {
            if (i < host_.size() && now[i] == host_[i]) continue;
            const auto &p = params_[i], &g = gradient(i);
            TORCH_CHECK(held(p), "adamw: parameter ", i, " has no memory");
            TORCH_CHECK(!g.defined() || !same_order(g, p.strides()) || held(g),
                        "adamw: the gradient of parameter ", i, " has no memory");
        }
    }

    const torch::Tensor &gradient(size_t i) const {
        const auto &src = grads_[i];
        return src.defined() && src.numel() ? src : params_[i].grad();
    }

    // elements of equal place in storage are equal elements
    static bool same_order(const torch::Tensor &t, at::IntArrayRef strides) {
        for (int64_t d = 0; d < t.dim(); ++d)
            if (t.size(d) > 1 && t.stride(d) != strides[d]) return false;
        return true;
    }

    static bool capturing() {
        hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
        auto st = at::hip::getCurrentHIPStream().stream();
        return hipStreamIsCapturing(st, &s) == hipSuccess &&
               s != hipStreamCaptureStatusNone;
    }

    c10::Device dev_ = c10::Device(c10::kCPU);
    std::vector<torch::Tensor> params_, grads_;
    torch::Tensor masters_;
    std::vector<torch::Tensor> moments_;
    std::vector<sodkit::aw::Info> infos_;
    // a parameter's order in storage, which is its states': contiguous (no
    // sizes and strides kept) or these
    struct Layout {
        at::ScalarType dtype;
        std::vector<int64_t> sizes, strides;
    };
    std::vector<Layout> layouts_;
    std::vector<int64_t> first_;
    int64_t n_chunks_ = 0;
    torch::Tensor info_, chunks_, steps_, rows_;
    std::vector<Row> host_, now_;           // rows_' content; this step's
    std::vector<const void *> apart_;       // parameters that do not overlap
    bool kept_ = false;                     // a captured graph reads rows_
    std::vector<torch::Tensor> graphs_;     // tables that graphs read
    // the streams that the states and that rows_ were allocated on
    c10::hip::HIPStream home_ = at::hip::getDefaultHIPStream();
    c10::hip::HIPStream made_on_ = home_;
};

// {m, v} of moments in 8 bits, bfloat16, in the states' places
std::vector<torch::Tensor> adamw8_decode(torch::Tensor cm, torch::Tensor cr,
                                         torch::Tensor sc) {
    using namespace sodkit::aw;
    long n = cm.numel();
    TORCH_CHECK(cm.is_cuda() && cr.numel() == n && n % BLOCK == 0 &&
                sc.numel() == n / BLOCK * 2 && cm.is_contiguous() &&
                cr.is_contiguous() && sc.is_contiguous());
    c10::DeviceGuard guard(cm.device());
    auto opt = cm.options().dtype(torch::kBFloat16);
    auto m = torch::empty({n}, opt), v = torch::empty({n}, opt);
    if (n == 0) return {m, v};
    long g = (n / 8 + 255) / 256;
    TORCH_CHECK(g < (1L << 24), "adamw: too many elements");
    hipLaunchKernelGGL(adamw8_decode_kernel, dim3(g), dim3(256), 0,
                       at::hip::getCurrentHIPStream().stream(),
                       cm.data_ptr<unsigned char>(),
                       cr.data_ptr<unsigned char>(),
                       reinterpret_cast<const float2 *>(sc.data_ptr<float>()),
                       reinterpret_cast<__hip_bfloat16 *>(m.data_ptr()),
                       reinterpret_cast<__hip_bfloat16 *>(v.data_ptr()), n);
    return {m, v};
}

void bind_adamw(pybind11::module_ &mod) {
    pybind11::class_<AdamWPlan>(mod, "AdamWPlan")
        .def(pybind11::init<std::vector<torch::Tensor>, std::vector<double>,
                            std::vector<int64_t>, std::vector<int64_t>,
                            torch::Tensor, std::vector<torch::Tensor>>())
        .def("set_decay", &AdamWPlan::set_decay)
        .def("set_grads", &AdamWPlan::set_grads)
        .def("get_steps", &AdamWPlan::get_steps)
        .def("set_steps", &AdamWPlan::set_steps)
        .def("step", &AdamWPlan::step);
    mod.def("adamw8_decode", &adamw8_decode);
}
