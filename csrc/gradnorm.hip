// sodkit — global gradient norm over many tensors at once, and from it the
// multiplier of the optimizer's step: clipping, the dynamic loss scale, and
// the skip of a step whose gradients overflowed.  No host round trip.
//
//   n    = prescale * sqrt(sum g^2) / L            L the loss scale, or 1
//   mult = min(1, max_norm / (n + 1e-6)) / L       0 where n is not finite
//
// Squares are summed in 64 bits: a bfloat16 gradient of 2e19 has a square
// past float32's range, which would read as an overflow that is none, and a
// sum of 1e9 terms keeps its low digits.  Every block writes one partial sum
// and a second kernel adds them in a fixed order (no atomics), so a repeated
// call gives the same bits.
//
// Bound by memory where there is much (1.56G bfloat16: 459 us, 6.8 TB/s), by
// the two dependent launches where there is little: 24.5M bfloat16 take 14 us
// where their bytes take 9 (12 and 4 us, each launch traced by itself).  A next
// chunk loaded while one is added up changes neither.

#include <torch/extension.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"

namespace sodkit {
namespace gn {

constexpr int SEGS = 160;       // tensors of one launch: 21 bytes each, and a
//                                 kernel's arguments hold 4096
constexpr int CHUNK = 8192;     // elements that a block reads at a time
constexpr int MAX_BLOCKS = 8192;
constexpr long SMALL = 16384;   // elements that one workgroup sums by itself:
//                                 111 vectors 6.9 us, in two launches 10.6

// The tensors travel as kernel arguments: nothing to allocate, to copy or to
// keep, and a captured graph has its own.
struct Segs {
    const void *ptr[SEGS];
    long numel[SEGS];
    int first[SEGS];            // chunks of the tensors before
    unsigned char dtype[SEGS];  // 0 float32, 1 bfloat16, 2 float16
    int n, chunks;
};

template <typename T> struct Vec;   // 16 bytes, at any element's address
template <> struct Vec<float> {
    typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Vec<__hip_bfloat16> {
    typedef short type __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Vec<__half> {
    typedef short type __attribute__((ext_vector_type(8), aligned(2)));
};

SOD_DEVINL float elem(const Vec<float>::type &v, int i, float) { return v[i]; }
template <typename T>
SOD_DEVINL float elem(const typename Vec<T>::type &v, int i, T) {
    return s16_as_f32<T>(v[i]);
}

template <typename T>
SOD_DEVINL double chunk_sum(const T *p, int n) {
    using V = typename Vec<T>::type;
    constexpr int W = 16 / sizeof(T);
    double a[4] = {0., 0., 0., 0.};
    if (n == CHUNK) {
#pragma unroll
        for (int k = 0; k < CHUNK / W / 256; k += 4) {
            V v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                v[u] = __builtin_nontemporal_load(reinterpret_cast<const V *>(
                    p + ((k + u) * 256 + threadIdx.x) * W));
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    double x = (double)elem(v[u], e, T());
                    a[u] = fma(x, x, a[u]);
                }
        }
    } else {
        for (int i = threadIdx.x; i < n; i += 256) {
            double x = (double)ElemTraits<T>::to_f32(p[i]);
            a[0] = fma(x, x, a[0]);
        }
    }
    return (a[0] + a[1]) + (a[2] + a[3]);
}

// sum over a block of 256; valid in thread 0
SOD_DEVINL double block_sum(double s, double *red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_down(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ void __launch_bounds__(256)
norm_partial_kernel(const Segs segs, double *__restrict__ partial) {
    __shared__ double red[4];
    double s = 0.;
    for (int c = blockIdx.x; c < segs.chunks; c += gridDim.x) {
        int lo = 0, hi = segs.n - 1;        // the last tensor with first <= c
        while (lo < hi) {
            int mid = (lo + hi + 1) >> 1;
            if (segs.first[mid] <= c) lo = mid; else hi = mid - 1;
        }
        long off = (long)(c - segs.first[lo]) * CHUNK;
        long left = segs.numel[lo] - off;
        // The comparison in 32 bits (CHUNK is a power of two): of a uniform
        // 64-bit one and its selections the compiler (ROCm 7.2) has put an
        // addition in between, whose carry the selections took for its result.
        int n = (int)(left / CHUNK) != 0 ? CHUNK : (int)left;
        const void *p = segs.ptr[lo];
        int d = segs.dtype[lo];
        if (d == 0)
            s += chunk_sum(reinterpret_cast<const float *>(p) + off, n);
        else if (d == 1)
            s += chunk_sum(reinterpret_cast<const __hip_bfloat16 *>(p) + off, n);
        else
            s += chunk_sum(reinterpret_cast<const __half *>(p) + off, n);
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

struct Final {
    double prescale, max_norm;
    float growth;               // good steps before the loss scale doubles
    float *loss_scale, *good, *skips;   // null: 1 / not moved
    float *norm, *mult;
};

SOD_DEVINL void finish(double sum, const Final &f) {
    double L = f.loss_scale ? (double)*f.loss_scale : 1.0;
    float norm = (float)(sqrt(sum) * f.prescale / L);
    bool fine = isfinite(norm);
    double m = 1.0;
    if (f.max_norm > 0) m = fmin(f.max_norm / ((double)norm + 1e-6), 1.0);
    // 0 means "skip the step": a finite norm never rounds to it
    float mult = fmaxf((float)(m / L), 1.17549435e-38f);
    *f.norm = norm;
    *f.mult = fine ? mult : 0.f;
    if (f.good) {
        float good = fine ? *f.good + 1.f : 0.f;
        bool grow = good >= f.growth;
        float s = (float)L;
        *f.loss_scale = !fine ? fmaxf(s * 0.5f, 1.f)
                              : grow ? fminf(s * 2.f, 65536.f) : s;
        *f.good = grow ? 0.f : good;
        if (!fine) *f.skips += 1.f;
    }
}

// sum over a block of 1024; valid in thread 0
SOD_DEVINL double block_sum16(double s, double *red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_down(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x < 64) {
        s = threadIdx.x < 16 ? red[threadIdx.x] : 0.;
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) s += __shfl_down(s, off, 64);
    }
    return s;
}

__global__ void __launch_bounds__(1024)
norm_final_kernel(const double *__restrict__ partial, int n, const Final f) {
    __shared__ double red[16];
    double s = 0.;
    for (int i = threadIdx.x; i < n; i += 2048) {
        double a = partial[i], b = i + 1024 < n ? partial[i + 1024] : 0.;
        s += a + b;
    }
    s = block_sum16(s, red);
    if (threadIdx.x == 0) finish(s, f);
}

// Few elements in one launch's tensors: one workgroup goes over all of them,
// flat, its threads looking their elements' tensors up in LDS, and finishes.
__global__ void __launch_bounds__(1024)
norm_small_kernel(const Segs segs, const Final f) {
    __shared__ int first[SEGS + 1];     // elements of the tensors before
    __shared__ double red[16];
    const int n = segs.n;
    if (threadIdx.x < 64) {
        // prefix sums by one wave, SEGS / 64 tensors a lane
        constexpr int K = (SEGS + 63) / 64;
        int c[K], sum = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int t = threadIdx.x * K + k;
            c[k] = t < n ? (int)segs.numel[t] : 0;
            sum += c[k];
        }
        int before = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            int o = __shfl_up(before, off, 64);
            if ((int)threadIdx.x >= off) before += o;
        }
        before -= sum;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int t = threadIdx.x * K + k;
            if (t <= n) first[t] = before;
            before += c[k];
        }
    }
    __syncthreads();
    const int total = first[n];
    double s = 0.;
    for (int i = threadIdx.x; i < total; i += 1024) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= i) lo = mid; else hi = mid - 1;
        }
        int j = i - first[lo];
        const void *p = segs.ptr[lo];
        int d = segs.dtype[lo];
        float x = d == 0 ? reinterpret_cast<const float *>(p)[j]
                  : d == 1 ? ElemTraits<__hip_bfloat16>::to_f32(
                                 reinterpret_cast<const __hip_bfloat16 *>(p)[j])
                           : ElemTraits<__half>::to_f32(
                                 reinterpret_cast<const __half *>(p)[j]);
        s = fma((double)x, (double)x, s);
    }
    s = block_sum16(s, red);
    if (threadIdx.x == 0) finish(s, f);
}

float *scalar(const torch::Tensor &t, const char *what,
              const c10::Device &dev) {
    if (!t.defined() || t.numel() == 0) return nullptr;
    TORCH_CHECK(t.device() == dev && t.scalar_type() == torch::kFloat32 &&
                t.numel() == 1, "grad_norm: ", what,
                " must be a float32 scalar on the gradients' device");
    return t.data_ptr<float>();
}

}  // namespace gn
}  // namespace sodkit

// grads: a list of tensors.  loss_scale / good / skips: float32 device scalars
// or empty; with good and skips the three move as a dynamic loss scale does.
// Returns {norm, mult}.
std::vector<torch::Tensor> grad_norm(pybind11::list list, double prescale,
                                     double max_norm, torch::Tensor loss_scale,
                                     torch::Tensor good, torch::Tensor skips,
                                     double growth) {
    using namespace sodkit::gn;
    at::NoGradGuard no_grad;
    const size_t T = list.size();
    TORCH_CHECK(T > 0, "grad_norm: no gradients");
    // read where they are: hundreds of handles cost more to copy than to use
    std::vector<const torch::Tensor *> grads(T);
    for (size_t i = 0; i < T; ++i) {
        PyObject *o = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
        TORCH_CHECK(THPVariable_Check(o), "grad_norm: gradients must be tensors");
        grads[i] = &THPVariable_Unpack(o);
    }
    auto dev = grads[0]->device();
    TORCH_CHECK(dev.is_cuda(), "grad_norm: gradients must be on the GPU");
    c10::DeviceGuard guard(dev);
    std::vector<unsigned char> codes(T);
    std::vector<torch::Tensor> copies;
    copies.reserve(T);
    for (size_t i = 0; i < T; ++i) {
        const auto &g = *grads[i];
        TORCH_CHECK(g.layout() == torch::kStrided && g.device() == dev,
                    "grad_norm: gradients must be dense and on one device");
        auto t = g.scalar_type();
        TORCH_CHECK(t == torch::kFloat32 || t == torch::kBFloat16 ||
                    t == torch::kFloat16, "grad_norm: gradients must be "
                    "float32, bfloat16 or float16, got ", t);
        codes[i] = t == torch::kFloat32 ? 0 : t == torch::kBFloat16 ? 1 : 2;
        // the order of the elements is of no consequence, holes and overlaps are
        if (!g.is_non_overlapping_and_dense()) {
            TORCH_CHECK(g.numel() == 0 || g.storage().nbytes() != 0,
                        "grad_norm: gradient ", i, " has no memory");
            copies.push_back(g.contiguous());
            grads[i] = &copies.back();
        }
    }
    auto opt = torch::TensorOptions().device(dev).dtype(torch::kFloat32);
    auto norm = torch::empty({}, opt), mult = torch::empty({}, opt);
    Final f;
    f.prescale = prescale;
    f.max_norm = max_norm;
    f.growth = (float)growth;
    f.loss_scale = scalar(loss_scale, "loss_scale", dev);
    f.good = scalar(good, "good_steps", dev);
    f.skips = scalar(skips, "skips", dev);
    TORCH_CHECK(!f.good == !f.skips && (!f.good || f.loss_scale),
                "grad_norm: good_steps and skips come together, and with a "
                "loss_scale");
    f.norm = norm.data_ptr<float>();
    f.mult = mult.data_ptr<float>();

    auto stream = at::hip::getCurrentHIPStream().stream();
    // Neighbours in one storage (the views of a bucket) are one stretch.  Those
    // of two storages are not: how the sum is grouped, and so its last bits,
    // would hang on where the allocator put them, on every rank elsewhere.
    struct Stretch {
        const char *ptr;
        long numel;
        unsigned char dtype;
        const c10::StorageImpl *storage;
    };
    std::vector<Stretch> parts;
    parts.reserve(T);
    for (size_t i = 0; i < T; ++i) {
        long n = grads[i]->numel();
        if (n == 0) continue;
        const char *p = static_cast<const char *>(grads[i]->data_ptr());
        const auto *storage = grads[i]->storage().unsafeGetStorageImpl();
        if (!parts.empty()) {
            auto &l = parts.back();
            if (l.storage == storage && l.dtype == codes[i] &&
                l.ptr + l.numel * (codes[i] == 0 ? 4 : 2) == p) {
                l.numel += n;
                continue;
            }
        }
        parts.push_back({p, n, codes[i], storage});
    }
    for (const auto &p : parts)     // a storage may have been resized
        TORCH_CHECK(p.ptr + p.numel * (p.dtype == 0 ? 4 : 2) <=
                        static_cast<const char *>(p.storage->data()) +
                            p.storage->nbytes(),
                    "grad_norm: a gradient has no memory");
    const size_t N = parts.size(), n_launch = std::max<size_t>(1, (N + SEGS - 1) / SEGS);
    torch::Tensor partial;
    double *out = nullptr;
    int blocks = 0;
    for (size_t at = 0; at < n_launch * SEGS; at += SEGS) {
        Segs s;
        s.n = 0;
        long chunks = 0, elems = 0;
        for (size_t i = at; i < N && i < at + SEGS; ++i) {
            s.ptr[s.n] = parts[i].ptr;
            s.numel[s.n] = parts[i].numel;
            s.first[s.n] = (int)chunks;
            s.dtype[s.n++] = parts[i].dtype;
            chunks += (parts[i].numel + CHUNK - 1) / CHUNK;
            elems += parts[i].numel;
            TORCH_CHECK(chunks < (1L << 31), "grad_norm: too many elements");
        }
        s.chunks = (int)chunks;
        if (n_launch == 1 && elems <= SMALL) {
            hipLaunchKernelGGL(norm_small_kernel, dim3(1), dim3(1024), 0, stream,
                               s, f);
            return {norm, mult};
        }
        if (!partial.defined()) {
            partial = torch::empty({(long)n_launch * MAX_BLOCKS},
                                   opt.dtype(torch::kFloat64));
            out = partial.data_ptr<double>();
        }
        // Up to 2048 workgroups, which are there at once, each with the same
        // number of chunks; past 16 chunks each more of them, up to MAX_BLOCKS:
        // 1.56G bfloat16 take 540 us with 2048 and 465 with 8192, 24M 16.6 us
        // with one a chunk (2993) and 14.9 with 2048.
        long most = std::min<long>(MAX_BLOCKS, std::max<long>(2048, chunks / 16));
        long each = (chunks + most - 1) / most;
        int g = (int)((chunks + each - 1) / each);
        hipLaunchKernelGGL(norm_partial_kernel, dim3(g), dim3(256), 0, stream,
                           s, out + blocks);
        blocks += g;
    }
    hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(1024), 0, stream, out,
                       blocks, f);
    return {norm, mult};
}
