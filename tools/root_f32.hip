// root_f32 (csrc/common.h) against the rounded float64 root, for every float32
// from 0 up to 2^63.  STANDALONE: hipcc -O3 --offload-arch=gfx950 -Xclang
// -target-feature -Xclang -packed-fp32-ops tools/root_f32.hip -o root_f32
#include <cstdio>

#include "../csrc/common.h"

// A float64 root rounded to float32 is the float32 root: 53 bits are more than
// 2 * 24 + 2.
__global__ void check(unsigned long long *bad, unsigned end) {
    unsigned long long n = 0;
    for (unsigned long long b = blockIdx.x * 256ull + threadIdx.x; b < end;
         b += gridDim.x * 256ull) {
        float v = __uint_as_float((unsigned)b);
        n += __float_as_uint(root_f32(v)) != __float_as_uint((float)sqrt((double)v));
    }
    if (n) atomicAdd(bad, n);
}

int main() {
    const unsigned end = 0x5F000000u;   // the bits of 2^63
    unsigned long long *d, n = 0;
    if (hipMalloc(&d, sizeof n) != hipSuccess ||
        hipMemcpy(d, &n, sizeof n, hipMemcpyHostToDevice) != hipSuccess)
        return 2;
    hipLaunchKernelGGL(check, dim3(4096), dim3(256), 0, 0, d, end);
    if (hipDeviceSynchronize() != hipSuccess ||
        hipMemcpy(&n, d, sizeof n, hipMemcpyDeviceToHost) != hipSuccess)
        return 2;
    printf("root_f32: %llu of %u differ from the float64 root, rounded\n", n, end);
    return n != 0;
}
