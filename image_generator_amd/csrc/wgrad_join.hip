// The partial sums of a weight gradient whose pixels are split over workgroups, added in the order of the splits.
#include "common.h"

namespace {

// out[i] = sum of part[s][i] over the splits, in their order, and behind it dbias[i] (+)= the sum of its partial rows.  VEC 4: out
// is 16-byte aligned (n is a multiple of 8).  Bound by reading the parts, most of them from the last-level cache: six of 2304 x 768
// (43 MB in, 7 out) 10.5 us; 28 of 320 x 9 x 8, 23 workgroups, 7.4 us, a chain of two trips to memory (18 us with four loads at a time).
template <int VEC>
__global__ __launch_bounds__(256) void wgrad_join_kernel(const float* __restrict__ part, float* __restrict__ out, size_t n, int splits,
                                                         const float* __restrict__ bpart, float* __restrict__ dbias, int cout, int add_bias) {
    typedef float vec __attribute__((ext_vector_type(VEC)));
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (i < n) {
        const float* v = part + i;
        vec acc = *(const vec*)v;
        int s = 1;
        for (; s + 16 <= splits; s += 16) {
            vec x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = *(const vec*)(v + (s + e) * n);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc += x[e];
        }
        for (; s + 4 <= splits; s += 4) {
            vec x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = *(const vec*)(v + (s + e) * n);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc += x[e];
        }
        for (; s < splits; ++s) acc += *(const vec*)(v + s * n);
        *(vec*)(out + i) = acc;
    } else if (dbias != nullptr) {
        const size_t c0 = i - n;
        for (size_t c = c0; c < c0 + VEC && c < (size_t)cout; ++c) {
            float acc = bpart[c];
#pragma unroll 8
            for (int s = 1; s < splits; ++s) acc += bpart[(size_t)s * cout + c];
            dbias[c] = add_bias ? dbias[c] + acc : acc;
        }
    }
}

}  // namespace

int wgrad_join(const float* part, float* dw, size_t n, int splits, const float* bpart, float* dbias, int cout, int add_bias, hipStream_t st) {
    const bool vec = ((uintptr_t)dw & 15) == 0;
    const size_t threads = (n + (dbias ? cout : 0)) / (vec ? 4 : 1);         // (n and cout are multiples of 8)
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (vec) hipLaunchKernelGGL(wgrad_join_kernel<4>, grid, dim3(256), 0, st, part, dw, n, splits, bpart, dbias, cout, add_bias);
    else hipLaunchKernelGGL(wgrad_join_kernel<1>, grid, dim3(256), 0, st, part, dw, n, splits, bpart, dbias, cout, add_bias);
    return mi355_check_launch("wgrad_join_kernel");
}
