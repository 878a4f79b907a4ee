// vt_mx_tile.cuh -- a matrix product of any two operands on the CUDA cores.
#pragma once

#include "vt_mx.cuh"

namespace vt {

// One 64 x 64 tile of C(i, j) = sum_k A(i, k) B(j, k) a CTA, 4 x 4 of it a thread, operands
// staged through shared memory 16 deep.  Sums are binary32.
template <typename A, typename B, typename S>
__global__ void __launch_bounds__(256) tile_product_kernel(uint64_t I, uint32_t J, uint64_t K, A a, B b, S store)
{
    __shared__ float sa[16][65], sb[16][65];
    const uint64_t i0 = (uint64_t)blockIdx.x * 64u;
    const uint32_t j0 = blockIdx.y * 64u, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (uint64_t k0 = 0; k0 < K; k0 += 16u) {
#pragma unroll
        for (uint32_t e = threadIdx.x; e < 1024u; e += 256u) {
            // consecutive threads take consecutive elements of a row of memory
            const uint32_t ka = A::K_INNER ? e & 15u : e >> 6, ra = A::K_INNER ? e >> 4 : e & 63u;
            const uint32_t kb = B::K_INNER ? e & 15u : e >> 6, rb = B::K_INNER ? e >> 4 : e & 63u;
            sa[ka][ra] = i0 + ra < I && k0 + ka < K ? a(i0 + ra, k0 + ka) : 0.0f;
            sb[kb][rb] = j0 + rb < J && k0 + kb < K ? b(j0 + rb, k0 + kb) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    acc[p][q] = fmaf(sa[k][ty + 16u * p], sb[k][tx + 16u * q], acc[p][q]);
        __syncthreads();
    }
    for (int p = 0; p < 4; ++p)
        for (int q = 0; q < 4; ++q) {
            const uint64_t i = i0 + ty + 16u * p;
            const uint32_t j = j0 + tx + 16u * q;
            if (i < I && j < J) store(i, j, acc[p][q]);
        }
}

template <typename T, int ACT> struct StoreY {
    T *p;
    const T *bias;
    uint32_t cols;
    __device__ void operator()(uint64_t i, uint32_t j, float v) const
    {
        p[i * cols + j] = from_f32<T>(act_value<ACT>(bias ? v + to_f32<T>(bias[j]) : v));
    }
};

}  // namespace vt
