// vt_mx_linear.cu -- matrix products on the microscaled formats (vt_mx.cuh):
//   vt_mx8_linear_bwd   gradients of y = act(z) W^T + b from an 8-bit checkpoint of z
//                       dz = (dy W) * act'(z8), dW = dy^T act(z8), db = column sums of dy
//   vt_mx4_linear       y = act(q4(x) w4^T + b), both matrices in 4 bits
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

template <typename T, bool KIN> struct Rows {  // element (i, k) of a row-major matrix, or of its transpose
    static constexpr bool K_INNER = KIN;
    const T *p;
    uint64_t stride;
    __device__ float operator()(uint64_t i, uint64_t k) const
    {
        return to_f32<T>(__ldg(p + (KIN ? i * stride + k : k * stride + i)));
    }
};

template <int ACT> struct Checkpoint8 {  // act(z8) at (column, row)
    static constexpr bool K_INNER = false;
    const int8_t *codes;
    const uint8_t *exps;
    uint32_t blocks;
    __device__ float z(uint64_t row, uint32_t col) const
    {
        return (float)codes[row * blocks * MX_BLOCK + col] * mx8_scale(exps[row * blocks + col / MX_BLOCK]);
    }
    __device__ float operator()(uint64_t col, uint64_t row) const { return act_value<ACT>(z(row, (uint32_t)col)); }
};

template <typename T, int ACT> struct StoreDz {
    Checkpoint8<ACT> ckpt;
    T *p;
    uint32_t cols;
    __device__ void operator()(uint64_t i, uint32_t j, float v) const
    {
        p[i * cols + j] = from_f32<T>(v * act_slope<ACT>(ckpt.z(i, j)));
    }
};

template <typename T, int ACT> struct StoreY {
    T *p;
    const T *bias;
    uint32_t cols;
    __device__ void operator()(uint64_t i, uint32_t j, float v) const
    {
        p[i * cols + j] = from_f32<T>(act_value<ACT>(bias ? v + to_f32<T>(bias[j]) : v));
    }
};

template <typename T> __global__ void column_sum_kernel(const T *p, uint64_t rows, uint32_t cols, uint64_t stride, T *out)
{
    __shared__ float part[256];
    float v = 0.0f;
    for (uint64_t i = threadIdx.x; i < rows; i += 256u) v += to_f32<T>(p[i * stride + blockIdx.x]);
    part[threadIdx.x] = v;
    __syncthreads();
    for (int n = 128; n; n >>= 1) {
        if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = from_f32<T>(part[0]);
}

template <bool QUANT, typename T> struct Matrix4 {  // values of a 4-bit matrix at (row, column)
    static constexpr bool K_INNER = true;
    const uint8_t *codes, *exps;
    uint32_t blocks;
    __device__ float operator()(uint64_t row, uint64_t col) const
    {
        const uint32_t c = codes[(row * blocks * MX_BLOCK + col) / 2u];
        return mx4_value(c >> (4u * (col & 1u)) & 15u) * mx4_scale(exps[row * blocks + col / MX_BLOCK]);
    }
};

template <typename T>
static vt_status zero(T *p, uint64_t n, cudaStream_t stream)
{
    if (!p || !n) return VT_OK;
    cudaError_t e = cudaMemsetAsync(p, 0, n * sizeof(T), stream);
    return e == cudaSuccess ? VT_OK : set_error(VT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
}

}  // namespace vt

extern "C" uint64_t vt_mx8_linear_bwd_workspace_bytes(uint64_t, uint32_t, uint32_t) { return 0; }

extern "C" vt_status vt_mx8_linear_bwd(const void *dy, uint64_t dy_stride, const void *weight, uint64_t weight_stride,
                                       int dtype, uint64_t rows, uint32_t cols, uint32_t outs, const int8_t *codes,
                                       const uint8_t *exps, int act, void *dz, void *dw, void *db, void *workspace,
                                       uint64_t workspace_bytes, uint32_t *err, vt_stream stream)
{
    VT_REQUIRE(rows <= (1ull << 31) - 256, "vt_mx8_linear_bwd: too many rows");
    VT_REQUIRE(cols <= (1u << 20) && outs <= (1u << 20), "vt_mx8_linear_bwd: layer too wide");
    cudaStream_t st = (cudaStream_t)stream;
    return vt::with_type16(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        if (rows == 0 || cols == 0 || outs == 0) {
            if (vt_status s = vt::zero((T *)dz, rows * cols, st)) return s;
            if (vt_status s = vt::zero((T *)dw, (uint64_t)outs * cols, st)) return s;
            if (rows == 0 || outs == 0) return vt::zero((T *)db, outs, st);
        }
        VT_REQUIRE(dy && (cols == 0 || (weight && codes && exps)), "vt_mx8_linear_bwd: null pointer");
        VT_REQUIRE(dy_stride >= outs && weight_stride >= cols,
                   "vt_mx8_linear_bwd: a row stride is less than a row");
        return vt::with_act(act, [&](auto a) -> vt_status {
            constexpr int ACT = decltype(a)::value;
            const vt::Checkpoint8<ACT> ckpt{codes, exps, vt::mx_blocks(cols)};
            if (dz && cols) {
                const dim3 grid((unsigned)((rows + 63) / 64), (cols + 63) / 64);
                vt::tile_product_kernel<<<grid, 256, 0, st>>>(
                    rows, cols, (uint64_t)outs, vt::Rows<T, true>{(const T *)dy, dy_stride},
                    vt::Rows<T, false>{(const T *)weight, weight_stride}, vt::StoreDz<T, ACT>{ckpt, (T *)dz, cols});
            }
            if (dw && cols) {
                const dim3 grid((outs + 63) / 64, (cols + 63) / 64);
                vt::tile_product_kernel<<<grid, 256, 0, st>>>(
                    (uint64_t)outs, cols, rows, vt::Rows<T, false>{(const T *)dy, dy_stride}, ckpt,
                    vt::StoreY<T, vt::ACT_IDENTITY>{(T *)dw, nullptr, cols});
            }
            if (db) vt::column_sum_kernel<T><<<outs, 256, 0, st>>>((const T *)dy, rows, outs, dy_stride, (T *)db);
            return vt::check_launch("vt_mx8_linear_bwd");
        });
    });
}

extern "C" uint64_t vt_mx4_linear_workspace_bytes(uint64_t rows, uint32_t cols, uint32_t)
{
    const uint64_t blocks = vt::mx_blocks(cols);
    return rows * blocks * 16u + (rows * blocks + 15u) / 16u * 16u;
}

extern "C" vt_status vt_mx4_linear(const void *x, uint64_t x_stride, int dtype, uint64_t rows, uint32_t cols,
                                   uint32_t outs, const uint8_t *codes, const uint8_t *exps, const void *bias, int act,
                                   void *y, void *workspace, uint64_t workspace_bytes, uint32_t *err, vt_stream stream)
{
    VT_REQUIRE(rows <= (1ull << 31) - 256, "vt_mx4_linear: too many rows");
    VT_REQUIRE(cols <= (1u << 20) && outs <= (1u << 20), "vt_mx4_linear: layer too wide");
    if (rows == 0 || outs == 0) return VT_OK;
    VT_REQUIRE(y && (cols == 0 || (x && codes && exps)), "vt_mx4_linear: null pointer");
    VT_REQUIRE(x_stride >= cols, "vt_mx4_linear: the row stride is less than a row");
    VT_REQUIRE(workspace_bytes >= vt_mx4_linear_workspace_bytes(rows, cols, outs) && (workspace || cols == 0) &&
                   vt::aligned16(workspace),
               "vt_mx4_linear: workspace too small or not 16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    const uint32_t blocks = vt::mx_blocks(cols);
    uint8_t *xc = (uint8_t *)workspace, *xe = xc + rows * blocks * 16u;
    return vt::with_type16(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        if (vt_status s = vt_mx4_quantize(x, dtype, rows, cols, x_stride, xc, xe, stream)) return s;
        return vt::with_act(act, [&](auto a) -> vt_status {
            const dim3 grid((unsigned)((rows + 63) / 64), (outs + 63) / 64);
            vt::tile_product_kernel<<<grid, 256, 0, st>>>(
                rows, outs, (uint64_t)cols, vt::Matrix4<true, T>{xc, xe, blocks},
                vt::Matrix4<false, T>{codes, exps, blocks},
                vt::StoreY<T, decltype(a)::value>{(T *)y, (const T *)bias, outs});
            return vt::check_launch("vt_mx4_linear");
        });
    });
}
