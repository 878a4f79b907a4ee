// vt_mx4_linear.cu -- y = act(q4(x) w4^T + b), both matrices in 4-bit microscaled blocks (vt_mx.cuh).
#include "vt_mx_tile.cuh"

namespace vt {

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

}  // namespace vt

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
