// vt_mx.cu -- elementwise operators on the microscaled formats (vt_mx.cuh):
// activation checkpoints in 8 bits, the activation's gradient from them, and
// 4-bit quantisation.
//
// All are one pass over the data and bound by HBM.  Four lanes share a block of
// 32 columns, 8 columns a lane, so a lane reads and writes 16-byte words of the
// 16-bit types, and a block's largest magnitude is two shuffles away.  Magnitudes
// are compared as integers: the bits of |x| order like |x|, with infinities and
// NaN on top, which is what the exponent rule wants.
//
// Measured (1088640 x 64, binary16, SiLU): checkpoint and gradient together 134 to 141 us, 5.0 to 5.2 TB/s
// of 6.45; 4 bits and back on 1000000 x 192 binary32: 310 us, 5.6 TB/s.  The exponential and the reciprocal
// of an activation share a pipe of 16 lanes an SM, which is half busy: conversions are kept off it.  Two
// items a thread in flight cost registers and were slower (186 us); so was a grid without a loop (151 us).
// Rows of odd widths are read and written a column at a time: 25842 x 1929 in binary16 245 us a step, three
// times the floor (a block a warp, a column a lane, measured 255 us).
#include "vt_mx.cuh"

namespace vt {

// Work item -> 8 columns of a row.  An item is a lane's share of one block.
struct MxShape {
    uint64_t rows;
    uint32_t cols, blocks;  // blocks a row
    uint64_t in_stride, out_stride;
    bool vec;  // rows start on 16 bytes and hold whole groups of 8 columns
    __host__ __device__ uint64_t items() const { return rows * blocks * 4u; }
};

struct MxItem {
    uint64_t row;
    uint32_t col, n;  // first column, columns inside the row (0..8)
};

__device__ __forceinline__ MxItem mx_item(const MxShape &s, uint64_t t)
{
    const uint32_t per_row = s.blocks * 4u;
    MxItem it;
    uint32_t in_row;
    if (t >> 32) {
        it.row = t / per_row;
        in_row = (uint32_t)(t % per_row);
    } else {
        it.row = (uint32_t)t / per_row;
        in_row = (uint32_t)t % per_row;
    }
    it.col = in_row * 8u;
    it.n = it.col >= s.cols ? 0u : min(8u, s.cols - it.col);
    return it;
}

template <typename T>
__device__ __forceinline__ void mx_load(const MxShape &s, const MxItem &it, const T *p, uint64_t stride,
                                        float *v)
{
    p += it.row * stride + it.col;
    if (s.vec) {
        Vec8<T> w;
        if (it.n) w.load(p); else w.zero();
        w.unpack(v);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = i < it.n ? to_f32<T>(__ldg(p + i)) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void mx_store(const MxShape &s, const MxItem &it, T *p, const float *v)
{
    p += it.row * s.out_stride + it.col;
    if (s.vec) {
        if (!it.n) return;
        Vec8<T> w;
        w.pack(v);
        w.store(p);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i < it.n) p[i] = from_f32<T>(v[i]);
    }
}

// Bits of the largest magnitude of the block that this lane and its three neighbours share.
// Called by whole groups of four lanes: the number of items is a multiple of four, and the
// groups' lanes are in step because a block has 256 threads and items are dealt in order.
__device__ __forceinline__ uint32_t block_top(const float *v)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t lanes = 0xfu << (threadIdx.x & 28u);
    top = max(top, __shfl_xor_sync(lanes, top, 1));
    return max(top, __shfl_xor_sync(lanes, top, 2));
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) mx8_checkpoint_kernel(MxShape s, const T *__restrict__ z,
                                                             T *__restrict__ h, int8_t *__restrict__ codes,
                                                             uint8_t *__restrict__ exps)
{
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; t < items; t += (uint64_t)gridDim.x * 256u) {
        const MxItem it = mx_item(s, t);
        float v[8];
        mx_load(s, it, z, s.in_stride, v);
        const uint32_t E = mx8_exponent(block_top(v));
        const f32x2 inv = both(mx8_inverse(E));
        f32x2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
        const uint2 c = make_uint2(mx8_codes(p[0], p[1], inv), mx8_codes(p[2], p[3], inv));
        reinterpret_cast<uint2 *>(codes)[t] = E == 255u ? make_uint2(0, 0) : c;
        if ((t & 3u) == 0) exps[t >> 2] = (uint8_t)E;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(act_value2<ACT>(p[i]));
            v[2 * i] = a.x;
            v[2 * i + 1] = a.y;
        }
        mx_store(s, it, h, v);
    }
}

// The four pairs of values of item t
__device__ __forceinline__ void mx8_values(const int8_t *codes, const uint8_t *exps, uint64_t t, f32x2 *v)
{
    const uint2 c = __ldg(reinterpret_cast<const uint2 *>(codes) + t);
    const f32x2 sc = both(mx8_scale(__ldg(exps + (t >> 2))));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(code_pair((i < 2 ? c.x : c.y) ^ 0x80808080u, i % 2 * 2), sc);
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) mx8_act_bwd_kernel(MxShape s, const T *__restrict__ dh,
                                                          const int8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ exps, T *__restrict__ dz)
{
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; t < items; t += (uint64_t)gridDim.x * 256u) {
        const MxItem it = mx_item(s, t);
        float g[8];
        f32x2 v[4];
        mx_load(s, it, dh, s.in_stride, g);
        mx8_values(codes, exps, t, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(mul2(pair(g[2 * i], g[2 * i + 1]), act_slope2<ACT>(v[i])));
            g[2 * i] = a.x;
            g[2 * i + 1] = a.y;
        }
        mx_store(s, it, dz, g);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_kernel(MxShape s, const int8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ exps, T *__restrict__ out)
{
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; t < items; t += (uint64_t)gridDim.x * 256u) {
        f32x2 p[4];
        float v[8];
        mx8_values(codes, exps, t, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(p[i]);
            v[2 * i] = a.x;
            v[2 * i + 1] = a.y;
        }
        mx_store(s, mx_item(s, t), out, v);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(MxShape s, const T *__restrict__ x,
                                                           uint32_t *__restrict__ codes, uint8_t *__restrict__ exps)
{
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; t < items; t += (uint64_t)gridDim.x * 256u) {
        float v[8];
        mx_load(s, mx_item(s, t), x, s.in_stride, v);
        const uint32_t E = mx4_exponent(block_top(v));
        const float inv = mx4_inverse(E == 255u ? 1u : E);
        f32x2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = mul2(pair(v[2 * i], v[2 * i + 1]), both(inv));
        codes[t] = E == 255u ? 0u : mx4_word(p);
        if ((t & 3u) == 0) exps[t >> 2] = (uint8_t)E;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(MxShape s, const uint32_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ exps, T *__restrict__ out)
{
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; t < items; t += (uint64_t)gridDim.x * 256u) {
        const uint32_t c = __ldg(codes + t);
        const float sc = mx4_scale(__ldg(exps + (t >> 2)));
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mx4_value(c >> (4 * i) & 15u) * sc;
        mx_store(s, mx_item(s, t), out, v);
    }
}

template <typename T>
static MxShape mx_shape(uint64_t rows, uint32_t cols, const void *in, uint64_t in_stride, const void *out,
                        uint64_t out_stride)
{
    MxShape s;
    s.rows = rows;
    s.cols = cols;
    s.blocks = mx_blocks(cols);
    s.in_stride = in_stride;
    s.out_stride = out_stride;
    const uint32_t group = 16u / sizeof(T);
    s.vec = cols % 8u == 0 && in_stride % group == 0 && out_stride % group == 0 && aligned16(in) &&
            aligned16(out);
    return s;
}

static unsigned mx_grid(const MxShape &s)
{
    const uint64_t want = (s.items() + 255u) / 256u, most = (uint64_t)sm_count() * 32u;
    return (unsigned)(want < most ? want : most);
}

}  // namespace vt

// rows * (blocks a row) has to leave room for item counts in 64 bits; cols fits 32 bits by type
#define MX_COMMON(name)                                                                            \
    VT_REQUIRE(rows <= (1ull << 40), name ": too many rows");                                      \
    VT_REQUIRE(cols <= (1u << 30), name ": too many columns");                                     \
    if (rows == 0 || cols == 0) return VT_OK

extern "C" vt_status vt_mx8_checkpoint(const void *z, int dtype, uint64_t rows, uint32_t cols, uint64_t z_stride,
                                       int act, void *h, int8_t *codes, uint8_t *exps, vt_stream stream)
{
    MX_COMMON("vt_mx8_checkpoint");
    VT_REQUIRE(z && h && codes && exps, "vt_mx8_checkpoint: null pointer");
    VT_REQUIRE(z_stride >= cols, "vt_mx8_checkpoint: the row stride is less than a row");
    VT_REQUIRE(vt::aligned32(codes), "vt_mx8_checkpoint: codes must be 32-byte aligned");
    return vt::with_type(dtype, [&](auto ty) {
        using T = typename decltype(ty)::type;
        return vt::with_act(act, [&](auto a) {
            const vt::MxShape s = vt::mx_shape<T>(rows, cols, z, z_stride, h, cols);
            vt::mx8_checkpoint_kernel<T, decltype(a)::value><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                s, (const T *)z, (T *)h, codes, exps);
            return vt::check_launch("mx8_checkpoint_kernel");
        });
    });
}

extern "C" vt_status vt_mx8_act_bwd(const void *dh, int dtype, uint64_t rows, uint32_t cols, uint64_t dh_stride,
                                    const int8_t *codes, const uint8_t *exps, int act, void *dz, vt_stream stream)
{
    MX_COMMON("vt_mx8_act_bwd");
    VT_REQUIRE(dh && codes && exps && dz, "vt_mx8_act_bwd: null pointer");
    VT_REQUIRE(dh_stride >= cols, "vt_mx8_act_bwd: the row stride is less than a row");
    VT_REQUIRE(vt::aligned32(codes), "vt_mx8_act_bwd: codes must be 32-byte aligned");
    return vt::with_type(dtype, [&](auto ty) {
        using T = typename decltype(ty)::type;
        return vt::with_act(act, [&](auto a) {
            const vt::MxShape s = vt::mx_shape<T>(rows, cols, dh, dh_stride, dz, cols);
            vt::mx8_act_bwd_kernel<T, decltype(a)::value><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                s, (const T *)dh, codes, exps, (T *)dz);
            return vt::check_launch("mx8_act_bwd_kernel");
        });
    });
}

extern "C" vt_status vt_mx8_dequantize(const int8_t *codes, const uint8_t *exps, uint64_t rows, uint32_t cols,
                                       int dtype, void *out, vt_stream stream)
{
    MX_COMMON("vt_mx8_dequantize");
    VT_REQUIRE(codes && exps && out, "vt_mx8_dequantize: null pointer");
    VT_REQUIRE(vt::aligned32(codes), "vt_mx8_dequantize: codes must be 32-byte aligned");
    return vt::with_type(dtype, [&](auto ty) {
        using T = typename decltype(ty)::type;
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, out, cols, out, cols);
        vt::mx8_dequantize_kernel<T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(s, codes, exps, (T *)out);
        return vt::check_launch("mx8_dequantize_kernel");
    });
}

extern "C" vt_status vt_mx4_quantize(const void *x, int dtype, uint64_t rows, uint32_t cols, uint64_t x_stride,
                                     uint8_t *codes, uint8_t *exps, vt_stream stream)
{
    MX_COMMON("vt_mx4_quantize");
    VT_REQUIRE(x && codes && exps, "vt_mx4_quantize: null pointer");
    VT_REQUIRE(x_stride >= cols, "vt_mx4_quantize: the row stride is less than a row");
    VT_REQUIRE(vt::aligned16(codes), "vt_mx4_quantize: codes must be 16-byte aligned");
    return vt::with_type(dtype, [&](auto ty) {
        using T = typename decltype(ty)::type;
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, x, x_stride, x, x_stride);
        vt::mx4_quantize_kernel<T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
            s, (const T *)x, (uint32_t *)codes, exps);
        return vt::check_launch("mx4_quantize_kernel");
    });
}

extern "C" vt_status vt_mx4_dequantize(const uint8_t *codes, const uint8_t *exps, uint64_t rows, uint32_t cols,
                                       int dtype, void *out, vt_stream stream)
{
    MX_COMMON("vt_mx4_dequantize");
    VT_REQUIRE(codes && exps && out, "vt_mx4_dequantize: null pointer");
    VT_REQUIRE(vt::aligned16(codes), "vt_mx4_dequantize: codes must be 16-byte aligned");
    return vt::with_type(dtype, [&](auto ty) {
        using T = typename decltype(ty)::type;
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, out, cols, out, cols);
        vt::mx4_dequantize_kernel<T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
            s, (const uint32_t *)codes, exps, (T *)out);
        return vt::check_launch("mx4_dequantize_kernel");
    });
}
