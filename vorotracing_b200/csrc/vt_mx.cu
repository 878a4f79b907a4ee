// vt_mx.cu -- elementwise operators on the microscaled formats (vt_mx.cuh):
// activation checkpoints in 8 bits, the activation's gradient from them, and
// 4-bit quantisation.
//
// All are one pass over the data, for which HBM is the floor.  Four lanes share a block of
// 32 columns, 8 columns a lane, so a lane reads and writes 16-byte words of the
// 16-bit types, and a block's largest magnitude is two shuffles away.  Magnitudes
// are compared as integers: the bits of |x| order like |x|, with infinities and
// NaN on top, which is what the exponent rule wants.
//
// Measured (1088640 x 64, binary16, SiLU): checkpoint and gradient together 134 to 149 us, 4.7 to 5.2 TB/s
// of 6.45 (floor 109 us); 4 bits and back on 1000000 x 192 binary32: 305 to 318 us, 5.5 TB/s; 8 bits to binary16 on the first
// matrix 44 us (floor 33), 4 bits to binary16 52 us (floor 27).  Neither HBM nor the issue slots are full: 38 to 46 % and
// 62 to 66 % under the counters.  The exponential and the reciprocal
// of an activation share a pipe of 16 lanes an SM, which is half busy: conversions are kept off it.  Two
// items a thread in flight cost registers and were slower (186 us); so was a grid without a loop (151 us).
#include "vt_mx.cuh"

namespace vt {

// Work item -> 8 columns of a row.  An item is a lane's share of one block.
struct MxShape {
    uint64_t rows;
    uint32_t cols, blocks;  // blocks a row
    uint64_t in_stride, out_stride;
    int word;  // bytes of the words that rows start on and hold whole (16, 8, 4 or an element's), or TURNED
    __host__ __device__ uint64_t items() const { return rows * blocks * 4u; }
};

// The row and the block in it that count blocks into the matrix lie at
__device__ __forceinline__ void mx_place(const MxShape &s, uint64_t block, uint64_t &row, uint32_t &in_row)
{
    row = block >> 32 ? block / s.blocks : (uint32_t)block / s.blocks;
    in_row = (uint32_t)(block - row * s.blocks);
}

// The 8 columns of an item, for a lane: as words of WORD bytes, as many as the row has.  Rows that only single elements
// divide are TURNED in shared memory if they are long: the warp's 8 blocks of 32 columns are read and written a block an
// access, a column a lane, where a lane that touched its own 8 columns would have every access cover 16 to 32 sectors
// (checkpoint and gradient of 25842 x 1929 in binary16: 156 us turned, 247 by elements).  In rows of few blocks the steps
// from row to row cost more than that saves (1500000 x 3 in binary32: 191 us turned, 85 by elements; 100000 x 257 in
// bfloat16, nine blocks: 129 either way).
constexpr int TURNED = 0;
constexpr uint32_t TURN_BLOCKS = 9;
template <int WORD> struct MxTurn { float4 w[WORD == TURNED ? 8 : 1][64]; };
template <int WORD> struct MxWord;
template <> struct MxWord<16> { using type = uint4; };
template <> struct MxWord<8> { using type = uint2; };
template <> struct MxWord<4> { using type = uint32_t; };
template <> struct MxWord<2> { using type = unsigned short; };

// Whether whole items are told from ragged ones, or each word has its condition: measured, checkpoint and gradient then 4 bits
// and back, 200000 x 65 in binary32 63 and 42 us against 62 and 71, 500000 x 100 in bfloat16 133 and 89 against 125 and 84.
template <int WORD, typename T> constexpr bool mx_whole_first = WORD == 16 || sizeof(T) == 4;

// Calls f(i, offset, whether it exists) for the warp's 8 blocks, a column a lane, with offsets into a matrix of that row
// stride.  Steps instead of products, and none inside a row: instructions bound the rows read this way.
template <typename F>
__device__ __forceinline__ void mx_blocks_of_warp(const MxShape &s, uint64_t t, uint64_t stride, const F &f)
{
    const uint32_t lane = threadIdx.x & 31u, last = s.blocks - 1u, tail = s.cols - last * 32u;
    const uint64_t first = t >> 5 << 3;
    uint64_t row;
    uint32_t in_row;
    mx_place(s, first, row, in_row);
    uint64_t at = row * stride + in_row * 32u + lane;
    if (in_row + 8u <= last) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) f(i, at + i * 32u, true);
    } else {
        const uint64_t after = s.rows * s.blocks - first, to_next = stride - last * 32u;
        const uint32_t left = after < 8u ? (uint32_t)after : 8u;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const bool ends = in_row == last;
            f(i, at, i < left && (!ends || lane < tail));
            at += ends ? to_next : 32u;
            in_row = ends ? 0u : in_row + 1u;
        }
    }
}

// Zeros for columns that do not exist.  Called by whole warps if TURNED.
template <int WORD, typename T>
__device__ __forceinline__ void mx_load(const MxShape &s, uint64_t t, const T *p, float *v, MxTurn<WORD> &turn)
{
    if constexpr (WORD == TURNED) {
        const uint32_t lane = threadIdx.x & 31u;
        float x[8];
        mx_blocks_of_warp(s, t, s.in_stride, [&](uint32_t i, uint64_t at, bool is) { x[i] = is ? to_f32<T>(__ldg(p + at)) : 0.0f; });
        float4 *w = turn.w[threadIdx.x / 32u];
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) reinterpret_cast<float *>(w)[i * 32u + lane] = x[i];
        __syncwarp();
        *reinterpret_cast<float4 *>(v) = w[lane * 2u];
        *reinterpret_cast<float4 *>(v + 4) = w[lane * 2u + 1u];
    } else {
        using W = typename MxWord<WORD>::type;
        constexpr uint32_t EACH = WORD / sizeof(T);
        constexpr bool WHOLE_FIRST = mx_whole_first<WORD, T>;
        uint64_t row;
        uint32_t in_row;
        mx_place(s, t >> 2, row, in_row);
        const uint32_t col = in_row * 32u + (uint32_t)(t & 3u) * 8u, have = col < s.cols ? s.cols - col : 0u;
        const W *q = reinterpret_cast<const W *>(p + row * s.in_stride + col);
        alignas(16) W w[8u / EACH];
        if (WHOLE_FIRST && have >= 8u) {
#pragma unroll
            for (uint32_t i = 0; i < 8u / EACH; ++i) w[i] = __ldg(q + i);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u / EACH; ++i) w[i] = i * EACH < have ? __ldg(q + i) : W();
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = to_f32<T>(reinterpret_cast<const T *>(w)[i]);
    }
}

// Called by whole warps if TURNED
template <int WORD, typename T>
__device__ __forceinline__ void mx_store(const MxShape &s, uint64_t t, T *p, const float *v, MxTurn<WORD> &turn)
{
    if constexpr (WORD == TURNED) {
        const uint32_t lane = threadIdx.x & 31u;
        float4 *w = turn.w[threadIdx.x / 32u];
        __syncwarp();
        w[lane * 2u] = make_float4(v[0], v[1], v[2], v[3]);
        w[lane * 2u + 1u] = make_float4(v[4], v[5], v[6], v[7]);
        __syncwarp();
        mx_blocks_of_warp(s, t, s.out_stride, [&](uint32_t i, uint64_t at, bool is) {
            if (is) p[at] = from_f32<T>(reinterpret_cast<const float *>(w)[i * 32u + lane]);
        });
    } else {
        using W = typename MxWord<WORD>::type;
        constexpr uint32_t EACH = WORD / sizeof(T);
        constexpr bool WHOLE_FIRST = mx_whole_first<WORD, T>;
        uint64_t row;
        uint32_t in_row;
        mx_place(s, t >> 2, row, in_row);
        const uint32_t col = in_row * 32u + (uint32_t)(t & 3u) * 8u, have = col < s.cols ? s.cols - col : 0u;
        W *q = reinterpret_cast<W *>(p + row * s.out_stride + col);
        alignas(16) W w[8u / EACH];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) reinterpret_cast<T *>(w)[i] = from_f32<T>(v[i]);
        if (WHOLE_FIRST && have >= 8u) {
#pragma unroll
            for (uint32_t i = 0; i < 8u / EACH; ++i) q[i] = w[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u / EACH; ++i)
                if (i * EACH < have) q[i] = w[i];
        }
    }
}

// Whether a thread's loop goes on at item t.  A warp that turns goes on as one, past the last item with it.
template <int WORD> __device__ __forceinline__ bool mx_goes_on(uint64_t t, uint64_t items)
{
    return (WORD == TURNED ? t & ~31ull : t) < items;
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

template <int WORD, typename T, int ACT>
__global__ void __launch_bounds__(256) mx8_checkpoint_kernel(MxShape s, const T *__restrict__ z,
                                                             T *__restrict__ h, int8_t *__restrict__ codes,
                                                             uint8_t *__restrict__ exps)
{
    __shared__ MxTurn<WORD> turn;
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; mx_goes_on<WORD>(t, items); t += (uint64_t)gridDim.x * 256u) {
        alignas(16) float v[8];
        mx_load<WORD>(s, t, z, v, turn);
        const uint32_t E = mx8_exponent(block_top(v));
        const f32x2 inv = both(mx8_inverse(E));
        f32x2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
        const uint2 c = make_uint2(mx8_codes(p[0], p[1], inv), mx8_codes(p[2], p[3], inv));
        if (WORD != TURNED || t < items) {
            reinterpret_cast<uint2 *>(codes)[t] = E == 255u ? make_uint2(0, 0) : c;
            if ((t & 3u) == 0) exps[t >> 2] = (uint8_t)E;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(act_value2<ACT>(p[i]));
            v[2 * i] = a.x;
            v[2 * i + 1] = a.y;
        }
        mx_store<WORD>(s, t, h, v, turn);
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

template <int WORD, typename T, int ACT>
__global__ void __launch_bounds__(256) mx8_act_bwd_kernel(MxShape s, const T *__restrict__ dh,
                                                          const int8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ exps, T *__restrict__ dz)
{
    __shared__ MxTurn<WORD> turn;
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; mx_goes_on<WORD>(t, items); t += (uint64_t)gridDim.x * 256u) {
        alignas(16) float g[8];
        f32x2 v[4];
        mx_load<WORD>(s, t, dh, g, turn);
        mx8_values(codes, exps, WORD != TURNED || t < items ? t : 0u, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(mul2(pair(g[2 * i], g[2 * i + 1]), act_slope2<ACT>(v[i])));
            g[2 * i] = a.x;
            g[2 * i + 1] = a.y;
        }
        mx_store<WORD>(s, t, dz, g, turn);
    }
}

template <int WORD, typename T>
__global__ void __launch_bounds__(256) mx8_dequantize_kernel(MxShape s, const int8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ exps, T *__restrict__ out)
{
    __shared__ MxTurn<WORD> turn;
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; mx_goes_on<WORD>(t, items); t += (uint64_t)gridDim.x * 256u) {
        f32x2 p[4];
        float v[8];
        mx8_values(codes, exps, WORD != TURNED || t < items ? t : 0u, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpair(p[i]);
            v[2 * i] = a.x;
            v[2 * i + 1] = a.y;
        }
        mx_store<WORD>(s, t, out, v, turn);
    }
}

template <int WORD, typename T>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(MxShape s, const T *__restrict__ x,
                                                           uint32_t *__restrict__ codes, uint8_t *__restrict__ exps)
{
    __shared__ MxTurn<WORD> turn;
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; mx_goes_on<WORD>(t, items); t += (uint64_t)gridDim.x * 256u) {
        alignas(16) float v[8];
        mx_load<WORD>(s, t, x, v, turn);
        const uint32_t E = mx4_exponent(block_top(v));
        const float inv = mx4_inverse(E == 255u ? 1u : E);
        f32x2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = mul2(pair(v[2 * i], v[2 * i + 1]), both(inv));
        if (WORD != TURNED || t < items) {
            codes[t] = E == 255u ? 0u : mx4_word(p);
            if ((t & 3u) == 0) exps[t >> 2] = (uint8_t)E;
        }
    }
}

template <int WORD, typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(MxShape s, const uint32_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ exps, T *__restrict__ out)
{
    __shared__ MxTurn<WORD> turn;
    const uint64_t items = s.items();
    for (uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x; mx_goes_on<WORD>(t, items); t += (uint64_t)gridDim.x * 256u) {
        const uint64_t at = WORD != TURNED || t < items ? t : 0u;
        const uint32_t c = __ldg(codes + at);
        const float sc = mx4_scale(__ldg(exps + (at >> 2)));
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mx4_value(c >> (4 * i) & 15u) * sc;
        mx_store<WORD>(s, t, out, v, turn);
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
    const uint64_t all = cols * sizeof(T) | in_stride * sizeof(T) | out_stride * sizeof(T) | (uintptr_t)in | (uintptr_t)out;
    s.word = all % 16u == 0 ? 16 : all % 8u == 0 ? 8 : all % 4u == 0 ? 4 : 2;
    if (s.word == (int)sizeof(T) && s.blocks >= TURN_BLOCKS) s.word = TURNED;
    return s;
}

// f with the word's size as a type
template <typename T, typename F> static vt_status with_word(const MxShape &s, F &&f)
{
    if (s.word == 16) return f(std::integral_constant<int, 16>());
    if (s.word == 8) return f(std::integral_constant<int, 8>());
    if (s.word == TURNED) return f(std::integral_constant<int, TURNED>());
    if constexpr (sizeof(T) == 2) {
        if (s.word == 2) return f(std::integral_constant<int, 2>());
    }
    return f(std::integral_constant<int, 4>());
}

static unsigned mx_grid(const MxShape &s)
{
    const uint64_t want = (s.items() + 255u) / 256u, most = (uint64_t)sm_count() * 32u;
    return (unsigned)(want < most ? want : most);
}

}  // namespace vt

// rows * (blocks a row) has to leave room for item counts and offsets in 64 bits
#define MX_COMMON(name)                                                                            \
    VT_REQUIRE(cols <= (1u << 30), name ": too many columns");                                     \
    if (rows == 0 || cols == 0) return VT_OK;                                                      \
    VT_REQUIRE(rows <= (1ull << 40) / vt::mx_blocks(cols), name ": too many rows")
#define MX_ELEMENTS(name, ...)                                                                     \
    VT_REQUIRE(vt::on_elements<T>(__VA_ARGS__), name ": a matrix does not start on an element")

extern "C" vt_status vt_mx8_checkpoint(const void *z, int dtype, uint64_t rows, uint32_t cols, uint64_t z_stride,
                                       int act, void *h, int8_t *codes, uint8_t *exps, vt_stream stream)
{
    MX_COMMON("vt_mx8_checkpoint");
    VT_REQUIRE(z && h && codes && exps, "vt_mx8_checkpoint: null pointer");
    VT_REQUIRE(z_stride >= cols, "vt_mx8_checkpoint: the row stride is less than a row");
    VT_REQUIRE(vt::aligned32(codes), "vt_mx8_checkpoint: codes must be 32-byte aligned");
    return vt::with_type(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        MX_ELEMENTS("vt_mx8_checkpoint", z, h);
        return vt::with_act(act, [&](auto a) {
            const vt::MxShape s = vt::mx_shape<T>(rows, cols, z, z_stride, h, cols);
            return vt::with_word<T>(s, [&](auto word) {
                vt::mx8_checkpoint_kernel<decltype(word)::value, T, decltype(a)::value><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                    s, (const T *)z, (T *)h, codes, exps);
                return vt::check_launch("mx8_checkpoint_kernel");
            });
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
    return vt::with_type(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        MX_ELEMENTS("vt_mx8_act_bwd", dh, dz);
        return vt::with_act(act, [&](auto a) {
            const vt::MxShape s = vt::mx_shape<T>(rows, cols, dh, dh_stride, dz, cols);
            return vt::with_word<T>(s, [&](auto word) {
                vt::mx8_act_bwd_kernel<decltype(word)::value, T, decltype(a)::value><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                    s, (const T *)dh, codes, exps, (T *)dz);
                return vt::check_launch("mx8_act_bwd_kernel");
            });
        });
    });
}

extern "C" vt_status vt_mx8_dequantize(const int8_t *codes, const uint8_t *exps, uint64_t rows, uint32_t cols,
                                       int dtype, void *out, vt_stream stream)
{
    MX_COMMON("vt_mx8_dequantize");
    VT_REQUIRE(codes && exps && out, "vt_mx8_dequantize: null pointer");
    VT_REQUIRE(vt::aligned32(codes), "vt_mx8_dequantize: codes must be 32-byte aligned");
    return vt::with_type(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        MX_ELEMENTS("vt_mx8_dequantize", out);
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, out, cols, out, cols);
        return vt::with_word<T>(s, [&](auto word) {
            vt::mx8_dequantize_kernel<decltype(word)::value, T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                s, codes, exps, (T *)out);
            return vt::check_launch("mx8_dequantize_kernel");
        });
    });
}

extern "C" vt_status vt_mx4_quantize(const void *x, int dtype, uint64_t rows, uint32_t cols, uint64_t x_stride,
                                     uint8_t *codes, uint8_t *exps, vt_stream stream)
{
    MX_COMMON("vt_mx4_quantize");
    VT_REQUIRE(x && codes && exps, "vt_mx4_quantize: null pointer");
    VT_REQUIRE(x_stride >= cols, "vt_mx4_quantize: the row stride is less than a row");
    VT_REQUIRE(vt::aligned16(codes), "vt_mx4_quantize: codes must be 16-byte aligned");
    return vt::with_type(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        MX_ELEMENTS("vt_mx4_quantize", x);
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, x, x_stride, x, x_stride);
        return vt::with_word<T>(s, [&](auto word) {
            vt::mx4_quantize_kernel<decltype(word)::value, T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                s, (const T *)x, (uint32_t *)codes, exps);
            return vt::check_launch("mx4_quantize_kernel");
        });
    });
}

extern "C" vt_status vt_mx4_dequantize(const uint8_t *codes, const uint8_t *exps, uint64_t rows, uint32_t cols,
                                       int dtype, void *out, vt_stream stream)
{
    MX_COMMON("vt_mx4_dequantize");
    VT_REQUIRE(codes && exps && out, "vt_mx4_dequantize: null pointer");
    VT_REQUIRE(vt::aligned16(codes), "vt_mx4_dequantize: codes must be 16-byte aligned");
    return vt::with_type(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        MX_ELEMENTS("vt_mx4_dequantize", out);
        const vt::MxShape s = vt::mx_shape<T>(rows, cols, out, cols, out, cols);
        return vt::with_word<T>(s, [&](auto word) {
            vt::mx4_dequantize_kernel<decltype(word)::value, T><<<vt::mx_grid(s), 256, 0, (cudaStream_t)stream>>>(
                s, (const uint32_t *)codes, exps, (T *)out);
            return vt::check_launch("mx4_dequantize_kernel");
        });
    });
}
