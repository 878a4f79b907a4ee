// vt_mx_rows.cuh -- row-major 16-bit matrices as TMA sources.
#pragma once

#include "vt_mx.cuh"
#include "vt_tc.cuh"

namespace vt {

inline uint64_t align_up(uint64_t n, uint64_t a) { return (n + a - 1) / a * a; }

// Rows of a matrix copied to a pitch of whole 16-byte words, which TMA asks for.
template <typename T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T *__restrict__ src, uint64_t rows, uint32_t cols, uint64_t stride,
                                                       T *__restrict__ dst, uint32_t pitch)
{
    const uint32_t words = pitch / 8u;
    const uint64_t n = rows * words;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256u) {
        const uint64_t row = n >> 32 ? i / words : (uint32_t)i / words;  // a 64-bit division takes some hundred instructions
        const uint32_t col = (uint32_t)(i - row * words) * 8u;
        const T *p = src + row * stride + col;
        Vec8<T> v;
        T *e = reinterpret_cast<T *>(v.w);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) e[k] = col + k < cols ? p[k] : from_f32<T>(0.0f);
        v.store(dst + row * pitch + col);
    }
}


// Whether a matrix's rows start on 16 bytes, which TMA asks for.
template <typename T> inline bool whole_words(const void *p, uint64_t stride) { return stride * sizeof(T) % 16u == 0 && aligned16(p); }

// p and its row stride, or a copy's whose rows are whole 16-byte words where p's are not.
template <typename T>
static vt_status whole_rows(const void *&p, uint64_t &stride, uint64_t rows, uint32_t cols, void *copy, cudaStream_t stream)
{
    if (!whole_words<T>(p, stride)) {
        const uint32_t to = (uint32_t)align_up(cols, 8);
        const uint64_t items = rows * (to / 8u), want = (items + 255u) / 256u;
        pad_rows_kernel<T><<<(unsigned)(want < 4096u ? want : 4096u), 256, 0, stream>>>((const T *)p, rows, cols, stride, (T *)copy, to);
        p = copy;
        stride = to;
        return check_launch("pad_rows_kernel");
    }
    return VT_OK;
}
template <typename T> constexpr CUtensorMapDataType tma_type()
{
    return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}
template <typename T>
static vt_status map_rows(CUtensorMap *map, const void *p, uint64_t stride, uint64_t rows, uint64_t cols, uint32_t box_rows)
{
    return tc::make_map(map, tma_type<T>(), p, rows, cols, stride * sizeof(T), box_rows, 64);
}

}  // namespace vt
