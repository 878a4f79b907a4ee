// vt_tc.cu -- host side of the tensor-core plumbing: TMA tensor maps; a wait that runs out; error words.
#include "vt_tc.cuh"

namespace vt {
namespace tc {

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's entry point, looked up once: the library does not link against the driver.
static EncodeTiled encode_tiled()
{
    static const EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (EncodeTiled)p;
    }();
    return f;
}

static vt_status encode_map(CUtensorMap *map, CUtensorMapDataType type, const void *p, int rank, const cuuint64_t *dims,
                            const cuuint64_t *strides, const cuuint32_t *box, bool swizzle)
{
    const EncodeTiled encode = encode_tiled();
    if (!encode) return set_error(VT_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint32_t one[3] = {1, 1, 1};
    const auto make = [&] {
        return encode(map, type, rank, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = make();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a thread that has made no runtime call yet, as autograd's
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = make();
    }
    if (r != CUDA_SUCCESS)
        return set_error(VT_ERR_CUDA, "cuTensorMapEncodeTiled: error %d (%llu x %llu, pitch %llu)", (int)r,
                         (unsigned long long)dims[1], (unsigned long long)dims[0], (unsigned long long)strides[0]);
    return VT_OK;
}

vt_status make_map(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t rows, uint64_t cols,
                   uint64_t pitch, uint32_t box_rows, uint32_t box_cols, bool swizzle)
{
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_cols, box_rows};
    return encode_map(map, type, p, 2, dims, strides, box, swizzle);
}

vt_status make_chunk_map(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t rows, uint32_t chunks,
                         uint64_t pitch, uint32_t box_rows, uint32_t box_cols, uint32_t bytes)
{
    const cuuint64_t dims[3] = {box_cols, rows, chunks}, strides[2] = {pitch, (cuuint64_t)box_cols * bytes};
    const cuuint32_t box[3] = {box_cols, box_rows, chunks};
    return encode_map(map, type, p, 3, dims, strides, box, true);
}

// One wait for a barrier that has no arrivals to come: it gives up as any wait does, and the kernel ends.
__global__ void wait_check_kernel(uint32_t *err)
{
    __shared__ uint64_t bar;
    __shared__ Fail fail;
    mbar_init(&bar, 1);
    fail.failed = 0;
    mbar_wait(&bar, 0, &fail, err);
}

}  // namespace tc
}  // namespace vt

extern "C" vt_status vt_wait_check(uint32_t *err, vt_stream stream)
{
    VT_REQUIRE(err, "vt_wait_check: null pointer");
    vt::tc::wait_check_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(err);
    return vt::check_launch("wait_check_kernel");
}

extern "C" vt_status vt_error_word_create(uint32_t **word)
{
    VT_REQUIRE(word, "vt_error_word_create: null pointer");
    // An allocation is no part of a graph that this thread may be capturing.
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    void *p = nullptr;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaSuccess) {
        e = cudaHostAlloc(&p, sizeof(uint32_t), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return vt::set_error(VT_ERR_CUDA, "vt_error_word_create: %s", cudaGetErrorString(e));
    }
    *word = (uint32_t *)p;
    **word = 0;
    return VT_OK;
}

extern "C" vt_status vt_error_word_free(uint32_t *word)
{
    if (!word) return VT_OK;
    const cudaError_t e = cudaFreeHost(word);
    if (e == cudaSuccess) return VT_OK;
    cudaGetLastError();
    return vt::set_error(VT_ERR_CUDA, "vt_error_word_free: %s", cudaGetErrorString(e));
}
