// Device memory of other libraries as tensors of this one.
//
// A copy into the framework's layout, f32 NCHW or binary16 NHWC with channels padded to 32: what it moves is the bytes in and out once.  Source
// and destination may run along different axes, so a block of threads takes 64 pixels x 64 channels through shared memory, reads along
// the axis on which the source is denser and writes along the one on which the destination is (rows of 65 values: no bank twice).
#include <exception>

#include "ln_common.h"

namespace {

constexpr int kThreads = 256, kTile = 64;

struct take_params {
    const void* src;
    void* dst;
    int64_t sn, sc, sh, sw;       // strides of the source, in values
    int64_t pixels, hw, w, c, cs;  // pixels of all images, of one; channels as stored (NHWC)
    int64_t tiles_c, tiles;
    int along_pixels;
};
template <typename T, bool NHWC>
__global__ void __launch_bounds__(kThreads) take_kernel(const take_params p) {
    __shared__ T tile[kTile][kTile + 1];  // [channel][pixel]
    __shared__ int64_t from[kTile], to[kTile];  // of the tile's pixels: first channel in the source and the destination
    for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x) {
        const int64_t q0 = t / p.tiles_c * kTile, c0 = t % p.tiles_c * kTile;
        if (threadIdx.x < kTile) {
            const int64_t q = q0 + threadIdx.x, n = q / p.hw, i = q - n * p.hw, y = i / p.w;
            from[threadIdx.x] = n * p.sn + y * p.sh + (i - y * p.w) * p.sw;
            to[threadIdx.x] = NHWC ? q * p.cs : n * p.c * p.hw + i;
        }
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < kTile * kTile; i += kThreads) {
            const int q = p.along_pixels ? i % kTile : i / kTile, c = p.along_pixels ? i / kTile : i % kTile;
            tile[c][q] = q0 + q < p.pixels && c0 + c < p.c ? ((const T*)p.src)[from[q] + (c0 + c) * p.sc] : T(0.0f);
        }
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < kTile * kTile; i += kThreads) {
            const int q = NHWC ? i / kTile : i % kTile, c = NHWC ? i % kTile : i / kTile;
            if (q0 + q >= p.pixels || c0 + c >= (NHWC ? p.cs : p.c)) continue;
            if (NHWC) ((T*)p.dst)[to[q] + c0 + c] = tile[c][q];
            else ((T*)p.dst)[to[q] + (c0 + c) * p.hw] = tile[c][q];
        }
        __syncthreads();
    }
}

// Whether [lo, hi) is memory of the ctx's device that this process has mapped.
bool device_range(ln_ctx* ctx, uint64_t lo, uint64_t hi) {
    while (lo < hi) {
        unsigned kind = 0;
        int device = -1;
        uint64_t start = 0;
        size_t size = 0;
        if (ctx->pointer_attribute(&kind, CU_POINTER_ATTRIBUTE_MEMORY_TYPE, (CUdeviceptr)lo) != CUDA_SUCCESS || kind != CU_MEMORYTYPE_DEVICE) return false;
        if (ctx->pointer_attribute(&device, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, (CUdeviceptr)lo) != CUDA_SUCCESS || device != ctx->device) return false;
        if (ctx->pointer_attribute(&start, CU_POINTER_ATTRIBUTE_RANGE_START_ADDR, (CUdeviceptr)lo) != CUDA_SUCCESS) return false;
        if (ctx->pointer_attribute(&size, CU_POINTER_ATTRIBUTE_RANGE_SIZE, (CUdeviceptr)lo) != CUDA_SUCCESS || start + size <= lo) return false;
        lo = start + size;  // (memory that is mapped in pieces)
    }
    return true;
}

}  // namespace

extern "C" {

int32_t ln_tensor_from_device(ln_ctx* ctx, const void* data, int32_t dtype, const int64_t shape[4], const int64_t strides[4], void* stream, ln_tensor** out) {
    const char* who = "ln_tensor_from_device";
    if (!ctx || !data || !shape || !strides || !out) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (dtype != LN_F32 && dtype != LN_F16) return ln_fail(ctx, LN_ERR_ARG, "%s: dtype must be LN_F32 or LN_F16", who);
    const int64_t size = dtype == LN_F32 ? 4 : 2;
    if ((uint64_t)data % (uint64_t)size) return ln_fail(ctx, LN_ERR_ARG, "%s: the address is not a multiple of a value's %lld bytes", who, (long long)size);
    __int128 count = 1, lo = (int64_t)0, hi = 0;  // values in front of and behind the first one that the strides reach
    bool dense = true;
    int64_t expect = 1;
    for (int i = 3; i >= 0; --i) {
        if (shape[i] < 1 || shape[i] >= (1ll << 40)) return ln_fail(ctx, LN_ERR_SHAPE, "%s: tensor shape [%lld,%lld,%lld,%lld]", who, (long long)shape[0], (long long)shape[1], (long long)shape[2], (long long)shape[3]);
        const __int128 reach = (__int128)(shape[i] - 1) * strides[i];
        (reach < 0 ? lo : hi) += reach;
        if (shape[i] > 1) dense = dense && strides[i] == expect;
        count *= shape[i];
        if (count >= ((__int128)1 << 40)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: 2^40 values or more", who);
        expect *= shape[i];
    }
    const __int128 first = (__int128)(uint64_t)data + lo * size, last = (__int128)(uint64_t)data + (hi + 1) * size;
    try {
        cudaSetDevice(ctx->device);
        if (first < 0 || last > (__int128)INT64_MAX || !device_range(ctx, (uint64_t)first, (uint64_t)last))
            return ln_fail(ctx, LN_ERR_ARG, "%s: the values do not lie in memory of device %d", who, ctx->device);
        int rc = ln_order_streams(ctx, (cudaStream_t)stream, ctx->stream, who);
        if (rc) return rc;
        ln_tensor* t = ln_tensor_new(ctx, dtype, shape[0], shape[1], shape[2], shape[3]);
        if (!t) return LN_ERR_CUDA;
        cudaError_t e;
        if (dtype == LN_F32 && dense) e = cudaMemcpyAsync(t->ptr, data, t->bytes, cudaMemcpyDeviceToDevice, ctx->stream);
        else {
            take_params p;
            p.src = data; p.dst = t->ptr;
            p.sn = strides[0]; p.sc = strides[1]; p.sh = strides[2]; p.sw = strides[3];
            p.pixels = t->n * t->h * t->w; p.hw = t->h * t->w; p.w = t->w; p.c = t->c; p.cs = t->cstride / 2;
            // along the pixels where their neighbours are nearer to each other than those of the channels
            auto far = [&](int axis) { return shape[axis] > 1 ? (strides[axis] < 0 ? -strides[axis] : strides[axis]) : INT64_MAX; };
            p.along_pixels = (t->w > 1 ? far(3) : (t->h > 1 ? far(2) : far(0))) < far(1);
            p.tiles_c = ((dtype == LN_F16 ? p.cs : p.c) + kTile - 1) / kTile;
            p.tiles = (p.pixels + kTile - 1) / kTile * p.tiles_c;
            const int64_t most = (int64_t)ctx->sm_count * 64;
            const int grid = (int)(p.tiles < most ? p.tiles : most);
            if (dtype == LN_F32) take_kernel<float, false><<<grid, kThreads, 0, ctx->stream>>>(p);
            else take_kernel<__half, true><<<grid, kThreads, 0, ctx->stream>>>(p);
            ctx->launches++;
            e = cudaGetLastError();
        }
        if (e != cudaSuccess) {
            ln_tensor_release(t);
            return ln_fail(ctx, LN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
        }
        rc = ln_order_streams(ctx, ctx->stream, (cudaStream_t)stream, who);  // (the source may be written or freed in the stream's order)
        if (rc) { ln_tensor_release(t); return rc; }
        *out = t;
        return LN_OK;
    } catch (const std::exception&) {
        return ln_fail(ctx, LN_ERR_CUDA, "%s: host memory exhausted", who);
    }
}

}  // extern "C"
