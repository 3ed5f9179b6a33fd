// Device memory of other libraries as tensors of this one.
//
// A copy into the framework's layout, f32 NCHW or binary16 NHWC with channels padded to 32: what it moves is the bytes in and out once.  Source
// and destination may run along different axes, so a block of threads takes 64 pixels x 64 channels through shared memory, reads along
// the axis on which the source is denser and writes along the one on which the destination is.  A thread has its 16 reads in flight before it
// stores the first (64 x 128 x 76 x 76 binary16 NCHW, 189 MB in and out: 47 us; with bounds checked for every value, which issued in 77 % of the
// cycles, 62, with four reads in flight and scalar stores 120).
#include <exception>

#include "ln_common.h"

namespace {

constexpr int kThreads = 256, kTile = 64, kEach = kTile * kTile / kThreads;

struct take_params {
    const void* src;
    void* dst;
    int64_t sn, sc, sh, sw;       // strides of the source, in values
    int64_t pixels, hw, w, c, cs;  // pixels of all images, of one; channels as stored (NHWC)
    int64_t tiles_c, tiles;
};
__device__ __forceinline__ int64_t source_of(const take_params& p, int64_t q) {  // first channel of a pixel
    const int64_t n = q / p.hw, i = q - n * p.hw, y = i / p.w;
    return n * p.sn + y * p.sh + (i - y * p.w) * p.sw;
}
// WHOLE: all of the tile's pixels and channels are there
template <typename T, bool NHWC, bool ALONG_PIXELS, bool WHOLE>
__device__ __forceinline__ void take_tile(const take_params& p, int64_t q0, int64_t c0, T (&tile)[kTile][kTile + (sizeof(T) == 2 ? 2 : 1)], int64_t (&from)[kTile]) {
    constexpr int kRows = kThreads / kTile;
    const int fast = threadIdx.x % kTile, slow = threadIdx.x / kTile;
    const int pixels = WHOLE || p.pixels - q0 > kTile ? kTile : (int)(p.pixels - q0), channels = WHOLE || p.c - c0 > kTile ? kTile : (int)(p.c - c0);
    T v[kEach];
    if (ALONG_PIXELS) {  // a pixel per thread, pairs of channels
        const T* src = (const T*)p.src + (WHOLE || fast < pixels ? source_of(p, q0 + fast) : 0) + (c0 + 2 * slow) * p.sc;
        const int64_t step = 2 * kRows * p.sc;
#pragma unroll
        for (int k = 0; k < kEach; k += 2) {
            const int c = 2 * (slow + kRows * (k / 2));
            v[k] = WHOLE || (fast < pixels && c < channels) ? src[0] : T(0.0f);
            v[k + 1] = WHOLE || (fast < pixels && c + 1 < channels) ? src[p.sc] : T(0.0f);
            src += step;
        }
#pragma unroll
        for (int k = 0; k < kEach; k += 2) {
            const int c = 2 * (slow + kRows * (k / 2));
            if (sizeof(T) == 2) *reinterpret_cast<__half2*>(&tile[fast][c]) = __halves2half2(v[k], v[k + 1]);
            else { tile[fast][c] = v[k]; tile[fast][c + 1] = v[k + 1]; }
        }
    } else {
        if (slow == 0) from[fast] = WHOLE || fast < pixels ? source_of(p, q0 + fast) : 0;
        __syncthreads();
        const T* src = (const T*)p.src + (c0 + fast) * p.sc;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int q = slow + kRows * k;
            v[k] = WHOLE || (q < pixels && fast < channels) ? src[from[q]] : T(0.0f);
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) tile[slow + kRows * k][fast] = v[k];
    }
    __syncthreads();
    if (NHWC) {  // two channels of a pixel per thread (cs is even)
        const int c = 2 * (threadIdx.x % (kTile / 2)), q1 = threadIdx.x / (kTile / 2);
        T* dst = (T*)p.dst + (q0 + q1) * p.cs + c0 + c;
#pragma unroll
        for (int q = 0; q < kTile; q += 2 * kRows) {
            if (WHOLE || (q + q1 < pixels && c0 + c < p.cs)) *reinterpret_cast<__half2*>(dst) = *reinterpret_cast<const __half2*>(&tile[q + q1][c]);
            dst += 2 * kRows * p.cs;
        }
    } else if (WHOLE || fast < pixels) {
        const int64_t n = (q0 + fast) / p.hw;
        T* dst = (T*)p.dst + n * p.c * p.hw + (q0 + fast - n * p.hw) + (c0 + slow) * p.hw;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (WHOLE || slow + kRows * k < channels) *dst = tile[fast][slow + kRows * k];
            dst += kRows * p.hw;
        }
    }
    __syncthreads();
}
template <typename T, bool NHWC, bool ALONG_PIXELS>
__global__ void __launch_bounds__(kThreads) take_kernel(const take_params p) {
    // (33 or 65 words from pixel to pixel: no bank twice along either axis)
    __shared__ __align__(4) T tile[kTile][kTile + (sizeof(T) == 2 ? 2 : 1)];
    __shared__ int64_t from[kTile];
    for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x) {
        const int64_t q0 = t / p.tiles_c * kTile, c0 = t % p.tiles_c * kTile;
        if (q0 + kTile <= p.pixels && c0 + kTile <= p.c) take_tile<T, NHWC, ALONG_PIXELS, true>(p, q0, c0, tile, from);
        else take_tile<T, NHWC, ALONG_PIXELS, false>(p, q0, c0, tile, from);
    }
}
template <typename T, bool NHWC>
void take(const take_params& p, bool along_pixels, int grid, cudaStream_t stream) {
    if (along_pixels) take_kernel<T, NHWC, true><<<grid, kThreads, 0, stream>>>(p);
    else take_kernel<T, NHWC, false><<<grid, kThreads, 0, stream>>>(p);
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
            const bool along_pixels = (t->w > 1 ? far(3) : (t->h > 1 ? far(2) : far(0))) < far(1);
            p.tiles_c = ((dtype == LN_F16 ? p.cs : p.c) + kTile - 1) / kTile;
            p.tiles = (p.pixels + kTile - 1) / kTile * p.tiles_c;
            const int64_t most = (int64_t)ctx->sm_count * 64;
            const int grid = (int)(p.tiles < most ? p.tiles : most);
            if (dtype == LN_F32) take<float, false>(p, along_pixels, grid, ctx->stream);
            else take<__half, true>(p, along_pixels, grid, ctx->stream);
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
