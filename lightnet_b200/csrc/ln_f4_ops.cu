// Microscaled 4-bit tensors: narrow, widen, weights and the convolution (LN_F4, LN_MX4; formats and storage in ln_f4.h).
//
// What bounds them: narrow and widen move 4.5 (binary16) to 9 (f32) bytes for each byte of codes, so HBM; the product has its own notes.
#include <exception>
#include <new>

#include "ln_conv_plan.h"
#include "ln_f4.h"

namespace {

constexpr int kThreads = 256;

// 16 bytes that are read once
__device__ __forceinline__ uint4 ln_ldg_stream(const __half* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }

// Up to 64 blocks per SM: with 16, few enough for loops of two or three rounds, the last round left SMs idle (64 x 128 x 76 x 76, LN_F4, to
// binary16 21.4 us, now 19.9, to f32 43.5, now 38.9).  The rows of narrow_rows_kernel go through shared memory and want 16 (33.8 us against
// 35.9 for 8192 x 4096).
int grid_for(ln_ctx* ctx, int64_t n, int per_sm = 64) {
    const int64_t b = (n + kThreads - 1) / kThreads, cap = (int64_t)ctx->sm_count * per_sm;
    return (int)(b < 1 ? 1 : (b > cap ? cap : b));
}
int check_launch(ln_ctx* ctx, const char* what, cudaError_t e) {
    if (e == cudaSuccess) return LN_OK;
    (void)cudaGetLastError();  // (the next launch is checked for its own error)
    return ln_fail(ctx, LN_ERR_CUDA, "%s: kernel launch failed: %s", what, cudaGetErrorString(e));
}
// A new tensor, or the status of why there is none.
int new_tensor(ln_ctx* ctx, int dtype, int64_t n, int64_t c, int64_t h, int64_t w, ln_tensor** out) {
    *out = ln_tensor_new(ctx, dtype, n, c, h, w);
    return *out ? LN_OK : (ctx->err.find("cudaMalloc") != std::string::npos ? LN_ERR_CUDA : LN_ERR_SHAPE);
}
// Nothing is thrown across the boundary: what the host code can throw is a failed allocation.
template <typename F>
int32_t guarded(ln_ctx* ctx, const char* who, F&& body) {
    try {
        return body();
    } catch (const std::exception&) {
        return ln_fail(ctx, LN_ERR_CUDA, "%s: host memory exhausted", who);
    }
}
// Tensor scales that keep 6 g, every product of g with a block scale and its reciprocal normal numbers.
bool usable_scale(int dtype, float s) { return dtype == LN_MX4 ? s == 1.0f : s >= 0x1p-100f && s <= 0x1p100f; }

// ---- narrow and widen -----------------------------------------------------------------------------------------------------------
// binary16 NHWC (narrow): a thread takes 32 channels of a pixel, consecutive threads consecutive groups of them, so that all accesses of a warp are
// contiguous; two neighbours, which always belong to one pixel (its channels are padded to 64), put their scale bytes together.
// f32 NCHW: the 32 lanes of a warp are 8 pixels x 4 blocks, so that a row of 8 pixels is a sector of a plane on one side and the four
// blocks of a pixel (32 or 64 bytes of codes, one word of scales) are contiguous on the other.
// I: 32-bit indexes where they suffice (a division per thread).

template <int FMT>
__device__ __forceinline__ uint32_t store_block(const float* x, float g, float six_g, uint8_t* codes) {
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    uint32_t w[B / 8];
    const uint32_t scale = ln_f4_quantise<FMT>(x, g, six_g, w);
    if (FMT == LN_F4) *reinterpret_cast<uint2*>(codes) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(codes) = make_uint4(w[0], w[1], w[B / 8 - 2], w[B / 8 - 1]);
    return scale;
}
template <int FMT, typename I>
__global__ void __launch_bounds__(kThreads, 5) narrow_f16_kernel(const __half* __restrict__ x, int64_t xs, uint8_t* __restrict__ codes, uint8_t* __restrict__ sf, int64_t pixels, int C, int groups,
                                                              int64_t cstride, int64_t sf_words, float g, float six_g) {
    ln_f4_after_predecessor();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    const I total = (I)(pixels * groups), step = (I)(gridDim.x * blockDim.x);
    const int lane = threadIdx.x & 31;
    for (I first = (I)blockIdx.x * blockDim.x + (threadIdx.x & ~31); first < total; first += step) {  // (whole warps, for the exchange)
        const bool real = first + lane < total;
        const I i = real ? first + lane : total - 1, pix = i / (I)groups;
        const int c0 = (int)(i - pix * (I)groups) * 32;
        uint4 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = c0 < C ? ln_ldg_stream(x + (int64_t)pix * xs + c0 + 8 * j) : make_uint4(0, 0, 0, 0);  // (a pixel's channels are padded to 32)
        float v[32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                v[8 * j + 2 * k] = f.x;
                v[8 * j + 2 * k + 1] = f.y;
            }
        }
        if (c0 + 32 > C) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c0 + j >= C) v[j] = 0.0f;
        }
        uint32_t w[4], s = 0;
#pragma unroll
        for (int b = 0; b < 32 / B; ++b) s |= ln_f4_quantise<FMT>(v + b * B, g, six_g, w + b * B / 8) << (8 * b);
        const uint32_t other = __shfl_down_sync(0xFFFFFFFFu, s, 1);  // (blocks take different ways through the quantisation: all lanes are named)
        if (!real) continue;
        *reinterpret_cast<uint4*>(codes + (int64_t)pix * cstride + c0 / 2) = make_uint4(w[0], w[1], w[2], w[3]);
        if ((c0 & 32) == 0) {
            uint8_t* dst = sf + ln_f4_sf_at(pix, c0 / (4 * B), sf_words) + c0 / B % 4;
            if (FMT == LN_F4) *reinterpret_cast<uint32_t*>(dst) = s | other << 16;
            else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)(s | other << 8);
        }
    }
}
template <int FMT, typename I>
__global__ void __launch_bounds__(kThreads) narrow_f32_kernel(const float* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ sf, int64_t pixels, int64_t hw, int C, int blocks,
                                                              int64_t cstride, int64_t sf_words, float g, float six_g) {
    ln_f4_after_predecessor();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    const I rows = (I)((pixels + 7) / 8), warps = rows * (I)((blocks + 3) / 4), step = (I)(gridDim.x * (blockDim.x / 32));
    const int lane = threadIdx.x & 31;
    for (I w = (I)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; w < warps; w += step) {
        const I quad = w / rows;
        const I pix = (w - quad * rows) * 8 + (lane >> 2);
        const int b = (int)quad * 4 + (lane & 3);
        uint32_t s = 0;
        if (pix < (I)pixels && b < blocks) {
            const I img = pix / (I)hw;
            const float* src = x + ((int64_t)img * C + b * B) * hw + (pix - img * (I)hw);
            float v[B];
            if (b * B + B <= C) {
#pragma unroll
                for (int j = 0; j < B; ++j) v[j] = __ldg(src + j * hw);
            } else {
#pragma unroll
                for (int j = 0; j < B; ++j) v[j] = b * B + j < C ? __ldg(src + j * hw) : 0.0f;
            }
            s = store_block<FMT>(v, g, six_g, codes + (int64_t)pix * cstride + b * (B / 2));
        }
        s |= __shfl_down_sync(0xFFFFFFFFu, s, 1) << 8;
        s |= __shfl_down_sync(0xFFFFFFFFu, s, 2) << 16;
        // (behind the last block of LN_MX4 a word may have two bytes that nothing uses)
        if ((lane & 3) == 0 && pix < (I)pixels) *reinterpret_cast<uint32_t*>(sf + ln_f4_sf_at(pix, b >> 2, sf_words)) = s;
    }
}

// 16 channels
template <int FMT>
__device__ __forceinline__ void widen_16(uint2 w, uint32_t scale, float g, float (&v)[16]) {
    const float d = ln_f4_factor<FMT>(scale, g);
    uint32_t h[8];
    ln_e2m1x8_to_h2(w.x, *reinterpret_cast<uint32_t(*)[4]>(h));
    ln_e2m1x8_to_h2(w.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
        v[2 * k] = __fmul_rn(f.x, d);
        v[2 * k + 1] = __fmul_rn(f.y, d);
    }
}
template <int FMT, typename I>
__global__ void __launch_bounds__(kThreads) widen_f16_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf, __half* __restrict__ y, int64_t ys, int64_t pixels, int C, int blocks,
                                                             int64_t cstride, int64_t sf_words, float g) {
    ln_f4_after_predecessor();  // (16 channels a thread: its 32 bytes are a sector of the output)
    const I total = (I)(pixels * blocks), step = (I)(gridDim.x * blockDim.x);
    for (I i = (I)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
        const I pix = i / (I)blocks;
        const int b16 = (int)(i - pix * (I)blocks), b = FMT == LN_F4 ? b16 : b16 >> 1;
        float v[16];
        widen_16<FMT>(__ldg(reinterpret_cast<const uint2*>(codes + (int64_t)pix * cstride + b16 * 8)), __ldg(sf + ln_f4_sf_at(pix, b >> 2, sf_words) + (b & 3)), g, v);
        if (b16 * 16 + 16 > C) {  // (a NaN block that ends inside the padding must not reach it)
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (b16 * 16 + j >= C) v[j] = 0.0f;
        }
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const __half2 p = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
            h[k] = *reinterpret_cast<const uint32_t*>(&p);
        }
        ln_store_32(y + (int64_t)pix * ys + b16 * 16, h);
    }
}
template <int FMT, typename I>
__global__ void __launch_bounds__(kThreads) widen_f32_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf, float* __restrict__ y, int64_t pixels, int64_t hw, int C, int blocks,
                                                             int64_t cstride, int64_t sf_words, float g) {
    ln_f4_after_predecessor();  // (blocks of 16 channels for both types)
    const I rows = (I)((pixels + 7) / 8), warps = rows * (I)((blocks + 3) / 4), step = (I)(gridDim.x * (blockDim.x / 32));
    const int lane = threadIdx.x & 31;
    for (I w = (I)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; w < warps; w += step) {
        const I quad = w / rows;
        const I pix = (w - quad * rows) * 8 + (lane >> 2);
        const int b16 = (int)quad * 4 + (lane & 3), b = FMT == LN_F4 ? b16 : b16 >> 1;
        if (pix >= (I)pixels || b16 >= blocks) continue;
        float v[16];
        widen_16<FMT>(__ldg(reinterpret_cast<const uint2*>(codes + (int64_t)pix * cstride + b16 * 8)), __ldg(sf + ln_f4_sf_at(pix, b >> 2, sf_words) + (b & 3)), g, v);
        const I img = pix / (I)hw;
        float* dst = y + ((int64_t)img * C + b16 * 16) * hw + (pix - img * (I)hw);
        if (b16 * 16 + 16 <= C) {
#pragma unroll
            for (int j = 0; j < 16; ++j) dst[j * hw] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (b16 * 16 + j < C) dst[j * hw] = v[j];
        }
    }
}
// f32 rows of tokens (1 x 1 images: a row is the channels of one).  A warp takes 32 consecutive blocks, whose values are one contiguous
// range wherever rows begin; it goes through shared memory (17 words per 16: no bank twice) so that every access to it is coalesced.
template <int FMT>
__global__ void __launch_bounds__(kThreads) narrow_rows_kernel(const float* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ sf, int64_t rows, int C, int blocks, int64_t cstride,
                                                               int64_t sf_words, float g, float six_g) {
    ln_f4_after_predecessor();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    __shared__ float stage[kThreads / 32][34 * B];
    float* mine = stage[threadIdx.x / 32];
    const int lane = threadIdx.x & 31;
    const int64_t total = rows * blocks;
    for (int64_t first = (blockIdx.x * (int64_t)(kThreads / 32) + threadIdx.x / 32) * 32; first < total; first += (int64_t)gridDim.x * kThreads) {
        const int64_t u = first + lane < total ? first + lane : total - 1, row = u / blocks;
        const int b = (int)(u - row * blocks), have = C - b * B < 0 ? 0 : (C - b * B < B ? C - b * B : B);
        const int64_t at = row * C + (b * B < C ? b * B : C), from = __shfl_sync(0xFFFFFFFFu, at, 0);
        const int o = (int)(at - from), end = __shfl_sync(0xFFFFFFFFu, o + have, 31);
        __syncwarp();
        for (int i = lane; i < end; i += 32) mine[i + (i >> 4)] = __ldcs(x + from + i);
        __syncwarp();
        float v[B];
#pragma unroll
        for (int j = 0; j < B; ++j) v[j] = j < have ? mine[o + j + ((o + j) >> 4)] : 0.0f;
        const bool real = first + lane < total;
        uint32_t s = real ? store_block<FMT>(v, g, six_g, codes + row * cstride + b * (B / 2)) : 0u;
        s |= __shfl_down_sync(0xFFFFFFFFu, s, 1) << 8;
        if (FMT == LN_F4) {  // (a row's blocks are a multiple of four, of LN_MX4 of two)
            s |= __shfl_down_sync(0xFFFFFFFFu, s, 2) << 16;
            if (real && (lane & 3) == 0) *reinterpret_cast<uint32_t*>(sf + ln_f4_sf_at(row, b >> 2, sf_words)) = s;
        } else if (real && (lane & 1) == 0)
            *reinterpret_cast<uint16_t*>(sf + ln_f4_sf_at(row, b >> 2, sf_words) + (b & 3)) = (uint16_t)s;
    }
}
template <int FMT>
__global__ void __launch_bounds__(kThreads) widen_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf, float* __restrict__ y, int64_t rows, int C, int blocks, int64_t cstride,
                                                              int64_t sf_words, float g) {
    ln_f4_after_predecessor();  // (blocks of 16 channels for both types)
    __shared__ float stage[kThreads / 32][34 * 16];
    float* mine = stage[threadIdx.x / 32];
    const int lane = threadIdx.x & 31;
    const int64_t total = rows * blocks;
    for (int64_t first = (blockIdx.x * (int64_t)(kThreads / 32) + threadIdx.x / 32) * 32; first < total; first += (int64_t)gridDim.x * kThreads) {
        const int64_t u = first + lane < total ? first + lane : total - 1, row = u / blocks;
        const int b16 = (int)(u - row * blocks), b = FMT == LN_F4 ? b16 : b16 >> 1, have = C - b16 * 16 < 16 ? C - b16 * 16 : 16;
        const int64_t at = row * C + b16 * 16, from = __shfl_sync(0xFFFFFFFFu, at, 0);
        const int o = (int)(at - from), end = __shfl_sync(0xFFFFFFFFu, o + have, 31);
        float v[16];
        widen_16<FMT>(__ldg(reinterpret_cast<const uint2*>(codes + row * cstride + b16 * 8)), __ldg(sf + ln_f4_sf_at(row, b >> 2, sf_words) + (b & 3)), g, v);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < have) mine[o + j + ((o + j) >> 4)] = v[j];
        __syncwarp();
        for (int i = lane; i < end; i += 32) y[from + i] = mine[i + (i >> 4)];
    }
}
// codes (one per byte) and scales in NCHW order
__global__ void unpack_f4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf, uint8_t* __restrict__ out_codes, uint8_t* __restrict__ out_sf, int64_t n, int64_t hw,
                                 int C, int sf_blocks, int64_t cstride, int64_t sf_words) {
    ln_f4_after_predecessor();
    const int64_t first = n * C * hw, total = first + n * sf_blocks * hw;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t k = i < first ? i : i - first;
        const int per = i < first ? C : sf_blocks;
        const int64_t p = k % hw, img = k / hw / per;
        const int c = (int)(k / hw % per);
        if (i < first) out_codes[k] = (codes[(img * hw + p) * cstride + c / 2] >> (4 * (c & 1))) & 15;
        else out_sf[k] = sf[ln_f4_sf_at(img * hw + p, c >> 2, sf_words) + (c & 3)];
    }
}

// ---- weights --------------------------------------------------------------------------------------------------------------------
// One thread block per filter: its largest magnitude, then the blocks of each tap (a filter's scale 0 leaves zero codes).
template <int FMT>
__global__ void pack_weights_f4_kernel(const float* __restrict__ w, int C, int k2, int64_t cstride, uint8_t* __restrict__ codes, uint8_t* __restrict__ sf, float* __restrict__ wscale,
                                       int64_t sf_words) {
    ln_f4_after_predecessor();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    const int f = blockIdx.x;
    const float* src = w + (int64_t)f * C * k2;
    float amax = 0.0f;
    for (int64_t i = threadIdx.x; i < (int64_t)C * k2; i += blockDim.x) amax = ln_max_nan(amax, fabsf(src[i]));
    for (int o = 16; o; o >>= 1) amax = ln_max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    __shared__ float part[32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) amax = ln_max_nan(amax, part[i]);
    // g stays in the range of tensor scales: 1 for a filter of zeros, the end of the range behind it.  A filter with a NaN is NaN as a whole, scale and
    // blocks: whether taps outside the image multiply it by zero or are left out then makes no difference.
    const bool nan = amax != amax;
    float g = 1.0f;
    if (FMT == LN_F4 && amax > 0.0f) g = fminf(fmaxf(__fdiv_rn(amax, 6.0f * 448.0f), 0x1p-100f), 0x1p100f);
    if (threadIdx.x == 0) wscale[f] = nan ? amax : g;
    const int blocks = (int)(cstride * 2 / B);
    for (int i = threadIdx.x; i < k2 * blocks; i += blockDim.x) {
        const int tap = i / blocks, b = i - tap * blocks;
        float v[B];
#pragma unroll
        for (int j = 0; j < B; ++j) v[j] = b * B + j < C ? src[(int64_t)(b * B + j) * k2 + tap] : 0.0f;
        const int64_t at = ln_f4_sf_at(f, (int64_t)tap * sf_words + (b >> 2), k2 * sf_words) + (b & 3);
        const uint32_t scale = store_block<FMT>(v, g, 6.0f * g, codes + ((int64_t)f * k2 + tap) * cstride + b * (B / 2));
        sf[at] = (uint8_t)(!nan ? scale : (FMT == LN_F4 ? 0x7Fu : 0xFFu));
    }
}

// ---- the product on the CUDA cores ----------------------------------------------------------------------------------------------
struct simt_params {
    const uint8_t *x, *xsf, *w, *wsf;
    const float *wscale, *bias;
    void* y;
    uint8_t* ysf;
    int64_t xs, xsf_words, ys, ysf_words, total;
    int H, W, F, fpad, k, sx, sy, pad, OH, OW, blocks, act, out_kind;  // fpad: filters as they are counted, F, or for a 4-bit output its padded channels
    float xscale, g, six_g;
};
// One thread per output value, filters fastest.  Takes every geometry.  A 4-bit output's channels are padded to 64, so that a warp is 32 filters of
// one pixel; the first lane of each block collects its values (a tensor between this kernel and a narrow would be memory that a
// caller who captures the call cannot keep for the replays).
template <int FMT, bool EXACT>
__global__ void conv_f4_simt_kernel(const simt_params p) {
    ln_f4_after_predecessor();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < p.total; i += (int64_t)gridDim.x * blockDim.x) {
        const int f = (int)(i % p.fpad);
        const int64_t pix = i / p.fpad;
        const int ox = (int)(pix % p.OW), oy = (int)(pix / p.OW % p.OH);
        const int64_t n = pix / p.OW / p.OH;
        float acc = 0.0f;
        for (int r = 0; r < p.k && f < p.F; ++r) {
            const int yy = oy * p.sy - p.pad + r;
            if (yy < 0 || yy >= p.H) continue;
            for (int s = 0; s < p.k; ++s) {
                const int xx = ox * p.sx - p.pad + s;
                if (xx < 0 || xx >= p.W) continue;
                const int64_t q = (n * p.H + yy) * p.W + xx;
                const int tap = r * p.k + s;
                const uint8_t* xc = p.x + q * p.xs;
                const uint8_t* wc = p.w + ((int64_t)f * p.k * p.k + tap) * p.xs;
                for (int b = 0; b < p.blocks; ++b) {
                    const int64_t at = ln_f4_sf_at(f, (int64_t)tap * p.xsf_words + (b >> 2), p.k * p.k * p.xsf_words) + (b & 3), xat = ln_f4_sf_at(q, b >> 2, p.xsf_words) + (b & 3);
                    float sum = 0.0f;  // exact: multiples of 0.25 below 2^11
#pragma unroll
                    for (int j = 0; j < B / 8; ++j) {
                        uint32_t a[4], c[4];
                        ln_e2m1x8_to_h2(*reinterpret_cast<const uint32_t*>(xc + b * (B / 2) + 4 * j), a);
                        ln_e2m1x8_to_h2(*reinterpret_cast<const uint32_t*>(wc + b * (B / 2) + 4 * j), c);
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&a[t])), v = __half22float2(*reinterpret_cast<const __half2*>(&c[t]));
                            sum = __fmaf_rn(u.x, v.x, sum);
                            sum = __fmaf_rn(u.y, v.y, sum);
                        }
                    }
                    // (block scales first: their product is exact for LN_F4; those of LN_MX4 need the range of 64 bits)
                    if (FMT == LN_F4) acc = __fmaf_rn(sum, __fmul_rn(ln_e4m3_value(p.xsf[xat]), ln_e4m3_value(p.wsf[at])), acc);
                    else acc += __double2float_rn((double)sum * ((double)ln_e8m0_value(p.xsf[xat]) * (double)ln_e8m0_value(p.wsf[at])));
                }
            }
        }
        const float v = f < p.F ? ln_f4_act<EXACT>(p.act, __fmaf_rn(acc, __fmul_rn(p.xscale, p.wscale[f]), p.bias[f])) : 0.0f;
        if (p.out_kind == LN_OUT_Q) {
            const int lane = threadIdx.x & 31;
            float b[B];
#pragma unroll
            for (int j = 0; j < B; ++j) b[j] = __shfl_sync(0xFFFFFFFFu, v, (lane & ~(B - 1)) + j);
            if (lane % B == 0) p.ysf[ln_f4_sf_at(pix, f / (4 * B), p.ysf_words) + f / B % 4] = (uint8_t)store_block<FMT>(b, p.g, p.six_g, (uint8_t*)p.y + pix * p.ys + f / 2);
        } else if (p.out_kind == LN_OUT_F16) ((__half*)p.y)[pix * p.ys + f] = __float2half_rn(v);
        else ((float*)p.y)[((n * p.F + f) * p.OH + oy) * p.OW + ox] = v;
    }
}

// ---- the product for few pixels --------------------------------------------------------------------------------------------------
// A 1x1 stride-1 convolution of up to 16 pixels (a token, or a few): the weights are read once and nothing else costs, so what counts is how
// many reads are in flight.  A block of 16 warps takes 32 filters and cuts their k range into chunks of 128 channels; a lane reads 16 bytes of
// a row (filter or pixel), widens them with their block scales to binary16 (LN_F4: a code times an E4M3 scale has 6 bits and at most 2688) or
// bfloat16 (LN_MX4: any power of two), both exact, and feeds warp-level instructions, whose k order may be any as long as both operands have
// the same: pixels fill 8 of their columns, the tensor pipe has time.  (tcgen05 works on 128 pixels and one CTA per 64 filters then walks the
// whole k range: 4096 -> 4096 for one token 8.5 us, this way 4.7.)  The warps' sums are added in order.
constexpr int kFewThreads = 512, kFewFilters = 32, kFewPixels = 16;
struct few_params {
    const uint8_t *x, *xsf, *w, *wsf;
    const float *wscale, *bias;
    void* y;
    uint8_t* ysf;
    int64_t xs, sf_words, ys, ysf_words;
    int pixels, F, chunks, act, exact, out_kind, hw;
    float xscale, g, six_g;
};
// 32 codes of a lane -> 16 scaled pairs
template <int FMT>
__device__ __forceinline__ void few_operand(const uint4& q, uint32_t scale, uint32_t (&h)[16]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) ln_e2m1x8_to_h2(w[i], *reinterpret_cast<uint32_t(*)[4]>(h + 4 * i));
    if (FMT == LN_F4) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const __half2 s = __float2half2_rn(ln_e4m3_value(scale >> (8 * b) & 0xFFu));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[8 * b + i]), s);
                h[8 * b + i] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
    } else {
        // (a quarter of the values: 6 * 2^126, a saturated infinity, is more than 16 bits hold; the sums are multiplied by 16)
        const float s = 0.25f * ln_e8m0_value(scale);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            h[i] = __byte_perm(__float_as_uint(__fmul_rn(f.x, s)), __float_as_uint(__fmul_rn(f.y, s)), 0x7632);  // (two bits and an exponent: the low halves are zero)
        }
    }
}
template <int FMT>
__device__ __forceinline__ void few_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (FMT == LN_F4)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int FMT>
__device__ __forceinline__ void few_load(const uint8_t* codes, const uint8_t* sf, int64_t row, bool there, int64_t stride, int64_t sf_words, int chunk, int t, uint4& q, uint32_t& scale) {
    const int64_t at = (int64_t)chunk * 64 + t * 16;
    q = make_uint4(0, 0, 0, 0);
    scale = 0;
    if (!there || at >= stride) return;
    q = __ldg(reinterpret_cast<const uint4*>(codes + row * stride + at));
    if (FMT == LN_F4) scale = __ldg(reinterpret_cast<const uint16_t*>(sf + ln_f4_sf_at(row, chunk * 2 + (t >> 1), sf_words) + (t & 1) * 2));
    else scale = __ldg(sf + ln_f4_sf_at(row, chunk, sf_words) + t);
}
template <int FMT, int NT>
__global__ void __launch_bounds__(kFewThreads) conv_f4_few_kernel(const few_params p) {
    ln_f4_after_predecessor();
    __shared__ float part[kFewThreads / 32][kFewFilters][8 * NT + 1];
    __shared__ float sums[8 * NT][kFewFilters + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, f0 = (int)blockIdx.x * kFewFilters;
    float acc[2][NT][4] = {};
#pragma unroll 2
    for (int chunk = warp; chunk < p.chunks; chunk += kFewThreads / 32) {
        uint4 wq[4], xq[NT];
        uint32_t ws[4], xsc[NT];
#pragma unroll
        for (int i = 0; i < 4; ++i) few_load<FMT>(p.w, p.wsf, f0 + g + 8 * i, f0 + g + 8 * i < p.F, p.xs, p.sf_words, chunk, t, wq[i], ws[i]);
#pragma unroll
        for (int n = 0; n < NT; ++n) few_load<FMT>(p.x, p.xsf, g + 8 * n, g + 8 * n < p.pixels, p.xs, p.sf_words, chunk, t, xq[n], xsc[n]);
        uint32_t b[NT][16];
#pragma unroll
        for (int n = 0; n < NT; ++n) few_operand<FMT>(xq[n], xsc[n], b[n]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint32_t lo[16], hi[16];
            few_operand<FMT>(wq[2 * m], ws[2 * m], lo);
            few_operand<FMT>(wq[2 * m + 1], ws[2 * m + 1], hi);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int s = 0; s < 8; ++s) few_mma<FMT>(acc[m][n], lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], b[n][2 * s], b[n][2 * s + 1]);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[warp][16 * m + g + (i >> 1) * 8][8 * n + 2 * t + (i & 1)] = acc[m][n][i];
    __syncthreads();
    const int i = threadIdx.x, f = f0 + (i & 31), n = i >> 5;  // (a warp: the 32 filters of a pixel)
    if (n < 8 * NT) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kFewThreads / 32; ++k) sum += part[k][i & 31][n];
        float v = 0.0f;
        if (f < p.F) {
            v = __fmaf_rn(sum, FMT == LN_F4 ? __fmul_rn(p.xscale, p.wscale[f]) : 16.0f, p.bias[f]);
            v = p.exact ? ln_f4_act<true>(p.act, v) : ln_f4_act<false>(p.act, v);
        }
        if (p.out_kind == LN_OUT_Q) sums[n][i & 31] = v;
        else if (n < p.pixels) {
            if (p.out_kind == LN_OUT_F16) ((__half*)p.y)[n * p.ys + f] = __float2half_rn(v);  // (filters are padded to 32)
            else if (f < p.F) {
                const int img = n / p.hw;
                ((float*)p.y)[((int64_t)img * p.F + f) * p.hw + n - img * p.hw] = v;
            }
        }
    }
    if (p.out_kind != LN_OUT_Q) return;
    __syncthreads();
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    const int pix = i / (32 / B), b = i % (32 / B);
    if (pix >= p.pixels || pix >= 8 * NT) return;
    float v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) v[j] = sums[pix][b * B + j];
    const int first = f0 + b * B;
    p.ysf[ln_f4_sf_at(pix, first / (4 * B), p.ysf_words) + first / B % 4] = (uint8_t)store_block<FMT>(v, p.g, p.six_g, (uint8_t*)p.y + pix * p.ys + first / 2);
}
int few_launch(ln_ctx* ctx, const ln_f4_conv& c, int64_t pixels) {
    const ln_tensor &x = *c.x, &y = *c.y;
    few_params p;
    p.x = (const uint8_t*)x.ptr; p.xsf = (const uint8_t*)x.sf; p.w = (const uint8_t*)c.w->w; p.wsf = (const uint8_t*)c.w->sf;
    p.wscale = c.w->wscale; p.bias = c.bias; p.y = y.ptr; p.ysf = (uint8_t*)y.sf;
    p.xs = x.cstride; p.sf_words = x.sf_words; p.ys = y.dtype == LN_F16 ? y.cstride / 2 : y.cstride; p.ysf_words = y.sf_words;
    p.pixels = (int)pixels; p.F = (int)y.c; p.chunks = (int)((x.cstride + 63) / 64); p.act = c.act; p.exact = ctx->exact_epilogue; p.out_kind = c.out_kind; p.hw = (int)(y.h * y.w);
    p.xscale = x.scale; p.g = y.scale; p.six_g = 6.0f * y.scale;
    const int grid = (int)(ln_round_up(y.c, c.out_kind == LN_OUT_Q ? 64 : 32) / kFewFilters);
    cudaError_t e;
    if (c.dtype == LN_F4) e = pixels <= 8 ? ln_f4_launch(ctx, conv_f4_few_kernel<LN_F4, 1>, grid, kFewThreads, 0, p) : ln_f4_launch(ctx, conv_f4_few_kernel<LN_F4, 2>, grid, kFewThreads, 0, p);
    else e = pixels <= 8 ? ln_f4_launch(ctx, conv_f4_few_kernel<LN_MX4, 1>, grid, kFewThreads, 0, p) : ln_f4_launch(ctx, conv_f4_few_kernel<LN_MX4, 2>, grid, kFewThreads, 0, p);
    return check_launch(ctx, "ln_conv2d_bias_act_f4", e);
}

// one launch with 32-bit indexes where every index, and the step behind the last one, stays below 2^31
#define LN_F4_CALL(KERNEL, FMT, SMALL, GRID, ...) \
    ((FMT) == LN_F4 ? ((SMALL) ? ln_f4_launch(ctx, KERNEL<LN_F4, uint32_t>, GRID, kThreads, 0, __VA_ARGS__) : ln_f4_launch(ctx, KERNEL<LN_F4, int64_t>, GRID, kThreads, 0, __VA_ARGS__)) \
                    : ((SMALL) ? ln_f4_launch(ctx, KERNEL<LN_MX4, uint32_t>, GRID, kThreads, 0, __VA_ARGS__) : ln_f4_launch(ctx, KERNEL<LN_MX4, int64_t>, GRID, kThreads, 0, __VA_ARGS__)))

int narrow_into(ln_ctx* ctx, const ln_tensor* t, ln_tensor* q) {
    const int64_t pixels = t->n * t->h * t->w, hw = t->h * t->w;
    uint8_t *codes = (uint8_t*)q->ptr, *sf = (uint8_t*)q->sf;
    const float g = q->scale, six_g = 6.0f * g;
    const bool small = q->cstride * pixels < (1ll << 30);
    cudaError_t e;
    const int blocks = (int)(q->cstride * 2 / ln_f4_block(q->dtype));
    if (t->dtype == LN_F32 && hw == 1) {
        const int grid = grid_for(ctx, pixels * blocks, 16);
        e = q->dtype == LN_F4 ? ln_f4_launch(ctx, narrow_rows_kernel<LN_F4>, grid, kThreads, 0, (const float*)t->ptr, codes, sf, pixels, (int)t->c, blocks, q->cstride, q->sf_words, g, six_g)
                              : ln_f4_launch(ctx, narrow_rows_kernel<LN_MX4>, grid, kThreads, 0, (const float*)t->ptr, codes, sf, pixels, (int)t->c, blocks, q->cstride, q->sf_words, g, six_g);
    } else if (t->dtype == LN_F32) {
        e = LN_F4_CALL(narrow_f32_kernel, q->dtype, small, grid_for(ctx, (pixels + 7) / 8 * ((blocks + 3) / 4) * 32), (const float*)t->ptr, codes, sf, pixels, hw, (int)t->c, blocks, q->cstride, q->sf_words, g,
                       six_g);
    } else {
        const int groups = (int)(q->cstride / 16);
        e = LN_F4_CALL(narrow_f16_kernel, q->dtype, small, grid_for(ctx, pixels * groups), (const __half*)t->ptr, t->cstride / 2, codes, sf, pixels, (int)t->c, groups, q->cstride, q->sf_words, g, six_g);
    }
    return check_launch(ctx, "ln_tensor_narrow_f4", e);
}
int widen_into(ln_ctx* ctx, const ln_tensor* t, ln_tensor* y) {
    const int64_t pixels = t->n * t->h * t->w, hw = t->h * t->w;
    const uint8_t *codes = (const uint8_t*)t->ptr, *sf = (const uint8_t*)t->sf;
    const bool small = t->cstride * pixels < (1ll << 30);
    cudaError_t e;
    const int blocks = (int)((t->c + 15) / 16);
    if (y->dtype == LN_F32 && hw == 1) {
        const int grid = grid_for(ctx, pixels * blocks);
        e = t->dtype == LN_F4 ? ln_f4_launch(ctx, widen_rows_kernel<LN_F4>, grid, kThreads, 0, codes, sf, (float*)y->ptr, pixels, (int)t->c, blocks, t->cstride, t->sf_words, t->scale)
                              : ln_f4_launch(ctx, widen_rows_kernel<LN_MX4>, grid, kThreads, 0, codes, sf, (float*)y->ptr, pixels, (int)t->c, blocks, t->cstride, t->sf_words, t->scale);
    } else if (y->dtype == LN_F32) {
        e = LN_F4_CALL(widen_f32_kernel, t->dtype, small, grid_for(ctx, (pixels + 7) / 8 * ((blocks + 3) / 4) * 32), codes, sf, (float*)y->ptr, pixels, hw, (int)t->c, blocks, t->cstride, t->sf_words, t->scale);
    } else {
        const int padded = (int)(y->cstride / 32);  // (the channels of binary16 are padded to 32)
        e = LN_F4_CALL(widen_f16_kernel, t->dtype, small, grid_for(ctx, pixels * padded), codes, sf, (__half*)y->ptr, y->cstride / 2, pixels, (int)t->c, padded, t->cstride, t->sf_words, t->scale);
    }
    return check_launch(ctx, "ln_tensor_widen_f4", e);
}
#undef LN_F4_CALL

}  // namespace

extern "C" {

int32_t ln_tensor_narrow_f4(ln_ctx* ctx, const ln_tensor* t, float scale, int32_t dtype, ln_tensor** out) {
    const char* who = "ln_tensor_narrow_f4";
    if (!ctx || !t || !out) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (t->dtype != LN_F32 && t->dtype != LN_F16) return ln_fail(ctx, LN_ERR_ARG, "%s: f32 or binary16 tensor required", who);
    if (t->ctx != ctx) return ln_fail(ctx, LN_ERR_ARG, "%s: the tensor belongs to another context", who);
    if (!ln_is_f4(dtype)) return ln_fail(ctx, LN_ERR_ARG, "%s: dtype must be LN_F4 or LN_MX4", who);
    if (t->c > (1 << 30)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: more than 2^30 channels", who);
    if (!usable_scale(dtype, scale)) return ln_fail(ctx, LN_ERR_ARG, "%s: scale %g is not %s", who, scale, dtype == LN_MX4 ? "1 (LN_MX4 has no tensor scale)" : "in [2^-100, 2^100]");
    return guarded(ctx, who, [&]() -> int32_t {
        cudaSetDevice(ctx->device);
        ln_tensor* q = nullptr;
        int rc = new_tensor(ctx, dtype, t->n, t->c, t->h, t->w, &q);
        if (rc) return rc;
        q->scale = scale;
        rc = narrow_into(ctx, t, q);
        if (rc) { ln_tensor_release(q); return rc; }
        *out = q;
        return LN_OK;
    });
}

int32_t ln_tensor_widen_f4(ln_ctx* ctx, const ln_tensor* t, int32_t dtype, ln_tensor** out) {
    const char* who = "ln_tensor_widen_f4";
    if (!ctx || !t || !out) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (!ln_is_f4(t->dtype)) return ln_fail(ctx, LN_ERR_ARG, "%s: 4-bit tensor required", who);
    if (t->ctx != ctx) return ln_fail(ctx, LN_ERR_ARG, "%s: the tensor belongs to another context", who);
    if (dtype != LN_F32 && dtype != LN_F16) return ln_fail(ctx, LN_ERR_ARG, "%s: dtype must be LN_F32 or LN_F16", who);
    return guarded(ctx, who, [&]() -> int32_t {
        cudaSetDevice(ctx->device);
        ln_tensor* y = nullptr;
        int rc = new_tensor(ctx, dtype, t->n, t->c, t->h, t->w, &y);
        if (rc) return rc;
        rc = widen_into(ctx, t, y);
        if (rc) { ln_tensor_release(y); return rc; }
        *out = y;
        return LN_OK;
    });
}

int32_t ln_tensor_download_f4(ln_ctx* ctx, const ln_tensor* t, uint8_t* host_codes, int64_t code_count, uint8_t* host_scales, int64_t scale_count) {
    const char* who = "ln_tensor_download_f4";
    if (!ctx || !t || !host_codes || !host_scales) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (!ln_is_f4(t->dtype)) return ln_fail(ctx, LN_ERR_ARG, "%s: 4-bit tensor required", who);
    if (t->ctx != ctx) return ln_fail(ctx, LN_ERR_ARG, "%s: the tensor belongs to another context", who);
    const int sf_blocks = (int)((t->c + ln_f4_block(t->dtype) - 1) / ln_f4_block(t->dtype));
    const int64_t hw = t->h * t->w, scales = t->n * sf_blocks * hw;
    if (code_count != t->count() || scale_count != scales)
        return ln_fail(ctx, LN_ERR_SHAPE, "%s: the tensor has %lld codes and %lld scales", who, (long long)t->count(), (long long)scales);
    return guarded(ctx, who, [&]() -> int32_t {
        cudaSetDevice(ctx->device);
        uint8_t* tmp = (uint8_t*)ln_pool_alloc(ctx, (size_t)(code_count + scales));
        if (!tmp) return LN_ERR_CUDA;
        cudaError_t e = ln_f4_launch(ctx, unpack_f4_kernel, grid_for(ctx, code_count + scales), kThreads, 0, (const uint8_t*)t->ptr, (const uint8_t*)t->sf, tmp, tmp + code_count, t->n, hw, (int)t->c, sf_blocks,
                                                                                         t->cstride, t->sf_words);
        int rc = check_launch(ctx, who, e);
        if (rc == LN_OK) {
            e = cudaMemcpyAsync(host_codes, tmp, (size_t)code_count, cudaMemcpyDeviceToHost, ctx->stream);
            if (e == cudaSuccess) e = cudaMemcpyAsync(host_scales, tmp + code_count, (size_t)scales, cudaMemcpyDeviceToHost, ctx->stream);
            const cudaError_t s = cudaStreamSynchronize(ctx->stream);
            if (e == cudaSuccess) e = s;
        }
        ln_pool_free(ctx, tmp, 0);
        if (e != cudaSuccess) return ln_fail(ctx, LN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
        return rc ? rc : ln_status(ctx, who);
    });
}

int32_t ln_conv_weights_f4(ln_ctx* ctx, const ln_tensor* weights_f32, int64_t filters, int64_t channels, int64_t kernel_size, int32_t dtype, ln_conv_weights** out) {
    const char* who = "ln_conv_weights_f4";
    if (!ctx || !weights_f32 || !out) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (weights_f32->dtype != LN_F32) return ln_fail(ctx, LN_ERR_ARG, "%s: f32 weights required", who);
    if (weights_f32->ctx != ctx) return ln_fail(ctx, LN_ERR_ARG, "%s: the tensor belongs to another context", who);
    if (!ln_is_f4(dtype)) return ln_fail(ctx, LN_ERR_ARG, "%s: dtype must be LN_F4 or LN_MX4", who);
    if (channels > 0 && kernel_size > 0 && kernel_size <= 64 && channels <= (1 << 24) && channels * kernel_size * kernel_size >= (1ll << 31))
        return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: a filter has 2^31 weights or more", who);
    if (filters < 1 || channels < 1 || kernel_size < 1 || filters > (1 << 24) || channels > (1 << 24) || kernel_size > 64 || weights_f32->count() != filters * channels * kernel_size * kernel_size)
        return ln_fail(ctx, LN_ERR_SHAPE, "%s: weight tensor has %lld elements, expected %lld x %lld x %lld x %lld", who, (long long)weights_f32->count(), (long long)filters, (long long)channels,
                       (long long)kernel_size, (long long)kernel_size);
    return guarded(ctx, who, [&]() -> int32_t {
        cudaSetDevice(ctx->device);
        const int64_t k2 = kernel_size * kernel_size;
        const int64_t sf_words = ln_f4_sf_words(dtype, channels);
        ln_conv_weights* w = new ln_conv_weights();
        w->ctx = ctx; w->dtype = dtype;
        w->filters = filters; w->channels = channels; w->k = kernel_size;
        w->fpad = ln_round_up(filters, 128) + kF4FilterPad; w->cpad = ln_f4_cstride(channels);
        const size_t sf_bytes = (size_t)(w->fpad / 128 * k2 * sf_words * 512);
        w->w = ln_pool_alloc(ctx, (size_t)(filters * k2 * w->cpad));
        w->sf = ln_pool_alloc(ctx, sf_bytes);
        w->wscale = (float*)ln_pool_alloc(ctx, (size_t)filters * 4);
        if (!w->w || !w->sf || !w->wscale) { ln_conv_weights_release(w); return LN_ERR_CUDA; }
        int rc = LN_OK;
        cudaError_t e = cudaMemsetAsync(w->sf, 0, sf_bytes, ctx->stream);
        if (e != cudaSuccess) rc = ln_fail(ctx, LN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
        if (rc == LN_OK) {
            if (dtype == LN_F4) e = ln_f4_launch(ctx, pack_weights_f4_kernel<LN_F4>, (int)filters, 256, 0, (const float*)weights_f32->ptr, (int)channels, (int)k2, w->cpad, (uint8_t*)w->w, (uint8_t*)w->sf, w->wscale, sf_words);
            else e = ln_f4_launch(ctx, pack_weights_f4_kernel<LN_MX4>, (int)filters, 256, 0, (const float*)weights_f32->ptr, (int)channels, (int)k2, w->cpad, (uint8_t*)w->w, (uint8_t*)w->sf, w->wscale, sf_words);
            rc = check_launch(ctx, who, e);
        }
        if (rc) { ln_conv_weights_release(w); return rc; }
        *out = w;
        return LN_OK;
    });
}

int32_t ln_conv2d_bias_act_f4(ln_ctx* ctx, const ln_tensor* x, const ln_conv_weights* weights, const ln_tensor* bias, const int64_t output_shape[4], int64_t channels,
                              int64_t input_height, int64_t input_width, int64_t filters, int64_t kernel_size, int64_t stride_x, int64_t stride_y, int64_t dilation,
                              int64_t padding, int64_t groups, int32_t activation, float y_scale, int32_t out_kind, ln_tensor** out) {
    const char* who = "ln_conv2d_bias_act_f4";
    if (!ctx || !x || !weights || !bias || !output_shape || !out) return ln_fail(ctx, LN_ERR_ARG, "%s: NULL argument", who);
    if (!ln_is_f4(x->dtype)) return ln_fail(ctx, LN_ERR_ARG, "%s: 4-bit input required", who);
    if (weights->dtype != x->dtype) return ln_fail(ctx, LN_ERR_ARG, "%s: input and weights have different types", who);
    if (x->ctx != ctx || weights->ctx != ctx || bias->ctx != ctx) return ln_fail(ctx, LN_ERR_ARG, "%s: an operand belongs to another context", who);
    if (bias->dtype != LN_F32 || bias->count() != filters) return ln_fail(ctx, LN_ERR_SHAPE, "%s: bias must be f32 [filters]", who);
    if (groups != 1 || dilation != 1) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: groups and dilation must be 1", who);
    if (kernel_size < 1 || stride_x < 1 || stride_y < 1 || stride_x > 64 || stride_y > 64 || padding < 0 || padding > 64) return ln_fail(ctx, LN_ERR_SHAPE, "%s: invalid geometry", who);
    if (x->c != channels || x->h != input_height || x->w != input_width || weights->filters != filters || weights->channels != channels || weights->k != kernel_size)
        return ln_fail(ctx, LN_ERR_SHAPE, "%s: geometry does not match the tensors", who);
    if (activation < LN_ACT_LINEAR || activation > LN_ACT_RELU) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: activation %d is not on the detector path", who, activation);
    if (out_kind != LN_OUT_Q && out_kind != LN_OUT_F32 && out_kind != LN_OUT_F16) return ln_fail(ctx, LN_ERR_ARG, "%s: out_kind must be LN_OUT_Q, LN_OUT_F32 or LN_OUT_F16", who);
    if (out_kind == LN_OUT_Q && !usable_scale(x->dtype, y_scale)) return ln_fail(ctx, LN_ERR_ARG, "%s: y_scale %g is not %s", who, y_scale, x->dtype == LN_MX4 ? "1 (LN_MX4 has no tensor scale)" : "in [2^-100, 2^100]");
    const int64_t oh = (input_height + 2 * padding - kernel_size < 0 ? 0 : input_height + 2 * padding - kernel_size) / stride_y + 1;
    const int64_t ow = (input_width + 2 * padding - kernel_size < 0 ? 0 : input_width + 2 * padding - kernel_size) / stride_x + 1;
    if (output_shape[0] != x->n || output_shape[1] != filters || output_shape[2] != oh || output_shape[3] != ow)
        return ln_fail(ctx, LN_ERR_SHAPE, "%s: output_shape does not match [%lld,%lld,%lld,%lld]", who, (long long)x->n, (long long)filters, (long long)oh, (long long)ow);
    if (input_height > (1 << 24) || input_width > (1 << 24)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: more than 2^24 rows or columns", who);
    int rc = ln_status(ctx, who);  // of an earlier call
    if (rc) return rc;
    ctx->f4_plan[0] = ctx->f4_plan[1] = ctx->f4_plan[2] = 0;
    return guarded(ctx, who, [&]() -> int32_t {
        cudaSetDevice(ctx->device);
        ln_tensor* y = nullptr;
        int rc = new_tensor(ctx, out_kind == LN_OUT_Q ? x->dtype : (out_kind == LN_OUT_F16 ? LN_F16 : LN_F32), x->n, filters, oh, ow, &y);
        ln_f4_conv c;
        c.dtype = x->dtype; c.x = x; c.w = weights; c.bias = (const float*)bias->ptr; c.y = y;
        c.k = (int)kernel_size; c.stride = (int)stride_x; c.pad = (int)padding; c.act = activation; c.out_kind = out_kind;
        if (rc == LN_OK && out_kind == LN_OUT_Q) y->scale = y_scale;
        const bool few = kernel_size == 1 && stride_x == 1 && stride_y == 1 && padding == 0 && x->n * oh * ow <= kFewPixels;
        if (rc == LN_OK && (few || ln_f4_umma_takes(c, stride_x, stride_y))) {
            rc = few ? few_launch(ctx, c, x->n * oh * ow) : ln_f4_umma_launch(ctx, c);
            if (rc) { ln_tensor_release(y); return rc; }
            *out = y;
            return LN_OK;
        }
        if (rc == LN_OK && y->dtype == LN_F16 && y->cstride != 2 * filters) {
            const cudaError_t e = cudaMemsetAsync(y->ptr, 0, y->bytes, ctx->stream);
            if (e != cudaSuccess) rc = ln_fail(ctx, LN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
        }
        if (rc == LN_OK) {
            simt_params p;
            p.x = (const uint8_t*)x->ptr; p.xsf = (const uint8_t*)x->sf; p.w = (const uint8_t*)weights->w; p.wsf = (const uint8_t*)weights->sf;
            p.wscale = weights->wscale; p.bias = (const float*)bias->ptr; p.y = y->ptr; p.ysf = (uint8_t*)y->sf;
            p.xs = x->cstride; p.xsf_words = x->sf_words; p.ys = out_kind == LN_OUT_F16 ? y->cstride / 2 : y->cstride; p.ysf_words = y->sf_words;
            p.fpad = out_kind == LN_OUT_Q ? (int)ln_round_up(filters, 64) : (int)filters; p.total = x->n * oh * ow * p.fpad;
            p.H = (int)input_height; p.W = (int)input_width; p.F = (int)filters; p.k = (int)kernel_size; p.sx = (int)stride_x; p.sy = (int)stride_y; p.pad = (int)padding;
            p.OH = (int)oh; p.OW = (int)ow; p.blocks = (int)(x->cstride * 2 / ln_f4_block(x->dtype));
            p.act = activation; p.out_kind = out_kind; p.xscale = x->scale; p.g = y->scale; p.six_g = 6.0f * y->scale;
            const int grid = grid_for(ctx, p.total);
            cudaError_t e;
            if (x->dtype == LN_F4) {
                if (ctx->exact_epilogue) e = ln_f4_launch(ctx, conv_f4_simt_kernel<LN_F4, true>, grid, kThreads, 0, p);
                else e = ln_f4_launch(ctx, conv_f4_simt_kernel<LN_F4, false>, grid, kThreads, 0, p);
            } else {
                if (ctx->exact_epilogue) e = ln_f4_launch(ctx, conv_f4_simt_kernel<LN_MX4, true>, grid, kThreads, 0, p);
                else e = ln_f4_launch(ctx, conv_f4_simt_kernel<LN_MX4, false>, grid, kThreads, 0, p);
            }
            rc = check_launch(ctx, who, e);
        }
        if (rc) { if (y) ln_tensor_release(y); return rc; }
        *out = y;
        return LN_OK;
    });
}

}  // extern "C"
