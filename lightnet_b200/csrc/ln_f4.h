// Storage of the microscaled 4-bit types, shared by their operators.
//
// A tensor is NHWC: per pixel two codes per byte (channel 2i in the low nibble), channels padded to 64, so that a pixel is a multiple
// of the 32 bytes that one tensor-core instruction consumes.  Weights are the same with a filter's taps in the place of a pixel.
// The k range of a product is cut into k-blocks of `bk` bytes of one tap (the last one of a tap may be shorter), a k-block's scales into
// `words` of 4 bytes: LN_F4 has one word for the 64 channels of an instruction, LN_MX4 one for the 128 of two.
// Block scales lie behind the codes in the order in which the tensor cores take them: per 128 pixels (filters) and k-block `words`
// groups of 512 bytes, [32 pixels][4 groups of 32 pixels][4 scale bytes], so that pixel q has its word at q % 32 * 16 + q / 32 % 4 * 4.
// A product over pixels in their own order copies them as they are; one whose taps shift the pixels gathers words.
// Codes and scales of the padding up to 64 channels are zero; the other scale bytes of a group are never used.
#pragma once

#include <cstdint>

#include "ln_umma.h"

inline bool ln_is_f4(int dtype) { return dtype == LN_F4 || dtype == LN_MX4; }
inline int ln_f4_block(int dtype) { return dtype == LN_MX4 ? 32 : 16; }
inline int64_t ln_f4_cstride(int64_t c) { return ln_round_up(c, 64) / 2; }
struct ln_f4_kblocks {
    int bk, cblocks, words;
};
inline ln_f4_kblocks ln_f4_kblocks_of(int dtype, int64_t c) {
    const int64_t cstride = ln_f4_cstride(c);
    ln_f4_kblocks k;
    k.bk = cstride <= 32 ? 32 : (cstride <= 64 ? 64 : 128);
    k.cblocks = (int)((cstride + k.bk - 1) / k.bk);
    k.words = dtype == LN_MX4 ? (k.bk + 63) / 64 : k.bk / 32;
    return k;
}
inline int64_t ln_f4_sf_words(int dtype, int64_t c) {  // of a pixel
    const ln_f4_kblocks k = ln_f4_kblocks_of(dtype, c);
    return (int64_t)k.cblocks * k.words;
}
inline int64_t ln_f4_sf_bytes(int dtype, int64_t pixels, int64_t c) { return (pixels + 127) / 128 * ln_f4_sf_words(dtype, c) * 512; }
// Scales are there for this many filters behind the last group of 128 (zeros): a tile of up to 256 filters may start at the last one.
constexpr int64_t kF4FilterPad = 256;

#ifdef __CUDACC__
// byte of the scales at which word w of pixel q starts
__host__ __device__ __forceinline__ int64_t ln_f4_sf_at(int64_t q, int64_t w, int64_t words_per_pixel) {
    return ((q >> 7) * words_per_pixel + w) * 512 + (q & 31) * 16 + (q >> 5 & 3) * 4;
}

// ---- the number formats -----------------------------------------------------------------------------------------------------------

// The 4-bit kernels are launched as programmatic dependents: they may start, and set up what is their own, while the kernel in front of
// them still runs.  Every thread comes by here before it reads or writes global memory.
__device__ __forceinline__ void ln_f4_after_predecessor() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void ln_store_32(void* dst, const uint32_t (&v)[8]) {  // a whole sector
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// max that hands a NaN on
__device__ __forceinline__ float ln_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// x >= 0 -> E4M3 (nearest even, saturating at 448; NaN is 0x7F) and back
__device__ __forceinline__ uint32_t ln_e4m3_of(float x) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(0.0f), "f"(x));  // second source -> low byte
    return d & 0xFFu;
}
__device__ __forceinline__ float ln_e4m3_value(uint32_t code) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}
// 2^(code - 127): 0 is 2^-127, 255 is NaN
__device__ __forceinline__ float ln_e8m0_value(uint32_t code) {
    return code == 255u ? __uint_as_float(0x7FC00000u) : (code ? __uint_as_float(code << 23) : __uint_as_float(0x00400000u));
}
// eight values -> eight E2M1 codes (nearest even, saturating at 6), the first in the lowest nibble
__device__ __forceinline__ uint32_t ln_e2m1x8(float a, float b, float c, float d, float e, float f, float g, float h) {
    uint32_t r;
    asm("{\n\t.reg .b8 p, q, r, s;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 p, %2, %1;\n\t"  // first source -> high nibble
        "cvt.rn.satfinite.e2m1x2.f32 q, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 r, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 s, %8, %7;\n\t"
        "mov.b32 %0, {p, q, r, s};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f), "f"(g), "f"(h));
    return r;
}
// eight codes -> four binary16 pairs, in order
__device__ __forceinline__ void ln_e2m1x8_to_h2(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 p, q, r, s;\n\t"
        "mov.b32 {p, q, r, s}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, p;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, q;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, r;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, s;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}

// Activations behind a product.  The 8-bit types clamp what goes into exp (their codes cannot show it); these types hold values of the whole range,
// where v / (1 + e^60) is no longer small.  Below the clamp, swish and mish are v e^v and the logistic e^v to 1e-26 of their value: e^v is the
// square of e^(v / 2), which is 0 after the clamp of ln_det_expf too.
template <bool EXACT>
__host__ __device__ constexpr float ln_f4_far(int act) {  // from here down; -inf for activations that need no exp
    return act == LN_ACT_MISH || act == LN_ACT_SWISH || act == LN_ACT_LOGISTIC ? (EXACT ? -87.0f : -60.0f) : -__builtin_huge_valf();
}
__device__ __forceinline__ float ln_f4_act_far(int act, float v) {
    const float h = ln_det_expf(0.5f * v);
    return act == LN_ACT_LOGISTIC ? __fmul_rn(h, h) : __fmul_rn(__fmul_rn(fmaxf(v, -1000.0f), h), h);  // (-inf times 0 is no number)
}
template <bool EXACT>
__device__ __forceinline__ float ln_f4_act(int act, float v) {
    if (act == LN_ACT_RELU) return ln_max_nan(v, 0.0f);
    const float a = v < ln_f4_far<EXACT>(act) ? ln_f4_act_far(act, v) : ln_epilogue_act<EXACT>(act, v);
    return v == v ? a : v;  // (a NaN stays one: the clamps of the 8-bit types drop it)
}

// Block scale: its stored byte and the binary32 factor d of the codes (g is not used for LN_MX4).
template <int FMT>
__device__ __forceinline__ uint32_t ln_f4_scale_of(float amax, float six_g) {
    if (FMT == LN_F4) return ln_e4m3_of(__fdiv_rn(amax, six_g));
    const uint32_t bits = __float_as_uint(amax), field = (bits >> 23) & 0xFFu;
    if (bits > 0x7F800000u) return 255u;
    return field > 2u ? field - 2u : 0u;  // e + 127 = (field - 127) - 2 + 127
}
template <int FMT>
__device__ __forceinline__ float ln_f4_factor(uint32_t scale, float g) {
    return FMT == LN_F4 ? __fmul_rn(ln_e4m3_value(scale), g) : ln_e8m0_value(scale);
}

// The codes of one block: B = 16 (LN_F4) or 32 (LN_MX4) values -> B / 8 words.  Returns the scale byte.
template <int FMT>
__device__ __forceinline__ uint32_t ln_f4_quantise(const float* x, float g, float six_g, uint32_t* codes) {
    constexpr int B = FMT == LN_F4 ? 16 : 32;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < B; ++i) amax = ln_max_nan(amax, fabsf(x[i]));
    const uint32_t scale = ln_f4_scale_of<FMT>(amax, six_g);
    float t[B];
    if (FMT == LN_F4) {
        // x / d by one correction of x * (1 / d), three operations instead of a division: the codes are those of the rounded quotient for every
        // d >= 2^-101 (for all 2^23 significands of d and the x next to each border between codes); below that the correction's remainder loses
        // bits, so smaller ones are taken 2^64 times as large.  Codes end at 6, so quotients end at 8 where the scale is the largest and they may be of any size
        // (|x / d| is at most 9 otherwise, at the smallest scale).
        float d = ln_f4_factor<FMT>(scale, g);
        if (scale == 126u || __float_as_uint(d) - 1u < 0x0F800000u - 1u) {  // 0 < d < 2^-96
            const float up = d < 0x1p-96f ? 0x1p64f : 1.0f, most = 8.0f * (d *= up);
#pragma unroll
            for (int i = 0; i < B; ++i) t[i] = fminf(fmaxf(__fmul_rn(x[i], up), -most), most);
        } else {
#pragma unroll
            for (int i = 0; i < B; ++i) t[i] = x[i];
        }
        const float r = scale ? __frcp_rn(d) : 0.0f;
#pragma unroll
        for (int i = 0; i < B; i += 2) {
            float q0, q1, e0, e1;
            fmul2(q0, q1, t[i], t[i + 1], r, r);
            ffma2(e0, e1, -q0, -q1, d, d, t[i], t[i + 1]);
            ffma2(t[i], t[i + 1], e0, e1, r, r, q0, q1);
        }
    } else {
        const float inv = __uint_as_float((254u - (scale > 253u ? 253u : scale)) << 23);  // 2^-e, exact
#pragma unroll
        for (int i = 0; i < B; ++i) t[i] = __fmul_rn(x[i], inv);
    }
#pragma unroll
    for (int w = 0; w < B / 8; ++w)
        codes[w] = ln_e2m1x8(t[8 * w], t[8 * w + 1], t[8 * w + 2], t[8 * w + 3], t[8 * w + 4], t[8 * w + 5], t[8 * w + 6], t[8 * w + 7]);
    return scale;
}
#endif

// ---- the product on the tensor cores (ln_f4_umma.cu) --------------------------------------------------------------------------------
struct ln_f4_conv {  // one convolution: operands, geometry, output
    int dtype = LN_F4;
    const ln_tensor* x = nullptr;
    const ln_conv_weights* w = nullptr;
    const float* bias = nullptr;
    ln_tensor* y = nullptr;
    int k = 1, stride = 1, pad = 0, act = 0, out_kind = LN_OUT_F32;
};
// launches a 4-bit kernel (all begin with ln_f4_after_predecessor) on the ctx stream, in clusters of `cluster` CTAs
template <typename... P, typename... A>
inline cudaError_t ln_f4_launch_clusters(ln_ctx* ctx, void (*kernel)(P...), int grid, int threads, size_t smem, int cluster, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)cluster;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    ctx->launches++;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... A>
inline cudaError_t ln_f4_launch(ln_ctx* ctx, void (*kernel)(P...), int grid, int threads, size_t smem, const A&... args) {
    return ln_f4_launch_clusters(ctx, kernel, grid, threads, smem, 1, args...);
}
bool ln_f4_umma_takes(const ln_f4_conv& c, int64_t stride_x, int64_t stride_y);
int ln_f4_umma_launch(ln_ctx* ctx, const ln_f4_conv& c);
