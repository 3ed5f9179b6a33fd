// The 4-bit product on the tensor cores: tcgen05.mma with block scales (kind::mxf4nvf4, scale_vec::4X for LN_F4; kind::mxf4,
// scale_vec::2X for LN_MX4), operands and scales in shared memory and TMEM, bias + activation + output conversion in the epilogue.
//
// GEMM view as for the 8-bit types: D[pixel, filter] = sum over (tap, channel block) of X[pixel shifted by the tap, c] * W[filter, tap, c];
// a tile is 128 output pixels (a TW x TH x TN box; a 1x1 stride-1 convolution is flattened to one row of pixels) by bn filters, a
// k-block 128 bytes = 256 channels of one tap (fewer where the tensor has fewer): four instructions of 64 channels.
// Codes come by TMA (taps outside the image are zero filled; stride 2 has one tensor map per parity class of the input).  The scales
// of the weights lie in memory as the tensor core takes them and come by bulk copies.  Those of the pixels cannot: every tap needs the
// scales of other pixels in the rows of the tile, so two warps gather them, one lane for the rows l, l + 32, l + 64, l + 96, whose four
// words it stores transposed as one 16-byte piece per instruction.  The issuing thread copies both from shared memory to TMEM
// (tcgen05.cp, executed in order with the instructions that read them) right before the k-block that they belong to.
//
// Roles: warp 0 loads, warp 1 issues, warps 2 and 3 gather scales (every second k-block each), 16 epilogue warps.  An accumulator tile is
// handed out as `subs` units of CH columns; a unit is read into registers whole and its part of TMEM handed back before any arithmetic.
// TMEM: 416 columns of accumulators (one tile of 256 filters, two of 192, three of 128, six of 64), 2 x 48 of scales.
// Every wait is bounded (see ln_umma.h).
#include <cstdlib>

#include "ln_f4.h"
#include "ln_umma.h"

namespace {

constexpr int kThreadsF4 = 32 * 20;
constexpr int kMaxStagesF4 = 8, kMaxBufsF4 = 6;
constexpr uint32_t kScaleCols = 416, kScaleSet = 48, kScaleB = 16;  // TMEM columns: two sets of [16 pixels' | 32 filters'] scale words
constexpr uint32_t kBarBytesF4 = 512;
constexpr uint32_t kTabBytesF4 = 16 * 512;  // {multiplier, bias} of the columns that a warp is at
constexpr int kMaxSmemF4 = 227 * 1024;

struct f4_params {
    CUtensorMap tmA[4], tmB;
    const uint8_t *xsf, *wsf;
    const float *wscale, *bias;
    void* y;
    uint8_t* ysf;
    int* status;
    long long ys, ysf_stride;  // bytes per pixel of an NHWC output, of its scales
    float xscale, g, six_g;    // tensor scale of the input; of a 4-bit output
    int sf_stride, cstride;
    int bk, bn, cblocks, words, wblocks;  // wblocks: groups of 128 filters a tile's scales are in
    int R, S, stride, pad, H, W, N, OH, OW, F, hw;
    int TW, TH, TN, log_tw, log_th, tiles_f, tiles_w, tiles_h, num_tiles;
    unsigned long long magic_f, magic_w, magic_h;
    int stages, nbuf, subs, act, exact;
    uint32_t off_b, off_sfa, off_sfb, stage_bytes;
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
// a wait of the whole warp: one answer for all lanes
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 32 rows of 16 bytes -> the four 32-lane quarters of TMEM, four columns
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void tc_mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (FMT == LN_F4)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
            : "memory");
}
// descriptor of 32 rows of 16 bytes (no swizzle, groups of 8 rows 128 bytes apart)
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) { return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46); }

template <int CH>
__device__ __forceinline__ void act_all(int act, bool exact, float (&v)[CH]) {
#define LN_ALL(E, A)                                                       \
    _Pragma("unroll") for (int i = 0; i < CH; ++i) v[i] = ln_epilogue_act<E>(A, v[i]); \
    break;
    switch (act) {
        case LN_ACT_LEAKY: LN_ALL(true, LN_ACT_LEAKY)
        case LN_ACT_RELU: LN_ALL(true, LN_ACT_RELU)
        case LN_ACT_MISH:
            if (exact) { LN_ALL(true, LN_ACT_MISH) }
            LN_ALL(false, LN_ACT_MISH)
        case LN_ACT_SWISH:
            if (exact) { LN_ALL(true, LN_ACT_SWISH) }
            LN_ALL(false, LN_ACT_SWISH)
        case LN_ACT_LOGISTIC:
            if (exact) { LN_ALL(true, LN_ACT_LOGISTIC) }
            LN_ALL(false, LN_ACT_LOGISTIC)
        default: break;
    }
#undef LN_ALL
}

// the tile's place: output box origin and first filter
struct f4_tile {
    int ow0, oh0, n0, f0;
};
__device__ __forceinline__ f4_tile tile_at(const f4_params& p, int unit) {
    const int q1 = fast_div(unit, p.magic_f), tf = unit - q1 * p.tiles_f;
    const int q2 = fast_div(q1, p.magic_w), tw = q1 - q2 * p.tiles_w;
    const int tn = fast_div(q2, p.magic_h), th = q2 - tn * p.tiles_h;
    return {tw * p.TW, th * p.TH, tn * p.TN, tf * p.bn};
}

template <int FMT, int OUT, int CH>
__global__ void __launch_bounds__(kThreadsF4, 1) f4_umma_kernel(const __grid_constant__ f4_params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + (uint32_t)p.stages * p.stage_bytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStagesF4 + s); };
    auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStagesF4 + b); };
    auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStagesF4 + kMaxBufsF4 + b); };
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(smem_raw + (bar_base - smem_u32(smem_raw)) + 8u * (2 * kMaxStagesF4 + 2 * kMaxBufsF4));
    volatile int* abort_flag = (volatile int*)(tmem_slot + 2);
    const uint32_t tab_base = bar_base + kBarBytesF4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full_bar(s), 2);  // the loader (with the copies' bytes) and the warp that gathers scales
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < p.nbuf; ++b) {
            mbar_init(tfull_bar(b), 1);
            mbar_init(tempty_bar(b), 4 * p.subs);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int kblocks = p.R * p.S * p.cblocks, step = (int)gridDim.x;

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        if (lane == 0) {
            const uint32_t bytes = (uint32_t)(128 + p.bn) * p.bk + (uint32_t)p.wblocks * p.words * 512u;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = (int)blockIdx.x; ok && unit < p.num_tiles; unit += step) {
                const f4_tile t = tile_at(p, unit);
                const uint8_t* wsf = p.wsf + (size_t)(t.f0 >> 7) * kblocks * p.words * 512u;
                int wcol = 0, kb = 0;
                for (int r = 0; ok && r < p.R; ++r)
                    for (int s = 0; ok && s < p.S; ++s, wcol += p.cstride) {
                        int ty = r - p.pad, tx = s - p.pad, map = 0;
                        if (p.stride == 2) {
                            const int py = ty & 1, px = tx & 1;  // parity class of the tap
                            ty = (ty - py) >> 1;
                            tx = (tx - px) >> 1;
                            map = py * 2 + px;
                        }
                        for (int c0 = 0; c0 < p.cstride; c0 += p.bk, ++kb) {
                            if (!(ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                            const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes, bar = full_bar(stage);
                            mbar_arrive_expect_tx(bar, bytes);
                            tma_load_4d(at, &p.tmA[map], c0, t.ow0 + tx, t.oh0 + ty, t.n0, bar);
                            tma_load_2d(at + p.off_b, &p.tmB, wcol + c0, t.f0, bar);
                            for (int b = 0; b < p.wblocks; ++b)
                                bulk_load(at + p.off_sfb + (uint32_t)(b * p.words) * 512u, wsf + ((size_t)b * kblocks + kb) * p.words * 512u, (uint32_t)p.words * 512u, bar);
                            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                        }
                    }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ instructions (the whole warp walks the loop; one lane issues)
        const bool leader = elect_one();
        // E2M1 operands (bits 7, 10: type 1), N / 8, scale type (bit 23: 1 = E8M0), M / 128, K-major; the scale ids go to bits 4 and 29
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | ((FMT == LN_MX4 ? 1u : 0u) << 23) | (1u << 27);
        const uint64_t desc_base = make_smem_desc(0u, p.bk);
        int stage = 0, t = 0;
        uint32_t phase = 0, set = 0;
        bool ok = true;
        for (int unit = (int)blockIdx.x; ok && unit < p.num_tiles; unit += step, ++t) {
            const int buf = t % p.nbuf;
            if (!(ok = warp_wait(tempty_bar(buf), (uint32_t)((t / p.nbuf) & 1) ^ 1u, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
            tc_fence_after();
            const uint32_t d = tmem_base + (uint32_t)(buf * p.bn);
            const int tf = unit - fast_div(unit, p.magic_f) * p.tiles_f;
            const uint32_t shift = (uint32_t)((tf * p.bn & 127) >> 5);  // first column of the tile's filters inside their group of 128
            int c0 = 0;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!(ok = warp_wait(full_bar(stage), phase, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
                tc_fence_after();
                const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes;
                const uint32_t sfa = tmem_base + kScaleCols + set * kScaleSet, sfb = sfa + kScaleB;
                const int left = p.cstride - c0, n = (left < p.bk ? left : p.bk) >> 5;  // instructions of this k-block
                if (leader) {
                    for (int j = 0; j < p.words; ++j) {
                        tc_copy_scales(sfa + 4u * j, scale_desc(at + p.off_sfa + 512u * j));
                        for (int b = 0; b < p.wblocks; ++b) tc_copy_scales(sfb + 4u * (j * p.wblocks + b), scale_desc(at + p.off_sfb + 512u * (b * p.words + j)));
                    }
                    const uint64_t a_desc = desc_base + (at >> 4), b_desc = desc_base + ((at + p.off_b) >> 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < n) {
                            const uint32_t word = FMT == LN_MX4 ? i >> 1 : i, id = FMT == LN_MX4 ? (uint32_t)(i & 1) * 2u : 0u;
                            tc_mma_scaled<FMT>(d, a_desc + 2u * i, b_desc + 2u * i, idesc | (id << 4) | (id << 29), sfa + 4u * word, sfb + 4u * word * p.wblocks + shift, (uint32_t)((kb | i) != 0));
                        }
                    tc_commit(empty_bar(stage));
                }
                __syncwarp();
                set ^= 1u;
                c0 += p.bk;
                if (c0 >= p.cstride) c0 = 0;
                if (++stage == p.stages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) break;
            if (leader) tc_commit(tfull_bar(buf));
            __syncwarp();
        }
    } else if (warp < 4) {
        // ------------------------------------------------------------------ scales of the pixels
        const int which = warp - 2;
        int unit = (int)blockIdx.x, r = 0, s = 0, cb = 0;
        int iy0[4], ix0[4], img[4];
        auto enter_tile = [&]() {
            if (unit >= p.num_tiles) return;
            const f4_tile t = tile_at(p, unit);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int row = g * 32 + lane;
                ix0[g] = (t.ow0 + (row & (p.TW - 1))) * p.stride - p.pad;
                iy0[g] = (t.oh0 + ((row >> p.log_tw) & (p.TH - 1))) * p.stride - p.pad;
                img[g] = t.n0 + (row >> (p.log_tw + p.log_th));
            }
        };
        auto advance = [&]() {
            if (++cb < p.cblocks) return;
            cb = 0;
            if (++s < p.S) return;
            s = 0;
            if (++r < p.R) return;
            r = 0;
            unit += step;
            enter_tile();
        };
        auto fetch = [&](uint32_t (&v)[4][4]) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int y = iy0[g] + r, x = ix0[g] + s;
                uint4 q = make_uint4(0u, 0u, 0u, 0u);
                if (y >= 0 && y < p.H && x >= 0 && x < p.W && img[g] < p.N) {
                    const uint8_t* src = p.xsf + (((long long)img[g] * p.H + y) * p.W + x) * p.sf_stride + (long long)cb * p.words * 4;
                    if (p.words == 4) q = __ldg((const uint4*)src);
                    else if (p.words == 2) { const uint2 h = __ldg((const uint2*)src); q.x = h.x; q.y = h.y; }
                    else q.x = __ldg((const uint32_t*)src);
                }
                v[g][0] = q.x; v[g][1] = q.y; v[g][2] = q.z; v[g][3] = q.w;
            }
        };
        enter_tile();
        if (which == 1) advance();
        int stage = which == 1 ? 1 % p.stages : 0;
        uint32_t phase = which == 1 && p.stages == 1 ? 1u : 0u;
        uint32_t now[4][4], next[4][4];
        bool more = unit < p.num_tiles, ok = true;
        if (more) fetch(now);
        while (more && ok) {
            advance();
            advance();
            more = unit < p.num_tiles;
            if (more) fetch(next);
            if (!(ok = warp_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
            const uint32_t dst = smem_base + (uint32_t)stage * p.stage_bytes + p.off_sfa + 16u * lane;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < p.words)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512u * j), "r"(now[0][j]), "r"(now[1][j]), "r"(now[2][j]), "r"(now[3][j]) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full_bar(stage));
            stage += 2;
            if (stage >= p.stages) { stage -= p.stages; phase ^= 1u; }
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) now[g][j] = next[g][j];
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        // Units (tile, sub) in order; group g takes those with number % groups == g.  Never more groups than nbuf * subs: a group that
        // waits for a tile's accumulator has finished a unit of the tile nbuf before it or a later one, so the parity is unambiguous.
        const int quad = warp & 3, group = (warp - 4) >> 2;
        const int groups = p.nbuf * p.subs < 4 ? p.nbuf * p.subs : 4;
        const int row = quad * 32 + lane, pw = row & (p.TW - 1), ph = (row >> p.log_tw) & (p.TH - 1), pn = row >> (p.log_tw + p.log_th);
        const uint32_t tab = tab_base + (uint32_t)(warp - 4) * 512u;
        int t = 0, turn = 0;
        bool ok = true;
        for (int unit = (int)blockIdx.x; ok && group < groups && unit < p.num_tiles; unit += step, ++t)
            for (int sub = 0; ok && sub < p.subs; ++sub, turn = turn + 1 == groups ? 0 : turn + 1) {
                if (turn != group) continue;
                const f4_tile at = tile_at(p, unit);
                const int ow = at.ow0 + pw, oh = at.oh0 + ph, n = at.n0 + pn, f0 = at.f0 + sub * CH;
                const bool valid = ow < p.OW && oh < p.OH && n < p.N;
                const long long pix = ((long long)n * p.OH + oh) * p.OW + ow;
                const int buf = t % p.nbuf;
                __syncwarp();  // (the table of the unit before has been read)
#pragma unroll
                for (int i = lane; i < CH; i += 32) {
                    const int f = f0 + i;
                    const float m = f < p.F ? __fmul_rn(p.xscale, __ldg(p.wscale + f)) : 0.0f, b = f < p.F ? __ldg(p.bias + f) : 0.0f;
                    asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(tab + 8u * i), "f"(m), "f"(b) : "memory");
                }
                __syncwarp();
                if (!(ok = warp_wait(tfull_bar(buf), (uint32_t)((t / p.nbuf) & 1), abort_flag, p.status, LN_STATUS_EPILOGUE_TIMEOUT))) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * p.bn + sub * CH);
                uint32_t acc[CH / 32][32];
#pragma unroll
                for (int c = 0; c < CH / 32; ++c) tmem_ld_32x32(taddr + 32u * c, acc[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(buf));
                if (f0 >= p.F && !(OUT == LN_OUT_Q && f0 < ((p.F + 63) & ~63))) continue;  // nothing but padding (the columns of a tile that no filter has)
                float v[CH];
#pragma unroll
                for (int i = 0; i < CH; i += 2) {
                    float4 e;  // (volatile: the table is another one for every unit)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(e.x), "=f"(e.y), "=f"(e.z), "=f"(e.w) : "r"(tab + 8u * i) : "memory");
                    v[i] = __fmaf_rn(__uint_as_float(acc[i >> 5][i & 31]), e.x, e.y);
                    v[i + 1] = __fmaf_rn(__uint_as_float(acc[i >> 5][(i & 31) + 1]), e.z, e.w);
                }
                act_all<CH>(p.act, p.exact != 0, v);
                if (f0 + CH > p.F) {
#pragma unroll
                    for (int i = 0; i < CH; ++i)
                        if (f0 + i >= p.F) v[i] = 0.0f;
                }
                if (!valid) continue;
                if (OUT == LN_OUT_F32) {
                    const long long img = pix / p.hw;
                    float* dst = (float*)p.y + (img * p.F + f0) * p.hw + (pix - img * p.hw);
#pragma unroll
                    for (int i = 0; i < CH; ++i)
                        if (f0 + i < p.F) dst[(long long)i * p.hw] = v[i];
                } else if (OUT == LN_OUT_F16) {
                    uint4* dst = (uint4*)((uint8_t*)p.y + pix * p.ys + 2 * f0);
#pragma unroll
                    for (int c = 0; c < CH; c += 8) {
                        if ((c & 31) == 0 && f0 + c >= p.F) break;  // (channels are padded to 32)
                        uint32_t h[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __half2 q = __floats2half2_rn(v[c + 2 * i], v[c + 2 * i + 1]);
                            h[i] = *reinterpret_cast<const uint32_t*>(&q);
                        }
                        dst[c >> 3] = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                } else {
                    constexpr int B = FMT == LN_F4 ? 16 : 32;
                    uint8_t* dst = (uint8_t*)p.y + pix * p.ys + f0 / 2;
                    uint8_t* sf = p.ysf + pix * p.ysf_stride + f0 / B;
#pragma unroll
                    for (int c = 0; c < CH; c += 32) {
                        uint32_t q[4];
#pragma unroll
                        for (int b = 0; b < 32 / B; ++b) sf[c / B + b] = (uint8_t)ln_f4_quantise<FMT>(v + c + b * B, p.g, p.six_g, q + b * B / 8);
                        *(uint4*)(dst + c / 2) = make_uint4(q[0], q[1], q[2], q[3]);
                    }
                }
            }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag && warp == 0 && lane == 0) {
        // a wait was abandoned: give copies that may still be in flight time to land before the shared memory is handed on
        for (int i = 0; i < 64; ++i) __nanosleep(20000);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

int log2_of(int v) {
    int l = 0;
    while ((1 << l) < v) ++l;
    return l;
}

template <int FMT, int OUT>
cudaError_t launch(ln_ctx* ctx, const f4_params& p, int grid, size_t smem) {
    auto go = [&](void (*k)(const f4_params)) -> cudaError_t {
        if (!ctx->configured_kernels.count((const void*)k)) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemF4);
            if (e != cudaSuccess) return e;
            ctx->configured_kernels.insert((const void*)k);
        }
        k<<<grid, kThreadsF4, smem, ctx->stream>>>(p);
        return cudaGetLastError();
    };
    return p.bn >= 192 ? go(f4_umma_kernel<FMT, OUT, 64>) : go(f4_umma_kernel<FMT, OUT, 32>);
}

}  // namespace

// Equal strides of 1 or 2; extents that the tensor maps and the 32-bit tile arithmetic hold.
bool ln_f4_umma_takes(const ln_f4_conv& c, int64_t stride_x, int64_t stride_y) {
    if (stride_x != stride_y || stride_x > 2) return false;
    // (a stride-2 convolution whose taps reach the odd rows and columns has to have some: their tensor maps are of those pixels)
    if (stride_x == 2 && (c.x->h == 1 || c.x->w == 1) && (c.k > 1 || c.pad > 0)) return false;
    const int64_t pixels = c.y->n * c.y->h * c.y->w, in = c.x->n * c.x->h * c.x->w;
    return pixels < (1ll << 30) && in < (1ll << 30) && c.w->filters < (1 << 20) && c.x->cstride * c.k * c.k < (1ll << 31) && c.x->h < (1 << 20) && c.x->w < (1 << 30);
}

int ln_f4_umma_launch(ln_ctx* ctx, const ln_f4_conv& c) {
    const char* who = "ln_conv2d_bias_act_f4";
    f4_params p;
    memset(&p, 0, sizeof p);
    const ln_tensor &x = *c.x, &y = *c.y;
    const ln_f4_kblocks kb = ln_f4_kblocks_of(c.dtype, x.c);
    const bool flat = c.k == 1 && c.stride == 1 && c.pad == 0;
    const int64_t pixels = y.n * y.h * y.w;
    p.H = flat ? 1 : (int)x.h; p.W = flat ? (int)pixels : (int)x.w; p.N = flat ? 1 : (int)x.n;
    p.OH = flat ? 1 : (int)y.h; p.OW = flat ? (int)pixels : (int)y.w;
    p.F = (int)y.c; p.hw = (int)(y.h * y.w);
    p.R = p.S = c.k; p.stride = c.stride; p.pad = c.pad;
    p.bk = kb.bk; p.cblocks = kb.cblocks; p.words = kb.words;
    p.cstride = (int)x.cstride; p.sf_stride = (int)x.sf_stride;
    // box of 128 output pixels: the fewest tiles, ties to the widest
    int64_t best = -1;
    for (int lw = 0; lw <= 7; ++lw)
        for (int lh = 0; lw + lh <= 7; ++lh) {
            const int tw = 1 << lw, th = 1 << lh, tn = 128 >> (lw + lh);
            const int64_t tiles = (int64_t)((p.OW + tw - 1) / tw) * ((p.OH + th - 1) / th) * ((p.N + tn - 1) / tn);
            if (best < 0 || tiles < best || (tiles == best && tw > p.TW)) { best = tiles; p.TW = tw; p.TH = th; p.TN = tn; }
        }
    p.log_tw = log2_of(p.TW); p.log_th = log2_of(p.TH);
    // filter tile
    const int64_t instructions = (int64_t)c.k * c.k * x.cstride / 32;
    int64_t least = -1;
    const int cand[4] = {256, 192, 128, 64};
    for (int bn : cand) {
        const int64_t rounds = (best * ((p.F + bn - 1) / bn) + ctx->sm_count - 1) / ctx->sm_count;
        const int64_t chain = instructions * (bn >= 128 ? bn / 2 + 8 : 100), out = (int64_t)bn * 12;
        const int64_t cost = rounds * (bn == 256 ? chain + 500 + (out > chain ? out - chain : 0) : (chain > out ? chain : out)) + out;
        if (least < 0 || cost < least) { least = cost; p.bn = bn; }
    }
    if (const char* e = getenv("LN_F4_BN")) {  // (A/B measurements: another filter tile)
        for (int bn : cand)
            if (atoi(e) == bn) p.bn = bn;
    }
    p.wblocks = p.bn > 128 ? 2 : 1;
    p.nbuf = (int)kScaleCols / p.bn;
    p.subs = p.bn >= 192 ? p.bn / 64 : p.bn / 32;
    p.tiles_f = (p.F + p.bn - 1) / p.bn; p.tiles_w = (p.OW + p.TW - 1) / p.TW; p.tiles_h = (p.OH + p.TH - 1) / p.TH;
    const int64_t num_tiles = best * p.tiles_f;
    if (num_tiles >= (1 << 20)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: %lld tiles", who, (long long)num_tiles);
    p.num_tiles = (int)num_tiles;
    auto magic = [](int d) { return ((1ull << 40) + (unsigned long long)d - 1) / (unsigned long long)d; };
    p.magic_f = magic(p.tiles_f); p.magic_w = magic(p.tiles_w); p.magic_h = magic(p.tiles_h);
    p.off_b = 128u * p.bk;
    p.off_sfa = p.off_b + (uint32_t)p.bn * p.bk;
    p.off_sfb = p.off_sfa + (uint32_t)p.words * 512u;
    p.stage_bytes = (uint32_t)ln_round_up(p.off_sfb + (uint32_t)(p.words * p.wblocks) * 512u, 1024);
    p.stages = (int)((kMaxSmemF4 - 1024 - kBarBytesF4 - kTabBytesF4) / p.stage_bytes);
    if (p.stages > kMaxStagesF4) p.stages = kMaxStagesF4;
    const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + kBarBytesF4 + kTabBytesF4;
    p.xsf = (const uint8_t*)x.sf; p.wsf = (const uint8_t*)c.w->sf; p.wscale = c.w->wscale; p.bias = c.bias;
    p.y = y.ptr; p.ys = y.cstride; p.ysf = (uint8_t*)y.sf; p.ysf_stride = y.sf_stride;
    p.xscale = x.scale; p.g = y.scale; p.six_g = 6.0f * y.scale;
    p.act = c.act; p.exact = ctx->exact_epilogue ? 1 : 0;
    p.status = ctx->h_status;

    const CUtensorMapSwizzle swz = p.bk == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (p.bk == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    for (int m = 0; m < (c.stride == 2 ? 4 : 1); ++m) {
        const int py = m >> 1, px = m & 1;  // input pixels (y, x) with y % stride == py, x % stride == px
        int64_t wm = (p.W - px + c.stride - 1) / c.stride, hm = (p.H - py + c.stride - 1) / c.stride;
        if (wm < 1) wm = 1;  // (a map that no tap uses)
        if (hm < 1) hm = 1;
        const cuuint64_t dims[4] = {(cuuint64_t)x.cstride, (cuuint64_t)wm, (cuuint64_t)hm, (cuuint64_t)p.N};
        const cuuint64_t strides[3] = {(cuuint64_t)(c.stride * x.cstride), (cuuint64_t)((int64_t)c.stride * p.W * x.cstride), (cuuint64_t)((int64_t)p.H * p.W * x.cstride)};
        const cuuint32_t box[4] = {(cuuint32_t)p.bk, (cuuint32_t)p.TW, (cuuint32_t)p.TH, (cuuint32_t)p.TN};
        void* base = (uint8_t*)x.ptr + ((int64_t)py * p.W + px) * x.cstride;
        const CUresult r = ctx->encode_tiled(&p.tmA[m], CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return ln_fail(ctx, LN_ERR_CUDA, "%s: cuTensorMapEncodeTiled(activations, map %d) failed with %d", who, m, (int)r);
    }
    {
        const cuuint64_t dims[2] = {(cuuint64_t)((int64_t)c.k * c.k * x.cstride), (cuuint64_t)p.F};
        const cuuint64_t strides[1] = {(cuuint64_t)((int64_t)c.k * c.k * x.cstride)};
        const cuuint32_t box[2] = {(cuuint32_t)p.bk, (cuuint32_t)p.bn};
        const CUresult r = ctx->encode_tiled(&p.tmB, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.w->w, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return ln_fail(ctx, LN_ERR_CUDA, "%s: cuTensorMapEncodeTiled(weights) failed with %d", who, (int)r);
    }
    const int grid = p.num_tiles < ctx->sm_count ? p.num_tiles : ctx->sm_count;
    cudaError_t e;
#define LN_F4_LAUNCH(FMT) \
    (c.out_kind == LN_OUT_F32 ? launch<FMT, LN_OUT_F32>(ctx, p, grid, smem) : c.out_kind == LN_OUT_F16 ? launch<FMT, LN_OUT_F16>(ctx, p, grid, smem) : launch<FMT, LN_OUT_Q>(ctx, p, grid, smem))
    e = c.dtype == LN_F4 ? LN_F4_LAUNCH(LN_F4) : LN_F4_LAUNCH(LN_MX4);
#undef LN_F4_LAUNCH
    ctx->launches++;
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return ln_fail(ctx, LN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    }
    return LN_OK;
}
