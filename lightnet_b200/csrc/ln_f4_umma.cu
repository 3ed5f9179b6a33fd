// The 4-bit product on the tensor cores: tcgen05.mma with block scales (kind::mxf4nvf4, scale_vec::4X for LN_F4; kind::mxf4,
// scale_vec::2X for LN_MX4), operands and scales in shared memory and TMEM, bias + activation + output conversion in the epilogue.
//
// GEMM view as for the 8-bit types: D[pixel, filter] = sum over (tap, channel block) of X[pixel shifted by the tap, c] * W[filter, tap, c];
// a tile is 128 output pixels (a TW x TH x TN box; a 1x1 stride-1 convolution is flattened to one row of pixels) by bn filters, a
// k-block 128 bytes = 256 channels of one tap (fewer where the tensor has fewer): four instructions of 64 channels.
// Codes come by TMA (taps outside the image are zero filled; stride 2 has one tensor map per parity class of the input).  Block scales
// lie in memory as the tensor core takes them: those of the weights, and of pixels in their own order, come by bulk copies.  Taps shift
// the pixels, so there four warps gather words, a lane for the rows l, l + 32, l + 64, l + 96, one 16-byte piece per instruction.  The
// issuing thread copies both from shared memory to TMEM (tcgen05.cp, executed in order with the instructions that read them) right
// before the k-block that they belong to.
//
// Roles: warps 0 and 6 load (pixels; weights), warp 1 issues, warps 2 to 5 gather scales (every fourth k-block each; the ring has at
// least four stages, so none comes back to a stage whose use before is still to be filled), warps 8 to 23 are the epilogue: four groups
// of four that take the units of 32 columns of the tiles in turn.  TMEM: 416 columns of accumulators, 2 x 48 of scales.  Two tiles of
// 192 filters, three of 128 or six of 64 fit; two of 256 overlap by 96 columns (0..255 and 160..415), so their epilogue reads the four
// units that hold the overlap first and the next tile starts as soon as those are in registers.
// Every wait is bounded (see ln_umma.h).
#include <cstdlib>

#include "ln_f4.h"
#include "ln_umma.h"

namespace {

constexpr int kThreadsF4 = 32 * 24, kFirstEpilogueWarp = 8, kGatherWarps = 4;
constexpr int kMaxStagesF4 = 8, kMaxBufsF4 = 6;
constexpr int CH = 32;  // columns of an epilogue unit
constexpr int kOverlapBase = 160;  // first column of the second accumulator of 256
constexpr uint32_t kScaleCols = 416, kScaleSet = 48, kScaleB = 16;  // TMEM columns: two sets of [16 pixels' | 32 filters'] scale words
constexpr uint32_t kBarBytesF4 = 512;
constexpr uint32_t kTabBytesF4 = 16 * 256;  // {multiplier, bias} of the columns that a warp is at
constexpr int kMaxSmemF4 = 227 * 1024;

struct f4_params {
    CUtensorMap tmA[4], tmB;
    const uint8_t *xsf, *wsf;
    const float *wscale, *bias;
    void* y;
    uint8_t* ysf;
    int* status;
    long long ys, ysf_words;  // bytes per pixel of an NHWC output, words of scales
    float xscale, g, six_g;    // tensor scale of the input; of a 4-bit output
    int sf_words, cstride;
    int bk, bn, cblocks, words;
    int R, S, stride, pad, H, W, N, OH, OW, F, hw;
    int TW, TH, TN, log_tw, log_th, tiles_f, tiles_w, tiles_h, num_tiles;
    unsigned long long magic_f, magic_w, magic_h;
    int stages, nbuf, acc_step, subs, act, exact, flat;
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

__device__ __forceinline__ void act_all(int act, bool exact, float (&v)[32]) {
#define LN_ALL(E, A)                                                       \
    _Pragma("unroll") for (int i = 0; i < 32; ++i) v[i] = ln_epilogue_act<E>(A, v[i]); \
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

__device__ __forceinline__ void store_32(uint8_t* dst, const uint32_t (&v)[8]) {  // a whole sector
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
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

template <int FMT, int OUT, int WBLOCKS>
__global__ void __launch_bounds__(kThreadsF4, 1) f4_umma_kernel(const __grid_constant__ f4_params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + (uint32_t)p.stages * p.stage_bytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStagesF4 + s); };
    auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStagesF4 + b); };
    auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStagesF4 + kMaxBufsF4 + b); };
    auto early_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStagesF4 + 2 * kMaxBufsF4 + b); };  // (overlapping accumulators)
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(smem_raw + (bar_base - smem_u32(smem_raw)) + 8u * (2 * kMaxStagesF4 + 2 * kMaxBufsF4 + 2));
    volatile int* abort_flag = (volatile int*)(tmem_slot + 2);
    const uint32_t tab_base = bar_base + kBarBytesF4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full_bar(s), p.flat ? 2 : 3);  // the two loaders (with their copies' bytes) and a warp that gathers scales
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < p.nbuf; ++b) {
            mbar_init(tfull_bar(b), 1);
            mbar_init(tempty_bar(b), 4 * p.subs);
        }
        mbar_init(early_bar(0), 16);
        mbar_init(early_bar(1), 16);
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
    const bool overlap = p.bn == 256;

    if (warp == 0) {
        // ------------------------------------------------------------------ loads of the pixels (whole warps walk these loops; one lane issues)
        const bool leader = elect_one();
        const uint32_t sf_bytes = (uint32_t)p.words * 512u, bytes = 128u * p.bk + (p.flat ? sf_bytes : 0u);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int unit = (int)blockIdx.x; ok && unit < p.num_tiles; unit += step) {
            const f4_tile t = tile_at(p, unit);
            const uint8_t* xsf = p.xsf + (size_t)(t.ow0 >> 7) * kblocks * sf_bytes;  // (flat)
            for (int r = 0; ok && r < p.R; ++r)
                for (int s = 0; ok && s < p.S; ++s) {
                    int ty = r - p.pad, tx = s - p.pad, map = 0;
                    if (p.stride == 2) {
                        const int py = ty & 1, px = tx & 1;  // parity class of the tap
                        ty = (ty - py) >> 1;
                        tx = (tx - px) >> 1;
                        map = py * 2 + px;
                    }
                    for (int c0 = 0; c0 < p.cstride; c0 += p.bk, xsf += sf_bytes) {
                        if (!(ok = warp_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                        if (leader) {
                            const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes, bar = full_bar(stage);
                            mbar_arrive_expect_tx(bar, bytes);
                            tma_load_4d(at, &p.tmA[map], c0, t.ow0 + tx, t.oh0 + ty, t.n0, bar);
                            if (p.flat) bulk_load(at + p.off_sfa, xsf, sf_bytes, bar);
                        }
                        __syncwarp();
                        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                    }
                }
        }
    } else if (warp == 6) {
        // ------------------------------------------------------------------ loads of the weights
        const bool leader = elect_one();
        const uint32_t sf_bytes = (uint32_t)p.words * 512u, bytes = (uint32_t)p.bn * p.bk + WBLOCKS * sf_bytes;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int unit = (int)blockIdx.x; ok && unit < p.num_tiles; unit += step) {
            const int f0 = (unit - fast_div(unit, p.magic_f) * p.tiles_f) * p.bn;
            const uint8_t* wsf = p.wsf + (size_t)(f0 >> 7) * kblocks * sf_bytes;
            int col = 0, c0 = 0;  // first byte of the tap, of the k-block inside it
            for (int kb = 0; kb < kblocks; ++kb, wsf += sf_bytes) {
                if (!(ok = warp_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                if (leader) {
                    const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes, bar = full_bar(stage);
                    mbar_arrive_expect_tx(bar, bytes);
                    tma_load_2d(at + p.off_b, &p.tmB, col + c0, f0, bar);
#pragma unroll
                    for (int b = 0; b < WBLOCKS; ++b) bulk_load(at + p.off_sfb + b * sf_bytes, wsf + (size_t)b * kblocks * sf_bytes, sf_bytes, bar);
                }
                __syncwarp();
                c0 += p.bk;
                if (c0 >= p.cstride) { c0 = 0; col += p.cstride; }
                if (++stage == p.stages) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ instructions (the whole warp walks the loop; one lane issues)
        const bool leader = elect_one();
        // E2M1 operands (bits 7, 10: type 1), N / 8, scale type (bit 23: 1 = E8M0), M / 128, K-major; the scale ids go to bits 4 and 29
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | ((FMT == LN_MX4 ? 1u : 0u) << 23) | (1u << 27);
        const uint64_t desc_base = make_smem_desc(0u, p.bk);
        constexpr int kWords = FMT == LN_MX4 ? 2 : 4, kBlocks = WBLOCKS;  // of a whole k-block
        const uint64_t sfa_desc = scale_desc(p.off_sfa), sfb_desc = scale_desc(p.off_sfb);
        int stage = 0, t = 0;
        uint32_t phase = 0, set = 0;
        bool ok = true;
        for (int unit = (int)blockIdx.x; ok && unit < p.num_tiles; unit += step, ++t) {
            const int buf = t % p.nbuf;
            if (!(ok = warp_wait(tempty_bar(buf), (uint32_t)((t / p.nbuf) & 1) ^ 1u, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
            if (overlap && t > 0 && !(ok = warp_wait(early_bar(buf ^ 1), (uint32_t)(((t - 1) >> 1) & 1), abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
            tc_fence_after();
            const uint32_t d = tmem_base + (uint32_t)(buf * p.acc_step);
            const int tf = unit - fast_div(unit, p.magic_f) * p.tiles_f;
            const uint32_t shift = (uint32_t)((tf * p.bn & 127) >> 5);  // first column of the tile's filters inside their group of 128
            int c0 = 0;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!(ok = warp_wait(full_bar(stage), phase, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
                tc_fence_after();
                const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes;
                const uint32_t sfa = tmem_base + kScaleCols + set * kScaleSet, sfb = sfa + kScaleB;
                const int left = p.cstride - c0, n = (left < p.bk ? left : p.bk) >> 5;  // instructions of this k-block
                const uint64_t a_desc = desc_base + (at >> 4), b_desc = desc_base + ((at + p.off_b) >> 4);
                if (n == 4) {
                    // a whole k-block of 128 bytes, unrolled with constant offsets: as loops with run-time bounds the copies and
                    // instructions of a k-block took their thread 1100 cycles, this way 420, less than the 530 that they run for
                    if (leader) {
#pragma unroll
                        for (int j = 0; j < kWords; ++j) {
                            tc_copy_scales(sfa + 4u * j, sfa_desc + ((at + 512u * j) >> 4));
#pragma unroll
                            for (int b = 0; b < kBlocks; ++b) tc_copy_scales(sfb + 4u * (j * kBlocks + b), sfb_desc + ((at + 512u * (b * kWords + j)) >> 4));
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t word = FMT == LN_MX4 ? i >> 1 : i, id = FMT == LN_MX4 ? (uint32_t)(i & 1) * 2u : 0u;
                            tc_mma_scaled<FMT>(d, a_desc + 2u * i, b_desc + 2u * i, idesc | (id << 4) | (id << 29), sfa + 4u * word, sfb + 4u * word * kBlocks + shift, i ? 1u : (uint32_t)(kb != 0));
                        }
                        tc_commit(empty_bar(stage));
                    }
                } else if (leader) {
                    for (int j = 0; j < p.words; ++j) {
                        tc_copy_scales(sfa + 4u * j, scale_desc(at + p.off_sfa + 512u * j));
                        for (int b = 0; b < WBLOCKS; ++b) tc_copy_scales(sfb + 4u * (j * WBLOCKS + b), scale_desc(at + p.off_sfb + 512u * (b * p.words + j)));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < n) {
                            const uint32_t word = FMT == LN_MX4 ? i >> 1 : i, id = FMT == LN_MX4 ? (uint32_t)(i & 1) * 2u : 0u;
                            tc_mma_scaled<FMT>(d, a_desc + 2u * i, b_desc + 2u * i, idesc | (id << 4) | (id << 29), sfa + 4u * word, sfb + 4u * word * WBLOCKS + shift, (uint32_t)((kb | i) != 0));
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
    } else if (warp < 2 + kGatherWarps) {
        // ------------------------------------------------------------------ scales of the pixels under shifted taps
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
                const bool inside = y >= 0 && y < p.H && x >= 0 && x < p.W && img[g] < p.N;
                const uint8_t* src = p.xsf + (inside ? ln_f4_sf_at((img[g] * p.H + y) * p.W + x, cb * p.words, p.sf_words) : 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[g][j] = inside && j < p.words ? __ldg((const uint32_t*)(src + 512 * j)) : 0u;
            }
        };
        if (!p.flat) {
            enter_tile();
            for (int i = 2; i < warp; ++i) advance();
            int stage = warp - 2;  // (fewer than stages)
            uint32_t phase = 0;
            uint32_t now[4][4], next[4][4];
            bool more = unit < p.num_tiles, ok = true;
            if (more) fetch(now);
            while (more && ok) {
                for (int i = 0; i < kGatherWarps; ++i) advance();
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
                stage += kGatherWarps;
                if (stage >= p.stages) { stage -= p.stages; phase ^= 1u; }
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int j = 0; j < 4; ++j) now[g][j] = next[g][j];
            }
        }
    } else if (warp >= kFirstEpilogueWarp) {
        // ------------------------------------------------------------------ epilogue
        // Group g takes the units with number % 4 == g.  (nbuf * subs >= 4: a group that waits for a tile's accumulator has finished a unit
        // of the tile nbuf before it or a later one, so the parity is unambiguous.)
        const int quad = warp & 3, group = (warp - kFirstEpilogueWarp) >> 2;
        const int row = quad * 32 + lane, pw = row & (p.TW - 1), ph = (row >> p.log_tw) & (p.TH - 1), pn = row >> (p.log_tw + p.log_th);
        const uint32_t tab = tab_base + (uint32_t)(warp - kFirstEpilogueWarp) * 256u;
        // {multiplier, bias} of the unit's column that this lane looks after: read one unit ahead
        auto table_of = [&](int f, float& m, float& b) {
            m = f < p.F ? __ldg(p.wscale + f) : 0.0f;
            b = f < p.F ? __ldg(p.bias + f) : 0.0f;
        };
        int t = 0, unit = (int)blockIdx.x, order = group;
        while (order >= p.subs) { order -= p.subs; unit += step; ++t; }
        auto filter_of = [&]() {
            const int sub = overlap && t % p.nbuf == 0 ? order ^ 4 : order;  // (what overlaps the other accumulator first)
            return (unit - fast_div(unit, p.magic_f) * p.tiles_f) * p.bn + sub * CH;
        };
        float mult = 0.0f, bias = 0.0f;
        if (unit < p.num_tiles) table_of(filter_of() + lane, mult, bias);
        bool ok = true;
        while (unit < p.num_tiles) {
            const f4_tile at = tile_at(p, unit);
            const int buf = t % p.nbuf, f0 = filter_of(), sub = (f0 - at.f0) / CH, this_t = t;
            const bool first = order < 4;
            const int ow = at.ow0 + pw, oh = at.oh0 + ph, n = at.n0 + pn;
            const bool valid = ow < p.OW && oh < p.OH && n < p.N;
            const long long pix = ((long long)n * p.OH + oh) * p.OW + ow;
            __syncwarp();  // (the table of the unit before has been read)
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(tab + 8u * lane), "f"(__fmul_rn(p.xscale, mult)), "f"(bias) : "memory");
            __syncwarp();
            order += 4;
            while (order >= p.subs) { order -= p.subs; unit += step; ++t; }
            if (unit < p.num_tiles) table_of(filter_of() + lane, mult, bias);
            if (!(ok = warp_wait(tfull_bar(buf), (uint32_t)((this_t / p.nbuf) & 1), abort_flag, p.status, LN_STATUS_EPILOGUE_TIMEOUT))) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * p.acc_step + sub * CH);
            uint32_t acc[32];
            tmem_ld_32x32(taddr, acc);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(tempty_bar(buf));
                if (overlap && first) mbar_arrive(early_bar(buf));
            }
            // (binary16 channels are padded to 32, 4-bit ones to 64: what is behind them is not stored)
            if (f0 >= (OUT == LN_OUT_Q ? (p.F + 63) & ~63 : p.F)) continue;
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float4 e;  // (volatile: the table is another one for every unit)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(e.x), "=f"(e.y), "=f"(e.z), "=f"(e.w) : "r"(tab + 8u * i) : "memory");
                v[i] = __fmaf_rn(__uint_as_float(acc[i]), e.x, e.y);
                v[i + 1] = __fmaf_rn(__uint_as_float(acc[i + 1]), e.z, e.w);
            }
            act_all(p.act, p.exact != 0, v);
            if (f0 + 32 > p.F) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (f0 + i >= p.F) v[i] = 0.0f;
            }
            if (OUT == LN_OUT_F32) {
                if (valid) {
                    const long long img = pix / p.hw;
                    float* dst = (float*)p.y + (img * p.F + f0) * p.hw + (pix - img * p.hw);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (f0 + i < p.F) dst[(long long)i * p.hw] = v[i];
                }
            } else if (OUT == LN_OUT_F16) {
                uint32_t h[2][8];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const __half2 q = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                    h[i >> 3][i & 7] = *reinterpret_cast<const uint32_t*>(&q);
                }
                if (valid) {
                    uint8_t* dst = (uint8_t*)p.y + pix * p.ys + 2 * f0;
                    store_32(dst, h[0]);
                    store_32(dst + 32, h[1]);
                }
            } else {
                constexpr int B = FMT == LN_F4 ? 16 : 32;
                uint32_t q[4], sf = 0;
#pragma unroll
                for (int b = 0; b < 32 / B; ++b) sf |= ln_f4_quantise<FMT>(v + b * B, p.g, p.six_g, q + b * B / 8) << (8 * b);
                if (valid) {
                    *(uint4*)((uint8_t*)p.y + pix * p.ys + f0 / 2) = make_uint4(q[0], q[1], q[2], q[3]);
                    uint8_t* at_sf = p.ysf + ln_f4_sf_at(pix, f0 / (4 * B), p.ysf_words) + f0 / B % 4;
                    if (FMT == LN_F4) *(uint16_t*)at_sf = (uint16_t)sf;
                    else *at_sf = (uint8_t)sf;
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
    return p.bn > 128 ? go(f4_umma_kernel<FMT, OUT, 2>) : go(f4_umma_kernel<FMT, OUT, 1>);
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
    p.cstride = (int)x.cstride; p.sf_words = (int)x.sf_words;
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
    const int wblocks = p.bn > 128 ? 2 : 1;
    p.nbuf = p.bn == 256 ? 2 : (int)kScaleCols / p.bn;
    p.acc_step = p.bn == 256 ? kOverlapBase : p.bn;
    p.subs = p.bn / CH;
    p.flat = flat ? 1 : 0;
    p.tiles_f = (p.F + p.bn - 1) / p.bn; p.tiles_w = (p.OW + p.TW - 1) / p.TW; p.tiles_h = (p.OH + p.TH - 1) / p.TH;
    const int64_t num_tiles = best * p.tiles_f;
    if (num_tiles >= (1 << 20)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: %lld tiles", who, (long long)num_tiles);
    p.num_tiles = (int)num_tiles;
    auto magic = [](int d) { return ((1ull << 40) + (unsigned long long)d - 1) / (unsigned long long)d; };
    p.magic_f = magic(p.tiles_f); p.magic_w = magic(p.tiles_w); p.magic_h = magic(p.tiles_h);
    p.off_b = 128u * p.bk;
    p.off_sfa = p.off_b + (uint32_t)p.bn * p.bk;
    p.off_sfb = p.off_sfa + (uint32_t)p.words * 512u;
    p.stage_bytes = (uint32_t)ln_round_up(p.off_sfb + (uint32_t)(p.words * wblocks) * 512u, 1024);
    p.stages = (int)((kMaxSmemF4 - 1024 - kBarBytesF4 - kTabBytesF4) / p.stage_bytes);
    if (p.stages > kMaxStagesF4) p.stages = kMaxStagesF4;
    const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + kBarBytesF4 + kTabBytesF4;
    p.xsf = (const uint8_t*)x.sf; p.wsf = (const uint8_t*)c.w->sf; p.wscale = c.w->wscale; p.bias = c.bias;
    p.y = y.ptr; p.ys = y.cstride; p.ysf = (uint8_t*)y.sf; p.ysf_words = y.sf_words;
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
