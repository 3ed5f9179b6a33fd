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
// of four that take the units of 32 columns of the tiles in turn.  TMEM: 416 columns of accumulators, 2 x 48 of scales.  Three tiles of
// 128 filters or six of 64 fit; two of 256 overlap by 96 columns (0..255 and 160..415), so their epilogue reads the four units that hold
// the overlap first, and the next tile starts when those have been read.
// Where all tiles leave SMs idle, long k ranges are split over clusters: each CTA takes a part, then one unit of the tile's sums, which
// the others write into its shared memory.  The last round of tiles, where it would leave SMs idle, is cut into units of fewer filters; each is the last one of its CTA, so nothing
// waits for its accumulator to be free.
// What bounds it: large k ranges the way from L2 to shared memory (54 KB per k-block of 256 filters at 64 bytes a cycle are 844 cycles, the
// instructions take 528, measured 830 to 900; 28 KB of 64 filters 437, measured 550) and, in runs of seconds, power (1500 MHz); short ones the
// epilogue.  K-blocks of half the size (8192 x 4096 x 4096 in 80 us instead of 63) pay the fixed cost of a k-block twice.  CTA pairs (cta_group::2, half of the filters' codes per CTA) were built and
// gave the same 64 us on 8192 x 4096 x 4096: a tcgen05.cp of a pair takes its thread 50 cycles and more, and twelve go with four instructions.
// Every wait is bounded (see ln_umma.h).
#include <cstdlib>
#include <cstring>
#include <type_traits>

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
constexpr uint32_t kRowBytesF4 = 32 * 17 * 4;  // of a warp, where f32 rows are stored through shared memory
constexpr int kMaxSmemF4 = 227 * 1024;
constexpr size_t kLeastSmemF4 = 118 * 1024;

struct f4_params {
    CUtensorMap tmA[4], tmB[2], tmXS, tmWS;  // codes of pixels and filters (whole tiles, narrow ones); their scales as rows of 512 bytes
    const uint8_t* xsf;
    const float *wscale, *bias;
    void* y;
    uint8_t* ysf;
    int* status;
    long long ys, ysf_words;  // bytes per pixel of an NHWC output, words of scales
    float xscale, g, six_g;    // tensor scale of the input; of a 4-bit output
    int sf_words, cstride;
    int bk, bn, cblocks, words;
    int R, S, stride, pad, H, W, N, OH, OW, F, hw;
    int TW, TH, TN, log_tw, log_th, tiles_f, tiles_w, tiles_h, num_units;  // units: pixel tiles x filter tiles
    int log_parts;  // CTAs of a cluster that share a tile's k range, as many as the tile has units of 32 columns
    int whole, log_split, narrow;  // the tiles behind the first `whole` are cut into 2^log_split units of `narrow` filters
    unsigned long long magic_f, magic_w, magic_h;
    int stages, nbuf, acc_step, subs, act, exact, flat;
    uint32_t off_b, off_sfa, off_sfb, stage_bytes;
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void cluster_sync() {  // (of whole warps)
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// whether a phase is complete, now
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// a wait of the whole warp: one answer for all lanes
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// 32 rows of 16 bytes -> the four 32-lane quarters of TMEM, four columns
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void tc_mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define LN_MMA(KIND)                                                                                                         \
    asm volatile(                                                                                                            \
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                                                    \
        "tcgen05.mma.cta_group::1.kind::" KIND " [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),                            \
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)                                                      \
        : "memory")
    if (FMT == LN_F4) LN_MMA("mxf4nvf4.block_scale.scale_vec::4X");
    else LN_MMA("mxf4.block_scale.scale_vec::2X");
#undef LN_MMA
}
// descriptor of 32 rows of 16 bytes (no swizzle, groups of 8 rows 128 bytes apart)
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) { return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46); }

// Fast activations, two values at a time.  exp is ex2.approx, the reciprocal a seed from the exponent's bits (12 % off) and three Newton
// steps on the FMA pipe (2e-4, then a rounding or two): with rcp.approx as well the special function unit, at a quarter of the lanes'
// rate, bounded the epilogue of the products with short k ranges.
__device__ __forceinline__ void reciprocal2(float& r0, float& r1, float d0, float d1) {
    r0 = __uint_as_float(0x7EF311C7u - __float_as_uint(d0));
    r1 = __uint_as_float(0x7EF311C7u - __float_as_uint(d1));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        float e0, e1;
        ffma2(e0, e1, -d0, -d1, r0, r1, 1.0f, 1.0f);
        ffma2(r0, r1, r0, r1, e0, e1, r0, r1);
    }
}
// FAR: for values below -60 too.  There the function is its value at -60, as far as exp goes, times e^(v + 60), a factor of 1 for all others.
// A warp takes this form for all its columns when one of them is below (3x3 C256->K512 at 38x38, 16 images, mish: 25.6 us, 28.0 where most
// warps do; with the factor inside the usual form 26.4 and 28.7, with a branch per lane 25.6 and 33.1, without the test 24.6).
template <int ACT, bool FAR>
__device__ __forceinline__ void act2(float& v0, float& v1) {
    float c0 = 1.0f, c1 = 1.0f;
    if (FAR) {
        v0 = v0 < -1000.0f ? -1000.0f : v0;  // (-inf times 0 is no number)
        v1 = v1 < -1000.0f ? -1000.0f : v1;
        c0 = ln_ex2_ftz(fminf(v0 + 60.0f, 0.0f) * 1.44269504f);
        c1 = ln_ex2_ftz(fminf(v1 + 60.0f, 0.0f) * 1.44269504f);
    }
    if (ACT == LN_ACT_MISH) {  // v w / (w + 2), w = e^v (e^v + 2), the ratio evaluated at min(v, 20) (it is 1 from there on)
        float e0, e1, w0, w1, d0, d1, r0, r1;
        e0 = fminf(v0, 20.0f);
        e1 = fminf(v1, 20.0f);
        if (FAR) { e0 = fmaxf(e0, -60.0f); e1 = fmaxf(e1, -60.0f); }
        fmul2(e0, e1, e0, e1, 1.44269504f, 1.44269504f);
        e0 = ln_ex2_ftz(e0);
        e1 = ln_ex2_ftz(e1);
        fadd2(w0, w1, e0, e1, 2.0f, 2.0f);
        fmul2(w0, w1, w0, w1, e0, e1);
        fadd2(d0, d1, w0, w1, 2.0f, 2.0f);
        reciprocal2(r0, r1, d0, d1);
        fmul2(w0, w1, w0, w1, r0, r1);
        fmul2(v0, v1, v0, v1, w0, w1);
        if (FAR) fmul2(v0, v1, v0, v1, c0, c1);
    } else {  // swish, logistic: 1 / (1 + e^-v) at max(v, -60)
        float e0, e1, r0, r1;
        fmul2(e0, e1, fmaxf(v0, -60.0f), fmaxf(v1, -60.0f), -1.44269504f, -1.44269504f);
        fadd2(e0, e1, ln_ex2_ftz(e0), ln_ex2_ftz(e1), 1.0f, 1.0f);
        reciprocal2(r0, r1, e0, e1);
        if (ACT == LN_ACT_SWISH) {
            fmul2(v0, v1, v0, v1, r0, r1);
            if (FAR) fmul2(v0, v1, v0, v1, c0, c1);
        } else {
            if (FAR) fmul2(r0, r1, r0, r1, c0, c1);
            v0 = v0 == v0 ? r0 : v0;  // (max drops a NaN)
            v1 = v1 == v1 ? r1 : v1;
        }
    }
}
template <int ACT, bool EXACT, int W>
__device__ __forceinline__ void act_all(float (&v)[W]) {
    constexpr bool fast = !EXACT && (ACT == LN_ACT_MISH || ACT == LN_ACT_SWISH || ACT == LN_ACT_LOGISTIC);
    if (fast) {
        float least = v[0];
#pragma unroll
        for (int i = 1; i < W; ++i) least = fminf(least, v[i]);
        if (__any_sync(0xFFFFFFFFu, least < ln_f4_far<false>(ACT))) {
#pragma unroll
            for (int i = 0; i < W; i += 2) act2<ACT, true>(v[i], v[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < W; i += 2) act2<ACT, false>(v[i], v[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = ln_f4_act<true>(ACT, v[i]);
    }
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x16(taddr, r); tmem_ld_wait(); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32(taddr, r); tmem_ld_wait(); }
// what a unit is: pixels and filters, and the output box's origin
struct f4_unit {
    int pixel_tile, f0;
};
__device__ __forceinline__ f4_unit unit_at(const f4_params& p, int unit) {
    const int v = unit - p.whole, tile = v < 0 ? unit : p.whole + (v >> p.log_split);
    const int pixel_tile = fast_div(tile, p.magic_f), f0 = (tile - pixel_tile * p.tiles_f) * p.bn;
    return {pixel_tile, v < 0 ? f0 : f0 + (v & ((1 << p.log_split) - 1)) * p.narrow};
}
struct f4_box {
    int ow0, oh0, n0;
};
__device__ __forceinline__ f4_box box_at(const f4_params& p, int unit) {
    const int q1 = unit_at(p, unit).pixel_tile;
    const int q2 = fast_div(q1, p.magic_w), tw = q1 - q2 * p.tiles_w;
    const int tn = fast_div(q2, p.magic_h), th = q2 - tn * p.tiles_h;
    return {tw * p.TW, th * p.TH, tn * p.TN};
}

// what the epilogue shares with the other roles: shared addresses of its table and barriers
struct f4_epilogue_at {
    uint32_t tmem, tab, rows, tfull, tempty, early, ring;  // rows: 32 rows of 17 words
    volatile int* abort_flag;
    int unit, step, rank;  // first unit; units from one to the next; place in the cluster
};
constexpr uint32_t kPartBytes = 128 * CH * 4;  // of a unit's partial sums: [quarter of 32 rows][4 columns][row][column]
// A split k range: every CTA of the cluster has partial sums of the whole tile.  It finishes one unit, and writes the others into the shared
// memory of the CTAs that do those; their stages are free then.
__device__ __forceinline__ void f4_exchange(const f4_params& p, const f4_epilogue_at& e) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3;
    const bool ok = warp_wait(e.tfull, 0, e.abort_flag, p.status, LN_STATUS_EPILOGUE_TIMEOUT);
    __syncwarp();
    cluster_sync();  // (all instructions of all CTAs are done)
    tc_fence_after();
    if (ok)
        for (int j = (warp - kFirstEpilogueWarp) >> 2; j < p.subs; j += 4) {
            if (j == e.rank) continue;
            const uint32_t dst = peer_smem(e.ring + (uint32_t)(e.rank < j ? e.rank : e.rank - 1) * kPartBytes + 4096u * quad + 16u * lane, j);
#pragma unroll 1
            for (int c0 = 0; c0 < CH; c0 += 16) {
                uint32_t acc[16];
                tmem_ld(e.tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(j * CH + c0), acc);
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 128u * (c0 + i)), "r"(acc[i]), "r"(acc[i + 1]), "r"(acc[i + 2]), "r"(acc[i + 3]) : "memory");
            }
        }
    __syncwarp();
    cluster_sync();
}
template <int FMT, int OUT, int WBLOCKS, bool PARTS, int ACT, bool EXACT>
__device__ __forceinline__ void f4_epilogue(const f4_params& p, const f4_epilogue_at& e) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = e.step;
    constexpr bool overlap = WBLOCKS == 2;
    // Group g takes the units with number % 4 == g.  (nbuf * subs >= 4: a group that waits for a tile's accumulator has finished a unit
    // of the tile nbuf before it or a later one, so the parity is unambiguous.)
    constexpr int W = OUT == LN_OUT_Q && FMT == LN_MX4 ? 32 : 16;  // columns at a time (a block of a 4-bit output)
    const int quad = warp & 3, group = (warp - kFirstEpilogueWarp) >> 2;
    const int row = quad * 32 + lane, pw = row & (p.TW - 1), ph = (row >> p.log_tw) & (p.TH - 1), pn = row >> (p.log_tw + p.log_th);
    const uint32_t tab = e.tab;
    // {multiplier, bias} of the unit's column that this lane looks after, read one unit ahead (volatile: otherwise the compiler moves the
    // loads down to their use, and every unit waits for them); LN_MX4 has no multiplier.  They go through a table in shared memory, 8
    // bytes per column and warp: 1024 cycles of its port for 128 x 128 outputs, which with 512 of binary16 stores is what bounds the
    // epilogue (measured 2400).
    constexpr bool scaled = FMT == LN_F4;
    float wscale = 0.0f, bias = 0.0f;
    int unit = e.unit, order = PARTS ? (group ? p.subs : e.rank) : group, buf = 0, pixel_tile = 0, col = 0, f0 = 0;  // of the next unit
    uint32_t phase = 0;
    auto settle = [&]() {  // units beyond the tile's: the next tiles
        while (unit < p.num_units && order >= (unit < p.whole ? p.subs : p.narrow / CH)) {
            order -= p.subs;  // (nothing follows a narrow unit)
            unit += step;
            if (++buf == p.nbuf) { buf = 0; phase ^= 1u; }
        }
    };
    auto prefetch = [&]() {
        if (unit >= p.num_units) return;
        const f4_unit u = unit_at(p, unit);
        pixel_tile = u.pixel_tile;
        col = (overlap && buf == 0 && unit < p.whole ? order ^ 4 : order) * CH;  // (what overlaps the other accumulator first)
        f0 = u.f0 + col;
        const int f = f0 + lane;
        wscale = bias = 0.0f;
        if (f >= p.F) return;
        if (scaled) asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(wscale) : "l"(p.wscale + f));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(bias) : "l"(p.bias + f));
    };
    settle();
    prefetch();
    bool ok = true;
    while (unit < p.num_units) {
        const int this_f0 = f0, this_buf = buf;
        const uint32_t this_phase = phase, taddr = e.tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(this_buf * p.acc_step + col);
        const bool first = order < 4;
        int pix = pixel_tile * 128 + row;  // (of a valid row below 2^30)
        bool valid = pix < p.OW;
        if (!p.flat) {
            const int q2 = fast_div(pixel_tile, p.magic_w), q3 = fast_div(q2, p.magic_h);
            const int ow = (pixel_tile - q2 * p.tiles_w) * p.TW + pw, oh = (q2 - q3 * p.tiles_h) * p.TH + ph, n = q3 * p.TN + pn;
            valid = ow < p.OW && oh < p.OH && n < p.N;
            pix = (n * p.OH + oh) * p.OW + ow;
        }
        // the table: {m 2i, m 2i + 1, b 2i, b 2i + 1}, or the biases alone
        __syncwarp();  // (that of the unit before has been read)
        if (scaled) {
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(tab + 16u * (lane >> 1) + 4u * (lane & 1)), "f"(__fmul_rn(p.xscale, wscale)) : "memory");
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(tab + 16u * (lane >> 1) + 8u + 4u * (lane & 1)), "f"(bias) : "memory");
        } else
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(tab + 4u * lane), "f"(bias) : "memory");
        __syncwarp();
        order += PARTS ? p.subs : 4;
        settle();
        prefetch();
        if (!(ok = warp_wait(e.tfull + 8u * this_buf, this_phase, e.abort_flag, p.status, LN_STATUS_EPILOGUE_TIMEOUT))) break;
        tc_fence_after();
        // A loop, not unrolled: 32 columns in one piece are more code than the instruction caches of four warps at different places of
        // it keep, and the epilogue then waited for instructions most of the time.
#pragma unroll 1
        for (int c0 = 0; c0 < CH; c0 += W) {
            uint32_t acc[W];
            __syncwarp();  // (rows behind the last pixel store nothing)
            tmem_ld(taddr + c0, acc);
            for (int part = 1; PARTS && part < 1 << p.log_parts; ++part) {  // (this CTA's own sum first, the others in their order)
#pragma unroll
                for (int i = 0; i < W; i += 4) {
                    float4 t;
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(t.x), "=f"(t.y), "=f"(t.z), "=f"(t.w) : "r"(e.ring + (uint32_t)(part - 1) * kPartBytes + 4096u * quad + 16u * lane + 128u * (c0 + i)));
                    acc[i] = __float_as_uint(__fadd_rn(__uint_as_float(acc[i]), t.x));
                    acc[i + 1] = __float_as_uint(__fadd_rn(__uint_as_float(acc[i + 1]), t.y));
                    acc[i + 2] = __float_as_uint(__fadd_rn(__uint_as_float(acc[i + 2]), t.z));
                    acc[i + 3] = __float_as_uint(__fadd_rn(__uint_as_float(acc[i + 3]), t.w));
                }
            }
            if (c0 + W == CH) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(e.tempty + 8u * this_buf);
                    if (overlap && first) mbar_arrive(e.early + 8u * this_buf);
                }
                __syncwarp();
            }
            const int f = this_f0 + c0;
            // (binary16 channels are padded to 32, 4-bit ones to 64: what is behind them is not stored)
            if (this_f0 >= (OUT == LN_OUT_Q ? (p.F + 63) & ~63 : p.F)) continue;
            float v[W];
#pragma unroll
            for (int i = 0; i < W; i += scaled ? 2 : 4) {
                float4 t;  // (volatile: the table is another one for every unit)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(t.x), "=f"(t.y), "=f"(t.z), "=f"(t.w) : "r"(tab + (scaled ? 8u : 4u) * (c0 + i)));
                if (scaled) ffma2(v[i], v[i + 1], __uint_as_float(acc[i]), __uint_as_float(acc[i + 1]), t.x, t.y, t.z, t.w);
                else {
                    fadd2(v[i], v[i + 1], __uint_as_float(acc[i]), __uint_as_float(acc[i + 1]), t.x, t.y);
                    fadd2(v[(i + 2) % W], v[(i + 3) % W], __uint_as_float(acc[(i + 2) % W]), __uint_as_float(acc[(i + 3) % W]), t.z, t.w);
                }
            }
            act_all<ACT, EXACT>(v);
            if (f + W > p.F) {
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (f + i >= p.F) v[i] = 0.0f;
            }
            if (OUT == LN_OUT_F32) {
                if (p.flat && p.hw == 1) {  // rows of F values
                    if (p.F % 8 == 0) {  // a lane's are consecutive and fill sectors
                        float* dst = (float*)p.y + (long long)pix * p.F + f;
#pragma unroll
                        for (int i = 0; i < W; i += 8) {
                            const uint32_t (&h)[8] = *reinterpret_cast<const uint32_t(*)[8]>(v + i);
                            if (valid && f + i < p.F) ln_store_32(dst + i, h);
                        }
                        continue;
                    }
                    // Rows begin anywhere: two rows at a time through shared memory (17 words apart: no bank twice), so that the 16 values of
                    // one go out together.  (65536 x 128 -> 255: 94 us with a lane writing its own row.)
                    const uint32_t rows = e.rows + 68u * lane;
#pragma unroll
                    for (int i = 0; i < W; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(rows + 4u * i), "f"(v[i]) : "memory");
                    __syncwarp();
                    const int c = lane & 15, first_row = pix - lane;  // (the rows of a warp are consecutive)
                    for (int r = lane >> 4; r < 32; r += 2) {
                        float one;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(one) : "r"(e.rows + 68u * r + 4u * c));
                        if (first_row + r < p.OW && f + c < p.F) ((float*)p.y)[(long long)(first_row + r) * p.F + f + c] = one;
                    }
                    continue;  // (the lanes meet before the next columns)
                }
                if (!valid) continue;
                const int img = pix / p.hw;
                float* dst = (float*)p.y + ((long long)img * p.F + f) * p.hw + (pix - img * p.hw);
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (f + i < p.F) dst[(long long)i * p.hw] = v[i];
            } else if (OUT == LN_OUT_F16) {
                uint32_t h[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const __half2 q = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                    h[i] = *reinterpret_cast<const uint32_t*>(&q);
                }
                if (valid) ln_store_32((uint8_t*)p.y + (long long)pix * p.ys + 2 * f, h);
            } else {
                uint32_t q[W / 8];
                const uint32_t sf = ln_f4_quantise<FMT>(v, p.g, p.six_g, q);
                if (!valid) continue;
                uint8_t* dst = (uint8_t*)p.y + (long long)pix * p.ys + f / 2;
                if (W == 16) *(uint2*)dst = make_uint2(q[0], q[1]);
                else *(uint4*)dst = make_uint4(q[0], q[1], q[W / 8 - 2], q[W / 8 - 1]);
                p.ysf[ln_f4_sf_at(pix, f / (4 * W), p.ysf_words) + f / W % 4] = (uint8_t)sf;
            }
        }
    }
}

// WBLOCKS: groups of 128 filters that a tile's scales are in; PARTS: clusters whose CTAs split the k range of one tile
template <int FMT, int OUT, int WBLOCKS, bool PARTS>
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
            mbar_init(full_bar(s), p.flat ? 2 : 3);  // the two loaders (with the copies' bytes) and the warps that gather scales
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
    ln_f4_after_predecessor();
    const uint32_t tmem_base = *tmem_slot;
    const int kblocks = p.R * p.S * p.cblocks, log_parts = PARTS ? p.log_parts : 0, rank = (int)blockIdx.x & ((1 << log_parts) - 1);
    const int first_unit = (int)blockIdx.x >> log_parts, step = (int)gridDim.x >> log_parts;
    const int k0 = (kblocks * rank) >> log_parts, k1 = (kblocks * (rank + 1)) >> log_parts;  // of this CTA
    const int tap0 = PARTS ? k0 / p.cblocks : 0, cb0 = k0 - tap0 * p.cblocks, r0 = PARTS ? tap0 / p.S : 0, s0 = tap0 - r0 * p.S;
    constexpr bool overlap = WBLOCKS == 2;

    if (warp == 0) {
        // ------------------------------------------------------------------ loads of the pixels
        if (elect_one()) {
            const uint32_t bytes = 128u * p.bk + (p.flat ? (uint32_t)p.words * 512u : 0u);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = first_unit; ok && unit < p.num_units; unit += step) {
                const f4_box t = box_at(p, unit);
                int sf_row = ((t.ow0 >> 7) * kblocks + k0) * p.words;  // (flat)
                int r = r0, s = s0, c0 = cb0 * p.bk;
                for (int kb = k0; kb < k1;) {  // a tap's k-blocks
                    int ty = r - p.pad, tx = s - p.pad, map = 0;
                    if (p.stride == 2) {
                        const int py = ty & 1, px = tx & 1;  // parity class of the tap
                        ty = (ty - py) >> 1;
                        tx = (tx - px) >> 1;
                        map = py * 2 + px;
                    }
                    for (; c0 < p.cstride && kb < k1; c0 += p.bk, ++kb, sf_row += p.words) {
                        if (!(ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                        const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes, bar = full_bar(stage);
                        mbar_arrive_expect_tx(bar, bytes);
                        tma_load_4d(at, &p.tmA[map], c0, t.ow0 + tx, t.oh0 + ty, t.n0, bar);
                        if (p.flat) tma_load_2d(at + p.off_sfa, &p.tmXS, 0, sf_row, bar);
                        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                    }
                    if (!ok) break;
                    c0 = 0;
                    if (++s == p.S) { s = 0; ++r; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 6) {
        // ------------------------------------------------------------------ loads of the weights
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = first_unit; ok && unit < p.num_units; unit += step) {
                const int f0 = unit_at(p, unit).f0;
                const CUtensorMap* codes = &p.tmB[unit < p.whole ? 0 : 1];
                const uint32_t bytes = (uint32_t)(unit < p.whole ? p.bn : p.narrow) * p.bk + WBLOCKS * (uint32_t)p.words * 512u;
                int col = tap0 * p.cstride, c0 = cb0 * p.bk;  // first byte of the tap, of the k-block inside it
                for (int kb = k0; kb < k1; ++kb) {
                    if (!(ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                    const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes, bar = full_bar(stage);
                    mbar_arrive_expect_tx(bar, bytes);
                    tma_load_2d(at + p.off_b, codes, col + c0, f0, bar);
                    tma_load_3d(at + p.off_sfb, &p.tmWS, 0, kb * p.words, f0 >> 7, bar);
                    c0 += p.bk;
                    if (c0 >= p.cstride) { c0 = 0; col += p.cstride; }
                    if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ instructions
        if (elect_one()) {
            // E2M1 operands (bits 7, 10: type 1), N / 8, scale type (bit 23: 1 = E8M0), M / 128, K-major; the scale ids go to bits 4 and 29
            const uint32_t idesc_base = (1u << 7) | (1u << 10) | ((FMT == LN_MX4 ? 1u : 0u) << 23) | (1u << 27);
            const uint64_t desc_base = make_smem_desc(0u, p.bk);
            const uint64_t sfa_desc = scale_desc(p.off_sfa), sfb_desc = scale_desc(p.off_sfb);
            int stage = 0, t = 0;
            uint32_t phase = 0, set = 0;
            bool ok = true, ready = false;  // ready: the next k-block was there when this one was issued
            for (int unit = first_unit; ok && unit < p.num_units; unit += step, ++t) {
                const int buf = t % p.nbuf;
                if (!(ok = mbar_wait(tempty_bar(buf), (uint32_t)((t / p.nbuf) & 1) ^ 1u, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
                if (overlap && t > 0 && !(ok = mbar_wait(early_bar(buf ^ 1), (uint32_t)(((t - 1) >> 1) & 1), abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(buf * p.acc_step);
                const uint32_t idesc = idesc_base | ((uint32_t)((unit < p.whole ? p.bn : p.narrow) >> 3) << 17);
                const uint32_t shift = (uint32_t)((unit_at(p, unit).f0 & 127) >> 5);  // first column of the tile's filters inside their group of 128
                int c0 = cb0 * p.bk;
                for (int kb = k0; kb < k1; ++kb) {
                    if (!ready && !(ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, LN_STATUS_MMA_TIMEOUT))) break;
                    const int next = stage + 1 == p.stages ? 0 : stage + 1;
                    const uint32_t next_phase = next ? phase : phase ^ 1u;
                    const uint32_t at = smem_base + (uint32_t)stage * p.stage_bytes;
                    const uint32_t sfa = tmem_base + kScaleCols + set * kScaleSet, sfb = sfa + kScaleB;
                    const int left = p.cstride - c0, n = (left < p.bk ? left : p.bk) >> 5;  // instructions of this k-block
                    const uint64_t a_desc = desc_base + (at >> 4), b_desc = desc_base + ((at + p.off_b) >> 4);
                    // Unrolled with constant offsets: as loops with run-time bounds the copies and instructions of a k-block of 128 bytes took
                    // their thread 1100 cycles, this way under 200, less than the 530 that they run for.
                    auto issue = [&](auto most, bool whole) {  // instructions of a whole k-block: 4, 2 or 1; the channels' last one may have fewer
                        constexpr int kN = decltype(most)::value, kWords = FMT == LN_MX4 ? (kN + 1) / 2 : kN;
#pragma unroll
                        for (int j = 0; j < kWords; ++j) {
                            tc_copy_scales(sfa + 4u * j, sfa_desc + ((at + 512u * j) >> 4));
#pragma unroll
                            for (int b = 0; b < WBLOCKS; ++b) tc_copy_scales(sfb + 4u * (j * WBLOCKS + b), sfb_desc + ((at + 512u * (b * kWords + j)) >> 4));
                        }
#pragma unroll
                        for (int i = 0; i < kN; ++i) {
                            const uint32_t word = FMT == LN_MX4 ? i >> 1 : i, id = FMT == LN_MX4 ? (uint32_t)(i & 1) * 2u : 0u;
                            if (whole || i < n) tc_mma_scaled<FMT>(d, a_desc + 2u * i, b_desc + 2u * i, idesc | (id << 4) | (id << 29), sfa + 4u * word, sfb + 4u * word * WBLOCKS + shift, i ? 1u : (uint32_t)(kb != k0));
                            // (asked for while instructions are still being issued: a wait takes its thread 150 cycles even where there is nothing to wait for)
                            if (i == (kN - 1) / 2) ready = mbar_test(full_bar(next), next_phase);
                        }
                    };
                    if (p.bk == 128) { if (n == 4) issue(std::integral_constant<int, 4>(), true); else issue(std::integral_constant<int, 4>(), false); }
                    else if (p.bk == 64) issue(std::integral_constant<int, 2>(), false);
                    else issue(std::integral_constant<int, 1>(), true);
                    tc_commit(empty_bar(stage));
                    set ^= 1u;
                    c0 += p.bk;
                    if (c0 >= p.cstride) c0 = 0;
                    stage = next;
                    phase = next_phase;
                }
                if (!ok) break;
                tc_commit(tfull_bar(buf));
            }
        }
        __syncwarp();
    } else if (warp < 2 + kGatherWarps) {
        // ------------------------------------------------------------------ scales of the pixels under shifted taps
        int unit = first_unit, r = r0, s = s0, cb = cb0, tap = r0 * p.W + s0;  // tap: pixels between the tap's and the first one's
        int iy0[4], ix0[4], q0[4];                             // of the lane's rows under the first tap: place and number of the input pixel
        auto enter_tile = [&]() {
            if (unit >= p.num_units) return;
            const f4_box t = box_at(p, unit);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int row = g * 32 + lane, img = t.n0 + (row >> (p.log_tw + p.log_th));
                ix0[g] = (t.ow0 + (row & (p.TW - 1))) * p.stride - p.pad;
                iy0[g] = (t.oh0 + ((row >> p.log_tw) & (p.TH - 1))) * p.stride - p.pad;
                q0[g] = (img * p.H + iy0[g]) * p.W + ix0[g];
                if (img >= p.N) iy0[g] = -(1 << 28);  // (outside under every tap)
            }
        };
        auto advance = [&]() {
            if (++cb < p.cblocks) return;
            cb = 0;
            ++tap;
            if (++s < p.S) return;
            s = 0;
            tap += p.W - p.S;
            if (++r < p.R) return;
            r = tap = 0;
            unit += step;
            enter_tile();
        };
        const size_t group_bytes = (size_t)p.sf_words * 512u;  // of the scales of 128 pixels
        auto fetch = [&](uint32_t (&v)[4][4]) {
            const uint8_t* base = p.xsf + cb * p.words * 512;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const bool inside = (unsigned)(iy0[g] + r) < (unsigned)p.H && (unsigned)(ix0[g] + s) < (unsigned)p.W;
                const unsigned q = (unsigned)(q0[g] + tap);
                const uint8_t* src = base + (size_t)(q >> 7) * group_bytes + ((q & 31u) * 16u + (q >> 5 & 3u) * 4u);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[g][j] = 0u;
                if (inside) {
                    v[g][0] = __ldg((const uint32_t*)src);
                    if (p.words > 1) v[g][1] = __ldg((const uint32_t*)(src + 512));
                    if (FMT == LN_F4 && p.words > 2) {
                        v[g][2] = __ldg((const uint32_t*)(src + 1024));
                        v[g][3] = __ldg((const uint32_t*)(src + 1536));
                    }
                }
            }
        };
        if (!p.flat) {
            enter_tile();
            for (int i = 2; i < warp; ++i) advance();
            int stage = warp - 2;  // (fewer than stages)
            uint32_t phase = 0;
            uint32_t v[4][4];
            int left = k1 - k0 - stage;  // k-blocks from this one on, where they end inside a unit
            bool ok = true;
            auto more = [&]() { return unit < p.num_units && (!PARTS || left > 0); };
            if (more()) fetch(v);
            while (ok && more()) {
                if (!(ok = warp_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, LN_STATUS_PRODUCER_TIMEOUT))) break;
                const uint32_t dst = smem_base + (uint32_t)stage * p.stage_bytes + p.off_sfa + 16u * lane;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < p.words)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512u * j), "r"(v[0][j]), "r"(v[1][j]), "r"(v[2][j]), "r"(v[3][j]) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(stage));
                stage += kGatherWarps;
                if (stage >= p.stages) { stage -= p.stages; phase ^= 1u; }
                // (behind the fence, which would wait for the reads; the other warps' k-blocks cover their latency)
                for (int i = 0; i < kGatherWarps; ++i) advance();
                left -= kGatherWarps;
                if (more()) fetch(v);
            }
        }
        __syncwarp();
    } else if (warp >= kFirstEpilogueWarp) {
        // ------------------------------------------------------------------ epilogue
        // (one loop per activation: a choice inside it put the code of a unit in pieces far apart, and its warps waited for instructions)
        const f4_epilogue_at at = {tmem_base, tab_base + (uint32_t)(warp - kFirstEpilogueWarp) * 256u, tab_base + kTabBytesF4 + (uint32_t)(warp - kFirstEpilogueWarp) * kRowBytesF4, tfull_bar(0), tempty_bar(0), early_bar(0), smem_base, abort_flag, first_unit, step, rank};
        if (PARTS) f4_exchange(p, at);
        switch (p.act + (p.exact ? 8 : 0)) {
            case LN_ACT_LEAKY: case LN_ACT_LEAKY + 8: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_LEAKY, true>(p, at); break;
            case LN_ACT_RELU: case LN_ACT_RELU + 8: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_RELU, true>(p, at); break;
            case LN_ACT_MISH: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_MISH, false>(p, at); break;
            case LN_ACT_SWISH: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_SWISH, false>(p, at); break;
            case LN_ACT_LOGISTIC: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_LOGISTIC, false>(p, at); break;
            case LN_ACT_MISH + 8: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_MISH, true>(p, at); break;
            case LN_ACT_SWISH + 8: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_SWISH, true>(p, at); break;
            case LN_ACT_LOGISTIC + 8: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_LOGISTIC, true>(p, at); break;
            default: f4_epilogue<FMT, OUT, WBLOCKS, PARTS, LN_ACT_LINEAR, true>(p, at); break;
        }
    }

    if (PARTS && warp < kFirstEpilogueWarp) {  // (the two barriers of the exchange: every warp of the cluster comes to both, whatever its waits ended with)
        cluster_sync();
        cluster_sync();
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
    void (*k)(const f4_params) = p.bn > 128 ? f4_umma_kernel<FMT, OUT, 2, false>
                                            : (p.log_parts ? f4_umma_kernel<FMT, OUT, 1, true> : f4_umma_kernel<FMT, OUT, 1, false>);
    if (!ctx->configured_kernels.count((const void*)k)) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemF4);
        if (e != cudaSuccess) return e;
        ctx->configured_kernels.insert((const void*)k);
    }
    return ln_f4_launch_clusters(ctx, k, grid, kThreadsF4, smem, 1 << p.log_parts, p);
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
    // A launch takes about start + (k-blocks of a tile + (rounds - 1) x the longer of k-blocks and epilogue), rounds = tiles per SM, in ns
    // as measured over 28 shapes of both types with binary16 output (leaky), 4 to 65 us, each with every tile; the choice was the best one or
    // within 3 % of it on all of them.  Where most SMs have nothing to do, a k-block of 256 filters comes faster.
    // The tiles of the last, partly filled round may be cut into units of fewer filters, where those fit into one round.  Where all tiles
    // leave SMs idle, the k range may be split over a cluster, which costs 3.1 us more (launch, two barriers, exchange; 4.3 where most SMs take part): worth it from about
    // 20 k-blocks on (128 x 11008 -> 4096, LN_F4: 16.8 us, split over four 11.4; 3x3 C1024->K512 at 13x13: 14.9 and 10.2).
    const int64_t kblocks = (int64_t)c.k * c.k * kb.cblocks, sms = ctx->sm_count;
    const int cand[3] = {256, 128, 64}, start[3] = {5400, 3650, 3300}, out[3] = {3300, 1750, 900}, flat_k[3] = {490, 360, 320}, tap_k[3] = {640, 520, 420};
    const bool rows = c.out_kind == LN_OUT_F32 && flat && p.hw == 1 && p.F % 8 != 0;  // (their way through shared memory leaves no four stages of the widest tile)
    int force = 0, force_narrow = 0, force_parts = 1;
    if (const char* e = getenv("LN_F4_BN")) {  // (A/B measurements: another filter tile where it can be; "256/64": with the last round in units of 64; "128*4": its k range over 4 CTAs)
        force = force_narrow = atoi(e);
        if (const char* slash = strchr(e, '/')) force_narrow = atoi(slash + 1);
        if (const char* star = strchr(e, '*')) force_parts = atoi(star + 1);
    }
    int64_t least = -1;
    int parts = 1;
    auto consider = [&](int bn, int narrow, int split, int64_t cost) {
        if (force && (bn != force || narrow != force_narrow || split != force_parts)) cost += 1ll << 50;
        if (least < 0 || cost < least) { least = cost; p.bn = bn; p.narrow = narrow; parts = split; }
    };
    for (int i = rows ? 1 : 0; i < 3; ++i) {
        const int64_t tiles = best * ((p.F + cand[i] - 1) / cand[i]), rounds = (tiles + sms - 1) / sms, rest = tiles % sms;
        const int64_t chain = kblocks * (!flat ? tap_k[i] : (i == 0 && 2 * tiles <= sms ? 330 : flat_k[i])), round = chain > out[i] ? chain : out[i];
        consider(cand[i], cand[i], 1, start[i] + chain + (rounds - 1) * round);
        for (int j = i + 1; j < 3; ++j) {
            const int64_t tail = kblocks * (flat ? flat_k[j] : tap_k[j]);
            if (rounds > 1 && rest && rest * (cand[i] / cand[j]) <= sms) consider(cand[i], cand[j], 1, start[j] + chain + (rounds - 2) * round + (tail > out[i] ? tail : out[i]));
        }
        const int split = cand[i] / CH;
        if (i && tiles * split <= sms && kblocks >= split) consider(cand[i], cand[i], split, start[i] + chain / split + (4 * tiles * split > 3 * sms ? 4300 : 3100));
    }
    const int wblocks = p.bn > 128 ? 2 : 1;
    p.nbuf = p.bn == 256 ? 2 : (int)kScaleCols / p.bn;
    p.acc_step = p.bn == 256 ? kOverlapBase : p.bn;
    p.subs = p.bn / CH;
    p.flat = flat ? 1 : 0;
    p.tiles_f = (p.F + p.bn - 1) / p.bn; p.tiles_w = (p.OW + p.TW - 1) / p.TW; p.tiles_h = (p.OH + p.TH - 1) / p.TH;
    const int64_t tiles = best * p.tiles_f;
    p.log_split = log2_of(p.bn / p.narrow);
    const int64_t cut = p.log_split ? tiles % sms : 0, num_units = tiles - cut + (cut << p.log_split);
    // fast_div(n, d) is exact for n < 2^24 and n d < 2^40; a magic number of 0 is a quotient of 0, for the pixels of one row of tiles
    const int most = p.tiles_f > p.tiles_h ? p.tiles_f : p.tiles_h, row = flat ? 1 : p.tiles_w;
    if (num_units >= (1 << 24) || num_units * (most > row ? most : row) >= (1ll << 40)) return ln_fail(ctx, LN_ERR_UNSUPPORTED, "%s: %lld tiles", who, (long long)num_units);
    p.num_units = (int)num_units;
    p.whole = (int)(tiles - cut);
    auto magic = [](int d) { return ((1ull << 40) + (unsigned long long)d - 1) / (unsigned long long)d; };
    p.magic_f = magic(p.tiles_f); p.magic_w = flat ? 0 : magic(p.tiles_w); p.magic_h = magic(p.tiles_h);
    p.off_b = 128u * p.bk;
    p.off_sfa = p.off_b + (uint32_t)p.bn * p.bk;
    p.off_sfb = p.off_sfa + (uint32_t)p.words * 512u;
    p.stage_bytes = (uint32_t)ln_round_up(p.off_sfb + (uint32_t)(p.words * wblocks) * 512u, 1024);
    const size_t rest = 1024 + kBarBytesF4 + kTabBytesF4 + (rows ? 16 * kRowBytesF4 : 0);
    p.stages = (int)((kMaxSmemF4 - rest) / p.stage_bytes);
    if (p.stages > kMaxStagesF4) p.stages = kMaxStagesF4;
    p.log_parts = log2_of(parts);
    size_t smem = rest + (size_t)p.stages * p.stage_bytes;
    // One CTA per SM: it takes all of TMEM and would wait while another one has it, so none asks for less than half of an SM's shared memory.
    if (smem < kLeastSmemF4) smem = kLeastSmemF4;
    // The CTAs of a cluster wait for each other: with one of another such kernel beside each, two clusters could hold the TMEM that the other
    // one waits for.  With all of the shared memory asked for none fits.
    if (parts > 1) smem = kMaxSmemF4;
    p.xsf = (const uint8_t*)x.sf; p.wscale = c.w->wscale; p.bias = c.bias;
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
        CUresult r = CUDA_SUCCESS;
        for (int m = 0; m < (p.log_split ? 2 : 1) && r == CUDA_SUCCESS; ++m) {
            const cuuint32_t box[2] = {(cuuint32_t)p.bk, (cuuint32_t)(m ? p.narrow : p.bn)};
            r = ctx->encode_tiled(&p.tmB[m], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.w->w, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        }
        if (r != CUDA_SUCCESS) return ln_fail(ctx, LN_ERR_CUDA, "%s: cuTensorMapEncodeTiled(weights) failed with %d", who, (int)r);
    }
    {
        const int64_t rows = (int64_t)c.k * c.k * kb.cblocks * kb.words, groups = c.w->fpad / 128;
        const cuuint64_t dims[3] = {128, (cuuint64_t)rows, (cuuint64_t)groups};
        const cuuint64_t strides[2] = {512, (cuuint64_t)rows * 512};
        const cuuint32_t box[3] = {128, (cuuint32_t)kb.words, (cuuint32_t)wblocks};
        CUresult r = ctx->encode_tiled(&p.tmWS, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, c.w->sf, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r == CUDA_SUCCESS && flat) {
            const cuuint64_t xdims[2] = {128, (cuuint64_t)((pixels + 127) / 128 * x.sf_words)};
            r = ctx->encode_tiled(&p.tmXS, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, x.sf, xdims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        }
        if (r != CUDA_SUCCESS) return ln_fail(ctx, LN_ERR_CUDA, "%s: cuTensorMapEncodeTiled(scales) failed with %d", who, (int)r);
    }
    const int grid = parts > 1 ? p.num_units * parts : (p.num_units < ctx->sm_count ? p.num_units : ctx->sm_count);
    cudaError_t e;
#define LN_F4_LAUNCH(FMT) \
    (c.out_kind == LN_OUT_F32 ? launch<FMT, LN_OUT_F32>(ctx, p, grid, smem) : c.out_kind == LN_OUT_F16 ? launch<FMT, LN_OUT_F16>(ctx, p, grid, smem) : launch<FMT, LN_OUT_Q>(ctx, p, grid, smem))
    e = c.dtype == LN_F4 ? LN_F4_LAUNCH(LN_F4) : LN_F4_LAUNCH(LN_MX4);
#undef LN_F4_LAUNCH
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return ln_fail(ctx, LN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    }
    ctx->f4_plan[0] = p.bn;
    ctx->f4_plan[1] = cut ? p.narrow : 0;
    ctx->f4_plan[2] = parts;
    return LN_OK;
}
