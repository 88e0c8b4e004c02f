// Gated feed-forward product and its gradient, bf16 / fp16 with 32-bit sums:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u          x: M x d; Wg, Wu: F x d
//   dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// The products run on one persistent, warp-specialised kernel (ff_gemm_kernel): tcgen05
// tiles with both operands by TMA, of single CTAs or of SM pairs.
//   forward    Half of B is rows of Wg and half the same rows of Wu (of a pair, one CTA
//              stages each), so a thread of the epilogue finds the gate and the up value
//              of one place in its own TMEM row: activation and product happen there and
//              h leaves through a TMA store.
//   gradient   One launch for both products.  dx contracts dg with Wg, then du with Wu,
//              into one accumulator, the weights read MN-major as they lie; dWg and dWu
//              contract over the rows with both operands MN-major: nothing is transposed
//              in memory.  dg and du come from a pointwise pass (ff_pointwise_kernel),
//              rounded to 16 bits as operands of the tensor cores (in float16 infinite
//              beyond 65504, as dh * u would be in that type).
// That pass reads g and u as the forward pass kept them, in 24 bits: in 16 their rounding
// would come beside those of dg, du and the result, and put the gradients' error at 1.8
// instead of 1.4 roundings (of either type; 32 bits would not lower it).
//
// Few rows without a gradient take ff_skinny_kernel.
//
// Measured, M x d x F = 4096 x 2048 x 8192 in bf16 (275 GFLOP a projection pair), two calls
// in a graph on a card that is not yet at its power cap: forward 167 us (1.65 PFLOP/s; a
// library product of the size, without activation, 170), 186 when g and u are kept;
// pointwise 68 us (5.9 TB/s); both gradient products 335 us (1.64 PFLOP/s; two library
// products 350).  Bound by the tensor cores at the clock that their power leaves them (1.6 of
// 1.9 GHz): 77 to 86 % of their cycles.  In a program's loop, at the cap (980 W, 1.40 to 1.55
// GHz), the same take 206, 229 and 420 us, the three library products 211 + 209 + 216.
#include <cuda.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "prof.cuh"
#include "tc.cuh"
#include "tmap.cuh"

namespace {

enum { FF_FORWARD = 0, FF_DX, FF_DW };      // what a work item computes

// Tiles: of one CTA, or of the two CTAs of a cluster (tcgen05.mma.cta_group::2), of which
// each stages its 128 (TALL: 256) rows of A and 128 columns of B.
enum { SINGLE = 0 /* 128 x 128 */, PAIR /* 256 x 256 */, TALL /* 512 x 256 */ };

constexpr uint32_t FOPB = 128 * 64 * 2;     // one 128 x 64 operand block, 16 KB
constexpr int FEPI_WARPS = 8;
constexpr uint32_t FOUTB = 32 * 64 * 2;     // a warp's 32 x 64 block of the result, 4 KB
constexpr int FTHREADS = 64 + 32 * FEPI_WARPS;
constexpr int FBAND_ROWS = 4096;            // rows per band of the tile order

template <int SHAPE>
struct FfShape {
    static constexpr int NC = SHAPE == SINGLE ? 1 : 2;      // CTAs of a tile
    static constexpr int HALVES = SHAPE == TALL ? 2 : 1;    // 128-row blocks of A in a CTA
    static constexpr int TM = 128 * NC * HALVES, TN = 128 * NC;
    static constexpr uint32_t STAGE = (HALVES + 1) * FOPB;
    static constexpr int STAGES = SHAPE == TALL ? 4 : 6;    // 192 KB either way
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + FEPI_WARPS * FOUTB;
};
static_assert(FfShape<TALL>::SMEM <= 231 * 1024 && FfShape<PAIR>::SMEM <= 231 * 1024, "shared memory");

// One product: `parts` results of rows x cols in mt x nt tiles, each the sum over
// `steps` 64-deep blocks, which `splits` items share.
struct FfWork {
    int mode, parts, mt, nt, splits, steps, rows, cols;
    int tma_out, vec;                       // results by TMA; else by stores of 4, 2 or (1) one or two values
    int count0;                             // split: this product's first counter,
    int64_t partial0;                       // and the first of its partial sums
    int64_t ldo;
    void* outp[2];
};

struct FfGemm {
    // boxes 64 wide: 128 rows of what is read K-major (64 of the weights for single CTAs),
    // 64 of what is read MN-major, 32 of the results (h, or dx, dWg, dWu)
    CUtensorMap x, w[2], dguk[2], dgum[2], out[3];
    FfWork work[2];                         // in the order in which a CTA (pair) takes them
    unsigned char* saved;                   // forward: g and u for the gradient, or null
    float* partial;                         // split tiles: sums of the items
    int* count;                             // split tiles: items done, per epilogue warp
    int* status;
    int extra;                              // see ff_item
    int dtype;
};

struct FfItem { int w, part, m, n, split, tile; };

// The n-th item of group g of G (a CTA or a pair): items of work[0] in turn, then those
// of work[1].  Where the first do not come out even, the groups that got one less
// take `extra` items of the second first: about as many as take the same time.
template <int BAND>
SCAO_DEV bool ff_item(const FfGemm& P, int g, int G, int n, FfItem& it) {
    const FfWork &a = P.work[0], &b = P.work[1];
    const int na = a.parts * a.mt * a.nt * a.splits, nb = b.parts * b.mt * b.nt * b.splits;
    const int mine = g < na ? (na - g + G - 1) / G : 0, r = na % G;
    int i;
    if (n < mine) {
        it.w = 0;
        i = g + n * G;
    } else {
        it.w = 1;
        n -= mine;
        const int late = r ? G - r : 0, early = min(late * P.extra, nb);
        if (late && g >= r) {
            i = g - r + n * late;
            if (n < P.extra && i < early) goto found;
            n -= P.extra;
            if (n < 0) return false;
        }
        i = early + g + n * G;
        if (i >= nb) return false;
    }
found:
    const FfWork& w = P.work[it.w];
    it.tile = i / w.splits;
    it.split = i - it.tile * w.splits;
    const int per = w.mt * w.nt;
    it.part = it.tile / per;
    int t = it.tile - it.part * per;
    // in bands of row tiles, row tiles fastest: the tiles that run at one time share few
    // operand panels, which stay in L2
    const int band = t / (BAND * w.nt);
    t -= band * BAND * w.nt;
    const int h = min(BAND, w.mt - band * BAND);
    it.n = t / h;
    it.m = band * BAND + t - it.n * h;
    return true;
}

// first step of a split
SCAO_DEV int ff_first(const FfWork& w, int split) { return (int)((int64_t)split * w.steps / w.splits); }

SCAO_DEV float ff_sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

constexpr float TANH_A = 0.7978845608028654f, TANH_B = 0.044715f;   // sqrt(2 / pi)

template <int ACT>
SCAO_DEV float ff_act(float g) {
    if (ACT == SCAO_ACT_SILU) return g * ff_sigmoid(g);
    if (ACT == SCAO_ACT_GELU) return g * normcdff(g);
    // 0.5 (1 + tanh y) = sigmoid(2 y)
    return g * ff_sigmoid(2.f * TANH_A * (g + TANH_B * g * g * g));
}

// act(g) and act'(g)
template <int ACT>
SCAO_DEV void ff_act_grad(float g, float& a, float& d) {
    if (ACT == SCAO_ACT_SILU) {
        const float s = ff_sigmoid(g);
        a = g * s;
        d = s * (1.f + g * (1.f - s));
    } else if (ACT == SCAO_ACT_GELU) {
        const float s = normcdff(g);
        a = g * s;
        d = s + g * 0.3989422804014327f * __expf(-0.5f * g * g);
    } else {
        const float s = ff_sigmoid(2.f * TANH_A * (g + TANH_B * g * g * g));
        a = g * s;
        const float t = a * (1.f - s);      // 0 far out, where g * g may be infinite
        d = t == 0.f ? s : s + t * 2.f * TANH_A * (1.f + 3.f * TANH_B * g * g);
    }
}

SCAO_DEV uint32_t pack2(float a, float b, int dt) {
    if (dt == SCAO_BF16) return (uint32_t)f_to_bf16_bits(a) | ((uint32_t)f_to_bf16_bits(b) << 16);
    return (uint32_t)f_to_f16_bits(a) | ((uint32_t)f_to_f16_bits(b) << 16);
}

// g and u as kept for the gradient: rounded to 24 bits (16 of the significand), 3 bytes a
// value, which is 2^-8 of a bfloat16 rounding, 2^-5 of a float16 one, and a quarter less to
// write and read than 32.
// Per whole 128-row x 128-column block the g values, then the u values, as [16-column
// group][16 bytes of its 48][row], so that a warp (a thread per row) writes 512
// consecutive bytes.
constexpr int SAVED_BLOCK = 128 * 128 * 3;
SCAO_DEV int64_t saved_off(int row, int col, int col_blocks) {
    return ((int64_t)(row >> 7) * col_blocks + (col >> 7)) * (2 * SAVED_BLOCK) +
           (((col & 127) >> 4) * 3 * 128 + (row & 127)) * 16;
}
constexpr int SAVED_PLANE = 128 * 16;

// to nearest, ties away; infinities and NaN as they are
SCAO_DEV uint32_t round24(uint32_t x) { return (x & 0x7fffffffu) < 0x7f800000u ? x + 0x80u : x; }

SCAO_DEV void save16(unsigned char* p, const uint32_t* v) {
    uint32_t w[12];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = round24(v[4 * i]), b = round24(v[4 * i + 1]), c = round24(v[4 * i + 2]),
                       d = round24(v[4 * i + 3]);
        w[3 * i] = __byte_perm(a, b, 0x5321);           // upper three bytes of each, in turn
        w[3 * i + 1] = __byte_perm(b, c, 0x6532);
        w[3 * i + 2] = __byte_perm(c, d, 0x7653);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        *(uint4*)(p + i * SAVED_PLANE) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// the four values of three of those words
SCAO_DEV void restore4(uint32_t w0, uint32_t w1, uint32_t w2, float* v) {
    v[0] = __uint_as_float(w0 << 8);
    v[1] = __uint_as_float(__byte_perm(w0, w1, 0x5433) & 0xffffff00u);
    v[2] = __uint_as_float(__byte_perm(w1, w2, 0x4322) & 0xffffff00u);
    v[3] = __uint_as_float(w2 & 0xffffff00u);
}

SCAO_DEV void ff_fail(int* status) { *(volatile int*)status = 2; }

// One warp's 32 x 64 block of a result, 16-bit values: into shared memory (after the
// block before it has left), 8 columns of this thread's row at a time, then a TMA store
// or guarded stores.
SCAO_DEV void ff_stage_ready(int lane) {
    if (lane == 0) bulk_wait_read0();
    __syncwarp();
}
SCAO_DEV void ff_stage_put(unsigned char* stage, int lane, int c, const uint32_t* v) {
    *(uint4*)(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) = make_uint4(v[0], v[1], v[2], v[3]);
}
SCAO_DEV void ff_stage_store(const FfWork& w, const CUtensorMap* map, int part, unsigned char* stage, int row0,
                             int col0, int lane) {
    if (w.tma_out) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (row0 < w.rows && col0 < w.cols) tma_store_2d(map, col0, row0, smem_u32(stage));
            bulk_commit();
        }
        return;
    }
    __syncwarp();
    // rows that are no multiple of 16 bytes apart: the widest stores that their pitch allows
    auto at = [&](int r, int c) { return stage + r * 128 + (((c >> 3) ^ (r & 7)) * 16) + (c & 7) * 2; };
    uint16_t* out = (uint16_t*)w.outp[part] + col0;
    const int rows = min(32, w.rows - row0), cols = min(64, w.cols - col0);
    if (w.vec == 4) {
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
            const int r = 2 * i + (lane >> 4), c = (lane & 15) * 4;
            if (r < rows && c < cols) *(uint2*)(out + (row0 + r) * w.ldo + c) = *(const uint2*)at(r, c);
        }
    } else if (w.vec == 2) {
#pragma unroll 4
        for (int r = 0; r < 32; ++r)
            if (r < rows && 2 * lane < cols)
                *(uint32_t*)(out + (row0 + r) * w.ldo + 2 * lane) = *(const uint32_t*)at(r, 2 * lane);
    } else {
        // a row that begins between two 32-bit words (every other one of an odd pitch): a lane's
        // word is then the upper half of its pair and the lower half of the next lane's
        uint16_t* d = out + row0 * w.ldo;
        auto even = [&](int r) {
            const uint32_t x = *(const uint32_t*)at(r, 2 * lane);
            uint16_t* p = d + r * w.ldo + 2 * lane;
            if (r >= rows) return;
            if (2 * lane + 1 < cols) *(uint32_t*)p = x;
            else if (2 * lane < cols) *p = (uint16_t)x;
        };
        auto odd = [&](int r) {
            const uint32_t x = *(const uint32_t*)at(r, 2 * lane);
            const uint32_t next = __shfl_down_sync(0xffffffffu, x, 1);
            uint16_t* p = d + r * w.ldo + 2 * lane + 1;
            if (r >= rows) return;
            if (lane < 31 && 2 * lane + 2 < cols) *(uint32_t*)p = __funnelshift_r(x, next, 16);
            else if (2 * lane + 1 < cols) *p = (uint16_t)(x >> 16);
            if (lane == 0 && cols > 0) p[-1] = (uint16_t)x;
        };
        if (!(w.ldo & 1)) {                 // a result that begins so: all its rows alike
#pragma unroll 1
            for (int r = 0; r < 32; ++r)
                if ((uintptr_t)d & 2) odd(r); else even(r);
        } else if ((uintptr_t)d & 2) {
#pragma unroll 4
            for (int r = 0; r < 32; r += 2) { odd(r); even(r + 1); }
        } else {
#pragma unroll 4
            for (int r = 0; r < 32; r += 2) { even(r); odd(r + 1); }
        }
    }
    __syncwarp();
}

SCAO_DEV void ff_store_block(const FfWork& w, const CUtensorMap* map, int part, const uint32_t* v,
                             unsigned char* stage, int row0, int col0, int lane) {
    ff_stage_ready(lane);
#pragma unroll
    for (int c = 0; c < 8; ++c) ff_stage_put(stage, lane, c, v + 4 * c);
    ff_stage_store(w, map, part, stage, row0, col0, lane);
}

// 16 columns of a row from their gate and up values: kept for the gradient, and their h.
template <int ACT>
SCAO_DEV void ff_finish16(const FfGemm& G, const FfWork& w, const uint32_t* g, const uint32_t* u, int row, int col,
                          uint32_t* out) {
    if (G.saved && row < w.rows && col < w.cols) {
        unsigned char* p = G.saved + saved_off(row, col, (w.cols + 127) >> 7);
        save16(p, g);
        save16(p + SAVED_BLOCK, u);
    }
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = ff_act<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]);
#pragma unroll
    for (int i = 0; i < 16; i += 2) out[i / 2] = pack2(y[i], y[i + 1], G.dtype);
}

// The product kernel.  Roles per CTA: warp 0 TMA producer; warp 1 TMEM owner and (first
// CTA) MMA issuer; warps 2-9 epilogue, which overlaps the next item's main loop.  TMEM
// holds two accumulators of 128 rows x TN columns per CTA: of alternate items, or, TALL,
// of the two row halves of one item.  TALL reads a quarter less for a result; its
// halves share every stage, so around the end of an item the order of the MMAs changes:
// a pipeline's length of the first half's last steps, then the second half's, then the
// same of the next item, which gives the epilogue that long for each half
// while the tensor cores go on.
// Every wait is bounded; when one runs out the CTA records it in *status, issues no
// more, waits for its copies in flight, and both CTAs still meet at the end.
template <int SHAPE, bool FORWARD, int ACT>
__global__ void __cluster_dims__(SHAPE == SINGLE ? 1 : 2, 1, 1) __launch_bounds__(FTHREADS, 1)
ff_gemm_kernel(const __grid_constant__ FfGemm G) {
    typedef FfShape<SHAPE> Sh;
    constexpr bool TWO = Sh::NC == 2;
    constexpr int NC = Sh::NC, HALVES = Sh::HALVES, TM = Sh::TM, TN = Sh::TN, FST = Sh::STAGES;
    constexpr uint32_t FSTAGE = Sh::STAGE;
    constexpr int BAND = FBAND_ROWS / TM;
    // the forward tile of one CTA has 64 columns: four warps read it
    constexpr int EPI = FORWARD && !TWO ? 4 : FEPI_WARPS;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[FST], empty[FST], accf[2], acce[2], fin;
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = TWO ? cluster_ctarank() : 0;
    const bool leader = rank == 0;
    auto sync_all = [] { if (TWO) cluster_sync_all(); else __syncthreads(); };
    auto commit = [](uint64_t* bar) { if (TWO) tc_commit_pair(bar, 0x3); else tc_commit(bar); };
    if (tid == 0) {
        for (int i = 0; i < FST; ++i) { mbar_init(&full[i], NC); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&accf[i], 1); mbar_init(&acce[i], NC * EPI); }
        mbar_init(&fin, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) { if (TWO) tc_alloc_pair(&tslot, 2 * TN); else tc_alloc(&tslot, 2 * TN); }
    if (tid == 96) {                        // the maps, on their way meanwhile
        if (FORWARD) {
            tc_prefetch_map(&G.x);
            tc_prefetch_map(&G.w[0]);
            tc_prefetch_map(&G.w[1]);
        } else {
            for (int i = 0; i < 2; ++i) {
                if (G.work[i].mode == FF_DW) tc_prefetch_map(&G.x);
                for (int k = 0; k < 2; ++k)
                    if (G.work[i].mode == FF_DX) {
                        tc_prefetch_map(&G.w[k]);
                        tc_prefetch_map(&G.dguk[k]);
                    } else if (G.work[i].mode == FF_DW) {
                        tc_prefetch_map(&G.dgum[k]);
                    }
            }
        }
    }
    tc_fence_before();
    sync_all();
    tc_fence_after();
    if (!FORWARD) tc_grid_wait();           // launched while the pointwise pass ran
    const uint32_t tmem = tslot;
    const int grp = blockIdx.x / NC, ngrp = gridDim.x / NC;
    FfItem it;
    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t ph = 0, issued = 0, last_ph = 0;
            for (int n = 0; !abort_flag && ff_item<BAND>(G, grp, ngrp, n, it); ++n) {
                const FfWork& w = G.work[it.w];
                const int i0 = it.m * TM + 128 * (int)rank;     // of the first half; the second 256 on
                const int j0 = FORWARD ? it.n * (TN / 2) : it.n * TN + 128 * (int)rank;
                const int s0 = ff_first(w, it.split), s1 = ff_first(w, it.split + 1), seg = w.steps >> 1;
                // one step: waits for its stage, announces its bytes and lets `fill` copy them
                auto run = [&](auto&& fill) {
                    for (int s = s0; s < s1; ++s) {
                        if (!mbar_wait(&empty[stage], ph ^ 1)) { abort_flag = 1; ff_fail(G.status); return; }
                        const uint32_t bar = TWO ? mapa_shared(smem_u32(&full[stage]), 0) : smem_u32(&full[stage]);
                        if (TWO) mbar_arrive_expect_tx_cl(bar, FSTAGE); else mbar_expect_tx(&full[stage], FSTAGE);
                        const uint32_t a = smem_u32(sm) + stage * FSTAGE;
                        fill(s, a, a + HALVES * FOPB, [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                            if (TWO) tma_load_2d_pair(dst, map, x, y, bar);
                            else tma_load_2d(dst, map, x, y, &full[stage]);
                        });
                        issued |= 1u << stage;
                        last_ph = (last_ph & ~(1u << stage)) | (ph << stage);
                        if (++stage == FST) { stage = 0; ph ^= 1; }
                    }
                };
                constexpr uint32_t HB = FOPB / 2;
                if (FORWARD) {
                    const CUtensorMap* wm = &G.w[rank];
                    run([&](int s, uint32_t a, uint32_t b, auto&& load) {
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) load(a + h * FOPB, &G.x, s * 64, i0 + 256 * h);
                        load(b, wm, s * 64, j0);
                        if (!TWO) load(b + HB, &G.w[1], s * 64, j0);
                    });
                } else if (w.mode == FF_DX) {
                    run([&](int s, uint32_t a, uint32_t b, auto&& load) {
                        const int g = s >= seg, k0 = (s - g * seg) * 64;
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) load(a + h * FOPB, &G.dguk[g], k0, i0 + 256 * h);
                        load(b, &G.w[g], j0, k0);
                        load(b + HB, &G.w[g], j0 + 64, k0);
                    });
                } else {
                    const CUtensorMap* am = &G.dgum[it.part];
                    run([&](int s, uint32_t a, uint32_t b, auto&& load) {
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) {
                            load(a + h * FOPB, am, i0 + 256 * h, s * 64);
                            load(a + h * FOPB + HB, am, i0 + 256 * h + 64, s * 64);
                        }
                        load(b, &G.x, j0, s * 64);
                        load(b + HB, &G.x, j0 + 64, s * 64);
                    });
                }
            }
            // no copy of either CTA is still landing (all complete on the leader's barriers)
            if (leader)
                for (int s = 0; s < FST; ++s)
                    if ((issued >> s) & 1u)
                        if (!mbar_wait(&full[s], (last_ph >> s) & 1u)) ff_fail(G.status);
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            int stage = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            auto need = [&](uint64_t* bar, uint32_t parity) {
                if (ok && !mbar_wait(bar, parity)) ok = false;
                tc_fence_after();
            };
            for (int n = 0; ok && !abort_flag && ff_item<BAND>(G, grp, ngrp, n, it); ++n) {
                const FfWork& w = G.work[it.w];
                const bool amn = !FORWARD && w.mode == FF_DW;
                uint32_t idesc = idesc_bf16(128 * NC, TN, 0, FORWARD ? 0 : 1) | (amn ? 1u << 15 : 0u);
                if (G.dtype == SCAO_F16) idesc &= ~((1u << 7) | (1u << 10));
                const int steps = ff_first(w, it.split + 1) - ff_first(w, it.split);
                auto run = [&](auto a_mn) {
                    // 16 deep: 32 bytes along a K-major row, 2 KB of MN-major rows
                    constexpr bool AMN = decltype(a_mn)::value;
                    const uint32_t a0 = smem_u32(sm), b0 = a0 + HALVES * FOPB;
                    const uint64_t ad0 = AMN ? smem_desc_sw128(a0, FOPB / 2, 1024) : smem_desc_sw128(a0, 16, 1024);
                    const uint64_t bd0 = FORWARD ? smem_desc_sw128(b0, 16, 1024) : smem_desc_sw128(b0, FOPB / 2, 1024);
                    // the products of stage `st` into accumulator `acc`, with A's row block h
                    auto mma = [&](int st, int h, int acc, bool first) {
                        const uint64_t at = (uint64_t)st * (FSTAGE >> 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint64_t ad = ad0 + at + h * (FOPB >> 4) + k * (AMN ? 2048 >> 4 : 32 >> 4);
                            const uint64_t bd = bd0 + at + k * (FORWARD ? 32 >> 4 : 2048 >> 4);
                            const uint32_t more = (!first || k > 0) ? 1u : 0u;
                            if (TWO) tc_mma_bf16_pair(tmem + acc * TN, ad, bd, idesc, more);
                            else tc_mma_bf16(tmem + acc * TN, ad, bd, idesc, more);
                        }
                    };
                    if constexpr (HALVES == 1) {
                        const int acc = n & 1;
                        need(&acce[acc], aph ^ 1);
                        for (int s = 0; s < steps; ++s) {
                            need(&full[stage], ph);
                            if (!ok) return;
                            mma(stage, 0, acc, s == 0);
                            commit(&empty[stage]);
                            if (++stage == FST) { stage = 0; ph ^= 1; }
                        }
                        commit(&accf[acc]);
                        if (acc == 1) aph ^= 1;
                    } else {
                        // `count` steps of the first half, then the same of the second
                        auto block = [&](int count, bool begins, bool ends) {
                            int st = stage;
                            uint32_t p = ph;
                            if (begins) need(&acce[0], aph ^ 1);
                            for (int i = 0; i < count; ++i) {
                                need(&full[st], p);
                                if (!ok) return;
                                mma(st, 0, 0, begins && i == 0);
                                if (++st == FST) { st = 0; p ^= 1; }
                            }
                            if (ends) commit(&accf[0]);
                            if (begins) need(&acce[1], aph ^ 1);
                            if (!ok) return;
                            for (int i = 0; i < count; ++i) {
                                mma(stage, 1, 1, begins && i == 0);
                                commit(&empty[stage]);
                                if (++stage == FST) stage = 0;
                            }
                            ph = p;
                            if (ends) commit(&accf[1]);
                        };
                        const int head = min(steps, FST), tail = min(steps - head, FST);
                        block(head, true, tail == 0);
                        for (int s = head; ok && s < steps - tail; ++s) block(1, false, false);
                        if (ok && tail) block(tail, false, true);
                        aph ^= 1;
                    }
                };
                if (amn) run(std::true_type()); else run(std::false_type());
            }
            if (!ok) { abort_flag = 1; ff_fail(G.status); }
            commit(&fin);
        }
        __syncwarp();
        if (!mbar_wait(&fin, 0)) ff_fail(G.status);
    } else if (warp - 2 < EPI) {
        const int q = warp & 3, h = (warp - 2) >> 2;     // TMEM lane quarter, column half
        unsigned char* stage = sm + (size_t)FST * FSTAGE + (warp - 2) * FOUTB;
        uint32_t aph = 0;
        // accumulator `acc` -> the rows of A's block `half` of item `it`; false to give up
        auto finish = [&](int acc, int half) {
            const FfWork& w = G.work[it.w];
            if (__any_sync(0xffffffffu, abort_flag)) return false;
            if (!__all_sync(0xffffffffu, mbar_wait(&accf[acc], aph))) {
                abort_flag = 1;
                ff_fail(G.status);
                return false;
            }
            tc_fence_after();
            auto release = [&] {                         // this warp has read the accumulator
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (TWO) mbar_arrive_cl(mapa_shared(smem_u32(&acce[acc]), 0));
                    else mbar_arrive(&acce[acc]);
                }
            };
            const int row0 = it.m * TM + 256 * half + 128 * (int)rank + q * 32, row = row0 + lane;
            const uint32_t tb = tmem + acc * TN + ((uint32_t)(q * 32) << 16);
            if constexpr (FORWARD) {
                const int c0 = it.n * (TN / 2) + h * 64;
                if constexpr (!TWO) {
                    // mostly run once: a short loop, whose instructions come from memory sooner
                    ff_stage_ready(lane);
#pragma unroll 1
                    for (int c = 0; c < 64; c += 16) {
                        uint32_t g[16], u[16], out[8];
                        tc_ld16_async(tb + c, g);
                        tc_ld16_async(tb + TN / 2 + c, u);
                        tc_ld16_wait(g);
                        tc_ld16_wait(u);
                        ff_finish16<ACT>(G, w, g, u, row, c0 + c, out);
                        ff_stage_put(stage, lane, c >> 3, out);
                        ff_stage_put(stage, lane, (c >> 3) + 1, out + 4);
                    }
                    release();
                    ff_stage_store(w, &G.out[0], 0, stage, row0, c0, lane);
                } else {
                    // everything out of TMEM first, so the next item's products wait for no store
                    uint32_t gr[64], ur[64], out[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        tc_ld16_async(tb + h * 64 + c, gr + c);
                        tc_ld16_async(tb + TN / 2 + h * 64 + c, ur + c);
                    }
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        tc_ld16_wait(gr + c);
                        tc_ld16_wait(ur + c);
                    }
                    release();
#pragma unroll
                    for (int c = 0; c < 64; c += 16)
                        ff_finish16<ACT>(G, w, gr + c, ur + c, row, c0 + c, out + c / 2);
                    ff_store_block(w, &G.out[0], 0, out, stage, row0, c0, lane);
                }
            } else {
                constexpr int COLS = TN / 2;            // of this warp
                const int cw = h * COLS;
                const CUtensorMap* map = &G.out[w.mode == FF_DX ? 0 : 1 + it.part];
                if (w.splits == 1) {
                    uint32_t out[COLS / 2], v[2][16];
                    tc_ld16_async(tb + cw, v[0]);
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) {        // the next 16 columns are on their way
                        uint32_t* y = v[(c >> 4) & 1];
                        tc_ld16_wait(y);
                        if (c + 16 < COLS) tc_ld16_async(tb + cw + c + 16, v[((c >> 4) + 1) & 1]);
#pragma unroll
                        for (int i = 0; i < 16; i += 2)
                            out[(c + i) / 2] = pack2(__uint_as_float(y[i]), __uint_as_float(y[i + 1]), G.dtype);
                    }
                    release();
#pragma unroll
                    for (int c0 = 0; c0 < COLS; c0 += 64)
                        ff_store_block(w, map, it.part, out + c0 / 2, stage, row0, it.n * TN + cw + c0, lane);
                } else {
                    // a share of the sum goes to memory; the warp that brings the last one adds
                    // them all in their order, whichever came last
                    const int64_t slot = (((int64_t)it.tile * NC + rank) * HALVES + half) * FEPI_WARPS + (warp - 2);
                    constexpr int64_t PART = 32 * COLS;
                    float* mine = G.partial + w.partial0 + (slot * w.splits + it.split) * PART;
#pragma unroll 1
                    for (int c = 0; c < COLS; c += 16) {
                        float v[16];
                        tc_ld16(tb + cw + c, v);
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *(float4*)(mine + ((c + i) / 4 * 32 + lane) * 4) =
                                make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                    release();
                    __threadfence();
                    __syncwarp();
                    int done = 0;
                    if (lane == 0) done = atomicAdd(G.count + w.count0 + slot, 1);
                    if (__shfl_sync(0xffffffffu, done, 0) == w.splits - 1) {
                        __threadfence();
                        const float* all = mine - it.split * PART;
#pragma unroll 1
                        for (int c0 = 0; c0 < COLS; c0 += 64) {
                            float y[64];
#pragma unroll
                            for (int i = 0; i < 64; ++i) y[i] = 0.f;
#pragma unroll 2
                            for (int p = 0; p < w.splits; ++p) {
                                const float4* z = (const float4*)(all + p * PART) + c0 * 8 + lane;
                                float4 t[16];               // one share's loads together
#pragma unroll
                                for (int i = 0; i < 16; ++i) t[i] = __ldcg(z + i * 32);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    y[4 * i] += t[i].x;
                                    y[4 * i + 1] += t[i].y;
                                    y[4 * i + 2] += t[i].z;
                                    y[4 * i + 3] += t[i].w;
                                }
                            }
                            uint32_t out[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) out[i] = pack2(y[2 * i], y[2 * i + 1], G.dtype);
                            ff_store_block(w, map, it.part, out, stage, row0, it.n * TN + cw + c0, lane);
                        }
                    }
                }
            }
            return true;
        };
        for (int n = 0; ff_item<BAND>(G, grp, ngrp, n, it); ++n) {
            if constexpr (HALVES == 1) {
                if (!finish(n & 1, 0)) break;
                if (n & 1) aph ^= 1;
            } else {
                bool more = true;
#pragma unroll 1
                for (int half = 0; more && half < 2; ++half) more = finish(half, half);
                if (!more) break;
                aph ^= 1;
            }
        }
        if (lane == 0) bulk_wait_read0();   // the stores have left shared memory
    }
    tc_fence_before();
    __syncthreads();
    sync_all();
    tc_fence_after();
    if (warp == 1) { if (TWO) tc_dealloc_pair(tmem, 2 * TN); else tc_dealloc(tmem, 2 * TN); }
}

// dg = dh u act'(g), du = dh act(g).  A block takes `span` rows of a 128-column block of
// g and u as they were kept; a warp 8 rows x 64 columns at a time, a thread 16 columns
// of a row: runs of 128 bytes of every array.  HBM bound (12 bytes a value): 4096 x 8192 in
// 68 us, 5.9 TB/s.  (4 columns a thread, 4 to 32 bytes a run, took 1.3 to 1.6 times as long.)
constexpr int PT = 256;

template <int ACT>
__global__ void __launch_bounds__(PT)
ff_pointwise_kernel(const unsigned char* __restrict__ saved, const uint16_t* __restrict__ dh, int64_t lddh,
                    uint16_t* __restrict__ dg, uint16_t* __restrict__ du, int64_t ldg, int rows,
                    int cols, int dtype, int vec, int span, int* count, int n_count) {
    tc_grid_release();                      // the products may set up while this runs
    // the counters of the products that follow
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * PT + threadIdx.x; i < n_count;
         i += (int64_t)gridDim.x * gridDim.y * PT)
        count[i] = 0;
    const int cb = (cols + 127) >> 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // once round, unless there are more blocks of columns than a grid has places
    for (int c = blockIdx.y * 128 + (warp & 1) * 64 + (lane & 3) * 16; c < cols; c += gridDim.y * 128) {
        for (int i = (warp >> 1) * 8 + (lane >> 2); i < span; i += 32) {
            const int r = blockIdx.x * span + i;
            if (r >= rows) break;
            const unsigned char* p = saved + saved_off(r, c, cb);
            uint4 gw[3], uw[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                gw[k] = *(const uint4*)(p + k * SAVED_PLANE);
                uw[k] = *(const uint4*)(p + SAVED_BLOCK + k * SAVED_PLANE);
            }
            const uint16_t* d = dh + r * lddh + c;
            uint32_t y[8];
            if (vec) {
                const bool all = c + 8 < cols;
                const uint4 a = *(const uint4*)d, b = all ? *(const uint4*)(d + 8) : make_uint4(0, 0, 0, 0);
                y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w;
                y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    y[k] = (c + 2 * k < cols ? (uint32_t)d[2 * k] : 0) |
                           (c + 2 * k + 1 < cols ? (uint32_t)d[2 * k + 1] << 16 : 0);
            }
            const uint32_t gq[12] = {gw[0].x, gw[0].y, gw[0].z, gw[0].w, gw[1].x, gw[1].y,
                                     gw[1].z, gw[1].w, gw[2].x, gw[2].y, gw[2].z, gw[2].w};
            const uint32_t uq[12] = {uw[0].x, uw[0].y, uw[0].z, uw[0].w, uw[1].x, uw[1].y,
                                     uw[1].z, uw[1].w, uw[2].x, uw[2].y, uw[2].z, uw[2].w};
            uint32_t og[8], ou[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float g[4], u[4], a[4], b[4], z[4];
                restore4(gq[3 * k], gq[3 * k + 1], gq[3 * k + 2], g);
                restore4(uq[3 * k], uq[3 * k + 1], uq[3 * k + 2], u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t bits = y[2 * k + (e >> 1)] >> (16 * (e & 1)) & 0xffff;
                    z[e] = dtype == SCAO_BF16 ? bf16_bits_to_f(bits) : f16_bits_to_f(bits);
                    ff_act_grad<ACT>(g[e], a[e], b[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    ou[2 * k + e / 2] = pack2(z[e] * a[e], z[e + 1] * a[e + 1], dtype);
                    og[2 * k + e / 2] = pack2(z[e] * u[e] * b[e], z[e + 1] * u[e + 1] * b[e + 1], dtype);
                }
            }
            // dg and du have a pitch of whole lines: this may write past `cols` within it, where the
            // products read nothing
            uint16_t *pg = dg + r * ldg + c, *pu = du + r * ldg + c;
            *(uint4*)pg = make_uint4(og[0], og[1], og[2], og[3]);
            *(uint4*)(pg + 8) = make_uint4(og[4], og[5], og[6], og[7]);
            *(uint4*)pu = make_uint4(ou[0], ou[1], ou[2], ou[3]);
            *(uint4*)(pu + 8) = make_uint4(ou[4], ou[5], ou[6], ou[7]);
        }
    }
}

// Few rows: the time is one reading of the weights, so no tile waits for a whole
// operand block.  A warp takes 8 FG inner columns: the 16 rows of an mma.m16n8k16 A
// operand are 8 gate and 8 up weight rows, loaded straight from global memory into the
// registers that the instruction reads (a contraction may take its terms in any order,
// so a lane's 16 consecutive bytes serve as the k places of two instructions, in x as
// in the weights).  Gate and up of one place meet in one thread.  The block's warps
// share a row's contraction and join in shared memory in a fixed order.
constexpr int SK_ROWS = 64;

SCAO_DEV void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                        uint32_t b1, bool bf16) {
    if (bf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the 8 values from p on, those beyond the row's end as zeros
SCAO_DEV uint4 load8_guard(const uint16_t* p, int left) {
    if (left >= 8) return *(const uint4*)p;
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < left; ++i) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Registers: up to 8 rows at most 72, so that seven blocks of four warps fit an SM (1024
// blocks, the columns of 8192, are then one wave).
constexpr int sk_registers(int nt) { return nt == 1 ? 72 : nt == 2 ? 64 : nt == 4 ? 128 : 144; }

template <int ACT, bool BF16, int NT, int FG>
__global__ void __maxnreg__(sk_registers(NT))
ff_skinny_kernel(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ wg, int64_t ldg,
                 const uint16_t* __restrict__ wu, int64_t ldu, uint16_t* __restrict__ h, int rows, int d,
                 int ff) {
    constexpr int U = NT == 1 ? 4 : NT <= 4 ? 2 : 1;      // 32-deep steps in flight
    extern __shared__ float part[];                       // [warp][NT * 4][lane]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int warps = blockDim.x >> 5, f0 = blockIdx.x * 8 * FG + g;
    float acc[FG][NT][4];
#pragma unroll
    for (int j = 0; j < FG; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][n][i] = 0.f;
    for (int k0 = warp * 32 * U; k0 < d; k0 += warps * 32 * U) {
        uint4 a[FG][U], b[FG][U], v[NT][U];
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const int k = k0 + 32 * s + 8 * t;
#pragma unroll
            for (int j = 0; j < FG; ++j) {
                const int64_t f = min(f0 + 8 * j, ff - 1);
                a[j][s] = load8_guard(wg + f * ldg + k, d - k);
                b[j][s] = load8_guard(wu + f * ldu + k, d - k);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = n * 8 + g;
                v[n][s] = load8_guard(x + (int64_t)min(r, rows - 1) * ldx + k, r < rows ? d - k : 0);
            }
        }
#pragma unroll
        for (int s = 0; s < U; ++s)
#pragma unroll
            for (int j = 0; j < FG; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 p = a[j][s], q = b[j][s], y = v[n][s];
                    mma_16816(acc[j][n], p.x, q.x, p.y, q.y, y.x, y.y, BF16);
                    mma_16816(acc[j][n], p.z, q.z, p.w, q.w, y.z, y.w, BF16);
                }
    }
#pragma unroll
    for (int j = 0; j < FG; ++j) {
        if (j) __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[(warp * NT * 4 + n * 4 + i) * 32 + lane] = acc[j][n][i];
        __syncthreads();
        // a warp per row group; rows 2t + i, gate in place i and up in 2 + i
        const int f = f0 + 8 * j;
        for (int n = warp; n < NT; n += warps)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float gate = 0.f, upv = 0.f;
                for (int w = 0; w < warps; ++w) {
                    gate += part[(w * NT * 4 + n * 4 + i) * 32 + lane];
                    upv += part[(w * NT * 4 + n * 4 + 2 + i) * 32 + lane];
                }
                const int r = n * 8 + 2 * t + i;
                if (f < ff && r < rows) {
                    const float y = ff_act<ACT>(gate) * upv;
                    h[(int64_t)r * ff + f] = BF16 ? f_to_bf16_bits(y) : f_to_f16_bits(y);
                }
            }
    }
}

// Copies of operands whose rows TMA cannot read, at a pitch of whole 128-byte lines (a
// tile's rows at 16-byte steps cost a fifth sector for every four), zeros behind each row:
// up to three matrices in one launch, a thread per 16 bytes written.  Where the two 16-byte words around a source run lie inside the
// matrix they are loaded whole and shifted, else (its first and last few values) by
// single values.
struct FfPack {
    const uint16_t* src[3];
    uint16_t* dst[3];
    int64_t pitch[3], vecs[3];              // of the source; 16-byte vectors of the copy
    int rows[3], cols[3], n;
};

__global__ void __launch_bounds__(256)
ff_pack_kernel(const __grid_constant__ FfPack P) {
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int m = 0;
    while (m < P.n && i >= P.vecs[m]) i -= P.vecs[m++];
    if (m == P.n) return;
    const int cols = P.cols[m], per = (cols + 63) >> 6 << 3;
    const int64_t row = i / per;
    const int c = (int)(i - row * per) * 8, left = cols - c;
    const uint16_t* p = P.src[m] + row * P.pitch[m] + c;
    const uint16_t* end = P.src[m] + (P.rows[m] - 1) * P.pitch[m] + cols;
    const int off = (int)((uintptr_t)p & 15);
    const uint16_t* lo = p - off / 2;
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left >= 8 && off == 0) {
        const uint4 a = *(const uint4*)p;
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else if (left > 0 && lo >= P.src[m] && lo + 16 <= end) {
        const uint4 a = *(const uint4*)lo, b = *(const uint4*)(lo + 8);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        if (off & 8)
#pragma unroll
            for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
        if (off & 4)
#pragma unroll
            for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
        if (off & 2)
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
#pragma unroll
        for (int k = 0; k < 4; ++k)         // nothing behind the row
            if (2 * k + 1 >= left) w[k] = 2 * k < left ? w[k] & 0xffff : 0;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) w[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
    }
    *(uint4*)(P.dst[m] + (row * per) * 8 + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t up64(int64_t n) { return (n + 63) / 64 * 64; }
int up(int64_t n, int k) { return (int)((n + k - 1) / k); }

template <int SHAPE, bool FORWARD, int ACT>
int launch_shape(const FfGemm& G, int items, cudaStream_t st) {
    auto* kernel = ff_gemm_kernel<SHAPE, FORWARD, ACT>;
    constexpr int NC = FfShape<SHAPE>::NC, SMEM = (int)FfShape<SHAPE>::SMEM;
    {
        // once per device, before any thread launches there
        static std::mutex mu;
        static PerDeviceOnce once;
        std::lock_guard<std::mutex> lk(mu);
        if (once.first() &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
            return SCAO_ERR_LAUNCH;
    }
    const int groups = scao_sm_count() / NC;
    ProfScope p(SLOT_GATED_FF, st);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((items < groups ? items : groups) * NC));
    cfg.blockDim = dim3(FTHREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    // The gradient's products set up beside the pointwise pass, which every earlier kernel
    // precedes (512 x 128 x 512: 1 us).  Not in front of other kernels (0.3 to 0.6 us a call):
    // the order of what came before would rest on their own waits.
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = FORWARD ? 0 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, G) != cudaSuccess) {
        (void)cudaGetLastError();
        return SCAO_ERR_LAUNCH;
    }
    return SCAO_OK;
}

template <bool FORWARD, int ACT>
int launch_gemm(int shape, const FfGemm& G, int items, cudaStream_t st) {
    if (shape == SINGLE) return launch_shape<SINGLE, FORWARD, ACT>(G, items, st);
    if (shape == PAIR) return launch_shape<PAIR, FORWARD, ACT>(G, items, st);
    return launch_shape<TALL, FORWARD, ACT>(G, items, st);
}

int tile_rows(int shape) { return shape == SINGLE ? 128 : shape == PAIR ? 256 : 512; }
int tile_cols(int shape) { return shape == SINGLE ? 128 : 256; }
int group_count(int shape) { return scao_sm_count() / (shape == SINGLE ? 1 : 2); }

// Time of the busiest group, as ff_item deals the items out: na of ta each, then nb of tb.
double longest(int64_t na, double ta, int64_t nb, double tb, int extra, int G) {
    const int64_t h = na / G, r = na % G, early = r ? (G - r) * extra < nb ? (G - r) * extra : nb : 0;
    const double rest = (double)((nb - early + G - 1) / G) * tb;
    const double x = (double)(h + (r > 0)) * ta + rest, y = (double)h * ta + (early ? extra : 0) * tb + rest;
    return x > y ? x : y;
}

// Microseconds, measured, of which the plan is chosen.  A step of a tile: a CTA takes in
// about 50 bytes of operands a clock, whatever the shape, so the 32 KB of SINGLE and PAIR
// bound their steps (the tensor cores need 256 and 512 clocks of them), the 48 KB of TALL
// take about its 1024 clocks.  An epilogue, which an item of few steps waits for.  Set-up,
// first copies and the last epilogue, beyond SINGLE's.  Joining a tile's shares.
double step_us(int shape) { return shape == SINGLE ? 0.35 : shape == PAIR ? 0.40 : 0.72; }
double item_us(int shape, int steps) {
    const double epilogue = shape == SINGLE ? 1.6 : shape == PAIR ? 2.4 : 4.8, main = step_us(shape) * steps;
    return main > epilogue ? main : epilogue;
}
double begin_us(int shape) { return shape == SINGLE ? 0.0 : shape == PAIR ? 1.2 : 1.6; }
double join_us(int shape, int splits) {
    return splits == 1 ? 0.0 : shape == SINGLE ? 1.5 + 0.3 * splits : 4.0 + 1.0 * splits;
}

struct FfPlan {
    int shape;
    FfWork dx, dw;
    int dx_items, dw_items, extra;
    bool dx_first;
    int64_t partial_floats, counts;
    double us;                              // below 0: too many tiles
};

// The gradient's products in tiles of one shape, dx and dW cut along the contraction
// into so many items.
FfPlan plan_shape(int shape, int rows, int d, int ff, int dx_splits, int dw_splits) {
    FfPlan p;
    memset(&p, 0, sizeof(p));
    p.shape = shape;
    const int tm = tile_rows(shape), tn = tile_cols(shape), groups = group_count(shape);
    auto set = [&](FfWork& w, int mode, int parts, int r, int steps, int splits) {
        w.splits = splits > 0 ? splits : 1;
        if (splits == 0) return (int64_t)0;             // not wanted
        w.mode = mode;
        w.parts = parts;
        w.mt = up(r, tm);
        w.nt = up(d, tn);
        w.steps = steps;
        w.rows = r;
        w.cols = d;
        w.ldo = d;
        return (int64_t)parts * w.mt * w.nt;
    };
    const int64_t nx = set(p.dx, FF_DX, 1, rows, 2 * up(ff, 64), dx_splits);
    const int64_t nw = set(p.dw, FF_DW, 2, ff, up(rows, 64), dw_splits);
    const int64_t per_tile = (int64_t)tm * tn, warps = tm / 128 * FEPI_WARPS;
    if (p.dx.splits > 1) {
        p.partial_floats = nx * p.dx.splits * per_tile;
        p.counts = nx * warps;
    }
    p.dw.partial0 = p.partial_floats;
    p.dw.count0 = (int)p.counts;
    if (p.dw.splits > 1) {
        p.partial_floats += nw * p.dw.splits * per_tile;
        p.counts += nw * warps;
    }
    const int64_t ix = nx * p.dx.splits, iw = nw * p.dw.splits;
    if (ix + iw > 1 << 30) {
        p.us = -1;
        return p;
    }
    p.dx_items = (int)ix;
    p.dw_items = (int)iw;
    // the product with the longer items first
    const double tx = nx ? item_us(shape, up(p.dx.steps, p.dx.splits)) : 0;
    const double tw = nw ? item_us(shape, up(p.dw.steps, p.dw.splits)) : 0;
    p.dx_first = tx >= tw;
    const double a = p.dx_first ? tx : tw, b = p.dx_first ? tw : tx;
    p.extra = b > 0 ? (int)(a / b + 0.5) : 0;
    const int most = p.dx.splits > p.dw.splits ? p.dx.splits : p.dw.splits;
    p.us = begin_us(shape) + join_us(shape, most) +
           (p.dx_first ? longest(ix, a, iw, b, p.extra, groups) : longest(iw, a, ix, b, p.extra, groups));
    return p;
}

// The shape and the cut whose busiest group is done first.  Cuts: items of 8 steps and
// more, in lengths a fifth apart, of the products that are longer than that, while their
// shares are no more than the groups.
FfPlan plan_backward_new(int rows, int d, int ff, bool want_dx, bool want_dw) {
    FfPlan best = plan_shape(TALL, rows, d, ff, want_dx, want_dw);
    auto take = [&](const FfPlan& p) { if (best.us < 0 || (p.us >= 0 && p.us < best.us)) best = p; };
    for (int shape = SINGLE; shape <= PAIR; ++shape) {
        const FfPlan whole = plan_shape(shape, rows, d, ff, want_dx, want_dw);
        take(whole);
        if (whole.us < 0) continue;
        const int64_t nx = whole.dx_items, nw = whole.dw_items, groups = group_count(shape);
        const int most = whole.dx.steps > whole.dw.steps ? whole.dx.steps : whole.dw.steps;
        for (int64_t len = 8; len < most; len += len / 5 > 1 ? len / 5 : 1) {
            const int sx = want_dx ? up(whole.dx.steps, (int)len) : 0, sw = want_dw ? up(whole.dw.steps, (int)len) : 0;
            if ((sx > 1 ? nx * sx : 0) + (sw > 1 ? nw * sw : 0) <= groups)
                take(plan_shape(shape, rows, d, ff, sx, sw));
        }
    }
    return best;
}

// The workspace query and the call that follows it ask for the same plan.
const FfPlan& plan_backward(int rows, int d, int ff, bool want_dx, bool want_dw) {
    static thread_local FfPlan plan;
    static thread_local int of[5] = {-1, 0, 0, 0, 0};
    const int now[5] = {rows, d, ff, want_dx, want_dw};
    if (memcmp(of, now, sizeof(of))) {
        plan = plan_backward_new(rows, d, ff, want_dx, want_dw);
        memcpy(of, now, sizeof(of));
    }
    return plan;
}

int64_t tiles_of(int64_t rows, int64_t cols, int tm, int tn) {
    return ((rows + tm - 1) / tm) * ((cols + tn - 1) / tn);
}

// Whether few rows go through ff_skinny_kernel: every block reads x again, so by the bytes
// it takes in (about 8 MB a microsecond) against the tensor-core tiles' steps.  At 32 rows
// 1024 x 4096 takes 8.5 and 12.2 us, 2048 x 8192 20.1 and 19.6.
bool plan_skinny(int rows, int d, int ff) {
    if (rows <= 16) return true;
    if (rows > SK_ROWS) return false;
    const double bytes = 4.0 * d * ff + 2.0 * up(ff, 16) * rows * d;
    if (rows > 32 && up(ff, 16) > scao_sm_count()) return false;        // one block an SM: its registers
    const int64_t waves = (tiles_of(rows, ff, 128, 64) + scao_sm_count() - 1) / scao_sm_count();
    return 2.5 + bytes / 8e6 < 6.0 + step_us(SINGLE) * up(d, 64) * (double)waves;
}

int plan_forward(int rows, int d, int ff) {
    const int steps = up(d, 64);
    int best = SINGLE;
    double least = 0;
    for (int shape = SINGLE; shape <= TALL; ++shape) {
        const int64_t n = tiles_of(rows, ff, tile_rows(shape), tile_cols(shape) / 2), g = group_count(shape);
        const double us = begin_us(shape) + step_us(shape) * steps * (double)((n + g - 1) / g);
        if (shape == SINGLE || us < least) best = shape, least = us;
    }
    return best;
}

// workspace: dg, du, the counters, the partial sums
struct FfSpace { int64_t du, count, partial, bytes; };

FfSpace space_of(const FfPlan& p, int rows, int ff) {
    FfSpace s;
    s.du = (int64_t)rows * up64(ff) * 2;
    s.count = 2 * s.du;
    s.partial = (s.count + p.counts * 4 + 15) / 16 * 16;
    s.bytes = s.partial + p.partial_floats * 4;
    return s;
}

bool map_operand(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int dtype, int box) {
    return scao_tensor_map_2d(m, dtype, base, rows, cols, ld, 64, box);
}
bool map_result(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int dtype) {
    return scao_tensor_map_2d(m, dtype, base, rows, cols, cols, 64, 32);
}

// Host word that the kernels write when a wait runs out and that the next call
// reads, without a copy or a synchronisation.  Allocated at the first call, which
// may be inside a stream capture: hence the relaxed mode for this thread.
int* status_word() {
    static std::mutex mu;
    static int* word = nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!word) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        void* p = nullptr;
        if (cudaHostAlloc(&p, 64, cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
            memset(p, 0, 64);
            word = (int*)p;
        }
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
        (void)cudaGetLastError();
    }
    return word;
}

int take_status() {
    int* w = status_word();
    if (!w) return SCAO_ERR_LAUNCH;
    return __atomic_exchange_n(w, 0, __ATOMIC_RELAXED) ? SCAO_ERR_TIMEOUT : SCAO_OK;
}

template <int ACT, bool BF16>
int launch_skinny(const ScaoGatedFf* f, cudaStream_t st) {
    const int groups = (f->rows + 7) / 8, nt = groups <= 2 ? groups : groups <= 4 ? 4 : 8;
    const int fg = nt > 2 ? 2 : 1, blocks = up(f->ff, 8 * fg);
    auto* kernel = nt == 1   ? ff_skinny_kernel<ACT, BF16, 1, 1>
                   : nt == 2 ? ff_skinny_kernel<ACT, BF16, 2, 1>
                   : nt == 4 ? ff_skinny_kernel<ACT, BF16, 4, 2> : ff_skinny_kernel<ACT, BF16, 8, 2>;
    // Warps that share a contraction: 4 fill the SMs where the columns are many (8192 columns
    // of 2048: 14.1 us, with 8 15.8), more where they are few (1000 of 2048: 7.2 us with 4, 4.7
    // with 8), as far as the contraction gives each a step.
    const int step = nt == 1 ? 128 : nt <= 4 ? 64 : 32, most = nt <= 2 ? 16 : 8;
    int warps = 4;
    while (warps < most && 2 * warps * blocks <= 24 * scao_sm_count() && warps * step < f->d) warps *= 2;
    ProfScope p(SLOT_GATED_FF, st);
    kernel<<<blocks, 32 * warps, (size_t)warps * nt * 4 * 32 * sizeof(float), st>>>(
        (const uint16_t*)f->x, f->ldx, (const uint16_t*)f->w_gate, f->ldg, (const uint16_t*)f->w_up, f->ldu,
        (uint16_t*)f->h, f->rows, f->d, f->ff);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
}

template <int ACT>
int launch_skinny(const ScaoGatedFf* f, cudaStream_t st) {
    return f->dtype == SCAO_BF16 ? launch_skinny<ACT, true>(f, st) : launch_skinny<ACT, false>(f, st);
}

bool aligned(const void* p, int64_t ld) { return p && ((uintptr_t)p & 15) == 0 && ld > 0 && (ld & 7) == 0; }

// how a product's packed results (one, or two) are stored
void set_store(FfWork& w, void* a, void* b) {
    w.outp[0] = a;
    w.outp[1] = b;
    const uintptr_t bits = (uintptr_t)a | (uintptr_t)b | (uintptr_t)(w.ldo * 2);
    w.tma_out = (bits & 15) == 0;
    w.vec = (bits & 7) == 0 ? 4 : (bits & 3) == 0 ? 2 : 1;
}

// x, Wg, Wu as TMA reads them
bool operands_ok(const ScaoGatedFf* f) {
    return f && f->rows >= 0 && f->d > 0 && f->ff > 0 && (f->dtype == SCAO_BF16 || f->dtype == SCAO_F16) &&
           f->act >= SCAO_ACT_SILU && f->act <= SCAO_ACT_GELU_TANH &&
           (f->rows == 0 || aligned(f->x, f->ldx)) && aligned(f->w_gate, f->ldg) && aligned(f->w_up, f->ldu) &&
           f->ldx >= (f->rows ? f->d : 0) && f->ldg >= f->d && f->ldu >= f->d;
}

// 16-bit values at their own alignment
bool even(const void* p) { return ((uintptr_t)p & 1) == 0; }

}  // namespace

extern "C" int* scao_gated_ff_status_word(void) { return status_word(); }

extern "C" int64_t scao_gated_ff_saved_bytes(int rows, int ff) {
    return (int64_t)up(rows, 128) * up(ff, 128) * (2 * SAVED_BLOCK);
}

extern "C" int64_t scao_gated_ff_workspace_bytes(int rows, int d, int ff, int which) {
    if (rows < 1 || d < 1 || ff < 1 || !(which & 3)) return 0;
    return space_of(plan_backward(rows, d, ff, which & 1, which & 2), rows, ff).bytes;
}

extern "C" int scao_gated_ff_plan(int rows, int d, int ff, int which, int32_t* out) {
    if (rows < 1 || d < 1 || ff < 1 || which < 0 || which > 3 || !out) return SCAO_ERR_ARG;
    if (which == 0) {
        out[0] = plan_forward(rows, d, ff);
        const int64_t items = tiles_of(rows, ff, tile_rows(out[0]), tile_cols(out[0]) / 2);
        if (items > 1 << 30) return SCAO_ERR_ARG;
        out[1] = (int32_t)items;
        out[2] = out[3] = 1;
    } else {
        const FfPlan& p = plan_backward(rows, d, ff, which & 1, which & 2);
        if (p.us < 0) return SCAO_ERR_ARG;
        out[0] = p.shape;
        out[1] = p.dx_items + p.dw_items;
        out[2] = p.dx.splits;
        out[3] = p.dw.splits;
    }
    out[4] = group_count(out[0]);
    return SCAO_OK;
}

extern "C" int scao_gated_ff_pack(const int64_t* table, int n, void* stream) {
    if (!table || n < 1 || n > 3) return SCAO_ERR_ARG;
    FfPack P;
    memset(&P, 0, sizeof(P));
    int64_t all = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t *t = table + 5 * i, rows = t[2], cols = t[3];
        if (!t[0] || !t[1] || (t[0] & 1) || (t[1] & 15) || rows < 1 || cols < 1 || rows > 0x7fffffff ||
            cols > 1 << 24 || t[4] < 0)
            return SCAO_ERR_ARG;
        P.src[i] = (const uint16_t*)t[0];
        P.dst[i] = (uint16_t*)t[1];
        P.rows[i] = (int)rows;
        P.cols[i] = (int)cols;
        P.pitch[i] = t[4];
        all += P.vecs[i] = rows * ((cols + 63) / 64 * 8);
    }
    P.n = n;
    if ((all + 255) / 256 > 0x7fffffff) return SCAO_ERR_ARG;
    const cudaStream_t st = (cudaStream_t)stream;
    ProfScope p(SLOT_GATED_FF, st);
    ff_pack_kernel<<<(unsigned)((all + 255) / 256), 256, 0, st>>>(P);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
}

extern "C" int scao_gated_ff_forward(const ScaoGatedFf* f, void* stream) {
    if (!operands_ok(f)) return SCAO_ERR_ARG;
    if (f->rows == 0) return SCAO_OK;
    if (!f->h || !even(f->h) || ((uintptr_t)f->saved & 15)) return SCAO_ERR_ARG;
    if (int rc = take_status()) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    if (!f->saved && plan_skinny(f->rows, f->d, f->ff)) {
        if (f->act == SCAO_ACT_SILU) return launch_skinny<SCAO_ACT_SILU>(f, st);
        if (f->act == SCAO_ACT_GELU) return launch_skinny<SCAO_ACT_GELU>(f, st);
        return launch_skinny<SCAO_ACT_GELU_TANH>(f, st);
    }
    FfGemm G;
    memset(&G, 0, sizeof(G));
    const int shape = plan_forward(f->rows, f->d, f->ff), box = shape == SINGLE ? 64 : 128;
    FfWork& w = G.work[0];
    w.mode = FF_FORWARD;
    w.mt = up(f->rows, tile_rows(shape));
    w.nt = up(f->ff, tile_cols(shape) / 2);
    w.parts = w.splits = G.work[1].splits = 1;
    w.steps = up(f->d, 64);
    w.rows = f->rows;
    w.cols = f->ff;
    w.ldo = f->ff;
    set_store(w, f->h, f->h);
    const int64_t items = (int64_t)w.mt * w.nt;
    if (items > 1 << 30) return SCAO_ERR_ARG;
    if (!map_operand(&G.x, f->x, f->rows, f->d, f->ldx, f->dtype, 128) ||
        !map_operand(&G.w[0], f->w_gate, f->ff, f->d, f->ldg, f->dtype, box) ||
        !map_operand(&G.w[1], f->w_up, f->ff, f->d, f->ldu, f->dtype, box) ||
        (w.tma_out && !map_result(&G.out[0], f->h, f->rows, f->ff, f->dtype)))
        return SCAO_ERR_LAUNCH;
    G.saved = (unsigned char*)f->saved;
    G.status = status_word();
    G.dtype = f->dtype;
    const int n = (int)items;
    if (f->act == SCAO_ACT_SILU) return launch_gemm<true, SCAO_ACT_SILU>(shape, G, n, st);
    if (f->act == SCAO_ACT_GELU) return launch_gemm<true, SCAO_ACT_GELU>(shape, G, n, st);
    return launch_gemm<true, SCAO_ACT_GELU_TANH>(shape, G, n, st);
}

extern "C" int scao_gated_ff_backward(const ScaoGatedFf* f, void* stream) {
    if (!operands_ok(f) || f->rows == 0 || !f->saved || !f->dh || f->lddh < 0 || !f->workspace ||
        ((uintptr_t)f->workspace & 15) || ((uintptr_t)f->saved & 15) || !even(f->dh) || !even(f->dx) ||
        !even(f->dw_gate) || !even(f->dw_up) || (!f->dw_gate != !f->dw_up))
        return SCAO_ERR_ARG;
    if (int rc = take_status()) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool want_dx = f->dx != nullptr, want_dw = f->dw_gate != nullptr;
    if (!want_dx && !want_dw) return SCAO_OK;
    FfPlan p = plan_backward(f->rows, f->d, f->ff, want_dx, want_dw);
    if (p.us < 0) return SCAO_ERR_ARG;
    const FfSpace space = space_of(p, f->rows, f->ff);
    const int64_t ld = up64(f->ff);
    char* ws = (char*)f->workspace;
    uint16_t *dg = (uint16_t*)ws, *du = (uint16_t*)(ws + space.du);
    {
        const int vec = ((uintptr_t)f->dh & 15) == 0 && (f->lddh & 7) == 0 && (f->ff & 7) == 0;
        ProfScope prof(SLOT_GATED_FF, st);
        auto* kernel = f->act == SCAO_ACT_SILU   ? ff_pointwise_kernel<SCAO_ACT_SILU>
                       : f->act == SCAO_ACT_GELU ? ff_pointwise_kernel<SCAO_ACT_GELU>
                                                 : ff_pointwise_kernel<SCAO_ACT_GELU_TANH>;
        // rows of a block: 128, fewer where that would leave SMs without one
        int span = 128;
        while (span > 32 && (int64_t)up(f->rows, span) * up(f->ff, 128) < 4 * scao_sm_count()) span >>= 1;
        const int across = up(f->ff, 128);
        kernel<<<dim3(up(f->rows, span), across < 65535 ? across : 65535), PT, 0, st>>>(
            (const unsigned char*)f->saved, (const uint16_t*)f->dh, f->lddh, dg, du, ld, f->rows, f->ff, f->dtype, vec,
            span, (int*)(ws + space.count), (int)p.counts);
        SCAO_CHECK_LAUNCH();
    }
    FfGemm G;
    memset(&G, 0, sizeof(G));
    G.status = status_word();
    G.dtype = f->dtype;
    G.count = (int*)(ws + space.count);
    G.partial = (float*)(ws + space.partial);
    if (want_dx) {
        if (!map_operand(&G.w[0], f->w_gate, f->ff, f->d, f->ldg, f->dtype, 64) ||
            !map_operand(&G.w[1], f->w_up, f->ff, f->d, f->ldu, f->dtype, 64) ||
            !map_operand(&G.dguk[0], dg, f->rows, f->ff, ld, f->dtype, 128) ||
            !map_operand(&G.dguk[1], du, f->rows, f->ff, ld, f->dtype, 128))
            return SCAO_ERR_LAUNCH;
        set_store(p.dx, f->dx, f->dx);
        if (p.dx.tma_out && !map_result(&G.out[0], f->dx, f->rows, f->d, f->dtype)) return SCAO_ERR_LAUNCH;
    }
    if (want_dw) {
        if (!map_operand(&G.x, f->x, f->rows, f->d, f->ldx, f->dtype, 64) ||
            !map_operand(&G.dgum[0], dg, f->rows, f->ff, ld, f->dtype, 64) ||
            !map_operand(&G.dgum[1], du, f->rows, f->ff, ld, f->dtype, 64))
            return SCAO_ERR_LAUNCH;
        set_store(p.dw, f->dw_gate, f->dw_up);
        if (p.dw.tma_out && (!map_result(&G.out[1], f->dw_gate, f->ff, f->d, f->dtype) ||
                             !map_result(&G.out[2], f->dw_up, f->ff, f->d, f->dtype)))
            return SCAO_ERR_LAUNCH;
    }
    G.work[0] = p.dx_first ? p.dx : p.dw;
    G.work[1] = p.dx_first ? p.dw : p.dx;
    G.extra = p.extra;
    return launch_gemm<false, 0>(p.shape, G, p.dx_items + p.dw_items, st);
}
