// Gated feed-forward product and its gradient, bf16 / fp16 with 32-bit sums:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u          x: M x d; Wg, Wu: F x d
//   dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Three products on one persistent, warp-specialised kernel (ff_gemm_kernel) on
// SM pairs, with tcgen05.mma.cta_group::2 tiles of 256 x 256 and both operands by
// TMA; each CTA stages its 128 rows of A and 128 of B.
//   forward    B is 128 rows of Wg (from the pair's first CTA) and the same 128 of
//              Wu (from the second), so a thread of the epilogue finds the gate and
//              the up value of one place in its own TMEM row: activation and product
//              happen there and h leaves through a TMA store.
//   dx         contraction over F of dg with Wg, then of du with Wu, into one
//              accumulator; the weights are read MN-major as they lie.
//   dW         dg^T x and du^T x over the rows, both operands MN-major: nothing is
//              transposed in memory.
// The pointwise part of the gradient (ff_pointwise_kernel) reads g and u as the
// forward pass kept them, in 32 bits: rounding them to 16 as well would add their
// rounding to those of dg, du (16 bits: they are operands of the tensor cores)
// and of the result, and put the gradients' error at 1.8 instead of 1.4 roundings.
#include <cuda.h>
#include <string.h>

#include <mutex>

#include "common.cuh"
#include "prof.cuh"
#include "tc.cuh"
#include "tmap.cuh"

namespace {

enum { FF_FORWARD = 0, FF_DX, FF_DW };

constexpr int FN = 256;                     // accumulator columns of a tile
constexpr int FST = 6;                      // pipeline stages
constexpr uint32_t FOPB = 128 * 64 * 2;     // one 128 x 64 operand block, 16 KB
constexpr uint32_t FSTAGE = 2 * FOPB;
constexpr int FEPI_WARPS = 8;
constexpr uint32_t FOUTB = 32 * 64 * 2;     // a warp's 32 x 64 block of the result, 4 KB
constexpr int FTHREADS = 64 + 32 * FEPI_WARPS;
constexpr int FBAND = 16;                   // row blocks per band of the tile order
constexpr size_t FSMEM = 1024 + (size_t)FST * FSTAGE + FEPI_WARPS * FOUTB;
static_assert(FSMEM <= 231 * 1024, "shared memory");

struct FfGemm {
    CUtensorMap a[2], b[2], out[2];
    void* outp[2];                          // the results, for the stores without TMA
    float* saved;                           // forward: g and u for the gradient, or null
    int* status;
    int64_t ldo;                            // row pitch of the results (values)
    int rows, cols;                         // of one result
    int mt, nt, parts;                      // row and column tiles; results (dW: 2)
    int ksteps, segs;                       // 64-deep steps of one segment; segments (dx: 2)
    int dtype, tma_out;
};

struct FfTile { int part, m, n; };          // result, row tile, column tile

// tiles in bands of FBAND row blocks, row blocks fastest: the tiles that run at
// one time share few operand panels, which stay in L2
__device__ __forceinline__ FfTile ff_tile(const FfGemm& G, int T) {
    FfTile w;
    const int per = G.mt * G.nt;
    w.part = T / per;
    int t = T - w.part * per;
    const int band = t / (FBAND * G.nt);
    t -= band * FBAND * G.nt;
    const int h = min(FBAND, G.mt - band * FBAND);
    w.n = t / h;
    w.m = band * FBAND + t - w.n * h;
    return w;
}

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
        d = s + g * s * (1.f - s) * 2.f * TANH_A * (1.f + 3.f * TANH_B * g * g);
    }
}

SCAO_DEV uint32_t pack2(float a, float b, int dt) {
    if (dt == SCAO_BF16) return (uint32_t)f_to_bf16_bits(a) | ((uint32_t)f_to_bf16_bits(b) << 16);
    return (uint32_t)f_to_f16_bits(a) | ((uint32_t)f_to_f16_bits(b) << 16);
}

// g and u as kept for the gradient: per 128-row x 128-column block the g values,
// then the u values, as [4-column group][row][4], so that a warp (a thread per row)
// writes 512 consecutive bytes.
SCAO_DEV int64_t saved_off(int row, int col, int col_blocks) {
    return ((int64_t)(row >> 7) * col_blocks + (col >> 7)) * (2 * 128 * 128) +
           (((col & 127) >> 2) * 128 + (row & 127)) * 4;
}
constexpr int SAVED_U = 128 * 128;

SCAO_DEV void ff_fail(int* status) { *(volatile int*)status = 2; }

// One warp's 32 x 64 block of a result, 16-bit values in `v` (32 pairs of this
// thread's row): through shared memory, then a TMA store or guarded stores.
SCAO_DEV void ff_store_block(const FfGemm& G, int part, const uint32_t* v, unsigned char* stage,
                             int row0, int col0, int lane) {
    if (lane == 0) bulk_wait_read0();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c)
        *(uint4*)(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) =
            make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    if (G.tma_out) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (row0 < G.rows && col0 < G.cols) tma_store_2d(&G.out[part], col0, row0, smem_u32(stage));
            bulk_commit();
        }
        return;
    }
    __syncwarp();
    for (int r = 0; r < 32 && row0 + r < G.rows; ++r) {
        uint16_t* dst = (uint16_t*)G.outp[part] + (int64_t)(row0 + r) * G.ldo;
#pragma unroll
        for (int c = lane; c < 64; c += 32)
            if (col0 + c < G.cols)
                dst[col0 + c] = *(const uint16_t*)(stage + r * 128 + (((c >> 3) ^ (r & 7)) * 16) + (c & 7) * 2);
    }
    __syncwarp();
}

// Roles per CTA: warp 0 TMA producer; warp 1 TMEM owner and (first CTA of the pair)
// MMA issuer; warps 2-9 epilogue, which overlaps the next tile's main loop (two
// accumulators).  Every wait is bounded; when one runs out the CTA records it in
// *status, issues no more, waits for its copies in flight and both CTAs still meet
// at the end.
template <int MODE, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(FTHREADS, 1)
ff_gemm_kernel(const __grid_constant__ FfGemm G) {
    extern __shared__ unsigned char raw[];
    unsigned char* sm = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[FST], empty[FST], accf[2], acce[2], fin;
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    if (tid == 0) {
        for (int i = 0; i < FST; ++i) { mbar_init(&full[i], 2); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&accf[i], 1); mbar_init(&acce[i], 2 * FEPI_WARPS); }
        mbar_init(&fin, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tc_alloc_pair(&tslot, 2 * FN);
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tslot;
    const int total = G.parts * G.mt * G.nt;
    const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
    const int steps = G.ksteps * G.segs;
    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t ph = 0, issued = 0, last_ph = 0;
            for (int T = cid; T < total && !abort_flag; T += ncl) {
                const FfTile w = ff_tile(G, T);
                const int i0 = w.m * 256 + 128 * (int)rank;
                const int j0 = MODE == FF_FORWARD ? w.n * 128 : w.n * FN + 128 * (int)rank;
                for (int s = 0; s < steps; ++s) {
                    if (!mbar_wait(&empty[stage], ph ^ 1)) { abort_flag = 1; ff_fail(G.status); break; }
                    const uint32_t fb = mapa_shared(smem_u32(&full[stage]), 0);
                    mbar_arrive_expect_tx_cl(fb, FSTAGE);
                    const uint32_t a = smem_u32(sm + (size_t)stage * FSTAGE), b = a + FOPB;
                    if (MODE == FF_FORWARD) {
                        tma_load_2d_pair(a, &G.a[0], s * 64, i0, fb);
                        tma_load_2d_pair(b, &G.b[rank], s * 64, j0, fb);
                    } else if (MODE == FF_DX) {
                        const int g = s >= G.ksteps, k0 = (s - g * G.ksteps) * 64;
                        tma_load_2d_pair(a, &G.a[g], k0, i0, fb);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            tma_load_2d_pair(b + h * (FOPB / 2), &G.b[g], j0 + 64 * h, k0, fb);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tma_load_2d_pair(a + h * (FOPB / 2), &G.a[w.part], i0 + 64 * h, s * 64, fb);
                            tma_load_2d_pair(b + h * (FOPB / 2), &G.b[0], j0 + 64 * h, s * 64, fb);
                        }
                    }
                    issued |= 1u << stage;
                    last_ph = (last_ph & ~(1u << stage)) | (ph << stage);
                    if (++stage == FST) { stage = 0; ph ^= 1; }
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
            constexpr int AMN = MODE == FF_DW, BMN = MODE != FF_FORWARD;
            uint32_t idesc = idesc_bf16(256, FN, AMN, BMN);
            if (G.dtype == SCAO_F16) idesc &= ~((1u << 7) | (1u << 10));
            int stage = 0, acc = 0;
            uint32_t ph = 0, aph = 0;
            for (int T = cid; T < total && !abort_flag; T += ncl) {
                if (!mbar_wait(&acce[acc], aph ^ 1)) { abort_flag = 1; ff_fail(G.status); break; }
                tc_fence_after();
                const uint32_t d = tmem + acc * FN;
                bool ok = true;
                for (int s = 0; s < steps; ++s) {
                    if (!mbar_wait(&full[stage], ph)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a = smem_u32(sm + (size_t)stage * FSTAGE), b = a + FOPB;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // 16 deep: 32 bytes along a K-major row, 2 KB of MN-major rows
                        const uint64_t ad = AMN ? smem_desc_sw128(a + k * 2048, FOPB / 2, 1024)
                                                : smem_desc_sw128(a + k * 32, 16, 1024);
                        const uint64_t bd = BMN ? smem_desc_sw128(b + k * 2048, FOPB / 2, 1024)
                                                : smem_desc_sw128(b + k * 32, 16, 1024);
                        tc_mma_bf16_pair(d, ad, bd, idesc, (s > 0 || k > 0) ? 1u : 0u);
                    }
                    tc_commit_pair(&empty[stage], 0x3);
                    if (++stage == FST) { stage = 0; ph ^= 1; }
                }
                if (!ok) { abort_flag = 1; ff_fail(G.status); break; }
                tc_commit_pair(&accf[acc], 0x3);
                acc ^= 1;
                if (acc == 0) aph ^= 1;
            }
            tc_commit_pair(&fin, 0x3);
        }
        __syncwarp();
        if (!mbar_wait(&fin, 0)) ff_fail(G.status);
    } else {
        const int q = warp & 3, h = (warp - 2) >> 2;     // TMEM lane quarter, column half
        unsigned char* stage = sm + (size_t)FST * FSTAGE + (warp - 2) * FOUTB;
        const uint32_t acce_cl[2] = {mapa_shared(smem_u32(&acce[0]), 0),
                                     mapa_shared(smem_u32(&acce[1]), 0)};
        int acc = 0;
        uint32_t aph = 0;
        for (int T = cid; T < total; T += ncl) {
            if (__any_sync(0xffffffffu, abort_flag)) break;
            const FfTile w = ff_tile(G, T);
            if (!__all_sync(0xffffffffu, mbar_wait(&accf[acc], aph))) {
                abort_flag = 1;
                ff_fail(G.status);
                break;
            }
            tc_fence_after();
            const int row0 = w.m * 256 + 128 * (int)rank + q * 32, row = row0 + lane;
            const uint32_t tb = tmem + acc * FN + ((uint32_t)(q * 32) << 16);
            if (MODE == FF_FORWARD) {
                const int c0 = w.n * 128 + h * 64, cb = (G.cols + 127) >> 7;
                uint32_t out[32], gr[2][16], ur[2][16];
                tc_ld16_async(tb + h * 64, gr[0]);
                tc_ld16_async(tb + 128 + h * 64, ur[0]);
#pragma unroll
                for (int c = 0; c < 64; c += 16) {      // the next 16 columns are on their way
                    uint32_t *g = gr[(c >> 4) & 1], *u = ur[(c >> 4) & 1];
                    tc_ld16_wait(g);
                    tc_ld16_wait(u);
                    if (c + 16 < 64) {
                        tc_ld16_async(tb + h * 64 + c + 16, gr[((c >> 4) + 1) & 1]);
                        tc_ld16_async(tb + 128 + h * 64 + c + 16, ur[((c >> 4) + 1) & 1]);
                    }
                    if (G.saved && row < G.rows && c0 + c < G.cols) {
                        float* p = G.saved + saved_off(row, c0 + c, cb);
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            *(uint4*)(p + i * 128) = make_uint4(g[i], g[i + 1], g[i + 2], g[i + 3]);
                            *(uint4*)(p + SAVED_U + i * 128) = make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]);
                        }
                    }
                    float y[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        y[i] = ff_act<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) out[(c + i) / 2] = pack2(y[i], y[i + 1], G.dtype);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cl(acce_cl[acc]);
                ff_store_block(G, 0, out, stage, row0, c0, lane);
            } else {
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    const int c0 = h * 128 + half * 64;
                    uint32_t out[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        float v[16];
                        tc_ld16(tb + c0 + c, v);
#pragma unroll
                        for (int i = 0; i < 16; i += 2) out[(c + i) / 2] = pack2(v[i], v[i + 1], G.dtype);
                    }
                    if (half == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cl(acce_cl[acc]);
                    }
                    ff_store_block(G, w.part, out, stage, row0, w.n * FN + c0, lane);
                }
            }
            acc ^= 1;
            if (acc == 0) aph ^= 1;
        }
        if (lane == 0) bulk_wait0();        // the stores have left shared memory and are visible
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) tc_dealloc_pair(tmem, 2 * FN);
}

// dg = dh u act'(g), du = dh act(g).  A warp takes 4 rows x 32 columns at a time:
// runs of 64 bytes and more of every array.  HBM bound (14 bytes a value).
constexpr int PT = 256;

template <int ACT>
__global__ void __launch_bounds__(PT)
ff_pointwise_kernel(const float* __restrict__ saved, const uint16_t* __restrict__ dh, int64_t lddh,
                    uint16_t* __restrict__ dg, uint16_t* __restrict__ du, int64_t ldg, int rows,
                    int cols, int dtype, int vec) {
    const int cb = (cols + 127) >> 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.y * 128 + (warp & 3) * 32 + (lane & 7) * 4;
    if (c >= cols) return;
    const int r0 = blockIdx.x * 128 + (warp >> 2) * 64 + (lane >> 3);
#pragma unroll 1
    for (int i = 0; i < 16; i += 4) {
        if (r0 + 4 * i >= rows) break;
        float4 g[4], u[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {                   // all loads first
            const int r = min(r0 + 4 * (i + k), rows - 1);
            const float* p = saved + saved_off(r, c, cb);
            g[k] = ldg_stream4(p);
            u[k] = ldg_stream4(p + SAVED_U);
            const uint16_t* d = dh + r * lddh + c;
            if (vec) {
                y[k] = load4_dt(d, 0, dtype);
            } else {
                y[k].x = load_dt(d, 0, dtype);
                y[k].y = c + 1 < cols ? load_dt(d, 1, dtype) : 0.f;
                y[k].z = c + 2 < cols ? load_dt(d, 2, dtype) : 0.f;
                y[k].w = c + 3 < cols ? load_dt(d, 3, dtype) : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + 4 * (i + k);
            if (r >= rows) break;
            float4 a, b;
            ff_act_grad<ACT>(g[k].x, a.x, b.x);
            ff_act_grad<ACT>(g[k].y, a.y, b.y);
            ff_act_grad<ACT>(g[k].z, a.z, b.z);
            ff_act_grad<ACT>(g[k].w, a.w, b.w);
            const float4 d = y[k];
            // the pitch of dg and du is a multiple of 8: the last group may write past
            // `cols` within it, where the products read nothing
            store4_dt(du + r * ldg + c, 0, dtype, make_float4(d.x * a.x, d.y * a.y, d.z * a.z, d.w * a.w));
            store4_dt(dg + r * ldg + c, 0, dtype,
                      make_float4(d.x * u[k].x * b.x, d.y * u[k].y * b.y, d.z * u[k].z * b.z,
                                  d.w * u[k].w * b.w));
        }
    }
}

// Few rows (at most SK_ROWS): the time is one reading of the weights, so no tile
// waits for a whole operand block.  A warp takes 8 inner columns: the 16 rows of an
// mma.m16n8k16 A operand are their 8 gate and 8 up weight rows, loaded straight
// from global memory into the registers that the instruction reads (a contraction
// may take its terms in any order, so a lane's 16 consecutive bytes serve as the
// k places of two instructions, in x as in the weights).  Gate and up of one place
// meet in one thread.  The block's warps share a row's contraction and join in
// shared memory in a fixed order.
constexpr int SK_WARPS = 8;
constexpr int SK_ROWS = 32;

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

template <int ACT, bool BF16, int NT>
__global__ void __launch_bounds__(32 * SK_WARPS)
ff_skinny_kernel(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ wg, int64_t ldg,
                 const uint16_t* __restrict__ wu, int64_t ldu, uint16_t* __restrict__ h, int rows, int d,
                 int ff) {
    constexpr int U = NT == 1 ? 4 : 2;          // 32-deep steps in flight
    __shared__ float part[SK_WARPS][NT * 4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int f = blockIdx.x * 8 + g;
    const bool has = f < ff;
    const uint16_t* pg = wg + (int64_t)min(f, ff - 1) * ldg;
    const uint16_t* pu = wu + (int64_t)min(f, ff - 1) * ldu;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    for (int k0 = warp * 32 * U; k0 < d; k0 += SK_WARPS * 32 * U) {
        uint4 a[U], b[U], v[NT][U];
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const int k = k0 + 32 * s + 8 * t;
            a[s] = load8_guard(pg + k, d - k);
            b[s] = load8_guard(pu + k, d - k);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = n * 8 + g;
                v[n][s] = load8_guard(x + (int64_t)min(r, rows - 1) * ldx + k, r < rows ? d - k : 0);
            }
        }
#pragma unroll
        for (int s = 0; s < U; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma_16816(acc[n], a[s].x, b[s].x, a[s].y, b[s].y, v[n][s].x, v[n][s].y, BF16);
                mma_16816(acc[n], a[s].z, b[s].z, a[s].w, b[s].w, v[n][s].z, v[n][s].w, BF16);
            }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][n * 4 + i][lane] = acc[n][i];
    __syncthreads();
    // thread (n, j): columns 2t + j of row group n, gate in place j and up in 2 + j
    if (warp < NT) {
        const int n = warp;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float gate = 0.f, upv = 0.f;
#pragma unroll
            for (int w = 0; w < SK_WARPS; ++w) {
                gate += part[w][n * 4 + j][lane];
                upv += part[w][n * 4 + 2 + j][lane];
            }
            const int r = n * 8 + 2 * t + j;
            if (has && r < rows) {
                const float y = ff_act<ACT>(gate) * upv;
                h[(int64_t)r * ff + f] = BF16 ? f_to_bf16_bits(y) : f_to_f16_bits(y);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
bool map2d(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int dtype, int bx,
           int by) {
    return scao_tensor_map_2d(m, dtype, base, rows, cols, ld, bx, by);
}

template <int MODE, int ACT = 0>
int launch_gemm(FfGemm& G, cudaStream_t st) {
    static PerDeviceOnce once;
    if (once.first() && cudaFuncSetAttribute(ff_gemm_kernel<MODE, ACT>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FSMEM) != cudaSuccess)
        return SCAO_ERR_LAUNCH;
    const int64_t tiles = (int64_t)G.parts * G.mt * G.nt;
    if (tiles > (1 << 30)) return SCAO_ERR_ARG;
    const int pairs = scao_sm_count() / 2;
    ProfScope p(SLOT_GATED_FF, st);
    ff_gemm_kernel<MODE, ACT><<<2 * (int)(tiles < pairs ? tiles : pairs), FTHREADS, FSMEM, st>>>(G);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
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
    const int nt = (f->rows + 7) / 8;
    auto* kernel = nt == 1 ? ff_skinny_kernel<ACT, BF16, 1>
                   : nt == 2 ? ff_skinny_kernel<ACT, BF16, 2> : ff_skinny_kernel<ACT, BF16, 4>;
    ProfScope p(SLOT_GATED_FF, st);
    kernel<<<(f->ff + 7) / 8, 32 * SK_WARPS, 0, st>>>(
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

// x, Wg, Wu as TMA reads them
bool operands_ok(const ScaoGatedFf* f) {
    return f && f->rows >= 0 && f->d > 0 && f->ff > 0 && (f->dtype == SCAO_BF16 || f->dtype == SCAO_F16) &&
           f->act >= SCAO_ACT_SILU && f->act <= SCAO_ACT_GELU_TANH &&
           (f->rows == 0 || aligned(f->x, f->ldx)) && aligned(f->w_gate, f->ldg) && aligned(f->w_up, f->ldu) &&
           f->ldx >= (f->rows ? f->d : 0) && f->ldg >= f->d && f->ldu >= f->d;
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
int up(int64_t n, int k) { return (int)((n + k - 1) / k); }

}  // namespace

extern "C" int* scao_gated_ff_status_word(void) { return status_word(); }

extern "C" int64_t scao_gated_ff_saved_bytes(int rows, int ff) {
    return (int64_t)up(rows, 128) * up(ff, 128) * (2 * 128 * 128) * (int64_t)sizeof(float);
}

extern "C" int64_t scao_gated_ff_workspace_bytes(int rows, int d, int ff) {
    (void)d;
    return 2 * (int64_t)rows * up8(ff) * 2 + 16;
}

extern "C" int scao_gated_ff_forward(const ScaoGatedFf* f, void* stream) {
    if (!operands_ok(f)) return SCAO_ERR_ARG;
    if (f->rows == 0) return SCAO_OK;
    if (!f->h) return SCAO_ERR_ARG;
    if (int rc = take_status()) return rc;
    if (!f->saved && f->rows <= SK_ROWS) {
        const cudaStream_t st = (cudaStream_t)stream;
        if (f->act == SCAO_ACT_SILU) return launch_skinny<SCAO_ACT_SILU>(f, st);
        if (f->act == SCAO_ACT_GELU) return launch_skinny<SCAO_ACT_GELU>(f, st);
        return launch_skinny<SCAO_ACT_GELU_TANH>(f, st);
    }
    FfGemm G;
    memset(&G, 0, sizeof(G));
    G.tma_out = aligned(f->h, f->ff);
    if (!map2d(&G.a[0], f->x, f->rows, f->d, f->ldx, f->dtype, 64, 128) ||
        !map2d(&G.b[0], f->w_gate, f->ff, f->d, f->ldg, f->dtype, 64, 128) ||
        !map2d(&G.b[1], f->w_up, f->ff, f->d, f->ldu, f->dtype, 64, 128) ||
        (G.tma_out && !map2d(&G.out[0], f->h, f->rows, f->ff, f->ff, f->dtype, 64, 32)))
        return SCAO_ERR_LAUNCH;
    G.outp[0] = f->h;
    G.saved = (float*)f->saved;
    G.status = status_word();
    G.ldo = f->ff;
    G.rows = f->rows;
    G.cols = f->ff;
    G.mt = up(f->rows, 256);
    G.nt = up(f->ff, 128);
    G.parts = G.segs = 1;
    G.ksteps = up(f->d, 64);
    G.dtype = f->dtype;
    const cudaStream_t st = (cudaStream_t)stream;
    if (f->act == SCAO_ACT_SILU) return launch_gemm<FF_FORWARD, SCAO_ACT_SILU>(G, st);
    if (f->act == SCAO_ACT_GELU) return launch_gemm<FF_FORWARD, SCAO_ACT_GELU>(G, st);
    return launch_gemm<FF_FORWARD, SCAO_ACT_GELU_TANH>(G, st);
}

extern "C" int scao_gated_ff_backward(const ScaoGatedFf* f, void* stream) {
    if (!operands_ok(f) || f->rows == 0 || !f->saved || !f->dh || f->lddh < 0 || !f->workspace ||
        ((uintptr_t)f->workspace & 15) || (!f->dw_gate != !f->dw_up))
        return SCAO_ERR_ARG;
    if (int rc = take_status()) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    const int64_t ld = up8(f->ff);
    uint16_t *dg = (uint16_t*)f->workspace, *du = dg + f->rows * ld;
    {
        const int vec = ((uintptr_t)f->dh & 7) == 0 && (f->lddh & 3) == 0 && (f->ff & 3) == 0;
        if (up(f->ff, 128) > 65535) return SCAO_ERR_ARG;
        ProfScope p(SLOT_GATED_FF, st);
        auto* kernel = f->act == SCAO_ACT_SILU   ? ff_pointwise_kernel<SCAO_ACT_SILU>
                       : f->act == SCAO_ACT_GELU ? ff_pointwise_kernel<SCAO_ACT_GELU>
                                                 : ff_pointwise_kernel<SCAO_ACT_GELU_TANH>;
        kernel<<<dim3(up(f->rows, 128), up(f->ff, 128)), PT, 0, st>>>(
            (const float*)f->saved, (const uint16_t*)f->dh, f->lddh, dg, du, ld, f->rows, f->ff, f->dtype, vec);
        SCAO_CHECK_LAUNCH();
    }
    FfGemm G;
    memset(&G, 0, sizeof(G));
    G.status = status_word();
    G.dtype = f->dtype;
    G.ldo = G.cols = f->d;
    G.nt = up(f->d, FN);
    if (f->dx) {
        G.tma_out = aligned(f->dx, f->d);
        if (!map2d(&G.a[0], dg, f->rows, f->ff, ld, f->dtype, 64, 128) ||
            !map2d(&G.a[1], du, f->rows, f->ff, ld, f->dtype, 64, 128) ||
            !map2d(&G.b[0], f->w_gate, f->ff, f->d, f->ldg, f->dtype, 64, 64) ||
            !map2d(&G.b[1], f->w_up, f->ff, f->d, f->ldu, f->dtype, 64, 64) ||
            (G.tma_out && !map2d(&G.out[0], f->dx, f->rows, f->d, f->d, f->dtype, 64, 32)))
            return SCAO_ERR_LAUNCH;
        G.outp[0] = f->dx;
        G.rows = f->rows;
        G.mt = up(f->rows, 256);
        G.parts = 1;
        G.segs = 2;
        G.ksteps = up(f->ff, 64);
        if (int rc = launch_gemm<FF_DX>(G, st)) return rc;
    }
    if (f->dw_gate) {
        G.tma_out = aligned(f->dw_gate, f->d) && aligned(f->dw_up, f->d);
        if (!map2d(&G.a[0], dg, f->rows, f->ff, ld, f->dtype, 64, 64) ||
            !map2d(&G.a[1], du, f->rows, f->ff, ld, f->dtype, 64, 64) ||
            !map2d(&G.b[0], f->x, f->rows, f->d, f->ldx, f->dtype, 64, 64) ||
            (G.tma_out && (!map2d(&G.out[0], f->dw_gate, f->ff, f->d, f->d, f->dtype, 64, 32) ||
                           !map2d(&G.out[1], f->dw_up, f->ff, f->d, f->d, f->dtype, 64, 32))))
            return SCAO_ERR_LAUNCH;
        G.outp[0] = f->dw_gate;
        G.outp[1] = f->dw_up;
        G.rows = f->ff;
        G.mt = up(f->ff, 256);
        G.parts = 2;
        G.segs = 1;
        G.ksteps = up(f->rows, 64);
        if (int rc = launch_gemm<FF_DW>(G, st)) return rc;
    }
    return SCAO_OK;
}
