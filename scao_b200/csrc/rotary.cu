// Rotary positions of query and key heads: for pair j of a head at position p
//
//   (y_a, y_b) = m (x_a cos t - x_b sin t,  x_a sin t + x_b cos t),  t = p w_j
//
// with (a, b) = (2j, 2j + 1) or (j, j + dim/2); values beyond dim pass through.
// The gradient is the transposed rotation: the same kernel with -sin.
//
// The angle is formed in turns, as a fixed-point fraction of 64 bits: p times the
// fraction w_j / 2 pi 2^64, of which a 64-bit product keeps what is left when whole turns are
// taken off (in 32-bit floats p w_j / 2 pi of far positions would be off by 1e-2 turns and
// more; doubles would do, at three conversions of a quarter of the rate each).  What it is
// off by is p times the error of the fraction, which comes as a double: at most 2^-55.2
// (w_j <= 1, two roundings of 53 bits, and the cut at 2^-64).  Its upper 32 bits, as a signed
// part of a turn, are rounded to a float for sincospif: 2^-26 of a turn, 1e-7 radian, as
// much as one rounding of a float32 result and nothing beside those of 16-bit types (a
// float32 result is off by 1.3 times what angles rounded only once would leave).  The
// frequencies travel as kernel arguments (dim <= 512: 2 KB), so there is no table in
// memory to keep or to outgrow.
//
// A block takes a few tokens: it forms their cosines and sines once into shared
// memory and applies them to every head of q and of k, each value read and
// written once with the widest vector that the strides allow.  HBM bound: 1 x 30011 x 14
// heads x 80 float32 (64 turned, interleaved) in 48 us, 5.6 TB/s; 2 x 5000 x 40 x 128 bf16 in
// 37 us, 5.5 TB/s.  Where the rows allow wider vectors than their pairs do (halves of an odd
// length, say), rotary_tile_kernel brings whole rows through shared memory.
#include <math.h>

#include "common.cuh"
#include "prof.cuh"
#include "tmap.cuh"

namespace {

constexpr int RT = 256;                 // threads per block, at most
constexpr int RMAX = 256;               // frequencies
constexpr int RTOK = 64;                // tokens per block, at most

struct RotArgs {
    uint64_t turn[RMAX];                // turns per position, of 2^-64
    const void* in[2];
    void* out[2];
    int64_t isb[2], ish[2], ist[2], osb[2], osh[2], ost[2];   // strides in values
    const void* pos;                    // int32 / int64, or null: start + t
    int64_t pos_sb, pos_st, start, tokens;
    int heads[2];
    int pos64, T, D, half, tb;
    int hb;                             // heads per block (rotary_tile_kernel)
    uint32_t inv_half, inv_per;         // of half and (rotary_tile_kernel) of a row's vectors: see small_div
    float cosm, sinm;                   // m and +-m
};
static_assert(sizeof(RotArgs) <= 4096, "kernel arguments");

template <int ES, int N> struct VecOf;
template <> struct VecOf<2, 8> { typedef uint4 type; };
template <> struct VecOf<2, 4> { typedef uint2 type; };
template <> struct VecOf<2, 2> { typedef uint32_t type; };
template <> struct VecOf<2, 1> { typedef uint16_t type; };
template <> struct VecOf<4, 4> { typedef uint4 type; };
template <> struct VecOf<4, 2> { typedef uint2 type; };
template <> struct VecOf<4, 1> { typedef uint32_t type; };

template <int DT> struct ElemOf { typedef uint16_t type; };
template <> struct ElemOf<SCAO_F32> { typedef float type; };

template <int DT>
SCAO_DEV float to_f(typename ElemOf<DT>::type x) {
    if constexpr (DT == SCAO_F32) return x;
    else if constexpr (DT == SCAO_BF16) return bf16_bits_to_f(x);
    else return f16_bits_to_f(x);
}
template <int DT>
SCAO_DEV typename ElemOf<DT>::type from_f(float x) {
    if constexpr (DT == SCAO_F32) return x;
    else if constexpr (DT == SCAO_BF16) return f_to_bf16_bits(x);
    else return f_to_f16_bits(x);
}

// NV values of one memory vector
template <int DT, int NV>
union Pack {
    typename VecOf<sizeof(typename ElemOf<DT>::type), NV>::type v;
    typename ElemOf<DT>::type e[NV];
};

// i / n for i < 2^14, from inv = 2^32 / n rounded up (0 for n = 1)
SCAO_DEV int small_div(int i, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)i, inv) : i; }

// Item of a thread, one of S per head: NV pairs of two vectors (halves apart),
// NV / 2 pairs of one vector (interleaved; one pair where NV is 1), or a
// vector behind the rotated part.  A thread keeps its item and goes over (token, head)
// rows, RROWS at a time with all their loads first; the first rows are on their way
// while the block forms its cosines and sines.
template <int DT, bool INTER, int NV>
__global__ void __launch_bounds__(RT)
rotary_kernel(const __grid_constant__ RotArgs A) {
    typedef typename ElemOf<DT>::type E;
    typedef Pack<DT, NV> V;
    typedef decltype(V::v) Word;
    constexpr bool TWO = !INTER || NV == 1;                       // a rotating item is two vectors
    constexpr int PAIRS = INTER ? (NV > 1 ? NV / 2 : 1) : NV;     // its pairs
    constexpr int RROWS = TWO && sizeof(Word) == 16 ? 2 : 4;
    // m cos, +-m sin of [token][two pairs of an item][item][2]: neighbouring items read
    // neighbouring 16 bytes (by pair, their reads met in the same banks)
    extern __shared__ float4 cs4[];
    float2* cs = (float2*)cs4;
    __shared__ int64_t base[RTOK][5];   // of the token in q, k, the results and the positions
    const int half = A.half, bx = blockDim.x, by = blockDim.y;
    const int64_t tok0 = (int64_t)blockIdx.x * A.tb;
    const int nt = (int)min((int64_t)A.tb, A.tokens - tok0);
    const int tid = threadIdx.y * bx + threadIdx.x, nthr = bx * by;
    if (tid < nt) {
        const int64_t b = (tok0 + tid) / A.T, t = (tok0 + tid) - b * A.T;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            base[tid][i] = b * A.isb[i] + t * A.ist[i];
            base[tid][2 + i] = b * A.osb[i] + t * A.ost[i];
        }
        base[tid][4] = A.pos ? b * A.pos_sb + t * A.pos_st : A.start + t;
    }
    __syncthreads();
    const int rot = half / PAIRS, S = rot + (A.D - 2 * half) / NV;
    const int H0 = A.heads[0], H = H0 + A.heads[1], rows = nt * H;
    const int ob = INTER ? 1 : half;                              // to an item's second vector
    int s = threadIdx.x, r = threadIdx.y, k = 0, h = threadIdx.y; // item; row, its token and head
    V a[RROWS], x2[RROWS];
    E* out[RROWS];
    int tok[RROWS];
    auto load = [&] {
        const bool turns = s < rot;
        const int oa = turns ? (INTER ? 2 : 1) * s * PAIRS : 2 * half + (s - rot) * NV;
#pragma unroll
        for (int u = 0; u < RROWS; ++u) {
            tok[u] = -1;
            if (r < rows) {
                while (h >= H) { h -= H; ++k; }
                const int w = h >= H0, hh = w ? h - H0 : h;
                const E* in = (const E*)A.in[w] + base[k][w] + hh * A.ish[w] + oa;
                out[u] = (E*)A.out[w] + base[k][2 + w] + hh * A.osh[w] + oa;
                a[u].v = *(const Word*)in;
                if (TWO && turns) x2[u].v = *(const Word*)(in + ob);
                tok[u] = k;
            }
            r += by;
            h += by;
        }
    };
    load();
    for (int i = tid; i < nt * half; i += nthr) {
        const int t = small_div(i, A.inv_half), j = i - t * half;
        int64_t p = base[t][4];
        if (A.pos) p = A.pos64 ? ((const int64_t*)A.pos)[p] : (int64_t)((const int32_t*)A.pos)[p];
        const int part = (int)(((uint64_t)p * A.turn[j]) >> 32);      // of a turn, times 2^32
        float sn, c;
        sincospif((float)part * 0x1p-31f, &sn, &c);
        const int item = j / PAIRS, e = j % PAIRS;
        cs[t * half + (PAIRS > 1 ? ((e >> 1) * rot + item) * 2 + (e & 1) : item)] =
            make_float2(A.cosm * c, A.sinm * sn);
    }
    __syncthreads();
    for (;;) {
#pragma unroll
        for (int u = 0; u < RROWS; ++u) {
            if (tok[u] < 0) break;
            if (s >= rot) {
                *(Word*)out[u] = a[u].v;
                continue;
            }
            const float2* c = cs + tok[u] * half;
            V y, y2;
            float4 two;
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) {
                if (PAIRS > 1 && e % 2 == 0) two = *(const float4*)(c + (e / 2 * rot + s) * 2);
                const float2 q = PAIRS == 1 ? c[s] : e % 2 ? make_float2(two.z, two.w) : make_float2(two.x, two.y);
                const float xa = to_f<DT>(TWO ? a[u].e[e] : a[u].e[2 * e % NV]);
                const float xb = to_f<DT>(TWO ? x2[u].e[e] : a[u].e[(2 * e + 1) % NV]);
                const E ya = from_f<DT>(xa * q.x - xb * q.y), yb = from_f<DT>(xa * q.y + xb * q.x);
                if (TWO) {
                    y.e[e] = ya;
                    y2.e[e] = yb;
                } else {
                    y.e[2 * e % NV] = ya;
                    y.e[(2 * e + 1) % NV] = yb;
                }
            }
            *(Word*)out[u] = y.v;
            if (TWO) *(Word*)(out[u] + ob) = y2.v;
        }
        if (r >= rows) {                                          // the next item
            s += bx;
            r = h = threadIdx.y;
            k = 0;
        }
        if (s >= S) break;
        load();
    }
}

// The same over whole rows, where they allow wider vectors than their pairs do:
// asynchronous copies of NV values each into shared memory, the pairs turned there, and the
// rows written as wide.  With the pairs' narrow vectors too few bytes are in flight (4 x
// 4000 x 10 x 100 bf16, 50 turned: 16 against 51 us, 92 turned: 21 against 25; float32 of
// 96, 38 turned: 22 against 52).  Where both are as wide, rotary_kernel spares the way
// through shared memory (2 x 5000 x 40 x 128 bf16: 37 against 52 us).
constexpr int TILE_BYTES = 16384;       // of rows per block
constexpr int TILE_ROWS = RT;           // at most

template <int BYTES>
SCAO_DEV void copy_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(BYTES) : "memory");
}

template <int DT, bool INTER, int NV>
__global__ void __launch_bounds__(RT)
rotary_tile_kernel(const __grid_constant__ RotArgs A) {
    typedef typename ElemOf<DT>::type E;
    typedef decltype(Pack<DT, NV>::v) Word;
    extern __shared__ float4 tile4[];   // rows, then [token][pair] m cos, +-m sin
    __shared__ const E* src[TILE_ROWS];
    __shared__ E* dst[TILE_ROWS];
    __shared__ int first[TILE_ROWS];    // of the row's cosines and sines
    __shared__ int64_t pos[RTOK];
    E* tile = (E*)tile4;
    float2* cs = (float2*)((char*)tile4 + TILE_BYTES);
    const int half = A.half, tid = threadIdx.x, H0 = A.heads[0];
    const int64_t tok0 = (int64_t)blockIdx.x * A.tb;
    const int nt = (int)min((int64_t)A.tb, A.tokens - tok0);
    const int h0 = blockIdx.y * A.hb, nh = min(A.hb, H0 + A.heads[1] - h0), rows = nt * nh;
    if (tid < rows) {
        const int k = tid / nh, h = h0 + tid - k * nh, w = h >= H0, hh = w ? h - H0 : h;
        const int64_t b = (tok0 + k) / A.T, t = (tok0 + k) - b * A.T;
        src[tid] = (const E*)A.in[w] + b * A.isb[w] + t * A.ist[w] + hh * A.ish[w];
        dst[tid] = (E*)A.out[w] + b * A.osb[w] + t * A.ost[w] + hh * A.osh[w];
        first[tid] = k * half;
        if (tid == k * nh) pos[k] = A.pos ? b * A.pos_sb + t * A.pos_st : A.start + t;
    }
    __syncthreads();
    const int per = A.D / NV, total = rows * per;
    for (int i = tid; i < total; i += RT) {
        const int row = small_div(i, A.inv_per);
        copy_async<NV * sizeof(E)>(tile + i * NV, src[row] + (i - row * per) * NV);
    }
    for (int i = tid; i < nt * half; i += RT) {
        const int t = small_div(i, A.inv_half), j = i - t * half;
        int64_t p = pos[t];
        if (A.pos) p = A.pos64 ? ((const int64_t*)A.pos)[p] : (int64_t)((const int32_t*)A.pos)[p];
        const int part = (int)(((uint64_t)p * A.turn[j]) >> 32);      // of a turn, times 2^32
        float sn, c;
        sincospif((float)part * 0x1p-31f, &sn, &c);
        cs[i] = make_float2(A.cosm * c, A.sinm * sn);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < rows * half; i += RT) {
        const int row = small_div(i, A.inv_half), j = i - row * half;
        E *a = tile + row * A.D + (INTER ? 2 * j : j), *b = a + (INTER ? 1 : half);
        const float2 q = cs[first[row] + j];
        const float xa = to_f<DT>(*a), xb = to_f<DT>(*b);
        *a = from_f<DT>(xa * q.x - xb * q.y);
        *b = from_f<DT>(xa * q.y + xb * q.x);
    }
    __syncthreads();
    for (int i = tid; i < total; i += RT) {
        const int row = small_div(i, A.inv_per);
        *(Word*)(dst[row] + (i - row * per) * NV) = *(const Word*)(tile + i * NV);
    }
}

uint32_t inverse(int n) { return n > 1 ? (uint32_t)((0x100000000ull + n - 1) / n) : 0; }

template <int DT, bool INTER, int NV>
int launch_tile(RotArgs& A, cudaStream_t st) {
    const int H = A.heads[0] + A.heads[1], row = A.D * (int)sizeof(typename ElemOf<DT>::type);
    int rows = TILE_BYTES / row;                                  // at least one: see launch_width
    if (rows > TILE_ROWS) rows = TILE_ROWS;
    A.hb = rows < H ? rows : H;
    int64_t tb = rows / A.hb;
    const int64_t spread = A.tokens / (2 * scao_sm_count());
    if (tb > spread) tb = spread;
    if (tb > RTOK) tb = RTOK;
    if (tb > 2048 / A.half) tb = 2048 / A.half;                   // 16 KB of cosines and sines
    if (tb < 1) tb = 1;
    A.tb = (int)tb;
    A.inv_per = inverse(A.D / NV);
    const int64_t grid = (A.tokens + tb - 1) / tb;
    const int chunks = (H + A.hb - 1) / A.hb;
    if (grid > 0x7fffffff || chunks > 65535) return SCAO_ERR_ARG;
    ProfScope p(SLOT_ROTARY, st);
    rotary_tile_kernel<DT, INTER, NV><<<dim3((unsigned)grid, chunks), RT,
                                 TILE_BYTES + (size_t)tb * A.half * sizeof(float2), st>>>(A);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
}

template <int DT, bool INTER, int NV>
int launch(RotArgs& A, cudaStream_t st) {
    constexpr int PAIRS = INTER ? (NV > 1 ? NV / 2 : 1) : NV;
    const int S = A.half / PAIRS + (A.D - 2 * A.half) / NV, H = A.heads[0] + A.heads[1];
    const int bx = S < RT ? S : RT, by = RT / bx;
    // up to four rows a thread, unless that would leave SMs without a block (eight, or a row
    // beyond four, took 10 to 20 % longer)
    int64_t tb = 4 * by / H;
    const int64_t spread = A.tokens / (2 * scao_sm_count());
    if (tb > spread) tb = spread;
    if (tb > RTOK) tb = RTOK;
    if (tb > 4096 / A.half) tb = 4096 / A.half;                   // 32 KB of cosines and sines
    if (tb < 1) tb = 1;
    A.tb = (int)tb;
    const int64_t grid = (A.tokens + tb - 1) / tb;
    if (grid > 0x7fffffff) return SCAO_ERR_ARG;
    ProfScope p(SLOT_ROTARY, st);
    rotary_kernel<DT, INTER, NV><<<(unsigned)grid, dim3(bx, by), (size_t)tb * A.half * sizeof(float2),
                                   st>>>(A);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
}

// nv: vectors of the pairs; row: of the rows
template <int DT, bool INTER>
int launch_width(RotArgs& A, int nv, int row, cudaStream_t st) {
    if (nv < row && A.D * (int)sizeof(typename ElemOf<DT>::type) <= TILE_BYTES) {
        if constexpr (DT != SCAO_F32)
            if (row == 8) return launch_tile<DT, INTER, 8>(A, st);
        return row == 4 ? launch_tile<DT, INTER, 4>(A, st) : launch_tile<DT, INTER, 2>(A, st);
    }
    if constexpr (DT != SCAO_F32)
        if (nv == 8) return launch<DT, INTER, 8>(A, st);
    if (nv >= 4) return launch<DT, INTER, 4>(A, st);
    if (nv >= 2) return launch<DT, INTER, 2>(A, st);
    return launch<DT, INTER, 1>(A, st);
}

template <int DT>
int launch_layout(RotArgs& A, bool inter, int nv, int row, cudaStream_t st) {
    return inter ? launch_width<DT, true>(A, nv, row, st) : launch_width<DT, false>(A, nv, row, st);
}

}  // namespace

extern "C" int scao_rotary(const ScaoRotary* r, void* stream) {
    if (!r || r->dtype < SCAO_F32 || r->dtype > SCAO_F16 || r->dim < 2 || (r->dim & 1) ||
        r->dim > 2 * RMAX || r->head_dim < r->dim || r->batch < 0 || r->len < 0 || !r->turns ||
        (uintptr_t)r->positions % (r->positions_64 ? 8 : 4))
        return SCAO_ERR_ARG;
    RotArgs A;
    A.T = r->len;
    A.D = r->head_dim;
    A.half = r->dim / 2;
    A.tokens = (int64_t)r->batch * r->len;
    A.pos = r->positions;
    A.pos64 = r->positions_64;
    A.pos_sb = r->pos_stride_b;
    A.pos_st = r->pos_stride_t;
    A.start = r->start;
    A.cosm = r->factor;
    A.sinm = r->inverse ? -r->factor : r->factor;
    const int es = r->dtype == SCAO_F32 ? 4 : 2;
    A.inv_half = inverse(A.half);
    for (int j = 0; j < A.half; ++j) {
        const double whole = floor(r->turns[j]), x = ldexp(r->turns[j] - whole, 64);
        if (!(x >= 0)) return SCAO_ERR_ARG;             // not a number, infinite
        A.turn[j] = x >= 0x1p64 ? 0 : (uint64_t)x;
    }
    // widest vector that every address and stride allows, and (nv) the parts of the head
    int64_t bits = A.D;
    for (int i = 0; i < 2; ++i) {
        A.heads[i] = r->heads[i];
        if (r->heads[i] < 0) return SCAO_ERR_ARG;
        A.in[i] = r->in[i];
        A.out[i] = r->out[i];
        A.isb[i] = r->in_stride[i][0];
        A.ish[i] = r->in_stride[i][1];
        A.ist[i] = r->in_stride[i][2];
        A.osb[i] = r->out_stride[i][0];
        A.osh[i] = r->out_stride[i][1];
        A.ost[i] = r->out_stride[i][2];
        if (!r->heads[i]) continue;
        if (A.tokens && (!A.in[i] || !A.out[i] || ((uintptr_t)A.in[i] | (uintptr_t)A.out[i]) % es))
            return SCAO_ERR_ARG;
        bits |= A.isb[i] | A.ish[i] | A.ist[i] | A.osb[i] | A.osh[i] | A.ost[i] |
                (int64_t)(((uintptr_t)A.in[i] | (uintptr_t)A.out[i]) / es);
    }
    if (A.tokens == 0 || A.heads[0] + A.heads[1] == 0) return SCAO_OK;
    int row = 16 / es;
    while (row > 1 && (bits & (row - 1))) row >>= 1;
    int nv = row;
    while (nv > 1 && ((r->interleaved ? r->dim : A.half) & (nv - 1))) nv >>= 1;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool in = r->interleaved != 0;
    if (r->dtype == SCAO_F32) return launch_layout<SCAO_F32>(A, in, nv, row, st);
    if (r->dtype == SCAO_BF16) return launch_layout<SCAO_BF16>(A, in, nv, row, st);
    return launch_layout<SCAO_F16>(A, in, nv, row, st);
}
