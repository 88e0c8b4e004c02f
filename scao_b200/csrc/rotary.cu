// Rotary positions of query and key heads: for pair j of a head at position p
//
//   (y_a, y_b) = m (x_a cos t - x_b sin t,  x_a sin t + x_b cos t),  t = p w_j
//
// with (a, b) = (2j, 2j + 1) or (j, j + dim/2); values beyond dim pass through.
// The gradient is the transposed rotation: the same kernel with -sin.
//
// The angle is kept in turns and in 64 bits until its whole turns are taken
// off (p w_j / 2 pi reaches 1e5 and more, where 32 bits would leave an error of
// 1e-2 turns); the remainder, below half a turn, goes to sincospif.  The
// frequencies travel as kernel arguments (dim <= 512: 2 KB), so there is no
// table in memory to keep or to outgrow.
//
// A block takes a few tokens: it forms their cosines and sines once into shared
// memory and applies them to every head of q and of k, each value read and
// written once with the widest vector that the strides allow.  HBM bound.
#include "common.cuh"
#include "prof.cuh"
#include "tmap.cuh"

namespace {

constexpr int RT = 256;                 // threads per block, at most
constexpr int RMAX = 256;               // frequencies
constexpr int RTOK = 16;                // tokens per block, at most

struct RotArgs {
    double turn[RMAX];                  // turns per position
    const void* in[2];
    void* out[2];
    int64_t isb[2], ish[2], ist[2], osb[2], osh[2], ost[2];   // strides in values
    const void* pos;                    // int32 / int64, or null: start + t
    int64_t pos_sb, pos_st, start, tokens;
    int heads[2];
    int pos64, T, D, half, tb;
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

// Item of a thread, one of S per head: NV pairs of two vectors (halves apart),
// NV / 2 pairs of one vector (interleaved; one pair where NV is 1), or a
// vector behind the rotated part.
template <int DT, bool INTER, int NV>
__global__ void __launch_bounds__(RT)
rotary_kernel(const __grid_constant__ RotArgs A) {
    typedef typename ElemOf<DT>::type E;
    typedef Pack<DT, NV> V;
    extern __shared__ float2 cs[];      // [token][pair]: m cos, +-m sin
    const int half = A.half;
    const int64_t tok0 = (int64_t)blockIdx.x * A.tb;
    const int nt = (int)min((int64_t)A.tb, A.tokens - tok0);
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthr = blockDim.x * blockDim.y;
    for (int i = tid; i < nt * half; i += nthr) {
        const int k = i / half, j = i - k * half;
        const int64_t b = (tok0 + k) / A.T, t = (tok0 + k) - b * A.T;
        int64_t p = A.start + t;
        if (A.pos) {
            const int64_t o = b * A.pos_sb + t * A.pos_st;
            p = A.pos64 ? ((const int64_t*)A.pos)[o] : (int64_t)((const int32_t*)A.pos)[o];
        }
        const double x = (double)p * A.turn[j];
        float s, c;
        sincospif((float)(2.0 * (x - rint(x))), &s, &c);
        cs[i] = make_float2(A.cosm * c, A.sinm * s);
    }
    __syncthreads();
    constexpr int PAIRS = INTER ? (NV > 1 ? NV / 2 : 1) : NV;     // pairs of a rotating item
    const int rot = half / PAIRS, S = rot + (A.D - 2 * half) / NV;
    const int H = A.heads[0] + A.heads[1], rows = nt * H;
    for (int s = threadIdx.x; s < S; s += blockDim.x) {
        const bool turns = s < rot;
        const int j = s * PAIRS;
        const int oa = turns ? (INTER ? 2 * j : j) : 2 * half + (s - rot) * NV;
        for (int r = threadIdx.y; r < rows; r += blockDim.y) {
            const int k = r / H;
            int h = r - k * H;
            const int w = h >= A.heads[0];
            if (w) h -= A.heads[0];
            const int64_t b = (tok0 + k) / A.T, t = (tok0 + k) - b * A.T;
            const E* in = (const E*)A.in[w] + b * A.isb[w] + h * A.ish[w] + t * A.ist[w] + oa;
            E* out = (E*)A.out[w] + b * A.osb[w] + h * A.osh[w] + t * A.ost[w] + oa;
            V a, y;
            a.v = *(const decltype(a.v)*)in;
            if (!turns) {
                *(decltype(a.v)*)out = a.v;
                continue;
            }
            const float2* c = cs + k * half + j;
            if constexpr (INTER && NV > 1) {
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    const float2 q = c[e];
                    const float xa = to_f<DT>(a.e[2 * e]), xb = to_f<DT>(a.e[2 * e + 1]);
                    y.e[2 * e] = from_f<DT>(xa * q.x - xb * q.y);
                    y.e[2 * e + 1] = from_f<DT>(xa * q.y + xb * q.x);
                }
                *(decltype(a.v)*)out = y.v;
            } else {
                const int ob = INTER ? 1 : half;
                V x2, y2;
                x2.v = *(const decltype(a.v)*)(in + ob);
#pragma unroll
                for (int e = 0; e < NV; ++e) {
                    const float2 q = c[e];
                    const float xa = to_f<DT>(a.e[e]), xb = to_f<DT>(x2.e[e]);
                    y.e[e] = from_f<DT>(xa * q.x - xb * q.y);
                    y2.e[e] = from_f<DT>(xa * q.y + xb * q.x);
                }
                *(decltype(a.v)*)out = y.v;
                *(decltype(a.v)*)(out + ob) = y2.v;
            }
        }
    }
}

template <int DT, bool INTER, int NV>
int launch(RotArgs& A, cudaStream_t st) {
    constexpr int PAIRS = INTER ? (NV > 1 ? NV / 2 : 1) : NV;
    const int S = A.half / PAIRS + (A.D - 2 * A.half) / NV, H = A.heads[0] + A.heads[1];
    const int bx = S < RT ? S : RT, by = RT / bx;
    // about four rows a thread, unless that would leave SMs without a block
    int64_t tb = (4 * by + H - 1) / H;
    const int64_t spread = A.tokens / (2 * scao_sm_count());
    if (tb > spread) tb = spread;
    if (tb > RTOK) tb = RTOK;
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

template <int DT, bool INTER>
int launch_width(RotArgs& A, int nv, cudaStream_t st) {
    if constexpr (DT != SCAO_F32)
        if (nv == 8) return launch<DT, INTER, 8>(A, st);
    if (nv >= 4) return launch<DT, INTER, 4>(A, st);
    if (nv >= 2) return launch<DT, INTER, 2>(A, st);
    return launch<DT, INTER, 1>(A, st);
}

template <int DT>
int launch_layout(RotArgs& A, bool inter, int nv, cudaStream_t st) {
    return inter ? launch_width<DT, true>(A, nv, st) : launch_width<DT, false>(A, nv, st);
}

}  // namespace

extern "C" int scao_rotary(const ScaoRotary* r, void* stream) {
    if (!r || r->dtype < SCAO_F32 || r->dtype > SCAO_F16 || r->dim < 2 || (r->dim & 1) ||
        r->dim > 2 * RMAX || r->head_dim < r->dim || r->batch < 0 || r->len < 0 || !r->turns)
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
    for (int j = 0; j < A.half; ++j) A.turn[j] = r->turns[j];
    // widest vector that every address, stride and part of the head allows
    int64_t bits = A.D | (r->interleaved ? r->dim : A.half);
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
    int nv = 16 / es;
    while (nv > 1 && (bits & (nv - 1))) nv >>= 1;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool in = r->interleaved != 0;
    if (r->dtype == SCAO_F32) return launch_layout<SCAO_F32>(A, in, nv, st);
    if (r->dtype == SCAO_BF16) return launch_layout<SCAO_BF16>(A, in, nv, st);
    return launch_layout<SCAO_F16>(A, in, nv, st);
}
