// Global norm of many gradients, and clipping by it.
//
//   n = (sum |g|^2)^(1/2), sum |g| or max |g| over every value of every tensor
//   c = min(1, max_norm / (n + 1e-6));  g <- c g
//
// Two launches for a step's gradients, whatever their number: grad_norm_kernel
// reads everything once and leaves one partial result per block, and
// grad_scale_kernel, in which every block joins the partials in the same fixed
// order (no atomics: the same inputs give the same bits), forms c and scales.
// Where c is 1 it ends there, so gradients within the threshold are read once
// and never written.  The tensors' addresses travel as kernel arguments: no
// table is copied to the device, and a captured graph holds its own.
//
// Bound by HBM: one reading (plus, where c < 1, a second reading and a write;
// the second reading runs over the tensors backwards, so it begins with what
// the first left in L2).  100 M float32 values: norm 65 us (6.2 TB/s), scaling
// 126 us (6.3 TB/s of reading and writing); 1.41 GB in 195 tensors, clipped, 684 us.
// A single launch with a barrier between its halves would save a launch of about
// 2 us and need every block resident.
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "prof.cuh"
#include "tmap.cuh"

namespace {

constexpr int CT = 512;                 // threads per block
constexpr int CBLOCKS = 2;              // blocks per SM
constexpr int CUNROLL = 4;              // 16-byte loads in flight per thread
// Tensors per launch: a step of up to 200 fits the 4 KB of kernel arguments
// every launch pays for; more take the 32 KB form, 1600 at a time.
constexpr int TAB_SMALL = 200, TAB_LARGE = 1600;
constexpr int NUMEL_BITS = 48;          // numel | dtype << 48

template <int MAXT>
struct GradTab {
    uint64_t ptr[MAXT];
    uint64_t meta[MAXT];
    uint32_t item0[MAXT];               // first work item of the tensor
    uint32_t items;
    int32_t n, chunk;                   // tensors; 16-byte vectors per work item
};
static_assert(sizeof(GradTab<TAB_SMALL>) + 64 <= 4096, "kernel arguments");
static_assert(sizeof(GradTab<TAB_LARGE>) + 64 <= 32764, "kernel arguments");

// One work item: vectors [v0, v1) of a tensor, and for the tensor's first item
// the values before the first and after the last whole 16-byte vector.
struct Item {
    char* base;                         // first whole vector
    int64_t v0, v1;
    int head, tail;                     // loose values of this item
    int64_t nvec;
    int dtype;
};

template <int MAXT>
SCAO_DEV Item find_item(const GradTab<MAXT>& t, uint32_t it) {
    int lo = 0, hi = t.n - 1;           // last tensor with item0 <= it
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.item0[mid] <= it) lo = mid; else hi = mid - 1;
    }
    Item w;
    const uint64_t meta = t.meta[lo];
    const int64_t numel = (int64_t)(meta & ((1ull << NUMEL_BITS) - 1));
    w.dtype = (int)(meta >> NUMEL_BITS);
    const int es = w.dtype == SCAO_F32 ? 4 : 2, per = 16 / es;
    const uint64_t p = t.ptr[lo];
    const int64_t head = min((int64_t)(((16 - (p & 15)) & 15) / es), numel);
    w.base = (char*)(p + head * es);
    w.nvec = (numel - head) / per;
    const int64_t c = it - t.item0[lo];
    w.v0 = c * t.chunk;
    w.v1 = min(w.v0 + t.chunk, w.nvec);
    w.head = c == 0 ? (int)head : 0;
    w.tail = c == 0 ? (int)(numel - head - w.nvec * per) : 0;
    return w;
}

template <int DT>
SCAO_DEV void unpack(uint4 v, float* x) {
    const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == SCAO_F32) {
            x[i] = __uint_as_float(r[i]);
        } else if (DT == SCAO_BF16) {
            x[2 * i] = bf16_bits_to_f(r[i] & 0xffff);
            x[2 * i + 1] = bf16_bits_to_f(r[i] >> 16);
        } else {
            x[2 * i] = f16_bits_to_f(r[i] & 0xffff);
            x[2 * i + 1] = f16_bits_to_f(r[i] >> 16);
        }
    }
}

template <int DT>
SCAO_DEV uint4 pack(const float* x) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == SCAO_F32) r[i] = __float_as_uint(x[i]);
        else if (DT == SCAO_BF16)
            r[i] = (uint32_t)f_to_bf16_bits(x[2 * i]) | ((uint32_t)f_to_bf16_bits(x[2 * i + 1]) << 16);
        else
            r[i] = (uint32_t)f_to_f16_bits(x[2 * i]) | ((uint32_t)f_to_f16_bits(x[2 * i + 1]) << 16);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Running result of one thread: a sum in 64 bits, or the largest |x| as its
// bits (as unsigned numbers NaN > inf > finite, so a NaN stays the largest).
struct Acc {
    double s = 0.0;
    uint32_t m = 0;
};

// Adds n values.  Up to 32 are summed in 32 bits first (their error is below
// 32 * 2^-24 of their sum) and joined to the rest in 64; a batch whose sum
// leaves the range where 32 bits neither overflow nor lose to underflow is
// summed again in 64 bits, so the norm holds over the whole range of float32.
template <int KIND, int N>
SCAO_DEV void add(Acc& a, const float* x) {
    if (KIND == SCAO_NORM_INF) {
#pragma unroll
        for (int i = 0; i < N; ++i) a.m = max(a.m, __float_as_uint(x[i]) & 0x7fffffffu);
        return;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = KIND == SCAO_NORM_2 ? fmaf(x[i], x[i], s) : s + fabsf(x[i]);
    if (s >= 0x1p-100f && s <= 0x1p126f) {
        a.s += (double)s;
        return;
    }
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= __float_as_uint(x[i]) & 0x7fffffffu;
    if (!any) return;                   // all zero: rows that had no gradient
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double y = (double)x[i];
        d += KIND == SCAO_NORM_2 ? y * y : fabs(y);
    }
    a.s += d;
}

template <int KIND, int DT>
SCAO_DEV void norm_item(const Item& w, Acc& a) {
    constexpr int PER = DT == SCAO_F32 ? 4 : 8;
    const uint4* p = (const uint4*)w.base;
    int64_t v = w.v0 + threadIdx.x;
    for (; v + (CUNROLL - 1) * CT < w.v1; v += CUNROLL * CT) {
        uint4 r[CUNROLL];
#pragma unroll
        for (int u = 0; u < CUNROLL; ++u) r[u] = p[v + u * CT];
        float x[CUNROLL * PER];
#pragma unroll
        for (int u = 0; u < CUNROLL; ++u) unpack<DT>(r[u], x + u * PER);
        add<KIND, CUNROLL * PER>(a, x);
    }
    for (; v < w.v1; v += CT) {
        float x[PER];
        unpack<DT>(p[v], x);
        add<KIND, PER>(a, x);
    }
    const int t = threadIdx.x;
    if (t < w.head) {
        const float x = load_dt(w.base, (int64_t)t - w.head, DT);
        add<KIND, 1>(a, &x);
    }
    if (t < w.tail) {
        const float x = load_dt(w.base, w.nvec * PER + t, DT);
        add<KIND, 1>(a, &x);
    }
}

// joins the threads' results in a fixed order; valid in thread 0
template <int KIND>
SCAO_DEV double block_join(double v, double* red) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double w = __shfl_xor_sync(0xffffffffu, v, o);
        v = KIND == SCAO_NORM_INF ? fmax(v, w) : v + w;
    }
    __syncthreads();
    if (lane == 0) red[wid] = v;
    __syncthreads();
    if (wid == 0) {
        v = lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double w = __shfl_xor_sync(0xffffffffu, v, o);
            v = KIND == SCAO_NORM_INF ? fmax(v, w) : v + w;
        }
    }
    return v;
}

// partial[block]: the block's sum, or (largest value) the largest |x|'s bits
// as a whole number
template <int MAXT, int KIND>
__global__ void __launch_bounds__(CT, CBLOCKS)
grad_norm_kernel(const __grid_constant__ GradTab<MAXT> tab, double* __restrict__ partial) {
    __shared__ double red[CT / 32];
    Acc a;
    for (uint32_t it = blockIdx.x; it < tab.items; it += gridDim.x) {
        const Item w = find_item(tab, it);
        if (w.dtype == SCAO_F32) norm_item<KIND, SCAO_F32>(w, a);
        else if (w.dtype == SCAO_BF16) norm_item<KIND, SCAO_BF16>(w, a);
        else norm_item<KIND, SCAO_F16>(w, a);
    }
    const double v = block_join<KIND>(KIND == SCAO_NORM_INF ? (double)a.m : a.s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

template <int DT>
SCAO_DEV void scale_item(const Item& w, float c) {
    constexpr int PER = DT == SCAO_F32 ? 4 : 8;
    uint4* p = (uint4*)w.base;
    int64_t v = w.v0 + threadIdx.x;
    auto scaled = [c](uint4 r) {
        float x[PER];
        unpack<DT>(r, x);
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] *= c;
        return pack<DT>(x);
    };
    for (; v + (CUNROLL - 1) * CT < w.v1; v += CUNROLL * CT) {
        uint4 r[CUNROLL];
#pragma unroll
        for (int u = 0; u < CUNROLL; ++u) r[u] = p[v + u * CT];
#pragma unroll
        for (int u = 0; u < CUNROLL; ++u) p[v + u * CT] = scaled(r[u]);
    }
    for (; v < w.v1; v += CT) p[v] = scaled(p[v]);
    const int t = threadIdx.x;
    if (t < w.head) store_dt(w.base, (int64_t)t - w.head, DT, load_dt(w.base, (int64_t)t - w.head, DT) * c);
    if (t < w.tail) {
        const int64_t i = w.nvec * PER + t;
        store_dt(w.base, i, DT, load_dt(w.base, i, DT) * c);
    }
}

// The norm from `n_partial` partials, or `total_in`; block 0 writes it to
// `total_out` where that is set.  Then c (formed in 64 bits, rounded to 32
// once) and the scaling: c g in 32 bits, rounded then to the gradient's type (in 16 bits a
// second rounding, of 2^-24, which moves a result only where the first falls on a border).
template <int MAXT>
__global__ void __launch_bounds__(CT, CBLOCKS)
grad_scale_kernel(const __grid_constant__ GradTab<MAXT> tab, const double* __restrict__ partial,
                  int n_partial, int kind, double max_norm, const float* __restrict__ total_in,
                  float* total_out) {
    __shared__ double red[CT / 32];
    __shared__ float coef;
    double n;
    if (total_in) {
        n = (double)*total_in;
    } else {
        double v = 0.0;
        if (kind == SCAO_NORM_INF) {
            for (int i = threadIdx.x; i < n_partial; i += CT) v = fmax(v, partial[i]);
            v = block_join<SCAO_NORM_INF>(v, red);
            n = (double)__uint_as_float((uint32_t)v);
        } else {
            for (int i = threadIdx.x; i < n_partial; i += CT) v += partial[i];
            v = block_join<SCAO_NORM_2>(v, red);
            n = kind == SCAO_NORM_2 ? sqrt(v) : v;
        }
    }
    if (threadIdx.x == 0) {
        const float nf = (float)n;                 // as reported: both forms scale alike
        if (total_out && blockIdx.x == 0) *total_out = nf;
        const double c = max_norm / ((double)nf + 1e-6);
        coef = c >= 1.0 ? 1.f : (float)c;          // a NaN stays one
    }
    __syncthreads();
    const float c = coef;
    if (c == 1.f) return;
    for (uint32_t i = blockIdx.x; i < tab.items; i += gridDim.x) {
        const Item w = find_item(tab, tab.items - 1 - i);
        if (w.dtype == SCAO_F32) scale_item<SCAO_F32>(w, c);
        else if (w.dtype == SCAO_BF16) scale_item<SCAO_BF16>(w, c);
        else scale_item<SCAO_F16>(w, c);
    }
}

struct Grad {
    uint64_t ptr;
    int64_t numel;
    int dtype;
    int64_t es() const { return dtype == SCAO_F32 ? 4 : 2; }
};

// rows (address, values, dtype) of the host table; false when one is bad
bool read_table(const int64_t* table, int n, std::vector<Grad>& out) {
    if (n < 0 || (n > 0 && !table)) return false;
    out.reserve(n);
    for (int i = 0; i < n; ++i) {
        const Grad g = {(uint64_t)table[3 * i], table[3 * i + 1], (int)table[3 * i + 2]};
        if (g.numel < 0 || g.numel >= (int64_t)1 << NUMEL_BITS || g.dtype < SCAO_F32 || g.dtype > SCAO_F16)
            return false;
        if (g.numel == 0) continue;
        if (!g.ptr || g.ptr % g.es()) return false;
        out.push_back(g);
    }
    return true;
}

int grid_limit() { return scao_sm_count() * CBLOCKS; }

// Vectors per work item: as many as leave every block one, at most 8 rounds
// of the block (64 KB), so few values are spread over all SMs and many do not
// pay the search of find_item often.
int chunk_of(const std::vector<Grad>& g) {
    int64_t vecs = 0;
    for (const Grad& x : g) vecs += x.numel * x.es() / 16 + 1;
    const int64_t rounds = vecs / ((int64_t)grid_limit() * CT);
    return CT * (int)std::min<int64_t>(std::max<int64_t>(rounds, 1), 8);
}

template <int MAXT>
void fill(GradTab<MAXT>& t, const Grad* g, int n, int chunk) {
    uint64_t item = 0;
    for (int i = 0; i < n; ++i) {
        t.ptr[i] = g[i].ptr;
        t.meta[i] = (uint64_t)g[i].numel | ((uint64_t)g[i].dtype << NUMEL_BITS);
        t.item0[i] = (uint32_t)item;
        const int64_t vecs = g[i].numel * g[i].es() / 16;
        item += (uint64_t)std::max<int64_t>((vecs + chunk - 1) / chunk, 1);
    }
    t.items = (uint32_t)item;
    t.n = n;
    t.chunk = chunk;
}

template <int MAXT>
int run_norm(const Grad* g, int n, int chunk, int kind, double* partial, int* used, cudaStream_t st) {
    static thread_local GradTab<MAXT> tab;
    fill(tab, g, n, chunk);
    const int grid = (int)std::min<int64_t>(tab.items, grid_limit());
    ProfScope p(SLOT_CLIP, st);
    if (kind == SCAO_NORM_2) grad_norm_kernel<MAXT, SCAO_NORM_2><<<grid, CT, 0, st>>>(tab, partial);
    else if (kind == SCAO_NORM_1) grad_norm_kernel<MAXT, SCAO_NORM_1><<<grid, CT, 0, st>>>(tab, partial);
    else grad_norm_kernel<MAXT, SCAO_NORM_INF><<<grid, CT, 0, st>>>(tab, partial);
    SCAO_CHECK_LAUNCH();
    *used = grid;
    return SCAO_OK;
}

template <int MAXT>
int run_scale(const Grad* g, int n, int chunk, const double* partial, int n_partial, int kind,
              double max_norm, const float* total_in, float* total_out, cudaStream_t st) {
    static thread_local GradTab<MAXT> tab;
    fill(tab, g, n, chunk);
    const int grid = (int)std::min<int64_t>(std::max<int64_t>(tab.items, 1), grid_limit());
    ProfScope p(SLOT_CLIP, st);
    grad_scale_kernel<MAXT><<<grid, CT, 0, st>>>(tab, partial, n_partial, kind, max_norm, total_in,
                                                 total_out);
    SCAO_CHECK_LAUNCH();
    return SCAO_OK;
}

// norm of all gradients to total_out, or (total_in) a given norm; then, where
// `clip` is set, the scaling
int norm_and_clip(const int64_t* table, int n, int kind, bool clip, double max_norm, double* partial,
                  const float* total_in, float* total_out, cudaStream_t st) {
    if (kind < SCAO_NORM_1 || kind > SCAO_NORM_INF) return SCAO_ERR_ARG;
    if (clip && !(max_norm >= 0)) return SCAO_ERR_ARG;
    if ((uintptr_t)partial % sizeof(double) || ((uintptr_t)total_in | (uintptr_t)total_out) % sizeof(float))
        return SCAO_ERR_ARG;
    try {
        std::vector<Grad> g;
        if (!read_table(table, n, g)) return SCAO_ERR_ARG;
        const int chunk = chunk_of(g), total = (int)g.size();
        auto slices = [&](auto&& small, auto&& large) {
            if (total <= TAB_SMALL) return small(0, total);
            for (int i = 0; i < total; i += TAB_LARGE)
                if (int rc = large(i, std::min(TAB_LARGE, total - i))) return rc;
            return SCAO_OK;
        };
        int n_partial = 0;
        if (!total_in && total > 0) {
            if (!partial) return SCAO_ERR_ARG;
            int used = 0;
            int rc = slices(
                [&](int i, int k) {
                    int r = run_norm<TAB_SMALL>(&g[i], k, chunk, kind, partial, &used, st);
                    n_partial += used;
                    return r;
                },
                [&](int i, int k) {
                    int r = run_norm<TAB_LARGE>(&g[i], k, chunk, kind, partial + n_partial, &used, st);
                    n_partial += used;
                    return r;
                });
            if (rc) return rc;
        }
        if (!clip) return run_scale<TAB_SMALL>(nullptr, 0, chunk, partial, n_partial, kind, 0.0, total_in,
                                               total_out, st);
        return slices(
            [&](int i, int k) {
                return run_scale<TAB_SMALL>(g.data() + i, k, chunk, partial, n_partial, kind, max_norm,
                                            total_in, total_out, st);
            },
            [&](int i, int k) {
                return run_scale<TAB_LARGE>(g.data() + i, k, chunk, partial, n_partial, kind, max_norm,
                                            total_in, i == 0 ? total_out : nullptr, st);
            });
    } catch (const std::bad_alloc&) {
        return SCAO_ERR_ARG;
    }
}

}  // namespace

extern "C" int64_t scao_grad_norm_workspace_bytes(int n) {
    const int64_t launches = n <= TAB_SMALL ? 1 : ((int64_t)n + TAB_LARGE - 1) / TAB_LARGE;
    return launches * grid_limit() * (int64_t)sizeof(double);
}

extern "C" int scao_grads_overlap(const int64_t* table, int n) {
    try {
        std::vector<Grad> g;
        if (!read_table(table, n, g)) return -1;
        std::sort(g.begin(), g.end(), [](const Grad& a, const Grad& b) { return a.ptr < b.ptr; });
        for (size_t i = 1; i < g.size(); ++i)
            if (g[i - 1].ptr + g[i - 1].numel * g[i - 1].es() > g[i].ptr) return 1;
        return 0;
    } catch (const std::bad_alloc&) {
        return -1;
    }
}

extern "C" int scao_grad_norm(const int64_t* table, int n, int kind, void* workspace, float* total,
                              void* stream) {
    if (!total) return SCAO_ERR_ARG;
    return norm_and_clip(table, n, kind, false, 0.0, (double*)workspace, nullptr, total,
                         (cudaStream_t)stream);
}

extern "C" int scao_grad_clip(const int64_t* table, int n, double max_norm, const float* total,
                              void* stream) {
    if (!total) return SCAO_ERR_ARG;
    return norm_and_clip(table, n, SCAO_NORM_2, true, max_norm, nullptr, total, nullptr,
                         (cudaStream_t)stream);
}

extern "C" int scao_grad_norm_clip(const int64_t* table, int n, int kind, double max_norm,
                                   void* workspace, float* total, void* stream) {
    if (!total) return SCAO_ERR_ARG;
    return norm_and_clip(table, n, kind, true, max_norm, (double*)workspace, nullptr, total,
                         (cudaStream_t)stream);
}
