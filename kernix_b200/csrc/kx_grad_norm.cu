// The 2-norm over all elements of a list of gradients, and the gradients
// scaled down to a largest norm.
//
//   norm = sqrt(sum over all tensors of g^2),  out = g * min(1, max_norm / norm)
//
// Squares are added in 64 bits in an order that the gradients' sizes, strides
// and places against 16 bytes and the device fix: the same gradients where they
// were give the same bits again, and elsewhere bits that may differ in the last
// place of the sum.  A norm that is not finite scales nothing: the outputs are
// the gradients as they were.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "kx_internal.hpp"

using namespace kx;

namespace {

const char *const kNorm = "grad_norm";
const char *const kClip = "clip_grad_norm";
constexpr int kThreads = 256;
constexpr int kSpans = 256;     // tensors of one launch
constexpr int kVectors = 4;     // 16-byte loads in flight for each thread

template <typename T> struct Vec;
template <> struct Vec<float> {
    using type = float4;
    static constexpr int n = 4;
};
template <> struct Vec<double> {
    using type = double2;
    static constexpr int n = 2;
};
template <typename T> constexpr int kChunk = kThreads * kVectors * Vec<T>::n;   // elements

// Tensors whose elements fill their span, in whatever order, as runs of
// memory cut into chunks; a launch's parameters hold the list, so a captured
// graph keeps it.
template <typename T> struct Spans {
    int n;
    uint32_t chunks;
    const T *src[kSpans];
    int64_t len[kSpans];
    uint32_t first[kSpans + 1];     // each span's first chunk, then their number
};
template <typename T> struct Outputs {
    T *dst[kSpans];
};

// A span's elements before its first 16-byte boundary, its vectors, the rest.
template <typename T> struct Cut {
    int head, tail;
    int64_t nv;
    __device__ __forceinline__ Cut(const T *p, int64_t len) {
        const int to = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
        head = to < len ? to : (int)len;
        nv = (len - head) / Vec<T>::n;
        tail = (int)(len - head - nv * Vec<T>::n);
    }
};

// One tensor (and its scaled copy) as C-order dims with each one's strides.
struct Geom {
    int rank;
    int64_t count;
    int64_t dims[KX_MAX_RANK], src[KX_MAX_RANK], dst[KX_MAX_RANK];
};

// I: what counts the elements; 32 bits where they do, as divisions take most of
// the time of a tensor with gaps.
template <typename I>
__device__ __forceinline__ void offsets(const Geom &g, I i, int64_t &so, int64_t &d_o) {
    so = d_o = 0;
    for (int d = g.rank - 1; d > 0; --d) {
        const I n = (I)g.dims[d], q = i / n, c = i - q * n;
        so += (int64_t)c * g.src[d];
        d_o += (int64_t)c * g.dst[d];
        i = q;
    }
    so += (int64_t)i * g.src[0];
    d_o += (int64_t)i * g.dst[0];
}

// Squares are added up in 64 bits, which no square of an f32 leaves.  Those of f64
// elements above 2^512 or below 2^-511 do, so three sums are kept: of the squares
// as they are, of those of the elements times 2^-600 and of those times 2^600.
// The first counts where it is finite and at least 2^-950 (what its squares lose
// below the normal numbers is none of its 53 bits, whatever their number), the
// second where it is infinite, the third where it is less: no square that
// matters leaves that one.  A block whose own first sum is ordinary has the
// second at hand and no part in the third; else it reads its elements again.
// (All three sums in one pass took 27.8 us for 16.8 million elements, where this
// takes 24.9 and the first sum alone 24.8.)
template <typename T> constexpr int kSums = sizeof(T) == 4 ? 1 : 3;
constexpr double kLarge = 0x1p-600, kSmall = 0x1p600, kLeast = 0x1p-950;

// A thread's N first sums, and whether an f64 element is not zero.
template <typename T, int N> struct Squares {
    double s[N] = {};
    bool any = false;
    __device__ __forceinline__ void add(int k, T x) {
        const double d = (double)x;
        s[k] = fma(d, d, s[k]);
        if constexpr (kSums<T> == 3) any = any || d != 0.0;
    }
    __device__ __forceinline__ double total() const {
        double t = 0.0;
#pragma unroll
        for (int k = 0; k < N; ++k) t += s[k];
        return t;
    }
};

// The same total in each thread of the block; a barrier lies between two calls.
__device__ double block_total(double v) {
    constexpr int kWarps = kThreads / 32;
    __shared__ double red[kWarps];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = (threadIdx.x & 31) < kWarps ? red[threadIdx.x & 31] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// The workspace: of each sum, the blocks' partial sums.
constexpr int64_t kRoom = 16384;       // partial sums that it holds; then they are folded
constexpr uint64_t kWorkspace = kSums<double> * kRoom * sizeof(double);

// The root of all squares' sum: of the one that counts.
template <typename T> __device__ __forceinline__ double root_of(double first, double large, double small) {
    if (kSums<T> == 3 && first < kLeast) return sqrt(small) * (1.0 / kSmall);
    if (kSums<T> == 3 && isinf(first)) return sqrt(large) * (1.0 / kLarge);
    return sqrt(first);
}

// The block's partial sums from each thread's first sum; anew(by) is its sum of
// the squares of its elements times `by`, of which any is not zero.  Their root.
template <typename T, typename F>
__device__ __forceinline__ double leave_partials(double mine, bool any, F anew, double *partial) {
    const double s = block_total(mine);
    double large = s * kLarge * kLarge, small = 0.0;
    if constexpr (kSums<T> == 3) {
        const bool less = s < kLeast;
        if ((less || isinf(s)) && __syncthreads_or(any)) {
            const double t = block_total(anew(less ? kSmall : kLarge));
            (less ? small : large) = t;
        }
        if (threadIdx.x == 0) {
            partial[kRoom + blockIdx.x] = large;
            partial[2 * kRoom + blockIdx.x] = small;
        }
    }
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
    return root_of<T>(s, large, small);
}

__device__ __forceinline__ double add_partials(const double *partial, int64_t n) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) s += partial[i];
    return s;
}

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A thread's sum of the squares of its block's elements times `by`, one by one:
// rarely taken, and in few registers.
template <typename T> __device__ __forceinline__ double chunks_anew(const Spans<T> &g, uint32_t lo, uint32_t hi, double by) {
    double s = 0.0;
    int k = 0;
    for (uint32_t c = lo; c < hi; ++c) {
        while (c >= g.first[k + 1]) ++k;
        const Cut<T> cut(g.src[k], g.len[k]);
        // the first chunk of a span has its edges too
        const uint32_t part = c - g.first[k];
        const int64_t a = cut.head + (int64_t)part * kChunk<T>, b = cut.head + cut.nv * Vec<T>::n;
        auto add = [&](int64_t from, int64_t to) {
#pragma unroll 1
            for (int64_t j = from + threadIdx.x; j < to; j += kThreads) {
                const double d = (double)g.src[k][j] * by;
                s = fma(d, d, s);
            }
        };
        add(part ? a : 0, min(a + kChunk<T>, b));
        if (part == 0) add(b, g.len[k]);
    }
    return s;
}

// Sums of squares, one for each block, over its share of the chunks.  The
// bound is the reading: 0.37 billion f32 elements take 214 us, 6.9 TB/s.  A
// square is converted and added in 64 bits, which keeps a tenth of the 64-bit
// pipe busy.
template <typename T>
__global__ void __launch_bounds__(kThreads) sum_spans_kernel(const __grid_constant__ Spans<T> g, double *partial) {
    using V = typename Vec<T>::type;
    constexpr int VN = Vec<T>::n;
    const uint32_t lo = (uint32_t)((uint64_t)blockIdx.x * g.chunks / gridDim.x);
    const uint32_t hi = (uint32_t)((uint64_t)(blockIdx.x + 1) * g.chunks / gridDim.x);
    Squares<T, VN> s;
    int k = 0;
    for (uint32_t c = lo; c < hi; ++c) {
        while (c >= g.first[k + 1]) ++k;
        const T *x = g.src[k];
        const Cut<T> cut(x, g.len[k]);
        const V *xv = reinterpret_cast<const V *>(x + cut.head);
        const int64_t i0 = (int64_t)(c - g.first[k]) * (kThreads * kVectors) + threadIdx.x;
        V v[kVectors];
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            v[u] = V{};
            if (i0 + u * kThreads < cut.nv) v[u] = __ldg(xv + i0 + u * kThreads);
        }
#pragma unroll
        for (int u = 0; u < kVectors; ++u)
#pragma unroll
            for (int e = 0; e < VN; ++e) s.add(e, reinterpret_cast<const T *>(&v[u])[e]);
        if (c == g.first[k]) {      // the span's edges
            if ((int)threadIdx.x < cut.head) s.add(0, x[threadIdx.x]);
            if ((int)threadIdx.x < cut.tail) s.add(0, x[cut.head + cut.nv * VN + threadIdx.x]);
        }
    }
    leave_partials<T>(s.total(), s.any, [&](double by) { return chunks_anew<T>(g, lo, hi, by); }, partial);
    launch_dependents();
}

// The same for a tensor with gaps between its elements, or with several at one
// place.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads) sum_strided_kernel(const T *__restrict__ x, const __grid_constant__ Geom g,
                                                               double *partial) {
    auto each = [&](auto add) {
        for (I i = blockIdx.x * kThreads + threadIdx.x; i < (I)g.count; i += gridDim.x * kThreads) {
            int64_t so, d_o;
            offsets<I>(g, i, so, d_o);
            add(x[so]);
        }
    };
    Squares<T, 1> s;
    each([&](T v) { s.add(0, v); });
    auto anew = [&](double by) {
        double t = 0.0;
        each([&](T v) { t = fma((double)v * by, (double)v * by, t); });
        return t;
    };
    leave_partials<T>(s.total(), s.any, anew, partial);
    launch_dependents();
}

// All partial sums by one block, in the order in which each block of the scaling
// adds them: their root, and the sums in the place of their first parts.
template <typename T> __global__ void __launch_bounds__(kThreads) fold_kernel(double *partial, int64_t n, T *norm) {
    wait_for_previous();
    auto anew = [&](double by) { return add_partials(partial + (by == kLarge ? 1 : 2) * kRoom, n); };
    const double root = leave_partials<T>(add_partials(partial, n), true, anew, partial);
    if (threadIdx.x == 0) *norm = (T)root;
}

// Loads and stores of 16 bytes whose lines are the first to leave the
// second-level cache again.
__device__ __forceinline__ uint64_t leave_first() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
template <typename V> __device__ __forceinline__ V load(const V *p, uint64_t policy) {
    uint4 q;
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "l"(p), "l"(policy));
    return *reinterpret_cast<V *>(&q);
}
template <typename V> __device__ __forceinline__ void store(V *p, const V &v, uint64_t policy) {
    const uint4 q = *reinterpret_cast<const uint4 *>(&v);
    asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(q.x), "r"(q.y), "r"(q.z),
                 "r"(q.w), "l"(policy)
                 : "memory");
}

// The factor of the scaling, and 1.  A factor below the normal numbers lacks
// digits that its products need not lack: it comes as one that has them and a
// power of two.  The first is 1/2 at most: its products fit the type, and it is
// not taken for the factor 1.
template <typename T> struct Scale {
    T by, then;
    __device__ __forceinline__ T operator()(T v) const { return v * by * then; }
};
template <typename T> __device__ Scale<T> split_factor(double max_norm, double root) {
    constexpr bool f32 = sizeof(T) == 4;
    // twice the smallest normal number or, for factors below it, the smallest of all
    const bool last = max_norm / root < (f32 ? 0x1p-149 : 0x1p-1074);
    const double up = f32 ? (last ? 0x1p74 : 0x1p63) : (last ? 0x1p537 : 0x1p511);
    const double down = f32 ? (last ? 0x1p-74 : 0x1p-62) : (last ? 0x1p-536 : 0x1p-510);
    return {(T)(max_norm * up / (root * down)), (T)(f32 ? (last ? 0x1p-148 : 0x1p-125) : (last ? 0x1p-1073 : 0x1p-1021))};
}
template <typename T>
__device__ __forceinline__ Scale<T> scale_of(const double *partial, int64_t n, double max_norm, T *norm) {
    const double s = block_total(add_partials(partial, n));
    double scaled = 0.0;
    if (kSums<T> == 3 && (s < kLeast || isinf(s))) {
        __syncthreads();
        scaled = block_total(add_partials(partial + (s < kLeast ? 2 : 1) * kRoom, n));
    }
    const double root = root_of<T>(s, scaled, scaled);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (T)root;
    if (!isfinite((T)root) || !(root > max_norm)) return {T(1), T(1)};
    const T by = (T)(max_norm / root);
    if (by < T(sizeof(T) == 4 ? FLT_MIN : DBL_MIN)) return split_factor<T>(max_norm, root);
    return {by, T(1)};
}

// The scaled copies.  Each block adds the partial sums for itself, in one
// order, which costs less than another launch would, and takes its chunks last
// to first: what the sums read last is still in the cache.  Where the cache has
// room for much of the gradients (SHORTLY), neither the copies nor gradients
// that have been read again take it from those that have not.  The bound is the
// two streams: 0.37 billion f32 elements take 465 us, 6.3 TB/s.
// Blocks of an SM that the registers are to leave room for (0: any number): five
// are faster at what the cache does not hold (0.37 billion f32 elements clipped:
// 706 us, with six 715, with four 720), the six of the other form at what it
// does (16.8 million: 36.4, with five 36.9).
template <bool SHORTLY> constexpr int kScaleBlocks = SHORTLY ? 0 : 5;

template <typename T, bool SHORTLY>
__global__ void __launch_bounds__(kThreads, kScaleBlocks<SHORTLY>) scale_spans_kernel(const __grid_constant__ Spans<T> g,
                                                               const __grid_constant__ Outputs<T> out,
                                                               const double *partial, int64_t n, double max_norm,
                                                               T *norm) {
    using V = typename Vec<T>::type;
    constexpr int VN = Vec<T>::n;
    wait_for_previous();
    const Scale<T> scale = scale_of<T>(partial, n, max_norm, norm);
    const uint32_t lo = (uint32_t)((uint64_t)blockIdx.x * g.chunks / gridDim.x);
    const uint32_t hi = (uint32_t)((uint64_t)(blockIdx.x + 1) * g.chunks / gridDim.x);
    const uint64_t policy = SHORTLY ? leave_first() : 0;
    int k = g.n - 1;
    for (uint32_t c = hi; c-- > lo;) {
        while (c < g.first[k]) --k;
        const T *x = g.src[k];
        T *y = out.dst[k];
        if (!y || (scale.by == T(1) && x == y)) continue;     // scaled by itself, or in place already
        const Cut<T> cut(x, g.len[k]);
        const uint32_t part = c - g.first[k];
        if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
            const V *xv = reinterpret_cast<const V *>(x + cut.head);
            V *yv = reinterpret_cast<V *>(y + cut.head);
            const int64_t i0 = (int64_t)part * (kThreads * kVectors) + threadIdx.x;
            V v[kVectors];
#pragma unroll
            for (int u = 0; u < kVectors; ++u)
                if (i0 + u * kThreads < cut.nv)
                    v[u] = SHORTLY ? load(xv + i0 + u * kThreads, policy) : xv[i0 + u * kThreads];
#pragma unroll
            for (int u = 0; u < kVectors; ++u) {
#pragma unroll
                for (int e = 0; e < VN; ++e) {
                    T &each = reinterpret_cast<T *>(&v[u])[e];
                    each = scale(each);
                }
                if (i0 + u * kThreads < cut.nv) {
                    if (SHORTLY) store(yv + i0 + u * kThreads, v[u], policy);
                    else yv[i0 + u * kThreads] = v[u];
                }
            }
            if (part == 0) {
                if ((int)threadIdx.x < cut.head) y[threadIdx.x] = scale(x[threadIdx.x]);
                const int64_t j = cut.head + cut.nv * VN + threadIdx.x;
                if ((int)threadIdx.x < cut.tail) y[j] = scale(x[j]);
            }
        } else {    // the two lie differently against 16 bytes
            const int64_t j0 = (int64_t)part * kChunk<T>;
            const int64_t j1 = c + 1 == g.first[k + 1] ? g.len[k] : j0 + kChunk<T>;
            for (int64_t j = j0 + threadIdx.x; j < j1; j += kThreads) y[j] = scale(x[j]);
        }
    }
}

template <typename T, typename I>
__global__ void __launch_bounds__(kThreads) scale_strided_kernel(const T *x, T *out, const __grid_constant__ Geom g,
                                                                 const double *partial, int64_t n, double max_norm,
                                                                 T *norm) {
    wait_for_previous();
    const Scale<T> scale = scale_of<T>(partial, n, max_norm, norm);
    for (I i = blockIdx.x * kThreads + threadIdx.x; i < (I)g.count; i += gridDim.x * kThreads) {
        int64_t so, d_o;
        offsets<I>(g, i, so, d_o);
        out[d_o] = scale(x[so]);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int64_t kPartials = 2048;    // most blocks of one launch over spans,
constexpr int64_t kStrided = 512;      // over a tensor by itself
constexpr uint64_t kMostTensors = 1u << 20;
constexpr int64_t kCount32 = 1ll << 31;    // 32 bits count fewer elements, and a block's step beyond them
constexpr int64_t kFold = 2048;        // most partial sums that each block of the scaling adds

// Bytes of gradients between which the scaling marks its accesses as the first to
// leave the cache of 126 MB: 48 MB are clipped in 25.9 us, without marks in 28.5,
// 64 MB in 32.5 and 35.3, 128 MB in 62.0 and 65.6.  Fewer have room beside their
// copies, which are there for who reads them next (clipped and read, 44 MB take
// 34.7 and 33.2, 48 MB 37.1 and 37.6); of more little is left to read again (192
// MB clipped and read: 134.9 both ways, 256 MB 179 and 176).  All of that is of
// copies apart; lists clipped in place follow the same rule, unmeasured.
constexpr int64_t kShortlyFrom = 46ll << 20, kShortlyTo = 192ll << 20;

struct Range {
    uintptr_t a, b;
    bool out;
};

// The same elements at the same addresses.
bool same_view(const kx_tensor &g, const kx_tensor &o) {
    bool same = g.data == o.data && g.origin == o.origin;
    for (uint32_t d = 0; d < g.rank; ++d) same = same && (g.dims[d] <= 1 || g.strides[d] == o.strides[d]);
    return same;
}

// Distinct elements at distinct addresses: with the strides in order of size,
// each steps over all that the smaller ones reach.
bool distinct_elements(const kx_tensor *t) {
    struct {
        i128 step, dim;
    } s[KX_MAX_RANK];
    int n = 0;
    for (uint32_t d = 0; d < t->rank; ++d) {
        if (t->dims[d] == 0) return true;
        if (t->dims[d] == 1) continue;
        const i128 step = t->strides[d] < 0 ? -(i128)t->strides[d] : (i128)t->strides[d];
        int i = n++;
        for (; i > 0 && s[i - 1].step > step; --i) s[i] = s[i - 1];
        s[i] = {step, (i128)t->dims[d]};
    }
    i128 reach = 0;   // largest offset of the strides so far
    for (int i = 0; i < n; ++i) {
        if (s[i].step <= reach) return false;
        reach += s[i].step * (s[i].dim - 1);
    }
    return true;
}

// Validates both lists; no device work.
template <typename T>
int check_lists(const kx_tensor *grads, uint64_t count, const kx_tensor *outs, const kx_tensor *norm,
                const void *workspace, uint64_t bytes, const char *op, kx_error *err) {
    if (count && !grads) return set_err(err, KX_E_PARAM, op, "null gradients");
    if (count > kMostTensors) return set_err(err, KX_E_UNSUPPORTED, op, "more than 2^20 gradients");
    Span s;
    int rc = validate_tensor(norm, sizeof(T), &s, err);
    if (rc) return rc;
    if (numel(norm->dims, norm->rank) != 1)
        return set_err(err, KX_E_LAYOUT, op, "norm (one element)", KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
    if (!workspace || bytes < kWorkspace || (uintptr_t)workspace % 8)
        return set_err(err, KX_E_PARAM, op, "workspace (8-byte aligned, of the size asked for)");
    std::vector<Range> all;
    all.reserve(2 * count + 2);
    auto add = [&](const kx_tensor *t, const Span &sp, bool out) {
        if (!sp.empty)
            all.push_back({(uintptr_t)t->data + sp.start * sizeof(T), (uintptr_t)t->data + sp.end * sizeof(T), out});
    };
    add(norm, s, true);
    all.push_back({(uintptr_t)workspace, (uintptr_t)workspace + kWorkspace, true});
    uint64_t total = 0;
    for (uint64_t i = 0; i < count; ++i) {
        rc = validate_tensor(&grads[i], sizeof(T), &s, err);
        if (rc) return rc;
        if (numel(grads[i].dims, grads[i].rank) > kIsizeMax - total)
            return set_err(err, KX_E_UNSUPPORTED, op, "too many elements");
        total += numel(grads[i].dims, grads[i].rank);
        if (!outs || !same_view(grads[i], outs[i])) add(&grads[i], s, false);
        if (!outs) continue;
        rc = validate_tensor(&outs[i], sizeof(T), &s, err);
        if (rc) return rc;
        bool same = outs[i].rank == grads[i].rank;
        for (uint32_t d = 0; same && d < outs[i].rank; ++d) same = outs[i].dims[d] == grads[i].dims[d];
        if (!same) return set_err(err, KX_E_LAYOUT, op, "output shape mismatch", KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
        if (!distinct_elements(&outs[i])) return set_err(err, KX_E_ALIAS, op, "output elements overlap");
        add(&outs[i], s, true);
    }
    // An output may be its own gradient, element for element (one range then),
    // and touches nothing else of the call.
    std::sort(all.begin(), all.end(), [](const Range &x, const Range &y) { return x.a < y.a; });
    uintptr_t end_out = 0, end_any = 0;   // furthest end of the outputs and of all ranges so far
    for (const Range &r : all) {
        if (r.a < (r.out ? end_any : end_out)) return set_err(err, KX_E_ALIAS, op, "output overlaps another operand");
        if (r.out) end_out = std::max(end_out, r.b);
        end_any = std::max(end_any, r.b);
    }
    return KX_OK;
}

template <typename T> T *at(const kx_tensor *t) { return static_cast<T *>(t->data) + t->origin; }

// Dims from the gradient's largest stride to its smallest, those of one element
// left out, neighbours that both tensors walk as one merged.
Geom geom(const kx_tensor *g, const kx_tensor *o) {
    Geom r;
    std::memset(&r, 0, sizeof(r));
    r.count = (int64_t)numel(g->dims, g->rank);
    auto size = [](int64_t s) { return s < 0 ? -(i128)s : (i128)s; };
    int n = 0;
    for (uint32_t d = 0; d < g->rank; ++d) {
        if (g->dims[d] == 1) continue;
        int at = n++;
        for (; at > 0 && size(r.src[at - 1]) < size(g->strides[d]); --at) {
            r.dims[at] = r.dims[at - 1];
            r.src[at] = r.src[at - 1];
            r.dst[at] = r.dst[at - 1];
        }
        r.dims[at] = (int64_t)g->dims[d];
        r.src[at] = g->strides[d];
        r.dst[at] = o ? o->strides[d] : 0;
    }
    int w = 0;
    for (int d = 0; d < n; ++d) {
        if (w > 0 && r.src[w - 1] == (i128)r.src[d] * r.dims[d] && r.dst[w - 1] == (i128)r.dst[d] * r.dims[d])
            r.dims[w - 1] *= r.dims[d];
        else
            r.dims[w++] = r.dims[d];
        r.src[w - 1] = r.src[d];
        r.dst[w - 1] = r.dst[d];
    }
    r.rank = w;
    return r;
}

// The offset of a nonempty tensor's lowest element from its origin, if its
// elements fill their span, each at a place of its own; 1 if they do not.
int64_t filled_span(const kx_tensor *t) {
    if (is_c_contiguous(t)) return 0;
    i128 low = 0, reach = 0;
    for (uint32_t d = 0; d < t->rank; ++d) {
        if (t->dims[d] == 1) continue;
        const i128 r = (i128)t->strides[d] * (i128)(t->dims[d] - 1);
        if (r < 0) low += r;
        reach += r < 0 ? -r : r;
    }
    if (reach + 1 != (i128)numel(t->dims, t->rank) || !distinct_elements(t)) return 1;
    return (int64_t)low;
}

bool same_strides(const kx_tensor *a, const kx_tensor *b) {
    for (uint32_t d = 0; d < a->rank; ++d)
        if (a->dims[d] > 1 && a->strides[d] != b->strides[d]) return false;
    return true;
}

unsigned blocks_for(int64_t count) {
    const int64_t b = (count + kThreads * 8 - 1) / (kThreads * 8);
    return (unsigned)std::min<int64_t>(kStrided, std::max<int64_t>(b, 1));
}

// One launch's worth of filled spans.
template <typename T> struct Batch {
    Spans<T> spans;
    Outputs<T> outs;
    // Eight blocks for each SM where they have four chunks or more each (0.37
    // billion f32 elements: 213 us, with four blocks 241), else four: every
    // block's sum is read by every block of the scaling (4.2 million elements,
    // clipped: 14 us, with eight blocks 16).
    unsigned blocks(const Handle *h) const {
        const unsigned some = std::min(spans.chunks, 4u * h->sm_count), more = std::min(spans.chunks / 4, 8u * h->sm_count);
        return std::min<unsigned>(kPartials, std::max(some, more));
    }
};

// A kernel that may start while the previous one ends; it waits by itself for
// that one's results (griddepcontrol.wait).
template <typename... Params, typename... Args>
void launch_after(Handle *h, void (*kernel)(Params...), unsigned blocks, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = h->stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
    ++h->launches;
}

template <typename T>
int norm_lists(Handle *h, const kx_tensor *grads, uint64_t count, double max_norm, const kx_tensor *outs,
               const kx_tensor *norm, void *workspace, const char *op, kx_error *err) {
    // which tensors are runs of memory; the rest go one by one, and so does the
    // scaling into an output of other strides, so that the sums are the same
    // whatever the outputs are
    std::vector<Batch<T>> batches;
    std::vector<uint64_t> strided, apart;
    int64_t bytes = 0;      // of the gradients
    for (uint64_t i = 0; i < count; ++i) {
        const int64_t n = (int64_t)numel(grads[i].dims, grads[i].rank);
        if (n == 0) continue;
        bytes += n * (int64_t)sizeof(T);
        const int64_t low = filled_span(&grads[i]);
        const bool alike = outs && same_strides(&grads[i], &outs[i]);
        if (outs && (low > 0 || !alike)) apart.push_back(i);
        if (low > 0) {
            strided.push_back(i);
            continue;
        }
        if (n / kChunk<T> > (1 << 30)) return set_err(err, KX_E_UNSUPPORTED, op, "too many elements");
        const uint32_t chunks = (uint32_t)std::max<int64_t>(1, (n + kChunk<T> - 1) / kChunk<T>);
        if (batches.empty() || batches.back().spans.n == kSpans || batches.back().spans.chunks > (1u << 30)) {
            batches.emplace_back();
            batches.back().spans.n = 0;
            batches.back().spans.chunks = 0;
        }
        Spans<T> &s = batches.back().spans;
        s.src[s.n] = at<T>(&grads[i]) + low;
        s.len[s.n] = n;
        s.first[s.n] = s.chunks;
        batches.back().outs.dst[s.n] = alike ? at<T>(&outs[i]) + low : nullptr;
        s.chunks += chunks;
        s.first[++s.n] = s.chunks;
    }
    double *partial = static_cast<double *>(workspace);
    T *to = at<T>(norm);
    int64_t used = 0;
    auto room = [&](int64_t blocks) {   // for that many partial sums more
        if (used + blocks <= kRoom) return;
        launch_after(h, fold_kernel<T>, 1, partial, used, to);
        used = 1;
    };
    for (const Batch<T> &b : batches) {
        room(b.blocks(h));
        sum_spans_kernel<T><<<b.blocks(h), kThreads, 0, h->stream>>>(b.spans, partial + used);
        ++h->launches;
        used += b.blocks(h);
    }
    for (uint64_t i : strided) {
        const Geom g = geom(&grads[i], nullptr);
        const unsigned blocks = blocks_for(g.count);
        room(blocks);
        if (g.count < kCount32)
            sum_strided_kernel<T, uint32_t><<<blocks, kThreads, 0, h->stream>>>(at<T>(&grads[i]), g, partial + used);
        else
            sum_strided_kernel<T, int64_t><<<blocks, kThreads, 0, h->stream>>>(at<T>(&grads[i]), g, partial + used);
        ++h->launches;
        used += blocks;
    }
    if (!outs || used == 0 || used > kFold) {
        launch_after(h, fold_kernel<T>, 1, partial, used, to);
        used = 1;
        to = nullptr;
    }
    if (outs) {
        const bool shortly = bytes > kShortlyFrom && bytes <= kShortlyTo;
        for (const Batch<T> &b : batches) {
            launch_after(h, shortly ? scale_spans_kernel<T, true> : scale_spans_kernel<T, false>, b.blocks(h),
                         b.spans, b.outs, partial, used, max_norm, to);
            to = nullptr;
        }
        for (uint64_t i : apart) {
            const Geom g = geom(&grads[i], &outs[i]);
            launch_after(h, g.count < kCount32 ? scale_strided_kernel<T, uint32_t> : scale_strided_kernel<T, int64_t>,
                         blocks_for(g.count), at<T>(&grads[i]), at<T>(&outs[i]), g, partial, used, max_norm, to);
            to = nullptr;
        }
    }
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, op);
    }
    h->last_kernel = op;
    return KX_OK;
}

template <typename T>
int norm_impl(kx_handle *hh, const kx_tensor *grads, uint64_t count, double max_norm, const kx_tensor *outs,
              const kx_tensor *norm, void *workspace, uint64_t bytes, const char *op, kx_error *err) {
    if (!hh) return set_err(err, KX_E_PARAM, op, "null handle");
    Handle *h = &hh->impl;
    if (outs && !(std::isfinite(max_norm) && max_norm > 0.0))
        return set_err(err, KX_E_PARAM, op, "max_norm (must be finite and > 0)");
    try {
        const int rc = check_lists<T>(grads, count, outs, norm, workspace, bytes, op, err);
        if (rc) return rc;
        DeviceGuard guard(h->device);
        if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, op, "cannot select device");
        return norm_lists<T>(h, grads, count, max_norm, outs, norm, workspace, op, err);
    } catch (const std::bad_alloc &) {
        return set_err(err, KX_E_PARAM, op, "out of host memory");
    }
}

}  // namespace

extern "C" {
int kx_grad_norm_workspace(uint64_t *bytes) {
    if (!bytes) return KX_E_PARAM;
    *bytes = kWorkspace;
    return KX_OK;
}
int kx_grad_norm_f32(kx_handle *h, const kx_tensor *grads, uint64_t count, const kx_tensor *norm, void *workspace,
                     uint64_t workspace_bytes, kx_error *err) {
    return norm_impl<float>(h, grads, count, 0.0, nullptr, norm, workspace, workspace_bytes, kNorm, err);
}
int kx_grad_norm_f64(kx_handle *h, const kx_tensor *grads, uint64_t count, const kx_tensor *norm, void *workspace,
                     uint64_t workspace_bytes, kx_error *err) {
    return norm_impl<double>(h, grads, count, 0.0, nullptr, norm, workspace, workspace_bytes, kNorm, err);
}
int kx_clip_grad_norm_f32(kx_handle *h, const kx_tensor *grads, uint64_t count, double max_norm, const kx_tensor *outs,
                          const kx_tensor *norm, void *workspace, uint64_t workspace_bytes, kx_error *err) {
    if (count && !outs) return set_err(err, KX_E_PARAM, kClip, "null outputs");
    const kx_tensor none = {};
    return norm_impl<float>(h, grads, count, max_norm, outs ? outs : &none, norm, workspace, workspace_bytes, kClip,
                            err);
}
int kx_clip_grad_norm_f64(kx_handle *h, const kx_tensor *grads, uint64_t count, double max_norm, const kx_tensor *outs,
                          const kx_tensor *norm, void *workspace, uint64_t workspace_bytes, kx_error *err) {
    if (count && !outs) return set_err(err, KX_E_PARAM, kClip, "null outputs");
    const kx_tensor none = {};
    return norm_impl<double>(h, grads, count, max_norm, outs ? outs : &none, norm, workspace, workspace_bytes, kClip,
                             err);
}
}
