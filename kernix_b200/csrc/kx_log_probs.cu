// Log probabilities of given tokens, with the entropy and the likeliest
// alternatives of each row of logits, and their gradient.
//
// With z = x / T over the last axis of the logits:
//   lse       = m/T + log S,  m = max x,  S = sum exp((x - m)/T)
//   log_prob  = (x_t - m)/T - log S            for the row's given token t
//   entropy   = log S - sum exp((x - m)/T) (x - m)/T / S
//   alternatives: the largest x, ties to the lower index, each as z - lse
//   gradient  = [p (g_lse - g_lp - g_H (log p + H)) + g_lp [j = t]] / T
// A logit of -inf is a token that a mask took out: probability 0, no part in
// the entropy, gradient 0.  Nothing here is read back by the host: rows that
// hold a NaN or +inf answer with NaN.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>
#include <limits>

#include "kx_internal.hpp"

namespace cg = cooperative_groups;
using namespace kx;

namespace {

constexpr int kMaxTop = 32;
constexpr int kRowOperands = 7;
enum RowOperand { kLogits, kTokens, kLse, kEntropy, kGradLp, kGradH, kGradLse };

// Where row r (C order over the leading dims) starts in each operand.
struct Rows {
    int64_t count;
    int ndims;
    int64_t dims[KX_MAX_RANK];
    int64_t str[kRowOperands][KX_MAX_RANK];
};

__device__ __forceinline__ int64_t row_offset(const Rows &g, int which, int64_t row) {
    int64_t o = 0;
    for (int d = g.ndims - 1; d > 0; --d) {
        const int64_t q = row / g.dims[d];
        o += (row - q * g.dims[d]) * g.str[which][d];
        row = q;
    }
    return g.ndims > 0 ? o + row * g.str[which][0] : o;
}

template <typename T> struct ForwardParams {
    const T *x;
    const int64_t *tokens;
    T *log_probs, *lse, *entropy, *top_lp;
    int64_t *top_ids;
    int64_t stride;
    int len, top, cluster;   // cluster: blocks that share a row
    T factor;                // exp_factor(temperature)
    double inverse;          // 1 / temperature
    Rows rows;
};

template <typename T> struct Vec;
template <> struct Vec<float> {
    using type = float4;
    static constexpr int n = 4;
};
template <> struct Vec<double> {
    using type = double2;
    static constexpr int n = 2;
};

// Exponentials of differences d = x - m <= 0.  They take d c, c = unit / T.
//
// f32: 2^a by the special-function unit, whose few half steps of error are
// below those of the difference itself; results under the smallest normal
// number are 0.
//
// f64: a counts sixteenths, 2^(a/16).  With n = round(a) and g = a - n, which
// is exact, it is 2^(n/16) 2^(g/16): the first factor is one of 16 roots with n's
// whole part in its exponent, the second 1 + g q(g), |g| <= 1/2, from the
// Taylor series of 2^x to the seventh power (the eighth is below 2^-59).  That
// is 12 operations in 64 bits instead of the about 25 of exp(), which with its
// registers held the f64 pass over the logits at a third of its speed.
// Below 2^-1020 nothing counts: neither in a sum beside exp(0) nor after
// multiplication with the difference, which may be -inf there.
template <typename T> struct Exp;

// 1.5 2^52, which leaves a sum's last place at 1, and log(2)^i / i! / 16^i from
// the seventh down: in constant memory an instruction takes them as they are,
// where 64-bit literals take two more instructions each.
__constant__ double kExpTerms[8] = {6755399441055744.0,
                                    0.000015252733804059840280 / 268435456,
                                    0.00015403530393381609954 / 16777216,
                                    0.0013333558146428443423 / 1048576,
                                    0.0096181291076284771620 / 65536,
                                    0.055504108664821579953 / 4096,
                                    0.24022650695910071233 / 256,
                                    0.69314718055994530942 / 16};

template <> struct Exp<float> {
    static constexpr double unit = 1.4426950408889634;      // log2(e)
    struct Table {};
    __device__ __forceinline__ explicit Exp(const Table &) {}
    __device__ __forceinline__ float operator()(float a) const {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a));
        return e;
    }
};
template <> struct Exp<double> {
    static constexpr double unit = 16 * 1.4426950408889634074;
    struct Table {
        double root[16];    // 2^(j/16)
    };
    const double *root;
    __device__ __forceinline__ explicit Exp(const Table &t) : root(t.root) {}
    __device__ __forceinline__ static bool counts(double a) { return !(a < -16.0 * 1020.0); }   // a NaN does
    __device__ __forceinline__ double operator()(double a) const {
        const double shifted = a + kExpTerms[0], g = a - (shifted - kExpTerms[0]);
        const int n = __double2loint(shifted);
        const double r = root[n & 15];
        const double scaled = __hiloint2double(__double2hiint(r) + ((n >> 4) << 20), __double2loint(r));
        double q = fma(kExpTerms[1], g, kExpTerms[2]);
#pragma unroll
        for (int i = 3; i < 8; ++i) q = fma(q, g, kExpTerms[i]);
        return fma(scaled, q * g, scaled);
    }
};
// The first threads of a block or warp fill the table; a barrier follows.
__device__ __forceinline__ void fill(Exp<float>::Table &, int) {}
__device__ __forceinline__ void fill(Exp<double>::Table &t, int tid) {
    if (tid < 16) t.root[tid] = exp2((double)tid / 16);
}
template <typename T> T exp_factor(T temperature) { return (T)(Exp<T>::unit / (double)temperature); }

template <typename T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -FLT_MAX; }
template <> __device__ __forceinline__ double lowest<double>() { return -DBL_MAX; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
// no instruction has it in 64 bits; b where a is NaN
__device__ __forceinline__ double larger(double a, double b) { return a > b ? a : b; }

__device__ __forceinline__ float warp_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// What a thread knows of the elements that it has seen: their maximum, the sum
// of exp((x - m)/T) and that of exp((x - m)/T) (x - m).  A NaN or +inf makes
// the sum NaN; it stays 0 where all elements are -inf, which makes -inf the
// neutral element that fills up a last vector.
template <typename T, bool ENT> struct Stats {
    T m = lowest<T>(), s = T(0), e = T(0);

    // adds the values and gives the largest of them
    template <int N> __device__ __forceinline__ T add(const T (&v)[N], T c, const Exp<T> &ex) {
        T most = lowest<T>();
#pragma unroll
        for (int i = 0; i < N; ++i) most = larger(v[i], most);
        const T nm = larger(most, m);
        // one more f32 exponential costs less than a branch around it
        if (sizeof(T) == 4 || nm != m) rebase(nm, c, ex);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const T d = v[i] - m;
            if constexpr (sizeof(T) == 4) {
                const T p = ex(d * c);
                s += p;
                // of a difference of -inf the exponential is 0, and so is the product
                if (ENT) e = fma(p, larger(d, lowest<T>()), e);
            } else {
                const T p = ex(d * c);      // and thrown away, rather than a branch for each
                if (Exp<T>::counts(d * c)) {
                    s += p;
                    if (ENT) e = fma(p, d, e);
                }
            }
        }
        return most;
    }
    __device__ __forceinline__ void rebase(T nm, T c, const Exp<T> &ex) {
        const T d = m - nm;
        T f;
        if constexpr (sizeof(T) == 4) f = ex(d * c);
        else f = Exp<T>::counts(d * c) ? ex(d * c) : T(0);
        if (ENT) e = f == T(0) ? T(0) : fma(d, s, e) * f;
        s *= f;
        m = nm;
    }
    // over N lanes that stand side by side, the same in each; all N are one and
    // the same in the other lanes' groups
    template <int N> __device__ __forceinline__ void join(T c, const Exp<T> &ex) {
        rebase(warp_max(m), c, ex);
#pragma unroll
        for (int o = N / 2; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            if (ENT) e += __shfl_xor_sync(0xffffffffu, e, o);
        }
    }
};

// One row's elements as this block walks them: a head up to the first 16-byte
// boundary, vectors, a tail; or single elements of any stride.
template <typename T, bool VEC> struct RowView {
    static constexpr int VN = VEC ? Vec<T>::n : 1;
    const T *x;
    int64_t stride;
    int head, tail, nv;   // elements before the vectors, after them; vectors

    // A stride of 1 that the compiler knows saves a 64-bit product for each
    // element (the gradient of 4096 x 1003 f32: 7.8 us, with it 9.1).
    __device__ __forceinline__ RowView(const T *row, int len, int64_t stride_) : x(row), stride(VEC ? 1 : stride_) {
        if (VEC) {
            const int to = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
            head = to < len ? to : len;
            nv = (len - head) / VN;
            tail = len - head - nv * VN;
        } else {
            head = tail = 0;
            nv = len;
        }
    }
    __device__ __forceinline__ void load(int i, bool ok, T (&v)[VN]) const {
        if (VEC) {
            typename Vec<T>::type q;
            if (ok) q = __ldg(reinterpret_cast<const typename Vec<T>::type *>(x + head) + i);
#pragma unroll
            for (int k = 0; k < VN; ++k) v[k] = ok ? reinterpret_cast<const T *>(&q)[k] : T(-INFINITY);
        } else {
            v[0] = ok ? __ldg(x + i * stride) : T(-INFINITY);
        }
    }
    __device__ __forceinline__ T at(int j) const { return __ldg(x + j * stride); }
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// An element as the alternatives are ordered: by value, then by place, the
// lower one first.  For f32 both are one whole number, so that a comparison is
// one too; the two zeros are equal.  none(n) are the 512 that a row does not
// have, behind all that it can have.
template <typename T> struct Key;
template <> struct Key<float> {
    uint64_t k;
    __device__ static Key of(float v, int i) {
        const int b = __float_as_int(v + 0.0f);
        const uint32_t rising = (uint32_t)(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
        return {(uint64_t)rising << 32 | (uint32_t)~i};
    }
    __device__ static Key first() { return {~0ull}; }
    __device__ static Key none(int n) { return of(-INFINITY, INT_MAX - 512 + n); }
    __device__ bool before(const Key &o) const { return k > o.k; }
    __device__ float value() const {
        const int b = (int)((uint32_t)(k >> 32) ^ 0x80000000u);
        return __int_as_float(b ^ ((b >> 31) & 0x7fffffff));
    }
    __device__ int place() const { return (int)~(uint32_t)k; }
    __device__ Key lane_xor(int o) const { return {__shfl_xor_sync(0xffffffffu, k, o)}; }
};
template <> struct __align__(16) Key<double> {
    double v;
    int i;
    __device__ static Key of(double v, int i) { return {v, i}; }
    __device__ static Key first() { return {(double)INFINITY, -1}; }
    __device__ static Key none(int n) { return {-(double)INFINITY, INT_MAX - 512 + n}; }
    __device__ bool before(const Key &o) const { return v > o.v || (v == o.v && i < o.i); }
    __device__ double value() const { return v; }
    __device__ int place() const { return i; }
    __device__ Key lane_xor(int o) const {
        return {__shfl_xor_sync(0xffffffffu, v, o), __shfl_xor_sync(0xffffffffu, i, o)};
    }
};

// The warp's lane values in falling order over its lanes (a bitonic network).
template <typename T> __device__ __forceinline__ T sorted_falling(T v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const T o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool up = (lane & j) == 0, falling = (lane & k) == 0;
            v = up == falling ? fmax(v, o) : fmin(v, o);
        }
    }
    return v;
}

// The same for values that rise and then fall, or the other way round.
template <typename T> __device__ __forceinline__ T falling_again(T v, int lane) {
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) {
        const T o = __shfl_xor_sync(0xffffffffu, v, j);
        v = (lane & j) == 0 ? fmax(v, o) : fmin(v, o);
    }
    return v;
}

// The q-th largest of the warp's lane values.  Up to six are found one by one,
// in blocks of four and eight warps (2500 x 30000 f32 with 8 alternatives: 57.4
// us, sorting always 58.4).
template <typename T> __device__ __forceinline__ T largest(T v, int q, int lane) {
    if (q > 6) return __shfl_sync(0xffffffffu, sorted_falling(v, lane), q - 1);
    for (; q > 1; --q) {
        const unsigned at = __ballot_sync(0xffffffffu, v == warp_max(v));
        if (lane == __ffs(at) - 1) v = T(-INFINITY);
    }
    return warp_max(v);
}

template <int NW> constexpr int kCandidates = NW == 1 ? 256 : 512;
constexpr int kMaxCluster = 8;
// Alternatives for which one warp's 32 maxima bound well: beyond them the bound
// comes from the maxima of the parts (4096 x 1000 f32 with 32 alternatives:
// 13 us, with the 32 maxima 46; with 16 alternatives 11.7 and 10.5).
constexpr int kWarpTop = 20;
template <int NW> constexpr int kSlots = NW == 1 ? 8 : 16;

template <typename T, int NW> struct Shared {
    T m[NW], s[NW], e[NW], bound[NW];     // each warp's
    T part_m[kMaxCluster], part_s[kMaxCluster], part_e[kMaxCluster];    // each block's of the cluster
    T slot[kSlots<NW>][NW * 32];          // each thread's maxima over parts of its elements
    typename Exp<T>::Table table;
    int found;
    Key<T> best[32];                      // the block's alternatives, in order
    Key<T> cand[kCandidates<NW>];
    Key<T> list[NW == 8 ? kMaxCluster : 1][32];         // the alternatives of each block of the cluster
};

// Blocks of one SM: 48 registers a thread for f32 (56 where a warp has a row,
// 64 with WIDE, which has twice the loads in flight), 64 for f64 (96).
template <typename T, int NW, bool WIDE>
constexpr int kBlocks = NW == 1 ? (sizeof(T) == 4 ? 9 : 5) : (sizeof(T) == 4 && !WIDE ? 40 : 32) / NW;

// The forward pass.  One pass over the logits keeps, for each thread, the
// maximum of its elements and the two sums against it; they meet by shuffles,
// then in shared memory, then (few rows) in that of the cluster's first block,
// so that one launch and no workspace do for any number of rows.  The bound is
// the reading of the logits: 4096 x 32000 f32 with entropies takes 80 us, 6.5
// TB/s.  In f64 an element takes 48 instructions, 17 of them of the 64-bit pipe,
// and 509 x 32003 with 4 alternatives 49 us: a third of the warps' places are
// taken, which leaves that pipe 46 % and the issue 57 % busy, and some SMs have
// four rows where the mean is 3.4.  (Copies into shared memory two steps ahead,
// with half as many elements of a thread at a time, took 61 us where this took
// 52: it is the number of independent exponentials that counts.)  Few rows wait
// for one memory round trip after another: 1 x 32000 f32 takes 3.7 us, with
// alternatives 5.8 to 6.4.
//
// The alternatives come from the threads' maxima: the K-th largest of them, or
// less, bounds the K-th alternative from below, so only elements at or above
// it matter.  Threads whose maximum reaches it (a few times K) read the parts
// of theirs again whose own maxima do, about 4 % of the row: going over all of
// their elements took 97 us where this took 72, and takes 63 now (1501 x 50021
// f32, 8 alternatives, half of the tokens masked).  A few dozen candidates are ranked
// by counting.  Should more than kCandidates elements reach the bound, the
// alternatives are found one after another instead, with a reading of the
// block's part for each: rows of equal values (64 x 32000 f32 with 8: 27 us for
// 7.5; 300 x 32000 with 20: 236 for 14.7; 1501 x 50021 with 8: 803 for 59), and
// rows of which a mask leaves one run so short that some warp has none of it and
// yet longer than kCandidates (700 tokens: 24, 224 and 58 us).
template <typename T, bool VEC, bool ENT, int NW, bool WIDE = false>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32, kBlocks<T, NW, WIDE>)
    log_probs_kernel(const __grid_constant__ ForwardParams<T> p) {
    constexpr int kRowsPerBlock = NW == 1 ? 4 : 1;
    constexpr int GT = NW * 32;           // threads that share a row in this block
    constexpr int VN = RowView<T, VEC>::VN;
    constexpr int U = VEC && !WIDE ? 4 : 8;     // loads in flight for each thread
    __shared__ Shared<T, NW> shared[kRowsPerBlock];
    const int lane = threadIdx.x & 31;
    const int warp = NW == 1 ? 0 : threadIdx.x >> 5;
    const int tid = NW == 1 ? lane : threadIdx.x;
    Shared<T, NW> &sh = shared[NW == 1 ? threadIdx.x >> 5 : 0];
    auto sync = [] {
        if (NW == 1) __syncwarp();
        else __syncthreads();
    };
    const int C = NW == 8 ? p.cluster : 1;    // only the widest blocks share a row
    const int rank = NW == 8 ? blockIdx.x % C : 0;
    const T c = p.factor;
    const Exp<T> ex(sh.table);
    if (sizeof(T) == 8) {
        fill(sh.table, tid);
        sync();
    }
    // the cluster's first block has to be there before the others write to it
    if (NW == 8 && C > 1) cluster_arrive();
    const int64_t step = (int64_t)(gridDim.x / C) * kRowsPerBlock;
    for (int64_t row = (int64_t)(blockIdx.x / C) * kRowsPerBlock + (NW == 1 ? threadIdx.x >> 5 : 0);
         row < p.rows.count; row += step) {
        const RowView<T, VEC> x(p.x + row_offset(p.rows, kLogits, row), p.len, p.stride);
        // the given token's logit, on its way while the row is read
        int64_t token = -1;
        if (p.log_probs && rank == 0 && tid == 0) token = p.tokens[row_offset(p.rows, kTokens, row)];
        const int per = (x.nv + C - 1) / C;
        const int v0 = min(rank * per, x.nv), v1 = min(v0 + per, x.nv);
        const bool edges = VEC && rank == 0 && warp == 0;   // the warp of the head and the tail
        const int tail0 = x.head + x.nv * VN;
        Stats<T, ENT> st;
        if (edges) {
            const T v[1] = {lane < x.head ? x.at(lane) : T(-INFINITY)};
            st.add(v, c, ex);
        }
        const int rounds = (per + GT * U - 1) / (GT * U), each = (rounds + kSlots<NW> - 1) / kSlots<NW>;
        const int slots_all = each > 0 ? (rounds + each - 1) / each : 0;
        int slots = 0, left = each;
        T most = lowest<T>();
        for (int i = v0 + tid; i < v1; i += GT * U) {
            T v[U][VN];
#pragma unroll
            for (int u = 0; u < U; ++u) x.load(i + u * GT, i + u * GT < v1, v[u]);
            most = fmax(most, st.add(reinterpret_cast<T(&)[U * VN]>(v), c, ex));
            if (p.top > 0 && --left == 0) {
                sh.slot[slots++][tid] = most;
                most = lowest<T>();
                left = each;
            }
        }
        if (left != each) sh.slot[slots++][tid] = most;
        if (edges) {
            const T v[1] = {lane >= 16 && lane < 16 + x.tail ? x.at(tail0 + lane - 16) : T(-INFINITY)};
            st.add(v, c, ex);
        }
        // its logit, now that asking for it holds up no load of the row
        const T given = token >= 0 && token < p.len ? x.at((int)token) : T(NAN);
        const T mine = st.m;
        st.template join<32>(c, ex);
        T bound = lowest<T>();
        // NW times the (K / NW)-th largest maximum of a warp are K elements
        if (NW == 1 && p.top > kWarpTop && slots_all > 1) {
            // of one warp's 32, the K-th would be too low: those of the parts
            T v = sorted_falling(slots > 0 ? sh.slot[0][lane] : lowest<T>(), lane);
            for (int q = 1; q < slots_all; ++q) {
                const T o = sorted_falling(q < slots ? sh.slot[q][lane] : lowest<T>(), lane);
                v = falling_again(larger(v, __shfl_xor_sync(0xffffffffu, o, 31)), lane);
            }
            bound = __shfl_sync(0xffffffffu, v, p.top - 1);
        } else if (p.top > 0) {
            bound = largest(mine, (p.top + NW - 1) / NW, lane);
        }
        if (NW > 1) {
            if (lane == 0) {
                sh.m[warp] = st.m;
                sh.s[warp] = st.s;
                sh.e[warp] = st.e;
                sh.bound[warp] = bound;
            }
            if (tid == 0) sh.found = 0;
            sync();
            st.m = sh.m[lane % NW];
            st.s = sh.s[lane % NW];
            st.e = sh.e[lane % NW];
            st.template join<NW>(c, ex);
            if (p.top > 0) {
#pragma unroll
                for (int w = 0; w < NW; ++w) bound = fmin(bound, sh.bound[w]);
            }
        } else {
            if (tid == 0) sh.found = 0;
            sync();
        }
        if (p.top > 0) {
            auto offer = [&](int j) {
                const int k = atomicAdd(&sh.found, 1);
                if (k < kCandidates<NW>) sh.cand[k] = Key<T>::of(x.at(j), j);
            };
            // Few threads have anything here, and each of them little: code
            // that is short to fetch counts, and an offered element is read
            // once more rather than picked out of registers.
            if (mine >= bound && st.s != T(0)) {
                unsigned wanted = 0;
#pragma unroll 4
                for (int q = 0; q < slots; ++q) wanted |= (unsigned)(sh.slot[q][tid] >= bound) << q;
                for (; wanted; wanted &= wanted - 1) {
                    const int q = __ffs(wanted) - 1;
                    for (int b = q * each; b < (q + 1) * each; ++b) {
                        const int i = v0 + tid + b * (GT * U);
                        T v[U][VN];
#pragma unroll
                        for (int u = 0; u < U; ++u) x.load(i + u * GT, i + u * GT < v1, v[u]);
                        unsigned hit = 0;
#pragma unroll
                        for (int k = 0; k < U * VN; ++k)
                            hit |= (unsigned)(v[k / VN][k % VN] >= bound && v[k / VN][k % VN] > T(-INFINITY)) << k;
                        for (; hit; hit &= hit - 1) {
                            const int k = __ffs(hit) - 1;
                            offer(x.head + (i + k / VN * GT) * VN + k % VN);
                        }
                    }
                }
                if (edges) {
                    const int j = lane < x.head ? lane : tail0 + lane - 16;
                    const bool there = lane < x.head || (lane >= 16 && lane < 16 + x.tail);
                    const T v = there ? x.at(j) : T(-INFINITY);
                    if (v >= bound && v > T(-INFINITY)) offer(j);
                }
            }
            sync();
            const int n = sh.found;
            if (n <= kCandidates<NW>) {
                for (int k = n + tid; k < p.top; k += GT) sh.best[k] = Key<T>::none(32 * rank + k);
                // Four lanes for each candidate where a row has eight warps (509
                // x 32003 f64, 4 alternatives: 49.2 us, one lane 50.7); four warps
                // have rows enough to wait for (4096 x 32000 f32: 80.6 us, with
                // the code of it in their kernel 80.8).
                constexpr int kLanes = NW == 8 ? 4 : 1;
                for (int k0 = tid / 32 * (32 / kLanes); k0 < n; k0 += GT / kLanes) {
                    const int k = k0 + lane / kLanes;
                    const Key<T> mine_k = sh.cand[min(k, n - 1)];
                    int place = 0;
#pragma unroll 8
                    for (int o = lane % kLanes; o < n; o += kLanes) place += sh.cand[o].before(mine_k);
#pragma unroll
                    for (int o = 1; o < kLanes; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
                    if (lane % kLanes == 0 && k < n && place < p.top) sh.best[place] = mine_k;
                }
            } else {
                Key<T> last = Key<T>::first();
                for (int k = 0; k < p.top; ++k) {
                    Key<T> best = Key<T>::none(32 * rank + k);
                    auto look = [&](T v, int j) {
                        const Key<T> key = Key<T>::of(v, j);
                        if (last.before(key) && key.before(best)) best = key;
                    };
                    for (int i = v0 + tid; i < v1; i += GT) {
                        T v[VN];
                        x.load(i, true, v);
#pragma unroll
                        for (int q = 0; q < VN; ++q) look(v[q], x.head + i * VN + q);
                    }
                    if (edges && lane < x.head) look(x.at(lane), lane);
                    if (edges && lane < x.tail) look(x.at(tail0 + lane), tail0 + lane);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const Key<T> other = best.lane_xor(o);
                        if (other.before(best)) best = other;
                    }
                    if (NW > 1) {
                        sync();
                        if (lane == 0) sh.cand[warp] = best;
                        sync();
#pragma unroll
                        for (int w = 0; w < NW; ++w)
                            if (sh.cand[w].before(best)) best = sh.cand[w];
                    }
                    if (tid == 0) sh.best[k] = best;
                    last = best;
                }
            }
            sync();
        }
        int total = p.top;      // alternatives in best, in order
        if (NW == 8 && C > 1) {  // one row for the cluster, which ends with it
            cg::cluster_group cluster = cg::this_cluster();
            Shared<T, NW> *first = cluster.map_shared_rank(&sh, 0);
            cluster_wait();
            if (tid == 0) {
                first->part_m[rank] = st.m;
                first->part_s[rank] = st.s;
                first->part_e[rank] = st.e;
            }
            if (tid < p.top) first->list[rank][tid] = sh.best[tid];
            cluster_arrive();
            cluster_wait();
            if (rank != 0) return;
            const int k = lane % kMaxCluster;
            st.m = k < C ? sh.part_m[k] : lowest<T>();
            st.s = k < C ? sh.part_s[k] : T(0);
            st.e = k < C ? sh.part_e[k] : T(0);
            st.template join<kMaxCluster>(c, ex);
            total = C * p.top;
        }
        // the row's answers, added up in 64 bits
        const bool bad = isnan(st.s), none = st.s == T(0);
        const double m = (double)st.m, log_s = none ? 0.0 : (double)log(st.s);
        auto log_prob = [&](T v) {
            if (bad) return T(NAN);
            if (v == T(-INFINITY)) return T(-INFINITY);
            return (T)fma((double)v - m, p.inverse, -log_s);
        };
        if (tid == 0) {
            if (p.lse) p.lse[row] = bad ? T(NAN) : none ? T(-INFINITY) : (T)fma(m, p.inverse, log_s);
            if (ENT && p.entropy)
                p.entropy[row] = bad ? T(NAN) : none ? T(0) : (T)fma((double)(st.e / st.s), -p.inverse, log_s);
            if (p.log_probs) p.log_probs[row] = token < 0 ? T(0) : token >= p.len ? T(NAN) : log_prob(given);
        }
        if (p.top > 0) {
            for (int k = tid; k < total; k += GT) {
                Key<T> key = sh.best[k % p.top];
                int at = k;
                if (NW == 8 && total > p.top) {
                    // the cluster's lists, in order each: how many elements of
                    // each come before this one, by halving, in all at once
                    key = sh.list[k / p.top][k % p.top];
                    int less[kMaxCluster] = {};
#pragma unroll 1
                    for (int by = 1 << (31 - __clz(p.top)); by > 0; by >>= 1) {
#pragma unroll
                        for (int l = 0; l < kMaxCluster; ++l) {
                            const int to = less[l] + by;
                            if (l < C && to <= p.top && sh.list[NW == 8 ? l : 0][to - 1].before(key)) less[l] = to;
                        }
                    }
                    at = 0;
#pragma unroll
                    for (int l = 0; l < kMaxCluster; ++l) at += less[l];
                    if (at >= p.top) continue;
                }
                const T v = key.value();
                p.top_lp[row * p.top + at] = log_prob(v);
                p.top_ids[row * p.top + at] = bad || v == T(-INFINITY) ? -1 : key.place();
            }
        }
        sync();     // the next row's candidates overwrite these
    }
}

template <typename T> struct BackwardParams {
    const T *x, *lse, *entropy, *g_lp, *g_h, *g_lse;
    const int64_t *tokens;
    T *out;
    int64_t stride;
    int len, per, parts;     // elements of one block's part of a row; parts of a row
    T factor;                // exp_factor(temperature)
    double temperature, inverse;
    double trusted;          // lse_trusted(temperature)
    T before;                // before x after = 1 / temperature
    double after;
    Rows rows;
};

// A row's lse is known to half a step of its own size; beyond 256 that would
// show in the probabilities, and the row's maximum and sum are taken anew
// instead.  So they are where T lse, which at temperatures near the type's
// largest number need not be finite in it, is beyond a quarter of that number's
// last place: a logit of the type's lowest value less T lse is finite.
template <typename T> double lse_trusted(T temperature) {
    using Limits = std::numeric_limits<T>;
    return std::min(256.0, (double)Limits::max() * ((double)Limits::epsilon() / 8) / (double)temperature);
}

// A row's numbers in the gradient of its elements:
//   l = (x - base) c - less, which is log p in the exponential's units,
//   dx = p (a - b l)  [+ at the token]
template <typename T> struct RowGrad {
    T base, less, a, b, at_token;
    T nothing;      // of an element whose probability is 0: NaN where the row's numbers are
    int token;
    __device__ __forceinline__ T operator()(T v, T c, const Exp<T> &ex) const {
        const T l = fma(v - base, c, -less);
        if constexpr (sizeof(T) == 4) {
            const T d = ex(l) * fma(-b, larger(l, T(-1e5)), a);
            return v == T(-INFINITY) ? T(0) : d;
        } else {
            if (Exp<T>::counts(l)) return ex(l) * fma(-b, l, a);
            return v == T(-INFINITY) ? T(0) : nothing;
        }
    }
};

// The vectors lo to hi (one by one without VEC) of a row, by GT threads, first
// the loads of a thread's first round, then everything else: the row's own
// numbers come from memory meanwhile.
template <typename T, bool VEC, int GT> struct GradPart {
    static constexpr int VN = RowView<T, VEC>::VN;
    static constexpr int U = VEC ? 4 : 64 / (int)sizeof(T);   // 64 bytes in flight for each thread
    T v[U][VN];
    const int lo, hi, tid;

    __device__ __forceinline__ GradPart(const RowView<T, VEC> &x, int lo_, int hi_, int tid_)
        : lo(lo_), hi(hi_), tid(tid_) {
        load(x, lo + tid);
    }
    __device__ __forceinline__ void load(const RowView<T, VEC> &x, int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) x.load(i + u * GT, i + u * GT < hi, v[u]);
    }
    __device__ __forceinline__ void run(const RowView<T, VEC> &x, T *out, const RowGrad<T> &g, T c, const Exp<T> &ex,
                                        bool first, bool last) {
        for (int i = lo + tid; i < hi; i += GT * U) {
            if (i != lo + tid) load(x, i);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = x.head + (i + u * GT) * VN;
                T d[VN];
#pragma unroll
                for (int k = 0; k < VN; ++k) d[k] = g(v[u][k], c, ex);
                if ((unsigned)(g.token - j) < (unsigned)VN) {
#pragma unroll
                    for (int k = 0; k < VN; ++k)
                        if (g.token == j + k && v[u][k] != T(-INFINITY)) d[k] += g.at_token;
                }
                if (i + u * GT < hi) {
                    if (VEC)
                        *reinterpret_cast<typename Vec<T>::type *>(out + j) =
                            *reinterpret_cast<const typename Vec<T>::type *>(d);
                    else
                        out[j] = d[0];
                }
            }
        }
        if (VEC && first && tid < x.head) one(x, out, tid, g, c, ex);
        if (VEC && last && tid < x.tail) one(x, out, x.head + x.nv * VN + tid, g, c, ex);
    }
    __device__ __forceinline__ static void one(const RowView<T, VEC> &x, T *out, int j, const RowGrad<T> &g, T c,
                                               const Exp<T> &ex) {
        const T value = x.at(j);
        T d = g(value, c, ex);
        if (j == g.token && value != T(-INFINITY)) d += g.at_token;
        out[j] = d;
    }
};

constexpr int kGradThreads = 256, kGradBlocks = 4;    // threads of a block, blocks of an SM

// A row's numbers for its gradient, by the NW warps that share it.
template <typename T, int NW>
__device__ __forceinline__ RowGrad<T> row_grad(const BackwardParams<T> &p, int64_t row, const T *xr, int64_t stride, int tid, T *sm,
                                               T *ss, const Exp<T> &ex) {
    const double unit = Exp<T>::unit;
    const double lse = (double)p.lse[row_offset(p.rows, kLse, row)];
    const int64_t t = p.tokens ? p.tokens[row_offset(p.rows, kTokens, row)] : -1;
    T gp = p.g_lp ? p.g_lp[row_offset(p.rows, kGradLp, row)] : T(0);
    T gh = p.g_h ? p.g_h[row_offset(p.rows, kGradH, row)] : T(0);
    const T h = p.g_h ? p.entropy[row_offset(p.rows, kEntropy, row)] : T(0);
    T gl = p.g_lse ? p.g_lse[row_offset(p.rows, kGradLse, row)] : T(0);
    RowGrad<T> g;
    if (fabs(lse) <= p.trusted) {
        const double b = lse * p.temperature;
        g.base = (T)b;
        g.less = (T)((b - (double)g.base) * (p.inverse * unit));
    } else {
        Stats<T, false> st;
        constexpr int U = 64 / (int)sizeof(T);
        const RowView<T, false> x(xr, p.len, stride);
        for (int j = tid; j < p.len; j += NW * 32 * U) {
            T v[U][1];
#pragma unroll
            for (int u = 0; u < U; ++u) x.load(j + u * NW * 32, j + u * NW * 32 < p.len, v[u]);
            st.add(reinterpret_cast<T(&)[U]>(v), p.factor, ex);
        }
        st.template join<32>(p.factor, ex);
        if (NW > 1) {
            __syncthreads();
            if ((tid & 31) == 0) {
                sm[tid >> 5] = st.m;
                ss[tid >> 5] = st.s;
            }
            __syncthreads();
            st.m = sm[tid % NW];
            st.s = ss[tid % NW];
            st.template join<NW>(p.factor, ex);
        }
        // a NaN or +inf in the row: NaN by way of g.a, and log p of -inf for a logit of -inf
        const bool bad = isnan(st.s);
        g.base = bad ? T(0) : st.m;
        g.less = bad || st.s == T(0) ? T(0) : (T)(log((double)st.s) * unit);
        if (bad) gl = T(NAN);
    }
    if (t < 0) gp = T(0);
    if (t >= p.len) gp = T(NAN);
    gp *= p.before;
    gh *= p.before;
    gl *= p.before;
    g.a = (T)((double)(gl - gp - gh * h) * p.after);
    g.b = (T)((double)gh * (p.after / unit));
    g.at_token = (T)((double)gp * p.after);
    g.nothing = g.a * T(0);
    g.token = t >= 0 && t < p.len ? (int)t : -1;
    return g;
}

// The gradient: one element in, one out, with a row's few numbers between
// them.  The bound is the two streams: 4096 x 32000 f32 takes 164 us, 6.4
// TB/s, and 169 where the two lie differently against 16 bytes.  A row that is
// taken anew is read once more by each of its parts: with lse = 600, at T =
// 0.05, the same takes 218 us, 8 x 131072 19.1 us for 3.8 and 1 x 131072 15.7 for
// 3.4.  At 64 registers a thread the f64 forms spill 56 to 132 bytes, the f32
// forms 32 at most.  A block takes a
// part of one row: parts of 32000 elements there, where parts of 8192 took 190 us
// and of 2048 343, as each begins with its row's numbers; or each of its warps a
// short row (4096 x 1000: 8 us, with a block for each row 23).
template <typename T, bool VEC, int NW>
__global__ void __launch_bounds__(kGradThreads, kGradBlocks)
    log_probs_backward_kernel(const __grid_constant__ BackwardParams<T> p) {
    constexpr int GT = NW * 32;
    constexpr int kGroups = kGradThreads / GT;
    __shared__ T sm[NW], ss[NW];
    __shared__ typename Exp<T>::Table table;
    const Exp<T> ex(table);
    if (sizeof(T) == 8) {
        fill(table, threadIdx.x);
        __syncthreads();
    }
    const int tid = threadIdx.x % GT;
    const int64_t total = p.rows.count * p.parts;
    for (int64_t w = (int64_t)blockIdx.x * kGroups + threadIdx.x / GT; w < total; w += (int64_t)gridDim.x * kGroups) {
        const int64_t row = w >> 32 ? w / p.parts : (uint32_t)w / (uint32_t)p.parts;
        const int part = (int)(w - row * p.parts);
        const T *xr = p.x + row_offset(p.rows, kLogits, row);
        T *out = p.out + row * p.len;
        const bool first = part == 0, last = part + 1 == p.parts;
        // vectors where logits and gradient lie alike against 16 bytes
        if (VEC && ((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
            const RowView<T, true> x(xr, p.len, p.stride);
            const int per = p.per / RowView<T, true>::VN, lo = min(part * per, x.nv);
            GradPart<T, true, GT> g(x, lo, last ? x.nv : min(lo + per, x.nv), tid);
            const RowGrad<T> numbers = row_grad<T, NW>(p, row, xr, VEC ? 1 : p.stride, tid, sm, ss, ex);
            g.run(x, out, numbers, p.factor, ex, first, last);
        } else {
            const RowView<T, false> x(xr, p.len, VEC ? 1 : p.stride);
            const int lo = min(part * p.per, p.len);
            GradPart<T, false, GT> g(x, lo, last ? p.len : min(lo + p.per, p.len), tid);
            const RowGrad<T> numbers = row_grad<T, NW>(p, row, xr, VEC ? 1 : p.stride, tid, sm, ss, ex);
            g.run(x, out, numbers, p.factor, ex, first, last);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
const char *const kFwd = "token_log_probs";
const char *const kBwd = "token_log_probs_backward";

constexpr int64_t kMaxGrid = 1 << 30;
// Longest row that one warp takes: where there are more rows than blocks of
// eight warps at once 16 KB (4096 x 2048 f32 with 8 alternatives: 12 us, with a
// block for each row 19; 4096 x 8192 with 20: 38 and 37; 1000 x 2048 f64 12 and
// 12), else what gives each thread of such a block less than 16 bytes (64 x
// 2000 f32 with 8 alternatives: 8.2 us, in blocks 6.2).
constexpr int kWarpRowBytes = 16384, kWarpRow = 1024;
constexpr int kWideRow = 16384;     // shortest row with eight loads in flight
// Longest row of the gradient that one warp takes: 4096 x 2000 f32 13 us, in
// blocks 27; 4096 x 4096 29 us, in blocks 27.
constexpr int kGradWarpRow = 2048;
// Elements of a block's part of a row in the gradient: no fewer, for the few
// rows that are cut for the SMs' sake (8 x 30208 f32: 5.5 us, in parts of 16384
// 7.5), and no more, for the last blocks to end together (2000 x 100000: 247 us,
// whole rows 257).
constexpr int kGradPartLeast = 4096, kGradPartMost = 32768;
// The temperature divides logits: it and its reciprocal are normal numbers.
template <typename T> bool temperature_ok(T t) {
    return std::isnormal((double)t) && t > T(0) && std::isnormal(exp_factor<T>(t));
}

// An operand with one element for each row: the logits' dims without the last.
int check_rows(const kx_tensor *t, const kx_tensor *logits, uint32_t es, const char *op, const char *name, Span *s,
               kx_error *err) {
    int rc = validate_tensor(t, es, s, err);
    if (rc) return rc;
    bool same = t->rank + 1 == logits->rank;
    for (uint32_t i = 0; same && i < t->rank; ++i) same = t->dims[i] == logits->dims[i];
    if (!same) return set_err(err, KX_E_PARAM, op, name);
    return KX_OK;
}

// An output: C-contiguous, clear of the inputs seen so far.
struct Seen {
    const void *data[8];
    Span span[8];
    uint32_t es[8];
    bool written[8];
    int n = 0;
    int add(const kx_tensor *t, const Span &s, uint32_t e, bool out, const char *op, kx_error *err) {
        const uintptr_t a0 = (uintptr_t)t->data + s.start * e, a1 = (uintptr_t)t->data + s.end * e;
        for (int i = 0; i < n && !s.empty; ++i) {
            if (span[i].empty || !(out || written[i])) continue;
            const uintptr_t b0 = (uintptr_t)data[i] + span[i].start * es[i],
                            b1 = (uintptr_t)data[i] + span[i].end * es[i];
            if (a0 < b1 && b0 < a1) return set_err(err, KX_E_ALIAS, op, "output overlaps another operand");
        }
        data[n] = t->data;
        span[n] = s;
        es[n] = e;
        written[n++] = out;
        return KX_OK;
    }
};

// Leading dims with their strides in every operand; size-one dims dropped, and
// neighbours that every operand walks as one merged.
struct RowsBuilder {
    Rows g;
    explicit RowsBuilder(const kx_tensor *logits) {
        std::memset(&g, 0, sizeof(g));
        g.count = 1;
        for (uint32_t d = 0; d + 1 < logits->rank; ++d) g.count *= (int64_t)logits->dims[d];
        int n = 0;
        for (uint32_t d = 0; d + 1 < logits->rank; ++d)
            if (logits->dims[d] != 1) g.dims[n++] = (int64_t)logits->dims[d];
        g.ndims = n;
    }
    void operand(int which, const kx_tensor *t, const kx_tensor *logits) {
        int n = 0;
        for (uint32_t d = 0; t && d + 1 < logits->rank; ++d)
            if (logits->dims[d] != 1) g.str[which][n++] = t->strides[d];
    }
    Rows done() {
        int w = 0;
        for (int d = 0; d < g.ndims; ++d) {
            bool merge = w > 0;
            for (int k = 0; merge && k < kRowOperands; ++k) merge = g.str[k][w - 1] == (i128)g.str[k][d] * g.dims[d];
            if (merge) {
                g.dims[w - 1] *= g.dims[d];
            } else {
                g.dims[w] = g.dims[d];
                ++w;
            }
            for (int k = 0; k < kRowOperands; ++k) g.str[k][w - 1] = g.str[k][d];
        }
        g.ndims = w;
        return g;
    }
};

template <typename E> E *at(const kx_tensor *t) { return t ? static_cast<E *>(t->data) + t->origin : nullptr; }

template <typename T>
int check_logits(const kx_tensor *logits, T temperature, const char *op, Span *s, kx_error *err) {
    if (!temperature_ok(temperature))
        return set_err(err, KX_E_PARAM, op, "temperature (must be finite and > 0, as must its reciprocal)");
    int rc = validate_tensor(logits, sizeof(T), s, err);
    if (rc) return rc;
    if (logits->rank == 0) return set_err(err, KX_E_INVALID_RANK, op, "rank", 1, 0);
    if (logits->dims[logits->rank - 1] > (1u << 30))
        return set_err(err, KX_E_UNSUPPORTED, op, "vocabulary above 2^30");
    // with an empty vocabulary the rows alone need not fit the element count
    rc = validate_dims(logits->dims, logits->rank - 1, err);
    if (rc) return rc;
    if (numel(logits->dims, logits->rank - 1) > kIsizeMax)
        return set_err(err, KX_E_UNSUPPORTED, op, "too many rows");
    return KX_OK;
}

int row_output(const kx_tensor *t, const kx_tensor *logits, uint32_t es, const char *op, const char *name, Seen *seen,
               kx_error *err) {
    if (!t) return KX_OK;
    Span s;
    int rc = validate_tensor(t, es, &s, err);
    if (rc) return rc;
    bool same = t->rank + 1 == logits->rank;
    for (uint32_t i = 0; same && i < t->rank; ++i) same = t->dims[i] == logits->dims[i];
    if (!same) return set_err(err, KX_E_LAYOUT, op, name, KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
    if (!is_c_contiguous(t))
        return set_err(err, KX_E_LAYOUT, op, "output must be C-contiguous", KX_LAYOUT_OUTPUT_NOT_C_CONTIGUOUS);
    return seen->add(t, s, es, true, op, err);
}

// Elements from which on another part of a row is worth its merging where the
// device has room for both: 296 x 17000 f64 with 8 alternatives takes 22.5 us in
// two parts, 19.3 in one.
template <typename T> constexpr int kLongPart = sizeof(T) == 4 ? 16384 : 12288;

template <typename T, bool VEC, bool ENT>
void launch_forward(Handle *h, ForwardParams<T> &p) {
    const int64_t at_once = (int64_t)kBlocks<T, 8, false> * h->sm_count;
    const bool many = p.rows.count > at_once;
    if (p.len <= (many ? kWarpRowBytes / (int)sizeof(T) : kWarpRow)) {
        const int64_t blocks = (p.rows.count + 3) / 4;
        log_probs_kernel<T, VEC, ENT, 1><<<(unsigned)std::min<int64_t>(blocks, kMaxGrid), 128, 0, h->stream>>>(p);
        h->last_kernel = "log_probs_warp";
        return;
    }
    // Rows that blocks of eight warps take at once have one each, or a cluster:
    // for the SMs that would have nothing (1 x 131072 f32: 6 us in eight parts,
    // 16 in one), or for long parts (64 x 131072: 10 us, with four parts 12; 200 x
    // 32003 f64 with 8 alternatives: 24.7 us, in one part 27.4).
    // More rows than that go to blocks of four warps: twice as many rows are on
    // their way at once while others end (4096 x 16384 with 20 alternatives:
    // 60 us, with eight warps 67; 600 x 65536: 36 us, with eight warps 30).
    // Long f32 rows have eight loads of each thread in flight, with eight such
    // blocks on an SM instead of ten, unless more places would stay empty in the
    // last round of rows than that gains (about 7 %): 1000 x 131072 with 8
    // alternatives 88 us, with four loads 94; 1300 x 50021 59 and 51; 4096 x
    // 10000 45 and 41.
    if (many) {
        h->last_kernel = "log_probs_block4";
        const unsigned grid = (unsigned)std::min<int64_t>(p.rows.count, kMaxGrid);
        if constexpr (sizeof(T) == 4 && VEC) {
            auto places = [&](int blocks) {
                const int64_t n = (int64_t)blocks * h->sm_count;
                return (p.rows.count + n - 1) / n * n;
            };
            if (p.len >= kWideRow && places(kBlocks<T, 4, true>) * 100 <= places(kBlocks<T, 4, false>) * 107) {
                log_probs_kernel<T, VEC, ENT, 4, true><<<grid, 128, 0, h->stream>>>(p);
                h->last_kernel = "log_probs_block4_wide";
                return;
            }
        }
        log_probs_kernel<T, VEC, ENT, 4><<<grid, 128, 0, h->stream>>>(p);
        return;
    }
    while (p.cluster < kMaxCluster) {
        const int64_t blocks = p.rows.count * p.cluster, piece = p.len / (2 * p.cluster);
        if (!(blocks < h->sm_count && piece >= 4096) && !(2 * blocks <= at_once && piece >= kLongPart<T>)) break;
        p.cluster *= 2;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows.count * p.cluster));
    cfg.blockDim = dim3(256);
    cfg.stream = h->stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, log_probs_kernel<T, VEC, ENT, 8>, p);
    h->last_kernel = p.cluster > 1 ? "log_probs_cluster" : "log_probs_block8";
}

// Into how many parts the gradient cuts a row: `wanted` or a few more, so that
// the last round of blocks is short or full, where each part costs the time of
// 13 KB beside its own elements (300 x 40000 f64: 42 us, in two parts 51; 700 x
// 20011 f64 52 and 57, f32 23 and 24; with 8 KB 2000 x 9000 f64 would be cut in two:
// 68 us, whole 63).
template <typename T> int parts_of_least_time(const Handle *h, int64_t rows, int64_t len, int64_t wanted) {
    const int64_t places = (int64_t)kGradBlocks * h->sm_count, most = std::max<int64_t>(1, len / kGradPartLeast);
    const int64_t from = std::min(std::max<int64_t>(1, wanted), most), to = std::min(from + 3, most);
    int64_t parts = from, least = INT64_MAX;
    for (int64_t n = from; n <= to; ++n) {
        const int64_t rounds = (rows * n + places - 1) / places;
        const int64_t time = rounds * (len / n + 13 * 1024 / (int64_t)sizeof(T));
        if (time < least) {
            least = time;
            parts = n;
        }
    }
    return (int)parts;
}

template <typename T, bool VEC, int NW> void launch_backward(Handle *h, const BackwardParams<T> &p) {
    constexpr int kGroups = kGradThreads / (NW * 32);
    const i128 groups = (i128)p.rows.count * p.parts;
    const unsigned grid = (unsigned)std::min<i128>((groups + kGroups - 1) / kGroups, kMaxGrid);
    log_probs_backward_kernel<T, VEC, NW><<<grid, kGradThreads, 0, h->stream>>>(p);
    h->last_kernel = NW == 1 ? "log_probs_backward_warp" : "log_probs_backward_block";
}

template <typename T>
int forward_impl(kx_handle *hh, const kx_tensor *logits, const kx_tensor *tokens, T temperature,
                 const kx_tensor *log_probs, const kx_tensor *lse, const kx_tensor *entropy,
                 const kx_tensor *top_log_probs, const kx_tensor *top_tokens, kx_error *err) {
    if (!hh) return set_err(err, KX_E_PARAM, kFwd, "null handle");
    Handle *h = &hh->impl;
    Span s;
    int rc = check_logits<T>(logits, temperature, kFwd, &s, err);
    if (rc) return rc;
    Seen seen;
    rc = seen.add(logits, s, sizeof(T), false, kFwd, err);
    if (rc) return rc;
    if ((tokens != nullptr) != (log_probs != nullptr))
        return set_err(err, KX_E_PARAM, kFwd, "tokens and log_probs go together");
    if ((top_log_probs != nullptr) != (top_tokens != nullptr))
        return set_err(err, KX_E_PARAM, kFwd, "top_log_probs and top_tokens go together");
    if (!log_probs && !lse && !entropy && !top_log_probs) return set_err(err, KX_E_PARAM, kFwd, "no output");
    if (tokens) {
        rc = check_rows(tokens, logits, 8, kFwd, "tokens (one for each row of logits)", &s, err);
        if (!rc) rc = seen.add(tokens, s, 8, false, kFwd, err);
        if (rc) return rc;
    }
    rc = row_output(log_probs, logits, sizeof(T), kFwd, "log_probs shape mismatch", &seen, err);
    if (!rc) rc = row_output(lse, logits, sizeof(T), kFwd, "lse shape mismatch", &seen, err);
    if (!rc) rc = row_output(entropy, logits, sizeof(T), kFwd, "entropy shape mismatch", &seen, err);
    if (rc) return rc;
    uint64_t top = 0;
    if (top_log_probs) {
        const kx_tensor *both[2] = {top_log_probs, top_tokens};
        for (const kx_tensor *t : both) {
            const uint32_t es = t == top_log_probs ? (uint32_t)sizeof(T) : 8u;
            rc = validate_tensor(t, es, &s, err);
            if (rc) return rc;
            bool same = t->rank == logits->rank;
            for (uint32_t i = 0; same && i + 1 < t->rank; ++i) same = t->dims[i] == logits->dims[i];
            same = same && t->dims[t->rank - 1] == top_log_probs->dims[top_log_probs->rank - 1];
            if (!same)
                return set_err(err, KX_E_LAYOUT, kFwd, "alternatives shape mismatch", KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
            if (!is_c_contiguous(t))
                return set_err(err, KX_E_LAYOUT, kFwd, "output must be C-contiguous",
                               KX_LAYOUT_OUTPUT_NOT_C_CONTIGUOUS);
            rc = seen.add(t, s, es, true, kFwd, err);
            if (rc) return rc;
        }
        top = top_log_probs->dims[top_log_probs->rank - 1];
        if (top > kMaxTop) return set_err(err, KX_E_PARAM, kFwd, "top (at most 32 alternatives)");
    }
    RowsBuilder rows(logits);
    if (rows.g.count == 0) return KX_OK;
    ForwardParams<T> p;
    std::memset(&p, 0, sizeof(p));
    rows.operand(kLogits, logits, logits);
    rows.operand(kTokens, tokens, logits);
    p.rows = rows.done();
    p.x = at<T>(logits);
    p.tokens = at<int64_t>(tokens);
    p.log_probs = at<T>(log_probs);
    p.lse = at<T>(lse);
    p.entropy = at<T>(entropy);
    p.top_lp = at<T>(top_log_probs);
    p.top_ids = at<int64_t>(top_tokens);
    p.len = (int)logits->dims[logits->rank - 1];
    p.stride = logits->strides[logits->rank - 1];
    p.top = (int)top;
    p.inverse = 1.0 / (double)temperature;
    p.factor = exp_factor<T>(temperature);
    p.cluster = 1;
    DeviceGuard guard(h->device);
    if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, kFwd, "cannot select device");
    const bool vec = p.stride == 1 || p.len <= 1;
    if (vec) entropy ? launch_forward<T, true, true>(h, p) : launch_forward<T, true, false>(h, p);
    else entropy ? launch_forward<T, false, true>(h, p) : launch_forward<T, false, false>(h, p);
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, kFwd);
    }
    ++h->launches;
    return KX_OK;
}

template <typename T>
int backward_impl(kx_handle *hh, const kx_tensor *logits, const kx_tensor *tokens, const kx_tensor *lse,
                  const kx_tensor *entropy, const kx_tensor *grad_log_probs, const kx_tensor *grad_entropy,
                  const kx_tensor *grad_lse, T temperature, const kx_tensor *grad_logits, kx_error *err) {
    if (!hh) return set_err(err, KX_E_PARAM, kBwd, "null handle");
    Handle *h = &hh->impl;
    Span s;
    int rc = check_logits<T>(logits, temperature, kBwd, &s, err);
    if (rc) return rc;
    Seen seen;
    rc = seen.add(logits, s, sizeof(T), false, kBwd, err);
    if (rc) return rc;
    if (!grad_log_probs && !grad_entropy && !grad_lse) return set_err(err, KX_E_PARAM, kBwd, "no incoming gradient");
    if (!lse) return set_err(err, KX_E_PARAM, kBwd, "lse (the forward pass's is needed)");
    if (grad_log_probs && !tokens) return set_err(err, KX_E_PARAM, kBwd, "tokens (needed with grad_log_probs)");
    if (grad_entropy && !entropy) return set_err(err, KX_E_PARAM, kBwd, "entropy (needed with grad_entropy)");
    const struct {
        const kx_tensor *t;
        uint32_t es;
        const char *name;
    } ins[] = {{tokens, 8, "tokens (one for each row of logits)"},
               {lse, sizeof(T), "lse (one for each row of logits)"},
               {entropy, sizeof(T), "entropy (one for each row of logits)"},
               {grad_log_probs, sizeof(T), "grad_log_probs (one for each row of logits)"},
               {grad_entropy, sizeof(T), "grad_entropy (one for each row of logits)"},
               {grad_lse, sizeof(T), "grad_lse (one for each row of logits)"}};
    for (const auto &in : ins) {
        if (!in.t) continue;
        rc = check_rows(in.t, logits, in.es, kBwd, in.name, &s, err);
        if (!rc) rc = seen.add(in.t, s, in.es, false, kBwd, err);
        if (rc) return rc;
    }
    rc = validate_tensor(grad_logits, sizeof(T), &s, err);
    if (rc) return rc;
    bool same = grad_logits->rank == logits->rank;
    for (uint32_t i = 0; same && i < logits->rank; ++i) same = grad_logits->dims[i] == logits->dims[i];
    if (!same) return set_err(err, KX_E_LAYOUT, kBwd, "output shape mismatch", KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
    if (!is_c_contiguous(grad_logits))
        return set_err(err, KX_E_LAYOUT, kBwd, "output must be C-contiguous", KX_LAYOUT_OUTPUT_NOT_C_CONTIGUOUS);
    rc = seen.add(grad_logits, s, sizeof(T), true, kBwd, err);
    if (rc) return rc;
    if (numel(logits->dims, logits->rank) == 0) return KX_OK;
    RowsBuilder rows(logits);
    BackwardParams<T> p;
    std::memset(&p, 0, sizeof(p));
    rows.operand(kLogits, logits, logits);
    rows.operand(kTokens, grad_log_probs ? tokens : nullptr, logits);
    rows.operand(kLse, lse, logits);
    rows.operand(kEntropy, grad_entropy ? entropy : nullptr, logits);
    rows.operand(kGradLp, grad_log_probs, logits);
    rows.operand(kGradH, grad_entropy, logits);
    rows.operand(kGradLse, grad_lse, logits);
    p.rows = rows.done();
    p.x = at<T>(logits);
    p.tokens = grad_log_probs ? at<int64_t>(tokens) : nullptr;
    p.lse = at<T>(lse);
    p.entropy = grad_entropy ? at<T>(entropy) : nullptr;
    p.g_lp = at<T>(grad_log_probs);
    p.g_h = at<T>(grad_entropy);
    p.g_lse = at<T>(grad_lse);
    p.out = at<T>(grad_logits);
    p.len = (int)logits->dims[logits->rank - 1];
    p.stride = logits->strides[logits->rank - 1];
    p.temperature = (double)temperature;
    p.inverse = 1.0 / (double)temperature;
    p.trusted = lse_trusted(temperature);
    // Gradients as large as a large temperature come out small, but their sum and
    // the product with an entropy (21 at most) need not fit the type.  Beside 2^64
    // nothing that the factor pushes below the normal numbers would be seen.
    p.before = (double)temperature < 0x1p64 ? T(1) : T(1) / 64;
    p.after = 1.0 / ((double)p.before * (double)temperature);
    p.factor = exp_factor<T>(temperature);
    DeviceGuard guard(h->device);
    if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, kBwd, "cannot select device");
    const bool vec = p.stride == 1 || p.len <= 1;
    if (p.len <= kGradWarpRow) {
        p.per = p.len;
        p.parts = 1;
        vec ? launch_backward<T, true, 1>(h, p) : launch_backward<T, false, 1>(h, p);
    } else {
        // even parts, as many as the device takes at once, or of the longest size
        const int64_t wanted = std::max<int64_t>((int64_t)kGradBlocks * h->sm_count / p.rows.count,
                                                 (p.len + kGradPartMost - 1) / kGradPartMost);
        p.parts = parts_of_least_time<T>(h, p.rows.count, p.len, wanted);
        p.per = ((p.len + p.parts - 1) / p.parts + 15) / 16 * 16;
        p.parts = (p.len + p.per - 1) / p.per;
        vec ? launch_backward<T, true, kGradThreads / 32>(h, p) : launch_backward<T, false, kGradThreads / 32>(h, p);
    }
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, kBwd);
    }
    ++h->launches;
    return KX_OK;
}

}  // namespace

extern "C" {
int kx_token_log_probs_f32(kx_handle *h, const kx_tensor *logits, const kx_tensor *tokens, float temperature,
                           const kx_tensor *log_probs, const kx_tensor *lse, const kx_tensor *entropy,
                           const kx_tensor *top_log_probs, const kx_tensor *top_tokens, kx_error *err) {
    return forward_impl<float>(h, logits, tokens, temperature, log_probs, lse, entropy, top_log_probs, top_tokens, err);
}
int kx_token_log_probs_f64(kx_handle *h, const kx_tensor *logits, const kx_tensor *tokens, double temperature,
                           const kx_tensor *log_probs, const kx_tensor *lse, const kx_tensor *entropy,
                           const kx_tensor *top_log_probs, const kx_tensor *top_tokens, kx_error *err) {
    return forward_impl<double>(h, logits, tokens, temperature, log_probs, lse, entropy, top_log_probs, top_tokens,
                                err);
}
int kx_token_log_probs_backward_f32(kx_handle *h, const kx_tensor *logits, const kx_tensor *tokens,
                                    const kx_tensor *lse, const kx_tensor *entropy, const kx_tensor *grad_log_probs,
                                    const kx_tensor *grad_entropy, const kx_tensor *grad_lse, float temperature,
                                    const kx_tensor *grad_logits, kx_error *err) {
    return backward_impl<float>(h, logits, tokens, lse, entropy, grad_log_probs, grad_entropy, grad_lse, temperature,
                                grad_logits, err);
}
int kx_token_log_probs_backward_f64(kx_handle *h, const kx_tensor *logits, const kx_tensor *tokens,
                                    const kx_tensor *lse, const kx_tensor *entropy, const kx_tensor *grad_log_probs,
                                    const kx_tensor *grad_entropy, const kx_tensor *grad_lse, double temperature,
                                    const kx_tensor *grad_logits, kx_error *err) {
    return backward_impl<double>(h, logits, tokens, lse, entropy, grad_log_probs, grad_entropy, grad_lse, temperature,
                                 grad_logits, err);
}
}
