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
#include <cfloat>
#include <cmath>
#include <cstring>

#include "kx_internal.hpp"

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

template <typename T> __device__ __forceinline__ T kexp(T x);
template <> __device__ __forceinline__ float kexp<float>(float x) { return expf(x); }
template <> __device__ __forceinline__ double kexp<double>(double x) { return exp(x); }

// The smallest (x - m)/T that enters a sum: exp of it is 0 in either type, and
// 0 times it is 0 where 0 times -inf would be NaN.
template <typename T> __device__ __forceinline__ T floor_of(T d) { return fmax(d, T(-1e5)); }

template <typename T> struct ForwardParams {
    const T *x;
    const int64_t *tokens;
    T *log_probs, *lse, *entropy, *top_lp;
    int64_t *top_ids;
    int64_t len, stride;
    int top;
    T temperature;
    Rows rows;
};

template <typename T>
__device__ __forceinline__ T block_sum(T v, T *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T s = T(0);
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
    return s;
}

template <typename T>
__device__ __forceinline__ T block_max(T v, T *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T s = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) s = fmax(s, red[w]);
    return s;
}

// Maximum, sum of exponentials and sum of exponential times difference of one
// row, by all threads of the block.
template <typename T>
__device__ void row_stats(const T *x, int64_t len, int64_t stride, T temperature, T *red, T &m, T &s, T &e) {
    m = -INFINITY;
    for (int64_t j = threadIdx.x; j < len; j += blockDim.x) m = fmax(m, x[j * stride]);
    m = block_max(m, red);
    const T base = m == T(-INFINITY) ? T(0) : m;
    s = T(0);
    e = T(0);
    for (int64_t j = threadIdx.x; j < len; j += blockDim.x) {
        const T d = (x[j * stride] - base) / temperature;
        const T p = kexp(d);
        s += p;
        e += p * floor_of(d);
    }
    s = block_sum(s, red);
    e = block_sum(e, red);
}

template <typename T>
__global__ void __launch_bounds__(256) log_probs_kernel(const __grid_constant__ ForwardParams<T> p) {
    __shared__ T red[8];
    __shared__ T best_v[8];
    __shared__ int64_t best_i[8];
    for (int64_t row = blockIdx.x; row < p.rows.count; row += gridDim.x) {
        const T *x = p.x + row_offset(p.rows, kLogits, row);
        T m, s, e;
        row_stats(x, p.len, p.stride, p.temperature, red, m, s, e);
        const bool bad = isnan(s), none = !bad && m == T(-INFINITY);
        const double log_s = log((double)s);
        if (threadIdx.x == 0) {
            if (p.lse) p.lse[row] = bad ? T(NAN) : none ? T(-INFINITY) : (T)((double)m / (double)p.temperature + log_s);
            if (p.entropy) p.entropy[row] = bad ? T(NAN) : none ? T(0) : (T)(log_s - (double)e / (double)s);
            if (p.log_probs) {
                const int64_t t = p.tokens[row_offset(p.rows, kTokens, row)];
                T lp = T(0);
                if (t >= p.len) lp = T(NAN);
                else if (t >= 0)
                    lp = bad ? T(NAN) : none ? T(-INFINITY)
                             : (T)(((double)x[t * p.stride] - (double)m) / (double)p.temperature - log_s);
                p.log_probs[row] = lp;
            }
        }
        // the alternatives, one pass each: the best element after the last one
        T last_v = INFINITY;
        int64_t last_i = -1;
        for (int k = 0; k < p.top; ++k) {
            T v = -INFINITY;
            int64_t i = INT64_MAX;
            if (!bad) {
                for (int64_t j = threadIdx.x; j < p.len; j += blockDim.x) {
                    const T c = x[j * p.stride];
                    if ((c < last_v || (c == last_v && j > last_i)) && (c > v || (c == v && j < i))) {
                        v = c;
                        i = j;
                    }
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const T ov = __shfl_xor_sync(0xffffffffu, v, o);
                const int64_t oi = __shfl_xor_sync(0xffffffffu, i, o);
                if (ov > v || (ov == v && oi < i)) {
                    v = ov;
                    i = oi;
                }
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 0) {
                best_v[threadIdx.x >> 5] = v;
                best_i[threadIdx.x >> 5] = i;
            }
            __syncthreads();
            v = best_v[0];
            i = best_i[0];
            for (int w = 1; w < 8; ++w)
                if (best_v[w] > v || (best_v[w] == v && best_i[w] < i)) {
                    v = best_v[w];
                    i = best_i[w];
                }
            if (threadIdx.x == 0) {
                const bool gone = v == T(-INFINITY);
                p.top_lp[row * p.top + k] =
                    bad ? T(NAN) : gone ? T(-INFINITY)
                                        : (T)(((double)v - (double)m) / (double)p.temperature - log_s);
                p.top_ids[row * p.top + k] = bad || gone ? -1 : i;
            }
            last_v = v;
            last_i = i;
        }
        __syncthreads();
    }
}

template <typename T> struct BackwardParams {
    const T *x, *lse, *entropy, *g_lp, *g_h, *g_lse;
    const int64_t *tokens;
    T *out;
    int64_t len, stride;
    T temperature;
    Rows rows;
};

// A row's lse is known to half a step of its own size; beyond this size that
// would show in the probabilities, and the row's maximum and sum are taken
// anew instead.
constexpr double kLseTrusted = 256.0;

template <typename T>
__global__ void __launch_bounds__(256) log_probs_backward_kernel(const __grid_constant__ BackwardParams<T> p) {
    __shared__ T red[8];
    for (int64_t row = blockIdx.x; row < p.rows.count; row += gridDim.x) {
        const T *x = p.x + row_offset(p.rows, kLogits, row);
        T *out = p.out + row * p.len;
        const double lse = (double)p.lse[row_offset(p.rows, kLse, row)];
        T base, less;   // log p = (x - base)/T - less
        if (fabs(lse) <= kLseTrusted) {
            const double b = lse * (double)p.temperature;
            base = (T)b;
            less = (T)((b - (double)base) / (double)p.temperature);
        } else {
            T m, s, e;
            row_stats(x, p.len, p.stride, p.temperature, red, m, s, e);
            base = m;
            less = isnan(s) ? T(NAN) : (T)log((double)s);
        }
        const int64_t t = p.tokens ? p.tokens[row_offset(p.rows, kTokens, row)] : -1;
        T g = p.g_lp && t >= 0 ? p.g_lp[row_offset(p.rows, kGradLp, row)] : T(0);
        const T gh = p.g_h ? p.g_h[row_offset(p.rows, kGradH, row)] : T(0);
        const T h = p.g_h ? p.entropy[row_offset(p.rows, kEntropy, row)] : T(0);
        const T gl = p.g_lse ? p.g_lse[row_offset(p.rows, kGradLse, row)] : T(0);
        if (p.g_lp && t >= p.len) g = T(NAN);
        const T factor = (gl - g - gh * h) / p.temperature;
        const T gh_t = gh / p.temperature, g_t = g / p.temperature;
        for (int64_t j = threadIdx.x; j < p.len; j += blockDim.x) {
            const T v = x[j * p.stride];
            const T lq = (v - base) / p.temperature - less;
            const T q = kexp(lq);
            T d = q * (factor - gh_t * floor_of(lq));
            if (j == t) d += g_t;
            out[j] = v == T(-INFINITY) ? T(0) : d;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
const char *const kFwd = "token_log_probs";
const char *const kBwd = "token_log_probs_backward";

// The temperature divides logits: it and its reciprocal are normal numbers.
template <typename T> bool temperature_ok(T t) {
    return std::isnormal((double)t) && t > T(0) && std::isnormal((T)(T(1.4426950408889634) / t));
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
    if (logits->dims[logits->rank - 1] > (uint64_t)INT32_MAX)
        return set_err(err, KX_E_UNSUPPORTED, op, "vocabulary above 2^31-1");
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
    p.len = (int64_t)logits->dims[logits->rank - 1];
    p.stride = logits->strides[logits->rank - 1];
    p.top = (int)top;
    p.temperature = temperature;
    DeviceGuard guard(h->device);
    if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, kFwd, "cannot select device");
    const int64_t cap = 16LL * h->sm_count;
    const unsigned grid = (unsigned)(p.rows.count < cap ? p.rows.count : cap);
    log_probs_kernel<T><<<grid, 256, 0, h->stream>>>(p);
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, kFwd);
    }
    ++h->launches;
    h->last_kernel = "log_probs";
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
    p.len = (int64_t)logits->dims[logits->rank - 1];
    p.stride = logits->strides[logits->rank - 1];
    p.temperature = temperature;
    DeviceGuard guard(h->device);
    if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, kBwd, "cannot select device");
    const int64_t cap = 16LL * h->sm_count;
    const unsigned grid = (unsigned)(p.rows.count < cap ? p.rows.count : cap);
    log_probs_backward_kernel<T><<<grid, 256, 0, h->stream>>>(p);
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, kBwd);
    }
    ++h->launches;
    h->last_kernel = "log_probs_backward";
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
