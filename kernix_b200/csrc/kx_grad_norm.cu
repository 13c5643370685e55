// The 2-norm over all elements of a list of gradients, and the gradients
// scaled down to a largest norm.
//
//   norm = sqrt(sum over all tensors of g^2),  out = g * min(1, max_norm / norm)
//
// Squares are added in 64 bits in an order that only the sizes and the device
// fix, so the same gradients give the same bits again.  A norm that is not
// finite scales nothing: the outputs are the gradients as they were.
#include <algorithm>
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

// One tensor (and its scaled copy) as C-order dims with each one's strides.
struct Geom {
    int rank;
    int64_t count;
    int64_t dims[KX_MAX_RANK], src[KX_MAX_RANK], dst[KX_MAX_RANK];
};

__device__ __forceinline__ void offsets(const Geom &g, int64_t i, int64_t &so, int64_t &d_o) {
    so = d_o = 0;
    for (int d = g.rank - 1; d >= 0; --d) {
        const int64_t q = i / g.dims[d], c = i - q * g.dims[d];
        so += c * g.src[d];
        d_o += c * g.dst[d];
        i = q;
    }
}

__device__ double block_total(double v) {
    __shared__ double red[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) s += red[w];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sum_squares_kernel(const T *__restrict__ x, const __grid_constant__ Geom g,
                                                               double *partial) {
    double s = 0.0;
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < g.count; i += (int64_t)gridDim.x * kThreads) {
        int64_t so, d_o;
        offsets(g, i, so, d_o);
        const double v = (double)x[so];
        s = fma(v, v, s);
    }
    s = block_total(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The norm and the scale from the partial sums, by one block.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(const double *partial, int64_t n, double max_norm, T *norm,
                                                        double *scale) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) s += partial[i];
    s = sqrt(block_total(s));
    if (threadIdx.x == 0) {
        *norm = (T)s;
        *scale = isfinite(s) && s > max_norm ? max_norm / s : 1.0;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) scale_kernel(const T *x, T *out, const __grid_constant__ Geom g,
                                                         const double *scale) {
    const T c = (T)*scale;
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < g.count; i += (int64_t)gridDim.x * kThreads) {
        int64_t so, d_o;
        offsets(g, i, so, d_o);
        out[d_o] = x[so] * c;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kPartials = 512;   // most blocks of one launch

uint64_t workspace_bytes(uint64_t count) { return (count + 1) * kPartials * sizeof(double); }

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
    if (count > (1u << 24)) return set_err(err, KX_E_UNSUPPORTED, op, "more than 2^24 gradients");
    Span s;
    int rc = validate_tensor(norm, sizeof(T), &s, err);
    if (rc) return rc;
    if (numel(norm->dims, norm->rank) != 1)
        return set_err(err, KX_E_LAYOUT, op, "norm (one element)", KX_LAYOUT_OUTPUT_SHAPE_MISMATCH);
    if (!workspace || bytes < workspace_bytes(count) || (uintptr_t)workspace % 8)
        return set_err(err, KX_E_PARAM, op, "workspace (8-byte aligned, of the size asked for)");
    std::vector<Range> all;
    all.reserve(2 * count + 2);
    auto add = [&](const kx_tensor *t, const Span &sp, bool out) {
        if (!sp.empty)
            all.push_back({(uintptr_t)t->data + sp.start * sizeof(T), (uintptr_t)t->data + sp.end * sizeof(T), out});
    };
    add(norm, s, true);
    all.push_back({(uintptr_t)workspace, (uintptr_t)workspace + workspace_bytes(count), true});
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

Geom geom(const kx_tensor *g, const kx_tensor *o) {
    Geom r;
    std::memset(&r, 0, sizeof(r));
    r.rank = (int)g->rank;
    r.count = (int64_t)numel(g->dims, g->rank);
    for (uint32_t d = 0; d < g->rank; ++d) {
        r.dims[d] = (int64_t)g->dims[d];
        r.src[d] = g->dims[d] > 1 ? g->strides[d] : 0;
        r.dst[d] = o && g->dims[d] > 1 ? o->strides[d] : 0;
    }
    return r;
}

unsigned blocks_for(int64_t count) {
    const int64_t b = (count + kThreads * 8 - 1) / (kThreads * 8);
    return (unsigned)std::min<int64_t>((int64_t)kPartials, std::max<int64_t>(b, 1));
}

template <typename T>
int norm_impl(kx_handle *hh, const kx_tensor *grads, uint64_t count, double max_norm, const kx_tensor *outs,
              const kx_tensor *norm, void *workspace, uint64_t bytes, const char *op, kx_error *err) {
    if (!hh) return set_err(err, KX_E_PARAM, op, "null handle");
    Handle *h = &hh->impl;
    if (outs && !(std::isfinite(max_norm) && max_norm > 0.0))
        return set_err(err, KX_E_PARAM, op, "max_norm (must be finite and > 0)");
    int rc;
    try {
        rc = check_lists<T>(grads, count, outs, norm, workspace, bytes, op, err);
    } catch (const std::bad_alloc &) {
        rc = set_err(err, KX_E_PARAM, op, "out of host memory");
    }
    if (rc) return rc;
    DeviceGuard guard(h->device);
    if (!guard.ok) return set_err(err, KX_E_NO_DEVICE, op, "cannot select device");
    double *scale = static_cast<double *>(workspace), *partial = scale + 1;
    int64_t used = 0;
    for (uint64_t i = 0; i < count; ++i) {
        const Geom g = geom(&grads[i], nullptr);
        if (g.count == 0) continue;
        const unsigned nb = blocks_for(g.count);
        sum_squares_kernel<T><<<nb, kThreads, 0, h->stream>>>(at<T>(&grads[i]), g, partial + used);
        ++h->launches;
        used += nb;
    }
    norm_kernel<T><<<1, kThreads, 0, h->stream>>>(partial, used, max_norm, at<T>(norm), scale);
    ++h->launches;
    for (uint64_t i = 0; outs && i < count; ++i) {
        const Geom g = geom(&grads[i], &outs[i]);
        if (g.count == 0) continue;
        scale_kernel<T><<<blocks_for(g.count), kThreads, 0, h->stream>>>(at<T>(&grads[i]), at<T>(&outs[i]), g, scale);
        ++h->launches;
    }
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) {
        h->cuda_fail(ce);
        return cuda_err(err, h, op);
    }
    h->last_kernel = op;
    return KX_OK;
}

}  // namespace

extern "C" {
int kx_grad_norm_workspace(uint64_t count, uint64_t *bytes) {
    if (!bytes || count > (1u << 24)) return KX_E_PARAM;
    *bytes = workspace_bytes(count);
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
