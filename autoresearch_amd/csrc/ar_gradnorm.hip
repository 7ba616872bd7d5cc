// ar_gradnorm.hip -- the norm of all gradients together, and clipping by it:
//   norm = sqrt(sum over all tensors of g^2), out = g min(1, max_norm / norm).
// Bound by HBM: the gradients are read once for the norm, read again to be
// scaled and written.  Sums are fp64 in a fixed order, so that the norm is
// right for gradients anywhere in fp32's range and the same every time.
// 201 MB in 60 tensors: norm 31.5 us (6.4 TB/s), scaling 64 us (6.3 TB/s).
#include <math.h>

#include <algorithm>
#include <new>

#include "ar_losses.hpp"

namespace ar {
namespace {

constexpr int kClipBlock = 256;
constexpr int kClipTensors = 124;                            // per launch: the table is a kernel argument
constexpr int kClipBlocks = 2048;                            // of 256 lanes with at most 64 registers: all resident
constexpr int kClipBatch = 4;                                // loads of 16 bytes that a lane has in flight
constexpr int64_t kClipUnit = 4096;                          // bytes a tensor takes up of the shares, at least
constexpr int64_t kClipStep = kClipBatch * kClipBlock * 16;  // shares are whole batches (46 MB: 16.4 -> 15.8 us)

// The tensors of a launch one after the other, each on a whole number of
// units; block b works on bytes [b share, (b + 1) share) of that, whatever
// tensors lie there, so that all blocks but the last have the same to do.
struct ClipTable {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    int64_t size[kClipTensors];       // elements
    int32_t start[kClipTensors + 1];  // units
    uint8_t bf16[kClipTensors];
    int32_t n;
};
static_assert(sizeof(ClipTable) <= 3800, "kernel arguments hold 4 KiB");

// f(tensor, first element, last element + 1) for the tensors in a block's share.
template <typename F>
__device__ __forceinline__ void each_tensor(const ClipTable& t, int64_t b, int64_t share, F f) {
    const int64_t end = min((b + 1) * share, t.start[t.n] * kClipUnit);
    int64_t at = b * share;
    int j = 0, hi = t.n - 1;
    while (j < hi) {
        const int mid = (j + hi + 1) / 2;
        if (t.start[mid] * kClipUnit <= at) j = mid;
        else hi = mid - 1;
    }
    for (; at < end; at = t.start[++j] * kClipUnit) {
        const int64_t es = t.bf16[j] ? 2 : 4, base = t.start[j] * kClipUnit;
        const int64_t lo = (at - base) / es, to = (min(end, t.start[j + 1] * kClipUnit) - base) / es;
        if (lo < t.size[j]) f(j, lo, min(to, t.size[j]));
    }
}

// f(chunk's first element, chunk) for every whole chunk of in[lo .. hi), and
// g(element, value) for the values behind the last one.
template <typename T, typename F, typename G>
__device__ __forceinline__ void each(const void* base, int64_t lo, int64_t hi, F f, G g) {
    using R = Row<T>;
    constexpr int64_t E = R::E, step = kClipBlock * E;
    const T* in = static_cast<const T*>(base);
    int64_t i = lo + threadIdx.x * E;
    for (; i + (kClipBatch - 1) * step + E <= hi; i += kClipBatch * step) {
        u32x4 q[kClipBatch];
#pragma unroll
        for (int k = 0; k < kClipBatch; ++k) q[k] = R::load(in + i + k * step);
#pragma unroll
        for (int k = 0; k < kClipBatch; ++k) f(i + k * step, q[k]);
    }
    for (; i + E <= hi; i += step) f(i, R::load(in + i));
    for (int64_t j = hi - (hi - lo) % E + threadIdx.x; j < hi; j += kClipBlock) g(j, to_f32<T>(in[j]));
}

template <typename T>
__device__ __forceinline__ double sum_squares(const void* in, int64_t lo, int64_t hi) {
    double s = 0.0;
    auto add = [&](float v) { s = fma((double)v, (double)v, s); };
    each<T>(in, lo, hi,
            [&](int64_t, u32x4 q) {
#pragma unroll
                for (int e = 0; e < Row<T>::E; ++e) add(Row<T>::get(q, e));
            },
            [&](int64_t, float v) { add(v); });
    return s;
}
template <typename T>
__device__ __forceinline__ void scale(const void* in, void* out, int64_t lo, int64_t hi, double c) {
    T* o = static_cast<T*>(out);
    each<T>(in, lo, hi,
            [&](int64_t i, u32x4 q) {
                float x[Row<T>::E];
#pragma unroll
                for (int e = 0; e < Row<T>::E; ++e) x[e] = (float)(Row<T>::get(q, e) * c);
                Row<T>::store_nt(o + i, Row<T>::pack(x));
            },
            [&](int64_t i, float v) { o[i] = from_f32<T>((float)(v * c)); });
}

__global__ __launch_bounds__(kClipBlock, 8) void clip_sum_k(ClipTable t, int64_t share, double* part) {
    __shared__ double red[kClipBlock / kWave];
    double s = 0.0;
    each_tensor(t, blockIdx.x, share, [&](int j, int64_t lo, int64_t hi) {
        s += t.bf16[j] ? sum_squares<bf16>(t.in[j], lo, hi) : sum_squares<float>(t.in[j], lo, hi);
    });
    s = block_total(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// Every block sums the np partials in the same order.  A norm that is not
// finite clips nothing.
__global__ __launch_bounds__(kClipBlock, 8) void clip_scale_k(ClipTable t, int64_t share, const double* part,
                                                              int64_t np, double max_norm, float* norm_out) {
    __shared__ double red[kClipBlock / kWave];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < np; i += kClipBlock) s += part[i];
    const double norm = sqrt(block_total(s, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
    if (t.n == 0) return;
    const double c = norm > max_norm && norm < INFINITY ? max_norm / norm : 1.0;
    // back to front: what the sums read last is the likeliest still cached
    each_tensor(t, gridDim.x - 1 - blockIdx.x, share, [&](int j, int64_t lo, int64_t hi) {
        if (c == 1.0 && t.in[j] == t.out[j]) return;
        if (t.bf16[j]) scale<bf16>(t.in[j], t.out[j], lo, hi, c);
        else scale<float>(t.in[j], t.out[j], lo, hi, c);
    });
}

struct Range {
    uintptr_t lo, hi;
    bool written;
};

// Whether a tensor is written while another one, or part of its own input,
// lies there too (a tensor clipped in place is one range).
int32_t check_overlap(const char* nm, void* const* outs, const void* const* grads, const int32_t* grads_bf16,
                      const int64_t* sizes, int64_t n) {
    Range* r = new (std::nothrow) Range[2 * n + 1];
    if (!r) return set_error(AR_ENOMEM, "%s: no host memory for %lld tensors", nm, (long long)n);
    int64_t k = 0;
    for (int64_t j = 0; j < n; ++j) {
        const size_t bytes = (size_t)sizes[j] * (grads_bf16 && grads_bf16[j] ? 2 : 4);
        if (!bytes) continue;
        const uintptr_t in = reinterpret_cast<uintptr_t>(grads[j]);
        const uintptr_t out = outs ? reinterpret_cast<uintptr_t>(outs[j]) : in;
        r[k++] = Range{out, out + bytes, true};
        if (out != in) r[k++] = Range{in, in + bytes, false};
    }
    std::sort(r, r + k, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t end_all = 0, end_written = 0;
    bool bad = false;
    for (int64_t i = 0; i < k; ++i) {
        bad = bad || r[i].lo < (r[i].written ? end_all : end_written);
        end_all = std::max(end_all, r[i].hi);
        if (r[i].written) end_written = std::max(end_written, r[i].hi);
    }
    delete[] r;
    AR_CHECK_ARG(!bad, "%s: tensors that are written overlap each other or the gradients", nm);
    return AR_OK;
}

int64_t clip_units(const int32_t* grads_bf16, const int64_t* sizes, int64_t j) {
    return cdiv(sizes[j] * (grads_bf16 && grads_bf16[j] ? 2 : 4), kClipUnit);
}
int64_t clip_share(const int32_t* grads_bf16, const int64_t* sizes, int64_t n) {
    int64_t total = 0;
    for (int64_t j = 0; j < n; ++j) total += clip_units(grads_bf16, sizes, j) * kClipUnit;
    const int64_t steps = cdiv(cdiv(total, kClipBlocks), kClipStep);
    return (steps < 1 ? 1 : steps) * kClipStep;
}
// The next launch's tensors, from j on; how many blocks they are.
int64_t clip_table(ClipTable& t, int64_t& j, void* const* outs, const void* const* grads, const int32_t* grads_bf16,
                   const int64_t* sizes, int64_t n, int64_t share) {
    t.n = 0;
    t.start[0] = 0;
    for (; j < n && t.n < kClipTensors; ++j) {
        if (sizes[j] == 0) continue;
        t.in[t.n] = grads[j];
        t.out[t.n] = outs ? outs[j] : const_cast<void*>(grads[j]);
        t.size[t.n] = sizes[j];
        t.bf16[t.n] = grads_bf16 && grads_bf16[j];
        t.start[t.n + 1] = (int32_t)(t.start[t.n] + clip_units(grads_bf16, sizes, j));
        ++t.n;
    }
    return cdiv(t.start[t.n] * kClipUnit, share);
}

}  // namespace

int64_t clip_partials(int64_t n) {  // a launch's last block is shorter than its share
    return kClipBlocks + cdiv(n, kClipTensors);
}

int32_t clip_grads(hipStream_t st, float* norm_out, void* const* outs, const void* const* grads,
                   const int32_t* grads_bf16, const int64_t* sizes, int64_t n, double max_norm, double* part) {
    const int64_t share = clip_share(grads_bf16, sizes, n);
    bool write = false;  // whether there is anything to write: a bound, or an output elsewhere
    for (int64_t j = 0; j < n; ++j)
        write = write || (sizes[j] && (max_norm < INFINITY || (outs && outs[j] != grads[j])));
    ClipTable t;
    int64_t np = 0;
    for (int64_t j = 0; j < n;)
        if (const int64_t b = clip_table(t, j, outs, grads, grads_bf16, sizes, n, share)) {
            clip_sum_k<<<(unsigned)b, kClipBlock, 0, st>>>(t, share, part + np);
            np += b;
        }
    bool norm_done = false;
    for (int64_t j = 0; j < n && write;)
        if (const int64_t b = clip_table(t, j, outs, grads, grads_bf16, sizes, n, share)) {
            clip_scale_k<<<(unsigned)b, kClipBlock, 0, st>>>(t, share, part, np, max_norm,
                                                             norm_done ? nullptr : norm_out);
            norm_done = true;
        }
    if (!norm_done) {
        t.n = 0;
        clip_scale_k<<<1, kClipBlock, 0, st>>>(t, share, part, np, max_norm, norm_out);
    }
    return check_launch("clip_grad_norm");
}

}  // namespace ar

using namespace ar;

extern "C" int32_t ar_clip_grad_norm(ar_stream_t stream, float* norm_out, void* const* outputs,
                                     const void* const* grads, const int32_t* grads_bf16, const int64_t* sizes,
                                     int64_t num_tensors, double max_norm) {
    const char* nm = "clip_grad_norm";
    AR_CHECK_ARG(norm_out && (num_tensors <= 0 || (grads && sizes)), "%s: null pointer", nm);
    AR_CHECK_ARG(num_tensors >= 0 && num_tensors <= (1 << 24), "%s: bad number of tensors", nm);
    AR_CHECK_ARG(max_norm > 0.0, "%s: max_norm must be positive", nm);
    for (int64_t j = 0; j < num_tensors; ++j) {
        const int32_t b = grads_bf16 ? grads_bf16[j] : 0;
        AR_CHECK_ARG(b == 0 || b == 1, "%s: grads_bf16[%lld] must be 0 or 1", nm, (long long)j);
        AR_CHECK_ARG(sizes[j] >= 0 && sizes[j] <= (int64_t(1) << 32), "%s: bad size of tensor %lld", nm, (long long)j);
        AR_CHECK_ARG(sizes[j] == 0 || (grads[j] && (!outputs || outputs[j])), "%s: null tensor %lld", nm,
                     (long long)j);
        const uintptr_t mis = reinterpret_cast<uintptr_t>(grads[j]) |
                              (outputs ? reinterpret_cast<uintptr_t>(outputs[j]) : uintptr_t(0));
        AR_CHECK_ARG(sizes[j] == 0 || (mis & (b ? 1 : 3)) == 0, "%s: tensor %lld not aligned to a value", nm,
                     (long long)j);
    }
    if (const int32_t r = check_overlap(nm, outputs, grads, grads_bf16, sizes, num_tensors)) return r;
    int32_t status;
    double* part = static_cast<double*>(
        workspace(S(stream), (size_t)clip_partials(num_tensors) * sizeof(double), &status));
    if (!part) return status;
    return clip_grads(S(stream), norm_out, outputs, grads, grads_bf16, sizes, num_tensors, max_norm, part);
}
