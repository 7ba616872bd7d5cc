// ar_logprob.hip -- log-probabilities of tokens from rows of logits, and the
// gradients that go back through them.
//
// A row z [V] with target y: lse = m + log sum_j exp(z_j - m), m = max_j z_j,
// logp = z_y - lse, and for a loss with gradient g by logp
//   d loss / d x_j = g ([j = y] - exp(z_j - lse)) (1 - (z_j / cap)^2),
// the last factor the derivative of z = cap tanh(x / cap) (1 without a cap).
// Bound by HBM: a row is read once (the running maximum and sum need one
// pass) and a row of the gradient written once.
#include <math.h>

#include "ar_losses.hpp"

namespace ar {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of a row: E values.  Rows start at any multiple of a value's size
// (any V, any view), which the vector accesses say.
template <typename T>
struct Row;
template <>
struct Row<float> {
    static constexpr int E = 4;
    typedef u32x4 vec __attribute__((aligned(4)));
    static __device__ __forceinline__ float get(u32x4 v, int i) { return __uint_as_float(v[i]); }
    static __device__ __forceinline__ u32x4 pack(const float* x) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(x[i]);
        return v;
    }
    static __device__ __forceinline__ u32x4 load(const float* p) { return *reinterpret_cast<const vec*>(p); }
    static __device__ __forceinline__ void store(float* p, u32x4 v) { *reinterpret_cast<vec*>(p) = v; }
    static __device__ __forceinline__ u32x4 fill(float x) { return u32x4{1, 1, 1, 1} * __float_as_uint(x); }
};
template <>
struct Row<bf16> {
    static constexpr int E = 8;
    typedef u32x4 vec __attribute__((aligned(2)));
    static __device__ __forceinline__ float get(u32x4 v, int i) {
        return __uint_as_float((i & 1) ? (v[i / 2] & 0xffff0000u) : (v[i / 2] << 16));
    }
    static __device__ __forceinline__ u32x4 pack(const float* x) {
        bf16x8 b;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (bf16)x[i];
        return __builtin_bit_cast(u32x4, b);
    }
    static __device__ __forceinline__ u32x4 load(const bf16* p) { return *reinterpret_cast<const vec*>(p); }
    static __device__ __forceinline__ void store(bf16* p, u32x4 v) { *reinterpret_cast<vec*>(p) = v; }
    static __device__ __forceinline__ u32x4 fill(float x) { return u32x4{1, 1, 1, 1} * (__float_as_uint(x) >> 16) * 0x10001u; }
};

// A row's values in chunks of 16 bytes: h values before them, V - tail0 < E
// behind them.  Accesses of 16 bytes cost the same at any multiple of 4 bytes
// (rows of 50001 fp32 values: 169 us either way), but more at odd multiples of
// 2: bf16 rows leave out their first value there (8191 x 32003: 221 -> 205 us).
template <typename T>
struct Span {
    int h, nb, tail0;
    __device__ __forceinline__ Span(const T* row, int V)
        : h(sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(row) & 2) ? 1 : 0),
          nb((V - h) / Row<T>::E),
          tail0(h + nb * Row<T>::E) {}
    // The value outside the chunks that thread i holds; -1: none.
    __device__ __forceinline__ int edge(int i, int V) const {
        return i < h ? i : i >= Row<T>::E && i - Row<T>::E < V - tail0 ? tail0 + i - Row<T>::E : -1;
    }
};

// The maximum so far and the sum of exp(z - m) under it.
struct MaxSum {
    float m = -INFINITY, s = 0.f;
    __device__ __forceinline__ void add(float om, float os) {
        const float nm = fmaxf(m, om);
        if (nm == -INFINITY) {
            s += os;  // both empty, or NaN
            return;
        }
        s = s * __expf(m - nm) + os * __expf(om - nm);
        m = nm;
    }
};
__device__ __forceinline__ MaxSum block_max_sum(MaxSum v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float om = __shfl_xor(v.m, o, kWave), os = __shfl_xor(v.s, o, kWave);
        v.add(om, os);
    }
    const int w = threadIdx.x / kWave, nw = blockDim.x / kWave;
    if (nw == 1) return v;
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
        red[2 * w] = v.m;
        red[2 * w + 1] = v.s;
    }
    __syncthreads();
    MaxSum t;
    for (int i = 0; i < nw; ++i) t.add(red[2 * i], red[2 * i + 1]);
    return t;
}

// What a token's gradient by its log-probability is, and for POLICY its terms;
// by one thread of a workgroup.
template <LpOp OP>
__device__ __forceinline__ float row_coef(const LpRows& a, int64_t r, float w, float logp) {
    if constexpr (OP == LpOp::POLICY) {
        const PolicyTerm t = policy_term(logp, r, a.policy);
        if (a.logp) a.logp[r] = logp;
        a.terms[r] = make_double2(w * t.loss, w * t.kl);
        return (float)(w * t.g * a.loss_scale);
    }
    return w;
}

// The gradient of a value that is not the target: -g p f; the target's has
// g f besides, f = 1 - (z / cap)^2.
struct RowGrad {
    float m, gs, rcap;  // gs = g / sum
    __device__ __forceinline__ RowGrad(const LpRows& a, float g, MaxSum v)
        : m(v.m), gs(-g / v.s), rcap(a.cap > 0.f ? 1.f / a.cap : 0.f) {}
    __device__ __forceinline__ float factor(float z) const {
        const float u = z * rcap;
        return fmaxf(0.f, fmaf(-u, u, 1.f));
    }
    __device__ __forceinline__ float operator()(float z) const { return gs * __expf(z - m) * factor(z); }
    __device__ __forceinline__ float target(float z, float g) const { return fmaf(gs, __expf(z - m), g) * factor(z); }
};

template <typename T>
__device__ __forceinline__ void zero_row(T* out, int V) {
    using R = Row<T>;
    const int nb = V / R::E;
    for (int c = threadIdx.x; c < nb; c += blockDim.x) R::store(out + c * R::E, u32x4{0, 0, 0, 0});
    for (int j = nb * R::E + threadIdx.x; j < V; j += blockDim.x) out[j] = from_f32<T>(0.f);
}

// Whether a token's logits are read; if not, its outputs are written here.
template <typename T, LpOp OP>
__device__ __forceinline__ bool row_counts(const LpRows& a, int64_t r, int64_t y, float& w) {
    w = 1.f;
    if constexpr (OP == LpOp::BWD) w = a.grad_logp[r];
    if constexpr (OP == LpOp::POLICY) w = a.weight[r];
    if (y >= 0 && y < a.V && w != 0.f) return true;
    if constexpr (OP != LpOp::BWD)
        if (threadIdx.x == 0 && a.logp) a.logp[r] = 0.f;
    if constexpr (OP == LpOp::POLICY)
        if (threadIdx.x == 0) a.terms[r] = make_double2(0.0, 0.0);
    if constexpr (OP != LpOp::FWD) zero_row(static_cast<T*>(a.grad) + r * a.V, (int)a.V);
    return false;
}

// The maximum and sum of 16 bytes of a row.
template <typename T>
__device__ __forceinline__ void add_chunk(MaxSum& v, u32x4 q) {
    using R = Row<T>;
    float cm = R::get(q, 0);
#pragma unroll
    for (int i = 1; i < R::E; ++i) cm = fmaxf(cm, R::get(q, i));
    const float use = fmaxf(v.m, cm) == -INFINITY ? 0.f : fmaxf(v.m, cm);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < R::E; ++i) s += __expf(R::get(q, i) - use);
    v.add(cm == -INFINITY ? -INFINITY : use, s);
}

// Between two passes over held chunks: what the first one made of them (bf16
// values widened to fp32: twice the registers) is made again, not kept.
__device__ __forceinline__ void again(u32x4& q) { asm volatile("" : "+v"(q)); }

constexpr int kRowBlock = 256;

// Rows of any length: the row is read again for the gradient.
template <typename T, LpOp OP>
__global__ __launch_bounds__(kRowBlock) void lp_row_k(LpRows a) {
    using R = Row<T>;
    constexpr int E = R::E;
    __shared__ float red[2 * kRowBlock / kWave];
    __shared__ float coef;
    const int64_t r = blockIdx.x;
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    T* out = static_cast<T*>(a.grad) + r * a.V;
    float w;
    if (!row_counts<T, OP>(a, r, y, w)) return;
    const Span<T> sp(row, V);
    const int h = sp.h, nb = sp.nb, ej = sp.edge(tid, V);
    const float zy = to_f32<T>(row[y]), ez = ej >= 0 ? to_f32<T>(row[ej]) : -INFINITY;
    MaxSum v;
    for (int c = tid; c < nb; c += kRowBlock) add_chunk<T>(v, R::load(row + h + c * E));
    v.add(ez, ez == -INFINITY ? 0.f : __expf(ez - ez));
    v = block_max_sum(v, red);
    if constexpr (OP == LpOp::FWD) {
        if (tid == 0) a.logp[r] = (zy - v.m) - logf(v.s);
        return;
    }
    if (tid == 0) coef = row_coef<OP>(a, r, w, (zy - v.m) - logf(v.s));
    __syncthreads();  // zy and the sums are read: from here the row may be overwritten
    const float g = coef;
    const RowGrad grad(a, g, v);
    for (int c = tid; c < nb; c += kRowBlock) {
        const u32x4 q = R::load(row + h + c * E);
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = h + c * E + i == y ? grad.target(zy, g) : grad(R::get(q, i));
        R::store(out + h + c * E, R::pack(x));
    }
    if (ej >= 0) out[ej] = from_f32<T>(ej == y ? grad.target(zy, g) : grad(ez));
}

// The same for rows of up to NV TB chunks of 16 bytes, held in registers: one
// read, and the maximum before the exponentials.
template <typename T, LpOp OP, int TB, int NV>
__global__ __launch_bounds__(TB, NV > 8 ? 4 : 6) void lp_held_k(LpRows a) {
    using R = Row<T>;
    constexpr int E = R::E;
    __shared__ float red[2 * (TB / kWave)];
    __shared__ float coef;
    const int64_t r = blockIdx.x;
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    T* out = static_cast<T*>(a.grad) + r * a.V;
    float w;
    if (!row_counts<T, OP>(a, r, y, w)) return;
    const Span<T> sp(row, V);
    const int h = sp.h, nb = sp.nb;
    const u32x4 none = R::fill(-INFINITY);
    u32x4 q[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (k * TB < nb) {
            const int c = tid + k * TB;
            q[k] = R::load(row + h + min(c, nb - 1) * E);
        }
    const int ej = sp.edge(tid, V);
    const float ez = ej >= 0 ? to_f32<T>(row[ej]) : -INFINITY;
    const float zy = to_f32<T>(row[y]);
    float mt = ez;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (k * TB < nb) {
            if (tid + k * TB >= nb) q[k] = none;
#pragma unroll
            for (int i = 0; i < E; ++i) mt = fmaxf(mt, R::get(q[k], i));
            again(q[k]);
        }
    MaxSum v;
    v.m = block_max(mt, red);
    const float use = v.m == -INFINITY ? 0.f : v.m;
    float st = __expf(ez - use);
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (k * TB < nb) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s += __expf(R::get(q[k], i) - use);
            st += s;
            again(q[k]);
        }
    v.s = block_sum(st, red + TB / kWave);
    if (tid == 0) coef = row_coef<OP>(a, r, w, (zy - v.m) - logf(v.s));
    __syncthreads();
    const float g = coef;
    const RowGrad grad(a, g, v);
    const int yc = y < h ? -1 : ((int)y - h) / E, yi = y < h ? 0 : ((int)y - h) % E;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (k * TB < nb) {
            const int c = tid + k * TB;
            float x[E];
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = grad(R::get(q[k], i));
            if (c == yc) {
                const float t = grad.target(zy, g);
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = i == yi ? t : x[i];
            }
            if (c < nb) R::store(out + h + c * E, R::pack(x));
        }
    if (ej >= 0) out[ej] = from_f32<T>(ej == y ? grad.target(zy, g) : grad(ez));
}

template <typename T, LpOp OP>
void launch_grad(hipStream_t st, const LpRows& a) {
    const unsigned g = (unsigned)a.n;
    const int64_t nc = cdiv(a.V, Row<T>::E);
    if (nc <= 128) lp_held_k<T, OP, 64, 2><<<g, 64, 0, st>>>(a);
    else if (nc <= 512) lp_held_k<T, OP, 64, 8><<<g, 64, 0, st>>>(a);
    else if (nc <= 2048) lp_held_k<T, OP, 256, 8><<<g, 256, 0, st>>>(a);
    else if (nc <= 4096) lp_held_k<T, OP, 256, 16><<<g, 256, 0, st>>>(a);
    else if (nc <= 8192) lp_held_k<T, OP, 512, 16><<<g, 512, 0, st>>>(a);
    else if (nc <= 16384) lp_held_k<T, OP, 1024, 16><<<g, 1024, 0, st>>>(a);
    else lp_row_k<T, OP><<<g, kRowBlock, 0, st>>>(a);
}

template <typename T>
int32_t launch(hipStream_t st, LpOp op, const LpRows& a, const char* nm) {
    if (op == LpOp::FWD) lp_row_k<T, LpOp::FWD><<<(unsigned)a.n, kRowBlock, 0, st>>>(a);
    else if (op == LpOp::BWD) launch_grad<T, LpOp::BWD>(st, a);
    else launch_grad<T, LpOp::POLICY>(st, a);
    return check_launch(nm);
}

}  // namespace

int32_t lp_rows(hipStream_t st, LpOp op, bool bf16_logits, const LpRows& a, const char* nm) {
    if (a.n == 0) return AR_OK;
    return bf16_logits ? launch<bf16>(st, op, a, nm) : launch<float>(st, op, a, nm);
}

int32_t check_rows(const char* nm, const void* logits, int32_t logits_bf16, const void* grad, const int64_t* targets,
                   int64_t n, int64_t V) {
    AR_CHECK_ARG(n >= 0 && V > 0, "%s: bad shape", nm);
    AR_CHECK_ARG(n == 0 || (logits && targets), "%s: null pointer", nm);
    AR_CHECK_ARG(logits_bf16 == 0 || logits_bf16 == 1, "%s: logits_bf16 must be 0 or 1", nm);
    if (n > INT32_MAX || V > INT32_MAX / 2)
        return set_error(AR_EUNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^30 logits per token", nm);
    const size_t es = logits_bf16 ? 2 : 4, bytes = (size_t)n * V * es;
    AR_CHECK_ARG(((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(grad)) & (es - 1)) == 0,
                 "%s: logits or their gradient not aligned to a value", nm);
    AR_CHECK_ARG(grad == logits || !overlaps(grad, bytes, logits, bytes),
                 "%s: the gradient overlaps the logits without being them", nm);
    return AR_OK;
}

}  // namespace ar

using namespace ar;

extern "C" int32_t ar_token_logprob_fwd(ar_stream_t stream, float* logp_out, const void* logits, int32_t logits_bf16,
                                        const int64_t* targets, int64_t num_tokens, int64_t vocab_size) {
    AR_CHECK_ARG(num_tokens <= 0 || logp_out, "token_logprob_fwd: null pointer");
    if (const int32_t r = check_rows("token_logprob_fwd", logits, logits_bf16, nullptr, targets, num_tokens, vocab_size))
        return r;
    LpRows a;
    a.logits = logits;
    a.targets = targets;
    a.logp = logp_out;
    a.n = num_tokens;
    a.V = vocab_size;
    return lp_rows(S(stream), LpOp::FWD, logits_bf16 != 0, a, "token_logprob_fwd");
}

extern "C" int32_t ar_token_logprob_bwd(ar_stream_t stream, void* grad_logits, const void* logits, int32_t logits_bf16,
                                        const int64_t* targets, const float* grad_logp, float cap, int64_t num_tokens,
                                        int64_t vocab_size) {
    AR_CHECK_ARG(num_tokens <= 0 || (grad_logits && grad_logp), "token_logprob_bwd: null pointer");
    AR_CHECK_ARG(cap >= 0.f, "token_logprob_bwd: cap must not be negative");
    if (const int32_t r =
            check_rows("token_logprob_bwd", logits, logits_bf16, grad_logits, targets, num_tokens, vocab_size))
        return r;
    LpRows a;
    a.logits = logits;
    a.grad = grad_logits;
    a.targets = targets;
    a.grad_logp = grad_logp;
    a.cap = cap;
    a.n = num_tokens;
    a.V = vocab_size;
    return lp_rows(S(stream), LpOp::BWD, logits_bf16 != 0, a, "token_logprob_bwd");
}
