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

constexpr int kRowBlock = 256;

template <typename T, LpOp OP>
__global__ __launch_bounds__(kRowBlock) void lp_row_k(LpRows a) {
    using R = Row<T>;
    constexpr int E = R::E;
    __shared__ float red[2 * kRowBlock / kWave];
    __shared__ float coef;
    const int64_t r = blockIdx.x;
    const int V = (int)a.V, nb = V / E;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    T* out = static_cast<T*>(a.grad) + r * a.V;
    float w = 1.f;
    if constexpr (OP == LpOp::BWD) w = a.grad_logp[r];
    if constexpr (OP == LpOp::POLICY) w = a.weight[r];
    if (y < 0 || y >= a.V || w == 0.f) {
        // a token that does not count: nothing is read, its gradient is zero
        if constexpr (OP != LpOp::BWD)
            if (threadIdx.x == 0 && a.logp) a.logp[r] = 0.f;
        if constexpr (OP == LpOp::POLICY)
            if (threadIdx.x == 0) a.terms[r] = make_double2(0.0, 0.0);
        if constexpr (OP != LpOp::FWD) {
            for (int c = threadIdx.x; c < nb; c += kRowBlock)
                reinterpret_cast<typename R::vec*>(out)[c] = u32x4{0, 0, 0, 0};
            for (int j = nb * E + threadIdx.x; j < V; j += kRowBlock) out[j] = from_f32<T>(0.f);
        }
        return;
    }
    const float zy = to_f32<T>(row[y]);
    MaxSum v;
    for (int c = threadIdx.x; c < nb; c += kRowBlock) {
        const u32x4 q = reinterpret_cast<const typename R::vec*>(row)[c];
        float cm = R::get(q, 0);
#pragma unroll
        for (int i = 1; i < E; ++i) cm = fmaxf(cm, R::get(q, i));
        const float use = fmaxf(v.m, cm) == -INFINITY ? 0.f : fmaxf(v.m, cm);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += __expf(R::get(q, i) - use);
        v.add(cm == -INFINITY ? -INFINITY : use, s);
    }
    for (int j = nb * E + threadIdx.x; j < V; j += kRowBlock) {
        const float z = to_f32<T>(row[j]);
        v.add(z, z == -INFINITY ? 0.f : __expf(z - z));
    }
    v = block_max_sum(v, red);
    if constexpr (OP == LpOp::FWD) {
        if (threadIdx.x == 0) a.logp[r] = (zy - v.m) - logf(v.s);
        return;
    }
    if (threadIdx.x == 0) {
        if constexpr (OP == LpOp::POLICY) {
            const float logp = (zy - v.m) - logf(v.s);
            const PolicyTerm t = policy_term(logp, r, a.policy);
            if (a.logp) a.logp[r] = logp;
            a.terms[r] = make_double2(w * t.loss, w * t.kl);
            coef = (float)(w * t.g * a.loss_scale);
        } else {
            coef = w;
        }
    }
    __syncthreads();  // zy and the sums are read: from here the row may be overwritten
    const float g = coef, gs = g / v.s, rcap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    auto grad_of = [&](float z, int j) {
        float d = -gs * __expf(z - v.m);
        if (j == y) d += g;
        const float u = z * rcap;
        return d * fmaxf(0.f, fmaf(-u, u, 1.f));
    };
    for (int c = threadIdx.x; c < nb; c += kRowBlock) {
        const u32x4 q = reinterpret_cast<const typename R::vec*>(row)[c];
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = grad_of(R::get(q, i), c * E + i);
        reinterpret_cast<typename R::vec*>(out)[c] = R::pack(x);
    }
    for (int j = nb * E + threadIdx.x; j < V; j += kRowBlock) out[j] = from_f32<T>(grad_of(to_f32<T>(row[j]), j));
}

template <typename T>
int32_t launch(hipStream_t st, LpOp op, const LpRows& a, const char* nm) {
    const unsigned g = (unsigned)a.n;
    if (op == LpOp::FWD) lp_row_k<T, LpOp::FWD><<<g, kRowBlock, 0, st>>>(a);
    else if (op == LpOp::BWD) lp_row_k<T, LpOp::BWD><<<g, kRowBlock, 0, st>>>(a);
    else lp_row_k<T, LpOp::POLICY><<<g, kRowBlock, 0, st>>>(a);
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
