// ar_losses.hpp -- shared by the post-training losses: token log-probabilities
// and their gradient (ar_logprob.hip), the policy and preference losses
// (ar_losses.hip).  fp32 or bf16 logits, fp64 for the few values per token.
#pragma once

#include "ar_internal.hpp"

namespace ar {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of an array: E values.  Arrays and rows start at any multiple of a
// value's size (any V, any view), which the vector accesses say.
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
    static __device__ __forceinline__ void store_nt(float* p, u32x4 v) {
        __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
    }
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
    static __device__ __forceinline__ void store_nt(bf16* p, u32x4 v) {
        __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
    }
    static __device__ __forceinline__ u32x4 fill(float x) {
        return u32x4{1, 1, 1, 1} * (__float_as_uint(x) >> 16) * 0x10001u;
    }
};

// What one token adds to the policy loss, before its weight:
//   pg = -A rho, rho = r = exp(logp - old) or the bound that binds it,
//   kl = exp(ref - logp) - (ref - logp) - 1, loss = pg + c kl, g = d loss / d logp.
// The bound binds where it lowers the gain: r > hi with A > 0, r < lo with
// A < 0; there pg does not depend on logp.
// F = double where log-probabilities are given: the difference of two fp32
// values is exact in it, and r meets the bounds unrounded.  F = float where
// they come out of a row of logits, to which it adds less than their own error
// (a few 1e-7).
struct PolicyIn {
    const float *old_logp, *ref_logp, *adv;  // old_logp null: old = logp; ref_logp null: no KL term
    double lo, hi, kl_coef;
};
struct PolicyToken {
    float adv, old_logp, ref_logp;
    __device__ __forceinline__ PolicyToken() {}
    __device__ __forceinline__ PolicyToken(const PolicyIn& in, int64_t t)
        : adv(in.adv[t]), old_logp(in.old_logp ? in.old_logp[t] : 0.f), ref_logp(in.ref_logp ? in.ref_logp[t] : 0.f) {}
};
template <typename F>
struct PolicyTerm {
    F loss, kl, g;
};
template <typename F>
__device__ __forceinline__ PolicyTerm<F> policy_term(F logp, const PolicyToken& t, const PolicyIn& in) {
    const F a = t.adv, lo = (F)in.lo, hi = (F)in.hi, c = (F)in.kl_coef;
    const F r = in.old_logp ? exp(logp - (F)t.old_logp) : (F)1;
    const bool above = a > (F)0 && r > hi, below = a < (F)0 && r < lo;
    PolicyTerm<F> o;
    o.loss = -a * (above ? hi : below ? lo : r);
    o.g = above || below ? (F)0 : -a * r;
    o.kl = (F)0;
    if (in.ref_logp) {
        const F k = (F)t.ref_logp - logp, e = expm1(k);
        o.kl = e - k;
        if (c != (F)0) {
            o.loss += c * o.kl;
            o.g -= c * e;
        }
    }
    return o;
}

// g alone, in fp32 with the hardware's exponential.
__device__ __forceinline__ float policy_slope(float logp, const PolicyToken& t, const PolicyIn& in) {
    constexpr float kL2e = 1.44269504f;
    const float a = t.adv, r = in.old_logp ? __builtin_amdgcn_exp2f((logp - t.old_logp) * kL2e) : 1.f;
    float g = (a > 0.f && r > (float)in.hi) || (a < 0.f && r < (float)in.lo) ? 0.f : -a * r;
    if (in.ref_logp && in.kl_coef != 0.0)
        g -= (float)in.kl_coef * (__builtin_amdgcn_exp2f((t.ref_logp - logp) * kL2e) - 1.f);
    return g;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
// As block_sum(float), for double and int; red holds blockDim.x / 64 values.
template <typename T>
__device__ __forceinline__ T block_total(T v, T* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    const int w = threadIdx.x / kWave, l = threadIdx.x % kWave, nw = blockDim.x / kWave;
    __syncthreads();
    if (l == 0) red[w] = v;
    __syncthreads();
    T t = 0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

// Rows of logits (ar_logprob.hip).  FWD: logp.  BWD: the gradient by the
// logits of sum_t grad_logp[t] logp[t].  POLICY: logp, each token's weighted
// loss and KL to terms, and the loss's gradient by the logits; weight[t] is
// what the token's term weighs in the loss, 0 for one that does not count.
enum class LpOp { FWD, BWD, POLICY };
struct LpRows {
    const void* logits = nullptr;
    void* grad = nullptr;  // may be logits
    const int64_t* targets = nullptr;
    float* logp = nullptr;
    const float* grad_logp = nullptr;  // BWD
    const float* weight = nullptr;     // POLICY
    double2* terms = nullptr;          // POLICY: {loss, kl} per token
    PolicyIn policy{};
    float cap = 0.f;         // the softcap the logits went through, 0: none
    float loss_scale = 1.f;  // POLICY
    int64_t n = 0, V = 0, first = 0;  // first: a launch's first row
    void* scratch = nullptr;  // lp_scratch(...) bytes; null: no row is split
};
size_t lp_scratch(LpOp op, bool bf16_logits, int64_t n, int64_t V);
int32_t lp_rows(hipStream_t st, LpOp op, bool bf16_logits, const LpRows& a, const char* nm);
// What the entry points on logits check alike; logp: an array by token that
// the call reads for one row, or writes, while it works on others.
int32_t check_rows(const char* nm, const void* logits, int32_t logits_bf16, const void* grad, const int64_t* targets,
                   const float* logp, int64_t n, int64_t V);

inline bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + nb && y < x + na;
}

}  // namespace ar
