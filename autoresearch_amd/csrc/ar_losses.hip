// ar_losses.hip -- the clipped policy loss with a KL term and the preference
// loss over pairs, each with its gradient by the tokens' log-probabilities.
//
// Tokens come in sequences: sequence s holds tokens seq_start[s] up to, but
// not including, seq_start[s + 1].  A token counts if its target is a token
// of the vocabulary and it lies in a sequence.  Bound by launches: a batch's
// tokens are a few numbers each, and every sum over them is a launch that the
// next one needs.  The sums are fp64 in a fixed order; counts are integers.
#include <math.h>

#include "ar_losses.hpp"

namespace ar {
namespace {

constexpr int kTokBlock = 256;
constexpr int kMaxSplitItems = 1024;  // sequences x parts, when sequences are split
constexpr int64_t kPartTokens = 4096;

struct Seqs {
    const int64_t *targets, *start;  // start null: the n tokens are one sequence
    int64_t n, S, V;
    int parts;  // of each sequence; item = s * parts + part
};

// Tokens of an item.  Offsets outside [0, n], or descending ones, give
// shortened or empty sequences, never an access out of range.
__device__ __forceinline__ void item_range(const Seqs& q, int64_t item, int64_t& lo, int64_t& hi) {
    const int64_t s = item / q.parts, p = item - s * q.parts;
    int64_t a = 0, b = q.n;
    if (q.start) {
        a = min(max(q.start[s], (int64_t)0), q.n);
        b = min(max(q.start[s + 1], a), q.n);
    }
    const int64_t len = b - a;
    lo = a + len * p / q.parts;
    hi = a + len * (p + 1) / q.parts;
}
__device__ __forceinline__ bool counts(const Seqs& q, int64_t t) {
    const int64_t y = q.targets[t];
    return y >= 0 && y < q.V;
}

// cnt[item] = tokens that count; zero[0 .. n) = 0.
__global__ __launch_bounds__(kTokBlock) void count_k(Seqs q, int* cnt, float* zero) {
    __shared__ int red[kTokBlock / kWave];
    const int64_t step = (int64_t)gridDim.x * kTokBlock;
    if (zero)
        for (int64_t t = (int64_t)blockIdx.x * kTokBlock + threadIdx.x; t < q.n; t += step) zero[t] = 0.f;
    const int64_t items = q.S * q.parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t lo, hi;
        item_range(q, item, lo, hi);
        int c = 0;
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock) c += counts(q, t);
        c = block_total(c, red);
        if (threadIdx.x == 0) cnt[item] = c;
    }
}

// total[0] = tokens that count, total[1] = sequences with one.
__global__ __launch_bounds__(1024) void totals_k(const int* cnt, int64_t S, int parts, int64_t* total) {
    __shared__ int64_t red[16];
    int64_t n = 0, alive = 0;
    for (int64_t s = threadIdx.x; s < S; s += blockDim.x) {
        int64_t c = 0;
        for (int p = 0; p < parts; ++p) c += cnt[s * parts + p];
        n += c;
        alive += c > 0;
    }
    n = block_total(n, red);
    alive = block_total(alive, red);
    if (threadIdx.x == 0) {
        total[0] = n;
        total[1] = alive;
    }
}

// What a token's term weighs: 1 / (all tokens that count), or 1 / (sequences
// with one x this sequence's), rounded once to fp32.
__global__ __launch_bounds__(kTokBlock) void weight_k(Seqs q, const int* cnt, const int64_t* total, int per_seq,
                                                      float* weight) {
    const int64_t items = q.S * q.parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t lo, hi, ns = 0;
        item_range(q, item, lo, hi);
        const int64_t s = item / q.parts;
        for (int p = 0; p < q.parts; ++p) ns += cnt[s * q.parts + p];
        if (ns == 0) continue;
        const float w = (float)(per_seq ? 1.0 / ((double)total[1] * (double)ns) : 1.0 / (double)total[0]);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock)
            if (counts(q, t)) weight[t] = w;
    }
}

__global__ __launch_bounds__(kTokBlock) void policy_tokens_k(const float* weight, const float* logp, PolicyIn in,
                                                             float loss_scale, int64_t n, float* grad, double2* part) {
    __shared__ double red[kTokBlock / kWave];
    double loss = 0.0, kl = 0.0;
    const int64_t step = (int64_t)gridDim.x * kTokBlock;
    for (int64_t t = (int64_t)blockIdx.x * kTokBlock + threadIdx.x; t < n; t += step) {
        const float w = weight[t];
        float g = 0.f;
        if (w != 0.f) {
            const PolicyTerm<double> o = policy_term<double>(logp[t], PolicyToken(in, t), in);
            loss += w * o.loss;
            kl += w * o.kl;
            g = (float)(w * o.g * loss_scale);
        }
        if (grad) grad[t] = g;
    }
    loss = block_total(loss, red);
    kl = block_total(kl, red);
    if (threadIdx.x == 0) part[blockIdx.x] = make_double2(loss, kl);
}

// out[0], out[1] = the sums of part's n pairs, in a fixed order.
__global__ __launch_bounds__(1024) void sum_pairs_k(const double2* part, int64_t n, float* out) {
    __shared__ double red[16];
    double a = 0.0, b = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const double2 v = part[i];
        a += v.x;
        b += v.y;
    }
    a = block_total(a, red);
    b = block_total(b, red);
    if (threadIdx.x == 0) {
        out[0] = (float)a;
        out[1] = (float)b;
    }
}

// ---- preference ----
// sum[item] = sum of logp - ref over an item's tokens that count, and cnt;
// grad[0 .. n) = 0.
__global__ __launch_bounds__(kTokBlock) void pair_sums_k(Seqs q, const float* logp, const float* ref, double* sum,
                                                         int* cnt, float* grad) {
    __shared__ double red[kTokBlock / kWave];
    __shared__ int redi[kTokBlock / kWave];
    const int64_t step = (int64_t)gridDim.x * kTokBlock;
    if (grad)
        for (int64_t t = (int64_t)blockIdx.x * kTokBlock + threadIdx.x; t < q.n; t += step) grad[t] = 0.f;
    const int64_t items = q.S * q.parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t lo, hi;
        item_range(q, item, lo, hi);
        double s = 0.0;
        int c = 0;
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock)
            if (counts(q, t)) {
                s += (double)logp[t] - (ref ? (double)ref[t] : 0.0);
                ++c;
            }
        s = block_total(s, red);
        c = block_total(c, redi);
        if (threadIdx.x == 0) {
            sum[item] = s;
            cnt[item] = c;
        }
    }
}

// The loss of each pair and its slope by h = beta (chosen's sum - rejected's):
//   l = (1 - e) softplus(-h) + e softplus(h), softplus(x) = max(x, 0) + log1p(exp(-|x|)),
//   dl/dh = e sigma(h) - (1 - e) sigma(-h).
// A pair with a sequence in which no token counts is left out; the mean is
// over the others.  slope[i] = beta dl/dh / pairs, 0 for a pair left out.
__global__ __launch_bounds__(1024) void pair_loss_k(const double* sum, const int* cnt, int64_t pairs, int parts,
                                                    double beta, double smooth, double* h_ws, double* slope,
                                                    float* loss_out, float* margin_out) {
    __shared__ double red[16];
    __shared__ int64_t redi[16];
    int64_t live = 0;
    double loss = 0.0;
    for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) {
        double s[2] = {0.0, 0.0};
        int64_t c[2] = {0, 0};
        for (int k = 0; k < 2; ++k)
            for (int p = 0; p < parts; ++p) {
                s[k] += sum[(2 * i + k) * parts + p];
                c[k] += cnt[(2 * i + k) * parts + p];
            }
        const bool ok = c[0] > 0 && c[1] > 0;
        const double h = beta * (s[0] - s[1]);
        double d = 0.0;
        if (ok) {
            const double e = exp(-fabs(h)), lg = log1p(e);
            const double up = (h >= 0.0 ? 1.0 : e) / (1.0 + e), down = (h >= 0.0 ? e : 1.0) / (1.0 + e);
            double l = 0.0;  // a term without weight is left out: it may be infinite
            if (smooth < 1.0) l += (1.0 - smooth) * (fmax(-h, 0.0) + lg);
            if (smooth > 0.0) l += smooth * (fmax(h, 0.0) + lg);
            d = smooth * up - (1.0 - smooth) * down;
            loss += l;  // NaN where h is: through lg
            ++live;
        }
        if (margin_out) margin_out[i] = ok ? (float)h : 0.f;
        h_ws[i] = d;
    }
    live = block_total(live, redi);
    loss = block_total(loss, red);
    if (threadIdx.x == 0) loss_out[0] = live ? (float)(loss / (double)live) : 0.f;
    for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) slope[i] = live ? beta * h_ws[i] / (double)live : 0.0;
}

__global__ __launch_bounds__(kTokBlock) void pair_grad_k(Seqs q, const double* slope, float loss_scale, float* grad) {
    const int64_t items = q.S * q.parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t lo, hi;
        item_range(q, item, lo, hi);
        const int64_t s = item / q.parts;
        const float g = (float)((s & 1 ? -slope[s / 2] : slope[s / 2]) * loss_scale);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock)
            if (counts(q, t)) grad[t] = g;
    }
}

// Sequences of more than kPartTokens on average are split, so that a few long
// ones fill more than a few CUs.
Seqs make_seqs(const int64_t* targets, const int64_t* start, int64_t n, int64_t S, int64_t V) {
    int64_t parts = S > 0 ? cdiv(cdiv(n, S), kPartTokens) : 1;
    if (S > 0 && parts > kMaxSplitItems / S) parts = kMaxSplitItems / S;
    if (parts < 1) parts = 1;
    return Seqs{targets, start, n, S, V, (int)parts};
}
unsigned item_grid(const Seqs& q) {
    const int64_t items = q.S * q.parts;
    return (unsigned)(items < 1 ? 1 : items > 16384 ? 16384 : items);
}

struct Scratch {  // a workspace cut into arrays, each on 256 bytes
    char* base;
    size_t used = 0;
    template <typename T>
    T* take(int64_t n) {
        T* p = reinterpret_cast<T*>(base + used);
        used += ((size_t)n * sizeof(T) + 255) & ~size_t(255);
        return p;
    }
};

int32_t check_seqs(const char* nm, const int64_t* targets, const int64_t* seq_start, int64_t n, int64_t S, int64_t V) {
    AR_CHECK_ARG(n >= 0 && S >= 0 && V > 0, "%s: bad shape", nm);
    AR_CHECK_ARG(n == 0 || targets, "%s: null pointer", nm);
    AR_CHECK_ARG(seq_start || S == 1, "%s: without seq_start the tokens are one sequence", nm);
    if (n > INT32_MAX || S > INT32_MAX / 2)
        return set_error(AR_EUNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^30 sequences", nm);
    return AR_OK;
}
int32_t check_policy(const char* nm, const float* adv, const float* ref, int64_t n, double lo, double hi, double kl) {
    AR_CHECK_ARG(n <= 0 || adv, "%s: null pointer", nm);
    AR_CHECK_ARG(lo >= 0.0 && hi >= 0.0, "%s: clip_low and clip_high must not be negative", nm);
    AR_CHECK_ARG(kl == kl && (kl == 0.0 || ref || n <= 0), "%s: a KL coefficient needs ref_logp", nm);
    return AR_OK;
}

struct PolicyWs {
    int* cnt;
    int64_t* total;
    float* weight;
    double2* part;
    size_t bytes;
};
PolicyWs policy_ws(char* base, const Seqs& q, int64_t nparts) {
    Scratch s{base};
    PolicyWs w;
    w.cnt = s.take<int>(q.S * q.parts);
    w.total = s.take<int64_t>(2);
    w.weight = s.take<float>(q.n);
    w.part = s.take<double2>(nparts);
    w.bytes = s.used;
    return w;
}
int32_t policy_weights(hipStream_t st, const Seqs& q, int per_seq, const PolicyWs& w, const char* nm) {
    const unsigned g = item_grid(q);
    count_k<<<g, kTokBlock, 0, st>>>(q, w.cnt, w.weight);
    totals_k<<<1, 1024, 0, st>>>(w.cnt, q.S, q.parts, w.total);
    weight_k<<<g, kTokBlock, 0, st>>>(q, w.cnt, w.total, per_seq, w.weight);
    return check_launch(nm);
}

}  // namespace
}  // namespace ar

using namespace ar;

extern "C" int32_t ar_policy_loss(ar_stream_t stream, float* loss_out, float* grad_logp, const float* logp,
                                  const float* old_logp, const float* ref_logp, const float* advantages,
                                  const int64_t* targets, const int64_t* seq_start, double clip_low, double clip_high,
                                  double kl_coef, int32_t per_seq, int64_t num_tokens, int64_t num_seqs,
                                  int64_t vocab_size, float loss_scale) {
    const char* nm = "policy_loss";
    AR_CHECK_ARG(loss_out && (num_tokens <= 0 || logp), "%s: null pointer", nm);
    if (const int32_t r = check_seqs(nm, targets, seq_start, num_tokens, num_seqs, vocab_size)) return r;
    if (const int32_t r = check_policy(nm, advantages, ref_logp, num_tokens, clip_low, clip_high, kl_coef)) return r;
    const Seqs q = make_seqs(targets, seq_start, num_tokens, num_seqs, vocab_size);
    int64_t blocks = cdiv(num_tokens, kTokBlock);
    if (blocks > 1024) blocks = 1024;
    if (blocks < 1) blocks = 1;
    int32_t status;
    char* base = static_cast<char*>(workspace(S(stream), policy_ws(nullptr, q, blocks).bytes, &status));
    if (!base) return status;
    const PolicyWs w = policy_ws(base, q, blocks);
    if (const int32_t r = policy_weights(S(stream), q, per_seq, w, nm)) return r;
    const PolicyIn in{old_logp, ref_logp, advantages, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
    policy_tokens_k<<<(unsigned)blocks, kTokBlock, 0, S(stream)>>>(w.weight, logp, in, loss_scale, num_tokens,
                                                                   grad_logp, w.part);
    sum_pairs_k<<<1, 1024, 0, S(stream)>>>(w.part, blocks, loss_out);
    return check_launch(nm);
}

extern "C" int32_t ar_policy_loss_logits(ar_stream_t stream, float* loss_out, float* logp_out, void* grad_logits,
                                         const void* logits, int32_t logits_bf16, const float* old_logp,
                                         const float* ref_logp, const float* advantages, const int64_t* targets,
                                         const int64_t* seq_start, float cap, double clip_low, double clip_high,
                                         double kl_coef, int32_t per_seq, int64_t num_tokens, int64_t num_seqs,
                                         int64_t vocab_size, float loss_scale) {
    const char* nm = "policy_loss_logits";
    AR_CHECK_ARG(loss_out && (num_tokens <= 0 || grad_logits), "%s: null pointer", nm);
    AR_CHECK_ARG(cap >= 0.f, "%s: cap must not be negative", nm);
    if (const int32_t r = check_rows(nm, logits, logits_bf16, grad_logits, targets, num_tokens, vocab_size)) return r;
    if (const int32_t r = check_seqs(nm, targets, seq_start, num_tokens, num_seqs, vocab_size)) return r;
    if (const int32_t r = check_policy(nm, advantages, ref_logp, num_tokens, clip_low, clip_high, kl_coef)) return r;
    const Seqs q = make_seqs(targets, seq_start, num_tokens, num_seqs, vocab_size);
    int32_t status;
    char* base = static_cast<char*>(workspace(S(stream), policy_ws(nullptr, q, num_tokens).bytes, &status));
    if (!base) return status;
    const PolicyWs w = policy_ws(base, q, num_tokens);
    if (const int32_t r = policy_weights(S(stream), q, per_seq, w, nm)) return r;
    LpRows a;
    a.logits = logits;
    a.grad = grad_logits;
    a.targets = targets;
    a.logp = logp_out;
    a.weight = w.weight;
    a.terms = w.part;
    a.policy = PolicyIn{old_logp, ref_logp, advantages, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
    a.cap = cap;
    a.loss_scale = loss_scale;
    a.n = num_tokens;
    a.V = vocab_size;
    if (const int32_t r = lp_rows(S(stream), LpOp::POLICY, logits_bf16 != 0, a, nm)) return r;
    sum_pairs_k<<<1, 1024, 0, S(stream)>>>(w.part, num_tokens, loss_out);
    return check_launch(nm);
}

extern "C" int32_t ar_preference_loss(ar_stream_t stream, float* loss_out, float* margin_out, float* grad_logp,
                                      const float* logp, const float* ref_logp, const int64_t* targets,
                                      const int64_t* seq_start, double beta, double label_smoothing,
                                      int64_t num_tokens, int64_t num_pairs, int64_t vocab_size, float loss_scale) {
    const char* nm = "preference_loss";
    AR_CHECK_ARG(loss_out && seq_start && (num_tokens <= 0 || logp), "%s: null pointer", nm);
    AR_CHECK_ARG(num_pairs >= 0 && num_pairs <= INT32_MAX / 4, "%s: bad number of pairs", nm);
    if (const int32_t r = check_seqs(nm, targets, seq_start, num_tokens, 2 * num_pairs, vocab_size)) return r;
    AR_CHECK_ARG(beta == beta && label_smoothing >= 0.0 && label_smoothing <= 1.0,
                 "%s: label_smoothing must lie in [0, 1]", nm);
    AR_CHECK_ARG(!overlaps(grad_logp, num_tokens * sizeof(float), logp, num_tokens * sizeof(float)) &&
                     !overlaps(grad_logp, num_tokens * sizeof(float), ref_logp, num_tokens * sizeof(float)),
                 "%s: grad_logp must not overlap logp or ref_logp", nm);
    const Seqs q = make_seqs(targets, seq_start, num_tokens, 2 * num_pairs, vocab_size);
    const int64_t items = q.S * q.parts;
    auto cut = [&](char* base, double*& sum, double*& d, double*& slope, int*& cnt) {
        Scratch s{base};
        sum = s.take<double>(items);
        d = s.take<double>(num_pairs);
        slope = s.take<double>(num_pairs);
        cnt = s.take<int>(items);
        return s.used;
    };
    double *sum, *d, *slope;
    int* cnt;
    int32_t status;
    char* base = static_cast<char*>(workspace(S(stream), cut(nullptr, sum, d, slope, cnt), &status));
    if (!base) return status;
    cut(base, sum, d, slope, cnt);
    const unsigned g = item_grid(q);
    pair_sums_k<<<g, kTokBlock, 0, S(stream)>>>(q, logp, ref_logp, sum, cnt, grad_logp);
    pair_loss_k<<<1, 1024, 0, S(stream)>>>(sum, cnt, num_pairs, q.parts, beta, label_smoothing, d, slope, loss_out,
                                           margin_out);
    if (grad_logp && num_tokens > 0) pair_grad_k<<<g, kTokBlock, 0, S(stream)>>>(q, slope, loss_scale, grad_logp);
    return check_launch(nm);
}
