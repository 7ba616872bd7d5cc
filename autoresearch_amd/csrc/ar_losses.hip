// ar_losses.hip -- the clipped policy loss with a KL term and the preference
// loss over pairs, each with its gradient by the tokens' log-probabilities.
//
// Tokens come in sequences: sequence s holds tokens seq_start[s] up to, but
// not including, seq_start[s + 1].  A token counts if its target is a token
// of the vocabulary and it lies in a sequence.  Bound by launches: a batch's
// tokens are a few numbers each, and every sum over them is a launch that the
// next one needs.  The sums are fp64 in a fixed order; counts are integers.
// Policy loss of 500 tokens 8.4 us, of 262144 15.7 (three launches); preference
// loss of 4 pairs (801 tokens) 7.9.
#include <math.h>

#include "ar_losses.hpp"

namespace ar {
namespace {

constexpr int kTokBlock = 256;
constexpr int64_t kMaxItems = 2048;     // sequences x parts, where sequences are split
constexpr int64_t kInlineItems = 1024;  // counts that every block adds up itself

struct Seqs {
    const int64_t *targets, *start;  // start null: the n tokens are one sequence
    int64_t n, S, V;
    int parts;  // of each sequence; item = s * parts + part
};

// Tokens of an item.  Offsets outside [0, n], or descending ones, give
// shortened or empty sequences, never an access out of range.
// (Divisions in 32 bits: at most 2^31 - 1 tokens, 2^30 sequences.)
__device__ __forceinline__ uint32_t item_seq(const Seqs& q, int64_t item) { return (uint32_t)item / (uint32_t)q.parts; }
__device__ __forceinline__ void item_range(const Seqs& q, int64_t item, int64_t& lo, int64_t& hi) {
    const uint32_t s = item_seq(q, item), p = (uint32_t)item - s * q.parts;
    int64_t a = 0, b = q.n;
    if (q.start) {
        a = min(max(q.start[s], (int64_t)0), q.n);
        b = min(max(q.start[s + 1], a), q.n);
    }
    const uint32_t len = (uint32_t)(b - a), step = (len + q.parts - 1) / (uint32_t)q.parts;
    lo = a + min(len, p * step);
    hi = a + min(len, (p + 1) * step);
}
__device__ __forceinline__ bool counts(const Seqs& q, int64_t t) {
    const int64_t y = q.targets[t];
    return y >= 0 && y < q.V;
}

// f(t) for every token that lies in no sequence, the grid's threads in turn.
template <typename F>
__device__ __forceinline__ void each_outside(const Seqs& q, F f) {
    const int64_t a = q.S > 0 ? (q.start ? min(max(q.start[0], (int64_t)0), q.n) : 0) : q.n;
    const int64_t b = q.S > 0 ? (q.start ? min(max(q.start[q.S], a), q.n) : q.n) : q.n;
    const int64_t step = (int64_t)gridDim.x * blockDim.x, me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t t = me; t < a; t += step) f(t);
    for (int64_t t = b + me; t < q.n; t += step) f(t);
}

// cnt[item] = tokens that count.
__global__ __launch_bounds__(kTokBlock) void count_k(Seqs q, int* cnt) {
    __shared__ int red[kTokBlock / kWave];
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

// All tokens that count and the sequences with one, by every thread of a
// block, from the items' counts.
struct Totals {
    int64_t n, alive;
};
struct TotalsLds {
    int64_t red[16];
    int alive[kMaxItems];  // of split sequences: at most one per item
};
__device__ __forceinline__ Totals sum_counts(const Seqs& q, const int* cnt, TotalsLds& l) {
    const int64_t items = q.S * q.parts;
    Totals t{0, 0};
    if (q.parts > 1) {
        for (int s = threadIdx.x; s < q.S; s += blockDim.x) l.alive[s] = 0;
        __syncthreads();
    }
    for (int64_t i = threadIdx.x; i < items; i += blockDim.x) {
        const int c = cnt[i];
        t.n += c;
        if (q.parts == 1) t.alive += c > 0;
        else if (c > 0) l.alive[item_seq(q, i)] = 1;
    }
    t.n = block_total(t.n, l.red);
    if (q.parts > 1)
        for (int s = threadIdx.x; s < q.S; s += blockDim.x) t.alive += l.alive[s];
    t.alive = block_total(t.alive, l.red);
    return t;
}
__global__ __launch_bounds__(1024) void totals_k(Seqs q, const int* cnt, Totals* total) {
    __shared__ TotalsLds l;
    const Totals t = sum_counts(q, cnt, l);
    if (threadIdx.x == 0) *total = t;
}

// What a token's term weighs: 1 / (all tokens that count), or 1 / (sequences
// with one x this sequence's); rounded to fp32 only on its way to rows of
// logits, whose gradients are rounded again.  Ahead of the sequences' items
// every block takes the totals: from the counts where they are few, or as
// totals_k left them.
struct Weights {
    Totals t;
    __device__ __forceinline__ Weights(const Seqs& q, const int* cnt, const Totals* total, TotalsLds& l) {
        if (total) t = *total;
        else t = sum_counts(q, cnt, l);
    }
    // of a token of an item, by every thread of the block
    __device__ __forceinline__ double of(const Seqs& q, const int* cnt, int64_t item, int per_seq, int64_t* red) const {
        if (!per_seq) return t.n ? 1.0 / (double)t.n : 0.0;
        const int64_t first = (int64_t)item_seq(q, item) * q.parts;
        int64_t ns = 0;
        if (q.parts == 1) {
            ns = cnt[first];
        } else {
            for (int p = threadIdx.x; p < q.parts; p += blockDim.x) ns += cnt[first + p];
            ns = block_total(ns, red);
        }
        return ns ? 1.0 / ((double)t.alive * (double)ns) : 0.0;
    }
};
__global__ __launch_bounds__(kTokBlock) void weight_k(Seqs q, const int* cnt, const Totals* total, int per_seq,
                                                      float* weight) {
    __shared__ TotalsLds l;
    const Weights w(q, cnt, total, l);
    const int64_t items = q.S * q.parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t lo, hi;
        item_range(q, item, lo, hi);
        const float ws = (float)w.of(q, cnt, item, per_seq, l.red);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock) weight[t] = counts(q, t) ? ws : 0.f;
    }
    each_outside(q, [&](int64_t t) { weight[t] = 0.f; });
}

struct PolicyTokens {
    const float* logp;
    PolicyIn in;
    int per_seq;
    float loss_scale;
    float* grad;  // may be null
};
// A token's inputs, and what becomes of them.
struct Token {
    PolicyToken in;
    float logp;
    bool live = false;
    __device__ __forceinline__ Token() {}
    __device__ __forceinline__ Token(const Seqs& q, const PolicyTokens& a, int64_t t)
        : in(a.in, t), logp(a.logp[t]), live(counts(q, t)) {}
    __device__ __forceinline__ void use(const PolicyTokens& a, int64_t t, double w, double& loss, double& kl) const {
        float g = 0.f;
        if (live && w != 0.0) {
            const PolicyTerm<double> o = policy_term<double>(logp, in, a.in);
            loss += w * o.loss;
            kl += w * o.kl;
            g = (float)(w * o.g * a.loss_scale);
        }
        if (a.grad) a.grad[t] = g;
    }
};
// part[block] = this block's items' loss and KL; every token's gradient.  The
// next token of a lane is on its way while one is worked on, the first before
// the counts are added up.  Bound by one chain of loads and the fp64
// exponentials behind it, not by bytes: 262144 tokens of 509 sequences (6.5 MB)
// 10.4 us, 8.4 of them without the counts (which would take a launch of 3.7).
template <int TB>
__global__ __launch_bounds__(TB) void policy_tokens_k(Seqs q, const int* cnt, const Totals* total, PolicyTokens a,
                                                      double2* part) {
    __shared__ double red[TB / kWave];
    __shared__ TotalsLds l;
    double loss = 0.0, kl = 0.0;
    const int64_t items = q.S * q.parts;
    int64_t item = blockIdx.x, lo = 0, hi = 0, t = 0;
    Token next;
    auto begin = [&]() {
        if (item >= items) return;
        item_range(q, item, lo, hi);
        t = lo + threadIdx.x;
        if (t < hi) next = Token(q, a, t);
    };
    begin();
    const Weights w(q, cnt, total, l);
    while (item < items) {
        const double ws = w.of(q, cnt, item, a.per_seq, l.red);
        for (; t < hi; t += TB) {
            const Token now = next;
            if (t + TB < hi) next = Token(q, a, t + TB);
            now.use(a, t, ws, loss, kl);
        }
        item += gridDim.x;
        begin();
    }
    if (a.grad) each_outside(q, [&](int64_t t) { a.grad[t] = 0.f; });
    loss = block_total(loss, red);
    kl = block_total(kl, red);
    if (threadIdx.x == 0) part[blockIdx.x] = make_double2(loss, kl);
}

// ---- small batches: one block ----
// The sequences' offsets, their counts and the tokens' sequences in LDS.
constexpr int kSmallBlock = 1024, kSmallSeqs = 1024;
constexpr int kSmallTokens = 8192;  // pairs: 12.8 us at 8000, three launches 13.2
constexpr int kSmallPolicy = 2048;  // policy loss: 8.4 us at 500, 10.2 at 2048, 15.0 at 4000, three launches 13.8
struct SmallSeqs {
    int start[kSmallSeqs + 1], cnt[kSmallSeqs];
    int16_t seq[kSmallTokens];  // -1: the token does not count
};
__device__ __forceinline__ void small_load(const Seqs& q, SmallSeqs& l) {
    for (int s = threadIdx.x; s <= q.S; s += kSmallBlock) {
        l.start[s] = q.start ? (int)min(max(q.start[s], (int64_t)0), q.n) : s ? (int)q.n : 0;
        if (s < q.S) l.cnt[s] = 0;
    }
    __syncthreads();
}
// The last sequence that starts at or before token t, if it holds it.
__device__ __forceinline__ int small_seq(const Seqs& q, const SmallSeqs& l, int t) {
    int lo = 0, hi = (int)q.S - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (l.start[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return hi >= 0 && l.start[lo] <= t && t < l.start[lo + 1] ? lo : -1;
}
// The sequences of all tokens and their counts (integers: in any order), and
// the totals.
__device__ __forceinline__ Totals small_totals(const Seqs& q, SmallSeqs& l, int64_t* red) {
    small_load(q, l);
    Totals n{0, 0};
    for (int t = threadIdx.x; t < q.n; t += kSmallBlock) {
        const bool in = counts(q, t);
        const int s = in ? small_seq(q, l, t) : -1;
        l.seq[t] = (int16_t)s;
        if (s >= 0) {
            atomicAdd(&l.cnt[s], 1);
            ++n.n;
        }
    }
    n.n = block_total(n.n, red);  // its barriers: the counts are whole
    for (int s = threadIdx.x; s < q.S; s += kSmallBlock) n.alive += l.cnt[s] > 0;
    n.alive = block_total(n.alive, red);
    return n;
}
__device__ __forceinline__ double small_weight(const SmallSeqs& l, const Totals& n, int t, int per_seq) {
    const int s = l.seq[t];
    return s < 0 ? 0.0 : per_seq ? 1.0 / ((double)n.alive * (double)l.cnt[s]) : 1.0 / (double)n.n;
}
__global__ __launch_bounds__(kSmallBlock) void weight_small_k(Seqs q, int per_seq, float* weight) {
    __shared__ SmallSeqs l;
    __shared__ int64_t red[kSmallBlock / kWave];
    const Totals n = small_totals(q, l, red);
    for (int t = threadIdx.x; t < q.n; t += kSmallBlock) weight[t] = (float)small_weight(l, n, t, per_seq);
}
__global__ __launch_bounds__(kSmallBlock) void policy_small_k(Seqs q, PolicyTokens a, float* loss_out) {
    __shared__ SmallSeqs l;
    __shared__ int64_t red[kSmallBlock / kWave];
    __shared__ double redd[kSmallBlock / kWave];
    int t = threadIdx.x;
    Token next;
    if (t < q.n) next = Token(q, a, t);
    const Totals n = small_totals(q, l, red);
    double loss = 0.0, kl = 0.0;
    for (; t < q.n; t += kSmallBlock) {
        const Token now = next;
        if (t + kSmallBlock < q.n) next = Token(q, a, t + kSmallBlock);
        now.use(a, t, small_weight(l, n, t, a.per_seq), loss, kl);
    }
    loss = block_total(loss, redd);
    kl = block_total(kl, redd);
    if (threadIdx.x == 0) {
        loss_out[0] = (float)loss;
        loss_out[1] = (float)kl;
    }
}

// The sums of a block's PAIRS of part's n pairs, in a fixed order: to out (one
// block), or to part2 for another such launch.  One block for all of 65536
// pairs took 36 us, with eight loads in flight 23, in two launches 11; up to
// kSumLast pairs one block is faster (8192: by 2.7 us, 16384: 1.5).
constexpr int64_t kSumPairs = 4096, kSumLast = 16384;
template <int64_t PAIRS>
__global__ __launch_bounds__(1024) void sum_pairs_k(const double2* part, int64_t n, double2* part2, float* out) {
    __shared__ double red[16];
    double a = 0.0, b = 0.0;
#pragma unroll
    for (int k = 0; k < PAIRS / 1024; ++k) {
        const int64_t i = blockIdx.x * PAIRS + threadIdx.x + k * 1024;
        const double2 v = i < n ? part[i] : make_double2(0.0, 0.0);
        a += v.x;
        b += v.y;
    }
    a = block_total(a, red);
    b = block_total(b, red);
    if (threadIdx.x == 0) {
        if (part2) {
            part2[blockIdx.x] = make_double2(a, b);
        } else {
            out[0] = (float)a;
            out[1] = (float)b;
        }
    }
}

// How many pairs sum_pairs needs, for the sums of sums behind the n.
int64_t pair_room(int64_t n) {
    int64_t room = n;
    while (n > kSumLast) room += n = cdiv(n, kSumPairs);
    return room;
}
void sum_pairs(hipStream_t st, double2* part, int64_t n, float* out) {
    for (; n > kSumLast; part += n, n = cdiv(n, kSumPairs))
        sum_pairs_k<kSumPairs><<<(unsigned)cdiv(n, kSumPairs), 1024, 0, st>>>(part, n, part + n, nullptr);
    if (n > kSumPairs) sum_pairs_k<kSumLast><<<1, 1024, 0, st>>>(part, n, nullptr, out);
    else sum_pairs_k<kSumPairs><<<1, 1024, 0, st>>>(part, n, nullptr, out);
}

// ---- preference ----
// sum[item] = sum of logp - ref over an item's tokens that count, and cnt.
__global__ __launch_bounds__(kTokBlock) void pair_sums_k(Seqs q, const float* logp, const float* ref, double* sum,
                                                         int* cnt) {
    __shared__ double red[kTokBlock / kWave];
    __shared__ int redi[kTokBlock / kWave];
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

// The loss of a pair and its slope by h = beta (chosen's sum - rejected's):
//   l = (1 - e) softplus(-h) + e softplus(h), softplus(x) = max(x, 0) + log1p(exp(-|x|)),
//   dl/dh = e sigma(h) - (1 - e) sigma(-h).
// A term without weight is left out: it may be infinite.
__device__ __forceinline__ double pair_loss(double h, double smooth, double& d) {
    const double e = exp(-fabs(h)), lg = log1p(e);
    const double up = (h >= 0.0 ? 1.0 : e) / (1.0 + e), down = (h >= 0.0 ? e : 1.0) / (1.0 + e);
    double l = 0.0;
    if (smooth < 1.0) l += (1.0 - smooth) * (fmax(-h, 0.0) + lg);
    if (smooth > 0.0) l += smooth * (fmax(h, 0.0) + lg);
    d = smooth * up - (1.0 - smooth) * down;
    return l;  // NaN where h is: through lg
}
// A pair with a sequence in which no token counts is left out; the mean is
// over the others.  slope[i] = beta dl/dh / pairs, 0 for a pair left out.
constexpr int kFewParts = 8, kManyParts = 16;
__global__ __launch_bounds__(1024) void pair_loss_k(const double* sum, const int* cnt, int64_t pairs, int parts,
                                                    double beta, double smooth, double* h_ws, double* slope,
                                                    float* loss_out, float* margin_out) {
    __shared__ double red[16];
    __shared__ int64_t redi[16];
    __shared__ double seq_sum[2 * kManyParts];
    __shared__ int seq_cnt[2 * kManyParts];
    const bool split = parts > kFewParts;  // then there are at most kManyParts pairs: a wave adds up a sequence
    if (split) {
        for (int64_t s = threadIdx.x / kWave; s < 2 * pairs; s += blockDim.x / kWave) {
            double v = 0.0;
            int c = 0;
            for (int p = threadIdx.x % kWave; p < parts; p += kWave) {
                v += sum[s * parts + p];
                c += cnt[s * parts + p];
            }
            v = wave_sum(v);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, kWave);
            if (threadIdx.x % kWave == 0) {
                seq_sum[s] = v;
                seq_cnt[s] = c;
            }
        }
        __syncthreads();
    }
    int64_t live = 0;
    double loss = 0.0;
    for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) {
        double s[2] = {0.0, 0.0};
        int64_t c[2] = {0, 0};
        for (int k = 0; k < 2; ++k)
            for (int p = 0; p < (split ? 1 : parts); ++p) {
                s[k] += split ? seq_sum[2 * i + k] : sum[(2 * i + k) * parts + p];
                c[k] += split ? seq_cnt[2 * i + k] : cnt[(2 * i + k) * parts + p];
            }
        const bool ok = c[0] > 0 && c[1] > 0;
        const double h = beta * (s[0] - s[1]);
        double d = 0.0;
        if (ok) {
            loss += pair_loss(h, smooth, d);
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
        const int64_t s = item_seq(q, item);
        const float g = (float)((s & 1 ? -slope[s / 2] : slope[s / 2]) * loss_scale);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kTokBlock) grad[t] = counts(q, t) ? g : 0.f;
    }
    each_outside(q, [&](int64_t t) { grad[t] = 0.f; });
}

// A few pairs in one block: a wave sums a sequence.
constexpr int kSmallPairs = 64;
__global__ __launch_bounds__(kSmallBlock) void pair_small_k(Seqs q, const float* logp, const float* ref, double beta,
                                                            double smooth, float loss_scale, float* loss_out,
                                                            float* margin_out, float* grad) {
    __shared__ SmallSeqs l;
    __shared__ double sum[2 * kSmallPairs], slope[kSmallPairs];
    small_load(q, l);
    const int lane = threadIdx.x % kWave;
    for (int s = threadIdx.x / kWave; s < q.S; s += kSmallBlock / kWave) {
        double v = 0.0;
        int c = 0;
        for (int t = l.start[s] + lane; t < l.start[s + 1]; t += kWave)
            if (counts(q, t)) {
                v += (double)logp[t] - (ref ? (double)ref[t] : 0.0);
                ++c;
            }
        v = wave_sum(v);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, kWave);
        if (lane == 0) {
            sum[s] = v;
            l.cnt[s] = c;
        }
    }
    __syncthreads();
    if (threadIdx.x < kWave) {  // a lane per pair
        const int i = lane;
        double loss = 0.0, d = 0.0;
        const bool in = 2 * i < q.S, ok = in && l.cnt[2 * i] > 0 && l.cnt[2 * i + 1] > 0;
        if (ok) loss = pair_loss(beta * (sum[2 * i] - sum[2 * i + 1]), smooth, d);
        if (in && margin_out) margin_out[i] = ok ? (float)(beta * (sum[2 * i] - sum[2 * i + 1])) : 0.f;
        const int live = __popcll(__ballot(ok));
        loss = wave_sum(loss);
        if (in) slope[i] = ok ? beta * d / (double)live : 0.0;
        if (i == 0) loss_out[0] = live ? (float)(loss / (double)live) : 0.f;
    }
    __syncthreads();
    if (grad)
        for (int t = threadIdx.x; t < q.n; t += kSmallBlock) {
            const int s = counts(q, t) ? small_seq(q, l, t) : -1;
            grad[t] = s < 0 ? 0.f : (float)((s & 1 ? -slope[s / 2] : slope[s / 2]) * loss_scale);
        }
}

// Sequences longer than part_tokens on average are split, into at most
// max_parts and kMaxItems in all.
Seqs make_seqs(const int64_t* targets, const int64_t* start, int64_t n, int64_t S, int64_t V, int64_t part_tokens,
               int64_t max_parts) {
    int64_t parts = S > 0 ? cdiv(cdiv(n, S), part_tokens) : 1;
    if (parts > max_parts) parts = max_parts;
    if (S > 0 && parts > kMaxItems / S) parts = kMaxItems / S;
    if (parts < 1) parts = 1;
    return Seqs{targets, start, n, S, V, (int)parts};
}
// A lane takes its tokens in turn: parts of a few per lane.
Seqs policy_seqs(const int64_t* targets, const int64_t* start, int64_t n, int64_t S, int64_t V) {
    return make_seqs(targets, start, n, S, V, 1024, kMaxItems);
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
    if (n > INT32_MAX || S > (int64_t(1) << 30))
        return set_error(AR_EUNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^30 sequences", nm);
    return AR_OK;
}
// out: an array of n floats that the call writes, one value per token, after
// it has read that token's inputs: it may be one of them, not overlap one.
int32_t check_policy(const char* nm, const float* out, const float* logp, const float* old, const float* ref,
                     const float* adv, int64_t n, double lo, double hi, double kl) {
    AR_CHECK_ARG(n <= 0 || adv, "%s: null pointer", nm);
    for (const float* in : {logp, old, ref, adv})
        AR_CHECK_ARG(out == in || !overlaps(out, n * sizeof(float), in, n * sizeof(float)),
                     "%s: an output overlaps an input without being it", nm);
    AR_CHECK_ARG(lo >= 0.0 && hi >= 0.0, "%s: clip_low and clip_high must not be negative", nm);
    AR_CHECK_ARG(kl == kl && (kl == 0.0 || ref || n <= 0), "%s: a KL coefficient needs ref_logp", nm);
    return AR_OK;
}

struct PolicyWs {
    int* cnt;
    Totals* total;
    float* weight;
    double2* part;
    char* rows;  // lp_rows' scratch
    size_t bytes;
};
PolicyWs policy_ws(char* base, const Seqs& q, int64_t nweights, int64_t nparts, size_t row_bytes = 0) {
    Scratch s{base};
    PolicyWs w;
    w.cnt = s.take<int>(q.S * q.parts);
    w.total = s.take<Totals>(1);
    w.weight = s.take<float>(nweights);
    w.part = s.take<double2>(pair_room(nparts));
    w.rows = s.take<char>(row_bytes);
    w.bytes = s.used;
    return w;
}
// The items' counts, and the totals if they are not summed inline.
const Totals* launch_counts(hipStream_t st, const Seqs& q, const PolicyWs& w) {
    const int64_t items = q.S * q.parts;
    count_k<<<item_grid(q), kTokBlock, 0, st>>>(q, w.cnt);
    if (items <= kInlineItems) return nullptr;
    totals_k<<<1, 1024, 0, st>>>(q, w.cnt, w.total);
    return w.total;
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
    if (const int32_t r = check_policy(nm, grad_logp, logp, old_logp, ref_logp, advantages, num_tokens, clip_low,
                                       clip_high, kl_coef))
        return r;
    const Seqs q = policy_seqs(targets, seq_start, num_tokens, num_seqs, vocab_size);
    const PolicyTokens a{logp, PolicyIn{old_logp, ref_logp, advantages, 1.0 - clip_low, 1.0 + clip_high, kl_coef},
                         per_seq, loss_scale, grad_logp};
    if (num_tokens <= kSmallPolicy && num_seqs <= kSmallSeqs) {
        policy_small_k<<<1, kSmallBlock, 0, S(stream)>>>(q, a, loss_out);
        return check_launch(nm);
    }
    const unsigned blocks = item_grid(q);
    int32_t status;
    char* base = static_cast<char*>(workspace(S(stream), policy_ws(nullptr, q, 0, blocks).bytes, &status));
    if (!base) return status;
    const PolicyWs w = policy_ws(base, q, 0, blocks);
    const Totals* total = launch_counts(S(stream), q, w);
    if (num_tokens / blocks > kTokBlock)
        policy_tokens_k<512><<<blocks, 512, 0, S(stream)>>>(q, w.cnt, total, a, w.part);
    else
        policy_tokens_k<kTokBlock><<<blocks, kTokBlock, 0, S(stream)>>>(q, w.cnt, total, a, w.part);
    sum_pairs(S(stream), w.part, blocks, loss_out);
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
    if (const int32_t r =
            check_rows(nm, logits, logits_bf16, grad_logits, targets, logp_out, num_tokens, vocab_size))
        return r;
    if (const int32_t r = check_seqs(nm, targets, seq_start, num_tokens, num_seqs, vocab_size)) return r;
    if (const int32_t r = check_policy(nm, logp_out, nullptr, old_logp, ref_logp, advantages, num_tokens, clip_low,
                                       clip_high, kl_coef))
        return r;
    const Seqs q = policy_seqs(targets, seq_start, num_tokens, num_seqs, vocab_size);
    const size_t row_bytes = lp_scratch(LpOp::POLICY, logits_bf16 != 0, num_tokens, vocab_size);
    int32_t status;
    char* base = static_cast<char*>(
        workspace(S(stream), policy_ws(nullptr, q, num_tokens, num_tokens, row_bytes).bytes, &status));
    if (!base) return status;
    const PolicyWs w = policy_ws(base, q, num_tokens, num_tokens, row_bytes);
    if (num_tokens <= kSmallPolicy && num_seqs <= kSmallSeqs) {
        weight_small_k<<<1, kSmallBlock, 0, S(stream)>>>(q, per_seq, w.weight);
    } else {
        const Totals* total = launch_counts(S(stream), q, w);
        weight_k<<<item_grid(q), kTokBlock, 0, S(stream)>>>(q, w.cnt, total, per_seq, w.weight);
    }
    if (const int32_t r = check_launch(nm)) return r;
    LpRows a;
    a.logits = logits;
    a.grad = grad_logits;
    a.targets = targets;
    a.logp = logp_out;
    a.weight = w.weight;
    a.terms = w.part;
    a.scratch = row_bytes ? w.rows : nullptr;
    a.policy = PolicyIn{old_logp, ref_logp, advantages, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
    a.cap = cap;
    a.loss_scale = loss_scale;
    a.n = num_tokens;
    a.V = vocab_size;
    if (const int32_t r = lp_rows(S(stream), LpOp::POLICY, logits_bf16 != 0, a, nm)) return r;
    sum_pairs(S(stream), w.part, num_tokens, loss_out);
    return check_launch(nm);
}

extern "C" int32_t ar_preference_loss(ar_stream_t stream, float* loss_out, float* margin_out, float* grad_logp,
                                      const float* logp, const float* ref_logp, const int64_t* targets,
                                      const int64_t* seq_start, double beta, double label_smoothing,
                                      int64_t num_tokens, int64_t num_pairs, int64_t vocab_size, float loss_scale) {
    const char* nm = "preference_loss";
    AR_CHECK_ARG(loss_out && seq_start && (num_tokens <= 0 || logp), "%s: null pointer", nm);
    AR_CHECK_ARG(num_pairs >= 0, "%s: bad number of pairs", nm);
    if (num_pairs > (1 << 29)) return set_error(AR_EUNSUPPORTED, "%s: more than 2^29 pairs", nm);
    if (const int32_t r = check_seqs(nm, targets, seq_start, num_tokens, 2 * num_pairs, vocab_size)) return r;
    AR_CHECK_ARG(beta == beta && label_smoothing >= 0.0 && label_smoothing <= 1.0,
                 "%s: label_smoothing must lie in [0, 1]", nm);
    AR_CHECK_ARG(!overlaps(grad_logp, num_tokens * sizeof(float), logp, num_tokens * sizeof(float)) &&
                     !overlaps(grad_logp, num_tokens * sizeof(float), ref_logp, num_tokens * sizeof(float)),
                 "%s: grad_logp must not overlap logp or ref_logp", nm);
    const Seqs q = make_seqs(targets, seq_start, num_tokens, 2 * num_pairs, vocab_size, 1024,
                             num_pairs <= kManyParts ? 64 : kFewParts);
    if (num_tokens <= kSmallTokens && num_pairs <= kSmallPairs) {
        pair_small_k<<<1, kSmallBlock, 0, S(stream)>>>(q, logp, ref_logp, beta, label_smoothing, loss_scale, loss_out,
                                                       margin_out, grad_logp);
        return check_launch(nm);
    }
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
    pair_sums_k<<<g, kTokBlock, 0, S(stream)>>>(q, logp, ref_logp, sum, cnt);
    pair_loss_k<<<1, 1024, 0, S(stream)>>>(sum, cnt, num_pairs, q.parts, beta, label_smoothing, d, slope, loss_out,
                                           margin_out);
    if (grad_logp && num_tokens > 0) pair_grad_k<<<g, kTokBlock, 0, S(stream)>>>(q, slope, loss_scale, grad_logp);
    return check_launch(nm);
}
