// ar_logprob.hip -- log-probabilities of tokens from rows of logits, and the
// gradients that go back through them.
//
// A row z [V] with target y: lse = m + log sum_j exp(z_j - m), m = max_j z_j,
// logp = z_y - lse, and for a loss with gradient g by logp
//   d loss / d x_j = g ([j = y] - exp(z_j - lse)) (1 - (z_j / cap)^2),
// the last factor the derivative of z = cap tanh(x / cap) (1 without a cap).
// Bound by HBM: a row is read once (the running maximum and sum need one
// pass) and a row of the gradient written once; a part of rows of more than
// 208 KiB, and few long rows, are read twice.  16384 rows of 32768 bf16 values:
// forward 173 us (6.2 TB/s), gradient 357 us (6.0); 65536 rows of 8192 fp32
// values: gradient 719 us (6.0), policy step with a quarter of the tokens not
// counting 704 us.
#include <math.h>

#include <algorithm>

#include "ar_losses.hpp"

namespace ar {
namespace {

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

// Reductions over a wave without LDS: lanes to the left within rows of 16 (row
// shift 1, 2, 4, 8), then rows to the right of them (broadcasts of lane 15 and
// 31), `none` where there is no lane; the last lane's result to all.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float none, float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
struct Max {
    static constexpr float none = -INFINITY;
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
struct Sum {
    static constexpr float none = 0.f;
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
template <typename O>
__device__ __forceinline__ float of_row16(float v) {  // lane 15 of each row
    v = O::of(v, dpp<0x111>(O::none, v));
    v = O::of(v, dpp<0x112>(O::none, v));
    v = O::of(v, dpp<0x114>(O::none, v));
    return O::of(v, dpp<0x118>(O::none, v));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
template <typename O>
__device__ __forceinline__ float of_wave(float v) {
    v = of_row16<O>(v);
    v = O::of(v, dpp<0x142, 0xa>(O::none, v));
    return lane_value(O::of(v, dpp<0x143, 0xc>(O::none, v)), 63);
}
// Over a block of up to 16 waves; red: a value per wave that nothing else of
// the kernel uses.  One barrier.
template <typename O>
__device__ __forceinline__ float of_block(float v, float* red) {
    v = of_wave<O>(v);
    const int lane = threadIdx.x % kWave, nw = blockDim.x / kWave;
    if (nw == 1) return v;
    if (lane == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    return lane_value(of_row16<O>(lane < nw ? red[lane] : O::none), 15);
}

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
    // the same sum under another maximum (-inf: of nothing)
    __device__ __forceinline__ float under(float nm) const { return s * __expf(m - (nm == -INFINITY ? 0.f : nm)); }
};
__device__ __forceinline__ MaxSum wave_max_sum(MaxSum v) {
    MaxSum t;
    t.m = of_wave<Max>(v.m);
    t.s = of_wave<Sum>(v.under(t.m));
    return t;
}
// red: two values per wave.
__device__ __forceinline__ MaxSum block_max_sum(MaxSum v, float* red) {
    v = wave_max_sum(v);
    const int w = threadIdx.x / kWave, lane = threadIdx.x % kWave, nw = blockDim.x / kWave;
    if (nw == 1) return v;
    if (lane == 0) {
        red[2 * w] = v.m;
        red[2 * w + 1] = v.s;
    }
    __syncthreads();
    MaxSum o, t;
    if (lane < nw) {
        o.m = red[2 * lane];
        o.s = red[2 * lane + 1];
    }
    t.m = lane_value(of_row16<Max>(o.m), 15);
    t.s = lane_value(of_row16<Sum>(o.under(t.m)), 15);
    return t;
}

// A token's values for POLICY, loaded ahead of its row; nothing otherwise.  The
// row waits for coef, its gradient by logp (w: the token's weight or
// gradient); what else the token has comes behind the row's last store, in one
// lane (65536 rows of 8192 fp32 values: both before the row in fp64 798 us, in
// fp32 725, so 704).
template <LpOp OP>
struct RowToken {
    __device__ __forceinline__ explicit RowToken(const PolicyToken&) {}
    __device__ __forceinline__ RowToken(const LpRows&, int64_t) {}
    __device__ __forceinline__ float coef(const LpRows&, float w, float) const { return w; }
    __device__ __forceinline__ void finish(const LpRows&, int64_t, float, float) const {}
};
template <>
struct RowToken<LpOp::POLICY> {
    PolicyToken t;
    __device__ __forceinline__ explicit RowToken(const PolicyToken& token) : t(token) {}
    __device__ __forceinline__ RowToken(const LpRows& a, int64_t r) : t(a.policy, r) {}
    __device__ __forceinline__ float coef(const LpRows& a, float w, float logp) const {
        return w * policy_slope(logp, t, a.policy) * a.loss_scale;
    }
    __device__ __forceinline__ void finish(const LpRows& a, int64_t r, float w, float logp) const {
        const PolicyTerm<float> o = policy_term<float>(logp, t, a.policy);
        if (a.logp) a.logp[r] = logp;
        a.terms[r] = make_double2((double)w * o.loss, (double)w * o.kl);
    }
};

// log2 of a sum: its exponent, and the logarithm of its mantissa (in
// [sqrt(1/2), sqrt(2)): off by 2^-25).  Sums over tokens add up what
// log-probabilities are off by, so they are put together in fp64 and rounded
// once (the forward of 131072 rows of 1024 bf16 values: 51 us; with all of the
// logarithm in fp64, 64).
__device__ __forceinline__ double log2_sum(float s) {
    float f = __builtin_amdgcn_frexp_mantf(s);
    int e = __builtin_amdgcn_frexp_expf(s);
    if (f < 0.707106781f) {
        f *= 2.f;
        --e;
    }
    return (double)e + (double)log2f(f);
}
constexpr double kLn2 = 0.6931471805599453;

// exp(z - m).  SUB: the difference first.  Otherwise one fma and the hardware's
// exponential: z log2 e - m log2 e, rounded once.  The second product's own
// rounding is a factor common to the whole row, which the sum has too; it is
// small up to |m| = 2^20, and the caller sees to that.
constexpr float kLog2e = 1.44269504f;
constexpr float kFar = 1048576.f;
template <bool SUB>
struct RowExp {
    float m, c;
    __device__ __forceinline__ explicit RowExp(float max) : m(max), c(max * -kLog2e) {}
    __device__ __forceinline__ float log2_of(float z) const {
        return SUB ? (z - m) * kLog2e : fmaf(z, kLog2e, c);
    }
    __device__ __forceinline__ float operator()(float z) const { return __builtin_amdgcn_exp2f(log2_of(z)); }
    // log-probability of z where the row's exponentials sum up to s
    __device__ __forceinline__ float logp(float z, float s) const {
        const float common = SUB ? 0.f : fmaf(m, kLog2e, c);  // log2 of the row's common factor
        return (float)((double)z - (double)m - (log2_sum(s) - (double)common) * kLn2);
    }
};

// The gradient of a value that is not the target: -g p f; the target's has
// g f besides, f = 1 - (z / cap)^2 (values past the cap by rounding: 0).
// z0: what the values were shortened by.
template <bool SUB>
struct RowGrad {
    RowExp<SUB> ex;
    float g, sum, gs, rcap, u0;  // gs = -g / sum
    __device__ __forceinline__ RowGrad(RowExp<SUB> e, float cap, float coef, float s, float z0)
        : ex(e), g(coef), sum(s), gs(-coef / s), rcap(cap > 0.f ? 1.f / cap : 0.f), u0(z0 * rcap) {}
    __device__ __forceinline__ float factor(float z) const {
        const float u = fmaf(z, rcap, u0);
        return fminf(fmaxf(fmaf(-u, u, 1.f), 0.f), 1.f);
    }
    __device__ __forceinline__ float operator()(float z) const { return gs * ex(z) * factor(z); }
    // (a target that holds the whole row: exactly 0)
    __device__ __forceinline__ float target(float z) const { return g * (1.f - ex(z) / sum) * factor(z); }
};

template <typename T>
__device__ __forceinline__ void zero_row(T* out, int V) {
    using R = Row<T>;
    const int nb = V / R::E;
    for (int c = threadIdx.x; c < nb; c += blockDim.x) R::store(out + c * R::E, u32x4{0, 0, 0, 0});
    for (int j = nb * R::E + threadIdx.x; j < V; j += blockDim.x) out[j] = from_f32<T>(0.f);
}

// Whether a token's logits are read; if not, its outputs but for the row are
// written here (out).
template <LpOp OP>
__device__ __forceinline__ bool row_live(const LpRows& a, int64_t r, int64_t y, float& w, bool out) {
    w = 1.f;
    if constexpr (OP == LpOp::BWD) w = a.grad_logp[r];
    if constexpr (OP == LpOp::POLICY) w = a.weight[r];
    if (y >= 0 && y < a.V && w != 0.f) return true;
    if constexpr (OP != LpOp::BWD)
        if (out && threadIdx.x == 0 && a.logp) a.logp[r] = 0.f;
    if constexpr (OP == LpOp::POLICY)
        if (out && threadIdx.x == 0) a.terms[r] = make_double2(0.0, 0.0);
    return false;
}
template <typename T, LpOp OP>
__device__ __forceinline__ bool row_counts(const LpRows& a, int64_t r, int64_t y, float& w) {
    if (row_live<OP>(a, r, y, w, true)) return true;
    if constexpr (OP != LpOp::FWD) zero_row(static_cast<T*>(a.grad) + r * a.V, (int)a.V);
    return false;
}

// The maximum and sum of N chunks of a row, the sum so far rescaled once.
template <typename T, int N>
__device__ __forceinline__ void add_chunks(MaxSum& v, const u32x4* q) {
    using R = Row<T>;
    float cm = R::get(q[0], 0);
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < R::E; ++i) cm = fmaxf(cm, R::get(q[k], i));
    const float nm = fmaxf(v.m, cm), use = nm == -INFINITY ? 0.f : nm;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < R::E; ++i) s += __expf(R::get(q[k], i) - use);
    v.s = fmaf(v.s, __expf(v.m - use), s);
    v.m = nm;
}

// Between two passes over held chunks: what the first one made of them (bf16
// values widened to fp32: twice the registers) is made again, not kept.
__device__ __forceinline__ void again(u32x4& q) { asm volatile("" : "+v"(q)); }

constexpr int kBatch = 4;  // chunks a lane has in flight

// The maximum and sum of a row's chunks [lo, hi), lane t's lo + t, lo + t + TB, ...
template <typename T, int TB>
__device__ __forceinline__ MaxSum max_sum(const T* chunks, int lo, int hi) {
    using R = Row<T>;
    MaxSum v;
    u32x4 q[kBatch];
    int c = lo + threadIdx.x;
    for (; c + (kBatch - 1) * TB < hi; c += kBatch * TB) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) q[k] = R::load(chunks + (c + k * TB) * R::E);
        add_chunks<T, kBatch>(v, q);
    }
    for (; c < hi; c += TB) {
        q[0] = R::load(chunks + c * R::E);
        add_chunks<T, 1>(v, q);
    }
    return v;
}
__device__ __forceinline__ void add_value(MaxSum& v, float z) { v.add(z, z == -INFINITY ? 0.f : __expf(z - z)); }

// The forward: rows of any length, read once.
template <typename T, int TB>
__global__ __launch_bounds__(TB) void lp_fwd_k(LpRows a) {
    __shared__ float red[2 * (TB / kWave)];
    const int64_t r = a.first + blockIdx.x;
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    float w;
    if (!row_live<LpOp::FWD>(a, r, y, w, true)) return;
    const Span<T> sp(row, V);
    const int ej = sp.edge(tid, V);
    const float zy = to_f32<T>(row[y]), ez = ej >= 0 ? to_f32<T>(row[ej]) : -INFINITY;
    MaxSum v = max_sum<T, TB>(row + sp.h, 0, sp.nb);
    add_value(v, ez);
    v = block_max_sum(v, red);
    if (tid == 0) a.logp[r] = RowExp<true>(v.m).logp(zy, v.s);
}

// The gradient of rows of up to (NV + NL) TB chunks of 16 bytes, held on the
// CU, NV a lane in registers and NL in LDS: one read, and the maximum before the
// exponentials.  REST: longer rows, of which what is not held is read again for
// the gradient, which is written past the caches (1000 rows of 300001 fp32
// values: 700 -> 640 us, and with a pass that reads the gradient next 940 -> 842;
// shorter rows gain nothing, and a pass over 128 MB of gradient takes 45 us for 21).
// Rows go last to first: what the forward or the logits' product left in the
// cache is read before it is gone, and what reads the gradient next finds its
// first rows there (256 MB of fp32 and a pass over it 175 -> 160 us).
// Only rows with a chunk may come to an instance with SURE > 0: its first SURE
// steps ask no question (the row's last chunk is loaded where a lane has none,
// and not used).
template <typename T, LpOp OP, int TB, int NV, int SURE, int NL = 0, bool REST = false>
__global__ __launch_bounds__(TB, NV > 9 ? 4 : 8) void lp_held_k(LpRows a) {
    using R = Row<T>;
    constexpr int E = R::E, N = NV + NL;
    constexpr bool kFirst = NV > 9;  // registers for the rest's chunks beside those held
    __shared__ float red[2 * (TB / kWave)];
    __shared__ u32x4 more[NL ? NL * TB : 1];  // lane t's: t, t + TB, ...
    const int64_t r = a.first + (gridDim.x - 1 - blockIdx.x);
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    T* out = static_cast<T*>(a.grad) + r * a.V;
    float w;
    if (!row_counts<T, OP>(a, r, y, w)) return;
    const RowToken<OP> token(a, r);
    const Span<T> sp(row, V);
    const int h = sp.h, nb = sp.nb;
    const u32x4 none = R::fill(-INFINITY);
    MaxSum rest;
    if constexpr (REST && !kFirst) {
        rest = max_sum<T, TB>(row + h, N * TB, nb);
        __builtin_amdgcn_sched_barrier(0);
    }
    u32x4 q[N];  // from NV on only until they are in LDS
    auto there = [&](int k) { return k < SURE || k * TB < nb; };
    auto chunk = [&](int k) { return k < NV ? q[k] : more[(k - NV) * TB + tid]; };
    auto keep = [&](int k, u32x4 v) {
        if (k < NV) q[k] = v;
        else more[(k - NV) * TB + tid] = v;
    };
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (there(k)) q[k] = R::load(row + h + min(tid + k * TB, nb - 1) * E);
    const int ej = sp.edge(tid, V);
    float ez = ej >= 0 ? to_f32<T>(row[ej]) : -INFINITY;
    float zy = to_f32<T>(row[y]);
    if constexpr (REST && kFirst) rest = max_sum<T, TB>(row + h, N * TB, nb);
    float mt = fmaxf(ez, rest.m);
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (there(k)) {
            if (tid + k * TB >= nb) q[k] = none;
#pragma unroll
            for (int i = 0; i < E; ++i) mt = fmaxf(mt, R::get(q[k], i));
            again(q[k]);
            if (k >= NV) keep(k, q[k]);
        }
    float m = of_block<Max>(mt, red);
    float z0 = 0.f;
    if (__builtin_amdgcn_readfirstlane(!(fabsf(m) < kFar))) {
        // the same in every lane: shorten the row by its maximum.  (Values
        // that bf16 rounds here differ from it by 2^12 or more: no weight.)
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (there(k)) {
                const u32x4 v = chunk(k);
                float x[E];
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = R::get(v, i) - m;
                keep(k, R::pack(x));
                if (k < NV) again(q[k]);
            }
        ez -= m;
        zy -= m;
        rest.m -= m;
        z0 = m;
        m = 0.f;
    }
    const RowExp<false> ex(m);
    float st = ex(ez);
    if constexpr (REST) st += rest.s * ex(rest.m);
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (there(k)) {
            const u32x4 v = chunk(k);
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s += ex(R::get(v, i));
            st += s;
            if (k < NV) again(q[k]);
        }
    st = of_block<Sum>(st, red + TB / kWave);
    const float logp = ex.logp(zy, st);
    const RowGrad<false> grad(ex, a.cap, token.coef(a, w, logp), st, z0);
    const int yc = y < h ? -1 : ((int)y - h) / E, yi = y < h ? 0 : ((int)y - h) % E;
    auto emit = [&](int c, u32x4 v, float less) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = grad(R::get(v, i) - less);
        if (c == yc) {
            const float t = grad.target(zy);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = i == yi ? t : x[i];
        }
        if constexpr (REST) R::store_nt(out + h + c * E, R::pack(x));
        else R::store(out + h + c * E, R::pack(x));
    };
    auto emit_rest = [&] {
        int c = N * TB + tid;
        for (; c + (kBatch - 1) * TB < nb; c += kBatch * TB) {
            u32x4 v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = R::load(row + h + (c + k * TB) * E);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) emit(c + k * TB, v[k], z0);
        }
        for (; c < nb; c += TB) emit(c, R::load(row + h + c * E), z0);
    };
    if constexpr (REST && kFirst) emit_rest();
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (there(k) && tid + k * TB < nb) emit(tid + k * TB, chunk(k), 0.f);
    if constexpr (REST && !kFirst) {
        __builtin_amdgcn_sched_barrier(0);
        emit_rest();
    }
    if (ej >= 0) out[ej] = from_f32<T>(ej == y ? grad.target(zy) : grad(ez));
    if (tid == 0) token.finish(a, r, w, logp);
}

// ---- few long rows: each split over several workgroups ----
// part[r][p]: the maximum and sum of part p's chunks, part 0 with the values
// outside the chunks; zy[r]: the target's; token[r]: POLICY's inputs, of which
// logp_out may be one (a row's workgroups end in any order).
struct Split {
    MaxSum* part;
    PolicyToken* token;
    float* zy;
    int parts;
    __device__ __forceinline__ int lo(int nb) const { return min(nb, (int)blockIdx.x * ((nb + parts - 1) / parts)); }
    __device__ __forceinline__ int hi(int nb) const { return min(nb, lo(nb) + (nb + parts - 1) / parts); }
};
constexpr int kSplitBlock = 256;

template <typename T, LpOp OP>
__global__ __launch_bounds__(kSplitBlock) void lp_part_k(LpRows a, Split sp) {
    __shared__ float red[2 * (kSplitBlock / kWave)];
    const int64_t r = blockIdx.y;
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    float w;
    if (!row_live<OP>(a, r, y, w, false)) return;
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    const Span<T> s(row, V);
    const int hi = sp.hi(s.nb), ej = blockIdx.x == 0 ? s.edge(tid, V) : -1;
    MaxSum v = max_sum<T, kSplitBlock>(row + s.h, sp.lo(s.nb), hi);
    if (ej >= 0) add_value(v, to_f32<T>(row[ej]));
    v = block_max_sum(v, red);
    if (tid == 0) {
        sp.part[r * sp.parts + blockIdx.x] = v;
        if (blockIdx.x == 0) sp.zy[r] = to_f32<T>(row[y]);
        if (OP == LpOp::POLICY && blockIdx.x == 0) sp.token[r] = PolicyToken(a.policy, r);
    }
}
// The whole row's, by every wave.
__device__ __forceinline__ MaxSum join_parts(const Split& sp, int64_t r) {
    const int lane = threadIdx.x % kWave;
    MaxSum v;
    if (lane < sp.parts) v = sp.part[r * sp.parts + lane];
    return wave_max_sum(v);
}
__global__ __launch_bounds__(kWave) void lp_join_k(LpRows a, Split sp) {
    const int64_t r = blockIdx.x;
    float w;
    if (!row_live<LpOp::FWD>(a, r, a.targets[r], w, true)) return;
    const MaxSum v = join_parts(sp, r);
    if (threadIdx.x == 0) a.logp[r] = RowExp<true>(v.m).logp(sp.zy[r], v.s);
}
template <typename T, LpOp OP>
__global__ __launch_bounds__(kSplitBlock) void lp_apply_k(LpRows a, Split sp) {
    using R = Row<T>;
    constexpr int E = R::E;
    const int64_t r = blockIdx.y;
    const int V = (int)a.V, tid = threadIdx.x;
    const int64_t y = a.targets[r];
    const T* row = static_cast<const T*>(a.logits) + r * a.V;
    T* out = static_cast<T*>(a.grad) + r * a.V;
    const Span<T> s(row, V);
    const int hi = sp.hi(s.nb), ej = blockIdx.x == 0 ? s.edge(tid, V) : -1;
    float w;
    if (!row_live<OP>(a, r, y, w, blockIdx.x == 0)) {
        for (int c = sp.lo(s.nb) + tid; c < hi; c += kSplitBlock) R::store(out + s.h + c * E, u32x4{0, 0, 0, 0});
        if (ej >= 0) out[ej] = from_f32<T>(0.f);
        return;
    }
    const RowToken<OP> token(OP == LpOp::POLICY ? sp.token[r] : PolicyToken());
    const MaxSum v = join_parts(sp, r);
    const float zy = sp.zy[r];
    const RowExp<true> ex(v.m);
    const float logp = ex.logp(zy, v.s);
    const RowGrad<true> grad(ex, a.cap, token.coef(a, w, logp), v.s, 0.f);
    for (int c = sp.lo(s.nb) + tid; c < hi; c += kSplitBlock) {
        const u32x4 z = R::load(row + s.h + c * E);
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = s.h + c * E + i == y ? grad.target(zy) : grad(R::get(z, i));
        R::store(out + s.h + c * E, R::pack(x));
    }
    if (ej >= 0) out[ej] = from_f32<T>(ej == y ? grad.target(zy) : grad(to_f32<T>(row[ej])));
    if (tid == 0 && blockIdx.x == 0) token.finish(a, r, w, logp);
}

// Splitting reads the row twice and takes two launches: for long rows of which
// there are too few to fill the card.  Unsplit and split, us a call (7 to 9 of
// them the host's): gradient of 1, 64, 128 rows of 131072 bf16 values 17.8 9.5,
// 20.8 11.6, 24.4 19.1; of 65536 fp32 10.2 9.4, 12.8 9.9, 17.6 17.1; the forward
// of 1, 128 rows of 150001 bf16 9.0 9.1, 11.0 11.0, of 300000 14.9 9.0, 17.9 16.9.
constexpr int64_t kSplitRows = 128, kSplitValues = 65536, kPartChunks = 4 * kSplitBlock;
int split_parts(LpOp op, int64_t n, int64_t V, int E) {
    if (n > kSplitRows || V < (op == LpOp::FWD ? 3 * kSplitValues : kSplitValues)) return 1;
    int64_t p = cdiv(cdiv(V, E), kPartChunks);
    if (p > 1024 / n) p = 1024 / n;
    return (int)(p > kWave ? kWave : p);
}

// Lanes and chunks per lane by the row's chunks (TB/s of the row read and the
// gradient written).  With as few chunks per lane as 1024 lanes allow, down to
// two, a row is in flight the shortest: 8192 fp32 values 1024 x 2 6.1, 512 x 4
// 5.4, 256 x 8 5.5; 16384 1024 x 4 6.0, 512 x 8 5.3.  bf16 has twice the values
// per chunk and takes four: 8192 values 256 x 4 5.8, 512 x 2 5.6, 1024 x 1 3.7.
// Two workgroups of 1024 fit a CU with up to 64 registers and 80 KiB of LDS
// each, one with more, whose reads, sums and writes then take turns: 90000 bf16
// values 8 chunks in registers and 4 in LDS 5.0, 16 in registers 4.6; 50001 fp32
// 5.0, 4.7.  Two with a part of the row read again or one, which reads less of it
// again and has the cache to itself: 131072 bf16 4.7 4.0, 150001 4.5 4.2, 180000
// 4.5 4.5, 256000 4.5 4.6; 65536 fp32 5.1 5.1, 80001 4.7 4.8, 300001 3.4 4.2.  (One
// that keeps 8 more chunks in LDS: 256000 bf16 4.6, 300001 fp32 4.1.)
template <typename T, LpOp OP>
void launch_grad(hipStream_t st, const LpRows& a, unsigned g) {
    const int64_t nc = cdiv(a.V, Row<T>::E);
#define AR_HELD(TB, NV) lp_held_k<T, OP, TB, NV, NV / 2><<<g, TB, 0, st>>>(a)
    constexpr int M = sizeof(T) == 2 ? 4 : 2, HR = sizeof(T) == 2 ? 8 : 9;
    if (nc <= 64 * 2) lp_held_k<T, OP, 64, 2, 0><<<g, 64, 0, st>>>(a);  // rows without a whole chunk too
    else if (nc <= 128 * M) AR_HELD(128, M);
    else if (nc <= 256 * M) AR_HELD(256, M);
    else if (nc <= 512 * M) AR_HELD(512, M);
    else if (nc <= 1024 * M) AR_HELD(1024, M);
    else if (nc <= 1024 * 4) AR_HELD(1024, 4);
    else if (nc <= 1024 * 8) AR_HELD(1024, 8);
    else if (nc <= 1024 * (HR + 4)) lp_held_k<T, OP, 1024, HR, 8, 4><<<g, 1024, 0, st>>>(a);
    else if (nc <= 1024 * 20) lp_held_k<T, OP, 1024, 8, 8, 4, true><<<g, 1024, 0, st>>>(a);
    else lp_held_k<T, OP, 1024, 16, 16, 0, true><<<g, 1024, 0, st>>>(a);
#undef AR_HELD
}

// The forward alone: TB/s of the rows read, by lanes: 1024 bf16 values 64 5.7,
// 256 2.4; 8192 bf16 256 6.4, 1024 3.2; 8192 fp32 256 6.4, 1024 5.2; 32768 bf16
// 256 6.1, 1024 6.4; 150001 fp32 256 5.8, 1024 6.2.  Few rows: as many lanes as
// a workgroup has.
template <typename T>
void launch_fwd(hipStream_t st, const LpRows& a, unsigned g) {
    const int64_t nc = cdiv(a.V, Row<T>::E);
    if (nc <= 256) lp_fwd_k<T, 64><<<g, 64, 0, st>>>(a);
    else if (nc <= 2048 && a.n > 256) lp_fwd_k<T, 256><<<g, 256, 0, st>>>(a);
    else lp_fwd_k<T, 1024><<<g, 1024, 0, st>>>(a);
}

template <typename T, LpOp OP>
void launch_split(hipStream_t st, const LpRows& a, int parts) {
    MaxSum* const part = static_cast<MaxSum*>(a.scratch);
    PolicyToken* const token = reinterpret_cast<PolicyToken*>(part + a.n * parts);
    const Split sp{part, token, reinterpret_cast<float*>(token + (OP == LpOp::POLICY ? a.n : 0)), parts};
    const dim3 g(parts, (unsigned)a.n);
    lp_part_k<T, OP><<<g, kSplitBlock, 0, st>>>(a, sp);
    if constexpr (OP == LpOp::FWD) lp_join_k<<<(unsigned)a.n, kWave, 0, st>>>(a, sp);
    else lp_apply_k<T, OP><<<g, kSplitBlock, 0, st>>>(a, sp);
}

template <typename T, LpOp OP>
void launch(hipStream_t st, const LpRows& a) {
    const int parts = a.scratch ? split_parts(OP, a.n, a.V, Row<T>::E) : 1;
    if (parts > 1) return launch_split<T, OP>(st, a, parts);
    // a launch holds fewer than 2^32 lanes: 2^22 rows of 1024
    constexpr int64_t kRows = 1 << 21;
    LpRows part = a;
    for (part.first = 0; part.first < a.n; part.first += kRows) {
        const unsigned rows = (unsigned)std::min(kRows, a.n - part.first);
        if constexpr (OP == LpOp::FWD) launch_fwd<T>(st, part, rows);
        else launch_grad<T, OP>(st, part, rows);
    }
}

}  // namespace

size_t lp_scratch(LpOp op, bool bf16_logits, int64_t n, int64_t V) {
    const int parts = n > 0 ? split_parts(op, n, V, bf16_logits ? Row<bf16>::E : Row<float>::E) : 1;
    const size_t token = op == LpOp::POLICY ? sizeof(PolicyToken) : 0;
    return parts > 1 ? n * (parts * sizeof(MaxSum) + token + sizeof(float)) : 0;
}

int32_t lp_rows(hipStream_t st, LpOp op, bool bf16_logits, const LpRows& a, const char* nm) {
    if (a.n == 0) return AR_OK;
    if (op == LpOp::FWD) bf16_logits ? launch<bf16, LpOp::FWD>(st, a) : launch<float, LpOp::FWD>(st, a);
    else if (op == LpOp::BWD) bf16_logits ? launch<bf16, LpOp::BWD>(st, a) : launch<float, LpOp::BWD>(st, a);
    else bf16_logits ? launch<bf16, LpOp::POLICY>(st, a) : launch<float, LpOp::POLICY>(st, a);
    return check_launch(nm);
}

int32_t check_rows(const char* nm, const void* logits, int32_t logits_bf16, const void* grad, const int64_t* targets,
                   const float* logp, int64_t n, int64_t V) {
    AR_CHECK_ARG(n >= 0 && V > 0, "%s: bad shape", nm);
    AR_CHECK_ARG(n == 0 || (logits && targets), "%s: null pointer", nm);
    AR_CHECK_ARG(logits_bf16 == 0 || logits_bf16 == 1, "%s: logits_bf16 must be 0 or 1", nm);
    if (n > INT32_MAX || V > (int64_t(1) << 30))
        return set_error(AR_EUNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^30 logits per token", nm);
    const size_t es = logits_bf16 ? 2 : 4, bytes = (size_t)n * V * es;
    AR_CHECK_ARG(((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(grad)) & (es - 1)) == 0,
                 "%s: logits or their gradient not aligned to a value", nm);
    AR_CHECK_ARG(grad == logits || !overlaps(grad, bytes, logits, bytes),
                 "%s: the gradient overlaps the logits without being them", nm);
    AR_CHECK_ARG(!overlaps(logp, n * sizeof(float), logits, bytes) && !overlaps(logp, n * sizeof(float), grad, bytes),
                 "%s: an array by token overlaps the logits or their gradient", nm);
    return AR_OK;
}

}  // namespace ar

using namespace ar;

static int32_t rows_entry(ar_stream_t stream, LpOp op, bool bf16_logits, LpRows& a, const char* nm) {
    if (const size_t bytes = lp_scratch(op, bf16_logits, a.n, a.V)) {
        int32_t status;
        a.scratch = workspace(S(stream), bytes, &status);
        if (!a.scratch) return status;
    }
    return lp_rows(S(stream), op, bf16_logits, a, nm);
}

extern "C" int32_t ar_token_logprob_fwd(ar_stream_t stream, float* logp_out, const void* logits, int32_t logits_bf16,
                                        const int64_t* targets, int64_t num_tokens, int64_t vocab_size) {
    AR_CHECK_ARG(num_tokens <= 0 || logp_out, "token_logprob_fwd: null pointer");
    if (const int32_t r =
            check_rows("token_logprob_fwd", logits, logits_bf16, nullptr, targets, logp_out, num_tokens, vocab_size))
        return r;
    LpRows a;
    a.logits = logits;
    a.targets = targets;
    a.logp = logp_out;
    a.n = num_tokens;
    a.V = vocab_size;
    return rows_entry(stream, LpOp::FWD, logits_bf16 != 0, a, "token_logprob_fwd");
}

extern "C" int32_t ar_token_logprob_bwd(ar_stream_t stream, void* grad_logits, const void* logits, int32_t logits_bf16,
                                        const int64_t* targets, const float* grad_logp, float cap, int64_t num_tokens,
                                        int64_t vocab_size) {
    AR_CHECK_ARG(num_tokens <= 0 || (grad_logits && grad_logp), "token_logprob_bwd: null pointer");
    AR_CHECK_ARG(cap >= 0.f, "token_logprob_bwd: cap must not be negative");
    if (const int32_t r = check_rows("token_logprob_bwd", logits, logits_bf16, grad_logits, targets, grad_logp,
                                     num_tokens, vocab_size))
        return r;
    LpRows a;
    a.logits = logits;
    a.grad = grad_logits;
    a.targets = targets;
    a.grad_logp = grad_logp;
    a.cap = cap;
    a.n = num_tokens;
    a.V = vocab_size;
    return rows_entry(stream, LpOp::BWD, logits_bf16 != 0, a, "token_logprob_bwd");
}
