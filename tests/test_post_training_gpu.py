"""The post-training operators against plain implementations in 64 bits:
token log-probabilities with their gradient, the policy loss (from
log-probabilities and from logits), the preference loss, gradient clipping,
and a run of them together on the model."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
TINY = 2.0 ** -120


@pytest.fixture(scope="module")
def env():
    import torch
    from autoresearch_amd import ops
    return torch, ops


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def half_step(torch, t):
    return torch.finfo(t).eps / 2


def sum_rel(V):
    """Relative error of sum_j exp(z_j - m).  An exponential: the difference and
    its product with log2 e are rounded (2^-24 of up to 40 each; smaller
    exponentials do not show) and the exponential is off by 2 ulp.  The sum: a
    value passes at most V / 256 + 32 additions of its thread and of the trees."""
    return (2 * 40 + 4 + V / 256 + 32) * U


def logp_tol(V, z_y, m, lse, logp):
    """z_y - m, log's argument and result (2 ulp), their difference."""
    return sum_rel(V) + U * ((z_y - m).abs() + 4 * (lse - m).abs() + logp.abs()) + TINY


def ref_rows(torch, z, y):
    """logp, probabilities, lse, maximum, and whether a token counts, in 64 bits."""
    Z, V = z.double(), z.shape[1]
    ok = (y >= 0) & (y < V)
    m = Z.amax(1)
    lse = torch.logsumexp(Z, 1)
    z_y = Z.gather(1, y.clamp(0, V - 1)[:, None])[:, 0]
    logp = torch.where(ok, z_y - lse, torch.zeros_like(lse))
    return logp, torch.softmax(Z, 1), lse, m, z_y, ok


def ref_grad(torch, z, y, p, ok, g, cap):
    """The gradient by the logits and how far one in 32 bits may be off before
    its last rounding: p's exponential and sum, the products, the subtraction
    at the target, the softcap's factor 1 - u^2 with u = z / cap (u off by two
    roundings, u^2 by twice that, and its own)."""
    V = z.shape[1]
    g = torch.where(ok, g.double(), torch.zeros(len(g), dtype=torch.float64, device="cuda"))
    hot = torch.zeros_like(p).scatter_(1, y.clamp(0, V - 1)[:, None], 1.0)
    f = 1 - (z.double() / cap) ** 2 if cap else torch.ones_like(p)
    d = (hot - p) * f
    live = g != 0
    d = torch.where(live[:, None], d * g[:, None], torch.zeros_like(d))
    tol = (g.abs()[:, None] * (p * f.abs() * (sum_rel(V) + 90 * U) + (hot - p).abs() * (f.abs() * 4 * U + 5 * U)
                              + hot * 2 * U))
    return d, torch.where(live[:, None], tol, torch.zeros_like(tol))


def make_logits(torch, n, V, dtype, seed, cap=0.0, off=0):
    """Rows of a head a few units wide, at an element offset into their storage."""
    g = gen(torch, seed)
    store = torch.full((n * V + off + 16,), 7.0, dtype=dtype, device="cuda")
    z = store[off:off + n * V].view(n, V)
    x = torch.randn(n, V, generator=g, device="cuda") * 3
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    x.scatter_add_(1, y[:, None], torch.rand(n, 1, generator=g, device="cuda") * 6)
    z.copy_(cap * torch.tanh(x / cap) if cap else x)
    return z, y, store


def close(torch, got, want, tol, dtype):
    tol = tol + half_step(torch, dtype) * want.abs() + (2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -126)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


SIZES = [1, 2, 3, 7, 8, 9, 255, 511, 512, 513, 1025, 2047, 2048, 2050, 8191, 8192, 8200, 16385, 32768, 40001, 70001]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", SIZES + [131072, 131079, 270001])
@pytest.mark.parametrize("n,off", [(19, 0), (2, 1)])
def test_logprob_and_gradient(env, V, dtype, n, off):
    check_logprob_and_gradient(env, V, dtype, n, off)


# long rows that are many enough not to be split over workgroups
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [32769, 65537, 131072, 131079, 150001])
@pytest.mark.parametrize("n,off", [(128, 1), (129, 0), (131, 1)])
def test_many_long_rows(env, V, dtype, n, off):
    check_logprob_and_gradient(env, V, dtype, n, off)


def test_more_rows_than_a_launch_holds(env):
    torch, ops = env
    n, V = (1 << 21) + 3, 5
    g = gen(torch, 3)
    z, y = torch.randn(n, V, generator=g, device="cuda"), torch.randint(0, V, (n,), generator=g, device="cuda")
    logp, out = torch.empty(n, device="cuda"), torch.empty_like(z)
    ops.token_logprob_fwd(logp, z, y, n, V)
    ops.token_logprob_bwd(out, z, y, torch.ones(n, device="cuda"), 0.0, n, V)
    want, p, lse, m, z_y, ok = ref_rows(torch, z, y)
    close(torch, logp, want, logp_tol(V, z_y, m, lse, want), torch.float32)
    d, tol = ref_grad(torch, z, y, p, ok, torch.ones(n, device="cuda"), 0.0)
    close(torch, out, d, tol, torch.float32)


def check_logprob_and_gradient(env, V, dtype, n, off):
    torch, ops = env
    dt = getattr(torch, dtype)
    cap = 15.0 if V % 2 else 0.0
    z, y, store = make_logits(torch, n, V, dt, V + n, cap, off)
    if n > 9:
        y[3], y[5], y[0], y[1] = -1, V, V - 1, 0
    logp = torch.full((n,), 7.0, device="cuda")
    ops.token_logprob_fwd(logp, z, y, n, V)
    want, p, lse, m, z_y, ok = ref_rows(torch, z, y)
    close(torch, logp, want, torch.where(ok, logp_tol(V, z_y, m, lse, want), torch.zeros_like(want)), torch.float32)
    g = torch.randn(n, generator=gen(torch, 1), device="cuda") * 0.3
    if n > 9:
        g[7] = 0.0
    gstore = torch.full_like(store, 5.0)
    out = gstore[off:off + n * V].view(n, V)
    ops.token_logprob_bwd(out, z, y, g, cap, n, V)
    d, tol = ref_grad(torch, z, y, p, ok, g, cap)
    close(torch, out, d, tol, dt)
    assert (gstore[:off] == 5).all() and (gstore[off + n * V:] == 5).all()
    # in place, and the same bits (at the same alignment: a row's sums are taken in its chunks' order)
    z2 = store.clone()[off:off + n * V].view(n, V)
    ops.token_logprob_bwd(z2, z2, y, g, cap, n, V)
    assert torch.equal(z2, out)


def test_gradient_of_other_alignment_than_logits(env):
    torch, ops = env
    for dt in (torch.float32, torch.bfloat16):
        n, V = 5, 4099
        z, y, _ = make_logits(torch, n, V, dt, 4, 15.0, off=2)
        g = torch.randn(n, device="cuda")
        a = torch.empty(n, V, dtype=dt, device="cuda")
        b = torch.empty(n * V + 3, dtype=dt, device="cuda")[3:].view(n, V)
        ops.token_logprob_bwd(a, z, y, g, 15.0, n, V)
        ops.token_logprob_bwd(b, z, y, g, 15.0, n, V)
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [5, 513, 8192, 40001, 131079])
@pytest.mark.parametrize("n", [8, 700])
def test_rows_of_infinities_and_nan(env, V, dtype, n):
    check_rows_of_infinities_and_nan(env, V, dtype, min(n, 10_000_000 // V))


# rows too many to be split over workgroups, of which a part is read again
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [70001, 131079, 270001])
def test_many_long_rows_of_infinities_and_nan(env, V, dtype):
    check_rows_of_infinities_and_nan(env, V, dtype, 130)


def check_rows_of_infinities_and_nan(env, V, dtype, n):
    torch, ops = env
    dt = getattr(torch, dtype)
    z, y, _ = make_logits(torch, n, V, dt, V, 0.0)
    y[:8] = torch.tensor([V - 1, 0, 0, 0, -1, V + 5, 1, 1], device="cuda")
    z[0, : V - 1] = -math.inf          # one value left
    z[1, V // 2 + 1:] = -math.inf      # whole chunks without a value
    z[2] = -math.inf                   # no value: no distribution
    z[3, V // 2] = math.nan
    z[4] = math.nan                    # tokens that do not count
    z[5, 0] = math.inf
    z[6] = torch.finfo(dt).min         # a mask by the type's lowest value, but for two
    z[6, 0], z[6, 1] = 1.0, 2.0
    z[7, 0] = math.inf
    g = torch.ones(n, device="cuda")
    logp, out = torch.full((n,), 7.0, device="cuda"), torch.full_like(z, 7.0)
    ops.token_logprob_fwd(logp, z, y, n, V)
    ops.token_logprob_bwd(out, z, y, g, 0.0, n, V)
    assert logp[0] == 0.0 and (out[0] == 0).all()
    assert logp[2:4].isnan().all() and logp[7].isnan() and out[3].isnan().all() and out[7].isnan().all()
    assert (logp[4:6] == 0).all() and (out[4:6] == 0).all()
    live = torch.tensor([1, 6] + list(range(8, n)), device="cuda")
    want, p, lse, m, z_y, ok = ref_rows(torch, z[live], y[live])
    close(torch, logp[live], want, logp_tol(V, z_y, m, lse, want), torch.float32)
    d, tol = ref_grad(torch, z[live], y[live], p, ok, g[live], 0.0)
    close(torch, out[live], d, tol, dt)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [9, 513, 8192, 40001, 150001, 270001])
def test_rows_of_far_values(env, V, dtype):
    check_rows_of_far_values(env, V, dtype, 1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [70001, 131079, 270001])
def test_many_long_rows_of_far_values(env, V, dtype):
    check_rows_of_far_values(env, V, dtype, 12)


def check_rows_of_far_values(env, V, dtype, times):
    """Rows whose largest value is far from zero, on both sides of 2^20, or the type's lowest or largest value."""
    torch, ops = env
    dt = getattr(torch, dtype)
    lowest, largest = torch.finfo(dt).min, torch.finfo(dt).max
    top = [1048575.0, 1048576.0, 1.0e6, 3.0e6, -1.0e6, -3.0e6, 1e9, -1e9, 3e37, lowest, largest] * times
    n = len(top)
    g = gen(torch, V)
    z = (torch.tensor(top, device="cuda", dtype=torch.float64)[:, None]
         - torch.rand(n, V, generator=g, device="cuda").double() * 4).clamp(lowest, largest).to(dt)
    z[:, 0] = torch.tensor(top, device="cuda", dtype=torch.float64).to(dt)
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    z[2, 1:] = 0.0  # one value holds all
    z[3, V // 2:] = -math.inf
    y[3] = 0
    gl = torch.ones(n, device="cuda")
    logp, out = torch.empty(n, device="cuda"), torch.empty_like(z)
    ops.token_logprob_fwd(logp, z, y, n, V)
    ops.token_logprob_bwd(out, z, y, gl, 0.0, n, V)
    want, p, lse, m, z_y, ok = ref_rows(torch, z, y)
    want = (z_y - m) - torch.log(torch.exp(z.double() - m[:, None]).sum(1))  # lse itself is rounded to the values' size
    close(torch, logp, want, logp_tol(V, z_y, m, m + torch.log(torch.exp(z.double() - m[:, None]).sum(1)), want)
          + U * 4 * math.log(V), torch.float32)
    d, tol = ref_grad(torch, z, y, p, ok, gl, 0.0)
    close(torch, out, d, tol, dt)


# ---------------------------------------------------------------- policy

def ref_weights(torch, y, start, V, per_seq):
    n = len(y)
    seq = torch.full((n,), -1, dtype=torch.int64)
    b = start.cpu().tolist()
    for s in range(len(b) - 1):
        seq[b[s]:b[s + 1]] = s
    seq = seq.cuda()
    ok = (y >= 0) & (y < V) & (seq >= 0)
    w = torch.zeros(n, dtype=torch.float64, device="cuda")
    cnt = [int((ok & (seq == s)).sum()) for s in range(len(b) - 1)]
    for s, c in enumerate(cnt):
        if c:
            w[ok & (seq == s)] = 1 / (c * sum(1 for x in cnt if x)) if per_seq else 1 / sum(cnt)
    return w, ok, seq, cnt


def ref_policy(torch, logp, old, ref, adv, w, ok, lo, hi, kl_coef):
    """loss, mean KL, gradient by logp, and the gradient's slope by an error of logp."""
    zero = torch.zeros_like(w)
    lp = logp.double()
    r = torch.exp(lp - old.double()) if old is not None else torch.ones_like(w)
    a = adv.double()
    binds = ((a > 0) & (r > 1 + hi)) | ((a < 0) & (r < 1 - lo))
    pg = torch.maximum(-a * r, -a * r.clamp(1 - lo, 1 + hi))
    k = ref.double() - lp if ref is not None else zero
    kl = torch.expm1(k) - k
    g = torch.where(binds, zero, -a * r) - kl_coef * torch.expm1(k)
    slope = torch.where(binds, zero, a.abs() * r) + abs(kl_coef) * torch.exp(k)
    pick = lambda x: torch.where(ok, w * x, zero)  # noqa: E731
    return pick(pg + kl_coef * kl), pick(kl), pick(g), pick(slope)


def make_tokens(torch, n, start, seed, V=100):
    g = gen(torch, seed)
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    y[torch.rand(n, generator=g, device="cuda") < 0.3] = -1
    y[torch.rand(n, generator=g, device="cuda") < 0.02] = V
    logp = -torch.rand(n, generator=g, device="cuda") * 8
    d = torch.randn(n, generator=g, device="cuda") * 0.4
    old, ref = logp - d, logp + torch.randn(n, generator=g, device="cuda") * 0.4
    adv = torch.randn(n, generator=g, device="cuda")
    return y, logp, old, ref, adv


BATCHES = [
    (1, [0, 1]), (1, [0, 0]), (5, [0, 5]), (64, [0, 0, 1, 1, 64, 64]), (1000, [10, 400, 400, 777]),
    (9000, [0, 9000]), (9001, [0, 1, 8999]), (20000, list(range(0, 20001, 5))), (300, None),
    (70001, list(range(0, 70001, 7000))), (50000, None),
]


def offsets(torch, n, start):
    return torch.tensor([0, n] if start is None else start, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("n,start", BATCHES)
@pytest.mark.parametrize("per_seq", [False, True])
@pytest.mark.parametrize("kind", ["full", "on_policy", "no_kl", "metric_kl"])
def test_policy_loss(env, n, start, per_seq, kind):
    torch, ops = env
    V, lo, hi = 100, 0.2, 0.3
    y, logp, old, ref, adv = make_tokens(torch, n, start, n)
    if kind == "on_policy":
        old = None
    if kind == "no_kl":
        ref = None
    c = 0.25 if kind in ("full", "on_policy") else 0.0
    # what tokens that do not count hold is not looked at
    for t in (logp, old, ref, adv):
        if t is not None:
            t[y < 0] = math.nan
    st = offsets(torch, n, start)
    S = st.numel() - 1
    loss, grad = torch.full((3,), 7.0, device="cuda"), torch.full((n + 1,), 7.0, device="cuda")
    args = (logp, old, ref, adv, y, None if start is None else st, lo, hi, c, per_seq, n, S, V)
    ops.policy_loss(loss, grad, *args, 0.5)
    w, ok, _, cnt = ref_weights(torch, y, st, V, per_seq)
    L, K, G, slope = ref_policy(torch, logp, old, ref, adv, w, ok, lo, hi, c)
    # fp64 but for the weight (half a step of fp32) and the results
    close(torch, loss[:1], L.sum()[None], U * L.abs().sum(), torch.float32)
    close(torch, loss[1:2], K.sum()[None], U * K.abs().sum(), torch.float32)
    close(torch, grad[:n], 0.5 * G, U * G.abs(), torch.float32)
    assert loss[2] == 7 and grad[n] == 7 and (grad[:n][~ok] == 0).all()
    if not any(cnt):
        assert (loss[:2] == 0).all()
    # the loss alone; the gradient over the log-probabilities; the same bits again
    again, over = torch.empty(2, device="cuda"), logp.clone()
    ops.policy_loss(again, None, *args, 0.5)
    assert torch.equal(again, loss[:2])
    ops.policy_loss(again, over, over, *args[1:], 0.5)
    assert torch.equal(again, loss[:2]) and torch.equal(over, grad[:n])


def test_policy_at_the_bounds(env):
    """Ratios on the bounds and a step to either side, by the definition in 64 bits."""
    torch, ops = env
    lo, hi = 0.25, 0.5
    base = torch.tensor([math.log(1 - lo), math.log(1 + hi), 0.0], dtype=torch.float32, device="cuda")
    d = torch.cat([base, torch.nextafter(base, base + 1), torch.nextafter(base, base - 1)])
    d = d.repeat(2)
    adv = torch.cat([torch.ones(9), -torch.ones(9)]).cuda()
    n = len(d)
    y, st = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.tensor([0, n], device="cuda")
    old = torch.zeros(n, device="cuda")
    loss, grad = torch.empty(2, device="cuda"), torch.empty(n, device="cuda")
    ops.policy_loss(loss, grad, d, old, None, adv, y, st, lo, hi, 0.0, False, n, 1, 1)
    r = torch.exp(d.double())
    binds = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    assert torch.equal(grad != 0, ~binds) and binds.any() and not binds.all()


def test_policy_of_infinite_log_probabilities(env):
    """A token the old policy held impossible and one that the new one does."""
    torch, ops = env
    inf = math.inf
    logp = torch.tensor([-1.0, -inf, -inf, -1.0], device="cuda")
    old = torch.tensor([-inf, -1.0, -1.0, -1.0], device="cuda")
    adv = torch.tensor([1.0, 1.0, -1.0, 1.0], device="cuda")
    y, st = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.tensor([0, 4], device="cuda")
    loss, grad = torch.empty(2, device="cuda"), torch.empty(4, device="cuda")
    ops.policy_loss(loss, grad, logp, old, None, adv, y, st, 0.25, 0.5, 0.0, False, 4, 1, 1)
    # r = inf binds; r = 0 gains nothing; r = 0 with A < 0 binds at 1 - lo; r = 1
    assert loss[0].item() == (-1.5 + 0.0 + 0.75 - 1.0) / 4 and grad.tolist() == [0.0, 0.0, 0.0, -0.25]


def test_descending_and_outside_offsets_stay_inside(env):
    torch, ops = env
    n = 257
    y, logp, old, ref, adv = make_tokens(torch, n, None, 3)
    for bad in ([0, 300, 200], [-50, 100, 90, 257], [257, 0, 0], [1 << 60, -(1 << 60), 12]):
        st = torch.tensor(bad, dtype=torch.int64, device="cuda")
        S = len(bad) - 1
        store = torch.full((n + 64,), 7.0, device="cuda")
        loss, m = torch.empty(2, device="cuda"), torch.empty(S, device="cuda")
        ops.policy_loss(loss, store[32:32 + n], logp, old, ref, adv, y, st, 0.2, 0.2, 0.1, True, n, S, 100)
        if S % 2 == 0:
            ops.preference_loss(loss, m, store[32:32 + n], logp, ref, y, st, 0.1, 0.0, n, S // 2, 100)
        torch.cuda.synchronize()
        assert (store[:32] == 7).all() and (store[32 + n:] == 7).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [9, 512, 2050, 8192, 32768, 40001, 131079])
@pytest.mark.parametrize("n,start,per_seq",
                         [(40, [0, 11, 11, 38], True), (3, [0, 3], False), (601, [1, 300, 600], True)])
def test_policy_loss_from_logits(env, V, dtype, n, start, per_seq):
    if n * V > 12_000_000:
        n, start = 80, [0, 3, 79]
    check_policy_loss_from_logits(env, V, dtype, n, start, per_seq)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [50001, 70001, 90002, 131079, 270001])
def test_policy_loss_from_many_long_rows(env, V, dtype):
    check_policy_loss_from_logits(env, V, dtype, 131, [0, 70, 130], True)


# the losses of so many tokens are added up in one launch and in two
@pytest.mark.parametrize("n", [2049, 4097, 16384, 16385, 70001])
def test_policy_loss_from_many_rows(env, n):
    check_policy_loss_from_logits(env, 9, "float32", n, [0, n // 3, n // 2, n - 7], n % 2 == 0)


def check_policy_loss_from_logits(env, V, dtype, n, start, per_seq):
    torch, ops = env
    dt = getattr(torch, dtype)
    cap = 15.0 if V % 2 == 0 else 0.0
    z, y, _ = make_logits(torch, n, V, dt, V + n, cap)
    y[1], y[2] = (-1, V) if n > 3 else (y[1], y[2])
    st = offsets(torch, n, start)
    S = st.numel() - 1
    lo, hi, c = 0.2, 0.3, 0.1
    logp64, p, lse, m, z_y, ok0 = ref_rows(torch, z, y)
    g = gen(torch, 8)
    d = torch.randn(n, generator=g, device="cuda") * 0.5
    for b in (math.log(1 - lo), math.log(1 + hi)):  # both gradients are right on a bound
        d = torch.where((d - b).abs() < 1e-3, torch.full_like(d, b + 3e-3), d)
    old = (logp64 - d).float()
    ref = (logp64 + torch.randn(n, generator=g, device="cuda") * 0.5).float()
    adv = torch.randn(n, generator=g, device="cuda")
    z[y < 0] = math.nan  # not read
    loss, logp = torch.empty(2, device="cuda"), torch.full((n,), 7.0, device="cuda")
    out = torch.full_like(z, 7.0)
    args = (old, ref, adv, y, st, cap, lo, hi, c, per_seq, n, S, V)
    ops.policy_loss_logits(loss, logp, out, z, *args, 2.0)
    w, ok, _, _ = ref_weights(torch, y, st, V, per_seq)
    want = torch.where(ok, logp64, torch.zeros_like(logp64))
    tol = torch.where(ok, logp_tol(V, z_y, m, lse, want), torch.zeros_like(want)).nan_to_num(0.0)
    close(torch, logp, want, tol, torch.float32)
    L, K, G, slope = ref_policy(torch, logp64, old, ref, adv, w, ok, lo, hi, c)
    err = tol * slope + 4 * U * G.abs()  # of the gradient by logp
    dL = ((w * tol * (adv.abs() * torch.exp(want - old.double()) + c * torch.expm1((ref - want)).abs())) + U * L.abs())
    close(torch, loss[:1], L.sum()[None], dL.nan_to_num(0.0).sum(), torch.float32)
    close(torch, loss[1:], K.sum()[None],
          (w * tol * torch.expm1(ref - want).abs() + U * K).nan_to_num(0.0).sum() + 1e-9, torch.float32)
    z0 = torch.where(ok[:, None], z, torch.zeros_like(z))
    p0 = torch.where(ok[:, None], p, torch.zeros_like(p))
    D, t = ref_grad(torch, z0, y, p0, ok, 2 * G, cap)
    hot = torch.zeros_like(p0).scatter_(1, y.clamp(0, V - 1)[:, None], 1.0)
    close(torch, out, D, t + 2 * err[:, None] * (hot - p0).abs(), dt)
    assert (out[~ok] == 0).all()
    # in place, without logp: the same bits
    again, z2 = torch.empty(2, device="cuda"), z.clone()
    ops.policy_loss_logits(again, None, z2, z2, *args, 2.0)
    assert torch.equal(again, loss) and torch.equal(z2, out)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,V", [(40, 131079), (128, 65537), (131, 65537), (300, 513), (9000, 64)])
def test_log_probabilities_over_an_input(env, dtype, n, V):
    """logp_out may be an input by token, also where a row is split over workgroups: the same bits."""
    torch, ops = env
    z, y, _ = make_logits(torch, n, V, getattr(torch, dtype), 3, 15.0)
    g = gen(torch, 5)
    old, ref, adv = (torch.randn(n, generator=g, device="cuda") for _ in range(3))
    old, ref = old * 0.3 - math.log(V), ref * 0.3 - math.log(V)
    st = torch.tensor([0, n // 3, n - 1], device="cuda")

    def call(over):
        ins = [old.clone(), ref.clone(), adv.clone()]
        loss, out = torch.empty(2, device="cuda"), torch.empty_like(z)
        logp = torch.empty(n, device="cuda") if over is None else ins[over]
        ops.policy_loss_logits(loss, logp, out, z, *ins, y, st, 15.0, 0.2, 0.2, 0.1, True, n, 2, V)
        return loss, logp, out

    want = call(None)
    for over in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, call(over))), over


def test_policy_gradient_against_differences(env):
    """<gradient, v> against the loss's central difference along v, both losses in 64 bits."""
    torch, ops = env
    n, V, cap = 30, 257, 15.0
    g = gen(torch, 11)
    x = (torch.randn(n, V, generator=g, device="cuda") * 3).double()
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    y[4] = -1
    st = torch.tensor([0, 9, 28], device="cuda")
    logp64 = lambda x: ref_rows(torch, cap * torch.tanh(x / cap), y)[0]  # noqa: E731
    lp = logp64(x)
    old, ref = (lp - 0.05).float(), (lp + 0.3).float()
    adv = torch.randn(n, generator=g, device="cuda")
    w, ok, _, _ = ref_weights(torch, y, st, V, True)
    f = lambda x: ref_policy(torch, logp64(x), old, ref, adv, w, ok, 0.2, 0.2, 0.1)[0].sum()  # noqa: E731
    z = (cap * torch.tanh(x / cap)).float()
    out, loss = torch.empty_like(z), torch.empty(2, device="cuda")
    ops.policy_loss_logits(loss, None, out, z, old, ref, adv, y, st, cap, 0.2, 0.2, 0.1, True, n, 2, V)
    for seed in range(4):
        v = torch.randn(n, V, generator=gen(torch, 20 + seed), device="cuda").double()
        h = 1e-4
        num = (f(x + h * v) - f(x - h * v)) / (2 * h)
        got = (out.double() * v).sum()
        # the difference's third derivative (h^2) and the gradient's 32 bits
        assert abs(num - got) <= 1e-6 * (out.double() * v).abs().sum() + 1e-7, (num.item(), got.item())


# ---------------------------------------------------------------- preference

PAIRS = [(2, [0, 1, 2]), (10, [0, 5, 5]), (10, [0, 0, 0]), (33, [0, 10, 20, 25, 32]),
         (9000, [0, 4000, 9000]), (30001, [0, 29000, 29001, 30000, 30001]), (24000, list(range(0, 24001, 10))),
         (6000, [0] + [3] * 3 + list(range(10, 6001, 10)) + [6000])]


@pytest.mark.parametrize("n,start", PAIRS)
@pytest.mark.parametrize("smooth", [0.0, 0.1])
@pytest.mark.parametrize("with_ref", [True, False])
def test_preference_loss(env, n, start, smooth, with_ref):
    torch, ops = env
    V, beta, P = 100, 0.1, (len(start) - 1) // 2
    start = start[:2 * P + 1]
    y, logp, _, ref, _ = make_tokens(torch, n, start, n + 1)
    st = offsets(torch, n, start)
    for t in (logp, ref):
        t[y < 0] = math.nan
    if not with_ref:
        ref = None
    loss, margin = torch.full((2,), 7.0, device="cuda"), torch.full((P + 1,), 7.0, device="cuda")
    grad = torch.full((n + 1,), 7.0, device="cuda")
    args = (logp, ref, y, st, beta, smooth, n, P, V)
    ops.preference_loss(loss, margin, grad, *args, 3.0)
    _, ok, seq, cnt = ref_weights(torch, y, st, V, False)
    diff = torch.where(ok, logp.double() - (ref.double() if with_ref else 0.0), 0.0)
    sums = torch.zeros(2 * P, dtype=torch.float64, device="cuda").index_add_(0, seq.clamp(min=0), diff)
    cnt = torch.tensor(cnt, device="cuda")
    live = (cnt[0::2] > 0) & (cnt[1::2] > 0)
    h = torch.where(live, beta * (sums[0::2] - sums[1::2]), torch.zeros(P, dtype=torch.float64, device="cuda"))
    sp = torch.nn.functional.softplus
    pairs = max(1, int(live.sum()))
    lp = torch.where(live, (1 - smooth) * sp(-h) + smooth * sp(h), torch.zeros_like(h))
    slope = torch.where(live, beta * (smooth * torch.sigmoid(h) - (1 - smooth) * torch.sigmoid(-h)) / pairs, 0.0)
    sign = torch.stack([slope, -slope], 1).reshape(-1)
    G = torch.where(ok, sign[seq.clamp(min=0)], torch.zeros_like(diff))
    close(torch, loss[:1], lp.sum()[None] / pairs, 2.0 ** -40, torch.float32)
    close(torch, margin[:P], h, 2.0 ** -40, torch.float32)
    close(torch, grad[:n], 3 * G, 2.0 ** -40 * G.abs(), torch.float32)
    assert loss[1] == 7 and margin[P] == 7 and grad[n] == 7 and (grad[:n][~ok] == 0).all()
    again = torch.empty(1, device="cuda")
    ops.preference_loss(again, None, None, *args)
    assert torch.equal(again, loss[:1])


def test_preference_of_far_margins(env):
    """Pairs decided by hundreds of nats, and by an impossible token."""
    torch, ops = env
    logp = torch.tensor([-1.0, -900.0, -900.0, -1.0, -1.0, -math.inf], device="cuda")
    ref = torch.zeros(6, device="cuda")
    y, st = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.arange(7, device="cuda")
    loss, margin, grad = torch.empty(1, device="cuda"), torch.empty(3, device="cuda"), torch.empty(6, device="cuda")
    ops.preference_loss(loss, margin, grad, logp, ref, y, st, 1.0, 0.0, 6, 3, 1)
    assert margin.tolist() == [899.0, -899.0, math.inf] and abs(loss.item() - 899.0 / 3) < 1e-4
    assert abs(grad[2] + 1 / 3) < 1e-7 and abs(grad[3] - 1 / 3) < 1e-7 and (grad[[0, 1, 4, 5]] == 0).all()


# ---------------------------------------------------------------- clipping

SHAPES = [[1], [0, 5, 0], [4096, 4097, 3], [1 << 20, 1, 12289, 513], [7] * 350, [5_000_001, 2, 65536]]


@pytest.mark.parametrize("sizes", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "mixed"])
@pytest.mark.parametrize("factor", [0.25, 4.0, math.inf])
@pytest.mark.parametrize("off", [0, 1])
def test_clip_grad_norm(env, sizes, dtype, factor, off):
    torch, ops = env
    g = gen(torch, len(sizes))
    grads = []
    for i, s in enumerate(sizes):
        dt = getattr(torch, dtype) if dtype != "mixed" else (torch.float32, torch.bfloat16)[i % 2]
        grads.append(torch.randn(s + off, generator=g, device="cuda").to(dt)[off:])
    n = sum(sizes)
    norm64 = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    bound = norm64 * factor
    norm = torch.full((2,), 7.0, device="cuda")
    outs = [torch.full_like(x, 3.0) for x in grads]
    ops.clip_grad_norm(norm, outs, grads, bound)
    # fp64 sums (n roundings of 2^-53 at most), one rounding
    assert abs(norm[0].item() - norm64) <= (U + n * 2.0 ** -53) * norm64 and norm[1] == 7
    c = min(1.0, factor)
    for x, o in zip(grads, outs):
        # product and quotient in fp64, a rounding to fp32 on the way to bf16
        rel = 2 * U if x.dtype == torch.bfloat16 else n * 2.0 ** -52
        close(torch, o, x.double() * c, rel * x.double().abs(), x.dtype)
        if c == 1.0:
            assert torch.equal(o, x)
    inplace = [x.clone() for x in grads]
    ops.clip_grad_norm(norm, None, inplace, bound)
    mixed = [x.clone() if i % 3 else x for i, x in enumerate(grads)]
    ops.clip_grad_norm(norm, [x if i % 3 else torch.empty_like(x) for i, x in enumerate(mixed)], mixed, bound)
    for i, (a, b, o) in enumerate(zip(inplace, mixed, outs)):
        assert torch.equal(a, o) and (i % 3 == 0 or torch.equal(b, o))


def test_clip_over_the_range_of_fp32(env):
    """Squares that fp32 could not hold, and norms that are not finite."""
    torch, ops = env
    norm = torch.empty(1, device="cuda")
    for scale in (1e30, 1e-30, 3e38, 1e-44):
        x = torch.full((1000,), scale, device="cuda")
        want = math.sqrt(1000) * x[0].double().item()
        out = torch.empty_like(x)
        bound = want / 2 if want < 1e300 else 1.0
        ops.clip_grad_norm(norm, [out], [x], bound)
        assert abs(norm.item() - want) <= 2 * U * want + 1e-45 if want < 3.4e38 else norm.item() == math.inf
        ref = x.double() * (bound / want)
        assert ((out.double() - ref).abs() <= 2 * U * ref + 1.5e-45).all()
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.ones(5000, device="cuda")
        x[4999] = bad
        y = x.clone()
        ops.clip_grad_norm(norm, None, [y], 0.5)
        assert not math.isfinite(norm.item()) and torch.equal(y[:4999], x[:4999])


def test_clip_of_no_gradients(env):
    torch, ops = env
    norm = torch.full((1,), 7.0, device="cuda")
    ops.clip_grad_norm(norm, None, [], 1.0)
    assert norm.item() == 0.0
    z = [torch.zeros(100, device="cuda")]
    ops.clip_grad_norm(norm, None, z, 1.0)
    assert norm.item() == 0.0 and (z[0] == 0).all()


# ---------------------------------------------------------------- calls

def test_empty_batches(env):
    torch, ops = env
    f, i = torch.empty(0, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    z = torch.empty(0, 8, device="cuda")
    ops.token_logprob_fwd(f, z, i, 0, 8)
    ops.token_logprob_bwd(z, z, i, f, 0.0, 0, 8)
    loss = torch.full((2,), 7.0, device="cuda")
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.policy_loss(loss, f, f, f, f, f, i, one, 0.2, 0.2, 0.1, True, 0, 0, 8)
    assert loss.tolist() == [0.0, 0.0]
    loss.fill_(7.0)
    ops.policy_loss_logits(loss, f, z, z, f, f, f, i, torch.zeros(3, dtype=torch.int64, device="cuda"), 0.0, 0.2, 0.2,
                           0.1, False, 0, 2, 8)
    assert loss.tolist() == [0.0, 0.0]
    loss.fill_(7.0)
    ops.preference_loss(loss, f, f, f, f, i, one, 0.1, 0.0, 0, 0, 8)
    assert loss[0].item() == 0.0


def test_refusals(env):
    torch, ops = env
    from autoresearch_amd._lib import ArError
    f, i = torch.zeros(64, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="needed"):
        ops.token_logprob_fwd(f, f, i, 9, 8)
    with pytest.raises(TypeError):
        ops.token_logprob_fwd(f, f.half(), i, 4, 8)
    with pytest.raises(TypeError):
        ops.token_logprob_bwd(f.bfloat16(), f, i, f, 0.0, 4, 8)
    with pytest.raises(TypeError):
        ops.token_logprob_fwd(f, f, i.int(), 4, 8)
    with pytest.raises(ValueError, match="contiguous"):
        ops.token_logprob_fwd(f, torch.zeros(8, 8, device="cuda").t(), i, 4, 8)
    with pytest.raises(ValueError, match="contiguous"):
        ops.clip_grad_norm(f, None, [torch.zeros(8, 8, device="cuda").t()], 1.0)
    with pytest.raises(ArError, match="overlap"):
        ops.clip_grad_norm(f[:1], None, [f[8:16], f[12:20]], 1.0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # no workspace is bound to it
        with pytest.raises(ArError, match="workspace"):
            ops.clip_grad_norm(f[:1], None, [f[8:]], 1.0)
        many, ids = torch.zeros(9000, device="cuda"), torch.zeros(9000, dtype=torch.int64, device="cuda")
        with pytest.raises(ArError, match="workspace"):
            ops.policy_loss(f, None, many, None, None, many, ids, None, 0.2, 0.2, 0.0, False, 9000, 1, 8)
        with pytest.raises(ArError, match="workspace"):
            ops.preference_loss(f, None, None, many, None, ids, ids, 0.1, 0.0, 9000, 100, 8)
        with pytest.raises(ArError, match="workspace"):
            ops.policy_loss_logits(f, None, many, many, None, None, f, i, None, 0.0, 0.2, 0.2, 0.0, False, 8, 1, 8)


def test_two_streams_with_their_own_workspaces(env):
    """Calls that overlap in time, each on its stream's workspace."""
    torch, ops = env
    n, V = 300, 8192
    z, y, _ = make_logits(torch, n, V, torch.float32, 5)
    st = torch.tensor([0, 100, 290], device="cuda")
    old = torch.full((n,), -3.0, device="cuda")
    adv = torch.randn(n, generator=gen(torch, 2), device="cuda")

    def call(a, scale):
        loss, out, norm = torch.empty(2, device="cuda"), torch.empty_like(z), torch.empty(1, device="cuda")
        clipped = torch.empty_like(z)
        for _ in range(3):
            ops.policy_loss_logits(loss, None, out, z, old, old, a, y, st, 0.0, 0.2, 0.2, 0.1, True, n, 2, V, scale)
            ops.clip_grad_norm(norm, [clipped], [out], 1e-3)
        return loss, out, norm, clipped

    want = call(adv, 1.0), call(-adv, 2.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = []
    for s in streams:
        with torch.cuda.stream(s):
            spaces.append(ops.Workspace(4 << 20).bind())
    got = []
    for s, a, c in zip(streams, (adv, -adv), (1.0, 2.0)):
        with torch.cuda.stream(s):
            got.append(call(a, c))
    torch.cuda.synchronize()
    for w in spaces:
        w.close()
    for a, b in zip(want, got):
        for x, t in zip(a, b):
            assert torch.equal(x, t)


# one block for the tokens, several launches, rows split over workgroups
@pytest.mark.parametrize("n,V", [(96, 2050), (9000, 130), (60, 131079)])
def test_captured_and_replayed(env, n, V):
    """A step's loss, gradient, preference loss and clipping in one graph, replayed on new inputs."""
    torch, ops = env
    S = 4
    st = torch.tensor([0, 20, 50, 51, n - 6], device="cuda")
    z, y, _ = make_logits(torch, n, V, torch.bfloat16, 1)
    old, ref, adv = (torch.empty(n, device="cuda") for _ in range(3))
    f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731

    def outputs():
        return dict(loss=f(2), logp=f(n), grad=torch.empty_like(z), pl=f(1), margin=f(2), gl=f(n), norm=f(1),
                    gt=torch.empty_like(z), lp2=f(n))

    def step(o):
        ops.policy_loss_logits(o["loss"], o["logp"], o["grad"], z, old, ref, adv, y, st, 15.0, 0.2, 0.2, 0.1, True, n,
                               S, V)
        ops.token_logprob_fwd(o["lp2"], z, y, n, V)
        ops.preference_loss(o["pl"], o["margin"], o["gl"], o["lp2"], ref, y, st, 0.1, 0.1, n, S // 2, V)
        ops.token_logprob_bwd(o["gt"], z, y, o["gl"], 15.0, n, V)
        ops.clip_grad_norm(o["norm"], None, [o["grad"], o["gt"]], 1e-3)

    def fill(seed):
        a, b, _ = make_logits(torch, n, V, torch.bfloat16, seed)
        z.copy_(a)
        y.copy_(b)
        y[seed % n] = -1
        g = gen(torch, seed)
        for t in (old, ref):
            t.copy_(-torch.rand(n, generator=g, device="cuda") * 4)
        adv.copy_(torch.randn(n, generator=g, device="cuda"))

    fill(1)
    s = torch.cuda.Stream()
    graph, rec = torch.cuda.CUDAGraph(), outputs()
    with torch.cuda.stream(s):
        ws = ops.Workspace(4 << 20).bind()
        step(rec)  # before the capture: the kernels are loaded
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            step(rec)
    torch.cuda.synchronize()
    for seed in range(2, 7):
        fill(seed)
        want = outputs()
        step(want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(rec[k], want[k]), (seed, k)
        _ = (z.float() * 2).sum().item()
    ws.close()


# ---------------------------------------------------------------- the model

CONFIG1 = dict(sequence_len=64, vocab_size=512, n_layer=2, n_head=2, n_kv_head=2, n_embd=128, head_dim=64, kv_dim=128)


def _model(torch, precision, seed=3):
    from autoresearch_amd.model import GPT, GPTConfig
    m = GPT(GPTConfig(**CONFIG1), 2, 64, precision=precision, rope_period=64)
    m.init_weights(seed)
    g = gen(torch, seed)
    x = torch.randint(0, 512, (128,), generator=g, device="cuda")
    y = torch.randint(0, 512, (128,), generator=g, device="cuda")
    # a head with something to say, so that logits differ and the softcap bends
    off, size = next((o, s) for k, o, s in m.tensors() if k == "lm_head")
    m.params()[off:off + size] = torch.randn(size, generator=g, device="cuda") * 0.6
    return m, x, y, off, size


@pytest.mark.parametrize("precision", [0, 1])
def test_policy_step_of_the_model(env, precision):
    """forward -> log-probabilities -> policy loss -> backward -> clip -> optimizer:
    the head's gradient against the loss's central difference, the norm against
    the arena's, and the parameters move."""
    torch, ops = env
    m, x, y, off, size = _model(torch, precision)
    n, V = 128, 512
    st = torch.tensor([0, 60, 128], device="cuda")
    y[:20] = -1
    g = gen(torch, 9)
    adv = torch.randn(n, generator=g, device="cuda")

    def logp():
        m.forward(x, y)
        return -m.token_loss()

    base = logp().clone()
    old = base - torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, 0.05, 0.5)
    ref = base + 0.3
    w, ok, _, _ = ref_weights(torch, y, st, V, True)
    f = lambda lp: ref_policy(torch, lp, old, ref, adv, w, ok, 0.2, 0.2, 0.1)[0].sum().item()  # noqa: E731
    loss, gl = torch.empty(2, device="cuda"), torch.empty(n, device="cuda")
    ops.policy_loss(loss, gl, base, old, ref, adv, y, st, 0.2, 0.2, 0.1, True, n, 2, V)
    assert abs(loss[0].item() - f(base)) <= 1e-6 * max(1.0, abs(f(base)))
    m.zero_grads()
    m.backward_logp(x, y, gl)
    grads = m.grads().clone()
    head = grads[off:off + size].double()
    P = m.params()
    keep = P[off:off + size].clone()
    v = head / head.norm()  # along the gradient itself: the largest change for its step
    h = 0.02
    P[off:off + size] = (keep.double() + h * v).float()
    up = f(logp())
    P[off:off + size] = (keep.double() - h * v).float()
    down = f(logp())
    P[off:off + size] = keep
    num, got = (up - down) / (2 * h), head.norm().item()
    # fp32: the second-order term of the difference; bf16: logits and their
    # gradient rounded to 8 bits, weights to 8 bits within the step
    assert abs(num - got) <= (0.02 if precision == 0 else 0.1) * got, (num, got)
    # the gradient by logp that cross entropy has, through the same backward as
    # the cross entropy but for the softcap's derivative: another head gradient
    norm = m.clip_grads(math.inf)
    want = grads.double().norm().item()
    assert abs(norm - want) <= 1e-6 * want and torch.equal(m.grads(), grads)
    norm = m.clip_grads(want / 3)
    assert abs(norm - want) <= 1e-6 * want
    assert ((m.grads().double() - grads.double() / 3).abs() <= 1e-6 * grads.double().abs() + 1e-40).all()
    before = P.clone()
    m.optimizer_step(0.0)
    assert P.isfinite().all() and (P != before).any()
    # the ordinary backward is what it was
    m.zero_grads()
    m.forward(x, y)
    m.backward(x, y, 1.0)
    a = m.grads().clone()
    m.zero_grads()
    m.forward(x, y)
    m.backward_logp(x, y, gl)
    m.zero_grads()
    m.backward(x, y, 1.0)
    assert torch.equal(a, m.grads())
    m.close()


@pytest.mark.parametrize("precision", [0, 1])
def test_train_step_with_clipping(env, precision):
    """train_step and its graph with a bound, against the pieces; without one, as ever."""
    torch, ops = env
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        models = [_model(torch, precision) for _ in range(3)]
        pieces, eager, graph = (mm[0] for mm in models)
        x, y = models[0][1], models[0][2]
        for step, bound in enumerate([0.0, 1e-3, 1e-3, 5e-4, 0.0]):
            eager.set_grad_clip(bound)
            graph.set_grad_clip(bound)
            pieces.zero_grads()
            pieces.forward(x, y)
            pieces.backward(x, y, 1.0)
            if bound:
                assert pieces.clip_grads(bound) > bound  # it clips
            pieces.optimizer_step(0.1 * step)
            eager.train_step(x, y, 0.1 * step)
            graph.train_step_graph(x, y, 0.1 * step)
            torch.cuda.synchronize()
            assert torch.equal(pieces.params(), eager.params()), step
            assert torch.equal(eager.params(), graph.params()), step
            assert torch.equal(eager.grads(), graph.grads()), step
        for mm in models:
            mm[0].close()


def test_backward_logp_refuses(env):
    torch, _ = env
    m, x, y, _, _ = _model(torch, 0)
    for bad in (torch.zeros(127, device="cuda"), torch.zeros(128), torch.zeros(128, device="cuda", dtype=torch.float64)):
        with pytest.raises(ValueError):
            m.backward_logp(x, y, bad)
    m.close()
