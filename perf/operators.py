"""Measured cases of the post-training operators: token log-probabilities of
logits with their gradient, the clipped policy loss with a KL term, the
preference loss over pairs, and the global gradient norm with clipping.

`run()` is one pass on what `prepare()` made: in elementary torch operations,
or, with `own` set, through this library's entry points.  `exact()` is the same
in 64 bits, from the definitions.

Logits are as the model leaves them after its softcap (cap 15), or plain ones
(cap 0).  Tokens come in sequences one after the other, seq_start their
offsets; a prompt's tokens carry the target -1, and so does the padding behind
the last sequence: they count nowhere and their gradient is zero.
"""
import math
import random

import torch

own = False

CAP = 15.0
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL_COEF = 0.04
BETA, SMOOTH = 0.1, 0.05
D = torch.float64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
CHUNK = 1 << 26  # logits at a time in making inputs and in 64 bits


def listed():
    return [
        # scoring the last few tokens under a long vocabulary: three rows to fill the card with
        {"name": "logprob_few_rows", "op": "logprob_fwd", "tokens": 3, "vocab": 131072, "type": "bf16"},
        # the reference policy's log-probabilities of two sequences of 2048
        {"name": "logprob_long_vocab", "op": "logprob_fwd", "tokens": 4096, "vocab": 131072, "type": "bf16"},
        # a caller's own loss on top of the log-probabilities; no size a multiple of anything
        {"name": "logprob_grad_odd", "op": "logprob_bwd", "tokens": 2047, "vocab": 50001, "type": "fp32", "cap": 0.0},
        # the same behind the softcapped head in bf16
        {"name": "logprob_grad_bf16", "op": "logprob_bwd", "tokens": 16384, "vocab": 32768, "type": "bf16",
         "cap": CAP},
        # the tiny test model's batch: latency and launches
        {"name": "policy_small", "op": "policy", "tokens": 128, "seqs": 2, "vocab": 512, "type": "fp32", "cap": CAP,
         "per_seq": False},
        # a policy step at the benchmark's batch: 32 answers of up to 2048 tokens, vocabulary 8192, fp32
        {"name": "policy_full", "op": "policy", "tokens": 65536, "seqs": 32, "vocab": 8192, "type": "fp32",
         "cap": CAP, "per_seq": True},
        # an odd vocabulary in bf16: rows off every alignment
        {"name": "policy_odd_bf16", "op": "policy", "tokens": 8191, "seqs": 11, "vocab": 32003, "type": "bf16",
         "cap": 0.0, "per_seq": False},
        # the loss alone, on log-probabilities a program already has: a rollout batch of short answers
        {"name": "policy_tokens", "op": "policy_tokens", "tokens": 262144, "seqs": 509, "vocab": 8192,
         "per_seq": True},
        # the loss of four pairs of short answers
        {"name": "preference_tokens", "op": "preference_tokens", "tokens": 801, "seqs": 8, "vocab": 8192},
        # a whole preference step from the logits of sixteen pairs to their gradient
        {"name": "preference_step", "op": "preference", "tokens": 12288, "seqs": 32, "vocab": 32768, "type": "bf16",
         "cap": CAP},
        # the gradients of the tiny test model
        {"name": "clip_small", "op": "clip", "depth": 2, "vocab": 512, "type": "fp32", "clips": True},
        # the gradients of the depth-8 model
        {"name": "clip_depth8", "op": "clip", "depth": 8, "vocab": 8192, "type": "fp32", "clips": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprob_fwd", "logprob_bwd", "policy", "policy", "policy_tokens", "preference_tokens",
                     "preference", "clip"])
    if op == "clip":
        return {"op": op, "depth": rng.randint(1, 14), "vocab": _log(rng, 500, 20000),
                "type": rng.choice(["fp32", "bf16"]), "clips": rng.random() < 0.75}
    if op in ("policy_tokens", "preference_tokens"):
        n = _log(rng, 64, 400000)
        seqs = min(_log(rng, 1, 2000), max(1, n // 8))
        case = {"op": op, "tokens": n, "seqs": seqs, "vocab": 8192}
    else:
        type_ = rng.choice(["fp32", "bf16"])
        while True:
            n, V = _log(rng, 1, 65536), _log(rng, 500, 150000)
            if rng.random() < 0.5:
                V = (V + 63) // 64 * 64
            if n * V * (4 if type_ == "fp32" else 2) < 1.5e9:
                break
        case = {"op": op, "tokens": n, "vocab": V, "type": type_}
        if op != "logprob_fwd":
            case["cap"] = rng.choice([0.0, CAP])
        if op in ("policy", "preference"):
            case["seqs"] = min(_log(rng, 1, 256), max(1, n // 8))
    if op.startswith("policy"):
        case["per_seq"] = rng.random() < 0.5
    if op.startswith("preference"):
        case["tokens"] = max(16, case["tokens"])
        case["seqs"] = max(2, case["seqs"] // 2 * 2)
    return case


# ---------------------------------------------------------------- layout of a batch

def _layout(case):
    """Offsets of the sequences and how many of each one's first tokens are
    the prompt, from the sizes alone: ragged lengths, a few rows of padding
    behind the last sequence."""
    n, S = case["tokens"], case.get("seqs", 1)
    r = random.Random(n * 1009 + S)
    used = n if n < 64 else n - n // 50
    weights = [r.uniform(0.25, 1.0) for _ in range(S)]
    total, acc, start = sum(weights), 0.0, [0]
    for w in weights:
        acc += w
        start.append(min(used, int(used * acc / total + 0.5)))
    start[-1] = used
    prompt = [int((b - a) * r.uniform(0.0, 0.4)) for a, b in zip(start, start[1:])]
    return start, prompt


def _mask(case):
    start, prompt = _layout(case)
    keep = torch.zeros(case["tokens"], dtype=torch.bool)
    for a, b, p in zip(start, start[1:], prompt):
        keep[a + p:b] = True
    return keep


def _shapes(case):
    """Every parameter of the model the depth rule gives."""
    V, C = case["vocab"], (case["depth"] * 64 + 127) // 128 * 128
    out = [(V, C), (V, C), (case["depth"],), (case["depth"],)]
    for i in range(case["depth"]):
        out += [(C, C)] * 4 + [(4 * C, C), (C, 4 * C)]
        if i % 2 == (case["depth"] - 1) % 2:
            out += [(V, C), (C // 128, 32)]
    return out


# ---------------------------------------------------------------- inputs

_scratch = None


def _workspace():
    """One workspace for the process, bound to its stream, as a program makes it once."""
    global _scratch
    if _scratch is None:
        from autoresearch_amd import ops
        _scratch = ops.Workspace(64 << 20).bind()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 23)
    return g


def _rows(case):
    step = max(1, CHUNK // case["vocab"])
    return [(i, min(case["tokens"], i + step)) for i in range(0, case["tokens"], step)]


def _away(d):
    """Log ratios as a policy a few updates on has them, none within 1e-3 of
    where the clip begins to bind: on it, both gradients are right."""
    for b in (math.log1p(CLIP_HIGH), math.log1p(-CLIP_LOW)):
        near = (d - b).abs() < 1e-3
        d = torch.where(near, torch.full_like(d, b + 2e-3), d)
    return d


def _logits(case, g):
    """Logits of a trained head (a few units wide, the sampled token well
    above the rest), softcapped if the case has a cap; and their targets."""
    n, V, t = case["tokens"], case["vocab"], TYPES[case["type"]]
    targets = torch.randint(0, V, (n,), generator=g, device="cuda")
    lift = torch.rand(n, generator=g, device="cuda") * 8 + 4
    z = torch.empty(n, V, dtype=t, device="cuda")
    for a, b in _rows(case):
        x = torch.randn(b - a, V, generator=g, device="cuda").mul_(2.5)
        x.scatter_add_(1, targets[a:b, None], lift[a:b, None])
        if case.get("cap"):
            x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
        z[a:b] = x
    return z, targets


def prepare(case, seed):
    g = _gen(seed)
    if own:
        _workspace()
    st = {"case": case}
    f = dict(dtype=torch.float32, device="cuda")
    if case["op"] == "clip":
        t = TYPES[case["type"]]
        grads = [(torch.randn(*s, generator=g, device="cuda") * (0.02 if len(s) == 2 else 0.5)).to(t)
                 for s in _shapes(case)]
        norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        # a bound well inside the norm, or one that training rarely meets
        st.update(grads=grads, out=[torch.empty_like(x) for x in grads], norm=torch.empty(1, **f),
                  max_norm=torch.tensor(norm * (0.3 if case["clips"] else 3.0), dtype=torch.float32).item())
        return st
    n, V = case["tokens"], case["vocab"]
    if case["op"].endswith("_tokens"):
        targets = torch.randint(0, V, (n,), generator=g, device="cuda")
        logp = -torch.empty(n, **f).exponential_(0.5, generator=g)
    else:
        st["z"], targets = _logits(case, g)
        if case["op"].startswith("policy"):
            logp = torch.empty(n, **f)
            for a, b in _rows(case):
                x = st["z"][a:b].float()
                logp[a:b] = x.gather(1, targets[a:b, None])[:, 0] - x.logsumexp(1)
    st["targets"] = targets
    st["logp"] = torch.empty(n, **f)
    if not case["op"].startswith("logprob"):
        keep = _mask(case).cuda()
        targets[~keep] = -1
        start = _layout(case)[0]
        st["start"] = torch.tensor(start, dtype=torch.int64, device="cuda")
        lengths = st["start"][1:] - st["start"][:-1]
    if case["op"] == "logprob_bwd":
        # a loss's gradient by each token: some tokens have none
        gl = torch.randn(n, generator=g, device="cuda") / n
        st["grad_logp"] = torch.where(torch.arange(n, device="cuda") % 16 == 5, torch.zeros_like(gl), gl)
    if case["op"].startswith("policy"):
        d = _away(torch.randn(n, generator=g, **f) * 0.25)
        st["old"], st["ref"] = logp - d, logp + torch.randn(n, generator=g, **f) * 0.3
        # each answer's reward against its group's mean, one for all its tokens
        adv = torch.randn(lengths.numel(), generator=g, **f).repeat_interleave(lengths)
        st["adv"] = torch.cat([adv, torch.zeros(n - adv.numel(), **f)])
        st["loss"] = torch.empty(2, **f)
    if case["op"].startswith("preference"):
        if "z" in st:
            logp = torch.empty(n, **f)
            for a, b in _rows(case):
                x = st["z"][a:b].float()
                logp[a:b] = x.gather(1, targets[a:b, None].clamp(min=0))[:, 0] - x.logsumexp(1)
        st["ref"] = logp + torch.randn(n, generator=g, **f) * 0.2
        st["loss"], st["margin"] = torch.empty(1, **f), torch.empty(case["seqs"] // 2, **f)
        st["grad_logp"] = torch.empty(n, **f)
    if case["op"].endswith("_tokens"):
        st["logp"] = logp
        st["grad_logp"] = torch.empty(n, **f)
    elif case["op"] != "logprob_fwd":
        st["grad"] = torch.empty_like(st["z"])
    return st


# ---------------------------------------------------------------- plain form

def _softmax_parts(z, targets):
    """logp of the targets (0 where there is none) and the probabilities, in 32 bits."""
    x = z.float()
    e = torch.exp(x - x.amax(1, keepdim=True))
    s = e.sum(1, keepdim=True)
    keep = (targets >= 0) & (targets < z.shape[1])
    at = targets.clamp(0, z.shape[1] - 1)[:, None]
    logp = (x.gather(1, at) - x.amax(1, keepdim=True) - torch.log(s))[:, 0]
    return torch.where(keep, logp, torch.zeros_like(logp)), e.div_(s), keep


def _logits_grad(z, p, targets, keep, g, cap):
    g = torch.where(keep, g, torch.zeros_like(g))
    d = p.neg_()
    d.scatter_add_(1, targets.clamp(0, z.shape[1] - 1)[:, None], torch.ones_like(g)[:, None])
    d.mul_(g[:, None])
    if cap:
        d.mul_(1 - (z.float() / cap).square())
    return torch.where((g != 0)[:, None], d, torch.zeros_like(d)).to(z.dtype)


def _weights(targets, start, vocab, per_seq):
    """What each token's term weighs in the loss (64 bits)."""
    n = targets.numel()
    t = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    S = start.numel() - 1
    keep = (targets >= 0) & (targets < vocab) & (seq >= 0) & (seq < S)
    seq = seq.clamp(0, S - 1)
    count = torch.zeros(S, dtype=D, device="cuda").index_add_(0, seq, keep.to(D))
    if per_seq:
        w = 1 / (count.clamp(min=1) * (count > 0).sum().clamp(min=1))[seq]
    else:
        w = (1 / count.sum().clamp(min=1)).expand(n)
    return torch.where(keep, w, torch.zeros_like(w)), keep, seq


def _policy(logp, st, case):
    """loss, mean KL and the loss's gradient by logp; the few operations per token in 64 bits."""
    w, keep, _ = _weights(st["targets"], st["start"], case["vocab"], case["per_seq"])
    logp = logp.to(D)
    a, r = st["adv"].to(D), torch.exp(logp - st["old"].to(D))
    k = st["ref"].to(D) - logp
    binds = ((a > 0) & (r > 1 + CLIP_HIGH)) | ((a < 0) & (r < 1 - CLIP_LOW))
    pg = torch.maximum(-a * r, -a * r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH))
    kl = torch.exp(k) - k - 1
    zero = torch.zeros_like(w)
    loss = torch.where(keep, w * (pg + KL_COEF * kl), zero).sum()
    mean_kl = torch.where(keep, w * kl, zero).sum()
    g = torch.where(binds, zero, -a * r) + KL_COEF * (1 - torch.exp(k))
    return torch.stack([loss, mean_kl]).float(), torch.where(keep, w * g, zero).float()


def _preference(logp, st, case):
    targets, start = st["targets"], st["start"]
    _, keep, seq = _weights(targets, start, case["vocab"], False)
    zero = torch.zeros(logp.numel(), dtype=D, device="cuda")
    diff = torch.where(keep, logp.to(D) - st["ref"].to(D), zero)
    S = start.numel() - 1
    total = torch.zeros(S, dtype=D, device="cuda").index_add_(0, seq, diff)
    count = torch.zeros(S, dtype=D, device="cuda").index_add_(0, seq, keep.to(D))
    live = (count[0::2] > 0) & (count[1::2] > 0)
    h = BETA * (total[0::2] - total[1::2])
    up, down = 1 / (1 + torch.exp(-h)), 1 / (1 + torch.exp(h))  # sigma(h), sigma(-h)
    loss = (1 - SMOOTH) * torch.log1p(torch.exp(-h)) + SMOOTH * torch.log1p(torch.exp(h))
    pairs = live.sum().clamp(min=1)
    zp = torch.zeros_like(h)
    c = torch.where(live, BETA / pairs * (SMOOTH * up - (1 - SMOOTH) * down), zp)
    sign = torch.stack([c, -c], 1).reshape(-1)
    return ((torch.where(live, loss, zp).sum() / pairs).float().reshape(1), torch.where(live, h, zp).float(),
            torch.where(keep, sign[seq], zero).float())


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "clip":
        total = torch.zeros((), dtype=D, device="cuda")
        for x in st["grads"]:
            total = total + x.float().square().sum().to(D)
        norm = torch.sqrt(total)
        c = torch.where(norm > st["max_norm"], st["max_norm"] / norm, torch.ones_like(norm)).float()
        return [norm.float().reshape(1)] + [(x.float() * c).to(x.dtype) for x in st["grads"]]
    if op == "policy_tokens":
        return list(_policy(st["logp"], st, case))
    if op == "preference_tokens":
        return list(_preference(st["logp"], st, case))
    logp, p, keep = _softmax_parts(st["z"], st["targets"])
    if op == "logprob_fwd":
        return [logp]
    if op == "logprob_bwd":
        return [_logits_grad(st["z"], p, st["targets"], keep, st["grad_logp"], case["cap"])]
    if op == "policy":
        loss, g = _policy(logp, st, case)
        return [loss, logp, _logits_grad(st["z"], p, st["targets"], keep, g, case["cap"])]
    loss, margin, g = _preference(logp, st, case)
    return [loss, margin, logp, _logits_grad(st["z"], p, st["targets"], keep, g, case["cap"])]


# ---------------------------------------------------------------- the library's operators

def _run_own(st):
    from autoresearch_amd import ops
    case = st["case"]
    op = case["op"]
    if op == "clip":
        ops.clip_grad_norm(st["norm"], st["out"], st["grads"], st["max_norm"])
        return [st["norm"]] + st["out"]
    n, V = case["tokens"], case["vocab"]
    if op == "logprob_fwd":
        ops.token_logprob_fwd(st["logp"], st["z"], st["targets"], n, V)
        return [st["logp"]]
    if op == "logprob_bwd":
        ops.token_logprob_bwd(st["grad"], st["z"], st["targets"], st["grad_logp"], case["cap"], n, V)
        return [st["grad"]]
    if op == "policy":
        ops.policy_loss_logits(st["loss"], st["logp"], st["grad"], st["z"], st["old"], st["ref"], st["adv"],
                               st["targets"], st["start"], case["cap"], CLIP_LOW, CLIP_HIGH, KL_COEF,
                               case["per_seq"], n, case["seqs"], V)
        return [st["loss"], st["logp"], st["grad"]]
    if op == "policy_tokens":
        ops.policy_loss(st["loss"], st["grad_logp"], st["logp"], st["old"], st["ref"], st["adv"], st["targets"],
                        st["start"], CLIP_LOW, CLIP_HIGH, KL_COEF, case["per_seq"], n, case["seqs"], V)
        return [st["loss"], st["grad_logp"]]
    if op == "preference":
        ops.token_logprob_fwd(st["logp"], st["z"], st["targets"], n, V)
    ops.preference_loss(st["loss"], st["margin"], st["grad_logp"], st["logp"], st["ref"], st["targets"], st["start"],
                        BETA, SMOOTH, n, case["seqs"] // 2, V)
    if op == "preference_tokens":
        return [st["loss"], st["margin"], st["grad_logp"]]
    ops.token_logprob_bwd(st["grad"], st["z"], st["targets"], st["grad_logp"], case["cap"], n, V)
    return [st["loss"], st["margin"], st["logp"], st["grad"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- work

def work(case):
    """Rows that count are read, every row of a gradient is written; a token's
    own few numbers once each; a multiply and an add are two operations."""
    op = case["op"]
    if op == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        es = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2 * n * es, "flops": 3 * n}
    n, V = case["tokens"], case["vocab"]
    counted = n if op.startswith("logprob") else int(_mask(case).sum())
    if op == "policy_tokens":
        return {"bytes": 12 * n + 16 * counted, "flops": 30 * counted}
    if op == "preference_tokens":
        return {"bytes": 12 * n + 8 * counted, "flops": 6 * counted}
    es = 4 if case["type"] == "fp32" else 2
    if op == "logprob_fwd":
        return {"bytes": counted * V * es + 12 * n, "flops": 4 * counted * V}
    if op == "logprob_bwd":
        counted -= len([i for i in range(n) if i % 16 == 5])  # no gradient: zeros, nothing read
    return {"bytes": (counted + n) * V * es + 12 * n + 16 * counted, "flops": 8 * counted * V}


# ---------------------------------------------------------------- 64 bits

def _exact_rows(case, st, token_grad):
    """logp, and the gradient by the logits when token_grad gives one by logp."""
    n, V, cap = case["tokens"], case["vocab"], case.get("cap", 0.0)
    tg = st["targets"]
    ok = (tg >= 0) & (tg < V)
    logp = torch.zeros(n, dtype=D, device="cuda")
    for a, b in _rows(case):
        z = st["z"][a:b].to(D)
        at = tg[a:b].clamp(0, V - 1).unsqueeze(1)
        logp[a:b] = torch.where(ok[a:b], torch.log_softmax(z, 1).gather(1, at).squeeze(1), logp[a:b])
    if token_grad is None:
        return logp, None
    g, rest = token_grad(logp)
    out = torch.zeros(n, V, dtype=D, device="cuda")
    for a, b in _rows(case):
        live = ok[a:b] & (g[a:b] != 0)
        if not bool(live.any()):
            continue
        z = st["z"][a:b][live].to(D)
        d = -torch.softmax(z, 1)
        d[torch.arange(d.shape[0], device="cuda"), tg[a:b][live]] += 1
        d *= g[a:b][live].unsqueeze(1)
        if cap:
            d *= (1 - z / cap) * (1 + z / cap)
        out[a:b][live] = d
    return logp, (out, rest)


def _exact_policy(case, st):
    start, V = st["start"].tolist(), case["vocab"]

    def by_token(logp):
        logp = logp.to(D)
        tg = st["targets"]
        ok = (tg >= 0) & (tg < V)
        spans = [(a, b, int(ok[a:b].sum())) for a, b in zip(start, start[1:])]
        total, alive = sum(c for _, _, c in spans), sum(1 for _, _, c in spans if c)
        loss = mean_kl = 0.0
        g = torch.zeros_like(logp)
        for a, b, c in spans:
            if not c:
                continue
            w = 1 / (alive * c) if case["per_seq"] else 1 / total
            i = torch.nonzero(ok[a:b]).squeeze(1) + a
            adv, ratio = st["adv"][i].to(D), (logp[i] - st["old"][i].to(D)).exp()
            k = st["ref"][i].to(D) - logp[i]
            bounded = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
            first = adv * ratio <= adv * bounded  # the smaller gain is the one that counts
            gain, kl = torch.minimum(adv * ratio, adv * bounded), torch.expm1(k) - k
            loss += w * float((KL_COEF * kl - gain).sum())
            mean_kl += w * float(kl.sum())
            g[i] = w * (-adv * ratio * first.to(D) - KL_COEF * torch.expm1(k))
        return g, torch.tensor([loss, mean_kl], dtype=D, device="cuda")
    return by_token


def _exact_preference(case, st):
    start, V = st["start"].tolist(), case["vocab"]

    def by_token(logp):
        logp = logp.to(D)
        tg = st["targets"]
        ok = (tg >= 0) & (tg < V)
        diff = logp - st["ref"].to(D)
        spans = list(zip(start, start[1:]))
        live = [bool(ok[a:b].any()) for a, b in spans]
        P = sum(1 for i in range(0, len(spans), 2) if live[i] and live[i + 1])
        g, loss, margins = torch.zeros_like(logp), 0.0, []
        for i in range(0, len(spans), 2):
            if not (live[i] and live[i + 1]):
                margins.append(0.0)
                continue
            s = [float(diff[a:b][ok[a:b]].sum()) for a, b in spans[i:i + 2]]
            h = torch.tensor(BETA * (s[0] - s[1]), dtype=D)
            margins.append(float(h))
            log_up, log_down = torch.nn.functional.logsigmoid(h), torch.nn.functional.logsigmoid(-h)
            loss -= float((1 - SMOOTH) * log_up + SMOOTH * log_down) / P
            slope = BETA / P * float(SMOOTH * log_up.exp() - (1 - SMOOTH) * log_down.exp())
            for (a, b), sign in zip(spans[i:i + 2], (1.0, -1.0)):
                g[a:b] = torch.where(ok[a:b], sign * slope, 0.0)
        dev = dict(dtype=D, device="cuda")
        return g, (torch.tensor([loss], **dev), torch.tensor(margins, **dev))
    return by_token


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        norm = math.sqrt(sum(float(x.to(D).square().sum()) for x in st["grads"]))
        c = min(1.0, st["max_norm"] / norm)
        return [torch.tensor([norm], dtype=D, device="cuda")] + [x.to(D) * c for x in st["grads"]]
    if op == "logprob_fwd":
        return [_exact_rows(case, st, None)[0]]
    if op == "logprob_bwd":
        return [_exact_rows(case, st, lambda logp: (st["grad_logp"].to(D), None))[1][0]]
    if op == "policy_tokens":
        g, loss = _exact_policy(case, st)(st["logp"])
        return [loss, g]
    if op == "preference_tokens":
        g, (loss, margins) = _exact_preference(case, st)(st["logp"])
        return [loss, margins, g]
    if op == "policy":
        logp, (grad, loss) = _exact_rows(case, st, _exact_policy(case, st))
        return [loss, logp, grad]
    logp, (grad, (loss, margins)) = _exact_rows(case, st, _exact_preference(case, st))
    return [loss, margins, logp, grad]
