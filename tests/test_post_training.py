"""Refusals of the post-training operators (token log-probabilities, policy
and preference losses, gradient clipping): arguments are checked before any
device work, so they run without a GPU on host buffers that nothing reads."""
import ctypes as ct
import math

import pytest

from autoresearch_amd import _lib

EINVAL, EUNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


class Buf:
    """Host memory for a pointer argument."""

    def __init__(self, nbytes=1 << 12):
        self.raw = (ct.c_char * (nbytes + 64))()
        self.at = (ct.addressof(self.raw) + 63) // 64 * 64


def refused(lib, status, code, *words):
    msg = lib.ar_last_error().decode()
    assert status == code, (status, msg)
    for w in words:
        assert w in msg, msg


BUFS = {k: Buf() for k in ("loss", "logp", "grad", "logits", "old", "ref", "adv", "targets", "start", "margin")}
A = {k: b.at for k, b in BUFS.items()}


def fwd(lib, **kw):
    a = {**A, "bf16": 0, "n": 4, "V": 8, **kw}
    return lib.ar_token_logprob_fwd(None, a["logp"], a["logits"], a["bf16"], a["targets"], a["n"], a["V"])


def bwd(lib, **kw):
    a = {**A, "bf16": 0, "cap": 0.0, "n": 4, "V": 8, **kw}
    return lib.ar_token_logprob_bwd(None, a["grad"], a["logits"], a["bf16"], a["targets"], a["logp"], a["cap"],
                                    a["n"], a["V"])


POLICY = {"lo": 0.2, "hi": 0.2, "kl": 0.1, "per_seq": 0, "n": 4, "S": 2, "V": 8, "scale": 1.0, "bf16": 0, "cap": 0.0}


def policy(lib, **kw):
    a = {**A, **POLICY, **kw}
    return lib.ar_policy_loss(None, a["loss"], a["grad"], a["logp"], a["old"], a["ref"], a["adv"], a["targets"],
                              a["start"], a["lo"], a["hi"], a["kl"], a["per_seq"], a["n"], a["S"], a["V"], a["scale"])


def policy_logits(lib, **kw):
    a = {**A, **POLICY, **kw}
    return lib.ar_policy_loss_logits(None, a["loss"], a["logp"], a["grad"], a["logits"], a["bf16"], a["old"],
                                     a["ref"], a["adv"], a["targets"], a["start"], a["cap"], a["lo"], a["hi"],
                                     a["kl"], a["per_seq"], a["n"], a["S"], a["V"], a["scale"])


def preference(lib, **kw):
    a = {**A, "beta": 0.1, "smooth": 0.0, "n": 4, "P": 1, "V": 8, "scale": 1.0, **kw}
    return lib.ar_preference_loss(None, a["loss"], a["margin"], a["grad"], a["logp"], a["ref"], a["targets"],
                                  a["start"], a["beta"], a["smooth"], a["n"], a["P"], a["V"], a["scale"])


ROWS = [fwd, bwd, policy_logits]
LOSSES = [policy, policy_logits, preference]


@pytest.mark.parametrize("call", ROWS)
@pytest.mark.parametrize("kw,code,word", [
    ({"logits": None}, EINVAL, "null"), ({"targets": None}, EINVAL, "null"),
    ({"n": -1}, EINVAL, "shape"), ({"V": 0}, EINVAL, "shape"), ({"V": -3}, EINVAL, "shape"),
    ({"bf16": 2}, EINVAL, "logits_bf16"), ({"logits": A["logits"] + 2}, EINVAL, "aligned"),
    ({"logits": A["logits"] + 1, "bf16": 1}, EINVAL, "aligned"),
    ({"n": 1 << 31}, EUNSUPPORTED, "2^31"), ({"V": 1 << 31}, EUNSUPPORTED, "2^30"),
])
def test_rows_of_logits(lib, call, kw, code, word):
    refused(lib, call(lib, **kw), code, word)


@pytest.mark.parametrize("call", [bwd, policy_logits])
@pytest.mark.parametrize("kw,word", [
    ({"grad": None}, "null"), ({"cap": -1.0}, "cap"), ({"cap": math.nan}, "cap"),
    ({"grad": A["logits"] + 4}, "overlaps"), ({"grad": A["logits"] - 64}, "overlaps"),
    ({"grad": A["grad"] + 2}, "aligned"),
])
def test_gradient_of_logits(lib, call, kw, word):
    refused(lib, call(lib, **kw), EINVAL, word)


@pytest.mark.parametrize("call", ROWS)
def test_arrays_by_token_over_the_logits(lib, call):
    refused(lib, call(lib, logp=A["logits"] + 8), EINVAL, "overlaps")
    if call is not fwd:
        refused(lib, call(lib, logp=A["grad"] + 100), EINVAL, "overlaps")


def test_null_log_probabilities(lib):
    refused(lib, fwd(lib, logp=None), EINVAL, "null")
    refused(lib, bwd(lib, logp=None), EINVAL, "null")
    refused(lib, policy(lib, logp=None), EINVAL, "null")
    refused(lib, preference(lib, logp=None), EINVAL, "null")


@pytest.mark.parametrize("call", LOSSES)
@pytest.mark.parametrize("kw,word", [({"loss": None}, "null"), ({"targets": None}, "null"), ({"n": -4}, "shape"),
                                     ({"V": 0}, "shape"), ({"start": None}, "")])
def test_losses(lib, call, kw, word):
    refused(lib, call(lib, **kw), EINVAL, word)


@pytest.mark.parametrize("call", [policy, policy_logits])
@pytest.mark.parametrize("kw,word", [
    ({"adv": None}, "null"), ({"lo": -0.1}, "clip"), ({"hi": math.nan}, "clip"), ({"ref": None}, "ref_logp"),
    ({"kl": math.nan}, "KL"), ({"S": -1}, "shape"), ({"start": None, "S": 3}, "seq_start"),
    ({"old": A["grad"] + 4, "ref": A["logp"] + 4}, "overlaps"), ({"adv": A["logp"] - 8, "grad": A["logp"]}, "overlaps"),
])
def test_policy(lib, call, kw, word):
    refused(lib, call(lib, **kw), EINVAL, word)


@pytest.mark.parametrize("kw,word", [
    ({"P": -1}, "pairs"), ({"smooth": -0.1}, "label_smoothing"), ({"smooth": 1.5}, "label_smoothing"),
    ({"beta": math.nan}, ""), ({"grad": A["logp"]}, "overlap"), ({"grad": A["ref"] + 4}, "overlap"),
])
def test_preference(lib, kw, word):
    refused(lib, preference(lib, **kw), EINVAL, word)


def test_more_than_there_is_room_for(lib):
    refused(lib, preference(lib, P=(1 << 29) + 1), EUNSUPPORTED, "2^29")
    for call in (policy, policy_logits):
        refused(lib, call(lib, S=(1 << 30) + 1), EUNSUPPORTED, "2^30")
    for call in ROWS:
        refused(lib, call(lib, V=(1 << 30) + 1), EUNSUPPORTED, "2^30")


def clip(lib, ptrs, sizes, bf16=None, outs=None, max_norm=1.0, norm=A["loss"], n=None):
    n = len(ptrs) if n is None else n
    arr = lambda t, v: None if v is None else (t * len(v))(*v)  # noqa: E731
    return lib.ar_clip_grad_norm(None, norm, arr(ct.c_void_p, outs), arr(ct.c_void_p, ptrs), arr(ct.c_int32, bf16),
                                 arr(ct.c_int64, sizes), n, max_norm)


def test_clip_grad_norm(lib):
    a, b = A["grad"], A["logits"]
    refused(lib, clip(lib, [a], [4], norm=None), EINVAL, "null")
    refused(lib, clip(lib, [a, None], [4, 4]), EINVAL, "null tensor 1")
    refused(lib, clip(lib, [a], [4], n=-1), EINVAL, "number")
    refused(lib, clip(lib, [a], [-4]), EINVAL, "size")
    for bad in (0.0, -1.0, math.nan, -math.inf):
        refused(lib, clip(lib, [a], [4], max_norm=bad), EINVAL, "max_norm")
    refused(lib, clip(lib, [a], [4], bf16=[2]), EINVAL, "grads_bf16")
    refused(lib, clip(lib, [a + 2], [4]), EINVAL, "aligned")
    refused(lib, clip(lib, [a + 1], [4], bf16=[1]), EINVAL, "aligned")
    # the same tensor twice, or two that share values, in place
    refused(lib, clip(lib, [a, b, a], [4, 4, 4]), EINVAL, "overlap")
    refused(lib, clip(lib, [a, b, a + 12], [4, 4, 4]), EINVAL, "overlap")
    # an output over another gradient, over another output, over half of its own gradient
    refused(lib, clip(lib, [a, b], [4, 4], outs=[b, A["old"]]), EINVAL, "overlap")
    refused(lib, clip(lib, [a, b], [4, 4], outs=[A["old"], A["old"] + 8]), EINVAL, "overlap")
    refused(lib, clip(lib, [a], [4], outs=[a + 8]), EINVAL, "overlap")
    refused(lib, clip(lib, [a], [4], outs=[None]), EINVAL, "null")


def test_model_calls(lib):
    assert lib.ar_gpt_backward_logp(None, A["targets"], A["targets"], A["grad"]) == EINVAL
    assert lib.ar_gpt_clip_grads(None, 1.0, None) == EINVAL
    assert lib.ar_gpt_set_grad_clip(None, 1.0) == EINVAL


def test_python_surface_refuses_host_tensors():
    import torch
    from autoresearch_amd import ops
    f, i = torch.zeros(64), torch.zeros(8, dtype=torch.int64)
    with pytest.raises(ValueError, match="device"):
        ops.token_logprob_fwd(f, f, i, 4, 8)
    with pytest.raises(ValueError, match="device"):
        ops.token_logprob_bwd(f, f, i, f, 0.0, 4, 8)
    with pytest.raises(ValueError, match="device"):
        ops.policy_loss(f, f, f, f, f, f, i, i, 0.2, 0.2, 0.1, False, 4, 2, 8)
    with pytest.raises(ValueError, match="device"):
        ops.policy_loss_logits(f, f, f, f, f, f, f, i, i, 0.0, 0.2, 0.2, 0.1, False, 4, 2, 8)
    with pytest.raises(ValueError, match="device"):
        ops.preference_loss(f, f, f, f, f, i, i, 0.1, 0.0, 4, 1, 8)
    with pytest.raises(ValueError, match="device"):
        ops.clip_grad_norm(f, None, [f], 1.0)
    with pytest.raises(ValueError, match="outputs"):
        ops.clip_grad_norm(f, [f, f], [f], 1.0)
