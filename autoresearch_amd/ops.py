"""Reference-named operator surface over the C ABI (kernels/ops.mojo,
optimizer.mojo, model.mojo kernels).

Each function takes device tensors (torch, on the GPU) in the reference
kernel's argument order and meaning, launches on torch's current stream and
raises ``ArError`` where the reference would raise.  Tensors must be
contiguous float32 (int64 for indices).  The post-training operators have no
counterpart in the reference; their logits and gradients are float32 or
bfloat16.  Nothing here computes on the host.
"""
from __future__ import annotations

from array import array

import torch

from ._lib import check, load

__all__ = [
    "Workspace", "embedding_fwd", "rmsnorm_fwd", "linear_fwd", "rope_fwd", "flash_attn_fwd",
    "flash_attn_bwd_precompute_d", "flash_attn_bwd_dq", "flash_attn_bwd_dkv", "relu_squared_fwd",
    "softcap_fwd", "ve_gate_fwd", "ve_apply_fwd", "add_residual_fwd", "scaled_add_fwd", "softmax_fwd",
    "cross_entropy_fwd", "mean_reduce", "cross_entropy_softcap_bwd", "linear_bwd_dx", "linear_bwd_dw",
    "rmsnorm_bwd", "rope_bwd", "relu_squared_bwd", "embedding_bwd", "scaled_add_bwd", "ve_apply_bwd",
    "ve_gate_bwd", "scalar_grad_reduce", "zero_buffer", "adamw_kernel", "adamw_step_group",
    "nesterov_momentum_kernel", "normalize_frobenius_kernel", "scale_add_kernel", "muon_update_kernel",
    "muon_step", "fill_normal_kernel", "fill_uniform_kernel", "fill_zeros_kernel", "fill_value_kernel",
    "precompute_rope", "token_logprob_fwd", "token_logprob_bwd", "policy_loss", "policy_loss_logits",
    "preference_loss", "clip_grad_norm",
]


def _stream():
    # torch.cuda.current_stream().cuda_stream without the stream object around
    # it, which takes 3 us to make: as long as a small call's kernel
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


class Workspace:
    """Device scratch for the entry points that need some (ar_workspace_*).

    Created once by the host (it is the one allocation), then bound to the
    streams whose per-op calls should use it.  Calls on a stream with no
    workspace bound, or one too small, raise ``ArError`` naming the bytes
    they need; no call allocates behind the caller's back."""

    def __init__(self, nbytes: int):
        import ctypes as ct
        self._lib = load()
        h = ct.c_void_p()
        check(self._lib.ar_workspace_create(ct.byref(h), int(nbytes)), "workspace_create")
        self.h = h

    @property
    def nbytes(self) -> int:
        return int(self._lib.ar_workspace_bytes(self.h))

    def bind(self, stream=None):
        """Bind to `stream` (a torch stream, a raw handle, or None = torch's current stream)."""
        s = _stream() if stream is None else getattr(stream, "cuda_stream", stream)
        check(self._lib.ar_workspace_bind(s, self.h), "workspace_bind")
        return self

    def close(self):
        if getattr(self, "h", None):
            check(self._lib.ar_workspace_destroy(self.h), "workspace_destroy")
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _p(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("device tensor required (no CPU path)")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    if t.dtype not in (torch.float32, torch.int64):
        raise TypeError(f"unsupported dtype {t.dtype}")
    return t.data_ptr()


def _call(name: str, *args):
    fn = getattr(load(), "ar_" + name)
    conv = [(_p(a) if isinstance(a, torch.Tensor) else a) for a in args]
    check(fn(_stream(), *conv), name)


def _sfx(bf16: bool) -> str:
    return "_bf16" if bf16 else ""


# ---- kernels/ops.mojo ----
def embedding_fwd(output, weight, indices, num_tokens, embd_dim):
    _call("embedding_fwd", output, weight, indices, num_tokens, embd_dim)


def rmsnorm_fwd(output, rms_out, input, num_rows, dim):
    _call("rmsnorm_fwd", output, rms_out, input, num_rows, dim)


def linear_fwd(output, input, weight, M, N, K, bf16=False):
    _call("linear_fwd" + _sfx(bf16), output, input, weight, M, N, K)


def rope_fwd(output, input, cos_buf, sin_buf, num_tokens, num_heads, head_dim):
    _call("rope_fwd", output, input, cos_buf, sin_buf, num_tokens, num_heads, head_dim)


def flash_attn_fwd(output, lse_out, q, k, v, B, T, num_heads, head_dim, window_size, bf16=False):
    _call("flash_attn_fwd" + _sfx(bf16), output, lse_out, q, k, v, B, T, num_heads, head_dim, window_size)


def flash_attn_bwd_precompute_d(d_out, output, grad_output, B, T, num_heads, head_dim, bf16=False):
    _call("flash_attn_bwd_precompute_d" + _sfx(bf16), d_out, output, grad_output, B, T, num_heads, head_dim)


def flash_attn_bwd_dq(grad_q, q, k, v, grad_output, lse, d_buf, B, T, num_heads, head_dim, window_size, bf16=False):
    _call("flash_attn_bwd_dq" + _sfx(bf16), grad_q, q, k, v, grad_output, lse, d_buf, B, T, num_heads, head_dim,
          window_size)


def flash_attn_bwd_dkv(grad_k, grad_v, q, k, v, grad_output, lse, d_buf, B, T, num_heads, head_dim, window_size,
                       bf16=False):
    _call("flash_attn_bwd_dkv" + _sfx(bf16), grad_k, grad_v, q, k, v, grad_output, lse, d_buf, B, T, num_heads,
          head_dim, window_size)


def relu_squared_fwd(output, input, size):
    _call("relu_squared_fwd", output, input, size)


def softcap_fwd(output, input, cap, size):
    _call("softcap_fwd", output, input, cap, size)


def ve_gate_fwd(gate_out, x_norm, gate_weight, num_tokens, n_kv_head, gate_channels, embd_dim):
    _call("ve_gate_fwd", gate_out, x_norm, gate_weight, num_tokens, n_kv_head, gate_channels, embd_dim)


def ve_apply_fwd(v, gate, ve, num_tokens, n_kv_head, head_dim):
    _call("ve_apply_fwd", v, gate, ve, num_tokens, n_kv_head, head_dim)


def add_residual_fwd(output, residual, input, size):
    _call("add_residual_fwd", output, residual, input, size)


def scaled_add_fwd(output, a, b, scale_a, scale_b, idx, size):
    _call("scaled_add_fwd", output, a, b, scale_a, scale_b, idx, size)


def softmax_fwd(output, input, num_rows, cols):
    _call("softmax_fwd", output, input, num_rows, cols)


def cross_entropy_fwd(loss_out, logits, targets, num_tokens, vocab_size):
    _call("cross_entropy_fwd", loss_out, logits, targets, num_tokens, vocab_size)


def mean_reduce(output, input, size):
    _call("mean_reduce", output, input, size)


def cross_entropy_softcap_bwd(grad_logits, logits, targets, cap, num_tokens, vocab_size, loss_scale):
    _call("cross_entropy_softcap_bwd", grad_logits, logits, targets, cap, num_tokens, vocab_size, loss_scale)


def linear_bwd_dx(grad_input, grad_output, weight, M, N, K, bf16=False):
    _call("linear_bwd_dx" + _sfx(bf16), grad_input, grad_output, weight, M, N, K)


def linear_bwd_dw(grad_weight, grad_output, input, M, N, K, bf16=False):
    _call("linear_bwd_dw" + _sfx(bf16), grad_weight, grad_output, input, M, N, K)


def rmsnorm_bwd(grad_input, grad_output, input, rms_saved, num_rows, dim):
    _call("rmsnorm_bwd", grad_input, grad_output, input, rms_saved, num_rows, dim)


def rope_bwd(grad_input, grad_output, cos_buf, sin_buf, num_tokens, num_heads, head_dim):
    _call("rope_bwd", grad_input, grad_output, cos_buf, sin_buf, num_tokens, num_heads, head_dim)


def relu_squared_bwd(grad_input, grad_output, input, size):
    _call("relu_squared_bwd", grad_input, grad_output, input, size)


def embedding_bwd(grad_weight, grad_output, indices, num_tokens, embd_dim):
    _call("embedding_bwd", grad_weight, grad_output, indices, num_tokens, embd_dim)


def scaled_add_bwd(grad_a, grad_b, grad_output, scale_a, scale_b, idx, size):
    _call("scaled_add_bwd", grad_a, grad_b, grad_output, scale_a, scale_b, idx, size)


def ve_apply_bwd(grad_ve, grad_gate, grad_v, gate, ve, num_tokens, n_kv_head, head_dim):
    _call("ve_apply_bwd", grad_ve, grad_gate, grad_v, gate, ve, num_tokens, n_kv_head, head_dim)


def ve_gate_bwd(grad_x_norm_out, grad_gate_weight, grad_gate, gate, x_norm, gate_weight, num_tokens, n_kv_head,
                gate_channels, embd_dim):
    _call("ve_gate_bwd", grad_x_norm_out, grad_gate_weight, grad_gate, gate, x_norm, gate_weight, num_tokens,
          n_kv_head, gate_channels, embd_dim)


def scalar_grad_reduce(grad_scalar, grad_output, input, idx, size):
    _call("scalar_grad_reduce", grad_scalar, grad_output, input, idx, size)


def zero_buffer(buf, size):
    _call("zero_buffer", buf, size)


# ---- optimizer.mojo ----
def adamw_kernel(params, grads, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, weight_decay, bias_corr1, bias_corr2,
                 size):
    _call("adamw", params, grads, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, weight_decay, bias_corr1, bias_corr2,
          size)


def adamw_step_group(params, grads, exp_avg, exp_avg_sq, size, lr, beta1, beta2, eps, weight_decay, lr_multiplier,
                     step):
    _call("adamw_step_group", params, grads, exp_avg, exp_avg_sq, size, lr, beta1, beta2, eps, weight_decay,
          lr_multiplier, step)


def nesterov_momentum_kernel(output, grads, momentum_buf, momentum, size):
    _call("nesterov_momentum", output, grads, momentum_buf, momentum, size)


def normalize_frobenius_kernel(data, size):
    _call("normalize_frobenius", data, size)


def scale_add_kernel(output, a, b, sa, sb, size):
    _call("scale_add", output, a, b, sa, sb, size)


def muon_update_kernel(params, grads, lr, wd, size):
    _call("muon_update", params, grads, lr, wd, size)


def muon_step(params, grads, momentum_buf, rows, cols, initial_lr, lr_multiplier, momentum, weight_decay,
              bf16=False):
    _call("muon_step", params, grads, momentum_buf, rows, cols, initial_lr, lr_multiplier, momentum, weight_decay,
          1 if bf16 else 0)


# ---- model.mojo init ----
def fill_normal_kernel(output, seed_base, std, size):
    _call("fill_normal", output, seed_base, std, size)


def fill_uniform_kernel(output, seed_base, low, high, size):
    _call("fill_uniform", output, seed_base, low, high, size)


def fill_zeros_kernel(output, size):
    _call("fill_zeros", output, size)


def fill_value_kernel(output, value, size):
    _call("fill_value", output, value, size)


def precompute_rope(cos_buf, sin_buf, seq_len, head_dim, base=10000.0):
    _call("precompute_rope", cos_buf, sin_buf, seq_len, head_dim, base)


# ---- post-training: token log-probabilities, losses, gradient clipping ----
_LOGITS = (torch.float32, torch.bfloat16)


def _device(nm: str, t) -> int:
    """The device of a call's first tensor: the current one."""
    d = -1 if t is None else t.get_device()
    if d < 0 or d != torch.cuda.current_device():
        raise ValueError(f"{nm}: tensors on the current device are required")
    return d


def _dev(nm: str, what: str, t, n: int, dev: int, dtype=torch.float32, optional: bool = False):
    """The address of an array of at least n elements of dtype on device dev."""
    if t is None and (optional or n == 0):
        return None
    if t is None or t.get_device() != dev:
        raise ValueError(f"{nm} {what}: a tensor on the current device is required")
    if t.dtype is not dtype:
        raise TypeError(f"{nm} {what}: unsupported dtype {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{nm} {what}: tensor must be contiguous")
    if t.numel() < n:
        raise ValueError(f"{nm} {what}: {t.numel()} elements, {n} needed")
    return t.data_ptr()


def _logits(nm: str, logits, grad, num_tokens, vocab_size, dev):
    """Addresses of the logits and their gradient, and whether they are bf16."""
    dtype = torch.float32 if logits is None else logits.dtype
    if dtype not in _LOGITS:
        raise TypeError(f"{nm} logits: unsupported dtype {dtype}")
    n = num_tokens * vocab_size
    return (_dev(nm, "logits", logits, n, dev, dtype),
            None if grad is None else _dev(nm, "grad_logits", grad, n, dev, dtype), int(dtype is torch.bfloat16))


def _launch(nm: str, *args):
    check(getattr(load(), "ar_" + nm)(_stream(), *args), nm)


def token_logprob_fwd(logp_out, logits, targets, num_tokens, vocab_size):
    """logp_out[t] = logits[t, targets[t]] - logsumexp(logits[t]); 0 where the target is no token."""
    nm, n, dev = "token_logprob_fwd", num_tokens, _device("token_logprob_fwd", logp_out)
    z, _, bf16 = _logits(nm, logits, None, n, vocab_size, dev)
    _launch(nm, _dev(nm, "logp_out", logp_out, n, dev), z, bf16, _dev(nm, "targets", targets, n, dev, torch.int64), n,
            vocab_size)


def token_logprob_bwd(grad_logits, logits, targets, grad_logp, cap, num_tokens, vocab_size):
    """The gradient of sum_t grad_logp[t] logp[t] by the logits before the softcap `cap` (0: none)."""
    nm, n, dev = "token_logprob_bwd", num_tokens, _device("token_logprob_bwd", grad_logits)
    z, g, bf16 = _logits(nm, logits, grad_logits, n, vocab_size, dev)
    _launch(nm, g, z, bf16, _dev(nm, "targets", targets, n, dev, torch.int64),
            _dev(nm, "grad_logp", grad_logp, n, dev), cap, n, vocab_size)


def _batch(nm, old_logp, ref_logp, advantages, targets, seq_start, n, num_seqs, dev):
    return (_dev(nm, "old_logp", old_logp, n, dev, optional=True),
            _dev(nm, "ref_logp", ref_logp, n, dev, optional=True), _dev(nm, "advantages", advantages, n, dev),
            _dev(nm, "targets", targets, n, dev, torch.int64),
            _dev(nm, "seq_start", seq_start, num_seqs + 1, dev, torch.int64, optional=True))


def policy_loss(loss_out, grad_logp, logp, old_logp, ref_logp, advantages, targets, seq_start, clip_low, clip_high,
                kl_coef, per_seq, num_tokens, num_seqs, vocab_size, loss_scale=1.0):
    """loss_out = (clipped policy loss with its KL term, mean KL); grad_logp = its gradient (None: not formed)."""
    nm, n, dev = "policy_loss", num_tokens, _device("policy_loss", loss_out)
    _launch(nm, _dev(nm, "loss_out", loss_out, 2, dev), _dev(nm, "grad_logp", grad_logp, n, dev, optional=True),
            _dev(nm, "logp", logp, n, dev),
            *_batch(nm, old_logp, ref_logp, advantages, targets, seq_start, n, num_seqs, dev), clip_low, clip_high,
            kl_coef, int(per_seq), n, num_seqs, vocab_size, loss_scale)


def policy_loss_logits(loss_out, logp_out, grad_logits, logits, old_logp, ref_logp, advantages, targets, seq_start,
                       cap, clip_low, clip_high, kl_coef, per_seq, num_tokens, num_seqs, vocab_size, loss_scale=1.0):
    """policy_loss from the logits, with its gradient by them (before the softcap), in one pass over them."""
    nm, n, dev = "policy_loss_logits", num_tokens, _device("policy_loss_logits", loss_out)
    z, g, bf16 = _logits(nm, logits, grad_logits, n, vocab_size, dev)
    _launch(nm, _dev(nm, "loss_out", loss_out, 2, dev), _dev(nm, "logp_out", logp_out, n, dev, optional=True), g, z,
            bf16, *_batch(nm, old_logp, ref_logp, advantages, targets, seq_start, n, num_seqs, dev), cap, clip_low,
            clip_high, kl_coef, int(per_seq), n, num_seqs, vocab_size, loss_scale)


def preference_loss(loss_out, margin_out, grad_logp, logp, ref_logp, targets, seq_start, beta, label_smoothing,
                    num_tokens, num_pairs, vocab_size, loss_scale=1.0):
    """The preference loss of pairs of sequences (2 i chosen, 2 i + 1 rejected), their margins and the gradient."""
    nm, n, dev = "preference_loss", num_tokens, _device("preference_loss", loss_out)
    _launch(nm, _dev(nm, "loss_out", loss_out, 1, dev),
            _dev(nm, "margin_out", margin_out, num_pairs, dev, optional=True),
            _dev(nm, "grad_logp", grad_logp, n, dev, optional=True), _dev(nm, "logp", logp, n, dev),
            _dev(nm, "ref_logp", ref_logp, n, dev, optional=True),
            _dev(nm, "targets", targets, n, dev, torch.int64),
            _dev(nm, "seq_start", seq_start, 2 * num_pairs + 1, dev, torch.int64), beta, label_smoothing, n, num_pairs,
            vocab_size, loss_scale)


def clip_grad_norm(norm_out, outputs, grads, max_norm):
    """norm_out = the 2-norm of all of grads; outputs[i] = grads[i] min(1, max_norm / norm).
    outputs None: in place.  max_norm math.inf: the norm alone."""
    if outputs is not None and len(outputs) != len(grads):
        raise ValueError(f"clip_grad_norm: {len(outputs)} outputs for {len(grads)} gradients")
    nm, n, dev = "clip_grad_norm", len(grads), _device("clip_grad_norm", norm_out)
    types, sizes = [g.dtype for g in grads], list(map(torch.Tensor.numel, grads))
    for t in set(types).difference(_LOGITS):
        raise TypeError(f"{nm} grads: unsupported dtype {t}")

    def addresses(what, tensors):
        # _dev's checks over all tensors at once: half its time for each
        if not (all(map(torch.Tensor.is_contiguous, tensors)) and set(map(torch.Tensor.get_device, tensors)) <= {dev}
                and [t.dtype for t in tensors] == types and list(map(torch.Tensor.numel, tensors)) == sizes):
            for t, k, d in zip(tensors, sizes, types):
                _dev(nm, what, t, k, dev, d)
            raise ValueError(f"{nm} {what}: as many elements as the gradients are required")
        return array("Q", map(torch.Tensor.data_ptr, tensors))

    def at(a):
        return None if a is None else a.buffer_info()[0]

    pg, po = addresses("grads", grads), None if outputs is None else addresses("outputs", outputs)
    bf16, sz = array("i", [t is torch.bfloat16 for t in types]), array("q", sizes)
    _launch(nm, _dev(nm, "norm_out", norm_out, 1, dev), at(po), at(pg), at(bf16), at(sz), n, max_norm)
