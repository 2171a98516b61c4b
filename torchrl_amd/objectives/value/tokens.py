"""Policies over tokens: what V-trace's ``log_pi`` / ``log_mu`` and a policy-gradient loss need of a network's logits.

:func:`process_logits` applies the penalties for repeated tokens, the bias, the temperature and the (grammar) mask that a token was
sampled under; :func:`token_log_prob` gives the log-probability of the stored tokens and the entropy under the same processing,
without ever writing the processed logits or a softmax to memory, and their gradient.  :class:`TokenActor` wraps a logits network into
the ``actor_network`` that :class:`~torchrl_amd.objectives.value.VTrace` calls.  The kernels are behind ``trl_process_logits_fwd`` /
``_bwd`` and ``trl_token_log_prob_fwd`` / ``_bwd`` of include/trl_value.h, which has the formulas.

The reference masks logits in ``MaskedCategorical`` (torchrl/modules/distributions/discrete.py) and has no counterpart of the rest.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import nn, Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from torchrl_amd import _extension
from torchrl_amd.objectives.value import functional as F
from torchrl_amd.objectives.value.functional import _host_done, _native, _ptr

__all__ = ["process_logits", "token_log_prob", "TokenActor"]

_DT = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}
_INT = (torch.int32, torch.int64)
_NONE, _BOOL, _BITS = 0, 1, 2
_LARGEST = torch.finfo(torch.float32).max

Scalar = Union[float, Tensor]


class _Processing(NamedTuple):
    """Validated processing of (B, T, V) logits, in the layout that the kernels read."""

    B: int
    T: int
    V: int
    logits: Tensor  # (B, T, V), last stride 1
    tokens: Optional[Tensor]  # (B, L), last stride 1
    lengths: Optional[Tensor]  # (B, T) dense
    prompt: Optional[Tensor]  # (B,) dense
    rep: float
    pres: float
    freq: float
    temp: float
    rep_t: Optional[Tensor]  # (B,) float32 dense, instead of the number
    pres_t: Optional[Tensor]
    freq_t: Optional[Tensor]
    temp_t: Optional[Tensor]
    bias: Optional[Tensor]  # (B, T, V), any leading strides
    mask: Optional[Tensor]  # (B, T, V) truth values or (B, T, words) bits


_TENSORS = ("logits", "tokens", "lengths", "prompt", "rep_t", "pres_t", "freq_t", "temp_t", "bias", "mask")


def _need(ok, error, text):
    if not ok:
        raise error(text)


def _rows_view(x: Tensor, batch, T: int, name: str) -> Tensor:
    """``x`` broadcast to ``[*batch, T, n]`` as a (B, T, n) tensor with last stride 1; only batch dims that cannot be merged are copied."""
    n = x.shape[-1]
    lead = tuple(x.shape[:-1])
    full = (*batch, T)
    _need(len(lead) <= len(full) and all(a in (1, b) for a, b in zip(lead[::-1], full[::-1])), RuntimeError,
          f"{name} of shape {tuple(x.shape)} does not broadcast to the logits' rows {full}")
    if x.stride(-1) != 1 and n > 1:
        x = x.contiguous()
    own_T = lead[-1] if lead else 1
    x = x.expand(*batch, own_T, n).reshape(math.prod(batch), own_T, n)
    return x.expand(-1, T, -1)


def _per_sequence(x: Scalar, batch, name: str, device, positive: bool) -> Tuple[float, Optional[Tensor]]:
    if not isinstance(x, Tensor):
        x = float(x)
        _need(math.isfinite(x) and abs(x) <= _LARGEST and (x >= 2.0 ** -126 or not positive), ValueError,
              f"{name} must be {'positive and ' if positive else ''}finite in float32, got {x}")
        return x, None
    _need(not (torch.is_grad_enabled() and x.requires_grad), NotImplementedError, f"gradients with respect to {name} are not implemented: detach it")
    _need(x.device == device, RuntimeError, f"{name} is on {x.device}, the logits on {device}")
    _need(x.dtype.is_floating_point, RuntimeError, f"{name} must be a floating-point tensor, got {x.dtype}")
    _need(x.ndim <= len(batch) and all(a in (1, b) for a, b in zip(x.shape[::-1], batch[::-1])), RuntimeError,
          f"{name} of shape {tuple(x.shape)} does not broadcast to the sequences {tuple(batch)}")
    return 1.0, x.to(torch.float32).expand(batch).reshape(-1).contiguous()


def _int_tensor(x, shape, name: str, device) -> Tensor:
    _need(isinstance(x, Tensor) and x.dtype in _INT, RuntimeError, f"{name} must be an int32 or int64 tensor")
    _need(x.device == device, RuntimeError, f"{name} is on {x.device}, the logits on {device}")
    _need(tuple(x.shape) == tuple(shape), RuntimeError, f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    return x.reshape(-1).contiguous()


def _processing(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, mask,
                temperature) -> _Processing:
    _need(isinstance(logits, Tensor), TypeError, "logits must be a tensor")
    _need(logits.dtype in _DT, NotImplementedError, f"torchrl_amd token operators support float32, bfloat16 and float16 logits, got {logits.dtype}")
    _need(logits.ndim >= 1 and logits.shape[-1] > 0, RuntimeError, f"logits need a vocabulary dim, got shape {tuple(logits.shape)}")
    dev, V, lead = logits.device, logits.shape[-1], tuple(logits.shape[:-1])
    _need(V <= 2 ** 31 - 1, RuntimeError, "a vocabulary of 2**31 tokens or more is not supported")
    if tokens is not None:
        _need(isinstance(tokens, Tensor) and tokens.dtype in _INT, RuntimeError, "tokens must be an int32 or int64 tensor")
        _need(tokens.device == dev, RuntimeError, f"tokens is on {tokens.device}, the logits on {dev}")
        _need(tokens.ndim in (logits.ndim, logits.ndim - 1) and tokens.ndim >= 1, RuntimeError,
              f"tokens must be [*B, L] for logits [*B, V] or [*B, T, V], got {tuple(tokens.shape)} for {tuple(logits.shape)}")
        steps = tokens.ndim == logits.ndim - 1
    else:
        steps = len(lead) >= 2
    batch, T = (lead[:-1], lead[-1]) if steps else (lead, 1)
    B = math.prod(batch)
    rep, rep_t = _per_sequence(repetition_penalty, batch, "repetition_penalty", dev, True)
    pres, pres_t = _per_sequence(presence_penalty, batch, "presence_penalty", dev, False)
    freq, freq_t = _per_sequence(frequency_penalty, batch, "frequency_penalty", dev, False)
    temp, temp_t = _per_sequence(temperature, batch, "temperature", dev, True)
    penalised = rep_t is not None or pres_t is not None or freq_t is not None or rep != 1.0 or pres != 0.0 or freq != 0.0
    prompt = None
    if tokens is None:
        _need(not penalised, ValueError, "penalties need the tokens that they are for")
        _need(lengths is None and prompt_lengths is None, ValueError, "lengths and prompt_lengths go with tokens")
    else:
        _need(tuple(tokens.shape[:-1]) == tuple(batch), RuntimeError,
              f"tokens of shape {tuple(tokens.shape)} do not belong to logits of shape {tuple(logits.shape)}")
        if lengths is None:
            _need(not steps, ValueError, "logits [*B, T, V] need lengths [*B, T]: how many tokens each row has seen")
        else:
            lengths = _int_tensor(lengths, lead, "lengths", dev)
        if prompt_lengths is not None:
            prompt = _int_tensor(prompt_lengths, batch, "prompt_lengths", dev)
        L = tokens.shape[-1]
        if not penalised or L == 0:
            tokens = lengths = prompt = None
        else:
            tokens = tokens.reshape(B, L)
            if tokens.stride(-1) != 1 and L > 1:
                tokens = tokens.contiguous()
    if bias is not None:
        _need(isinstance(bias, Tensor) and bias.dtype in _DT, RuntimeError, "bias must be a float32, bfloat16 or float16 tensor")
        _need(bias.device == dev, RuntimeError, f"bias is on {bias.device}, the logits on {dev}")
        _need(not (torch.is_grad_enabled() and bias.requires_grad), NotImplementedError,
              "gradients with respect to bias are not implemented: detach it, or add it to the logits")
        _need(bias.ndim >= 1 and bias.shape[-1] == V, RuntimeError, f"bias must have {V} entries in its last dim, got shape {tuple(bias.shape)}")
        bias = _rows_view(bias if steps else bias.unsqueeze(-2), batch, T, "bias")
    if mask is not None:
        _need(isinstance(mask, Tensor) and mask.dtype in (torch.bool, torch.int32), RuntimeError,
              "mask must be a bool tensor [..., V] or an int32 tensor of bits [..., ceil(V / 32)]")
        _need(mask.device == dev, RuntimeError, f"mask is on {mask.device}, the logits on {dev}")
        n = V if mask.dtype == torch.bool else (V + 31) // 32
        _need(mask.ndim >= 1 and mask.shape[-1] == n, RuntimeError, f"a {mask.dtype} mask must have {n} entries in its last dim, got shape {tuple(mask.shape)}")
        mask = _rows_view(mask if steps else mask.unsqueeze(-2), batch, T, "mask")
    for t, name in ((logits, "logits"), (bias, "bias"), *((s, "a penalty or the temperature") for s in (rep_t, pres_t, freq_t, temp_t))):
        _need(t is None or forward_ad.unpack_dual(t).tangent is None, NotImplementedError, f"forward-mode derivatives with respect to {name} are not implemented")
    if logits.device.type != "cuda":
        raise RuntimeError(f"torchrl_amd token operators run on MI355X (HIP, device type 'cuda') tensors only; got a tensor on {logits.device}.")
    x = logits.detach()
    return _Processing(B, T, V, _rows_view(x if steps else x.unsqueeze(-2), batch, T, "logits"), tokens, lengths, prompt, rep, pres, freq, temp,
                       rep_t, pres_t, freq_t, temp_t, bias, mask)


def _wide(x):
    return 0 if x is None or x.dtype == torch.int32 else 1


def _args(p: _Processing, **more) -> "_extension.TokenArgs":
    z, tok, bias, mask = p.logits, p.tokens, p.bias, p.mask
    a = _extension.TokenArgs(
        _DT[z.dtype], _NONE if mask is None else _BOOL if mask.dtype == torch.bool else _BITS, 0 if bias is None else 1 + _DT[bias.dtype],
        _wide(tok), _wide(p.lengths), _wide(p.prompt), 0, p.rep, p.pres, p.freq, p.temp, p.B, p.T, p.V, 0 if tok is None else tok.shape[1],
        z.data_ptr(), z.stride(0), z.stride(1), _ptr(tok), 0 if tok is None else tok.stride(0), _ptr(p.lengths), _ptr(p.prompt),
        _ptr(p.rep_t), _ptr(p.pres_t), _ptr(p.freq_t), _ptr(p.temp_t))
    if bias is not None:
        size = bias.element_size()
        a.bias, a.bias_sb, a.bias_st = bias.data_ptr(), bias.stride(0) * size, bias.stride(1) * size
    if mask is not None:
        size = mask.element_size()
        a.mask, a.mask_sb, a.mask_st = mask.data_ptr(), mask.stride(0) * size, mask.stride(1) * size
    for k, v in more.items():
        setattr(a, k, v)
    return a


def _save(ctx, p: _Processing, *more, logits: bool = True):
    """Keeps a call's tensors with autograd, which notices when one is written in place before the backward pass."""
    saved = [getattr(p, k) for k in _TENSORS]
    if not logits:
        saved[0] = None
    ctx.save_for_backward(*saved, *more)
    ctx.forms = [F._kept_form(t) for t in (*saved, *more)]
    ctx.numbers = p._replace(**dict.fromkeys(_TENSORS))


def _saved(ctx):
    kept = ctx.saved_tensors
    F._check_kept(kept, ctx.forms)
    # a hook may hand back another layout: rows of vectors need a last stride of 1, the rest has to be dense
    rows = ("logits", "tokens", "bias", "mask")
    tensors = {k: t if t is None or (k in rows and t.stride(-1) == 1) else t.contiguous() for k, t in zip(_TENSORS, kept)}
    return ctx.numbers._replace(**tensors), [None if t is None else t.contiguous() for t in kept[len(_TENSORS):]]


# ---- process_logits ---------------------------------------------------------------------------------------------------------
def _process_fwd(p: _Processing, out: Tensor) -> None:
    if p.B * p.T:
        _native("trl_process_logits_fwd", out.device, _args(p, out=out.data_ptr(), out_sb=out.stride(0), out_st=out.stride(1)))


def _process_new(p: _Processing, shape) -> Tensor:
    """The processed logits in a tensor of their own; not a view, so that it may be written in place whatever its history."""
    out = torch.empty(shape, dtype=p.logits.dtype, device=p.logits.device)
    _process_fwd(p, out.view(p.B, p.T, p.V))
    return out


def _process_bwd(p: _Processing, grad: Tensor) -> Tensor:
    """d_logits (B, T, V); ``p.logits`` may be ``grad`` itself where the logits are not read (no repetition penalty)."""
    grad = grad.reshape(p.B, p.T, p.V).contiguous()
    d = torch.empty_like(grad)
    if p.B * p.T:
        _native("trl_process_logits_bwd", grad.device, _args(p, grad_out=grad.data_ptr(), out=d.data_ptr(), out_sb=d.stride(0), out_st=d.stride(1)))
    return d


def _reads_sign(p: _Processing) -> bool:
    return p.tokens is not None and (p.rep_t is not None or p.rep != 1.0)


class _ProcessLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, p):
        out = _process_new(p, logits.shape)
        _save(ctx, p, logits=_reads_sign(p))
        ctx.shape = logits.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, _ = _saved(ctx)
        if p.logits is None:
            p = p._replace(logits=grad.reshape(p.B, p.T, p.V).contiguous())
        return _process_bwd(p, grad).view(ctx.shape), None


def _apart(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors with dense rows share no byte: they lie one behind the other, or their rows lie beside each other in rows of one buffer."""
    def span(x):
        return x.data_ptr(), x.data_ptr() + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return True
    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    step = math.gcd(*(s * x.element_size() for x in (a, b) for n, s in zip(x.shape[:-1], x.stride()) if n > 1))
    off = (b0 - a0) % step if step else 0
    return off >= a.shape[-1] * a.element_size() and off + b.shape[-1] * b.element_size() <= step


def _out_rows(p: _Processing, logits: Tensor, out: Tensor) -> Tensor:
    """``out`` as (B, T, V), after what :func:`process_logits` promises of it has been checked."""
    _need(isinstance(out, Tensor) and out.shape == logits.shape and out.dtype == logits.dtype and out.device == logits.device, RuntimeError,
          "out must have the logits' shape, dtype and device")
    _need(not (torch.is_grad_enabled() and out.requires_grad), RuntimeError, "process_logits(out=...) does not support automatic differentiation")
    try:
        o = out.view(p.B, p.T, p.V)
    except RuntimeError:
        o = None
    _need(o is not None and (o.stride(2) == 1 or p.V == 1) and (o.stride(1) >= p.V or p.T == 1) and (o.stride(0) >= p.V or p.B == 1), RuntimeError,
          "out must have rows that are dense and do not overlap, and batch dims that can be merged")
    _need(p.B == 1 or p.T == 1 or o.stride(0) >= p.T * o.stride(1) or o.stride(1) >= p.B * o.stride(0), RuntimeError,
          "out must have rows that do not overlap")
    # in place every element is read and written by one thread; a bias or a mask is read by all rows
    same = out.data_ptr() == p.logits.data_ptr() and out.stride() == logits.stride()
    _need(all(t is None or _apart(o, t) for k, t in ((k, getattr(p, k)) for k in _TENSORS) if not (same and k == "logits")), RuntimeError,
          "out must be the logits themselves or share no memory with the inputs")
    return o


def process_logits(logits: Tensor, *, tokens: Optional[Tensor] = None, lengths: Optional[Tensor] = None, prompt_lengths: Optional[Tensor] = None,
                   repetition_penalty: Scalar = 1.0, presence_penalty: Scalar = 0.0, frequency_penalty: Scalar = 0.0,
                   bias: Optional[Tensor] = None, mask: Optional[Tensor] = None, temperature: Scalar = 1.0,
                   out: Optional[Tensor] = None) -> Tensor:
    """The logits that a token is sampled from: penalties for repeated tokens, a bias, a temperature and a mask.

    ``logits`` is ``[*B, V]`` (one decoding step) or ``[*B, T, V]`` (a rollout), float32, bfloat16 or float16; arithmetic is float32 and
    the result is rounded once to the logits' dtype.  In this order::

        z = z / repetition_penalty  where z > 0, else  z * repetition_penalty     for tokens in the row's history
        z = z - frequency_penalty * n - presence_penalty * (n > 0)                n: how often the token stands behind the prompt
        z = (z + bias) / temperature
        z = -inf                                                                  where the mask does not allow the token

    ``tokens`` ``[*B, L]`` holds each sequence's ids (ids outside ``[0, V)``, such as a padding id of -1, are no tokens).  A row's history is
    its first ``lengths`` tokens (shape of the logits without the last dim; may be left out for one decoding step: all of them).  For the
    logits of a rollout that is what had been seen when the row's token was picked.  ``prompt_lengths`` ``[*B]``: where the
    presence and frequency penalties begin to count (0: at the start); the repetition penalty counts the prompt too.  Penalties and temperature are
    numbers or tensors that broadcast to ``[*B]`` (tensors are not read on the host: repetition penalties and temperatures in them have to be positive).  ``bias`` broadcasts to the logits.  ``mask`` broadcasts to the logits too: truth values, or
    bits of int32 words ``[..., ceil(V / 32)]`` (token j: bit ``j % 32`` of word ``j // 32``); what the logits hold in masked places does not matter.

    Differentiable in ``logits``; masked places get no gradient.  ``out`` (not under autograd) may be ``logits`` itself, and shares no
    memory with any other input."""
    compiling = torch.compiler.is_compiling()
    host = None if compiling else F._HOST if F._HOST_TRIED else F._host_module()
    if host is not None and out is None:  # the plain layouts in one C++ hop (csrc/host_policy.cpp)
        got = host.process_logits(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, mask,
                                  temperature)
        if got is not None:
            return _host_done(got)
    if compiling or F._recorded():
        _need(out is None, NotImplementedError, "process_logits(out=...) is not supported under torch.compile, make_fx and torch.jit.trace")
        from torchrl_amd.objectives.value import _ops
        return _ops.process_logits(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, mask,
                                   temperature)
    p = _processing(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, mask, temperature)
    if F._needs_grad(logits):
        _need(out is None, RuntimeError, "process_logits(out=...) does not support automatic differentiation")
        return _ProcessLogits.apply(logits, p)
    if out is None:
        return _process_new(p, logits.shape)
    _process_fwd(p, _out_rows(p, logits, out))
    torch.autograd.graph.increment_version(out)
    return out


# ---- token_log_prob ---------------------------------------------------------------------------------------------------------
def _log_prob_fwd(p: _Processing, action: Tensor, shape, entropy: bool, stats: bool):
    """log_prob and entropy of ``shape`` (tensors of their own, no views), and {max, log2 of the sum} a row."""
    dev = action.device
    n = p.B * p.T
    log_prob = torch.empty(shape, dtype=torch.float32, device=dev)
    H = torch.empty(shape, dtype=torch.float32, device=dev) if entropy else None
    st = torch.empty(n, 2, dtype=torch.float32, device=dev) if stats else None
    if n:
        need = _extension.get_lib().trl_token_workspace_bytes(p.B, p.T, p.V)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _native("trl_token_log_prob_fwd", dev, _args(p, action=action.data_ptr(), action_wide=_wide(action), log_prob=log_prob.data_ptr(),
                                                   entropy=_ptr(H), stats=_ptr(st)), ws.data_ptr(), need)
    return log_prob, H, st


def _row_grad(g: Optional[Tensor]) -> Optional[Tensor]:
    return None if g is None else g.reshape(-1).to(torch.float32).contiguous()


def _log_prob_bwd(p: _Processing, action: Tensor, H: Optional[Tensor], stats: Tensor, g_lp: Optional[Tensor], g_H: Optional[Tensor]) -> Tensor:
    d = torch.empty(p.B, p.T, p.V, dtype=p.logits.dtype, device=action.device)
    n = p.B * p.T
    F._check_kept((stats,), ((torch.float32, (n, 2), p.logits.device),))
    if n:
        g_lp, g_H = _row_grad(g_lp), _row_grad(g_H)
        _native("trl_token_log_prob_bwd", action.device, _args(p, action=action.data_ptr(), action_wide=_wide(action), entropy=_ptr(H),
                                                             stats=stats.data_ptr(), g_log_prob=_ptr(g_lp), g_entropy=_ptr(g_H), out=d.data_ptr(),
                                                             out_sb=d.stride(0), out_st=d.stride(1)))
    return d


class _TokenLogProb(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, p, action, entropy):
        ctx.set_materialize_grads(False)
        log_prob, H, stats = _log_prob_fwd(p, action, logits.shape[:-1], entropy, True)
        _save(ctx, p, action, H, stats)
        ctx.shape = logits.shape
        return log_prob, H

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_H):
        if g_lp is None and g_H is None:
            return None, None, None, None
        p, (action, H, stats) = _saved(ctx)
        return _log_prob_bwd(p, action, H, stats, g_lp, g_H).view(ctx.shape), None, None, None


def token_log_prob(logits: Tensor, action: Tensor, *, entropy: bool = False, tokens: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                   prompt_lengths: Optional[Tensor] = None, repetition_penalty: Scalar = 1.0, presence_penalty: Scalar = 0.0,
                   frequency_penalty: Scalar = 0.0, bias: Optional[Tensor] = None, mask: Optional[Tensor] = None,
                   temperature: Scalar = 1.0) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Log-probability of the stored tokens (and the entropy) under the processed logits, float32, shape of ``action``.

    ``action`` (int32 or int64, shape of the logits without the last dim) holds the picked ids; every other argument is
    :func:`process_logits`'s, and the result is that of a log-softmax of its (unrounded) output.  A negative action marks padding: 0, no
    gradient, and the row is not read.  In a row that allows nothing the log-probability is ``-inf`` and the entropy 0, without a gradient; an
    action that the mask does not allow has ``-inf`` too; an id of ``V`` or more gives NaN.

    Differentiable in ``logits`` (whose gradient has their dtype); neither a softmax nor the processed logits are kept for that."""
    compiling = torch.compiler.is_compiling()
    host = None if compiling else F._HOST if F._HOST_TRIED else F._host_module()
    if host is not None:  # the plain layouts in one C++ hop (csrc/host_policy.cpp)
        got = host.token_log_prob(logits, action, bool(entropy), tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty,
                                  frequency_penalty, bias, mask, temperature)
        if got is not None:
            return _host_done(got)
    if compiling or F._recorded():
        from torchrl_amd.objectives.value import _ops
        return _ops.token_log_prob(logits, action, entropy, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty,
                                   bias, mask, temperature)
    _need(isinstance(logits, Tensor), TypeError, "logits must be a tensor")
    lead = logits.shape[:-1]
    act = _int_tensor(action, lead, "action", logits.device)
    p = _processing(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, mask, temperature)
    if F._needs_grad(logits):
        log_prob, H = _TokenLogProb.apply(logits, p, act, bool(entropy))
    else:
        log_prob, H, _ = _log_prob_fwd(p, act, lead, bool(entropy), False)
    return (log_prob, H) if entropy else log_prob


class TokenActor(nn.Module):
    """A logits network as the ``actor_network`` of :class:`~torchrl_amd.objectives.value.VTrace`: ``actor(data)`` is the log-probability of the
    stored tokens under the distribution that they are sampled from.

    ``network``: any callable ``data -> logits [*B, T, V]`` (or a collection that holds them under ``logits_key``).  The keys name where the
    data keeps the picked ids, the sequences (``tokens`` / ``lengths`` / ``prompt_lengths`` of :func:`process_logits`) and a mask a row;
    ``bias``, ``temperature`` and the penalties are :func:`process_logits`'s; tensors among them move with the module."""

    def __init__(self, network, *, action_key="action", logits_key="logits", tokens_key=None, lengths_key=None, prompt_lengths_key=None, mask_key=None,
                 bias: Optional[Tensor] = None, temperature: Scalar = 1.0, repetition_penalty: Scalar = 1.0, presence_penalty: Scalar = 0.0,
                 frequency_penalty: Scalar = 0.0):
        super().__init__()
        self.network = network
        self.action_key, self.logits_key = action_key, logits_key
        self.data_keys = {"tokens": tokens_key, "lengths": lengths_key, "prompt_lengths": prompt_lengths_key, "mask": mask_key}
        self.register_buffer("bias", bias)
        self.settings = {"temperature": temperature, "repetition_penalty": repetition_penalty, "presence_penalty": presence_penalty,
                         "frequency_penalty": frequency_penalty}

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        for k, v in self.settings.items():  # tensors follow to the module's device; what they hold is float32 arithmetic's and keeps its type
            if isinstance(v, Tensor):
                self.settings[k] = v.to(fn(v).device)
        return self

    def _inputs(self, data):
        logits = self.network(data)
        if not isinstance(logits, Tensor):
            logits = logits.get(self.logits_key)
        return logits, {"bias": self.bias, **self.settings, **{k: data.get(key) for k, key in self.data_keys.items() if key is not None}}

    def logits(self, data) -> Tensor:
        """The processed logits: what to sample from."""
        logits, kwargs = self._inputs(data)
        return process_logits(logits, **kwargs)

    def evaluate(self, data) -> Tuple[Tensor, Tensor]:
        """(log-probability of the stored tokens, entropy), both differentiable in the network: what a policy-gradient loss needs."""
        logits, kwargs = self._inputs(data)
        return token_log_prob(logits, data.get(self.action_key).reshape(logits.shape[:-1]), entropy=True, **kwargs)

    def forward(self, data) -> Tensor:
        logits, kwargs = self._inputs(data)
        return token_log_prob(logits, data.get(self.action_key).reshape(logits.shape[:-1]), **kwargs)
