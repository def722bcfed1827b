"""Scoring of given tokens: log-probability, entropy and the most likely alternatives of a row, from logits
(csrc/kernels/logprobs.cu) or straight from hidden states and the output projection (csrc/kernels/head_logprobs.cu).

With x a row of scores, T its temperature (1 without one, and where it is not above 0) and u = x / T:

    logprob = u[id] - log sum exp u        entropy = log sum exp u - sum softmax(u) u

A negative id asks for nothing and gets 0.  An id beyond the vocabulary cannot occur: -inf.  A row whose scores are all -inf
has no distribution: logprob -inf, entropy 0, no alternatives.  A NaN or +inf in a row makes its results NaN.
Sums, maxima and results are fp32 whatever the scores' type.
"""
from __future__ import annotations

import functools

import torch

from . import _count, _debug, _lib
from ._lib import I, L, P, check, ptr, stream_on

_lib.register_signature("xllm_token_logprobs", [P, L, I, I, I, P, P, I, P, P, P, P, P])
_lib.register_signature("xllm_head_logprobs", [P, L, P, L, I, I, I, P, P, P, P, P, P])
_lib.register_signature("xllm_head_logprobs_workspace", [I, I, I], L)
_lib.register_signature("xllm_head_logprobs_error_status", [], I)

MAX_TOP = 128          # alternatives a row can list
MAX_ROWS = 1 << 30     # of a call: tiles of rows are counted in 32 bits
MAX_COLUMNS = 1 << 30  # of a row, and tokens of a vocabulary: as are the places in a row


def _results(d, x_id, ids, vocab):
    """(logprob, entropy, log normaliser) of rows d = u - max(u), the given tokens' d in x_id."""
    e = torch.exp(d)
    z = e.sum(-1)
    log_z = torch.log(z)
    entropy = log_z - torch.where(e == 0, 0.0, e * d).sum(-1) / z
    logprob = torch.where(ids >= vocab, float("-inf"), x_id - log_z)
    logprob = torch.where(z == 0, float("-inf"), logprob)
    return torch.where(ids < 0, 0.0, logprob), torch.where(z == 0, 0.0, entropy), log_z


def token_logprobs_reference(logits, ids, n_top=0, temperature=None):
    x = logits.float()
    top = x.amax(-1, keepdim=True) if x.numel() else x[:, :1]
    top = torch.where(torch.isnan(x), float("-inf"), x).amax(-1, keepdim=True) if bool(torch.isnan(top).any()) else top
    d = x - torch.where(top == float("-inf"), 0.0, top)
    if temperature is not None:
        d = d / torch.where(temperature > 0, temperature.float(), 1.0)[:, None]
    at = ids.clamp(0, x.shape[1] - 1)[:, None]
    logprob, entropy, log_z = _results(d, d.gather(1, at)[:, 0], ids, x.shape[1])
    if n_top == 0:
        return logprob, entropy, None, None
    order = torch.where(torch.isnan(x), float("-inf"), x)
    order = torch.sort(order, dim=-1, descending=True, stable=True)
    barred = order.values[:, :n_top] == float("-inf")
    i = order.indices[:, :n_top]
    lps = d.gather(1, i) - log_z[:, None]
    return (logprob, entropy, torch.where(barred, -1, i).to(torch.int32), torch.where(barred, float("-inf"), lps))


def _check_rows(x, ids, temperature, name):
    """Refuses what no kernel reads; returns (rows, columns, device)."""
    dev = x.device
    if x.dim() != 2 or x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError(f"{name}: rows [rows, columns] with adjacent columns expected, got {tuple(x.shape)} strides {x.stride()}")
    n, columns = x.shape
    if n > MAX_ROWS:
        raise ValueError(f"{name}: at most {MAX_ROWS} rows, got {n}")
    if columns > MAX_COLUMNS:
        raise ValueError(f"{name}: at most {MAX_COLUMNS} columns, got {columns}")
    if ids.dtype is not torch.int64 or ids.shape != (n,) or ids.device != dev:
        raise TypeError(f"{name}: ids are int64 [{n}] on {dev}, got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
    if temperature is not None and (temperature.dtype is not torch.float32 or temperature.shape != (n,) or temperature.device != dev):
        raise TypeError(f"{name}: temperatures are fp32 [{n}] on {dev}")
    return n, columns, dev


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def token_logprobs(logits, ids, n_top=0, temperature=None):
    """logits [rows, vocab] (bf16 or fp32; other floating types are converted to fp32), rows at any stride; ids int64 [rows]; temperature fp32
    [rows] or None.  Returns (logprob fp32 [rows], entropy fp32 [rows], alternatives int32 [rows, n_top], their
    log-probabilities fp32 [rows, n_top]); the alternatives are the n_top largest logits, largest first, ties to the lowest index, -1 and
    -inf where the row has no more tokens above -inf, and None without n_top.  The sums' order, and with it a result's last bits, depends
    on how many rows there are and how they lie in memory."""
    rows, vocab, dev = _check_rows(logits, ids, temperature, "token_logprobs")
    if vocab < 1 or not 0 <= n_top <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: 0 to {min(MAX_TOP, vocab)} alternatives of a vocabulary of {vocab}, asked for {n_top}")
    if _debug.enabled():
        _debug.check_range(ids, 0, vocab, "token_logprobs ids", allow_negative_skip=True)
    index = dev.index
    dt = 0 if logits.dtype is torch.bfloat16 else 1
    if dt == 1 and logits.dtype is not torch.float32:
        if not logits.is_floating_point():
            raise TypeError(f"token_logprobs: floating-point logits expected, got {logits.dtype}")
        logits = logits.float()
    if not logits.is_cuda:
        return token_logprobs_reference(logits, ids, n_top, temperature)
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return token_logprobs(logits, ids, n_top, temperature)
    ids, temperature = _dense(ids), _dense(temperature)
    lp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(lp)
    top = top_lp = None
    if n_top:
        top_lp = lp.new_empty((rows, n_top))
        top = torch.empty_like(top_lp, dtype=torch.int32)
    check(_lib.load().xllm_token_logprobs(ptr(logits), logits.stride(0), dt, rows, vocab, ptr(ids), ptr(temperature), int(n_top),
                                          ptr(lp), ptr(entropy), ptr(top), ptr(top_lp), stream_on(index)), "token_logprobs")
    _count()
    return lp, entropy, top, top_lp


def head_logprobs_reference(hidden, weight, ids, temperature=None):
    return token_logprobs_reference(hidden.float() @ weight.float().T, ids, 0, temperature)[:2]


def _stride(t):
    """Elements between rows; a single row has none of its own."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def head_supported(hidden, weight):
    """Whether `head_logprobs` takes these on CUDA: bf16, rows of 16-byte multiples that start on such a boundary."""
    return (hidden.is_cuda and hidden.dtype == weight.dtype == torch.bfloat16 and hidden.shape[1] % 8 == 0
            and not (_stride(hidden) | _stride(weight)) % 8 and not (hidden.data_ptr() | weight.data_ptr()) % 16)


@functools.lru_cache(maxsize=4096)
def _head_workspace(rows, vocab, width):
    return _lib.load().xllm_head_logprobs_workspace(rows, vocab, width)


def head_logprobs(hidden, weight, ids, temperature=None):
    """The log-probabilities and entropies of token_logprobs(hidden @ weight^T, ids) without the logits: hidden [rows, width]
    and weight [vocab, width] bf16, the products' sums fp32 and never rounded to bf16 (so not the bits of the two steps, which
    round every logit).  Returns (logprob, entropy) fp32 [rows].  A workspace of 16 bytes for each row and up to 256 tokens of
    the vocabulary is allocated.  On CUDA the width is a multiple of 8 and rows start on 16-byte boundaries.  Where a bounded wait of the
    kernel expires, all results of the call are NaN and `error_status` tells."""
    rows, width, dev = _check_rows(hidden, ids, temperature, "head_logprobs")
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[1] or weight.stride(-1) != 1 or weight.dtype != hidden.dtype \
            or weight.shape[0] < 1 or width < 1 or weight.device != hidden.device:
        raise ValueError(f"head_logprobs: weight [vocab, {hidden.shape[1]}] {hidden.dtype} on {hidden.device} expected, got "
                         f"{tuple(weight.shape)} {weight.dtype} on {weight.device}")
    vocab = weight.shape[0]
    if vocab > MAX_COLUMNS:
        raise ValueError(f"head_logprobs: a vocabulary of at most {MAX_COLUMNS} tokens, got {vocab}")
    if _debug.enabled():
        _debug.check_range(ids, 0, vocab, "head_logprobs ids", allow_negative_skip=True)
    if not hidden.is_cuda:
        return head_logprobs_reference(hidden, weight, ids, temperature)
    if not head_supported(hidden, weight):
        raise ValueError(f"head_logprobs: bf16 with a width in multiples of 8 and 16-byte aligned rows expected, got {hidden.dtype} "
                         f"{tuple(hidden.shape)} strides {hidden.stride()}, weight strides {weight.stride()}")
    index = dev.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return head_logprobs(hidden, weight, ids, temperature)
    ids, temperature = _dense(ids), _dense(temperature)
    if _stride(hidden) < width:                     # one row for all, or overlapping ones
        hidden = hidden.contiguous()
    if _stride(weight) < width:
        weight = weight.contiguous()
    lp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(lp)
    work = torch.empty(_head_workspace(rows, vocab, width), dtype=torch.uint8, device=dev)
    check(_lib.load().xllm_head_logprobs(ptr(hidden), _stride(hidden), ptr(weight), _stride(weight), rows, vocab, width, ptr(ids),
                                         ptr(temperature), ptr(work), ptr(lp), ptr(entropy), stream_on(index)), "head_logprobs")
    _count(2)
    return lp, entropy


_expired = 0           # what `expired` has read and `error_status` has not told yet


def expired() -> bool:
    """Whether a bounded wait inside `head_logprobs` expired; the next `error_status` tells it too."""
    global _expired
    _expired |= int(_lib.load().xllm_head_logprobs_error_status())
    return _expired != 0


def error_status() -> int:
    """Non-zero when a bounded wait inside `head_logprobs` expired since the last query."""
    global _expired
    v, _expired = _expired | int(_lib.load().xllm_head_logprobs_error_status()), 0
    return v
