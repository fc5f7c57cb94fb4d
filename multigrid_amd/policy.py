"""What stands between the simulator and a policy network, as launches of the HIP library.

An environment shows cells (``image``: type, colour and state of every cell of a view) and a mission text; a policy
answers with logits.  Here the one becomes the input of a dense layer and the other an action:

* ``embed`` - rows of a table by cell or by token, with scaling; its gradient is summed by token (``embed_grad``);
* ``adjust_logits`` - penalties for what was answered before, a bias, a mask of what may be answered;
* ``draw`` - an answer from logits and a uniform number of the caller's;
* ``token_logprobs`` - log-probabilities and entropies of answers, what a policy gradient trains on.

``embed``, ``adjust_logits`` and ``token_logprobs`` are differentiable, once and backwards: a tangent of forward-mode
differentiation is refused (NotImplementedError).  Every call is enqueued on the current stream of its tensors' device,
waits for nothing and may be captured into a HIP graph; tensors may have any strides, and a last dimension that is not
adjacent in memory is copied.  What a backward pass reads again (``logits``, ``history``, ``lengths``, ``mask``, ``tokens``)
must hold the same values until then; ``ids`` may change, a copy is kept (the simulator writes its images in place).
float32, bfloat16 and float16; sums are held in 32 bits or more and rounded once.

Arguments that do not fit raise ValueError, what the library itself refuses ``_lib.MgError`` (a RuntimeError; out of a backward
pass it comes as a plain RuntimeError with the same text).

A backward pass that is captured must not meet a leaf that an eager graph of the default stream still holds: the leaf's
gradient would be accumulated on that stream, which ends the process.  A differentiable call under capture looks for such
a leaf and raises RuntimeError; ``embed_grad`` is the table's gradient without autograd.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib

CELL_FIELDS = (11, 6, 7)  # rows of a cell's type, colour and state: the planes of multigrid/wrappers.py:95

_ENTRIES = ("mg_last_error", "mg_embed", "mg_embed_grad_workspace", "mg_embed_grad", "mg_adjust_logits",
            "mg_adjust_logits_grad", "mg_draw_workspace", "mg_draw", "mg_token_logprobs_workspace", "mg_token_logprobs",
            "mg_token_logprobs_grad")
_bound = None


def _native():
    """The torch side of the library (csrc/policy_torch.cpp), with the C entry points handed to it."""
    global _bound
    if _bound is None:
        lib = _lib.lib()
        try:
            from . import _policy_torch
        except ImportError as e:
            raise RuntimeError(f"{_lib.TORCH_LIB_PATH} is missing or does not load ({e}): build it with `python -c 'import "
                               "__graft_entry__ as g; g.build()'`") from e
        _policy_torch.bind([ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES], _lib.MgError)
        _bound = _policy_torch
    return _bound


def embed(ids: torch.Tensor, table: torch.Tensor, *, fields: Optional[Sequence[int]] = None, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` in the table's type: ``ids`` ``[...]`` of whole numbers, ``table`` ``[rows, dim]`` -> ``[..., dim]``.

    With ``fields`` (how many rows belong to each field, in order) ``ids`` is ``[..., len(fields)]`` and a token's rows are
    added up: ``embed(image, table, fields=CELL_FIELDS)`` is the one-hot image times the table, without the one-hot image.
    An id below 0 or beyond its field's rows reads nothing and passes no gradient, so it serves as padding."""
    return (_bound or _native()).embed(ids, table, fields, scale)


def embed_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, *, fields: Optional[Sequence[int]] = None,
               scale: float = 1.0) -> torch.Tensor:
    """The gradient ``[rows, dim]`` of ``embed``'s table for the gradient ``grad`` ``[..., dim]`` of its output, summed by
    token in an order that depends on the shapes and ids alone, in ``grad``'s type.  Not differentiable."""
    return (_bound or _native()).embed_grad(grad, ids, rows, fields, scale)


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  repetition=1.0, presence=0.0, frequency=0.0, bias: Optional[torch.Tensor] = None,
                  mask: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits ``[..., k]`` as an answer is to be drawn from them, in their own type.

    ``history`` ``[..., t]`` (or ``[t]`` for all rows): what was answered before, whole numbers; of row i the first
    ``lengths[i]`` count (all without ``lengths``), entries outside 0 .. k - 1 do not.  A token that stands there c > 0 times
    has its logit x made ``x * (1 / repetition)`` where positive and ``x * repetition`` elsewhere, less ``presence``, less
    ``frequency * c``; each of the three is a number or a tensor of one per row, ``repetition`` positive.  ``bias`` ``[k]`` or ``[..., k]`` is added.
    ``mask`` says what may be answered - ``bool`` / ``uint8`` ``[k]`` or ``[..., k]``, or one bit per token in ``int32``
    ``[ceil(k / 32)]`` or ``[..., ceil(k / 32)]``, lowest bit first; everything else becomes -inf, also all of a row.

    Differentiable with respect to the logits.  ``out`` (contiguous, may be the logits) is written instead of a new
    tensor, then nothing is differentiable; a backward pass that has kept ``out``'s old values raises RuntimeError, as after
    torch's own operations in place (the replay of a captured graph writes uncounted)."""
    return (_bound or _native()).adjust_logits(logits, history, lengths, repetition, presence, frequency, bias, mask, out)


def draw(logits: torch.Tensor, uniforms: Optional[torch.Tensor] = None, *, temperature=1.0,
         dtype: torch.dtype = torch.int64):
    """One token of every row of ``logits`` ``[..., k]`` and its log-probability (float32): ``([...], [...])``.

    ``uniforms`` ``[...]`` in [0, 1), float32 or float64: the lowest token up to which the probabilities add up to more
    than it, worked out in 64 bits.  Without: the lowest token of the largest logit.  ``temperature`` is a number or a
    tensor of one per row.  A row that is no distribution - everything -inf, a NaN, +inf, no positive temperature - gives
    token -1 (255 in uint8) and log-probability -inf or NaN.  ``dtype`` of the tokens: int64, int32, or uint8 for up to 255 tokens, which is what
    ``step`` takes as actions (255 is no action).  Not differentiable: ``token_logprobs`` is."""
    return (_bound or _native()).draw(logits, uniforms, temperature, dtype)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature=1.0):
    """Log-probability of ``tokens`` ``[...]`` (int64, int32, or uint8 for up to 255 tokens) under ``logits`` ``[..., k]``, and
    the entropy of every row: two float32 tensors ``[...]``, both differentiable with respect to the logits.  A token outside
    0 .. k - 1 is ignored: its log-probability is 0 and passes no gradient.  -inf logits (what ``adjust_logits`` bars) have probability 0 and
    gradient 0; a row of nothing else has log-probability -inf, entropy 0 and no gradient.  ``temperature`` is a number
    or a tensor of one per row (a row whose number is no temperature - below 2^-126, infinite or NaN - gives NaN); it passes
    no gradient."""
    return (_bound or _native()).token_logprobs(logits, tokens, temperature)
