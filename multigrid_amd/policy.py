"""What stands between the simulator and a policy network, as launches of the HIP library.

An environment shows cells (``image``: type, colour and state of every cell of a view) and a mission text; a policy
answers with logits.  Here the one becomes the input of a dense layer and the other an action:

* ``embed`` - rows of a table by cell or by token, with scaling; its gradient is summed by token (``embed_grad``);
* ``adjust_logits`` - penalties for what was answered before, a bias, a mask of what may be answered;
* ``draw`` - an answer from logits and a uniform number of the caller's;
* ``token_logprobs`` - log-probabilities and entropies of answers, what a policy gradient trains on.

``embed``, ``adjust_logits`` and ``token_logprobs`` are differentiable.  Every call is enqueued on the current stream of
its tensors' device, waits for nothing and may be captured into a HIP graph; tensors may have any strides, and a last
dimension that is not adjacent in memory is copied.  What a backward pass reads again (``history``, ``lengths``,
``mask``, ``tokens``) must hold the same values until then; ``ids`` may change, a copy is kept (the simulator writes
its images in place).  float32, bfloat16 and float16; sums are held in 32 bits or more and rounded once.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import MgAdjust, MgEmbed, MgLogits, check

CELL_FIELDS = (11, 6, 7)  # rows of a cell's type, colour and state: the planes of multigrid/wrappers.py:95

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_INTS = {torch.uint8: _lib.U8, torch.int32: _lib.I32, torch.int64: _lib.I64}
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _on:
    """The device made the current one where it is not already, and its current stream."""

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return ctypes.c_void_p(_RAW_STREAM(self.index) if _RAW_STREAM is not None else torch.cuda.current_stream(self.index).cuda_stream)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _on_gpu(name: str, t, device: Optional[torch.device] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU (there is no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors are on {device}")
    return t


def _floating(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _whole(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _INTS:
        raise ValueError(f"{name} must be uint8, int32 or int64, got {t.dtype}")
    return _INTS[t.dtype]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[..., k]`` as ``[n, k]`` with adjacent elements in a row; a view wherever there is one."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.shape[1] == 1 or t.stride(1) == 1 else t.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may share memory, by their first and last element."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
                          for t in (a, b))
    return a0 < b1 and b0 < a1


def _workspace(need: int, device: torch.device) -> Optional[torch.Tensor]:
    if need < 0:
        check(int(need))
    return torch.empty((need,), dtype=torch.uint8, device=device) if need else None


# ---- embedding -------------------------------------------------------------------------------------------------------


def _embed_spec(ids: torch.Tensor, fields: Optional[Sequence[int]], rows: int, dim: int, dtype: int, scale: float):
    """The descriptor of a lookup, the ids as ``[n, fields]`` and the tokens' shape."""
    if fields is None:
        sizes, shape = (rows,), tuple(ids.shape)
        ids = ids.reshape(-1, 1)
    else:
        sizes = tuple(int(f) for f in fields)
        if not 1 <= len(sizes) <= _lib.MAX_FIELDS or min(sizes) < 1 or sum(sizes) != rows:
            raise ValueError(f"fields {sizes} must be 1 to {_lib.MAX_FIELDS} positive numbers that add up to the {rows} rows of the table")
        if ids.dim() < 1 or ids.shape[-1] != len(sizes):
            raise ValueError(f"ids of shape {tuple(ids.shape)} must have {len(sizes)} fields in their last dimension")
        shape = tuple(ids.shape[:-1])
        ids = ids.reshape(-1, len(sizes))
    n = ids.shape[0]
    e = MgEmbed(n=n, fields=len(sizes), dim=dim, ids_type=_whole("ids", ids), dtype=dtype, ids_stride=ids.stride(0) if n > 1 else 0,
                field_stride=ids.stride(1), scale=scale)
    e.sizes[:len(sizes)] = sizes
    return e, ids, shape


def _embed_forward(ids, table, fields, scale):
    rows, dim = table.shape
    if table.stride(1) != 1 and dim > 1:
        table = table.contiguous()
    e, ids, shape = _embed_spec(ids, fields, rows, dim, _floating("table", table), scale)
    e.row_stride = table.stride(0) if rows > 1 else 0
    out = torch.empty(shape + (dim,), dtype=table.dtype, device=table.device)
    if out.numel():
        with _on(table.device) as stream:
            check(_lib.lib().mg_embed(ctypes.byref(e), _ptr(ids), _ptr(table), _ptr(out), stream))
    return out


def embed_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, *, fields: Optional[Sequence[int]] = None,
               scale: float = 1.0) -> torch.Tensor:
    """The gradient ``[rows, dim]`` of ``embed``'s table for the gradient ``grad`` ``[..., dim]`` of its output, summed by
    token in an order that depends on the shapes and ids alone, in ``grad``'s type."""
    _on_gpu("grad", grad)
    _on_gpu("ids", ids, grad.device)
    if grad.dim() < 1 or grad.shape[-1] < 1 or rows < 1:
        raise ValueError(f"grad of shape {tuple(grad.shape)} and {rows} rows: both must hold something")
    e, ids, shape = _embed_spec(ids, fields, int(rows), grad.shape[-1], _floating("grad", grad), float(scale))
    if tuple(grad.shape[:-1]) != shape:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, the ids are of shape {shape}")
    g = _rows(grad)
    e.row_stride = g.stride(0) if g.shape[0] > 1 else 0
    out = torch.empty((int(rows), grad.shape[-1]), dtype=grad.dtype, device=grad.device)
    with _on(grad.device) as stream:
        lib = _lib.lib()
        ws = _workspace(lib.mg_embed_grad_workspace(ctypes.byref(e)), grad.device)
        check(lib.mg_embed_grad(ctypes.byref(e), _ptr(ids), _ptr(g), _ptr(out), _ptr(ws), 0 if ws is None else ws.numel(), stream))
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, fields, scale):
        ctx.fields, ctx.scale, ctx.rows = fields, scale, table.shape[0]
        ctx.save_for_backward(ids.clone())
        return _embed_forward(ids, table, fields, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, embed_grad(grad, ids, ctx.rows, fields=ctx.fields, scale=ctx.scale), None, None


def embed(ids: torch.Tensor, table: torch.Tensor, *, fields: Optional[Sequence[int]] = None, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` in the table's type: ``ids`` ``[...]`` of whole numbers, ``table`` ``[rows, dim]`` -> ``[..., dim]``.

    With ``fields`` (how many rows belong to each field, in order) ``ids`` is ``[..., len(fields)]`` and a token's rows are
    added up: ``embed(image, table, fields=CELL_FIELDS)`` is the one-hot image times the table, without the one-hot image.
    An id below 0 or beyond its field's rows reads nothing and passes no gradient, so it serves as padding."""
    _on_gpu("table", table)
    _on_gpu("ids", ids, table.device)
    if table.dim() != 2 or not table.shape[0] or not table.shape[1]:
        raise ValueError(f"table must be [rows, dim] and hold something, got {tuple(table.shape)}")
    if table.requires_grad and torch.is_grad_enabled():
        return _Embed.apply(ids, table, fields, float(scale))
    return _embed_forward(ids, table, fields, float(scale))


# ---- adjustment of logits ----------------------------------------------------------------------------------------------


def _per_row(name: str, v, lead, device):
    """A number, or a float32 tensor ``[n]`` of one number per row: (tensor or None, number)."""
    if not isinstance(v, torch.Tensor):
        return None, float(v)
    _on_gpu(name, v, device)
    if v.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} passes no gradient: detach it")
    if v.dim() == 0:
        v = v.expand(lead)
    if tuple(v.shape) != tuple(lead):
        raise ValueError(f"{name} must be a number or of shape {tuple(lead)}, got {tuple(v.shape)}")
    return v.to(torch.float32).reshape(-1).contiguous(), 0.0


def _table(name: str, t: torch.Tensor, lead, width: int, device):
    """``[width]`` for every row, or ``[..., width]``: (2-D tensor, elements between rows)."""
    _on_gpu(name, t, device)
    if t.dim() == 1 and t.shape[0] == width:
        t = t.contiguous()
        return t, 0
    if tuple(t.shape) != tuple(lead) + (width,):
        raise ValueError(f"{name} must be of shape {(width,)} or {tuple(lead) + (width,)}, got {tuple(t.shape)}")
    t = _rows(t)
    return t, t.stride(0) if t.shape[0] > 1 else 0


def _adjust_spec(logits, history, lengths, repetition, presence, frequency, bias, mask):
    """The descriptor of an adjustment, and the tensors whose memory it names."""
    _on_gpu("logits", logits)
    dev, lead = logits.device, logits.shape[:-1]
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., k], got {tuple(logits.shape)}")
    k, n = logits.shape[-1], logits[..., 0].numel()
    a = MgAdjust(n=n, k=k, dtype=_floating("logits", logits))
    keep = []
    if history is not None:
        _whole("history", _on_gpu("history", history, dev))
        h, a.history_stride = _table("history", history, lead, history.shape[-1] if history.dim() else 0, dev)
        a.history_dev, a.history_type, a.t = (_ptr(h) if h.shape[-1] else None), _INTS[h.dtype], h.shape[-1]
        keep.append(h)
        if lengths is not None:
            _on_gpu("lengths", lengths, dev)
            if lengths.dtype not in (torch.int32, torch.int64) or tuple(lengths.shape) != tuple(lead):
                raise ValueError(f"lengths must be int32 or int64 of shape {tuple(lead)}, got {lengths.dtype} {tuple(lengths.shape)}")
            lengths = lengths.clamp(0, h.shape[-1]) if lengths.dtype == torch.int64 else lengths
            lengths = lengths.to(torch.int32).reshape(-1).contiguous()
            a.lengths_dev = _ptr(lengths)
            keep.append(lengths)
    elif lengths is not None:
        raise ValueError("lengths without a history")
    for name, v in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        t, number = _per_row(name, v, lead, dev)
        if t is None:
            setattr(a, name, number)
        else:
            setattr(a, name + "_dev", _ptr(t))
            keep.append(t)
    if bias is not None:
        if isinstance(bias, torch.Tensor) and bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("bias passes no gradient: add one that is trained to the logits")
        b, a.bias_stride = _table("bias", bias, lead, k, dev)
        b = b if b.dtype == torch.float32 else b.to(torch.float32)
        a.bias_stride = 0 if b.dim() == 1 or n <= 1 else b.stride(0)
        a.bias_dev = _ptr(b)
        keep.append(b)
    if mask is not None:
        _on_gpu("mask", mask, dev)
        if mask.dtype in (torch.bool, torch.uint8):
            a.mask_kind, width = _lib.MASK_BYTES, k
        elif mask.dtype == torch.int32:
            a.mask_kind, width = _lib.MASK_BITS, (k + 31) // 32
        else:
            raise ValueError(f"mask must be bool or uint8 (one for each token) or int32 (one bit for each token), got {mask.dtype}")
        m, a.mask_stride = _table("mask", mask, lead, width, dev)
        a.mask_dev = _ptr(m)
        keep.append(m)
    return a, keep


def _adjust_forward(logits, out, *more):
    a, keep = _adjust_spec(logits, *more)
    x = _rows(logits)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    a.logits_stride, a.out_stride = x.stride(0), a.k if a.n <= 1 or out.dim() < 2 else out.reshape(-1, a.k).stride(0)
    if a.n:
        with _on(logits.device) as stream:
            check(_lib.lib().mg_adjust_logits(ctypes.byref(a), _ptr(x), _ptr(out), stream))
    return out


class _Adjust(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, history, lengths, repetition, presence, frequency, bias, mask):
        tensors = (logits, history, lengths, repetition, mask)
        ctx.save_for_backward(*(t if isinstance(t, torch.Tensor) else None for t in tensors))
        ctx.repetition = None if isinstance(repetition, torch.Tensor) else repetition
        return _adjust_forward(logits, None, history, lengths, repetition, presence, frequency, bias, mask)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, history, lengths, repetition, mask = ctx.saved_tensors
        a, keep = _adjust_spec(logits, history, lengths, ctx.repetition if repetition is None else repetition, 0.0, 0.0, None, mask)
        x, g = _rows(logits), _rows(grad)
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a.logits_stride, a.grad_stride, a.out_stride = x.stride(0), g.stride(0), a.k
        if a.n:
            with _on(logits.device) as stream:
                check(_lib.lib().mg_adjust_logits_grad(ctypes.byref(a), _ptr(x), _ptr(g), _ptr(out), stream))
        return (out,) + (None,) * 7


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  repetition=1.0, presence=0.0, frequency=0.0, bias: Optional[torch.Tensor] = None,
                  mask: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits ``[..., k]`` as an answer is to be drawn from them, in their own type.

    ``history`` ``[..., t]`` (or ``[t]`` for all rows): what was answered before, whole numbers; of row i the first
    ``lengths[i]`` count (all without ``lengths``), entries outside 0 .. k - 1 do not.  A token that stands there c > 0 times
    has its logit x made ``x / repetition`` where positive and ``x * repetition`` elsewhere, less ``presence``, less
    ``frequency * c``; each of the three is a number or a tensor of one per row.  ``bias`` ``[k]`` or ``[..., k]`` is added.
    ``mask`` says what may be answered - ``bool`` / ``uint8`` ``[k]`` or ``[..., k]``, or one bit per token in ``int32``
    ``[ceil(k / 32)]`` or ``[..., ceil(k / 32)]``, lowest bit first; everything else becomes -inf, also all of a row.

    Differentiable with respect to the logits.  ``out`` (contiguous, may be the logits) is written instead of a new
    tensor, then nothing is differentiable."""
    more = (history, lengths, repetition, presence, frequency, bias, mask)
    if out is not None:
        _on_gpu("logits", logits)
        if (logits.requires_grad or (isinstance(out, torch.Tensor) and out.requires_grad)) and torch.is_grad_enabled():
            raise ValueError("out is not differentiable: leave it out, or call under torch.no_grad()")
        _on_gpu("out", out, logits.device)
        if out.shape != logits.shape or out.dtype != logits.dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous, {logits.dtype} and of shape {tuple(logits.shape)}")
        if _overlap(out, logits) and not (out.data_ptr() == logits.data_ptr() and logits.is_contiguous()):
            raise ValueError("out may be the logits or lie beside them, not across them")
    elif isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return _Adjust.apply(logits, *more)
    return _adjust_forward(logits, out, *more)


# ---- draw ----------------------------------------------------------------------------------------------------------------


def _logits_spec(logits, temperature, tokens_type):
    _on_gpu("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., k], got {tuple(logits.shape)}")
    x = _rows(logits)
    t, number = _per_row("temperature", temperature, logits.shape[:-1], logits.device)
    l = MgLogits(n=x.shape[0], k=x.shape[1], dtype=_floating("logits", logits), stride=x.stride(0) if x.shape[0] > 1 else 0,
                 temperature_dev=_ptr(t), temperature=number, tokens_type=tokens_type)
    return l, x, t


def draw(logits: torch.Tensor, uniforms: Optional[torch.Tensor] = None, *, temperature=1.0,
         dtype: torch.dtype = torch.int64):
    """One token of every row of ``logits`` ``[..., k]`` and its log-probability (float32): ``([...], [...])``.

    ``uniforms`` ``[...]`` in [0, 1), float32 or float64: the lowest token up to which the probabilities add up to more
    than it, worked out in 64 bits.  Without: the lowest token of the largest logit.  ``temperature`` is a number or a
    tensor of one per row.  A row that is no distribution - everything -inf, a NaN, +inf - gives token -1 (255 in uint8)
    and log-probability -inf or NaN.  ``dtype`` of the tokens: int64, int32, or uint8 for up to 255 tokens, which is what
    ``step`` takes as actions (255 is no action).  Not differentiable: ``token_logprobs`` is."""
    if dtype not in _INTS:
        raise ValueError(f"tokens are uint8, int32 or int64, not {dtype}")
    l, x, t = _logits_spec(logits, temperature, _INTS[dtype])
    lead, dev = logits.shape[:-1], logits.device
    kind = 0
    if uniforms is not None:
        _on_gpu("uniforms", uniforms, dev)
        if uniforms.dtype not in (torch.float32, torch.float64) or uniforms.shape != lead:
            raise ValueError(f"uniforms must be float32 or float64 of shape {tuple(lead)}, got {uniforms.dtype} {tuple(uniforms.shape)}")
        kind = _lib.F64 if uniforms.dtype == torch.float64 else _lib.F32
        uniforms = uniforms.contiguous()
    tokens = torch.empty(lead, dtype=dtype, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev)
    with _on(dev) as stream:
        lib = _lib.lib()
        ws = _workspace(lib.mg_draw_workspace(ctypes.byref(l)), dev)
        check(lib.mg_draw(ctypes.byref(l), _ptr(x), _ptr(uniforms), kind, _ptr(tokens), _ptr(logprobs), _ptr(ws),
                          0 if ws is None else ws.numel(), stream))
    return tokens, logprobs


# ---- log-probabilities and entropies ---------------------------------------------------------------------------------------


def _logprobs_forward(logits, tokens, temperature, stats: bool):
    _whole("tokens", _on_gpu("tokens", tokens, logits.device))
    l, x, t = _logits_spec(logits, temperature, _INTS[tokens.dtype])
    lead, dev = logits.shape[:-1], logits.device
    if tokens.shape != lead:
        raise ValueError(f"tokens must be of shape {tuple(lead)}, got {tuple(tokens.shape)}")
    tokens = tokens.contiguous()
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev)
    entropies = torch.empty(lead, dtype=torch.float32, device=dev)
    kept = torch.empty((l.n, 4), dtype=torch.float32, device=dev) if stats and l.k > 32 else None
    with _on(dev) as stream:
        lib = _lib.lib()
        ws = _workspace(lib.mg_token_logprobs_workspace(ctypes.byref(l)), dev)
        check(lib.mg_token_logprobs(ctypes.byref(l), _ptr(x), _ptr(tokens), _ptr(logprobs), _ptr(entropies), _ptr(kept), _ptr(ws),
                                    0 if ws is None else ws.numel(), stream))
    return logprobs, entropies, kept


def _strided(g: Optional[torch.Tensor]):
    """A gradient of one number per row as the kernel reads it: (tensor, elements between rows)."""
    if g is None:
        return None, 0
    g = g if g.dtype == torch.float32 else g.float()
    if g.dim() != 1:
        g = g.reshape(-1)
    return g, g.stride(0) if g.shape[0] > 1 else 0


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        logprobs, entropies, stats = _logprobs_forward(logits, tokens, temperature, True)
        ctx.number = None if isinstance(temperature, torch.Tensor) else temperature
        ctx.save_for_backward(logits, tokens, temperature if ctx.number is None else None, stats)
        ctx.set_materialize_grads(False)
        return logprobs, entropies

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprobs, grad_entropies):
        logits, tokens, temperature, stats = ctx.saved_tensors
        l, x, t = _logits_spec(logits, ctx.number if temperature is None else temperature, _INTS[tokens.dtype])
        tokens = tokens.contiguous()
        (g, gs), (h, hs) = _strided(grad_logprobs), _strided(grad_entropies)
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with _on(logits.device) as stream:
            check(_lib.lib().mg_token_logprobs_grad(ctypes.byref(l), _ptr(x), _ptr(tokens), _ptr(stats), _ptr(g), gs, _ptr(h), hs,
                                                    _ptr(out), stream))
        return out, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature=1.0):
    """Log-probability of ``tokens`` ``[...]`` (whole numbers) under ``logits`` ``[..., k]``, and the entropy of every row:
    two float32 tensors ``[...]``, both differentiable with respect to the logits.  A token outside 0 .. k - 1 is ignored: its
    log-probability is 0 and passes no gradient.  -inf logits (what ``adjust_logits`` bars) have probability 0 and
    gradient 0; a row of nothing else has log-probability -inf, entropy 0 and no gradient.  ``temperature`` is a number
    or a tensor of one per row; it passes no gradient."""
    _on_gpu("logits", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Logprobs.apply(logits, tokens, temperature)
    return _logprobs_forward(logits, tokens, temperature, False)[:2]
