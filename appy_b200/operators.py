"""Language-model operators on arrays, beside the annotated loops: embedding lookup and its gradient, the gated
linear recurrence and its gradient, log probabilities of given tokens with entropy and top alternatives and their
gradient.  They are what three kinds of loops would say that the loop lowering refuses: a parallel store whose row
repeats, a scalar carried from one iteration to the next, and a reduction over (value, index) pairs.

Every function launches prebuilt kernels of libappy_sm100 (include/appy_sm100.h) on torch's current stream of the
arguments' device and returns without waiting.  Arguments are torch CUDA tensors, used in place; if the first one is
a NumPy array or a CPU tensor, all host arrays are uploaded, and results come back as the first argument's kind, or in
the arrays given for them, as with annotated loops.  Element types are float32, float16 and bfloat16; arithmetic is float32, a result is rounded
once.  Token and offset arrays are int32 or int64.  Inputs may have any strides (a layout that the kernels do not read
in place, such as a transposed last dimension, is copied first); arrays that are written need a unit last stride.

Gradients are functions of their own: nothing is recorded for autograd; a tensor that requires grad is refused while
grad mode is on, and one that carries a forward-mode tangent.  A ``torch.autograd.Function`` whose ``forward`` calls
``f`` and whose ``backward`` calls ``f_grad`` puts an operator into a graph.  Calls may be captured into CUDA graphs,
gradients included, once each kind of call has run outside of one (kernels are loaded with their first call).  An array
that is written must not overlap an argument, unless it says so.
"""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

import numpy as np
import torch
from torch.autograd import forward_ad

from .backends.cuda_sm100 import runtime as rt

__all__ = ["embedding", "embedding_grad", "gated_scan", "gated_scan_grad", "token_logprobs", "token_logprobs_grad", "LogProbs"]

_FLOATS = {torch.float32: 0, torch.float16: 4, torch.bfloat16: 5}      # the codes of include/appy_sm100.h
_INTS = {torch.int32: 2, torch.int64: 3}

LogProbs = namedtuple("LogProbs", "logprobs entropy stats top_logprobs top_tokens")
LogProbs.__doc__ = "Result of token_logprobs; `stats` is for token_logprobs_grad, the last two are None unless `top` is given."


# ------------------------------------------------------------------------------------------------ arguments

def _is_host(a) -> bool:
    return not (isinstance(a, torch.Tensor) and a.is_cuda)


def _touch(h):
    """A host array was written here: loops that keep it on the device upload it again."""
    from .backends.cuda_sm100 import codegen
    if isinstance(h, np.ndarray):
        codegen.touch_bytes(*np.lib.array_utils.byte_bounds(h))
    else:
        lo = h.untyped_storage().data_ptr()
        codegen.touch_bytes(lo, lo + h.untyped_storage().nbytes())


def _through_host(fn, args, kwargs):
    """Run `fn` on uploaded copies of host arguments and bring results (and written arguments) back."""
    from . import to_gpu

    def up(a):
        if isinstance(a, np.ndarray):
            return to_gpu(a).view(a.shape)         # which hands a single number back as an array of one
        return to_gpu(a) if isinstance(a, torch.Tensor) and not a.is_cuda else a

    def up_any(a):
        return tuple(up(x) for x in a) if isinstance(a, (tuple, list)) else up(a)

    first = args[0]
    if not isinstance(first, (np.ndarray, torch.Tensor)):
        raise TypeError(f"{fn.__name__}: expected a NumPy array or a torch tensor, got {type(first).__name__}")
    for name in ("out", "last"):
        given = kwargs.get(name)
        for h in given if isinstance(given, (tuple, list)) else (given,):
            if isinstance(h, np.ndarray) and not h.flags.writeable:
                raise ValueError(f"{name} is read-only")
    dev_args, dev_kwargs = [up(a) for a in args], {k: up_any(a) for k, a in kwargs.items()}
    result = fn(*dev_args, **dev_kwargs)
    written = {}                                   # device tensor -> the array that the caller gave for it
    for name in ("out", "last"):
        given, dev = kwargs.get(name), dev_kwargs.get(name)
        pairs = zip(given, dev) if isinstance(given, (tuple, list)) else ((given, dev),)
        for h, d in pairs:
            if h is None:
                continue
            if h is not d:
                if isinstance(h, np.ndarray):
                    np.copyto(h, d.cpu().numpy())
                else:
                    h.copy_(d)
                _touch(h)
            written[id(d)] = h

    def down(t):
        if not isinstance(t, torch.Tensor):
            return t
        if id(t) in written:
            return written[id(t)]
        return t.cpu().numpy() if isinstance(first, np.ndarray) else t.cpu()

    if isinstance(result, tuple):
        return type(result)(*map(down, result)) if hasattr(result, "_fields") else tuple(map(down, result))
    return down(result)


def _fail(fn, what):
    raise ValueError(f"{fn}: {what}")


def _floats(fn, name, t):
    if type(t) is not torch.Tensor and not isinstance(t, torch.Tensor):
        raise TypeError(f"{fn}: {name} must be a torch CUDA tensor like the first argument, got {type(t).__name__}")
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{fn}: {name} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def _ints(fn, name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{fn}: {name} must be a torch CUDA tensor like the first argument, got {type(t).__name__}")
    code = _INTS.get(t.dtype)
    if code is None:
        raise TypeError(f"{fn}: {name} must be int32 or int64, got {t.dtype}")
    return code


def _together(fn, first, *others):
    """All on the device of `first`, none of them part of an autograd graph, backwards or forwards."""
    device = first.device
    grad = torch.is_grad_enabled()
    if grad and first.requires_grad:
        _no_graph(fn)
    for t in others:
        if t is None:
            continue
        if t.device != device:
            _fail(fn, f"arguments are on {device} and {t.device}")
        if grad and t.requires_grad:
            _no_graph(fn)
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in (first, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{fn}: an argument carries a forward-mode tangent, but autograd does not see this operator: "
                                   "call it on primal values, or inside a torch.autograd.Function that has a jvp")
    return device.index


def _no_graph(fn):
    raise RuntimeError(f"{fn}: an argument requires grad, but nothing is recorded for autograd here: call it under "
                       "torch.no_grad() or inside a torch.autograd.Function, and use the operator's _grad function")


def _row_stride(t):
    """Elements from one row to the next if the rows of all leading dimensions are evenly spaced, else None."""
    width = t.shape[-1]
    if t.is_contiguous():
        return width
    if width > 1 and t.stride(-1) != 1:
        return None
    step = None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step, span = stride, stride * size
        elif stride != span:
            return None
        else:
            span = stride * size
    if step is None:
        return width
    return step if step >= width else None


def _rows_in(t):
    step = _row_stride(t)
    return (t, step) if step is not None else (t.contiguous(), t.shape[-1])


def _rows_out(fn, name, t, shape, dtype):
    _like(fn, name, t, shape, dtype)
    step = _row_stride(t)
    if step is None:
        _fail(fn, f"{name} needs a unit last stride and evenly spaced, separate rows")
    return step


def _like(fn, name, t, shape, dtype):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{fn}: {name} must be a torch CUDA tensor like the first argument, got {type(t).__name__}")
    if t.shape != shape or t.dtype != dtype:
        _fail(fn, f"{name} must be {dtype} of shape {tuple(shape)}, got {t.dtype} of {tuple(t.shape)}")


_entries: dict = {}
_one_device = None


def _entry(name):
    """The C function `name`; the library's own set-up of the device comes with the first."""
    global _one_device
    if _one_device is None:
        _one_device = torch.cuda.device_count() == 1
        rt.init(torch.cuda.current_device())
    fn = _entries[name] = getattr(rt.lib(), name)
    return fn


def _run(entry, device, *args):
    """Call the C entry on torch's current stream of `device`."""
    if torch._C._cuda_getDevice() != device:
        with torch.cuda.device(device):
            return _run(entry, device, *args)
    fn = _entries.get(entry) or _entry(entry)
    if not _one_device:
        rt.init(device)                            # with several, the library's idea of the current one follows torch's
    if fn(*args, torch._C._cuda_getCurrentRawStream(device)):
        rt.check(-1)


# ------------------------------------------------------------------------------------------------ embedding

def embedding(weight, tokens, scale=1.0, out=None):
    """``out[..., :] = scale * weight[tokens[...], :]``; a token outside the rows of `weight` gives zeros.

    weight: [rows, width]; tokens: any shape, int32 or int64.  Returns `out`, [*tokens.shape, width] of weight's type.
    """
    fn = "embedding"
    if _is_host(weight):
        return _through_host(embedding, (weight, tokens), {"scale": scale, "out": out})
    code, int_code = _floats(fn, "weight", weight), _ints(fn, "tokens", tokens)
    if weight.dim() != 2:
        _fail(fn, f"weight must have two dimensions, got {weight.dim()}")
    device = _together(fn, weight, tokens, out)
    rows, width = weight.shape
    weight, ldw = _rows_in(weight)
    tokens = tokens.contiguous()
    shape = tokens.shape + (width,)
    if out is None:
        out, ldo = torch.empty(shape, dtype=weight.dtype, device=weight.device), width
    else:
        ldo = _rows_out(fn, "out", out, shape, weight.dtype)
    _run("appy_embedding", device, weight.data_ptr(), code, ldw, rows, width, tokens.data_ptr(), int_code, tokens.numel(),
         float(scale), out.data_ptr(), ldo)
    return out


_grad_bytes: dict = {}


def _embedding_grad_bytes(n, rows, width):
    known = _grad_bytes.get((n, rows, width))
    if known is None:
        size = C.c_size_t()
        rt.check(rt.lib().appy_embedding_grad_bytes(n, rows, width, C.byref(size)))
        if len(_grad_bytes) >= 1024:
            _grad_bytes.clear()
        known = _grad_bytes[n, rows, width] = size.value
    return known


def embedding_grad(grad, tokens, rows=None, scale=1.0, out=None, accumulate=False):
    """Gradient of ``embedding`` with respect to its weight: row v is ``scale`` times the sum of grad's rows whose
    token is v, added up in float32 in the order of the positions, whatever the schedule.

    grad: [*tokens.shape, width].  rows: number of rows of the weight, needed unless `out` is given.  out: [rows, width]
    of grad's type or float32; with ``accumulate=True`` the gradient is added to it and rows without tokens are not
    touched, else every row is written.  Tokens outside [0, rows) are dropped.
    """
    fn = "embedding_grad"
    if _is_host(grad):
        return _through_host(embedding_grad, (grad, tokens, rows), {"scale": scale, "out": out, "accumulate": accumulate})
    code, int_code = _floats(fn, "grad", grad), _ints(fn, "tokens", tokens)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape:
        _fail(fn, f"grad must have the shape of tokens and one more dimension, got {tuple(grad.shape)} for {tuple(tokens.shape)}")
    device = _together(fn, grad, tokens, out)
    width = grad.shape[-1]
    if out is None:
        if rows is None:
            _fail(fn, "rows or out is needed")
        if accumulate:
            _fail(fn, "accumulate needs out")
        out, ldo = torch.empty((rows, width), dtype=grad.dtype, device=grad.device), width
    else:
        if rows is None:
            rows = out.shape[0]
        ldo = _rows_out(fn, "out", out, (rows, width), torch.float32 if out.dtype == torch.float32 else grad.dtype)
    grad, ldg = _rows_in(grad)
    tokens = tokens.contiguous()
    n = tokens.numel()
    workspace = torch.empty(_embedding_grad_bytes(n, rows, width), dtype=torch.uint8, device=grad.device)
    _run("appy_embedding_grad", device, grad.data_ptr(), code, ldg, tokens.data_ptr(), int_code, n, rows, width, float(scale), bool(accumulate),
         out.data_ptr(), _FLOATS[out.dtype], ldo, workspace.data_ptr(), workspace.numel())
    return out


# ------------------------------------------------------------------------------------------------ gated recurrence

def _sequences(fn, x, offsets):
    """(sequences, tokens, shape of a state, offsets, their type) of a dense [batch, tokens, width] or packed
    [tokens, width] array."""
    if offsets is None:
        if x.dim() != 3:
            _fail(fn, f"x must be [batch, tokens, width], or [tokens, width] with offsets; got {x.dim()} dimensions")
        return x.shape[0], x.shape[1], None, 2
    code = _ints(fn, "offsets", offsets)
    if x.dim() != 2:
        _fail(fn, f"with offsets, x must be [tokens, width]; got {x.dim()} dimensions")
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        _fail(fn, "offsets must have one dimension and sequences + 1 entries")
    return offsets.shape[0] - 1, x.shape[0], offsets.contiguous(), code


def _scan_in(fn, name, t, x):
    if t is not x:
        _like(fn, name, t, x.shape, x.dtype)
    if t.is_contiguous():
        return t
    strides = [stride for stride, size in zip(t.stride(), t.shape) if size > 1]
    return t.contiguous() if 0 in strides or (t.shape[-1] > 1 and t.stride(-1) != 1) else t


def _scan_out(fn, name, t, x):
    _like(fn, name, t, x.shape, x.dtype)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _fail(fn, f"{name} needs a unit last stride")
    # two elements at one address would be written by different threads
    dims = sorted((stride, size) for stride, size in zip(t.stride(), t.shape) if size > 1)
    span = 1
    for stride, size in dims:
        if stride < span:
            _fail(fn, f"elements of {name} overlap")
        span = stride * (size - 1) + span
    return t


def _strided(t):
    return (t.data_ptr(), t.stride(0), t.stride(1)) if t.dim() == 3 else (t.data_ptr(), 0, t.stride(0))


def _state(fn, name, t, shape):
    if t is None:
        return None
    _like(fn, name, t, shape, torch.float32)
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def gated_scan(x, gate, initial=None, offsets=None, out=None, last=None):
    """Gated linear recurrence: ``h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t]`` with ``f = sigmoid(gate)``, each channel for
    itself.  Returns (h, last): all states, of x's type, and the state behind each sequence's last token, float32.

    x, gate: [batch, tokens, width]; or, with `offsets` (sequences + 1 positions, not decreasing), packed [tokens, width],
    where sequence s is rows offsets[s] to offsets[s+1].  An empty sequence keeps its initial state.  Rows of no sequence
    become zero, or are left as they are where `out` is given.  initial: float32 [sequences, width], zeros if None.
    `last` may be given, and may be `initial`, which then moves on in place: the step of a serving loop is a call with
    one token.
    """
    fn = "gated_scan"
    if _is_host(x):
        return _through_host(gated_scan, (x, gate), {"initial": initial, "offsets": offsets, "out": out, "last": last})
    code = _floats(fn, "x", x)
    sequences, tokens, offsets, int_code = _sequences(fn, x, offsets)
    shape = (sequences, x.shape[-1])
    x, gate = _scan_in(fn, "x", x, x), _scan_in(fn, "gate", gate, x)
    initial = _state(fn, "initial", initial, shape)
    fill = out is None
    if fill:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _scan_out(fn, "out", out, x)
    if last is None:
        last = torch.empty(shape, dtype=torch.float32, device=x.device)
    else:
        _like(fn, "last", last, shape, torch.float32)
        if not last.is_contiguous():
            _fail(fn, "last must be contiguous")
    device = _together(fn, x, gate, initial, offsets, out, last)
    _run("appy_gated_scan", device, *_strided(x), *_strided(gate), code, _ptr(offsets), int_code, sequences, tokens, x.shape[-1],
         _ptr(initial), *_strided(out), last.data_ptr(), fill)
    return out, last


def gated_scan_grad(grad, x, gate, h, initial=None, offsets=None, grad_last=None, out=None):
    """Gradients of ``gated_scan`` with respect to (x, gate, initial), given those with respect to its results.

    grad: gradient of h, or None; h: the states that gated_scan returned, of x's type (the gradient of gate takes h[t-1] - x[t]
    from them, so in 16 bits it has their rounding beside its own); x, gate, initial, offsets: as given to it;
    grad_last: gradient of the last states, float32, or None.  out: a pair of arrays for the gradients of x and gate
    (slices of one array, for instance).  The gradient of `initial` is float32 and returned even where it was None.
    """
    fn = "gated_scan_grad"
    if _is_host(x):
        if not isinstance(x, (np.ndarray, torch.Tensor)):
            raise TypeError(f"{fn}: expected a NumPy array or a torch tensor for x, got {type(x).__name__}")
        return _through_host(lambda x, *a, **k: gated_scan_grad(a[0], x, *a[1:], **k), (x, grad, gate, h),
                             {"initial": initial, "offsets": offsets, "grad_last": grad_last, "out": out})
    code = _floats(fn, "x", x)
    sequences, tokens, offsets, int_code = _sequences(fn, x, offsets)
    shape = (sequences, x.shape[-1])
    x, gate, h = _scan_in(fn, "x", x, x), _scan_in(fn, "gate", gate, x), _scan_in(fn, "h", h, x)
    if grad is not None:
        grad = _scan_in(fn, "grad", grad, x)
    initial, grad_last = _state(fn, "initial", initial, shape), _state(fn, "grad_last", grad_last, shape)
    fill = out is None
    if fill:
        dx, dgate = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        dx, dgate = out
        _scan_out(fn, "out[0]", dx, x)
        _scan_out(fn, "out[1]", dgate, x)
    dinitial = torch.empty(shape, dtype=torch.float32, device=x.device)
    device = _together(fn, x, gate, h, grad, initial, offsets, grad_last, dx, dgate)
    _run("appy_gated_scan_grad", device, *(_strided(grad) if grad is not None else (None, 0, 0)), *_strided(x), *_strided(gate), *_strided(h),
         code, _ptr(offsets), int_code, sequences, tokens, x.shape[-1], _ptr(initial), _ptr(grad_last), *_strided(dx), *_strided(dgate),
         dinitial.data_ptr(), fill)
    return dx, dgate, dinitial


# ------------------------------------------------------------------------------------------------ log probabilities

def _check_rows(fn, logits, tokens):
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        _fail(fn, f"logits must have the shape of tokens and one more dimension, got {tuple(logits.shape)} for {tuple(tokens.shape)}")
    if logits.shape[-1] < 1:
        _fail(fn, "a row of logits must have at least one entry")


def token_logprobs(logits, tokens, top=0, temperature=1.0):
    """Log probabilities of given tokens under ``softmax(logits / temperature)``, the entropy of each row, and its `top`
    (at most 32) most likely alternatives; equal logits are ordered by index.

    logits: [*tokens.shape, vocabulary].  Returns LogProbs(logprobs, entropy, stats, top_logprobs, top_tokens), float32
    ([..., top] for the last two; top_tokens of tokens' type).  A token outside the vocabulary (padding) has log probability
    0 and no gradient.  Logits of -inf are masked; a row with nothing else has log probability -inf, entropy 0, and no
    gradient.  A row with NaN or +inf gives NaN.
    """
    fn = "token_logprobs"
    if _is_host(logits):
        return _through_host(token_logprobs, (logits, tokens), {"top": top, "temperature": temperature})
    code, int_code = _floats(fn, "logits", logits), _ints(fn, "tokens", tokens)
    _check_rows(fn, logits, tokens)
    cols = logits.shape[-1]
    if not 0 <= top <= min(32, cols):
        _fail(fn, f"top must be in [0, {min(32, cols)}], got {top}")
    device = _together(fn, logits, tokens)
    logits, ld = _rows_in(logits)
    tokens = tokens.contiguous()
    shape, n = tokens.shape, tokens.numel()
    # arrays of their own: pieces of one allocation would be views, which autograd does not let a caller write in place
    logprobs = logits.new_empty(shape, dtype=torch.float32)
    entropy, stats = torch.empty_like(logprobs), logprobs.new_empty(shape + (3,))
    top_logprobs = top_tokens = None
    if top:
        top_logprobs, top_tokens = logprobs.new_empty(shape + (top,)), tokens.new_empty(shape + (top,))
    _run("appy_token_logprobs", device, logits.data_ptr(), code, ld, n, cols, tokens.data_ptr(), int_code, float(temperature), top,
         logprobs.data_ptr(), entropy.data_ptr(), stats.data_ptr(), _ptr(top_logprobs), _ptr(top_tokens))
    return LogProbs(logprobs, entropy, stats, top_logprobs, top_tokens)


def _per_row(fn, name, t, shape):
    """(array or None, stride) of one float32 per row; a broadcast scalar keeps its stride of 0."""
    if t is None:
        return None, 0
    _like(fn, name, t, shape, torch.float32)
    if t.is_contiguous():
        return t, 1
    if all(s == 0 or n == 1 for s, n in zip(t.stride(), t.shape)):
        return t, 0
    return t.contiguous(), 1


def token_logprobs_grad(logits, tokens, stats, grad_logprobs=None, grad_entropy=None, temperature=1.0, out=None):
    """Gradient of ``token_logprobs`` with respect to the logits, of their type, for the gradients of its logprobs and
    entropy (float32, or None; the top alternatives are answers and have none).  stats: as token_logprobs returned them for
    the same logits, tokens and temperature.  `out` may be `logits`, which is then overwritten.
    """
    fn = "token_logprobs_grad"
    if _is_host(logits):
        return _through_host(token_logprobs_grad, (logits, tokens, stats),
                             {"grad_logprobs": grad_logprobs, "grad_entropy": grad_entropy, "temperature": temperature, "out": out})
    code, int_code = _floats(fn, "logits", logits), _ints(fn, "tokens", tokens)
    _check_rows(fn, logits, tokens)
    _like(fn, "stats", stats, tokens.shape + (3,), torch.float32)
    g, g_stride = _per_row(fn, "grad_logprobs", grad_logprobs, tokens.shape)
    gh, gh_stride = _per_row(fn, "grad_entropy", grad_entropy, tokens.shape)
    device = _together(fn, logits, tokens, stats, g, gh, out)
    if out is None:
        out, ldo = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), logits.shape[-1]
    else:
        ldo = _rows_out(fn, "out", out, logits.shape, logits.dtype)
    logits, ld = _rows_in(logits)
    tokens, stats = tokens.contiguous(), stats.contiguous()
    _run("appy_token_logprobs_grad", device, logits.data_ptr(), code, ld, tokens.numel(), logits.shape[-1], tokens.data_ptr(), int_code,
         float(temperature), stats.data_ptr(), _ptr(g), g_stride, _ptr(gh), gh_stride, out.data_ptr(), ldo)
    return out
