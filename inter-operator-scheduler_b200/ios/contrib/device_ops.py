"""
Operators on device tensors: a mixture-of-experts layer and its 8-bit products.

Unlike the graph entry points, which take host arrays, these take tensors that already live on a GPU (``torch.Tensor``)
and return tensors on the same device.  The work goes to torch's current stream of that device and is not waited for;
the calls may be captured into CUDA graphs.  They compute no gradients and refuse tensors that ask for one.

A layer, from its router logits to its output::

    plan = ios_runtime.route_experts(logits, k)
    h = ios_runtime.grouped_matmul(x, w_in, plan.offsets, rows=plan.rows, act='silu', gated=True)
    y = ios_runtime.grouped_matmul(h, w_out, plan.offsets)
    out = ios_runtime.combine_experts(y, plan.gates, plan.slots)

See ``include/ios_runtime.h`` for the formulas.  (The reference has no counterpart: its operators are those of
convolution networks.)
"""
import ctypes
from collections import namedtuple

_ACTS = {'identity': 0, 'relu': 1, 'sigmoid': 2, 'tanh': 3, 'silu': 4}

Routing = namedtuple('Routing', ['experts', 'gates', 'offsets', 'rows', 'slots'])

_INT, _LONG, _PTR, _SIZE = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_size_t


def declare(handle):
    """Argument types of this module's entry points; called by the library loader."""
    handle.ios_route_experts_workspace.argtypes = [_INT, _INT, ctypes.POINTER(_SIZE)]
    handle.ios_route_experts.argtypes = [_PTR, _INT, _INT, _INT, _LONG, _INT, _INT] + [_PTR] * 6 + [_SIZE, _PTR]
    handle.ios_grouped_matmul.argtypes = [_PTR, _INT, _LONG, _LONG, _PTR, _INT, _INT, _INT, _LONG, _LONG, _PTR, _PTR, _INT,
                                          _PTR, _PTR, _PTR, _INT, _INT, _PTR, _INT, _LONG, _PTR]
    handle.ios_matmul_int8.argtypes = [_PTR, _LONG, _PTR, _LONG, _INT, _INT, _INT, _PTR, _PTR, _PTR, _INT, _PTR, _INT,
                                       _LONG, _PTR]
    handle.ios_quantize_rows.argtypes = [_PTR, _INT, _LONG, _LONG, _INT, _PTR, _LONG, _PTR, _LONG, _PTR, _PTR]
    handle.ios_device_ops_status.argtypes = [_INT, _PTR]
    handle.ios_combine_experts.argtypes = [_PTR, _INT, _LONG, _LONG, _PTR, _PTR, _LONG, _INT, _INT, _PTR, _INT, _LONG, _PTR]


class _Torch:
    """torch and its types, looked up on the first call (the rest of the package does not need torch)."""
    module = None
    codes = {}

    @classmethod
    def get(cls):
        if cls.module is None:
            import torch
            cls.codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
            cls.module = torch
        return cls.module


def _matrix(tensor, name, dims, codes):
    """Checks a tensor whose last axis is dense and returns the code of its type."""
    torch = _Torch.get()
    if not isinstance(tensor, torch.Tensor):
        raise ValueError(f'{name} must be a torch.Tensor')
    if tensor.dim() != dims:
        raise ValueError(f'{name} must have {dims} axes, not {tensor.dim()}')
    code = _Torch.codes.get(tensor.dtype)
    if code is None or code not in codes:
        raise ValueError(f'{name} has type {tensor.dtype}, which this operator does not take')
    if not tensor.is_cuda:
        raise ValueError(f'{name} must be on a GPU')
    if tensor.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{name} asks for a gradient: this operator has none, call it under torch.no_grad()')
    if tensor.shape[-1] > 1 and tensor.stride(-1) != 1:
        raise ValueError(f'the last axis of {name} must be dense (its stride is {tensor.stride(-1)})')
    return code


def _dense(tensor, name, shape, dtype, device):
    """Checks an optional dense tensor of known shape; returns its address."""
    if tensor is None:
        return None
    if not isinstance(tensor, _Torch.get().Tensor) or tensor.dtype != dtype or tuple(tensor.shape) != shape:
        raise ValueError(f'{name} must be a {dtype} tensor of shape {shape}')
    if tensor.device != device:
        raise ValueError(f'{name} is on {tensor.device}, the operands are on {device}')
    if not tensor.is_contiguous():
        raise ValueError(f'{name} must be contiguous')
    if tensor.requires_grad and _Torch.module.is_grad_enabled():
        raise ValueError(f'{name} asks for a gradient: this operator has none, call it under torch.no_grad()')
    return tensor.data_ptr()


def _same_device(tensor, name, device):
    if tensor.device != device:
        raise ValueError(f'{name} is on {tensor.device}, the operands are on {device}')


def _output(out, shape, dtype, device):
    """The output tensor: a new one, or the caller's after a check."""
    if out is None:
        return _Torch.module.empty(shape, dtype=dtype, device=device)
    _matrix(out, 'out', len(shape), (0, 1, 2))
    if tuple(out.shape) != shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f'out must be a {dtype} tensor of shape {shape}')
    _same_device(out, 'out', device)
    return out


def _stream(device):
    return _Torch.module.cuda.current_stream(device).cuda_stream


def _call(entry, *args):
    from . import ios_runtime
    ios_runtime._check(getattr(ios_runtime._library(), entry)(*args))


def route_experts(logits, k, renormalize=True):
    """
    The router: the ``k`` best experts of every token of ``logits`` [tokens, experts], their gates, and the plan that
    sorts the (token, expert) pairs by expert.  Returns a ``Routing``: ``experts`` [tokens, k], ``gates`` [tokens, k]
    float32, ``offsets`` [experts + 1], ``rows`` [tokens * k] (the token of every sorted row, -1 behind the last) and
    ``slots`` [tokens, k] (the sorted row of every pair).  Equal logits: the lower index first.  Logits of -inf or NaN are
    never chosen; a token with fewer than ``k`` others gets experts and slots of -1 and gates of 0 in their place.
    ``renormalize``: the gates of a token sum to one; otherwise they are its softmax over all experts.
    """
    code = _matrix(logits, 'logits', 2, (0, 1, 2))
    torch = _Torch.module
    tokens, experts = logits.shape
    k = int(k)
    if not 1 <= k <= experts:
        raise ValueError(f'k must be in 1..{experts}, not {k}')
    device = logits.device
    need = _SIZE(0)
    _call('ios_route_experts_workspace', tokens, experts, ctypes.byref(need))
    pairs = tokens * k
    # one allocation: [experts | slots | rows | offsets], then the workspace
    whole = torch.empty(3 * pairs + experts + 1 + (need.value + 3) // 4, dtype=torch.int32, device=device)
    chosen, slots, rows, offsets, work = whole.split([pairs, pairs, pairs, experts + 1, whole.numel() - 3 * pairs - experts - 1])
    gates = torch.empty((tokens, k), dtype=torch.float32, device=device)
    _call('ios_route_experts', logits.data_ptr(), code, tokens, experts, logits.stride(0), k, 1 if renormalize else 0,
          chosen.data_ptr(), gates.data_ptr(), offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(),
          work.data_ptr() if need.value else None, need.value, _stream(device))
    return Routing(chosen.view(tokens, k), gates, offsets, rows, slots.view(tokens, k))


def grouped_matmul(x, weight, offsets, rows=None, bias=None, act='identity', gated=False, row_scale=None,
                   channel_scale=None, out_dtype=None, out=None):
    """
    Products over ragged groups of rows.  Row ``r`` of the result, in group ``g`` (``offsets[g] <= r < offsets[g + 1]``), is
    ``act(x[src] @ weight[g].T * row_scale[src] * channel_scale[g] + bias[g])`` with ``src = rows[r]`` where ``rows`` is given,
    else ``r``.  ``x`` [rows of x, inner] and ``weight`` [groups, channels, inner] are bfloat16, float16, float32 or int8;
    ``offsets`` [groups + 1] and ``rows`` int32; the scales and ``bias`` float32.  ``gated``: ``weight`` holds 2 * channels
    rows per group and the result is ``act(first half) * second half``.  The result has as many rows as ``rows`` (else
    ``x``); those behind ``offsets[-1]`` are not written.  ``out_dtype``: the type of ``x`` unless given (int8: bfloat16).
    """
    code = _matrix(x, 'x', 2, (0, 1, 2, 3))
    torch = _Torch.module
    if _matrix(weight, 'weight', 3, (0, 1, 2, 3)) != code:
        raise ValueError(f'x is {x.dtype}, weight {weight.dtype}: they must have one type')
    device = x.device
    _same_device(weight, 'weight', device)
    groups, channels, inner = weight.shape
    if x.shape[1] != inner:
        raise ValueError(f'x has rows of {x.shape[1]} elements, weight of {inner}')
    per_group = channels
    if gated:
        if channels % 2:
            raise ValueError(f'a gated product needs an even number of weight rows, not {channels}')
        channels //= 2
    if act not in _ACTS:
        raise ValueError(f'act must be one of {", ".join(_ACTS)}')
    offsets_at = _dense(offsets, 'offsets', (groups + 1,), torch.int32, device)
    if offsets_at is None:
        raise ValueError('offsets must not be None')
    total = x.shape[0]
    if rows is not None:
        if not isinstance(rows, torch.Tensor) or rows.dim() != 1:
            raise ValueError('rows must be a tensor of one axis')
        total = rows.shape[0]
    rows_at = _dense(rows, 'rows', (total,), torch.int32, device)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else (torch.bfloat16 if code == 3 else x.dtype)
    if _Torch.codes.get(out_dtype) not in (0, 1, 2):
        raise ValueError(f'the result cannot have type {out_dtype}')
    out = _output(out, (total, channels), out_dtype, device)
    _call('ios_grouped_matmul', x.data_ptr(), code, x.shape[0], x.stride(0), weight.data_ptr(), groups, channels, inner,
          weight.stride(1), weight.stride(0), offsets_at, rows_at, total,
          _dense(row_scale, 'row_scale', (x.shape[0],), torch.float32, device),
          _dense(channel_scale, 'channel_scale', (groups, per_group), torch.float32, device),
          _dense(bias, 'bias', (groups, per_group), torch.float32, device),
          _ACTS[act], 1 if gated else 0, out.data_ptr(), _Torch.codes[out_dtype], out.stride(0), _stream(device))
    return out


def matmul_int8(a, b, row_scale=None, channel_scale=None, bias=None, act='identity', out_dtype=None, out=None):
    """
    ``act(a @ b.T * row_scale[:, None] * channel_scale + bias)`` for int8 ``a`` [rows, inner] and ``b`` [channels, inner], the
    sums exact; scales and bias float32.  The result is bfloat16 unless ``out_dtype`` says otherwise.
    """
    _matrix(a, 'a', 2, (3,))
    _matrix(b, 'b', 2, (3,))
    torch, device = _Torch.module, a.device
    _same_device(b, 'b', device)
    rows, inner = a.shape
    channels = b.shape[0]
    if b.shape[1] != inner:
        raise ValueError(f'a has rows of {inner} elements, b of {b.shape[1]}')
    if act not in _ACTS:
        raise ValueError(f'act must be one of {", ".join(_ACTS)}')
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.bfloat16
    if _Torch.codes.get(out_dtype) not in (0, 1, 2):
        raise ValueError(f'the result cannot have type {out_dtype}')
    out = _output(out, (rows, channels), out_dtype, device)
    _call('ios_matmul_int8', a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), rows, channels, inner,
          _dense(row_scale, 'row_scale', (rows,), torch.float32, device),
          _dense(channel_scale, 'channel_scale', (channels,), torch.float32, device),
          _dense(bias, 'bias', (channels,), torch.float32, device),
          _ACTS[act], out.data_ptr(), _Torch.codes[out_dtype], out.stride(0), _stream(device))
    return out


def quantize_rows(x, rows=None):
    """
    The rows of ``x`` [rows, inner] (or those that the int32 tensor ``rows`` names) in 8-bit integers with a float32 scale
    each: ``(q, scale)`` with ``q * scale[:, None]`` nearest to the row and the largest magnitude of a row at 127.  NaN
    becomes 0, an infinity +-127.  On a weight matrix it gives the scale per channel that ``matmul_int8`` takes.
    """
    code = _matrix(x, 'x', 2, (0, 1, 2))
    torch, device = _Torch.module, x.device
    total = x.shape[0]
    if rows is not None:
        if not isinstance(rows, torch.Tensor) or rows.dim() != 1:
            raise ValueError('rows must be a tensor of one axis')
        total = rows.shape[0]
    rows_at = _dense(rows, 'rows', (total,), torch.int32, device)
    q = torch.empty((total, x.shape[1]), dtype=torch.int8, device=device)
    scale = torch.empty((total,), dtype=torch.float32, device=device)
    _call('ios_quantize_rows', x.data_ptr(), code, x.shape[0], x.stride(0), x.shape[1], rows_at, total, q.data_ptr(),
          x.shape[1], scale.data_ptr(), _stream(device))
    return q, scale


def combine_experts(y, gates, slots, out_dtype=None, out=None):
    """
    The gate-weighted sum of every token's expert rows: ``out[t] = sum_j gates[t, j] * y[slots[t, j]]`` in float32, in the
    order of ``j``.  A slot outside the rows of ``y`` (-1) adds nothing.  The result has the type of ``y`` unless given.
    """
    code = _matrix(y, 'y', 2, (0, 1, 2))
    torch, device = _Torch.module, y.device
    if not isinstance(slots, torch.Tensor) or slots.dim() != 2:
        raise ValueError('slots must be a tensor of two axes')
    tokens, k = slots.shape
    slots_at = _dense(slots, 'slots', (tokens, k), torch.int32, device)
    gates_at = _dense(gates, 'gates', (tokens, k), torch.float32, device)
    if gates_at is None:
        raise ValueError('gates must not be None')
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else y.dtype
    if _Torch.codes.get(out_dtype) not in (0, 1, 2):
        raise ValueError(f'the result cannot have type {out_dtype}')
    out = _output(out, (tokens, y.shape[1]), out_dtype, device)
    _call('ios_combine_experts', y.data_ptr(), code, y.shape[0], y.stride(0), gates_at, slots_at, tokens, k, y.shape[1],
          out.data_ptr(), _Torch.codes[out_dtype], out.stride(0), _stream(device))
    return out


def device_ops_status(device=None):
    """Waits for torch's current stream of ``device`` and raises if a bounded wait inside a product ran out since the last call."""
    torch = _Torch.get()
    index = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    _call('ios_device_ops_status', index, _stream(index))
