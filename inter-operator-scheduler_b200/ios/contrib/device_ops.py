"""
Operators on device tensors: a mixture-of-experts layer and its 8-bit products.

Unlike the graph entry points, which take host arrays, these take tensors that already live on a GPU (``torch.Tensor``)
and return tensors on the same device; an ``out`` must not overlap what the call reads.  The work goes to torch's current
stream of that device and is not waited for; the calls may be captured into CUDA graphs.  They compute no gradients, and refuse
tensors that ask for one or carry a tangent.

A layer, from its router logits to its output::

    plan = ios_runtime.route_experts(logits, k)
    h = ios_runtime.grouped_matmul(x, w_in, plan.offsets, rows=plan.rows, act='silu', gated=True)
    y = ios_runtime.grouped_matmul(h, w_out, plan.offsets)
    out = ios_runtime.combine_experts(y, plan.gates, plan.slots)

See ``include/ios_runtime.h`` for the formulas.  (The reference has no counterpart: its operators are those of
convolution networks.)
"""
import ctypes
import functools
from collections import namedtuple

_ACTS = {'identity': 0, 'relu': 1, 'sigmoid': 2, 'tanh': 3, 'silu': 4}

Routing = namedtuple('Routing', ['experts', 'gates', 'offsets', 'rows', 'slots'])

_INT, _LONG, _PTR, _SIZE = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_size_t


def declare(handle):
    """Argument types of this module's entry points; called by the library loader."""
    handle.ios_route_experts_workspace.argtypes = [_INT, _INT, _INT, ctypes.POINTER(_SIZE)]
    handle.ios_route_experts.argtypes = [_PTR, _INT, _INT, _INT, _LONG, _INT, _INT] + [_PTR] * 6 + [_SIZE, _PTR]
    handle.ios_grouped_matmul.argtypes = [_PTR, _INT, _LONG, _LONG, _PTR, _INT, _INT, _INT, _LONG, _LONG, _PTR, _PTR, _INT,
                                          _PTR, _PTR, _PTR, _INT, _INT, _PTR, _INT, _LONG, _PTR]
    handle.ios_matmul_int8.argtypes = [_PTR, _LONG, _PTR, _LONG, _INT, _INT, _INT, _PTR, _PTR, _PTR, _INT, _PTR, _INT,
                                       _LONG, _PTR]
    handle.ios_quantize_rows.argtypes = [_PTR, _INT, _LONG, _LONG, _INT, _PTR, _LONG, _PTR, _LONG, _PTR, _PTR]
    handle.ios_device_ops_status.argtypes = [_INT, _PTR]
    handle.ios_combine_experts.argtypes = [_PTR, _INT, _LONG, _LONG, _PTR, _PTR, _LONG, _INT, _INT, _PTR, _INT, _LONG, _PTR]


torch = None          # looked up on the first call: the rest of the package does not need it
_codes = {}           # torch type -> element type of the C interface
_lib = None
_raw_stream = None
_forward_ad = None    # torch.autograd.forward_ad; where its level is below zero, no tensor carries a tangent
_FLOATS, _ALL, _INT8 = (0, 1, 2), (0, 1, 2, 3), (3,)
_MOST_ROWS, _MOST = 1 << 30, (1 << 31) - 1      # rows of a call; any other size: the C interface counts in 32 bits


def _load():
    global torch, _lib, _raw_stream, _forward_ad
    import torch as module
    import torch.autograd.forward_ad as _forward_ad
    from . import ios_runtime
    _codes.update({module.float32: 0, module.float16: 1, module.bfloat16: 2, module.int8: 3})
    # the stream's handle without a Stream object around it, where torch offers that: these calls are short
    _raw_stream = getattr(module._C, '_cuda_getCurrentRawStream', None) or (lambda index: module.cuda.current_stream(index).cuda_stream)
    _lib = ios_runtime._library()
    torch = module


def _no_derivative(tensor, name):
    if tensor.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{name} asks for a gradient: this operator has none, call it under torch.no_grad()')
    if _forward_ad.unpack_dual(tensor).tangent is not None:
        raise ValueError(f'{name} carries a tangent: this operator has no derivative, give it the primal of unpack_dual()')


def _matrix(tensor, name, dims, codes):
    """Checks a tensor whose last axis is dense and returns the code of its type."""
    if torch is None:
        _load()
    if not isinstance(tensor, torch.Tensor):
        raise ValueError(f'{name} must be a torch.Tensor')
    code = _codes.get(tensor.dtype)
    if code not in codes:
        raise ValueError(f'{name} has type {tensor.dtype}, which this operator does not take')
    if tensor.dim() != dims:
        raise ValueError(f'{name} must have {dims} axes, not {tensor.dim()}')
    if not tensor.is_cuda:
        raise ValueError(f'{name} must be on a GPU')
    if (tensor.requires_grad and torch.is_grad_enabled()) or getattr(_forward_ad, '_current_level', 0) >= 0:
        _no_derivative(tensor, name)
    if tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
        raise ValueError(f'the last axis of {name} must be dense (its stride is {tensor.stride(-1)})')
    return code


def _dense(tensor, name, shape, dtype, index):
    """Checks an optional dense tensor of known shape; returns its address."""
    if tensor is None:
        return None
    if not isinstance(tensor, torch.Tensor) or tensor.dtype != dtype or tensor.shape != shape:
        raise ValueError(f'{name} must be a {dtype} tensor of shape {tuple(shape)}')
    if tensor.get_device() != index:
        raise ValueError(f'{name} is on {tensor.device}, the operands are on cuda:{index}')
    if not tensor.is_contiguous():
        raise ValueError(f'{name} must be contiguous')
    if (tensor.requires_grad and torch.is_grad_enabled()) or getattr(_forward_ad, '_current_level', 0) >= 0:
        _no_derivative(tensor, name)
    return tensor.data_ptr()


def _needed(tensor, name, shape, dtype, index):
    if tensor is None:
        raise ValueError(f'{name} must not be None')
    return _dense(tensor, name, shape, dtype, index)


def _same_device(tensor, name, index):
    if tensor.get_device() != index:
        raise ValueError(f'{name} is on {tensor.device}, the operands are on cuda:{index}')


def _length(rows, name='rows'):
    if not isinstance(rows, torch.Tensor) or rows.dim() != 1:
        raise ValueError(f'{name} must be a tensor of one axis')
    return rows.shape[0]


def _output(out, out_dtype, default, like, shape):
    """
    (tensor, code of its type, row stride): a new one of `out_dtype`, else `default`, or the caller's after a check, marked
    as changed for whatever autograd has saved it for.
    """
    if out is None:
        dtype = default if out_dtype is None else out_dtype
        code = _codes.get(dtype)
        if code not in _FLOATS:
            raise ValueError(f'the result cannot have type {dtype}')
        return like.new_empty(shape, dtype=dtype), code, shape[1]
    code = _matrix(out, 'out', 2, _FLOATS)
    if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f'out must be a {out.dtype if out_dtype is None else out_dtype} tensor of shape {shape}')
    _same_device(out, 'out', like.get_device())
    torch.autograd.graph.increment_version(out)
    return out, code, max(out.stride(0), shape[1]) if shape[0] == 1 else out.stride(0)


def _too_large(what):
    raise ValueError(f'more than 2^30 rows, or rows of 2^31 elements or more: {what}')


def _act(act):
    code = _ACTS.get(act)
    if code is None:
        raise ValueError(f'act must be one of {", ".join(_ACTS)}')
    return code


def _check(status):
    if status != 0:
        from . import ios_runtime
        ios_runtime._check(status)


@functools.lru_cache(maxsize=1024)
def _route_workspace(tokens, experts, k):
    need = _SIZE(0)
    _check(_lib.ios_route_experts_workspace(tokens, experts, k, ctypes.byref(need)))
    return need.value


def route_experts(logits, k, renormalize=True):
    """
    The router: the ``k`` best experts of every token of ``logits`` [tokens, experts], their gates, and the plan that
    sorts the (token, expert) pairs by expert.  Returns a ``Routing``: ``experts`` [tokens, k], ``gates`` [tokens, k]
    float32, ``offsets`` [experts + 1], ``rows`` [tokens * k] (the token of every sorted row, -1 behind the last) and
    ``slots`` [tokens, k] (the sorted row of every pair).  Equal logits: the lower index first.  Logits of -inf or NaN are
    never chosen; a token with fewer than ``k`` others gets experts and slots of -1 and gates of 0 in their place.
    ``renormalize``: the gates of a token sum to one; otherwise they are its softmax over all experts.
    """
    code = _matrix(logits, 'logits', 2, _FLOATS)
    tokens, experts = logits.shape
    k = int(k)
    if tokens * k > _MOST_ROWS or experts > _MOST:
        _too_large(f'logits of shape {tuple(logits.shape)}, k = {k}')
    if not 1 <= k <= experts:
        raise ValueError(f'k must be in 1..{experts}, not {k}')
    pairs, need = tokens * k, _route_workspace(tokens, experts, k)
    # one allocation for everything: experts, slots, gates, rows, offsets, workspace
    whole = logits.new_empty(4 * pairs + experts + 1 + (need + 3) // 4, dtype=torch.int32)
    square, apart = (tokens, k), (k, 1)
    chosen, slots = whole.as_strided(square, apart, 0), whole.as_strided(square, apart, pairs)
    gates = whole.as_strided(square, apart, 2 * pairs).view(torch.float32)
    rows, offsets = whole.as_strided((pairs,), (1,), 3 * pairs), whole.as_strided((experts + 1,), (1,), 4 * pairs)
    base = whole.data_ptr()
    _check(_lib.ios_route_experts(
        logits.data_ptr(), code, tokens, experts, logits.stride(0), k, 1 if renormalize else 0, base, base + 8 * pairs,
        base + 16 * pairs, base + 12 * pairs, base + 4 * pairs, base + 4 * (4 * pairs + experts + 1) if need else None, need,
        _raw_stream(logits.get_device())))
    return Routing(chosen, gates, offsets, rows, slots)


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
    code = _matrix(x, 'x', 2, _ALL)
    if _matrix(weight, 'weight', 3, _ALL) != code:
        raise ValueError(f'x is {x.dtype}, weight {weight.dtype}: they must have one type')
    index = x.get_device()
    _same_device(weight, 'weight', index)
    x_rows, inner = x.shape
    groups, per_group, weight_inner = weight.shape
    if weight_inner != inner:
        raise ValueError(f'x has rows of {inner} elements, weight of {weight_inner}')
    channels = per_group
    if gated:
        if per_group % 2:
            raise ValueError(f'a gated product needs an even number of weight rows, not {per_group}')
        channels = per_group // 2
    total = x_rows if rows is None else _length(rows)
    if total > _MOST_ROWS or per_group > _MOST or inner > _MOST or groups > _MOST:
        _too_large(f'{total} rows, weight of shape {tuple(weight.shape)}')
    f32, i32 = torch.float32, torch.int32
    out, out_code, out_stride = _output(out, out_dtype, torch.bfloat16 if code == 3 else x.dtype, x, (total, channels))
    _check(_lib.ios_grouped_matmul(
        x.data_ptr(), code, x_rows, x.stride(0), weight.data_ptr(), groups, channels, inner, weight.stride(1), weight.stride(0),
        _needed(offsets, 'offsets', (groups + 1,), i32, index), _dense(rows, 'rows', (total,), i32, index), total,
        _dense(row_scale, 'row_scale', (x_rows,), f32, index),
        _dense(channel_scale, 'channel_scale', (groups, per_group), f32, index),
        _dense(bias, 'bias', (groups, per_group), f32, index), _act(act), 1 if gated else 0, out.data_ptr(), out_code, out_stride,
        _raw_stream(index)))
    return out


def matmul_int8(a, b, row_scale=None, channel_scale=None, bias=None, act='identity', out_dtype=None, out=None):
    """
    ``act(a @ b.T * row_scale[:, None] * channel_scale + bias)`` for int8 ``a`` [rows, inner] and ``b`` [channels, inner], the
    sums exact; scales and bias float32.  The result is bfloat16 unless ``out_dtype`` says otherwise.
    """
    _matrix(a, 'a', 2, _INT8)
    _matrix(b, 'b', 2, _INT8)
    index = a.get_device()
    _same_device(b, 'b', index)
    rows, inner = a.shape
    channels, b_inner = b.shape
    if b_inner != inner:
        raise ValueError(f'a has rows of {inner} elements, b of {b_inner}')
    if rows > _MOST_ROWS or channels > _MOST or inner > _MOST:
        _too_large(f'a of shape {tuple(a.shape)}, b of shape {tuple(b.shape)}')
    f32 = torch.float32
    out, out_code, out_stride = _output(out, out_dtype, torch.bfloat16, a, (rows, channels))
    _check(_lib.ios_matmul_int8(
        a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), rows, channels, inner, _dense(row_scale, 'row_scale', (rows,), f32, index),
        _dense(channel_scale, 'channel_scale', (channels,), f32, index), _dense(bias, 'bias', (channels,), f32, index), _act(act),
        out.data_ptr(), out_code, out_stride, _raw_stream(index)))
    return out


def quantize_rows(x, rows=None):
    """
    The rows of ``x`` [rows, inner] (or those that the int32 tensor ``rows`` names) in 8-bit integers with a float32 scale
    each: ``(q, scale)`` with ``q * scale[:, None]`` nearest to the row and the largest magnitude of a row at 127.  NaN
    becomes 0, an infinity +-127.  On a weight matrix it gives the scale per channel that ``matmul_int8`` takes.
    """
    code = _matrix(x, 'x', 2, _FLOATS)
    index = x.get_device()
    x_rows, inner = x.shape
    total = x_rows if rows is None else _length(rows)
    if total > _MOST_ROWS or inner > _MOST:
        _too_large(f'{total} rows of {inner} elements')
    q, scale = x.new_empty((total, inner), dtype=torch.int8), x.new_empty((total,), dtype=torch.float32)
    _check(_lib.ios_quantize_rows(
        x.data_ptr(), code, x_rows, x.stride(0), inner, _dense(rows, 'rows', (total,), torch.int32, index), total, q.data_ptr(), inner,
        scale.data_ptr(), _raw_stream(index)))
    return q, scale


def combine_experts(y, gates, slots, out_dtype=None, out=None):
    """
    The gate-weighted sum of every token's expert rows: ``out[t] = sum_j gates[t, j] * y[slots[t, j]]`` in float32, in the
    order of ``j``.  A slot outside the rows of ``y`` (-1) adds nothing.  The result has the type of ``y`` unless given.
    """
    code = _matrix(y, 'y', 2, _FLOATS)
    if not isinstance(slots, torch.Tensor) or slots.dim() != 2:
        raise ValueError('slots must be a tensor of two axes')
    index = y.get_device()
    y_rows, channels = y.shape
    shape = tokens, k = slots.shape
    if tokens > _MOST_ROWS or k > _MOST or channels > _MOST:
        _too_large(f'y of shape {tuple(y.shape)}, slots of shape {tuple(shape)}')
    out, out_code, out_stride = _output(out, out_dtype, y.dtype, y, (tokens, channels))
    _check(_lib.ios_combine_experts(
        y.data_ptr(), code, y_rows, y.stride(0), _needed(gates, 'gates', shape, torch.float32, index),
        _dense(slots, 'slots', shape, torch.int32, index), tokens, k, channels, out.data_ptr(), out_code, out_stride,
        _raw_stream(index)))
    return out


def device_ops_status(device=None):
    """
    Waits for torch's current stream of ``device`` and raises if a bounded wait inside a product there, on any stream, ran out
    since the calling thread last asked (or ever): the output of that product is incomplete, which nothing else tells.
    """
    if torch is None:
        _load()
    index = None
    if device is not None:
        device = torch.device(device)
        if device.type != 'cuda':
            raise ValueError(f'{device} is not a GPU')
        index = device.index
    if index is None:                            # None, or 'cuda' without a number
        index = torch.cuda.current_device()
    _check(_lib.ios_device_ops_status(index, _raw_stream(index)))
