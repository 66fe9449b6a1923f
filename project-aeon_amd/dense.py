"""Products over unquantised fp16 / bf16 weights, dense and by expert, over the C ABI: the functions
take torch tensors on one GPU, run on that GPU's current stream and allocate what they return (and
the workspace) from torch's allocator, so they can be captured into a graph.

    y   = linear(x, w, bias, activation="gelu", residual=r)
    lists = expert_lists(ids, experts)
    h   = expert_linear(x, w1, lists.offsets, lists.rows, weight_up=w3, activation="swiglu", swiglu_limit=7.0)
    out = expert_combine(h, w2, lists.offsets, lists.draws, ids, weights, base=shared)
"""
import collections
import ctypes as C

import torch

from . import capi

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "swiglu": 4}


# offsets [experts + 1], draws and rows (= draw // slots) [tokens * slots], int32
ExpertLists = collections.namedtuple("ExpertLists", "offsets draws rows")


class Projection(C.Structure):
    """aeon_projection of the C ABI."""
    _fields_ = [("dtype", C.c_int), ("in_dim", C.c_int), ("out_dim", C.c_int), ("activation", C.c_int),
                ("d_weight", C.c_void_p), ("d_weight_up", C.c_void_p), ("weight_stride", C.c_long),
                ("d_bias", C.c_void_p), ("d_bias_up", C.c_void_p), ("swiglu_limit", C.c_float)]


def _check(t, name, like, shape, dtype=None):
    """One operand: on x's GPU, of its type (or `dtype`), of this shape, its rows contiguous."""
    dtype = like.dtype if dtype is None else dtype
    if t.dtype != dtype:
        raise ValueError("%s is %s, not %s" % (name, t.dtype, dtype))
    if t.device != like.device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, like.device))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s: elements of a row have to follow each other" % name)
    return t


def _pitch(t):
    """Row pitch of a 2-d tensor: a tensor of one row may carry any stride for it."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _projection(x, weight, bias, activation, weight_up, bias_up, limit, lead):
    if x.dim() != 2 or x.dtype not in _DTYPES or not x.is_cuda:
        raise ValueError("x has to be a 2-d fp16 or bf16 tensor on a GPU")
    if activation not in ACTIVATIONS:
        raise ValueError("unknown activation %r" % (activation,))
    if weight.dim() != 2 + lead:
        raise ValueError("weight has to have %d dimensions" % (2 + lead))
    out_dim, in_dim = weight.shape[-2:]
    _check(x, "x", x, (x.shape[0], in_dim))
    _check(weight, "weight", x, weight.shape)
    stride = weight.stride(-2) if out_dim > 1 else max(weight.stride(-2), in_dim)
    if weight_up is not None:
        _check(weight_up, "weight_up", x, weight.shape)
        if weight_up.stride() != weight.stride():
            raise ValueError("weight and weight_up have to have the same strides")
    for b, name in ((bias, "bias"), (bias_up, "bias_up")):
        if b is not None:
            _check(b, name, x, weight.shape[:-1])
            if not b.is_contiguous():
                raise ValueError("%s has to be contiguous" % name)
    return Projection(_DTYPES[x.dtype], in_dim, out_dim, ACTIVATIONS[activation], weight.data_ptr(), _ptr(weight_up),
                      stride, _ptr(bias), _ptr(bias_up), limit)


def _call(x, name, *args):
    """One entry point on the current stream of x's GPU, with that GPU current."""
    stream = torch.cuda.current_stream(x.device).cuda_stream
    if x.device.index == torch.cuda.current_device():
        capi.call(name, *args, C.c_void_p(stream))
    else:
        with torch.cuda.device(x.device):
            capi.call(name, *args, C.c_void_p(stream))


def _output(out, x, shape):
    return torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else _check(out, "out", x, shape)


def _workspace(x, need):
    return torch.empty(need, dtype=torch.uint8, device=x.device) if need else None


def linear(x, weight, bias=None, activation="none", weight_up=None, bias_up=None, swiglu_limit=float("inf"),
           residual=None, out=None):
    """act(x @ weight.T + bias) + residual (aeon_linear). x [tokens][in_dim], weight [out_dim][in_dim];
    "swiglu" takes the second matrix as weight_up. `out` may be the residual itself."""
    p = _projection(x, weight, bias, activation, weight_up, bias_up, swiglu_limit, 0)
    shape = (x.shape[0], p.out_dim)
    if residual is not None:
        _check(residual, "residual", x, shape)
    out = _output(out, x, shape)
    need = capi.lib().aeon_linear_workspace_bytes(C.byref(p), shape[0])
    ws = _workspace(x, need)
    _call(x, "aeon_linear", C.byref(p), capi.vp(x), C.c_long(_pitch(x)), shape[0], capi.vp(residual),
          C.c_long(0 if residual is None else _pitch(residual)), capi.vp(out), C.c_long(_pitch(out)), capi.vp(ws),
          C.c_size_t(need))
    return out


def expert_lists(ids, experts):
    """The ragged lists of a routing, ids int32 [tokens][slots] (aeon_expert_permutation): expert e holds
    positions offsets[e] .. offsets[e+1]-1, its draws (token * slots + slot) ascending; ids outside
    [0, experts) are in no list."""
    if ids.dim() != 2 or ids.dtype != torch.int32 or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("ids has to be a contiguous int32 tensor [tokens][slots] on a GPU")
    new = lambda n: torch.empty(n, dtype=torch.int32, device=ids.device)
    lists = ExpertLists(new(experts + 1), new(ids.numel()), new(ids.numel()))
    _call(ids, "aeon_expert_permutation", capi.vp(ids), ids.shape[0], ids.shape[1], experts, capi.vp(lists.offsets),
          capi.vp(lists.rows), capi.vp(lists.draws), None, None)
    return lists


def _lists(x, experts, offsets, positions, **more):
    _check(offsets, "offsets", x, (experts + 1,), torch.int32)
    for name, t in more.items():
        if t is not None:
            _check(t, name, x, (positions,), torch.int32)


def _expert_stride(weight, p):
    return weight.stride(0) if weight.shape[0] > 1 else max(weight.stride(0), p.out_dim * p.weight_stride)


def expert_linear(x, weight, offsets, rows=None, bias=None, activation="none", weight_up=None, bias_up=None,
                  swiglu_limit=float("inf"), out=None):
    """The same product by expert (aeon_expert_linear): weight [experts][out_dim][in_dim]; expert e's
    positions are offsets[e] .. offsets[e+1]-1, position p takes row rows[p] of x (without `rows`: row p).
    Returns [positions][out_dim]; rows behind the last list are not written."""
    p = _projection(x, weight, bias, activation, weight_up, bias_up, swiglu_limit, 1)
    positions = x.shape[0] if rows is None else rows.shape[0]
    _lists(x, weight.shape[0], offsets, positions, rows=rows)
    out = _output(out, x, (positions, p.out_dim))
    _call(x, "aeon_expert_linear", C.byref(p), weight.shape[0], C.c_long(_expert_stride(weight, p)), capi.vp(x),
          C.c_long(_pitch(x)), x.shape[0], capi.vp(offsets), capi.vp(rows), positions, capi.vp(out),
          C.c_long(_pitch(out)))
    return out


def expert_combine(h, weight, offsets, draws, ids, weights, bias=None, base=None, out=None):
    """base + the weighted sum of each token's expert products, in slot order (aeon_expert_combine).
    h [tokens * slots][in_dim] by position, weight [experts][out_dim][in_dim], ids int32 and weights fp32
    [tokens][slots]. Returns [tokens][out_dim]; `out` may be the base itself."""
    p = _projection(h, weight, bias, "none", None, None, 0.0, 1)
    if ids.dim() != 2:
        raise ValueError("ids has to be [tokens][slots]")
    tokens, slots = ids.shape
    _check(h, "h", h, (tokens * slots, p.in_dim))
    _lists(h, weight.shape[0], offsets, tokens * slots, draws=draws)
    _check(ids, "ids", h, (tokens, slots), torch.int32)
    _check(weights, "weights", h, (tokens, slots), torch.float32)
    if not (ids.is_contiguous() and weights.is_contiguous()):
        raise ValueError("ids and weights have to be contiguous")
    if base is not None:
        _check(base, "base", h, (tokens, p.out_dim))
    out = _output(out, h, (tokens, p.out_dim))
    need = capi.lib().aeon_expert_combine_workspace_bytes(C.byref(p), tokens, slots)
    ws = _workspace(h, need)
    _call(h, "aeon_expert_combine", C.byref(p), weight.shape[0], C.c_long(_expert_stride(weight, p)), capi.vp(h),
          C.c_long(_pitch(h)), capi.vp(offsets), capi.vp(draws), capi.vp(ids), capi.vp(weights), tokens, slots,
          capi.vp(base), C.c_long(0 if base is None else _pitch(base)), capi.vp(out), C.c_long(_pitch(out)),
          capi.vp(ws), C.c_size_t(need))
    return out
