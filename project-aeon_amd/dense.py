"""Products over unquantised fp16 / bf16 weights, dense and by expert, over the C ABI: the functions
take torch tensors on one GPU, run on that GPU's current stream and allocate what they return (and
the workspace) from torch's allocator, so they can be captured into a graph. They have no backward
pass: where one would be recorded (gradients enabled, an operand that requires one) they refuse.

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


# These functions are called once per projection and token: what they check, they check with a few attribute
# reads, and one call costs the host about as much as one of torch's own element-wise operators.


def _check(t, name, device, dtype, shape):
    """Of this type, on this GPU, of this shape, the elements of a row next to each other."""
    if (t.dtype is dtype and t.get_device() == device and t.shape == shape
            and (t.stride(-1) == 1 or shape[-1] <= 1)):
        return
    if t.dtype is not dtype:
        raise ValueError("%s is %s, not %s" % (name, t.dtype, dtype))
    if t.get_device() != device:
        raise ValueError("%s is on %s, not on GPU %d" % (name, t.device, device))
    if t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    raise ValueError("%s: elements of a row have to follow each other" % name)


def pitch(t):
    """Row pitch of a 2-d tensor: a tensor of one row may carry any stride for it."""
    rows, cols = t.shape
    pitch = t.stride(0)
    return pitch if rows > 1 or pitch > cols else cols


def check_rows(t, name, like, cols):
    """A 2-d tensor of `cols` columns, of the type and on the GPU of `like`."""
    if t.dim() != 2:
        raise ValueError("%s has to be a 2-d tensor" % name)
    _check(t, name, like.get_device(), like.dtype, (t.shape[0], cols))


def _forward_only(*operands):
    """A result without a backward pass would drop the operands' gradients and say nothing."""
    if torch._C._any_requires_grad(*operands) and torch.is_grad_enabled():
        raise ValueError("an operand requires a gradient, and there is no backward pass: call under torch.no_grad(), or "
                         "give the operands detached")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _projection(x, weight, bias, activation, weight_up, bias_up, limit, lead):
    kind, shape, device = x.dtype, weight.shape, x.get_device()
    dtype, act = _DTYPES.get(kind), ACTIVATIONS.get(activation)
    if dtype is None or device < 0 or x.dim() != 2:
        raise ValueError("x has to be a 2-d fp16 or bf16 tensor on a GPU")
    if act is None:
        raise ValueError("unknown activation %r" % (activation,))
    if len(shape) != 2 + lead:
        raise ValueError("weight has to have %d dimensions" % (2 + lead))
    out_dim, in_dim = shape[-2], shape[-1]
    _check(x, "x", device, kind, (x.shape[0], in_dim))
    _check(weight, "weight", device, kind, shape)
    stride = weight.stride(-2)
    if out_dim == 1 and stride < in_dim:
        stride = in_dim
    if weight_up is not None:
        _check(weight_up, "weight_up", device, kind, shape)
        if weight_up.stride() != weight.stride():
            raise ValueError("weight and weight_up have to have the same strides")
    if bias is not None:
        _check_bias(bias, "bias", device, kind, shape)
    if bias_up is not None:
        _check_bias(bias_up, "bias_up", device, kind, shape)
    return Projection(dtype, in_dim, out_dim, act, weight.data_ptr(), _ptr(weight_up), stride, _ptr(bias), _ptr(bias_up), limit)


def _check_bias(b, name, device, kind, shape):
    _check(b, name, device, kind, shape[:-1])
    if not b.is_contiguous():
        raise ValueError("%s has to be contiguous" % name)


def _call(device, entry, *args):
    """One entry point on the current stream of a GPU, with that GPU current."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch._C._cuda_getDevice():
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    if rc != capi.OK:
        capi.check(rc)


def _output(out, x, shape):
    if out is None:
        return x.new_empty(shape)
    _check(out, "out", x.get_device(), x.dtype, shape)
    return out


def _workspace(x, need):
    return x.new_empty(need, dtype=torch.uint8) if need else None


def linear(x, weight, bias=None, activation="none", weight_up=None, bias_up=None, swiglu_limit=float("inf"),
           residual=None, out=None):
    """act(x @ weight.T + bias) + residual (aeon_linear). x [tokens][in_dim], weight [out_dim][in_dim];
    "swiglu" takes the second matrix as weight_up. `out` may be the residual itself."""
    _forward_only(x, weight, bias, weight_up, bias_up, residual)
    p = _projection(x, weight, bias, activation, weight_up, bias_up, swiglu_limit, 0)
    device, tokens = x.get_device(), x.shape[0]
    shape = (tokens, p.out_dim)
    if residual is not None:
        _check(residual, "residual", device, x.dtype, shape)
    out = _output(out, x, shape)
    at, lib = C.addressof(p), capi.lib()
    need = lib.aeon_linear_workspace_bytes(at, tokens)
    ws = _workspace(x, need)
    _call(device, lib.aeon_linear, at, x.data_ptr(), pitch(x), tokens, _ptr(residual),
          0 if residual is None else pitch(residual), out.data_ptr(), pitch(out), _ptr(ws), need)
    return out


def router_logits(x, gate):
    """fp32 [tokens][experts]: the sums x @ gate.T of a bf16 gate [experts][hidden], unrounded
    (aeon_router_logits_bf16)."""
    _forward_only(x, gate)
    if gate.dim() != 2 or gate.dtype is not torch.bfloat16 or not gate.is_cuda:
        raise ValueError("gate has to be a 2-d bf16 tensor on a GPU")
    experts, hidden = gate.shape
    check_rows(gate, "gate", gate, hidden)
    check_rows(x, "x", gate, hidden)
    device, tokens, lib = gate.get_device(), x.shape[0], capi.lib()
    out = x.new_empty((tokens, experts), dtype=torch.float32)
    need = lib.aeon_router_logits_bf16_workspace_bytes(tokens, hidden, experts)
    ws = _workspace(x, need)
    _call(device, lib.aeon_router_logits_bf16, x.data_ptr(), pitch(x), gate.data_ptr(), pitch(gate), out.data_ptr(), tokens,
          hidden, experts, _ptr(ws), need)
    return out


def expert_lists(ids, experts):
    """The ragged lists of a routing, ids int32 [tokens][slots] (aeon_expert_permutation): expert e holds
    positions offsets[e] .. offsets[e+1]-1, its draws (token * slots + slot) ascending; ids outside
    [0, experts) are in no list."""
    if ids.dim() != 2 or ids.dtype != torch.int32 or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("ids has to be a contiguous int32 tensor [tokens][slots] on a GPU")
    new = lambda n: torch.empty(n, dtype=torch.int32, device=ids.device)
    if ids.numel() == 0:
        return ExpertLists(torch.zeros(experts + 1, dtype=torch.int32, device=ids.device), new(0), new(0))
    lists = ExpertLists(new(experts + 1), new(ids.numel()), new(ids.numel()))
    stream = lambda: C.c_void_p(torch.cuda.current_stream(ids.device).cuda_stream)
    with torch.cuda.device(ids.device):
        capi.call("aeon_expert_permutation", capi.vp(ids), ids.shape[0], ids.shape[1], experts, capi.vp(lists.offsets),
                  capi.vp(lists.rows), capi.vp(lists.draws), None, None, stream())
    return lists


def _lists(device, experts, offsets, positions, lists, name):
    _check(offsets, "offsets", device, torch.int32, (experts + 1,))
    if lists is not None:
        _check(lists, name, device, torch.int32, (positions,))


def _expert_stride(weight, p):
    stride = weight.stride(0)
    return stride if weight.shape[0] > 1 else max(stride, p.out_dim * p.weight_stride)


def expert_linear(x, weight, offsets, rows=None, bias=None, activation="none", weight_up=None, bias_up=None,
                  swiglu_limit=float("inf"), out=None):
    """The same product by expert (aeon_expert_linear): weight [experts][out_dim][in_dim]; expert e's
    positions are offsets[e] .. offsets[e+1]-1, position p takes row rows[p] of x (without `rows`: row p).
    Returns [positions][out_dim]; rows behind the last list are not written."""
    _forward_only(x, weight, bias, weight_up, bias_up)
    p = _projection(x, weight, bias, activation, weight_up, bias_up, swiglu_limit, 1)
    device, x_rows = x.get_device(), x.shape[0]
    positions = x_rows if rows is None else rows.shape[0]
    _lists(device, weight.shape[0], offsets, positions, rows, "rows")
    out = _output(out, x, (positions, p.out_dim))
    _call(device, capi.lib().aeon_expert_linear, C.addressof(p), weight.shape[0], _expert_stride(weight, p), x.data_ptr(), pitch(x),
          x_rows, offsets.data_ptr(), _ptr(rows), positions, out.data_ptr(), pitch(out))
    return out


def expert_combine(h, weight, offsets, draws, ids, weights, bias=None, base=None, out=None):
    """base + the weighted sum of each token's expert products, in slot order (aeon_expert_combine).
    h [tokens * slots][in_dim] by position, weight [experts][out_dim][in_dim], ids int32 and weights fp32
    [tokens][slots], offsets and draws the lists of these ids: a draw is left out by an id outside
    [0, experts), not by taking it from a list. Returns [tokens][out_dim]; `out` may be the base itself."""
    _forward_only(h, weight, bias, weights, base)
    p = _projection(h, weight, bias, "none", None, None, 0.0, 1)
    if ids.dim() != 2:
        raise ValueError("ids has to be [tokens][slots]")
    tokens, slots = ids.shape
    device = h.get_device()
    if h.shape[0] != tokens * slots:
        raise ValueError("h has %d rows, not %d" % (h.shape[0], tokens * slots))
    _lists(device, weight.shape[0], offsets, tokens * slots, draws, "draws")
    _check(ids, "ids", device, torch.int32, ids.shape)
    _check(weights, "weights", device, torch.float32, ids.shape)
    if not (ids.is_contiguous() and weights.is_contiguous()):
        raise ValueError("ids and weights have to be contiguous")
    shape = (tokens, p.out_dim)
    if base is not None:
        _check(base, "base", device, h.dtype, shape)
    out = _output(out, h, shape)
    at, lib = C.addressof(p), capi.lib()
    need = lib.aeon_expert_combine_workspace_bytes(at, tokens, slots)
    ws = _workspace(h, need)
    _call(device, lib.aeon_expert_combine, at, weight.shape[0], _expert_stride(weight, p), h.data_ptr(), pitch(h),
          offsets.data_ptr(), draws.data_ptr(), ids.data_ptr(), weights.data_ptr(), tokens, slots, _ptr(base),
          0 if base is None else pitch(base), out.data_ptr(), pitch(out), _ptr(ws), need)
    return out
