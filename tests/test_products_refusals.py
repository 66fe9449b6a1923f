"""What the entry points of the unquantised products refuse, before any device work."""
import ctypes as C

import pytest

from project_aeon_amd import capi, dense

A = C.c_void_p(1 << 20)        # never dereferenced: every call below is refused first, or has nothing to do
B = C.c_void_p(1 << 21)
ODD = C.c_void_p((1 << 20) + 1)


def _p(**change):
    fields = dict(dtype=0, in_dim=64, out_dim=32, activation=0, d_weight=1 << 22, d_weight_up=None, weight_stride=64,
                  d_bias=None, d_bias_up=None, swiglu_limit=0.0)
    fields.update(change)
    return dense.Projection(**fields)


def _linear(p, x=A, xs=64, tokens=4, res=None, rs=0, y=B, ys=32, ws=None, wb=0):
    capi.call("aeon_linear", None if p is None else C.byref(p), x, C.c_long(xs), tokens, res, C.c_long(rs), y, C.c_long(ys),
              ws, C.c_size_t(wb), None)


def _experts(p, experts=4, es=2048, x=A, xs=64, x_rows=8, off=A, rows=None, positions=8, y=B, ys=32):
    capi.call("aeon_expert_linear", C.byref(p), experts, C.c_long(es), x, C.c_long(xs), x_rows, off, rows, positions, y,
              C.c_long(ys), None)


def _combine(p, experts=4, es=2048, h=A, hs=64, off=A, draws=A, ids=A, w=A, tokens=4, slots=2, base=None, bs=0, out=B,
             os=32, ws=A, wb=1 << 30):
    capi.call("aeon_expert_combine", C.byref(p), experts, C.c_long(es), h, C.c_long(hs), off, draws, ids, w, tokens, slots,
              base, C.c_long(bs), out, C.c_long(os), ws, C.c_size_t(wb), None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "unknown dtype"), (dict(dtype=-1), "unknown dtype"),
    (dict(in_dim=0), "bad shape"), (dict(out_dim=-3), "bad shape"), (dict(in_dim=1 << 25, weight_stride=1 << 25), "bad shape"),
    (dict(weight_stride=63), "overlap"), (dict(activation=5), "unknown activation"), (dict(activation=-1), "unknown activation"),
    (dict(d_weight=None), "null weight"), (dict(activation=4, swiglu_limit=7.0), "second weight matrix"),
    (dict(d_weight_up=1 << 23), "second weight matrix"), (dict(d_bias_up=1 << 23), "second bias"),
    (dict(activation=4, d_weight_up=1 << 23), "swiglu_limit"),
    (dict(activation=4, d_weight_up=1 << 23, swiglu_limit=float("nan")), "swiglu_limit"),
    (dict(d_weight=(1 << 22) + 1), "odd address"), (dict(d_bias=(1 << 22) + 1), "odd address")])
def test_projection_refusals(change, text):
    for call in (_linear, _experts, _combine):
        with pytest.raises(ValueError, match=text):
            call(_p(**change))
    assert capi.lib().aeon_linear_workspace_bytes(C.byref(_p(**change)), 4) == 0
    assert capi.lib().aeon_expert_combine_workspace_bytes(C.byref(_p(**change)), 4, 2) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(tokens=-1), "out of range"), (dict(tokens=(1 << 30) + 1), "out of range"), (dict(x=None), "null buffer"), (dict(y=None), "null buffer"), (dict(x=ODD), "odd address"),
    (dict(y=ODD), "odd address"), (dict(res=ODD, rs=32), "odd address"), (dict(xs=63), "row pitch"), (dict(ys=31), "row pitch"),
    (dict(res=A, rs=31), "row pitch"), (dict(y=A), "must not alias"), (dict(y=C.c_void_p(1 << 22)), "must not alias"),
    (dict(res=B, rs=40), "residual's row pitch")])
def test_linear_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _linear(_p(), **kw)


def test_linear_refuses_a_short_workspace():
    p = _p(in_dim=7168, weight_stride=7168, out_dim=256)
    need = capi.lib().aeon_linear_workspace_bytes(C.byref(p), 20)
    assert need > 0 and need % (256 * 4) == 0
    for ws, wb in ((None, need), (A, need - 1), (C.c_void_p((1 << 20) + 4), need)):
        with pytest.raises(ValueError, match="workspace of"):
            _linear(p, xs=7168, ys=256, tokens=20, ws=ws, wb=wb)


@pytest.mark.parametrize("kw,text", [
    (dict(experts=0), "expert count"), (dict(experts=1025), "expert count"), (dict(es=2047), "overlap"),
    (dict(positions=-1), "out of range"), (dict(positions=(1 << 30) + 1, rows=A), "out of range"), (dict(x=None), "null buffer"), (dict(off=None), "null buffer"),
    (dict(y=None), "null buffer"), (dict(x_rows=7), "7 rows for 8"), (dict(x_rows=0, rows=A), "0 rows"),
    (dict(x=ODD), "boundary"), (dict(off=C.c_void_p((1 << 20) + 2)), "boundary"), (dict(xs=8), "row pitch"),
    (dict(ys=8), "row pitch"), (dict(y=A), "must not alias")])
def test_expert_linear_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _experts(_p(), **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(experts=2000), "expert count"), (dict(es=100), "overlap"), (dict(tokens=-1), "bad draw shape"),
    (dict(slots=0), "bad draw shape"), (dict(tokens=1 << 30, slots=4), "bad draw shape"), (dict(h=None), "null buffer"),
    (dict(draws=None), "null buffer"), (dict(ids=None), "null buffer"), (dict(w=None), "null buffer"),
    (dict(out=None), "null buffer"), (dict(h=ODD), "boundary"), (dict(w=C.c_void_p(2)), "boundary"), (dict(hs=1), "row pitch"),
    (dict(os=1), "row pitch"), (dict(base=A, bs=1), "row pitch"), (dict(out=A), "must not alias"),
    (dict(base=B, bs=40), "base's row pitch"), (dict(tokens=40, ws=None), "workspace of"), (dict(tokens=40, wb=8), "workspace of")])
def test_expert_combine_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _combine(_p(), **kw)


def test_combine_takes_no_activation():
    with pytest.raises(ValueError, match="no activation"):
        _combine(_p(activation=1))


def test_null_projection_and_calls_with_nothing_to_do():
    with pytest.raises(ValueError, match="null projection"):
        _linear(None)
    _linear(_p(), tokens=0, x=None, y=None)
    _experts(_p(), positions=0, x=None, y=None)
    _combine(_p(), tokens=0, h=None, out=None)


def test_the_tensor_functions_check_their_operands():
    import torch
    x, w = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="on a GPU"):
        dense.linear(x, w)
    with pytest.raises(ValueError, match="on a GPU"):
        dense.linear(x.double(), w)
    with pytest.raises(ValueError, match="on a GPU"):
        dense.expert_lists(torch.zeros(2, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="hidden"):
        from project_aeon_amd import moe
        moe.UnquantisedMoeLayer(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), 1, 7.0)


def test_calls_of_more_threads_than_a_launch_holds():
    wide = dict(out_dim=1 << 24)
    calls = (lambda: _linear(_p(out_dim=1 << 20), tokens=1 << 30, ys=1 << 20),
             lambda: _experts(_p(**wide), experts=1024, es=1 << 30, positions=1024, x_rows=1024, ys=1 << 24),
             lambda: _combine(_p(), tokens=1 << 25, slots=1, wb=1 << 40))
    for call in calls:
        with pytest.raises(ValueError, match="more than one launch holds"):
            call()


def test_a_layer_without_a_router_takes_given_routing_only():
    import torch
    from project_aeon_amd import moe
    w = torch.zeros(2, 4, 4, dtype=torch.float16)
    with pytest.raises(ValueError, match="no router"):
        moe.UnquantisedMoeLayer(w, w, w, 1, 7.0).decode(torch.zeros(1, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="fp16 activations"):
        moe.UnquantisedMoeLayer(w.bfloat16(), w.bfloat16(), w.bfloat16(), 1, 7.0, router_weight=torch.zeros(4, 2))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_a_layer_checks_the_shape_of_its_16_bit_gate(dtype):
    """The router is told `experts` logits a token: a gate of another row count would make it read behind
    them, or at shifted places. Rows wider than the matrix are taken."""
    import torch
    from project_aeon_amd import moe
    dt, E, I, H = getattr(torch, dtype), 8, 4, 16
    w1, w2 = torch.zeros(E, I, H, dtype=dt), torch.zeros(E, H, I, dtype=dt)
    other = torch.float16 if dt is torch.bfloat16 else torch.bfloat16
    for gate in (torch.zeros(E - 1, H, dtype=dt), torch.zeros(E + 1, H, dtype=dt), torch.zeros(E, H - 1, dtype=dt),
                 torch.zeros(E, H, dtype=other), torch.zeros(E, H), torch.zeros(E * H, dtype=dt),
                 torch.zeros(H, E, dtype=dt).t(), torch.zeros(E, H, dtype=dt, device="meta")):
        with pytest.raises(ValueError, match="router_weight_16"):
            moe.UnquantisedMoeLayer(w1, w1, w2, 2, 7.0, router_weight_16=gate)
    moe.UnquantisedMoeLayer(w1, w1, w2, 2, 7.0, router_weight_16=torch.zeros(E, H + 3, dtype=dt)[:, :H])


def test_a_layer_refuses_a_routing_of_other_tokens():
    """ids and weights are [tokens][slots] of the given x: rows of ids beyond x would be sums over hidden rows that
    no product wrote, fewer would leave tokens out."""
    import torch
    from project_aeon_amd import moe
    E, I, H = 4, 4, 16
    w1, w2 = torch.zeros(E, I, H, dtype=torch.float16), torch.zeros(E, H, I, dtype=torch.float16)
    layer = moe.UnquantisedMoeLayer(w1, w1, w2, 2, 7.0)
    x = torch.zeros(3, H, dtype=torch.float16)
    ids, weights = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for bad in (ids[:2], torch.zeros(5, 2, dtype=torch.int32), ids.reshape(-1), ids[:0]):
        with pytest.raises(ValueError, match="ids has to be .*3 tokens"):
            layer.routed(x, bad, torch.zeros(bad.shape))
    for bad in (weights[:2], weights[:, :1], torch.zeros(5, 2)):
        with pytest.raises(ValueError, match="weights has to be"):
            layer.routed(x, ids, bad)


def test_a_layer_refuses_rows_too_far_apart_for_the_fp32_gate():
    """aeon_router_logits takes the row pitch as an int; 2^32 + 16 elements would pass as 16."""
    import torch
    from project_aeon_amd import moe
    E, I, H = 4, 4, 16
    w1 = torch.zeros(E, I, H, dtype=torch.float16, device="meta")
    w2 = torch.zeros(E, H, I, dtype=torch.float16, device="meta")
    layer = moe.UnquantisedMoeLayer(w1, w1, w2, 2, 7.0, router_weight=torch.zeros(H, E, device="meta"))
    far = torch.empty((1 << 33), dtype=torch.float16, device="meta").as_strided((2, H), ((1 << 32) + H, 1))
    with pytest.raises(ValueError, match="pitch"):
        layer.router_logits(far)


def test_a_stack_takes_unquantised_layers_of_fp16_only():
    """The residual streams and their mixes are fp16. Layers without the fused tail run in the three launches."""
    import torch
    from project_aeon_amd import moe

    def layer(dtype):
        w1, w2 = torch.zeros(2, 4, 8, dtype=dtype), torch.zeros(2, 8, 4, dtype=dtype)
        return moe.UnquantisedMoeLayer(w1, w1, w2, 1, 7.0)

    assert moe.LayerStack([layer(torch.float16)], [None]).fused is False
    assert moe.LayerStack([], []).fused is True
    with pytest.raises(ValueError, match="fp16"):
        moe.LayerStack([layer(torch.float16), layer(torch.bfloat16)], [None, None])


@pytest.mark.parametrize("kw,text", [
    (dict(tokens=-1), "out of range"), (dict(x=None), "null buffer"), (dict(y=None), "null buffer"), (dict(gate=None), "null weight"),
    (dict(x=ODD), "boundary"), (dict(y=C.c_void_p((1 << 21) + 2)), "boundary"), (dict(gate=ODD), "odd address"),
    (dict(xs=7167), "row pitch"), (dict(gs=7167), "overlap"), (dict(y=A), "must not alias"), (dict(experts=0), "bad shape"),
    (dict(ws=None), "workspace of"), (dict(wb=4), "workspace of")])
def test_bf16_gate_refusals(kw, text):
    a = dict(x=A, xs=7168, gate=C.c_void_p(1 << 22), gs=7168, y=B, tokens=20, hidden=7168, experts=256, ws=A, wb=1 << 30)
    a.update(kw)
    assert capi.lib().aeon_router_logits_bf16_workspace_bytes(20, 7168, 256) > 0
    with pytest.raises(ValueError, match=text):
        capi.call("aeon_router_logits_bf16", a["x"], a["xs"], a["gate"], a["gs"], a["y"], a["tokens"], a["hidden"],
                  a["experts"], a["ws"], a["wb"], None)


def test_the_bf16_gate_checks_its_operands():
    import torch
    for gate in (torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.float16), torch.zeros(8, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="gate has to be"):
            dense.router_logits(torch.zeros(2, 8, dtype=torch.bfloat16), gate)


def test_nothing_drops_a_gradient_silently():
    """An operand that requires a gradient is refused while gradients are recorded, whichever it is; without
    recording, or detached, the call goes on to its other checks (here: no GPU)."""
    import torch
    h = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16)
    lists = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    ids = torch.zeros(2, 2, dtype=torch.int32)
    x, y, w, w3, b = h(2, 8), h(4, 8), h(6, 8), h(2, 6, 8), h(6)
    calls = ((dense.linear, dict(x=x, weight=w, bias=b, weight_up=h(6, 8), bias_up=h(6), residual=h(2, 6), activation="swiglu")),
             (dense.expert_linear, dict(x=x, weight=w3, offsets=lists[0], rows=lists[1], bias=h(2, 6), weight_up=h(2, 6, 8),
                                        bias_up=h(2, 6), activation="swiglu")),
             (dense.expert_combine, dict(h=y, weight=w3, offsets=lists[0], draws=lists[1], ids=ids, weights=torch.zeros(2, 2),
                                         bias=h(2, 6), base=h(2, 6))),
             (dense.router_logits, dict(x=x, gate=w)))
    for call, kw in calls:
        for name, t in kw.items():
            if not (isinstance(t, torch.Tensor) and t.is_floating_point()):
                continue
            given = dict(kw)
            given[name] = t.clone().requires_grad_()
            with pytest.raises(ValueError, match="no backward pass"):
                call(**given)
            with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
                call(**given)
            given[name] = given[name].detach()
            with pytest.raises(ValueError, match="on a GPU"):
                call(**given)
