"""GPU parity of the unquantised layer and its products where a call is unlike the usual one: outputs on the input,
routing weights that are not finite or far larger than a value, gates whose logits need more than 16 bits."""
import pytest

pytestmark = pytest.mark.gpu

LIMIT = 2.5


def _setup():
    import torch
    assert torch.cuda.is_available()
    from project_aeon_amd import dense, moe
    return torch, dense, moe


def _normal(torch, shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [1, 40])
def test_a_layer_may_write_its_output_over_its_input(tokens, shared):
    """out=x: the layer's own result with an always-on expert, x plus the routed sum without one."""
    torch, dense, moe = _setup()
    dt, E, H, I, k = torch.bfloat16, 8, 256, 128, 2
    w1, w3 = (_normal(torch, (E, I, H), dt, s, H ** -0.5) for s in (1, 2))
    w2 = _normal(torch, (E, H, I), dt, 3, I ** -0.5)
    sh = tuple(_normal(torch, s, dt, 5 + i, s[1] ** -0.5) for i, s in enumerate(((I, H), (I, H), (H, I)))) if shared else None
    layer = moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, router_weight_16=_normal(torch, (E, H), dt, 4, H ** -0.5),
                                    dense_shared=sh)
    x = _normal(torch, (tokens, H), dt, 8)
    start = torch.empty_like(x) if shared else x.clone()
    want, ids, weights = layer.decode(x.clone(), out=start)
    got = layer.decode(x, out=x)
    assert got[0].data_ptr() == x.data_ptr()
    assert torch.equal(got[0], want) and torch.equal(got[1], ids) and torch.equal(got[2], weights)
