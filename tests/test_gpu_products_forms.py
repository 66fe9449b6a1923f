"""GPU parity of the unquantised layer and its products where a call is unlike the usual one: outputs on the input,
routing weights that are not finite or far larger than a value, gates whose logits need more than 16 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LIMIT = 2.5


def _setup():
    import torch
    assert torch.cuda.is_available()
    from project_aeon_amd import dense, moe
    return torch, dense, moe


def _whole(torch, shape, dtype, seed, span=2):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(-span, span + 1, shape, generator=g, device="cuda").to(dtype)


def _normal(torch, shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _mm64(x, w):
    return x.double() @ w.double().t().contiguous()


def _same(torch, got, want):
    """Equal, NaN where NaN is due and nowhere else."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


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


def _spread(torch, tokens, slots, experts):
    """ids that put the draws of a token on different experts, and their lists."""
    ids = (torch.arange(tokens * slots, device="cuda") * 3 % experts).to(torch.int32).view(tokens, slots)
    return ids


# draws and matrices on both sides of what one launch takes, K with and without a last partial chunk of 512, K of
# one lane, K of more chunks than waves
COMBINE_SHAPES = [(1, 8, 16, 1030, 48), (1, 8, 16, 2048, 520), (3, 4, 16, 72, 130), (2, 1, 5, 8, 9), (8, 2, 7, 4104, 24),
                  (1, 3, 5, 7, 16), (1, 64, 80, 520, 24), (2, 32, 7, 1030, 9), (20, 4, 16, 1030, 48), (40, 2, 16, 520, 130)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", COMBINE_SHAPES)
def test_combine_takes_weights_that_are_not_finite(tokens, slots, experts, k, n, dtype):
    """weight * (W_e h + b): an infinite weight gives the product's sign, NaN gives NaN, whatever way the product
    was summed. Whole numbers, so that the products are exact and the 64-bit formula has the same infinities."""
    torch, dense, moe = _setup()
    dt = getattr(torch, dtype)
    ids = _spread(torch, tokens, slots, experts)
    lists = dense.expert_lists(ids, experts)
    draws = lists.draws.long()
    h, w = _whole(torch, (tokens * slots, k), dt, 1), _whole(torch, (experts, n, k), dt, 2)
    b = _whole(torch, (experts, n), dt, 3, 9)
    by_draw = torch.empty(tokens * slots, n, dtype=torch.float64, device="cuda")
    flat = ids.reshape(-1).long()
    for p, d in enumerate(draws.tolist()):
        by_draw[d] = _mm64(h[p:p + 1], w[flat[d]])[0] + b[flat[d]].double()
    by_draw = by_draw.view(tokens, slots, n)
    inf, nan = float("inf"), float("nan")
    for i, special in enumerate((inf, -inf, nan, 0.0)):
        weights = _whole(torch, (tokens, slots), torch.float32, 5)
        weights[i % tokens, i % slots] = special
        print("combine", tokens, slots, experts, k, n, dtype, special, flush=True)
        want = (by_draw * weights.double().unsqueeze(2)).sum(dim=1)
        got = dense.expert_combine(h, w, lists.offsets, lists.draws, ids, weights, bias=b)
        assert _same(torch, got, want.to(dt))
    weights = torch.ones(tokens, slots, device="cuda")
    weights[0, 0], weights[0, slots - 1] = inf, -inf  # NaN where the products have one sign, infinity elsewhere
    want = (by_draw * weights.double().unsqueeze(2)).sum(dim=1)
    assert _same(torch, dense.expert_combine(h, w, lists.offsets, lists.draws, ids, weights, bias=b), want.to(dt))


@pytest.mark.parametrize("tokens", [1, 80])   # in one launch, and in two
@pytest.mark.parametrize("k", [512, 1024, 4096])
def test_combine_weighs_the_product_and_not_its_parts(tokens, k):
    """Parts of 2^11 that cancel to 2^4, times a weight of 2^118: the result is 2^122, though a weighed part would
    be beyond fp32."""
    torch, dense, moe = _setup()
    dt, n = torch.bfloat16, 40
    h = torch.full((tokens, k), 16.0, dtype=dt, device="cuda")
    h[:, torch.arange(k, device="cuda") // 8 % 2 == 1] = -16.0
    h[:, 0] = 17.0
    w = torch.full((2, n, k), 16.0, dtype=dt, device="cuda")
    ids = torch.ones(tokens, 1, dtype=torch.int32, device="cuda")
    lists = dense.expert_lists(ids, 2)
    out = dense.expert_combine(h, w, lists.offsets, lists.draws, ids, torch.full((tokens, 1), 2.0 ** 118, device="cuda"))
    assert bool((out.double() == 2.0 ** 122).all())


@pytest.mark.parametrize("tokens,hidden,experts", [(2100, 4168, 8000), (2100, 4167, 8000), (128, 7168, 1024), (1, 4096, 4096),
                                                   (9000, 72, 256), (0, 64, 8), (4, 64, 1)])
def test_logits_of_any_size(tokens, hidden, experts):
    """dense.router_logits alone, uncut products on the largest tiles among them, into memory that ends with them."""
    torch, dense, moe = _setup()
    x, gate = _whole(torch, (tokens, hidden), torch.bfloat16, 1, 9), _whole(torch, (experts, hidden), torch.bfloat16, 2, 9)
    print("logits", tokens, hidden, experts, flush=True)
    got = dense.router_logits(x, gate)
    assert got.shape == (tokens, experts) and torch.equal(got.double(), _mm64(x, gate))


def test_a_stack_of_unquantised_layers_as_it_defaults():
    """LayerStack(layers, mixes) with nothing else said: the bits of the stack without the fused tail."""
    torch, dense, moe = _setup()
    from project_aeon_amd import synth
    H, I, E, k, tokens, dt = 256, 128, 16, 2, 9, torch.float16
    layers, mixes = [], []
    for l in range(2):
        w1, w3 = (_normal(torch, (E, I, H), dt, 10 * l + s, H ** -0.5) for s in (2, 3))
        w2 = _normal(torch, (E, H, I), dt, 10 * l + 4, I ** -0.5)
        gate = torch.from_numpy(synth.router_weight(l, H, E)).cuda()
        layers.append(moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, router_weight=gate))
        mixes.append(moe.HyperConnection(np.random.default_rng(l).normal(size=24)))
    residual = _normal(torch, (4, tokens, H), dt, 1)
    got = moe.LayerStack(layers, mixes).step(residual.clone())
    want = moe.LayerStack(layers, mixes, fused=False).step(residual.clone())
    assert torch.equal(got, want) and bool(got.isfinite().all())
    # buffers that every layer reuses, twice: nothing of an earlier step stays in them
    scratch = (torch.empty_like(residual), torch.empty_like(residual[0]), torch.empty_like(residual[0]),
               torch.empty(tokens, k, dtype=torch.int32, device="cuda"), torch.empty(tokens, k, device="cuda"))
    for _ in range(2):
        assert torch.equal(moe.LayerStack(layers, mixes).step(residual.clone(), scratch=scratch), want)


@pytest.mark.parametrize("tokens,hidden,experts", [(1, 4096, 256), (1, 100, 7), (3, 512, 24), (20, 7168, 256), (33, 520, 40),
                                                   (64, 4100, 80), (300, 520, 130), (9, 2049, 16), (40, 4101, 80), (5, 7, 4)])
def test_logits_of_a_bf16_gate_are_not_rounded(tokens, hidden, experts):
    """Whole numbers whose sums need more than the 8 bits of bf16: exact in fp32, so the logits have to be the sums.
    Gate rows wider than the matrix, and a routing that only the lower bits decide."""
    torch, dense, moe = _setup()
    dt, I = torch.bfloat16, 8
    w1, w2 = _normal(torch, (experts, I, hidden), dt, 1), _normal(torch, (experts, hidden, I), dt, 2)
    gate = _whole(torch, (experts, hidden + 3), dt, 3, 9)[:, :hidden]
    x = _whole(torch, (tokens, hidden), dt, 4, 9)
    layer = moe.UnquantisedMoeLayer(w1, w1, w2, 2, LIMIT, router_weight_16=gate, score_kind=1)
    got = layer.router_logits(x)
    assert got.dtype == torch.float32
    assert torch.equal(got.double(), _mm64(x, gate))
    # logits 1 + e / 1024, one step of bf16 at 1 apart at most
    x = torch.zeros(tokens, hidden, dtype=dt, device="cuda")
    gate = torch.zeros(experts, hidden, dtype=dt, device="cuda")
    x[:, 0] = x[:, 1] = 1.0
    gate[:, 0], gate[:, 1] = 1.0, torch.arange(experts, device="cuda") % 8 / 1024.0
    layer = moe.UnquantisedMoeLayer(w1, w1, w2, 2, LIMIT, router_weight_16=gate, score_kind=1)
    _, ids, _ = layer.decode(x)
    scores = torch.sigmoid(_mm64(x, gate))
    assert torch.equal(ids.long(), torch.sort(scores, dim=1, descending=True, stable=True).indices[:, :2])


def _gated_halves(torch, product, run, dt):
    """silu(g) * 1 and silu(9) * u of whole-number sums, no clamp: a sum that lacks a term, or has another row's, is
    off by one at least. fp32 moves the exponential in silu by a few |g| * 2^-24 of itself, and the rest by at
    most 16 units of 2^-23; half the type's smallest step may be lost, or 2^-120 of fp32's range."""
    step = torch.finfo(dt).eps / 2
    least = torch.finfo(dt).smallest_normal * step if dt is torch.float16 else 2.0 ** -120
    silu9 = 9.0 * torch.special.expit(torch.tensor(9.0, dtype=torch.float64)).item()
    for up, want, loss in ((False, product * torch.special.expit(product), (4 * product.abs() + 16) * 2.0 ** -23),
                           (True, product * silu9, 64 * 2.0 ** -23)):
        got = run(up)
        loss = want.abs() * loss + least
        assert not bool(((got.double() - want).abs() > step * (want.abs() + loss) + loss).any())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tokens,k,n", [(2100, 4168, 4000), (3000, 4104, 2052), (2100, 4167, 4000), (600, 1000, 1030), (70, 1000, 130),
                                        (3, 512, 48)])
def test_both_halves_of_a_gated_product(tokens, k, n, dtype):
    torch, dense, moe = _setup()
    dt = getattr(torch, dtype)
    x, w = _whole(torch, (tokens, k), dt, 1, 1), _whole(torch, (n, k), dt, 2, 1)
    none, flat = torch.zeros_like(w), lambda v: torch.full((n,), v, dtype=dt, device="cuda")
    print("gated", tokens, k, n, dtype, flush=True)

    def run(up):
        if up:
            return dense.linear(x, none, flat(9.0), activation="swiglu", weight_up=w)
        return dense.linear(x, w, activation="swiglu", weight_up=none, bias_up=flat(1.0))

    product = _mm64(x, w)
    _gated_halves(torch, product, run, dt)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", [(600, 2, 4, 4200, 2080), (300, 6, 24, 264, 1200), (300, 6, 24, 265, 1200),
                                                      (1, 8, 32, 1024, 96), (64, 4, 16, 520, 130)])
def test_both_halves_of_a_gated_expert_product(tokens, slots, experts, k, n, dtype):
    torch, dense, moe = _setup()
    dt = getattr(torch, dtype)
    ids = _spread(torch, tokens, slots, experts)
    lists = dense.expert_lists(ids, experts)
    x, w = _whole(torch, (tokens, k), dt, 1, 1), _whole(torch, (experts, n, k), dt, 2, 1)
    none, flat = torch.zeros_like(w), lambda v: torch.full((experts, n), v, dtype=dt, device="cuda")
    print("gated experts", tokens, slots, experts, k, n, dtype, flush=True)

    def run(up):
        if up:
            return dense.expert_linear(x, none, lists.offsets, lists.rows, bias=flat(9.0), activation="swiglu", weight_up=w)
        return dense.expert_linear(x, w, lists.offsets, lists.rows, activation="swiglu", weight_up=none, bias_up=flat(1.0))

    product = torch.zeros(tokens * slots, n, dtype=torch.float64, device="cuda")
    bounds = lists.offsets.tolist()
    for e in range(experts):
        at = slice(bounds[e], bounds[e + 1])
        product[at] = _mm64(x[lists.rows[at].long()], w[e])
    _gated_halves(torch, product, run, dt)
