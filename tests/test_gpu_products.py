"""GPU parity of the products over unquantised fp16 / bf16 weights (aeon_linear, aeon_expert_linear,
aeon_expert_combine) against 64-bit evaluations of their definitions.

Two kinds of inputs. Small whole numbers: every product and partial sum is exact in fp32 whatever the
order, so the result has to be the exact sum rounded once, bit for bit. Normal values: an element may be
off by half a step of its type (finfo.eps / 2 of its size) plus what an fp32 sum of K terms can lose,
K * 2^-23 * sum |x w| for any order, times the slope of what follows (at most 1.13 for silu and both gelus)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LIMIT = 2.5


def _setup():
    import torch
    assert torch.cuda.is_available()
    from project_aeon_amd import dense
    return torch, dense


def _dtype(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


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


def _act64(torch, kind, g, u=None):
    if kind == "silu":
        return g * torch.special.expit(g)
    if kind == "gelu":
        return 0.5 * g * torch.special.erfc(-g * 0.5 ** 0.5)
    if kind == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh((2 / np.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    if kind == "swiglu":
        g = torch.where(g > LIMIT, torch.full_like(g, LIMIT), g)
        u = torch.where(u > LIMIT, torch.full_like(u, LIMIT), torch.where(u < -LIMIT, torch.full_like(u, -LIMIT), u))
        return g * torch.special.expit(g) * u
    return g


def _near(torch, got, want, loss):
    """|got - want| <= half a step of want's size + loss (a 64-bit tensor or number)."""
    step = torch.finfo(got.dtype).eps / 2
    bad = (got.double() - want).abs() > step * (want.abs() + loss) + loss
    assert not bool(bad.any()), "%d of %d off, worst %.3e" % (
        int(bad.sum()), bad.numel(), float((got.double() - want).abs().max()))


def _loss(x, w, slope=1.2):
    return slope * x.shape[1] * 2.0 ** -23 * _mm64(x.abs(), w.abs())


# tokens x in x out: every tile form, each with ragged edges in all three dimensions, K below one step, K of
# one step, K with and without a last partial step, K long enough to be cut into shares
LINEAR_SHAPES = [(1, 64, 16), (1, 4096, 256), (1, 1, 1), (2, 7, 3), (3, 72, 130), (15, 128, 64), (16, 2048, 65), (17, 192, 96),
                 (32, 1032, 200), (33, 64, 64), (64, 4100, 80), (65, 320, 1000), (130, 136, 4104),
                 (300, 200, 5000), (1000, 64, 4300), (4000, 200, 3300), (2050, 8, 8200)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,k,n", LINEAR_SHAPES)
def test_linear_of_whole_numbers_is_exact(tokens, k, n, dtype):
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    x, w = _whole(torch, (tokens, k), dt, 1), _whole(torch, (n, k), dt, 2)
    b, r = _whole(torch, (n,), dt, 3, 9), _whole(torch, (tokens, n), dt, 4, 9)
    guard = torch.full((tokens + 1, n), 77.0, dtype=dt, device="cuda")
    print("linear", tokens, k, n, dtype, flush=True)
    dense.linear(x, w, out=guard[:tokens])
    want = _mm64(x, w)
    assert torch.equal(guard[:tokens], want.to(dt))
    assert bool((guard[tokens] == 77.0).all())
    assert torch.equal(dense.linear(x, w, b, residual=r), (want + b.double() + r.double()).to(dt))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("x_pad,w_pad,y_pad,shift", [(8, 16, 4, 0), (3, 8, 1, 0), (8, 8, 8, 1), (1, 1, 3, 5), (4, 4, 2, 4)])
@pytest.mark.parametrize("tokens,k,n", [(5, 200, 72), (40, 130, 33), (260, 65, 300), (3000, 72, 5001)])
def test_linear_with_pitches_and_bases_off_every_boundary(tokens, k, n, x_pad, w_pad, y_pad, shift, dtype):
    """Rows wider than the matrices and bases that start `shift` elements into their buffers: the exact result,
    and nothing written between the rows."""
    torch, dense = _setup()
    dt = _dtype(torch, dtype)

    def inside(rows, cols, pad, fill, seed=None):
        flat = torch.full((rows * (cols + pad) + shift,), fill, dtype=dt, device="cuda")
        view = flat[shift:].view(rows, cols + pad)
        if seed is not None:
            view[:, :cols] = _whole(torch, (rows, cols), dt, seed)
        return view

    x, w, r = inside(tokens, k, x_pad, float("nan"), 1), inside(n, k, w_pad, float("nan"), 2), inside(tokens, n, y_pad, 5.0, 3)
    y = inside(tokens, n, y_pad, 77.0)
    dense.linear(x[:, :k], w[:, :k], residual=r[:, :n], out=y[:, :n])
    assert torch.equal(y[:, :n], (_mm64(x[:, :k], w[:, :k]) + r[:, :n].double()).to(dt))
    assert bool((y[:, n:] == 77.0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("tokens,k,n", [(1, 512, 48), (1, 2048, 100), (20, 333, 129), (70, 1000, 260), (600, 256, 2304), (4100, 96, 2052)])
def test_linear_activations(tokens, k, n, act, dtype):
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    x = _normal(torch, (tokens, k), dt, 5)
    w = _normal(torch, (n, k), dt, 6, 1.5 / k ** 0.5)
    b = _normal(torch, (n,), dt, 7)
    r = _normal(torch, (tokens, n), dt, 8)
    kw, g, u = {}, _mm64(x, w) + b.double(), None
    loss = _loss(x, w)
    if act == "swiglu":
        w3, b3 = _normal(torch, (n, k), dt, 9, 1.5 / k ** 0.5), _normal(torch, (n,), dt, 10)
        kw = dict(weight_up=w3, bias_up=b3, swiglu_limit=LIMIT)
        u = _mm64(x, w3) + b3.double()
        loss = LIMIT * (loss + _loss(x, w3))   # silu(g) and u are at most LIMIT
    want = _act64(torch, act, g, u) + r.double()
    got = dense.linear(x, w, b, activation=act, residual=r, **kw)
    _near(torch, got, want, loss + 2.0 ** -20 * (want.abs() + r.double().abs() + 1))
    # the same with the output on the residual, twice: the summation order is fixed
    assert torch.equal(dense.linear(x, w, b, activation=act, residual=r, out=r, **kw), got)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,k", [(3, 100), (40, 1024), (700, 264)])
def test_linear_keeps_inf_and_nan_in_their_own_rows(tokens, k, dtype):
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    n = 96
    x, w = _normal(torch, (tokens, k), dt, 1), _normal(torch, (n, k), dt, 2, k ** -0.5)
    w3 = _normal(torch, (n, k), dt, 3, k ** -0.5)
    clean = dense.linear(x, w, weight_up=w3, activation="swiglu", swiglu_limit=LIMIT)
    bad = x.clone()
    bad[1, k - 1] = float("nan")
    got = dense.linear(bad, w, weight_up=w3, activation="swiglu", swiglu_limit=LIMIT)
    assert bool(got[1].isnan().all())
    keep = torch.arange(tokens, device="cuda") != 1
    assert torch.equal(got[keep], clean[keep])
    w[5, 0] = float("inf")
    x[0, 0], x[2, 0] = 1.0, -1.0
    got = dense.linear(x, w)
    assert float(got[0, 5]) == float("inf") and float(got[2, 5]) == float("-inf")
    others = torch.arange(n, device="cuda") != 5
    assert bool(got[:, others].isfinite().all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_activations_far_from_zero(act, dtype):
    """act(g) of exact g from -14 to 14 (g times a one in the first column), element by element: half a step of
    the type, plus what fp32 loses: an argument z of an exponential, rounded in a few operations, moves the
    exponential by a few |z| * 2^-24 of itself, and the rest is at most 16 units of 2^-23. What is below the
    type's smallest step, or 2^-120 in fp32, may be lost."""
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    g = torch.linspace(-14, 14, 3601, dtype=torch.float64, device="cuda").to(dt)
    x, w = torch.zeros(g.numel(), 64, dtype=dt, device="cuda"), torch.zeros(16, 64, dtype=dt, device="cuda")
    x[:, 0], w[:, 0] = g, 1.0
    got, g = dense.linear(x, w, activation=act), g.double()
    z = {"silu": g, "gelu": g * g / 2, "gelu_tanh": 2 * (2 / np.pi) ** 0.5 * (g + 0.044715 * g ** 3)}[act]
    want = 0.5 * g * torch.special.erfc(-g * 0.5 ** 0.5) if act == "gelu" else g * torch.special.expit(z)
    loss = want.abs() * (4 * z.abs() + 16) * 2.0 ** -23
    least = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 if dtype == "f16" else 2.0 ** -120
    _near(torch, got, want[:, None].expand_as(got), (loss + least)[:, None])


@pytest.mark.parametrize("tokens", [1, 8, 40, 300])
def test_linear_keeps_subnormal_numbers(tokens):
    """Subnormal inputs with exact sums, and sums that are subnormal themselves: 64 equal powers of two."""
    torch, dense = _setup()
    for dt, low, high in ((torch.float16, -24, 10), (torch.bfloat16, -133, 100), (torch.float16, -14, -15),
                          (torch.bfloat16, -70, -66)):
        x = torch.full((tokens, 64), 2.0 ** low, dtype=torch.float64, device="cuda").to(dt)
        w = torch.full((128, 64), 2.0 ** high, dtype=dt, device="cuda")
        assert bool((dense.linear(x, w).double() == 64 * 2.0 ** (low + high)).all())


# long enough for the largest tiles: a last round cut into halves and a last window of 52 positions, shares of
# K of the two largest tiles with a partial last step, and a row pitch that is off every 4-byte boundary
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,k,n", [(2100, 4168, 8000), (400, 7170, 7100), (520, 4104, 2100), (250, 7176, 7000),
                                        (3000, 4104, 4104), (2100, 4167, 8000)])
def test_linear_on_the_largest_tiles_is_exact(tokens, k, n, gated, dtype):
    """Whole numbers as above. Gated, the gate is a constant 0 + bias beyond the clamp, so that the result is
    silu(LIMIT) times the clamped whole-number product."""
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    print("linear", tokens, k, n, gated, dtype, flush=True)
    x = _whole(torch, (tokens, k), dt, 1)
    if not gated:
        w, b, r = _whole(torch, (n, k), dt, 2), _whole(torch, (n,), dt, 3, 9), _whole(torch, (tokens, n), dt, 4, 9)
        guard = torch.full((tokens + 1, n), 77.0, dtype=dt, device="cuda")
        dense.linear(x, w, b, residual=r, out=guard[:tokens])
        assert torch.equal(guard[:tokens], (_mm64(x, w) + b.double() + r.double()).to(dt))
        assert bool((guard[tokens] == 77.0).all())
        return
    w, up = _whole(torch, (2, n // 2, k), dt, 2, 1)
    w.zero_()
    b = torch.full((n // 2,), 9.0, dtype=dt, device="cuda")
    got = dense.linear(x, w, b, activation="swiglu", weight_up=up, swiglu_limit=LIMIT)
    silu = LIMIT * torch.special.expit(torch.tensor(LIMIT, dtype=torch.float64)).item()
    want = _mm64(x, up).clamp(-LIMIT, LIMIT) * silu
    _near(torch, got, want, 2.0 ** -20 * want.abs())


def _lists(torch, ids, experts):
    """What the permutation defines: draws sorted by expert, ascending inside one; ids outside are dropped."""
    flat = ids.reshape(-1).cpu().numpy()
    order = [d for e in range(experts) for d in np.nonzero(flat == e)[0]]
    counts = [int((flat == e).sum()) for e in range(experts)]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    draws = torch.zeros(flat.size, dtype=torch.int32, device="cuda")
    draws[:len(order)] = torch.tensor(np.array(order, dtype=np.int32), device="cuda")
    return offsets, draws


def _ids(torch, kind, tokens, slots, experts, seed):
    rng = np.random.default_rng(seed)
    if kind == "even":
        ids = rng.integers(0, experts, (tokens, slots))
    elif kind == "one":          # every draw the same expert, twice in a token too
        ids = np.full((tokens, slots), experts - 1)
    elif kind == "ends":         # only the first and the last expert
        ids = rng.choice([0, experts - 1], (tokens, slots))
    elif kind == "dropped":      # some ids name no expert
        ids = rng.integers(-2, experts + 2, (tokens, slots))
    else:                        # none does
        ids = np.full((tokens, slots), experts)
    return torch.tensor(ids, dtype=torch.int32, device="cuda")


EXPERT_SHAPES = [(1, 1, 1, 64, 32), (1, 8, 256, 128, 64), (3, 2, 5, 100, 33), (16, 4, 64, 256, 40), (50, 3, 7, 65, 129),
                 (129, 2, 1000, 64, 48), (400, 6, 24, 136, 200), (900, 2, 3, 72, 260), (700, 1, 1, 64, 520),
                 (200, 2, 4, 72, 5000), (700, 2, 3, 72, 8200), (1100, 1, 1, 264, 12000), (700, 3, 9, 193, 2600),
                 (300, 6, 24, 72, 2300), (300, 6, 24, 67, 2300), (33, 2, 140, 128, 64), (8, 1, 16, 4104, 680),
                 (33, 2, 66, 128, 64), (8, 1, 9, 4104, 680)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["even", "one", "ends", "dropped", "none"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", EXPERT_SHAPES)
def test_expert_products_of_whole_numbers_are_exact(tokens, slots, experts, k, n, kind, dtype):
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    ids = _ids(torch, kind, tokens, slots, experts, tokens)
    offsets, draws = _lists(torch, ids, experts)
    live = int(offsets[-1])
    rows = draws // slots
    x, w = _whole(torch, (tokens, k), dt, 1), _whole(torch, (experts, n, k), dt, 2)
    b = _whole(torch, (experts, n), dt, 3, 9)
    print("experts", tokens, slots, experts, k, n, kind, dtype, flush=True)
    y = torch.full((tokens * slots, n), 77.0, dtype=dt, device="cuda")
    dense.expert_linear(x, w, offsets, rows, bias=b, out=y)
    want = torch.full((tokens * slots, n), 77.0, dtype=torch.float64, device="cuda")
    bounds = offsets.tolist()
    for e in range(experts):
        at = slice(bounds[e], bounds[e + 1])
        if bounds[e] < bounds[e + 1]:
            want[at] = _mm64(x[rows[at].long()], w[e]) + b[e].double()
    assert torch.equal(y, want.to(dt))           # rows behind the last list among them
    # without a row list position p takes row p
    gathered = x[rows.long()]
    again = torch.full_like(y, 77.0)
    dense.expert_linear(gathered, w, offsets, bias=b, out=again)
    assert torch.equal(again, y)
    # the way back: whole weights, so the sums over the slots are exact too
    h = gathered
    weights = _whole(torch, (tokens, slots), torch.float32, 5)
    base = _whole(torch, (tokens, n), dt, 6, 9)
    out = base.double()
    for s in range(slots):
        for t_ids in (ids[:, s],):
            ok = (t_ids >= 0) & (t_ids < experts)
            by_draw = torch.zeros(tokens * slots, n, dtype=torch.float64, device="cuda")
            by_draw[draws[:live].long()] = want[:live]
            got = by_draw.view(tokens, slots, n)[:, s] * weights[:, s].double().unsqueeze(1)
            out = out + torch.where(ok.unsqueeze(1), got, torch.zeros_like(got))
    got = dense.expert_combine(h, w, offsets, draws, ids, weights, bias=b, base=base)
    assert torch.equal(got, out.to(dt))
    assert torch.equal(dense.expert_combine(h, w, offsets, draws, ids, weights, bias=b, base=base, out=base), got)
    no_base = dense.expert_combine(h, w, offsets, draws, ids, weights)
    if live == 0:
        assert bool((no_base == 0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", [(1, 8, 32, 1024, 96), (2, 8, 32, 1030, 96), (64, 4, 16, 520, 130),
                                                      (600, 2, 6, 256, 192), (600, 2, 4, 4200, 4160), (300, 6, 24, 264, 1200),
                                                      (300, 6, 24, 265, 1200)])
def test_expert_gate_up_and_combine_of_normal_values(tokens, slots, experts, k, n, dtype):
    torch, dense = _setup()
    dt = _dtype(torch, dtype)
    ids = _ids(torch, "even", tokens, slots, experts, 3)
    offsets, draws = _lists(torch, ids, experts)
    rows = draws // slots
    bounds = offsets.tolist()
    x = _normal(torch, (tokens, k), dt, 1)
    w1, w3 = (_normal(torch, (experts, n, k), dt, s, 1.5 / k ** 0.5) for s in (2, 3))
    h = dense.expert_linear(x, w1, offsets, rows, weight_up=w3, activation="swiglu", swiglu_limit=LIMIT)
    for e in range(experts):
        at = slice(bounds[e], bounds[e + 1])
        xe = x[rows[at].long()]
        loss = LIMIT * (_loss(xe, w1[e]) + _loss(xe, w3[e])) + 2.0 ** -18
        _near(torch, h[at], _act64(torch, "swiglu", _mm64(xe, w1[e]), _mm64(xe, w3[e])), loss)
    w2 = _normal(torch, (experts, k, n), dt, 4, 1.5 / n ** 0.5)
    weights = torch.rand(tokens, slots, device="cuda") + 0.1
    base = _normal(torch, (tokens, k), dt, 5)
    out = dense.expert_combine(h, w2, offsets, draws, ids, weights, base=base)
    want, loss = base.double(), torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    for e in range(experts):
        at = slice(bounds[e], bounds[e + 1])
        d = draws[at].long()
        scale = weights.reshape(-1)[d].double().unsqueeze(1)
        want.index_add_(0, d // slots, _mm64(h[at], w2[e]) * scale)
        loss.index_add_(0, d // slots, _loss(h[at], w2[e]) * scale)
    # slots + 2 more fp32 roundings of values no larger than the sum of the sizes
    loss = loss + (slots + 2) * 2.0 ** -23 * (want.abs() + loss * k + 8)
    _near(torch, out, want, loss)


def test_rows_out_of_range_are_left_alone():
    """A row index that names no row of x: the position's output stays as it was, the others are exact."""
    torch, dense = _setup()
    dt = torch.bfloat16
    x, w = _whole(torch, (6, 64), dt, 1), _whole(torch, (2, 48, 64), dt, 2)
    offsets = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, -1, 5, 6, 3, 3, 1 << 30, 2], dtype=torch.int32, device="cuda")
    y = torch.full((8, 48), 77.0, dtype=dt, device="cuda")
    dense.expert_linear(x, w, offsets, rows, out=y)
    for p, r in enumerate(rows.tolist()):
        want = _mm64(x[r:r + 1], w[0 if p < 3 else 1])[0].to(dt) if 0 <= r < 6 else torch.full_like(y[p], 77.0)
        assert torch.equal(y[p], want)


def test_offsets_past_32_bits():
    """Expert matrices, activation rows and output rows more than 2^32 bytes into their buffers."""
    torch, dense = _setup()
    dt = torch.float16
    far = 1 << 30                                  # elements: 2 GiB apart
    w = torch.empty(4 * far + 64 * 72, dtype=dt, device="cuda").as_strided((5, 64, 72), (far, 72, 1))
    values = _whole(torch, (5, 64, 72), dt, 1)
    w.copy_(values)
    x = torch.empty(5 * far + 72, dtype=dt, device="cuda").as_strided((6, 72), (far, 1))
    x.copy_(_whole(torch, (6, 72), dt, 2))
    offsets = torch.tensor([0, 1, 2, 4, 5, 6], dtype=torch.int32, device="cuda")
    y = torch.empty(5 * far + 64, dtype=dt, device="cuda").as_strided((6, 64), (far, 1))
    dense.expert_linear(x, w, offsets, out=y)
    expert = [0, 1, 2, 2, 3, 4]
    for p, e in enumerate(expert):
        assert torch.equal(y[p], _mm64(x[p:p + 1], values[e])[0].to(dt))
    dense.linear(x, values[0], residual=y, out=y)
    for p, e in enumerate(expert):
        assert torch.equal(y[p], (_mm64(x[p:p + 1], values[e]) + _mm64(x[p:p + 1], values[0]))[0].to(dt))


def test_empty_calls():
    torch, dense = _setup()
    dt = torch.bfloat16
    w = _whole(torch, (3, 16, 24), dt, 1)
    none = torch.empty(0, 24, dtype=dt, device="cuda")
    assert dense.linear(none, w[0]).shape == (0, 16)
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    rows = torch.empty(0, dtype=torch.int32, device="cuda")
    assert dense.expert_linear(_whole(torch, (2, 24), dt, 2), w, offsets, rows).shape == (0, 16)
    ids = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    assert dense.expert_combine(none, w, offsets, rows, ids, ids.float()).shape == (0, 16)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_layer_of_no_tokens_and_what_it_refuses(dtype):
    torch, dense = _setup()
    from project_aeon_amd import moe
    dt = _dtype(torch, dtype)
    E, H, I, k = 4, 128, 64, 2
    w1, w3, w2 = _normal(torch, (E, I, H), dt, 1), _normal(torch, (E, I, H), dt, 2), _normal(torch, (E, H, I), dt, 3)
    kw = (dict(router_weight=_normal(torch, (H, E), torch.float32, 4)) if dtype == "f16"
          else dict(router_weight_16=_normal(torch, (E, H), dt, 4)))
    layer = moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, **kw)
    out, ids, weights = layer.decode(torch.empty(0, H, dtype=dt, device="cuda"))
    assert out.shape == (0, H) and ids.shape == (0, k) and weights.shape == (0, k)
    x = _normal(torch, (3, H), dt, 5)
    for bad in (x[:, :64], x.float(), x.reshape(-1), x.cpu(), x.bfloat16() if dtype == "f16" else x.half()):
        with pytest.raises((ValueError, IndexError)):
            layer.decode(bad)
    for given in (dict(ids=torch.empty(3, k, dtype=torch.int64, device="cuda")), dict(ids=torch.empty(2, k, dtype=torch.int32, device="cuda")),
                  dict(weights=torch.empty(3, k, dtype=dt, device="cuda"))):
        with pytest.raises(ValueError):
            layer.decode(x, **given)
    with pytest.raises(ValueError, match="router_bias"):
        moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, router_bias=_normal(torch, (E + 1,), torch.float32, 6), **kw)
    # one row that carries a stride of its own
    row = _normal(torch, (H, 1), dt, 7).t()
    assert row.stride() != (H, 1)
    a, b = layer.decode(row), layer.decode(row.contiguous().clone())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_side_stream_and_two_captured_graphs():
    """The calls on a stream of their own, captured into two graphs that replay in turns between eager
    calls: every replay has the eager result of what its inputs hold then."""
    torch, dense = _setup()
    dt = torch.bfloat16
    tokens, slots, experts, k, n = 12, 2, 6, 1024, 96
    w = _normal(torch, (n, k), dt, 1, k ** -0.5)
    we = _normal(torch, (experts, n, k), dt, 2, k ** -0.5)
    wd = _normal(torch, (experts, k, n), dt, 3, n ** -0.5)
    ids = _ids(torch, "even", tokens, slots, experts, 1)
    offsets, draws = _lists(torch, ids, experts)
    rows = draws // slots
    weights = torch.rand(tokens, slots, device="cuda")

    def step(x):
        h = dense.expert_linear(x, we, offsets, rows, activation="silu")
        return dense.linear(x, w), dense.expert_combine(h, wd, offsets, draws, ids, weights, base=x)

    x = [_normal(torch, (tokens, k), dt, 10 + i) for i in range(2)]
    eager = [step(v) for v in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for v, e in zip(x, eager):
            assert all(torch.equal(a, b) for a, b in zip(step(v), e))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(v))
        graphs.append(g)
    for i in range(4):
        for v in x:
            v.copy_(_normal(torch, (tokens, k), dt, 100 + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for v, o in zip(x, outs):
            assert all(torch.equal(a, b) for a, b in zip(o, step(v)))


def test_expert_lists_are_the_permutation():
    torch, dense = _setup()
    for kind in ("even", "one", "dropped"):
        ids = _ids(torch, kind, 40, 3, 9, 4)
        offsets, draws = _lists(torch, ids, 9)
        got = dense.expert_lists(ids, 9)
        live = int(offsets[-1])
        assert torch.equal(got.offsets, offsets) and torch.equal(got.draws[:live], draws[:live])
        assert torch.equal(got.rows[:live], draws[:live] // 3)


def _routed64(torch, x, w1, w3, w2, ids, weights, limit, base):
    """The layer's expert part in 64 bits with the hidden rows rounded to their type."""
    out = base.double()
    for e in range(w1.shape[0]):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        g, u = _mm64(x[t], w1[e]).clamp(max=limit), _mm64(x[t], w3[e]).clamp(-limit, limit)
        h = (g * torch.special.expit(g) * u).to(x.dtype)
        out.index_add_(0, t, _mm64(h, w2[e]) * weights[t, s].double().unsqueeze(1))
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [1, 7, 64, 500])
def test_unquantised_layer_as_used(tokens, shared, dtype):
    """Router, lists, gate and up, the weighted sum and the always-on expert run together. The hidden row's
    rounding may fall to the other side of a tie in fp32 (one step of a hidden value, weighed by w2), so the
    output is held to two steps of its type over the size of what was summed."""
    torch, dense = _setup()
    from project_aeon_amd import moe
    dt = _dtype(torch, dtype)
    H, I, E, k = 512, 256, 16, 4
    x = _normal(torch, (tokens, H), dt, 1)
    w1, w3 = (_normal(torch, (E, I, H), dt, s, 1.5 / H ** 0.5) for s in (2, 3))
    w2 = _normal(torch, (E, H, I), dt, 4, I ** -0.5)
    sh = tuple(_normal(torch, s, dt, 5 + i, s[1] ** -0.5) for i, s in enumerate(((I, H), (I, H), (H, I)))) if shared else None
    gate = _normal(torch, (E, H), dt, 9, H ** -0.5)
    bias = _normal(torch, (E,), torch.float32, 10, 0.1)
    layer = moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, router_bias=bias, router_weight_16=gate, dense_shared=sh)
    out, ids, weights = layer.decode(x)
    scores = torch.sigmoid(layer.router_logits(x).double())
    want_ids = torch.sort(scores + bias.double(), dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    assert torch.equal(ids, want_ids)
    picked = torch.gather(scores, 1, ids.long())
    assert float((weights.double() - picked / picked.sum(1, keepdim=True)).abs().max()) < 1e-6
    base = torch.zeros(tokens, H, dtype=dt, device="cuda")
    if shared:
        g, u = _mm64(x, sh[0]).clamp(max=LIMIT), _mm64(x, sh[1]).clamp(-LIMIT, LIMIT)
        base = _mm64((g * torch.special.expit(g) * u).to(dt), sh[2]).to(dt)
    want = _routed64(torch, x, w1, w3, w2, ids, weights, LIMIT, base)
    assert float((out.double() - want).abs().max()) <= 2 * torch.finfo(dt).eps * float(want.abs().max())
    # the routed part alone adds to what the output holds
    if not shared:
        start = _normal(torch, (tokens, H), dt, 20)
        want = _routed64(torch, x, w1, w3, w2, ids, weights, LIMIT, start)
        got = layer.routed(x, ids, weights, out=start)
        assert got.data_ptr() == start.data_ptr()
        assert float((got.double() - want).abs().max()) <= 2 * torch.finfo(dt).eps * float(want.abs().max())


def test_unquantised_layers_in_a_stack():
    """LayerStack runs over unquantised layers: the new residual is the static mix of each layer's output, and
    a layer with the fp32 gate selects what MoeLayer's router entry points select."""
    torch, dense = _setup()
    from project_aeon_amd import moe, synth
    H, I, E, k, tokens = 256, 128, 16, 2, 9
    dt = torch.float16
    layers, mixes = [], []
    for l in range(2):
        w1, w3 = (_normal(torch, (E, I, H), dt, 10 * l + s, H ** -0.5) for s in (2, 3))
        w2 = _normal(torch, (E, H, I), dt, 10 * l + 4, I ** -0.5)
        gate = torch.from_numpy(synth.router_weight(l, H, E)).cuda()
        layers.append(moe.UnquantisedMoeLayer(w1, w3, w2, k, LIMIT, router_weight=gate))
        mixes.append(moe.HyperConnection(np.random.default_rng(l).normal(size=24)))
    residual = _normal(torch, (4, tokens, H), dt, 1)
    trace = []
    final = moe.LayerStack(layers, mixes, fused=False).step(residual.clone(), trace=trace)
    assert len(trace) == 2 and bool(final.isfinite().all())
    for layer, hc, (r_in, x_pre, x, ids, w, y, r_out) in zip(layers, mixes, trace):
        assert torch.equal(layer.decode(x)[0], y)
        want = _routed64(torch, x, layer.w1, layer.w3, layer.w2, ids, w, LIMIT, torch.zeros_like(x))
        assert float((y.double() - want).abs().max()) <= 2 * torch.finfo(dt).eps * float(want.abs().max())
        again = torch.empty_like(r_out)
        assert torch.equal(hc.post_mix(y, r_in, again), r_out)
