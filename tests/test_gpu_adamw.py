"""The AdamW step over many tensors (adamw.hip) against 64 bits.

Bounds, with u = 2^-24 and e the half step of the type that is written (finfo.eps / 2):
  g   the factor and the product: 2 u |g| (none without a norm)
  m   b1 and 1 - b1 rounded to fp32, a product and a sum rounded: 3 u (|b1 m| + |(1 - b1) g|) + g's
  v   the same and the square's rounding: 4 u v + 2 g's
  p   decay and product 2 u |p|, sum u; step: size, root and eps rounded, square root, sum,
      quotient and product: 7 u of it, m's error, half of v's: then e |p|
8 bits: a code is that of the 64-bit moment, rounded with the same random bits, unless its fp32 error
(4 u, 8 units of the 20 random bits' 2^-23 or less) crosses the border: 2^-17 of them on average, and then
its neighbour in value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
MANY = [(256, 256), (256,), (1,), (0, 5), (3, 7, 5), (27, 8, 3, 3), (27,), (130, 129)] * 20
SHAPES = {"one": [(1,)], "two": [(5,), (3, 3)], "edges": [(127,), (128,), (129,), (2047,), (2049,)],
          "many": MANY, "large": [(2 ** 20 + 5,), (3,)], "empty": [(0,), (0, 3), (4,)]}
BLOCK = 128


def _up(n):
    return -(-n // BLOCK) * BLOCK


def _flat(tensors):
    """As the moments lie, in 64 bits, zeros between."""
    out = torch.zeros(sum(_up(t.numel()) for t in tensors), dtype=torch.float64)
    at = 0
    for t in tensors:
        out[at:at + t.numel()] = t.detach().cpu().double().flatten()
        at += _up(t.numel())
    return out


def _mix(x):
    for shift, mult in ((15, 0x9E3779B1), (13, 0xB504F333), (16, 0x9E3779B1)):
        x = (x & 0xffffffff) * mult & 0xffffffff  # wraps in int64, the low 32 bits are right
        x = x ^ (x >> shift)
    return x


def _random(total, step, seed):
    key = torch.zeros(1, dtype=torch.int64)
    for word in (seed & 0xffffffff, seed >> 32, step & 0xffffffff, step >> 32):
        key = _mix(key + word)
    return _mix(torch.arange(total) + _mix(key))


def _encode(v, random, top):
    bits = v.float().view(torch.int32).long()
    scale = ((bits.view(-1, BLOCK).amax(1) + 0xfffff) >> 23).clamp(top + 1, 255)
    q = ((bits + random * 16 + 8) >> 20) - ((scale - top) * 8).repeat_interleave(BLOCK)
    least = (v > 0) * 8 if top == 31 else torch.zeros_like(q)
    return torch.where(q < 8, least, q.clamp(max=top * 8 + 7)), scale


def _decode(codes, scale, top):
    q = codes.long() & (top * 8 + 7)
    bits = (q + ((scale.long() - top) * 8).repeat_interleave(BLOCK)) << 20
    return torch.where(q < 8, 0, bits).int().view(torch.float32).double()


def _signed(codes, scale):
    return _decode(codes, scale, 15) * torch.where(codes >= 128, -1.0, 1.0)


def _moments(state):
    if state["exp_avg"].dtype == torch.float32:
        return state["exp_avg"].cpu().double(), state["exp_avg_sq"].cpu().double()
    return (_signed(state["exp_avg"].cpu(), state["exp_avg_scale"].cpu()),
            _decode(state["exp_avg_sq"].cpu(), state["exp_avg_sq_scale"].cpu(), 31))


class Reference:
    """One step in 64 bits from what the tensors hold now."""

    def __init__(self, params, grads, state, lr, betas, eps, wd, norm, max_norm):
        (b1, b2), t = betas, state["step"].item() + 1
        m, v = _moments(state)
        p, g = _flat(params), _flat(grads)
        by = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
        g = g * by
        g_err = 0 if max_norm is None else 2 * U * g.abs()
        self.m_err = 3 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + (1 - b1) * g_err
        self.m = b1 * m + (1 - b1) * g
        self.v = b2 * v + (1 - b2) * g * g
        self.v_err = 4 * U * self.v + 2 * (1 - b2) * g.abs() * g_err
        den = torch.sqrt(self.v / (1 - b2 ** t)) + eps
        up = lr / (1 - b1 ** t) * torch.where(self.m == 0, 0.0, self.m / den)
        self.p = (1 - lr * wd) * p - up
        rel = 7 * U + 0.5 * self.v_err / self.v.clamp(min=1e-300)
        self.p_err = 3 * U * (p.abs() + up.abs()) + up.abs() * rel + lr / (1 - b1 ** t) * torch.where(
            self.m_err == 0, 0.0, self.m_err / den)
        self.random = _random(p.numel(), t, state.get("seed", 0))


def _inside(got, want, err, dtype, what):
    half = torch.finfo(dtype).eps / 2
    bound = err + half * (want.abs() + err) + torch.finfo(dtype).smallest_normal * half
    off = (got - want).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


def _setup(shapes, ptypes, gtypes, seed, scale=0.01):
    g = torch.Generator().manual_seed(seed)
    params = [(0.1 * torch.randn(*s, generator=g)).to(ptypes[k % len(ptypes)]).to(DEV) for k, s in enumerate(shapes)]
    grads = [[(scale * torch.randn(*s, generator=g)).to(gtypes[k % len(gtypes)]).to(DEV)
              for k, s in enumerate(shapes)] for _ in range(3)]
    return params, grads


def _near_codes(got, want, top, what):
    got, want = got.cpu().long(), want.long()
    far = (got - want).abs()
    off = int((far > 0).sum())
    assert off <= 2 + got.numel() * 2.0 ** -15, f"{what}: {off} of {got.numel()} codes"
    assert far.max() <= 1 or top == 31 and far.max() <= 8, what


def _check_step(params, grads, state, lr, betas, eps, wd, max_norm, copies):
    import modulated_deform_conv as mdc
    norm = mdc.grad_norm(grads) if max_norm is not None else None
    r = Reference(params, grads, state, lr, betas, eps, wd, norm.item() if max_norm is not None else None,
                  max_norm)
    before = state["step"].item()
    mdc.adamw_step_(params, grads, state, lr=lr, betas=betas, eps=eps, weight_decay=wd, norm=norm,
                    max_norm=max_norm, copies=copies)
    assert state["step"].item() == before + 1
    at = 0
    for k, p in enumerate(params):
        part = slice(at, at + p.numel())
        for got in [p] + ([copies[k]] if copies is not None else []):
            # a copy is rounded from the fp32 value, as the parameter is
            _inside(got.cpu().double().flatten(), r.p[part], r.p_err[part], got.dtype, f"tensor {k}")
        at += _up(p.numel())
    if state["exp_avg"].dtype == torch.float32:
        _inside(state["exp_avg"].cpu().double(), r.m, r.m_err, torch.float32, "exp_avg")
        _inside(state["exp_avg_sq"].cpu().double(), r.v, r.v_err, torch.float32, "exp_avg_sq")
    else:
        codes, scale = _encode(r.m.abs(), r.random >> 16, 15)
        assert torch.equal(state["exp_avg_scale"].cpu().long(), scale)
        _near_codes(state["exp_avg"].cpu() % 128, codes, 15, "exp_avg")
        minus = state["exp_avg"].cpu() >= 128
        assert torch.equal(minus & (codes > 0), (r.m < 0) & (codes > 0))
        codes, scale = _encode(r.v, r.random & 0xffff, 31)
        assert torch.equal(state["exp_avg_sq_scale"].cpu().long(), scale)
        _near_codes(state["exp_avg_sq"], codes, 31, "exp_avg_sq")
        m, v = mdc.adamw_moments(state)
        mine = _moments(state)
        assert torch.equal(m.cpu().double(), mine[0]) and torch.equal(v.cpu().double(), mine[1])
        half = mdc.adamw_moments(state, torch.bfloat16)
        assert torch.equal(half[0].float(), m) and torch.equal(half[1].float(), v)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", [(("fp32",), ("fp32",)), (("fp32",), ("bf16",)), (("bf16",), ("bf16",)),
                                   (("fp16", "fp32", "bf16"), ("fp32", "fp16"))],
                         ids=["fp32", "mixed", "bf16", "all"])
@pytest.mark.parametrize("shapes", list(SHAPES))
def test_adamw(shapes, types, bits):
    import modulated_deform_conv as mdc
    params, grads = _setup(SHAPES[shapes], [TYPES[t] for t in types[0]], [TYPES[t] for t in types[1]],
                           len(shapes) + bits)
    state = mdc.adamw_state(params, bits, seed=2 ** 40 + 17)
    copies = [torch.empty(p.shape, dtype=torch.bfloat16, device=DEV) for p in params]
    for k, (g, max_norm) in enumerate(zip(grads, (None, 0.05, 1e9))):
        _check_step(params, g, state, 3e-3, (0.9, 0.999), 1e-8, 0.01, max_norm, copies if k else None)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_at_the_ends(bits):
    """Zero gradients, values whose squares leave fp32's normal range, eps 0, no memory (betas 0)."""
    import modulated_deform_conv as mdc
    params = [torch.ones(300, device=DEV), torch.full((129,), -2.0, device=DEV)]
    grads = [torch.zeros(300, device=DEV), torch.cat([torch.full((64,), 1e-12), torch.full((65,), 1e6)]).to(DEV)]
    grads[0][::7] = 1e-15
    grads[0][0] = 0.5
    state = mdc.adamw_state(params, bits)
    for betas, eps in (((0.9, 0.999), 1e-8), ((0.9, 0.999), 1e-8), ((0.0, 0.0), 1e-3)):
        _check_step(params, grads, state, 0.1, betas, eps, 0.0, None, None)


def test_views_and_strides():
    """Tensors off 16-byte boundaries, channels-last ones, one value of a larger tensor."""
    import modulated_deform_conv as mdc
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(4000, generator=g).to(DEV)
    conv = torch.randn(8, 3, 3, 4, generator=g).to(DEV).permute(0, 3, 1, 2)
    params = [wide[1:1001], wide[2003:2004], conv, wide[3000:3999].view(27, 37)]
    keep = wide.clone()
    grads = [torch.randn(1003, generator=g).to(DEV).half()[3:], torch.ones(1, device=DEV),
             torch.randn(8, 3, 3, 4, generator=g).to(DEV).permute(0, 3, 1, 2), torch.randn(27, 37, generator=g).to(DEV)]
    r = [(p.clone(), q.clone()) for p, q in zip(params, grads)]
    state = mdc.adamw_state(params)
    mdc.adamw_step_(params, grads, state, lr=0.01)
    for p, (p0, g0) in zip(params, r):
        want = p0.double() * (1 - 1e-4) - 0.01 * g0.double() / (g0.double().abs() + 1e-8)
        assert ((p.double() - want).abs() <= 20 * U * (p0.double().abs() + 0.01)).all()
    rest = torch.ones(4000, dtype=torch.bool)
    rest[1:1001] = rest[2003:2004] = rest[3000:3999] = False
    assert torch.equal(wide.cpu()[rest], keep.cpu()[rest])


def test_random_rounding_is_right_on_average():
    """200 steps of gradients of one spread: the mean over 2^17 places of v against the exact one. A
    place's spread is at most 0.3 v, so the mean's 2^-17/2 of that; m's is below 0.1 |m| + 0.1 sigma."""
    import modulated_deform_conv as mdc
    n = 2 ** 17
    p = torch.zeros(n, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(5)
    state, exact = mdc.adamw_state(p, 8, seed=9), mdc.adamw_state(p, 32)
    q = p.clone()
    for _ in range(200):
        g = 0.01 + 0.01 * torch.randn(n, device=DEV, generator=gen)
        mdc.adamw_step_(p, g, state, lr=1e-4)
        mdc.adamw_step_(q, g, exact, lr=1e-4)
    m, v = (t.double().mean().item() for t in mdc.adamw_moments(state))
    m0, v0 = (t.double().mean().item() for t in mdc.adamw_moments(exact))
    assert abs(v / v0 - 1) <= 6 * 0.3 * n ** -0.5 and abs(m / m0 - 1) <= 6 * 0.2 * n ** -0.5


def test_same_results_on_every_run_and_by_seed():
    import modulated_deform_conv as mdc
    out = []
    for seed in (4, 4, 5):
        params, grads = _setup(MANY, [torch.float32], [torch.bfloat16], 1)
        state = mdc.adamw_state(params, 8, seed=seed)
        for g in grads:
            mdc.adamw_step_(params, g, state, lr=1e-3, max_norm=0.1)
        out.append([state["exp_avg"], state["exp_avg_sq"], *params])
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    assert not torch.equal(out[0][0], out[2][0])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """A captured step against eager ones on its own stream, the rate read from the device."""
    import modulated_deform_conv as mdc
    a, grads = _setup(MANY[:20], [torch.float32], [torch.float32], 7)
    b = [p.clone() for p in a]
    sa, sb = mdc.adamw_state(a, bits, 3), mdc.adamw_state(b, bits, 3)
    lr = torch.full((1,), 1e-3, device=DEV)
    still = [g.clone() for g in grads[0]]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mdc.adamw_step_(a, still, sa, lr=lr, max_norm=0.1)  # the first step, eager
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        mdc.adamw_step_(a, still, sa, lr=lr, max_norm=0.1)
    mdc.adamw_step_(b, still, sb, lr=lr.item(), max_norm=0.1)  # the rate as fp32 holds it
    for k in range(4):
        rate = 1e-3 / (k + 1)
        lr.fill_(rate)
        for s, g in zip(still, grads[k % 3]):
            s.copy_(g)
        graph.replay()
        mdc.adamw_step_(b, still, sb, lr=lr.item(), max_norm=0.1)
        torch.cuda.synchronize()
        assert sa["step"].item() == sb["step"].item() == k + 2
        for x, y in zip([*a, sa["exp_avg"], sa["exp_avg_sq"]], [*b, sb["exp_avg"], sb["exp_avg_sq"]]):
            assert torch.equal(x, y)


def test_saved_and_loaded(tmp_path):
    import modulated_deform_conv as mdc
    params, grads = _setup(MANY[:9], [torch.float32], [torch.float32], 11)
    state = mdc.adamw_state(params, 8, seed=6)
    mdc.adamw_step_(params, grads[0], state, lr=1e-3)
    torch.save(state, tmp_path / "state.pt")
    loaded = torch.load(tmp_path / "state.pt", weights_only=True)
    again = [p.clone() for p in params]
    mdc.adamw_step_(params, grads[1], state, lr=1e-3)
    mdc.adamw_step_(again, grads[1], loaded, lr=1e-3)
    assert all(torch.equal(x, y) for x, y in zip(params, again))


def test_versions_and_parameters():
    """Leaves that record gradients are taken, and a graph that saved one says that it was changed."""
    import modulated_deform_conv as mdc
    w = torch.nn.Parameter(torch.ones(64, device=DEV))
    y = (w * w).sum()
    state = mdc.adamw_state([w])
    mdc.adamw_step_([w], [torch.ones(64, device=DEV)], state, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals_on_the_device():
    import modulated_deform_conv as mdc
    p = [torch.ones(256, device=DEV), torch.ones(5, device=DEV)]
    g = [torch.ones(256, device=DEV), torch.ones(5, device=DEV)]
    state = mdc.adamw_state(p)

    def step(params=p, grads=g, st=state, **kw):
        mdc.adamw_step_(params, grads, st, lr=0.1, **kw)

    for kw, match in ((dict(params=[p[0], p[0][:5]]), "overlap"), (dict(grads=[p[0], g[1]]), "overlap"),
                      (dict(copies=[p[0], torch.ones(5, device=DEV)]), "overlap"),
                      (dict(grads=g[:1]), "1 gradients"), (dict(grads=[g[1], g[0]]), "shape"),
                      (dict(params=p[:1], grads=g[:1]), "moments of"), (dict(betas=(1.0, 0.9)), "betas"),
                      (dict(eps=-1.0), "negative"), (dict(max_norm=-1.0), "negative"),
                      (dict(norm=torch.ones((), device=DEV)), "without max_norm"),
                      (dict(norm=torch.ones(()), max_norm=1.0), "norm must be"),
                      (dict(grads=[g[0].cpu(), g[1]]), "HIP"), (dict(params=[p[0].cpu(), p[1]]), "HIP"),
                      (dict(st={k: v for k, v in state.items() if k != "step"}), "no 'step'"),
                      (dict(st=dict(state, exp_avg=state["exp_avg"].half())), "float32 or uint8"),
                      (dict(st=dict(state, exp_avg_sq=state["exp_avg_sq"][:128])), "one size"),
                      (dict(st=dict(state, step=torch.zeros(1, dtype=torch.int64))), "HIP"),
                      (dict(copies=[torch.ones(256, device=DEV, dtype=torch.int32), g[1].clone()]), "not supported")):
        with pytest.raises(RuntimeError, match=match):
            step(**kw)
    assert torch.equal(p[0], torch.ones_like(p[0])) and state["step"].item() == 0
