"""Embedding lookup (embedding.hip) against plain indexing in 64 bits.

Bounds, with u = 2^-24 and e the half step of the type (finfo.eps / 2): a looked-up row takes the
scale's and the product's rounding, 2 u, then e; a gradient adds up k rows in runs of at most 128
and the runs in turn, at most 128 + k / 64 fp32 sums in a row, u of the sum of magnitudes each,
then the scale and e as above."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _index(kind, rows, n, g):
    if kind == "uniform":
        return torch.randint(0, rows, (n,), generator=g)
    if kind == "same":
        return torch.full((n,), rows - 1)
    if kind == "skewed":  # frequency as one over the rank
        return (torch.exp(torch.rand(n, generator=g).double()
                          * torch.tensor(rows + 1.0).double().log()).long() - 1).clamp(0, rows - 1)
    if kind == "padded":  # and indices past both ends of the table
        i = torch.randint(0, rows, (n,), generator=g)
        i[torch.rand(n, generator=g) < 0.3] = -1
        i[::7], i[3::11] = rows, -2 ** 31
        return i
    if kind == "sorted":
        return torch.randint(0, rows, (n,), generator=g).sort().values
    return torch.full((n,), -1)  # nothing


def _reference(w, i, g, scale, padding):
    rows, there = w.shape[0], (i >= 0) & (i < w.shape[0])
    safe = torch.where(there, i, 0)
    out = w.double()[safe] * there.unsqueeze(-1) * scale
    gd = g.double() * (there & (i != (-5 if padding is None else padding))).unsqueeze(-1)
    flat, gd = safe.flatten(), gd.reshape(-1, w.shape[1])
    grad = torch.zeros(w.shape, dtype=torch.float64).index_add_(0, flat, gd)
    mag = torch.zeros(w.shape, dtype=torch.float64).index_add_(0, flat, gd.abs())
    k = torch.bincount(flat, minlength=rows).double().unsqueeze(-1)
    return out, grad * scale, mag * scale * U * (k.clamp(max=128) + k / 64 + 2)


def _near(got, ref, err, what):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    bound = err + half * (ref.abs() + err) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


def _check(w, i, g, scale=1.0, padding=None):
    import msda_opt2
    leaf = w.to(DEV).requires_grad_()
    out = msda_opt2.embedding_lookup(leaf, i.to(DEV), scale, padding)
    assert out.shape == (*i.shape, w.shape[1]) and out.dtype == w.dtype
    grad, = torch.autograd.grad(out, leaf, g.to(DEV))
    ref, ref_grad, err = _reference(w, i.long(), g, scale, padding)
    _near(out, ref, 2 * U * ref.abs(), "rows")
    assert grad.shape == w.shape and grad.dtype == w.dtype
    _near(grad, ref_grad, err, "gradient")
    untouched = err.sum(1) == 0
    assert not grad.detach().cpu()[untouched].any()
    return out.detach(), grad


def _problem(rows, dim, n, kind, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    i = _index(kind, rows, n, g)
    return (torch.randn(rows, dim, generator=g).to(dtype), i,
            torch.randn(n, dim, generator=g).to(dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,n,kind", [
    (1, 1, 1, "uniform"), (5, 3, 7, "uniform"), (300, 256, 300, "sorted"), (7, 128, 4001, "uniform"),
    (1, 256, 1000, "same"), (1000, 257, 65, "uniform"), (40000, 64, 3000, "padded"),
    (513, 1001, 777, "padded"), (2000, 320, 9000, "skewed"), (100, 2048, 300, "uniform"),
    (900, 8, 20000, "skewed"), (65, 96, 64, "nothing"), (3, 512, 129, "uniform"),
    (70000, 16, 70000, "skewed"), (2, 40, 40000, "padded"), (4099, 250, 33333, "sorted")])
def test_lookup(rows, dim, n, kind, dtype):
    _check(*_problem(rows, dim, n, kind, TYPES[dtype], rows + n), scale=dim ** 0.5)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_int32_shapes_and_padding_row(dtype):
    w, i, g = _problem(50, 64, 360, "padded", TYPES[dtype], 1)
    i = i.clamp(min=-9).int().view(3, 4, 30)
    a = _check(w, i, g.view(3, 4, 30, 64), 0.5, padding=7)
    b = _check(w, i.long(), g.view(3, 4, 30, 64), 0.5, padding=7)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_strides_and_scalars():
    import msda_opt2
    w, i, g = _problem(40, 30, 24, "uniform", torch.float32, 2)
    idx = i.view(4, 6).to(DEV).t()
    assert not idx.is_contiguous()
    leaf = w.t().contiguous().to(DEV).t().requires_grad_()
    out = msda_opt2.embedding_lookup(leaf, idx)
    out.backward(torch.ones(1, device=DEV).expand(out.shape))
    ref, grad, err = _reference(w, idx.cpu(), torch.ones(6, 4, 30), 1.0, None)
    _near(out, ref, 0 * ref, "rows")
    _near(leaf.grad, grad, err, "gradient")
    assert torch.equal(msda_opt2.embedding_lookup(leaf, idx[2, 1]), leaf[idx[2, 1]])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_offset_views(dtype):
    """Tables and gradients that start off a 16-byte boundary."""
    import _modulated_deform_conv_ext as ext
    w, i, g = _problem(90, 64, 500, "skewed", TYPES[dtype], 3)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    ref, grad, err = _reference(w, i, g, 3.0, None)
    _near(ext.embedding_forward(shifted(w), i.to(DEV), 3.0), ref, 2 * U * ref.abs(), "rows")
    _near(ext.embedding_backward(shifted(g), i.to(DEV), 90, 3.0), grad, err, "gradient")


def test_empty():
    import msda_opt2
    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    none = torch.empty(0, 3, dtype=torch.int64, device=DEV)
    out = msda_opt2.embedding_lookup(w, none)
    grad, = torch.autograd.grad(out, w, torch.empty_like(out))
    assert out.shape == (0, 3, 8) and grad.shape == (5, 8) and not grad.any()
    table = torch.empty(0, 8, device=DEV, requires_grad=True)
    out = msda_opt2.embedding_lookup(table, torch.tensor([0, -1, 3], device=DEV))
    grad, = torch.autograd.grad(out, table, torch.ones_like(out))
    assert out.shape == (3, 8) and not out.any() and grad.shape == (0, 8)
    flat = torch.empty(4, 0, device=DEV)
    assert msda_opt2.embedding_lookup(flat, torch.tensor([1, 2], device=DEV)).shape == (2, 0)


def test_nonfinite_rows_reach_their_own_index_only():
    import msda_opt2
    w, i, g = _problem(30, 64, 3000, "padded", torch.float32, 4)
    w[3], g[10], g[5] = float("nan"), float("inf"), float("nan")
    i[10], i[5], i[6] = 8, -1, 3
    leaf = w.to(DEV).requires_grad_()
    out = msda_opt2.embedding_lookup(leaf, i.to(DEV))
    grad, = torch.autograd.grad(out, leaf, g.to(DEV))
    assert torch.equal(out.isnan().any(1).cpu(), i == 3)
    assert not out[(i < 0).to(DEV)].any()
    assert (grad[8] == float("inf")).all() and torch.isfinite(grad).all(1).sum() == 29


def test_same_on_every_run():
    w, i, g = _problem(500, 256, 50000, "skewed", torch.float32, 5)
    a, b = _check(w, i, g), _check(w, i, g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_differences():
    """The lookup is linear in the table: the gradient against differences along a direction, whose
    only error is fp32's, u of the magnitudes for each of about 20 sums."""
    w, i, g = _problem(40, 16, 200, "skewed", torch.float32, 6)
    _, grad = _check(w, i, g, 2.0)
    v = torch.randn(w.shape, generator=torch.Generator().manual_seed(7)).double()

    def f(step):
        return (_reference(w.double() + step * v, i, g, 2.0, None)[0] * g.double()).sum().item()

    terms = grad.cpu().double() * v
    assert abs(terms.sum().item() - (f(0.5) - f(-0.5))) <= 128 * U * terms.abs().sum().item()


def test_graph_and_streams():
    """Captured training steps replayed with new indices, eager calls on another stream between."""
    import msda_opt2
    w, i, g = (t.to(DEV) for t in _problem(700, 128, 5000, "skewed", torch.bfloat16, 8))

    def step(w, i, g):
        leaf = w.detach().requires_grad_()
        out = msda_opt2.embedding_lookup(leaf, i, 2.0)
        return out.detach(), *torch.autograd.grad(out, leaf, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w, i, g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(w, i, g)
    torch.cuda.current_stream().wait_stream(side)
    for seed, kind in ((9, "uniform"), (10, "same"), (11, "padded")):
        new = [t.to(DEV) for t in _problem(700, 128, 5000, kind, torch.bfloat16, seed)]
        for t, v in zip((w, i, g), new):
            t.copy_(v)
        graph.replay()
        got = [o.clone() for o in outs]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step(*new)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_camera_queries_through_attention():
    """The cells that each camera sees, padded with -1, looked up, attended to and learned: the
    gradient of the grid is the sum over the cameras that see a cell."""
    import msda_opt2
    from oracle import inputs
    g = torch.Generator().manual_seed(12)
    grid = (0.1 * torch.randn(400, 256, generator=g)).to(DEV).requires_grad_()
    index = torch.rand(3, 400, generator=g).argsort(1)[:, :50].sort(1).values
    index[1, 30:], index[2, 45:] = -1, -1
    index = index.to(DEV)
    q = msda_opt2.embedding_lookup(grid, index)                       # [3, 50, 256]
    d = inputs.msda_random(3, [(9, 7)], 50, 8, 32, 4)
    d = {k: v.to(DEV) for k, v in d.items()}
    attn = torch.softmax(q.view(3, 50, 8, 32)[..., :4], -1).view(3, 50, 8, 1, 4)
    out = msda_opt2.multi_scale_deformable_attn(d["value"], d["spatial_shapes"],
                                                d["level_start_index"], d["sampling_loc"], attn)
    gq, = torch.autograd.grad(out.square().sum(), q, retain_graph=True)
    grad, = torch.autograd.grad(out.square().sum(), grid)
    _, ref, err = _reference(grid.detach().cpu(), index.cpu(), gq.cpu(), 1.0, None)
    _near(grad, ref, err, "gradient")
    assert grad.any() and not grad[~torch.isin(torch.arange(400, device=DEV), index)].any()
