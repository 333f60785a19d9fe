"""The norm of many gradients and their clipping (grad_clip.hip) against 64 bits.

Bounds, with u = 2^-24 and e the half step of the output's type (finfo.eps / 2): the norm is summed
in fp64 and rounded once, u (2 u with all of fp64's own); the factor is rounded to fp32 and the
product once, 2 u, then e."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
MANY = [(256, 256), (256,), (1,), (0, 5), (3, 7, 5), (27, 256, 3, 3), (27,)] * 30 + [(1000, 257)]


def _grads(shapes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(*s, generator=g)).to(dtypes[k % len(dtypes)])
            for k, s in enumerate(shapes)]


def _norm(grads):
    return sum((g.double().square().sum() for g in grads), torch.zeros((), dtype=torch.float64)).sqrt()


def _check(grads, norm, outs, max_norm):
    ref = _norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(norm.item() - ref.item()) <= 2 * U * ref.item()
    by = min(1.0, max_norm / (ref.item() + 1e-6))
    for g, o in zip(grads, outs):
        want = g.double() * by
        half = torch.finfo(o.dtype).eps / 2
        bound = (2.5 * U + half) * want.abs() + torch.finfo(o.dtype).smallest_normal * half
        assert o.shape == g.shape and ((o.cpu().double() - want).abs() <= bound).all()
        if by == 1.0 and o.dtype == g.dtype:
            assert torch.equal(o.cpu(), g)


@pytest.mark.parametrize("max_norm", [0.0, 0.1, 35.0, 1e9])
@pytest.mark.parametrize("types", [("fp32",), ("fp16",), ("bf16",), ("bf16", "fp32", "fp16")],
                         ids=lambda t: "-".join(t))
@pytest.mark.parametrize("shapes", [[(1,)], [(5,), (3, 3)], [(8191,), (8192,), (8193,)], MANY,
                                    [(2 ** 22 + 5,)], [(0,), (0, 3), (4,)]],
                         ids=["one", "two", "edges", "many", "large", "empty"])
def test_clip(shapes, types, max_norm):
    import modulated_deform_conv as mdc
    grads = _grads(shapes, [TYPES[t] for t in types], len(shapes), 0.05)
    ours = [g.to(DEV) for g in grads]
    out = [torch.full(g.shape, float("nan"), device=DEV) for g in grads]
    norm = mdc.clip_gradients_(ours, max_norm, out=out)
    assert all(torch.equal(o.cpu(), g) for o, g in zip(ours, grads))
    _check(grads, norm, out, max_norm)
    half = [torch.empty(g.shape, dtype=torch.bfloat16, device=DEV) for g in grads]
    _check(grads, mdc.clip_gradients_(ours, max_norm, out=half), half, max_norm)
    assert torch.equal(mdc.grad_norm(ours), norm)
    again = mdc.clip_gradients_(ours, max_norm)
    assert torch.equal(again, norm)
    _check(grads, again, ours, max_norm)


def test_unaligned_and_other_orders():
    """Views into one buffer at odd places, channels-last and transposed memory."""
    import modulated_deform_conv as mdc
    for dtype in TYPES.values():
        flat = torch.full((40000,), 7.0, dtype=dtype, device=DEV)
        ours, at = [], 1
        for n in (5, 300, 4096, 9001, 1, 13000):
            ours.append(flat[at:at + n])
            at += n + 1  # a value between that no tensor has
        grads = _grads([tuple(v.shape) for v in ours], [dtype], 3)
        [v.copy_(g) for v, g in zip(ours, grads)]
        _check(grads, mdc.clip_gradients_(ours, 2.0), ours, 2.0)
        used = sum(v.numel() for v in ours)
        assert (flat == 7.0).sum().item() >= 40000 - used
        assert (flat[0] == 7.0) and (flat[at:] == 7.0).all() and (flat[6] == 7.0)
    x = torch.randn(6, 16, 5, 7, device=DEV).to(memory_format=torch.channels_last)
    y = torch.randn(30, 50, device=DEV).t()
    grads = [x.cpu(), y.cpu()]
    _check(grads, mdc.clip_gradients_([x, y], 1.5), [x, y], 1.5)


def test_values_beyond_fp32_squares():
    """Squares past fp32's range on both sides, and the smallest fp16 and bf16 values."""
    import modulated_deform_conv as mdc
    big = [torch.full((300,), 1e30), torch.full((7,), -2e30)]
    ours = [g.to(DEV) for g in big]
    _check(big, mdc.clip_gradients_(ours, 1.0), ours, 1.0)
    small = [torch.full((1000,), 1e-30), torch.full((64,), 2.0 ** -24, dtype=torch.float16)]
    ref = _norm(small).item()
    assert abs(mdc.grad_norm([g.to(DEV) for g in small]).item() - ref) <= 2 * U * ref


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_nonfinite(bad):
    """As torch.nn.utils.clip_grad_norm_: Inf makes the factor 0 (and Inf itself NaN), NaN makes all NaN."""
    import modulated_deform_conv as mdc
    a, b = torch.ones(500, device=DEV), torch.ones(70, device=DEV)
    a[3] = bad
    norm = mdc.clip_gradients_([a, b], 1.0)
    if bad != bad:
        assert norm.isnan() and a.isnan().all() and b.isnan().all()
    else:
        assert norm.isinf() and a.isnan().sum() == 1 and a[3].isnan() and not b.any()


def test_parameters_of_a_layer():
    """clip_grad_norm_ after a layer's backward: torch's own result; parameters without a gradient
    are passed over; an in-place write is seen by autograd's check."""
    import modulated_deform_conv as mdc
    torch.manual_seed(4)
    layer = mdc.ModulatedDeformConv2dPack(64, 64, 3, padding=1).to(DEV)
    layer.unused = torch.nn.Parameter(torch.ones(3, device=DEV))
    torch.nn.init.normal_(layer.conv_offset.weight, std=0.01)
    layer(torch.randn(1, 64, 12, 12, device=DEV)).square().sum().backward()
    grads = [p.grad.clone() for p in layer.parameters() if p.grad is not None]
    version = layer.weight.grad._version
    norm = mdc.clip_grad_norm_(layer.parameters(), 3.0)
    assert layer.unused.grad is None and layer.weight.grad._version > version
    _check([g.cpu() for g in grads], norm, [p.grad for p in layer.parameters() if p.grad is not None], 3.0)
    assert mdc.clip_grad_norm_([], 1.0).item() == 0.0 and mdc.grad_norm([]).item() == 0.0


def test_same_on_every_run_and_graph():
    """Captured once, replayed on new gradients with eager work on another stream between."""
    import modulated_deform_conv as mdc
    shapes, types = MANY, [torch.bfloat16, torch.float32]
    ours = [g.to(DEV) for g in _grads(shapes, types, 5)]
    flat = [torch.empty(g.shape, device=DEV) for g in ours]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mdc.clip_gradients_(ours, 1.0, out=flat)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = mdc.clip_gradients_(ours, 1.0, out=flat)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (6, 7, 8):
        new = [g.to(DEV) for g in _grads(shapes, types, seed)]
        [t.copy_(v) for t, v in zip(ours, new)]
        graph.replay()
        got = [norm.clone()] + [f.clone() for f in flat]
        out = [torch.empty(g.shape, device=DEV) for g in ours]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [mdc.clip_gradients_(new, 1.0, out=out)] + out
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refused_overlaps():
    """Nothing is launched for outputs that overlap: found from the addresses on the host."""
    import modulated_deform_conv as mdc
    a = torch.ones(100, device=DEV)
    with pytest.raises(RuntimeError, match="two outputs overlap"):
        mdc.clip_gradients_([a, a], 1.0)
    with pytest.raises(RuntimeError, match="two outputs overlap"):
        mdc.clip_gradients_([a[:60], a[50:]], 1.0)
    with pytest.raises(RuntimeError, match="not its own"):
        mdc.clip_gradients_([a[:50]], 1.0, out=[a[1:51]])
    with pytest.raises(RuntimeError, match="not its own"):
        b = torch.ones(50, device=DEV)
        mdc.clip_gradients_([a[:50], b], 1.0, out=[b, a[:50]])
    assert (a == 1).all() and abs(mdc.grad_norm([a, a]).item() - 200 ** 0.5) < 1e-5
