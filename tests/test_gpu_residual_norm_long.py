"""The gradients of long rows, which take two passes (more than 4,096 channels), against the formulas in 64 bits with the
bounds of test_gpu_residual_norm.py: sums in many parts, gates by set, some gradients alone, every type."""
import pytest
import torch

from test_gpu_residual_norm import DEV, NAMES, TYPES, Reference, _check, _inputs, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate,block", [(None, False), ("channels", True), ("sets", True), ("sets", False)])
@pytest.mark.parametrize("shape", [(2, 150, 4104), (1, 90, 9000), (3, 41, 8192), (1, 1, 16384)], ids=str)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_long_rows(shape, dtype, gate, block, kind):
    """9,000 and 16,384 channels are two vectors a thread of 16 bits; in fp32 they pass over the row."""
    t, grads = _inputs(shape, TYPES[dtype], shape[1], gate, block)
    _check(t, grads, 0.7, block, kind)


@pytest.mark.parametrize("sets,rows", [(700, 1), (300, 3), (7, 100)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_numbers_of_sets(dtype, sets, rows):
    """More sets than parts, and parts of a set."""
    t, grads = _inputs((sets, rows, 4104), TYPES[dtype], sets, "sets", True)
    _check(t, grads, 1.0)


@pytest.mark.parametrize("residual,stream,affine", [(False, True, True), (True, False, True), (True, True, False)])
def test_without_some_inputs(residual, stream, affine):
    t, grads = _inputs((2, 33, 5000), torch.bfloat16, 5, None, True, affine=affine, residual=residual)
    _check(t, grads, 0.5, True, stream=stream)


def test_fp32_parameters():
    t, grads = _inputs((2, 40, 8192), torch.float16, 6, "sets", True, torch.float32)
    _check(t, grads, 0.5)


def test_some_gradients():
    """Each input's gradient alone is that of all together (and the first pass alone where no sum is wanted)."""
    from msda_opt2 import residual_norm
    t, (gy, gs) = _inputs((2, 50, 8192), torch.bfloat16, 7, "sets", True)
    gy, gs = gy.to(DEV), gs.to(DEV)

    def run(of):
        return residual_norm(of["x"], of["residual"], of["weight"], of["bias"], of["gate"], 0.5,
                             (of["block_weight"], of["block_bias"]))

    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    want = torch.autograd.grad(run(leaves), list(leaves.values()), (gy, gs))
    for n, w in zip(NAMES, want):
        rest = {m: v if m == n else v.detach() for m, v in leaves.items()}
        y, h = run(rest)
        outs = [(o, g) for o, g in ((y, gy), (h, gs)) if o.requires_grad]
        got, = torch.autograd.grad([o for o, _ in outs], leaves[n], [g for _, g in outs])
        assert torch.equal(got, w), n


def test_captured():
    from msda_opt2 import residual_norm
    t, grads = _inputs((3, 60, 8192), torch.float16, 8, "sets", True)
    still = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    g = [v.to(DEV) for v in grads]

    def step(of):
        out = residual_norm(of["x"], of["residual"], of["weight"], of["bias"], of["gate"], 0.5,
                            (of["block_weight"], of["block_bias"]))
        return [*(o.detach() for o in out), *torch.autograd.grad(out, list(of.values()), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(still)
    for k in range(4):
        new, _ = _inputs((3, 60, 8192), torch.float16, 20 + k, "sets", True)
        with torch.no_grad():
            for n, v in new.items():
                still[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step({n: v.to(DEV).requires_grad_() for n, v in new.items()})):
            assert torch.equal(a, b)


def test_non_finite_rows_stay_in_their_rows():
    from msda_opt2 import residual_norm
    t, (gy, gs) = _inputs((1, 300, 8192), torch.bfloat16, 9, None, True)

    def rows(x):
        leaves = [x.to(DEV).requires_grad_(), t["residual"].to(DEV).requires_grad_()]
        out = residual_norm(*leaves, t["weight"].to(DEV), t["bias"].to(DEV),
                            block_norm=(t["block_weight"].to(DEV), t["block_bias"].to(DEV)))
        return torch.autograd.grad(out, leaves, (gy.to(DEV), gs.to(DEV)))

    good = rows(t["x"])
    x = t["x"].clone()
    x[0, 77, 5000] = float("nan")
    rest = torch.arange(300, device=DEV) != 77
    for a, b in zip(rows(x), good):
        assert torch.equal(a[0, rest], b[0, rest]) and a[0, 77].isnan().all()
