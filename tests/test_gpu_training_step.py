"""A training step of a small camera encoder with the operators in a row: grid cells looked up for
each camera, a deformable layer with group norm for the camera's map, attention between them,
backward, clipping. Each operator's part is held to the 64-bit formulas on what it was given, at
the bounds of its own tests."""
import pytest
import torch

import modulated_deform_conv as mdc
import msda_opt2
from modulated_deform_conv.dcn_split_nhwc import dcn_split_nhwc

from test_gpu_embedding import _near, _reference
from test_gpu_grad_clip import _check as _check_clip
from test_gpu_group_norm import Reference, _near as _near_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
CAMS, H, W, CELLS, SEEN = 3, 13, 17, 400, 60


def _leaves(dtype, seed):
    g = torch.Generator().manual_seed(seed)

    def leaf(*size, s=1.0, mean=0.0):
        return (mean + s * torch.randn(*size, generator=g)).to(dtype).to(DEV).requires_grad_()

    index = torch.rand(CAMS, CELLS, generator=g).argsort(1)[:, :SEEN].sort(1).values
    index[1, 41:] = -1
    loc = torch.rand(CAMS, SEEN, 8, 1, 4, 2, generator=g).to(dtype).to(DEV)
    params = [leaf(CELLS, 256, s=0.1), leaf(27, 64, 3, 3, s=0.02), leaf(27, s=0.3),
              leaf(256, 64, 3, 3, s=0.05), leaf(256, s=0.2, mean=1.0), leaf(256, s=0.2),
              leaf(32, 256, s=0.1)]
    return params, index.to(DEV), loc, leaf(CAMS, H, W, 64).detach(), leaf(CAMS, SEEN, 256).detach()


@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16],
                         ids=["fp32", "fp16", "bf16"])
def test_step(dtype, act):
    params, index, loc, x, go = _leaves(dtype, 1)
    grid, w_off, b_off, w, gn_w, gn_b, w_attn = params
    shapes = torch.tensor([[H, W]], device=DEV)
    starts = torch.zeros(1, dtype=torch.int64, device=DEV)

    q = msda_opt2.embedding_lookup(grid, index, 2.0)
    y = dcn_split_nhwc(x, w_off, b_off, w)
    m = mdc.group_norm_act_nhwc(y, 32, gn_w, gn_b, act=act)
    for t in (q, y, m):
        t.retain_grad()
    attn = torch.softmax(torch.nn.functional.linear(q, w_attn).view(CAMS, SEEN, 8, 1, 4), -1)
    out = msda_opt2.multi_scale_deformable_attn(m.view(CAMS, H * W, 8, 32), shapes, starts, loc, attn)
    out.backward(go)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in params)

    cpu = lambda t: t.detach().cpu()  # noqa: E731
    rows, grad, err = _reference(cpu(grid), cpu(index), cpu(q.grad), 2.0, None)
    _near(q, rows, 2 * 2.0 ** -24 * rows.abs(), "rows")
    _near(grid.grad, grad, err, "grid")
    r = Reference(cpu(y), cpu(gn_w), cpu(gn_b), cpu(m.grad), 32, act)
    for got, ref, bound in ((m, r.y, r.y_err), (y.grad, r.gx, r.gx_err), (gn_w.grad, r.gw, r.gw_err),
                            (gn_b.grad, r.gb, r.gb_err)):
        _near_norm(got, ref, bound, "norm")

    before = [cpu(p.grad).clone() for p in params]
    total = sum(t.double().square().sum() for t in before).sqrt().item()
    norm = mdc.clip_grad_norm_(params, total / 3)
    _check_clip(before, norm, [p.grad for p in params], total / 3)


def test_step_captured():
    """The whole step recorded once; replays with new inputs agree with the eager step up to what
    the attention's and the convolution's own atomics reorder: u = 2^-24 for each of at most
    some thousand sums of a gradient, against its largest value."""
    params, index, loc, x, go = _leaves(torch.float32, 2)
    shapes = torch.tensor([[H, W]], device=DEV)
    starts = torch.zeros(1, dtype=torch.int64, device=DEV)

    def step(params, index, loc, x, go):
        leaves = [p.detach().requires_grad_() for p in params]
        grid, w_off, b_off, w, gn_w, gn_b, w_attn = leaves
        q = msda_opt2.embedding_lookup(grid, index, 2.0)
        m = mdc.group_norm_act_nhwc(dcn_split_nhwc(x, w_off, b_off, w), 32, gn_w, gn_b, act="silu")
        attn = torch.softmax((q.reshape(-1, 256) @ w_attn.t()).view(CAMS, SEEN, 8, 1, 4), -1)
        out = msda_opt2.multi_scale_deformable_attn(m.view(CAMS, H * W, 8, 32), shapes, starts, loc, attn)
        grads = list(torch.autograd.grad(out, leaves, go))
        return [out.detach(), mdc.clip_gradients_(grads, 1.0), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(params, index, loc, x, go)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(params, index, loc, x, go)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (3, 4, 5):
        new = _leaves(torch.float32, seed)
        with torch.no_grad():
            for t, v in zip([*params, index, loc, x, go], [*new[0], *new[1:]]):
                t.copy_(v)
        graph.replay()
        got = [o.clone() for o in outs]
        want = step(*new)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert (a - b).abs().max().item() <= 4096 * 2.0 ** -24 * b.abs().max().item()


def test_without_gradients():
    """Under no_grad and inference_mode: the same values, nothing recorded; refusals stay."""
    params, index, _, x, _ = _leaves(torch.bfloat16, 6)
    grid, gn_w, gn_b = params[0], params[4], params[5]
    maps = x.repeat(1, 1, 1, 4).permute(0, 2, 1, 3)  # not contiguous
    want = [msda_opt2.embedding_lookup(grid, index, 2.0, 3), mdc.group_norm_act_nhwc(maps, 32, gn_w, gn_b)]
    assert all(t.requires_grad for t in want)
    for mode in (torch.no_grad(), torch.inference_mode()):
        with mode:
            got = [msda_opt2.embedding_lookup(grid, index.t().contiguous().t(), 2.0, 3),
                   mdc.group_norm_act_nhwc(maps, 32, gn_w, gn_b)]
            assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
            with pytest.raises(RuntimeError, match="padding_idx"):
                msda_opt2.embedding_lookup(grid, index, 1.0, CELLS)
            with pytest.raises(RuntimeError, match="act must be"):
                mdc.group_norm_act_nhwc(maps, 32, gn_w, gn_b, act="gelu")


def test_two_streams_at_once():
    """The same operators on two streams without a wait between: each call has its own workspace."""
    def work(seed):
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(6, 40, 50, 256, generator=g).half().to(DEV).requires_grad_()
        w = torch.rand(256, generator=g).half().to(DEV).requires_grad_()
        table = torch.randn(3000, 128, generator=g).to(DEV).requires_grad_()
        index = torch.randint(-1, 3000, (40000,), generator=g).to(DEV)
        return x, w, table, index, torch.ones(40000, 128, device=DEV)

    def run(x, w, table, index, g):
        y = mdc.group_norm_act_nhwc(x, 32, w, None, act="relu")
        grads = list(torch.autograd.grad(y, (x, w), y.detach()))
        grads += torch.autograd.grad(msda_opt2.embedding_lookup(table, index), table, g)
        return [y.detach(), mdc.clip_gradients_(grads, 1.0), *grads]

    inputs = [work(1), work(2)]
    want = [run(*i) for i in inputs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))
