"""Calls of the operators over feature rows that their documentation allows, beyond those of test_decoder_ops_gpu.py."""
import threading

import numpy as np
import pytest
import torch

from test_decoder_ops_gpu import check_linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from neuralgaussiansplatting_amd import decoder_ops
    return decoder_ops


def test_dropout_of_a_long_flat_tensor(ops):
    """More than 2^31 elements in one dimension: the mask is a function of the element's number, so it is that of the same
    elements as rows (which test_far_offsets compares with the definition)."""
    x = torch.ones((1 << 31) + 24, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = ops.dropout(x, 0.5, 3)
    assert torch.equal(y.detach().view(-1, 8), ops.dropout(x.detach().view(-1, 8), 0.5, 3))
    (dx,) = torch.autograd.grad(y, [x], x.detach())
    assert torch.equal(dx, y.detach())


def test_capture_refuses_views_of_a_leaf_of_a_living_graph(ops):
    """What holds for a leaf holds for a slice of its rows and for weights that lie in one flat parameter: the gradient
    ends in the leaf's accumulator."""
    flat = torch.linspace(-1, 1, 256, device=DEV).requires_grad_()
    other = torch.ones(8, 8, device=DEV)
    calls = [lambda: ops.linear(flat.view(16, 16)[:, 3:11], other), lambda: ops.linear(other, flat[64:128].view(8, 8)),
             lambda: ops.layer_norm(other, flat[:8], flat[8:16]), lambda: ops.layer_norm(flat.view(32, 8)),
             lambda: ops.dropout(flat.view(16, 16)[2:], 0.5, 1),
             lambda: ops.dropout(other, 0.5, 1, residual=flat[:64].view(8, 8))]
    for call in calls:
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="graph of the same tensor is alive"):
            with torch.cuda.graph(graph):
                torch.zeros(1, device=DEV)  # (an empty capture would warn)
                call()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
            (d,) = torch.autograd.grad(y, [flat], torch.ones_like(y))
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            want = call()
            assert torch.equal(y.detach(), want.detach())
            assert torch.equal(d, torch.autograd.grad(want, [flat], torch.ones_like(want))[0])
            del want
        del y, d


def test_dropout_takes_whole_numbers_of_any_kind(ops):
    """numpy's whole numbers count as Python's; what is not whole is refused, and so is a tensor as offset."""
    x = torch.ones(500, device=DEV)
    want = ops.dropout(x, 0.5, 7, offset=3)
    for kind in (np.int32, np.int64, np.uint8):
        assert torch.equal(ops.dropout(x, 0.5, kind(7), offset=kind(3)), want)
    assert torch.equal(ops.dropout(x, 0.5, np.int64(-1)), ops.dropout(x, 0.5, -1))
    for bad in (np.float32(7), 7.0, "7", None, [7]):
        with pytest.raises((RuntimeError, TypeError)):
            ops.dropout(x, 0.5, bad)
        with pytest.raises((RuntimeError, TypeError)):
            ops.dropout(x, 0.5, 7, offset=bad)
    with pytest.raises(RuntimeError):
        ops.dropout(x, 0.5, 7, offset=torch.tensor(3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["gelu", "sigmoid"])
@pytest.mark.parametrize("size", [(300, 512, 515), (130, 1024, 321), (523, 520, 514)], ids=str)
def test_stored_derivative_at_widths_that_end_inside_a_tile(ops, size, act, dtype):
    check_linear(ops, *size, dtype, act, True, True)


def step_of(ops, g, dtype, rows, k, n):
    """-> inputs of a training step through tiles (or padded copies) and a wide norm, and the step"""
    make = lambda *s, scale=1.0: (torch.randn(s, generator=g, device=DEV) * scale).to(dtype)
    x, w, b = make(rows, k).requires_grad_(), make(n, k, scale=k ** -0.5).requires_grad_(), make(n).requires_grad_()
    dy = make(rows, n)

    def step():
        y = ops.layer_norm(ops.linear(x, w, b, activation="silu"))
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]

    return (x, w, b, dy), step


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [(700, 1001, 1203), (2100, 1208, 1203), (512, 512, 9000)], ids=str)
def test_tiles_captured_and_replayed(ops, size, dtype):
    """Two graphs in one memory pool, replayed in turn with eager work between, on new inputs each time: the bits of
    eager steps."""
    graphs = []
    pool = torch.cuda.graph_pool_handle()
    for seed in (1, 2):
        inputs, step = step_of(ops, torch.Generator(device=DEV).manual_seed(seed), dtype, *size)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = step()
        graphs.append((inputs, step, graph, out))
    g = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(3):
        for inputs, step, graph, out in graphs:
            with torch.no_grad():
                for t in inputs:
                    t.copy_(torch.randn(t.shape, generator=g, device=DEV) * 0.1)
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in out]
            for a, b in zip(kept, step()):
                assert torch.equal(a, b)


def test_threads_on_streams_of_their_own(ops):
    """Four threads, each on its own stream: the bits of a lone call."""
    work = [step_of(ops, torch.Generator(device=DEV).manual_seed(i), dtype, *size) for i, (dtype, size) in enumerate(
        [(torch.float32, (900, 64, 48)), (torch.bfloat16, (700, 600, 777)), (torch.float16, (40, 1000, 90)),
         (torch.bfloat16, (3000, 39, 130))])]
    want = [step() for _, step in work]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = work[i][1]()
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        failed.append(i)
        except Exception as e:  # reported by the test's thread
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_dropout_reads_a_lazily_negated_seed_by_its_value(ops):
    x = torch.ones(1000, device=DEV, requires_grad=True)
    lazy = torch._neg_view(torch.tensor([5], device=DEV))
    assert lazy.is_neg()
    y = ops.dropout(x, 0.4, lazy)
    assert torch.equal(y, ops.dropout(x, 0.4, -5))
    assert torch.equal(torch.autograd.grad(y, [x], torch.ones_like(y))[0], y.detach())
