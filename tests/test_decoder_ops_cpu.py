"""What the operators over feature rows refuse before anything reaches a GPU, through the C ABI and through torch, and
what the 64-bit definitions the GPU tests rest on say about themselves."""
import ctypes

import pytest
import torch

import decoder_reference as ref


@pytest.fixture(scope="module")
def lib():
    from neuralgaussiansplatting_amd.diff_gaussian_rasterization import _lib
    L = _lib.lib()
    for name in ("ngs_linear_forward_workspace_bytes", "ngs_linear_backward_workspace_bytes",
                 "ngs_layer_norm_backward_workspace_bytes"):
        getattr(L, name).restype = ctypes.c_size_t
    return L


LL, P = ctypes.c_longlong, ctypes.c_void_p
SOME = P(4096)  # an address that is never used: every call here is refused or has nothing to do


def linear(lib, rows=4, k=8, n=3, dtype=0, act=0, x=SOME, ldx=8, w=SOME, ldw=8, y=SOME, res=None, ldr=0, ws=SOME):
    return lib.ngs_linear_forward(LL(rows), k, n, dtype, act, x, LL(ldx), w, LL(ldw), None, res, LL(ldr), y, None, ws, None)


def linear_backward(lib, rows=4, k=8, n=3, dtype=0, act=0, x=SOME, w=SOME, slope=None, dy=SOME, lddy=3, dx=SOME, ws=SOME):
    return lib.ngs_linear_backward(LL(rows), k, n, dtype, act, x, LL(8), w, LL(8), None, slope, dy, LL(lddy), dx, SOME, SOME, ws, None)


def norm(lib, rows=4, d=8, dtype=0, wtype=0, eps=1e-5, x=SOME, ldx=8, y=SOME):
    return lib.ngs_layer_norm_forward(LL(rows), d, dtype, wtype, ctypes.c_float(eps), x, LL(ldx), None, None, y, None, None, None)


def norm_backward(lib, rows=4, d=8, dtype=0, wtype=0, x=SOME, mean=SOME, dy=SOME, ws=SOME):
    return lib.ngs_layer_norm_backward(LL(rows), d, dtype, wtype, x, LL(8), None, mean, SOME, dy, LL(8), SOME, SOME, SOME, ws, None)


def dropout(lib, rows=4, d=8, dtype=0, p=0.5, x=SOME, ldx=8, y=SOME):
    return lib.ngs_dropout(LL(rows), LL(d), dtype, ctypes.c_double(p), ctypes.c_ulonglong(1), None, ctypes.c_ulonglong(0), x,
                           LL(ldx), None, LL(0), y, None)


REFUSED = [
    (linear, dict(rows=-1)), (linear, dict(k=-1)), (linear, dict(n=-1)), (linear, dict(dtype=3)), (linear, dict(dtype=-1)),
    (linear, dict(act=5)), (linear, dict(act=-1)), (linear, dict(x=None)), (linear, dict(w=None)), (linear, dict(y=None)),
    (linear, dict(ldx=-8)), (linear, dict(ldw=-8)), (linear, dict(res=SOME, ldr=-1)), (linear, dict(rows=1 << 41)),
    (linear, dict(rows=1 << 40, ldx=1 << 20)), (linear, dict(rows=8, k=40000, ldx=40000, ldw=40000, ws=None)),
    (linear_backward, dict(rows=-1)), (linear_backward, dict(dtype=7)), (linear_backward, dict(act=9)),
    (linear_backward, dict(x=None)), (linear_backward, dict(w=None)), (linear_backward, dict(dy=None)),
    (linear_backward, dict(act=2, slope=None)), (linear_backward, dict(lddy=-3)), (linear_backward, dict(ws=None)),
    (norm, dict(rows=-1)), (norm, dict(d=-1)), (norm, dict(dtype=5)), (norm, dict(wtype=1)), (norm, dict(dtype=1, wtype=2)),
    (norm, dict(eps=-1.0)), (norm, dict(eps=float("nan"))), (norm, dict(x=None)), (norm, dict(y=None)), (norm, dict(ldx=-1)),
    (norm_backward, dict(rows=-1)), (norm_backward, dict(x=None)), (norm_backward, dict(dy=None)),
    (norm_backward, dict(mean=None)), (norm_backward, dict(ws=None)), (norm_backward, dict(wtype=2)),
    (dropout, dict(rows=-1)), (dropout, dict(d=-1)), (dropout, dict(dtype=3)), (dropout, dict(p=-0.01)),
    (dropout, dict(p=1.01)), (dropout, dict(p=float("nan"))), (dropout, dict(x=None)), (dropout, dict(y=None)),
    (dropout, dict(ldx=-8)), (dropout, dict(rows=1 << 50, d=1 << 20)),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_c_entries_refuse(lib, case):
    call, kw = REFUSED[case]
    assert call(lib, **kw) == 1, kw
    assert lib.ngs_last_error()


@pytest.mark.parametrize("call,args", [
    (linear, dict(rows=1 << 31, k=300, n=32, ldx=0, ldw=300)), (linear, dict(k=8, n=(1 << 31) - 1)),
    (linear, dict(k=(1 << 31) - 1)),
    (linear_backward, dict(n=(1 << 31) - 1)), (norm, dict(d=(1 << 31) - 1)), (norm, dict(rows=1 << 23, d=20000, ldx=0)), (dropout, dict(rows=1, d=1 << 36, ldx=0)),
])
def test_c_entries_refuse_what_one_launch_does_not_hold(lib, call, args):
    assert call(lib, **args) != 0
    lib.ngs_last_error.restype = ctypes.c_char_p
    assert b"too many elements for one launch" in lib.ngs_last_error()


def test_c_entries_with_nothing_to_do(lib):
    """Sizes of zero return without touching an address (or a GPU)."""
    assert linear(lib, rows=0, x=None, y=None, ws=None) == 0
    assert linear(lib, n=0, w=None, y=None, ws=None) == 0
    assert norm(lib, rows=0, x=None, y=None) == 0 and norm(lib, d=0, x=None, y=None) == 0
    assert dropout(lib, rows=0, x=None, y=None) == 0 and dropout(lib, d=0, x=None, y=None) == 0


def test_workspace_sizes(lib):
    f = lambda r, k, n, t: lib.ngs_linear_forward_workspace_bytes(LL(r), k, n, t)
    assert f(0, 64, 64, 0) == 0 and f(-1, 64, 64, 0) == 0 and f(100, 64, 0, 0) == 0 and f(100, 64, 64, 9) == 0
    assert f(1920 * 1080, 64, 128, 0) == 0  # enough rows to fill the chip: nothing is cut
    b = lambda r, k, n, t, a: lib.ngs_linear_backward_workspace_bytes(LL(r), k, n, t, a)
    assert b(1000, 64, 128, 2, 2) >= 1000 * 128 * 2  # dz
    assert 0 < b(1 << 21, 64, 128, 0, 0) < 1 << 30   # the cut reduction's parts stay small beside the operands
    assert b(-1, 64, 128, 0, 0) == 0
    for r, k, n_ in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (0, 0, 0)):
        for t in range(3):
            assert b(r, k, n_, t, 2) < 1 << 16 and f(r, k, n_, t) == 0
    n = lambda r, d, t: lib.ngs_layer_norm_backward_workspace_bytes(LL(r), d, t)
    assert n(0, 64, 0) == 0 and n(10, 0, 0) == 0 and 0 < n(1, 64, 0) <= n(1 << 21, 64, 0) < 1 << 24


def test_torch_functions_want_the_gpu():
    from neuralgaussiansplatting_amd import decoder_ops
    x = torch.zeros(4, 8)
    for call in (lambda: decoder_ops.linear(x, torch.zeros(3, 8)), lambda: decoder_ops.layer_norm(x),
                 lambda: decoder_ops.dropout(x, 0.5, 0)):
        with pytest.raises(RuntimeError, match="on the GPU only"):
            call()


def test_reference_agrees_with_torch():
    """The 64-bit definitions, their gradients included, are those of torch's own operators."""
    g = torch.Generator().manual_seed(0)
    d = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    acts = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
            "sigmoid": torch.sigmoid}
    x, w, b, r, dy = (t.float() for t in (d(7, 12), d(5, 12), d(5), d(7, 5), d(7, 5)))
    for act, f in acts.items():
        leaves = [t.double().requires_grad_() for t in (x, w, b, r)]
        y = f(leaves[0] @ leaves[1].t() + leaves[2]) + leaves[3]
        want = [y, *torch.autograd.grad(y, leaves, dy.double())]
        got = ref.linear(x, w, b, act, r, dy)
        for name, t in zip(("y", "dx", "dweight", "dbias", "dresidual"), want):
            torch.testing.assert_close(got[name][0], t.detach(), rtol=1e-12, atol=1e-12)
    x, w, b, dy = (t.float() for t in (d(6, 11), d(11), d(11), d(6, 11)))
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (11,), leaves[1], leaves[2], 1e-5)
    want = [y, *torch.autograd.grad(y, leaves, dy.double())]
    got = ref.layer_norm(x, w, b, 1e-5, dy)
    for name, t in zip(("y", "dx", "dweight", "dbias"), want):
        torch.testing.assert_close(got[name][0], t.detach(), rtol=1e-11, atol=1e-11)


def test_reference_mask_is_the_published_generator():
    """Block 0 of an all-zero key and counter, and one with every word set, of Philox 4x32 with 7 rounds (the published
    known-answer vectors of the method's authors), as 16-bit halves against thresholds on either side of each."""
    zero = [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    halves = [w >> s & 0xFFFF for w in zero for s in (0, 16)]
    for i, h in enumerate(halves):
        assert bool(ref.kept(8, h / 65536, 0, 0)[i])
        assert not bool(ref.kept(8, (h + 1) / 65536, 0, 0)[i])
