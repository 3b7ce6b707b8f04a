"""The C entries of the operators over feature rows between guards: operands lie in buffers whose every other element is
NaN (a value read from beside a row would show in the results), and every output and workspace is exactly as large as the
entry says, with known bytes in front and behind that have to survive.  Sizes, strides and offsets are drawn, a new
set per case; values are checked against the 64-bit definitions."""
import ctypes
import random

import pytest
import torch

import decoder_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]  # in the order of NGS_FLOAT32 and so on
ACTS = ["none", "relu", "gelu", "silu", "sigmoid"]
LL, P, I = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int
GUARD = 4096


@pytest.fixture(scope="module")
def lib():
    from neuralgaussiansplatting_amd.diff_gaussian_rasterization import _lib
    L = _lib.lib()
    for name in ("ngs_linear_forward_workspace_bytes", "ngs_linear_backward_workspace_bytes", "ngs_linear_slope_bytes",
                 "ngs_layer_norm_backward_workspace_bytes"):
        getattr(L, name).restype = ctypes.c_size_t
    L.ngs_last_error.restype = ctypes.c_char_p
    return L


class Guarded:
    """`size` bytes, 16-byte aligned (plus `shift`), between known bytes."""

    def __init__(self, size, shift=0):
        self.size, self.start = size, GUARD + shift
        self.bytes = torch.full((size + 2 * GUARD + shift,), 0xA5, device=DEV, dtype=torch.uint8)
        self.ptr = P(self.bytes.data_ptr() + self.start)

    def check(self, what):
        for part in (self.bytes[:self.start], self.bytes[self.start + self.size:]):
            assert (part == 0xA5).all(), what + " was written outside its bounds"

    def tensor(self, dtype, *shape):
        return self.bytes[self.start:self.start + self.size].clone().view(dtype).view(shape)


def rows_between_nan(g, rng, rows, width, dtype, scale=1.0):
    """-> tensor [rows, width], its row stride; what lies between and around the rows is NaN"""
    stride = width + rng.choice([0, 0, 1, 2, 8, 25])
    first = rng.choice([0, 0, 1, 8, 25])
    buffer = torch.full((first + rows * stride + 64,), float("nan"), device=DEV, dtype=dtype)
    t = buffer.as_strided((rows, width), (stride, 1), first)
    t.copy_(torch.randn(rows, width, generator=g, device=DEV) * scale)
    return t, stride


def at(t):
    return P(t.data_ptr()) if t is not None else None


def draw_linear(rng):
    kind = rng.choice(["few", "narrow", "narrow", "tiles", "tiles", "wide"])
    pick = lambda lo, hi: rng.choice([rng.randint(lo, hi), rng.randint(lo, hi) // 8 * 8 or 8])
    if kind == "few":
        return rng.randint(1, 64), pick(1, 2100), pick(1, 600)
    if kind == "narrow":
        return rng.randint(65, 9000), pick(1, 256), pick(1, 256)
    if kind == "tiles":
        return rng.randint(1, 1200), pick(1, 1300), pick(1, 1300)
    return rng.randint(900, 2600), pick(600, 1400), pick(600, 1400)


@pytest.mark.parametrize("case", range(120))
def test_linear_between_guards(lib, case):
    rng = random.Random(1000 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    number = case % 3
    dtype, act = DTYPES[number], rng.randrange(5)
    rows, k, n = draw_linear(rng)
    size = torch.empty((), dtype=dtype).element_size()
    x, ldx = rows_between_nan(g, rng, rows, k, dtype)
    w, ldw = rows_between_nan(g, rng, n, k, dtype, k ** -0.5)
    dy, lddy = rows_between_nan(g, rng, rows, n, dtype, 0.1)
    r, ldr = rows_between_nan(g, rng, rows, n, dtype) if rng.random() < 0.5 else (None, 0)
    b = rows_between_nan(g, rng, 1, n, dtype, 0.3)[0] if rng.random() < 0.7 else None
    stream = P(torch.cuda.current_stream().cuda_stream)
    odd = lambda: rng.choice([0, size])  # outputs need their type's alignment only
    y = Guarded(rows * n * size, odd())
    slope_bytes = lib.ngs_linear_slope_bytes(LL(rows), k, n, number, act)
    slope = Guarded(slope_bytes, rng.choice([0, 4])) if slope_bytes else None
    ws = Guarded(lib.ngs_linear_forward_workspace_bytes(LL(rows), k, n, number))
    rc = lib.ngs_linear_forward(LL(rows), k, n, number, act, at(x), LL(ldx), at(w), LL(ldw), at(b), at(r), LL(ldr), y.ptr,
                                slope.ptr if slope else None, ws.ptr, stream)
    assert rc == 0, lib.ngs_last_error()
    dx, dw, db = Guarded(rows * k * size, odd()), Guarded(n * k * size, odd()), Guarded(n * size, odd())
    back = Guarded(lib.ngs_linear_backward_workspace_bytes(LL(rows), k, n, number, act))
    rc = lib.ngs_linear_backward(LL(rows), k, n, number, act, at(x), LL(ldx), at(w), LL(ldw), at(b),
                                 slope.ptr if slope else None, at(dy), LL(lddy), dx.ptr, dw.ptr, db.ptr, back.ptr, stream)
    assert rc == 0, lib.ngs_last_error()
    torch.cuda.synchronize()
    for name, buffer in dict(y=y, slope=slope, workspace=ws, dx=dx, dw=dw, db=db, backward_workspace=back).items():
        if buffer is not None:
            buffer.check("%s of %s" % (name, (rows, k, n, dtype, ACTS[act])))
    if ACTS[act] == "relu":  # (its derivative jumps where z is zero but for rounding)
        z = x.double() @ w.double().t() + (b.double() if b is not None else 0)
        sure = z.abs() > 2 * (k + 2) * ref.E * (x.double().abs() @ w.double().abs().t() + 1)
        if not sure.all():
            assert torch.isfinite(dx.tensor(dtype, rows, k)).all()
            return
    want = ref.linear(x, w, b[0] if b is not None else None, ACTS[act], r, dy)
    ref.assert_within(y.tensor(dtype, rows, n), want["y"], "y")
    ref.assert_within(dx.tensor(dtype, rows, k), want["dx"], "dx")
    ref.assert_within(dw.tensor(dtype, n, k), want["dweight"], "dweight")
    ref.assert_within(db.tensor(dtype, n), want["dbias"], "dbias")


@pytest.mark.parametrize("case", range(60))
def test_layer_norm_between_guards(lib, case):
    rng = random.Random(2000 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    number = case % 3
    dtype = DTYPES[number]
    wnumber = rng.choice([number, 0])
    rows = rng.choice([rng.randint(1, 20), rng.randint(1, 3000)])
    width = rng.choice([rng.randint(1, 300), rng.randint(1, 300), rng.randint(300, 5000), rng.randint(5000, 20000)])
    if rows * width > 6000000:
        rows = max(6000000 // width, 1)
    size, wsize = torch.empty((), dtype=dtype).element_size(), torch.empty((), dtype=DTYPES[wnumber]).element_size()
    x, ldx = rows_between_nan(g, rng, rows, width, dtype)
    dy, lddy = rows_between_nan(g, rng, rows, width, dtype)
    w = rows_between_nan(g, rng, 1, width, DTYPES[wnumber])[0] if rng.random() < 0.8 else None
    b = rows_between_nan(g, rng, 1, width, DTYPES[wnumber])[0] if rng.random() < 0.8 else None
    stream = P(torch.cuda.current_stream().cuda_stream)
    odd = lambda s: rng.choice([0, s])
    y, mean, rstd = Guarded(rows * width * size, odd(size)), Guarded(rows * 4, odd(4)), Guarded(rows * 4, odd(4))
    eps = 1e-5
    rc = lib.ngs_layer_norm_forward(LL(rows), width, number, wnumber, ctypes.c_float(eps), at(x), LL(ldx), at(w), at(b), y.ptr,
                                    mean.ptr, rstd.ptr, stream)
    assert rc == 0, lib.ngs_last_error()
    dx, dw, db = Guarded(rows * width * size, odd(size)), Guarded(width * wsize, odd(wsize)), Guarded(width * wsize, odd(wsize))
    ws = Guarded(lib.ngs_layer_norm_backward_workspace_bytes(LL(rows), width, number))
    rc = lib.ngs_layer_norm_backward(LL(rows), width, number, wnumber, at(x), LL(ldx), at(w), mean.ptr, rstd.ptr, at(dy), LL(lddy),
                                     dx.ptr, dw.ptr, db.ptr, ws.ptr, stream)
    assert rc == 0, lib.ngs_last_error()
    torch.cuda.synchronize()
    for name, buffer in dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db, workspace=ws).items():
        buffer.check("%s of %s" % (name, (rows, width, dtype)))
    want = ref.layer_norm(x, w[0] if w is not None else None, b[0] if b is not None else None, eps, dy)
    ref.assert_within(y.tensor(dtype, rows, width), want["y"], "y")
    ref.assert_within(dx.tensor(dtype, rows, width), want["dx"], "dx")
    for name, got in (("dweight", dw), ("dbias", db)):
        value, bound = want[name]
        if w is None and b is None:  # (the reference rounds to x's type then, the entry to weight_dtype, which may be finer)
            bound = bound + ref.half_step(dtype) * value.abs()
        ref.assert_within(got.tensor(DTYPES[wnumber], width), (value, bound), name)


@pytest.mark.parametrize("case", range(40))
def test_dropout_between_guards(lib, case):
    rng = random.Random(3000 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    number = case % 3
    dtype = DTYPES[number]
    rows, cols = rng.randint(1, 200), rng.choice([rng.randint(1, 100), rng.randint(1, 1000)])
    size = torch.empty((), dtype=dtype).element_size()
    x, ldx = rows_between_nan(g, rng, rows, cols, dtype)
    r, ldr = rows_between_nan(g, rng, rows, cols, dtype) if rng.random() < 0.5 else (None, 0)
    y = Guarded(rows * cols * size, rng.choice([0, size]))
    p, seed, offset = rng.random(), rng.getrandbits(64), rng.getrandbits(64)
    rc = lib.ngs_dropout(LL(rows), LL(cols), number, ctypes.c_double(p), ctypes.c_ulonglong(seed), None, ctypes.c_ulonglong(offset),
                         at(x), LL(ldx), at(r), LL(ldr), y.ptr, P(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.ngs_last_error()
    torch.cuda.synchronize()
    y.check("y of %s" % ((rows, cols, dtype),))
    mask = ref.kept(rows * cols, p, seed, offset).view(rows, cols).to(DEV)
    ref.assert_within(y.tensor(dtype, rows, cols), ref.dropout(x, mask, p, r, None)["y"], "y")
