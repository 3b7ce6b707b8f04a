"""The operators over feature rows (decoder_ops) against their definitions in 64 bits: sizes and types, strides, zero
sizes, special values, gradients, streams, graph capture, far offsets.  Bounds are derived in decoder_reference.py."""
import pytest
import torch

import decoder_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu", "sigmoid"]


@pytest.fixture(scope="module")
def ops():
    from neuralgaussiansplatting_amd import decoder_ops
    return decoder_ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def gradients(y, leaves, dy):
    names = [n for n, t in leaves.items() if t is not None]
    return dict(zip(names, torch.autograd.grad(y, [leaves[n] for n in names], dy)))


def check_linear(ops, rows, k, n, dtype, act, bias, residual, train=True, first=0, pitch=None, integers=False, seed=0):
    g = gen(seed + rows * 31 + k * 7 + n)

    def make(*shape, scale=1.0):
        if integers:
            return torch.randint(-3, 4, shape, generator=g, device=DEV).to(dtype)
        return normal(g, *shape, dtype=dtype, scale=scale)

    x = make(rows, pitch or k)[:, first:first + k].detach().requires_grad_(train)
    w = make(n, k, scale=max(k, 1) ** -0.5).requires_grad_(train)
    b = make(n, scale=0.3).requires_grad_(train) if bias else None
    r = make(rows, n).requires_grad_(train) if residual else None
    dy = make(rows, n, scale=0.1) if train else None
    y = ops.linear(x, w, b, activation=act, residual=r)
    assert y.dtype == dtype and y.shape == (rows, n) and y.is_contiguous() and y.requires_grad == train
    want = ref.linear(x.detach(), w.detach(), None if b is None else b.detach(), act,
                      None if r is None else r.detach(), dy)
    ref.assert_within(y, want["y"], "y")
    if train:
        for name, got in gradients(y, {"dx": x, "dweight": w, "dbias": b, "dresidual": r}, dy).items():
            assert got.dtype == dtype
            ref.assert_within(got, want[name], name)


LINEAR_SIZES = [(1, 1, 1), (1, 64, 128), (3, 39, 3), (5, 17, 31), (16, 8, 40), (33, 100, 65), (127, 128, 129),
                (128, 64, 128), (130, 200, 300), (257, 513, 40), (1000, 39, 3), (300, 1030, 520), (4100, 24, 16),
                (2, 4096, 1000), (64, 5000, 48), (7, 3, 700), (40, 2050, 33), (2600, 128, 128), (2049, 64, 96), (8192, 64, 1024), (3000, 1000, 1000), (2048, 264, 3400), (600, 4104, 600), (2300, 1001, 1003), (1500, 1203, 1208), (1500, 1208, 1203), (8200, 304, 2000), (4099, 1001, 2003),
                (515, 256, 256), (9, 1027, 2051), (12, 512, 512), (1, 8192, 70), (4, 1111, 999), (8, 2048, 3), (15, 640, 4097), (16, 33, 5), (17, 700, 64), (33, 1001, 50), (64, 3711, 40), (60, 9, 17),
                # many narrow rows
                (4096, 1, 1), (4097, 3, 5), (5000, 39, 3), (4999, 128, 128), (4100, 127, 129), (6001, 200, 24), (4200, 17, 100),
                (4111, 256, 40), (9000, 64, 128), (4500, 8, 250), (5003, 65, 33), (4099, 33, 64), (70001, 40, 48), (4100, 2, 70),
                (4101, 7, 7), (5000, 3, 2), (4300, 100, 200), (4400, 250, 60), (4200, 60, 255), (4150, 256, 3), (4160, 3, 256),
                (4170, 130, 256), (8300, 16, 152)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", LINEAR_SIZES, ids=str)
def test_linear_sizes(ops, size, dtype):
    i = LINEAR_SIZES.index(size)
    act = ["gelu", "silu", "none", "sigmoid"][i % 4]
    check_linear(ops, *size, dtype, act, bias=i % 3 != 0, residual=i % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(70, 72, 40), (700, 39, 3), (3, 300, 260), (300, 64, 128), (4300, 39, 3),
                                  (4301, 72, 40), (4302, 128, 128)], ids=str)
def test_linear_activations(ops, size, act, dtype):
    """Every activation with and without bias and residual.  Small whole numbers give exact sums, so that relu's
    derivative at and next to zero is decided by the definition."""
    for bias in (False, True):
        for residual in (False, True):
            check_linear(ops, *size, dtype, act, bias, residual, integers=act in ("none", "relu"))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", [(300, 39, 3, 25, 64), (2500, 39, 64, 25, 64), (1, 39, 20, 25, 64), (140, 128, 130, 8, 144),
                                  (300, 63, 64, 1, 65), (5, 256, 32, 0, 300), (5000, 39, 64, 25, 64), (4500, 39, 3, 25, 64),
                                  (4501, 128, 128, 0, 130), (4502, 63, 30, 1, 67), (4503, 5, 72, 25, 30)], ids=str)
def test_linear_slices(ops, case, dtype):
    """Rows that are slices of wider ones (the 39 copied features of a feature row), aligned or not."""
    rows, k, n, first, pitch = case
    check_linear(ops, rows, k, n, dtype, "gelu", True, True, first=first, pitch=pitch)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear_layouts(ops, dtype):
    """Leading dimensions, transposed operands, broadcast residual and gradient, strided weight and bias."""
    g = gen(5)
    x = normal(g, 2, 5, 7, 24, dtype=dtype)
    w = normal(g, 24, 40, dtype=dtype, scale=0.2).t()          # columns contiguous
    b = normal(g, 80, dtype=dtype)[::2]
    r = normal(g, 40, dtype=dtype).expand(2, 5, 7, 40)
    for t in (x, x.transpose(1, 2), x.flip(0).transpose(0, 2), x[:, ::2], x[..., 3:11]):
        wt = w[:, :t.shape[-1]]
        rt = r[:1, :1, :1].expand(*t.shape[:-1], 40)
        leaves = {"dx": t.detach().requires_grad_(), "dweight": wt.detach().requires_grad_(),
                  "dbias": b.detach().requires_grad_(), "dresidual": rt.detach().requires_grad_()}
        y = ops.linear(*[leaves[n] for n in ("dx", "dweight", "dbias")], activation="silu", residual=leaves["dresidual"])
        assert y.shape == (*t.shape[:-1], 40)
        dy = normal(g, 40, dtype=dtype).expand(y.shape)
        want = ref.linear(t, wt, b, "silu", rt, dy)
        ref.assert_within(y, want["y"], "y")
        for name, got in gradients(y, leaves, dy).items():
            assert got.shape == leaves[name].shape
            ref.assert_within(got, want[name], name)
    x1 = normal(g, 24, dtype=dtype)  # a single row without leading dimensions
    y = ops.linear(x1, w, b)
    assert y.shape == (40,)
    ref.assert_within(y, ref.linear(x1, w, b, "none", None, None)["y"], "y")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(0, 8, 4), (0, 8, 0), (5, 0, 4), (5, 8, 0), (0, 0, 0), (300, 0, 64)], ids=str)
def test_linear_zero_sizes(ops, size, dtype):
    rows, k, n = size
    for act in ("none", "gelu"):
        x = torch.ones(rows, k, device=DEV, dtype=dtype, requires_grad=True)
        w = torch.ones(n, k, device=DEV, dtype=dtype, requires_grad=True)
        b = torch.full((n,), 2.0, device=DEV, dtype=dtype, requires_grad=True)
        y = ops.linear(x, w, b, activation=act)
        want = torch.nn.functional.gelu(b.detach().double()) if act == "gelu" else b.detach().double()
        torch.testing.assert_close(y.double(), want.expand(rows, n), atol=0, rtol=2.0 ** -8)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        if rows == 0 or n == 0 or k == 0:
            assert (dx == 0).all() and (dw == 0).all()
        if act == "none":
            assert (db == rows).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear_special_values(ops, dtype):
    """Infinities and NaN stay in their rows and columns, at every size of kernel."""
    for rows, k, n in ((1, 100, 200), (6, 100, 200), (200, 39, 70), (300, 256, 256), (5001, 39, 70), (4101, 128, 64)):
        g = gen(rows)
        x, w = normal(g, rows, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=0.1)
        clean = ops.linear(x, w)
        x[rows - 1, k - 1] = float("nan")
        w[n - 1, 0] = float("inf")
        y = ops.linear(x, w)
        assert torch.isnan(y[rows - 1]).all()
        assert not torch.isfinite(y[:, n - 1]).any()
        assert torch.equal(y[:rows - 1, :n - 1], clean[:rows - 1, :n - 1])
        y = ops.linear(x, w, activation="relu")
        assert torch.isnan(y[rows - 1, :n - 1]).all()
    big = torch.tensor([[1.0], [-1.0], [60.0], [-60.0], [1e4], [-1e4]], device=DEV, dtype=dtype, requires_grad=True)
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    for act in ACTS:  # far out nothing overflows on the way
        y = ops.linear(big, one, activation=act)
        (dx,) = torch.autograd.grad(y, [big], torch.ones_like(y))
        want = ref.linear(big.detach(), one, None, act, None, torch.ones_like(y))
        ref.assert_within(y, want["y"], act)
        ref.assert_within(dx, want["dx"], act)


def test_linear_partial_gradients(ops):
    """Every subset of inputs that want gradients gets the gradients that all of them get."""
    g = gen(3)
    for rows in (300, 5000):
        partial_gradients(ops, g, rows)


def partial_gradients(ops, g, rows):
    tensors = [normal(g, rows, 40), normal(g, 24, 40, scale=0.2), normal(g, 24), normal(g, rows, 24)]
    dy = normal(g, rows, 24)

    def run(subset, act):
        ts = [t.clone().requires_grad_(i in subset) for i, t in enumerate(tensors)]
        y = ops.linear(ts[0], ts[1], ts[2], activation=act, residual=ts[3])
        return dict(zip(subset, torch.autograd.grad(y, [ts[i] for i in subset], dy)))

    for act in ("none", "gelu"):
        every = run((0, 1, 2, 3), act)
        for m in range(1, 15):
            subset = tuple(i for i in range(4) if m >> i & 1)
            for i, d in run(subset, act).items():
                assert torch.equal(d, every[i]), (act, subset, i)


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid"])
def test_linear_gradient_against_differences(ops, act):
    """Central differences of the 32-bit forward pass: with a step h the difference quotient of a scalar loss is off by
    h^2 times its third derivative and by the loss's own rounding over h; both stay below 1e-2 of the gradient's norm
    for the sizes here (|third derivatives| < 1, rounding about 1e-6 a unit of loss, h = 2^-6)."""
    g = gen(17)
    ts = [normal(g, 6, 20, scale=0.5), normal(g, 10, 20, scale=0.3), normal(g, 10, scale=0.3), normal(g, 6, 10)]
    dy = normal(g, 6, 10)
    leaves = [t.clone().requires_grad_() for t in ts]
    y = ops.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    grads = torch.autograd.grad(y, leaves, dy)
    h = 2.0 ** -6
    loss = lambda a: (ops.linear(a[0], a[1], a[2], activation=act, residual=a[3]).double() * dy.double()).sum().item()
    for i, t in enumerate(ts):
        way = normal(g, *t.shape)
        way /= way.norm()
        up, down = [list(ts) for _ in range(2)]
        up[i], down[i] = t + h * way, t - h * way
        quotient = (loss(up) - loss(down)) / (2 * h)
        assert abs(quotient - (grads[i].double() * way.double()).sum().item()) < 1e-2 * max(grads[i].norm().item(), 1.0)


# ---- layer norm ----

NORM_SIZES = [(1, 1), (3, 2), (5, 3), (17, 8), (64, 9), (33, 16), (20, 24), (1000, 39), (513, 64), (100, 65), (50, 100),
              (70, 128), (31, 200), (12, 255), (40, 512), (9, 513), (7, 1000), (5, 1024), (3, 2047), (2, 2048), (6, 2500),
              (3, 4096), (2, 5001), (1, 8192), (3, 9000), (2, 16384), (2, 20001), (3, 33000), (3000, 40), (1, 4096)]


def check_norm(ops, rows, d, dtype, wtype, weight=True, bias=True, first=0, pitch=None, eps=1e-5, offset=0.5):
    g = gen(rows * 131 + d)
    x = (normal(g, rows, pitch or d) + offset).to(dtype)[:, first:first + d].detach().requires_grad_()
    w = normal(g, d, dtype=wtype).requires_grad_() if weight else None
    b = normal(g, d, dtype=wtype).requires_grad_() if bias else None
    y = ops.layer_norm(x, w, b, eps=eps)
    assert y.dtype == dtype and y.shape == (rows, d) and y.is_contiguous()
    dy = normal(g, rows, d, dtype=dtype)
    want = ref.layer_norm(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), eps, dy)
    ref.assert_within(y, want["y"], "y")
    for name, got in gradients(y, {"dx": x, "dweight": w, "dbias": b}, dy).items():
        ref.assert_within(got, want[name], name)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps=eps), y)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", NORM_SIZES, ids=str)
def test_norm_sizes(ops, size, dtype):
    check_norm(ops, *size, dtype, torch.float32 if NORM_SIZES.index(size) % 2 else dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", [(300, 39, 25, 64), (70, 500, 3, 504), (3, 2001, 8, 2048), (2, 17000, 1, 17001)], ids=str)
def test_norm_slices_and_absent_weights(ops, case, dtype):
    rows, d, first, pitch = case
    for weight, bias in ((True, True), (True, False), (False, True), (False, False)):
        check_norm(ops, rows, d, dtype, dtype, weight, bias, first=first, pitch=pitch)


def test_norm_rows_far_from_zero(ops):
    """A mean a thousand times the spread costs the digits that the mean takes, not twice as many: the variance is
    taken about the mean."""
    for d in (64, 600, 5000, 40000):
        check_norm(ops, 5, d, torch.float32, torch.float32, offset=1000.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_norm_special_rows(ops, dtype):
    """A constant row gives the bias; a row with NaN or infinity is NaN and the rows beside it do not notice."""
    for d in (24, 700, 3000, 20000):
        g = gen(d)
        x, w, b = normal(g, 9, d, dtype=dtype), normal(g, d, dtype=dtype), normal(g, d, dtype=dtype)
        x[4] = 2.0
        clean = ops.layer_norm(x, w, b)
        assert torch.equal(clean[4], b)
        x[2, d - 1], x[6, 0] = float("nan"), float("inf")
        y = ops.layer_norm(x, w, b)
        assert torch.isnan(y[2]).all() and torch.isnan(y[6]).all()
        others = [0, 1, 3, 4, 5, 7, 8]
        assert torch.equal(y[others], clean[others])


@pytest.mark.parametrize("size", [(0, 8), (5, 0), (0, 0)], ids=str)
def test_norm_zero_sizes(ops, size):
    rows, d = size
    x = torch.ones(rows, d, device=DEV, requires_grad=True)
    w, b = torch.ones(d, device=DEV, requires_grad=True), torch.ones(d, device=DEV, requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
    assert y.shape == dx.shape == x.shape and (dw == 0).all() and (db == 0).all() and dw.shape == (d,)


def test_norm_partial_gradients(ops):
    g = gen(8)
    for d in (40, 3000, 20000):
        ts = [normal(g, 30, d), normal(g, d), normal(g, d)]
        dy = normal(g, 30, d)

        def run(subset):
            a = [t.clone().requires_grad_(i in subset) for i, t in enumerate(ts)]
            return dict(zip(subset, torch.autograd.grad(ops.layer_norm(*a), [a[i] for i in subset], dy)))

        every = run((0, 1, 2))
        for subset in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
            for i, got in run(subset).items():
                assert torch.equal(got, every[i]), (d, subset, i)


def test_norm_gradient_against_differences(ops):
    """As test_linear_gradient_against_differences; 1e-2 covers h^2 times the third derivative along a unit step (below
    10 at a spread of one) and the rounding over h."""
    g = gen(23)
    ts = [normal(g, 6, 30), normal(g, 30), normal(g, 30)]
    dy = normal(g, 6, 30)
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    h = 2.0 ** -6
    loss = lambda a: (ops.layer_norm(*a).double() * dy.double()).sum().item()
    for i, t in enumerate(ts):
        way = normal(g, *t.shape)
        way /= way.norm()
        up, down = [list(ts) for _ in range(2)]
        up[i], down[i] = t + h * way, t - h * way
        quotient = (loss(up) - loss(down)) / (2 * h)
        assert abs(quotient - (grads[i].double() * way.double()).sum().item()) < 1e-2 * max(grads[i].norm().item(), 1.0)


# ---- dropout ----

@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (7, 1), (1, 8), (3, 5), (64, 64), (13, 39), (2, 3, 10), (5, 1001), (9, 7), (3, 2047), (2, 2049), (700, 39)], ids=str)
def test_dropout_mask_and_values(ops, shape, dtype):
    g = gen(sum(shape))
    numel = torch.Size(shape).numel()
    for p, seed, offset in ((0.1, 0, 0), (0.5, 2 ** 63 + 12345, 7), (0.25, 77, 2 ** 40 + 3), (0.0, 5, 5), (1.0, 5, 5)):
        mask = ref.kept(numel, p, seed, offset).view(shape).to(DEV)
        x = normal(g, *shape, dtype=dtype).requires_grad_()
        r = normal(g, *shape, dtype=dtype).requires_grad_()
        dy = normal(g, *shape, dtype=dtype)
        for residual in (None, r):
            y = ops.dropout(x, p, seed, offset=offset, residual=residual)
            want = ref.dropout(x.detach(), mask, p, None if residual is None else r.detach(), dy)
            assert y.dtype == dtype and y.shape == x.shape
            for name, got in [("y", y)] + list(gradients(y, {"dx": x, "dresidual": residual}, dy).items()):
                ref.assert_within(got, want[name], name)
            if residual is None:
                assert torch.equal(y != 0, mask & (x != 0))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dropout_strides_do_not_matter(ops, dtype):
    """The mask goes by an element's place among the rows, not by where it lies."""
    g = gen(1)
    wide, res = normal(g, 50, 64, dtype=dtype), normal(g, 50, 80, dtype=dtype)
    for first, k in ((25, 39), (0, 24), (8, 40), (1, 63), (3, 1), (0, 2)):
        x, r = wide[:, first:first + k], res[:, first:first + k]
        want = ops.dropout(x.contiguous(), 0.3, 9, offset=2, residual=r.contiguous())
        assert torch.equal(ops.dropout(x, 0.3, 9, offset=2, residual=r), want)
        assert torch.equal(ops.dropout(x.contiguous(), 0.3, 9, offset=2, residual=r), want)
        assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.3, 9, offset=2, residual=r), want)
    for k in (2047, 2048, 2049, 5003):  # rows with gaps, about as long as what a workgroup takes
        x = normal(g, 40, k + 2, dtype=dtype)[:, 1:k + 1]
        assert torch.equal(ops.dropout(x, 0.3, 9, offset=2), ops.dropout(x.contiguous(), 0.3, 9, offset=2))
    row = normal(g, 40, dtype=dtype).expand(50, 40)
    assert torch.equal(ops.dropout(row, 0.3, 9), ops.dropout(row.contiguous(), 0.3, 9))


def test_dropout_drops_what_is_not_finite(ops):
    x = torch.full((64, 64), float("nan"), device=DEV)
    x[::2] = float("inf")
    y = ops.dropout(x, 0.5, 3)
    mask = ref.kept(64 * 64, 0.5, 3, 0).view(64, 64).to(DEV)
    assert (y[~mask] == 0).all() and not torch.isfinite(y[mask]).any()
    assert (ops.dropout(x, 1.0, 3) == 0).all()


def test_dropout_keeps_the_right_share(ops):
    """n draws with probability q keep n q, give or take 6 standard deviations sqrt(n q (1 - q)); masks of two
    offsets or seeds agree in q^2 + (1 - q)^2 of the places."""
    n = 1 << 22
    x = torch.ones(n, device=DEV)
    masks = [ops.dropout(x, 0.3, s, offset=o) != 0 for s, o in ((1, 0), (1, 1), (2, 0), (1 << 32, 0))]
    q = 1 - round(0.3 * 65536) / 65536
    for m in masks:
        assert abs(m.sum().item() - n * q) < 6 * (n * q * (1 - q)) ** 0.5
    same = q * q + (1 - q) ** 2
    for i in range(4):
        for j in range(i):
            assert abs((masks[i] == masks[j]).sum().item() - n * same) < 6 * (n * same * (1 - same)) ** 0.5


def test_dropout_seed_on_the_device(ops):
    x = torch.ones(1000, device=DEV, requires_grad=True)
    for seed in (0, 5, -1, 2 ** 62 + 9):
        t = torch.tensor([seed], device=DEV, dtype=torch.int64)
        y = ops.dropout(x, 0.4, t, offset=3)
        assert torch.equal(y, ops.dropout(x, 0.4, seed, offset=3))
        (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        assert torch.equal(dx, y.detach())
    t = torch.tensor([1], device=DEV)
    y = ops.dropout(x, 0.4, t)
    t.add_(1)  # the mask of the forward pass is gone
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], torch.ones_like(y))


def test_dropout_zero_sizes(ops):
    for shape in ((0,), (0, 8), (5, 0), (2, 0, 3)):
        x = torch.ones(shape, device=DEV, requires_grad=True)
        y = ops.dropout(x, 0.5, 1, residual=torch.ones(shape, device=DEV))
        assert y.shape == x.shape
        assert torch.autograd.grad(y, [x], torch.ones_like(y))[0].shape == x.shape


# ---- refusals that need a GPU tensor (the others are in test_decoder_ops_cpu.py) ----

def test_refusals(ops):
    f = lambda *s, dtype=torch.float32: torch.zeros(s, device=DEV, dtype=dtype)
    bad = [lambda: ops.linear(f(4, 8), f(3, 7)), lambda: ops.linear(f(4, 8), f(8)),
           lambda: ops.linear(f(4, 8), f(3, 8), f(4)), lambda: ops.linear(f(4, 8), f(3, 8), f(3, 1)),
           lambda: ops.linear(f(4, 8), f(3, 8), residual=f(3)), lambda: ops.linear(f(4, 8), f(3, 8), residual=f(4, 4)),
           lambda: ops.linear(f(4, 8), f(3, 8, dtype=torch.float16)), lambda: ops.linear(f(4, 8), torch.zeros(3, 8)),
           lambda: ops.linear(f(4, 8, dtype=torch.float64), f(3, 8, dtype=torch.float64)),
           lambda: ops.linear(f(4, 8), f(3, 8), activation="tanh"), lambda: ops.linear(f(), f(3, 8)),
           lambda: ops.linear(f(4, 8), f(3, 8), residual=f(4, 3, dtype=torch.bfloat16)),
           lambda: ops.layer_norm(f(4, 8), f(7)), lambda: ops.layer_norm(f(4, 8), f(8), f(9)),
           lambda: ops.layer_norm(f(4, 8), f(8, dtype=torch.float16)), lambda: ops.layer_norm(f(4, 8), eps=-1.0),
           lambda: ops.layer_norm(f(4, 8, dtype=torch.float16), f(8, dtype=torch.float16), f(8)),
           lambda: ops.layer_norm(f(4, 8, dtype=torch.int32)),
           lambda: ops.dropout(f(4, 8), -0.1, 0), lambda: ops.dropout(f(4, 8), 1.1, 0),
           lambda: ops.dropout(f(4, 8), float("nan"), 0), lambda: ops.dropout(f(4, 8), 0.5, 0.5),
           lambda: ops.dropout(f(4, 8), 0.5, f(1)), lambda: ops.dropout(f(4, 8), 0.5, torch.zeros(1, dtype=torch.int64)),
           lambda: ops.dropout(f(4, 8), 0.5, 0, residual=f(8)), lambda: ops.dropout(f(4, 8), 0.5, 0, offset=1.5)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            pytest.fail("call %d was not refused" % i)
    x = f(4, 8).requires_grad_()
    for y in (ops.linear(x, f(3, 8)), ops.layer_norm(x), ops.dropout(x, 0.5, 0)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y, [x], torch.ones_like(y), create_graph=True)


# ---- together, and the ways they are called ----

def block(ops, x, p, seed, t):
    """Norm, product with activation, product, dropout and sum: a residual block."""
    h = ops.layer_norm(x, t["g"], t["b"])
    h = ops.linear(h, t["w1"], t["b1"], activation="gelu")
    h = ops.linear(h, t["w2"], t["b2"])
    return ops.dropout(h, p, seed, offset=1, residual=x)


def block_tensors(dtype, d=64, wide=128, seed=2):
    g = gen(seed)
    t = {"g": normal(g, d, dtype=dtype, scale=0.1) + 1, "b": normal(g, d, dtype=dtype, scale=0.1),
         "w1": normal(g, wide, d, dtype=dtype, scale=d ** -0.5), "b1": normal(g, wide, dtype=dtype, scale=0.1),
         "w2": normal(g, d, wide, dtype=dtype, scale=wide ** -0.5), "b2": normal(g, d, dtype=dtype, scale=0.1)}
    return {n: v.requires_grad_() for n, v in t.items()}


def block_reference(x, p, seed, t, dy):
    x = x.detach().double().requires_grad_()
    t = {n: v.detach().double().requires_grad_() for n, v in t.items()}
    h = torch.nn.functional.layer_norm(x, x.shape[-1:], t["g"], t["b"])
    h = torch.nn.functional.gelu(h @ t["w1"].t() + t["b1"]) @ t["w2"].t() + t["b2"]
    mask = ref.kept(x.numel(), p, seed, 1).view(x.shape).to(DEV)
    y = x + torch.where(mask, h * (65536 / (65536 - round(p * 65536))), 0.0)
    grads = torch.autograd.grad(y, [x, *t.values()], dy.double())
    return y, dict(zip(["x", *t], grads))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 37, 2000])
def test_block(ops, rows, dtype):
    """A residual block and its gradients against 64 bits.  Each of the block's four operators rounds to the type once
    on the way there and (dz included) up to twice on the way back, and no later step amplifies a relative error by more
    than 4 here (norms with weights about one, products of variance-preserving weights): at most 12 roundings of half a
    step times 4, in the norm of a tensor; float32 adds its sums' (at most 2000 terms) about 2000 e."""
    t = block_tensors(dtype)
    g = gen(rows)
    x, dy = normal(g, rows, 64, dtype=dtype).requires_grad_(), normal(g, rows, 64, dtype=dtype)
    y = block(ops, x, 0.2, 11, t)
    grads = dict(zip(["x", *t], torch.autograd.grad(y, [x, *t.values()], dy)))
    want, want_grads = block_reference(x, 0.2, 11, t, dy)
    bar = 48 * ref.half_step(dtype) + (2000 * ref.E if dtype == torch.float32 else 0.0)
    assert (y.double() - want).norm() <= bar * want.norm()
    for n, w in want_grads.items():
        assert (grads[n].double() - w).norm() <= bar * w.norm(), n


def test_same_bits_every_time(ops):
    """No atomics: a second run of forward and backward gives the same bits, also while another stream is busy."""
    t = block_tensors(torch.bfloat16)
    g = gen(4)
    x, dy = normal(g, 5000, 64, dtype=torch.bfloat16).requires_grad_(), normal(g, 5000, 64, dtype=torch.bfloat16)
    run = lambda: [block(ops, x, 0.2, 11, t)] + list(torch.autograd.grad(block(ops, x, 0.2, 11, t), [x, *t.values()], dy))
    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        noise = run()
    second = run()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, noise):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_works_on_the_current_stream(ops):
    """Inputs made on a side stream and used there, without a synchronisation in between."""
    side = torch.cuda.Stream()
    t = {n: v.detach() for n, v in block_tensors(torch.float32).items()}
    base = normal(gen(6), 100000, 64)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = base
        for _ in range(20):
            x = x * 1.01 + 0.001
        y = block(ops, x, 0.1, 1, t)
    side.synchronize()
    assert torch.equal(y, block(ops, x, 0.1, 1, t))


def test_captured_and_replayed(ops):
    """A training step of the block in a graph: every replay gives what the eager step gives for the inputs and the
    seed of the moment, with eager work between the replays."""
    t = block_tensors(torch.float32)
    g = gen(12)
    x, dy = normal(g, 777, 64).requires_grad_(), normal(g, 777, 64)
    seed = torch.tensor([5], device=DEV)

    def step():
        y = block(ops, x, 0.2, seed, t)
        return [y.detach(), *torch.autograd.grad(y, [x, *t.values()], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(normal(g, 777, 64))
            dy.copy_(normal(g, 777, 64))
            seed.fill_(100 + i)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b), i


def test_capture_refuses_a_leaf_of_a_living_graph(ops):
    """A gradient's accumulator that an eager graph keeps alive belongs to that graph's stream; a captured backward pass
    would have to wait for it across streams.  Refused in the forward call, before anything is captured."""
    x = torch.ones(8, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, 8, device=DEV)
    calls = [lambda: ops.linear(x, w), lambda: ops.layer_norm(x), lambda: ops.dropout(x, 0.5, 1)]
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
            (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(y.detach(), want.detach())
        assert torch.equal(dx, torch.autograd.grad(want, [x], torch.ones_like(want))[0])
        del y, dx, want


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [300, 4200])
def test_linear_gradients_beside_infinities(ops, rows, dtype):
    """Where the derivative is finite although z is not (relu, sigmoid), so are the gradients, at widths that fill no
    step; rows without infinities do not notice."""
    for k, n in ((40, 17), (17, 3), (24, 40)):
        g = gen(n)
        x, w = normal(g, rows, k, dtype=dtype), normal(g, n, k, dtype=dtype)
        w[w == 0] = 1
        x[7, 2], x[rows - 1, k - 1] = float("inf"), -float("inf")
        dy = torch.randint(-3, 4, (rows, n), generator=g, device=DEV).to(dtype)
        for act in ("relu", "sigmoid"):
            xl = x.clone().requires_grad_()
            y = ops.linear(xl, w, activation=act)
            (dx,) = torch.autograd.grad(y, [xl], dy)
            assert torch.isfinite(dx).all()
            for r, c in ((7, 2), (rows - 1, k - 1)):
                up = (w[:, c] > 0) == (x[r, c] > 0)  # z = +inf there, -inf elsewhere
                assert torch.equal(y[r], torch.where(up, float("inf") if act == "relu" else 1.0, 0.0).to(dtype))
                slope = up.double() if act == "relu" else torch.zeros(n, device=DEV, dtype=torch.float64)
                want = (dy[r].double() * slope) @ w.double()
                bound = (n + 2) * 2 * ref.E * ((dy[r].double() * slope).abs() @ w.double().abs())
                ref.assert_within(dx[r], (want, ref.rounded(want, bound, dtype)), act)


def test_far_offsets(ops):
    """More than 2^31 elements: the last rows come out as they do on their own."""
    rows, d = (1 << 21) + 300, 1032
    x = torch.empty(rows, d, device=DEV, dtype=torch.bfloat16).fill_(0.5)
    tail = normal(gen(1), 300, d, dtype=torch.bfloat16)
    x[-300:] = tail
    w = normal(gen(2), 5, d, dtype=torch.bfloat16, scale=0.03)
    ref.assert_within(ops.linear(x, w)[-300:], ref.linear(tail, w, None, "none", None, None)["y"], "y")
    assert torch.equal(ops.layer_norm(x)[-300:], ops.layer_norm(tail))
    y = ops.dropout(x, 0.5, 3)
    kept = y[-300:] != 0
    assert torch.equal(y[-300:], torch.where(kept, tail * 2, 0.0))
    first = rows * d - 8000  # (a multiple of 8: whole blocks)
    mask = [bool(v) for v in kept.reshape(-1)[-8000:].tolist()]
    bits = _kept_from(first, 8000, 0.5, 3)
    assert mask == [b and v for b, v in zip(bits, (tail.reshape(-1)[-8000:] != 0).tolist())]
    # the reduction over that many rows: ones, whose sums are exact
    del y, kept
    x.fill_(1.0)
    dy = torch.zeros(rows, 5, device=DEV, dtype=torch.bfloat16)
    dy[-256:] = 1.0
    wl, xl = w.requires_grad_(), x.requires_grad_()
    b = torch.zeros(5, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    dx, dw, db = torch.autograd.grad(ops.linear(xl, wl, b), [xl, wl, b], dy)
    assert (dw == 256).all() and (db == 256).all() and (dx[:-256] == 0).all() and (dx[-256:] == dx[-1]).all()


def _kept_from(first, count, p, seed):
    word, out = 0xFFFFFFFF, []
    for block in range(first // 8, (first + count) // 8):
        a, b, c, d, k0, k1 = block & word, block >> 32, 0, 0, seed, 0
        for _ in range(7):
            l, h = a * 0xD2511F53, c * 0xCD9E8D57
            a, b, c, d = (h >> 32) ^ b ^ k0, h & word, (l >> 32) ^ d ^ k1, l & word
            k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
        out += [(v >> s & 0xFFFF) >= round(p * 65536) for v in (a, b, c, d) for s in (0, 16)]
    return out


@pytest.mark.parametrize("dtype", DTYPES)
def test_lazily_negated_tensors(ops, dtype):
    """A view whose memory holds the negated values counts as its values: the same bits as from a plain copy."""
    g = gen(12)

    def pair(*shape):
        lazy = torch._neg_view(normal(g, *shape, dtype=dtype))
        assert lazy.is_neg()
        return lazy, lazy.clone().resolve_neg()

    (x, px), (w, pw), (b, pb), (r, pr), (dy, pdy) = pair(200, 40), pair(24, 40), pair(24), pair(200, 24), pair(200, 24)
    (v, pv), (c, pc) = pair(40), pair(40)
    calls = [lambda x, w, b, r, v, c: ops.linear(x, w, b, activation="gelu", residual=r),
             lambda x, w, b, r, v, c: ops.layer_norm(x, v, c) @ torch.ones(40, 24, device=DEV, dtype=dtype),
             lambda x, w, b, r, v, c: ops.dropout(x, 0.3, 5)[:, :24] + r]
    for call in calls:
        assert torch.equal(call(x, w, b, r, v, c), call(px, pw, pb, pr, pv, pc))
    leaf = px.clone().requires_grad_(True)
    lazy, plain = (torch.autograd.grad(ops.linear(leaf, pw, pb, activation="silu"), leaf, d)[0] for d in (dy, pdy))
    assert torch.equal(lazy, plain)
