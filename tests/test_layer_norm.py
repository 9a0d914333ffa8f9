"""Layer norm forwards and backwards (include/pt_feed_forward.h) against
float64, element by element.

Tolerances: a result is rounded once to its type (unit roundoff u) and
computed in float32 (unit roundoff e = 2^-24).  A thread adds at most 32
elements in a row and the partial sums are joined by trees of at most 10
levels, so a row's mean is within 48 e of the mean of |x|; with the roundings
of the difference, the variance and the products around it, 64 e times the
magnitudes that enter covers an element.  A sum over R rows is within R + 64
roundings of the sum of its terms' magnitudes.
"""
import ctypes

import pytest

import phptensors as P

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
E = 2.0 ** -24
EPS = 1e-5


def arr(t):
    return None if t is None else P.CudaArray.from_torch(t)


def make(rows, cols, dtype, seed, layout):
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = torch.rand(cols, generator=g, device="cuda") + 0.5

    def one(offset):
        v = torch.randn(rows, cols, generator=g, device="cuda") * spread + offset
        if layout == "padded":        # rows at a pitch that breaks 16-byte alignment
            base = torch.full((rows, cols + 3), float("nan"), device="cuda", dtype=DT[dtype])
            base[:, 1:cols + 1] = v
            return base[:, 1:cols + 1]
        if layout == "transposed":
            return v.to(DT[dtype]).t().contiguous().t()
        return v.to(DT[dtype])
    return (one(0.5), one(0.0), (torch.randn(cols, generator=g, device="cuda") + 1).to(DT[dtype]),
            torch.randn(cols, generator=g, device="cuda").to(DT[dtype]))


def check_forward(x, gamma, beta, y, mean, rstd, dtype):
    x = x.double()
    g = torch.ones(x.shape[-1], device="cuda").double() if gamma is None else gamma.double()
    b = torch.zeros_like(g) if beta is None else beta.double()
    m = x.mean(-1, keepdim=True)
    r = ((x - m).square().mean(-1, keepdim=True) + EPS) ** -0.5
    n = (x - m) * r
    want = n * g + b
    big = x.abs().amax(-1, keepdim=True) * r
    tol = UNIT[dtype] * want.abs() + 64 * E * (g.abs() * (big + n.abs() * (1 + big)) + b.abs())
    if dtype == "float16":
        tol += 2.0 ** -25             # spacing of its smallest values
    assert torch.all((y.double() - want).abs() <= tol)
    if mean is not None:
        assert torch.all((mean.double() - m[..., 0]).abs() <= 64 * E * x.abs().amax(-1))
        assert torch.all((rstd.double() / r[..., 0] - 1).abs() <= 64 * E * (1 + big[..., 0]))


CASES = [(1, 1), (1, 7), (3, 8), (5, 64), (2, 100), (130, 257), (64, 768), (9, 1531), (33, 2050),
         (700, 1024), (7, 4096), (3, 8192), (2, 20000), (2, 40001)]


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,cols", CASES)
@pytest.mark.parametrize("layout", ["plain", "padded", "transposed"])
def test_forward_and_backward(dtype, rows, cols, layout):
    x, grad, gamma, beta = make(rows, cols, dtype, rows * 31 + cols, layout)
    y, mean, rstd = arr(x).layer_norm(arr(gamma), arr(beta), EPS, save_stats=True)
    check_forward(x, gamma, beta, y.to_torch(), mean.to_torch(), rstd.to_torch(), dtype)
    dx, dg, db = P.layer_norm_backward(arr(grad), arr(x), arr(gamma), mean, rstd)
    m, r = mean.to_torch().double()[:, None], rstd.to_torch().double()[:, None]
    n = (x.double() - m) * r
    a = grad.double() * gamma.double()
    an = (a * n).mean(1, keepdim=True)
    want = r * (a - a.mean(1, keepdim=True) - n * an)
    big = (x.double().abs() + m.abs()) * r         # what n is the difference of
    ma, mn = a.abs().mean(1, keepdim=True), (a.abs() * big).mean(1, keepdim=True)
    tol = UNIT[dtype] * want.abs() + 64 * E * r * (a.abs() + ma + (n.abs() + big) * mn)
    if dtype == "float16":
        tol += 2.0 ** -25
    assert torch.all((dx.to_torch().double() - want).abs() <= tol)
    terms = grad.double() * n
    slack = (rows + 64) * E
    assert torch.all((dg.to_torch().double() - terms.sum(0)).abs()
                     <= slack * (grad.double().abs() * (n.abs() + big)).sum(0))
    assert torch.all((db.to_torch().double() - grad.double().sum(0)).abs()
                     <= slack * grad.double().abs().sum(0))


@gpu
def test_gradient_against_differences():
    """dx, dgamma and dbeta against central differences of the float64 norm."""
    x, grad, gamma, beta = make(4, 40, "float32", 5, "plain")
    y, mean, rstd = arr(x).layer_norm(arr(gamma), arr(beta), EPS, save_stats=True)
    dx, dg, db = P.layer_norm_backward(arr(grad), arr(x), arr(gamma), mean, rstd)

    def loss(x, gamma, beta):
        m = x.mean(1, keepdim=True)
        n = (x - m) * ((x - m).square().mean(1, keepdim=True) + EPS) ** -0.5
        return ((n * gamma + beta) * grad.double()).sum()
    at = [x.double(), gamma.double(), beta.double()]
    h = 1e-5
    for k, got in enumerate((dx, dg, db)):
        flat = at[k].reshape(-1)
        num = torch.empty_like(flat)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss(*at)
            flat[i] = keep - h
            num[i] = (up - loss(*at)) / (2 * h)
            flat[i] = keep
        # differences: h^2 times a third derivative of order 10; float32: 1e-5
        assert torch.allclose(got.to_torch().double().reshape(-1), num, rtol=1e-4, atol=1e-4)


@gpu
def test_float32_parameters_no_parameters_and_ranks():
    x, grad, gamma, beta = make(24, 96, "bfloat16", 3, "plain")
    y = arr(x).layer_norm(arr(gamma.float()), arr(beta.float()), EPS)
    assert torch.equal(y.to_torch(), arr(x).layer_norm(arr(gamma), arr(beta), EPS).to_torch())
    y = arr(x).layer_norm(eps=EPS).to_torch()
    check_forward(x, None, None, y, None, None, "bfloat16")
    x4 = x.view(2, 3, 4, 96).permute(2, 0, 1, 3)          # leading axes that do not merge
    y4, m4, r4 = arr(x4).layer_norm(eps=EPS, save_stats=True)
    assert y4.getShape() == [4, 2, 3, 96] and m4.getShape() == [4, 2, 3]
    assert torch.equal(y4.to_torch(), y.view(2, 3, 4, 96).permute(2, 0, 1, 3))
    one = arr(x[0]).layer_norm(eps=EPS)                   # a single row as rank 1
    assert torch.equal(one.to_torch(), y[0])
    dx, dg, db = P.layer_norm_backward(
        arr(grad.view(2, 3, 4, 96).permute(2, 0, 1, 3)), arr(x4), None, m4, r4)
    y2, m2, r2 = arr(x).layer_norm(eps=EPS, save_stats=True)
    flat, _, fb = P.layer_norm_backward(arr(grad), arr(x), None, m2, r2)
    assert torch.equal(dx.to_torch(), flat.to_torch().view(2, 3, 4, 96).permute(2, 0, 1, 3))
    assert torch.allclose(db.to_torch(), fb.to_torch(), rtol=1e-5, atol=1e-5)


@gpu
def test_constant_rows_nonfinite_rows_and_no_rows():
    x = torch.full((3, 33), 7.0, device="cuda", dtype=torch.float16)
    beta = torch.arange(33, device="cuda").half()
    y = arr(x).layer_norm(None, arr(beta), EPS).to_torch()
    assert torch.equal(y, beta.expand(3, 33))            # no variance: beta alone
    x = torch.randn(4, 64, device="cuda")
    x[1, 5], x[2, 9] = float("nan"), float("inf")
    y, mean, rstd = arr(x).layer_norm(eps=EPS, save_stats=True)
    check_forward(x[[0, 3]], None, None, y.to_torch()[[0, 3]], None, None, "float32")
    assert torch.isnan(y.to_torch()[[1, 2]]).all()       # only their own rows are lost
    e = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = arr(e).layer_norm(save_stats=True)
    dx, dg, db = P.layer_norm_backward(arr(e), arr(e), None, mean, rstd)
    assert y.getShape() == [0, 16] and not dg.to_torch().any() and not db.to_torch().any()


@gpu
def test_same_bits_again_and_on_another_stream():
    x, grad, gamma, beta = make(3000, 520, "bfloat16", 11, "plain")
    y, mean, rstd = arr(x).layer_norm(arr(gamma), arr(beta), EPS, save_stats=True)
    first = [t.to_torch() for t in P.layer_norm_backward(arr(grad), arr(x), arr(gamma), mean, rstd)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [t.to_torch()
                 for t in P.layer_norm_backward(arr(grad), arr(x), arr(gamma), mean, rstd)]
    side.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@gpu
def test_offsets_beyond_32_bits():
    """2.2e9 elements: the last rows are those of a call on them alone."""
    rows, cols = 270001, 8192
    x = torch.randn(rows, cols, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = arr(x).layer_norm(save_stats=True)
    tail = x[rows - 3:].contiguous()
    few, fm, fr = arr(tail).layer_norm(save_stats=True)
    check_forward(tail, None, None, y.to_torch()[rows - 3:], mean.to_torch()[rows - 3:],
                  rstd.to_torch()[rows - 3:], "bfloat16")
    dx, dg, db = P.layer_norm_backward(y, arr(x), None, mean, rstd)
    fx, _, _ = P.layer_norm_backward(arr(y.to_torch()[rows - 3:].contiguous()), arr(tail), None,
                                     arr(mean.to_torch()[rows - 3:].contiguous()),
                                     arr(rstd.to_torch()[rows - 3:].contiguous()))
    assert torch.equal(dx.to_torch()[rows - 3:], fx.to_torch())
    want = torch.zeros(cols, device="cuda").double()
    for a in range(0, rows, 30000):
        want += y.to_torch()[a:a + 30000].double().sum(0)
    slack = (rows + 64) * E * y.to_torch()[:1000].double().abs().mean() * rows
    assert torch.all((db.to_torch().double() - want).abs() <= slack)


def _pt(shape, dtype):
    t = P.PtTensor()
    t.data, t.dtype, t.ndims = 4096, P.DTYPE_CODES[dtype], len(shape)
    for i, (d, s) in enumerate(zip(shape, P._contiguous_strides(shape))):
        t.shape[i], t.strides[i] = d, s
    return t


def test_refusals():
    """Arguments are refused before any CUDA call."""
    lib, ref = P.library(), ctypes.byref
    x, y, g = _pt([4, 8], "float16"), _pt([4, 8], "float16"), _pt([8], "float16")

    def forward(x=x, gamma=g, beta=g, eps=1e-5, y=y, mean=16, rstd=16):
        return lib.pt_layer_norm(ref(x), ref(gamma), ref(beta), eps, ref(y), mean, rstd, None)
    for bad in (dict(x=_pt([4, 8], "float64")), dict(y=_pt([4, 8], "float32")),
                dict(y=_pt([8, 4], "float16")), dict(gamma=_pt([7], "float16")),
                dict(beta=_pt([8], "bfloat16")), dict(eps=-1.0), dict(eps=float("nan")),
                dict(mean=None), dict(x=_pt([4, 0], "float16"), y=_pt([4, 0], "float16"))):
        assert forward(**bad) == P.PT_INVALID_ARGUMENT, bad
        assert lib.pt_last_error().startswith(b"layer norm")
    wide = _pt([2, 2, 2, 2, 2, 8], "float16")
    for i in range(5):
        wide.strides[i] = 1000 * (3 * i + 1)             # five axes that do not merge
    assert forward(x=wide, y=_pt([2, 2, 2, 2, 2, 8], "float16")) == P.PT_INVALID_ARGUMENT
    strided = _pt([4, 8], "float16")
    strided.strides[0] = 16
    assert forward(y=strided) == P.PT_INVALID_ARGUMENT
    size = ctypes.c_size_t(0)
    assert lib.pt_layer_norm_backward(ref(x), ref(x), ref(g), 16, 16, ref(y), 16, 16, None,
                                      ref(size), None) == P.PT_WORKSPACE
    assert size.value == lib.pt_layer_norm_backward_workspace(4, 8) > 0
    assert lib.pt_layer_norm_backward(ref(_pt([4, 9], "float16")), ref(x), ref(g), 16, 16, ref(y),
                                      16, 16, None, ref(size), None) == P.PT_INVALID_ARGUMENT


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("rows,cols", [(5, 40), (9, 1024), (4, 1531), (3, 8192), (2, 20000)])
@pytest.mark.parametrize("offset", [1e3, 1e4])
def test_backward_of_rows_far_from_zero(dtype, rows, cols, offset):
    """n = (x - mean) rstd from the statistics given: the difference of two
    near floats is exact, so n is within 4 e of its own size however far the
    row is from zero, a constant row (the last one) has n = 0, and the
    tolerance holds no |x| rstd."""
    x, grad, gamma, _ = make(rows, cols, dtype, cols, "plain")
    x = (x.float() + offset).to(DT[dtype])
    x[-1] = offset + 0.3
    mean = x.double().mean(1).float()
    mean[-1] = x[-1, 0].float()
    d = x.double() - mean.double()[:, None]
    rstd = ((d.square().mean(1) + EPS) ** -0.5).float()
    dx, dg, db = P.layer_norm_backward(arr(grad), arr(x), arr(gamma), arr(mean), arr(rstd))
    r = rstd.double()[:, None]
    n = d * r
    assert not n[-1].any()
    a = grad.double() * gamma.double()
    want = r * (a - a.mean(1, keepdim=True) - n * (a * n).mean(1, keepdim=True))
    ma, mn = a.abs().mean(1, keepdim=True), (a * n).abs().mean(1, keepdim=True)
    tol = UNIT[dtype] * want.abs() + 64 * E * r * (a.abs() + ma + n.abs() * mn)
    if dtype == "float16":
        tol += 2.0 ** -25
    assert torch.all((dx.to_torch().double() - want).abs() <= tol)
    terms = grad.double() * n
    assert torch.all((dg.to_torch().double() - terms.sum(0)).abs()
                     <= (rows + 64) * E * terms.abs().sum(0))


def test_sizes_that_pass_32_bits_are_refused():
    """Rows stay 1024 columns below 2^31: a thread's column steps past the end
    before it compares.  Refused before any CUDA call."""
    lib, ref = P.library(), ctypes.byref
    x = _pt([1, 2 ** 31 - 1024], "bfloat16")
    assert lib.pt_layer_norm(ref(x), None, None, 1e-5, ref(x), None, None,
                             None) == P.PT_INVALID_ARGUMENT
    assert b"2^31" in lib.pt_last_error()
    size = ctypes.c_size_t(0)
    assert lib.pt_layer_norm_backward(ref(x), ref(x), None, 16, 16, ref(x), 16, 16, None,
                                      ref(size), None) == P.PT_INVALID_ARGUMENT
    assert b"2^31" in lib.pt_last_error()


@gpu
def test_parameter_gradients_beyond_32_bits():
    """Sums over 2.2e9 elements as wholes: rows left out behind element 2^31, 3 %
    of them, would be 17 % of dbeta's norm and 3 % of dgamma's.  A sum is joined
    from chains of fewer than 1000 additions in float32, each within e of a
    partial sum that is no larger than the whole in the mean: below 1000 e."""
    rows, cols = 270001, 8192
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = arr(x).layer_norm(save_stats=True)
    dx, dg, db = P.layer_norm_backward(y, arr(x), None, mean, rstd)
    grad, m, r = y.to_torch(), mean.to_torch(), rstd.to_torch()
    sums = torch.zeros(2, cols, device="cuda").double()
    for at in range(0, rows, 15000):
        part = slice(at, at + 15000)
        dy = grad[part].double()
        sums[0] += (dy * ((x[part].double() - m[part, None]) * r[part, None].double())).sum(0)
        sums[1] += dy.sum(0)
    for got, want in ((dg, sums[0]), (db, sums[1])):
        assert (got.to_torch().double() - want).norm() <= 1000 * E * want.norm()
