"""Linear layers, plain and grouped by expert (include/pt_feed_forward.h),
against float64, element by element.

Tolerances, with u the unit roundoff of the operands' type and A = |x| . |w|
the magnitudes a dot product of length K adds: products of 16-bit values are
exact in float32 and the tensor core truncates its sum, so a product is within
(K + 8) 2^-23 A; float32 operands lose less than 2^-22 A in their parts as
well.  Activations have slopes below 1.2 and are computed to 2^-16 of their
argument (16-bit results) or 2^-20.  A result is rounded once, and backwards
the 16-bit dz once before it, which moves a product by at most u |dz| . |w|.
"""
import ctypes
import math

import pytest

import phptensors as P

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}
ALL = ["bfloat16", "float16", "float32"]


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        assert P.device_status() == 0


def arr(t):
    return None if t is None else P.CudaArray.from_torch(t)


def act64(z, name):
    F = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: F.relu(z), "tanh": lambda: torch.tanh(z),
            "sigmoid": lambda: torch.sigmoid(z), "silu": lambda: F.silu(z),
            "gelu": lambda: F.gelu(z), "gelu_tanh": lambda: F.gelu(z, approximate="tanh")}[name]()


def slope64(z, name):
    z = z.clone().requires_grad_()
    return torch.autograd.grad(act64(z, name).sum(), z)[0]


def product_slack(k, dtype):
    return (k + 8) * 2.0 ** -23 + (2.0 ** -22 if dtype == "float32" else 0.0)


def act_slack(z, dtype):
    return (2.0 ** -16 if UNIT[dtype] > 2.0 ** -20 else 2.0 ** -20) * z.abs()


def strided(t, layout):
    """The values of t in another layout."""
    if layout == "column":
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    if layout == "padded":          # rows at an odd pitch, off by one element
        shape = list(t.shape)
        shape[-1] += 3
        base = torch.full(shape, float("nan"), dtype=t.dtype, device=t.device)
        base[..., 1:1 + t.shape[-1]] = t
        return base[..., 1:1 + t.shape[-1]]
    if layout == "gaps":            # every second element
        base = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)
        base[..., ::2] = t
        return base[..., ::2]
    return t


def spans_of(ends, rows):
    spans, at = [], 0
    for e in ends:
        e = min(max(e, at), rows)
        spans.append((at, e))
        at = e
    return spans


def case(rows, inner, cols, dtype, seed, groups=None, layout="plain"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return strided((torch.randn(*shape, generator=g, device="cuda") * scale).to(DT[dtype]),
                       layout)
    lead = [] if groups is None else [groups]
    return {"x": rnd(rows, inner), "w": rnd(*lead, inner, cols, scale=inner ** -0.5),
            "bias": (torch.randn(*lead, cols, generator=g, device="cuda") * 0.5).to(DT[dtype]),
            "res": rnd(rows, cols), "grad": rnd(rows, cols), "pre": rnd(rows, cols)}


def check_forward(c, y, pre, dtype, act, spans, bias=True, res=True):
    x, w = c["x"].double(), c["w"].double().reshape(len(spans), *c["w"].shape[-2:])
    y, pre = y.double(), None if pre is None else pre.double()
    for e, (a, b) in enumerate(spans):
        z = x[a:b] @ w[e]
        mag = x[a:b].abs() @ w[e].abs()
        if bias:
            be = c["bias"].double().reshape(len(spans), -1)[e]
            z, mag = z + be, mag + be.abs()
        slack = product_slack(x.shape[1], dtype) * mag + TINY[dtype]
        want = act64(z, act)
        if pre is not None:
            assert torch.all((pre[a:b] - z).abs() <= slack + UNIT[dtype] * z.abs()), (act, e)
        if res:
            want = want + c["res"][a:b].double()
        tol = 1.2 * slack + act_slack(z, dtype) + UNIT[dtype] * want.abs()
        tol = tol * (1 + 2 * UNIT[dtype]) + (2.0 ** -23 * c["res"][a:b].double().abs() if res else 0)
        assert torch.all((y[a:b] - want).abs() <= tol), (act, e)
    rest = spans[-1][1]
    assert not y[rest:].any() and (pre is None or not pre[rest:].any())


def check_backward(c, out, dtype, act, spans, dw_dtype=None):
    dx, dw, db = [t.to_torch().double() for t in out]
    x, w = c["x"].double(), c["w"].double().reshape(len(spans), *c["w"].shape[-2:])
    u = UNIT[dtype]
    dw, db = dw.reshape(w.shape), db.reshape(len(spans), -1)
    for e, (a, b) in enumerate(spans):
        z, grad = c["pre"][a:b].double(), c["grad"][a:b].double()
        slope = slope64(z, act) if act != "none" else torch.ones_like(z)
        dz = grad * slope
        off = grad.abs() * 4 * act_slack(z.abs() + 1, dtype) if act != "none" else 0 * grad
        mag = dz.abs() + off
        # dz: its activation's error, and its rounding when it is one
        dz_off = off + (u * mag if act != "none" and dtype != "float32" else 0) + TINY[dtype]
        k = w.shape[2]
        tol = dz_off @ w[e].abs().T + product_slack(k, dtype) * (mag @ w[e].abs().T)
        want = dz @ w[e].T
        assert torch.all((dx[a:b] - want).abs() <= tol * (1 + u) + u * want.abs() + TINY[dtype]), e
        tol = x[a:b].abs().T @ dz_off + product_slack(b - a, dtype) * (x[a:b].abs().T @ mag)
        want = x[a:b].T @ dz
        ud = UNIT[dw_dtype or dtype]
        assert torch.all((dw[e] - want).abs()
                         <= tol * (1 + ud) + ud * want.abs() + TINY[dtype]), e
        tol = off.sum(0) + (b - a + 64) * 2.0 ** -24 * mag.sum(0)
        assert torch.all((db[e] - dz.sum(0)).abs() <= tol), e
    assert not dx[spans[-1][1]:].any()


# a case beyond one tile of each kernel in every direction, and odd ones
SIZES = [(1, 64, 64), (65, 2100, 130), (2100, 130, 72), (2, 8, 8), (3, 7, 5), (8, 128, 264), (31, 65, 1), (33, 1, 70), (129, 72, 520),
         (256, 256, 256), (257, 200, 96), (300, 1000, 136), (700, 264, 312)]


PATHS = ["auto", "tensor-core", "tensor-core-pair", "simt"]


@pytest.fixture
def path(request):
    """One of the kernel families: few rows, CTA pairs, CUDA cores."""
    before = P.set_kernel_path(request.param)
    yield request.param
    P.library().gemm_sm100_set_path(before)


@gpu
@pytest.mark.parametrize("path", PATHS, indirect=True)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,inner,cols", SIZES)
def test_linear(dtype, rows, inner, cols, path):
    c = case(rows, inner, cols, dtype, rows + inner)
    for act, bias, res in (("gelu", True, True), ("none", False, False), ("silu", True, False)):
        y, pre = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]) if bias else None, act,
                                    arr(c["res"]) if res else None, save_pre=True)
        check_forward(c, y.to_torch(), pre.to_torch(), dtype, act, [(0, rows)], bias, res)
    for act in ("gelu", "none"):
        out = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), arr(c["pre"]), act)
        check_backward(c, out, dtype, act, [(0, rows)])


@gpu
@pytest.mark.parametrize("path", PATHS[1:], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("act", sorted(P.ACTIVATIONS))
def test_activations(dtype, act, path):
    c = case(70, 96, 200, dtype, 5)
    c["bias"] = (c["bias"] * 8).contiguous()             # far into both tails
    c["pre"] = c["pre"] * 4
    y = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]), act, arr(c["res"]))
    check_forward(c, y.to_torch(), None, dtype, act, [(0, 70)])
    out = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), arr(c["pre"]), act)
    check_backward(c, out, dtype, act, [(0, 70)])


@gpu
@pytest.mark.parametrize("path", PATHS[1:], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["column", "padded", "gaps"])
def test_layouts(dtype, layout, path):
    c = case(150, 88, 264, dtype, 9, layout=layout)
    y, pre = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"].float()), "silu", arr(c["res"]),
                                save_pre=True)
    check_forward(c, y.to_torch(), pre.to_torch(), dtype, "silu", [(0, 150)])
    out = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), arr(c["pre"]), "silu")
    check_backward(c, out, dtype, "silu", [(0, 150)])
    # a residual row that serves every row
    c["res"] = c["res"][:1].expand(150, 264)
    y = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]), "silu", arr(c["res"]))
    check_forward(c, y.to_torch(), None, dtype, "silu", [(0, 150)])


ENDS = [[0, 0, 5, 5, 40], [1800, 1800, 1843], [64, 128, 192, 256], [1, 2, 3, 400], [300], [0, 0, 0],
        [255, 256, 513, 514, 600], [10, 4, 90, 70, 5000]]      # the last one: not in order


@gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ends", ENDS)
@pytest.mark.parametrize("layout,path", [("plain", p) for p in PATHS] + [
    ("column", "tensor-core-pair"), ("column", "simt"), ("padded", "tensor-core"),
    ("padded", "simt")], indirect=["path"])
def test_grouped(dtype, ends, layout, path):
    rows, inner, cols = max(e for e in ends if e < 5000) + 7, 136, 264
    c = case(rows, inner, cols, dtype, 21, groups=len(ends), layout=layout)
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")
    spans = spans_of(ends, rows)
    # rows of no group hold NaN: nothing of them may reach any result
    for k in ("x", "grad", "pre", "res"):
        c[k][spans[-1][1]:] = float("nan")
    y, pre = arr(c["x"]).grouped_linear(arr(c["w"]), at, arr(c["bias"]), "gelu_tanh",
                                        arr(c["res"]), save_pre=True)
    check_forward(c, y.to_torch(), pre.to_torch(), dtype, "gelu_tanh", spans)
    for act in ("gelu_tanh", "none"):
        out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at,
                                        arr(c["pre"]), act)
        check_backward(c, out, dtype, act, spans)


@gpu
@pytest.mark.parametrize("path", PATHS[1:], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
def test_nonfinite_rows_stay_in_their_group(dtype, path):
    ends = [70, 75, 140]
    c = case(140, 72, 80, dtype, 4, groups=3)
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")
    spans = spans_of(ends, 140)
    for k in ("x", "grad", "res"):
        c[k][70:75] = float("nan")
        c[k][72] = float("inf")
    y = arr(c["x"]).grouped_linear(arr(c["w"]), at, None, "none", arr(c["res"])).to_torch()
    dx, dw, db = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at)
    for t, rows in ((y, True), (dx.to_torch(), True), (dw.to_torch(), False),
                    (db.to_torch(), False)):
        bad = t[70:75] if rows else t[1]
        good = torch.cat([t[:70], t[75:]]) if rows else t[[0, 2]]
        assert not torch.isfinite(bad).any() and torch.isfinite(good).all()


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_weight_gradient_in_float32(dtype):
    ends = [33, 33, 200]
    c = case(200, 96, 168, dtype, 8, groups=3)
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")
    out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at,
                                    weight_grad_dtype="float32")
    assert out[1].dtype() == "float32"
    check_backward(c, out, dtype, "none", spans_of(ends, 200), dw_dtype="float32")


@gpu
def test_float32_modes():
    """Strict float32 is near float64 as a whole as well; the tf32 mode keeps
    16 bits of each operand (parts of 8 and 8: 2^-15 of the magnitudes)."""
    c = case(400, 2048, 264, "float32", 6)
    before = P.set_kernel_path("tensor-core-pair")
    y = arr(c["x"]).linear(arr(c["w"])).to_torch().double()
    want = c["x"].double() @ c["w"].double()
    assert (y - want).norm() <= 1e-6 * want.norm()
    P.cuda_set_matmul_precision("tf32")
    try:
        t = arr(c["x"]).linear(arr(c["w"])).to_torch().double()
    finally:
        P.cuda_set_matmul_precision("fp32-strict")
        P.library().gemm_sm100_set_path(before)
    mag = c["x"].double().abs() @ c["w"].double().abs()
    assert torch.all((t - want).abs() <= (2.0 ** -15 + 2056 * 2.0 ** -23) * mag)


@gpu
def test_gradient_against_differences():
    c = case(9, 12, 10, "float32", 2, groups=3)
    ends = torch.tensor([4, 4, 9], dtype=torch.int32, device="cuda")
    spans = [(0, 4), (4, 4), (4, 9)]
    y, pre = arr(c["x"]).grouped_linear(arr(c["w"]), ends, arr(c["bias"]), "gelu", save_pre=True)
    out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), ends, pre, "gelu")
    at = [c["x"].double(), c["w"].double(), c["bias"].double()]

    def loss():
        z = torch.cat([at[0][a:b] @ at[1][e] + at[2][e] for e, (a, b) in enumerate(spans)])
        return (act64(z, "gelu") * c["grad"].double()).sum()
    h = 1e-5
    for k, got in enumerate(out):
        flat = at[k].reshape(-1)
        num = torch.empty_like(flat)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss()
            flat[i] = keep - h
            num[i] = (up - loss()) / (2 * h)
            flat[i] = keep
        # differences: h^2 times a third derivative of order 10; float32: 1e-5
        assert torch.allclose(got.to_torch().double().reshape(-1), num, rtol=1e-4, atol=1e-4)


@gpu
def test_ranks_empty_tensors_and_parts_of_the_gradient():
    c = case(24, 64, 72, "bfloat16", 12)
    y = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]), "relu").to_torch()
    x4 = c["x"].view(2, 3, 4, 64).permute(2, 0, 1, 3)
    y4 = arr(x4).linear(arr(c["w"]), arr(c["bias"]), "relu")
    assert y4.getShape() == [4, 2, 3, 72]
    assert torch.equal(y4.to_torch(), y.view(2, 3, 4, 72).permute(2, 0, 1, 3))
    res4 = c["res"].view(2, 3, 4, 72).permute(2, 0, 1, 3)      # rows of no single stride
    y4 = arr(x4).linear(arr(c["w"]), arr(c["bias"]), "relu", arr(res4))
    y = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]), "relu", arr(c["res"])).to_torch()
    assert torch.equal(y4.to_torch(), y.view(2, 3, 4, 72).permute(2, 0, 1, 3))
    full = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), arr(c["pre"]), "relu")
    for k, want in enumerate(("inputs", "weights", "bias")):
        only = {n: n == want for n in ("inputs", "weights", "bias")}
        got = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), arr(c["pre"]), "relu",
                                **only)
        assert [t is not None for t in got] == [i == k for i in range(3)]
        assert torch.equal(got[k].to_torch(), full[k].to_torch())
    none = c["x"][:0]
    assert arr(none).linear(arr(c["w"])).getShape() == [0, 72]
    dx, dw, db = P.linear_backward(arr(c["grad"][:0]), arr(none), arr(c["w"]), arr(c["pre"][:0]),
                                   "relu")
    assert not dw.to_torch().any() and not db.to_torch().any()
    # an inner size of zero leaves the epilogue alone
    y = arr(c["x"][:, :0]).linear(arr(c["w"][:0]), arr(c["bias"]), "silu", arr(c["res"]))
    c0 = dict(c, x=c["x"][:, :0], w=c["w"][:0])
    check_forward(c0, y.to_torch(), None, "bfloat16", "silu", [(0, 24)])


@gpu
def test_choice_of_kernel():
    """By the work and the rows, with the name of the last one kept."""
    def kernel(rows, inner, cols, dtype, layout="plain"):
        c = case(rows, inner, cols, dtype, 1, layout=layout)
        arr(c["x"]).linear(arr(c["w"]))
        return P.cuda_get_backend_info()["kernel"]
    assert kernel(8, 512, 512, "bfloat16") == "ragged-bf16-128x64"
    assert kernel(4096, 256, 2048, "float16") == "ragged2-f16-256x256"
    assert kernel(4096, 1024, 1024, "float32") == "ragged2-bf16x3-256x256"
    assert kernel(16, 256, 256, "float32") == "ragged-simt-f32"
    assert kernel(16, 255, 257, "float16") == "ragged-simt-f16"


@gpu
@pytest.mark.parametrize("path", PATHS[1:], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
def test_same_bits_again_on_another_stream_and_in_a_graph(dtype, path):
    c = case(500, 328, 264, dtype, 15, groups=4)
    ends = torch.tensor([100, 101, 380, 500], dtype=torch.int32, device="cuda")

    def both():
        y, pre = arr(c["x"]).grouped_linear(arr(c["w"]), ends, arr(c["bias"]), "gelu",
                                            arr(c["res"]), save_pre=True)
        out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), ends, pre, "gelu")
        return [t.to_torch() for t in (y, pre, *out)]
    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = both()
        graph.replay()
    side.synchronize()
    for a, b, k in zip(first, again, kept):
        assert torch.equal(a, b) and torch.equal(a, k)


@gpu
@pytest.mark.parametrize("path", PATHS, indirect=True)
@pytest.mark.parametrize("dtype", ALL)
def test_broadcast_operands(dtype, path):
    """One weight for all groups, one row for all rows, one upstream gradient:
    strides of zero.  Each group still has its own gradient."""
    ends = [40, 40, 100]
    c = case(100, 72, 136, dtype, 17, groups=3)
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")
    spans = spans_of(ends, 100)
    for name, shape in (("w", (3, 72, 136)), ("x", (100, 72)), ("grad", (100, 136)),
                        ("pre", (100, 136)), ("res", (100, 136))):
        c[name] = c[name][:1].expand(shape)
    y = arr(c["x"]).grouped_linear(arr(c["w"]), at, arr(c["bias"]), "silu", arr(c["res"]))
    check_forward(c, y.to_torch(), None, dtype, "silu", spans)
    for act in ("silu", "none"):
        out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at,
                                        arr(c["pre"]), act)
        check_backward(c, out, dtype, act, spans)


@gpu
def test_offsets_beyond_32_bits():
    """2.2e9 elements: the last rows, and the sums over all of them."""
    rows, inner, cols = 270001, 24, 8192
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, inner, generator=g, device="cuda").bfloat16()
    w = (torch.randn(inner, cols, generator=g, device="cuda") * 0.2).bfloat16()
    c = {"x": x, "w": w}
    y, pre = arr(x).linear(arr(w), None, "silu", save_pre=True)
    tail = slice(rows - 300, rows)
    check_forward(dict(c, x=x[tail]), y.to_torch()[tail], pre.to_torch()[tail], "bfloat16", "silu",
                  [(0, 300)], bias=False, res=False)
    grad, z = y.to_torch(), pre.to_torch()
    dx, dw, db = P.linear_backward(y, arr(x), arr(w), pre, "silu")
    k = dict(c, x=x[tail], grad=grad[tail], pre=z[tail])
    want = P.linear_backward(arr(k["grad"].contiguous()), arr(k["x"].contiguous()), arr(w),
                             arr(k["pre"].contiguous()), "silu")
    assert torch.equal(dx.to_torch()[tail], want[0].to_torch())
    sw, sb = torch.zeros(inner, cols, device="cuda").double(), torch.zeros(cols, device="cuda").double()
    for a in range(0, rows, 30000):
        dz = grad[a:a + 30000].double() * slope64(z[a:a + 30000].double(), "silu")
        sw += x[a:a + 30000].double().T @ dz
        sb += dz.sum(0)
    # as wholes: dz's and the result's rounding, 2^-8 each
    assert (dw.to_torch().double() - sw).norm() <= 2.0 ** -7 * sw.norm()
    assert (db.to_torch().double() - sb).norm() <= 1e-5 * sb.norm()


def _pt(shape, dtype):
    t = P.PtTensor()
    t.data, t.dtype, t.ndims = 4096, P.DTYPE_CODES[dtype], len(shape)
    for i, (d, s) in enumerate(zip(shape, P._contiguous_strides(shape))):
        t.shape[i], t.strides[i] = d, s
    return t


def test_refusals():
    """Arguments are refused before any CUDA call."""
    lib, ref = P.library(), ctypes.byref
    x, w, y = _pt([4, 8], "float16"), _pt([8, 16], "float16"), _pt([4, 16], "float16")
    size = ctypes.c_size_t(0)

    def forward(x=x, w=w, ends=None, bias=None, act=0, res=None, y=y, pre=None, work=None):
        return lib.pt_linear(ref(x), ref(w), ends, bias and ref(bias), act, res and ref(res),
                             ref(y), pre and ref(pre), work, ref(size), None)
    strided_y = _pt([4, 16], "float16")
    strided_y.strides[0] = 32
    for bad in (dict(x=_pt([4, 8], "float64")), dict(w=_pt([8, 16], "bfloat16")),
                dict(x=_pt([4, 9], "float16")), dict(y=_pt([5, 16], "float16")),
                dict(y=_pt([4, 15], "float16")), dict(y=strided_y), dict(act=7), dict(act=-1),
                dict(bias=_pt([15], "float16")), dict(bias=_pt([16], "bfloat16")),
                dict(res=_pt([4, 15], "float16")), dict(res=_pt([4, 16], "float32")),
                dict(pre=_pt([4, 16], "float32")), dict(ends=4096),
                dict(w=_pt([2, 8, 16], "float16")), dict(work=4097),
                dict(w=_pt([2049, 8, 16], "float16"), ends=4096),
                dict(w=_pt([0, 8, 16], "float16"), ends=4096),
                dict(x=_pt([8], "float16"), y=_pt([16], "float16"))):
        assert forward(**bad) == P.PT_INVALID_ARGUMENT, bad
        assert b"linear" in lib.pt_last_error() or b"workspace" in lib.pt_last_error()
    back = lib.pt_linear_backward
    assert back(ref(y), ref(x), ref(w), None, None, 4, ref(x), ref(w), None, None, ref(size),
                None) == P.PT_INVALID_ARGUMENT            # an activation without pre
    assert back(ref(y), ref(x), ref(w), None, None, 0, ref(x), ref(_pt([8, 16], "bfloat16")), None,
                None, ref(size), None) == P.PT_INVALID_ARGUMENT
    # float32 operands on the tensor cores need a place for their parts, and say
    # how large
    x, w, y = _pt([4, 8], "float32"), _pt([8, 16], "float32"), _pt([4, 16], "float32")
    before = P.set_kernel_path("tensor-core-pair")
    assert forward(x=x, w=w, y=y) == P.PT_WORKSPACE
    lib.gemm_sm100_set_path(before)
    assert size.value >= 3 * 2 * (4 * 8 + 8 * 16)
    with pytest.raises(P.InvalidArgumentException):
        P._activation_code("swish")


TAIL = [-9.5, -8.0, -7.25, -6.0, -5.0, -4.0, -3.5, -3.0, -1.0, -0.25, 0.25, 1.0, 3.0, 6.0, 9.0]


@gpu
@pytest.mark.parametrize("path", PATHS[1:], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
def test_gelu_keeps_its_digits_in_the_tail(dtype, path):
    """z P(z) relative to itself, through a product that is z exactly.  float16
    values below its spacing aside, what enters is the exponential and the
    argument's roundings, z^2 / 2 times a few e, the tail's fit (2^-17, 16-bit
    results) and the result's rounding."""
    z = torch.tensor(TAIL, device="cuda", dtype=DT[dtype])
    x = torch.zeros(len(TAIL), 64, device="cuda", dtype=DT[dtype])
    x[:, 3] = z
    w = torch.zeros(64, 72, device="cuda", dtype=DT[dtype])
    w[3] = 1
    y = arr(x).linear(arr(w), activation="gelu").to_torch().double()
    z = z.double()
    want = z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    tol = UNIT[dtype] + (2 * z * z + 16) * 2.0 ** -24 + (0 if dtype == "float32" else 2.0 ** -17)
    assert torch.all((y - want[:, None]).abs() <= (tol * want.abs() + TINY[dtype])[:, None])


def slope_of(act, z, dtype):
    """act'(z) in float32: dbias of one row whose upstream gradient is one."""
    n = z.numel()
    one = torch.ones(1, n, device="cuda", dtype=DT[dtype])
    x, w = (torch.zeros(s, device="cuda", dtype=DT[dtype]) for s in ((1, 8), (8, n)))
    return P.linear_backward(arr(one), arr(x), arr(w), arr(z[None]), act, inputs=False,
                             weights=False)[2].to_torch().double()


@gpu
@pytest.mark.parametrize("dtype", ALL)
def test_gelu_slope_keeps_its_digits_in_the_tail(dtype):
    """P(z) + z p(z), relative to its terms, of the same sources as above."""
    z = torch.tensor(TAIL, device="cuda", dtype=DT[dtype])
    v = z.double()
    p = torch.exp(-0.5 * v * v) * (0.5 / math.pi) ** 0.5
    cdf = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
    tol = (2 * v * v + 16) * 2.0 ** -24 + (0 if dtype == "float32" else 2.0 ** -17)
    assert torch.all((slope_of("gelu", z, dtype) - (cdf + v * p)).abs()
                     <= tol * (cdf + (v * p).abs()))


@gpu
@pytest.mark.parametrize("dtype", ALL)
def test_tanh_and_sigmoid_slopes_keep_their_digits_in_the_tail(dtype):
    """1 - tanh^2 and s (1 - s) relative to themselves: an exponential of at most
    2 |z|, within (2.4 |z| + 4) units of 2^-23 (16-bit operands), and a few
    roundings."""
    z = torch.tensor(TAIL, device="cuda", dtype=DT[dtype])
    v = z.double()
    tol = (5 * v.abs() + 32) * 2.0 ** -24
    for act, want in (("tanh", torch.cosh(v) ** -2), ("sigmoid", 0.25 * torch.cosh(0.5 * v) ** -2)):
        assert torch.all((slope_of(act, z, dtype) - want).abs() <= tol * want), act


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [64, 65])
def test_float32_weight_gradient_with_an_activation(dtype, rows):
    """On both sides of 16384 elements of dz: asking for dw in float32 changes
    dw's rounding alone, and a kernel path that is none of the linear layers'
    changes nothing."""
    ends = [20, 20, rows - 1]
    c = case(rows, 96, 256, dtype, 31, groups=3)
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")

    def back(path, dw=None):
        before = P.set_kernel_path(path)
        try:
            return P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at,
                                             arr(c["pre"]), "gelu", weight_grad_dtype=dw)
        finally:
            P.library().gemm_sm100_set_path(before)
    want = back("auto")
    check_backward(c, want, dtype, "gelu", spans_of(ends, rows))
    for path in ("auto", "skinny", "tensor-core-wide"):
        for dw in (None, "float32"):
            got = back(path, dw)
            for a, b in zip(want, got):
                assert torch.equal(a.to_torch(), b.to_torch().to(a.to_torch().dtype)), (path, dw)
            if dw:
                check_backward(c, got, dtype, "gelu", spans_of(ends, rows), dw_dtype="float32")
    # the CUDA-core path stays what was asked for
    got = back("simt", "float32")
    assert P.cuda_get_backend_info()["kernel"] == "ragged-simt-" + {"bfloat16": "bf16"}.get(
        dtype, "f16")
    check_backward(c, got, dtype, "gelu", spans_of(ends, rows), dw_dtype="float32")


def test_sizes_that_pass_32_bits_are_refused():
    """Column and inner counts stay 1024 below 2^31, as row counts do: loops and
    tiles may step past the end before they compare.  Refused before any CUDA
    call; no memory of these sizes is touched."""
    lib, ref = P.library(), ctypes.byref
    size = ctypes.c_size_t(0)
    big = 2 ** 31 - 1024
    for x, w, y in (([1, 8], [8, big], [1, big]), ([1, big], [big, 1], [1, 1])):
        x, w, y = (_pt(s, "bfloat16") for s in (x, w, y))
        assert lib.pt_linear(ref(x), ref(w), None, None, 0, None, ref(y), None, None, ref(size),
                             None) == P.PT_INVALID_ARGUMENT
        assert lib.pt_linear_backward(ref(y), ref(x), ref(w), None, None, 0, ref(x), ref(w), None,
                                      None, ref(size), None) == P.PT_INVALID_ARGUMENT
        assert b"2^31" in lib.pt_last_error()


@gpu
@pytest.mark.parametrize("path,block,clusters", [
    ("tensor-core", 192, (1, 2, 4, 8)), ("tensor-core-pair", 608, (2,)),
    ("simt", 256, (1, 2, 4, 8))], indirect=["path"])
def test_last_launch(path, block, clusters):
    """gemm_sm100_last_launch describes the product's launch, the bias
    gradient's or the norm's where the call has no product."""
    c = case(130, 512, 264, "bfloat16", 3)
    for call in (lambda: arr(c["x"]).linear(arr(c["w"])),
                 lambda: P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), weights=False)):
        call()
        grid, threads, cluster = P.last_launch()
        assert threads == block and cluster in clusters and grid > 0 and grid % cluster == 0
    P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), inputs=False, weights=False)
    grid, threads, cluster = P.last_launch()
    assert grid == 2 * 3 and threads == 256 and cluster == 1     # column strips x row tiles
    arr(c["x"]).layer_norm()
    grid, threads, cluster = P.last_launch()
    assert 0 < grid <= 130 and threads in (256, 512) and cluster == 1


def test_python_refusals():
    """What is missing or of another kind is refused as an argument, before
    torch or the device are asked for anything."""
    def host(*shape, dtype="float32"):
        return P.CudaArray(torch.zeros(math.prod(shape)), shape, dtype=dtype)
    x, w, y = host(4, 8), host(8, 16), host(4, 16)
    stats = host(4)
    for call in (lambda: x.linear(None), lambda: x.grouped_linear(None, None),
                 lambda: x.linear(w, bias=torch.zeros(16)),
                 lambda: P.linear_backward(None, x, w), lambda: P.linear_backward(y, None, w),
                 lambda: P.linear_backward(y, x, None),
                 lambda: P.linear_backward(y, x, w, weight_grad_dtype="int8"),
                 lambda: P.grouped_linear_backward(y, x, None, None),
                 lambda: P.grouped_linear_backward(None, x, w, None),
                 lambda: P.layer_norm_backward(None, x, None, stats, stats),
                 lambda: P.layer_norm_backward(x, None, None, stats, stats),
                 lambda: P.layer_norm_backward(x, x, None, None, stats),
                 lambda: P.layer_norm_backward(x, x, None, stats, None),
                 lambda: x.view([2, 8], [-8, 1], 8)._packed()):
        with pytest.raises(P.InvalidArgumentException):
            call()


@gpu
@pytest.mark.parametrize("path", ["auto", "tensor-core", "tensor-core-pair"], indirect=True)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,inner,cols,ends", [
    (300, 128, 320, [0, 70, 70, 71, 260]),          # chunked maps, three feature tiles of dx
    (3200, 256, 192, [1500, 1501, 3190]),           # a group's rows in parts for dw
    (40, 1024, 384, [3, 3, 20, 37])])               # few rows, the inner axis over a cluster
def test_grouped_widths_of_64(dtype, path, rows, inner, cols, ends):
    """Widths that are multiples of 64, as real experts have them: operands
    whose maps walk chunks of 64 beside the group's coordinate, as they lie
    and with the weight transposed."""
    at = torch.tensor(ends, dtype=torch.int32, device="cuda")
    spans = spans_of(ends, rows)
    for layout in ("plain", "column"):
        c = case(rows, inner, cols, dtype, 41, groups=len(ends))
        c["w"] = strided(c["w"], layout)
        for k in ("x", "grad", "pre", "res"):
            c[k][spans[-1][1]:] = float("nan")
        y, pre = arr(c["x"]).grouped_linear(arr(c["w"]), at, arr(c["bias"]), "silu",
                                            arr(c["res"]), save_pre=True)
        check_forward(c, y.to_torch(), pre.to_torch(), dtype, "silu", spans)
        for act in ("silu", "none"):
            out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at,
                                            arr(c["pre"]), act)
            check_backward(c, out, dtype, act, spans)


@gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("groups", [None, 3])
def test_more_tiles_than_pairs(dtype, groups):
    """Every pair takes several tiles of eight k-blocks and more, both
    accumulators in turn."""
    rows, inner, cols = 2100, 576, 4352
    ends = [rows] if groups is None else [700, 1405, 2099]
    spans = spans_of(ends, rows)
    c = case(rows, inner, cols, dtype, 43, groups=groups)
    before = P.set_kernel_path("tensor-core-pair")
    try:
        if groups is None:
            y = arr(c["x"]).linear(arr(c["w"]), arr(c["bias"]), "none", arr(c["res"]))
            out = P.linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]))
        else:
            at = torch.tensor(ends, dtype=torch.int32, device="cuda")
            y = arr(c["x"]).grouped_linear(arr(c["w"]), at, arr(c["bias"]), "none", arr(c["res"]))
            out = P.grouped_linear_backward(arr(c["grad"]), arr(c["x"]), arr(c["w"]), at)
    finally:
        P.library().gemm_sm100_set_path(before)
    check_forward(c, y.to_torch(), None, dtype, "none", spans)
    check_backward(c, out, dtype, "none", spans)


@gpu
@pytest.mark.parametrize("act", sorted(set(P.ACTIVATIONS) - {"none", "relu"}))
@pytest.mark.parametrize("dtype", ALL)
def test_slopes_are_float32(dtype, act):
    """dbias sums slopes in float32, so these are held to float32 whatever the
    operands' type: a few roundings and an exponential within (|x| + 4) 2^-23 come
    to some 2^-23 of their norm; a fit made for 16-bit results would be
    ten times that."""
    g = torch.Generator(device="cuda").manual_seed(51)
    z = torch.randn(1 << 16, generator=g, device="cuda").to(DT[dtype])
    want = slope64(z.double(), act)
    assert (slope_of(act, z, dtype) - want).norm() <= 2.0 ** -22.5 * want.norm()
