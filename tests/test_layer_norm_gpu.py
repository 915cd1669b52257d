"""Layer norm, with and without a residual added first, on the GPU against its definition in 64 bits.

Tolerances. One rounding to the type of the result, half a step: finfo.eps / 2 of the value. The rest are errors of 32-bit
sums over a row, of at most 64 terms one after the other and 10 levels of pairs: below 2^-17 of the sum of the absolute
values. The mean's error moves every difference to it, so what n = (x - mean) r is off by is relative to
N = |n| + r (|mean| + mean|x|) ("size" below), and what is formed from n inherits that. 2^-15 of such sizes leaves room for
the three or four factors that meet in a gradient.
"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
SUMS = 2.0**-15
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def functions():
    from flashy_linear_attention_b200 import AddLayerNorm, LayerNorm

    return LayerNorm, AddLayerNorm


def reference(x, w, b, eps, dy=None, ds=None):
    """{name: (value, size)} in 64 bits for the rows `x` that are normalised; w, b [D], [H, D] or None."""
    shape = lambda t: None if t is None else (t.double() if t.dim() == 1 else t.double().unsqueeze(1))  # noqa: E731
    x, W, B = x.double(), shape(w), shape(b)
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    n = (x - mean) * r
    N = n.abs() + r * (mean.abs() + x.abs().mean(-1, keepdim=True))
    y, y_size = n, N
    if W is not None:
        y, y_size = y * W, y_size * W.abs()
    if B is not None:
        y, y_size = y + B, y_size + B.abs()
    res = {"y": (y, y_size)}
    if dy is None:
        return res
    dy = dy.double()
    u = dy if W is None else dy * W
    m = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dx = r * (u - m(u) - n * m(u * n))
    size = r * (u.abs() + m(u.abs()) + N * m(u.abs() * N))
    if ds is not None:
        dx, size = dx + ds.double(), size + ds.double().abs()
    res["dx"] = (dx, size)
    per_head = any(t is not None and t.dim() == 2 for t in (w, b))
    rows = [d for d in range(x.dim() - 1) if not (per_head and d == 1)]
    over = lambda t: t.sum(rows) if rows else t  # noqa: E731  (a sum over no dimensions is one over all)
    res["dw"] = (over(dy * n), over(dy.abs() * N))
    res["db"] = (over(dy), over(dy.abs()))
    return res


def check(name, got, want):
    value, size = want
    bound = torch.finfo(got.dtype).eps / 2 * (value.abs() + torch.finfo(got.dtype).tiny) + SUMS * size
    assert got.shape == value.shape, name
    assert torch.isfinite(got).all(), name
    over = (got.double() - value).abs() - bound
    assert (over <= 0).all(), f"{name}: {over.max().item():.3e} over the bound, largest value {value.abs().max().item():.3e}"


def make(shape, dtype=BF, param=None, heads=False, layout="bhnd", seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    lay = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "bnhd" else t  # noqa: E731
    x = lay((randn(*shape) * 2 + randn(*shape[:-1], 1)).to(dtype))
    z, dy, ds = (lay(randn(*shape).to(dtype)) for _ in range(3))
    ws = (shape[1], shape[-1]) if heads else (shape[-1],)
    w, b = ((1 + 0.3 * randn(*ws)).to(param or dtype), randn(*ws).to(param or dtype))
    return x, z, w, b, dy, ds


def run(x, z, w, b, dy, ds, eps=1e-5):
    """Outputs and gradients of LayerNorm (z None) or AddLayerNorm."""
    LayerNorm, AddLayerNorm = functions()
    leaves = {n: t.detach().requires_grad_(True) for n, t in (("dx", x), ("dz", z), ("dw", w), ("db", b)) if t is not None}
    x, z, w, b = (leaves.get(n) for n in ("dx", "dz", "dw", "db"))
    if z is None:
        outs, grads = (LayerNorm.apply(x, w, b, eps),), (dy,)
    else:
        outs, grads = AddLayerNorm.apply(x, z, w, b, eps), (dy, ds)
    res = dict(zip(("y", "sum"), (o.detach() for o in outs)))
    res.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    return res


def verify(x, z, w, b, dy, ds, eps=1e-5):
    got = run(x, z, w, b, dy, ds, eps)
    rows = x if z is None else (x.float() + z.float()).to(x.dtype)
    want = reference(rows, w, b, eps, dy, None if z is None else ds)
    if z is not None:
        assert torch.equal(got["sum"], rows)
        assert torch.equal(got["dx"], got["dz"])
    for name, value in want.items():
        if name in got:
            assert got[name].dtype == (w if name == "dw" else b if name == "db" else x).dtype
            check(name, got[name], value)
    return got


WIDTHS = [1, 2, 3, 7, 8, 9, 16, 24, 31, 32, 33, 63, 64, 65, 83, 100, 127, 128, 129, 130, 255, 256, 257, 264, 273, 500, 511,
          512, 513, 520, 1000, 1016, 1024, 1025, 1032, 2048, 4096, 4097, 4104, 5120, 8192, 8193, 8200, 16384, 16390, 32760, 32768]


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(D, dtype):
    x, z, w, b, dy, ds = make((2, 11, D), dtype, seed=D)
    verify(x, None, w, b, dy, None)
    verify(x, z, w.float(), b.float(), dy, ds)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 32, 33, 255, 1000, 5003])
@pytest.mark.parametrize("D", [64, 83, 128, 1024, 2048])
def test_rows(rows, D):
    x, z, w, b, dy, ds = make((rows, D), seed=rows)
    verify(x, None, w, b, dy, None)
    verify(x, z, w, b, dy, ds)


def test_many_narrow_rows():
    verify(*make((300_001, 8), FP)[:1], None, *make((300_001, 8), FP)[2:5], None)


@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("shape", [(2, 5, 70, 64), (1, 3, 1, 128), (3, 1, 40, 83), (2, 7, 33, 256), (4, 32, 9, 16), (1, 2, 600, 1024), (2, 3, 5, 2056)])
def test_heads(shape, layout):
    for heads in (False, True):
        for dtype, param in ((BF, BF), (HF, FP), (FP, FP)):
            x, z, w, b, dy, ds = make(shape, dtype, param, heads, layout, seed=shape[2])
            verify(x, None, w, b, dy, None)
            verify(x, z, w, b, dy, ds)


def test_layouts_that_differ_between_tensors():
    x, z, w, b, dy, ds = make((3, 4, 50, 64), heads=True)
    turn = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    want = run(x, z, w, b, dy, ds)
    for which in itertools.product((False, True), repeat=4):
        args = [turn(t) if f else t for t, f in zip((x, z, dy, ds), which)]
        got = run(args[0], args[1], w, b, args[2], args[3])
        assert all(torch.equal(got[n], want[n]) for n in ("y", "sum", "dx"))
        for n in ("dw", "db"):
            check(n, got[n], reference(want["sum"], w, b, 1e-5, dy, ds)[n])


def test_ranks_and_strides():
    LayerNorm, _ = functions()
    for shape in ((40,), (3, 40), (2, 3, 40), (2, 3, 4, 40), (2, 2, 3, 4, 40), (1, 2, 1, 2, 3, 40)):
        x, z, w, b, dy, ds = make((1, *shape), seed=len(shape))
        verify(x[0], None, w, b, dy[0], None)
        verify(x[0], z[0], w, b, dy[0], ds[0])
    base = torch.randn(3, 20, 5, 200, device=DEV).to(BF)
    _, _, w, b, dy, _ = make((3, 5, 20, 64))
    for offset in (0, 1, 2, 4, 8):
        verify(base[..., offset:offset + 64].transpose(1, 2), None, w, b, dy, None)
    verify(base.transpose(1, 3)[:, :64].transpose(1, 3).transpose(1, 2), None, w, b, dy, None)
    # columns that are not neighbours, rows that are one row, a gradient that is one number
    turned = torch.randn(5, 64, 33, device=DEV).to(BF).transpose(1, 2)
    _, _, w, b, dy, _ = make((5, 33, 64))
    verify(turned, None, w, b, dy.transpose(0, 1).contiguous().transpose(0, 1), None)
    verify(torch.randn(1, 1, 64, device=DEV).to(BF).expand(5, 33, 64), None, w, b, dy, None)
    leaf = turned.detach().requires_grad_(True)
    LayerNorm.apply(leaf, w, b).sum().backward()
    check("dx", leaf.grad, reference(turned, w, b, 1e-5, torch.ones_like(turned))["dx"])
    # weights that begin inside a 16-byte piece
    wide = torch.randn(2, 65, device=DEV).to(BF)
    verify(turned, None, wide[0, 1:], wide[1, 1:].contiguous(), dy, None)


@pytest.mark.parametrize("shape,order", [((3, 5, 70, 64), (0, 2, 1, 3)), ((3, 5, 70, 64), (2, 1, 0, 3)), ((3, 5, 70, 64), (1, 2, 0, 3)),
                                         ((2, 1, 33, 83), (2, 0, 1, 3)), ((3, 40, 128), (1, 0, 2)), ((2, 3, 4, 5, 32), (1, 3, 2, 0, 4))])
@pytest.mark.parametrize("add", [False, True])
def test_kept_tensors_that_come_back_with_other_strides(shape, order, add):
    """What autograd keeps can be packed away and unpacked contiguous; rows in memory order `order` (from outside in)."""
    x, z, w, b, dy, ds = make(shape)
    back = [order.index(i) for i in range(len(order))]
    x, z = (t.permute(order).contiguous().permute(back) for t in (x, z))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.contiguous()):
        verify(x, z if add else None, w, b, dy, ds)
    verify(x, z if add else None, w, b, dy, ds)


@pytest.mark.parametrize("shape,heads", [((2, 9, 96), False), ((2, 3, 9, 96), True), ((4, 2048), False)])
def test_without_weights_and_some_gradients_only(shape, heads):
    LayerNorm, AddLayerNorm = functions()
    x, z, w, b, dy, ds = make(shape, heads=heads)
    for weight, bias in ((None, None), (w, None), (None, b)):
        verify(x, None, weight, bias, dy, None)
        verify(x, z, weight, bias, dy, ds)
    full = run(x, z, w, b, dy, ds)
    for wanted in itertools.product((False, True), repeat=4):
        if not any(wanted):
            continue
        leaves = [t.detach().requires_grad_(f) for t, f in zip((x, z, w, b), wanted)]
        grads = torch.autograd.grad(AddLayerNorm.apply(*leaves)[0], [t for t in leaves if t.requires_grad], dy)
        want = reference(full["sum"], w, b, 1e-5, dy)
        for name, got in zip([n for n, f in zip(("dx", "dx", "dw", "db"), wanted) if f], grads):
            check(name, got, want[name])
    # the sum alone
    leaves = [t.detach().requires_grad_(True) for t in (x, z)]
    got = torch.autograd.grad(AddLayerNorm.apply(*leaves, w, b)[1], leaves, ds)
    assert all(torch.equal(t, ds) for t in got)
    # the same tensor twice
    leaf = x.detach().requires_grad_(True)
    (got,) = torch.autograd.grad(AddLayerNorm.apply(leaf, leaf, w, b)[0], leaf, dy)
    value, size = reference((x.float() + x.float()).to(x.dtype), w, b, 1e-5, dy)["dx"]
    check("dx twice", got, (2 * value, 2 * size + 2.0**-8 / SUMS * value.abs()))
    assert LayerNorm.apply(x).requires_grad is False


def test_eps_and_rows_without_variance():
    for D in (1, 40, 64, 2048):
        x, _, w, b, dy, _ = make((7, D), FP)
        x = x[:, :1].expand(7, D).contiguous()
        for eps in (1e-5, 1e-2, 3.0):
            got = run(x, None, w, b, dy, None, eps)
            # every difference to the mean is a rounding of it, 2^-20 of the value at most
            off = (2.0**-20 * x.abs().max() / eps**0.5).item()
            assert ((got["y"] - b).abs() <= off * w.abs() + 1e-6).all()
        verify(make((7, D), FP)[0], None, w, b, dy, None, eps=1e-3)
    # large means: differences first, then squares
    x, _, w, b, dy, _ = make((9, 512), FP, seed=5)
    verify(x + 100.0, None, w, b, dy, None)


@pytest.mark.parametrize("D", [64, 83, 1024, 4096])
def test_a_bad_row_stays_alone(D):
    """Infinities and NaN in a row spoil that row of the result and of the gradient, and no other."""
    x, z, w, b, dy, ds = make((30, D))
    clean = run(x, z, w, b, dy, ds)
    for bad in (float("inf"), float("-inf"), float("nan")):
        spoiled = x.clone()
        spoiled[4, D // 2] = bad
        got = run(spoiled, z, w, b, dy, ds)
        for name in ("y", "dx"):
            others = [i for i in range(30) if i != 4]
            assert torch.equal(got[name][others], clean[name][others])
            assert got[name][4].isnan().any()
        assert torch.equal(got["db"], clean["db"])


def test_gradients_against_differences():
    """Central differences of the fp32 call. Loss sum(w y): rounding noise 2^-24 * 24 * 3 / (2 * 0.01), and the third
    derivative's share h^2 / 6 times a value of a few: 2e-3."""
    LayerNorm, _ = functions()
    x, _, w, b, dy, _ = make((2, 12), FP)
    got = run(x, None, w, b, dy, None)
    step = 0.01
    for i, name in enumerate(("dx", "dw", "db")):
        for at in range(got[name].numel()):
            hi, lo = ([t.clone() for t in (x, w, b)] for _ in range(2))
            hi[i].view(-1)[at] += step
            lo[i].view(-1)[at] -= step
            moved = hi[i].view(-1)[at].item() - lo[i].view(-1)[at].item()
            rise = sum(s * (LayerNorm.apply(*t).double() * dy.double()).sum().item() for s, t in ((1, hi), (-1, lo)))
            assert abs(rise / moved - got[name].view(-1)[at].item()) < 2e-3 * max(1.0, abs(got[name].view(-1)[at].item())), name


@pytest.mark.parametrize("shape", [(0, 8), (3, 0), (2, 0, 5, 8), (0,)])
def test_nothing_to_do(shape):
    LayerNorm, AddLayerNorm = functions()
    x = torch.randn(shape, device=DEV).requires_grad_(True)
    w = torch.ones(shape[-1], device=DEV).requires_grad_(True)
    b = torch.zeros(shape[-1], device=DEV).requires_grad_(True)
    y = LayerNorm.apply(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == x.shape == dx.shape and (dw == 0).all() and (db == 0).all() and dw.shape == w.shape
    y, s = AddLayerNorm.apply(x, x, w, b)
    assert y.shape == s.shape == x.shape


def test_far_offsets():
    """Rows more than 2^31 elements apart, read and written."""
    LayerNorm, _ = functions()
    buf = torch.zeros(2**31 + 2**30 + 64, dtype=BF, device=DEV)
    x, _, w, b, dy, _ = make((4, 64))
    far = buf.as_strided((4, 64), (2**30, 1))
    far.copy_(x)
    verify(far, None, w, b, dy, None)
    far.copy_(dy)
    verify(x, None, w, b, far, None)


def test_the_same_bits_every_time():
    for shape, heads in (((3000, 64), False), ((2, 8, 300, 128), True), ((700, 4096), False), ((900, 83), False)):
        t = make(shape, heads=heads)
        first = run(*t)
        for _ in range(20):
            again = run(*t)
            assert all(torch.equal(first[n], again[n]) for n in first)


def test_streams_graphs_and_the_path_without_the_extension(monkeypatch):
    from flashy_linear_attention_b200 import _lib, graphs

    for shape, heads in (((8, 1, 4096), False), ((2, 3, 200, 64), True), ((500, 83), False), ((5, 96), False)):
        t = make(shape, heads=heads)
        want = run(*t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run(*t)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(got[n], want[n]) for n in want)
        leaves = [a.clone() for a in t]
        steps = [graphs.capture_step(lambda: run(*leaves)) for _ in range(2)]
        for seed in range(3):
            for a, b in zip(leaves, make(shape, heads=heads, seed=seed)):
                a.copy_(b)
            want_now = run(*leaves)
            both = [{n: v.clone() for n, v in step().items()} for step in steps]
            for got in both:
                assert all(torch.equal(got[n], want_now[n]) for n in want_now)
        monkeypatch.setattr(_lib, "host", lambda: None)
        got = run(*t)
        monkeypatch.undo()
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_autocast_leaves_types_alone():
    LayerNorm, _ = functions()
    x, _, w, b, dy, _ = make((5, 64), FP)
    with torch.autocast("cuda", dtype=BF):
        y = LayerNorm.apply(x, w, b)
    assert y.dtype == FP and torch.equal(y, LayerNorm.apply(x, w, b))


def test_rows_around_the_outputs_stay_as_they_are():
    import ctypes

    from flashy_linear_attention_b200 import _lib, layer_norm as ln

    lib = _lib.load()
    for rows, D, dtype in ((1, 33, FP), (3, 64, BF), (45, 83, HF), (130, 1024, BF), (9, 2048, BF), (5, 8199, FP)):
        x, z, w, b, dy, ds = make((rows, D), dtype)
        x, z, dy, ds = (ln._rows(t) for t in (x, z, dy, ds))
        pad = 16 // x.element_size()
        bands = [torch.full((1, 1, rows + 4, D + 2 * pad), 7.0, dtype=dtype, device=DEV) for _ in range(3)]
        y, total, dx = (t[:, :, 2:-2, pad:-pad] for t in bands)
        flat = torch.full((4, D + 16), 7.0, dtype=dtype, device=DEV)
        stats = torch.full((2 * rows + 8,), 7.0, device=DEV)
        a = ln._args(x, w, b, 1e-5)
        a.residual, a.sum, a.y, a.stats = ln._desc(z), ln._desc(total), ln._desc(y), stats[2:].data_ptr()
        ln._call("fla_sm100_layer_norm_fwd", a, x.device)
        want = reference(total, w, b, 1e-5, dy, ds)
        check("y", y, want["y"])
        a.x, a.d_y, a.d_sum, a.d_x = ln._desc(total), ln._desc(dy), ln._desc(ds), ln._desc(dx)
        a.d_weight, a.d_bias = flat[1, 8:].data_ptr(), flat[2, 8:].data_ptr()
        need = lib.fla_sm100_layer_norm_workspace_bytes(ctypes.byref(a))
        ws = torch.full((need // 4 + 64,), 7.0, device=DEV)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        ln._call("fla_sm100_layer_norm_bwd", a, x.device)
        check("dx", dx, want["dx"])
        check("dw", flat[1, 8:8 + D], want["dw"])
        check("db", flat[2, 8:8 + D], want["db"])
        assert (ws[need // 4:] == 7).all() and (stats[:2] == 7).all() and (stats[2 + 2 * rows:] == 7).all()
        for band, view in zip(bands, (y, total, dx)):
            view.fill_(7.0)
            assert (band == 7).all()
        flat[1:3, 8:8 + D] = 7.0
        assert (flat == 7).all()
