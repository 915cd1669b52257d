"""Gated linear recurrence on the GPU against the recurrence token by token in 64 bits.

Tolerances. A result is the exact one but for (1) one rounding to the type of the tensor, at most half a step,
finfo.eps / 2 of the value, and (2) the errors of the 32-bit sums, which are relative to the same sums with absolute values
(`scale` below). Within a run of 16 tokens a decay is off by 2^-22 for the fast exponential and 2^-24 for its product,
so a run's sum by 16 * 1.3 * 2^-22 < 2^-17; joining a run to what came before costs 3 roundings of 2^-24, over at most
2048 / 8 = 256 runs 2^-14.4 if they all pointed the same way. Hence 2^-14 of `scale` for states and gradients of x, and
twice that for the gradient of the decay, a product of two such sums.
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
SUMS = 2.0**-14


def recurrence():
    from flashy_linear_attention_b200 import GatedLinearRecurrence

    return GatedLinearRecurrence


def reference(x, g, s, dy=None, ds=None):
    """out, s_final and, with dy, (dx, dg, ds_init), all in 64 bits, and the scales that their sums are relative to."""
    x, g = x.double(), g.double()
    B, H, N, D = x.shape
    zero = torch.zeros(B, H, D, dtype=torch.float64, device=x.device)
    s = zero if s is None else s.double()
    h, size = s, s.abs()
    out, out_size, before, before_size = [], [], [], []
    for t in range(N):
        drop = g[:, :, t] == -math.inf
        a = g[:, :, t].exp()
        before.append(h)
        before_size.append(size)
        h = torch.where(drop, x[:, :, t], a * h + x[:, :, t])
        size = torch.where(drop, x[:, :, t].abs(), a * size + x[:, :, t].abs())
        out.append(h)
        out_size.append(size)
    res = {"out": (torch.stack(out, 2), torch.stack(out_size, 2)), "s_final": (h, size)}
    if dy is None:
        return res
    back = zero if ds is None else ds.double()
    back_size = back.abs()
    dx, dx_size, dg, dg_size = ([None] * N for _ in range(4))
    for t in reversed(range(N)):
        drop = g[:, :, t] == -math.inf
        a = g[:, :, t].exp()
        back, back_size = back + dy[:, :, t].double(), back_size + dy[:, :, t].double().abs()
        dx[t], dx_size[t] = back, back_size
        back, back_size = torch.where(drop, zero, a * back), torch.where(drop, zero, a * back_size)
        dg[t] = torch.where(drop, zero, back * before[t])
        dg_size[t] = torch.where(drop, zero, 2 * back_size * before_size[t])
    res["dx"] = (torch.stack(dx, 2), torch.stack(dx_size, 2))
    res["dg"] = (torch.stack(dg, 2), torch.stack(dg_size, 2))
    res["ds"] = (back, back_size)
    return res


def check(name, got, want):
    value, scale = want
    # (below its smallest normal number a type has steps of a fixed size)
    bound = torch.finfo(got.dtype).eps / 2 * (value.abs() + torch.finfo(got.dtype).tiny) + SUMS * scale
    over = (got.double() - value).abs() - bound
    assert torch.isfinite(got).all(), name
    assert (over <= 0).all(), f"{name}: {over.max().item():.3e} over the bound, largest value {value.abs().max().item():.3e}"


def make(B, H, N, D, dtype=torch.bfloat16, gate=None, layout="bhnd", seed=0, reset=0.02, rate=(1e-3, 2.0)):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    lo, hi = (math.log(r) for r in rate)
    r = torch.exp(torch.rand(H, 1, D, device=DEV, generator=gen) * (hi - lo) + lo)
    g = -r * torch.exp(0.5 * randn(B, H, N, D))
    g.masked_fill_(torch.rand(B, H, N, 1, device=DEV, generator=gen) < reset, -math.inf)

    def lay(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "bnhd" else t

    x, dy = lay(randn(B, H, N, D).to(dtype)), lay(randn(B, H, N, D).to(dtype))
    return x, lay(g.to(gate or dtype)), randn(B, H, D), dy, randn(B, H, D)


def run(x, g, s, dy, ds):
    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    out, s_final = recurrence().apply(*leaves)
    grads = torch.autograd.grad((out, s_final), leaves, (dy, ds))
    return dict(zip(("out", "s_final", "dx", "dg", "ds"), (out.detach(), s_final.detach(), *grads)))


def verify(x, g, s, dy, ds):
    got, want = run(x, g, s, dy, ds), reference(x, g, s, dy, ds)
    for name in got:
        assert got[name].dtype == {"out": x, "dx": x, "dg": g}.get(name, s).dtype
        check(name, got[name], want[name])
    return got


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 700, 1025, 2048])
def test_lengths(N):
    verify(*make(2, 3, N, 64, seed=N))


@pytest.mark.parametrize("N", [1, 20, 40, 300, 1030])
@pytest.mark.parametrize("types", [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)], ids=str)
def test_types(types, N):
    verify(*make(1, 2, N, 128, *types, seed=N))


@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("D", [1, 2, 3, 8, 16, 30, 31, 32, 33, 34, 63, 64, 65, 83, 128, 130, 273])
def test_widths(D, layout):
    for N, dtype in ((5, BF), (150, BF), (150, FP)):
        verify(*make(2, 3, N, D, dtype, layout=layout, seed=D))


@pytest.mark.parametrize("heads", [1, 2, 5, 40, 200])
def test_few_and_many_tiles(heads):
    """From clusters of eight CTAs to one CTA a tile; long enough for several steps of each."""
    verify(*make(2, heads, 1500, 64, seed=heads))


def test_no_state_before():
    x, g, _, dy, _ = make(2, 2, 200, 64)
    out, s_final = recurrence().apply(x, g)
    want = reference(x, g, None)
    check("out", out, want["out"])
    check("s_final", s_final, want["s_final"])


@pytest.mark.parametrize("N", [24, 500])
def test_extreme_gates(N):
    """No decay at all, decays that underflow, growth, and every token a reset."""
    x, g, s, dy, ds = make(1, 2, N, 64, FP, reset=0.0)
    for value in (0.0, -1e4, -60.0, 0.01, -math.inf):
        verify(x, torch.full_like(g, value), s, dy, ds)


@pytest.mark.parametrize("N", [20, 400])
@pytest.mark.parametrize("poison", [math.inf, -math.inf, math.nan])
def test_nothing_passes_a_reset(poison, N):
    """What a document holds, infinities and NaN included, reaches neither the next one nor, backward, the one before."""
    for at in (1, 5, N // 2, N - 1):
        x, g, s, dy, ds = make(1, 2, N, 64, reset=0.0, seed=at)
        g[:, :, at] = -math.inf
        clean = run(x, g, s, dy, ds)
        bad = x.clone()
        bad[:, :, at - 1] = poison
        got = run(bad, g, s, dy, ds)
        assert torch.equal(got["out"][:, :, at:], clean["out"][:, :, at:])
        assert torch.equal(got["s_final"], clean["s_final"])
        for name in ("dx", "dg"):
            assert torch.equal(got[name][:, :, at:], clean[name][:, :, at:]), name
        bad = dy.clone()
        bad[:, :, at] = poison
        got = run(x, g, s, bad, ds)
        for name in ("dx", "dg"):
            assert torch.equal(got[name][:, :, :at], clean[name][:, :, :at]), name
        assert torch.equal(got["ds"], clean["ds"])
        got = run(x, g, torch.full_like(s, poison), dy, ds)
        assert torch.equal(got["out"][:, :, at:], clean["out"][:, :, at:])


def test_a_wait_that_runs_out():
    """A peer whose sums never come: the wait ends at its limit, bit 0 of the status is set, what hangs on it is NaN,
    and the next call is right again. (The limit is that of the call; nothing is left waiting.)"""
    import ctypes

    from flashy_linear_attention_b200 import _lib, ops, recurrence as rec

    x, g, s, _, _ = make(1, 1, 5000, 64)
    ops.check_status(x.device)
    out, s_final = torch.zeros_like(x), torch.zeros(1, 1, 64, device=DEV)
    a = rec._args(x, g)
    a.o, a.s_init, a.s_final = rec._desc(out), s.data_ptr(), s_final.data_ptr()
    a.status, a.stream = ops._status_word(x.device).data_ptr(), torch.cuda.current_stream().cuda_stream
    a.wait_limit_us, a.debug_flags = 20000, _lib.FLA_DEBUG_WITHHOLD_FIRST_TILE
    assert _lib.load().fla_sm100_recurrence_fwd(ctypes.byref(a)) == 0
    with pytest.raises(RuntimeError, match="status 1"):
        ops.check_status(x.device)
    assert out.isnan().any() and s_final.isnan().all()
    got = recurrence().apply(x, g, s)
    ops.check_status(x.device)
    check("out", got[0], reference(x, g, s)["out"])


@pytest.mark.parametrize("N", [20, 700])
def test_an_infinity_stays_until_it_is_dropped(N):
    x, g, s, _, _ = make(1, 1, N, 64, reset=0.0, rate=(1e-3, 8.0))
    x[:, :, 3] = math.inf
    out, s_final = recurrence().apply(x, g, s)
    assert torch.isfinite(out[:, :, :3]).all() and (out[:, :, 3:] == math.inf).all() and (s_final == math.inf).all()


def test_tokens_passed_over():
    """x = 0 with a decay of 0 (padding) leaves the state alone to the bit, and its gradient passes through."""
    x, g, s, dy, ds = make(2, 2, 100, 64)
    short = run(x, g, s, dy, ds)
    pad = lambda t: torch.cat([t, torch.zeros_like(t[:, :, :60])], 2)  # noqa: E731
    long = run(pad(x), pad(g), s, pad(dy), ds)
    assert torch.equal(long["s_final"], short["s_final"])
    assert torch.equal(long["out"][:, :, :100], short["out"])
    for name in ("dx", "dg"):
        check(name, long[name][:, :, :100], reference(x, g, s, dy, ds)[name])


@pytest.mark.parametrize("cuts", [(1,) * 12, (1, 31, 33, 2, 200), (128, 128, 44), (0, 17, 0, 90)])
def test_pieces_of_a_sequence(cuts):
    """States handed on from call to call, and gradients back through them, as one call over all tokens."""
    N = sum(cuts)
    x, g, s, dy, ds = make(2, 2, N, 64, FP, seed=N)
    want = reference(x, g, s, dy, ds)
    leaves = [t.requires_grad_(True) for t in (x, g, s)]
    state, outs, at = s, [], 0
    for n in cuts:
        out, state = recurrence().apply(x[:, :, at:at + n], g[:, :, at:at + n], state)
        outs.append(out)
        at += n
    out = torch.cat(outs, 2)
    grads = torch.autograd.grad((out, state), leaves, (dy, ds))
    for name, got in zip(("out", "s_final", "dx", "dg", "ds"), (out.detach(), state.detach(), *grads)):
        check(name, got, want[name])


def test_long_memory_in_32_bits():
    """A decay of exp(-1e-4), rounded to 32 bits, is off by 3e-8 a token; over ten thousand tokens that is 3e-4. Held
    as two floats a run, what is left are roundings without a direction: 2^-24 each, about 20 of them add up to one
    part in 2^20 over the 1250 runs of the memory. Bound: four times that."""
    N = 16384
    for rate in (1.03e-4, 0.97e-4, 2.9e-5):
        x, g = torch.ones(1, 1, N, 8, device=DEV), torch.full((1, 1, N, 8), -rate, device=DEV)
        out, _ = recurrence().apply(x, g)
        a = math.exp(g[0, 0, 0, 0].item())
        t = torch.arange(1, N + 1, device=DEV, dtype=torch.float64)
        want = (1 - a**t) / (1 - a)
        assert ((out[0, 0, :, 3].double() - want).abs() / want).max() < 2.0**-18


def test_gradients_against_differences():
    """Central differences of the fp32 call. Loss sum(w out) + sum(v s_final), 33 tokens: rounding noise of the loss
    2^-24 * 33 * 5 / (2 * 0.01), and the third derivative's share h^2 / 6 times a value of a few: 2e-3."""
    x, g, s, dy, ds = make(1, 1, 33, 4, FP, reset=0.0, rate=(0.1, 1.0))
    got = run(x, g, s, dy, ds)

    def loss(*t):
        out, s_final = recurrence().apply(*t)
        return ((out.double() * dy.double()).sum() + (s_final.double() * ds.double()).sum()).item()

    step = 0.01
    for i, name in enumerate(("dx", "dg", "ds")):
        flat = got[name].reshape(-1)
        for at in range(0, flat.numel(), 7):
            hi, lo = ([t.clone() for t in (x, g, s)] for _ in range(2))
            hi[i].view(-1)[at] += step
            lo[i].view(-1)[at] -= step
            moved = hi[i].view(-1)[at].item() - lo[i].view(-1)[at].item()
            assert abs((loss(*hi) - loss(*lo)) / moved - flat[at].item()) < 2e-3 * max(1.0, abs(flat[at].item())), name


@pytest.mark.parametrize("N", [1, 20, 300])
def test_strides(N):
    """Rows cut out of wider ones, a transposed innermost dim, odd storage offsets, and gates that heads, tokens or
    channels share, with their gradients summed."""
    x, g, s, dy, ds = make(2, 3, N, 64, seed=3)
    want = reference(x, g, s, dy, ds)
    wide = torch.randn(2, N, 3, 3 * 64 + 1, device=DEV).to(BF)
    for offset in (0, 1, 2):
        view = wide[..., offset:offset + 64].transpose(1, 2)
        view.copy_(x)
        other = wide[..., 128 - offset:192 - offset].transpose(1, 2)
        other.copy_(g)
        got = run(view, other, s, dy, ds)
        for name in got:
            check(name, got[name], want[name])
    turned = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
    got = run(turned(x), turned(g), turned(s.unsqueeze(0)).squeeze(0), turned(dy), ds.flip(0).flip(0))
    for name in got:
        check(name, got[name], want[name])
    for shape in ((1, 3, 1, 64), (2, 3, N, 1), (1, 1, N, 64), (1, 1, 1, 1)):
        shared = (-torch.rand(shape, device=DEV)).to(BF).requires_grad_(True)
        full = shared.detach().expand(2, 3, N, 64)
        out, s_final = recurrence().apply(x, shared.expand(2, 3, N, 64), s)
        (got_g,) = torch.autograd.grad((out, s_final), shared, (dy, ds))
        ref = reference(x, full, s, dy, ds)
        check("out", out.detach(), ref["out"])
        dims = [d for d in range(4) if shape[d] == 1]
        # every summand has been rounded to bf16, and the sum once more (in 32 bits: its roundings are below SUMS)
        value, scale = ref["dg"]
        bound = 2.0**-8 * value.abs().sum(dims, True) * 2 + 2 * SUMS * scale.sum(dims, True)
        assert ((got_g.double() - value.sum(dims, True)).abs() <= bound).all()
    # a broadcast gradient (that of a sum) and none at all
    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    recurrence().apply(*leaves)[0].sum().backward()
    ref = reference(x, g, s, torch.ones_like(dy), None)
    for name, leaf in zip(("dx", "dg", "ds"), leaves):
        check(name, leaf.grad, ref[name])


def test_some_gradients_only():
    x, g, s, dy, ds = make(2, 2, 130, 64)
    full = run(x, g, s, dy, ds)
    for wanted in itertools.product((False, True), repeat=3):
        if not any(wanted):
            continue
        leaves = [t.detach().requires_grad_(w) for t, w in zip((x, g, s), wanted)]
        out, s_final = recurrence().apply(*leaves)
        grads = torch.autograd.grad((out, s_final), [t for t in leaves if t.requires_grad], (dy, ds))
        for name, got in zip([n for n, w in zip(("dx", "dg", "ds"), wanted) if w], grads):
            assert torch.equal(got, full[name]), name
    # a gradient of the state alone
    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    got = torch.autograd.grad(recurrence().apply(*leaves)[1], leaves, ds)
    want = reference(x, g, s, torch.zeros_like(dy), ds)
    for name, t in zip(("dx", "dg", "ds"), got):
        check(name, t, want[name])
    # without a state, and called with two arguments
    leaves = [t.detach().requires_grad_(True) for t in (x, g)]
    got = torch.autograd.grad(recurrence().apply(*leaves)[0], leaves, dy)
    want = reference(x, g, None, dy, None)
    check("dx", got[0], want["dx"])
    check("dg", got[1], want["dg"])


@pytest.mark.parametrize("shape", [(2, 3, 0, 64), (0, 3, 5, 64), (2, 0, 5, 64), (2, 3, 5, 0)])
def test_nothing_to_do(shape):
    B, H, N, D = shape
    x = torch.randn(shape, device=DEV).requires_grad_(True)
    g, s = (-torch.rand(shape, device=DEV)).requires_grad_(True), torch.randn(B, H, D, device=DEV).requires_grad_(True)
    out, s_final = recurrence().apply(x, g, s)
    assert out.shape == x.shape and torch.equal(s_final, s)
    grads = torch.autograd.grad((out, s_final), (x, g, s), (torch.ones_like(out), torch.full_like(s, 2.0)))
    assert grads[0].shape == x.shape and grads[1].shape == x.shape and torch.equal(grads[2], torch.full_like(s, 2.0))
    assert (recurrence().apply(x, g)[1] == 0).all()


def test_far_offsets():
    """Rows more than 2^31 elements apart."""
    buf = torch.empty(2**31 + 2**30 + 64, dtype=BF, device=DEV)
    x, g, s, _, _ = make(1, 1, 4, 64)
    far = buf.as_strided((1, 1, 4, 64), (0, 0, 2**30, 1))
    far.copy_(x)
    out, s_final = recurrence().apply(far, g, s)
    want = reference(x, g, s)
    check("out", out, want["out"])
    check("s_final", s_final, want["s_final"])


@pytest.mark.parametrize("N,apart", [(40, 2**26), (8192, 2**18)])
def test_offsets_past_32_bits(N, apart):
    """Rows that are read and written 2^26 elements apart (a step's offsets pass 32 bits) and 2^18 (those of the sequence do)."""
    far = [torch.empty(N * apart, dtype=BF, device=DEV).as_strided((1, 1, N, 64), (0, 0, apart, 1)) for _ in range(2)]
    x, g, s, dy, ds = make(1, 1, N, 64)
    far[0].copy_(x)
    far[1].copy_(dy)
    want = run(x, g, s, dy, ds)
    got = run(far[0], g, s, far[1], ds)
    ref = reference(x[:, :, :40], g[:, :, :40], s)
    check("out", got["out"][:, :, :40], ref["out"])
    for name in got:  # (the same sums in another order where the step is another)
        off, size = (got[name].double() - want[name].double()).norm(), want[name].double().norm()  # (zero behind a reset)
        assert off <= (torch.finfo(got[name].dtype).eps + 1e-5) * size, name


@pytest.mark.parametrize("N", [5, 700])
def test_negative_strides(N):
    """Tokens from the last to the first, which the C interface can be given."""
    from flashy_linear_attention_b200 import recurrence as rec

    x, g, s, _, _ = make(2, 3, N, 64)
    out, s_final = torch.empty_like(x), torch.empty_like(s)
    a = rec._args(x, g)
    a.o = rec._desc(out)
    for t, of in ((a.x, x), (a.g, g), (a.o, out)):
        t.ptr += (N - 1) * of.stride(2) * of.element_size()
        t.stride_n = -of.stride(2)
    a.s_init, a.s_final = s.data_ptr(), s_final.data_ptr()
    rec._call("fla_sm100_recurrence_fwd", a, x.device)
    want = reference(x.flip(2), g.flip(2), s)
    check("out", out.flip(2), want["out"])
    check("s_final", s_final, want["s_final"])


def test_the_same_bits_every_time():
    for shape in ((1, 2, 2000, 64), (4, 40, 300, 64), (2, 3, 500, 83)):
        t = make(*shape)
        first = run(*t)
        for _ in range(20):
            again = run(*t)
            assert all(torch.equal(first[n], again[n]) for n in first)


def test_streams_graphs_and_the_path_without_the_extension(monkeypatch):
    from flashy_linear_attention_b200 import _lib, graphs

    for shape in ((2, 2, 1, 64), (1, 3, 700, 64)):
        t = make(*shape)
        want = run(*t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run(*t)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(got[n], want[n]) for n in want)
        # two graphs over the same inputs, replayed in turn with other values
        leaves = [a.clone() for a in t]
        steps = [graphs.capture_step(lambda: run(*leaves)) for _ in range(2)]
        for seed in range(3):
            for a, b in zip(leaves, make(*shape, seed=seed)):
                a.copy_(b)
            want_now = run(*leaves)
            both = [{n: v.clone() for n, v in step().items()} for step in steps]
            for got in both:
                assert all(torch.equal(got[n], want_now[n]) for n in want_now)
        monkeypatch.setattr(_lib, "host", lambda: None)
        got = run(*t)
        monkeypatch.undo()
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_autocast():
    x, g, s, dy, ds = make(1, 2, 50, 64, FP)
    with torch.autocast("cuda", dtype=BF):
        out, s_final = recurrence().apply(x, g, s)
    want = recurrence().apply(x.to(BF), g, s)
    assert out.dtype == BF and s_final.dtype == FP
    assert torch.equal(out, want[0]) and torch.equal(s_final, want[1])
    leaf = x.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=BF):
        out, _ = recurrence().apply(leaf, g.to(HF), s)
    out.backward(dy.to(BF))
    assert leaf.grad.dtype == FP


def test_rows_around_the_outputs_stay_as_they_are():
    """The kernels called on rows inside guard bands: nothing outside [0, N) x [0, D) is written."""
    import ctypes

    from flashy_linear_attention_b200 import _lib, recurrence as rec

    lib = _lib.load()
    for N, D in ((1, 33), (3, 64), (45, 83), (130, 64), (300, 31)):
        x, g, s, dy, ds = make(1, 2, N, D, FP)
        guard = lambda: torch.full((1, 2, N + 4, D + 6), 7.0, device=DEV)  # noqa: E731
        bands = [guard() for _ in range(3)]
        views = [b[:, :, 2:-2, 3:-3] for b in bands]
        a = rec._args(x, g)
        state = torch.full((2 * 2 * D + 2,), 7.0, device=DEV)
        a.o, a.s_init, a.s_final = rec._desc(views[0]), s.data_ptr(), state[1:].data_ptr()
        a.states_bytes = lib.fla_sm100_recurrence_states_bytes(ctypes.byref(a))
        states = torch.full((a.states_bytes // 4 + 64,), 7.0, device=DEV)
        a.states = states.data_ptr()
        rec._call("fla_sm100_recurrence_fwd", a, x.device)
        assert (states[a.states_bytes // 4:] == 7).all()
        a.d_o, a.d_x, a.d_g = rec._desc(dy), rec._desc(views[1]), rec._desc(views[2])
        a.r_init, a.r_final = ds.data_ptr(), state[1 + 2 * D:].data_ptr()
        rec._call("fla_sm100_recurrence_bwd", a, x.device)
        want = reference(x, g, s, dy, ds)
        got = [v.clone() for v in views]
        for name, t in zip(("out", "dx", "dg"), got):
            check(name, t, want[name])
        check("s_final", state[1:1 + 2 * D].view(1, 2, D), want["s_final"])
        check("ds", state[1 + 2 * D:1 + 4 * D].view(1, 2, D), want["ds"])
        assert state[0] == 7 and state[-1] == 7
        for b, v in zip(bands, views):
            v.fill_(7.0)
            assert (b == 7).all()
