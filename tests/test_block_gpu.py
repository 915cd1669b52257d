"""The operators around an attention as a block uses them, and their native autograd nodes.

A block of heads: s1, n = AddLayerNorm(branch, residual); q, k, v from n; y = LinearAttention(q, k, v) normalised head by head
by LayerNorm; GatedLinearRecurrence over y; its output is the branch of the next AddLayerNorm. In 16 bits each of the seven
operators rounds its result once, by 2^-9 of it on average over a tensor (bf16); norms pass relative errors on unchanged, the
recurrence and the attention average over tokens. Seven such errors, unlike one another, and as many backward: sqrt(14) 2^-9 =
7.3e-3 of a tensor's norm. Bound: 2e-2, the bound of the attention alone in its tests.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
B, H, D = 2, 3, 64
C = H * D


def functions():
    import flashy_linear_attention_b200 as fla

    return fla


def heads(t):  # [B, N, C] -> the [B, H, N, D] view of a projection
    return t.unflatten(-1, (H, D)).transpose(1, 2)


def weights(seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    ws = {name: randn(C, C) / C**0.5 for name in ("q", "k", "v", "g")}
    ws.update(n1=1 + 0.1 * randn(C), b1=0.1 * randn(C), nh=1 + 0.1 * randn(H, D), bh=0.1 * randn(H, D), n2=1 + 0.1 * randn(C), b2=0.1 * randn(C))
    return ws


def phi(t):
    return torch.nn.functional.elu(t) + 1


def block(w, branch, residual, states=None):
    """out, sum and the states behind the tokens, through the library's Functions."""
    fla = functions()
    n, s1 = fla.AddLayerNorm.apply(branch, residual, w["n1"], w["b1"])
    q, k, v, g = (heads(n @ w[name]) for name in ("q", "k", "v", "g"))
    y, kv = fla.LinearAttentionResumable.apply(phi(q) / D, phi(k), v, None if states is None else states[0])
    y = fla.LayerNorm.apply(y, w["nh"], w["bh"])
    h, state = fla.GatedLinearRecurrence.apply(y, -torch.nn.functional.softplus(g.float()), None if states is None else states[1])
    out, s2 = fla.AddLayerNorm.apply(h.transpose(1, 2).flatten(-2), s1, w["n2"], w["b2"])
    return out, s2, (kv, state)


def plain(w, branch, residual):
    """The same in 64 bits, from elementary operations."""
    w = {name: t.double() for name, t in w.items()}

    def norm(x, a, b):
        c = x - x.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * a + b

    s1 = branch + residual
    n = norm(s1, w["n1"], w["b1"])
    q, k, v, g = (heads(n @ w[name]) for name in ("q", "k", "v", "g"))
    y = ((phi(q) / D) @ phi(k).transpose(-1, -2)).tril() @ v
    y = norm(y, w["nh"].unsqueeze(1), w["bh"].unsqueeze(1))
    a, h, outs = torch.exp(-torch.nn.functional.softplus(g)), 0.0, []
    for t in range(y.shape[2]):
        h = a[:, :, t] * h + y[:, :, t]
        outs.append(h)
    s2 = torch.stack(outs, 2).transpose(1, 2).flatten(-2) + s1
    return norm(s2, w["n2"], w["b2"]), s2


def inputs(N, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(B, N, C, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(4)]


def test_a_block_and_its_gradients():
    branch, residual, d_out, d_sum = inputs(192)
    w16 = {name: t.to(torch.bfloat16) for name, t in weights().items()}
    names = list(w16)
    got_leaves = [t.detach().requires_grad_(True) for t in (branch, residual, *w16.values())]
    out, s2, _ = block(dict(zip(names, got_leaves[2:])), *got_leaves[:2])
    got = (out.detach(), s2.detach(), *torch.autograd.grad((out, s2), got_leaves, (d_out, d_sum)))
    leaves = [t.detach().double().requires_grad_(True) for t in (branch, residual, *w16.values())]
    out, s2 = plain(dict(zip(names, leaves[2:])), *leaves[:2])
    want = (out.detach(), s2.detach(), *torch.autograd.grad((out, s2), leaves, (d_out.double(), d_sum.double())))
    for name, a, b in zip(["out", "sum", "branch", "residual", *names], got, want):
        assert a.dtype == torch.bfloat16
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off < 2e-2, f"{name}: {off:.3e}"


def test_prefill_and_single_tokens_give_what_one_call_gives():
    branch, residual, _, _ = inputs(60)
    w = {name: t.to(torch.bfloat16) for name, t in weights().items()}
    with torch.no_grad():
        want, want_sum, want_states = block(w, branch, residual)
        outs, states = [], None
        for at, n in ((0, 40), *((i, 1) for i in range(40, 60))):
            out, s2, states = block(w, branch[:, at:at + n], residual[:, at:at + n], states)
            outs.append(out)
    got = torch.cat(outs, 1)
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() < 2e-2
    for a, b in zip(states, want_states):
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() < 2e-2


def test_a_step_of_a_block_in_a_graph_beside_eager_ones():
    """Captured forward and backward, replayed with other inputs, and eager steps over the same leaves before, between and
    behind the replays. (Not while an eager graph of the same leaves lives on the default stream: autograd then makes that stream
    wait for the captured one, which CUDA refuses whatever the operators are.)"""
    from flashy_linear_attention_b200 import graphs

    w = {name: t.to(torch.bfloat16) for name, t in weights().items()}
    tensors = inputs(70)
    leaves = [t.requires_grad_(True) for t in (*tensors[:2], *w.values())]
    names = list(w)

    def step():
        out, s2, _ = block(dict(zip(names, leaves[2:])), *leaves[:2])
        return (out.detach(), s2.detach(), *torch.autograd.grad((out, s2), leaves, tensors[2:]))

    step()
    captured = graphs.capture_step(step)
    for seed in (3, 4):
        with torch.no_grad():
            for t, new in zip(tensors, inputs(70, seed)):
                t.copy_(new)
        want = step()
        got = captured()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def calls():
    """(name, call of leaves, leaves, number of outputs)"""
    fla = functions()
    gen = torch.Generator(device=DEV).manual_seed(5)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    x, z, g = randn(2, 3, 50, 64), randn(2, 3, 50, 64), -torch.rand(2, 3, 50, 64, device=DEV, generator=gen)
    s, w, b = randn(2, 3, 64), randn(64), randn(64)
    return [
        ("recurrence", lambda *t: fla.GatedLinearRecurrence.apply(*t), (x, g, s)),
        ("norm", lambda *t: (fla.LayerNorm.apply(*t),), (x, w, b)),
        ("add_norm", lambda *t: fla.AddLayerNorm.apply(*t), (x, z, w, b)),
    ]


def test_native_nodes_and_python_functions_do_the_same(monkeypatch):
    from flashy_linear_attention_b200 import _lib

    for name, call, inputs_ in calls():
        results = []
        for native in (True, False):
            if not native:
                monkeypatch.setattr(_lib, "host", lambda: None)
            leaves = [t.detach().clone().requires_grad_(True) for t in inputs_]
            outs = call(*leaves)
            assert ("Node" in type(outs[0].grad_fn).__name__ or "Node" in outs[0].grad_fn.name()) == native, (name, outs[0].grad_fn)
            total = sum((o * (i + 1)).sum() for i, o in enumerate(outs))
            total.backward(retain_graph=True)
            first = [t.grad.clone() for t in leaves]
            total.backward()  # again: gradients add up
            assert all(torch.equal(t.grad, 2 * f) for t, f in zip(leaves, first)), name
            results.append([o.detach() for o in outs] + first)
            with pytest.raises(RuntimeError):
                total.backward()  # the graph is gone
            # an input changed in place between the passes
            leaves = [t.detach().clone().requires_grad_(True) for t in inputs_]
            middle = leaves[0] * 1.0
            outs = call(middle, *leaves[1:])
            if name != "add_norm":  # (which keeps the sum instead)
                middle.data.add_(0)
                with torch.no_grad():
                    middle.add_(1.0)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    outs[0].sum().backward()
            # gradients of gradients are refused, not wrong
            leaves = [t.detach().clone().requires_grad_(True) for t in inputs_]
            grads = torch.autograd.grad(call(*leaves)[0].square().sum(), leaves, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                grads[0].sum().backward()
            # nothing wanted, nothing kept
            with torch.no_grad():
                assert all(o.grad_fn is None and not o.requires_grad for o in call(*leaves))
            assert all(not o.requires_grad for o in call(*inputs_))
        monkeypatch.undo()
        assert all(torch.equal(a, b) for a, b in zip(*results)), name


def test_gradients_of_any_layout_and_threads():
    """Upstream gradients that are broadcast or transposed, and two backward passes at once from two threads."""
    import threading

    for name, call, inputs_ in calls():
        leaves = [t.detach().requires_grad_(True) for t in inputs_]
        outs = call(*leaves)
        ups = [torch.randn(o.shape[:-2] + (o.shape[-1], o.shape[-2]), device=DEV).transpose(-1, -2) for o in outs]
        got = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
        want = torch.autograd.grad(outs, leaves, [u.contiguous() for u in ups], retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        one = [torch.ones((), device=DEV).expand(o.shape) for o in outs]
        got = torch.autograd.grad(outs, leaves, one, retain_graph=True)
        want = torch.autograd.grad(outs, leaves, [u.contiguous() for u in one], retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        found, errors = [None, None], []

        def work(i):
            try:
                with torch.cuda.stream(torch.cuda.Stream()):
                    mine = [t.detach().requires_grad_(True) for t in inputs_]
                    for _ in range(20):
                        found[i] = torch.autograd.grad(call(*mine), mine, [u.contiguous() for u in one])
                    torch.cuda.current_stream().synchronize()
            except Exception as e:  # noqa: BLE001
                errors.append(e)

        torch.cuda.synchronize()
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
        for res in found:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), name
