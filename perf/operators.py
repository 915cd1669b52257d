"""Timing cases of the operators that stand beside the attention Functions: the gated linear recurrence, layer norm
and layer norm behind the addition of a residual. A case is a plain dict:

  op      "recurrence"  GatedLinearRecurrence:  h_t = exp(g_t) h_(t-1) + x_t, with an fp32 state in and out
          "norm"        LayerNorm:              y = (x - mean) / sqrt(var + eps) * w + b over the last dim
          "add_norm"    AddLayerNorm:           s = x + z, y = LayerNorm(s); returns both
  mode    "train"       forward + backward; "forward": without gradients (prefill, decode, scoring)
  B, H, N, D            batch, heads, tokens, columns; tensors are [B, H, N, D], or [B, N, D] where H is 0
  dtype   "bf16" | "fp16" | "fp32": of the tensors
  param   "same" | "fp32": type of the log decays resp. of the weights
  layout  "bhnd": contiguous; "bnhd": the [B, H, N, D] view of a [B, N, H, D] projection
  heads   (norms) whether every head has weights of its own, [H, D]

Log decays: a rate for each channel, log-uniform from 1e-4 (a memory of ten thousand tokens) to 1, varied from token to
token, and -inf where a packed document starts. Inputs of the recurrence are scaled so that its state stays near one.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _recurrence(mode, B, H, N, D, dtype="bf16", param="same", layout="bhnd", name=None):
    case = {"op": "recurrence", "mode": mode, "B": B, "H": H, "N": N, "D": D, "dtype": dtype, "param": param, "layout": layout}
    return case if name is None else dict(case, name=name)


def _norm(op, mode, B, H, N, D, dtype="bf16", param="same", layout="bhnd", heads=False, name=None):
    case = {"op": op, "mode": mode, "B": B, "H": H, "N": N, "D": D, "dtype": dtype, "param": param, "layout": layout,
            "heads": heads}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one decode step of a served batch: 8 sequences x 32 heads, one token each; launch and host time
        _recurrence("forward", 8, 32, 1, 128, name="recurrence_1_token"),
        # chunked prefill: the next 1000 tokens of two sequences in fp16, straight from a projection, no multiple of a tile
        _recurrence("forward", 2, 32, 1000, 128, dtype="fp16", layout="bnhd", name="recurrence_prefill_1000"),
        # an odd head dim and length (the acceptance tests' largest), in 32 bits
        _recurrence("train", 3, 24, 1984, 83, dtype="fp32", name="recurrence_odd_fp32"),
        # ordinary training layer of the headline benchmark's size: the largest case
        _recurrence("train", 4, 32, 8192, 128, name="recurrence_train"),
        # long context, few channels, decays kept in 32 bits: the scan over tokens is what counts
        _recurrence("train", 1, 8, 65536, 128, param="fp32", name="recurrence_long"),
        # layer norm of one decode step over model rows of 32 x 128 columns, added to the residual
        _norm("add_norm", "forward", 8, 0, 1, 4096, name="add_norm_1_token"),
        # pre-norm of a training layer with its residual, weights kept in 32 bits
        _norm("add_norm", "train", 4, 0, 8192, 4096, param="fp32", name="add_norm_train"),
        # norm of the unnormalised attention output head by head, weights of each head's own, in the projection's layout
        _norm("norm", "train", 4, 32, 8192, 128, layout="bnhd", heads=True, name="norm_heads_train"),
        # narrow heads, scoring
        _norm("norm", "forward", 8, 16, 4096, 64, dtype="fp16", name="norm_d64_forward"),
        # rows that are no multiple of 16 bytes, in 32 bits
        _norm("norm", "train", 3, 24, 1984, 83, dtype="fp32", name="norm_odd_fp32"),
        # an ordinary small training step over model rows
        _norm("norm", "train", 2, 0, 256, 1024, name="norm_small_train"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        mode = rng.choice(["train", "train", "forward"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        param = rng.choice(["same", "same", "fp32"])
        layout = rng.choice(["bhnd", "bhnd", "bnhd"])
        B, N = _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 65536)
        if rng.random() < 0.5:
            H = rng.choice([1, 2, 4, 8, 16, 24, 32, rng.randint(1, 32)])
            D = rng.choice([32, 64, 128, 256, rng.randint(8, 300)])
            case = _recurrence(mode, B, H, N, D, dtype, param, layout)
        else:
            op = rng.choice(["norm", "norm", "add_norm"])
            if rng.random() < 0.5:  # heads
                H = rng.choice([1, 2, 4, 8, 16, 24, 32, rng.randint(1, 32)])
                D, heads = rng.choice([32, 64, 128, 256, rng.randint(8, 300)]), rng.random() < 0.5
            else:  # model rows
                H, heads, layout = 0, False, "bhnd"
                D = rng.choice([512, 1024, 2048, 4096, 8192, _log_uniform(rng, 128, 16384)])
            case = _norm(op, mode, B, H, N, D, dtype, param, layout, heads)
        if 2e4 < work(case)["bytes"] < 0.6 * most:
            return case


def _shape(case):
    B, H, N, D = (case[x] for x in ("B", "H", "N", "D"))
    return (B, H, N, D) if H else (B, N, D)


def _layout(case, t):
    return t.transpose(1, 2).contiguous().transpose(1, 2) if case["layout"] == "bnhd" else t


def _inputs(case, seed):
    """Every tensor of the case, with the values and types that the call gets."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape, dtype = _shape(case), DTYPES[case["dtype"]]
    param = torch.float32 if case["param"] == "fp32" else dtype
    train = case["mode"] == "train"

    def randn(*sizes):
        return torch.randn(*sizes, device="cuda", generator=gen)

    t = {}
    if case["op"] == "recurrence":
        B, H, N, D = shape
        rate = torch.exp(torch.rand(H, 1, D, device="cuda", generator=gen) * math.log(1e4) - math.log(1e4))
        g = -rate * torch.exp(0.5 * randn(*shape))
        x = randn(*shape) * torch.sqrt(-torch.expm1(2 * g))
        g.masked_fill_(torch.rand(B, 1, N, 1, device="cuda", generator=gen) < 1 / 2048, -math.inf)
        t["x"], t["g"] = _layout(case, x.to(dtype)), _layout(case, g.to(param))
        t["s"] = randn(B, H, D)
        if train:
            t["dy"], t["ds"] = _layout(case, randn(*shape).to(dtype)), randn(B, H, D)
        return t
    # rows with a mean of their own and columns of unlike size, as in a residual stream
    scale = torch.exp(0.5 * randn(shape[-1]))
    t["x"] = _layout(case, (randn(*shape) * scale + 0.5 * randn(*shape[:-1], 1)).to(dtype))
    weights = (case["H"], case["D"]) if case["heads"] else (case["D"],)
    t["w"], t["b"] = (1 + 0.2 * randn(*weights)).to(param), (0.2 * randn(*weights)).to(param)
    if case["op"] == "add_norm":
        t["z"] = _layout(case, (randn(*shape) * scale).to(dtype))
    if train:
        t["dy"] = _layout(case, randn(*shape).to(dtype))
        if case["op"] == "add_norm":
            t["ds"] = _layout(case, randn(*shape).to(dtype))
    return t


def prepare(case, seed):
    state = dict(_inputs(case, seed), op=case["op"], train=case["mode"] == "train")
    if state["train"]:
        for name in ("x", "g", "s", "z", "w", "b"):
            if name in state:
                state[name].requires_grad_(True)
    return state


def _scan(decay, x):
    """h_t = decay_t h_(t-1) + x_t over dim 2, starting from zero: pairs of neighbours, then of pairs, and so on (the
    composition of two steps is a step), log2(N) passes over the tensors. A scan has no other form in elementary
    operations that neither overflows nor takes a pass a token."""
    decay, x, span = decay.clone(), x.clone(), 1
    while span < x.shape[2]:
        x[:, :, span:] += decay[:, :, span:] * x[:, :, :-span]
        decay[:, :, span:] *= decay[:, :, :-span].clone()
        span *= 2
    return x


def _plain_recurrence(s):
    # in 64 bits: a decay of exp(-1e-4), rounded to 32, is off by 3e-8 every token, over ten thousand tokens
    x, g, s0 = s["x"].detach().double(), s["g"].detach().double(), s["s"].detach().double()
    a = g.exp()
    first = x.clone()
    first[:, :, 0] += a[:, :, 0] * s0
    h = _scan(a, first)
    out, s_final = h.to(s["x"].dtype), h[:, :, -1].float()
    if not s["train"]:
        return out, s_final
    # R_t = exp(g_t) G_t with G_t = dy_t + R_(t+1): the same scan from the end, whose decay is that of the token behind
    dy = s["dy"].double()
    dy[:, :, -1] += s["ds"].double()
    behind = torch.cat([a[:, :, 1:], torch.zeros_like(a[:, :, :1])], dim=2)
    G = _scan(behind.flip(2), dy.flip(2)).flip(2)
    R = a * G
    before = torch.cat([s0.unsqueeze(2), h[:, :, :-1]], dim=2)
    return out, s_final, G.to(out.dtype), (R * before).to(s["g"].dtype), R[:, :, 0].float()


def _plain_norm(s):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    total = None
    if s["op"] == "add_norm":
        total = (x.float() + s["z"].detach().float()).to(x.dtype)
        x = total
    wide = (w.float(), b.float()) if w.dim() == 1 else (w.float().unsqueeze(1), b.float().unsqueeze(1))
    c = x.float()
    c = c - c.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * r
    y = (n * wide[0] + wide[1]).to(x.dtype)
    outs = (y,) if total is None else (y, total)
    if not s["train"]:
        return outs
    dy = s["dy"].float()
    u = dy * wide[0]
    dx = r * (u - u.mean(-1, keepdim=True) - n * (u * n).mean(-1, keepdim=True))
    rows = tuple(d for d in range(x.dim() - 1) if w.dim() == 1 or d != 1)
    dw, db = (dy * n).sum(rows).to(w.dtype), dy.sum(rows).to(w.dtype)
    if total is None:
        return outs + (dx.to(x.dtype), dw, db)
    dx = (dx + s["ds"].float()).to(x.dtype)
    return outs + (dx, dx.clone(), dw, db)


def _own(s):
    from flashy_linear_attention_b200 import AddLayerNorm, GatedLinearRecurrence, LayerNorm

    if s["op"] == "recurrence":
        call, inputs = (lambda: GatedLinearRecurrence.apply(s["x"], s["g"], s["s"])), ("x", "g", "s")
    elif s["op"] == "norm":
        call, inputs = (lambda: (LayerNorm.apply(s["x"], s["w"], s["b"], EPS),)), ("x", "w", "b")
    else:
        call, inputs = (lambda: AddLayerNorm.apply(s["x"], s["z"], s["w"], s["b"], EPS)), ("x", "z", "w", "b")
    if not s["train"]:
        with torch.no_grad():
            return call()
    outs = call()
    grads = [s["dy"], s["ds"]] if len(outs) == 2 else [s["dy"]]
    return tuple(outs) + torch.autograd.grad(outs, [s[name] for name in inputs], grads)


def run(state):
    if own:
        return _own(state)
    return _plain_recurrence(state) if state["op"] == "recurrence" else _plain_norm(state)


def work(case):
    """Each input once and each output once; forward and backward are two calls, and what they read fits no cache."""
    elements = math.prod(_shape(case))
    size, train = 4 if case["dtype"] == "fp32" else 2, case["mode"] == "train"
    param = 4 if case["param"] == "fp32" else size
    if case["op"] == "recurrence":
        state = 4 * case["B"] * case["H"] * case["D"]
        per, flops = 2 * size + param, 3
        if train:
            per, flops = per + 3 * size + 2 * param, flops + 8
        return {"bytes": per * elements + (5 if train else 2) * state, "flops": flops * elements}
    weights = param * case["D"] * (max(case["H"], 1) if case["heads"] else 1)
    more = case["op"] == "add_norm"
    per, flops = 2 + 2 * more, 8 + more
    if train:
        per, flops = per + 3 + more, flops + 14 + more
    return {"bytes": per * size * elements + (5 if train else 2) * weights, "flops": flops * elements}


def exact(case, seed):
    """The definitions in 64 bits: the recurrence token by token, the norm with its gradient written out from the
    derivative of each step."""
    t = {name: x.double() for name, x in _inputs(case, seed).items()}
    train = case["mode"] == "train"
    if case["op"] == "recurrence":
        a, state, N = torch.exp(t["g"]), t["s"], case["N"]
        h = torch.empty_like(t["x"])
        for i in range(N):
            state = torch.addcmul(t["x"][:, :, i], a[:, :, i], state)
            h[:, :, i] = state
        if not train:
            return h, state
        dx, dg, back = torch.empty_like(h), torch.empty_like(h), t["ds"]
        for i in reversed(range(N)):
            back = back + t["dy"][:, :, i]
            dx[:, :, i] = back
            back = back * a[:, :, i]
            dg[:, :, i] = back * (h[:, :, i - 1] if i else t["s"])
        return h, state, dx, dg, back
    D, x = case["D"], t["x"]
    per_head = t["w"].dim() == 2
    w, b = (p[:, None, :] if per_head else p for p in (t["w"], t["b"]))
    if case["op"] == "add_norm":
        # what is normalised is the sum as it is stored
        x = (x + t["z"]).to(DTYPES[case["dtype"]]).double()
    mean = x.sum(-1, keepdim=True) / D
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / D
    root = torch.sqrt(var + EPS)
    y = (x - mean) / root * w + b
    sums = (x,) if case["op"] == "add_norm" else ()
    if not train:
        return (y,) + sums
    dy = t["dy"]
    dn = dy * w
    droot = -(dn * (x - mean)).sum(-1, keepdim=True) / root**2
    dc = dn / root + droot / root * (x - mean) / D
    dx = dc - dc.sum(-1, keepdim=True) / D
    axes = [0, 2] if per_head else list(range(x.dim() - 1))
    dw, db = (dy * (x - mean) / root).sum(axes), dy.sum(axes)
    if case["op"] == "add_norm":
        dx = dx + t["ds"]
        return (y,) + sums + (dx, dx, dw, db)
    return (y,) + sums + (dx, dw, db)
