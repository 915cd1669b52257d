"""Gated linear recurrence without a GPU: refusals of the Function and of the C interface, sizes, struct layout."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header():
    from flashy_linear_attention_b200._lib import FlaRecurrenceArgs

    header = open(os.path.join(ROOT, "include", "flashlinear_sm100.h")).read()
    body = header[header.index("typedef struct FlaRecurrenceArgs {") + len("typedef struct FlaRecurrenceArgs {"):header.index("} FlaRecurrenceArgs;")]
    names = [n.split()[-1] for stmt in body.replace("*", " ").split(";") if stmt.strip() for n in stmt.split(",")]
    assert names == [f[0] for f in FlaRecurrenceArgs._fields_]


def test_no_cpu_fallback():
    from flashy_linear_attention_b200 import GatedLinearRecurrence

    x = torch.zeros(1, 1, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        GatedLinearRecurrence.apply(x, x)


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks come before anything is launched."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def test_types_and_shapes_are_checked():
    from flashy_linear_attention_b200 import recurrence as rec

    x = fake(2, 3, 5, 8)
    rec.check_inputs(x, fake(2, 3, 5, 8), fake(2, 3, 8))
    rec.check_inputs(fake(2, 3, 5, 8, dtype=torch.bfloat16), x)
    with pytest.raises(TypeError):
        rec.check_inputs(fake(2, 3, 5, 8, dtype=torch.float64), x)
    with pytest.raises(TypeError):
        rec.check_inputs(x, fake(2, 3, 5, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        rec.check_inputs(fake(2, 3, 5, 8, dtype=torch.bfloat16), fake(2, 3, 5, 8, dtype=torch.float16))
    with pytest.raises(TypeError):
        rec.check_inputs(x, x, fake(2, 3, 8, dtype=torch.int32))
    with pytest.raises(ValueError):
        rec.check_inputs(fake(2, 5, 8), fake(2, 5, 8))
    with pytest.raises(ValueError):
        rec.check_inputs(x, fake(2, 3, 1, 8))
    with pytest.raises(ValueError):
        rec.check_inputs(x, x, fake(2, 3, 1, 8))


def test_c_interface_refuses():
    from flashy_linear_attention_b200 import _lib
    from flashy_linear_attention_b200._lib import FlaRecurrenceArgs, FlaTensor

    lib = _lib.load()
    fwd, bwd, size = lib.fla_sm100_recurrence_fwd, lib.fla_sm100_recurrence_bwd, lib.fla_sm100_recurrence_states_bytes
    assert fwd(None) == -1 and bwd(None) == -1 and size(None) == 0

    def args(**more):
        a = FlaRecurrenceArgs()
        a.batch, a.heads, a.seqlen, a.dim = 2, 3, 40, 8
        a.x = a.g = a.o = a.d_o = a.d_x = a.d_g = FlaTensor(64, 960, 320, 8)
        a.states, a.states_bytes = 64, 1 << 20
        for k, v in more.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for k in ("batch", "heads", "seqlen", "dim"):
        assert fwd(args(**{k: 0})) == -1 and fwd(args(**{k: -1})) == -1 and size(args(**{k: 0})) == 0
    none, odd = FlaTensor(None, 0, 0, 0), FlaTensor(65, 0, 0, 0)
    assert fwd(args(x=none)) == -1 and fwd(args(g=none)) == -1 and fwd(args(o=none)) == -1
    assert bwd(args(d_x=none, d_g=none)) == -1
    assert fwd(args(dtype=3)) == -1 and fwd(args(g_dtype=1)) == -1 and fwd(args(dtype=2, g_dtype=0)) == -1
    assert fwd(args(x=odd)) == -3 and bwd(args(d_g=odd)) == -3 and fwd(args(s_init=66)) == -3 and fwd(args(states=68)) == -3
    assert fwd(args(seqlen=(1 << 30) + 1)) == -2 and fwd(args(batch=1 << 20, heads=1 << 20)) == -2
    assert fwd(args(dim=(1 << 30) + 1)) == -2 and bwd(args(dim=2**31 - 1, states_bytes=1 << 40)) == -2
    # the state before every 16 tokens, 8 where a row or the gates are fp32
    assert size(args()) == 4 * 2 * 3 * 8 * 3 and size(args(g_dtype=2)) == 4 * 2 * 3 * 8 * 5
    assert fwd(args(states_bytes=575)) == -5 and bwd(args(states_bytes=575)) == -5 and bwd(args(states=None)) == -5
    if not torch.cuda.is_available():
        assert fwd(args()) in (-4, -6) and bwd(args()) in (-4, -6)
