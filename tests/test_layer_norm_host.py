"""Layer norm without a GPU: refusals of the Functions and of the C interface, sizes, struct layout."""
import ctypes
import os

import pytest
import torch

from test_recurrence_host import fake

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header():
    from flashy_linear_attention_b200._lib import FlaLayerNormArgs

    header = open(os.path.join(ROOT, "include", "flashlinear_sm100.h")).read()
    start = "typedef struct FlaLayerNormArgs {"
    body = header[header.index(start) + len(start):header.index("} FlaLayerNormArgs;")]
    names = [n.split()[-1] for stmt in body.replace("*", " ").split(";") if stmt.strip() for n in stmt.split(",")]
    assert names == [f[0] for f in FlaLayerNormArgs._fields_]


def test_no_cpu_fallback():
    from flashy_linear_attention_b200 import AddLayerNorm, LayerNorm

    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        LayerNorm.apply(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        AddLayerNorm.apply(x, x)


def test_types_and_shapes_are_checked():
    from flashy_linear_attention_b200.layer_norm import check_inputs

    x, w, b = fake(2, 3, 5, 8), fake(8), fake(8)
    half = torch.bfloat16
    check_inputs(x, w, b, 1e-5)
    check_inputs(x, fake(3, 8), fake(3, 8), 0.0, fake(2, 3, 5, 8))
    check_inputs(fake(5, 8, dtype=half), w, b, 1e-5)
    check_inputs(x, None, None, 1e-5)
    for bad in (fake(7), fake(1), fake(5, 8), fake(2, 8), fake(3, 1, 8), fake(1, 8)):
        with pytest.raises(ValueError):
            check_inputs(x, bad, None, 1e-5)
    with pytest.raises(ValueError):
        check_inputs(fake(5, 3, 8), fake(3, 8), None, 1e-5)  # heads only where there is a dimension of them
    with pytest.raises(ValueError):
        check_inputs(x, w, fake(3, 8), 1e-5)
    with pytest.raises(ValueError):
        check_inputs(fake(5, 8, dtype=half), w, fake(8, dtype=half), 1e-5)
    with pytest.raises(TypeError):
        check_inputs(x, fake(8, dtype=half), None, 1e-5)
    with pytest.raises(TypeError):
        check_inputs(fake(5, 8, dtype=half), fake(8, dtype=torch.float16), None, 1e-5)
    with pytest.raises(TypeError):
        check_inputs(fake(5, 8, dtype=torch.float64), None, None, 1e-5)
    with pytest.raises(ValueError):
        check_inputs(x, w, b, 1e-5, fake(2, 3, 5, 7))
    with pytest.raises(ValueError):
        check_inputs(x, w, b, 1e-5, fake(2, 3, 5, 8, dtype=half))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError):
            check_inputs(x, w, b, eps)
    with pytest.raises(ValueError):
        check_inputs(fake(2, 32769), None, None, 1e-5)
    with pytest.raises(ValueError):
        check_inputs(fake(1).squeeze(0), None, None, 1e-5)
    with pytest.raises(ValueError):
        check_inputs(fake(1).expand(2**31, 1), None, None, 1e-5)


def test_c_interface_refuses():
    from flashy_linear_attention_b200 import _lib
    from flashy_linear_attention_b200._lib import FlaLayerNormArgs, FlaTensor

    lib = _lib.load()
    fwd, bwd, size = lib.fla_sm100_layer_norm_fwd, lib.fla_sm100_layer_norm_bwd, lib.fla_sm100_layer_norm_workspace_bytes
    assert fwd(None) == -1 and bwd(None) == -1 and size(None) == 0

    def args(**more):
        a = FlaLayerNormArgs()
        a.batch, a.heads, a.tokens, a.dim = 2, 3, 40, 8
        a.x = a.y = a.d_y = a.d_x = FlaTensor(64, 960, 320, 8)
        a.stats, a.d_weight, a.workspace, a.workspace_bytes, a.eps = 64, 64, 64, 1 << 30, 1e-5
        for k, v in more.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    none, odd = FlaTensor(None, 0, 0, 0), FlaTensor(65, 0, 0, 0)
    for k in ("batch", "heads", "tokens", "dim"):
        assert fwd(args(**{k: 0})) == -1 and bwd(args(**{k: -1})) == -1 and size(args(**{k: 0})) == 0
    assert fwd(args(x=none)) == -1 and fwd(args(y=none)) == -1 and bwd(args(d_y=none)) == -1 and bwd(args(stats=None)) == -1
    assert fwd(args(residual=FlaTensor(64, 960, 320, 8))) == -1 and fwd(args(sum=FlaTensor(64, 960, 320, 8))) == -1
    assert bwd(args(d_x=none, d_weight=None)) == -1
    assert fwd(args(dtype=3)) == -1 and fwd(args(w_dtype=1)) == -1 and fwd(args(dtype=2, w_dtype=0)) == -1
    assert fwd(args(eps=-1.0)) == -1 and fwd(args(eps=float("nan"))) == -1
    assert fwd(args(x=odd)) == -3 and bwd(args(d_sum=odd)) == -3 and fwd(args(weight=65)) == -3 and bwd(args(workspace=72)) == -3
    assert fwd(args(dim=32769)) == -2 and fwd(args(heads=65536, per_head=1)) == -2 and fwd(args(batch=1 << 20, tokens=1 << 12)) == -2
    need = size(args())
    assert need > 0 and size(args(d_weight=None)) == 0 and size(args(per_head=1)) >= 3 * 2 * 8 * 4
    assert bwd(args(workspace=None)) in (-5, -4, -6) and bwd(args(workspace_bytes=need - 1)) in (-5, -4, -6)
    if not torch.cuda.is_available():
        assert fwd(args()) in (-4, -6) and bwd(args()) in (-4, -6)
