"""The gated linear recurrence at the ends of its range: rows whose bytes do not fit 32 bits. Values are checked at both
ends of the rows against the recurrence in 64 bits; tolerances are those of test_recurrence_gpu.py."""
import pytest
import torch

from test_recurrence_gpu import BF, DEV, FP, check, reference

pytestmark = pytest.mark.gpu


def needs(gigabytes):
    free = torch.cuda.mem_get_info()[0] / 2**30
    if free < gigabytes + 4:
        pytest.skip(f"needs {gigabytes} GB")


def repeated(columns, dtype, seed):
    """A row of `columns` with period 997."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    few = torch.rand(997, device=DEV, generator=gen).to(dtype)
    return few.repeat(columns // 997 + 1)[:columns]


def ends(t, n=200):
    return torch.cat([t[..., :n], t[..., -n:]], -1)


@pytest.mark.parametrize("columns,tokens,dtype,gigabytes", [
    (2**28 + 32, 1, BF, 6),     # ten times the columns pass 32 bits
    (2**29 + 33, 1, FP, 15),    # a row's bytes do
])
def test_wide_rows(columns, tokens, dtype, gigabytes):
    from flashy_linear_attention_b200 import GatedLinearRecurrence

    torch.cuda.empty_cache()
    needs(gigabytes)
    x, g = repeated(columns, dtype, 1), repeated(columns, dtype, 2).neg_()
    x, g = (t.expand(1, 1, tokens, columns) for t in (x, g))
    out, s_final = GatedLinearRecurrence.apply(x, g)
    want = reference(ends(x), ends(g), None)
    check("out", ends(out), want["out"])
    check("s_final", ends(s_final), want["s_final"])
    del out, s_final
    torch.cuda.empty_cache()
