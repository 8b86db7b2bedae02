"""The gate's backward pass by itself, from kept values as they are: every stripe of 16 rows and every group of columns is one workgroup's.

Tolerance: the activation and its slope are off by 2^-15 of a value (their terms are at most 1.2), products in fp32 by 2^-22, results are rounded to bf16."""
import pytest
import torch

from test_gated_mlp_gpu import act64, kept_values, near, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,f", [(1, 8), (16, 128), (17, 136), (127, 1000), (129, 120), (1000, 264), (2065, 15336), (40000, 40), (257, 65544)])
def test_every_row_and_column(T, f, act):
    from easyllm_amd import kernels as K
    print("gate_bwd", T, f, act, flush=True)
    x, wg, wu = rnd(T, 8), rnd(f, 8, seed=1), rnd(f, 8, seed=2)
    _, kept = K.gated_fwd(act, x, wg, wu, True)
    d = rnd(T, f, seed=3)
    dgate, dup = K.gate_bwd(act, d, kept)
    for first in range(0, T, 4096):
        rows = slice(first, first + 4096)
        g, u = kept_values(kept, T, f, rows)
        y, slope = act64(g, act)
        near(dup[rows], d[rows].double() * y, d[rows].double().abs() * (y.abs() + g.abs()) * 2.0 ** -15, "dup")
        near(dgate[rows], d[rows].double() * u * slope, (d[rows].double() * u).abs() * (slope.abs() + 1.2) * 2.0 ** -15, "dgate")
