"""Prompts of heads of one to three v dims, over many workgroups: no output is anything but its own workgroup's."""
import pytest

from test_linear_factors_gpu import _check, _inputs

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [9, 33, 777, 2000])
@pytest.mark.parametrize("geo", [(3, 9, 251, 1), (2, 8, 64, 2), (1, 16, 32, 3), (4, 64, 5, 1), (1, 1, 128, 2), (2, 4, 100, 5)])
def test_narrow_heads(state, geo, n):
    for seed in range(3):
        q, k, v, g, s, _ = _inputs(geo, n, n + seed)
        _check(state, geo, q, k, v, g, s if seed else None)
