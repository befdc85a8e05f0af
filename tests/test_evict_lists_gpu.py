"""Evictions from more rows than one workgroup chooses from, on every element and head: their moves go by the list of movers, which K's and V's
workgroups read while K's write it."""
import pytest

from test_evict_gpu import ELEMENTS, _check, _layer, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,keep", [(17001, 9000), (17001, 16985), (33003, 15)])
@pytest.mark.parametrize("geo", [(8, 2, 128), (2, 2, 90), (2, 1, 256)])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("with_kept", [True, False])
def test_movers_from_a_list(state, element, geo, rows, keep, with_kept):
    kv, before, rng = _layer(state, element, geo, rows, rows + keep)
    _check(kv, before, _weights(rng, geo[1], rows), keep, 4, 9, with_kept=with_kept)


@pytest.mark.parametrize("element", ELEMENTS)
def test_longer_than_the_threads_hold(state, element):
    """More than 32768 rows, whose weights are read anew in every pass; an odd page at the end and a budget that ends inside one."""
    kv, before, rng = _layer(state, element, (4, 2, 96), 70001, 3)
    _check(kv, before, _weights(rng, 2, 70001), 34567, 0, 100)
