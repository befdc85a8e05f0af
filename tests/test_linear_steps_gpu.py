"""The recurrence of linear attention, in few tokens and single ones, to the bounds of f32 numbers."""
import pytest

from linear_bounds import bounds
from linear_reference import close
from test_linear_factors_gpu import GEOMETRIES, _check, _inputs

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 8])
@pytest.mark.parametrize("geo", GEOMETRIES + [(1, 1, 1, 1), (2, 6, 33, 7)])
def test_few_tokens(state, geo, n):
    q, k, v, g, s, gen = _inputs(geo, n, n)
    _check(state, geo, q, k, v, g, s, step=1)
    for x in (q, k):
        x *= torch.nn.functional.one_hot(torch.randint(geo[2], (n,), generator=gen), geo[2])[:, None, :]
    _check(state, geo, q, k, v, g, s, step=1, single=True)


@pytest.mark.parametrize("seqs", [1, 3, 17])
@pytest.mark.parametrize("geo", GEOMETRIES)
def test_single_tokens(state, geo, seqs):
    kh, vh, dk, dv = geo
    q, k, v, g, _, gen = _inputs(geo, seqs, seqs)
    for x in (q, k):
        x *= torch.nn.functional.one_hot(torch.randint(dk, (seqs,), generator=gen), dk)[:, None, :]
    s = torch.randn(seqs, vh, dk, dv, generator=gen)
    op = state.linear_attention(*geo, 0.25)
    dev = [x.cuda().contiguous() for x in (q, k, v, g)]
    st, out = s.cuda(), torch.empty(seqs, vh, dv, device="cuda")
    at = [st[i].data_ptr() for i in range(seqs)]
    op.encode_step(torch.cuda.current_stream().cuda_stream, dev[0].data_ptr(), 0, dev[1].data_ptr(), 0, dev[2].data_ptr(), 0, dev[3].data_ptr(), vh, at, at,
                   out.data_ptr())
    for i in range(seqs):
        want, tol, last, last_tol = bounds(q[i:i + 1], k[i:i + 1], v[i:i + 1], g[i:i + 1], s[i], 0.25, single=True, step=1)
        close(out[i:i + 1], want, tol, f"sequence {i}")
        close(st[i], last, last_tol, f"state {i}")
