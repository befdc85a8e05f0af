"""Prompts of linear attention whose numbers lie far apart: every factor counts for what it is, whatever the chunk holds beside it."""
import pytest

from linear_bounds import bounds
from linear_reference import close

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

GEOMETRIES = [(1, 2, 32, 64), (2, 2, 64, 80), (1, 2, 128, 128), (1, 1, 100, 200), (1, 1, 256, 128), (1, 1, 256, 40)]


def _inputs(geo, n, seed):
    kh, vh, dk, dv = geo
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(n, kh, dk, generator=gen) for _ in range(2))
    v = torch.randn(n, vh, dv, generator=gen)
    g = -torch.exp(torch.linspace(-5.0, 1.0, vh)) * torch.rand(n, vh, generator=gen)
    return q, k, v, g, torch.randn(vh, dk, dv, generator=gen), gen


def _run(ctx, geo, q, k, v, g, s, scale):
    kh, vh, dk, dv = geo
    n = q.shape[0]
    op = ctx.linear_attention(*geo, scale)
    dev = [x.cuda().contiguous() for x in (q, k, v, g)]
    st = None if s is None else s.cuda()
    out, new = torch.empty(n, vh, dv, device="cuda"), torch.empty(vh, dk, dv, device="cuda")
    op.encode_rows(torch.cuda.current_stream().cuda_stream, dev[0].data_ptr(), 0, dev[1].data_ptr(), 0, dev[2].data_ptr(), 0, dev[3].data_ptr(), vh, n,
                   None if st is None else st.data_ptr(), new.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    return out, new


def _check(ctx, geo, q, k, v, g, s, scale=0.25, **how):
    want, tol, last, last_tol = bounds(q, k, v, g, s, scale, **how)
    out, new = _run(ctx, geo, q, k, v, g, s, scale)
    close(out, want, tol, "outputs")
    close(new, last, last_tol, "state")


@pytest.mark.parametrize("n", [9, 40, 300, 1500])
@pytest.mark.parametrize("geo", GEOMETRIES)
def test_single_products(state, geo, n):
    """One dim of q and one of k a token, so that a sum has few terms: factors of fewer bits than f32's show."""
    q, k, v, g, s, gen = _inputs(geo, n, n)
    dk = geo[2]
    for x, dims in ((k, torch.arange(n) * 5 % dk), (q, torch.randint(dk, (n,), generator=gen))):
        x *= torch.nn.functional.one_hot(dims, dk)[:, None, :]
    _check(state, geo, q, k, v, g, s, single=True)


@pytest.mark.parametrize("n", [33, 64, 700])
@pytest.mark.parametrize("apart", [20, 40, 60])
@pytest.mark.parametrize("geo", [(1, 2, 32, 64), (1, 2, 128, 128), (1, 1, 256, 64)])
def test_a_large_value_leaves_the_others_alone(state, geo, apart, n):
    """The last v of a chunk 2^apart times the others: earlier outputs are made of those alone."""
    q, k, v, g, s, _ = _inputs(geo, n, n + apart)
    v[31], v[-1] = v[31] * 2.0 ** apart, v[-1] * 2.0 ** apart
    _check(state, geo, q, k, v, g, s)


@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("geo", [(1, 2, 32, 64), (1, 2, 128, 128), (1, 1, 256, 64)])
def test_values_of_tokens_far_apart(state, geo, n):
    q, k, v, g, s, gen = _inputs(geo, n, n)
    _check(state, geo, q, k, v * torch.exp2(torch.randint(-40, 41, (n, geo[1], 1), generator=gen).float()), g, s)


@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("geo", [(1, 2, 64, 64), (1, 2, 128, 128)])
def test_keys_of_dims_far_apart(state, geo, n):
    """A large k in one dim, which q does not ask for, leaves the dims that it does ask for alone."""
    q, k, v, g, s, _ = _inputs(geo, n, n)
    k[n // 3, :, 7], q[:, :, 7] = 2.0 ** 50, 0.0
    _check(state, geo, q, k, v, g, s)


@pytest.mark.parametrize("powers", [(-100, 0, 0, 0), (0, -100, 40, -60), (0, 0, -100, -100), (60, 40, -80, -40), (-40, 100, -60, 0), (90, -100, 0, -90)])
@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("geo", [(1, 2, 32, 64), (1, 2, 128, 128)])
def test_small_factors(state, geo, n, powers):
    """q, k, v and the state of any of f32's sizes."""
    q, k, v, g, s, _ = _inputs(geo, n, n)
    _check(state, geo, *(x * 2.0 ** p for x, p in zip((q, k, v), powers)), g, s * 2.0 ** powers[3], scale=1.0)


@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("size", [30, 45, 90])
@pytest.mark.parametrize("geo", [(1, 2, 64, 64), (1, 2, 128, 128)])
def test_a_large_row_of_the_state_leaves_the_others_alone(state, geo, n, size):
    q, k, v, g, s, _ = _inputs(geo, n, n + size)
    g = g * 0.0
    s[:, 9], q[:, :, 9], k[:, :, 9] = s[:, 9] * 2.0 ** size, 0.0, 0.0
    _check(state, geo, q, k, v, g, s)


@pytest.mark.parametrize("n,there,back", [(70, (3, 9), (40, 44)), (70, (3, 9), (15, 20)), (700, (130, 140), (300, 310)), (700, (20, 130), (200, 400))])
@pytest.mark.parametrize("size,growth", [(-100, 55.0), (100, -55.0), (0, -60.0)])
def test_decays_beyond_what_f32_holds(state, n, there, back, size, growth):
    """Two tokens together take the state up or down by 2^158 and two others bring it back, within one chunk, from chunk to chunk and
    from part to part: the states are ordinary numbers all the way, so a factor between two of them may not be infinite or 0."""
    geo = (1, 2, 64, 80)
    q, k, v, g, s, _ = _inputs(geo, n, n)
    for t in there:
        g[t] = growth
    for t in back:
        g[t] = -growth
    small = 2.0 ** (min(size, 0) / 2 - 10)
    if growth < 0:  # nothing new: what comes back is what was there
        k[there[0]:back[1]] = 0.0
    _check(state, geo, q, k * small, v * small, g, s * 2.0 ** size)
