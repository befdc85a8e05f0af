"""The 4-bit element of the cache: rows as codes of 4 bits with a power of two per 32 dims, against the definition in 64
bits (fp4_reference.py). Rows read back are equal, value for value; contexts are within the bound that `fp4_reference.attention`
derives from the kernels' roundings."""
import os

import numpy as np
import pytest

import saragossa_amd as skv
from fp4_reference import attention, stored

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DIMS = [(32, 8, 128), (16, 2, 256), (8, 2, 64), (12, 4, 96), (8, 8, 80), (8, 2, 512), (4, 2, 32), (6, 2, 40), (5, 1, 33), (3, 3, 7),
        (20, 1, 320), (40, 2, 128)]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _rows(rng, n, kv_dim):
    """Normal rows on channels of different sizes."""
    size = np.exp(0.7 * rng.standard_normal(kv_dim)).astype(np.float32)
    return rng.standard_normal((n, kv_dim), dtype=np.float32) * size


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _layer(state, rng, dims, capacity, window=0, rollback=None):
    kv = state.full_attention_with_element(capacity, *dims, skv.DTYPE_FP4, window, rollback)
    kv.set_block_table(rng.permutation(kv.pages()).astype(np.int32))
    return kv


class Pair:
    """A layer and the rows that it should hold, once stored."""

    def __init__(self, state, dims, capacity, seed, window=0, rollback=None):
        self.rng = np.random.default_rng(seed)
        self.dims, self.window = dims, window
        self.kv = _layer(state, self.rng, dims, capacity, window, rollback)
        self.kv_dim, self.q_dim = dims[1] * dims[2], dims[0] * dims[2]
        self.k = np.empty((0, self.kv_dim))
        self.v = np.empty((0, self.kv_dim))

    def new(self, n):
        return _rows(self.rng, n, self.kv_dim), _rows(self.rng, n, self.kv_dim), self.rng.standard_normal((n, self.q_dim), dtype=np.float32)

    def holds(self, k, v):
        self.k = np.concatenate([self.k, stored(k, self.dims[2])])
        self.v = np.concatenate([self.v, stored(v, self.dims[2])])

    def append(self, n):
        if n == 0:
            return
        k, v, _ = self.new(n)
        kd, vd = _dev(k), _dev(v)
        self.kv.encode_append_batch(_stream(), kd.data_ptr(), vd.data_ptr(), n)
        torch.cuda.synchronize()
        self.holds(k, v)

    def truncate(self, n):
        self.kv.truncate(n)
        self.k, self.v = self.k[:n], self.v[:n]

    def step(self, call=None):
        k, v, q = self.new(1)
        kd, vd, qd = _dev(k), _dev(v), _dev(q)
        out = torch.full((self.q_dim,), float("nan"), device="cuda")
        (call or self.kv.encode_decode_step)(_stream(), kd.data_ptr(), 0, vd.data_ptr(), 0, qd.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        self.holds(k, v)
        self.check(q, out.cpu().numpy()[None])

    def chunk(self, n):
        k, v, q = self.new(n)
        kd, vd, qd = _dev(k), _dev(v), _dev(q)
        out = torch.full((n, self.q_dim), float("nan"), device="cuda")
        self.kv.encode_prefill_rows(_stream(), qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), n, out.data_ptr())
        torch.cuda.synchronize()
        self.holds(k, v)
        self.check(q, out.cpu().numpy())

    def check(self, q, got, window_start=0):
        want, tol = attention(q, self.k, self.v, self.dims, window=self.window, window_start=window_start)
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) / tol).max()
        assert worst <= 1.0, f"{worst:.3g} times the bound"

    def check_rows(self, first=0):
        gk, gv = self.kv.read_rows_f32(first)
        assert np.array_equal(gk, self.k[first:].astype(np.float32))
        assert np.array_equal(gv, self.v[first:].astype(np.float32))


# ---- rows ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_rows_read_back_are_what_the_definition_says(state, dims):
    p = Pair(state, dims, 400, seed=dims[2])
    for n in (1, 4, 3, 24, 1, 130, 16, 77):  # starts and ends in the middle of pages, and of quads of rows
        p.append(n)
    p.check_rows()
    k, v, _ = p.new(1)
    p.kv.append_row(k[0], v[0])
    p.holds(k, v)
    p.check_rows(p.kv.len() - 20)
    bits_k, bits_v = p.kv.read_rows(3, 50)  # bf16 holds every value
    gk, gv = p.kv.read_rows_f32(3, 50)
    assert np.array_equal((bits_k.astype(np.uint32) << 16).view(np.float32), gk)
    assert np.array_equal((bits_v.astype(np.uint32) << 16).view(np.float32), gv)


def test_special_values_of_a_group(state):
    dims = (2, 2, 64)
    p = Pair(state, dims, 64, seed=1)
    f = np.float32
    groups = [
        np.zeros(32), np.full(32, -0.0), np.array([7.0, 6.999, 5.0, -5.0, 4.99, 3.5, -3.5, 2.5, 1.75, 1.25, 0.75, -0.75, 0.25, 0.26] + [0] * 18),
        np.array([7.0000005] + [0.5, 0.50001, -1.5, 1.0, 10.0] + [0] * 26), np.full(32, 1e-45), np.full(32, -1e-38),
        np.full(32, 3.4e38), np.array([2.0 ** 127 * 1.75, 2.0 ** 126] + [1.0] * 30), np.array([2.0 ** -124 * 7, 2.0 ** -126] + [2.0 ** -127] * 30),
        np.array([np.inf] + [1.0] * 31), np.array([1.0] * 31 + [np.nan]), np.array([-np.inf, np.nan] + [0.0] * 30),
        np.array([448.0] + [2.0 ** -k for k in range(31)]), np.array([2.0 ** 100] + [2.0 ** -100] * 31),
    ]
    rows = np.resize(np.concatenate(groups).astype(f), (16, p.kv_dim))
    kd, vd = _dev(rows), _dev(rows[::-1].copy())
    p.kv.encode_append_batch(_stream(), kd.data_ptr(), vd.data_ptr(), 16)
    torch.cuda.synchronize()
    gk, gv = p.kv.read_rows_f32()
    want_k, want_v = stored(rows, 64), stored(rows[::-1], 64)
    assert np.array_equal(gk, want_k.astype(f), equal_nan=True)
    assert np.array_equal(gv, want_v.astype(f), equal_nan=True)


@pytest.mark.parametrize("dims", [(8, 2, 64), (8, 8, 80), (16, 2, 256)], ids=str)
def test_rows_from_any_float_address_and_to_any_bf16_address(state, dims):
    p = Pair(state, dims, 64, seed=5)
    k, v, _ = p.new(37)
    kd, vd = torch.zeros(k.size + 3, device="cuda"), torch.zeros(v.size + 3, device="cuda")
    kd[1:1 + k.size], vd[3:] = _dev(k).flatten(), _dev(v).flatten()
    p.kv.encode_append_batch(_stream(), kd.data_ptr() + 4, vd.data_ptr() + 12, 37)
    p.holds(k, v)
    p.check_rows()
    ko = torch.zeros(20 * p.kv_dim + 1, device="cuda", dtype=torch.bfloat16)
    vo = torch.zeros(20 * p.kv_dim + 1, device="cuda", dtype=torch.bfloat16)
    p.kv.encode_gather(_stream(), 9, 20, ko.data_ptr() + 2, vo.data_ptr() + 2)
    p.kv.encode_gather(_stream(), 9, 20, None, None)  # nothing asked for
    torch.cuda.synchronize()
    assert ko[0] == 0 and vo[0] == 0
    assert np.array_equal(ko[1:].float().cpu().numpy().reshape(20, -1), p.k[9:29].astype(np.float32))
    assert np.array_equal(vo[1:].float().cpu().numpy().reshape(20, -1), p.v[9:29].astype(np.float32))


# ---- contexts ------------------------------------------------------------------------------

@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_decode_steps_from_the_first_row_on(state, dims):
    p = Pair(state, dims, 64, seed=dims[2] + 1)
    for _ in range(20):
        p.step()
    p.check_rows()


@pytest.mark.parametrize("rows", [31, 100, 257, 1000, 5003])
@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512), (12, 4, 96), (40, 2, 128)], ids=str)
def test_decode_steps_over_a_context(state, dims, rows):
    p = Pair(state, dims, rows + 8, seed=rows)
    p.append(rows)
    for _ in range(3):
        p.step()
    p.truncate(rows - 5)
    p.step()
    p.check_rows(rows - 20)


@pytest.mark.parametrize("window_start", [0, 1, 15, 16, 300, 699, 700])
def test_windows_of_the_callers_choice(state, window_start):
    dims = (8, 2, 128)
    p = Pair(state, dims, 701, seed=9)
    p.append(701)
    q = p.rng.standard_normal((1, p.q_dim), dtype=np.float32)
    p.check(q, p.kv.attention_decode_windowed(q, window_start)[None], window_start)


@pytest.mark.parametrize("dims", [(8, 2, 64), (16, 8, 256), (8, 2, 512), (5, 1, 33)], ids=str)
@pytest.mark.parametrize("window,rollback", [(48, None), (100, 0), (64, 0)])
def test_rings_that_wrap(state, dims, window, rollback):
    p = Pair(state, dims, 1000, seed=window, window=window, rollback=rollback)
    for n in (40, 100, 1):
        p.append(n)
        p.step()
    for n in (1, 2, 15, 16, 17, 70, 200):
        p.chunk(n)
        p.step()
    p.check_rows(p.kv.len() - window)


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512), (12, 4, 96), (5, 1, 33), (4, 2, 32), (40, 2, 128)], ids=str)
@pytest.mark.parametrize("base,n", [(0, 1), (0, 2), (0, 33), (7, 6), (300, 17), (1000, 64), (50, 200)])
def test_chunks(state, dims, base, n):
    p = Pair(state, dims, base + n + 4, seed=base + n)
    p.append(base)
    p.chunk(n)
    p.step()
    p.check_rows()


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512), (40, 2, 128)], ids=str)
def test_batches_of_sequences(state, dims):
    """Each sequence's context is its own, whatever lies beside it: lengths from none to some thousand, more than a launch takes."""
    lengths = [0, 1, 15, 16, 17, 300, 2000, 31, 5, 900, 64, 33, 48, 7, 129, 640, 3, 255]
    seqs = [Pair(state, dims, n + 4, seed=i) for i, n in enumerate(lengths)]
    for p, n in zip(seqs, lengths):
        p.append(n)
    for _ in range(2):
        rows = [p.new(1) for p in seqs]
        dev = [[_dev(a) for a in r] for r in rows]
        outs = [torch.full((p.q_dim,), float("nan"), device="cuda") for p in seqs]
        skv.encode_decode_step_batch([p.kv for p in seqs], _stream(), [d[0].data_ptr() for d in dev], [d[1].data_ptr() for d in dev],
                                     [d[2].data_ptr() for d in dev], [o.data_ptr() for o in outs])
        torch.cuda.synchronize()
        for p, (k, v, q), o in zip(seqs, rows, outs):
            p.holds(k, v)
            p.check(q, o.cpu().numpy()[None])
    for p in seqs:
        p.check_rows()


def test_batches_over_wrapped_rings(state):
    dims = (16, 8, 256)
    lengths = [200, 10, 64, 131]
    seqs = [Pair(state, dims, 300, seed=i, window=48, rollback=0) for i in range(4)]
    for p, n in zip(seqs, lengths):
        p.append(n)
    for _ in range(3):
        rows = [p.new(1) for p in seqs]
        dev = [[_dev(a) for a in r] for r in rows]
        outs = [torch.full((p.q_dim,), float("nan"), device="cuda") for p in seqs]
        skv.encode_decode_step_batch([p.kv for p in seqs], _stream(), *([d[i].data_ptr() for d in dev] for i in range(3)),
                                     [o.data_ptr() for o in outs])
        torch.cuda.synchronize()
        for p, (k, v, q), o in zip(seqs, rows, outs):
            p.holds(k, v)
            p.check(q, o.cpu().numpy()[None])


def test_steps_that_may_not_allocate(state):
    for dims, rows in (((32, 8, 128), 3000), ((16, 2, 256), 700), ((40, 2, 64), 90)):
        p = Pair(state, dims, rows + 3, seed=rows)
        p.append(rows)
        for _ in range(3):
            p.step(p.kv.encode_decode_step_static)
        p.check_rows(rows - 8)


# the shapes of the chunk kernel: by the chunk's size, or one for all chunks of 64 query slots and more
SHAPES = {"by-size": {}, "always": {"SKV_PREFILL_TILES": "2"},
          "one-tile": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "1000000"},
          "two-tiles": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "0"}, "never": {"SKV_PREFILL_TILES": "0"}}


@pytest.fixture(params=SHAPES, ids=str)
def chunk_shape(request):
    env = SHAPES[request.param]
    saved = {k: os.environ.get(k) for k in env}
    os.environ.update(env)
    skv.flags.reload()
    yield request.param
    for k, v in saved.items():
        os.environ.pop(k) if v is None else os.environ.__setitem__(k, v)
    skv.flags.reload()


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512), (12, 4, 96), (5, 1, 33), (4, 2, 32), (40, 2, 128)], ids=str)
@pytest.mark.parametrize("base,n", [(0, 65), (777, 100), (3000, 37), (129, 300)])
def test_chunks_in_every_shape(state, chunk_shape, dims, base, n):
    p = Pair(state, dims, base + n, seed=base + n)
    p.append(base)
    p.chunk(n)


@pytest.mark.parametrize("dims", [(16, 8, 256), (8, 2, 64), (8, 2, 512), (5, 1, 33), (16, 2, 128)], ids=str)
def test_chunks_over_rings_in_every_shape(state, chunk_shape, dims):
    p = Pair(state, dims, 1200, seed=3, window=150, rollback=20)
    p.append(60)
    for n in (64, 33, 200, 90, 128):
        p.chunk(n)
    p.step()
    p.check_rows(p.kv.len() - 150)


@pytest.mark.parametrize("dims", [(16, 2, 256), (32, 8, 128), (8, 2, 64), (8, 2, 512)], ids=str)
@pytest.mark.parametrize("n", [7, 40, 150])
def test_rows_that_are_nan_reach_the_queries_that_attend_them_and_no_other(state, chunk_shape, dims, n):
    """A padded chunk: rows behind a query's own are NaN or infinite, in K, in V or in some groups of dims."""
    p = Pair(state, dims, 400, seed=n)
    p.append(100)
    k, v, q = p.new(n)
    bad = n - 3
    v[bad, :32] = np.nan           # the first group of dims of the first head
    v[bad + 1, -5] = np.inf        # of the last group of the last head
    k[bad + 2] = np.nan
    kd, vd, qd = _dev(k), _dev(v), _dev(q)
    out = torch.zeros((n, p.q_dim), device="cuda")
    p.kv.encode_prefill_rows(_stream(), qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), n, out.data_ptr())
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(n, dims[0], dims[2])
    clean_k, clean_v = k.copy(), v.copy()
    clean_k[bad + 2], clean_v[bad, :32], clean_v[bad + 1, -32:] = 0, 0, 0
    keys = np.concatenate([p.k, stored(clean_k, dims[2])])
    vals = np.concatenate([p.v, stored(clean_v, dims[2])])
    want, tol = attention(q[:bad + 2], keys[:-1], vals[:-1], dims)
    want, tol = want.reshape(bad + 2, *got.shape[1:]), tol.reshape(bad + 2, *got.shape[1:])
    group = dims[0] // dims[1]
    want[bad:, :group, :32] = np.nan
    want[bad + 1:, -group:, -min(32, dims[2]):] = np.nan
    assert np.array_equal(np.isnan(got[:bad + 2]), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(got[:bad + 2] - want)[ok] <= tol[ok]).all()
    assert np.isnan(got[bad + 2]).all()
