"""The 4-bit element on the rest of the entry points: rows behind the last one, captured graphs, contexts over their inputs, steps with
the norm and rotation in front, the plain kernel, knobs, snapshots and caches of prompts, streams side by side, pools beyond 4 GiB, refusals,
and a sequence's whole life."""
import contextlib
import os

import numpy as np
import pytest

import oracle
import saragossa_amd as skv
from fp4_reference import attention, stored
from test_fp4_kv_gpu import Pair, _dev, _layer, _rows, _stream

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@contextlib.contextmanager
def _env(**env):
    saved = {k: os.environ.get(k) for k in env}
    os.environ.update(env)
    skv.flags.reload()
    try:
        yield
    finally:
        for k, was in saved.items():
            os.environ.pop(k) if was is None else os.environ.__setitem__(k, was)
        skv.flags.reload()


CHUNKS = {"by-size": {}, "halves": {"SKV_PREFILL_TILES": "2"},
          "one-tile": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "1000000"},
          "two-tiles": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "0"}, "streaming": {"SKV_PREFILL_TILES": "0"}}


@pytest.fixture(params=CHUNKS, ids=str)
def chunk_kernel(request):
    with _env(**CHUNKS[request.param]):
        yield request.param


def _poison(rng, n, kv_dim):
    rows = _rows(rng, n, kv_dim)
    rows[0::3] = np.nan
    rows[1::3] = np.inf
    rows[2::3] = -np.inf
    return rows


def _twins(state, dims, rows, seed, capacity, window=0):
    """Two layers of the same rows and block table."""
    rng = np.random.default_rng(seed)
    k, v = _rows(rng, rows, dims[1] * dims[2]), _rows(rng, rows, dims[1] * dims[2])
    pair, table = [], None
    for _ in range(2):
        kv = state.full_attention_fp4(capacity, *dims, window=window)
        table = rng.permutation(kv.pages()).astype(np.int32) if table is None else table
        kv.set_block_table(table)
        if rows:
            kv.seed(k, v, rows)
        pair.append(kv)
    return pair, rng


# ---- rows that the cache does not count ------------------------------------------------------------

@pytest.mark.parametrize("dims,base,window", [((16, 2, 256), 700, 0), ((32, 8, 128), 37, 0), ((8, 2, 64), 100, 48), ((16, 8, 512), 300, 0),
                                              ((5, 1, 33), 45, 0)], ids=str)
def test_rolled_back_nan_and_inf_rows_leave_no_trace(state, chunk_kernel, dims, base, window):
    kv_dim, q_dim = dims[1] * dims[2], dims[0] * dims[2]
    (dirty, clean), rng = _twins(state, dims, base, base + dims[2], base + 160, window)
    bad = _poison(rng, 7, kv_dim)
    dirty.prefill_rows(rng.standard_normal((7, q_dim), dtype=np.float32), bad, bad)
    dirty.truncate(base)
    for _ in range(3):
        k, v, q = _rows(rng, 1, kv_dim), _rows(rng, 1, kv_dim), rng.standard_normal(q_dim, dtype=np.float32)
        outs = []
        for kv in (dirty, clean):
            kv.append_row(k[0], v[0])
            outs.append(kv.attention_decode_windowed(q, skv.flags.window_start(kv.len() - 1, window)))
        assert np.isfinite(outs[0]).all() and np.array_equal(*outs)
    k, v, q = _dev(_rows(rng, 1, kv_dim)), _dev(_rows(rng, 1, kv_dim)), _dev(rng.standard_normal(q_dim, dtype=np.float32))
    outs = []
    for kv in (dirty, clean):
        outs.append(torch.full((q_dim,), float("nan"), device="cuda"))
        kv.encode_decode_step(_stream(), k.data_ptr(), 0, v.data_ptr(), 0, q.data_ptr(), outs[-1].data_ptr())
    assert torch.isfinite(outs[0]).all() and torch.equal(*outs)
    for n in (2, 70):
        bad = _poison(rng, 30, kv_dim)  # (a ring keeps 32 rows behind its window)
        dirty.prefill_rows(rng.standard_normal((30, q_dim), dtype=np.float32), bad, bad)
        dirty.truncate(clean.len())
        qn, kn, vn = rng.standard_normal((n, q_dim), dtype=np.float32), _rows(rng, n, kv_dim), _rows(rng, n, kv_dim)
        outs = [kv.prefill_rows(qn, kn, vn) for kv in (dirty, clean)]
        assert np.isfinite(outs[0]).all() and np.array_equal(*outs)
    first = max(0, clean.len() - window) if window else 0
    for a, b in zip(dirty.read_rows_f32(first), clean.read_rows_f32(first)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("dims,window,base", [((8, 2, 64), 48, 101), ((16, 8, 256), 100, 333), ((4, 1, 40), 250, 261), ((8, 2, 512), 70, 99)], ids=str)
def test_rows_of_an_earlier_ring_chunk_leave_no_trace(chunk_kernel, dims, window, base):
    kv_dim, q_dim = dims[1] * dims[2], dims[0] * dims[2]
    rng = np.random.default_rng(base)
    k, v, q = _rows(rng, base + 160, kv_dim), _rows(rng, base + 160, kv_dim), rng.standard_normal((160, q_dim), dtype=np.float32)
    outs = []
    for poisoned in (True, False):
        ctx = skv.DecodeResidentState(0)
        kv = ctx.full_attention_fp4(base + 160, *dims, window=window)
        kv.seed(k[:base], v[:base], base)
        if poisoned:
            other = ctx.full_attention_fp4(base + 400, *dims, window=window)
            other.seed(k[:base], v[:base], base)
            bad = _poison(rng, 333, kv_dim)
            other.prefill_rows(np.ones((333, q_dim), np.float32), bad, bad)
        outs.append(np.concatenate([kv.prefill_rows(q[:90], k[base:base + 90], v[base:base + 90]),
                                    kv.prefill_rows(q[90:], k[base + 90:], v[base + 90:])]))
    assert np.isfinite(outs[0]).all() and np.array_equal(*outs)


@pytest.mark.parametrize("window,rollback", [(64, 0), (60, 0), (64, None), (33, 3), (1, 0), (5, 20), (16, 0)])
@pytest.mark.parametrize("dims", [(16, 8, 256), (8, 2, 64), (12, 4, 96), (8, 2, 512)], ids=str)
def test_chunks_about_as_long_as_their_ring(state, chunk_kernel, dims, window, rollback):
    """Up to a ring's rows are stored before the chunk attends, with what they overwrite kept aside, more of them after it."""
    p = Pair(state, dims, 2000, seed=window, window=window, rollback=rollback)
    ring = p.kv.pages() * 16
    p.append(ring + 5)
    for n in (ring - 6, ring, 3, ring - 16, 13, ring + 1, 2, 2 * ring + 7, 16, 17, ring - 1):
        p.chunk(max(n, 1))
        p.step()
        p.check_rows(p.kv.len() - window)


# ---- values of any size --------------------------------------------------------------------------

@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (12, 4, 96), (8, 2, 512), (5, 1, 33)], ids=str)
@pytest.mark.parametrize("case", ["tiny", "huge", "some rows", "some groups", "zeros"])
def test_values_whose_powers_half_precision_does_not_have(state, chunk_kernel, dims, case):
    """V from 1e-30 to 1e30, whole caches of it, or rows and groups of dims among others; rows of zeros."""
    p = Pair(state, dims, 700, seed=8)
    fresh = p.new

    def new(n):
        k, v, q = fresh(n)
        v = v.reshape(n, dims[1], dims[2])
        if case == "tiny":
            v *= np.float32(1e-12)
        elif case == "huge":
            v *= np.float32(1e30)
        elif case == "some rows":
            v[::7] *= np.float32(2.0 ** -18)
            v[3::11] *= np.float32(2.0 ** 17)
        elif case == "some groups":
            v[::5, :, :32] *= np.float32(1e-30)
            v[1::5, -1, -32:] *= np.float32(1e-6)
        else:
            v[::2] = 0
            v[1::4, :, :32] = 0
        return k, v.reshape(n, -1), q

    p.new = new
    p.append(333)
    p.step()
    for n in (5, 90, 70):
        p.chunk(n)
        p.step()
    p.check_rows()


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512), (5, 1, 33)], ids=str)
def test_queries_of_any_size(state, chunk_kernel, dims):
    """Rows of zeros, groups of zeros, 1e-36 and 1e4 times normal rows, and one large dim among small ones."""
    p = Pair(state, dims, 500, seed=12)
    fresh = p.new

    def new(n):
        k, v, q = fresh(n)
        q = q.reshape(n, dims[0], dims[2])
        q[0::6] = 0
        q[1::6, :, :32] = 0
        q[2::6] *= np.float32(1e-36)
        q[3::6] *= np.float32(1e4)
        q[4::6, :, 3] *= np.float32(1e5)
        return k, v, q.reshape(n, -1)

    p.new = new
    p.append(260)
    p.step()
    p.chunk(12)
    p.chunk(80)


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 512)], ids=str)
@pytest.mark.parametrize("attn_scalar", [1e-8, 1e-3, 1e8])
def test_steps_of_any_scale(state, dims, attn_scalar):
    p = Pair(state, dims, 400, seed=13)
    p.append(300)
    for zeros in (False, True):
        k, v, q = p.new(1)
        if zeros:
            q[:, :dims[2] // 2] = 0
        kd, vd, qd, out = _dev(k), _dev(v), _dev(q), torch.zeros(p.q_dim, device="cuda")
        p.kv.encode_decode_step_prekv(_stream(), None, 0, qd.data_ptr(), 0, kd.data_ptr(), 0, vd.data_ptr(), 0, None, None, 1e-6, attn_scalar, out.data_ptr())
        p.holds(k, v)
        want, tol = attention(q, p.k, p.v, dims, attn_scalar=attn_scalar)
        assert (np.abs(out.cpu().numpy()[None] - want) <= tol).all()


# ---- graphs ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dims,window,base,rows", [((16, 2, 256), 0, 2000, 6), ((8, 2, 64), 0, 900, 130), ((32, 8, 128), 0, 2000, 128),
                                                   ((8, 2, 64), 100, 300, 130), ((16, 8, 256), 100, 300, 20)], ids=str)
def test_captured_chunks_and_steps_replay_the_eager_result(dims, window, base, rows):
    ctx = skv.DecodeResidentState(0)
    kv_dim, q_dim = dims[1] * dims[2], dims[0] * dims[2]
    rng = np.random.default_rng(base + rows)
    kv = _layer(ctx, rng, dims, base + rows + 1, window)
    side = torch.cuda.Stream()
    old = [_dev(_rows(rng, base, kv_dim)) for _ in range(2)]
    k, v = (_dev(_rows(rng, rows + 1, kv_dim)) for _ in range(2))
    q = _dev(rng.standard_normal((rows + 1, q_dim), dtype=np.float32))
    out = torch.zeros(rows + 1, q_dim, device="cuda")
    torch.cuda.synchronize()

    def refill():
        kv.truncate(0)
        kv.encode_append_batch(side.cuda_stream, old[0].data_ptr(), old[1].data_ptr(), base)

    def run():
        kv.encode_prefill_rows(side.cuda_stream, q.data_ptr(), k.data_ptr(), v.data_ptr(), rows, out.data_ptr())
        kv.encode_decode_step(side.cuda_stream, k[rows].data_ptr(), 0, v[rows].data_ptr(), 0, q[rows].data_ptr(), out[rows].data_ptr())

    with torch.cuda.stream(side):
        refill()
        run()
        side.synchronize()
        want = out.clone()
        assert torch.isfinite(want).all()
        refill()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        for replay in range(4):
            refill()
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want), replay
            # eager work that outgrows the stream's scratch
            more = ctx.full_attention_fp4(4000 + 900 * replay, *dims)
            n = 1000 + 800 * replay
            x = torch.randn(n, q_dim, device="cuda")
            r = torch.randn(n, kv_dim, device="cuda")
            more.encode_prefill_rows(side.cuda_stream, x.data_ptr(), r.data_ptr(), r.data_ptr(), n, x.data_ptr())
            side.synchronize()
            more.close()
        refill()
        out.zero_()
        run()
        side.synchronize()
        assert torch.equal(out, want)


# ---- a context over what its launch reads --------------------------------------------------------

def _apart(kv, first=0):
    """How far two launches over the same rows and queries may be from each other, split differently: they have the same scores, and each rounds
    its weights by 2^-18 at most and its exponentials and sums by 2^-20 (fp4_reference.py), relative to the mean of |v|: at most the largest |v|."""
    return 2 * (2.0 ** -18 + 2.0 ** -20) * float(np.abs(kv.read_rows_f32(first)[1]).max())


def _placed(src, lead, room):
    buf = torch.zeros(max(room, lead + src.numel()), device="cuda")
    buf[lead:lead + src.numel()] = src.reshape(-1)
    return buf


@pytest.mark.parametrize("dims", [(32, 8, 128), (8, 2, 64), (24, 1, 128), (8, 8, 80), (4, 2, 512)], ids=str)
@pytest.mark.parametrize("rows", [15, 100, 700])
@pytest.mark.parametrize("over", ["q", "in place", "k", "v"])
@pytest.mark.parametrize("env", [{}, {"RETI_RUST_SDPA_2PASS": "0"}, {"SKV_FUSED_APPEND": "0"}, {"RETI_RUST_FLASH_SDPA": "0"}],
                         ids=["", "unsplit", "append apart", "plain"])
def test_steps_over_their_inputs(state, dims, rows, over, env):
    with _env(**env):
        (one, other), rng = _twins(state, dims, rows, rows, rows + 1)
        q, k, v = (_dev(rng.standard_normal(n * dims[2], dtype=np.float32)) for n in (dims[0], dims[1], dims[1]))
        want = torch.zeros(q.numel(), device="cuda")
        other.encode_decode_step(_stream(), k.data_ptr(), 0, v.data_ptr(), 0, q.data_ptr(), want.data_ptr())
        lead = 0 if over == "in place" else dims[2]
        under = over if over in "kv" else "q"
        buf = {n: _placed(a, lead if n == under else 0, lead + q.numel()) for n, a in zip("qkv", (q, k, v))}
        at = {n: b.data_ptr() + (lead * 4 if n == under else 0) for n, b in buf.items()}
        one.encode_decode_step(_stream(), at["k"], 0, at["v"], 0, at["q"], buf[under].data_ptr())
        torch.cuda.synchronize()
        assert (buf[under][:q.numel()] - want).abs().max().item() <= _apart(other)
        assert one.len() == rows + 1
        for a, b in zip(one.read_rows_f32(rows), other.read_rows_f32(rows)):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("dims,rows,chunk,window", [((32, 8, 128), 0, 512, 0), ((32, 8, 128), 0, 200, 0), ((8, 2, 64), 60, 6, 0), ((8, 2, 64), 3000, 12, 0),
                                                    ((16, 8, 256), 500, 512, 1024), ((32, 8, 128), 600, 512, 512), ((16, 8, 256), 1100, 64, 1024),
                                                    ((8, 2, 512), 30, 32, 0)], ids=str)
@pytest.mark.parametrize("over", ["q", "in place", "k", "v"])
def test_chunks_over_their_inputs(state, dims, rows, chunk, window, over):
    (one, other), rng = _twins(state, dims, rows, rows + chunk, rows + chunk, window)
    q, k, v = (_dev(rng.standard_normal((chunk, n * dims[2]), dtype=np.float32)) for n in (dims[0], dims[1], dims[1]))
    want = torch.zeros(q.numel(), device="cuda")
    other.encode_prefill_rows(_stream(), q.data_ptr(), k.data_ptr(), v.data_ptr(), chunk, want.data_ptr())
    lead = 0 if over == "in place" else 3 * dims[2]
    under = over if over in "kv" else "q"
    buf = {n: _placed(a, lead if n == under else 0, lead + q.numel()) for n, a in zip("qkv", (q, k, v))}
    at = {n: b.data_ptr() + (lead * 4 if n == under else 0) for n, b in buf.items()}
    one.encode_prefill_rows(_stream(), at["q"], at["k"], at["v"], chunk, buf[under].data_ptr())
    torch.cuda.synchronize()
    first = max(0, one.len() - window) if window else 0
    assert (buf[under][:q.numel()] - want).abs().max().item() <= _apart(other, first)
    for a, b in zip(one.read_rows_f32(first), other.read_rows_f32(first)):
        assert np.array_equal(a, b)


# ---- norm, rotation and gate around the step --------------------------------------------------------

@pytest.mark.parametrize("dims,window,start,rope_dims", [((16, 2, 256), 0, 700, 64), ((32, 8, 128), 0, 40, 128), ((8, 4, 64), 32, 5, 64), ((6, 2, 96), 0, 0, 48),
                                                         ((4, 2, 512), 0, 100, 128), ((24, 1, 64), 0, 30, 64)], ids=str)
@pytest.mark.parametrize("env", [{}, {"SKV_FUSED_APPEND": "0"}, {"RETI_RUST_FLASH_SDPA": "0"}], ids=["", "append apart", "plain"])
@pytest.mark.parametrize("gated", [False, True])
def test_steps_from_the_projections(state, dims, window, start, rope_dims, env, gated):
    """Norm and rotation are bit-exact against the oracle's, so that the stored rows are equal and the context is within the bound."""
    heads, kv_heads, hd = dims
    q_dim, kv_dim, steps, eps, theta = heads * hd, kv_heads * hd, 12, 1e-6, 1e6
    with _env(**env):
        p = Pair(state, dims, start + steps, seed=start + hd, window=window)
        p.append(start)
        rope = state.rope_table(start + steps, rope_dims, theta)
        qw, kw = (p.rng.random(hd, dtype=np.float32) + np.float32(0.5) for _ in range(2))
        qwd, kwd = _dev(qw), _dev(kw)
        lead = 2 * q_dim if gated else q_dim
        for t in range(start, start + steps):
            raw = p.rng.standard_normal(lead + 2 * kv_dim, dtype=np.float32)
            rd, out = _dev(raw), torch.zeros(q_dim, device="cuda")
            call = p.kv.encode_decode_step_gated if gated else p.kv.encode_decode_step_prekv
            call(_stream(), rope, t, rd.data_ptr(), 0, rd.data_ptr(), lead * 4, rd.data_ptr(), (lead + kv_dim) * 4, qwd.data_ptr(), kwd.data_ptr(),
                 eps, float(hd), out.data_ptr())
            q_raw, gate = oracle.split_attention_gate(raw[:lead], heads, hd) if gated else (raw[None, :q_dim], None)
            q = oracle.rms_norm_rope_heads_at(q_raw[0], heads, hd, rope_dims, qw, eps, theta, t)
            k = oracle.rms_norm_rope_heads_at(raw[lead:lead + kv_dim], kv_heads, hd, rope_dims, kw, eps, theta, t)
            p.holds(k.reshape(1, -1), raw[lead + kv_dim:].reshape(1, -1))
            want, tol = attention(q.reshape(1, -1), p.k, p.v, dims, window=window)
            if gated:  # the gate's sigmoid in f32: an exponential, a sum and a quotient, 8 halves of a step, and the product's rounding
                g = 1.0 / (1.0 + np.exp(-gate[0].astype(np.float64).reshape(1, -1)))
                tol, want = tol * g + np.abs(want) * g * 10 * 2.0 ** -24, want * g
            assert (np.abs(out.cpu().numpy()[None] - want) <= tol).all(), t
        first = max(0, start + steps - window) if window else 0
        p.check_rows(first)
        rope.close()


# ---- the plain kernel, the host's calls, the knobs --------------------------------------------------

@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 8, 80), (8, 2, 512), (5, 1, 33), (40, 2, 128)], ids=str)
def test_the_plain_kernel(state, dims):
    with _env(RETI_RUST_FLASH_SDPA="0"):
        p = Pair(state, dims, 400, seed=3)
        for n in (0, 1, 40, 300):
            p.append(n)
            p.step()
        for ws in (0, 17, 300):
            q = p.rng.standard_normal(p.q_dim, dtype=np.float32)
            p.check(q[None], p.kv.attention_decode_windowed(q, ws)[None], window_start=ws)


KNOBS = [{"SKV_DECODE_WAVES": "4"}, {"SKV_DECODE_WAVES": "8", "SKV_DECODE_WGS": "1024"}, {"SKV_DECODE_WGS": "16"}, {"SKV_DECODE_MIN_PAGES": "4"},
         {"SKV_DECODE_MIN_PAGES": "1"}, {"SKV_FUSED_APPEND": "0"}, {"SKV_Q_VEC": "0"}, {"RETI_RUST_SDPA_2PASS": "0"},
         {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_WGS": "64"}, {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_MAX_SPLITS": "1"}]


@pytest.mark.parametrize("knobs", KNOBS, ids=lambda k: ",".join("%s=%s" % kv for kv in k.items()))
@pytest.mark.parametrize("dims,n,window", [((16, 2, 256), 1500, 0), ((32, 8, 128), 60, 0), ((8, 2, 64), 70, 48)], ids=str)
def test_knobs_choose_among_kernels_never_among_results(state, knobs, dims, n, window):
    with _env(**knobs):
        p = Pair(state, dims, n + 300, seed=n, window=window)
        p.append(n)
        for _ in range(3):
            p.step()
        for rows in (3, 20, 130):
            p.chunk(rows)
            p.step()
        p.check_rows(max(0, p.kv.len() - window) if window else 0)


def test_probes_of_the_pages_run(state):
    for dims, window in (((32, 8, 128), 0), ((16, 2, 256), 100), ((8, 2, 512), 0)):
        p = Pair(state, dims, 1000, seed=5, window=window)
        p.append(900)
        p.step()
        out = torch.zeros(p.q_dim, device="cuda")
        p.kv.encode_probe_read_pages(_stream())
        p.kv.encode_probe_read_store_pages(_stream())
        p.kv.encode_probe_merge(_stream(), out.data_ptr())
        torch.cuda.synchronize()
        p.step()
        p.check_rows(max(0, p.kv.len() - window) if window else 0)


# ---- batches -----------------------------------------------------------------------------

@pytest.mark.parametrize("case", range(12))
def test_batches_of_any_lengths(state, case):
    rng = np.random.default_rng(900 + case)
    kv_heads = int(rng.integers(1, 5))
    dims = (kv_heads * int(rng.integers(1, 9)), kv_heads, int(rng.choice([17, 32, 64, 96, 128, 200, 256, 512])))
    window = int(rng.choice([0, 0, 40, 129]))
    seqs = [Pair(state, dims, 700, seed=100 * case + i, window=window) for i in range(int(rng.integers(1, 17)))]
    for p in seqs:
        p.append(int(rng.choice([0, 1, 15, 16, 31, 100, 333, 600])))
    for _ in range(int(rng.integers(1, 4))):
        new = [p.new(1) for p in seqs]
        dev = [[_dev(a) for a in r] for r in new]
        outs = torch.full((len(seqs), seqs[0].q_dim), float("nan"), device="cuda")
        skv.encode_decode_step_batch([p.kv for p in seqs], _stream(), [d[0].data_ptr() for d in dev], [d[1].data_ptr() for d in dev],
                                     [d[2].data_ptr() for d in dev], [o.data_ptr() for o in outs])
        got = outs.cpu().numpy()
        for p, (k, v, q), o in zip(seqs, new, got):
            p.holds(k, v)
            p.check(q, o[None])
    for p in seqs:
        p.check_rows(max(0, p.kv.len() - window) if window else 0)
        p.kv.close()


# ---- snapshots and caches -----------------------------------------------------------------

def test_snapshots_hold_the_codes(state):
    dims, n = (16, 2, 256), 96
    a = [Pair(state, dims, n, seed=i) for i in range(3)]
    b = [Pair(state, dims, n, seed=10 + i) for i in range(3)]
    for p in a + b:
        p.append(n)
    snap = skv.snapshot_blocks(state, [p.kv for p in a], [1, 2, 4], stream=_stream())
    assert snap.estimated_bytes() == 3 * 3 * 2 * 16 * 512 * 17 // 32
    copy = snap.clone(stream=_stream())
    skv.restore_blocks(state, copy, [p.kv for p in b], [0, 5, 3], stream=_stream())
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        for src, dst in ((1, 0), (2, 5), (4, 3)):
            y.k[dst * 16:dst * 16 + 16] = x.k[src * 16:src * 16 + 16]
            y.v[dst * 16:dst * 16 + 16] = x.v[src * 16:src * 16 + 16]
        y.check_rows()
    # pages of another element do not fit, not even of the same geometry
    for make in (state.full_attention_bf16, state.full_attention_f32):
        others = [make(n, *dims) for _ in range(3)]
        for kv, p in zip(others, a):
            kv.seed(p.k.astype(np.float32), p.v.astype(np.float32), n)
        with pytest.raises(skv.DimensionError):
            skv.restore_blocks(state, snap, others, [1, 2, 4])
        theirs = skv.snapshot_blocks(state, others, [1, 2, 4], stream=_stream())
        with pytest.raises(skv.DimensionError):
            skv.restore_blocks(state, theirs, [p.kv for p in a], [1, 2, 4])
    for p in a:
        p.check_rows()


@pytest.mark.parametrize("window", [0, 40])
def test_caches_of_whole_prompts(state, window):
    dims, n = (8, 2, 64), 77
    rng = np.random.default_rng(1)
    cache = skv.WholePromptCache(state, 2)
    prompt = list(range(n))
    one = [Pair(state, dims, 200, seed=i, window=window) for i in range(2)]
    for p in one:
        p.append(n)
    cache.put(prompt, [p.kv for p in one], stream=_stream())
    other = [Pair(state, dims, 200, seed=20 + i, window=window) for i in range(2)]
    assert cache.lookup(prompt, [p.kv for p in other], stream=_stream()) == n
    torch.cuda.synchronize()
    for x, y in zip(one, other):
        y.k, y.v = x.k.copy(), x.v.copy()
        y.check_rows(max(0, n - window) if window else 0)
        y.step()
        y.chunk(20)


def test_the_hot_cache_restores_blocks(state):
    dims, n, bt = (8, 2, 64), 64, 16
    tokens = list(range(1000, 1000 + n))
    layers = [Pair(state, dims, 128, seed=i) for i in range(2)]
    for p in layers:
        p.append(n)
    kvs = [p.kv for p in layers]
    hot = skv.HotCache(state, bt, 8, 8, kvs)
    assert hot.block_bytes() == 2 * 2 * bt * 128 * 17 // 32
    session = skv.BlockHash.root()
    h, hashes = session, []
    for i in range(0, n, bt):
        h = skv.BlockHash.chain(h, tokens[i:i + bt])
        hashes.append(h)
    hot.remember_prefix_blocks(session, hashes, bt, kvs, stream=_stream())
    fresh = [Pair(state, dims, 128, seed=30 + i) for i in range(2)]
    reused, _ = hot.match_restore(session, tokens + [1], [p.kv for p in fresh], stream=_stream())
    torch.cuda.synchronize()
    assert reused == n
    for x, y in zip(layers, fresh):
        y.k, y.v = x.k.copy(), x.v.copy()
        y.check_rows()
        y.step()
    bf = [state.full_attention_bf16(128, *dims) for _ in range(2)]
    with pytest.raises(skv.DimensionError):
        hot.match_restore(session, tokens + [1], bf, stream=_stream())


# ---- streams, sizes, refusals ---------------------------------------------------------------

def test_two_streams_at_once(state):
    dims = (16, 2, 256)
    streams = [torch.cuda.Stream() for _ in range(2)]
    pairs = [Pair(state, dims, 3000, seed=40 + i) for i in range(2)]
    for p in pairs:
        p.append(2500)
    new = [[p.new(40) for _ in range(4)] + [p.new(1) for _ in range(20)] for p in pairs]
    dev = [[[_dev(a) for a in r] for r in rows] for rows in new]
    outs = [[torch.full(r[2].shape, float("nan"), device="cuda") for r in rows] for rows in new]
    torch.cuda.synchronize()
    for i in range(24):
        for s, p, rows, o in zip(streams, pairs, dev, outs):
            k, v, q = rows[i]
            if len(q) > 1:
                p.kv.encode_prefill_rows(s.cuda_stream, q.data_ptr(), k.data_ptr(), v.data_ptr(), len(q), o[i].data_ptr())
            else:
                p.kv.encode_decode_step(s.cuda_stream, k.data_ptr(), 0, v.data_ptr(), 0, q.data_ptr(), o[i].data_ptr())
    torch.cuda.synchronize()
    for p, rows, o in zip(pairs, new, outs):
        for (k, v, q), out in zip(rows, o):
            p.holds(k, v)
            p.check(q, out.cpu().numpy())
        p.check_rows()


def test_pools_beyond_four_gib(state):
    """Pages at the far end of pools of 4.6 GB each: byte offsets that 32 bits do not hold."""
    dims, capacity = (8, 8, 512), 2_100_000
    kv = state.full_attention_fp4(capacity, *dims)
    assert kv.pages() * 16 * 8 * 512 * 17 // 32 > 2 ** 32
    kv.set_block_table(np.arange(kv.pages(), dtype=np.int32)[::-1].copy())
    p = Pair.__new__(Pair)
    p.rng, p.dims, p.window, p.kv, p.kv_dim, p.q_dim = np.random.default_rng(2), dims, 0, kv, 4096, 4096
    p.k, p.v = np.empty((0, 4096)), np.empty((0, 4096))
    p.append(45)
    p.step()
    p.chunk(5)
    with _env(SKV_PREFILL_TILES="2"):
        p.chunk(70)
    with _env(RETI_RUST_FLASH_SDPA="0"):
        p.step()
    p.check_rows()
    kv.close()


def test_refusals(state):
    kv = state.full_attention_fp4(64, 8, 2, 64)
    bf = state.full_attention_bf16(64, 8, 2, 64)
    x = torch.zeros(64 * 512, device="cuda")
    at = x.data_ptr()
    with pytest.raises(skv.DimensionError):
        kv.encode_append_batch(_stream(), at, at, 65)
    with pytest.raises(skv.DimensionError):
        kv.encode_prefill_rows(_stream(), at, at, at, 65, at)
    with pytest.raises(skv.DimensionError):
        kv.encode_gather(_stream(), 0, 1, at, at)  # no rows yet
    with pytest.raises(skv.KvError):
        skv.encode_decode_step_batch([kv, bf], _stream(), [at] * 2, [at] * 2, [at] * 2, [at] * 2)  # two elements
    with pytest.raises(skv.ConfigError):
        state.full_attention_with_element(64, 8, 2, 64, 3)
    with pytest.raises(skv.ConfigError):
        state.full_attention_fp4(64, 8, 2, 513)
    assert kv.len() == 0 and bf.len() == 0
    kv.append_row(np.ones(128, np.float32), np.ones(128, np.float32))
    with pytest.raises(skv.DimensionError):
        kv.attention_decode_windowed(np.ones(512, np.float32), 1)  # nothing left to attend
    assert kv.len() == 1


# ---- together -----------------------------------------------------------------------------

def test_a_sequence_from_its_prompt_to_its_snapshot(state):
    """Four layers, two of them with a window: a prompt in chunks, tokens one at a time, drafts of six verified and rolled back, the rows
    read back, and the sequence taken up again from a cache of prompts."""
    dims, windows = (8, 2, 128), (0, 64, 0, 64)
    layers = [Pair(state, dims, 600, seed=60 + i, window=w) for i, w in enumerate(windows)]
    for n in (100, 100, 37):
        for p in layers:
            p.chunk(n)
    for token in range(12):
        for p in layers:
            p.step()
        if token % 4 == 3:
            for p in layers:
                n = p.kv.len()
                p.chunk(6)
                p.truncate(n + 2)
    n = layers[0].kv.len()
    for p, w in zip(layers, windows):
        assert p.kv.len() == n
        p.check_rows(max(0, n - w) if w else 0)
    cache = skv.WholePromptCache(state, 1)
    cache.put(list(range(n)), [p.kv for p in layers], stream=_stream())
    again = [Pair(state, dims, 600, seed=70 + i, window=w) for i, w in enumerate(windows)]
    assert cache.lookup(list(range(n)), [p.kv for p in again], stream=_stream()) == n
    torch.cuda.synchronize()
    for x, y in zip(layers, again):
        y.k, y.v = x.k, x.v
        y.step()
        y.chunk(9)
