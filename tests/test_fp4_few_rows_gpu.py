"""Chunks of up to 16 rows on full 4-bit layers that have 64 query slots to a kv head: by size and by SKV_PREFILL_TILES they take the streaming launch, which
stores their rows itself, or a store and the chunk kernel."""
import contextlib
import os

import numpy as np
import pytest

import saragossa_amd as skv
from test_fp4_kv_gpu import Pair, _dev, _rows, _stream

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


@pytest.mark.parametrize("dims,rows", [((32, 8, 128), 16), ((16, 1, 128), 4), ((16, 1, 256), 7), ((8, 2, 512), 16), ((8, 1, 64), 11), ((40, 2, 96), 5)], ids=str)
def test_the_knob_holds_for_few_rows(state, dims, rows):
    """With SKV_PREFILL_TILES=2 they take the chunk kernel, bit for bit as where the store is a launch apart; with 0 the streaming one, which
    rounds elsewhere; the rows stored are the same."""
    kv_dim, q_dim, base = dims[1] * dims[2], dims[0] * dims[2], 700
    rng = np.random.default_rng(rows)
    k, v, q = _rows(rng, base + rows, kv_dim), _rows(rng, base + rows, kv_dim), rng.standard_normal((rows, q_dim), dtype=np.float32)
    table = None

    def run(**env):
        nonlocal table
        kv = state.full_attention_fp4(base + rows, *dims)
        table = rng.permutation(kv.pages()).astype(np.int32) if table is None else table
        kv.set_block_table(table)
        kv.seed(k[:base], v[:base], base)
        qd, kd, vd, out = _dev(q), _dev(k[base:]), _dev(v[base:]), torch.zeros(rows, q_dim, device="cuda")
        with _env(**env):
            kv.encode_prefill_rows(_stream(), qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), rows, out.data_ptr())
        result = out.cpu().numpy(), *kv.read_rows_f32()
        kv.close()
        return result

    tiles, apart, streamed = run(SKV_PREFILL_TILES="2"), run(SKV_PREFILL_TILES="2", SKV_FUSED_APPEND="0"), run(SKV_PREFILL_TILES="0")
    assert np.array_equal(tiles[0], apart[0]) and not np.array_equal(tiles[0], streamed[0])
    for other in (apart, streamed):
        assert np.array_equal(tiles[1], other[1]) and np.array_equal(tiles[2], other[2])


@pytest.mark.parametrize("dims,rows,base", [((16, 1, 128), 16, 51000), ((16, 1, 128), 16, 53000), ((8, 1, 512), 16, 33000)], ids=str)
def test_few_rows_over_long_contexts(state, dims, rows, base):
    """On both sides of the line in (16 slots, page) pairs, and a step behind them."""
    p = Pair(state, dims, base + rows + 2, seed=base)
    p.append(base)
    p.chunk(rows)
    p.step()
    p.check_rows(base - 20)


def test_captured_few_rows_over_a_long_context():
    dims, rows, base = (16, 1, 128), 16, 60000
    ctx = skv.DecodeResidentState(0)
    rng = np.random.default_rng(1)
    kv = ctx.full_attention_fp4(base + rows, *dims)
    side = torch.cuda.Stream()
    old = [_dev(_rows(rng, base, 128)) for _ in range(2)]
    k, v, q = _dev(_rows(rng, rows, 128)), _dev(_rows(rng, rows, 128)), _dev(rng.standard_normal((rows, 2048), dtype=np.float32))
    out = torch.zeros(rows, 2048, device="cuda")
    torch.cuda.synchronize()

    def refill():
        kv.truncate(0)
        kv.encode_append_batch(side.cuda_stream, old[0].data_ptr(), old[1].data_ptr(), base)

    def run():
        kv.encode_prefill_rows(side.cuda_stream, q.data_ptr(), k.data_ptr(), v.data_ptr(), rows, out.data_ptr())

    with torch.cuda.stream(side):
        refill()
        run()
        side.synchronize()
        want = out.clone()
        refill()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        for replay in range(3):
            refill()
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want), replay
        refill()
        run()
        side.synchronize()
        assert torch.equal(out, want)
