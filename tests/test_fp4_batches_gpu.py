"""Batches of 4-bit decode steps: all contexts stay whole, or none does that can be split."""
import contextlib
import os

import numpy as np
import pytest

import saragossa_amd as skv
from test_fp4_kv_gpu import Pair, _dev, _stream

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


@pytest.mark.parametrize("dims,rows", [((32, 8, 128), (500, 500, 500, 2000)), ((32, 8, 128), (250, 90, 250, 1000)), ((8, 2, 64), (600,) * 7 + (4000,)),
                                       ((16, 2, 256), (300, 10, 300, 4000))], ids=str)
def test_one_split_context_splits_them_all(state, dims, rows):
    """The threshold of splits at its default value, given, leaves none whole for longer: a batch with one split context has the same bits. One of
    short contexts alone has those of unsplit ones."""
    seqs = [Pair(state, dims, n + 1, seed=i) for i, n in enumerate(rows)]
    new = [p.new(1) for p in seqs]
    for p, n in zip(seqs, rows):
        p.append(n)
    dev = [[_dev(a) for a in r] for r in new]

    def run(count, **env):
        outs = [torch.zeros(p.q_dim, device="cuda") for p in seqs]
        with _env(**env):
            skv.encode_decode_step_batch([p.kv for p in seqs[:count]], _stream(), *[[d[i].data_ptr() for d in dev[:count]] for i in range(3)],
                                         [o.data_ptr() for o in outs[:count]])
        torch.cuda.synchronize()
        for p, n in zip(seqs[:count], rows):
            p.kv.truncate(n)
        return [o.cpu().numpy() for o in outs[:count]]

    mixed, split = run(len(rows)), run(len(rows), RETI_RUST_SDPA_2PASS_MIN_LEN="128")
    assert all(np.array_equal(a, b) for a, b in zip(mixed, split))
    short, whole = run(len(rows) - 1), run(len(rows) - 1, RETI_RUST_SDPA_2PASS="0")
    assert all(np.array_equal(a, b) for a, b in zip(short, whole))
    for p, (k, v, q), out in zip(seqs, new, mixed):
        p.holds(k, v)
        p.check(q, out[None])
        p.kv.close()
