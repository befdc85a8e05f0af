"""More than 256 splits of a context, and more than 512, which the knobs of the launches allow: every one is merged."""
import contextlib
import os

import numpy as np
import pytest

import saragossa_amd as skv

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DIMS, ROWS = (4, 1, 32), 140000
MAKE = {"bf16": skv.DTYPE_BF16, "f32": skv.DTYPE_F32, "fp4": skv.DTYPE_FP4}


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


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _filled(state, element, more):
    """Keys of zeros, so that a context is the mean of the values: 1 in the first half of the rows, 3 in the others, every sum of which is exact."""
    kv = state.full_attention_with_element(ROWS + more, *DIMS, MAKE[element], 0)
    k = torch.zeros(ROWS, 32, device="cuda")
    v = torch.ones(ROWS, 32, device="cuda")
    v[ROWS // 2:] = 3.0
    kv.encode_append_batch(_stream(), k.data_ptr(), v.data_ptr(), ROWS)
    torch.cuda.synchronize()
    return kv


def _mean(extra):
    return (ROWS // 2 + 3 * (ROWS - ROWS // 2 + extra)) / (ROWS + extra)


TOL = 600 * 2.0 ** -24 * 3  # partials joined, a rounding each


@pytest.mark.parametrize("element", MAKE)
@pytest.mark.parametrize("wgs", ["256", "300", "100000"])
def test_steps_and_batches(state, element, wgs):
    with _env(SKV_DECODE_WGS=wgs, SKV_DECODE_MIN_PAGES="1"):
        seqs = [_filled(state, element, 2) for _ in range(2)]
        x = torch.full((32,), 3.0, device="cuda")
        q = torch.randn(128, device="cuda")
        outs = [torch.zeros(128, device="cuda") for _ in seqs]
        zero = torch.zeros(32, device="cuda")
        for kv, out in zip(seqs, outs):
            kv.encode_decode_step(_stream(), zero.data_ptr(), 0, x.data_ptr(), 0, q.data_ptr(), out.data_ptr())
            assert np.abs(out.cpu().numpy() - _mean(1)).max() <= TOL
        with _env(SKV_DECODE_WGS=str(2 * int(wgs))):
            skv.encode_decode_step_batch(seqs, _stream(), [zero.data_ptr()] * 2, [x.data_ptr()] * 2, [q.data_ptr()] * 2, [o.data_ptr() for o in outs])
        for kv, out in zip(seqs, outs):
            assert np.abs(out.cpu().numpy() - _mean(2)).max() <= TOL
            kv.close()


@pytest.mark.parametrize("element", MAKE)
@pytest.mark.parametrize("tiles", ["0", "2"])
@pytest.mark.parametrize("splits", ["300", "1000000"])
@pytest.mark.parametrize("rows", [6, 40])
def test_chunks(state, element, tiles, splits, rows):
    with _env(SKV_DECODE_WGS="100000", SKV_DECODE_MIN_PAGES="1", SKV_PREFILL_WGS="1000000", SKV_PREFILL_MAX_SPLITS=splits, SKV_PREFILL_TILES=tiles):
        kv = _filled(state, element, rows)
        x, zero = torch.full((rows, 32), 3.0, device="cuda"), torch.zeros(rows, 32, device="cuda")
        q = torch.randn(rows, 128, device="cuda")
        out = torch.zeros(rows, 128, device="cuda")
        kv.encode_prefill_rows(_stream(), q.data_ptr(), zero.data_ptr(), x.data_ptr(), rows, out.data_ptr())
        got = out.cpu().numpy()
        for i in range(rows):
            assert np.abs(got[i] - _mean(i + 1)).max() <= TOL, i
        kv.close()
