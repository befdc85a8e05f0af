"""The 4-bit element's softmax where its base and its weights' steps show: scores so large that a step of 32 bits is 8 and more, and many
keys far below one."""
import contextlib
import os

import numpy as np
import pytest

import saragossa_amd as skv

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


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


def _step(kv, k, v, q):
    kd, vd, qd, out = _dev(k), _dev(v), _dev(q), torch.zeros(q.size, device="cuda")
    kv.encode_decode_step(_stream(), kd.data_ptr(), 0, vd.data_ptr(), 0, qd.data_ptr(), out.data_ptr())
    return out.cpu().numpy().reshape(1, -1)


def _projections(kv, k, v, q):
    kd, vd, qd, out = _dev(k), _dev(v), _dev(q), torch.zeros(q.size, device="cuda")
    kv.encode_decode_step_prekv(_stream(), None, 0, qd.data_ptr(), 0, kd.data_ptr(), 0, vd.data_ptr(), 0, None, None, 1e-6, float(kv.head_dim()), out.data_ptr())
    return out.cpu().numpy().reshape(1, -1)


def _chunk(kv, k, v, q):
    return kv.prefill_rows(q, k, v).reshape(len(q), -1)


# how the last rows are attended: their number, the call, the environment
CALLS = {"step": (1, _step, {}), "whole step": (1, _step, {"RETI_RUST_SDPA_2PASS": "0"}), "from the projections": (1, _projections, {}), "few rows": (6, _chunk, {}),
         "streaming chunk": (70, _chunk, {"SKV_PREFILL_TILES": "0"}), "chunk kernel": (70, _chunk, {"SKV_PREFILL_TILES": "2"})}


def _layer_of(state, rng, dims, n, window):
    kv = state.full_attention_fp4(n, *dims, window=window)
    kv.set_block_table(rng.permutation(kv.pages()).astype(np.int32))
    return kv


def _ties(rng, dims, n, m, sign, octave):
    """n rows whose keys have one dim that is not zero, 2^(octave - 7) or half of that, and m queries of one dim that is not zero, so that a score in
    base 2 is exact in 32 bits and lies in [2^octave, 2^(octave + 1)), or is half of one that does: keys of the same size tie, the others are 2^(octave - 1)
    away. The rows' keys and values, the queries, and a mask [n] of the larger keys."""
    heads, kv_heads, hd = dims
    large = rng.random(n) < 0.5
    k = np.zeros((n, kv_heads, hd), np.float32)
    k[:, :, 3] = np.where(large, 2.0, 1.0)[:, None] * 2.0 ** (octave - 8)
    v = np.sign(rng.standard_normal((n, kv_heads, hd))) * rng.choice([1.0, 2.0, 4.0], (n, kv_heads, hd))
    q = np.zeros((m, heads, hd), np.float32)
    qscale = np.float32(np.float32(1.0) / np.sqrt(np.float32(hd))) * np.float32(1.4426950408889634)
    q[:, :, 3] = sign * np.exp2(7.1 + 0.8 * rng.random((m, heads))) / qscale
    if octave == 27:  # (steps of 16: about half of the largest scores are odd multiples)
        s = np.abs(q[:, :, 3] * qscale).astype(np.float64) * 2.0 ** 20
        assert (s / 16 % 2 == 1).any()
    return k.reshape(n, -1), v.astype(np.float32).reshape(n, -1), q.reshape(m, -1), large


def _mean_of_ties(dims, v, large, m, sign, window):
    """The contexts of the last m rows: the mean over the keys of the largest score that a row sees, and how far sums of that many values in 32 bits
    may be off in any order, a quotient and the joining of partials with them: half a step of the sum of magnitudes each."""
    heads, kv_heads, hd = dims
    n = len(v)
    vv = np.repeat(v.astype(np.float64).reshape(n, kv_heads, hd), heads // kv_heads, 1)
    want, tol = np.empty((m, heads, hd)), np.empty((m, heads, hd))
    for i in range(m):
        hi = n - m + i + 1
        lo = max(0, hi - window) if window else 0
        top = large[lo:hi] if sign > 0 else ~large[lo:hi]
        keys = vv[lo:hi][top if top.any() else ~top]
        want[i] = keys.mean(0)
        tol[i] = (len(keys) + 40) * 2.0 ** -24 * np.abs(keys).mean(0)
    return want.reshape(m, -1), tol.reshape(m, -1)


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512)], ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("octave,window", [(26, 0), (27, 0), (27, 100), (40, 100)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size_have_finite_weights(state, dims, call, octave, sign, window):
    m, run, env = CALLS[call]
    rng = np.random.default_rng(octave + dims[2])
    n = 333
    k, v, q, large = _ties(rng, dims, n, m, sign, octave)
    want, tol = _mean_of_ties(dims, v, large, m, sign, window)
    kv = _layer_of(state, rng, dims, n, window)
    kv.seed(k[:n - m], v[:n - m], n - m)
    with _env(**env):
        got = run(kv, k[n - m:], v[n - m:], q)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.abs((got - want) / tol).max()
    kv.close()


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512)], ids=str)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size_in_batches(state, dims, sign):
    rng = np.random.default_rng(dims[2])
    seqs = []
    for n in (1, 17, 200, 333, 900):
        k, v, q, large = _ties(rng, dims, n, 1, sign, 27)
        kv = _layer_of(state, rng, dims, n, 0)
        if n > 1:
            kv.seed(k[:-1], v[:-1], n - 1)
        seqs.append((kv, _dev(k[-1]), _dev(v[-1]), _dev(q), torch.zeros(q.size, device="cuda"), _mean_of_ties(dims, v, large, 1, sign, 0)))
    at = [[s[i].data_ptr() for s in seqs] for i in range(1, 5)]
    skv.encode_decode_step_batch([s[0] for s in seqs], _stream(), *at)
    for kv, _, _, _, out, (want, tol) in seqs:
        got = out.cpu().numpy()[None]
        assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()
        kv.close()


# The kernels of chunks of many rows
SHAPES = {"halves": {"SKV_PREFILL_TILES": "2"}, "one tile": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "1000000"},
          "two tiles": {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_TILES2_MIN_PAGES": "0"}, "streaming": {"SKV_PREFILL_TILES": "0"}}


@pytest.mark.parametrize("dims", [(8, 2, 64), (8, 1, 128), (4, 1, 256), (4, 1, 512)], ids=str)
@pytest.mark.parametrize("shape", SHAPES)
def test_many_far_keys_behind_one_large_one_are_counted(state, dims, shape):
    """Row 0 has a score of 29.5 (in base 2) and values of 0, 12 rows of each page a score of 0 and values of 1, the rest no weight to speak of: the
    context is what the 12 rows' weights, 2^-29.5 each of the largest, are together, 3.2e-5.

    Weights are in steps of 2^-24, the largest is 2^7 or more: each may be off by 2^-32 of the largest. Beside that by 2^-22 of itself, the
    exponential by 2^-22, the score of 29.5 by its four roundings of 2^-24, which is 5e-6 of the weights' ratio, and sums of 2052 sums by half a step of 2^-24
    each: 1.3e-4 of the context together."""
    heads, kv_heads, hd = dims
    n, m = 32768, 64
    rng = np.random.default_rng(hd)
    k = np.zeros((n + m, kv_heads, hd), np.float32)
    row = np.arange(n + m) % 16
    k[row < 4, :, 3] = -1.0
    k[0, :, 3] = 1.0
    v = np.ones((n + m, kv_heads * hd), np.float32)
    v[0] = 0
    q = np.zeros((m, heads, hd), np.float32)
    q[:, :, 3] = 29.5 * np.sqrt(hd) / 1.4426950408889634
    kv = _layer_of(state, rng, dims, n + m, 0)
    k = k.reshape(n + m, -1)
    for i in range(0, n, 8192):
        kd, vd = _dev(k[i:i + 8192]), _dev(v[i:i + 8192])
        kv.encode_append_batch(_stream(), kd.data_ptr(), vd.data_ptr(), 8192)
        torch.cuda.synchronize()
    with _env(SKV_PREFILL_MAX_SPLITS="1", **SHAPES[shape]):
        got = _chunk(kv, k[n:], v[n:], q.reshape(m, -1))
    for i in range(m):
        far = (row[:n + i + 1] >= 4).sum() * 2.0 ** -29.5
        want = far / (1 + far)
        assert np.abs(got[i] - want).max() <= (row[:n + i + 1] >= 4).sum() * 2.0 ** -32 + 1.4e-4 * want, i
    kv.close()


@pytest.mark.parametrize("dims", [(32, 8, 128), (16, 2, 256), (8, 2, 64), (8, 2, 512)], ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("power", [0, 60, -60])
def test_weights_are_as_exact_for_values_that_half_precision_does_not_have(state, dims, call, power):
    """Two rows have weights to speak of, and the one of less weight values: a context is that row's weight times its values, which are 2^power times
    small ones. (The largest weight is a power of two, whose terms are exact.)

    Relative to itself it may be off by the score's four roundings (2 * 4 * 2^-24 of 1 / log2(e) at most), an exponential either way, 2^-22
    each, the weight as terms, 2^-22, and the sum, the quotient and the products' sums, 6 * 2^-24. Streaming chunks of heads up to 128 dims hold a
    weight in two terms of bf16 against such values: a rest of 2^-8 at most whose step is 2^-16, 2^-17."""
    m, run, env = CALLS[call]
    heads, kv_heads, hd = dims
    n = 200
    rng = np.random.default_rng(hd)
    k = np.zeros((n, kv_heads, hd), np.float32)
    k[:, :, 5] = -64.0  # no weight
    k[0, :, 5], k[1, :, 5] = 1.0, 0.0
    v = np.zeros((n, kv_heads, hd), np.float32)
    v[1] = rng.choice([-6.0, -2.0, 1.0, 3.0, 4.0, 6.0], (kv_heads, hd)) * 2.0 ** power
    q = np.zeros((m, heads, hd), np.float32)
    q[:, :, 5] = rng.uniform(0.8, 2.0, (m, heads)) * np.sqrt(hd) / 1.4426950408889634
    k, v2, q = k.reshape(n, -1), v.reshape(n, -1), q.reshape(m, -1)
    kv = _layer_of(state, rng, dims, n, 0)
    kv.seed(k[:n - m], v2[:n - m], n - m)
    with _env(**env):
        got = run(kv, k[n - m:], v2[n - m:], q)
    weight = 1.0 / (1.0 + np.exp(q.reshape(m, heads, hd)[:, :, 5].astype(np.float64) / np.sqrt(hd)))
    want = (weight[:, :, None] * np.repeat(v[1].astype(np.float64), heads // kv_heads, 0)[None]).reshape(m, -1)
    tol = 2 * 4 * 2.0 ** -24 * 0.7 + 3 * 2.0 ** -22 + 6 * 2.0 ** -24
    if power and call == "streaming chunk" and hd <= 128:
        tol += 2.0 ** -17
    else:
        assert tol < 1.5e-6
    assert (np.abs(got / want - 1.0) <= tol).all(), np.abs(got / want - 1.0).max()
    kv.close()
