"""A 4-bit layer of more than 2^28 rows: 2^24 pages among 256 and more splits, a product that 32 bits do not hold."""
import os

import numpy as np
import pytest

import saragossa_amd as skv

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BLOCK, BLOCKS, MORE = 1 << 20, 256, 100


def _stream():
    return torch.cuda.current_stream().cuda_stream


def test_every_row_of_a_long_cache_is_attended_once(state):
    """Keys of zeros, so that a context is the mean of the values: blocks of 2^20 equal rows. Weights are equal and powers of two, and the values
    multiples of a half, so that sums are exact until the 512 partials or fewer are joined, each a rounding of half a step."""
    dims = (4, 1, 32)
    rng = np.random.default_rng(0)
    kv = state.full_attention_fp4(BLOCK * BLOCKS + MORE, *dims)
    assert kv.pages() * 256 > 1 << 32
    levels = np.array([0.5, 1, 1.5, 2, 3, 4, 6])
    blocks = rng.choice(np.concatenate([levels, -levels]), (BLOCKS, 32))
    zeros = torch.zeros(BLOCK, 32, device="cuda")
    total = np.zeros(32)
    for block in blocks:
        rows = torch.from_numpy(block.astype(np.float32)).cuda().expand(BLOCK, 32).contiguous()
        kv.encode_append_batch(_stream(), zeros.data_ptr(), rows.data_ptr(), BLOCK)
        torch.cuda.synchronize()
        total += block * BLOCK
    size = np.abs(blocks).mean(0)
    n = BLOCK * BLOCKS

    def attended(rows, env):
        nonlocal total, n
        saved = {k: os.environ.get(k) for k in env}
        os.environ.update(env)
        skv.flags.reload()
        v = rng.choice(levels, (rows, 32))
        vd = torch.from_numpy(v.astype(np.float32)).cuda()
        q = torch.from_numpy(rng.standard_normal((rows, 128)).astype(np.float32)).cuda()
        out = torch.zeros(rows, 128, device="cuda")
        if rows == 1:
            kv.encode_decode_step(_stream(), zeros.data_ptr(), 0, vd.data_ptr(), 0, q.data_ptr(), out.data_ptr())
        else:
            kv.encode_prefill_rows(_stream(), q.data_ptr(), zeros.data_ptr(), vd.data_ptr(), rows, out.data_ptr())
        got = out.cpu().numpy().reshape(rows, 4, 32)
        for k, was in saved.items():
            os.environ.pop(k) if was is None else os.environ.__setitem__(k, was)
        skv.flags.reload()
        for i in range(rows):
            total = total + v[i]
            n += 1
            assert (np.abs(got[i] - total / n) <= 600 * 2.0 ** -24 * size).all(), (rows, i)

    attended(1, {})
    attended(6, {})
    attended(70, {"SKV_PREFILL_TILES": "0"})
    attended(20, {"SKV_PREFILL_TILES": "2", "SKV_PREFILL_WGS": "4096"})
    kv.close()
