"""The mark of an eviction goes with the rows: whatever way evicted rows come back into a layer, they are no prompt's."""
import numpy as np
import pytest

import saragossa_amd as skv

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

GEO, DIM = (8, 2, 64), 128


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _append(kv, n, stream=None):
    k = torch.randn(n, DIM, device="cuda")
    kv.encode_append_batch(_stream() if stream is None else stream, k.data_ptr(), k.data_ptr(), n)
    torch.cuda.synchronize()


def _layer(state, rows=64, capacity=128):
    kv = state.full_attention_bf16(capacity, *GEO)
    _append(kv, rows)
    return kv, torch.rand(2, capacity, device="cuda")


def _evict(kv, w, keep):
    kv.encode_evict(_stream(), w.data_ptr(), keep, 0, 0)


def _remember(state, kv):
    hot = skv.HotCache(state, 16, 8, 8, [kv])
    root = skv.BlockHash.for_session("s")
    hot.remember_prefix_block(root, root, 16, [kv], stream=_stream())
    skv.WholePromptCache(state, 2).put(range(kv.len()), [kv], [], [], _stream())


def _refused(state, kv):
    assert kv.evicted_rows() > 0
    hot = skv.HotCache(state, 16, 8, 8, [kv])
    root = skv.BlockHash.for_session("s")
    with pytest.raises(skv.ConfigError):
        hot.remember_prefix_block(root, root, 16, [kv], stream=_stream())
    with pytest.raises(skv.ConfigError):
        skv.WholePromptCache(state, 2).put(range(kv.len()), [kv], [], [], _stream())


@pytest.mark.parametrize("clone", [False, True])
@pytest.mark.parametrize("fresh", [False, True])
def test_a_snapshot_brings_the_mark_along(state, fresh, clone):
    kv, w = _layer(state)
    _evict(kv, w, 40)
    shot = skv.snapshot_blocks(state, [kv], [0, 1, 2], _stream())
    if clone:
        shot = shot.clone(_stream())
    to = state.full_attention_bf16(128, *GEO) if fresh else kv
    to.truncate(0)
    assert to.evicted_rows() == 0
    skv.restore_blocks(state, shot, [to], [0, 1, 2], _stream())
    to.truncate(40)
    _refused(state, to)
    assert to.evicted_rows() == 40
    with pytest.raises(skv.DimensionError):
        to.truncate(39)
    to.truncate(0)
    _append(to, 64)
    _remember(state, to)


def test_only_the_blocks_in_front_of_it_are_an_eviction_s(state):
    kv, w = _layer(state)
    _evict(kv, w, 20)
    _append(kv, 44)
    shot = skv.snapshot_blocks(state, [kv], [1, 2, 3], _stream())  # rows 16 .. 63, of which 16 .. 19 have been evicted to
    to = state.full_attention_bf16(128, *GEO)
    _append(to, 16)
    skv.restore_blocks(state, shot, [to], [4, 1, 2], _stream())
    to.truncate(48)
    assert to.evicted_rows() == 0  # the evicted block lies behind these
    _remember(state, to)
    to.truncate(80)
    assert to.evicted_rows() == 80
    _refused(state, to)


def test_a_block_restored_into_rows_in_use(state):
    kv, w = _layer(state)
    _evict(kv, w, 30)
    shot = skv.snapshot_blocks(state, [kv], [1], _stream())
    to, _ = _layer(state, 60)
    skv.restore_blocks(state, shot, [to], [2], _stream())
    assert to.evicted_rows() == 48
    _refused(state, to)


def test_rows_that_come_back_without_a_restore(state):
    kv, w = _layer(state)
    _evict(kv, w, 40)
    kv.truncate(0)
    kv.truncate(40)
    _refused(state, kv)
    kv.truncate(0)
    _append(kv, 20)
    kv.truncate(20)
    _remember(state, kv)   # written anew
    kv.truncate(40)        # and 20 .. 39, which were not
    _refused(state, kv)
    kv.seed(np.zeros((3, DIM), np.float32), np.zeros((3, DIM), np.float32), 3)
    kv.truncate(2)
    assert kv.evicted_rows() == 0
    kv.truncate(20)
    _refused(state, kv)


def test_a_layer_written_anew_is_a_prompt_s_again(state):
    kv, w = _layer(state)
    clean = skv.snapshot_blocks(state, [kv], [0, 1, 2, 3], _stream())
    _evict(kv, w, 40)
    kv.truncate(0)
    skv.restore_blocks(state, clean, [kv], [0, 1, 2, 3], _stream())
    kv.truncate(64)
    assert kv.evicted_rows() == 0
    _remember(state, kv)
    _evict(kv, w, 40)
    kv.truncate(0)
    _append(kv, 64)
    kv.truncate(10)
    kv.truncate(64)  # a draft's length, there and back
    _remember(state, kv)
    _evict(kv, w, 10)
    prompts = skv.WholePromptCache(state, 2)
    other, _ = _layer(state, 50)
    prompts.put(range(50), [other], [], [], _stream())
    assert prompts.get(range(50), [kv], lambda first, last: None, [], [], _stream()) == 50
    kv.truncate(50)
    _remember(state, kv)


@pytest.mark.parametrize("steady", [False, True])
def test_a_replayed_eviction(state, steady):
    """Recorded once; the host says after each replay what length it left, also where that is the length already."""
    kv, w = _layer(state, 40 if steady else 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    k = torch.randn(64, DIM, device="cuda")

    def pass_of():
        if steady:
            kv.encode_append_batch(side.cuda_stream, k.data_ptr(), k.data_ptr(), 1)
        kv.encode_evict(side.cuda_stream, w.data_ptr(), 40, 2, 3)
    with torch.cuda.stream(side):
        pass_of()
        kv.truncate(0)
        _append(kv, 40 if steady else 64, side.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            pass_of()
        for _ in range(3):
            kv.truncate(0)
            assert kv.evicted_rows() == 0
            _append(kv, 40 if steady else 64, side.cuda_stream)
            side.synchronize()
            graph.replay()
            side.synchronize()
            kv.truncate(40)
            _refused(state, kv)
            with pytest.raises(skv.DimensionError):
                kv.truncate(39)


def test_a_new_block_table_takes_the_mark_along(state):
    kv, w = _layer(state)
    _evict(kv, w, 20)  # pages 0 and 1 of eight
    kv.truncate(0)
    kv.set_block_table(np.array([2, 3, 4, 5, 6, 1, 7, 0], np.int32))
    kv.truncate(80)
    assert kv.evicted_rows() == 0
    kv.truncate(96)
    assert kv.evicted_rows() == 96
    _refused(state, kv)
