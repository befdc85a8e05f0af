"""skv_gather_device: rows of any head, from and to any place, one of K and V alone, and nothing written beside them."""
import numpy as np
import pytest

import saragossa_amd as skv

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("geo", [(2, 2, 1), (3, 3, 5), (4, 4, 18), (2, 1, 33), (8, 8, 84), (6, 3, 99), (6, 3, 100), (2, 2, 131), (2, 1, 509), (8, 2, 512)])
@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_rows_go_out_as_they_are(state, element, geo):
    rows, width = 70, geo[1] * geo[2]
    dtype = torch.float32 if element == "f32" else torch.bfloat16
    kv = state.full_attention_with_element(rows, *geo, {"bf16": skv.DTYPE_BF16, "f32": skv.DTYPE_F32}[element])
    kv.set_block_table(np.random.default_rng(width).permutation(kv.pages()).astype(np.int32))
    gen = torch.Generator(device="cuda").manual_seed(width)
    held = [torch.randn(rows, width, device="cuda", generator=gen) for _ in range(2)]
    stream = torch.cuda.current_stream().cuda_stream
    kv.encode_append_batch(stream, held[0].data_ptr(), held[1].data_ptr(), rows)
    held = [x.to(dtype) for x in held]
    for first, n, shift in ((0, 70, 0), (0, 1, 1), (69, 1, 3), (3, 64, 2), (17, 30, 5), (15, 2, 7)):
        for which in ((True, True), (True, False), (False, True)):
            out = [torch.full((8 + n * width + 8,), 7.0, device="cuda", dtype=dtype) for _ in range(2)]
            at = [x.data_ptr() + shift * x.element_size() if want else None for x, want in zip(out, which)]
            kv.encode_gather(stream, first, n, *at)
            for x, rows_of, want in zip(out, held, which):
                assert (x[:shift] == 7.0).all() and (x[shift + n * width:] == 7.0).all()
                if want:
                    assert torch.equal(x[shift:shift + n * width], rows_of[first:first + n].flatten())
                else:
                    assert (x == 7.0).all()
