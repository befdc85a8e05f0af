"""skv_attention_weights_device over rows and queries whose scores or operands would not fit its scratch: taken in parts, as exactly as ever."""
import math

import pytest

import saragossa_amd as skv

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("n,gqa", [(64, 1), (8, 8)])
@pytest.mark.parametrize("element", ["bf16", "fp4"])
def test_few_queries_over_many_rows_are_those_of_f32(state, element, n, gqa):
    """Scores of 64 slots of 128 kv heads over 8300 rows take more than 256 MiB. A score is one product, q's f32 dim 1 times a
    key of -1 .. 1 that every element holds, of up to 100: its queries have all 24 bits (two bf16 terms would leave 2^-17 of them, 7e-4 of a
    weight). A query is off by the terms' 2 u and the scale's 3 u, a score by as much and 3 products' u: 8 u of 100, twice in a weight (of
    itself and of the largest one): 1600 u; the sums of rows / 4 + 600 and of 64 slots, exponentials and the reciprocal 16 u, arguments 3 u times up to 300
    powers of two: (rows / 4 + 1600) u more."""
    kvh, rows, d = 128, 8300, 4
    gen = torch.Generator(device="cuda").manual_seed(n)
    kv = state.full_attention_with_element(rows, kvh * gqa, kvh, d, {"bf16": skv.DTYPE_BF16, "fp4": skv.DTYPE_FP4}[element])
    k = torch.zeros(rows, kvh, d, device="cuda")
    k[..., 1] = torch.randint(-2, 3, (rows, kvh), device="cuda", generator=gen) * 0.5
    k[..., 2] = 1.0  # (a group's largest number, q is 0 there)
    kv.encode_append_batch(_stream(), k.data_ptr(), k.data_ptr(), rows)
    q = torch.zeros(n, kvh, gqa, d, device="cuda")
    q[..., 1] = 200.0 * (0.5 + 0.5 * torch.rand(kvh, 1, device="cuda", generator=gen))
    w = torch.zeros(kvh, rows, device="cuda")
    kv.encode_attention_weights(_stream(), q.data_ptr(), n, w.data_ptr())
    s = (q[0, :, 0, 1].double() / math.sqrt(d))[:, None] * k[..., 1].double().T  # [kvh, rows], every query's
    want = torch.zeros(kvh, rows, device="cuda", dtype=torch.float64)
    for i in range(n):
        seen = rows - n + i + 1
        want[:, :seen] += gqa * torch.softmax(s[:, :seen], 1)
    off = (w.double() - want).abs()
    assert (off <= want * (rows / 4 + 3200) * U + 1e-36).all(), (off / want).max().item()


def test_many_queries_share_a_bounded_scratch(state):
    """Operands of 32768 queries of eight heads of 512 dims would be 512 MiB: they are taken in parts, and are the sum of the parts."""
    heads, d, rows = 8, 512, 32768
    kv = state.full_attention_bf16(rows, heads, 1, d)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(rows, d, device="cuda", generator=gen)
    kv.encode_append_batch(_stream(), k.data_ptr(), k.data_ptr(), rows)
    q = torch.randn(rows, heads * d, device="cuda", generator=gen)
    w, parts = torch.zeros(1, rows, device="cuda"), torch.zeros(1, rows, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    with torch.cuda.stream(side):
        kv.encode_attention_weights(side.cuda_stream, q.data_ptr(), rows, w.data_ptr())
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] <= 200 << 20
    for first in range(0, rows, 4096):
        kv.truncate(first + 4096)
        kv.encode_attention_weights(_stream(), q[first].data_ptr(), 4096, parts.data_ptr())
    torch.cuda.synchronize()
    # every weight of either is a softmax over bf16 scores of two-term queries by the same products: they differ by the order of sums over slots
    assert torch.allclose(w, parts, rtol=(rows / 4096 + 2 * math.sqrt(rows * heads) + 600) * U, atol=1e-6)
    assert abs(w.double().sum().item() / (rows * heads) - 1.0) < 1e-5
