"""The operators of the 4-bit cache element as measurable cases.

The element (`DTYPE_FP4`) keeps a row of K or V as codes of 4 bits, e2m1, in groups of 32 dims of a
head that share a power of two:

    2^e    the smallest with max |x| of the group <= 7 * 2^e, e in [-125, 125]
    code   x / 2^e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, above 6 to 6
    value  code * 2^e (of a group with an infinity or NaN: NaN)

Four operators work on it: rows stored as codes (`encode_append_batch`), rows read back (`encode_gather`,
in bf16, which holds every value exactly), a decode step, which stores one row per sequence and attends the
cache with one query row per head (`encode_decode_step`, `encode_decode_step_batch`), and a chunk, which stores
its rows and attends the cache with each of them, causally (`encode_prefill_rows`). Attention reads the
values that the codes stand for, of the call's own rows as well.

Every pass first takes the caches back to the length the case starts from (`truncate`, host bookkeeping
only, what a rollback does). The rows a pass stores are attended by it, so its contexts carry the
updated caches too. The head geometries are those of the benchmark's configurations; drawn cases add the
narrower, odd and wider heads of the tests.
"""
import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

GROUP = 32
_CTX = []


def _context():
    import saragossa_amd as skv
    if not _CTX:  # one context per process, as a serving program has
        _CTX.append(skv.DecodeResidentState(0))
    return _CTX[0]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def listed():
    dense = {"q_heads": 32, "kv_heads": 8, "head_dim": 128}
    hybrid = {"q_heads": 16, "kv_heads": 2, "head_dim": 256}
    sliding = {"q_heads": 16, "kv_heads": 8, "head_dim": 256}
    return [
        # one new row behind a chat's 2048: the smallest store there is, and its row read back
        {"name": "store_1_row", "kind": "store", **dense, "rows": 2048, "new": 1},
        # a whole long prompt's rows at once, read back as a disaggregated prefill hands them on
        {"name": "store_32k", "kind": "store", **dense, "rows": 0, "new": 32768},
        # a few hundred rows from the middle of a page on, heads of 80 dims (a last group of 16)
        {"name": "read_777_rows", "kind": "read", "q_heads": 8, "kv_heads": 8, "head_dim": 80, "rows": 1500, "first": 5, "new": 777},
        # a long context of the hybrid model moved elsewhere
        {"name": "read_32k", "kind": "read", **hybrid, "rows": 32768, "first": 0, "new": 32768},
        # one step of one attention layer at 1024 cached rows: the smallest attention a host asks for
        {"name": "decode_one_layer_1k", "kind": "decode", **dense, "layers": 1, "window": 0, "rows": 1024, "tokens": 1, "seqs": 1},
        # a chat answer after a 2048-token prompt: two tokens through all 36 layers
        {"name": "decode_36_layers_2k", "kind": "decode", **dense, "layers": 36, "window": 0, "rows": 2048, "tokens": 2, "seqs": 1},
        # long-context decode of the hybrid model's 10 full-attention layers
        {"name": "decode_32k", "kind": "decode", **hybrid, "layers": 10, "window": 0, "rows": 32768, "tokens": 2, "seqs": 1},
        # four users of the sliding-window model at 65536 context, one period of its layers
        {"name": "batch4_sliding_64k", "kind": "decode", **sliding, "layers": 6, "window": 1024, "global_layers": 1,
         "rows": 65536, "tokens": 2, "seqs": 4},
        # speculative decoding: a draft of six tokens verified over 8k rows, then rolled back
        {"name": "verify_6_rows_8k", "kind": "chunk", **hybrid, "layers": 10, "window": 0, "rows": 8192, "new": 6, "chunk": 6},
        # a prompt of 2000 tokens (not a multiple of the chunk) prefilled in chunks of 512
        {"name": "prompt_2000", "kind": "chunk", **dense, "layers": 4, "window": 0, "rows": 0, "new": 2000, "chunk": 512},
        # one more chunk of a long document
        {"name": "chunk_512_over_32k", "kind": "chunk", **hybrid, "layers": 2, "window": 0, "rows": 32768, "new": 512, "chunk": 512},
        # a prompt through the sliding-window model's local layers (ring caches)
        {"name": "prompt_ring_3000", "kind": "chunk", **sliding, "layers": 5, "window": 1024, "rows": 0, "new": 3000, "chunk": 512},
    ]


GEOMETRIES = [(32, 8, 128), (16, 2, 256), (16, 8, 256), (8, 2, 64), (12, 4, 96), (8, 8, 80), (28, 4, 128), (8, 2, 512),
              (24, 8, 128), (4, 2, 32)]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 4e14


def draw(rng):
    q, kv, hd = rng.choice(GEOMETRIES)
    case = {"kind": rng.choice(["store", "read", "decode", "decode", "decode", "chunk", "chunk", "chunk"]),
            "q_heads": q, "kv_heads": kv, "head_dim": hd}
    kind = case["kind"]
    if kind == "store":
        case.update(rows=rng.choice([0, _log_int(rng, 1, 3000)]), new=_log_int(rng, 1, 32768))
    elif kind == "read":
        n = _log_int(rng, 1, 32768)
        case.update(rows=n + rng.randint(0, 200), new=n, first=0)
        case["first"] = rng.randint(0, case["rows"] - n)
    elif kind == "decode":
        seqs = rng.choice([1, 1, 1, 2, 4, 7])
        case.update(layers=rng.randint(1, 6 if seqs > 1 else 24), window=rng.choice([0, 0, 0, 512, 1024]),
                    rows=_log_int(rng, 17, 32768), tokens=rng.randint(1, 2), seqs=seqs)
    elif rng.random() < 0.5:  # more rows over a cache
        n = _log_int(rng, 2, 512)
        case.update(layers=rng.randint(1, 2), window=0, rows=_log_int(rng, 64, 24000), new=n, chunk=n)
    else:  # a prompt
        case.update(layers=rng.randint(1, 3), window=rng.choice([0, 0, 512, 1024]), rows=0, new=_log_int(rng, 33, 2500),
                    chunk=rng.choice([256, 512, 512, 1024]))
    # no drawn case costs more than the largest listed one
    limit = max(_cost(c) for c in listed())
    while _cost(case) > limit:
        if case.get("layers", 1) > 1:
            case["layers"] = (case["layers"] + 1) // 2
        elif case["rows"] >= case["new"] if kind == "chunk" else kind == "decode":
            case["rows"] = case["rows"] * 2 // 3
        else:
            case["new"] = case["new"] * 2 // 3
            case["first"] = 0
    return case


# ---- inputs ------------------------------------------------------------------------------

class _Inputs:
    def __init__(self, seed, case):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.host = np.random.default_rng(seed)
        self.kv_heads, self.hd = case["kv_heads"], case["head_dim"]

    def normal(self, *shape):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=self.gen)

    def keys(self, *shape):
        """Rows of K: channels of different sizes, some many times the others', as rotated keys have them."""
        size = torch.exp(0.5 * torch.randn(self.kv_heads * self.hd, device="cuda", generator=self.gen))
        return self.normal(*shape, self.kv_heads * self.hd) * (size / size.square().mean().sqrt())

    def values(self, *shape):
        return self.normal(*shape, self.kv_heads * self.hd)

    def history(self, rows):
        """The cached rows of one sequence, in order, 16384 at a time."""
        for first in range(0, rows, 16384):
            n = min(16384, rows - first)
            yield self.keys(n), self.values(n)


def _seq_rows(case, i):  # independent sequences, lengths of their own
    return case["rows"] - 37 * i if case["rows"] > 400 else case["rows"]


def _windows(case):  # of the layers; the last `global_layers` of them have none
    full = case.get("global_layers", 0)
    return [case["window"]] * (case["layers"] - full) + [0] * full


def _layers(case):
    """(window, sequence, rows cached before the pass, rows the pass adds) of every cache of a case."""
    if case["kind"] == "decode":
        return [(w, i, _seq_rows(case, i), case["tokens"]) for w in _windows(case) for i in range(case["seqs"])]
    if case["kind"] == "chunk":
        return [(case["window"], 0, case["rows"], case["new"])] * case["layers"]
    return [(0, 0, case["rows"], case["new"] if case["kind"] == "store" else 0)]


def _new_inputs(case, x):
    """q, k and v of the pass: a decode step's [tokens, layers, sequences], a chunk's [layers, rows]."""
    q_dim = case["q_heads"] * case["head_dim"]
    if case["kind"] == "decode":
        lead = (case["tokens"], case["layers"], case["seqs"])
    elif case["kind"] == "chunk":
        lead = (case["layers"], case["new"])
    elif case["kind"] == "store":
        return None, x.keys(case["new"]), x.values(case["new"])
    else:
        return None, None, None
    return x.normal(*lead, q_dim), x.keys(*lead), x.values(*lead)


def prepare(case, seed):
    x = _Inputs(seed, case)
    s = {"case": case, "caches": []}
    for window, _, rows, new in _layers(case):
        if own:
            import saragossa_amd as skv
            kv = _context().full_attention_with_element(rows + new, case["q_heads"], case["kv_heads"], case["head_dim"],
                                                        skv.DTYPE_FP4, window)
            kv.set_block_table(x.host.permutation(kv.pages()).astype(np.int32))
            for k, v in x.history(rows):
                kv.encode_append_batch(_stream(), k.data_ptr(), v.data_ptr(), k.shape[0])
            s["caches"].append((kv, rows))
        else:
            s["caches"].append(_plain_cache(case, x, window, rows, new))
    s["q"], s["k"], s["v"] = _new_inputs(case, x)
    if s["q"] is not None:
        s["out"] = torch.empty_like(s["q"])
    elif own:
        s["out"] = torch.empty(2, case["new"], case["kv_heads"] * case["head_dim"], device="cuda", dtype=torch.bfloat16)
    return s


# ---- passes ------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"store": _plain_rows, "read": _plain_rows, "decode": _plain_decode, "chunk": _plain_chunk}[kind](s)
    return {"store": _run_rows, "read": _run_rows, "decode": _run_decode, "chunk": _run_chunk}[kind](s)


def _run_rows(s):
    case, (kv, rows), out, stream = s["case"], s["caches"][0], s["out"], _stream()
    n, first = case["new"], case.get("first", 0)
    if case["kind"] == "store":
        kv.truncate(rows)
        kv.encode_append_batch(stream, s["k"].data_ptr(), s["v"].data_ptr(), n)
        first = rows
    kv.encode_gather(stream, first, n, out[0].data_ptr(), out[1].data_ptr())
    return [out[0], out[1]]


def _run_decode(s):
    import saragossa_amd as skv
    case, stream = s["case"], _stream()
    q, k, v, out = s["q"], s["k"], s["v"], s["out"]
    tokens, n_layers, seqs = k.shape[:3]
    for kv, rows in s["caches"]:
        kv.truncate(rows)
    qs, ks = q.shape[3] * 4, k.shape[3] * 4
    q0, k0, v0, o0 = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    for t in range(tokens):
        for li in range(n_layers):
            at = (t * n_layers + li) * seqs
            if seqs > 1:
                skv.encode_decode_step_batch([s["caches"][li * seqs + i][0] for i in range(seqs)], stream,
                                             [k0 + (at + i) * ks for i in range(seqs)], [v0 + (at + i) * ks for i in range(seqs)],
                                             [q0 + (at + i) * qs for i in range(seqs)], [o0 + (at + i) * qs for i in range(seqs)])
            else:
                s["caches"][li][0].encode_decode_step(stream, k0 + at * ks, 0, v0 + at * ks, 0, q0 + at * qs, o0 + at * qs)
    return out


def _run_chunk(s):
    case, stream = s["case"], _stream()
    q, k, v, out = s["q"], s["k"], s["v"], s["out"]
    for kv, rows in s["caches"]:
        kv.truncate(rows)
    for first in range(0, case["new"], case["chunk"]):
        n = min(case["chunk"], case["new"] - first)
        for li, (kv, _) in enumerate(s["caches"]):
            kv.encode_prefill_rows(stream, q[li, first].data_ptr(), k[li, first].data_ptr(), v[li, first].data_ptr(), n,
                                   out[li, first].data_ptr())
    return out


# ---- plain forms -------------------------------------------------------------------------

def _quantise(x, heads, hd):
    """Rows [n, heads * hd] -> codes [n, heads, groups, 32] (uint8, sign in bit 3) and scales [n, heads, groups, 1]."""
    groups = -(-hd // GROUP)
    x = torch.nn.functional.pad(x.view(-1, heads, hd), (0, groups * GROUP - hd)).view(-1, heads, groups, GROUP)
    top = x.abs().amax(-1, keepdim=True)
    # the exponent field of max |x|, one more where the leading bits pass 1.75, less two (7 = 1.75 * 2^2)
    e = (((top.view(torch.int32) + 0x1fffff) >> 23) - 129).clamp(-125, 125)
    scale = torch.ldexp(torch.ones_like(top), e)
    y = (x / scale).abs()
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    return (code + 8 * (x < 0)).to(torch.uint8), scale


_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values(code, scale, hd):
    """[n, heads, groups, 32] -> [n, heads, hd] in 32 bits."""
    table = torch.tensor(_LEVELS + [-a for a in _LEVELS], device=code.device)
    return (table[code.int()] * scale).flatten(2)[..., :hd]


def _plain_cache(case, x, window, rows, new):
    """Codes and scales of the rows that the pass can see, and room for its own: position p lies at row p - base."""
    h, hd = case["kv_heads"], case["head_dim"]
    base = max(0, rows - window) if window else 0
    groups = -(-hd // GROUP)
    cache = [torch.zeros(rows - base + new, h, groups, GROUP, device="cuda", dtype=torch.uint8),
             torch.ones(rows - base + new, h, groups, 1, device="cuda"),
             torch.zeros(rows - base + new, h, groups, GROUP, device="cuda", dtype=torch.uint8),
             torch.ones(rows - base + new, h, groups, 1, device="cuda")]
    at = 0
    for k, v in x.history(rows):
        skip = min(max(base - at, 0), k.shape[0])
        at += skip
        if skip < k.shape[0]:
            _plain_store(case, cache, at - base, k[skip:], v[skip:])
        at += k.shape[0] - skip
    return cache, rows, base, window


def _plain_store(case, cache, at, k, v):
    n = k.shape[0]
    cache[0][at:at + n], cache[1][at:at + n] = _quantise(k, case["kv_heads"], case["head_dim"])
    cache[2][at:at + n], cache[3][at:at + n] = _quantise(v, case["kv_heads"], case["head_dim"])


def _plain_rows(s):
    case, (cache, rows, _, _) = s["case"], s["caches"][0]
    n, first = case["new"], case.get("first", 0)
    if case["kind"] == "store":
        _plain_store(case, cache, rows, s["k"], s["v"])
        first = rows
    here = slice(first, first + n)
    return [_values(cache[i][here], cache[i + 1][here], case["head_dim"]).flatten(1).to(torch.bfloat16) for i in (0, 2)]


def _plain_attend(case, cache, base, window, first, q):
    """Rows q [n, q_heads * hd] at positions first .. over the cache, each up to its own position."""
    h, hd, n = case["kv_heads"], case["head_dim"], q.shape[0]
    lo = max(base, first + 1 - window) if window else 0
    here = slice(lo - base, first + n - base)
    k, v = (_values(cache[i][here], cache[i + 1][here], hd).permute(1, 0, 2).contiguous() for i in (0, 2))
    g = case["q_heads"] // h
    rows = q.view(n, h, g, hd).permute(1, 0, 2, 3).reshape(h, n * g, hd)
    scores = torch.matmul(rows, k.transpose(1, 2)) / hd ** 0.5
    if n > 1 or window:
        pos = torch.arange(lo, first + n, device=q.device)
        own_pos = torch.arange(first, first + n, device=q.device).repeat_interleave(g)[:, None]
        seen = pos <= own_pos
        if window:
            seen &= pos > own_pos - window
        scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return out.view(h, n, g, hd).permute(1, 0, 2, 3).reshape(n, -1)


def _plain_decode(s):
    case, out = s["case"], s["out"]
    tokens, n_layers, seqs = s["k"].shape[:3]
    for t in range(tokens):
        for li in range(n_layers):
            for i in range(seqs):
                cache, rows, base, window = s["caches"][li * seqs + i]
                _plain_store(case, cache, rows + t - base, s["k"][t, li, i][None], s["v"][t, li, i][None])
                out[t, li, i] = _plain_attend(case, cache, base, window, rows + t, s["q"][t, li, i][None])[0]
    return out


def _plain_chunk(s):
    case, out = s["case"], s["out"]
    for first in range(0, case["new"], case["chunk"]):
        last = min(first + case["chunk"], case["new"])
        for li, (cache, rows, base, window) in enumerate(s["caches"]):
            _plain_store(case, cache, rows + first - base, s["k"][li, first:last], s["v"][li, first:last])
            out[li, first:last] = _plain_attend(case, cache, base, window, rows + first, s["q"][li, first:last])
    return out


# ---- from the definition, in 64 bits -------------------------------------------------------

def _exact_rows(x, hd):
    """What rows are worth once stored."""
    w = x.double().unflatten(-1, (-1, hd))
    out = torch.empty_like(w)
    levels = torch.tensor(_LEVELS, device=x.device, dtype=torch.float64)
    for d in range(0, hd, GROUP):
        part = w[..., d:d + GROUP]
        mantissa, exponent = torch.frexp(part.abs().amax(-1, keepdim=True) / 7.0)  # mantissa in [1/2, 1)
        power = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(-125, 125)
        scale = torch.pow(2.0, power.double())
        y = part.abs() / scale
        above = torch.bucketize(y, levels).clamp(1, 7)
        below = above - 1
        near, far = y - levels[below], levels[above] - y
        up = (far < near) | ((far == near) & (above % 2 == 0))
        out[..., d:d + GROUP] = torch.sign(part) * levels[torch.where(up, above, below)] * scale
    return out.flatten(-2)


def exact(case, seed):
    x = _Inputs(seed, case)
    h, hd, g = case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    pasts = []
    for window, _, rows, _ in _layers(case):
        parts = [(k, v) for k, v in x.history(rows)]
        keep = window if window else rows
        pasts.append([torch.cat([p[i] for p in parts])[-keep:] if parts and keep else None for i in (0, 1)])
    q, k, v = _new_inputs(case, x)
    if case["kind"] == "store":
        return [_exact_rows(k, hd), _exact_rows(v, hd)]
    if case["kind"] == "read":
        here = slice(case["first"], case["first"] + case["new"])
        return [_exact_rows(pasts[0][0][here], hd), _exact_rows(pasts[0][1][here], hd)]
    out = torch.empty(q.shape, device=q.device, dtype=torch.float64)

    def attend(past, window, rows, new_k, new_v, new_q, dst):
        """All new rows of one cache at once, 256 at a time: row i sees the past and the new rows up to its own."""
        keys, vals = (_exact_rows(torch.cat([p, n]) if p is not None else n, hd).view(-1, h, hd) for p, n in
                      ((past[0], new_k), (past[1], new_v)))
        start = rows + new_k.shape[0] - keys.shape[0]  # position of keys[0]
        for i0 in range(0, new_q.shape[0], 256):
            part = new_q[i0:i0 + 256].double().view(-1, h, g, hd)
            end = rows + i0 + part.shape[0] - start
            begin = max(0, rows + i0 + 1 - window - start) if window else 0
            pos = torch.arange(begin, end, device=q.device) + start
            mine = torch.arange(part.shape[0], device=q.device) + rows + i0
            hidden = pos[None, :] > mine[:, None]
            if window:
                hidden |= pos[None, :] + window <= mine[:, None]
            for head in range(h):
                logits = part[:, head].flatten(0, 1) @ keys[begin:end, head].T / float(hd) ** 0.5
                logits = logits.unflatten(0, (-1, g)).masked_fill(hidden[:, None, :], float("-inf"))
                weights = torch.softmax(logits, -1).flatten(0, 1)
                dst[i0:i0 + 256].view(-1, h, g, hd)[:, head] = (weights @ vals[begin:end, head]).unflatten(0, (-1, g))

    for at, (window, i, rows, _) in enumerate(_layers(case)):
        if case["kind"] == "chunk":
            attend(pasts[at], window, rows, k[at], v[at], q[at], out[at])
        else:
            li = at // case["seqs"]
            attend(pasts[at], window, rows, k[:, li, i], v[:, li, i], q[:, li, i], out[:, li, i])
    return out


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    h, hd, n = case["kv_heads"], case["head_dim"], case.get("new", 0)
    q_dim, kv_dim = case["q_heads"] * hd, h * hd
    held = 2 * h * (hd / 2 + -(-hd // GROUP))  # bytes of a row's K and V as codes and scales
    if case["kind"] == "store":  # f32 rows in, codes out; codes in, bf16 rows out
        return {"bytes": int(n * (8 * kv_dim + 2 * held + 4 * kv_dim)), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": int(n * (held + 4 * kv_dim)), "flops": 0}
    nbytes = flops = 0
    for window, _, rows, new in _layers(case):
        step = 1 if case["kind"] == "decode" else case["chunk"]
        for first in range(0, new, step):
            c = min(step, new - first)
            old = rows + first
            kept = min(old, window - 1) if window else old
            # cached rows in, the new rows in (f32) and out, q in and the context out
            nbytes += kept * held + c * (held + 8 * kv_dim + 8 * q_dim)
            for p in range(old + 1, old + c + 1):
                flops += 4 * q_dim * (min(p, window) if window else p)
    return {"bytes": int(nbytes), "flops": int(flops)}
