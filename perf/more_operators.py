"""Operators that keep a long context in bounded memory, as measurable cases.

Rows of a cache leave it by the attention they have had:

    weights   w[h, r] += sum over the queries i and the heads g of kv head h of softmax_r(q[i, g] . K[h, r] / sqrt(d)), rows
              r up to the query's own (the n queries are those of the cache's last n rows) -- `encode_attention_weights`
    evict     of a cache of `rows` rows, per kv head, `keep` stay: the first `first`, the last `last` and the heaviest of
              those between (of equal ones the lower); those below `keep` stay where they are, the gaps take the others
              in order; the weights move along, those behind `keep` become 0 -- `encode_evict`

and the other layers of a hybrid model keep a state instead of rows, S [k_dim, v_dim] per v head, linear attention with a
decay: v head h reads q and k of head h / (v_heads / k_heads),

    S_t = exp(g_t) S_(t-1) + k_t v_t^T,     o_t = scale * q_t^T S_t

    linear_rows   n tokens of one sequence -- `LinearAttention.encode_rows`
    linear_step   one token each of several sequences -- `LinearAttention.encode_step`

with a decay g of each token and head, or one of each head. Passes that change caches or weights begin by putting back the
weights (one copy) and the cache's length (host bookkeeping): an eviction leaves the rows behind the new length as they were and
moves nothing but those into the gaps, so passes repeat. The cached rows are numbers that every element of a cache holds exactly
(4-bit codes times a power of two per 32 dims, in bf16 and f32 too). Head geometries are those of the benchmark's
configurations, linear ones those of its hybrid model's recurrent state; drawn cases add narrower, odd and wider heads.
"""
import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

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
    delta = {"k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128}
    return [
        # one layer's weights of one decoded token over a short chat: the smallest call
        {"name": "weights_one_layer_1k", "kind": "weights", **dense, "element": "bf16", "layers": 1, "rows": 1024, "queries": 1},
        # a decoded token over a long context, all full-attention layers of the hybrid model
        {"name": "weights_step_32k", "kind": "weights", **hybrid, "element": "bf16", "layers": 10, "rows": 32768, "queries": 1},
        # the same on a 4-bit cache, an odd length, one global layer of each period
        {"name": "weights_step_fp4_30001", "kind": "weights", **sliding, "element": "fp4", "layers": 8, "rows": 30001, "queries": 1},
        # the last 32 tokens of a prompt say which of its rows a greedy request (f32 rows) keeps
        {"name": "weights_window_32_f32", "kind": "weights", **dense, "element": "f32", "layers": 4, "rows": 5003, "queries": 32},
        # a prompt's chunk of 512 rows weighs all that came before it
        {"name": "weights_chunk_512_16k", "kind": "weights", **hybrid, "element": "bf16", "layers": 2, "rows": 16896, "queries": 512},
        # a cache at its budget: every decoded token one row leaves
        {"name": "evict_one_of_2049", "kind": "evict", **dense, "element": "bf16", "layers": 36, "rows": 2049, "keep": 2048,
         "first": 4, "last": 512},
        # a long prompt cut to half before decoding
        {"name": "evict_half_of_32k", "kind": "evict", **hybrid, "element": "bf16", "layers": 10, "rows": 32768, "keep": 16384,
         "first": 4, "last": 1024},
        # f32 rows, heads of 96 dims, an odd length to an odd budget
        {"name": "evict_5003_to_1111_f32", "kind": "evict", "q_heads": 12, "kv_heads": 4, "head_dim": 96, "element": "f32",
         "layers": 4, "rows": 5003, "keep": 1111, "first": 0, "last": 33},
        # one token through the hybrid model's 30 linear layers
        {"name": "linear_step_30_layers", "kind": "linear_step", **delta, "layers": 30, "seqs": 1, "per_token": True},
        # eleven sequences a step, a fixed decay a head, dims that are no powers of two
        {"name": "linear_step_11_seqs", "kind": "linear_step", "k_heads": 8, "v_heads": 8, "k_dim": 96, "v_dim": 200, "layers": 4,
         "seqs": 11, "per_token": False},
        # a prompt of 2000 tokens through four linear layers
        {"name": "linear_prompt_2000", "kind": "linear_rows", **delta, "layers": 4, "rows": 2000, "per_token": True},
        # a long document
        {"name": "linear_prompt_16k", "kind": "linear_rows", **delta, "layers": 2, "rows": 16384, "per_token": True},
    ]


GEOMETRIES = [(32, 8, 128), (16, 2, 256), (16, 8, 256), (8, 2, 64), (12, 4, 96), (8, 8, 80), (28, 4, 128), (8, 2, 512),
              (24, 8, 128), (4, 2, 32)]
LINEAR = [(16, 32, 128, 128), (16, 32, 128, 128), (8, 8, 64, 64), (4, 8, 96, 80), (2, 2, 256, 256), (16, 16, 64, 128), (3, 9, 100, 36),
          (1, 4, 32, 256), (32, 32, 128, 64)]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1e14


def draw(rng):
    kind = rng.choice(["weights", "weights", "weights", "evict", "evict", "linear_step", "linear_rows", "linear_rows"])
    if kind in ("weights", "evict"):
        q, kv, hd = rng.choice(GEOMETRIES)
        case = {"kind": kind, "q_heads": q, "kv_heads": kv, "head_dim": hd, "element": rng.choice(["bf16", "bf16", "f32", "fp4"]),
                "layers": rng.randint(1, 10), "rows": _log_int(rng, 20, 32768)}
        if kind == "weights":
            case["queries"] = min(case["rows"], rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 700)]))
            if case["queries"] > 1:
                case["layers"] = min(case["layers"], 2)
        else:
            case["keep"] = rng.choice([case["rows"] - 1, rng.randint(1, case["rows"] - 1), rng.randint(1, case["rows"] - 1)])
            case["first"] = min(rng.choice([0, 4, 16]), case["keep"])
            case["last"] = rng.randint(0, case["keep"] - case["first"]) // rng.choice([1, 4, 16])
    else:
        kh, vh, dk, dv = rng.choice(LINEAR)
        case = {"kind": kind, "k_heads": kh, "v_heads": vh, "k_dim": dk, "v_dim": dv, "layers": rng.randint(1, 4),
                "per_token": rng.random() < 0.7}
        if kind == "linear_step":
            case.update(seqs=rng.choice([1, 2, 5, 11, 16, 33]), layers=rng.randint(1, 30))
        else:
            case["rows"] = _log_int(rng, 1, 16384)
    # no drawn case costs more than the largest listed one
    limit = max(_cost(c) for c in listed())
    while _cost(case) > limit:
        if case["layers"] > 1:
            case["layers"] = (case["layers"] + 1) // 2
        elif case["kind"] == "weights":
            case["queries"] = (case["queries"] + 1) // 2
        else:
            case["rows"] = case["rows"] * 2 // 3
    return case


# ---- inputs ------------------------------------------------------------------------------

SPARE = 40  # rows of a cache that are free when a pass begins


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _cached(case, gen, keys):
    """Rows [heads, rows, dims] of one layer: 4-bit codes, a 4 or -4 in each group of 32 dims, times a power of two per group; keys have
    channels of different sizes, as rotated keys have them."""
    h, n, hd = case["kv_heads"], case["rows"], case["head_dim"]
    size = _normal(gen, h, 1, hd) * 0.5 if keys else torch.zeros(h, 1, hd, device="cuda")
    x = _normal(gen, h, n, hd) * torch.exp(size) * 2.0
    x = torch.clamp(torch.round(x), -4.0, 4.0)  # whole numbers that the codes have
    x[..., ::32] = torch.where(x[..., ::32] < 0, -4.0, 4.0)
    groups = torch.repeat_interleave(torch.randint(-3, 0, (h, n, -(-hd // 32)), device="cuda", generator=gen), 32, dim=-1)
    return torch.ldexp(x, groups[..., :hd])


def _rows_inputs(case, seed):
    """Layers' K and V [layers, heads, rows, dims], queries of the last rows, and the weights so far [layers, heads, rows + spare]."""
    gen = _generator(seed)
    layers, h, hd = case["layers"], case["kv_heads"], case["head_dim"]
    kv = [torch.empty(layers, h, case["rows"], hd, device="cuda") for _ in range(2)]
    for li in range(layers):
        kv[0][li], kv[1][li] = _cached(case, gen, True), _cached(case, gen, False)
    q = _normal(gen, layers, case.get("queries", 1), case["q_heads"] * hd) * 3.0
    # a few rows get most of the attention, many get none that 32 bits would hold
    w = torch.exp(2.0 * _normal(gen, layers, h, case["rows"] + SPARE))
    w = torch.where(w < 0.1, 0.0, w)
    if case["kind"] == "weights":  # of the order of what the pass adds
        w *= case["queries"] * case["q_heads"] / (8.0 * h * case["rows"])
    w[..., case["rows"]:] = 0.0
    return kv[0], kv[1], q, w


def _linear_inputs(case, seed):
    """q, k and v as one projection per token, as they come from a layer's convolution; log decays; the state so far."""
    gen = _generator(seed)
    layers, kh, vh, dk, dv = (case[n] for n in ("layers", "k_heads", "v_heads", "k_dim", "v_dim"))
    n = case["seqs"] if case["kind"] == "linear_step" else case["rows"]
    qkv = torch.nn.functional.silu(_normal(gen, layers, n, 2 * kh * dk + vh * dv) * 1.5)
    if case["per_token"]:
        rate = torch.exp(torch.linspace(-4.0, 2.7, vh, device="cuda"))
        g = -rate * torch.nn.functional.softplus(_normal(gen, layers, n, vh) - 4.0)
    else:
        g = torch.log1p(-torch.exp2(-torch.linspace(3.0, 9.0, vh, device="cuda"))).repeat(layers, 1)
    states = (layers, case["seqs"]) if case["kind"] == "linear_step" else (layers,)
    return qkv, g, _normal(gen, *states, vh, dk, dv)


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] in ("linear_rows", "linear_step"):
        s["qkv"], s["g"], s["state"] = _linear_inputs(case, seed)
        s["new"] = torch.empty_like(s["state"])
        s["out"] = torch.empty(*s["qkv"].shape[:2], case["v_heads"] * case["v_dim"], device="cuda")
        if own:
            s["op"] = _context().linear_attention(case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"],
                                                  case["k_dim"] ** -0.5)
        return s
    k, v, s["q"], s["w0"] = _rows_inputs(case, seed)
    s["w"] = torch.empty_like(s["w0"])
    dtype = torch.float32 if case["element"] == "f32" else torch.bfloat16
    if case["kind"] == "evict":
        s["kept"] = torch.empty(case["layers"], case["kv_heads"], case["keep"], device="cuda", dtype=torch.int32)
        s["rows"] = torch.empty(2, case["layers"], case["keep"], case["kv_heads"] * case["head_dim"], device="cuda", dtype=dtype)
    if own:
        s["caches"] = _caches(case, k, v, seed)
    elif case["kind"] == "evict":
        s["k"], s["v"] = k.to(dtype), v.to(dtype)
    else:
        s["k"] = k
    return s


def _caches(case, k, v, seed):
    import saragossa_amd as skv
    host = np.random.default_rng(seed)
    element = {"bf16": skv.DTYPE_BF16, "f32": skv.DTYPE_F32, "fp4": skv.DTYPE_FP4}[case["element"]]
    caches = []
    for li in range(case["layers"]):
        kv = _context().full_attention_with_element(case["rows"] + SPARE, case["q_heads"], case["kv_heads"], case["head_dim"], element)
        kv.set_block_table(host.permutation(kv.pages()).astype(np.int32))
        rows = [x[li].transpose(0, 1).contiguous() for x in (k, v)]
        kv.encode_append_batch(_stream(), rows[0].data_ptr(), rows[1].data_ptr(), case["rows"])
        caches.append(kv)
    return caches


# ---- passes ------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"weights": _plain_weights, "evict": _plain_evict, "linear_rows": _plain_linear_rows,
                "linear_step": _plain_linear_step}[kind](s)
    return {"weights": _run_weights, "evict": _run_evict, "linear_rows": _run_linear_rows, "linear_step": _run_linear_step}[kind](s)


def _run_weights(s):
    stream, q, w = _stream(), s["q"], s["w"]
    w.copy_(s["w0"])
    qs, ws = q[0].numel() * 4, w[0].numel() * 4
    for li, kv in enumerate(s["caches"]):
        kv.encode_attention_weights(stream, q.data_ptr() + li * qs, q.shape[1], w.data_ptr() + li * ws)
    return w


def _run_evict(s):
    case, stream, w, kept, rows = s["case"], _stream(), s["w"], s["kept"], s["rows"]
    w.copy_(s["w0"])
    ws, ks, rs = w[0].numel() * 4, kept[0].numel() * 4, rows[0, 0].numel() * rows.element_size()
    k0, v0 = rows[0].data_ptr(), rows[1].data_ptr()
    for li, kv in enumerate(s["caches"]):
        kv.truncate(case["rows"])
        kv.encode_evict(stream, w.data_ptr() + li * ws, case["keep"], case["first"], case["last"], kept.data_ptr() + li * ks)
        kv.encode_gather(stream, 0, case["keep"], k0 + li * rs, v0 + li * rs)
    return [rows[0], rows[1], kept, w]


def _linear_pointers(s):
    case, stride = s["case"], s["qkv"].shape[2] * 4
    base, keys = s["qkv"].data_ptr(), case["k_heads"] * case["k_dim"] * 4
    decays = case["v_heads"] if case["per_token"] else 0
    for li in range(case["layers"]):
        at = base + li * s["qkv"].shape[1] * stride
        yield li, at, at + keys, at + 2 * keys, stride // 4, s["g"][li].data_ptr(), decays


def _run_linear_rows(s):
    stream, op, out = _stream(), s["op"], s["out"]
    for li, q, k, v, stride, g, decays in _linear_pointers(s):
        op.encode_rows(stream, q, stride, k, stride, v, stride, g, decays, out.shape[1], s["state"][li].data_ptr(),
                       s["new"][li].data_ptr(), out[li].data_ptr())
    return [out, s["new"]]


def _run_linear_step(s):
    stream, op, out, seqs = _stream(), s["op"], s["out"], s["case"]["seqs"]
    size = s["state"][0, 0].numel() * 4
    for li, q, k, v, stride, g, decays in _linear_pointers(s):
        old, new = s["state"][li].data_ptr(), s["new"][li].data_ptr()
        op.encode_step(stream, q, stride, k, stride, v, stride, g, decays, [old + i * size for i in range(seqs)],
                       [new + i * size for i in range(seqs)], out[li].data_ptr())
    return [out, s["new"]]


# ---- plain forms -------------------------------------------------------------------------

def _plain_weights(s):
    case, k, q = s["case"], s["k"], s["q"]
    layers, h, rows, hd = k.shape
    n, g = q.shape[1], case["q_heads"] // h
    queries = q.view(layers, n, h, g, hd).permute(0, 2, 1, 3, 4).reshape(layers, h, n * g, hd)
    scores = torch.matmul(queries, k.transpose(2, 3)) / hd ** 0.5
    if n > 1:
        own_row = torch.arange(rows - n, rows, device=k.device).repeat_interleave(g)
        scores = scores.masked_fill(torch.arange(rows, device=k.device) > own_row[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    w = s["w"].copy_(s["w0"])
    w[..., :rows] += p.sum(2)
    return w


def _plain_evict(s):
    case, w = s["case"], s["w"].copy_(s["w0"])
    rows, keep, first, last = case["rows"], case["keep"], case["first"], case["last"]
    middle = w[..., first:rows - last]
    heaviest = torch.sort(middle, dim=-1, descending=True, stable=True).indices[..., :keep - first - last]
    stays = torch.zeros(*w.shape[:2], rows, device=w.device, dtype=torch.bool)
    stays[..., :first] = True
    stays[..., rows - last:] = True
    stays.scatter_(2, heaviest + first, True)
    movers = torch.sort((~stays[..., keep:]).to(torch.uint8), dim=-1, stable=True).indices + keep  # those that stay in front
    gaps = ~stays[..., :keep]
    turn = (torch.cumsum(gaps, -1) - 1).clamp(0, rows - keep - 1)  # which of the movers a gap takes
    kept = torch.where(gaps, torch.gather(movers, 2, turn), torch.arange(keep, device=w.device))
    out = s["rows"]
    for i, x in enumerate((s["k"], s["v"])):
        here = torch.gather(x, 2, kept[..., None].expand(-1, -1, -1, x.shape[3]))
        out[i] = here.transpose(1, 2).flatten(2)
    moved = torch.gather(w, 2, kept)
    w[..., keep:rows] = 0.0
    w[..., :keep] = moved
    s["kept"].copy_(kept)
    return [out[0], out[1], s["kept"], w]


def _heads(case, qkv):
    """q and k of every v head [..., v_heads, tokens, k_dim], v [..., v_heads, tokens, v_dim]."""
    kh, vh, dk, dv = (case[n] for n in ("k_heads", "v_heads", "k_dim", "v_dim"))
    q, k, v = torch.split(qkv, [kh * dk, kh * dk, vh * dv], dim=-1)
    q, k = (x.unflatten(-1, (kh, dk)).repeat_interleave(vh // kh, dim=-2).transpose(-2, -3) for x in (q, k))
    return q, k, v.unflatten(-1, (vh, dv)).transpose(-2, -3)


CHUNK = 64


def _plain_linear_rows(s):
    """Chunks of tokens: inside one by its scores, from what came before through the state in front of it."""
    case, scale = s["case"], s["case"]["k_dim"] ** -0.5
    layers, n = s["qkv"].shape[:2]
    pad = -n % CHUNK
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)).unflatten(2, (-1, CHUNK)) for x in _heads(case, s["qkv"]))
    g = s["g"] if case["per_token"] else s["g"][:, None].expand(-1, n, -1)
    g = torch.nn.functional.pad(g.double().transpose(1, 2), (0, pad)).unflatten(2, (-1, CHUNK))
    b = torch.cumsum(g, -1)  # log decay from in front of the chunk up to each token
    seen = torch.ones(CHUNK, CHUNK, device=q.device, dtype=torch.bool).tril()
    between = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~seen, float("-inf"))).float()
    out = torch.matmul(torch.matmul(q, k.transpose(3, 4)) * between, v)
    added = torch.matmul((k * torch.exp(b[..., -1:] - b).float()[..., None]).transpose(3, 4), v)
    whole = torch.exp(b[..., -1]).float()[..., None, None]
    before = torch.empty_like(added)
    state = s["state"]
    for c in range(added.shape[2]):
        before[:, :, c] = state
        state = whole[:, :, c] * state + added[:, :, c]
    out += torch.matmul(q * torch.exp(b).float()[..., None], before)
    s["out"].copy_((out * scale).flatten(2, 3)[:, :, :n].transpose(1, 2).flatten(2))
    s["new"].copy_(state)
    return [s["out"], s["new"]]


def _plain_linear_step(s):
    case = s["case"]
    q, k, v = (x.squeeze(-2) for x in _heads(case, s["qkv"][:, :, None]))
    g = s["g"] if case["per_token"] else s["g"][:, None]
    new = torch.exp(g)[..., None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    s["new"].copy_(new)
    s["out"].copy_((torch.matmul(q[..., None, :], new).squeeze(-2) * case["k_dim"] ** -0.5).flatten(2))
    return [s["out"], s["new"]]


# ---- from the definition, in 64 bits -------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "weights":
        return _exact_weights(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(case, seed)
    return _exact_linear(case, seed)


def _exact_weights(case, seed):
    k, _, q, w = _rows_inputs(case, seed)
    w = w.double()
    n, rows, hd, group = case["queries"], case["rows"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    later = torch.arange(rows, device=w.device)[None, :] - torch.arange(rows - n, rows, device=w.device)[:, None] > 0
    for li in range(case["layers"]):
        for head in range(case["q_heads"]):
            logits = q[li, :, head * hd:(head + 1) * hd].double() @ k[li, head // group].double().T / float(hd) ** 0.5
            w[li, head // group, :rows] += torch.softmax(logits.masked_fill(later, float("-inf")), -1).sum(0)
    return w


def _exact_evict(case, seed):
    k, v, _, w = _rows_inputs(case, seed)
    rows, keep, first, last = case["rows"], case["keep"], case["first"], case["last"]
    host, order = w.double().cpu().numpy(), np.empty((case["layers"], case["kv_heads"], keep), np.int64)
    for li in range(case["layers"]):
        for head in range(case["kv_heads"]):
            between = np.arange(first, rows - last)
            chosen = between[np.lexsort((between, -host[li, head, first:rows - last]))][:keep - first - last]
            stay = np.sort(np.concatenate([np.arange(first), chosen, np.arange(rows - last, rows)]))
            low, high = stay[stay < keep], stay[stay >= keep]
            order[li, head] = np.arange(keep)
            order[li, head, np.setdiff1d(np.arange(keep), low)] = high
    at = torch.from_numpy(order).cuda()
    out = [torch.stack([torch.stack([x[li, head, at[li, head]] for head in range(case["kv_heads"])], 1) for li in range(case["layers"])])
           for x in (k, v)]
    moved = torch.zeros_like(w, dtype=torch.float64)
    moved[..., :keep] = torch.gather(w.double(), 2, at)
    return [out[0].flatten(2).double(), out[1].flatten(2).double(), at.to(torch.int32), moved]


def _exact_linear(case, seed):
    qkv, g, state = _linear_inputs(case, seed)
    kh, vh, dk, dv = (case[n] for n in ("k_heads", "v_heads", "k_dim", "v_dim"))
    scale, group, n = 1.0 / float(dk) ** 0.5, vh // kh, qkv.shape[1]
    x, state = qkv.double(), state.double()
    q, k, v = x[..., :kh * dk], x[..., kh * dk:2 * kh * dk], x[..., 2 * kh * dk:]
    decay = torch.exp(g.double()) if case["per_token"] else torch.exp(g.double())[:, None, :].expand(-1, n, -1)
    q, k = (t.reshape(*t.shape[:2], kh, 1, dk).expand(-1, -1, -1, group, -1).reshape(*t.shape[:2], vh, dk) for t in (q, k))
    v = v.reshape(*v.shape[:2], vh, dv)
    out = torch.empty(case["layers"], n, vh, dv, device="cuda", dtype=torch.float64)
    if case["kind"] == "linear_step":
        state = decay[..., None, None] * state + k[..., None] * v[..., None, :]
        out = scale * (q[..., None] * state).sum(-2)
    else:
        for t in range(n):
            state = torch.baddbmm((decay[:, t, :, None, None] * state).flatten(0, 1), k[:, t].flatten(0, 1)[:, :, None].contiguous(),
                                  v[:, t].flatten(0, 1)[:, None, :].contiguous()).unflatten(0, (case["layers"], vh))
            out[:, t] = scale * torch.matmul(q[:, t, :, None, :], state).squeeze(-2)
    return [out.flatten(2), state]


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    if case["kind"] in ("linear_rows", "linear_step"):
        kh, vh, dk, dv = (case[n] for n in ("k_heads", "v_heads", "k_dim", "v_dim"))
        seqs = case.get("seqs", 1)
        n = case.get("rows", 1) * seqs
        decays = n * vh if case["per_token"] else vh
        nbytes = 4 * (n * (2 * kh * dk + 2 * vh * dv) + decays + 2 * seqs * vh * dk * dv)
        return {"bytes": case["layers"] * nbytes, "flops": case["layers"] * n * vh * 4 * dk * dv}
    h, hd, rows = case["kv_heads"], case["head_dim"], case["rows"]
    held = h * {"bf16": 2 * hd, "f32": 4 * hd, "fp4": (hd + 1) // 2 + -(-hd // 32)}[case["element"]]  # bytes of a row of K, or of V
    if case["kind"] == "weights":  # K and the weights in, the queries in, the weights out
        n = case["queries"]
        nbytes = rows * held + 8 * h * rows + 4 * n * case["q_heads"] * hd
        return {"bytes": case["layers"] * nbytes, "flops": case["layers"] * 2 * case["q_heads"] * hd * sum(range(rows - n + 1, rows + 1))}
    # the weights in and out, the kept rows' numbers out, the rows that move in and out; then all rows in, and out as row-major ones
    keep = case["keep"]
    between = rows - case["first"] - case["last"]
    gaps = min(rows - keep, max(0, min(keep, rows - case["last"]) - case["first"]) * (rows - keep) // max(between, 1))
    plain = held if case["element"] != "fp4" else 2 * h * hd
    nbytes = 4 * h * (2 * rows + keep) + 2 * (2 * max(gaps, 1) * held + keep * (held + plain))
    return {"bytes": case["layers"] * nbytes, "flops": 0}
