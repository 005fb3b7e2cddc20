"""Cases that measure the operators a GPT needs to answer with what it has learned: rotary positions, the paged
key-value cache (written, quantised, read back) and the attention of one new token over it.

`run` computes an operator either in its plain form, from elementary torch operations in 32 bits (64 for the angles of
the rotary positions), or, where `own` is true, by the calls a user of torch_engine_b200 makes.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}

_backends = {}


def _backend():
    """The framework's handle for the current device, made once as a user's program makes it."""
    from torch_engine_b200 import ops
    dev = torch.cuda.current_device()
    if dev not in _backends:
        _backends[dev] = ops.Backend(dev, workspace_bytes=64 << 20)
    return _backends[dev]


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step: 32 query and 8 key heads of eight sequences far into a long context, as one view
        _rotary("rotary decode", batch=8, heads=40, tokens=1, d=128, rot=128, far=131072),
        # the GPT step of the benchmark configuration: q and k head views inside the projections' buffer, forward
        _rotary("rotary gpt step", batch=64, heads=12, tokens=256, d=64, rot=64, far=0, packed=True),
        # a training step on a long sequence: backward, interleaved pairs, half of the head, positions stretched by parts
        _rotary("rotary backward long", batch=1, heads=32, tokens=8191, d=128, rot=64, far=0, interleaved=True, backward=True, stretch=8.0),
        # one new token of each of 64 sequences goes into the cache
        _append("append decode bf16", dtype="bf16", batch=64, heads=8, tokens=1, d=128, page=16),
        # the GPT configuration's keys and values, taken from the projections' buffer, kept at full precision
        _append("append gpt f32", dtype="f32", batch=64, heads=6, tokens=256, d=64, page=16, packed=True),
        # prompts of unlike length, padded to the longest, into a half-precision cache
        _append("append prompt bf16", dtype="bf16", batch=8, heads=8, tokens=2001, d=128, page=16, ragged=True),
        # prompts quantised as they are written and read back, pages larger than the remainder of a prompt
        _append("append read e4m3", dtype="e4m3", batch=4, heads=8, tokens=4093, d=128, page=64, ragged=True, read=True),
        # one sequence of the GPT configuration: a call where latency counts
        _attention("attention gpt one", dtype="f32", rows=1, q_heads=6, kv_heads=6, d=64, page=16, longest=200),
        # the GPT configuration's batch at a context four times its own
        _attention("attention gpt batch", dtype="f32", rows=64, q_heads=6, kv_heads=6, d=64, page=16, longest=1024),
        # serving with shared key heads, lengths spread over two decades
        _attention("attention grouped bf16", dtype="bf16", rows=32, q_heads=32, kv_heads=8, d=128, page=16, longest=16384),
        # every head with its own keys, an uncommon head size, odd pages, the last 4096 tokens only
        _attention("attention window bf16", dtype="bf16", rows=16, q_heads=20, kv_heads=20, d=80, page=13, longest=9001, window=4096),
        # two very long contexts in a quantised cache, eight query heads a key head
        _attention("attention long e4m3", dtype="e4m3", rows=2, q_heads=64, kv_heads=8, d=128, page=64, longest=131072),
    ]


def _rotary(name, *, batch, heads, tokens, d, rot, far, packed=False, interleaved=False, backward=False, stretch=1.0):
    return {"name": name, "op": "rotary", "batch": batch, "heads": heads, "tokens": tokens, "d": d, "rot": rot, "far": far, "packed": packed,
            "interleaved": interleaved, "backward": backward, "stretch": stretch}


def _append(name, *, dtype, batch, heads, tokens, d, page, packed=False, ragged=False, read=False):
    return {"name": name, "op": "append", "dtype": dtype, "batch": batch, "heads": heads, "tokens": tokens, "d": d, "page": page,
            "packed": packed, "ragged": ragged, "read": read}


def _attention(name, *, dtype, rows, q_heads, kv_heads, d, page, longest, window=0):
    return {"name": name, "op": "attention", "dtype": dtype, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "d": d, "page": page,
            "longest": longest, "window": window}


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attention"))
    d = rng.choice((32, 48, 64, 64, 80, 96, 112, 128, 128, 128, 192, 256))
    page = rng.choice((16, 16, 32, 64, 128, _spread(rng, 1, 300)))
    if op == "rotary":
        heads = rng.randint(1, 48)
        elements = _spread(rng, 2000, 32 * 8191 * 128)
        tokens = max(1, elements // (heads * d))
        batch = rng.choice((1, tokens, max(1, min(tokens, _spread(rng, 1, 64)))))
        case = _rotary("", batch=batch, heads=heads, tokens=max(1, tokens // batch), d=d, rot=rng.choice((d, d, d // 2, 2 * rng.randint(1, d // 2))),
                       far=rng.choice((0, _spread(rng, 1, 1000000))), packed=rng.random() < 0.4, interleaved=rng.random() < 0.5,
                       backward=rng.random() < 0.5, stretch=rng.choice((1.0, 1.0, round(rng.uniform(2.0, 32.0), 2))))
    elif op == "append":
        heads = rng.randint(1, 16)
        elements = _spread(rng, 2000, 4 * 8 * 4093 * 128)
        tokens = max(1, elements // (heads * d))
        batch = rng.choice((tokens, max(1, min(tokens, _spread(rng, 1, 64))))) if tokens <= 512 else min(tokens, _spread(rng, 1, 64))
        dtype = rng.choice(("f32", "bf16", "e4m3"))
        case = _append("", dtype=dtype, batch=batch, heads=heads, tokens=max(1, tokens // batch), d=d, page=page, packed=rng.random() < 0.4,
                       ragged=rng.random() < 0.5, read=dtype == "e4m3" or rng.random() < 0.3)
    else:
        dtype = rng.choice(("f32", "bf16", "bf16", "e4m3"))
        kv_heads = rng.choice((1, 2, 4, 6, 8, 8, 16, rng.randint(1, 20)))
        group = rng.choice((1, 1, 2, 4, 4, 8, 16, rng.randint(1, 16)))
        elements = _spread(rng, 4000, 2 * 8 * 131072 * 128 // 4)     # of the keys, at the longest length in every row
        places = max(1, elements // (kv_heads * d))
        rows = rng.choice((1, max(1, min(places, _spread(rng, 1, 256))), max(1, min(places, _spread(rng, 1, 256)))))
        longest = min(131072, max(1, places // rows))
        case = _attention("", dtype=dtype, rows=rows, q_heads=kv_heads * group, kv_heads=kv_heads, d=d, page=page, longest=longest,
                          window=rng.choice((0, 0, 0, _spread(rng, 1, longest))))
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"rotary": _prepare_rotary, "append": _prepare_append, "attention": _prepare_attention}[case["op"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen)


def _integers(gen, low, high, *shape):
    """Whole numbers in [low, high]."""
    return torch.randint(low, high + 1, shape, device="cuda", dtype=torch.int64, generator=gen)


def _head_views(gen, case, count):
    """`count` head views [batch, heads, tokens, d]: column blocks of one projections' buffer where packed, else tensors of their own."""
    b, h, t, d = case["batch"], case["heads"], case["tokens"], case["d"]
    if case["packed"]:
        # rotary: the q and k blocks of a buffer whose last third is v; append: the k and v blocks behind q
        skip, extra = (0, (h + 1) // 2) if count == 1 else (h, 0)
        buffer = _normal(gen, b, t, (skip + count * h + extra) * d)
        return [buffer[:, :, (skip + i * h) * d:(skip + (i + 1) * h) * d].view(b, t, h, d).transpose(1, 2) for i in range(count)]
    return [_normal(gen, b, h, t, d) for _ in range(count)]


def _prepare_rotary(case, gen):
    (x,) = _head_views(gen, case, 1)
    rot, stretch = case["rot"], case["stretch"]
    j = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64)
    inv_freq, amplitude = 10000.0 ** (-j / rot), 1.0
    if stretch != 1.0:      # long contexts: slow pairs are stretched, fast ones kept, a ramp between 1 and 32 turns over 4096 tokens
        keep = ((4096 * inv_freq / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        inv_freq = inv_freq * (keep + (1.0 - keep) / stretch)
        amplitude = 0.1 * math.log(stretch) + 1.0
    start = _integers(gen, 0, case["far"], case["batch"], 1)
    positions = start + torch.arange(case["tokens"], device="cuda")
    return {"case": dict(case), "x": x, "positions": positions, "inv_freq": inv_freq.contiguous(), "amplitude": amplitude}


def _page_table(gen, lengths, page, pages):
    """Pages for rows of these lengths (host numbers), in the scattered order that a cache in use has; -1 where a row needs none.
    `pages`: how many the cache has, None for a few more than the rows need."""
    need = [-(-n // page) for n in lengths]
    width, total = max(1, max(need)), pages or sum(need) + 2
    order = torch.randperm(total, device="cuda", generator=gen)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda").unsqueeze(1)
    count = torch.tensor(need, device="cuda").unsqueeze(1)
    i = torch.arange(width, device="cuda").unsqueeze(0)
    return torch.where(i < count, order[(first + i).clamp(max=total - 1)], -1), total


def _ragged(gen, count, longest):
    """Lengths spread over two decades up to `longest`, the first the longest itself."""
    u = torch.rand(count, device="cuda", generator=gen)
    n = (longest * 100.0 ** (-u)).round().long().clamp(min=min(1, longest))
    n[0] = longest
    return n


def _prepare_append(case, gen):
    b, h, t, d, page, dtype = (case[n] for n in ("batch", "heads", "tokens", "d", "page", "dtype"))
    k, v = _head_views(gen, case, 2)
    n = _ragged(gen, b, t) if case["ragged"] else torch.full((b,), t, device="cuda")
    before = 37 if t == 1 else 0          # a decode step finds some tokens in the cache
    lengths = (n + before).tolist()
    page_table, pages = _page_table(gen, lengths, page, b * -(-(t + before) // page) + 1)
    at = torch.arange(t, device="cuda").unsqueeze(0)
    positions = torch.where(at < n.unsqueeze(1), at + before, -1)
    k_cache, v_cache, k_scale, v_scale = _cache(gen, case, pages)
    s = {"case": dict(case), "k": k, "v": v, "page_table": page_table, "positions": positions, "k_cache": k_cache, "v_cache": v_cache,
         "k_scale": k_scale, "v_scale": v_scale}
    if own:
        s["handle"] = _handle(s)
    return s


def _handle(s):
    from torch_engine_b200 import ops
    return ops.KvCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])


def _cache(gen, case, pages):
    """A cache of this many pages, [pages, heads, page, d], filled as by earlier tokens."""
    shape = (pages, case.get("heads") or case["kv_heads"], case["page"], case["d"])
    dtype = case["dtype"]
    k, v = _normal(gen, *shape), _normal(gen, *shape)
    k *= 1.0 + 0.5 * torch.sin(torch.arange(shape[3], device="cuda"))    # some columns of keys are larger than others
    if dtype != "e4m3":
        return k.to(_DTYPES[dtype]), v.to(_DTYPES[dtype]), None, None
    (k, k_scale), (v, v_scale) = _quantised(k), _quantised(v)
    return k, v, k_scale, v_scale


def _prepare_attention(case, gen):
    rows, longest, page = case["rows"], case["longest"], case["page"]
    lens = _ragged(gen, rows, longest)
    if rows > 2:
        lens[rows // 2] = 0               # a row of the batch that holds no sequence
    page_table, pages = _page_table(gen, lens.tolist(), page, None)
    k_cache, v_cache, k_scale, v_scale = _cache(gen, case, pages)
    q = 1.5 * _normal(gen, rows, case["q_heads"], case["d"])
    s = {"case": dict(case), "q": q, "lens": lens, "page_table": page_table, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale,
         "v_scale": v_scale}
    if own:
        s["handle"] = _handle(s)
    return s


# -------------------------------------------------------------------------------------------------------- the operators
def run(state):
    return {"rotary": _run_rotary, "append": _run_append, "attention": _run_attention}[state["case"]["op"]](state)


def _run_rotary(s):
    c = s["case"]
    if own:
        be = _backend()
        call = be.rotary_backward if c["backward"] else be.rotary
        return call(s["x"], s["positions"], s["inv_freq"], interleaved=c["interleaved"], scale=s["amplitude"])
    x, rot = s["x"], c["rot"]
    angle = s["positions"].unsqueeze(-1).double() * s["inv_freq"]
    cos, sin = (s["amplitude"] * torch.cos(angle)).float().unsqueeze(1), (s["amplitude"] * torch.sin(angle)).float().unsqueeze(1)
    if c["backward"]:
        sin = -sin
    if c["interleaved"]:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1).flatten(-2)
    else:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _quantised(x):
    """e4m3 values and the power of two each row is measured in: the smallest that brings the row's largest magnitude to at most 448."""
    amax = x.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(amax)              # amax = mantissa * 2^exponent, mantissa in [1/2, 1); 448 = 7/8 * 2^9
    e = (exponent - 9 + (mantissa > 0.875)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(amax), e)
    return (x * torch.ldexp(torch.ones_like(amax), -e).unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def _places(page_table, positions, page):
    index = (positions.clamp(min=0) // page).clamp(max=page_table.shape[1] - 1)
    return page_table.gather(1, index).clamp(min=0), positions.clamp(min=0) % page


def _run_append(s):
    c = s["case"]
    if own:
        be = _backend()
        be.kv_append(s["handle"], s["k"], s["v"], s["page_table"], s["positions"])
        if c["read"]:
            return be.kv_read(s["handle"], s["page_table"], s["positions"])
        return s["k_cache"], s["v_cache"]
    pages, slots = _places(s["page_table"], s["positions"], c["page"])
    there = s["positions"] >= 0
    p, o = pages[there], slots[there]
    read = []
    for cache, scales, x in ((s["k_cache"], s["k_scale"], s["k"]), (s["v_cache"], s["v_scale"], s["v"])):
        rows = x.transpose(1, 2)[there]                 # [tokens that are there, heads, d]
        if scales is None:
            cache[p, :, o] = rows.to(cache.dtype)
        else:
            codes, scale = _quantised(rows)
            cache.view(torch.uint8)[p, :, o] = codes.view(torch.uint8)
            scales[p, :, o] = scale
        if c["read"]:
            if scales is None:
                back = cache[pages, :, slots].float()
            else:
                back = cache.view(torch.uint8)[pages, :, slots].view(torch.float8_e4m3fn).float() * scales[pages, :, slots].unsqueeze(-1)
            read.append(torch.where(there[:, :, None, None], back, 0.0).transpose(1, 2))
    return tuple(read) if c["read"] else (s["k_cache"], s["v_cache"])


def _run_attention(s):
    c = s["case"]
    if own:
        return _backend().paged_attention(s["q"], s["handle"], s["page_table"], s["lens"], window=c["window"], want_lse=True)
    rows, hq, hk, d = c["rows"], c["q_heads"], c["kv_heads"], c["d"]
    at = torch.arange(c["longest"], device="cuda").unsqueeze(0).expand(rows, -1)
    pages, slots = _places(s["page_table"], at, c["page"])
    lens = s["lens"].unsqueeze(1)
    seen = at < lens
    if c["window"]:
        seen = seen & (at >= lens - c["window"])
    k, v = _gathered(s["k_cache"], s["k_scale"], pages, slots), _gathered(s["v_cache"], s["v_scale"], pages, slots)
    q = s["q"].view(rows, hk, hq // hk, d)
    scores = torch.einsum("rhgd,rlhd->rhgl", q, k) * d ** -0.5
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(dim=-1, keepdim=True)
    o = torch.einsum("rhgl,rlhd->rhgd", weights, v) / torch.where(total == 0.0, 1.0, total)
    return o.reshape(rows, hq, d), (top + torch.log(total)).reshape(rows, hq)


def _gathered(cache, scales, pages, slots):
    if scales is None:
        return cache[pages, :, slots].float()
    return cache.view(torch.uint8)[pages, :, slots].view(torch.float8_e4m3fn).float() * scales[pages, :, slots].unsqueeze(-1)


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        return {"bytes": 8.0 * tokens * case["heads"] * case["d"] + 8.0 * tokens, "flops": 3.0 * tokens * case["heads"] * case["rot"]}
    size = _BYTES[case["dtype"]]
    if case["op"] == "append":
        share = _mean_share(case["tokens"]) if case["ragged"] else 1.0
        rows = 2.0 * case["batch"] * case["tokens"] * case["heads"]         # of keys and of values
        kept = rows * (case["d"] * size + (4 if case["dtype"] == "e4m3" else 0))
        moved = share * (4.0 * rows * case["d"] + kept) + 8.0 * case["batch"] * case["tokens"]
        if case["read"]:
            moved += share * kept + 4.0 * rows * case["d"]
        return {"bytes": moved, "flops": rows * case["d"]}
    longest, window = case["longest"], case["window"]
    sizes = [longest] + [_mean_length(longest, window)] * (case["rows"] - 1 - (case["rows"] > 2))
    places = sum(min(n, window) if window else n for n in sizes)
    bytes_ = 2.0 * places * case["kv_heads"] * (case["d"] * size + (4 if case["dtype"] == "e4m3" else 0)) + 8.0 * case["rows"] * case["q_heads"] * case["d"]
    return {"bytes": bytes_, "flops": 4.0 * places * case["q_heads"] * case["d"]}


def _mean_share(longest):
    return _mean_length(longest, 0) / longest


def _mean_length(longest, window):
    """The mean of min(longest * 100^-u, window) over u in [0, 1], at least 1."""
    steps = 512
    values = [max(1.0, longest * 100.0 ** (-(i + 0.5) / steps)) for i in range(steps)]
    return sum(min(n, window) if window else n for n in values) / steps


# ----------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attention": _exact_attention}[case["op"]](s)


def _exact_rotary(s):
    c, rot = s["case"], s["case"]["rot"]
    turn = torch.polar(torch.full_like(s["inv_freq"], s["amplitude"]).expand(c["batch"], 1, c["tokens"], rot // 2).contiguous(),
                       (s["positions"].double()[:, None, :, None] * s["inv_freq"]))
    if c["backward"]:
        turn = turn.conj()
    out = s["x"].double().contiguous()
    parts = out[..., :rot].unflatten(-1, (rot // 2, 2) if c["interleaved"] else (2, rot // 2))
    axis = -1 if c["interleaved"] else -2
    z = torch.complex(parts.select(axis, 0), parts.select(axis, 1)) * turn
    out[..., :rot] = torch.stack((z.real, z.imag), dim=axis).flatten(-2)
    return out


def _to_grid(x):
    """Rows of x [..., d] on the e4m3 grid of their own power of two, half way to even."""
    x = x.double()
    top = x.abs().amax(dim=-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -110) / E4M3_MAX)))
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * unit


def _exact_append(s):
    c = s["case"]
    quantised = c["dtype"] == "e4m3"
    outs = []
    for cache, x in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        if c["read"]:
            out = torch.zeros(x.shape, device="cuda", dtype=torch.float64)
        else:
            out = cache.double()
        for b in range(c["batch"]):
            where = (s["positions"][b] >= 0).nonzero().flatten()
            at = s["positions"][b, where]
            rows = _to_grid(x[b, :, where]) if quantised else x[b, :, where].double()
            if c["read"]:
                out[b, :, where] = rows if quantised else rows.to(_DTYPES[c["dtype"]]).double()
            else:
                out[s["page_table"][b, torch.div(at, c["page"], rounding_mode="floor")], :, at % c["page"]] = rows.transpose(0, 1)
        outs.append(out)
    return tuple(outs)


def _exact_attention(s):
    c = s["case"]
    hk, group, d = c["kv_heads"], c["q_heads"] // c["kv_heads"], c["d"]
    o = torch.zeros(c["rows"], c["q_heads"], d, device="cuda", dtype=torch.float64)
    lse = torch.full((c["rows"], c["q_heads"]), -math.inf, device="cuda", dtype=torch.float64)
    for r, n in enumerate(s["lens"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n <= first:
            continue
        used = s["page_table"][r, :-(-n // c["page"])]
        k, v = (_exact_pages(s[x + "_cache"], s[x + "_scale"], used)[:, first:n] for x in "kv")
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            scores = (s["q"][r, heads].double() @ k[h].T) / math.sqrt(d)
            lse[r, heads] = torch.logsumexp(scores, dim=-1)
            o[r, heads] = torch.softmax(scores, dim=-1) @ v[h]
    return o, lse


def _exact_pages(cache, scales, used):
    """The tokens of these pages one after another, [heads, tokens, d]."""
    x = cache[used].double() if scales is None else cache.view(torch.uint8)[used].view(torch.float8_e4m3fn).double() * scales[used].double().unsqueeze(-1)
    return x.transpose(0, 1).flatten(1, 2)
