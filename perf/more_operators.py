"""Performance cases of the decoding operators: what a program that generates several
sequences behind a shared prompt does at every step, besides its projections.

  append     the heads of new tokens, read in place from the packed projection
             [batch, token, q | k | v]: queries and keys turned by their positions, keys
             and values written to the pages of a cache; padded tokens are not written
  attention  queries over a prefix that several sequences share (read once for all of
             them) and each sequence's own keys, causal, through tables of pages
  beams      the best continuations of every group of beams over the whole vocabulary,
             log-softmax included, and the rows of states (token histories, page tables,
             a recurrent state) put in the order of the beams they go on from

With `own` false, run() computes a case from elementary torch operations;
with `own` true it calls the framework's C ABI on the same tensors, whose
values are complete when run() is called; its outputs are complete once the
device has been synchronised (the framework has a stream of its own).  A case is
a dict of plain values.
`listed()` gives the named cases and `draw(rng)` one more of the same ranges.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float64": torch.float64}


# ------------------------------------------------------------------- cases

def _append(batch, tokens, heads, key_heads, width, rotary, layout, page, start, padded,
            dtype="float32"):
    return {"kind": "append", "batch": batch, "tokens": tokens, "heads": heads,
            "key_heads": key_heads, "width": width, "rotary": rotary, "layout": layout,
            "page": page, "start": start, "padded": padded, "dtype": dtype}


def _attention(batch, prefixes, heads, key_heads, width, queries, prefix, prefix_shortest,
               prefix_page, tokens, shortest, page, dtype="float32"):
    return {"kind": "attention", "batch": batch, "prefixes": prefixes, "heads": heads,
            "key_heads": key_heads, "width": width, "queries": queries, "prefix": prefix,
            "prefix_shortest": prefix_shortest, "prefix_page": prefix_page, "tokens": tokens,
            "shortest": shortest, "page": page, "dtype": dtype}


def _beams(groups, beams, vocabulary, picks, first, ended, masked, history, slots, state,
           dtype="float32"):
    return {"kind": "beams", "groups": groups, "beams": beams, "vocabulary": vocabulary,
            "picks": picks, "first": first, "ended": ended, "masked": masked, "history": history,
            "slots": slots, "state": state, "dtype": dtype}


def listed():
    return [
        # the next token of 64 sequences into pages of 16: launches count
        {"name": "append_token", **_append(64, 1, 32, 8, 128, 128, "half", 16, 900, False)},
        # four prompts of 4096 tokens
        {"name": "append_prompts", **_append(4, 4096, 32, 8, 128, 128, "half", 64, 0, False)},
        # double precision, heads turned in part, odd pages, prompts padded in front
        {"name": "append_odd", **_append(3, 1021, 12, 3, 80, 32, "interleaved", 5, 17, True,
                                         "float64")},
        # the next token of 4 answers to one short prompt: latency counts
        {"name": "attention_small", **_attention(4, 1, 16, 4, 64, 1, 512, 512, 0, 48, 1, 16)},
        # the next token of 16 conversations behind one long instruction
        {"name": "attention_token", **_attention(16, 1, 32, 8, 128, 1, 8192, 8192, 0, 2048, 500,
                                                 16)},
        # the next token of 64 conversations behind a longer one in pages
        {"name": "attention_shared", **_attention(64, 1, 32, 8, 128, 1, 16384, 16384, 64, 2048,
                                                  257, 64)},
        # beam search over 8 prompts of different lengths with 8 beams each, whose own
        # tokens move between beams by page tables: pages of one token
        {"name": "attention_beams", **_attention(64, 8, 16, 16, 64, 1, 2048, 900, 128, 200, 100,
                                                 1)},
        # 256 tokens at a time of 4 prompts behind one instruction
        {"name": "attention_chunk", **_attention(4, 1, 32, 8, 128, 256, 4096, 4096, 0, 1024, 300,
                                                 32)},
        # double precision, odd sizes, a prompt and sequences of no tokens
        {"name": "attention_double", **_attention(6, 2, 6, 2, 72, 3, 333, 0, 5, 50, 0, 5,
                                                  "float64")},
        # the next tokens of 4 beams of one prompt: latency counts
        {"name": "beams_small", **_beams(1, 4, 32000, 4, False, False, False, 256, 256, 0)},
        # 32 prompts of 8 beams and a large vocabulary
        {"name": "beams_batch", **_beams(32, 8, 131072, 8, False, True, False, 512, 2048, 0)},
        # twice as many picks as beams, banned tokens, an odd vocabulary and a recurrent
        # state to move
        {"name": "beams_state", **_beams(16, 5, 50257, 10, False, False, True, 77, 0, 65536)},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low),
                                                             math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "beams"])
    dtype = "float32" if rng.random() < 0.85 else "float64"
    if kind == "beams":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16])
        groups = _log(rng, 1, 64)
        vocabulary = _log(rng, 8, min(200000, (1 << 25) // (groups * beams)))
        picks = rng.choice([beams, beams, 2 * beams])
        return _beams(groups, beams, vocabulary, picks, rng.random() < 0.2, rng.random() < 0.4,
                      rng.random() < 0.3, _log(rng, 1, 4096), rng.choice([0, _log(rng, 1, 4096)]),
                      rng.choice([0, 0, _log(rng, 1, min(1 << 17, (1 << 25) // (groups * beams)))]),
                      dtype)
    width = rng.choice([32, 40, 64, 64, 72, 80, 96, 100, 128, 128, 128, 160, 192, 256])
    key_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    heads = min(32, key_heads * group) // key_heads * key_heads
    page = rng.choice([1, 5, 16, 16, 32, 64, 128])
    if kind == "append":
        rotary = width if rng.random() < 0.6 else 2 * rng.randint(0, width // 2)
        token = rng.random() < 0.4
        most = (1 << (26 if dtype == "float32" else 25)) // (width * (heads + 2 * key_heads))
        batch = _log(rng, 1, 256 if token else 16)
        tokens = 1 if token else _log(rng, 2, max(2, min(8192, most // batch)))
        return _append(batch, tokens, heads, key_heads, width, rotary,
                       rng.choice(["half", "interleaved"]), page, _log(rng, 1, 2000),
                       rng.random() < 0.3, dtype)
    prefixes = rng.choice([1, 1, 1, 2, 3, 8])
    batch = prefixes * _log(rng, 1, 64 // prefixes)
    queries = rng.choice([1, 1, 1, 1, 2, 4, 7, _log(rng, 1, 256)])
    # at most 2^26 elements in each of the prefixes' keys and the sequences' own, and 2^35
    # operations of either (2^34 in double)
    most = (1 << (33 if dtype == "float32" else 32)) // (batch * heads * queries * width)
    prefix = _log(rng, 1, min(16384, (1 << 26) // (prefixes * key_heads * width), most))
    tokens = _log(rng, queries, min(4096, (1 << 26) // (batch * key_heads * width), most))
    return _attention(batch, prefixes, heads, key_heads, width, queries, prefix,
                      prefix if rng.random() < 0.5 else rng.randint(0, prefix),
                      rng.choice([0, 1, 16, 64, 100, 128]), tokens, rng.randint(0, tokens), page,
                      dtype)


def _spread(most, least, count):
    """Lengths from `most` down to `least`."""
    return [most - (most - least) * i // max(1, count - 1) for i in range(count)]


# ------------------------------------------------------------- preparation

def _table(lengths, width, page, generator, device):
    """Tables of pages in no order, -1 behind each sequence's last page, and the number
    of pages."""
    needs = torch.tensor([(n + page - 1) // page for n in lengths], device=device)
    used = torch.arange(width, device=device) < needs[:, None]
    pages = int(needs.sum())
    table = torch.full(used.shape, -1, dtype=torch.int32, device=device)
    table[used] = torch.randperm(pages, generator=generator, device=device).int()
    return table, pages


def prepare(case, seed):
    """What a program holds before the call, on the GPU."""
    device = torch.device("cuda")
    dtype = _DTYPES[case["dtype"]]
    generator = torch.Generator(device=device)
    generator.manual_seed(int(seed) * 1000003 + 31)

    def normal(*shape):
        return torch.randn(shape, generator=generator, device=device, dtype=dtype)

    def whole(low, high, shape, kind):
        return torch.randint(low, high, shape, generator=generator, device=device, dtype=kind)

    state = {"case": case}
    if case["kind"] == "beams":
        rows, v = case["groups"] * case["beams"], case["vocabulary"]
        state["logits"] = normal(rows, v) * 3
        if case["masked"]:
            state["logits"][:, torch.rand(v, generator=generator, device=device) < 0.1] = -math.inf
        state["scores"] = -10 * torch.rand(rows, generator=generator, device=device, dtype=dtype)
        if case["first"]:  # all beams are the prompt: the first goes on alone
            state["scores"] = torch.full((case["groups"], case["beams"]), -math.inf, device=device,
                                         dtype=dtype)
            state["scores"][:, 0] = 0
            state["scores"] = state["scores"].flatten()
        state["end"] = v // 3
        state["ended"] = None
        if case["ended"]:
            state["ended"] = (torch.rand(rows, generator=generator, device=device) < 0.2).int()
        state["states"] = [whole(0, v, (rows, case["history"]), torch.int64)]
        if case["slots"]:
            state["states"].append(whole(0, 1 << 20, (rows, case["slots"]), torch.int32))
        if case["state"]:
            state["states"].append(normal(rows, case["state"]))
        return state
    b, h, hk, d, page = (case[k] for k in ("batch", "heads", "key_heads", "width", "page"))
    if case["kind"] == "append":
        t = case["tokens"]
        starts = _spread(case["start"], case["start"] // 2, b)
        lengths = torch.tensor(starts, device=device) + t
        most = (case["start"] + t + page - 1) // page
        state["table"], pages = _table(lengths.tolist(), most, page, generator, device)
        state["places"] = lengths[:, None] - t + torch.arange(t, device=device)
        if case["padded"]:  # all but the last of a sequence's tokens may be padding
            padding = whole(0, t, (b, 1), torch.int64)
            state["places"] = torch.where(torch.arange(t, device=device) < padding, -1,
                                          state["places"])
        state["positions"] = state["places"].clamp(min=0) + 100
        r = case["rotary"]
        state["frequencies"] = 10000.0 ** (
            -torch.arange(r // 2, device=device, dtype=torch.float64) * 2 / max(r, 1))
        state["packed"] = normal(b, t, (h + 2 * hk) * d)
        state["key"], state["value"] = normal(pages, hk, page, d), normal(pages, hk, page, d)
        return state
    t = case["queries"]
    state["query"] = normal(b, t, h, d)
    lengths = _spread(case["tokens"], case["shortest"], b)
    width = (case["tokens"] + page - 1) // page
    state["table"], pages = _table(lengths, width, page, generator, device)
    state["key"], state["value"] = normal(pages, hk, page, d), normal(pages, hk, page, d)
    state["lengths"] = torch.tensor(lengths, device=device, dtype=torch.int32)
    lengths = _spread(case["prefix"], case["prefix_shortest"], case["prefixes"])
    page = case["prefix_page"]
    state["prefix_table"], pages = None, case["prefixes"]
    if page:
        width = (case["prefix"] + page - 1) // page
        state["prefix_table"], pages = _table(lengths, width, page, generator, device)
    shape = (pages, hk, page or case["prefix"], d)
    state["prefix_key"], state["prefix_value"] = normal(*shape), normal(*shape)
    state["prefix_lengths"] = torch.tensor(lengths, device=device, dtype=torch.int32)
    return state


def _heads(state):
    """The views of the query, key and value heads in the packed projection."""
    case = state["case"]
    b, t, h, hk, d = (case[k] for k in ("batch", "tokens", "heads", "key_heads", "width"))
    every = state["packed"].view(b, t, h + 2 * hk, d)
    return every[:, :, :h], every[:, :, h:h + hk], every[:, :, h + hk:]


# -------------------------------------------------------------- plain forms

def _turned(x, cos, sin, case):
    r = case["rotary"]
    y = x.clone()
    if case["layout"] == "half":
        first, second = slice(0, r // 2), slice(r // 2, r)
    else:
        first, second = slice(0, r, 2), slice(1, r, 2)
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., second] * cos + x[..., first] * sin
    return y


def _plain_append(state):
    case = state["case"]
    query, key, value = _heads(state)
    page, places = case["page"], state["places"]
    angle = (state["positions"].double()[:, :, None] * state["frequencies"])[:, :, None]
    cos, sin = angle.cos().to(query.dtype), angle.sin().to(query.dtype)
    sequence, token = torch.nonzero(places >= 0, as_tuple=True)
    place = places[sequence, token]
    at = state["table"][sequence, place // page].long(), slice(None), place % page
    state["key"][at] = _turned(key, cos, sin, case)[sequence, token]
    state["value"][at] = value[sequence, token]
    return {"query": _turned(query, cos, sin, case), "key": state["key"], "value": state["value"]}


def _gathered(pool, table):
    """[row, key head, token, width] of a pool's pages."""
    if table is None:
        return pool
    rows, n = table.shape
    pages = pool[table.clamp(min=0).long()]
    return pages.permute(0, 2, 1, 3, 4).reshape(rows, pool.shape[1], n * pool.shape[2],
                                                pool.shape[3])


def _plain_attention(state):
    case, query = state["case"], state["query"]
    b, p, h, hk, d, t = (case[k] for k in ("batch", "prefixes", "heads", "key_heads", "width",
                                           "queries"))
    g, s, device = h // hk, b // p, query.device
    scaled = (query * (1 / math.sqrt(d))).view(b, t, hk, g, d)
    at = state["lengths"].long()[:, None] - t + torch.arange(t, device=device)  # [b, t]

    # the sharers' rows of a prefix together: [p, hk, s * t * g, d]
    shared = scaled.view(p, s, t, hk, g, d).permute(0, 3, 1, 2, 4, 5).reshape(p, hk, s * t * g, d)
    key = _gathered(state["prefix_key"], state["prefix_table"])
    scores = torch.matmul(shared, key.transpose(2, 3)).view(p, hk, s, t, g, -1)
    behind = torch.arange(key.shape[2], device=device) >= state["prefix_lengths"].long()[:, None]
    scores.masked_fill_(behind[:, None, None, None, None] |
                        (at < 0).view(p, 1, s, t, 1, 1), -math.inf)
    single = scaled.permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, d)
    key = _gathered(state["key"], state["table"])
    own_scores = torch.matmul(single, key.transpose(2, 3)).view(b, hk, t, g, -1)
    hidden = torch.arange(key.shape[2], device=device) > at[:, :, None]
    own_scores.masked_fill_(hidden[:, None, :, None], -math.inf)

    def by_row(x):  # [p, hk, s, t, g, n] in the order of [b, hk, t, g, n]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(b, hk, t, g, -1)

    top = torch.maximum(by_row(scores.amax(-1, keepdim=True)), own_scores.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(top.view(p, s, hk, t, g, 1).transpose(1, 2)).exp_()
    own_weights = own_scores.sub_(top).exp_()
    total = by_row(weights.sum(-1, keepdim=True)) + own_weights.sum(-1, keepdim=True)
    value = _gathered(state["prefix_value"], state["prefix_table"])
    out = torch.matmul(weights.view(p, hk, s * t * g, -1), value).view(p, hk, s, t, g, d)
    value = _gathered(state["value"], state["table"])
    out = by_row(out) + torch.matmul(own_weights.view(b, hk, t * g, -1),
                                     value).view(b, hk, t, g, d)
    out = out / torch.where(total == 0, 1.0, total)
    return {"output": out.permute(0, 2, 1, 3, 4).reshape(b, t, h, d)}


def _plain_beams(state):
    case, logits = state["case"], state["logits"]
    groups, beams, v = case["groups"], case["beams"], case["vocabulary"]
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    log_sum = (x - top).exp_().sum(-1, keepdim=True).log()
    totals = state["scores"].double()[:, None] + (x - (top + log_sum))
    totals = torch.where(totals.isnan(), -math.inf, totals)
    if state["ended"] is not None:  # goes on with the end token alone, at no cost
        alone = torch.full_like(totals, -math.inf)
        alone[:, state["end"]] = state["scores"].double()
        totals = torch.where(state["ended"][:, None] != 0, alone, totals)
    order = totals.view(groups, beams * v).sort(dim=-1, descending=True, stable=True)
    picked = order.indices[:, :case["picks"]]
    parents = (picked // v + beams * torch.arange(groups, device=x.device)[:, None])
    tokens = picked % v
    made = {"scores": order.values[:, :case["picks"]].to(logits.dtype), "parents": parents,
            "tokens": tokens}
    if state["ended"] is not None:
        made["ended"] = ((state["ended"][parents] != 0) | (tokens == state["end"])).int()
    made["states"] = [x[parents.flatten()] for x in state["states"]]
    return made


# --------------------------------------------------- the framework's calls

def _strides(x):
    """(batch, head, token) strides of a [batch, token, head, width] tensor."""
    return x.stride(0), x.stride(2), x.stride(1)


def _pages(key, value, table, lengths_bound):
    """A pool [page, key head, token, width] with its table, or rows that are a page each."""
    from spar_amd import hip

    return hip.pages(key.data_ptr(), key.stride()[:3], value.data_ptr(), value.stride()[:3],
                     key.shape[0], key.shape[2] if table is not None else lengths_bound,
                     None if table is None else table.data_ptr(),
                     0 if table is None else table.stride(0),
                     1 if table is None else table.shape[1])


def _scratch(state, name, like, count, dtype=None):
    """Device memory that calls write and read but do not return.  The state keeps it,
    as a program does: torch would hand memory dropped here to kernels of its own
    stream while the framework's stream still works in it."""
    held = state.setdefault("scratch", {})
    if name not in held:
        held[name] = torch.empty(count, dtype=dtype or like.dtype, device=like.device)
    return held[name]


def _own_append(state):
    from spar_amd import hip

    case = state["case"]
    query, key, value = _heads(state)
    b, t, h, d = query.shape
    places, positions = state["places"], state["positions"]
    turned = query.new_empty(b, t, h, d)
    rotary = hip.rotary(positions.data_ptr(), positions.stride(0), hip.INT64,
                        state["frequencies"].data_ptr(), case["rotary"], 1.0,
                        hip.ROTARY_HALF if case["layout"] == "half" else hip.ROTARY_INTERLEAVED)
    hip.call("spar_hip_launch_cache_append",
             _pages(state["key"], state["value"], state["table"], 0),
             hip.heads(turned.data_ptr(), _strides(turned)),
             hip.heads(query.data_ptr(), _strides(query)), h,
             hip.heads(key.data_ptr(), _strides(key)), hip.heads(value.data_ptr(), _strides(value)),
             b, case["key_heads"], t, d, places.data_ptr(), places.stride(0), hip.INT64, rotary,
             hip.dtype_tag(case["dtype"]), 0)
    return {"query": turned, "key": state["key"], "value": state["value"]}


def _own_attention(state):
    from spar_amd import hip

    case, query = state["case"], state["query"]
    b, t, h, d = query.shape
    output = torch.empty_like(query)
    shape = hip.cache_attention(b, case["prefixes"], h, case["key_heads"], t, d, 1 / math.sqrt(d),
                                state["lengths"].data_ptr(), state["prefix_lengths"].data_ptr(),
                                hip.INT32, hip.dtype_tag(case["dtype"]))
    cache = _pages(state["key"], state["value"], state["table"], 0)
    prefix = _pages(state["prefix_key"], state["prefix_value"], state["prefix_table"],
                    case["prefix"])
    need = hip.cache_attention_workspace(cache, prefix, shape)
    workspace = _scratch(state, "attention", query, need, torch.uint8)
    hip.call("spar_hip_launch_cache_attention", hip.heads(output.data_ptr(), _strides(output)),
             hip.heads(query.data_ptr(), _strides(query)), cache, prefix, shape,
             workspace.data_ptr(), need, 0)
    return {"output": output}


def _own_beams(state):
    from spar_amd import hip

    case, logits, scores, ended = (state[k] for k in ("case", "logits", "scores", "ended"))
    shape = hip.beams(case["groups"], case["beams"], case["vocabulary"], case["picks"],
                      logits.stride(0), None if ended is None else ended.data_ptr(), state["end"],
                      hip.dtype_tag(case["dtype"]))
    need = hip.beam_select_workspace(shape)
    workspace = _scratch(state, "select", logits, need, torch.uint8)
    picks = case["groups"], case["picks"]
    made = {"scores": logits.new_empty(picks),
            "parents": torch.empty(picks, dtype=torch.int64, device=logits.device),
            "tokens": torch.empty(picks, dtype=torch.int64, device=logits.device)}
    if ended is not None:
        made["ended"] = torch.empty(picks, dtype=torch.int32, device=logits.device)
    hip.call("spar_hip_launch_beam_select", made["scores"].data_ptr(), made["parents"].data_ptr(),
             made["tokens"].data_ptr(), None if ended is None else made["ended"].data_ptr(),
             logits.data_ptr(), scores.data_ptr(), shape, workspace.data_ptr(), need, 0)
    rows = picks[0] * picks[1]
    made["states"] = [x.new_empty(rows, x.shape[1]) for x in state["states"]]
    hip.call("spar_hip_launch_reorder",
             hip.reorders(*((y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), x.shape[1],
                             x.element_size()) for x, y in zip(state["states"], made["states"]))),
             len(state["states"]), made["parents"].data_ptr(), rows, logits.shape[0], 0)
    return made


def run(state):
    """One pass through the operator, or for beams the choice and the states' order."""
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "beams": _own_beams}[kind](state)
    return {"append": _plain_append, "attention": _plain_attention,
            "beams": _plain_beams}[kind](state)


# -------------------------------------------------------------- definitions

def _exact_append(state):
    """Each pair as a complex number times exp(i * position * frequency), written token by
    token of the flattened cache."""
    case = state["case"]
    r, page, hk = case["rotary"], case["page"], case["key_heads"]
    angle = state["positions"].double()[:, :, None, None] * state["frequencies"]
    factor = torch.polar(torch.ones_like(angle), angle)

    def turn(x):
        if case["layout"] == "half":
            pair = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous())
            parts = [(pair * factor).real, (pair * factor).imag]
            return torch.cat([*parts, x[..., r:]], -1)
        pair = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * factor
        return torch.cat([torch.stack([pair.real, pair.imag], -1).flatten(-2), x[..., r:]], -1)

    query, key, value = _heads(state)
    places = state["places"]
    written = (places >= 0).flatten()
    page_of = torch.gather(state["table"].long(), 1, places.clamp(min=0) // page)
    token = (page_of * page + places.clamp(min=0) % page).flatten()[written]
    made = {"query": turn(query)}
    for name, new in (("key", turn(key)), ("value", value)):
        pool = state[name].transpose(1, 2).reshape(-1, hk, case["width"]).clone()
        pool[token] = new.reshape(-1, hk, case["width"])[written]
        made[name] = pool.view(-1, page, hk, case["width"]).transpose(1, 2).contiguous()
    return made


def _exact_attention(state):
    """Sequence by sequence: the softmax over the keys it sees, laid side by side."""
    case = state["case"]
    t, g = case["queries"], case["heads"] // case["key_heads"]
    sharers = case["batch"] // case["prefixes"]
    output = torch.zeros_like(state["query"])

    def tokens(name, row, count):
        pool, table = state[name], state["prefix_table" if "prefix" in name else "table"]
        if table is None:
            found = pool[row]
        else:
            found = pool[table[row][table[row] >= 0].long()].transpose(0, 1).flatten(1, 2)
        return found[:, :count].repeat_interleave(g, 0)

    lengths, prefix_lengths = state["lengths"].tolist(), state["prefix_lengths"].tolist()
    for b, length in enumerate(lengths):
        p = b // sharers
        key, value = (torch.cat([tokens("prefix_" + name, p, prefix_lengths[p]),
                                 tokens(name, b, length)], 1) for name in ("key", "value"))
        first = max(0, t - length)  # queries before it are no tokens of the sequence
        if first == t:
            continue
        scores = torch.matmul(state["query"][b, first:].transpose(0, 1), key.transpose(1, 2))
        ends = prefix_lengths[p] + length - t + torch.arange(first, t, device=key.device)
        future = torch.arange(key.shape[1], device=key.device) > ends[:, None]
        scores = (scores / math.sqrt(case["width"])).masked_fill(future, -math.inf)
        output[b, first:] = torch.matmul(torch.softmax(scores, -1), value).transpose(0, 1)
    return {"output": output}


def _exact_beams(state):
    """Row by row: the best of each row's log-probabilities, then the best of the rows'."""
    case, ended = state["case"], state["ended"]
    beams, v, picks = case["beams"], case["vocabulary"], case["picks"]
    kept = min(picks, v)
    found = []
    for row in range(case["groups"] * beams):
        score = state["scores"][row].item()
        x = torch.log_softmax(state["logits"][row], 0).add(score).nan_to_num(
            nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        if ended is not None and ended[row].item():
            x = torch.full_like(x, -math.inf)
            x[state["end"]] = score
        order = torch.argsort(x, descending=True, stable=True)[:kept]
        found.append((x[order].tolist(), order.tolist()))
    scores, parents, tokens = [], [], []
    for group in range(case["groups"]):
        every = [(-score, row, token) for row in range(group * beams, (group + 1) * beams)
                 for score, token in zip(*found[row])]
        best = sorted(every)[:picks]
        scores.append([-x[0] for x in best])
        parents.append([x[1] for x in best])
        tokens.append([x[2] for x in best])
    device = state["logits"].device
    made = {"scores": torch.tensor(scores, device=device, dtype=torch.float64),
            "parents": torch.tensor(parents, device=device),
            "tokens": torch.tensor(tokens, device=device)}
    if ended is not None:
        flags = [[int(ended[r].item() != 0 or k == state["end"]) for r, k in zip(*both)]
                 for both in zip(parents, tokens)]
        made["ended"] = torch.tensor(flags, device=device, dtype=torch.int32)
    made["states"] = [torch.stack([x[r] for group in parents for r in group])
                      for x in state["states"]]
    return made


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    state = prepare(case, seed)
    for name, x in state.items():
        if isinstance(x, torch.Tensor) and x.is_floating_point():
            state[name] = x.double()
    state["states"] = [x.double() if x.is_floating_point() else x for x in state.get("states", [])]
    return {"append": _exact_append, "attention": _exact_attention,
            "beams": _exact_beams}[case["kind"]](state)


# --------------------------------------------------------------------- work

def work(case):
    """Each input read once and each output written once; of the caches what some query
    sees, a prefix once for all that share it.  Additions and products, and one operation
    for an exponential."""
    size = 4 if case["dtype"] == "float32" else 8
    if case["kind"] == "beams":
        rows, v = case["groups"] * case["beams"], case["vocabulary"]
        moved = 8 * case["history"] + 4 * case["slots"] + size * case["state"]
        picks = case["groups"] * case["picks"]
        # rows of states: as many parents as there are rows at most, read once each
        return {"bytes": rows * v * size + (min(rows, picks) + picks) * moved,
                "flops": 4 * rows * v}
    b, h, hk, d = (case[k] for k in ("batch", "heads", "key_heads", "width"))
    if case["kind"] == "append":
        n = b * case["tokens"]
        return {"bytes": 2 * n * (h + 2 * hk) * d * size,
                "flops": 3 * n * (h + hk) * max(case["rotary"], 1)}
    t, s = case["queries"], b // case["prefixes"]
    lengths = _spread(case["tokens"], case["shortest"], b)
    prefix_lengths = _spread(case["prefix"], case["prefix_shortest"], case["prefixes"])
    pairs = 0
    for i, length in enumerate(lengths):
        queries = min(t, length)
        pairs += queries * prefix_lengths[i // s] + sum(length - j for j in range(queries))
    keys = sum(lengths) + sum(prefix_lengths)
    return {"bytes": size * (2 * keys * hk * d + 2 * b * t * h * d),
            "flops": pairs * h * (4 * d + 4)}
