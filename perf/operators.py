"""Performance cases of the attention operators: what a decoder layer does with
the heads of its queries, keys and values between the projections.

  rotary     the rotary position embedding of [batch, token, head, width] heads:
             half or interleaved pairs, the whole head or its first part,
             frequencies as trained or scaled for longer contexts; training adds
             the gradient
  norm       RMSNorm of every query and key head followed by the rotation, read
             in place from the packed projection [batch, token, q | k | v];
             training adds the gradients of both inputs and both weights
  attention  causal attention with a sliding window and a few first tokens that
             stay visible: query heads share key heads, queries are the last
             tokens of their sequence; over a whole sequence (training, with the
             gradients), a chunk of queries or one token over a cache

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
_EPSILON = 1.0e-5


# ------------------------------------------------------------------- cases

def _rotary(batch, tokens, heads, width, rotary, layout, start, scaling, train, dtype="float32"):
    return {"kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "width": width,
            "rotary": rotary, "layout": layout, "start": start, "scaling": scaling, "train": train,
            "dtype": dtype}


def _norm(batch, tokens, heads, key_heads, width, rotary, layout, start, scaling, train,
          dtype="float32"):
    return {"kind": "norm", "batch": batch, "tokens": tokens, "heads": heads,
            "key_heads": key_heads, "width": width, "rotary": rotary, "layout": layout,
            "start": start, "scaling": scaling, "train": train, "dtype": dtype}


def _attention(batch, heads, key_heads, width, queries, keys, shortest, window, sinks, cache, train,
               dtype="float32"):
    return {"kind": "attention", "batch": batch, "heads": heads, "key_heads": key_heads,
            "width": width, "queries": queries, "keys": keys, "shortest": shortest,
            "window": window, "sinks": sinks, "cache": cache, "train": train, "dtype": dtype}


def listed():
    return [
        # the next token of 16 sequences of different lengths: launches count
        {"name": "rotary_token", **_rotary(16, 1, 16, 64, 64, "half", 900, "none", False)},
        # 16 sequences of 1024 tokens, 16 heads of 64, training
        {"name": "rotary_tokens", **_rotary(16, 1024, 16, 64, 64, "half", 0, "none", True)},
        # part of an odd head, interleaved pairs, an odd number of tokens far behind
        # the trained length, whose frequencies are scaled by parts; training
        {"name": "rotary_partial", **_rotary(3, 2047, 12, 80, 32, "interleaved", 100000, "parts",
                                             True)},
        # the next token of 16 sequences, heads of queries and keys in one call
        {"name": "norm_token", **_norm(16, 1, 16, 4, 128, 128, "half", 900, "none", False)},
        # a training batch of 16384 tokens with 32 query and 8 key heads
        {"name": "norm_tokens", **_norm(4, 4096, 32, 8, 128, 128, "half", 0, "linear", True)},
        # double precision, an odd number of tokens, half of the head turned
        {"name": "norm_double", **_norm(2, 1023, 12, 3, 64, 32, "interleaved", 17, "none", True,
                                        "float64")},
        # the next token of 16 sequences of 2049 to 4096 tokens under a window
        {"name": "attention_token", **_attention(16, 16, 4, 64, 1, 4096, 2049, 1024, 4, True,
                                                 False)},
        # the next token of 4 long sequences that see all of their cache
        {"name": "attention_cache", **_attention(4, 32, 8, 128, 1, 65536, 50001, 0, 0, True,
                                                 False)},
        # a chunk of 512 queries of one prompt behind 7680 tokens of its cache
        {"name": "attention_chunk", **_attention(1, 32, 8, 128, 512, 8192, 8192, 4096, 4, True,
                                                 False)},
        # 16 sequences of 1024 tokens, 16 heads of 64, training
        {"name": "attention_train", **_attention(16, 16, 16, 64, 1024, 1024, 1024, 256, 4, False,
                                                 True)},
        # one long sequence with shared key heads, training: the largest
        {"name": "attention_long", **_attention(1, 32, 8, 128, 8192, 8192, 8192, 1024, 4, False,
                                                True)},
        # double precision, odd sizes, a batch padded in front whose shortest
        # sequence is empty, training
        {"name": "attention_double", **_attention(3, 6, 2, 72, 333, 333, 0, 100, 3, False, True,
                                                  "float64")},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low),
                                                             math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["rotary", "norm", "attention"])
    dtype = "float32" if rng.random() < 0.85 else "float64"
    width = rng.choice([32, 40, 64, 64, 72, 80, 96, 100, 128, 128, 128, 160, 192, 256])
    key_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    heads = min(32, key_heads * group) // key_heads * key_heads
    if kind != "attention":
        rotary = width if rng.random() < 0.6 else 2 * rng.randint(1, width // 2)
        rest = (rotary, rng.choice(["half", "interleaved"]), _log(rng, 1, 200000),
                rng.choice(["none", "linear", "parts"]))
        token = rng.random() < 0.25
        most = (1 << 26) // (width * (heads + key_heads))
        batch = _log(rng, 1, 64 if token else 16)
        tokens = 1 if token else _log(rng, 2, max(2, min(8192, most // batch)))
        if kind == "rotary":
            return _rotary(batch, tokens, heads, width, *rest, not token, dtype)
        return _norm(batch, tokens, heads, key_heads, width, *rest, not token, dtype)
    sinks = rng.choice([0, 1, 4, 4, 7, 16])
    form = rng.choice(["token", "chunk", "train", "train"])
    if form == "token":
        keys = _log(rng, 1, 65536)
        batch = _log(rng, 1, max(1, min(32, (1 << 28) // (key_heads * keys * width))))
        window = rng.choice([0, _log(rng, 1, 4096)])
        queries = rng.choice([1, 1, 1, 2, 4])
        return _attention(batch, heads, key_heads, width, queries, keys, _log(rng, 1, keys), window,
                          sinks, True, False, dtype)
    # score matrices of at most 2^30 elements (2^28 in double)
    most = 1 << (30 if dtype == "float32" else 28)
    if form == "chunk":
        keys = _log(rng, 64, 16384)
        queries = _log(rng, 8, min(1024, keys, most // (heads * keys)))
        return _attention(1, heads, key_heads, width, queries, keys, keys,
                          rng.choice([0, _log(rng, 16, 4096)]), sinks, True, False, dtype)
    tokens = _log(rng, 2, min(8192, math.isqrt(most // heads)))
    batch = _log(rng, 1, max(1, min(16, most // (heads * tokens * tokens))))
    shortest = tokens if rng.random() < 0.7 else rng.randint(0, tokens)
    window = rng.choice([0, _log(rng, 1, 2048), _log(rng, 64, 2048)])
    return _attention(batch, heads, key_heads, width, tokens, tokens, shortest, window, sinks, False,
                      True, dtype)


def _lengths(case):
    """Tokens of each sequence, from the whole cache down to the shortest."""
    b = case["batch"]
    return [case["keys"] - (case["keys"] - case["shortest"]) * i // max(1, b - 1) for i in range(b)]


def _ragged(case):
    return case["shortest"] != case["keys"]


# ------------------------------------------------------------- preparation

def _frequencies(rotary, scaling, device):
    """Radians per position of each pair, base 10000: as trained, every one divided
    by 8, or by parts: those of pairs that turn less than once in the trained 8192
    positions divided by 8, those that turn more than 32 times kept, a linear blend
    between; with the factor of the rotated values."""
    f = 10000.0 ** (-torch.arange(rotary // 2, device=device, dtype=torch.float64) * 2 / rotary)
    if scaling == "linear":
        return f / 8, 1.0
    if scaling == "parts":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * keep + f / 8 * (1 - keep), 0.1 * math.log(8) + 1
    return f, 1.0


def prepare(case, seed):
    """What a program holds before the call, on the GPU: the projections' outputs
    or the cache, positions or lengths, frequencies, weights, and in training the
    gradient that arrives."""
    device = torch.device("cuda")
    dtype = _DTYPES[case["dtype"]]
    generator = torch.Generator(device=device)
    generator.manual_seed(int(seed) * 1000003 + 29)

    def normal(*shape):
        return torch.randn(shape, generator=generator, device=device, dtype=dtype)

    b, h, d = case["batch"], case["heads"], case["width"]
    state = {"case": case}
    if case["kind"] == "attention":
        hk, t, s = case["key_heads"], case["queries"], case["keys"]
        cache = (b, hk, s, d) if case["cache"] else (b, s, hk, d)
        state["query"] = normal(b, t, h, d)
        state["key"], state["value"] = normal(*cache), normal(*cache)
        state["lengths"] = None
        if _ragged(case):
            state["lengths"] = torch.tensor(_lengths(case), device=device, dtype=torch.int32)
        if case["train"]:
            state["gradient"] = normal(b, t, h, d)
        return state
    t = case["tokens"]
    starts = case["start"] - torch.arange(b, device=device) * case["start"] // (2 * b)
    state["positions"] = starts[:, None] + torch.arange(t, device=device)
    state["frequencies"], state["magnitude"] = _frequencies(case["rotary"], case["scaling"], device)
    if case["kind"] == "rotary":
        state["x"] = normal(b, t, h, d)
        if case["train"]:
            state["gradient"] = normal(b, t, h, d)
        return state
    hk = case["key_heads"]
    state["packed"] = normal(b, t, (h + 2 * hk) * d) * 1.5
    state["query_weight"] = 1 + 0.2 * normal(d)
    state["key_weight"] = 1 + 0.2 * normal(d)
    if case["train"]:
        state["query_gradient"], state["key_gradient"] = normal(b, t, h, d), normal(b, t, hk, d)
    return state


def _heads(state):
    """The views of the query and key heads in the packed projection."""
    case = state["case"]
    b, t, h, hk, d = (case[k] for k in ("batch", "tokens", "heads", "key_heads", "width"))
    packed = state["packed"]
    return (packed[:, :, :h * d].view(b, t, h, d),
            packed[:, :, h * d:(h + hk) * d].view(b, t, hk, d))


# -------------------------------------------------------------- plain forms

def _angles(state, dtype):
    """Cosines and sines [batch, token, 1, pair], the angles in 64 bits."""
    angle = (state["positions"].double()[:, :, None] * state["frequencies"])[:, :, None]
    return ((angle.cos() * state["magnitude"]).to(dtype),
            (angle.sin() * state["magnitude"]).to(dtype))


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


def _plain_rotary(state):
    case, x = state["case"], state["x"]
    cos, sin = _angles(state, x.dtype)
    made = {"output": _turned(x, cos, sin, case)}
    if case["train"]:
        made["gradient"] = _turned(state["gradient"], cos, -sin, case)
    return made


def _plain_norm(state):
    case = state["case"]
    query, key = _heads(state)
    cos, sin = _angles(state, query.dtype)

    def forward(x, weight):
        unit = x / (x.square().mean(-1, keepdim=True) + _EPSILON).sqrt()
        return _turned(unit * weight, cos, sin, case)

    def backward(x, weight, gradient):
        d = (x.square().mean(-1, keepdim=True) + _EPSILON).sqrt()
        unit = x / d
        g = _turned(gradient, cos, -sin, case)
        gw = g * weight
        return (gw - unit * (gw * unit).mean(-1, keepdim=True)) / d, (g * unit).sum((0, 1, 2))

    made = {"query": forward(query, state["query_weight"]),
            "key": forward(key, state["key_weight"])}
    if case["train"]:
        made["query_gradient"], made["query_weight_gradient"] = backward(
            query, state["query_weight"], state["query_gradient"])
        made["key_gradient"], made["key_weight_gradient"] = backward(
            key, state["key_weight"], state["key_gradient"])
    return made


def _visible(case, lengths, device):
    """[batch, query, key]: which keys a query sees.  Query i of n is token
    length - n + i of its sequence."""
    s, t = case["keys"], case["queries"]
    if lengths is None:
        lengths = torch.full((case["batch"],), s, device=device)
    key = torch.arange(s, device=device)
    at = (lengths.long()[:, None] - t + torch.arange(t, device=device))[:, :, None]
    seen = key <= at
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    return seen


def _plain_attention(state):
    case = state["case"]
    b, h, hk, d, t, s = (case[k] for k in ("batch", "heads", "key_heads", "width", "queries",
                                           "keys"))
    g = h // hk
    scale = 1 / math.sqrt(d)

    def grouped(x):  # [b, t, h, d] -> [b, hk, g * t, d]: a key head's query heads together
        return x.permute(0, 2, 1, 3).reshape(b, hk, g * t, d)

    def ungrouped(x):
        return x.view(b, h, t, d).permute(0, 2, 1, 3).contiguous()

    query = grouped(state["query"])
    key, value = state["key"], state["value"]
    if not case["cache"]:
        key, value = key.permute(0, 2, 1, 3).contiguous(), value.permute(0, 2, 1, 3).contiguous()
    hidden = ~_visible(case, state["lengths"], query.device)[:, None, None]
    scores = torch.matmul(query, key.transpose(2, 3)).mul_(scale)
    scores.view(b, hk, g, t, s).masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    weights = weights.div_(torch.where(total == 0, 1.0, total))
    output = torch.matmul(weights, value)
    made = {"output": ungrouped(output)}
    if case["train"]:
        gradient = grouped(state["gradient"])
        by_value = torch.matmul(weights.transpose(2, 3), gradient)
        toward = torch.matmul(gradient, value.transpose(2, 3))
        toward.sub_((gradient * output).sum(-1, keepdim=True)).mul_(weights).mul_(scale)
        made["query_gradient"] = ungrouped(torch.matmul(toward, key))
        by_key = torch.matmul(toward.transpose(2, 3), query)
        made["key_gradient"] = by_key.permute(0, 2, 1, 3).contiguous()
        made["value_gradient"] = by_value.permute(0, 2, 1, 3).contiguous()
    return made


# --------------------------------------------------- the framework's calls

def _strides(x):
    """(batch, head, token) strides of a [batch, token, head, width] tensor."""
    return x.stride(0), x.stride(2), x.stride(1)


def _scratch(state, name, like, count, dtype=None):
    """Device memory that calls write and read but do not return.  The state keeps it,
    as a program does: torch would hand memory dropped here to kernels of its own
    stream while the framework's stream still works in it."""
    held = state.setdefault("scratch", {})
    if name not in held:
        held[name] = torch.empty(count, dtype=dtype or like.dtype, device=like.device)
    return held[name]


def _own_rotary(state):
    from spar_amd import hip

    case, x = state["case"], state["x"]
    b, t, h, d = x.shape
    layout = hip.ROTARY_HALF if case["layout"] == "half" else hip.ROTARY_INTERLEAVED
    positions = state["positions"]

    def turn(source, inverse):
        made = torch.empty_like(source)
        hip.call("spar_hip_launch_rotary", hip.heads(made.data_ptr(), _strides(made)),
                 hip.heads(source.data_ptr(), _strides(source)), b, h, t, d,
                 hip.rotary(positions.data_ptr(), positions.stride(0), hip.INT64,
                            state["frequencies"].data_ptr(), case["rotary"], state["magnitude"],
                            layout),
                 inverse, hip.dtype_tag(case["dtype"]), 0)
        return made

    made = {"output": turn(x, 0)}
    if case["train"]:
        made["gradient"] = turn(state["gradient"], 1)
    return made


def _own_norm(state):
    from spar_amd import hip

    case = state["case"]
    query, key = _heads(state)
    b, t, h, d = query.shape
    hk = key.shape[2]
    dtype = hip.dtype_tag(case["dtype"])
    positions = state["positions"]
    rotary = hip.rotary(positions.data_ptr(), positions.stride(0), hip.INT64,
                        state["frequencies"].data_ptr(), case["rotary"], state["magnitude"],
                        hip.ROTARY_HALF if case["layout"] == "half" else hip.ROTARY_INTERLEAVED)
    made = {"query": query.new_empty(b, t, h, d), "key": query.new_empty(b, t, hk, d)}
    saved = _scratch(state, "denominators", query, b * t * (h + hk))
    split = saved.data_ptr() + b * t * h * saved.element_size()
    parts = hip.head_norms(
        (made["query"].data_ptr(), _strides(made["query"]), saved.data_ptr(), query.data_ptr(),
         _strides(query), state["query_weight"].data_ptr(), h),
        (made["key"].data_ptr(), _strides(made["key"]), split, key.data_ptr(), _strides(key),
         state["key_weight"].data_ptr(), hk))
    hip.call("spar_hip_launch_head_norm_rotary_forward", parts, 2, b, t, d, rotary, _EPSILON, dtype,
             0)
    if case["train"]:
        for name, like in (("query", made["query"]), ("key", made["key"])):
            made[name + "_gradient"] = torch.empty_like(like)
            made[name + "_weight_gradient"] = query.new_empty(d)
        need = hip.head_norm_rotary_workspace(b, t, h + hk, d, dtype)
        workspace = _scratch(state, "backward", query, need, torch.uint8)
        gradients = hip.head_norm_gradients(
            (made["query_gradient"].data_ptr(), _strides(made["query_gradient"]),
             made["query_weight_gradient"].data_ptr(), state["query_gradient"].data_ptr(),
             _strides(state["query_gradient"]), query.data_ptr(), _strides(query),
             state["query_weight"].data_ptr(), saved.data_ptr(), h),
            (made["key_gradient"].data_ptr(), _strides(made["key_gradient"]),
             made["key_weight_gradient"].data_ptr(), state["key_gradient"].data_ptr(),
             _strides(state["key_gradient"]), key.data_ptr(), _strides(key),
             state["key_weight"].data_ptr(), split, hk))
        hip.call("spar_hip_launch_head_norm_rotary_backward", gradients, 2, b, t, d, rotary,
                 workspace.data_ptr(), need, dtype, 0)
    return made


def _own_attention(state):
    from spar_amd import hip

    case, query = state["case"], state["query"]
    b, t, h, d = query.shape
    lengths = state["lengths"]

    def cached(x):  # a cache holds its heads outermost
        strides = (x.stride(0), x.stride(1), x.stride(2)) if case["cache"] else _strides(x)
        return hip.heads(x.data_ptr(), strides)

    def heads(x):
        return hip.heads(x.data_ptr(), _strides(x))

    shape = hip.attention(b, h, case["key_heads"], t, case["keys"], d, case["window"],
                          case["sinks"], 1 / math.sqrt(d),
                          None if lengths is None else lengths.data_ptr(), hip.INT32,
                          hip.dtype_tag(case["dtype"]))
    output = torch.empty_like(query)
    saved = _scratch(state, "logsumexp", query, b * h * t) if case["train"] else None
    need = hip.attention_workspace(shape, 0)
    workspace = _scratch(state, "forward", query, need, torch.uint8)
    key, value = cached(state["key"]), cached(state["value"])
    hip.call("spar_hip_launch_attention_forward", heads(output),
             None if saved is None else saved.data_ptr(), heads(query), key, value, shape,
             workspace.data_ptr(), need, 0)
    made = {"output": output}
    if case["train"]:
        need = hip.attention_workspace(shape, 1)
        workspace = _scratch(state, "backward", query, need, torch.uint8)
        made["query_gradient"] = torch.empty_like(query)
        made["key_gradient"] = torch.empty_like(state["key"])
        made["value_gradient"] = torch.empty_like(state["value"])
        hip.call("spar_hip_launch_attention_backward", heads(made["query_gradient"]),
                 cached(made["key_gradient"]), cached(made["value_gradient"]),
                 heads(state["gradient"]), heads(output), saved.data_ptr(), heads(query), key, value,
                 shape, workspace.data_ptr(), need, 0)
    return made


def run(state):
    """One pass: the operator, and in training its gradients."""
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "norm": _own_norm, "attention": _own_attention}[kind](state)
    return {"rotary": _plain_rotary, "norm": _plain_norm,
            "attention": _plain_attention}[kind](state)


# -------------------------------------------------------------- definitions

def _exact_turn(x, state):
    """Each pair as a complex number times magnitude * exp(i * position * frequency)."""
    case = state["case"]
    r = case["rotary"]
    angle = state["positions"].double()[:, :, None, None] * state["frequencies"]
    factor = torch.polar(torch.full_like(angle, state["magnitude"]), angle)
    if case["layout"] == "half":
        pair = torch.complex(x[..., :r // 2], x[..., r // 2:r])
    else:
        pair = torch.complex(x[..., 0:r:2], x[..., 1:r:2])
    pair = pair * factor
    if case["layout"] == "half":
        turned = torch.cat([pair.real, pair.imag], -1)
    else:
        turned = torch.stack([pair.real, pair.imag], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _exact_attention(query, key, value, case, lengths):
    g = case["heads"] // case["key_heads"]
    q = query.transpose(1, 2)
    if not case["cache"]:
        key, value = key.transpose(1, 2), value.transpose(1, 2)
    k, v = (x.repeat_interleave(g, 1) for x in (key, value))
    seen = _visible(case, lengths, q.device)[:, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(case["width"])
    # a row that sees nothing: any finite scores, then weights of zero
    weights = torch.softmax(torch.where(seen, scores, -1.0e300), -1) * seen
    return torch.matmul(weights, v).transpose(1, 2)


def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by automatic differentiation."""
    state = prepare(case, seed)
    for name, x in state.items():
        if isinstance(x, torch.Tensor) and x.is_floating_point():
            state[name] = x.double()
    train = case["train"]
    if case["kind"] == "rotary":
        x = state["x"].requires_grad_(train)
        output = _exact_turn(x, state)
        made = {"output": output.detach()}
        if train:
            made["gradient"], = torch.autograd.grad(output, x, state["gradient"])
        return made
    if case["kind"] == "norm":
        made = {}
        for name, x in zip(("query", "key"), _heads(state)):
            x = x.contiguous().requires_grad_(train)
            weight = state[name + "_weight"].requires_grad_(train)
            size = torch.sqrt(torch.mean(x * x, -1, keepdim=True) + _EPSILON)
            output = _exact_turn(x / size * weight, state)
            made[name] = output.detach()
            if train:
                made[name + "_gradient"], made[name + "_weight_gradient"] = torch.autograd.grad(
                    output, (x, weight), state[name + "_gradient"])
        return made
    inputs = [state[k].requires_grad_(train) for k in ("query", "key", "value")]
    output = _exact_attention(*inputs, case, state["lengths"])
    made = {"output": output.detach().contiguous()}
    if train:
        for name, x in zip(("query", "key", "value"),
                           torch.autograd.grad(output, inputs, state["gradient"])):
            made[name + "_gradient"] = x.contiguous()
    return made


# --------------------------------------------------------------------- work

def _seen_by(case, at):
    """Keys that token `at` sees."""
    if at < 0:
        return 0
    if not case["window"] or at < case["window"]:
        return at + 1
    return case["window"] + min(case["sinks"], at + 1 - case["window"])


def work(case):
    """Each input read once and each output written once; of the keys and values
    those that some query sees.  Additions and products, and one operation for an
    exponential."""
    size = 4 if case["dtype"] == "float32" else 8
    b, h, d = case["batch"], case["heads"], case["width"]
    passes = 2 if case["train"] else 1
    if case["kind"] == "rotary":
        n = b * case["tokens"] * h
        return {"bytes": passes * 2 * n * d * size, "flops": passes * 3 * n * case["rotary"]}
    if case["kind"] == "norm":
        n = b * case["tokens"] * (h + case["key_heads"])
        moved = 2 if not case["train"] else 5  # x and y; then x, the gradient and x's gradient
        return {"bytes": moved * n * d * size,
                "flops": n * (4 * d + 3 * case["rotary"]) * (3 if case["train"] else 1)}
    t = case["queries"]
    pairs = rows = 0
    for length in _lengths(case):
        first = length - t
        pairs += sum(_seen_by(case, first + i) for i in range(t))
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        rows += length - low + min(case["sinks"], low)
    queries, keys = b * t * h * d, rows * case["key_heads"] * d
    if not case["train"]:
        return {"bytes": size * (2 * queries + 2 * keys), "flops": pairs * h * (4 * d + 4)}
    # backward: the two products again, those of both sides' gradients, and the gradient's with v
    return {"bytes": size * (2 * queries + 2 * keys + 4 * queries + 4 * keys),
            "flops": pairs * h * (14 * d + 8)}
