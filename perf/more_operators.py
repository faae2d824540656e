"""The operators of a decoder that runs in 8-bit integers, as users call them on device arrays.

Three families, each over the range its users meet:

  product  int8 products of tokens: activations quantised row by row (a scale for each token), weights with a scale for each
           channel, bias and activation behind; from one token to a long prompt
  cache    keys and values quantised as they are written into the pages of a cache, and read back
  attend   causal attention of each sequence's last tokens over its pages: decoding steps, a few tokens at a time, long prompts;
           a prefix that all sequences share is read once for all

`run` computes them in elementary operations, or, where `own` is set, through the entry points of this repository.
The seed makes the inputs: activations as normalised layers leave them, with channels far from the others.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEAST = 2.0 ** -100  # a row whose largest magnitude is below this is held as zeros
_PACKAGE = []


def _pkg():
    """The package lives in a folder whose name is no Python identifier; the repository's entry file loads it."""
    if not _PACKAGE:
        spec = importlib.util.spec_from_file_location("repository_entry", os.path.join(os.getcwd(), "__graft_entry__.py"))
        entry = importlib.util.module_from_spec(spec)
        sys.modules["repository_entry"] = entry
        spec.loader.exec_module(entry)
        _PACKAGE.append(entry.load_package())
    return _PACKAGE[0]


def listed():
    return [
        # one token through a projection: nothing but the weights' bytes
        {"name": "product_step", "family": "product", "type": "bf16", "m": 1, "k": 4096, "n": 4096, "bias": False, "act": "none"},
        # the tokens of a decoding batch through the wide layer of a feed-forward block
        {"name": "product_batch", "family": "product", "type": "f16", "m": 64, "k": 4096, "n": 11008, "bias": True, "act": "swish"},
        # sizes of no round number, in the runtime's own fp32
        {"name": "product_odd", "family": "product", "type": "f32", "m": 333, "k": 1000, "n": 1234, "bias": True, "act": "gelu"},
        # a long prompt
        {"name": "product_prompt", "family": "product", "type": "bf16", "m": 8192, "k": 4096, "n": 8192, "bias": True, "act": "none"},
        # the new tokens of a decoding batch: a call that is all latency
        {"name": "cache_step", "family": "cache", "type": "bf16", "b": 64, "new": 1, "ragged": False, "context": 2048, "kv_heads": 8, "d": 128, "page": 16},
        # prompts of different lengths, written whole
        {"name": "cache_prompt", "family": "cache", "type": "f16", "b": 8, "new": 8192, "ragged": True, "context": 0, "kv_heads": 8, "d": 128, "page": 64},
        # heads of 72, three of them, behind contexts that end inside a page
        {"name": "cache_odd", "family": "cache", "type": "f32", "b": 5, "new": 700, "ragged": True, "context": 333, "kv_heads": 3, "d": 72, "page": 32},
        # a decoding step of one sequence
        {"name": "attend_one", "family": "attend", "type": "bf16", "b": 1, "new": 1, "context": 4096, "ragged": False, "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "shared": 0},
        # a decoding step of many sequences of different lengths
        {"name": "attend_batch", "family": "attend", "type": "f16", "b": 64, "new": 1, "context": 8191, "ragged": True, "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "shared": 0},
        # prompts taken in pieces, each piece behind what is already in the cache
        {"name": "attend_prompt", "family": "attend", "type": "bf16", "b": 4, "new": 2048, "context": 4096, "ragged": True, "heads": 32, "kv_heads": 8, "d": 128, "page": 64, "shared": 0},
        # a decoding step of many sequences behind one long common prefix
        {"name": "attend_shared", "family": "attend", "type": "bf16", "b": 64, "new": 1, "context": 512, "ragged": True, "heads": 32, "kv_heads": 8, "d": 128, "page": 32, "shared": 8192},
        # a few tokens at a time (guesses to be checked), heads of 80, fp32
        {"name": "attend_odd", "family": "attend", "type": "f32", "b": 7, "new": 5, "context": 1000, "ragged": True, "heads": 12, "kv_heads": 4, "d": 80, "page": 16, "shared": 0},
    ]


def _log_int(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    family = rng.choice(["product", "product", "cache", "attend", "attend", "attend"])
    kind = rng.choice(["f16", "bf16", "bf16", "f32"])
    if family == "product":
        k, n = _log_int(rng, 64, 12288), _log_int(rng, 32, 14336)
        if rng.random() < 0.7:
            k, n = max(64, k // 64 * 64), max(32, n // 32 * 32)
        m = min(_log_int(rng, 1, 8192), (1 << 38) // (k * n))
        return {"family": "product", "type": kind, "m": m, "k": k, "n": n, "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "none", "relu", "swish", "gelu"])}
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    d = rng.choice([40, 64, 64, 72, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    if family == "cache":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        b = max(1, min(_log_int(rng, 1, 256), (1 << 26) // (new * kv_heads * d)))
        return {"family": "cache", "type": kind, "b": b, "new": new, "ragged": rng.random() < 0.6, "context": _log_int(rng, 1, 4096) - 1,
                "kv_heads": kv_heads, "d": d, "page": page}
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    which = rng.random()
    new = 1 if which < 0.45 else _log_int(rng, 2, 8) if which < 0.65 else _log_int(rng, 9, 2048)
    shared = page * _log_int(rng, 1, 8192 // page) if rng.random() < 0.3 else 0
    context = _log_int(rng, 1, 8192) - 1
    b = _log_int(rng, 1, 64)
    # the products of a case stay below the largest listed one's (fp32: a hundredth of them), its keys below 2^29
    most = (1 << 37) if kind != "f32" else (1 << 30)
    while b > 1 and (b * new * (shared + context + new) * heads * d > most or b * (shared + context + new) * kv_heads * d > 1 << 29):
        b //= 2
    while b * new * (shared + context + new) * heads * d > most:
        new, context = max(1, new // 2), context // 2
        shared = shared // (2 * page) * page
    return {"family": "attend", "type": kind, "b": b, "new": new, "context": context, "ragged": rng.random() < 0.6, "heads": heads,
            "kv_heads": kv_heads, "d": d, "page": page, "shared": shared}


def _counts(case):
    """Each sequence's new tokens and the tokens of its own that are there already: evenly spread where they are ragged."""
    b, new, context = case["b"], case["new"], case["context"]
    if not case["ragged"]:
        return [new] * b, [context] * b
    return [max(1, new * (i + 1) // b) for i in range(b)], [context * ((i * 5 + 3) % b + 1) // b for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["family"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = (normal(m, k) * normal(k).abs_().add_(0.3)).to(kind)
        # rows of weights start at multiples of 16 bytes, as they are laid out once
        s["pitch"] = (k + 15) // 16 * 16
        s["w"] = torch.zeros(n, s["pitch"], dtype=torch.int8, device="cuda")
        s["w"][:, :k] = torch.randn(n, k, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s["steps"] = normal(n).abs_().add_(0.5).mul_(1 / (32 * math.sqrt(k)))
        s["bias"] = normal(n) if case["bias"] else None
        s["y"] = torch.empty(m, n, dtype=kind, device="cuda")
        return s
    b, page, kv_heads, d = (case[x] for x in ("b", "page", "kv_heads", "d"))
    shared = case.get("shared", 0)
    new, context = _counts(case)
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    new, context = [new[i] for i in order], [context[i] for i in order]
    lens = [shared + c + t for c, t in zip(context, new)]
    width = (max(lens) + page - 1) // page
    # a sequence's pages lie anywhere; those of the shared prefix are the same ones for all
    own_pages = [(length + page - 1) // page - shared // page for length in lens]
    pages = shared // page + sum(own_pages) + 3
    free = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device="cuda")
    table[:, :shared // page] = free[:shared // page]
    used = shared // page
    for i, count in enumerate(own_pages):
        table[i, shared // page:shared // page + count] = free[used:used + count]
        used += count
    s["table"], s["width"], s["pages"] = table, width, pages
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["new"] > 1 else None
    s["tokens"], s["most"], s["longest"] = starts[-1], max(new), max(lens)
    row = (d + 15) // 16 * 16
    for name in ("k", "v"):
        ints = torch.zeros(pages, kv_heads, page, row, dtype=torch.int8, device="cuda")
        if case["family"] == "attend":
            for at in range(0, pages, 4096):  # (in pieces: these are the large ones)
                size = min(4096, pages - at)
                ints[at:at + size, ..., :d] = torch.randn(size, kv_heads, page, d, generator=g, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)
        s[name + "_cache"] = ints
        s[name + "_steps"] = normal(pages, kv_heads, page).abs_().add_(0.5).mul_(1 / 40)
    if case["family"] == "cache":
        for name in ("k", "v"):
            s[name] = (normal(s["tokens"], kv_heads, d) * normal(d).abs_().add_(0.3)).to(kind)
            s[name + "_read"] = torch.empty_like(s[name])
    else:
        s["q"] = normal(s["tokens"], case["heads"], d).mul_(1.2).to(kind)
        s["o"] = torch.empty_like(s["q"])
    return s


def _quantise(x):
    """A row's integers (in 64 bits: halves are ties) and its step."""
    t = x.double()
    top = t.abs().amax(-1, keepdim=True)
    live = top >= LEAST
    q = t * 127 / torch.where(live, top, 1.0)
    q = torch.where(live, torch.trunc(q + torch.copysign(torch.full_like(q, 0.5), q)), 0.0)
    return q, torch.where(live, top, 0.0).float()[..., 0] / 127


def _activation(t, act):
    if act == "relu":
        return t.clamp_min(0)
    if act == "swish":
        return t / (1 + torch.exp(-t))
    if act == "gelu":
        return t * 0.5 * (1 + torch.erf(t * math.sqrt(0.5)))
    return t


def _product(s):
    case = s["case"]
    q, steps = _quantise(s["x"])
    t = (q.float() @ s["w"][:, :case["k"]].float().T) * (steps[:, None] * s["steps"])
    if s["bias"] is not None:
        t = t + s["bias"]
    return _activation(t, case["act"]).to(s["x"].dtype)


def _places(s):
    """Of each new token: its sequence, its position there, its page and its row of the page."""
    case = s["case"]
    token = torch.arange(s["tokens"], device="cuda")
    if s["starts"] is None:
        sequence, behind = token, torch.ones_like(token)
    else:
        sequence = torch.searchsorted(s["starts"][1:].long(), token, right=True)
        behind = s["starts"].long()[sequence + 1] - token
    position = s["lens"].long()[sequence] - behind
    return sequence, position, s["table"].long()[sequence, position // case["page"]], position % case["page"]


def _cache(s):
    d = s["case"]["d"]
    _, _, page, at = _places(s)
    out = []
    for name in ("k", "v"):
        q, steps = _quantise(s[name])
        s[name + "_cache"][page, :, at, :d] = q.to(torch.int8)
        s[name + "_steps"][page, :, at] = steps
        out.append((s[name + "_cache"][page, :, at, :d].float() * s[name + "_steps"][page, :, at][..., None]).to(s[name].dtype))
    return out


def _attend(s):
    case = s["case"]
    b, heads, kv_heads, d, size = (case[x] for x in ("b", "heads", "kv_heads", "d", "page"))
    sequence, position, _, _ = _places(s)
    length, most, rows = s["longest"], s["most"], heads // kv_heads
    first = s["starts"].long()[:-1] if s["starts"] is not None else torch.arange(b, device="cuda")
    inside = torch.arange(s["tokens"], device="cuda") - first[sequence]
    # [sequence][key head][new token][query head of it][component], and which keys each may see
    q = torch.zeros(b, most, heads, d, device="cuda")
    q[sequence, inside] = s["q"].float()
    q = q.view(b, most, kv_heads, rows, d).permute(0, 2, 1, 3, 4).reshape(b, kv_heads, most * rows, d)
    last = torch.full((b, most), -1, device="cuda")
    last[sequence, inside] = position
    keys = torch.arange(length, device="cuda")
    page, at = s["table"].long()[:, keys // size], keys % size

    def held(name):
        return (s[name + "_cache"][page, :, at, :d].float() * s[name + "_steps"][page, :, at][..., None]).permute(0, 2, 1, 3)

    scores = q.mul_(1 / math.sqrt(d)) @ held("k").transpose(2, 3)
    hidden = (keys > last[..., None]).repeat_interleave(rows, 1)
    scores.masked_fill_(hidden[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ held("v")) / torch.where(total == 0, 1.0, total)
    o = o.view(b, kv_heads, most, rows, d).permute(0, 2, 1, 3, 4).reshape(b, most, heads, d)
    return o[sequence, inside].to(s["q"].dtype)


def _pointer(t):
    return None if t is None else t.data_ptr()


def run(s):
    case = s["case"]
    if not own:
        return {"product": _product, "cache": _cache, "attend": _attend}[case["family"]](s)
    nb = _pkg()
    if case["family"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        if "space" not in s:
            s["space"] = torch.empty(nb.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
        nb.op_inner_product_tokens(s["x"].data_ptr(), s["y"].data_ptr(), case["type"], m, k, n, s["w"].data_ptr(), s["steps"].data_ptr(),
                                   s["space"].data_ptr(), s["space"].numel(), bias_ptr=_pointer(s["bias"]), activation=case["act"],
                                   weight_pitch=s["pitch"])
        return s["y"]
    if "cache" not in s:
        s["cache"] = nb.Cache(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["k_steps"].data_ptr(), s["v_steps"].data_ptr(), s["pages"],
                              case["page"], case["kv_heads"], case["d"])
        s["batch"] = nb.CacheBatch(s["table"].data_ptr(), s["lens"].data_ptr(), _pointer(s["starts"]), case["b"], s["tokens"], s["width"],
                                   s["most"], s["longest"])
    if case["family"] == "cache":
        nb.op_cache_write(s["cache"], s["batch"], s["k"].data_ptr(), s["v"].data_ptr(), case["type"])
        nb.op_cache_read(s["cache"], s["batch"], s["k_read"].data_ptr(), s["v_read"].data_ptr(), case["type"])
        return [s["k_read"], s["v_read"]]
    if "space" not in s:
        s["space"] = torch.empty(max(1, nb.op_cache_attention_workspace(s["cache"], s["batch"], case["heads"], case["shared"])),
                                 dtype=torch.uint8, device="cuda")
    nb.op_cache_attention(s["cache"], s["batch"], s["q"].data_ptr(), s["o"].data_ptr(), case["type"], case["heads"], case["shared"],
                          workspace_ptr=s["space"].data_ptr(), workspace_bytes=s["space"].numel())
    return s["o"]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["family"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": size * m * (k + n) + n * k + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * k * n}
    new, context = _counts(case)
    d, kv_heads = case["d"], case["kv_heads"]
    if case["family"] == "cache":
        # values in, integers and steps out and in again, values out
        rows = 2 * sum(new) * kv_heads
        return {"bytes": rows * (2 * size * d + 2 * (d + 4)), "flops": 8 * rows * d}
    keys = case["shared"] + sum(c + t for c, t in zip(context, new))
    seen = sum(t * (case["shared"] + c) + t * (t + 1) // 2 for c, t in zip(context, new))
    return {"bytes": 2 * size * sum(new) * case["heads"] * d + 2 * keys * kv_heads * (d + 4), "flops": 4 * seen * case["heads"] * d}


def _exact_rows(x):
    """Integers and steps of rows, in 64 bits, by whole numbers of halves."""
    x = x.double()
    top = x.abs().max(-1).values
    halves = torch.floor(254 * x.abs() / top.clamp_min(LEAST)[..., None])
    q = torch.sign(x) * torch.div(halves + 1, 2, rounding_mode="floor")
    return q * (top >= LEAST)[..., None], top * (top >= LEAST) / 127


def exact(case, seed):
    s = prepare(case, seed)
    if case["family"] == "product":
        q, steps = _exact_rows(s["x"])
        out = []
        for rows, step in zip(q.split(1024), steps.split(1024)):
            t = torch.einsum("mk,nk->mn", rows, s["w"][:, :case["k"]].double()) * step[:, None] * s["steps"].double()
            t = t if s["bias"] is None else t + s["bias"].double()
            out.append({"none": lambda a: a, "relu": torch.relu, "swish": lambda a: a * torch.sigmoid(a),
                        "gelu": lambda a: a * torch.special.ndtr(a)}[case["act"]](t))
        return torch.cat(out)
    d, size = case["d"], case["page"]
    if case["family"] == "cache":
        out = []
        for name in ("k", "v"):
            q, steps = _exact_rows(s[name])
            out.append(q * steps[..., None])
        return out
    q, rows = s["q"].double(), case["heads"] // case["kv_heads"]
    o = torch.empty_like(q)
    starts = list(range(case["b"] + 1)) if s["starts"] is None else s["starts"].tolist()
    for i, length in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :(length + size - 1) // size].long()
        count = starts[i + 1] - starts[i]
        see = torch.arange(length, device="cuda")[None] <= torch.arange(length - count, length, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k, v = ((s[n + "_cache"][pages, h, :, :d].double() * s[n + "_steps"][pages, h].double()[..., None]).reshape(-1, d)[:length] for n in ("k", "v"))
            for r in range(h * rows, (h + 1) * rows):
                scores = (q[starts[i]:starts[i + 1], r] @ k.T / math.sqrt(d)).masked_fill(~see, -math.inf)
                o[starts[i]:starts[i + 1], r] = torch.softmax(scores, -1) @ v
    return o
