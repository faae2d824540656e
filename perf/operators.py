"""The operators on device arrays that feature maps and their tokens pass through, as users call them.

Three families, each over the range its users meet:

  norm    group norm with an activation over channel-last feature maps: [image][pixel][channel]
  attend  attention of an image's (or a decoder's) tokens to an encoder's states of another length, from the single token
          of a decoding step to the tokens of a whole image; key heads shared by query heads, ragged lengths, key masks
  rotary  rotary positions with several axes (row and column of an image, and time of a video) on query or key heads

`run` computes them in elementary operations, or, where `own` is set, through the entry points of this repository.
The seed makes the inputs: activations as normalised layers leave them, a few channels far from the others.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
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
        # the last feature map of a classifier, one image: a call that is all latency
        {"name": "norm_last_map", "family": "norm", "type": "f16", "n": 1, "h": 7, "w": 7, "c": 512, "groups": 32, "act": "swish"},
        # a middle block of an image generator at its usual batch
        {"name": "norm_block", "family": "norm", "type": "bf16", "n": 8, "h": 64, "w": 64, "c": 320, "groups": 32, "act": "swish"},
        # channels and pixels of no round number
        {"name": "norm_odd", "family": "norm", "type": "f16", "n": 3, "h": 33, "w": 47, "c": 91, "groups": 7, "act": "gelu"},
        # the full-size maps at the end of an image decoder, in the runtime's own fp32
        {"name": "norm_full_size", "family": "norm", "type": "f32", "n": 2, "h": 512, "w": 512, "c": 128, "groups": 32, "act": "none"},
        # one decoding step of a recogniser over its encoder's frames
        {"name": "attend_step", "family": "attend", "type": "f16", "b": 1, "lq": 1, "lk": 1500, "heads": 16, "kv_heads": 16, "d": 64, "lens": "full", "mask": False},
        # a decoding step of many requests whose encoders saw inputs of different lengths, key heads shared
        {"name": "attend_step_batch", "family": "attend", "type": "bf16", "b": 64, "lq": 1, "lk": 4096, "heads": 32, "kv_heads": 8, "d": 128, "lens": "ragged", "mask": False},
        # every pixel of a feature map over the few tokens of a text
        {"name": "attend_text", "family": "attend", "type": "f16", "b": 8, "lq": 4096, "lk": 77, "heads": 10, "kv_heads": 10, "d": 64, "lens": "full", "mask": False},
        # the pixels of an image over another image's, prompts of different lengths behind one another
        {"name": "attend_image", "family": "attend", "type": "bf16", "b": 2, "lq": 4096, "lk": 4500, "heads": 16, "kv_heads": 16, "d": 128, "lens": "ragged", "mask": False},
        # fp32 as the runtime's graphs hold it, with a mask of keys and heads of 40
        {"name": "attend_exact", "family": "attend", "type": "f32", "b": 1, "lq": 1000, "lk": 333, "heads": 8, "kv_heads": 8, "d": 40, "lens": "full", "mask": True},
        # one decoding step of a batch: three axes that share one spectrum of frequencies
        {"name": "rotary_step", "family": "rotary", "type": "bf16", "b": 16, "l": 1, "heads": 32, "d": 128, "sections": "16,24,24", "interleaved": False, "shared": True, "far": 100000},
        # a video of 21 x 30 x 52 patches
        {"name": "rotary_video", "family": "rotary", "type": "bf16", "b": 1, "l": 32760, "heads": 24, "d": 128, "sections": "22,21,21", "interleaved": True, "shared": False, "far": 64},
        # images of 32 x 32 patches and a class token, the last components of each head left as they are
        {"name": "rotary_image", "family": "rotary", "type": "f32", "b": 4, "l": 1025, "heads": 16, "d": 72, "sections": "16,16", "interleaved": False, "shared": False, "far": 32},
    ]


def _log_int(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    family = rng.choice(["norm", "attend", "attend", "attend", "rotary"])
    kind = rng.choice(["f16", "bf16", "bf16", "f32"])
    if family == "norm":
        # any map whose elements fit in the largest listed one
        groups = rng.choice([1, 4, 7, 16, 32, 32])
        c = groups * _log_int(rng, 1, 40)
        n = _log_int(rng, 1, 16)
        side = min(512, max(1, int(math.sqrt((1 << 25) / (n * c)))))
        return {"family": "norm", "type": kind, "n": n, "h": _log_int(rng, 1, side), "w": _log_int(rng, 1, side), "c": c, "groups": groups,
                "act": rng.choice(["none", "relu", "swish", "swish", "gelu"])}
    if family == "rotary":
        sections = rng.choice(["16,24,24", "22,21,21", "32,32", "16,16", "20,20", "8,12,12", "9,9", "64"])
        pairs = sum(int(s) for s in sections.split(","))
        d = 2 * pairs + rng.choice([0, 0, 8])
        heads = _log_int(rng, 1, 48)
        b = _log_int(rng, 1, 16)
        return {"family": "rotary", "type": kind, "b": b, "l": _log_int(rng, 1, max(1, min(40000, (1 << 25) // (heads * d * b)))), "heads": heads, "d": d,
                "sections": sections, "interleaved": rng.random() < 0.5, "shared": rng.random() < 0.5, "far": _log_int(rng, 16, 1000000)}
    kv_heads = rng.choice([1, 2, 8, 10, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    d = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128, 160])
    lq = 1 if rng.random() < 0.35 else _log_int(rng, 2, 4500)
    lk = _log_int(rng, 1, 8192)
    # the products of a case stay below the largest listed one's (fp32: a tenth of them), its keys below 2^27
    most = (3 << 33) if kind != "f32" else (1 << 31)
    b = max(1, min(_log_int(rng, 1, 64), most // (lq * lk * heads * d), (1 << 27) // (lk * kv_heads * d)))
    while b * lq * lk * heads * d > most:
        lq = max(1, lq // 2)
        lk = max(1, lk // 2)
    return {"family": "attend", "type": kind, "b": b, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads, "d": d,
            "lens": rng.choice(["full", "ragged"]), "mask": rng.random() < 0.25}


def _lengths(case):
    """The sequences' key counts: all of them, or spread evenly up to all of them (the same ones for every seed, in another order)."""
    b, lk = case["b"], case["lk"]
    return [lk] * b if case["lens"] == "full" else [max(1, lk * (i + 1) // b) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["family"] == "norm":
        n, p, c = case["n"], case["h"] * case["w"], case["c"]
        # channels of different sizes and offsets, as convolutions leave them
        s["x"] = torch.randn(n, p, c, generator=g, device="cuda").mul_(normal(c).abs_().add_(0.25)).add_(normal(c)).to(kind)
        s["gamma"] = normal(c).mul_(0.2).add_(1.0)
        s["beta"] = normal(c).mul_(0.2)
        s["y"] = torch.empty_like(s["x"])
    elif case["family"] == "rotary":
        b, l, heads, d = case["b"], case["l"], case["heads"], case["d"]
        s["sections"] = [int(x) for x in case["sections"].split(",")]
        s["x"] = normal(b * l, heads, d).to(kind)
        s["positions"] = torch.randint(0, case["far"], (b * l, len(s["sections"])), generator=g, device="cuda", dtype=torch.int32)
        s["y"] = torch.empty_like(s["x"])
    else:
        b, lq, lk, heads, kv_heads, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "d"))
        # scores of a standard deviation of about 1.5: some keys stand out, none alone
        s["q"] = normal(b, lq, heads, d).mul_(1.5).to(kind)
        s["k"] = normal(b, lk, kv_heads, d).to(kind)
        s["v"] = normal(b, lk, kv_heads, d).to(kind)
        s["o"] = torch.empty_like(s["q"])
        lens = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        s["lens"] = lens[torch.randperm(b, generator=g, device="cuda")].contiguous() if case["lens"] == "ragged" else None
        s["mask"] = torch.rand(b, lk, generator=g, device="cuda").lt_(0.7).to(torch.uint8) if case["mask"] else None
    return s


def _norm(s):
    case, x = s["case"], s["x"]
    n, p, c = x.shape
    t = x.float().view(n, p, case["groups"], c // case["groups"])
    t = t - t.mean((1, 3), keepdim=True)
    t = t * torch.rsqrt(t.square().mean((1, 3), keepdim=True) + 1e-5)
    t = t.view(n, p, c) * s["gamma"] + s["beta"]
    if case["act"] == "relu":
        t = t.clamp_min(0)
    elif case["act"] == "swish":
        t = t / (1 + torch.exp(-t))
    elif case["act"] == "gelu":
        t = t * 0.5 * (1 + torch.erf(t * math.sqrt(0.5)))
    return t.to(x.dtype)


def _spectrum(case, sections, device):
    """The axis of each pair and its frequency (radians a position), in 64 bits."""
    pairs = sum(sections)
    axis = torch.tensor([a for a, p in enumerate(sections) for _ in range(p)], device=device)
    part = [j / pairs for j in range(pairs)] if case["shared"] else [j / p for p in sections for j in range(p)]
    return axis, torch.exp(torch.tensor(part, dtype=torch.float64, device=device) * -math.log(10000.0))


def _rotary(s):
    case, x = s["case"], s["x"]
    axis, frequency = _spectrum(case, s["sections"], x.device)
    angle = s["positions"].double()[:, axis] * frequency  # far positions: angles in 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    r = 2 * axis.numel()
    t = x.float()
    u, v = (t[..., 0:r:2], t[..., 1:r:2]) if case["interleaved"] else (t[..., : r // 2], t[..., r // 2 : r])
    pairs = (u * cos - v * sin, u * sin + v * cos)
    turned = torch.stack(pairs, -1).flatten(-2) if case["interleaved"] else torch.cat(pairs, -1)
    return torch.cat((turned, t[..., r:]), -1).to(x.dtype)


def _attend(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, lq, heads, d = q.shape
    lk, kv_heads = k.shape[1:3]
    shared = heads // kv_heads
    # [sequence][key head][query head of it x query][component]: the heads that share keys are rows of one product
    t = (q.float() * (1 / math.sqrt(d))).view(b, lq, kv_heads, shared, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, shared * lq, d)
    scores = t @ k.float().permute(0, 2, 3, 1)
    allowed = None
    if s["lens"] is not None:
        allowed = torch.arange(lk, device=q.device) < s["lens"][:, None]
    if s["mask"] is not None:
        allowed = s["mask"].bool() if allowed is None else allowed & s["mask"].bool()
    if allowed is not None:
        scores = scores.masked_fill(~allowed[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ v.float().permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return o.view(b, kv_heads, shared, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, heads, d).to(q.dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"norm": _norm, "rotary": _rotary, "attend": _attend}[case["family"]](s)
    nb = _pkg()
    if case["family"] == "norm":
        x, y = s["x"], s["y"]
        nb.op_group_norm(x.data_ptr(), y.data_ptr(), case["type"], case["n"], case["h"] * case["w"], case["c"], case["groups"],
                         s["gamma"].data_ptr(), s["beta"].data_ptr(), 1e-5, case["act"])
        return y
    if case["family"] == "rotary":
        x, y = s["x"], s["y"]
        nb.op_rotary_axes(x.data_ptr(), y.data_ptr(), case["type"], x.shape[0], case["heads"], case["d"], s["positions"].data_ptr(),
                          s["sections"], 10000.0, case["interleaved"], case["shared"])
        return y
    o = s["o"]
    nb.op_cross_attention(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), o.data_ptr(), case["type"], case["b"], case["lq"],
                          case["lk"], case["heads"], case["kv_heads"], case["d"],
                          None if s["lens"] is None else s["lens"].data_ptr(), None if s["mask"] is None else s["mask"].data_ptr())
    return o


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["family"] == "norm":
        elements = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": 2 * size * elements + 8 * case["c"], "flops": 8 * elements}
    if case["family"] == "rotary":
        tokens = case["b"] * case["l"]
        sections = case["sections"].split(",")
        return {"bytes": 2 * size * tokens * case["heads"] * case["d"] + 4 * tokens * len(sections),
                "flops": 6 * tokens * case["heads"] * sum(int(x) for x in sections)}
    keys = sum(_lengths(case))
    return {"bytes": size * (2 * case["b"] * case["lq"] * case["heads"] * case["d"] + 2 * keys * case["kv_heads"] * case["d"])
            + (case["b"] * case["lk"] if case["mask"] else 0) + (4 * case["b"] if case["lens"] == "ragged" else 0),
            "flops": 4 * case["lq"] * keys * case["heads"] * case["d"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["family"] == "norm":
        x, out = s["x"], []
        size = case["c"] // case["groups"]
        for image in x:
            groups = []
            for g in range(case["groups"]):
                t = image[:, g * size:(g + 1) * size].double()
                deviation, mean = torch.std_mean(t, correction=0)
                groups.append((t - mean) / torch.sqrt(deviation ** 2 + 1e-5))
            t = torch.cat(groups, 1) * s["gamma"].double() + s["beta"].double()
            out.append({"none": lambda a: a, "relu": torch.relu, "swish": lambda a: a * torch.sigmoid(a),
                        "gelu": lambda a: torch.special.ndtr(a) * a}[case["act"]](t))
        return torch.stack(out)
    if case["family"] == "rotary":
        x, out, first = s["x"].double(), [], 0
        pairs = sum(s["sections"])
        for a, count in enumerate(s["sections"]):
            for j in range(count):
                rate = 10000.0 ** -((first + j) / pairs if case["shared"] else j / count)
                turn = torch.polar(torch.ones_like(x[:, 0, 0]), s["positions"][:, a].double() * rate)[:, None]
                at = (2 * (first + j), 2 * (first + j) + 1) if case["interleaved"] else (first + j, first + j + pairs)
                out.append((at, torch.complex(x[..., at[0]], x[..., at[1]]) * turn))
            first += count
        y = x.clone()
        for at, z in out:
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
        return y
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o = torch.zeros_like(q)
    shared = case["heads"] // case["kv_heads"]
    for i in range(case["b"]):
        keep = torch.ones(case["lk"], dtype=torch.bool, device="cuda")
        if s["lens"] is not None:
            keep[int(s["lens"][i]):] = False
        if s["mask"] is not None:
            keep &= s["mask"][i] != 0
        if not bool(keep.any()):
            continue
        for h in range(case["heads"]):
            kh, vh = k[i, keep, h // shared], v[i, keep, h // shared]
            o[i, :, h] = torch.softmax(q[i, :, h] @ kh.T / case["d"] ** 0.5, -1) @ vh
    return o
