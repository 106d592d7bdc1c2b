"""The low-bit operators of language-model serving as measured work: the 4-bit
linear layer, the block-scaled key/value cache, and the single-token
attention that reads that cache.

With ``own`` false, ``run`` computes each operator in its plain form from
elementary torch operations in 32 bits; with ``own`` true it makes the calls
a program makes of this package. Shapes: x [rows, k], y [rows, n]; keys and
values [tokens, kv_heads, dim]; q and out [sequences, q_heads, dim].
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # a narrow layer (the widest layer of the binary convolution sweep, as a linear layer) on one token: latency
        {"name": "linear 1x512x512", "op": "linear", "rows": 1, "k": 512, "n": 512, "group": 128, "type": "bf16",
         "zeros": False, "bias": False},
        # one token of a single stream through a wide projection: bound by reading the weights
        {"name": "linear 1x8192x8192", "op": "linear", "rows": 1, "k": 8192, "n": 8192, "group": 128, "type": "bf16",
         "zeros": True, "bias": False},
        # a few streams, a last group that is cut short, odd counts everywhere
        {"name": "linear 3x1000x777", "op": "linear", "rows": 3, "k": 1000, "n": 777, "group": 32, "type": "fp16",
         "zeros": True, "bias": True},
        # a small serving batch, fine groups
        {"name": "linear 16x4096x16384", "op": "linear", "rows": 16, "k": 4096, "n": 16384, "group": 64, "type": "bf16",
         "zeros": False, "bias": False},
        # a prompt of two thousand tokens: bound by the products
        {"name": "linear 2048x4096x4096", "op": "linear", "rows": 2048, "k": 4096, "n": 4096, "group": 128,
         "type": "bf16", "zeros": True, "bias": True},
        # one new token for each of 64 running sequences, stored in 8 bits and read back
        {"name": "cache 64 steps 8-bit", "op": "cache", "seqs": 64, "longest": 1, "start": 1500, "pad": 0, "kv_heads": 8,
         "dim": 128, "page": 64, "bits": 8, "group": 128, "type": "bf16"},
        # ragged prompts in a padded batch, stored in 4 bits with a scale for 32 channels
        {"name": "cache prompts 4-bit", "op": "cache", "seqs": 12, "longest": 4096, "start": 0, "pad": 77, "kv_heads": 8,
         "dim": 128, "page": 64, "bits": 4, "group": 32, "type": "bf16"},
        # short chunks behind an odd start, a head width that fills no power of two, small pages
        {"name": "cache odd chunks", "op": "cache", "seqs": 5, "longest": 131, "start": 37, "pad": 3, "kv_heads": 3,
         "dim": 80, "page": 16, "bits": 8, "group": 32, "type": "fp16"},
        # one short conversation: latency
        {"name": "attend 1 short", "op": "attend", "seqs": 1, "longest": 190, "prefix": 0, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "bits": 8, "group": 128, "type": "bf16"},
        # one very long document: the work has to be split along it
        {"name": "attend 1 long", "op": "attend", "seqs": 1, "longest": 100_003, "prefix": 0, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "bits": 8, "group": 128, "type": "bf16"},
        # a serving batch of unequal lengths in 4 bits, one sequence with nothing in it
        {"name": "attend 64 ragged 4-bit", "op": "attend", "seqs": 64, "longest": 8192, "prefix": 0, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "bits": 4, "group": 32, "type": "bf16"},
        # many questions about one document that all share: its keys and values are read once for all
        {"name": "attend 48 shared prefix", "op": "attend", "seqs": 48, "longest": 300, "prefix": 8190, "q_heads": 16,
         "kv_heads": 4, "dim": 64, "page": 32, "bits": 8, "group": 64, "type": "fp16"},
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "cache", "attend"])
    kind = rng.choice(["bf16", "fp16"])
    if op == "linear":
        while True:
            rows, k, n = _spread(rng, 1, 2048), _spread(rng, 64, 16384), _spread(rng, 64, 16384)
            if rng.random() < 0.5:
                k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
            if rows * k * n <= 2048 * 4096 * 4096 and k * n <= 8192 * 8192:
                break
        return {"op": op, "rows": rows, "k": k, "n": n, "group": rng.choice([32, 64, 128]), "type": kind,
                "zeros": rng.random() < 0.5, "bias": rng.random() < 0.5}
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    case = {"op": op, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "bits": rng.choice([4, 8]),
            "group": rng.choice([32, 64, dim]), "type": kind}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if op == "cache":
        if rng.random() < 0.4:
            seqs, longest = _spread(rng, 1, 512), 1
        else:
            seqs, longest = _spread(rng, 1, 24), _spread(rng, 2, 4096)
        return {**case, "seqs": seqs, "longest": longest, "start": rng.randrange(0, 2000), "pad": rng.randrange(0, 90),
                "kv_heads": kv_heads}
    while True:
        seqs, longest = _spread(rng, 1, 128), _spread(rng, 1, 100_000)
        prefix = 0 if rng.random() < 0.6 else _spread(rng, 16, 16384)
        if seqs * (longest + prefix) * kv_heads * dim <= 64 * 8192 * 8 * 128:
            break
    return {**case, "seqs": seqs, "longest": longest, "prefix": prefix, "kv_heads": kv_heads,
            "q_heads": kv_heads * rng.choice([1, 2, 4, 6, 8, 16])}


def _lengths(case):
    """Unequal lengths up to the longest, one of them empty where there are
    many: a case's own, so that its work is known."""
    n, top = case["seqs"], case["longest"]
    rng = random.Random(n * 1_000_003 + top)
    got = [top] + [_spread(rng, max(1, top // 16), top) for _ in range(n - 1)]
    if n > 3 and top > 1:
        got[2] = 0
    return got


def work(case):
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        groups = -(-k // case["group"])
        read = n * ((k + 1) // 2) + 2 * n * groups + (n * groups if case["zeros"] else 0) + (4 * n if case["bias"] else 0)
        return {"bytes": read + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}
    tokens = sum(_lengths(case)) + case.get("prefix", 0)
    # one token's keys and values in the cache: codes and the scales of its groups
    stored = 2 * case["kv_heads"] * (case["dim"] * case["bits"] / 8 + 2 * -(-case["dim"] // case["group"]))
    if case["op"] == "cache":
        values = 2 * tokens * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * 2 * values + 2 * tokens * stored, "flops": 6 * values}
    seen = sum(n + case["prefix"] for n in _lengths(case))
    rows = case["seqs"] * case["q_heads"]
    return {"bytes": tokens * stored + rows * (4 * case["dim"] + 4), "flops": 4 * seen * case["q_heads"] * case["dim"]}


# ---------------------------------------------------------------- the inputs
def _values(gen, *shape):
    """Activations as transformers have them: near normal, a few channels
    many times the others."""
    x = torch.randn(*shape, device="cuda", generator=gen)
    loud = torch.rand(shape[-1], device="cuda", generator=gen) < 0.02
    return x * torch.where(loud, 6.0, 1.0)


def _linear_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, n, kind = case["rows"], case["k"], case["n"], TYPES[case["type"]]
    groups = -(-k // case["group"])
    return {
        "x": _values(gen, m, k).to(kind),
        # two codes a byte, the even channel in the low half
        "codes": torch.randint(0, 256, (n, (k + 1) // 2), device="cuda", generator=gen, dtype=torch.uint8),
        "scales": ((0.5 + torch.rand(n, groups, device="cuda", generator=gen)) / (4.6 * math.sqrt(k))).to(kind),
        "zeros": torch.randint(4, 12, (n, groups), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None,
        "bias": torch.randn(n, device="cuda", generator=gen) if case["bias"] else None,
    }


def _cache_inputs(case, seed):
    """Keys and values of all tokens, the sequences' pages in a shuffled
    order, and where each sequence's tokens stand."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, page = TYPES[case["type"]], case["page"]
    lengths, start = _lengths(case), case.get("start", 0)
    tokens = sum(lengths) + case.get("pad", 0)
    width = -(-(start + max(lengths)) // page)
    prefix_pages = -(-case.get("prefix", 0) // page)
    pages = case["seqs"] * width + prefix_pages
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    whole = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    d = {
        "k": _values(gen, tokens, case["kv_heads"], case["dim"]).to(kind),
        "v": _values(gen, tokens, case["kv_heads"], case["dim"]).to(kind),
        "pages": pages,
        "table": order[: case["seqs"] * width].view(case["seqs"], width).contiguous(),
        "prefix_table": order[case["seqs"] * width:].contiguous(),
        "offsets": whole(ends),
        "start": torch.full((case["seqs"],), start, device="cuda", dtype=torch.int32),
        "lengths": whole(lengths),
    }
    if case["op"] == "attend":
        d["q"] = _values(gen, case["seqs"], case["q_heads"], case["dim"]).to(kind)
        d["prefix_k"] = _values(gen, case["prefix"], case["kv_heads"], case["dim"]).to(kind)
        d["prefix_v"] = _values(gen, case["prefix"], case["kv_heads"], case["dim"]).to(kind)
        d["scale"] = 1.0 / math.sqrt(case["dim"])
    return d


# ---------------------------------------------------------------- the plain forms
def _plain_linear(s):
    c = s["codes"]
    q = torch.stack((c & 15, c >> 4), -1).flatten(1)[:, : s["x"].shape[1]].float()
    of = torch.arange(q.shape[1], device=q.device) // s["group"]
    zero = s["zeros"].float()[:, of] if s["zeros"] is not None else 8.0
    y = s["x"].float() @ ((q - zero) * s["scales"].float()[:, of]).T
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _quantised(x, bits, group):
    """Codes [.., dim] and the scales [.., groups] in 16 bits: the largest
    magnitude of a group over the largest code, rounded to bf16; each value
    over its scale, rounded to even. The quotient is taken in 64 bits: a
    value next to the border of two codes has to fall on its own side."""
    top, dim = 2 ** (bits - 1) - 1, x.shape[-1]
    groups = -(-dim // group)
    x = torch.nn.functional.pad(x, (0, groups * group - dim)).unflatten(-1, (groups, group))
    scale = (x.float().abs().amax(-1) / top).to(torch.bfloat16)
    s = scale.double().unsqueeze(-1)
    codes = torch.where(s > 0, (x.double() / s).round().clamp(-top, top), 0.0)
    return codes.to(torch.int8).flatten(-2)[..., :dim], scale


def _slots(table, page, seq, pos):
    return table[seq, pos // page].long() * page + pos % page


def _plain_store(s, store, slots, x):
    codes, scales = _quantised(x, s["bits"], s["group"])
    store[0][slots], store[1][slots] = codes, scales


def _plain_load(s, store, slots):
    codes, scales = store[0][slots].float(), store[1][slots].float()
    return codes * scales.repeat_interleave(s["group"], -1)[..., : codes.shape[-1]]


def _token_slots(s):
    """The slot of each given token; rows behind the last sequence go to the
    spare slot at the end."""
    t = torch.arange(s["k"].shape[0], device="cuda")
    seq = (torch.searchsorted(s["offsets"].long(), t, right=True) - 1).clamp(max=s["table"].shape[0] - 1)
    pos = s["start"].long()[seq] + t - s["offsets"].long()[seq]
    there = t < s["offsets"][-1]
    pos = torch.where(there, pos, 0)
    return torch.where(there, _slots(s["table"], s["page"], seq, pos), s["stores"][0][0].shape[0] - 1), there


def _plain_cache(s):
    slots, there = _token_slots(s)
    out = []
    for x, store in zip((s["k"], s["v"]), s["stores"]):
        _plain_store(s, store, slots, x)
        back = _plain_load(s, store, slots)
        out.append(torch.where(there[:, None, None], back, 0.0).to(x.dtype))
    return {"k": out[0], "v": out[1]}


def _plain_attend(s):
    q, page = s["q"].float(), s["page"]
    b, heads, dim = q.shape
    kv = s["stores"][0][0].shape[1]
    q = q.view(b, kv, heads // kv, dim) * s["scale"]
    at = torch.arange(s["longest"], device="cuda")
    slots = _slots(s["table"], page, torch.arange(b, device="cuda")[:, None], at[None])
    k = _plain_load(s, s["stores"][0], slots)
    score = torch.einsum("bhgd,blhd->bhgl", q, k)
    del k
    score.masked_fill_((at[None] >= s["lengths"][:, None])[:, None, None], -math.inf)
    if s["prefix"]:
        at = torch.arange(s["prefix"], device="cuda")
        prefix = _slots(s["prefix_table"][None], page, torch.zeros_like(at), at)
        score = torch.cat((torch.einsum("bhgd,phd->bhgp", q, _plain_load(s, s["stores"][0], prefix)), score), -1)
    top = score.amax(-1, keepdim=True)
    p = (score - top.clamp(min=-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.clamp(min=1e-30)
    v = _plain_load(s, s["stores"][1], slots)
    out = torch.einsum("bhgl,blhd->bhgd", p[..., s["prefix"]:], v)
    if s["prefix"]:
        out += torch.einsum("bhgp,phd->bhgd", p[..., : s["prefix"]], _plain_load(s, s["stores"][1], prefix))
    return {"out": out.reshape(b, heads, dim).to(s["q"].dtype), "lse": (top + total.log()).view(b, heads)}


# ---------------------------------------------------------------- a program's state and calls
def _cache(case, d):
    import bnns_to_c_b200 as bn

    return bn.KVCache(torch.cuda.current_device(), d["pages"], case["page"], case["kv_heads"], case["dim"],
                      bits=case["bits"], group=case["group"], dtype=case["type"])


def _filled(case, d, s):
    """The cache of an attention case, as earlier steps left it."""
    one = {"offsets": torch.tensor([0, case["prefix"]], device="cuda", dtype=torch.int32),
           "start": torch.zeros(1, device="cuda", dtype=torch.int32), "table": d["prefix_table"][None]}
    parts = [(d["k"], d["v"], d)] + ([(d["prefix_k"], d["prefix_v"], one)] if case["prefix"] else [])
    for k, v, at in parts:
        if own:
            s["cache"].write(k, v, at["table"], at["start"], offsets=at["offsets"], stream=torch.cuda.current_stream())
        else:
            slots, _ = _token_slots({**s, "k": k, **{x: at[x] for x in one}})
            for x, store in zip((k, v), s["stores"]):
                _plain_store(s, store, slots, x)


def prepare(case, seed):
    if case["op"] == "linear":
        s = {"op": "linear", "group": case["group"], **_linear_inputs(case, seed)}
        if own:
            import bnns_to_c_b200 as bn

            s["layer"] = bn.Q4Linear(torch.cuda.current_device(), case["k"], case["n"], s["codes"], s["scales"],
                                     zeros=s["zeros"], bias=s["bias"], group=case["group"], dtype=case["type"])
            s["y"] = torch.empty(case["rows"], case["n"], device="cuda", dtype=s["x"].dtype)
        return s
    d = _cache_inputs(case, seed)
    s = {"op": case["op"], "bits": case["bits"], "group": case["group"], "page": case["page"]}
    if own:
        s["cache"] = _cache(case, d)
    else:
        groups, slots = -(-case["dim"] // case["group"]), d["pages"] * case["page"] + 1
        s["stores"] = [(torch.zeros(slots, case["kv_heads"], case["dim"], device="cuda", dtype=torch.int8),
                        torch.zeros(slots, case["kv_heads"], groups, device="cuda", dtype=torch.bfloat16)) for _ in range(2)]
    if case["op"] == "cache":
        s.update({k: d[k] for k in ("k", "v", "table", "offsets", "start")})
        if own:
            s["out"] = {"k": torch.zeros_like(d["k"]), "v": torch.zeros_like(d["v"])}
        return s
    _filled(case, d, s)
    s.update({k: d[k] for k in ("q", "table", "prefix_table", "lengths", "scale")})
    s["prefix"], s["longest"] = case["prefix"], case["longest"]
    if own:
        s["out"] = {"out": torch.empty_like(d["q"]),
                    "lse": torch.empty(case["seqs"], case["q_heads"], device="cuda", dtype=torch.float32)}
        s["work"] = torch.empty(s["cache"].attend_work(case["seqs"], case["q_heads"], case["prefix"]), device="cuda",
                                dtype=torch.uint8)
    return s


def run(s):
    if not own:
        return {"linear": _plain_linear, "cache": _plain_cache, "attend": _plain_attend}[s["op"]](s)
    stream = torch.cuda.current_stream()
    if s["op"] == "linear":
        s["layer"].run(s["x"], s["y"], stream=stream)
        return s["y"]
    if s["op"] == "cache":
        s["cache"].write(s["k"], s["v"], s["table"], s["start"], offsets=s["offsets"], stream=stream)
        s["cache"].read(s["out"]["k"], s["out"]["v"], s["table"], s["start"], offsets=s["offsets"], stream=stream)
        return s["out"]
    s["cache"].attend(s["q"], s["lengths"], s["table"], s["out"]["out"], lse=s["out"]["lse"], scale=s["scale"],
                      prefix=s["prefix_table"], prefix_tokens=s["prefix"], work=s["work"], stream=stream)
    return s["out"]


# ---------------------------------------------------------------- the definitions in 64 bits
def _bf16(x):
    """A positive number in 64 bits rounded to the nearest with 8 bits, ties to even."""
    f, e = torch.frexp(x)
    return torch.ldexp((f * 256).round() / 256, e)


def _back(x, bits, group):
    """What a cache gives back for x, in 64 bits."""
    top, out = 2 ** (bits - 1) - 1, torch.empty_like(x, dtype=torch.float64)
    for at in range(0, x.shape[-1], group):
        part = x[..., at:at + group].double()
        scale = _bf16(part.abs().max(-1, keepdim=True).values / top)
        out[..., at:at + group] = torch.round(part / scale.clamp(min=1e-300)).clamp(-top, top) * scale
    return out


def exact(case, seed):
    if case["op"] == "linear":
        d = _linear_inputs(case, seed)
        k = case["k"]
        q = torch.empty(case["n"], k, device="cuda", dtype=torch.float64)
        q[:, 0::2], q[:, 1::2] = (d["codes"] % 16)[:, : (k + 1) // 2], torch.div(d["codes"], 16, rounding_mode="floor")[:, : k // 2]
        for g, at in enumerate(range(0, k, case["group"])):
            part = q[:, at:at + case["group"]]
            part -= d["zeros"][:, g, None] if case["zeros"] else 8
            part *= d["scales"][:, g, None].double()
        y = torch.mm(d["x"].double(), q.t())
        return y if d["bias"] is None else y + d["bias"].double()
    d = _cache_inputs(case, seed)
    k, v = _back(d["k"], case["bits"], case["group"]), _back(d["v"], case["bits"], case["group"])
    lengths = _lengths(case)
    if case["op"] == "cache":
        k[sum(lengths):], v[sum(lengths):] = 0, 0
        return {"k": k, "v": v}
    pk, pv = (_back(d["prefix_" + x], case["bits"], case["group"]) for x in "kv")
    out = torch.zeros_like(d["q"], dtype=torch.float64)
    lse = torch.full(out.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    share, at = case["q_heads"] // case["kv_heads"], 0
    for b, n in enumerate(lengths):
        keys, values = torch.cat((pk, k[at:at + n])), torch.cat((pv, v[at:at + n]))
        at += n
        if not keys.shape[0]:
            continue
        for h in range(case["kv_heads"]):
            mine = slice(h * share, (h + 1) * share)
            logits = d["q"][b, mine].double() @ keys[:, h].t() / math.sqrt(case["dim"])
            lse[b, mine] = torch.logsumexp(logits, 1)
            out[b, mine] = torch.exp(logits - lse[b, mine, None]) @ values[:, h]
    return {"out": out, "lse": lse}
