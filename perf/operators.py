"""Operators of one token step next to the vocoder: what is measured, on which sizes, and their plain forms.

Four operators of the token models whose codes the vocoder turns into sound:

  cache    keys and values are written into a paged cache (as they are, or in 8 bits with a scale per token and head) and read back
  attend   one new token per sequence attends over its pages
  norm     root-mean-square norm with the residual's addition, in the input's type or in 8 bits with scales
  project  products of a few rows with 4-bit weights and group scales; with 8-bit rows they come from the norm before them

`own = False` computes them from elementary torch operations, `own = True` through the library's entry points."""
import math

import torch

own = False

DEV = "cuda"
ACT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}            # the largest code of an 8-bit type
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------------
# cases
def listed():
    return [
        # sixteen streams take one step each: the new token's keys and values go in, the last pages come back for a check or a move
        dict(name="cache_step", op="cache", act="bf16", store="int8", seqs=16, longest=1, past=96, kv=8, hd=128, page=16),
        # four voice prompts of unequal length enter a cache in 8-bit floats; heads of 64 as in the vocoder's own transformer
        dict(name="cache_prompts", op="cache", act="f16", store="e4m3", seqs=4, longest=1900, past=0, kv=16, hd=64, page=64),
        # long prompts behind a shared past, kept in their own type
        dict(name="cache_long", op="cache", act="bf16", store="same", seqs=8, longest=4001, past=4096, kv=8, hd=128, page=256),
        # one stream inside a window of 72, the heads of the vocoder's transformer: latency is all that counts
        dict(name="attend_window", op="attend", act="bf16", store="same", seqs=1, longest=125, heads=16, kv=16, hd=64, page=16, window=72),
        # a served batch of unequal lengths, two query heads to a key head
        dict(name="attend_batch", op="attend", act="bf16", store="same", seqs=32, longest=4095, heads=16, kv=8, hd=128, page=16, window=0),
        # one very long context: few rows, a long axis
        dict(name="attend_long", op="attend", act="f16", store="same", seqs=1, longest=131071, heads=32, kv=8, hd=128, page=256, window=0),
        # a full batch on an 8-bit cache, four query heads to a key head
        dict(name="attend_int8", op="attend", act="bf16", store="int8", seqs=64, longest=8192, heads=32, kv=8, hd=128, page=64, window=0),
        # one token's norm between two layers
        dict(name="norm_one", op="norm", act="bf16", out="same", rows=1, cols=1024, group=0, residual=True),
        # a prompt's rows on their way to an 8-bit product
        dict(name="norm_rows", op="norm", act="bf16", out="e4m3", rows=8192, cols=2048, group=128, residual=True),
        # one token through norm and projection in 8 bits: the smallest step
        dict(name="project_one", op="project", x="int8", act="bf16", rows=1, cols=1024, outs=2048, group=32, mins=False),
        # four streams through a feed-forward layer
        dict(name="project_four", op="project", x="same", act="bf16", rows=4, cols=2048, outs=6144, group=128, mins=False),
        # sixteen streams into a large vocabulary, weights with a scale and a least value per group
        dict(name="project_vocab", op="project", x="same", act="f16", rows=16, cols=4096, outs=65536, group=64, mins=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["cache", "attend", "norm", "project"])
    act = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        cols = _log(rng, 64, 8192)
        group = rng.choice([0, 0, 32, 64, 128])
        cols = max(group, cols // group * group) if group else cols
        return dict(op=op, act=act, out=rng.choice(["same", "e4m3"]) if not group else "e4m3", group=group, cols=cols,
                    rows=_log(rng, 1, max(1, min(16384, (1 << 23) // cols))), residual=rng.random() < 0.75)
    if op == "project":
        group = rng.choice([32, 64, 128])
        cols = group * max(1, _log(rng, 128, 8192) // group)
        return dict(op=op, act=act, x="int8" if rng.random() < 0.4 else "same", group=group, cols=cols,
                    outs=_log(rng, 33, min(65536, (1 << 27) // cols)), rows=_log(rng, 1, 16), mins=rng.random() < 0.4)
    kv = rng.choice([1, 2, 4, 8, 16])
    case = dict(op=op, act=act, store=rng.choice(["same", "int8", "e4m3"]), kv=kv, hd=rng.choice([64, 128]), page=rng.choice([8, 16, 32, 64, 256]))
    if op == "cache":
        seqs = _log(rng, 1, 32)
        return dict(case, seqs=seqs, longest=1 if rng.random() < 0.3 else _log(rng, 2, max(2, 16384 // seqs)), past=rng.choice([0, _log(rng, 1, 1024)]))
    seqs = _log(rng, 1, 64)
    row = 2 * kv * case["hd"] * BYTES[act if case["store"] == "same" else case["store"]]
    longest = _log(rng, 1, min(131071, 500_000_000 // (seqs * row)))
    return dict(case, seqs=seqs, longest=longest, heads=kv * rng.choice([1, 2, 3, 4, 7, 8]), window=rng.choice([0, 0, _log(rng, 1, max(2, longest))]))


def _lengths(seqs, longest):
    """Unequal lengths of a served batch: the longest first, one of a single token, one empty slot, the rest spread evenly."""
    spread = [1 + int((longest - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(seqs)]
    return [longest if i == 0 else 1 if i == 2 else 0 if i == 5 else n for i, n in enumerate(spread)]


def _cache_lengths(c):
    """(tokens there already, tokens that are new) of each sequence."""
    new = [1] * c["seqs"] if c["longest"] == 1 else _lengths(c["seqs"], c["longest"])
    past = _lengths(c["seqs"], c["past"]) if c["past"] else [0] * c["seqs"]
    return past, new


def work(c):
    if c["op"] == "cache":
        past, new = _cache_lengths(c)
        row = 2 * c["kv"] * c["hd"]
        held = BYTES[c["act"] if c["store"] == "same" else c["store"]] * row + (8 * c["kv"] if c["store"] != "same" else 0)
        total = sum(past) + sum(new)
        return {"bytes": sum(new) * (BYTES[c["act"]] * row + held) + total * (held + BYTES[c["act"]] * row), "flops": 4 * row * sum(new)}
    if c["op"] == "attend":
        seen = sum(min(n, c["window"] or n) for n in _lengths(c["seqs"], c["longest"]))
        held = BYTES[c["act"] if c["store"] == "same" else c["store"]] * c["hd"] + (4 if c["store"] != "same" else 0)
        return {"bytes": 2 * seen * c["kv"] * held + c["seqs"] * c["heads"] * (2 * c["hd"] * BYTES[c["act"]] + 4), "flops": 4 * seen * c["heads"] * c["hd"]}
    if c["op"] == "norm":
        n, a = c["rows"] * c["cols"], BYTES[c["act"]]
        out = n * a if c["out"] == "same" else n + 4 * (n // c["group"] if c["group"] else c["rows"])
        return {"bytes": n * a * (3 if c["residual"] else 1) + out + c["cols"] * a, "flops": 5 * n}
    k, n, m, a = c["cols"], c["outs"], c["rows"], BYTES[c["act"]]
    both = n * k // 2 + n * (k // c["group"]) * (4 if c["mins"] else 2) + m * (k + n) * a + (m * k * 2 * a + k * a if c["x"] == "int8" else 0)
    return {"bytes": both, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
def _normal(gen, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * spread).to(dtype)


def _channels(gen, c):
    """Keys have a few channels that are much larger than the others."""
    return 1.0 + 5.0 * (torch.rand((c["kv"], c["hd"]), generator=gen, device=DEV) < 0.04)


def _held(x, store):
    """(codes, scales) of keys or values [..., hd] in the cache's type."""
    if store == "same":
        return x, None
    x = x.to(torch.float32)
    scale = x.abs().amax(-1) / TOP[store]
    y = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros((), device=x.device))
    return (torch.round(y).to(torch.int8) if store == "int8" else y.to(torch.float8_e4m3fn)), scale


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    act = ACT[c["act"]]
    if c["op"] == "norm":
        shape = (c["rows"], c["cols"])
        size = 1.0 + 20.0 * (torch.rand((c["cols"],), generator=gen, device=DEV) < 0.01)      # a stream's large channels
        return dict(c, x=_normal(gen, shape, act), residual=(_normal(gen, shape, torch.float32, 3.0) * size).to(act) if c["residual"] else None,
                    weight=(1.0 + 0.2 * torch.randn((c["cols"],), generator=gen, device=DEV)).to(act))
    if c["op"] == "project":
        m, k, n, groups = c["rows"], c["cols"], c["outs"], c["cols"] // c["group"]
        s = dict(c, codes=torch.randint(0, 256, (n, k // 2), generator=gen, device=DEV, dtype=torch.uint8),
                 scales=((0.5 + torch.rand((n, groups), generator=gen, device=DEV)) / (4.0 * math.sqrt(k))).to(torch.float16))
        s["mins"] = (-7.5 * s["scales"].float() * (0.8 + 0.4 * torch.rand((n, groups), generator=gen, device=DEV))).to(torch.float16) if c["mins"] else None
        s["input"] = _normal(gen, (m, k), act)
        if c["x"] == "int8":
            s["residual"] = _normal(gen, (m, k), act, 3.0)
            s["weight"] = (1.0 + 0.2 * torch.randn((k,), generator=gen, device=DEV)).to(act)
        return s
    past, new = _cache_lengths(c) if c["op"] == "cache" else ([0] * c["seqs"], _lengths(c["seqs"], c["longest"]))
    width = max(1, max(-(-(p + n) // c["page"]) for p, n in zip(past, new)))
    pages = c["seqs"] * width
    order = torch.randperm(pages, generator=gen, device=DEV)
    s = dict(c, table=order.reshape(c["seqs"], width).to(torch.int32))
    shape = (pages, c["kv"], c["page"], c["hd"])
    scale = _channels(gen, c)[None, :, None, :]
    s["k"], s["k_scale"] = _held((torch.randn(shape, generator=gen, device=DEV) * scale).to(act), c["store"])
    s["v"], s["v_scale"] = _held(_normal(gen, shape, act), c["store"])
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    if c["op"] == "attend":
        s["q"] = _normal(gen, (c["seqs"], c["heads"], c["hd"]), act)
        s["lens"] = ints(new)
        return s
    sums = lambda v: ints([sum(v[:i]) for i in range(len(v) + 1)])  # noqa: E731
    s["first"], s["cu"], s["zero"] = ints(past), sums(new), ints([0] * c["seqs"])
    s["all_cu"], s["all_rows"] = sums([p + n for p, n in zip(past, new)]), sum(past) + sum(new)
    s["new_k"] = (torch.randn((sum(new), c["kv"], c["hd"]), generator=gen, device=DEV) * scale[0, :, 0]).to(act)
    s["new_v"] = _normal(gen, (sum(new), c["kv"], c["hd"]), act)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
def _slots(s, cu, first, rows):
    """(page, place in the page) of each of `rows` tokens: sequence b's rows cu[b] .. cu[b+1] stand at its positions first[b] ..."""
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].long(), row, right=True)
    pos = first[seq].long() + row - cu[seq].long()
    return s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _put(s, which, rows, page, at):
    codes, scale = _held(rows, s["store"])
    _bytes(s[which])[page, :, at] = _bytes(codes)
    if scale is not None:
        s[which + "_scale"][page, :, at] = scale


def _value(s, which, index):
    """The cache's values at an index, in 32 bits."""
    x = _bytes(s[which])[index].view(s[which].dtype).to(torch.float32)
    return x if s["store"] == "same" else x * s[which + "_scale"][index][..., None]


def _cache(s):
    page, at = _slots(s, s["cu"], s["first"], s["new_k"].shape[0])
    _put(s, "k", s["new_k"], page, at)
    _put(s, "v", s["new_v"], page, at)
    where = _slots(s, s["all_cu"], s["zero"], s["all_rows"])
    back = (where[0], slice(None), where[1])
    return {"k": _value(s, "k", back).to(ACT[s["act"]]), "v": _value(s, "v", back).to(ACT[s["act"]])}


def _attend(s):
    b, heads, hd = s["q"].shape
    kv, group = s["kv"], heads // s["kv"]
    k = _value(s, "k", s["table"].long()).transpose(1, 2).reshape(b, kv, -1, hd)          # [seq, kv, position, hd]
    v = _value(s, "v", s["table"].long()).transpose(1, 2).reshape(b, kv, -1, hd)
    q = s["q"].to(torch.float32).reshape(b, kv, group, hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    pos, n = torch.arange(k.shape[2], device=DEV)[None], s["lens"].long()[:, None]
    seen = (pos < n) & (pos >= (n - s["window"] if s["window"] else 0))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": out.reshape(b, heads, hd).to(ACT[s["act"]]), "lse": (top + torch.log(total)).reshape(b, heads)}


def _rms(x, residual, weight):
    """(the sum, its norm) in 32 bits."""
    total = x.to(torch.float32) if residual is None else x.to(torch.float32) + residual.to(torch.float32)
    return total, total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS) * weight.to(torch.float32)


def _norm(s):
    total, y = _rms(s["x"], s["residual"], s["weight"])
    kept = {} if s["residual"] is None else {"sum": total.to(ACT[s["act"]])}
    if s["out"] == "same":
        return dict(kept, y=y.to(ACT[s["act"]]))
    codes, scales = _held(y.reshape(s["rows"], -1, s["group"] or s["cols"]), s["out"])
    return dict(kept, codes=codes.reshape(y.shape), scales=scales)


def _weights(s):
    """The 4-bit weights [outs, cols] in 32 bits: scale times (code - 8), or scale times code plus the group's least value."""
    n, k = s["outs"], s["cols"]
    code = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).reshape(n, -1, s["group"]).to(torch.float32)
    scale = s["scales"].to(torch.float32)[..., None]
    return (scale * (code - 8.0) if s["mins"] is None else scale * code + s["mins"].to(torch.float32)[..., None]).reshape(n, k)


def _project(s):
    act = ACT[s["act"]]
    if s["x"] == "same":
        return {"y": torch.matmul(s["input"].to(torch.float32), _weights(s).t()).to(act)}
    total, y = _rms(s["input"], s["residual"], s["weight"])
    codes, scales = _held(y.reshape(s["rows"], -1, s["group"]), "int8")
    x = (codes.to(torch.float32) * scales[..., None]).reshape(y.shape)
    return {"sum": total.to(act), "y": torch.matmul(x, _weights(s).t()).to(act)}


# ---------------------------------------------------------------------------------------------------------------------
# the library's calls
_kept = {}


def _ops():
    """The handle that a program opens once."""
    if not _kept:
        import _pkgload
        _kept["ops"] = _pkgload.load_pkg().HipOps.open(0)
    return _kept["ops"]


def _own(s):
    ops = _ops()
    if s["op"] == "norm":
        if s["out"] == "same":
            total, y = ops.add_rmsnorm(s["x"], s["weight"], s["residual"], eps=EPS)
            return {"y": y} if total is None else {"sum": total, "y": y}
        total, codes, scales = ops.add_rmsnorm(s["x"], s["weight"], s["residual"], eps=EPS, quant=s["out"], group=s["group"])
        return {"codes": codes, "scales": scales} if total is None else {"sum": total, "codes": codes, "scales": scales}
    if s["op"] == "project":
        if s["x"] == "same":
            return {"y": ops.q4_matvec(s["codes"], s["scales"], s["input"], mins=s["mins"])}
        total, codes, scales = ops.add_rmsnorm(s["input"], s["weight"], s["residual"], eps=EPS, quant="int8", group=s["group"])
        return {"sum": total, "y": ops.q4_matvec(s["codes"], s["scales"], codes, mins=s["mins"], x_scale=scales, dtype=ACT[s["act"]])}
    if "cache" not in s:                        # names the tensors of the cache once, as a program does that keeps them
        s["cache"] = ops.kv_cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "attend":
        out, lse = ops.attention(s["q"], s["cache"], s["table"], s["lens"], window=s["window"], max_len=s["longest"], lse=True)
        return {"out": out, "lse": lse}
    ops.kv_write(s["cache"], s["new_k"], s["new_v"], s["table"], s["cu"], s["first"])
    k, v = ops.kv_read(s["cache"], s["table"], s["all_cu"], s["zero"], s["all_rows"], dtype=ACT[s["act"]])
    return {"k": k, "v": v}


def run(s):
    if own:
        return _own(s)
    return {"cache": _cache, "attend": _attend, "norm": _norm, "project": _project}[s["op"]](s)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
def _exact8(y, kind):
    """The values that 8 bits with one scale hold for [..., n]; the scale, and a value over its scale, are numbers of 32 bits by definition
    (inputs of few bits meet the border between two codes exactly, and often)."""
    scale = (y.abs().max(-1, keepdim=True).values / TOP[kind]).float().double()
    t = (y / scale.clamp_min(1e-300)).float().double()
    if kind == "int8":
        step = torch.ones_like(t)
    else:
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3.0)      # four significant bits, the least exponent -6
    return torch.round(t / step) * step, scale


def exact(c, seed):
    s = prepare(c, seed)
    d = lambda t: t.to(torch.float64)  # noqa: E731
    if c["op"] in ("norm", "project"):
        x = d(s["x"] if c["op"] == "norm" else s["input"])
        kept = {}
        quant = c["out"] if c["op"] == "norm" else c["x"]
        if c["op"] == "norm" or c["x"] == "int8":
            if s["residual"] is not None:
                x = x + d(s["residual"])
                kept["sum"] = x
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["cols"] + EPS) * d(s["weight"])
        if quant != "same":
            codes, scale = _exact8(x.reshape(c["rows"], -1, c["group"] or c["cols"]), quant)
            if c["op"] == "norm":
                return dict(kept, codes=codes.reshape(x.shape), scales=scale[..., 0])
            x = (codes * scale).reshape(x.shape)
        if c["op"] == "norm":
            return dict(kept, y=x)
        low, high = d(s["codes"] % 16), d(s["codes"] // 16)
        per = lambda t: d(t).repeat_interleave(c["group"] // 2, 1)  # noqa: E731
        scale, least = per(s["scales"]), per(s["mins"]) if c["mins"] else -8.0 * per(s["scales"])
        return dict(kept, y=torch.mm(x[:, 0::2], (low * scale + least).t()) + torch.mm(x[:, 1::2], (high * scale + least).t()))
    hold = lambda which: d(s[which]) if c["store"] == "same" else d(s[which]) * d(s[which + "_scale"])[..., None]  # noqa: E731
    if c["op"] == "attend":
        outs, sums = [], []
        k, v, q = hold("k"), hold("v"), d(s["q"])
        for b, n in enumerate(s["lens"].tolist()):
            low = max(0, n - c["window"]) if c["window"] else 0
            if n == 0:
                outs.append(torch.zeros_like(q[b]))
                sums.append(torch.full((c["heads"],), -math.inf, dtype=torch.float64, device=DEV))
                continue
            rows = lambda t: t[s["table"][b].long()].permute(1, 0, 2, 3).flatten(1, 2)[:, low:n].repeat_interleave(c["heads"] // c["kv"], 0)  # noqa: E731
            score = (rows(k) * q[b][:, None]).sum(-1) / math.sqrt(c["hd"])
            outs.append((torch.softmax(score, -1)[..., None] * rows(v)).sum(1))
            sums.append(torch.logsumexp(score, -1))
        return {"out": torch.stack(outs), "lse": torch.stack(sums)}
    past, new = _cache_lengths(c)
    found = {"k": [], "v": []}
    for which in found:
        old, fresh = hold(which), d(s["new_" + which])
        if c["store"] != "same":
            codes, scale = _exact8(fresh, c["store"])
            fresh = codes * scale
        at = 0
        for b, (p, n) in enumerate(zip(past, new)):
            found[which] += [old[s["table"][b].long()].transpose(1, 2).flatten(0, 1)[:p], fresh[at:at + n]]
            at += n
    return {which: torch.cat(rows) for which, rows in found.items()}
