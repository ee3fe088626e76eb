"""What is measured of the 4-bit key / value cache and of the fused residual norm: the cases, their inputs, the operators
in plain torch, and what each pass cannot do without.

The cache.  A pool of pages; a page holds `page` tokens of every kv head, head-major: codes [pages, heads, page, dim / 2]
bytes and params [pages, heads, page, dim / group, 2] f16, for the keys and for the values.  A group of `group`
consecutive elements of one head of one token is stored as s = f16((max - min) / 15), m = f16(min) and the codes
c = clamp(round((x - m) / s), 0, 15) (half to even; 0 where s is 0), and stands for c * s + m.  Two codes a byte, the
even element in the low nibble.  The eight-element words of a row are transposed in it, so that a lane of a matrix
instruction finds what it needs in one place: word 4 i + c of a key row lies at place c * (dim / 32) + i, word 8 i + c of a
value row at place c * (dim / 64) + i.
Tokens belong to sequences: sequence b owns tokens cu[b] .. cu[b + 1] of the call, which are its last ones: the last of
them is at position lens[b] - 1, and position p lives in page table[b, p // page].
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a batch: each sequence's new token goes into the cache (and is read back)
        _cache("append_decode", "append", 32, 1, 64, 900, 8, 8, 128, 64, 64, "bf16", "bf16"),
        # a prompt's keys and values, still columns of the fused projection's output, go into the cache and come back as
        # the cache holds them
        _cache("append_prompt", "append", 1, 8192, 8192, 8192, 48, 8, 128, 64, 64, "bf16", "bf16"),
        # whole ragged sequences are taken out of the cache (another kernel's input, a move to another pool)
        _cache("read_ragged", "read", 16, 0, 700, 16000, 8, 8, 128, 128, 64, "bf16", "bf16"),
        # a few short sequences of narrow heads, single precision out
        _cache("read_small", "read", 3, 0, 17, 331, 5, 5, 64, 64, 16, "f16", "f32"),
        # one user, one token: latency counts
        _attn("decode_one", 1, 1, 4096, 4096, 8, 4, 128, 64, 64, 0, "bf16", True),
        # a serving batch of ragged contexts
        _attn("decode_batch", 32, 1, 50, 16000, 8, 4, 128, 64, 64, 0, "bf16", True),
        # long contexts, the shape of one of the wide layers (64 query heads on 8)
        _attn("decode_long", 4, 1, 100000, 131072, 8, 8, 128, 128, 128, 0, "bf16", False),
        # a drafted run of tokens is checked at once; odd group of query heads, narrow heads, small pages
        _attn("verify_drafts", 13, 5, 1, 5003, 4, 3, 64, 64, 16, 0, "f16", True),
        # a chunk of a long prompt, with a sliding window that starts inside a tile
        _attn("chunk_window", 3, 1000, 1009, 9001, 8, 4, 128, 64, 32, 4001, "bf16", False),
        # a whole prompt
        _attn("prompt", 1, 8192, 8192, 8192, 8, 4, 128, 64, 64, 0, "bf16", False),
        # the seam between two blocks of a decode step: residual, next norm, E4M3 for the next product
        _norm("norm_decode", 32, 8192, False, "none", "bf16", True),
        # the same seam on a prompt, with the norm behind the block and a gate of every element
        _norm("norm_prompt", 8190, 8192, True, "full", "bf16", False),
    ]


def _cache(name, op, seqs, new, lo, hi, heads_in, heads, dim, group, page, dtype, out):
    c = {"op": op, "seqs": seqs, "new": new, "lo": lo, "hi": hi, "heads_in": heads_in, "heads": heads, "dim": dim, "group": group,
         "page": page, "dtype": dtype, "out": out}
    return dict(c, name=name) if name else c


def _attn(name, seqs, new, lo, hi, heads, per, dim, group, page, window, dtype, lse):
    c = {"op": "attention", "seqs": seqs, "new": new, "lo": lo, "hi": hi, "heads": heads, "per": per, "dim": dim, "group": group, "page": page,
         "window": window, "dtype": dtype, "lse": lse}
    return dict(c, name=name) if name else c


def _norm(name, rows, cols, post, gate, dtype, fp8):
    c = {"op": "norm", "rows": rows, "cols": cols, "post": post, "gate": gate, "dtype": dtype, "fp8": fp8}
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """A case of the same ranges: head counts, groups, pages, lengths from one token up, odd sizes as they fall."""
    kind = rng.choice(["append", "read", "decode", "decode", "chunk", "norm"])
    if kind == "norm":
        cols = 8 * _log(rng, 8, 2048)
        return _norm(None, _log(rng, 1, max(1, (1 << 26) // cols)), cols, rng.random() < 0.5, rng.choice(["none", "row", "full"]), rng.choice(["bf16", "f16"]), rng.random() < 0.5)
    dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (64, 128) if g <= dim])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads = rng.choice([1, 2, 3, 4, 8, 8])
    if kind == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 8192 // seqs)
        lo = new + rng.randrange(300)
        return _cache(None, "append", seqs, new, lo, lo + rng.randrange(1000), heads * rng.choice([1, 3, 6]), heads, dim, group, page, dtype, dtype)
    if kind == "read":
        seqs = _log(rng, 1, 64)
        lo = _log(rng, 1, 2000)
        return _cache(None, "read", seqs, 0, lo, lo + _log(rng, 1, max(1, 140000 // seqs - lo)), heads, heads, dim, group, page, dtype, rng.choice([dtype, "f32"]))
    if kind == "decode":
        seqs, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        per = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        lo = _log(rng, new, 4000)
        hi = lo + _log(rng, 1, min(130000, 500000 // seqs))
        window = 0 if rng.random() < 0.7 else _log(rng, 1, 5000)
        return _attn(None, seqs, new, lo, hi, heads, per, dim, group, page, window, dtype, rng.random() < 0.5)
    seqs = rng.choice([1, 1, 2, 3, 5])
    new = _log(rng, 20, 8192 // seqs)
    lo = new + rng.randrange(200)
    hi = lo + rng.randrange(max(1, min(8000, (1 << 26) // (2 * seqs * new))))
    return _attn(None, seqs, new, lo, hi, heads, rng.choice([1, 2, 4, 4]), dim, group, page, 0 if rng.random() < 0.7 else _log(rng, 30, 5000), "bf16", False)


def _lens(case):
    """The sequences' lengths: spread over lo .. hi, the same for every seed."""
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    return [lo + int((hi - lo) * ((0.6180339887 * i + 0.999) % 1.0 if n > 1 else 1.0) + 0.5) for i in range(n)]


def _new(case):
    return [case["new"] or length for length in _lens(case)]


def _pairs(case):
    """How many keys the query tokens see, all together."""
    total = 0
    for n, length in zip(_new(case), _lens(case)):
        for j in range(n):
            at = length - n + j + 1
            if at > 0:
                total += min(at, case["window"]) if case["window"] else at
    return total


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["cols"], DT[case["dtype"]].itemsize
        gate = n if case["gate"] == "full" else case["cols"] if case["gate"] == "row" else 0
        return {"bytes": n * (3 * b + (1 if case["fp8"] else b)) + gate * b + case["cols"] * 4 * (2 if case["post"] else 1), "flops": 0}
    h, d = case["heads"], case["dim"]
    row = d // 2 + 4 * (d // case["group"])                     # one head of one token, keys or values
    if case["op"] in ("append", "read"):
        n = sum(_new(case))
        b = 2 * n * h * (row + d * DT[case["out"]].itemsize)
        return {"bytes": b + (2 * n * h * (row + d * DT[case["dtype"]].itemsize) if case["op"] == "append" else 0), "flops": 0}
    hq = h * case["per"]
    kept = sum(min(length, case["window"] + n - 1) if case["window"] else length for n, length in zip(_new(case), _lens(case)))
    n = sum(_new(case))
    return {"bytes": 2 * kept * h * row + 4 * n * hq * d + (4 * n * hq if case["lse"] else 0), "flops": 4 * _pairs(case) * hq * d}


# ------------------------------------------------------------------------------------------------- inputs

def _quantize(x, group):
    """f32 [..., dim] -> codes as int64 [..., dim], params f16 [..., dim / group, 2], by the definition above."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, m = ((hi - lo) / torch.full_like(hi, 15)).half(), lo.half()          # a true division: by a Python number it is a product with 1 / 15
    c = torch.where(s > 0, torch.round((g - m.float()) / s.float()).clamp(0, 15), 0.0)
    return c.flatten(-2).to(torch.uint8), torch.cat([s, m], -1)


def _pack(codes, keys):
    """uint8 codes [..., dim], one an element -> bytes [..., dim / 2], as a key or a value row lies in a page."""
    codes = codes.unflatten(-1, (-1, 4 if keys else 8, 8)).transpose(-3, -2).flatten(-3)
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(packed, params, keys):
    """Bytes and params of rows -> the f32 values that they stand for."""
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    c = c.unflatten(-1, (4 if keys else 8, -1, 8)).transpose(-3, -2).flatten(-3)
    g = c.float().unflatten(-1, (params.shape[-2], -1))
    return (g * params[..., :1].float() + params[..., 1:].float()).flatten(-2)


def prepare(case, seed):
    dev = "cuda"
    r = torch.Generator(device=dev)
    r.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=r, device=dev, dtype=torch.float32).to(dtype)

    s = {"case": case}
    dt = DT[case["dtype"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["y"] = normal(rows, cols, dtype=dt)
        s["residual"] = (normal(rows, cols) * 2).to(dt)
        s["weight"] = 1 + 0.2 * normal(cols)
        s["post"] = 1 + 0.2 * normal(cols) if case["post"] else None
        s["gate"] = None if case["gate"] == "none" else normal(rows, cols, dtype=dt) if case["gate"] == "full" else normal(cols, dtype=dt)
        s["alpha"], s["eps"] = 0.7, 1e-5
        s["scale"] = torch.tensor([0.02], device=dev)
        return s
    lens, new = _lens(case), _new(case)
    heads, dim, page = case["heads"], case["dim"], case["page"]
    need = [-(-length // page) for length in lens]
    pages, wide = sum(need) + 3, max(need) + 1
    order = torch.randperm(pages, generator=r, device=dev).tolist()
    table = torch.zeros(len(lens), wide, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.to(dev)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["cu"] = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)
    s["total"], s["most_new"], s["longest"] = sum(new), max(new), max(lens)
    # a few channels of the keys are much larger than the rest, as they are after a rotary embedding's slow channels
    channel = 1 + 7 * (torch.rand(heads, 1, dim, generator=r, device=dev) < 0.04).float()
    for name, big in (("k", channel), ("v", 0.5)):
        if case["op"] == "append":                              # what earlier steps left: zeros stand for it, nothing reads it
            s[name + "_codes"] = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device=dev)
            s[name + "_params"] = torch.zeros(pages, heads, page, dim // case["group"], 2, dtype=torch.float16, device=dev)
        else:
            codes, params = _quantize((normal(pages, heads, page, dim) * big).to(dt).float(), case["group"])
            s[name + "_codes"], s[name + "_params"] = _pack(codes, name == "k").contiguous(), params.contiguous()
            del codes
    if case["op"] == "append":
        # keys and values are columns of one projection's output: heads_in heads wide, the last 2 * heads of them theirs
        wide_in = max(case["heads_in"], 2 * heads)
        x = normal(s["total"], wide_in, dim)
        x[:, wide_in - 2 * heads:wide_in - heads] *= channel[:, 0]
        x = x.to(dt)
        s["k"], s["v"] = x[:, wide_in - 2 * heads:wide_in - heads], x[:, wide_in - heads:]
    if case["op"] == "attention":
        s["q"] = normal(s["total"], heads * case["per"], dim, dtype=dt)
        s["scale"] = dim ** -0.5
    return s


# ------------------------------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return _own_norm(s) if op == "norm" else _own_attention(s) if op == "attention" else _own_cache(s)
    return _plain_norm(s) if op == "norm" else _plain_attention(s) if op == "attention" else _plain_cache(s)


def _own_cache(s):
    from oxicuda_b200 import ops
    cache = ops.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
    if s["case"]["op"] == "append":
        ops.kv4_append(cache, s["k"], s["v"], s["table"], s["lens"], s["cu"])
    return ops.kv4_read(cache, s["table"], s["lens"], s["cu"], s["total"], dtype=DT[s["case"]["out"]])


def _own_attention(s):
    from oxicuda_b200 import ops
    cache = ops.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
    return ops.kv4_attention(s["q"], cache, s["table"], s["lens"], s["cu"], max_tokens=s["most_new"], scale=s["scale"], window=s["case"]["window"],
                             want_lse=s["case"]["lse"])


def _own_norm(s):
    from oxicuda_b200 import ops
    more = {"post_weight": s["post"], "gate": s["gate"], "alpha": s["alpha"], "eps": s["eps"]}
    if s["case"]["fp8"]:
        r, q = ops.residual_rmsnorm_fp8(s["y"], s["residual"], s["weight"], s["scale"], **more)
        return r, q.view(torch.float8_e4m3fn)
    return ops.residual_rmsnorm(s["y"], s["residual"], s["weight"], **more)


def _places(s):
    """Sequence, position, page and place in the page of every token of the call."""
    cu, page = s["cu"].long(), s["case"]["page"]
    t = torch.arange(s["total"], device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    at = s["lens"].long()[b] - cu[b + 1] + t
    return b, at, s["table"].long()[b, at // page], at % page


def _plain_cache(s):
    _, _, pg, slot = _places(s)
    if s["case"]["op"] == "append":
        for name in ("k", "v"):
            codes, params = _quantize(s[name].float().clamp(-65504, 65504), s["case"]["group"])
            s[name + "_codes"][pg, :, slot] = _pack(codes, name == "k")
            s[name + "_params"][pg, :, slot] = params
    out = DT[s["case"]["out"]]
    return tuple(_values(s[name + "_codes"][pg, :, slot], s[name + "_params"][pg, :, slot], name == "k").to(out) for name in ("k", "v"))


def _plain_attention(s):
    """All sequences at once, padded to the longest: scores, mask, softmax, weighted sum, in 32 bits."""
    case = s["case"]
    dev, page, heads, dim = s["q"].device, case["page"], case["heads"], case["dim"]
    cu, lens = s["cu"].long(), s["lens"].long()
    at = torch.arange(s["longest"], device=dev)
    pg, slot = s["table"].long()[:, at // page], (at % page).expand(len(lens), -1)
    k = _values(s["k_codes"][pg, :, slot], s["k_params"][pg, :, slot], True).transpose(1, 2)           # [seqs, heads, keys, dim]
    j = torch.arange(s["most_new"], device=dev)
    n = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + j).clamp(max=s["total"] - 1)                                                # [seqs, new]
    q = s["q"].float()[row].unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)             # [seqs, heads, per * new, dim]
    x = (q @ k.transpose(-1, -2)).mul_(s["scale"]).unflatten(2, (-1, s["most_new"]))
    del k
    mine = (lens - n)[:, None] + j                                                                     # the position of each query token
    see = (at <= mine[..., None]) & (at < lens[:, None, None])
    if case["window"]:
        see &= at > mine[..., None] - case["window"]
    x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_(min=-1e30)
    x.sub_(top).exp_()
    total = x.sum(-1)
    v = _values(s["v_codes"][pg, :, slot], s["v_params"][pg, :, slot], False).transpose(1, 2)
    o = (x.flatten(2, 3) @ v).unflatten(2, (-1, s["most_new"])) / total.clamp(min=1e-30)[..., None]
    o = torch.where(total[..., None] > 0, o, 0.0)
    real = j < n[:, None]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(s["q"].dtype)
    if not case["lse"]:
        return out
    return out, (top[..., 0] + total.log()).permute(0, 3, 1, 2).flatten(2, 3)[real]


def _rms(x, weight, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _plain_norm(s):
    t = s["y"].float()
    if s["post"] is not None:
        t = _rms(t, s["post"], s["eps"])
    if s["gate"] is not None:
        t = t * s["gate"].float()
    r = s["residual"].float() + s["alpha"] * t
    h = _rms(r, s["weight"], s["eps"])
    if s["case"]["fp8"]:
        h = (h / s["scale"]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return r.to(s["y"].dtype), h.to(h.dtype if s["case"]["fp8"] else s["y"].dtype)


# ------------------------------------------------------------------------------------------------- in 64 bits

def _exact_row(packed, params, keys, group):
    """One head's rows of a page table walk, [tokens, dim / 2] bytes and [tokens, dim / group, 2] params, as f64 values: element d is
    in word d // 8, which lies where the layout says; nibble d % 8 of it."""
    dim = packed.shape[-1] * 2
    d = torch.arange(dim, device=packed.device)
    word = d // 8
    place = (word % 4) * (dim // 32) + word // 4 if keys else (word % 8) * (dim // 64) + word // 8
    byte = place * 4 + (d % 8) // 2
    code = (packed[:, byte].long() >> (4 * (d % 2))) & 15
    p = params.double()[:, d // group]
    return code.double() * p[..., 0] + p[..., 1]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        y = s["y"].double()
        if case["post"]:
            y = y * s["post"].double() / (y.square().sum(1, keepdim=True) / case["cols"] + s["eps"]).sqrt()
        if s["gate"] is not None:
            y = s["gate"].double() * y
        r = y.mul(s["alpha"]).add(s["residual"].double())
        h = r * s["weight"].double() / (r.square().sum(1, keepdim=True) / case["cols"] + s["eps"]).sqrt()
        return r, (h / s["scale"].double()).clamp(-448, 448) if case["fp8"] else h
    lens, cu, page, group = s["lens"].tolist(), s["cu"].tolist(), case["page"], case["group"]
    if case["op"] == "append":
        # which of the sixteen levels stands for a value: the nearest one to it, of the stored step and offset
        out = []
        for x in (s["k"], s["v"]):
            x = x.double().clamp(-65504, 65504).unflatten(-1, (-1, group))
            low, high = x.min(-1).values[..., None], x.max(-1).values[..., None]
            step, low = ((high - low) / torch.full_like(high, 15)).float().half().double(), low.half().double()
            level = torch.where(step > 0, ((x - low) / step).round().clamp(0, 15), 0.0)
            out.append((low + level * step).flatten(-2))
        return tuple(out)
    keys, values = [], []
    outs = []
    sums = []
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        ids = s["table"][b].long()
        at = torch.arange(length, device=ids.device)
        rows = []
        for name in ("k", "v"):
            codes, params = s[name + "_codes"][ids[at // page], :, at % page], s[name + "_params"][ids[at // page], :, at % page]
            rows.append([_exact_row(codes[:, h], params[:, h], name == "k", group) for h in range(case["heads"])])
        if case["op"] == "read":
            keys.append(torch.stack(rows[0], 1)[length - n:])
            values.append(torch.stack(rows[1], 1)[length - n:])
            continue
        o = torch.zeros(n, case["heads"] * case["per"], case["dim"], dtype=torch.float64, device=ids.device)
        z = torch.full((n, case["heads"] * case["per"]), -math.inf, dtype=torch.float64, device=ids.device)
        for first in range(0, n, 2048):
            many = min(2048, n - first)
            p = length - n + first + torch.arange(many, device=ids.device)[:, None]
            hidden = (at[None] > p) | ((at[None] <= p - case["window"]) if case["window"] else torch.zeros_like(at[None] > p))
            blank = hidden.all(1)
            for h in range(case["heads"] * case["per"]):
                q = s["q"][cu[b] + first:cu[b] + first + many, h].double()
                x = torch.einsum("nd,kd->nk", q, rows[0][h // case["per"]]) * s["scale"]
                x[hidden] = -math.inf
                z[first:first + many, h] = torch.logsumexp(x, 1)
                w = torch.softmax(x, 1)
                w[blank] = 0
                o[first:first + many, h] = w @ rows[1][h // case["per"]]
        outs.append(o)
        sums.append(z)
    if case["op"] == "read":
        return torch.cat(keys), torch.cat(values)
    return (torch.cat(outs), torch.cat(sums)) if case["lse"] else torch.cat(outs)
