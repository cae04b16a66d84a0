"""Cases and plain forms of the operators that serve a sequence model over codes: rotary positions, a cache of keys and
values held in 8 bits (written, read back) and attention over that cache.

`own` false: elementary torch operations, 32-bit arithmetic (64 for angles), rounded once.  `own` true: the same pass
through vision_amd.  `exact` restates each operator in 64 bits, apart from both.
"""
import math

import torch

own = False

GPU = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LARGEST = {"e4m3": 448.0, "int8": 127.0}       # what a code can stand for, in units of its block's scale
LOWEST, HIGHEST = -110, 122                    # exponents a scale can have


# ---------------------------------------------------------------------------------------------------- cases

def _rotary(name, tokens, q_heads, k_heads, dim, turned, layout, scaling, far, type, train):
    return {"name": name, "op": "rotary", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "turned": turned, "layout": layout, "scaling": scaling, "far": far, "type": type, "train": train}


def _write(name, sequences, most, before, kv_heads, dim, block, format, type):
    return {"name": name, "op": "write", "sequences": sequences, "most": most, "before": before, "kv_heads": kv_heads,
            "dim": dim, "block": block, "format": format, "type": type}


def _attend(name, sequences, most, before, kv_heads, group, dim, block, format, type, window=0, sinks=0):
    return {"name": name, "op": "attend", "sequences": sequences, "most": most, "before": before, "kv_heads": kv_heads,
            "group": group, "dim": dim, "block": block, "format": format, "type": type, "window": window, "sinks": sinks}


def listed():
    return [
        # the next code of one picture: a single token's queries and keys, nothing but latency
        _rotary("turn-token", 1, 8, 8, 64, 64, "half", "none", 48, "bf16", False),
        # a batch of prompts, packed, grouped heads, a context stretched fourfold
        _rotary("turn-prompts", 16383, 32, 8, 128, 128, "half", "yarn", 32768, "bf16", False),
        # a training step in float32: neighbouring pairs, two thirds of the head turned, forward and backward
        _rotary("turn-training", 4099, 16, 16, 96, 64, "interleaved", "ntk", 0, "f32", True),
        # a decoding step of a batch: each sequence writes one token into a block that is partly full
        _write("write-tokens", 48, 1, 2047, 8, 128, 64, "e4m3", "bf16"),
        # prompts of unequal length written at once, the cache read back for another consumer
        _write("write-prompts", 8, 4096, 0, 8, 128, 128, "int8", "bf16"),
        # a float32 model's chunk, an odd number of heads and a narrow head, starting inside blocks
        _write("write-chunk-f32", 3, 333, 200, 5, 80, 64, "e4m3", "f32"),
        # one picture's codes (a 7 x 7 grid): the smallest call
        _attend("attend-picture", 1, 1, 48, 8, 1, 64, 64, "e4m3", "bf16"),
        # a decoding step of a batch with contexts of very unequal length
        _attend("attend-batch", 64, 1, 4095, 8, 4, 128, 64, "e4m3", "bf16"),
        # a decoding step over one long context: the work has to be split along it
        _attend("attend-long", 1, 1, 131070, 4, 8, 128, 256, "int8", "bf16"),
        # a decoding step that looks back over a window and keeps the first tokens in sight
        _attend("attend-window", 16, 1, 32767, 8, 4, 128, 64, "e4m3", "bf16", 2000, 4),
        # prompts behind a shared beginning: bound by the matrix cores
        _attend("attend-prompts", 2, 4096, 1000, 8, 4, 128, 64, "e4m3", "bf16"),
        # a float32 model's chunk over an earlier context, with a window shorter than it
        _attend("attend-chunk-f32", 3, 100, 1500, 5, 2, 96, 128, "int8", "f32", 700, 4),
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most_work = {}
    for c in listed():
        w = work(c)
        for key in w:
            most_work[c["op"], key] = max(most_work.get((c["op"], key), 0), w[key])
    while True:
        op = rng.choice(["rotary", "write", "attend", "attend"])
        type = rng.choice(["bf16", "bf16", "f32"])
        dim = rng.choice([32, 48, 64, 80, 96, 112, 128, 128, 160, 192, 256])
        if op == "rotary":
            k_heads = rng.randint(1, 12)
            turned = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
            case = _rotary("", _between(rng, 1, 20000), k_heads * rng.choice([1, 1, 2, 4]), k_heads, dim, turned,
                           rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "ntk", "yarn"]),
                           _between(rng, 1, 1000000), type, rng.random() < 0.4)
        elif op == "write":
            step = rng.random() < 0.4
            case = _write("", _between(rng, 1, 64), 1 if step else _between(rng, 2, 4096), _between(rng, 1, 2000), rng.randint(1, 8),
                          dim, rng.choice([64, 128, 256]), rng.choice(["e4m3", "int8"]), type)
        else:
            step = rng.random() < 0.5
            window = _between(rng, 1, 4000) if rng.random() < 0.3 else 0
            case = _attend("", _between(rng, 1, 64), 1 if step else _between(rng, 2, 2000), _between(rng, 1, 100000 if step else 4000),
                           rng.randint(1, 8), rng.choice([1, 2, 3, 4, 5, 8]), dim, rng.choice([64, 128, 256]),
                           rng.choice(["e4m3", "int8"]), type, window, rng.randint(0, 8) if window else 0)
            # the plain form holds every score in 32 bits, and every key as a float
            pairs = case["sequences"] * (case["most"] + case["before"])
            if pairs * case["kv_heads"] * case["group"] * case["most"] > 2.4e9 or pairs * case["kv_heads"] * dim > 1.2e9:
                continue
            if type == "f32" and work(case)["flops"] > 2e10:
                continue
        w = work(case)
        if all(w[key] <= most_work[op, key] for key in w):
            del case["name"]
            return case


def _ragged(count, most, least=1):
    """Lengths of a batch, least..most, unequal and in no order; the same for every seed.  The longest is among them."""
    got = [least + (most - least) * ((i * 29 + 7) % 31) // 31 for i in range(count)]
    got[count // 2] = most
    return got


def _lengths(case):
    """(tokens a sequence holds before the call, tokens the call brings) of each sequence."""
    before = _ragged(case["sequences"], case["before"], 0)
    new = [case["most"]] * case["sequences"] if case["most"] == 1 else _ragged(case["sequences"], case["most"])
    return before, new


def _visible(case):
    """(pairs of a query and a key it sees, keys that some query sees) over a batch."""
    before, new = _lengths(case)
    window, sinks = case["window"], case["sinks"]
    pairs = keys = 0
    for b, n in zip(before, new):
        if not window:
            pairs += n * b + n * (n + 1) // 2
            keys += b + n
            continue
        for p in (range(b, b + n)):
            pairs += min(p + 1, window) + min(sinks, max(p + 1 - window, 0))
        keys += min(b + n, window + n - 1) + min(sinks, max(b + 1 - window, 0))
    return pairs, keys


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "rotary":
        pairs = case["tokens"] * (case["q_heads"] + case["k_heads"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * pairs * case["dim"] * size + 8 * case["tokens"]), "flops": passes * 3 * pairs * case["turned"]}
    before, new = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "write":
        # new rows in, their codes out; the blocks' rows read back: codes in, values out
        back = sum(n + b % case["block"] for b, n in zip(before, new))
        return {"bytes": 2 * row * (sum(new) * (size + 1) + back * (1 + 2)), "flops": 2 * row * (sum(new) * 3 + back)}
    pairs, keys = _visible(case)
    return {"bytes": 2 * keys * row + 2 * sum(new) * row * case["group"] * size, "flops": 4 * pairs * row * case["group"]}


# ---------------------------------------------------------------------------------------------------- inputs

def _offsets(counts):
    got = [0]
    for c in counts:
        got.append(got[-1] + c)
    return torch.tensor(got, dtype=torch.int32, device=GPU)


def _rows(counts, heads, dim, type, gen, spread=0.0):
    """Normal rows; with `spread`, tokens and channels of unequal size, as keys and values have them."""
    n = sum(counts)
    x = torch.randn((n, heads, dim), generator=gen, device=GPU)
    if spread:
        x *= torch.exp(spread * torch.randn((n, 1, 1), generator=gen, device=GPU))
        x *= torch.exp(spread * torch.randn((1, heads, dim), generator=gen, device=GPU))
    return x.to(TYPES[type])


def _scaling(case):
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 4.0},
            "yarn": {"type": "yarn", "factor": 4.0, "original": 8192}}[case["scaling"]]


def _inputs(case, seed):
    gen = torch.Generator(GPU).manual_seed(seed)
    if case["op"] == "rotary":
        shape = (case["tokens"],)
        first = int(torch.randint(0, case["far"] + 1, (1,), generator=gen, device=GPU))
        s = {"positions": first + torch.arange(case["tokens"], dtype=torch.int64, device=GPU)}
        for name, heads in (("q", case["q_heads"]), ("k", case["k_heads"])):
            s[name] = _rows(shape, heads, case["dim"], case["type"], gen)
            if case["train"]:
                s["d" + name] = _rows(shape, heads, case["dim"], case["type"], gen)
        return s
    before, new = _lengths(case)
    block, heads, dim = case["block"], case["kv_heads"], case["dim"]
    width = max((b + n + block - 1) // block for b, n in zip(before, new))
    blocks = case["sequences"] * width + 3
    table = torch.randperm(blocks, generator=gen, device=GPU)[:case["sequences"] * width].to(torch.int32).view(-1, width)
    s = {"table": table, "blocks": blocks, "start": torch.tensor(before, dtype=torch.int32, device=GPU), "offsets": _offsets(new),
         "zeros": torch.zeros(case["sequences"], dtype=torch.int32, device=GPU)}
    if case["op"] == "write":
        s["past"] = [_rows(before, heads, dim, case["type"], gen, 0.4) for _ in "kv"]
        s["past_offsets"] = _offsets(before)
        s["k"], s["v"] = (_rows(new, heads, dim, case["type"], gen, 0.4) for _ in "kv")
        s["since"] = torch.tensor([b // block * block for b in before], dtype=torch.int32, device=GPU)
        back = [n + b % block for b, n in zip(before, new)]
        s["back"], s["back_offsets"], s["back_most"] = sum(back), _offsets(back), max(back)
    else:
        length = [b + n for b, n in zip(before, new)]
        s["past"] = [_rows(length, heads, dim, case["type"], gen, 0.4) for _ in "kv"]
        s["past_offsets"] = _offsets(length)
        s["lengths"] = torch.tensor(length, dtype=torch.int32, device=GPU)
        s["q"] = _rows(new, heads * case["group"], dim, case["type"], gen)
    return s


def prepare(case, seed):
    """Inputs and the handle a program keeps: the frequencies' plan, the cache with what was written earlier."""
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "rotary":
        if own:
            from vision_amd.rotary import Rotary
            s["rotary"] = Rotary(case["dim"], case["turned"], layout=case["layout"], scaling=_scaling(case), device=GPU)
            if case["train"]:
                s["q"].requires_grad_()
                s["k"].requires_grad_()
        else:
            s["frequencies"], s["amplitude"] = _frequencies(case)
        return s
    past, offsets = s.pop("past"), s.pop("past_offsets")
    before, new = _lengths(case)
    most = max(before) if case["op"] == "write" else max(b + n for b, n in zip(before, new))
    s["longest"] = max(b + n for b, n in zip(before, new))
    if own:
        from vision_amd.kvcache import KVCache
        s["cache"] = KVCache(s["blocks"], case["kv_heads"], case["dim"], block=case["block"], format=case["format"], device=GPU)
        if past[0].shape[0]:
            s["cache"].append(past[0], past[1], s["table"], s["zeros"], offsets=offsets, most=most)
    else:
        held = torch.float8_e4m3fn if case["format"] == "e4m3" else torch.int8
        shape = (s["blocks"], case["kv_heads"], case["block"], case["dim"])
        s["codes"] = [torch.zeros(shape, dtype=torch.int8, device=GPU).view(held) for _ in "kv"]
        s["scales"] = [torch.zeros(shape[:2], device=GPU) for _ in "kv"]
        for x, codes, scales in zip(past, s["codes"], s["scales"]):
            if x.shape[0]:
                _plain_append(case, x, codes, scales, s["table"], s["zeros"], offsets, most)
    return s


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if case["op"] == "rotary":
        if own:
            q, k = s["rotary"](s["positions"], s["q"], s["k"])
            if not case["train"]:
                return q, k
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
            return q.detach(), k.detach(), dq, dk
        cos, sin = _plain_angles(case, s)
        got = [_plain_turn(case, s[n], cos, sin) for n in "qk"]
        if case["train"]:
            got += [_plain_turn(case, s[n], cos, -sin) for n in ("dq", "dk")]
        return tuple(got)
    if case["op"] == "write":
        if own:
            s["cache"].append(s["k"], s["v"], s["table"], s["start"], offsets=s["offsets"], most=case["most"])
            return s["cache"].read(s["table"], s["since"], s["back"], offsets=s["back_offsets"], most=s["back_most"])
        for x, codes, scales in zip((s["k"], s["v"]), s["codes"], s["scales"]):
            _plain_append(case, x, codes, scales, s["table"], s["start"], s["offsets"], case["most"])
        return tuple(_plain_read(case, codes, scales, s["table"], s["since"], s["back_offsets"], s["back"]).to(torch.bfloat16)
                     for codes, scales in zip(s["codes"], s["scales"]))
    if own:
        return s["cache"].attend(s["q"], s["table"], s["lengths"], offsets=s["offsets"], most=case["most"], longest=s["longest"],
                                 window=case["window"], sinks=case["sinks"])
    return _plain_attend(case, s)


# ---------------------------------------------------------------------------------------------------- plain forms

def _frequencies(case):
    """Radians a position, one for each pair, in 64 bits, and the amplitude of the turned part."""
    R, base, amplitude = case["turned"], 10000.0, 1.0
    scaling = _scaling(case) or {"type": "none"}
    if scaling["type"] == "ntk" and R > 2:
        base *= scaling["factor"] ** (R / (R - 2))
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64, device=GPU) / R)
    if scaling["type"] == "linear":
        f = f / scaling["factor"]
    if scaling["type"] == "yarn":
        turns = scaling["original"] * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = f * keep + f / scaling["factor"] * (1 - keep)
        amplitude = 0.1 * math.log(scaling["factor"]) + 1
    return f, amplitude


def _plain_angles(case, s):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    return (torch.cos(angle) * s["amplitude"]).float()[:, None], (torch.sin(angle) * s["amplitude"]).float()[:, None]


def _plain_turn(case, x, cos, sin):
    R = case["turned"]
    t = x[..., :R].float()
    if case["layout"] == "half":
        a, b = t[..., :R // 2], t[..., R // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = t[..., 0::2], t[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y.to(x.dtype), x[..., R:]], -1)


def _plain_round(x, format):
    """To the nearest code, ties to even."""
    return x.to(torch.float8_e4m3fn).float() if format == "e4m3" else torch.round(x)


def _plain_append(case, x, codes, scales, table, start, offsets, most):
    block, largest = case["block"], LARGEST[case["format"]]
    count = (offsets[1:] - offsets[:-1])[:, None, None]
    touched = (most + block - 2) // block + 1
    nth = (start // block)[:, None] + torch.arange(touched, device=x.device)              # [B, T] blocks of the sequence
    slot = torch.arange(block, device=x.device)
    i = nth[..., None] * block + slot - start[:, None, None]                              # [B, T, block] row of the call
    fresh = (i >= 0) & (i < count)
    i = (i + offsets[:-1, None, None]).clamp(0, x.shape[0] - 1)
    page = table.gather(1, nth.clamp(max=table.shape[1] - 1).long()).long()               # [B, T]
    rows = x[i].float().transpose(2, 3)                                                   # [B, T, H, block, D]
    fresh = fresh[:, :, None, :, None]
    amax = (rows.abs() * fresh).amax((3, 4))
    mantissa, exponent = torch.frexp(amax.double() / largest)                             # 64 bits: next to a power of two
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(LOWEST, HIGHEST)
    need = torch.where(amax > 0, ((exponent + 127) << 23).view(torch.float32), 2.0 ** LOWEST)
    begun = (nth * block >= start[:, None])[..., None]
    old = torch.where(begun, 0.0, scales[page])
    scale = torch.maximum(old, need)
    kept = _plain_round(codes[page].float() * (old / scale)[..., None, None], case["format"])
    new = _plain_round(rows / scale[..., None, None], case["format"])
    got = torch.where(fresh, new, kept).to(codes.dtype)
    live = fresh.any(3).flatten(2)[..., 0]                                                # [B, T] blocks with rows of this call
    codes.view(torch.int8)[page[live]] = got.view(torch.int8)[live]
    scales[page[live]] = scale[live]


def _plain_read(case, codes, scales, table, start, offsets, rows):
    row = torch.arange(rows, device=table.device, dtype=torch.int32)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    at = start[seq] + row - offsets[seq]
    page = table[seq, at // case["block"]].long()
    return codes.view(torch.int8)[page, :, at % case["block"]].view(codes.dtype).float() * scales[page][..., None]


def _plain_attend(case, s):
    B, most, H, G, D, block = (case[n] for n in ("sequences", "most", "kv_heads", "group", "dim", "block"))
    q, table, offsets = s["q"], s["table"], s["offsets"]
    k, v = ((codes[table.long()].float() * scales[table.long()][..., None, None]).transpose(1, 2).reshape(B, H, -1, D)
            for codes, scales in zip(s["codes"], s["scales"]))
    n = (offsets[1:] - offsets[:-1])[:, None]
    i = torch.arange(most, device=q.device)
    rows = (offsets[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q[rows].float().view(B, most, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * most, D)
    scores = torch.matmul(x, k.transpose(2, 3)).view(B, H, G, most, -1) * D ** -0.5
    p = (s["lengths"][:, None] - n + i)[:, :, None]                                       # [B, most, 1] position of a query
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j <= p) & (i < n)[:, :, None]
    if case["window"]:
        seen &= (j < case["sinks"]) | (p - j < case["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    v = torch.where((j < s["lengths"][:, None])[:, None, :, None], v, 0.0)
    out = torch.matmul((e / torch.where(total == 0, 1.0, total)).view(B, H, G * most, -1), v).view(B, H, G, most, D)
    row = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    return out.permute(0, 3, 1, 2, 4)[seq, (row - offsets[seq]).long()].reshape(q.shape).to(q.dtype)


# ---------------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        f, amplitude = _frequencies(case)
        turn = torch.polar(torch.full((), amplitude, dtype=torch.float64, device=GPU), s["positions"].double()[:, None] * f)[:, None]

        def turned(x, by):
            R = case["turned"]
            y = x.double().clone()
            t = y[..., :R]
            t = t.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else t.unflatten(-1, (R // 2, 2))
            t = torch.view_as_real(torch.view_as_complex(t.contiguous()) * by)
            y[..., :R] = (t.transpose(-1, -2) if case["layout"] == "half" else t).flatten(-2)
            return y

        got = [turned(s["q"], turn), turned(s["k"], turn)]
        if case["train"]:
            got += [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())]
        return tuple(got)
    before, new = _lengths(case)
    bases = [0]
    for b, n in zip(before, new):
        bases.append(bases[-1] + (b if case["op"] == "write" else b + n))
    if case["op"] == "write":
        starts = s["offsets"].tolist()
        got = []
        for past, x in zip(s["past"], (s["k"], s["v"])):
            parts = []
            for b, (held, fresh) in enumerate(zip(before, new)):
                block, since = case["block"], held // case["block"] * case["block"]
                old = past[bases[b] + since:bases[b] + held].double().transpose(0, 1)                # [H, rows, D]
                rows = x[starts[b]:starts[b] + fresh].double().transpose(0, 1)
                first = block - (held - since)
                scale = _exact_scale(old, case["format"]) if held > since else None
                if scale is not None:
                    bigger = torch.maximum(scale, _exact_scale(rows[:, :first], case["format"]))
                    old = _exact_round(old / scale, case["format"])
                    parts.append((_exact_round(old * (scale / bigger), case["format"]) * bigger).transpose(0, 1))
                    parts.append((_exact_round(rows[:, :first] / bigger, case["format"]) * bigger).transpose(0, 1))
                    rows = rows[:, first:]
                parts += [(_exact_round(r / _exact_scale(r, case["format"]), case["format"]) * _exact_scale(r, case["format"])).transpose(0, 1)
                          for r in rows.split(block, 1) if r.shape[1]]
            got.append(torch.cat(parts))
        return tuple(got)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    starts = s["offsets"].tolist()
    G, D = case["group"], case["dim"]
    for b, n in enumerate(new):
        length = before[b] + n
        if case["window"] and n == 1:                        # keys that nobody sees are left out
            lo = max(0, length - case["window"])
            seen = torch.cat([torch.arange(min(case["sinks"], lo)), torch.arange(lo, length)]).to(GPU)
        else:
            seen = torch.arange(length, device=GPU)
        kv = []
        for past in s["past"]:
            x = past[bases[b]:bases[b] + length].double()
            pad = -length % case["block"]
            blocks = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).unflatten(0, (-1, case["block"])).transpose(1, 2)
            scale = _exact_scale(blocks.flatten(0, 1), case["format"]).unflatten(0, blocks.shape[:2])
            kv.append((_exact_round(blocks / scale, case["format"]) * scale).transpose(1, 2).flatten(0, 1)[seen])
        p = torch.arange(before[b], length, device=GPU)[:, None]
        hidden = seen > p
        if case["window"]:
            hidden |= (seen >= case["sinks"]) & (seen <= p - case["window"])
        for h in range(case["kv_heads"]):
            k, v = kv[0][:, h], kv[1][:, h]
            for g in range(G):
                q = s["q"][starts[b]:starts[b] + n, h * G + g].double()
                w = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
                out[starts[b]:starts[b] + n, h * G + g] = w @ v
    return out


def _exact_scale(x, format):
    """[H, rows, D] -> [H, 1, 1]: the smallest power of two whose largest code reaches the largest value."""
    top = x.abs().amax((1, 2), keepdim=True)
    e = torch.ceil(torch.log2(top / LARGEST[format]))
    e = e.clamp(LOWEST, HIGHEST)
    e = torch.where((_power(e - 1) * LARGEST[format] >= top) & (e > LOWEST), e - 1, e)
    e = torch.where((_power(e) * LARGEST[format] < top) & (e < HIGHEST), e + 1, e)
    return _power(e)


def _power(e):
    """2^e, to the last bit."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x, format):
    if format == "int8":
        return torch.round(x)
    step = _power(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step
