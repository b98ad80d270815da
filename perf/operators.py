"""The operators around a key/value cache held in 4 bits, as measurable cases.

  kind "rotary"   rotary positions of queries and keys: both layouts, part of the head, scaled frequencies
  kind "append"   queries and keys rotated, keys and values written to the cache in 4 bits, and the written
                  rows read back as the values that they stand for
  kind "attend"   attention of new tokens over the cache: one token a sequence, a few, or a prompt

A cache row of a head is groups of 64 values, each with a scale s and a lowest value l as FP16; value = s c + l
with a code c of 0..15.  Eight neighbouring values lie in four bytes: value 2 i in nibble i, value 2 i + 1 in
nibble i + 4.  Sequence b of a call has the rows first[b] .. first[b + 1] - 1 of its tensors, which sit at the
positions lens[b] - n .. lens[b] - 1 of the cache.

run() with own = False computes the operators with elementary torch operations; exact() computes the same from
their definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP, LIMIT = 64, 61440.0
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the next token of one conversation: a launch
        dict(name="rotary_1_fp16", kind="rotary", type="fp16", tokens=1, heads=32, kv_heads=8, dim=64, rot=64, half=False, base=500000.0,
             scaling="none", start=1500),
        # a piece of a long document, far behind the length that a model was trained on
        dict(name="rotary_8192_far_bf16", kind="rotary", type="bf16", tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, half=True,
             base=10000.0, scaling="yarn", start=120000),
        # a prompt of a 32-bit model that turns a part of each head
        dict(name="rotary_1531_part_fp32", kind="rotary", type="fp32", tokens=1531, heads=32, kv_heads=32, dim=80, rot=32, half=True,
             base=10000.0, scaling="linear", start=0),
        # one token for each of 24 sequences of a small server
        dict(name="append_24_bf16", kind="append", type="bf16", batch=24, new=1, lo=300, hi=8000, heads=32, kv_heads=8, dim=128, half=True,
             base=500000.0, scaling="llama3"),
        # three prompts at once, of different lengths
        dict(name="append_3_prompts_fp16", kind="append", type="fp16", batch=3, new=2003, lo=0, hi=0, heads=32, kv_heads=8, dim=64, half=False,
             base=500000.0, scaling="none"),
        # the next token of one conversation of a small model
        dict(name="attend_1x300_fp16", kind="attend", type="fp16", batch=1, new=1, lo=300, hi=300, heads=32, kv_heads=8, dim=64),
        # the next token behind a book
        dict(name="attend_1x131000_bf16", kind="attend", type="bf16", batch=1, new=1, lo=131000, hi=131000, heads=32, kv_heads=8, dim=128),
        # one token for each sequence of a server, short and long ones
        dict(name="attend_32_ragged_fp16", kind="attend", type="fp16", batch=32, new=1, lo=16, hi=8000, heads=32, kv_heads=8, dim=128),
        # up to five proposed tokens a sequence, checked in one call
        dict(name="attend_6x5_bf16", kind="attend", type="bf16", batch=6, new=5, lo=800, hi=3600, heads=32, kv_heads=8, dim=128),
        # a document as a prompt
        dict(name="attend_prompt_2000_fp16", kind="attend", type="fp16", batch=1, new=2000, lo=0, hi=0, heads=32, kv_heads=8, dim=128),
        # a piece of a long document behind what was read before
        dict(name="attend_512x16000_bf16", kind="attend", type="bf16", batch=1, new=512, lo=16000, hi=16000, heads=32, kv_heads=8, dim=128),
        # new questions and continued ones in one call
        dict(name="attend_9_prompts_fp16", kind="attend", type="fp16", batch=9, new=701, lo=5, hi=2500, heads=32, kv_heads=8, dim=64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(32, 8), (32, 8), (16, 4), (16, 16), (8, 1), (12, 4), (40, 8), (6, 2)]


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend"])
    heads, kv_heads = rng.choice(HEADS)
    base, scaling = rng.choice([10000.0, 500000.0]), rng.choice(["none", "linear", "yarn", "llama3"])
    half = rng.random() < 0.5
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = dim if rng.random() < 0.5 else 16 * rng.randint(1, dim // 16)
        return dict(kind=kind, type=rng.choice(["fp16", "bf16", "fp32"]), tokens=_log_int(rng, 1, 4096), heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rot, half=half, base=base, scaling=scaling, start=rng.randint(0, 200000))
    kind_type, dim = rng.choice(["fp16", "bf16"]), rng.choice([64, 128, 128])
    if kind == "append":
        batch, new = (rng.randint(1, 48), 1) if rng.random() < 0.5 else (rng.randint(1, 4), _log_int(rng, 2, 2000))
        lo = _log_int(rng, 1, 4000) - 1
        return dict(kind=kind, type=kind_type, batch=batch, new=new, lo=lo, hi=lo + rng.randint(0, 4000), heads=heads, kv_heads=kv_heads, dim=dim,
                    half=half, base=base, scaling=scaling)
    form = rng.choice(["step", "step", "few", "prompt", "prompt"])
    if form == "step":
        batch = _log_int(rng, 1, 48)
        lo = _log_int(rng, 1, 160000 // batch) - 1
        return dict(kind=kind, type=kind_type, batch=batch, new=1, lo=lo, hi=_log_int(rng, lo + 1, 160000 // batch + 1), heads=heads,
                    kv_heads=kv_heads, dim=dim)
    if form == "few":
        lo = _log_int(rng, 1, 4000) - 1
        return dict(kind=kind, type=kind_type, batch=rng.randint(1, 16), new=rng.randint(2, 16), lo=lo, hi=lo + rng.randint(0, 4000), heads=heads,
                    kv_heads=kv_heads, dim=dim)
    batch, new = rng.randint(1, 4), _log_int(rng, 17, 1500)
    lo = rng.choice([0, 0, rng.randint(1, 3000)])
    return dict(kind=kind, type=kind_type, batch=batch, new=new, lo=lo, hi=lo, heads=heads, kv_heads=kv_heads, dim=dim)


# ---- inputs ------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """(positions before the call, new tokens) of each sequence: spread over the logarithm of the range, the first
    sequence at its top; new tokens of several sequences from a fifth of the most on."""
    before, new = [], []
    for b in range(case["batch"]):
        u = b * 0.6180339887498949 % 1.0
        before.append(round(math.exp((1 - u) * math.log(case["hi"] + 1) + u * math.log(case["lo"] + 1))) - 1)
        new.append(max(1, round(case["new"] * (1 - 0.8 * (b * 0.7548776662466927 % 1.0)))))
    return before, new


SCALINGS = {
    "none": None,
    "linear": dict(type="linear", factor=4.0),
    "yarn": dict(type="yarn", factor=32.0, original=4096, beta_fast=32.0, beta_slow=1.0),
    "llama3": dict(type="llama3", factor=32.0, original=8192, low=1.0, high=4.0),
}


def _frequencies(rot, base, scaling):
    """Angles a position, one for each pair, and the factor of the result."""
    f = [base ** (-2 * i / rot) for i in range(rot // 2)]
    s = SCALINGS[scaling]
    if scaling == "linear":
        f = [v / s["factor"] for v in f]
    elif scaling == "yarn":
        def pair_of(turns):                       # the pair that turns so often over the original length
            return rot * math.log(s["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair_of(s["beta_fast"])), 0), min(math.ceil(pair_of(s["beta_slow"])), rot - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        return [v / s["factor"] * r + v * (1 - r) for v, r in zip(f, ramp)], 0.1 * math.log(s["factor"]) + 1.0
    elif scaling == "llama3":
        def scaled(v):
            turns = s["original"] * v / (2 * math.pi)
            mix = min(max((turns - s["low"]) / (s["high"] - s["low"]), 0.0), 1.0)
            return (1 - mix) * v / s["factor"] + mix * v
        f = [scaled(v) for v in f]
    return f, 1.0


def _pack(c):
    """Codes [.., dim] as bytes [.., dim / 2]."""
    w = c.reshape(*c.shape[:-1], -1, 4, 2).transpose(-1, -2).reshape(*c.shape[:-1], -1, 8)
    return (w[..., 0::2] | w[..., 1::2] << 4).to(torch.uint8).reshape(*c.shape[:-1], -1)


def _unpack(b):
    w = torch.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], -1, 2, 4).transpose(-1, -2)
    return w.reshape(*b.shape[:-1], -1)


def _quantise(x):
    """Bytes [.., dim / 2] and (s, l) [.., dim / 64, 2] of FP32 values [.., dim]."""
    x = x.clamp(-LIMIT, LIMIT).reshape(*x.shape[:-1], -1, GROUP)
    low = x.amin(-1).half()
    s = ((x.amax(-1) - low.float()) / 15.0).half()
    t = (x - low.float()[..., None]) / torch.where(s > 0, s, 1).float()[..., None]
    c = torch.where(s[..., None] > 0, t.round().clamp(0, 15), 0).to(torch.uint8)
    return _pack(c.flatten(-2)), torch.stack((s, low), -1)


def _values(codes, params):
    """FP32 values [.., dim]."""
    c = _unpack(codes).float().reshape(*codes.shape[:-1], -1, GROUP)
    p = params.float()
    return (c * p[..., :1] + p[..., 1:]).flatten(-2)


def _random_cache(gen, batch, kv_heads, rows, dim):
    """A cache whose rows hold keys and values as attention layers have them: a mean and a spread of their own for each channel."""
    out = []
    for spread in (1.0, 0.5):
        mean = 0.5 * torch.randn(kv_heads, 1, dim, generator=gen, device="cuda")
        size = spread * (0.6 + 0.8 * torch.rand(kv_heads, 1, dim, generator=gen, device="cuda"))
        codes = torch.empty(batch, kv_heads, rows, dim // 2, dtype=torch.uint8, device="cuda")
        params = torch.empty(batch, kv_heads, rows, dim // GROUP, 2, dtype=torch.float16, device="cuda")
        for b in range(batch):
            codes[b], params[b] = _quantise(mean + size * torch.randn(kv_heads, rows, dim, generator=gen, device="cuda"))
        out += [codes, params]
    return out


def prepare(case, seed):
    gen, t = _gen(seed), TYPES[case["type"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(t)

    state = dict(case=case)
    if case["kind"] != "attend":
        rot = case.get("rot", dim)
        freq, state["amplitude"] = _frequencies(rot, case["base"], case["scaling"])
        state["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
        if own:
            from ternary_llm_b200 import cache4_ops
            state["table"] = cache4_ops.RotaryTable(rot, case["base"], half=case["half"], scaling=SCALINGS[case["scaling"]])
    if case["kind"] == "rotary":
        n = case["tokens"]
        state.update(q=rand(n, heads, dim), k=rand(n, kv_heads, dim), positions=torch.arange(case["start"], case["start"] + n, dtype=torch.int32, device="cuda"))
        state.update(q_out=torch.empty_like(state["q"]), k_out=torch.empty_like(state["k"]))
        return state
    before, new = _lengths(case)
    lens = [a + b for a, b in zip(before, new)]
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    rows = (max(lens) + 127) // 128 * 128
    state.update(first=torch.tensor(first, dtype=torch.int32, device="cuda"), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 q=rand(first[-1], heads, dim), most_new=max(new), most_len=max(lens))
    if case["kind"] == "append":
        state.update(k=rand(first[-1], kv_heads, dim), v=rand(first[-1], kv_heads, dim))
        state.update(q_out=torch.empty_like(state["q"]), k_back=torch.empty_like(state["k"]), v_back=torch.empty_like(state["v"]))
        cache = [torch.zeros(case["batch"], kv_heads, rows, *last, dtype=dt, device="cuda")
                 for last, dt in (((dim // 2,), torch.uint8), ((dim // GROUP, 2), torch.float16)) * 2]
    else:
        state["out"] = torch.empty_like(state["q"])
        cache = _random_cache(gen, case["batch"], kv_heads, rows, dim)
    state["cache"] = cache
    if own:
        from ternary_llm_b200 import cache4_ops
        state["handle"] = cache4_ops.Cache4(*cache)
    return state


# ---- the operators ----------------------------------------------------------------------
def _places(first, lens, tokens):
    """(sequence, position) of each row."""
    row = torch.arange(tokens, device=first.device)
    seq = torch.searchsorted(first[1:].long(), row, right=True)
    return seq, lens.long()[seq] - first.long()[seq + 1] + row


def _rotate(x, positions, freq, amplitude, half):
    """x [tokens, heads, dim] in 32 bits, the angles in 64."""
    angle = positions.double()[:, None] * freq
    cos, sin = ((f(angle) * amplitude).float()[:, None] for f in (torch.cos, torch.sin))
    rot = 2 * freq.numel()
    y = x.float()
    a, b = (y[..., :rot // 2], y[..., rot // 2:rot]) if half else (y[..., 0:rot:2], y[..., 1:rot:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((a, b), -1) if half else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((turned, y[..., rot:]), -1)


def _plain_attend(s):
    """All sequences side by side, padded to the longest."""
    case, (kc, kp, vc, vp) = s["case"], s["cache"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    seq, position = _places(s["first"], s["lens"], s["q"].shape[0])
    place = torch.arange(s["q"].shape[0], device="cuda") - s["first"].long()[seq]
    n, m = s["most_new"], s["most_len"]
    q = torch.zeros(case["batch"], n, kv_heads, heads // kv_heads, dim, device="cuda")
    q[seq, place] = s["q"].float().reshape(-1, kv_heads, heads // kv_heads, dim)
    last = torch.zeros(case["batch"], n, dtype=torch.long, device="cuda")
    last[seq, place] = position
    k, v = _values(kc[:, :, :m], kp[:, :, :m]), _values(vc[:, :, :m], vp[:, :, :m])
    score = torch.einsum("bngrd,bgmd->bgrnm", q, k) * dim ** -0.5
    sees = torch.arange(m, device="cuda") <= last[..., None]
    score = score.masked_fill_(~sees[:, None, None], -torch.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    o = torch.einsum("bgrnm,bgmd->bngrd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    return o[seq, place].reshape(-1, heads, dim).to(s["q"].dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        from ternary_llm_b200 import cache4_ops as ops
        if case["kind"] == "rotary":
            ops.rotary(s["q"], s["k"], s["positions"], s["table"], s["q_out"], s["k_out"])
            return s["q_out"], s["k_out"]
        if case["kind"] == "append":
            ops.append(s["handle"], s["q"], s["k"], s["v"], s["first"], s["lens"], s["table"], s["q_out"])
            ops.read(s["handle"], s["k_back"], s["v_back"], s["first"], s["lens"])
            return s["q_out"], s["k_back"], s["v_back"]
        ops.attention(s["handle"], s["q"], s["out"], s["first"], s["lens"], max_new=s["most_new"], max_len=s["most_len"])
        return s["out"]
    if case["kind"] == "rotary":
        return tuple(_rotate(s[n], s["positions"], s["freq"], s["amplitude"], case["half"]).to(s[n].dtype) for n in ("q", "k"))
    if case["kind"] == "append":
        t = s["q"].dtype
        seq, position = _places(s["first"], s["lens"], s["q"].shape[0])
        q, k = (_rotate(s[n], position, s["freq"], s["amplitude"], case["half"]).to(t) for n in ("q", "k"))
        kc, kp, vc, vp = s["cache"]
        kc[seq, :, position], kp[seq, :, position] = _quantise(k.float())
        vc[seq, :, position], vp[seq, :, position] = _quantise(s["v"].float())
        return q, _values(kc[seq, :, position], kp[seq, :, position]).to(t), _values(vc[seq, :, position], vp[seq, :, position]).to(t)
    return _plain_attend(s)


def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["type"] == "fp32" else 2
    if case["kind"] == "rotary":
        values = case["tokens"] * (heads + kv_heads) * dim
        return {"bytes": 2 * size * values + 4 * case["tokens"], "flops": 3 * values * case["rot"] / dim}
    before, new = _lengths(case)
    tokens, row = sum(new), kv_heads * (dim // 2 + dim // GROUP * 4)
    if case["kind"] == "append":                  # q turned, k and v written as codes, read again as values
        return {"bytes": size * tokens * dim * (2 * heads + 4 * kv_heads) + 4 * tokens * row, "flops": tokens * dim * (3 * heads + 17 * kv_heads)}
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(before, new))
    return {"bytes": 2 * size * tokens * heads * dim + 2 * row * sum(a + n for a, n in zip(before, new)), "flops": 4 * dim * heads * pairs}


# ---- 64 bits ------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)

    def turned(x, positions):
        """As a product with e^(i angle)."""
        x, pairs = x.double(), s["freq"].numel()
        head, tail = x[..., :2 * pairs], x[..., 2 * pairs:]
        z = torch.complex(*(head.unflatten(-1, (2, pairs)).unbind(-2) if case["half"] else head.unflatten(-1, (pairs, 2)).unbind(-1)))
        angle = torch.outer(positions.double(), s["freq"])
        z = z * torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, None]
        parts = (z.real, z.imag)
        return torch.cat((torch.cat(parts, -1) if case["half"] else torch.stack(parts, -1).flatten(-2), tail), -1)

    if case["kind"] == "rotary":
        return turned(s["q"], s["positions"]), turned(s["k"], s["positions"])
    bounds, lens = s["first"].tolist(), s["lens"].tolist()
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(m - (e - b), m, device="cuda") for b, e, m in zip(bounds, bounds[1:], lens)])

        def held(x):
            """The value of 16 evenly spaced ones that is nearest, between the lowest and the highest of 64 neighbours."""
            x = x.to(TYPES[case["type"]]).double().unflatten(-1, (-1, GROUP)).clamp(-LIMIT, LIMIT)
            low = x.min(-1, keepdim=True).values.half().double()
            step = ((x.max(-1, keepdim=True).values - low) / 15).half().double()
            code = ((x - low) / step).nan_to_num(0.0).round().clamp(0, 15)
            return (low + step * code).flatten(-2)

        return turned(s["q"], positions), held(turned(s["k"], positions)), held(s["v"])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    kc, kp, vc, vp = s["cache"]
    per = case["heads"] // case["kv_heads"]
    nibble = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device="cuda")
    for b, m in enumerate(lens):
        def table(codes, params):
            word = codes[b, :, :m].unflatten(-1, (-1, 4)).long()
            word = word[..., 0] + (word[..., 1] << 8) + (word[..., 2] << 16) + (word[..., 3] << 24)
            c = (word[..., None] >> 4 * nibble) % 16
            p = params[b, :, :m].double().repeat_interleave(GROUP, -2)
            return p[..., 0] * c.flatten(-2) + p[..., 1]
        k, v = table(kc, kp), table(vc, vp)
        at = torch.arange(m, device="cuda")
        for h in range(case["heads"]):
            rows = s["q"][bounds[b]:bounds[b + 1], h].double()
            x = rows @ k[h // per].T / math.sqrt(case["dim"])
            x[at[None] > at[m - len(rows):, None]] = -torch.inf
            out[bounds[b]:bounds[b + 1], h] = torch.softmax(x, -1) @ v[h // per]
    return out
