"""What the token mixers are timed on: attention over a paged key-value cache, and the gated delta rule.

A layer of the model is a token mixer (attention in one layer of four, the gated
delta rule in the others) and the MoE block.  Each case is one call on one layer:

  op "append":   rotary positions (one axis, or time, height and width) on a call's
                 q and k, and k and v written to their places in the cache's pages.
  op "prompt":   causal attention of each sequence's new tokens over its pages, the
                 tokens of the call included (they are in the cache already).
  op "decode":   attention of one new token per sequence over its pages.
  op "delta":    the gated delta rule over packed prompts, states taken and left.
  op "step":     the gated delta rule for one token per sequence.

`lens` are the new tokens of the call's sequences and `ctx` what each had before.
`hq` query heads share `hkv` key-value heads of `dim` in order; for the delta rule
`hv` value heads share `hk` key heads.  With own set, run() calls the library;
otherwise it computes the same with elementary torch operations in 32 bits (64
for rotation angles and sums of log decays).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6  # of the L2 norm of the delta rule's q and k
CHUNK = 64  # tokens the plain delta rule takes together


def _mixer():
    path = os.path.join(os.getcwd(), "qe-qwen36-b50_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qe_mixer

    return qe_mixer


# -- the cases -----------------------------------------------------------------
# the model's layers: 16 query heads over 2 key-value heads of 256, rotation of the
# first 64 elements on three axes, pages of 256 positions; 16 key heads and 32 value
# heads of 128 in the delta rule
MODEL = {"hq": 16, "hkv": 2, "dim": 256, "page": 256, "rot": 64, "axes": 3}
DELTA = {"hk": 16, "hv": 32, "dk": 128, "dv": 128}


def listed():
    return [
        # eight sequences decoded together: the smallest append
        {"name": "append_decode_8", "op": "append", "dtype": "bf16", **MODEL, "lens": "1,1,1,1,1,1,1,1",
         "ctx": "0,17,255,256,1000,2047,4095,8191"},
        # a long prompt's keys and values, every element rotated, grouped heads of 128
        {"name": "append_8192", "op": "append", "dtype": "f16", "hq": 32, "hkv": 8, "dim": 128, "page": 64, "rot": 128,
         "axes": 1, "lens": "8192", "ctx": "0"},
        # a chat turn
        {"name": "prompt_100", "op": "prompt", "dtype": "bf16", **MODEL, "lens": "100", "ctx": "0"},
        # five prompts packed into one call, one of them with a cached beginning
        {"name": "prompt_packed_1999", "op": "prompt", "dtype": "f16", "hq": 32, "hkv": 8, "dim": 128, "page": 64,
         "rot": 128, "axes": 1, "lens": "1,37,512,1000,449", "ctx": "0,0,0,0,700"},
        # the benchmark's long prompt
        {"name": "prompt_8192", "op": "prompt", "dtype": "bf16", **MODEL, "lens": "8192", "ctx": "0"},
        # one token of one chat
        {"name": "decode_1_700", "op": "decode", "dtype": "bf16", **MODEL, "lens": "1", "ctx": "699"},
        # one token of one very long conversation
        {"name": "decode_1_100000", "op": "decode", "dtype": "bf16", **MODEL, "lens": "1", "ctx": "99999"},
        # a server's batch of ragged conversations
        {"name": "decode_24_ragged", "op": "decode", "dtype": "f16", "hq": 32, "hkv": 8, "dim": 128, "page": 64, "rot": 128,
         "axes": 1, "lens": ",".join(["1"] * 24), "ctx": ",".join(str(37 + 13 * i * i * i % 8111) for i in range(24))},
        # one token of one sequence through a delta-rule layer, the library's fp32 activations
        {"name": "step_1", "op": "step", "dtype": "f32", **DELTA, "lens": "1"},
        # a server's decode step
        {"name": "step_64", "op": "step", "dtype": "bf16", **DELTA, "lens": ",".join(["1"] * 64)},
        # three prompts packed into one call, fp32 activations
        {"name": "delta_packed_1999", "op": "delta", "dtype": "f32", **DELTA, "lens": "1200,99,700"},
        # the benchmark's long prompt
        {"name": "delta_8192", "op": "delta", "dtype": "bf16", **DELTA, "lens": "8192"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def ragged(total, n):
        """n lengths of at least one that sum to total (or to n, if that is more)."""
        w = [rng.uniform(0.05, 1.0) for _ in range(n)]
        return [max(1, int(total * x / sum(w))) for x in w]

    def text(v):
        return ",".join(str(x) for x in v)

    op = rng.choice(("append", "prompt", "prompt", "decode", "decode", "step", "delta", "delta"))
    if op in ("step", "delta"):
        hk, group = rng.choice(((16, 2), (8, 4), (12, 1), (4, 3)))
        case = {"op": op, "dtype": rng.choice(("f32", "bf16", "f16")), "hk": hk, "hv": hk * group,
                "dk": rng.choice((64, 128)), "dv": rng.choice((64, 128))}
        lens = [1] * spread(1, 64) if op == "step" else ragged(spread(1, 8000), rng.choice((1, 1, 2, 3, 7)))
        return {**case, "lens": text(lens)}
    hq, hkv, dim = rng.choice(((16, 2, 256), (32, 8, 128), (14, 2, 128), (12, 12, 64), (24, 8, 64), (8, 1, 256)))
    case = {"op": op, "dtype": rng.choice(("bf16", "f16")), "hq": hq, "hkv": hkv, "dim": dim,
            "page": rng.choice((16, 32, 64, 128, 256)), "rot": dim // rng.choice((1, 2, 4)), "axes": rng.choice((1, 3))}
    while True:
        if op == "decode":
            n = spread(1, 48)
            lens, ctx = [1] * n, [spread(1, 60000) - 1 for _ in range(n)]
        else:
            n = rng.choice((1, 1, 2, 3, 6))
            lens = ragged(spread(1, 8000), n)
            ctx = [rng.choice((0, spread(1, 20000))) for _ in range(n)]
        most = max(a + b for a, b in zip(lens, ctx))
        # no dearer than the listed ones, in work and in what the padded plain form holds
        if n * most * hkv * dim <= 24 * 8192 * 8 * 128 and hq * n * max(lens) * most <= 16 * 8192 * 8192 // 2:
            return {**case, "lens": text(lens), "ctx": text(ctx)}


# -- inputs ---------------------------------------------------------------------
def _ints(s):
    return [int(x) for x in s.split(",")]


def _sections(case):
    """Rotated pairs of each axis: time gets what height and width leave, as 11, 11 and 10 of 32."""
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return (pairs,)
    h = (pairs + 1) // 3
    w = (pairs - h) // 2
    return (pairs - h - w, h, w)


def _device_ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    lens = _ints(case["lens"])
    n, T = len(lens), sum(lens)
    starts = [sum(lens[:i]) for i in range(n + 1)]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case, "lens": lens, "T": T, "cu": _device_ints(starts)}
    if case["op"] in ("step", "delta"):
        hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
        # q, k and v leave a short convolution and a SiLU; a head's decay rate is its own, a token's gate scales it
        act = torch.nn.functional.silu
        s["q"], s["k"] = (act(normal(T, hk, dk, dtype=torch.float32)).to(dt) for _ in range(2))
        s["v"] = act(normal(T, hv, dv, dtype=torch.float32)).to(dt)
        rate = torch.exp(torch.rand(hv, generator=g, device="cuda") * math.log(2000.0) + math.log(1e-3))
        s["g"] = -rate * torch.nn.functional.softplus(normal(T, hv, dtype=torch.float32))
        s["beta"] = torch.sigmoid(normal(T, hv, dtype=torch.float32))
        # a pool of states: sequence i continues slot 2i (the first of several prompts starts from nothing) and
        # leaves its state in slot 2i + 1
        s["pool"] = normal(2 * n, hv, dk, dv, std=0.1, dtype=torch.float32)
        into = [2 * i for i in range(n)]
        if case["op"] == "delta" and n > 1:
            into[0] = -1
        s["into"], s["slots_in"], s["slots_out"] = into, _device_ints(into), _device_ints([2 * i + 1 for i in range(n)])
        s["out"] = torch.empty(T, hv, dv, dtype=dt, device="cuda")
        if own:
            s["handle"] = _mixer().GatedDelta(hk, hv, dk, dv, dtype=dt, t_max=max(T, 64), l2norm=True)
        return s
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    kv = [a + b for a, b in zip(lens, _ints(case["ctx"]))]
    per = [-(-x // page) for x in kv]
    width, total = max(per), sum(per)
    # pages in the order a busy server hands them out: any
    order = torch.randperm(total + 3, generator=g, device="cuda")[:total].to(torch.int32)
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(per, device="cuda"))
    col = torch.cat([torch.arange(x, device="cuda") for x in per])
    s["table"] = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    s["table"][row, col] = order
    s["kv"], s["kv_len"] = kv, _device_ints(kv)
    s["kc"], s["vc"] = (torch.empty(total + 3, hkv, page, dim, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2))
    # one projection makes q, k and v of a token side by side
    s["qkv"] = normal(T, hq + 2 * hkv, dim)
    s["q"], s["k"], s["v"] = s["qkv"].split((hq, hkv, hkv), dim=1)
    if case["op"] != "append":
        s["q"] = normal(T, hq, dim, std=2.0)  # scores as peaked as normalised heads with trained weights have them
    s["out"] = torch.empty(T, hq, dim, dtype=dt, device="cuda")
    # an image's tokens share a time and have a row and a column of it
    at = torch.cat([torch.arange(b - a, b, device="cuda") for a, b in zip(lens, kv)])
    s["pos"] = torch.stack([at // 3, at // 7 + 5, at % 61])[: case["axes"]].to(torch.int32) if case["axes"] == 3 else at[None].to(torch.int32)
    if own:
        m = _mixer()
        s["handle"] = m.Attention(hq, hkv, dim, page, dtype=dt, rotary=case["rot"], theta=1e7, sections=_sections(case),
                                  interleaved=case["axes"] == 3)
        s["batch"] = m.Batch(s["kv_len"], s["table"], None if case["op"] == "decode" else s["cu"], max_len=max(kv))
    return s


# -- one pass ---------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s, torch.cuda.current_stream())
    return {"append": _append, "prompt": _attend, "decode": _attend, "step": _step, "delta": _delta}[op](s)


def _own(op, s, stream):
    h = s["handle"]
    if op == "append":
        h.append(s["batch"], s["q"], s["k"], s["v"], s["kc"], s["vc"], s["out"], pos=s["pos"], stream=stream)
        return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}
    if op == "prompt":
        h.prompt(s["batch"], s["q"], s["kc"], s["vc"], s["out"], stream=stream)
        return {"out": s["out"]}
    if op == "decode":
        h.decode(s["batch"], s["q"], s["kc"], s["vc"], s["out"], stream=stream)
        return {"out": s["out"]}
    if op == "step":
        h.decode(s["q"], s["k"], s["v"], s["g"], s["beta"], s["pool"], s["slots_in"], s["slots_out"], s["out"], stream=stream)
    else:
        h.prompt(s["q"], s["k"], s["v"], s["g"], s["beta"], s["pool"], s["slots_in"], s["slots_out"], s["cu"], s["out"],
                 stream=stream)
    return {"out": s["out"], "pool": s["pool"]}


def _axes(case):
    """Axis of each rotated pair: axes take turns (time, height, width, time, ...) until height and width are used up."""
    pairs = case["rot"] // 2
    i = torch.arange(pairs, device="cuda")
    if case["axes"] == 1:
        return torch.zeros_like(i)
    _, h, w = _sections(case)
    return torch.where((i % 3 == 1) & (i < 3 * h), 1, torch.where((i % 3 == 2) & (i < 3 * w), 2, 0))


def _append(s):
    case, page = s["case"], s["case"]["page"]
    rot = case["rot"]
    inv = torch.pow(torch.tensor(1e7, dtype=torch.float64, device="cuda"),
                    -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = s["pos"].double()[_axes(case)].T * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        x = x.float()
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], dim=-1).to(s["kc"].dtype)

    s["out"].copy_(turn(s["q"]))
    token = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(s["cu"], token, right=True, out_int32=True) - 1
    at = s["kv_len"][seq] - s["cu"][seq + 1] + token
    p = s["table"][seq, at // page]
    s["kc"][p, :, at % page] = turn(s["k"])
    s["vc"][p, :, at % page] = s["v"]
    return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}


def _attend(s):
    case = s["case"]
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    n, most_q, most_kv = len(s["lens"]), max(s["lens"]), max(s["kv"])
    # sequences padded to the longest: queries [n, hkv, group * most_q, dim], keys and values [n, hkv, most_kv, dim]
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    j = torch.arange(most_q, device="cuda")
    there = j < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(there, cu[:-1, None] + j, 0)
    q = s["q"][rows].float().reshape(n, most_q, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)

    def cached(c):
        return c[s["table"].long()].transpose(1, 2).reshape(n, hkv, -1, dim)[:, :, :most_kv].float()

    scores = q @ cached(s["kc"]).transpose(2, 3) * dim ** -0.5
    place = (kv_len - (cu[1:] - cu[:-1]))[:, None] + j  # of each query in its sequence
    key = torch.arange(most_kv, device="cuda")
    seen = (key <= place[..., None]) & there[..., None]
    scores = scores.view(n, hkv, hq // hkv, most_q, most_kv).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = cached(s["vc"]).masked_fill_((key >= kv_len[:, None])[:, None, :, None], 0.0)
    o = (p.view(n, hkv, -1, most_kv) @ v).view(n, hkv, hq // hkv, most_q, dim) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, most_q, hq, dim)[there])
    return {"out": s["out"]}


def _heads(s):
    """q and k normalised and repeated for the value heads, and v, in 32 bits."""
    case = s["case"]
    group = case["hv"] // case["hk"]
    q, k = (x.float() for x in (s["q"], s["k"]))
    q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS) * case["dk"] ** -0.5
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS)
    return q.repeat_interleave(group, 1), k.repeat_interleave(group, 1), s["v"].float()


def _initial(s):
    first = s["pool"][s["slots_in"].clamp(min=0).long()]
    return torch.where((s["slots_in"] >= 0)[:, None, None, None], first, 0.0)


def _step(s):
    q, k, v = _heads(s)
    S = _initial(s) * s["g"].exp()[..., None, None]
    u = s["beta"][..., None] * (v - (k[..., None] * S).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    s["out"].copy_((q[..., None] * S).sum(-2))
    s["pool"][s["slots_out"].long()] = S
    return {"out": s["out"], "pool": s["pool"]}


def _delta(s):
    case = s["case"]
    n, chunks = len(s["lens"]), -(-max(s["lens"]) // CHUNK)
    cu = s["cu"].long()
    j = torch.arange(chunks * CHUNK, device="cuda")
    there = j < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(there, cu[:-1, None] + j, 0)

    def cut(x):  # [T, heads, ...] -> [n, heads, chunks, CHUNK, ...], nothing where a sequence has ended
        x = torch.where(there.view(n, -1, *[1] * (x.dim() - 1)), x[rows], 0)
        return x.view(n, chunks, CHUNK, *x.shape[2:]).movedim(3, 1)

    q, k, v = (cut(x) for x in _heads(s))
    beta, b = cut(s["beta"])[..., None], cut(s["g"]).double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    fade = torch.where(lower, b[..., :, None] - b[..., None, :], -math.inf).exp().float()
    eye = torch.eye(CHUNK, device="cuda")
    # (I + A)^-1 of a strictly lower A: (I - A)(I + A^2)(I + A^4) ... ends at A^32 of 64 rows
    A = (beta * (k @ k.transpose(-1, -2)) * fade).tril(-1)
    inverse, power = eye - A, A
    for _ in range(CHUNK.bit_length() - 2):
        power = power @ power
        inverse = inverse @ (eye + power)
    within = q @ k.transpose(-1, -2) * fade
    grown, last = b.exp().float()[..., None], b[..., -1:]
    left = (last - b).exp().float()[..., None] * k
    S, outs = _initial(s), []
    for c in range(chunks):
        u = inverse[:, :, c] @ (beta[:, :, c] * (v[:, :, c] - grown[:, :, c] * (k[:, :, c] @ S)))
        outs.append(grown[:, :, c] * (q[:, :, c] @ S) + within[:, :, c] @ u)
        S = last[:, :, c, :, None].exp().float() * S + left[:, :, c].transpose(-1, -2) @ u
    o = torch.stack(outs, 2).movedim(1, 3).reshape(n, chunks * CHUNK, case["hv"], case["dv"])
    s["out"].copy_(o[there])
    s["pool"][s["slots_out"].long()] = S
    return {"out": s["out"], "pool": s["pool"]}


# -- what a pass cannot do without -------------------------------------------------
def work(case):
    lens = _ints(case["lens"])
    n, T, size = len(lens), sum(lens), 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("step", "delta"):
        hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
        states = 2 * n - (1 if case["op"] == "delta" and n > 1 else 0)
        # a token: the state faded, read for k, added to, read for q
        return {"bytes": T * (2 * hk * dk + 2 * hv * dv) * size + T * hv * 8 + states * hv * dk * dv * 4,
                "flops": 7 * T * hv * dk * dv}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["op"] == "append":
        return {"bytes": T * (2 * hq + 4 * hkv) * dim * size + T * case["axes"] * 4, "flops": 3 * T * (hq + hkv) * case["rot"]}
    ctx = _ints(case["ctx"])
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(lens, ctx))
    return {"bytes": 2 * T * hq * dim * size + 2 * sum(lens + ctx) * hkv * dim * size, "flops": 4 * pairs * hq * dim}


# -- the definitions, in 64 bits ------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("step", "delta"):
        return _exact_delta(case, s)
    table, page, group = s["table"].cpu(), case["page"], case["hq"] // case["hkv"]
    if case["op"] == "append":
        out = {"q": s["q"].double(), "kc": s["kc"].double(), "vc": s["vc"].double()}
        k, half = s["k"].double(), case["rot"] // 2
        turns = [_sections(case)[1] if case["axes"] == 3 else 0, _sections(case)[2] if case["axes"] == 3 else 0]
        for i in range(half):
            axis = 1 if i % 3 == 1 and i // 3 < turns[0] else 2 if i % 3 == 2 and i // 3 < turns[1] else 0
            z = torch.polar(torch.ones_like(s["pos"][0], dtype=torch.float64), s["pos"][axis].double() * 1e7 ** (-2 * i / case["rot"]))
            for x in (out["q"], k):
                r = torch.complex(x[:, :, i], x[:, :, i + half]) * z[:, None]
                x[:, :, i], x[:, :, i + half] = r.real, r.imag
        t = 0
        for i, (new, kv) in enumerate(zip(s["lens"], s["kv"])):
            at = torch.arange(kv - new, kv)
            p = table[i, at // page].long().cuda()
            out["kc"][p, :, (at % page).cuda()] = k[t: t + new]
            out["vc"][p, :, (at % page).cuda()] = s["v"][t: t + new].double()
            t += new
        return out
    if case["hq"] * sum(s["kv"]) * max(s["lens"]) > 4e9:
        return None
    out, t = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (new, kv) in enumerate(zip(s["lens"], s["kv"])):
        pages = table[i, : -(-kv // page)].long().cuda()
        later = torch.arange(kv, device="cuda") > torch.arange(kv - new, kv, device="cuda")[:, None]
        for h in range(case["hq"]):
            k, v = (c[pages, h // group].reshape(-1, case["dim"])[:kv].double() for c in (s["kc"], s["vc"]))
            x = s["q"][t: t + new, h].double() @ k.T / math.sqrt(case["dim"])
            out[t: t + new, h] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v
        t += new
    return {"out": out}


def _exact_delta(case, s):
    group = case["hv"] // case["hk"]
    pool = s["pool"].double()
    q, k = (torch.repeat_interleave(x.double() / torch.sqrt(x.double().pow(2).sum(-1, keepdim=True) + EPS), group, 1)
            for x in (s["q"], s["k"]))
    v, fade, beta = s["v"].double(), s["g"].double().exp(), s["beta"].double()
    q = q / math.sqrt(case["dk"])
    out, t = torch.empty(v.shape, dtype=torch.float64, device="cuda"), 0
    for i, new in enumerate(s["lens"]):
        S = pool[2 * i].clone() if s["into"][i] >= 0 else torch.zeros_like(pool[0])
        for t in range(t, t + new):
            S *= fade[t, :, None, None]
            seen = (k[t, :, None] @ S)[:, 0]
            S += k[t, :, :, None] * (beta[t, :, None] * (v[t] - seen))[:, None]
            out[t] = (q[t, :, None] @ S)[:, 0]
        t += 1
        pool[2 * i + 1] = S
    return {"out": out, "pool": pool}
