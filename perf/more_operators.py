"""What attention over an 8-bit cache, and of a batch with a shared beginning, is timed on.

Each case is one call on one attention layer; `cache` is the pages' type ("i8": integers with a
scale for each position and head, "f8": the same with 8-bit floating point of 4 exponent bits,
"16": the activations' type):

  op "append":   q and k normalised per head and rotated (one axis, or time, height and
                 width), k and v written to their places in the cache's pages; what was
                 written to an 8-bit cache is read back.
  op "read":     positions of an 8-bit cache back in 16 bits.
  op "prompt":   causal attention of each sequence's new tokens over its 8-bit pages, the
                 tokens of the call included (they are in the cache already).
  op "decode":   attention of one new token per sequence over its 8-bit pages.
  op "shared":   the same for sequences that share their beginning with others of a group:
                 `members` sequences in each group, the first `prefix` positions shared.

`lens` are the new tokens of the call's sequences and `ctx` what each had before (behind the
shared beginning).  `hq` query heads share `hkv` key-value heads of `dim` in order.  With own
set, run() calls the library; otherwise it computes the same with elementary torch operations
in 32 bits (64 for rotation angles).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"i8": torch.int8, "f8": torch.float8_e4m3fn}
MOST = {"i8": 127.0, "f8": 448.0}  # the greatest code
EPS = 1e-6  # of the norms


def _mixer():
    path = os.path.join(os.getcwd(), "qe-qwen36-b50_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qe_mixer

    return qe_mixer


# -- the cases -----------------------------------------------------------------
# the model's attention layers: 16 query heads over 2 key-value heads of 256, rotation of the first
# 64 elements on three axes, pages of 256 positions; and a common geometry with heads of 128
MODEL = {"hq": 16, "hkv": 2, "dim": 256, "page": 256, "rot": 64, "axes": 3}
WIDE = {"hq": 32, "hkv": 8, "dim": 128, "page": 64, "rot": 128, "axes": 1}


def _text(v):
    return ",".join(str(x) for x in v)


def listed():
    ones = lambda n: _text([1] * n)  # noqa: E731
    return [
        # eight sequences decoded together: the smallest append
        {"name": "append8_decode_8", "op": "append", "dtype": "bf16", "cache": "i8", "in": "f32", **MODEL, "lens": ones(8),
         "ctx": "0,17,255,256,1000,2047,4095,8191"},
        # a long prompt into an 8-bit cache, every element rotated
        {"name": "append8_8000", "op": "append", "dtype": "f16", "cache": "f8", "in": "f16", **WIDE, "lens": "8000", "ctx": "0"},
        # a prompt into a 16-bit cache: the norms in the rotation's pass
        {"name": "append_normed_2000", "op": "append", "dtype": "bf16", "cache": "16", "in": "bf16", **MODEL, "lens": "2000", "ctx": "333"},
        # one conversation handed over in 16 bits, and a server's, ragged
        {"name": "read_700", "op": "read", "dtype": "bf16", "cache": "i8", **MODEL, "lens": "700", "ctx": "0"},
        {"name": "read_ragged", "op": "read", "dtype": "f16", "cache": "f8", **WIDE, "lens": "5001,37,9999,1,2500,640", "ctx": "0,0,0,900,0,0"},
        # one token of one chat
        {"name": "decode8_1_900", "op": "decode", "dtype": "bf16", "cache": "i8", **MODEL, "lens": "1", "ctx": "899"},
        # a server's batch of ragged conversations
        {"name": "decode8_24_ragged", "op": "decode", "dtype": "f16", "cache": "f8", **WIDE, "lens": ones(24),
         "ctx": _text(37 + 13 * i * i * i % 8111 for i in range(24))},
        # three prompts packed into one call, one of them with a cached beginning
        {"name": "prompt8_packed_1500", "op": "prompt", "dtype": "f16", "cache": "i8", **WIDE, "lens": "200,333,967", "ctx": "0,1700,0"},
        # the benchmark's long prompt
        {"name": "prompt8_8192", "op": "prompt", "dtype": "bf16", "cache": "f8", **MODEL, "lens": "8192", "ctx": "0"},
        # four answers to one question
        {"name": "shared_4_1000", "op": "shared", "dtype": "bf16", "cache": "i8", **MODEL, "lens": ones(4), "ctx": "0,5,60,150", "members": "4",
         "prefix": "1000"},
        # a server's batch behind one long system prompt
        {"name": "shared_32_8000", "op": "shared", "dtype": "bf16", "cache": "16", **MODEL, "lens": ones(32),
         "ctx": _text(11 + 37 * i * i % 1501 for i in range(32)), "members": "32", "prefix": "8000"},
        # three system prompts
        {"name": "shared_64_groups", "op": "shared", "dtype": "f16", "cache": "f8", **WIDE, "lens": ones(64),
         "ctx": _text(29 * i * i % 997 for i in range(64)), "members": "40,16,8", "prefix": "6003,2500,300"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def ragged(total, n):
        """n lengths of at least one that sum to total (or to n, if that is more)."""
        w = [rng.uniform(0.05, 1.0) for _ in range(n)]
        return [max(1, int(total * x / sum(w))) for x in w]

    op = rng.choice(("append", "append", "read", "prompt", "prompt", "decode", "decode", "shared", "shared"))
    dtype = rng.choice(("bf16", "f16"))
    hq, hkv, dim = rng.choice(((16, 2, 256), (32, 8, 128), (14, 2, 128), (12, 12, 64), (24, 8, 64), (8, 1, 256)))
    case = {"op": op, "dtype": dtype, "cache": rng.choice(("i8", "f8", "16") if op in ("append", "shared") else ("i8", "f8")), "hq": hq, "hkv": hkv,
            "dim": dim, "page": rng.choice((16, 32, 64, 128, 256)), "rot": dim // rng.choice((1, 2, 4)), "axes": rng.choice((1, 3))}
    if op == "append":
        case["in"] = rng.choice((dtype, "f32"))
    while True:
        if op == "shared":
            n_groups = rng.choice((1, 1, 1, 2, 4))
            members = ragged(spread(max(2, n_groups), 64), n_groups)
            n = sum(members)
            prefix = [spread(16, 16000) for _ in members]
            lens, ctx = [1] * n, [spread(1, 2000) - 1 for _ in range(n)]
            # no dearer than the listed ones, in rows by keys and in what the padded plain form holds
            if hq * n * max(prefix) <= 32 * 64 * 6003 and (n_groups * max(prefix) + n * max(ctx)) * hkv * dim <= 120000 * 1024:
                return {**case, "lens": _text(lens), "ctx": _text(ctx), "members": _text(members), "prefix": _text(prefix)}
            continue
        if op == "decode":
            n = spread(1, 48)
            lens, ctx = [1] * n, [spread(1, 60000) - 1 for _ in range(n)]
        else:
            n = rng.choice((1, 1, 2, 3, 6))
            lens = ragged(spread(1, 8000), n)
            ctx = [rng.choice((0, spread(1, 20000))) for _ in range(n)]
        most = max(a + b for a, b in zip(lens, ctx))
        if n * most * hkv * dim <= 24 * 8192 * 8 * 128 and (op != "prompt" or hq * n * max(lens) * most <= 16 * 8192 * 8192 // 2):
            return {**case, "lens": _text(lens), "ctx": _text(ctx)}


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


def _lengths(case):
    """Positions of each sequence, and how many of them are its group's."""
    lens, ctx = _ints(case["lens"]), _ints(case["ctx"])
    if case["op"] != "shared":
        return [a + b for a, b in zip(lens, ctx)], [0] * len(lens)
    of = [p for m, p in zip(_ints(case["members"]), _ints(case["prefix"])) for _ in range(m)]
    return [a + b + p for a, b, p in zip(lens, ctx, of)], of


def _quantised(x, cache):
    """Codes and scales of the last axis's rows."""
    scale = x.abs().amax(-1) / MOST[cache]
    y = x / torch.where(scale == 0, 1.0, scale)[..., None]
    return (y.round() if cache == "i8" else y).to(CODES[cache]), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, cache = DTYPES[case["dtype"]], case["cache"]
    lens = _ints(case["lens"])
    n, T = len(lens), sum(lens)
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    kv, of_group = _lengths(case)

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case, "lens": lens, "T": T, "kv": kv, "kv_len": _device_ints(kv), "cu": _device_ints([sum(lens[:i]) for i in range(n + 1)])}
    # a sequence has the pages that are not wholly its group's to itself, but for the first of a group, whose pages hold
    # the shared positions
    members = _ints(case["members"]) if case["op"] == "shared" else [1] * n
    starts = [sum(members[:i]) for i in range(len(members) + 1)]
    per = [-(-x // page) for x in kv]
    theirs = [0 if i in starts else of_group[i] // page for i in range(n)]
    width, total = max(per), sum(per) - sum(theirs)
    # pages in the order a busy server hands them out: any
    order = torch.randperm(total + 3, generator=g, device="cuda")[:total].to(torch.int32)
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor([a - b for a, b in zip(per, theirs)], device="cuda"))
    col = torch.cat([torch.arange(b, a, device="cuda") for a, b in zip(per, theirs)])
    s["table"] = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    s["table"][row, col] = order
    for a, b in zip(starts[:-1], starts[1:]):
        s["table"][a + 1: b, : of_group[a] // page] = s["table"][a, : of_group[a] // page]
    shape = (total + 3, hkv, page, dim)
    if cache == "16":
        s["kc"], s["vc"] = (torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2))
    else:
        for c in ("k", "v"):
            s[c + "c"], s[c + "s"] = _quantised(torch.empty(shape, device="cuda").normal_(generator=g), cache)
    s["out"] = torch.empty(T, hq, dim, dtype=dt, device="cuda")
    if case["op"] in ("append", "read"):
        s["k_back"], s["v_back"] = (torch.empty(T, hkv, dim, dtype=dt, device="cuda") for _ in range(2))
    if case["op"] == "append":
        # one projection makes q, k and v of a token side by side; trained norms' weights are near one
        s["qkv"] = normal(T, hq + 2 * hkv, dim, std=3.0, dtype=DTYPES[case["in"]])
        s["q"], s["k"], s["v"] = s["qkv"].split((hq, hkv, hkv), dim=1)
        s["wq"], s["wk"] = (1.0 + normal(dim, std=0.2, dtype=torch.float32) for _ in range(2))
        # an image's tokens share a time and have a row and a column of it
        at = torch.cat([torch.arange(b - a, b, device="cuda") for a, b in zip(lens, kv)])
        s["pos"] = (torch.stack([at // 3, at // 7 + 5, at % 61]) if case["axes"] == 3 else at[None]).to(torch.int32)
    else:
        s["q"] = normal(T, hq, dim, std=2.0)  # scores as peaked as normalised heads with trained weights have them
    if case["op"] == "shared":
        s["members"], s["starts"], s["prefix"] = members, _device_ints(starts), _device_ints(_ints(case["prefix"]))
    if own:
        m = _mixer()
        s["handle"] = m.Attention(hq, hkv, dim, page, dtype=dt, rotary=case["rot"], theta=1e7, sections=_sections(case),
                                  interleaved=case["axes"] == 3)
        s["batch"] = m.Batch(s["kv_len"], s["table"], None if case["op"] in ("decode", "shared") else s["cu"], max_len=max(kv))
        if cache != "16":
            s["cache8"] = m.Cache8(s["kc"], s["vc"], s["ks"], s["vs"])
        if case["op"] == "append":
            s["norms"] = m.Norms(s["wq"], s["wk"], EPS)
        if case["op"] == "shared":
            s["shared"] = m.Shared(s["starts"], s["prefix"], max_prefix=max(_ints(case["prefix"])))
    return s


# -- one pass ---------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s, torch.cuda.current_stream())
    return {"append": _append, "read": _read, "prompt": _attend, "decode": _attend, "shared": _shared}[op](s)


def _own(op, s, stream):
    h, b = s["handle"], s["batch"]
    if op == "append":
        if s["case"]["cache"] == "16":
            h.append(b, s["q"], s["k"], s["v"], s["kc"], s["vc"], s["out"], pos=s["pos"], norms=s["norms"], stream=stream)
            return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}
        h.append8(b, s["q"], s["k"], s["v"], s["cache8"], s["out"], pos=s["pos"], norms=s["norms"], stream=stream)
        h.read8(b, s["cache8"], s["k_back"], s["v_back"], stream=stream)
        return {"q": s["out"], "k": s["k_back"], "v": s["v_back"], "ks": s["ks"], "vs": s["vs"]}
    if op == "read":
        h.read8(b, s["cache8"], s["k_back"], s["v_back"], stream=stream)
        return {"k": s["k_back"], "v": s["v_back"]}
    if op == "prompt":
        h.prompt8(b, s["q"], s["cache8"], s["out"], stream=stream)
    elif op == "decode":
        h.decode8(b, s["q"], s["cache8"], s["out"], stream=stream)
    elif s["case"]["cache"] == "16":
        h.decode_shared(b, s["shared"], s["q"], s["kc"], s["vc"], s["out"], stream=stream)
    else:
        h.decode8_shared(b, s["shared"], s["q"], s["cache8"], s["out"], stream=stream)
    return {"out": s["out"]}


def _axes(case):
    """Axis of each rotated pair: axes take turns (time, height, width, time, ...) until height and width are used up."""
    pairs = case["rot"] // 2
    i = torch.arange(pairs, device="cuda")
    if case["axes"] == 1:
        return torch.zeros_like(i)
    _, h, w = _sections(case)
    return torch.where((i % 3 == 1) & (i < 3 * h), 1, torch.where((i % 3 == 2) & (i < 3 * w), 2, 0))


def _places(s):
    """Page and row in it of each of the call's tokens."""
    page, token = s["case"]["page"], torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(s["cu"], token, right=True, out_int32=True) - 1
    at = s["kv_len"][seq] - s["cu"][seq + 1] + token
    return s["table"][seq, at // page], at % page


def _append(s):
    case, dt = s["case"], s["out"].dtype
    rot = case["rot"]
    inv = torch.pow(torch.tensor(1e7, dtype=torch.float64, device="cuda"),
                    -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = s["pos"].double()[_axes(case)].T * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], dim=-1)

    s["out"].copy_(turn(s["q"], s["wq"]))
    k, v = turn(s["k"], s["wk"]), s["v"].float()
    p, r = _places(s)
    if case["cache"] == "16":
        s["kc"][p, :, r], s["vc"][p, :, r] = k.to(dt), v.to(dt)
        return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}
    for x, c, scale in ((k, "kc", "ks"), (v, "vc", "vs")):
        codes, s[scale][p, :, r] = _quantised(x, case["cache"])
        s[c].view(torch.int8)[p, :, r] = codes.view(torch.int8)
    return {"q": s["out"], **_read(s), "ks": s["ks"], "vs": s["vs"]}


def _values(s, c, p, r):
    """What the codes of rows r of pages p stand for, in 32 bits."""
    return s[c + "c"].view(torch.int8)[p, :, r].view(CODES[s["case"]["cache"]]).float() * s[c + "s"][p, :, r][..., None]


def _read(s):
    p, r = _places(s)
    s["k_back"].copy_(_values(s, "k", p, r))
    s["v_back"].copy_(_values(s, "v", p, r))
    return {"k": s["k_back"], "v": s["v_back"]}


def _pages(s, c, table):
    """[n, hkv, positions, dim] of the pages in table [n, pages], in 32 bits."""
    case, t = s["case"], table.long()
    if case["cache"] == "16":
        x = s[c + "c"][t].float()
    else:
        x = s[c + "c"].view(torch.int8)[t].view(CODES[case["cache"]]).float() * s[c + "s"][t][..., None]
    return x.transpose(1, 2).reshape(t.shape[0], case["hkv"], -1, case["dim"])


def _attend(s):
    case = s["case"]
    hq, hkv, dim = (case[x] for x in ("hq", "hkv", "dim"))
    n, most_q, most_kv = len(s["lens"]), max(s["lens"]), max(s["kv"])
    # sequences padded to the longest: queries [n, hkv, group * most_q, dim], keys and values [n, hkv, most_kv, dim]
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    j = torch.arange(most_q, device="cuda")
    there = j < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(there, cu[:-1, None] + j, 0)
    q = s["q"][rows].float().reshape(n, most_q, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)
    scores = q @ _pages(s, "k", s["table"])[:, :, :most_kv].transpose(2, 3) * dim ** -0.5
    place = (kv_len - (cu[1:] - cu[:-1]))[:, None] + j  # of each query in its sequence
    key = torch.arange(most_kv, device="cuda")
    seen = (key <= place[..., None]) & there[..., None]
    scores = scores.view(n, hkv, hq // hkv, most_q, most_kv).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _pages(s, "v", s["table"])[:, :, :most_kv].masked_fill((key >= kv_len[:, None])[:, None, :, None], 0.0)
    o = (p.view(n, hkv, -1, most_kv) @ v).view(n, hkv, hq // hkv, most_q, dim) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, most_q, hq, dim)[there])
    return {"out": s["out"]}


def _shared(s):
    case = s["case"]
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    n, G, most, most_p = len(s["lens"]), len(s["members"]), max(s["members"]), max(_ints(case["prefix"]))
    group = hq // hkv
    q = s["q"].float().view(n, hkv, group, dim)
    # the beginnings: all of a group's queries over its keys, groups padded to the largest
    starts, prefix = s["starts"].long(), s["prefix"].long()
    j = torch.arange(most, device="cuda")
    there = j < (starts[1:] - starts[:-1])[:, None]
    rows = torch.where(there, starts[:-1, None] + j, 0)
    key = torch.arange(most_p, device="cuda")
    table = s["table"][starts[:-1], : -(-most_p // page)]
    kp, vp = _pages(s, "k", table)[:, :, :most_p], _pages(s, "v", table)[:, :, :most_p]
    behind = (key >= prefix[:, None])[:, None, :, None]
    a = (q[rows].transpose(1, 2).reshape(G, hkv, most * group, dim) @ kp.transpose(2, 3)) * dim ** -0.5
    a = a.masked_fill_(behind.transpose(2, 3), -math.inf)
    # each sequence's own positions, from its first own page on
    of = torch.searchsorted(starts, torch.arange(n, device="cuda"), right=True) - 1
    skip = prefix[of] // page
    most_own = max(x - p // page * page for x, p in zip(s["kv"], _lengths(case)[1]))
    cols = skip[:, None] + torch.arange(-(-most_own // page), device="cuda")
    mine = s["table"].gather(1, cols.clamp(max=s["table"].shape[1] - 1))
    at = skip[:, None] * page + torch.arange(mine.shape[1] * page, device="cuda")
    no = ((at < prefix[of][:, None]) | (at >= s["kv_len"].long()[:, None]))[:, None, :, None]
    b = (q @ _pages(s, "k", mine).transpose(2, 3) * dim ** -0.5).masked_fill_(no.transpose(2, 3), -math.inf)
    # one softmax over both
    a = a.view(G, hkv, most, group, most_p).transpose(1, 2)
    top = torch.maximum(a[there].amax(-1), b.amax(-1))[..., None]
    wide = torch.zeros(G, most, hkv, group, 1, device="cuda")
    wide[there] = top
    a, b = (a - wide).exp_(), (b - top).exp_()
    total = a[there].sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    o = a.transpose(1, 2).reshape(G, hkv, most * group, most_p) @ vp.masked_fill(behind, 0.0)
    o = o.view(G, hkv, most, group, dim).transpose(1, 2)[there] + b @ _pages(s, "v", mine).masked_fill_(no, 0.0)
    s["out"].copy_((o / total).view(n, hq, dim))
    return {"out": s["out"]}


# -- what a pass cannot do without -------------------------------------------------
def work(case):
    lens = _ints(case["lens"])
    n, T = len(lens), sum(lens)
    hq, hkv, dim, cache = case["hq"], case["hkv"], case["dim"], case["cache"]
    entry = 2 * hkv * (2 * dim if cache == "16" else dim + 4)  # a position's keys and values
    if case["op"] == "append":
        size = 4 if case["in"] == "f32" else 2
        back = 0 if cache == "16" else 2 * hkv * dim * 2
        return {"bytes": T * ((hq + 2 * hkv) * dim * size + hq * dim * 2 + entry + back + case["axes"] * 4),
                "flops": T * (hq + hkv) * (4 * dim + 3 * case["rot"])}
    if case["op"] == "read":
        return {"bytes": T * (entry + 2 * hkv * dim * 2), "flops": 2 * T * hkv * dim}
    kv, of_group = _lengths(case)
    ctx = [a - b for a, b in zip(kv, lens)]
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(lens, ctx))
    positions = sum(kv) - sum(of_group) + (sum(_ints(case["prefix"])) if case["op"] == "shared" else 0)
    return {"bytes": 2 * T * hq * dim * 2 + positions * entry, "flops": 4 * pairs * hq * dim}


# -- the definitions, in 64 bits ------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    page, group, dim = case["page"], case["hq"] // case["hkv"], case["dim"]
    table, cache = s["table"].cpu(), case["cache"]

    def cached(c, pages, h, count):
        x = s[c + "c"].view(torch.int8)[pages, h].view(CODES[cache]) if cache != "16" else s[c + "c"][pages, h]
        x = x.double()
        if cache != "16":
            x = x * s[c + "s"][pages, h].double()[..., None]
        return x.reshape(-1, dim)[:count]

    if case["op"] == "append":
        return _exact_append(case, s, table)
    if case["op"] == "read":
        out = {c: torch.empty(s["T"], case["hkv"], dim, dtype=torch.float64, device="cuda") for c in ("k", "v")}
        t = 0
        for i, (new, kv) in enumerate(zip(s["lens"], s["kv"])):
            pages = table[i, : -(-kv // page)].long().cuda()
            for c in out:
                for h in range(case["hkv"]):
                    out[c][t: t + new, h] = cached(c, pages, h, kv)[kv - new:]
            t += new
        return out
    if case["hq"] * sum(s["kv"]) * max(s["lens"]) > 4e9:
        return None
    out, t = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda"), 0
    first = [sum(s["members"][:g]) for g, m in enumerate(s["members"]) for _ in range(m)] if case["op"] == "shared" else None
    of_group = _lengths(case)[1]
    for i, (new, kv) in enumerate(zip(s["lens"], s["kv"])):
        pages = table[i, : -(-kv // page)].long().cuda()
        later = torch.arange(kv, device="cuda") > torch.arange(kv - new, kv, device="cuda")[:, None]
        for h in range(case["hkv"]):
            k, v = (cached(c, pages, h, kv) for c in ("k", "v"))
            if first:  # the shared positions are the first sequence's
                p = of_group[i]
                theirs = table[first[i], : -(-p // page)].long().cuda()
                k, v = (torch.cat([cached(c, theirs, h, p), x[p:]]) for c, x in (("k", k), ("v", v)))
            for j in range(h * group, (h + 1) * group):
                x = s["q"][t: t + new, j].double() @ k.T / math.sqrt(dim)
                out[t: t + new, j] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v
        t += new
    return {"out": out}


def _exact_append(case, s, table):
    page, half = case["page"], case["rot"] // 2
    turns = _sections(case)[1:] if case["axes"] == 3 else (0, 0)
    out = []
    for x, w in ((s["q"].double(), s["wq"]), (s["k"].double(), s["wk"])):
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        for i in range(half):
            axis = 1 if i % 3 == 1 and i // 3 < turns[0] else 2 if i % 3 == 2 and i // 3 < turns[1] else 0
            z = torch.polar(torch.ones_like(s["pos"][0], dtype=torch.float64), s["pos"][axis].double() * 1e7 ** (-2 * i / case["rot"]))
            r = torch.complex(x[:, :, i], x[:, :, i + half]) * z[:, None]
            x[:, :, i], x[:, :, i + half] = r.real, r.imag
        out.append(x)
    new = {"k": out[1], "v": s["v"].double()}
    back = {}
    for c in ("k", "v"):
        if case["cache"] == "16":
            back[c + "c"], values = s[c + "c"].double(), new[c]
        else:
            back[c + "s"], scale = s[c + "s"].double(), new[c].abs().amax(-1) / MOST[case["cache"]]
            y = new[c] / scale[..., None]
            if case["cache"] == "i8":
                y = torch.round(y)
            else:  # three bits behind the leading one, steps of 2^-9 at least
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                y = torch.round(y / step) * step
            back[c] = y * scale[..., None]
        t = 0
        for i, (n, kv) in enumerate(zip(s["lens"], s["kv"])):
            at = torch.arange(kv - n, kv)
            p = table[i, at // page].long().cuda()
            if case["cache"] == "16":
                back[c + "c"][p, :, (at % page).cuda()] = values[t: t + n]
            else:
                back[c + "s"][p, :, (at % page).cuda()] = scale[t: t + n]
            t += n
    return {"q": out[0], **back}
