"""What is measured: rotary positions for long contexts, and a cache of 4-bit keys and values.

The operators, in the order in which a step calls them: tables of cosines and
sines for positions that may lie past the length that a model was trained on, the
rotation of queries and keys by them (in training with its gradient), the
4-bit cache that the new keys and values are quantised into and can be read
back from, and attention over it. Each case is one call of one of them. The
fields of a case (each kind uses some):

  op      "angles", "rotate", "store", "read" or "attend"
  B       sequences; lo, hi and nlo, nhi: tokens of each that the cache holds
          before the step, and new ones, drawn from [lo, hi] and [nlo, nhi] over
          their logarithm by `lens`, a seed of its own, so that the work of a case
          does not depend on the seed of its values
  page    tokens of a page (0: contiguous caches)
  cache   "fp4"; for "read" "int8" or "e4m3" too, a scale for `block` tokens
  dtype   what the model computes in, table: what cosines and sines are held in
  H, Hk, D  query heads, key / value heads, head dimension; rd: rotated part of it
  layout  rotate: "dense" (batch, rows), "ragged" (sequences one behind the other)
          or "step" (tokens of many requests, each at a position of its own)
  inter   pairs are neighbours (else: the halves of the rotated part)
  grad    with the backward pass
  scaling, factor, base, length, att: how positions are scaled, and the tables
  causal, left (left window, -1: none), softcap (0: none)

The 4-bit cache: 32 channels of a token and head share a scale 2^e (held as e +
127), the smallest with max |x| <= 6 * 2^e and e >= -100, and x / 2^e is held as the
nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign, ties to the even code. Two
codes are a byte, the lower half first. Codes are returned as their values: the
rows that were stored are read back.
"""
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
GROUP = 32  # channels of a scale
DEFAULTS = dict(op="attend", B=1, lo=1, hi=1, lens=0, nlo=1, nhi=1, page=64, block=16, cache="fp4", dtype="bf16",
                table="fp32", H=32, Hk=8, D=128, rd=128, layout="dense", inter=False, grad=False, scaling="none",
                factor=1.0, base=10000.0, length=8192, att=1.0, causal=True, left=-1, softcap=0.0)
# no drawn case costs more than the largest listed ones (attend_chunk, rotate_train)
MOST_FLOPS, MOST_BYTES = 7.5e11, 1.3e9
MOST_PADDED = 2.5e9  # scores, or key and value numbers, of the plain form's rectangles


def _case(**kw):
    return dict(DEFAULTS, **kw)


def listed():
    return [
        # the positions of one step of 64 users, a context four times the trained one
        _case(name="angles_step", op="angles", layout="step", B=64, lo=512, hi=131072, scaling="by_parts", factor=4.0,
              att=1.1386),
        # the table of one rank's share of a context split over several, 131072 positions from wherever its share begins
        _case(name="angles_context", op="angles", B=131072, hi=917504, layout="dense", scaling="ntk", factor=16.0),
        # q and k of one step of 64 users
        _case(name="rotate_step", op="rotate", layout="step", B=64, lo=512, hi=131072, lens=2),
        # a training step of sequences of 4096, forward and backward
        _case(name="rotate_train", op="rotate", B=4, nlo=4096, nhi=4096, grad=True),
        # packed documents of every length, neighbours paired, three quarters of an odd head, fp16, forward and backward
        _case(name="rotate_packed", op="rotate", layout="ragged", B=37, nlo=16, nhi=2048, lens=3, H=12, Hk=3, D=80, rd=64,
              inter=True, dtype="fp16", table="fp16", grad=True),
        # the next token of 64 users goes into the cache
        _case(name="store_step", op="store", B=64, lo=512, hi=32768, lens=4, page=16),
        # prompts of every length
        _case(name="store_prompts", op="store", B=16, lo=1, hi=64, lens=5, nlo=256, nhi=8192, page=256),
        # contexts read back, for a kernel that wants 16 bits or another server
        _case(name="read_context", op="read", B=13, lo=300, hi=16384, lens=6, page=48, Hk=5, D=96, dtype="fp16"),
        # one user's next token over a short context: nothing to fill the chip with
        _case(name="attend_one", B=1, lo=777, hi=777, page=16),
        # a serving step over a paged cache with lengths of every size
        _case(name="attend_paged", B=64, lo=512, hi=32768, lens=7, H=64, page=256),
        # verification of 4 speculated tokens, sliding window over long contexts, soft cap, fp16
        _case(name="attend_verify", B=8, lo=16384, hi=65536, lens=8, nlo=4, nhi=4, left=4096, softcap=50.0, dtype="fp16",
              page=16),
        # a prompt's next chunk over what the cache holds of it, the chunk itself appended
        _case(name="attend_chunk", B=4, lo=4096, hi=4096, nlo=2048, nhi=2048, page=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return a, b


def _draw(rng):
    op = rng.choice(["angles", "rotate", "rotate", "store", "read", "attend", "attend", "attend"])
    c = _case(op=op, lens=rng.randrange(1 << 20), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "angles":
        lo, hi = _range(rng, 1, 1 << 20)
        return dict(c, B=_log(rng, 1, 131072), lo=lo, hi=hi, layout=rng.choice(["dense", "step"]),
                    rd=16 * rng.randint(1, 16), scaling=rng.choice(["none", "linear", "ntk", "by_parts"]),
                    factor=round(rng.uniform(1.0, 32.0), 2), base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    length=_log(rng, 2048, 32768), att=round(rng.uniform(1.0, 1.4), 3),
                    table=rng.choice(["fp32", "bf16", "fp16"]))
    hk = rng.choice([1, 2, 4, 5, 8, 8, 16])
    c.update(Hk=hk, H=hk * rng.choice([1, 3, 4, 4, 8]))
    if op == "rotate":
        d = 8 * _log(rng, 4, 32)
        c.update(D=d, rd=rng.choice([d // 16 * 16, 16 * rng.randint(1, d // 16)]), inter=rng.random() < 0.5,
                 grad=rng.random() < 0.6, table=rng.choice(["fp32", c["dtype"]]), layout=rng.choice(["dense", "ragged", "step"]))
        lo, hi = _range(rng, 1, 8192)
        if c["layout"] == "dense":
            return dict(c, B=_log(rng, 1, 16), nlo=hi, nhi=hi, lo=0, hi=0)
        if c["layout"] == "step":
            return dict(c, B=_log(rng, 1, 512), lo=lo, hi=_log(rng, hi, 131072))
        return dict(c, B=_log(rng, 1, 64), nlo=lo, nhi=hi)
    c["D"] = rng.choice([32, 64, 96, 128, 128, 128, 160, 192, 256])
    c["page"] = rng.choice([0, 16, 16, 32, 48, 64, 80, 128, 256])
    lo, hi = _range(rng, 1, 32768)
    if op == "store":
        nlo, nhi = rng.choice([(1, 1), (2, 9), _range(rng, 1, 8192)])
        return dict(c, B=_log(rng, 1, 64), lo=min(lo, 4096), hi=min(hi, 4096), nlo=nlo, nhi=nhi)
    if op == "read":
        c["cache"] = rng.choice(["fp4", "fp4", "int8", "e4m3"])
        return dict(c, B=_log(rng, 1, 64), lo=lo, hi=hi, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    c.update(B=_log(rng, 1, 64), lo=lo, hi=hi)
    if kind == "verify":
        c.update(nlo=2, nhi=rng.choice([2, 4, 7]), left=rng.choice([-1, 1024, 4096]))
    if kind == "chunk":
        n = _log(rng, 64, 2048)
        c.update(B=_log(rng, 1, 8), lo=min(lo, 8192), hi=min(hi, 8192), nlo=n, nhi=n)
    if kind == "mixed":
        c.update(hi=min(hi, 8192), lo=min(lo, 8192), nlo=1, nhi=_log(rng, 2, 1024))
    if rng.random() < 0.2:
        c["softcap"] = rng.choice([15.0, 30.0, 50.0])
    if kind in ("verify", "chunk") and rng.random() < 0.2:
        c["causal"] = False
    return c


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
            continue
        if c["op"] in ("store", "read", "attend"):
            reqs = _lengths(c)
            wide, rows = max(L + n for L, n in reqs), max(n for _, n in reqs)
            if c["B"] * wide * max(2 * c["Hk"] * c["D"], c["H"] * rows if c["op"] == "attend" else 0) > MOST_PADDED:
                continue
        return c


def _lengths(c):
    """(tokens in the cache, new tokens) of each sequence."""
    r = random.Random(c["lens"])
    pick = lambda lo, hi: _log(r, lo, hi) if hi > lo else lo  # noqa: E731
    return [(pick(c["lo"], c["hi"]), pick(c["nlo"], c["nhi"])) for _ in range(c["B"])]


def _seen(c, sq, sk):
    """(pairs that the mask leaves, keys that some query sees)."""
    i = torch.arange(sq, dtype=torch.int64) + (sk - sq)
    hi = i if c["causal"] or c["left"] >= 0 else torch.full_like(i, sk - 1)
    lo = (i - c["left"]).clamp(min=0) if c["left"] >= 0 else torch.zeros_like(i)
    return int((hi - lo + 1).sum()), int(hi.max() - lo.min() + 1)


def _held(c):
    """Bytes of a key and a value row in the cache."""
    if c["cache"] == "fp4":
        return 2 * c["Hk"] * (c["D"] // 2 + c["D"] // GROUP)
    return 2 * c["Hk"] * (c["D"] + 4 / c["block"])


def work(c):
    if c["op"] == "angles":
        size = 4 if c["table"] == "fp32" else 2
        # positions in 32 bits; cosines and sines; an angle and its two functions
        return {"bytes": c["B"] * (4 + c["rd"] * size), "flops": 4 * c["B"] * c["rd"]}
    if c["op"] == "rotate":
        rows = sum(n for _, n in _lengths(c)) if c["layout"] != "step" else c["B"]
        heads, size = c["H"] + c["Hk"], 4 if c["table"] == "fp32" else 2
        places = max(n for _, n in _lengths(c)) if c["layout"] != "step" else c["B"]
        # rows in and out, gradients in and out; the tables' rows, each once a pass
        passes = 2 if c["grad"] else 1
        return {"bytes": passes * (4 * rows * heads * c["D"] + places * c["rd"] * size), "flops": passes * 3 * rows * heads * c["rd"]}
    reqs, row = _lengths(c), 2 * c["Hk"] * c["D"]
    if c["op"] == "store":
        new = sum(n for _, n in reqs)
        # rows in and their values out in 16 bits, slots; codes and scales written and read
        return {"bytes": new * (4 * row + 8 + 2 * _held(c)), "flops": 5 * new * row}
    if c["op"] == "read":
        keys = sum(L for L, _ in reqs)
        pages = sum(-(-L // c["page"]) for L, _ in reqs) if c["page"] else 0
        return {"bytes": keys * (_held(c) + row * (4 if c["dtype"] == "fp32" else 2)) + 4 * pages, "flops": keys * row}
    pairs = rows = keys = 0
    known = {}
    for L, n in reqs:
        p, k = known.setdefault((L, n), _seen(c, n, L + n))
        pairs, rows, keys = pairs + p, rows + n, keys + k
    # q and out, lse; codes and scales, lengths, pages
    moved = rows * c["H"] * (c["D"] * 4 + 4) + keys * _held(c) + 4 * c["B"]
    moved += 4 * sum(-(-(L + n) // c["page"]) for L, n in reqs) if c["page"] else 0
    return {"bytes": moved, "flops": pairs * c["H"] * c["D"] * 4}


# ---- what a program holds before the call ----------------------------------------------------


def _scatter_pages(need, g):
    """A page table whose rows hold `need` pages each, in any order."""
    ids = torch.randperm(sum(need) + 4, generator=g, device=DEVICE).to(torch.int32)
    col = torch.arange(max(need), device=DEVICE)[None]
    used = torch.tensor(need, device=DEVICE)[:, None]
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEVICE)
    table[col < used] = ids[:sum(need)]
    return table


def _like_keys(g, dt, *shape):
    """Rows as a model makes them: normal, some channels of a head larger than others."""
    x = torch.empty(shape, dtype=dt, device=DEVICE).normal_(generator=g)
    return x.mul_(torch.empty(shape[-2:], device=DEVICE).normal_(0.0, 0.5, generator=g).exp().to(dt))


def _cache(c, g, pages, size):
    """Codes and scales of a cache that earlier steps filled."""
    if c["cache"] != "fp4":
        x = torch.empty(pages, size, c["Hk"], c["D"], dtype=torch.bfloat16, device=DEVICE).normal_(generator=g)
        top = CODE_MAX[c["cache"]]
        x.mul_(top / 3.5).clamp_(-top, top)
        codes = x.round_().to(torch.int8) if c["cache"] == "int8" else x.to(CODES["e4m3"])
        s = torch.empty(pages, size // c["block"], c["Hk"], device=DEVICE).normal_(0.0, 0.3, generator=g).exp_()
        return codes, s * (3.5 / top)
    x = _like_keys(g, torch.bfloat16, pages, size, c["Hk"], c["D"])
    parts = [_quantise(p) for p in x.split(max(1, (1 << 26) // x[0].numel()))]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=DEVICE)
    s = {"case": c}
    if c["op"] == "angles":
        # each position for itself, or a run of them
        one = c["layout"] == "dense"
        s["pos"] = torch.randint(c["lo"], c["hi"] + 1, (1 if one else c["B"],), generator=g, **i32)
        if one:
            s["pos"] = s["pos"] + torch.arange(c["B"], **i32)
        return s
    dt = TYPES[c["dtype"]]
    reqs = _lengths(c)
    random.Random(seed).shuffle(reqs)
    if c["op"] == "rotate":
        rows = [n for _, n in reqs]
        most = max(rows)
        if c["layout"] == "dense":
            shape = (c["B"], rows[0])
        elif c["layout"] == "step":
            shape, most = (c["B"],), c["hi"] + 1
            s["pos"] = torch.tensor([L for L, _ in reqs], **i32)
        else:
            shape = (sum(rows),)
            s["cu"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **i32)
        f = 10000.0 ** (-torch.arange(0, c["rd"], 2, dtype=torch.float64, device=DEVICE) / c["rd"])
        angle = torch.arange(most, dtype=torch.float64, device=DEVICE)[:, None] * f
        s["cos"], s["sin"] = angle.cos().to(TYPES[c["table"]]), angle.sin().to(TYPES[c["table"]])
        for name, heads in (("q", c["H"]), ("k", c["Hk"])):
            s[name] = _like_keys(g, dt, *shape, heads, c["D"])
            if c["grad"]:
                s[name].requires_grad_()
                s["d" + name] = _like_keys(g, dt, *shape, heads, c["D"])
        return s
    P, Hk, D = c["page"], c["Hk"], c["D"]
    s["reqs"] = reqs = [(L, 0) for L, _ in reqs] if c["op"] == "read" else reqs
    after = [L + n for L, n in reqs]
    s["after"] = torch.tensor(after, **i32)
    if P:
        need = [-(-t // P) for t in after]
        s["table"], pages, size = _scatter_pages(need, g), sum(need) + 4, P
    else:
        pages, size = c["B"], -(-max(after) // 16) * 16
    if c["op"] == "store":
        s["kc"], s["vc"] = (torch.zeros(pages, size, Hk, D // 2, dtype=torch.uint8, device=DEVICE) for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros(pages, size, Hk, D // GROUP, dtype=torch.uint8, device=DEVICE) for _ in range(2))
        total = sum(n for _, n in reqs)
        s["k"], s["v"] = _like_keys(g, dt, total, Hk, D), _like_keys(g, dt, total, Hk, D)
        at = torch.cat([torch.arange(L, L + n) for L, n in reqs]).to(DEVICE)
        req = torch.repeat_interleave(torch.arange(c["B"]), torch.tensor([n for _, n in reqs])).to(DEVICE)
        s["slots"] = s["table"][req, at // P].long() * P + at % P if P else req * size + at
        return s
    s["kc"], s["ks"] = _cache(c, g, pages, size)
    s["vc"], s["vs"] = _cache(c, g, pages, size)
    if c["op"] == "read":
        s["cu"] = torch.tensor([sum(after[:i]) for i in range(len(after) + 1)], **i32)
        s["total"] = sum(after)
        return s
    rows = [n for _, n in reqs]
    s["ragged"] = c["nhi"] > c["nlo"]
    shape = (sum(rows), c["H"], D) if s["ragged"] else (c["B"], rows[0], c["H"], D)
    s["q"] = torch.empty(shape, device=DEVICE).normal_(generator=g).to(dt)
    s["rows"] = max(rows)
    if s["ragged"]:
        s["cu"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **i32)
    return s


# ---- one pass ----------------------------------------------------------------------------------


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-npu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import flash_attn_npu_v3 as fa

    c = s["case"]
    if c["op"] == "angles":
        cos, sin = fa.rotary_cos_sin(s["pos"], c["rd"], base=c["base"], scaling=None if c["scaling"] == "none" else c["scaling"],
                                     factor=c["factor"], original_length=c["length"], attention_factor=c["att"],
                                     dtype=TYPES[c["table"]])
        return {"cos": cos, "sin": sin}
    if c["op"] == "rotate":
        q, k = fa.apply_rotary_emb(s["q"], s["k"], s["cos"], s["sin"], positions=s.get("pos"), cu_seqlens=s.get("cu"),
                                   rotary_interleaved=c["inter"])
        if not c["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if c["op"] == "store":
        fa.append_quantized_kvcache(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        k, v = fa.read_quantized_kvcache(s["kc"], s["vc"], s["ks"], s["vs"], slot_mapping=s["slots"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    if c["op"] == "read":
        k, v = fa.read_quantized_kvcache(s["kc"], s["vc"], s["ks"], s["vs"], cu_seqlens_k=s["cu"], total_k=s["total"],
                                         page_table=s.get("table"), dtype=TYPES[c["dtype"]])
        return {"k": k, "v": v}
    more = dict(cu_seqlens_q=s["cu"], max_seqlen_q=s["rows"]) if s["ragged"] else {}
    window = (c["left"], 0 if c["causal"] or c["left"] >= 0 else -1)
    out, lse = fa.flash_attn_with_quantized_kvcache(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["after"],
                                                    page_table=s.get("table"), causal=c["causal"], window_size=window,
                                                    softcap=c["softcap"], return_softmax_lse=True, **more)
    return {"out": out, "lse": lse}


def _run_plain(s):
    return {"angles": _plain_angles, "rotate": _plain_rotate, "store": _plain_store, "read": _plain_read,
            "attend": _plain_attend}[s["case"]["op"]](s)


def _plain_angles(s):
    # in 64 bits: an angle of a far position leaves 32 no bits behind the point
    c, dt = s["case"], TYPES[s["case"]["table"]]
    rd, base = c["rd"], c["base"]
    if c["scaling"] == "ntk":
        base = base * c["factor"] ** (rd / (rd - 2))
    f = base ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=DEVICE) / rd)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "by_parts":
        turns = c["length"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / c["factor"])
    angle = s["pos"].double()[:, None] * f
    return {"cos": (angle.cos() * c["att"]).to(dt), "sin": (angle.sin() * c["att"]).to(dt)}


def _plain_rotate(s):
    c = s["case"]
    if c["layout"] == "dense":
        at = torch.arange(s["q"].shape[1], device=DEVICE)
    elif c["layout"] == "step":
        at = s["pos"].long()
    else:
        t = torch.arange(s["q"].shape[0], device=DEVICE, dtype=torch.int32)
        at = (t - s["cu"][torch.searchsorted(s["cu"][1:], t, right=True)]).long()
    cos, sin = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]
    half = c["rd"] // 2

    def turn(x, sin):
        y = x.detach().float()
        if c["inter"]:
            a, b = y[..., 0:c["rd"]:2], y[..., 1:c["rd"]:2]
            z = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:c["rd"]]
            z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((z, y[..., c["rd"]:]), -1).to(x.dtype)

    out = {"q": turn(s["q"], sin), "k": turn(s["k"], sin)}
    if c["grad"]:
        out.update(dq=turn(s["dq"], -sin), dk=turn(s["dk"], -sin))
    return out


def _two_to(e):
    """2 ** e of whole numbers from -126 to 127, by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """Codes (two to a byte) and scales of rows."""
    y = x.float().unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(y.abs().amax(-1))
    e = (e - 3 + (m > 0.75).int()).clamp(min=-100)  # the smallest with most <= 6 * 2 ** e
    e = torch.where(m > 0, e, -100)
    a = y.abs() * _two_to(-e)[..., None]
    # the border between two neighbours goes to the even code
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + torch.signbit(y).to(torch.uint8) * 8).flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, (e + 127).to(torch.uint8)


def _values(c, codes, scale):
    """Values in 32 bits of rows of codes (..., Hk, D) and their scales (of fp4: of each row)."""
    if c["cache"] != "fp4":
        return codes.float() * scale[..., None]
    known = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEVICE)
    known = torch.cat((known, -known))
    x = known[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    return (x.unflatten(-1, (-1, GROUP)) * _two_to(scale.int() - 127)[..., None]).flatten(-2)


def _plain_store(s):
    c, out = s["case"], {}
    for name, cache, scale in (("k", s["kc"], s["ks"]), ("v", s["vc"], s["vs"])):
        codes, e = _quantise(s[name])
        cache.view(-1, *cache.shape[2:])[s["slots"]] = codes
        scale.view(-1, *scale.shape[2:])[s["slots"]] = e
        out[name] = _values(c, codes, e).to(s[name].dtype)
    return out


def _at(s, req, j):
    """Rows of the caches, and of the scales, of keys j of sequences req."""
    c, size = s["case"], s["kc"].shape[1]
    page = s["table"][req, j // size].long() if c["page"] else req
    row = page * size + j % size
    return row, row if c["cache"] == "fp4" else row // c["block"]


def _take(s, row, part):
    """Values of keys and of values at those rows."""
    c = s["case"]
    got = []
    for cache, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        raw = cache.view(torch.uint8).view(-1, *cache.shape[2:])[row]
        got.append(_values(c, raw.view(cache.dtype), scale.view(-1, *scale.shape[2:])[part]))
    return got


def _plain_read(s):
    t = torch.arange(s["total"], device=DEVICE, dtype=torch.int32)
    req = torch.searchsorted(s["cu"][1:], t, right=True)
    k, v = _take(s, *_at(s, req, (t - s["cu"][req]).long()))
    dt = TYPES[s["case"]["dtype"]]
    return {"k": k.to(dt), "v": v.to(dt)}


def _plain_attend(s):
    c = s["case"]
    H, Hk, D, B, n = c["H"], c["Hk"], c["D"], c["B"], s["rows"]
    g = H // Hk
    sk = s["after"].long()
    wide = max(L + m for L, m in s["reqs"])
    j = torch.arange(wide, device=DEVICE)[None]
    req = torch.arange(B, device=DEVICE)[:, None]
    k, v = _take(s, *_at(s, req, torch.minimum(j, sk[:, None] - 1)))
    q = s["q"].float()
    if s["ragged"]:  # rows of every sequence side by side, the last ones of the longest
        cu = s["cu"].long()
        i = torch.arange(n, device=DEVICE)[None]
        own_row = cu[:-1, None] + i
        there = own_row < cu[1:, None]
        first = (cu[1:] - cu[:-1])[:, None]
        q = q[own_row.clamp(max=q.shape[0] - 1)]
        place = sk[:, None] - first + i
    else:
        place = sk[:, None] - n + torch.arange(n, device=DEVICE)[None]
    x = q.view(B, n, Hk, g, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, n * g, D)
    x = torch.matmul(x, k.permute(0, 2, 3, 1).contiguous()).mul_(D ** -0.5)
    if c["softcap"]:
        x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    hidden = (j >= sk[:, None])[:, None]
    if c["causal"] or c["left"] >= 0:
        hidden = hidden | (j[:, None] > place[:, :, None])
    if c["left"] >= 0:
        hidden = hidden | (j[:, None] < place[:, :, None] - c["left"])
    x.view(B, Hk, n, g, wide).masked_fill_(hidden[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()) / z
    out = o.view(B, Hk, n, g, D).permute(0, 2, 1, 3, 4).reshape(B, n, H, D).to(s["q"].dtype)
    lse = (m + z.log()).view(B, Hk, n, g).permute(0, 1, 3, 2).reshape(B, H, n)
    if s["ragged"]:
        return {"out": out[there], "lse": lse.permute(0, 2, 1)[there].t().contiguous()}
    return {"out": out, "lse": lse}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(c, seed):
    return {"angles": _exact_angles, "rotate": _exact_rotate, "store": _exact_store, "read": _exact_read,
            "attend": _exact_attend}[c["op"]](prepare(c, seed))


def _exact_angles(s):
    c = s["case"]
    pos, rd = s["pos"].double(), c["rd"]
    cos = torch.empty(pos.numel(), rd // 2, dtype=torch.float64, device=DEVICE)
    sin = torch.empty_like(cos)
    for i in range(rd // 2):
        f = math.exp(-2.0 * i / rd * math.log(c["base"]))
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "ntk":
            f /= c["factor"] ** (2.0 * i / (rd - 2))
        elif c["scaling"] == "by_parts":
            share = min(max((c["length"] / (2 * math.pi / f) - 1.0) / (32.0 - 1.0), 0.0), 1.0)
            f = (1.0 - share) * f / c["factor"] + share * f
        cos[:, i] = torch.cos(pos * f) * c["att"]
        sin[:, i] = torch.sin(pos * f) * c["att"]
    return {"cos": cos, "sin": sin}


def _exact_rotate(s):
    # as products with complex numbers
    c = s["case"]
    if "cu" in s:
        at = torch.cat([torch.arange(b - a, device=DEVICE) for a, b in zip(s["cu"].tolist(), s["cu"].tolist()[1:])])
    else:
        at = s["pos"].long() if "pos" in s else torch.arange(s["q"].shape[1], device=DEVICE)
    unit = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    rd = c["rd"]

    def turn(x, unit):
        y = x.detach().double().clone()
        pairs = y[..., :rd].unflatten(-1, (rd // 2, 2) if c["inter"] else (2, rd // 2))
        pairs = pairs if c["inter"] else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
        y[..., :rd] = (z if c["inter"] else z.transpose(-1, -2)).flatten(-2)
        return y

    out = {"q": turn(s["q"], unit), "k": turn(s["k"], unit)}
    if c["grad"]:
        out.update(dq=turn(s["dq"], unit.conj()), dk=turn(s["dk"], unit.conj()))
    return out


def _exact_store(s):
    # the nearest of the 15 values, the even code of two that are equally near
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=DEVICE)
    out = {}
    for name in ("k", "v"):
        parts = []
        for x in s[name].split(2048):
            y = x.double().unflatten(-1, (-1, GROUP))
            most = y.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -120) / 6.0))
            e = torch.where(most > 6.0 * 2.0 ** e, e + 1, torch.where(most <= 6.0 * 2.0 ** (e - 1), e - 1, e)).clamp(min=-100.0)
            off = (y.abs()[..., None] / 2.0 ** e[..., None] - grid).abs()
            off = off + torch.where(torch.arange(8, device=DEVICE) % 2 == 1, 1e-9, 0.0)
            parts.append((grid[off.argmin(-1)] * torch.sign(y) * 2.0 ** e).flatten(-2))
        out[name] = torch.cat(parts)
    return out


def _exact_rows(s, b, cache, scale):
    """Values 0 .. L - 1 of sequence b in 64 bits."""
    c, L, size = s["case"], s["after"].tolist()[b], cache.shape[1]
    j = torch.arange(L, device=DEVICE)
    page = s["table"][b].long()[j // size] if c["page"] else torch.full_like(j, b)
    if c["cache"] != "fp4":
        raw = cache.view(torch.uint8)[page, j % size].view(cache.dtype).double()
        return raw * scale[page, j % size // c["block"]].double()[..., None]
    byte = cache[page, j % size].long()
    code = torch.empty(*byte.shape[:-1], 2 * byte.shape[-1], dtype=torch.int64, device=DEVICE)
    code[..., 0::2], code[..., 1::2] = byte % 16, byte // 16
    low, high = code % 2, code % 8 // 2  # a bit behind the point and the exponent
    size = torch.where(high > 0, (1.0 + 0.5 * low) * 2.0 ** (high - 1.0), 0.5 * low)
    e = scale[page, j % cache.shape[1]].double().repeat_interleave(GROUP, -1) - 127.0
    return torch.where(code >= 8, -size, size) * 2.0 ** e


def _exact_read(s):
    return {name: torch.cat([_exact_rows(s, b, s[name + "c"], s[name + "s"]) for b in range(s["case"]["B"])])
            for name in ("k", "v")}


def _exact_attend(s):
    c = s["case"]
    g = c["H"] // c["Hk"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.zeros((c["H"], q.shape[0]) if s["ragged"] else (c["B"], c["H"], q.shape[1]), dtype=torch.float64,
                      device=DEVICE)
    start = 0
    for b, (L, n) in enumerate(s["reqs"]):
        rows = slice(start, start + n) if s["ragged"] else b
        start += n
        ks, vs = _exact_rows(s, b, s["kc"], s["ks"]), _exact_rows(s, b, s["vc"], s["vs"])
        i, j = torch.arange(L, L + n, device=DEVICE), torch.arange(L + n, device=DEVICE)
        seen = torch.ones(n, L + n, dtype=torch.bool, device=DEVICE)
        if c["causal"] or c["left"] >= 0:
            seen &= j[None] <= i[:, None]
        if c["left"] >= 0:
            seen &= j[None] >= i[:, None] - c["left"]
        for h in range(c["H"]):
            x = (q[rows][:, h] @ ks[:, h // g].t()) / math.sqrt(c["D"])
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            x = torch.where(seen, x, -math.inf)
            z = torch.logsumexp(x, -1)
            out[rows][:, h] = torch.exp(x - z[:, None]) @ vs[:, h // g]
            (lse[:, rows] if s["ragged"] else lse[b])[h] = z
    return {"out": out, "lse": lse}
