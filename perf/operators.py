"""What is measured: serving over a paged cache of 8-bit keys and values.

Three operators, in the order in which a serving step calls them: the page
table grows and shrinks with the requests and gives every new token its slot,
the new tokens are quantised into their slots, and attention reads the cache.
Each case is one call of one of them. The fields of a case:

  op      "table", "append" or "attend"
  B       requests of the step
  lo, hi  tokens that the cache holds of a request before the step, drawn from
          [lo, hi] over their logarithm by `lens`, a seed of its own, so that
          the work of a case does not depend on the seed of its values
  nlo, nhi  new tokens of a request, drawn alike (the query rows for "attend")
  done    table: requests in 100 that end in this step and give their pages back
  page    tokens of a page (0: contiguous caches, attend only)
  block   tokens that share a scale
  cache   "int8" or "e4m3", what the cache holds
  dtype   "bf16" or "fp16", what the model computes in
  H, Hk, D  query heads, key / value heads, head dimension
  causal, left (left window, -1: none), softcap (0: none)

A scale holds for the rows of a block and one head: a stored code c stands for
c * scale. The append takes the smallest power of two that brings the block's
largest value into the codes' range, and a block that it continues keeps its
scale or moves to the larger one; its results are therefore the same numbers in
32 and 64 bits, codes and scales alike.
"""
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
FLOOR = -100  # exponent of the smallest scale
DEFAULTS = dict(op="attend", B=1, lo=1, hi=1, lens=0, nlo=1, nhi=1, done=0, page=64, block=64, cache="e4m3",
                dtype="bf16", H=32, Hk=8, D=128, causal=True, left=-1, softcap=0.0)
# no drawn case costs more than the largest listed ones (attend_paged, attend_chunk)
MOST_FLOPS, MOST_BYTES = 1.0e12, 1.4e9


def _case(**kw):
    return dict(DEFAULTS, **kw)


def listed():
    return [
        # the next token of 64 users: a few of them come to a new page
        _case(name="table_decode", op="table", B=64, lo=512, hi=32768, lens=1, page=16),
        # a full server: an eighth of 1024 requests end and give their pages back
        _case(name="table_busy", op="table", B=1024, lo=64, hi=16384, lens=2, nlo=1, nhi=8, done=12, page=64),
        # prompts come in together, every page of them is new
        _case(name="table_prompts", op="table", B=96, lo=1, hi=64, lens=3, nlo=512, nhi=8192, page=16),
        # the next token of 64 users goes into blocks that earlier ones began
        _case(name="append_decode", op="append", B=64, lo=512, hi=32768, lens=4, cache="int8"),
        # prompts of every length
        _case(name="append_prompts", op="append", B=16, lo=1, hi=64, lens=5, nlo=256, nhi=8192, page=256),
        # speculated tokens of a model with odd heads, short blocks, fp16
        _case(name="append_odd", op="append", B=25, lo=64, hi=4096, lens=6, nlo=2, nhi=9, page=48, block=16, Hk=5, D=80,
              dtype="fp16"),
        # one user's next token over a short context: nothing to fill the chip with
        _case(name="attend_one", B=1, lo=777, hi=777, page=256),
        # a serving step of 32 users with contiguous int8 caches
        _case(name="attend_batch", B=32, lo=1024, hi=8191, lens=7, page=0, block=128, cache="int8"),
        # a serving step over a paged cache with lengths of every size
        _case(name="attend_paged", B=64, lo=512, hi=32768, lens=3, H=64, page=256, block=64),
        # verification of 4 speculated tokens, sliding window over long contexts, soft cap, fp16
        _case(name="attend_verify", B=8, lo=16384, hi=65536, lens=5, nlo=4, nhi=4, left=4096, softcap=50.0, dtype="fp16",
              cache="int8", block=16),
        # a prompt's next chunk over what the cache holds of it, the chunk itself appended
        _case(name="attend_chunk", B=4, lo=4096, hi=4096, nlo=2048, nhi=2048, page=256, block=64),
        # a step that mixes users at their next token with users in their prompt, head dimension 64
        _case(name="attend_mixed", B=40, lo=64, hi=8192, lens=9, nlo=1, nhi=700, H=24, Hk=8, D=64, cache="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["table", "append", "attend", "attend", "attend"])
    c = _case(op=op, lens=rng.randrange(1 << 20), cache=rng.choice(["int8", "e4m3"]),
              dtype=rng.choice(["bf16", "bf16", "fp16"]), page=16 * _log(rng, 1, 16))
    c["block"] = rng.choice([b for b in range(16, c["page"] + 1, 16) if c["page"] % b == 0])
    lo, hi = sorted((_log(rng, 1, 32768), _log(rng, 1, 32768)))
    if op == "table":
        lo, hi = sorted((_log(rng, 1, 16384), _log(rng, 1, 16384)))
        nlo, nhi = sorted((_log(rng, 1, 4096), _log(rng, 1, 4096)))
        return dict(c, B=_log(rng, 1, 1024), lo=lo, hi=hi, nlo=nlo, nhi=nhi, done=rng.choice([0, 0, 10, 30]))
    hk = rng.choice([1, 2, 4, 5, 8, 8, 16])
    c.update(Hk=hk, H=hk * rng.choice([1, 3, 4, 4, 8]), D=rng.choice([64, 80, 96, 128, 128, 128, 192, 256]))
    if op == "append":
        nlo, nhi = rng.choice([(1, 1), (2, 9), tuple(sorted((_log(rng, 1, 8192), _log(rng, 1, 8192))))])
        return dict(c, B=_log(rng, 1, 64), lo=min(lo, 4096), hi=min(hi, 4096), nlo=nlo, nhi=nhi)
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    c.update(B=_log(rng, 1, 64), lo=lo, hi=hi)
    if kind == "decode" and rng.random() < 0.3:
        c["page"] = 0
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
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return c


def _lengths(c):
    """(tokens in the cache, new tokens, whether it ends) of each request."""
    r = random.Random(c["lens"])
    pick = lambda lo, hi: _log(r, lo, hi) if hi > lo else lo  # noqa: E731
    return [(pick(c["lo"], c["hi"]), pick(c["nlo"], c["nhi"]), r.randrange(100) < c["done"]) for _ in range(c["B"])]


def _seen(c, sq, sk):
    """(pairs that the mask leaves, keys that some query sees)."""
    i = torch.arange(sq, dtype=torch.int64) + (sk - sq)
    hi = i if c["causal"] or c["left"] >= 0 else torch.full_like(i, sk - 1)
    lo = (i - c["left"]).clamp(min=0) if c["left"] >= 0 else torch.zeros_like(i)
    return int((hi - lo + 1).sum()), int(hi.max() - lo.min() + 1)


def work(c):
    reqs, row = _lengths(c), c["Hk"] * c["D"]
    if c["op"] == "table":
        new = sum(n for _, n, end in reqs if not end)
        moved = sum(-(-L // c["page"]) if end else -(-(L + n) // c["page"]) - -(-L // c["page"]) for L, n, end in reqs)
        # lengths before and after; pages read and written; slots, starts, the free count
        return {"bytes": 8 * c["B"] + 8 * moved + 8 * new + 4 * (c["B"] + 1) + 8, "flops": c["B"] + new}
    if c["op"] == "append":
        new = sum(n for _, n, _ in reqs)
        blocks = sum(-(-(L + n) // c["block"]) - L // c["block"] for L, n, _ in reqs)
        # k and v read in 16 bits and written in 8, slots, scales read and written
        return {"bytes": 2 * new * row * 3 + 8 * new + 2 * 8 * blocks * c["Hk"], "flops": 4 * new * row}
    pairs = rows = keys = scales = 0
    known = {}
    for L, n, _ in reqs:
        p, k = known.setdefault((L, n), _seen(c, n, L + n))
        pairs, rows, keys, scales = pairs + p, rows + n, keys + k, scales + -(-k // c["block"])
    # q and out, lse; keys and values in 8 bits, their scales, lengths, pages
    moved = rows * c["H"] * (c["D"] * 4 + 4) + 2 * keys * row + 8 * scales * c["Hk"] + 4 * c["B"]
    moved += 4 * sum(-(-(L + n) // c["page"]) for L, n, _ in reqs) if c["page"] else 0
    return {"bytes": moved, "flops": pairs * c["H"] * c["D"] * 4}


# ---- what a program holds before the call ----------------------------------------------------


def _scatter_pages(c, g, need, spare):
    """A page table whose rows hold `need` pages each, in any order, and the pages that are left."""
    ids = torch.randperm(sum(need) + spare, generator=g, device=DEVICE).to(torch.int32)
    width = max(need)
    col = torch.arange(width, device=DEVICE)[None]
    used = torch.tensor(need, device=DEVICE)[:, None]
    table = torch.zeros(len(need), width, dtype=torch.int32, device=DEVICE)
    table[col < used] = ids[:sum(need)]
    return table, ids[sum(need):]


def _codes(c, g, *shape):
    """Codes as a cache holds them: roughly normal, the largest of a block near the end of the range."""
    x = torch.empty(shape, dtype=torch.bfloat16, device=DEVICE).normal_(generator=g)
    top = CODE_MAX[c["cache"]]
    x.mul_(top / 3.5).clamp_(-top, top)
    return x.round_().to(torch.int8) if c["cache"] == "int8" else x.to(torch.float8_e4m3fn)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=DEVICE)
    reqs = _lengths(c)
    random.Random(seed).shuffle(reqs)
    P, Hk, D = c["page"], c["Hk"], c["D"]
    s = {"case": c, "reqs": reqs, "lens": torch.tensor([L for L, _, _ in reqs], **i32)}
    after = [0 if c["op"] == "table" and end else L + n for L, n, end in reqs]
    s["after"] = torch.tensor(after, **i32)
    if c["op"] == "table":
        have, need = [-(-L // P) for L, _, _ in reqs], [-(-t // P) for t in after]
        s["table"], left = _scatter_pages(c, g, have, sum(max(b - a, 0) for a, b in zip(have, need)) + 64)
        wide = max(max(have), max(need)) + 8
        s["table"] = torch.nn.functional.pad(s["table"], (0, wide - s["table"].shape[1])).contiguous()
        # the stack has room for every page there is
        s["free"] = torch.zeros(sum(have) + left.numel(), **i32)
        s["free"][:left.numel()] = left
        s["num_free"] = torch.tensor([left.numel()], **i32)
        s["new"] = sum(n for _, n, end in reqs if not end)
        return s
    dt = TYPES[c["dtype"]]
    if P:
        s["table"], _ = _scatter_pages(c, g, [-(-t // P) for t in after], 4)
        pages, size = sum(-(-t // P) for t in after) + 4, P
    else:
        pages, size = c["B"], -(-max(after) // c["block"]) * c["block"]
    s["k"], s["v"] = _codes(c, g, pages, size, Hk, D), _codes(c, g, pages, size, Hk, D)
    shape = (pages, size // c["block"], Hk)
    if c["op"] == "append":
        # scales as earlier appends left them: powers of two
        for name in ("ks", "vs"):
            s[name] = _two_to(torch.randint(-7, -4, shape, generator=g, device=DEVICE) - (2 if c["cache"] == "e4m3" else 0))
        total = sum(n for _, n, _ in reqs)
        for name in ("k_new", "v_new"):
            x = torch.empty(total, Hk, D, device=DEVICE).normal_(generator=g)
            s[name] = (x * torch.empty(Hk, D, device=DEVICE).normal_(0.0, 0.5, generator=g).exp()).to(dt)
        at = torch.cat([torch.arange(L, L + n) for L, n, _ in reqs]).to(DEVICE)
        req = torch.repeat_interleave(torch.arange(c["B"]), torch.tensor([n for _, n, _ in reqs])).to(DEVICE)
        s["slots"] = s["table"][req, at // P].long() * P + at % P
        return s
    # scales of any value, calibrated ones among them
    for name in ("ks", "vs"):
        s[name] = torch.empty(shape, device=DEVICE).normal_(0.0, 0.3, generator=g).exp_() * (3.5 / CODE_MAX[c["cache"]])
    rows = [n for _, n, _ in reqs]
    s["ragged"] = c["nhi"] > c["nlo"]
    shape = (sum(rows), c["H"], D) if s["ragged"] else (c["B"], rows[0], c["H"], D)
    s["q"] = torch.empty(shape, device=DEVICE).normal_(generator=g).to(dt)
    if s["ragged"]:
        s["cu"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **i32)
        s["max"] = c["nhi"]
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
    if c["op"] == "table":
        slots, cu, left = fa.update_page_table(s["table"], s["lens"], s["after"], s["free"], s["num_free"], c["page"],
                                               s["new"])
        return {"table": s["table"], "free": s["free"], "slots": slots, "cu": cu, "num_free": left}
    if c["op"] == "append":
        fa.append_quantized_kvcache(s["k_new"], s["v_new"], s["k"], s["v"], s["ks"], s["vs"], s["slots"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
    more = dict(cu_seqlens_q=s["cu"], max_seqlen_q=s["max"]) if s["ragged"] else {}
    window = (c["left"], 0 if c["causal"] or c["left"] >= 0 else -1)
    out, lse = fa.flash_attn_with_quantized_kvcache(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["after"],
                                                    page_table=s.get("table"), causal=c["causal"], window_size=window,
                                                    softcap=c["softcap"], return_softmax_lse=True, **more)
    return {"out": out, "lse": lse}


def _run_plain(s):
    return {"table": _plain_table, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


def _plain_table(s):
    P, table, free = s["case"]["page"], s["table"], s["free"]
    width, room = table.shape[1], free.numel()
    before, after = s["lens"].long().clamp(min=0), s["after"].long().clamp(min=0)
    have, need = (((x.clamp(max=width * P) + P - 1) // P)[:, None] for x in (before, after))
    col = torch.arange(width, device=DEVICE)[None]
    start = s["num_free"].long().clamp(0, room)
    # pages of requests that shrink or end go onto the stack
    back = (col >= need) & (col < have) & (table >= 0)
    place = start + torch.cumsum(back.flatten(), 0) - 1
    place = torch.where(back.flatten() & (place < room), place, room)
    stack = torch.cat([free, free.new_zeros(1)])
    stack.scatter_(0, place, table.flatten())
    free.copy_(stack[:room])
    top = (start + back.sum()).clamp(max=room)
    # pages for requests that grow come off its top
    take = (col >= have) & (col < need)
    place = top - torch.cumsum(take.flatten(), 0).view_as(take)
    page = torch.where(place >= 0, free[place.clamp(min=0)], -1)
    table.copy_(torch.where(take, page, table))
    count = (after - before).clamp(min=0)
    cu = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)])
    i = torch.arange(s["new"], device=DEVICE)
    b = torch.searchsorted(cu[1:], i, right=True)
    inside = b < count.numel()
    b = b.clamp(max=count.numel() - 1)
    at = before[b] + i - cu[b]
    page = table[b, (at // P).clamp(max=width - 1)].long()
    slots = torch.where(inside & (at < width * P) & (page >= 0), page * P + at % P, -1)
    return {"table": table, "free": free, "slots": slots, "cu": cu.to(torch.int32),
            "num_free": (top - take.sum()).to(torch.int32)}


def _two_to(e):
    """2 ** e of whole numbers from -126 to 127, by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _store(c, x):
    return x.round().to(torch.int8) if c["cache"] == "int8" else x.to(torch.float8_e4m3fn)


def _plain_append(s):
    c, slots = s["case"], s["slots"]
    bl, top = c["block"], CODE_MAX[c["cache"]]
    block, place = slots // bl, slots % bl
    begins = torch.ones_like(block, dtype=torch.bool)
    begins[1:] = block[1:] != block[:-1]
    first = begins.nonzero()[:, 0]
    where, old_rows = block[first], place[first]
    part = (torch.cumsum(begins, 0) - 1)[:, None].expand(-1, c["Hk"])  # which of `first` a token belongs to
    for new, cache, scale in ((s["k_new"], s["k"], s["ks"]), (s["v_new"], s["v"], s["vs"])):
        x = new.float()
        most = torch.zeros(first.numel(), c["Hk"], device=DEVICE).scatter_reduce(0, part, x.abs().amax(-1), "amax")
        m, e = torch.frexp(most)
        e = e - math.frexp(top)[1] + (m > math.frexp(top)[0]).int()  # the smallest with most / 2 ** e <= top
        needed = _two_to(torch.where(most > 0, e, FLOOR).clamp(min=FLOOR))
        flat = scale.view(-1, c["Hk"])
        old = flat[where]
        now = torch.where(old_rows[:, None] > 0, torch.maximum(old, needed), needed)
        flat[where] = now
        rows = cache.view(torch.uint8).view(-1, bl, c["Hk"], c["D"])
        held = rows[where].view(cache.dtype)
        moved = _store(c, held.float() * (old / now)[:, None, :, None])
        keep = (torch.arange(bl, device=DEVICE)[None] >= old_rows[:, None])[:, :, None, None]
        rows[where] = torch.where(keep, held.view(torch.uint8), moved.view(torch.uint8))
        codes = _store(c, x / now[part[:, 0]][:, :, None])
        cache.view(torch.uint8).view(-1, c["Hk"], c["D"])[slots] = codes.view(torch.uint8)
    return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _rows_of(s, b, L):
    """Keys and values 0 .. L - 1 of request b in 32 bits: (Hk, L, D) each."""
    c = s["case"]
    got = []
    for cache, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        raw = cache.view(torch.uint8)
        if c["page"]:
            pages = s["table"][b, :-(-L // c["page"])].long()
            x, f = raw[pages].flatten(0, 1)[:L], scale[pages].flatten(0, 1)
        else:
            x, f = raw[b, :L], scale[b]
        x = x.contiguous().view(cache.dtype).float()
        f = f.repeat_interleave(c["block"], 0)[:L]
        got.append((x * f[:, :, None]).transpose(0, 1).contiguous())
    return got


def _plain_attend(s):
    c = s["case"]
    H, Hk, D, g = c["H"], c["Hk"], c["D"], c["H"] // c["Hk"]
    outs, lses = [], []
    start = 0
    for b, (L, n, _) in enumerate(s["reqs"]):
        q = s["q"][start:start + n] if s["ragged"] else s["q"][b]
        start += n
        sk = L + n
        k, v = _rows_of(s, b, sk)
        x = q.float().view(n, Hk, g, D).permute(1, 0, 2, 3).reshape(Hk, n * g, D)
        x = torch.matmul(x, k.transpose(1, 2)) * D ** -0.5
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        if n > 1 or c["left"] >= 0:
            i = torch.arange(L, sk, device=DEVICE)[:, None]
            j = torch.arange(sk, device=DEVICE)[None]
            hidden = (j > i) if c["causal"] or c["left"] >= 0 else torch.zeros(n, sk, dtype=torch.bool, device=DEVICE)
            if c["left"] >= 0:
                hidden = hidden | (j < i - c["left"])
            x.view(Hk, n, g, sk).masked_fill_(hidden[None, :, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        p = x.sub_(m).exp_()
        z = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v) / z
        outs.append(o.view(Hk, n, g, D).permute(1, 0, 2, 3).reshape(n, H, D).to(s["q"].dtype))
        lses.append((m + z.log()).view(Hk, n, g).permute(0, 2, 1).reshape(H, n))
    if s["ragged"]:
        return {"out": torch.cat(outs), "lse": torch.cat(lses, 1)}
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(c, seed):
    return {"table": _exact_table, "append": _exact_append, "attend": _exact_attend}[c["op"]](prepare(c, seed))


def _exact_table(s):
    P = s["case"]["page"]
    table, free, after = s["table"].tolist(), s["free"].tolist(), s["after"].tolist()
    room, top = len(free), s["num_free"].item()
    for row, (L, _, _), t in zip(table, s["reqs"], after):
        for j in range(-(-t // P), -(-L // P)):
            if top < room:
                free[top] = row[j]
                top += 1
    slots, cu = [], [0]
    for row, (L, _, _), t in zip(table, s["reqs"], after):
        for j in range(-(-L // P), -(-t // P)):
            top -= 1
            row[j] = free[top] if top >= 0 else -1
        slots += [row[x // P] * P + x % P if row[x // P] >= 0 else -1 for x in range(L, t)]
        cu.append(len(slots))
    t32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"table": t32(table), "free": t32(free), "slots": torch.tensor(slots, device=DEVICE), "cu": t32(cu),
            "num_free": t32([top])}


def _exact_append(s):
    c = s["case"]
    bl, top, Hk, D = c["block"], CODE_MAX[c["cache"]], c["Hk"], c["D"]
    runs, at = [], s["slots"].tolist()
    for i, slot in enumerate(at):
        if runs and runs[-1][0] == slot // bl:
            runs[-1][2] += 1
        else:
            runs.append([slot // bl, i, i + 1, slot % bl])
    if len(runs) > 8192:
        return None
    half = torch.round  # to even
    for new, cache, scale in ((s["k_new"], s["k"], s["ks"]), (s["v_new"], s["v"], s["vs"])):
        new, flat = new.double(), scale.view(-1, Hk)
        raw = cache.view(torch.uint8).view(-1, bl, Hk, D)
        most = new.abs().amax(-1)
        for block, i0, i1, first in runs:
            # the smallest e with most / 2^e <= top
            m = most[i0:i1].amax(0)
            e = torch.ceil(torch.log2(torch.clamp(m, min=2.0 ** -120) / top))
            e = torch.where(m / 2.0 ** e > top, e + 1, torch.where(m / 2.0 ** (e - 1) <= top, e - 1, e))
            now = (2.0 ** torch.clamp(e, min=float(FLOOR))).float().double()
            if first:
                old = flat[block].double()
                now = torch.maximum(now, old)
                x = raw[block, :first].view(cache.dtype).double() * (old / now)[None, :, None]
                x = half(x).to(torch.int8) if c["cache"] == "int8" else x.to(cache.dtype)
                raw[block, :first] = x.view(torch.uint8)
            flat[block] = now.float()
            x = new[i0:i1] / now[None, :, None]
            x = half(x).to(torch.int8) if c["cache"] == "int8" else x.to(cache.dtype)
            raw[block, first:first + i1 - i0] = x.view(torch.uint8)
    return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _exact_attend(s):
    c = s["case"]
    g = c["H"] // c["Hk"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.zeros((c["H"], q.shape[0]) if s["ragged"] else (c["B"], c["H"], q.shape[1]), dtype=torch.float64,
                      device=DEVICE)
    start = 0
    for b, (L, n, _) in enumerate(s["reqs"]):
        rows = slice(start, start + n) if s["ragged"] else b
        start += n
        sk = L + n
        j = torch.arange(sk, device=DEVICE)
        page = s["table"][b].long()[j // c["page"]] if c["page"] else torch.full_like(j, b)
        place = j % c["page"] if c["page"] else j
        i = torch.arange(L, sk, device=DEVICE)
        seen = torch.ones(n, sk, dtype=torch.bool, device=DEVICE)
        if c["causal"] or c["left"] >= 0:
            seen &= j[None] <= i[:, None]
        if c["left"] >= 0:
            seen &= j[None] >= i[:, None] - c["left"]
        for h in range(c["Hk"]):
            k, v = (x.view(torch.uint8)[page, place, h].view(x.dtype).double() * f[page, place // c["block"], h, None].double()
                    for x, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for o in range(h * g, (h + 1) * g):
                x = (q[rows][:, o] @ k.t()) / math.sqrt(c["D"])
                if c["softcap"]:
                    x = torch.tanh(x / c["softcap"]) * c["softcap"]
                x = torch.where(seen, x, -math.inf)
                z = torch.logsumexp(x, -1)
                out[rows][:, o] = torch.exp(x - z[:, None]) @ v
                (lse[:, rows] if s["ragged"] else lse[b])[o] = z
    return {"out": out, "lse": lse}
