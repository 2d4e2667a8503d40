"""The operators between the q, k, v products and the o product when many
requests share a GPU, as measurable cases:

  plan      block tables, slot map, positions and row starts of a pass, from
            the requests' lengths
  rope      rotary positions of q and k (half and interleaved layouts, whole
            heads or their first dims, scaled frequencies)
  append    new k and v rows into pages of 8-bit codes with one scale for each
            page and head, and the whole cache read back as the values it holds
  attn      attention of the requests' new tokens over such pages: one token
            each (decode), several (a draft being checked), prompts, or a mix

`run` computes each in its plain form, or where `own` is set by the calls that
a user of agention-infer_amd/gq.py makes.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_FLOOR = 2.0 ** -60  # the smallest scale of a page


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode pass of 64 requests: a token each, a new page for some.
        dict(name="plan_64", kind="plan", requests=64, cached_lo=1, cached_hi=8192, new_lo=1, new_hi=1, page=64),
        # A long pass over very many requests: prompts' chunks and single tokens.
        dict(name="plan_2048", kind="plan", requests=2048, cached_lo=0, cached_hi=32768, new_lo=1, new_hi=63, page=16),
        # One decoded token of the 7B shape: half layout over the whole head.
        dict(name="rope_1", kind="rope", tokens=1, heads=28, kv_heads=4, hd=128, rot=128, layout="half",
             type="f32", theta=1e6, scaling="none", factor=1.0, pos_hi=4096),
        # A pass of prompts at far positions: interleaved pairs in half of
        # each head, frequencies stretched four times (YaRN).
        dict(name="rope_8192", kind="rope", tokens=8192, heads=32, kv_heads=8, hd=128, rot=64, layout="interleaved",
             type="bf16", theta=1e4, scaling="yarn", factor=4.0, pos_hi=131072),
        # The new rows of 64 decoding requests of the 7B shape.
        dict(name="append_64", kind="append", requests=64, cached_lo=0, cached_hi=63, new_lo=1, new_hi=1, page=16,
             kv_heads=4, hd=128, type="f32"),
        # The rows of a pass of ragged prompts.
        dict(name="append_8192", kind="append", requests=24, cached_lo=0, cached_hi=63, new_lo=1, new_hi=681, page=64,
             kv_heads=8, hd=128, type="bf16"),
        # One request's next token at the 7B shape, 4096 positions cached.
        dict(name="decode_1", kind="attn", requests=1, cached_lo=4096, cached_hi=4096, new_lo=1, new_hi=1, page=64,
             heads=28, kv_heads=4, hd=128, type="f32", window=0),
        # The next tokens of 64 requests of very different lengths.
        dict(name="decode_64", kind="attn", requests=64, cached_lo=127, cached_hi=8191, new_lo=1, new_hi=1, page=16,
             heads=32, kv_heads=8, hd=128, type="bf16", window=0),
        # The next tokens of a few very long requests.
        dict(name="decode_long", kind="attn", requests=3, cached_lo=100001, cached_hi=131071, new_lo=1, new_hi=1,
             page=128, heads=28, kv_heads=4, hd=128, type="f16", window=0),
        # Drafts of five tokens being checked, heads of 64 that see a window.
        dict(name="draft_24", kind="attn", requests=24, cached_lo=50, cached_hi=3000, new_lo=5, new_hi=5, page=32,
             heads=16, kv_heads=4, hd=64, type="f32", window=1024),
        # 512 tokens of a prompt after 3584, the 7B shape.
        dict(name="prefill_512", kind="attn", requests=1, cached_lo=3584, cached_hi=3584, new_lo=512, new_hi=512,
             page=64, heads=28, kv_heads=4, hd=128, type="f32", window=0),
        # A mixed pass: ragged prompts' chunks beside single tokens.
        dict(name="mixed_12", kind="attn", requests=12, cached_lo=0, cached_hi=2100, new_lo=1, new_hi=2048, page=64,
             heads=32, kv_heads=8, hd=128, type="bf16", window=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 48, 64, 64, 128, 256])
    kvh = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    hd = rng.choice([64, 128, 128])
    kt = rng.choice(["f32", "f16", "bf16"])
    if kind == "plan":
        b, hi = _log(rng, 1, 4096), rng.choice([1, 1, _log(rng, 2, 600)])
        while b * (hi + 1) > 2048 * 64:
            hi = hi // 2 + 1
            b = b // 2 + 1
        return dict(kind=kind, requests=b, cached_lo=0, cached_hi=_log(rng, 1, 32768), new_lo=rng.choice([0, 1]),
                    new_hi=hi, page=page)
    if kind == "rope":
        n = _log(rng, 1, 8192)
        while n * kvh * (group + 1) * hd > 8192 * 40 * 128:
            n = n // 2 + 1
        scaling = rng.choice(["none", "linear", "yarn", "llama3"])
        return dict(kind=kind, tokens=n, heads=kvh * group, kv_heads=kvh, hd=hd, rot=rng.choice([hd, hd, hd // 2, hd // 4, 48]),
                    layout=rng.choice(["half", "interleaved"]), type=kt, theta=rng.choice([1e4, 5e5, 1e6]), scaling=scaling,
                    factor=1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 40])), pos_hi=_log(rng, 100, 1 << 20))
    if kind == "append":
        b = _log(rng, 1, 256)
        hi = rng.choice([1, _log(rng, 2, 2048)])
        while b * (hi + page) * kvh * hd > 8192 * 8 * 128:
            hi = hi // 2 + 1
            b = b // 2 + (b > 1)
        return dict(kind=kind, requests=b, cached_lo=0, cached_hi=rng.randint(0, 2 * page), new_lo=1, new_hi=hi, page=page,
                    kv_heads=kvh, hd=hd, type=kt)
    b = _log(rng, 1, 64)
    hi = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 1024)])
    ctx = _log(rng, 1, 65536 if hi == 1 else 6000)
    lo = rng.choice([1, hi])
    while b * ctx * kvh * hd > 64 * 4160 * 8 * 128 or b * hi * (ctx + hi) * kvh * group * hd > 6 * 1024 * 3100 * 32 * 128:
        b = b // 2 + (b > 1)
        ctx = ctx * 3 // 4 + 1
        hi = hi * 3 // 4 + 1 if hi > 8 else hi
    return dict(kind=kind, requests=b, cached_lo=rng.choice([0, ctx]), cached_hi=ctx, new_lo=min(lo, hi), new_hi=hi, page=page,
                heads=kvh * group, kv_heads=kvh, hd=hd, type=kt, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))


# ---------------------------------------------------------------- lengths
def _spread(lo, hi, n, turn):
    """n whole numbers from lo to hi, the k-th of them at place k * turn mod n."""
    vals = [lo + (hi - lo) * k // max(1, n - 1) if n > 1 else hi for k in range(n)]
    while math.gcd(turn, n) > 1:
        turn += 1
    return [vals[k * turn % n] for k in range(n)]


def _lengths(case):
    """(cached, new) of each request: the case's alone, so that its work is too."""
    n = case["requests"]
    return _spread(case["cached_lo"], case["cached_hi"], n, 7), _spread(case["new_lo"], case["new_hi"], n, 1)


def _pages(tokens, page):
    return (tokens + page - 1) // page


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["hd"] * _SIZE[case["type"]] + 4 * case["tokens"] + 4 * case["rot"],
                "flops": 3 * n * case["rot"]}
    cached, new = _lengths(case)
    page, t = case["page"], sum(new)
    if kind == "plan":
        took = sum(_pages(c + m, page) - _pages(c, page) for c, m in zip(cached, new))
        held = sum(1 for c in cached if c % page)
        return {"bytes": 4 * (2 * len(new) + held + 2 * took + 2 * t + 2 * len(new) + 1 + 2), "flops": 0}
    row = case["kv_heads"] * case["hd"]
    if kind == "append":
        # k and v once, their codes and scales once, and the whole cache read
        # (codes) and given back as values
        touched = sum(_pages(c + m, page) - c // page for c, m in zip(cached, new))
        scales = 2 * 4 * case["kv_heads"]
        pool = touched + 3
        return {"bytes": 2 * t * row * (_SIZE[case["type"]] + 1) + 4 * t + scales * (touched + pool) + pool * page * (4 + 2 * row * 5),
                "flops": 4 * t * row}
    keys, pairs = 0, 0
    for c, m in zip(cached, new):
        w = case["window"] or c + m
        keys += c + m - max(0, c - w + 1) if m else 0
        pairs += sum(min(c + i + 1, w) for i in range(m))
    return {"bytes": 2 * t * case["heads"] * case["hd"] * _SIZE[case["type"]] + 2 * keys * row
            + 8 * case["kv_heads"] * _pages(keys, page) + 4 * _pages(keys, page) + 8 * len(new),
            "flops": 4 * pairs * case["heads"] * case["hd"]}


# ----------------------------------------------------------------- inputs
def _freqs(rot, theta, scaling, factor):
    """Radians a position of each pair, in 64 bits, and the factor of the
    rotated values: a model's table, made once.  The scaled ones are for a
    model trained on 8192 positions."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2.0 * i / rot)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    turns = 8192 * f / (2 * math.pi)  # over the trained context
    if scaling == "llama3":  # slow pairs stretched, fast ones kept, between 1 and 4 turns a mix
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    at = [rot * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
    lo, hi = max(0.0, math.floor(at[0])), min(rot - 1.0, math.ceil(at[1]))
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = dict(case)
    if kind == "rope":
        t = _TYPES[case["type"]]
        f, m = _freqs(case["rot"], case["theta"], case["scaling"], case["factor"])
        s["freqs"], s["mscale"] = f.cuda(), m
        n = case["tokens"]
        s["positions"] = torch.randint(0, case["pos_hi"], (n,), dtype=torch.int32, device="cuda", generator=g)
        s["q"] = torch.randn((n, case["heads"], case["hd"]), device="cuda", generator=g).to(t)
        s["k"] = torch.randn((n, case["kv_heads"], case["hd"]), device="cuda", generator=g).to(t)
        return s
    rng = random.Random(seed)
    cached, new = _lengths(case)
    order = list(range(len(new)))
    rng.shuffle(order)
    cached, new = [cached[i] for i in order], [new[i] for i in order]
    page, n = case["page"], len(new)
    if kind == "append":  # only the page that each request is in and its new ones are held here
        cached = [c % page for c in cached]
    total = [c + m for c, m in zip(cached, new)]
    wide = max(1, max(_pages(v, page) for v in total))
    held = [_pages(c if kind == "plan" else v, page) for c, v in zip(cached, total)]
    took = sum(_pages(v, page) for v in total) - sum(held)
    pool = sum(held) + took + 3
    free = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((n, wide), -1, dtype=torch.int32)
    ids, at = free.cpu(), 0
    for i, h in enumerate(held):
        tables[i, :h] = ids[at:at + h]
        at += h
    s["tables"], s["free"] = tables.cuda(), free[at:].clone()
    s["tokens"], s["pool"] = sum(new), pool
    s["cached"], s["new"] = _ints(cached), _ints(new)
    if kind == "plan":
        return s
    t = _TYPES[case["type"]]
    shape = (pool, case["kv_heads"], page, case["hd"])
    for name in ("k", "v"):  # rows of standard deviation about 1, scales of trained heads' spread
        c = torch.empty(shape, dtype=torch.int8, device="cuda")
        for part in c.split(max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))):
            part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(32).round_().clamp_(-127, 127))
        s[name + "_codes"] = c
        s[name + "_scales"] = torch.exp2(torch.randn(shape[:2], device="cuda", generator=g) * 0.5) / 32
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    if kind == "append":
        pos = [c + j for c, m in zip(cached, new) for j in range(m)]
        req = [i for i, m in enumerate(new) for _ in range(m)]
        tb = tables[torch.tensor(req), torch.tensor(pos) // page]
        s["slots"] = (tb * page + torch.tensor(pos) % page).to(torch.int32).cuda()
        s["every_slot"] = torch.arange(pool * page, dtype=torch.int32, device="cuda")
        loud = torch.exp2(torch.randn((s["tokens"], 1, 1), device="cuda", generator=g) * 0.5)  # tokens differ in size
        for name in ("k", "v"):
            x = torch.randn((s["tokens"], case["kv_heads"], case["hd"]), device="cuda", generator=g)
            s[name] = (x * loud).to(t)
        return s
    s["q"] = torch.randn((s["tokens"], case["heads"], case["hd"]), device="cuda", generator=g).to(t)
    s["q_start"], s["ctx"] = _ints(starts), _ints(total)
    s["max_new"], s["max_ctx"] = max(new), max(total)
    s["scale"] = 1.0 / math.sqrt(case["hd"])
    return s


# ------------------------------------------------------------ plain forms
def _plan(s):
    page, tables, free = s["page"], s["tables"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    n, wide = tables.shape
    dev = tables.device
    before = ((cached + page - 1) // page).clamp(max=wide)
    after = ((cached + new + page - 1) // page).clamp(max=wide)
    need = after - before
    first = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    q_start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), ends])
    j = torch.arange(wide, device=dev).unsqueeze(0)
    at = first.unsqueeze(1) + j - before.unsqueeze(1)
    given = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)].long(), -1)
    fresh = (j >= before.unsqueeze(1)) & (j < after.unsqueeze(1))
    tables.copy_(torch.where(fresh, given, tables.long()))
    t = torch.arange(s["tokens"], device=dev)
    r = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    pos = cached[r] + t - q_start[r]
    p = torch.where(pos // page < wide, tables[r, (pos // page).clamp(max=wide - 1)].long(), -1)
    slots = torch.where(p >= 0, p * page + pos % page, -1)
    i32 = torch.int32
    return dict(tables=tables, q_start=q_start.to(i32), ctx=(cached + new).to(i32), positions=pos.to(i32),
                slots=slots.to(i32), counts=torch.stack([ends[-1], need.sum()]).to(i32))


def _turned(x, c, sn, rot, layout):
    h = rot // 2
    f = x.float()
    a, b = (f[..., :h], f[..., h:rot]) if layout == "half" else (f[..., 0:rot:2], f[..., 1:rot:2])
    y0, y1 = a * c - b * sn, a * sn + b * c
    y = torch.cat([y0, y1], -1) if layout == "half" else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, f[..., rot:]], -1).to(x.dtype)


def _rope(s):
    a = s["positions"].double().unsqueeze(-1) * s["freqs"]
    c, sn = ((w * s["mscale"]).float().unsqueeze(1) for w in (torch.cos(a), torch.sin(a)))
    return dict(q=_turned(s["q"], c, sn, s["rot"], s["layout"]), k=_turned(s["k"], c, sn, s["rot"], s["layout"]))


def _append(x, codes, scales, slots, page):
    """One of k and v into its pages; the values that the whole cache then holds."""
    pool, h, _, d = codes.shape
    at, off = slots.long() // page, slots.long() % page
    x = x.float()
    top = torch.zeros((pool, h), device=x.device).scatter_reduce_(0, at.unsqueeze(1).expand(-1, h), x.abs().amax(-1), "amax")
    base = torch.full((pool,), page, device=x.device).scatter_reduce_(0, at, off, "amin")
    old = torch.where((base == 0).unsqueeze(1), 0.0, scales)
    now = torch.where((base < page).unsqueeze(1), torch.maximum(old, (top.double() / 127).float()).clamp(min=_FLOOR), scales)
    earlier = torch.arange(page, device=x.device) < torch.where(base < page, base, 0).unsqueeze(1)
    again = torch.round(codes.double() * old.double()[:, :, None, None] / now.double()[:, :, None, None]).to(torch.int8)
    codes.copy_(torch.where(earlier[:, None, :, None], again, codes))
    scales.copy_(now)
    codes[at, :, off] = torch.round(x.double() / now[at].double().unsqueeze(-1)).to(torch.int8)
    return (codes.float() * now[:, :, None, None]).permute(0, 2, 1, 3).reshape(pool * page, h, d)


def _attn(s):
    page, kvh, hd = s["page"], s["kv_heads"], s["hd"]
    group = s["heads"] // kvh
    n, m = s["requests"], s["max_new"]
    dev = s["q"].device
    wide = _pages(s["max_ctx"], page)
    ids = s["tables"][:, :wide].long()
    at = ids.clamp(min=0)

    def dense(codes, scales):  # [request][head][position][dim]
        x = codes[at].float() * scales[at][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, kvh, wide * page, hd)

    start, ctx = s["q_start"].long(), s["ctx"].long()
    new = start[1:] - start[:-1]
    i = torch.arange(m, device=dev)
    row = (start[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[row].view(n, m, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, m * group, hd)
    w = torch.matmul(q, dense(s["k_codes"], s["k_scales"]).transpose(2, 3).contiguous()).mul_(s["scale"])
    pos = (ctx - new)[:, None] + i
    key = torch.arange(wide * page, device=dev)
    sees = (key <= pos[..., None]) & (ids >= 0).repeat_interleave(page, 1)[:, None]
    if s["window"]:
        sees &= key > pos[..., None] - s["window"]
    w = w.view(n, kvh, m, group, wide * page).masked_fill_(~sees[:, None, :, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n, kvh, m * group, wide * page), dense(s["v_codes"], s["v_scales"])).view(n, kvh, m, group, hd)
    o = (o / torch.where(total > 0, total, 1.0)).permute(0, 2, 1, 3, 4).reshape(n, m, s["heads"], hd)
    t = torch.arange(s["tokens"], device=dev)
    r = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=n - 1)
    return o[r, t - start[r]].to(s["q"].dtype)


# -------------------------------------------------------- the library's
_be = None


def _backend():
    global _be
    if _be is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "agention-infer_amd"))
        import gq
        _be = gq.create_backend("hip")
    return _be


def _own(s):
    be, kind = _backend(), s["kind"]
    if kind == "plan":
        p = be.page_plan(s["cached"], s["new"], s["page"], s["free"], s["tables"], s["tokens"])
        return dict(tables=s["tables"], q_start=p.q_start, ctx=p.ctx_lens, positions=p.positions, slots=p.slots, counts=p.counts)
    if kind == "rope":
        q, k = be.rope(s["q"], s["k"], s["positions"], s["freqs"], layout=s["layout"], mscale=s["mscale"])
        return dict(q=q, k=k)
    cache = (s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    if kind == "append":
        be.kv8_append(cache, s["k"], s["v"], s["slots"])
        k, v = be.kv8_read(cache, s["every_slot"])
        return dict(k=k, v=v, k_scales=s["k_scales"], v_scales=s["v_scales"])
    return be.attn_kv8(s["q"], cache, s["tables"], s["q_start"], s["ctx"], s["max_new"], s["max_ctx"], scale=s["scale"],
                       window=s["window"])


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "plan":
        return _plan(s)
    if kind == "rope":
        return _rope(s)
    if kind == "append":
        return dict(k=_append(s["k"], s["k_codes"], s["k_scales"], s["slots"], s["page"]),
                    v=_append(s["v"], s["v_codes"], s["v_scales"], s["slots"], s["page"]),
                    k_scales=s["k_scales"], v_scales=s["v_scales"])
    return _attn(s)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    if case["kind"] == "rope":  # complex products
        z = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda"),
                        s["positions"].double()[:, None, None] * s["freqs"])
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            rot, y = case["rot"], x.clone()
            if case["layout"] == "half":
                w = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
                y[..., :rot // 2], y[..., rot // 2:rot] = w.real, w.imag
            else:
                w = torch.view_as_complex(x[..., :rot].contiguous().view(*x.shape[:2], rot // 2, 2)) * z
                y[..., :rot] = torch.view_as_real(w).flatten(-2)
            out[name] = y
        return out
    page = case["page"]
    if case["kind"] == "append":  # page by page, in the order of the slots
        out = {}
        slots = s["slots"].cpu().tolist()
        runs, t = [], 0
        while t < len(slots):
            e = t + 1
            while e < len(slots) and slots[e] == slots[e - 1] + 1 and slots[e] % page:
                e += 1
            runs.append((slots[t] // page, slots[t] % page, t, e))
            t = e
        for name in ("k", "v"):
            c, sc, x = s[name + "_codes"].double(), s[name + "_scales"], s[name].double()
            for p, o, t, e in runs:
                new = x[t:e].abs().amax((0, 2))
                want = (new / 127).float()  # a scale is held in 32 bits
                was = sc[p].clone()
                sc[p] = torch.maximum(want, was if o else torch.full_like(was, _FLOOR)).clamp(min=_FLOOR)
                if o:
                    c[p, :, :o] = torch.round(c[p, :, :o] * was.double()[:, None, None] / sc[p].double()[:, None, None])
                c[p, :, o:o + e - t] = torch.round(x[t:e].permute(1, 0, 2) / sc[p].double()[:, None, None])
            out[name] = (c * sc.double()[:, :, None, None]).permute(0, 2, 1, 3).reshape(s["pool"] * page, case["kv_heads"], -1)
            out[name + "_scales"] = sc.double()
        return out
    group, start, ctx = case["heads"] // case["kv_heads"], s["q_start"].tolist(), s["ctx"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["requests"]):
        ids = s["tables"][b, :_pages(ctx[b], page)].long()
        m = start[b + 1] - start[b]
        for h in range(case["kv_heads"] if m else 0):
            k, v = ((s[x + "_codes"][ids, h].double() * s[x + "_scales"][ids, h].double()[:, None, None]).flatten(0, 1)[:ctx[b]]
                    for x in ("k", "v"))
            for lo in range(0, m, 256):  # some rows of queries at a time
                i = torch.arange(lo, min(m, lo + 256), device="cuda")
                pos = ctx[b] - m + i
                q = s["q"][start[b] + i, h * group:(h + 1) * group].double()
                w = torch.matmul(q, k.T.contiguous()) * s["scale"]
                key = torch.arange(ctx[b], device="cuda")
                hides = key > pos[:, None]
                if case["window"]:
                    hides |= key <= pos[:, None] - case["window"]
                w = torch.softmax(w.masked_fill(hides[:, None], -math.inf), -1)
                out[start[b] + i, h * group:(h + 1) * group] = torch.matmul(w, v)
    return out
