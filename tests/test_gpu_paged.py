"""Page plan, rotary positions and the paged 8-bit cache's append and read
against their definitions in 64 bits (numpy)."""
import numpy as np
import pytest

import gq

pytestmark = pytest.mark.gpu
INT_MAX = 2**31 - 1


def say(*a):
    print(*a, flush=True)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(v):
    return dev(np.array(v, np.int32).reshape(-1))


# -------------------------------------------------------------- page plan
def plan_ref(cached, new, page, free, tables, max_tokens):
    """Request by request and token by token."""
    wide = tables.shape[1]
    tables, at, starts = tables.copy(), 0, [0]
    pos, slots = np.zeros(max_tokens, np.int64), np.full(max_tokens, -1, np.int64)
    ctx = []
    for r, (c, m) in enumerate(zip(cached, new)):
        c, m = max(c, 0), max(m, 0)
        held, want = min(-(-c // page), wide), min(-(-(c + m) // page), wide)
        for j in range(held, want):
            tables[r, j] = free[at] if at < len(free) else -1
            at += 1
        for i in range(min(m, max_tokens - starts[-1]) if starts[-1] < max_tokens else 0):
            p = c + i
            pos[starts[-1] + i] = p
            if p // page < wide and tables[r, p // page] >= 0:
                s = int(tables[r, p // page]) * page + p % page
                slots[starts[-1] + i] = s if s <= INT_MAX else -1  # (an int holds it, or there is none)
        starts.append(starts[-1] + m)
        ctx.append(c + m)
    return tables, starts, ctx, pos, slots, [starts[-1], at]


def check_plan(backend, cached, new, page, free, tables, max_tokens):
    want = plan_ref(cached, new, page, free, tables, max_tokens)
    t = dev(tables)
    got = backend.page_plan(i32(cached), i32(new), page, i32(free), t, max_tokens)
    for name, a, b in zip(("tables", *got._fields), (t, *got), want):
        np.testing.assert_array_equal(a.cpu().numpy(), b, err_msg=name)
    return got


def held_tables(rng, cached, page, wide, ids):
    t = rng.integers(0, 1000, (len(cached), wide)).astype(np.int32)  # entries past the held ones: anything
    at = 0
    for r, c in enumerate(cached):
        for j in range(min(-(-max(c, 0) // page), wide)):
            t[r, j] = ids[at]
            at += 1
    return t, ids[at:]


@pytest.mark.parametrize("n,page,hi_c,hi_n,wide,short,spare", [
    (1, 16, 0, 1, 1, 0, 0), (1, 64, 5000, 700, 100, 0, 9), (7, 48, 300, 5, 8, 0, 0), (64, 64, 8192, 1, 130, 0, 64),
    (65, 16, 100, 40, 10, 3, 5), (257, 256, 3000, 300, 20, 0, 1), (300, 32, 500, 60, 4, 0, 3), (4096, 16, 50, 3, 5, 40, 0),
    (1000, 128, 40, 0, 3, 0, 7)])
def test_page_plan(backend, n, page, hi_c, hi_n, wide, short, spare):
    """short: pages too few; wide 4, 5, 10: tables too narrow for some."""
    say(f"plan n={n} page={page}")
    rng = np.random.default_rng(n + page)
    cached, new = rng.integers(0, hi_c + 1, n), rng.integers(0, hi_n + 1, n)
    if n > 5:
        cached[2], new[3], new[4] = 0, 0, -7
    ids = rng.permutation(n * (wide + 1) + 64).astype(np.int32)
    tables, rest = held_tables(rng, cached, page, wide, ids)
    if n > 20:
        tables[11, 0] = -1  # a page given back (behind a window)
    need = plan_ref(cached, new, page, rest, tables, 0)[5][1]
    total = int(np.maximum(new, 0).sum())
    check_plan(backend, cached, new, page, rest[:max(0, need - short)], tables, total + spare)
    if total > 3:  # fewer rows than tokens
        check_plan(backend, cached, new, page, rest[:need], tables, total - 3)


def test_page_plan_edges(backend):
    """No requests; no free pages; huge and negative lengths; slots that do
    not fit; nothing to write."""
    none = np.zeros((0, 4), np.int32)
    check_plan(backend, [], [], 16, [3], none, 5)
    check_plan(backend, [5, 0], [3, 0], 16, [], np.array([[7, 0], [0, 0]], np.int32), 4)
    check_plan(backend, [5, 20], [3, 40], 16, [], np.array([[7, 0], [2, 3]], np.int32), 50)
    check_plan(backend, [15, 0], [3, 17], 16, [2**27, -5, 2**27 - 1], np.array([[2**27 - 1, 0], [0, 0]], np.int32), 20)
    check_plan(backend, [3], [2], 16, [1], np.zeros((1, 0), np.int32), 3)
    t = dev(np.zeros((3, 2), np.int32))
    p = backend.page_plan(i32([INT_MAX, -3, 4]), i32([INT_MAX, INT_MAX, 1]), 16, i32([8, 9]), t, 2)
    assert p.q_start.tolist() == [0, INT_MAX, INT_MAX, INT_MAX] and p.ctx_lens.tolist() == [INT_MAX, INT_MAX, 5]
    assert p.slots.tolist() == [-1, -1] and p.positions.tolist() == [INT_MAX, INT_MAX]
    assert p.counts.tolist() == [INT_MAX, 2] and t.tolist() == [[0, 0], [8, 9], [0, 0]]


def test_page_plan_replayed(backend):
    """A captured plan takes new lengths at every replay; rows behind the
    tokens of this replay have no slot."""
    import torch
    rng = np.random.default_rng(5)
    n, page, wide, most = 9, 16, 6, 64
    cached, new, tables = i32([0] * n), i32([0] * n), dev(np.zeros((n, wide), np.int32))
    free = i32(rng.permutation(80))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        backend.page_plan(cached, new, page, free, tables, most)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            p = backend.page_plan(cached, new, page, free, tables, most)
    for k in range(4):
        c, m = rng.integers(0, 60, n), rng.integers(0, 8, n)
        t = rng.integers(0, 80, (n, wide)).astype(np.int32)
        cached.copy_(dev(c.astype(np.int32)))
        new.copy_(dev(m.astype(np.int32)))
        tables.copy_(dev(t))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((tables, *p), plan_ref(c, m, page, free.tolist(), t, most)):
            np.testing.assert_array_equal(a.cpu().numpy(), b)


# ------------------------------------------------------- rotary positions
TYPES = ("float32", "float16", "bfloat16")
HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}


def rope_ref(x, pos, f, m, rot, layout):
    """float64, and |x0| + |x1| of each value's pair."""
    h, y, mag = rot // 2, x.copy(), np.zeros_like(x)
    a = pos.astype(np.float64)[:, None] * f
    c, s = (m * np.cos(a))[:, None], (m * np.sin(a))[:, None]
    i0, i1 = (np.arange(h), np.arange(h) + h) if layout == "half" else (2 * np.arange(h), 2 * np.arange(h) + 1)
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
    mag[..., i0] = mag[..., i1] = np.abs(x[..., i0]) + np.abs(x[..., i1])
    return y, mag


def check_rope(got, x, pos, f, m, rot, layout, dtype):
    """A sine or cosine is off by at most 2.5e-7: the fraction of a turn is
    rounded at 2^-25 of a half turn (9.4e-8 rad), the function by 2 steps of
    2^-24 (1.2e-7), the 64-bit angle by 1e-9.  With the factor m and the two
    products rounded at 2^-24 each, a value is off by at most 4e-7 m (|x0| +
    |x1|), and by half a step of its type."""
    x = x.double().cpu().numpy()
    want, mag = rope_ref(x, pos, f, m, rot, layout)
    err = np.abs(got.double().cpu().numpy() - want)
    tol = 4e-7 * m * mag + HALF_STEP[dtype] * (np.abs(want) + 4e-7 * m * mag) + (2.0**-25 if dtype == "float16" else 0)
    assert (err <= tol).all(), (err - tol).max()
    if rot < x.shape[-1]:
        np.testing.assert_array_equal(got.double().cpu().numpy()[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,nq,nk,hd,rot,hi", [
    (1, 28, 4, 128, 128, 4096), (3, 4, 4, 64, 32, 100), (5, 3, 1, 128, 48, 1 << 20), (2, 1, 0, 64, 64, 1 << 30),
    (4, 2, 2, 96, 24, 5000), (3, 5, 3, 80, 10, 5000), (2, 2, 1, 7, 6, 50), (33, 32, 8, 128, 64, 131072)])
def test_rope(backend, dtype, layout, n, nq, nk, hd, rot, hi):
    import torch
    say(f"rope {dtype} {layout} n={n} heads={nq},{nk} hd={hd} rot={rot}")
    t = getattr(torch, dtype)
    rng = np.random.default_rng(n + hd + rot)
    pos = rng.integers(0, hi, n).astype(np.int32)
    pos[0] = hi - 1
    f, m = gq.rope_freqs(rot, 1e4, "yarn", 4.0, orig_ctx=4096)
    q = dev(rng.standard_normal((n, nq, hd), np.float32)).to(t)
    k = dev(rng.standard_normal((n, nk, hd), np.float32)).to(t) if nk else None
    qo, ko = backend.rope(q, k, dev(pos), dev(f), layout=layout, mscale=m)
    check_rope(qo, q, pos, f, m, rot, layout, dtype)
    if nk:
        check_rope(ko, k, pos, f, m, rot, layout, dtype)
    # in place, the same bits
    q2, k2 = q.clone(), k.clone() if nk else None
    assert backend.rope(q2, k2, dev(pos), dev(f), layout=layout, mscale=m, q_out=q2, k_out=k2)[0] is q2
    assert torch.equal(q2, qo) and (not nk or torch.equal(k2, ko))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("gap,shift", [(0, 0), (3, 0), (8, 1), (16, 8)])
def test_rope_strided(backend, dtype, layout, gap, shift):
    """q and k as parts of one matrix, aligned and not; what lies between
    the rows stays."""
    import torch
    t = getattr(torch, dtype)
    rng = np.random.default_rng(gap + shift)
    n, nq, nk, hd, rot = 6, 4, 2, 64, 64
    f, m = gq.rope_freqs(rot, 1e6)
    pos = rng.integers(0, 9000, n).astype(np.int32)
    wide = shift + (nq + nk) * hd + gap
    all_ = dev(rng.standard_normal((n, wide), np.float32)).to(t)
    ref = all_.clone()
    q = all_[:, shift:shift + nq * hd].unflatten(1, (nq, hd))
    k = all_[:, shift + nq * hd:shift + (nq + nk) * hd].unflatten(1, (nk, hd))
    qo, ko = backend.rope(q, k, dev(pos), dev(f), layout=layout)
    assert torch.equal(all_, ref)
    check_rope(qo, q, pos, f, m, rot, layout, dtype)
    check_rope(ko, k, pos, f, m, rot, layout, dtype)
    backend.rope(q, k, dev(pos), dev(f), layout=layout, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(all_[:, :shift], ref[:, :shift]) and torch.equal(all_[:, wide - gap:], ref[:, wide - gap:])


def test_rope_refuses_tensors(backend):
    import torch
    q, k = torch.zeros((2, 4, 64), device="cuda"), torch.zeros((2, 2, 64), device="cuda")
    pos, f = i32([0, 1]), dev(gq.rope_freqs(64)[0])
    for bad in (dict(q=q.double()), dict(q=q[0]), dict(q=q.transpose(1, 2)), dict(k=k.half()), dict(k=k[:1]),
                dict(k=k[..., :32]), dict(positions=pos.long()), dict(positions=pos[:1]), dict(positions=pos.cpu()),
                dict(inv_freq=f.float()), dict(inv_freq=f.cpu()), dict(layout="whole"), dict(q_out=q[:1]), dict(k_out=q),
                dict(q=q[:1].expand(2, 4, 64))):
        with pytest.raises((ValueError, gq.GqError)):
            backend.rope(**{**dict(q=q, k=k, positions=pos, inv_freq=f), **bad})


# --------------------------------------------------------- append and read
class RefCache:
    """Codes and scales as the definition has them."""

    def __init__(self, n_pages, page, heads, hd, rng):
        self.page = page
        self.codes = [rng.integers(-127, 128, (n_pages, heads, page, hd)).astype(np.int8) for _ in "kv"]
        # (an untouched page's scale may hold anything)
        self.scales = [np.where(rng.random((n_pages, heads)) < 0.3, np.nan, rng.random((n_pages, heads)) + 0.01)
                       .astype(np.float32) for _ in "kv"]

    def on_gpu(self):
        return gq.Kv8Cache(dev(self.codes[0]), dev(self.codes[1]), dev(self.scales[0]), dev(self.scales[1]))

    def append(self, rows, slots):
        pages = {}
        for t, s in enumerate(slots):
            if 0 <= s < self.codes[0].shape[0] * self.page:
                pages.setdefault(s // self.page, []).append((s % self.page, t))
        for codes, scales, x in zip(self.codes, self.scales, rows):
            for p, at in pages.items():
                new = x[[t for _, t in at]].astype(np.float64)  # [rows][heads][hd]
                first = at[0][0]
                for h in range(scales.shape[1]):
                    old = np.float32(0) if first == 0 else scales[p, h]
                    if not np.isfinite(new[:, h]).all() or np.isnan(old):
                        s = np.float32(np.nan)
                    else:
                        s = max(old, np.float32(np.abs(new[:, h]).max() / 127), np.float32(2.0**-60))
                    if s > old > 0:
                        codes[p, h, :first] = np.rint(codes[p, h, :first] * np.float64(old) / np.float64(s))
                    for o, t in at:
                        codes[p, h, o] = 0 if np.isnan(s) else np.rint(x[t, h].astype(np.float64) / np.float64(s))
                    scales[p, h] = s


def same_cache(cache, ref):
    for i, name in enumerate("kv"):
        np.testing.assert_array_equal(cache[2 + i].cpu().numpy(), ref.scales[i], err_msg=name + " scale")
        np.testing.assert_array_equal(cache[i].cpu().numpy(), ref.codes[i], err_msg=name + " codes")


def rows_of(rng, n, heads, hd, t, loud):
    """k, v as device tensors of type t, and as the float32 they hold."""
    out = []
    for _ in "kv":
        x = rng.standard_normal((n, heads, hd), np.float32) * loud
        out.append(dev(x).to(t))
    return out, [o.float().cpu().numpy() for o in out]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,heads,hd", [(16, 2, 64), (64, 3, 128), (48, 1, 128), (256, 2, 64)])
def test_append_and_read(backend, dtype, page, heads, hd):
    """Five requests growing by ragged steps (none, one, several, past a
    page's end), rows that get louder and quieter, rows without a slot."""
    import torch
    say(f"append {dtype} page={page} heads={heads} hd={hd}")
    t = getattr(torch, dtype)
    rng = np.random.default_rng(page + hd)
    n_pages = 24
    ref = RefCache(n_pages, page, heads, hd, rng)
    cache = ref.on_gpu()
    order, ctx = rng.permutation(n_pages), [0] * 5
    for step in range(6):
        slots = []
        for r in range(5):
            m = [0, 1, 1, int(rng.integers(2, 12)), min(page + 3, 4 * page - ctx[r])][int(rng.integers(0, 5))] if step else r * 5
            m = min(m, 4 * page - ctx[r])
            slots += [int(order[4 * r + p // page]) * page + p % page for p in range(ctx[r], ctx[r] + m)]
            ctx[r] += m
        slots += [-1, n_pages * page, -2**31, INT_MAX]
        x, vals = rows_of(rng, len(slots), heads, hd, t, 2.0 ** rng.integers(-3, 4, (len(slots), heads, 1)).astype(np.float32))
        ref.append(vals, slots)
        backend.kv8_append(cache, x[0], x[1], i32(slots))
        same_cache(cache, ref)
    at = np.concatenate([rng.permutation(n_pages * page)[:200], [-1, n_pages * page, -2**31, 0, 0]]).astype(np.int32)
    for rt in TYPES:
        k, v = backend.kv8_read(cache, dev(at), dtype=getattr(torch, rt))
        for got, codes, scales in zip((k, v), ref.codes, ref.scales):
            ok = (at >= 0) & (at < n_pages * page)
            p, o = np.where(ok, at, 0) // page, np.where(ok, at, 0) % page
            want = np.where(ok[:, None, None], codes[p, :, o].astype(np.float64) * scales[p][:, :, None].astype(np.float64), 0)
            got = got.double().cpu().numpy()
            assert np.array_equal(np.isnan(got), np.isnan(want)) and (got[~ok] == 0).all()
            # the product is rounded once, or to f32 (half a step: 2^-24) and then to its type; a
            # float16 below 2^-14 by at most 2^-25
            tol = (HALF_STEP[rt] + (2.0**-24 if rt != "float32" else 0)) * np.abs(want) + (2.0**-25 if rt == "float16" else 0)
            assert (np.abs(got - want)[~np.isnan(want)] <= tol[~np.isnan(want)]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hd,page,lengths", [
    (3, 64, 16, [1] * 900 + [5] * 90),              # single tokens, drafts
    (8, 128, 64, [700, 1, 64, 1, 2, 129, 300, 17] + [1] * 40),
    (8, 64, 256, [1500, 255, 257, 1, 2000, 31, 33]),
    (16, 64, 48, [1, 2, 3, 16, 17, 18, 47, 48, 49] * 11),
    (32, 64, 64, [1] * 70 + [1000, 15, 64, 333, 2, 129, 2000, 63, 65, 700])])
def test_append_many(backend, dtype, heads, hd, page, lengths):
    """Passes of hundreds and thousands of rows: runs of every length that
    begin anywhere, twice, the second time behind the first."""
    import torch
    say(f"append {dtype} heads={heads} page={page} rows={sum(lengths)}")
    t = getattr(torch, dtype)
    rng = np.random.default_rng(heads + page)
    need = [-(-2 * m // page) for m in lengths]
    n_pages = sum(need)
    ref = RefCache(n_pages, page, heads, hd, rng)
    cache = ref.on_gpu()
    ids, first = rng.permutation(n_pages), np.concatenate([[0], np.cumsum(need)])
    for turn in range(2):
        slots = [int(ids[first[r] + p // page]) * page + p % page for r, m in enumerate(lengths) for p in range(turn * m, turn * m + m)]
        x, vals = rows_of(rng, len(slots), heads, hd, t, np.float32(1 + turn))
        ref.append(vals, slots)
        backend.kv8_append(cache, x[0], x[1], i32(slots))
        same_cache(cache, ref)


def test_append_ties_and_ranges(backend):
    """Quotients at, just below and just above a half; values so small that
    the smallest scale holds; the largest finite ones; zeros."""
    import torch
    rng = np.random.default_rng(8)
    ref = RefCache(6, 16, 2, 64, rng)
    cache = ref.on_gpu()
    x = np.zeros((6, 2, 64), np.float32)
    half = (np.arange(64) - 32 + 0.5).astype(np.float32)
    x[0, 0], x[0, 0, 0] = half, 127.0  # scale 1: every quotient a tie
    x[0, 1], x[0, 1, 0] = half * np.float32(0.37), np.float32(127 * 0.37)
    x[1, 0], x[1, 0, 0] = np.nextafter(half, np.float32(100)), 127.0
    x[1, 1], x[1, 1, 0] = np.nextafter(half, np.float32(-100)), 127.0
    x[2] = rng.standard_normal((2, 64)) * 1e-30
    x[3] = rng.standard_normal((2, 64)).astype(np.float32) * np.float32(2.0**-60 * 3)
    x[4, 0, 0], x[4, 0, 1], x[4, 1] = 3.4028234663852886e38, -3.4028234663852886e38, 1e38
    slots = [0, 16, 32, 48, 64, 80]
    ref.append((x, -x), slots)
    backend.kv8_append(cache, dev(x), dev(-x), i32(slots))
    same_cache(cache, ref)
    # and a row behind each, up to a hundred times as loud: the codes before it are rounded again
    y = (np.abs(x).max((1, 2), keepdims=True) * rng.random((6, 2, 64))).astype(np.float32)
    y[:4] *= np.array([1, 2, 100, 1.5], np.float32)[:, None, None]
    slots = [s + 1 for s in slots]
    ref.append((y, y), slots)
    backend.kv8_append(cache, dev(y), dev(y), i32(slots))
    same_cache(cache, ref)


def test_append_every_tie_again(backend):
    """Rescaling by exact ratios: codes at ties go to even."""
    rng = np.random.default_rng(9)
    ref = RefCache(2, 256, 1, 64, rng)
    cache = ref.on_gpu()
    x = np.zeros((255, 1, 64), np.float32)
    x[:] = np.arange(-127, 128, dtype=np.float32)[:, None, None]
    slots = np.arange(255)
    ref.append((x, x), slots)
    backend.kv8_append(cache, dev(x), dev(x), i32(slots))
    same_cache(cache, ref)
    y = np.full((1, 1, 64), 254, np.float32)  # twice the scale: every odd code is a tie
    ref.append((y, y), [255])
    backend.kv8_append(cache, dev(y), dev(y), i32([255]))
    same_cache(cache, ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_not_finite(backend, dtype, bad):
    """A value that is not finite marks its page and head, nothing else; a
    later row does not clear it, rows that start the page anew do."""
    import torch
    t = getattr(torch, dtype)
    rng = np.random.default_rng(4)
    ref = RefCache(3, 16, 2, 64, rng)
    cache = ref.on_gpu()
    for step, slots in enumerate(([0, 1, 16, 32], [2, 17], [0, 1])):
        x, _ = rows_of(rng, len(slots), 2, 64, t, np.float32(1))
        if step == 0:
            x[0][1, 1, 63] = bad
        vals = [a.float().cpu().numpy() for a in x]
        ref.append(vals, slots)
        backend.kv8_append(cache, x[0], x[1], i32(slots))
        same_cache(cache, ref)
        assert np.isnan(ref.scales[0][0, 1]) == (step < 2) and np.isfinite(ref.scales[0][0, 0])


def test_append_strided_and_streams(backend):
    """k and v as parts of one matrix, on a stream of their own."""
    import torch
    rng = np.random.default_rng(6)
    ref = RefCache(8, 32, 2, 64, rng)
    cache = ref.on_gpu()
    all_ = dev(rng.standard_normal((70, 3 * 128 + 4), np.float32))
    k, v = (all_[:, a:a + 128].unflatten(1, (2, 64)) for a in (128, 256))
    slots = list(range(40, 110))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    backend.kv8_append(cache, k, v, i32(slots), stream=s.cuda_stream)
    s.synchronize()
    ref.append([a.cpu().numpy() for a in (k, v)], slots)
    same_cache(cache, ref)


def test_cache_refuses_tensors(backend):
    import torch
    c = gq.kv8_cache(4, 16, 2, 64)
    k, slots = torch.zeros((3, 2, 64), device="cuda"), i32([0, 1, 2])
    for bad in (c._replace(k=c.k[:3]), c._replace(v=c.v.to(torch.uint8)), c._replace(k_scale=c.k_scale[:, :1]),
                c._replace(v_scale=c.v_scale.double()), c._replace(k=c.k[0]), c._replace(v=c.v.transpose(2, 3)),
                c._replace(k=c.k.cpu())):
        with pytest.raises(ValueError):
            backend.kv8_append(bad, k, k, slots)
        with pytest.raises(ValueError):
            backend.kv8_read(bad, slots)
    for a, b, s in ((k[:2], k, slots), (k, k[:2], slots), (k.half(), k, slots), (k[:, :1], k, slots), (k, k, slots[:2]),
                    (k, k, slots.long()), (k[..., ::2], k, slots), (k.cpu(), k.cpu(), slots)):
        with pytest.raises(ValueError):
            backend.kv8_append(c, a, b, s)
    with pytest.raises(gq.GqError):
        backend.kv8_append(c, k.double(), k.double(), slots)
