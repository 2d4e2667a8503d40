"""Attention over the paged 8-bit cache against its definition in 64 bits.

Tolerances.  Scores: q is carried to 2^-23 of its row's largest value (f32)
or exactly (16-bit types), a product of hd terms is summed in f32, and two f32
operations put it into base 2, so a score is off by at most
  E_s = scale (2^-23 max|q| sum|k| + (hd + 8) 2^-24 sum|q k|) + 2^-22 (|s| + 61)
(61: the largest log2 of a scale in these tests, with room).  A weight is then
off by E_s + 2^-20 of itself (exp2, two f16 parts), or with one f16 part by
E_s + 2^-11 + 2^-20; numerator and denominator each carry that once, and the sum
of N products in f32 adds (N / 32 + 64) 2^-24.  Together, per value,
  (2 E_s + 2^-18 (+ 2^-11 for 16-bit types) + (N / 32 + 64) 2^-24) sum p|v| + half a step of |o|.
Small weights: a weight times its page's V scale is held as f16, the largest
of a row between 2^14 and 2^15.9, and f16 has no steps below 2^-24, so each (its
last part, where there are two) is also off by up to 2^-25 / 2^14 of the largest:
2^-39 max(p vs) sum|code|.
"""
import numpy as np
import pytest

import gq

pytestmark = pytest.mark.gpu
TYPES = ("float32", "float16", "bfloat16")
HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}


def say(*a):
    print(*a, flush=True)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(v):
    return dev(np.array(v, np.int32).reshape(-1))


class Case:
    """Requests [(cached, new)] over a shuffled pool; pages that no request
    has hold NaN scales, and slots behind a request's last key any codes."""

    def __init__(self, reqs, page, kvh, group, hd, dtype, seed=0, loud=1.0, spare=3, gap=0):
        import torch
        rng = self.rng = np.random.default_rng(seed)
        self.page, self.kvh, self.group, self.hd, self.dtype = page, kvh, group, hd, dtype
        self.t = getattr(torch, dtype)
        self.new = [m for _, m in reqs]
        self.ctx = [c + m for c, m in reqs]
        need = [-(-c // page) for c in self.ctx]
        pool = sum(need) + spare
        self.wide = max(max(need), 1) + 1
        ids = rng.permutation(pool)
        self.tables, at = np.full((len(reqs), self.wide), 10**6, np.int32), 0
        for i, k in enumerate(need):
            self.tables[i, :k] = ids[at:at + k]
            at += k
        self.codes = [rng.integers(-128, 128, (pool, kvh, page, hd)).astype(np.int8) for _ in "kv"]
        self.scales = [np.exp2(rng.normal(0, 1, (pool, kvh))).astype(np.float32) / 73 for _ in "kv"]
        for s in self.scales:
            s[ids[at:]] = np.nan
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(int)
        self.n = int(self.starts[-1]) + 2  # and two rows of nobody
        x = rng.standard_normal((self.n, kvh * group * hd + gap), np.float32) * np.float32(loud)
        self.q = dev(x).to(self.t)[:, :kvh * group * hd].unflatten(1, (kvh * group, hd))
        self.scale = hd ** -0.5

    def cache(self):
        return gq.Kv8Cache(*map(dev, self.codes), *map(dev, self.scales))

    def want(self, window=0, most=2**31):
        """(out, tolerance) float64; NaN where a row sees a NaN."""
        q = self.q.double().cpu().numpy()
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        for b, m in enumerate(self.new):
            ctx = self.ctx[b]
            pos = np.arange(ctx)
            ids = self.tables[b, pos // self.page] if ctx else np.zeros(0, int)
            ok = (ids >= 0) & (ids < self.codes[0].shape[0]) & (pos < most)
            ids = np.where(ok, ids, 0)
            for h in range(self.kvh):
                k, v = (c[ids, h, pos % self.page].astype(np.float64) * s[ids, h][:, None].astype(np.float64)
                        for c, s in zip(self.codes, self.scales))
                for i in range(m):
                    p = ctx - m + i
                    sees = ok & (pos <= p) & (pos > p - window if window else True)
                    if not sees.any():
                        continue
                    ks, vs = k[sees], v[sees]
                    vsc = self.scales[1][ids, h][sees].astype(np.float64)
                    small = 2.0**-39 * np.abs(vs / vsc[:, None]).sum(0)
                    for g in range(self.group):
                        r, c = self.starts[b] + i, h * self.group + g
                        x = q[r, c]
                        s = ks @ x * self.scale
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        out[r, c] = w @ vs
                        hi = 2.0**-23 * np.abs(x).max() if self.dtype == "float32" else 0.0
                        e = np.abs(self.scale) * (hi * np.abs(ks).sum(1) + (self.hd + 8) * 2.0**-24 * (np.abs(ks) @ np.abs(x))) \
                            + 2.0**-22 * (np.abs(s) + 61)
                        one = 0 if self.dtype == "float32" else 2.0**-11
                        tol[r, c] = (2 * e.max() + 2.0**-18 + one + (len(s) / 32 + 64) * 2.0**-24) * (w @ np.abs(vs)) \
                            + HALF_STEP[self.dtype] * np.abs(out[r, c]) + (2.0**-25 if self.dtype == "float16" else 0) + small * (w * vsc).max()
        return out, tol

    def args(self, max_new=None, max_ctx=None):
        return (dev(self.tables), i32(self.starts), i32(self.ctx), max(self.new) if max_new is None else max_new,
                max(self.ctx) if max_ctx is None else max_ctx)

    def check(self, backend, window=0, cache=None, **kw):
        import torch
        out = torch.full(self.q.shape, 7.5, dtype=self.t, device="cuda")
        got = backend.attn_kv8(self.q, cache or self.cache(), *self.args(), scale=self.scale, window=window, out=out, **kw)
        assert got is out
        want, tol = self.want(window)
        mine = self.starts[-1]
        assert (out[mine:] == 7.5).all()  # rows of nobody stay
        got = out[:mine].double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want[:mine]))
        if self.dtype == "float16":  # values past its largest, 65504, are infinities
            over = np.abs(want[:mine]) - np.nan_to_num(tol[:mine]) > 65520
            assert (got[over] == np.sign(want[:mine][over]) * np.inf).all()
            near = np.isinf(got) & (np.abs(want[:mine]) + tol[:mine] > 65504) & (np.sign(got) == np.sign(want[:mine]))
            got[near] = want[:mine][near]
        err = np.nan_to_num(np.abs(got - want[:mine]))
        assert (err <= np.nan_to_num(tol[:mine], nan=1)).all(), (err / np.nan_to_num(tol[:mine], nan=1)).max()
        return out


RAGGED = [(0, 1), (15, 1), (16, 1), (700, 1), (0, 0), (63, 1), (5, 0), (1000, 1)]
SHAPES = [  # requests, page, KV heads, query heads of each, head_dim, window
    ([(0, 1)], 16, 1, 1, 64, 0),
    ([(4096, 1)], 64, 4, 7, 128, 0),
    (RAGGED, 16, 2, 4, 128, 0),
    (RAGGED, 48, 3, 5, 64, 100),
    (RAGGED, 256, 1, 8, 128, 1),
    ([(100, 3), (0, 5), (511, 2), (64, 9)], 32, 2, 7, 128, 0),
    ([(300, 4), (2, 8)], 128, 1, 71, 64, 40),
    ([(0, 130), (77, 61), (200, 1)], 64, 2, 3, 128, 0),
    ([(0, 40), (333, 300)], 16, 1, 16, 64, 64),
    ([(0, 600), (30, 1)], 64, 1, 4, 128, 0),
    ([(2500, 70)], 48, 1, 2, 64, 1000),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", range(len(SHAPES)))
def test_attention(backend, dtype, at):
    reqs, page, kvh, group, hd, window = SHAPES[at]
    say(f"attention {dtype} {reqs} page={page} kv={kvh} group={group} hd={hd} window={window}")
    Case(reqs, page, kvh, group, hd, dtype, seed=at).check(backend, window)


@pytest.mark.parametrize("dtype", TYPES)
def test_holes_and_empty_rows(backend, dtype):
    """Entries that are no pages (before a window, wild ones, all of them):
    their keys are not seen, rows that see nothing are zeros; ctx_lens shorter
    than the rows."""
    c = Case([(100, 4), (40, 2), (200, 70), (0, 3)], 16, 2, 3, 64, dtype, seed=5)
    c.tables[0, :5] = [-1, 2**31 - 1, -2**31, -1, 10**6]
    c.tables[1] = -1
    c.tables[2, 3:9] = -7
    c.ctx[3] = 2  # its first row sees nothing
    out = c.check(backend)
    assert (out[4:6] == 0).all() and (out[76] == 0).all()
    c.check(backend, window=20)


@pytest.mark.parametrize("reqs", [[(100, 4), (40, 2), (9, 1)], [(100, 70), (40, 30), (9, 1)]])
def test_bounds_hide_keys(backend, reqs):
    """Keys past max_ctx, and past what the table holds, are not seen."""
    for window in (0, 20):
        for most in (25, 64, 100):
            c = Case(reqs, 16, 2, 3, 64, "float32", seed=17)
            got = backend.attn_kv8(c.q, c.cache(), *c.args(max_ctx=most), window=window)[:c.starts[-1]]
            whole = c.tables.copy()
            want, tol = c.want(window, most)
            assert (np.abs(got.double().cpu().numpy() - want[:c.starts[-1]]) <= tol[:c.starts[-1]]).all()
            wide = most // 16  # a table that ends there
            c.tables = np.ascontiguousarray(whole[:, :wide])
            got = backend.attn_kv8(c.q, c.cache(), *c.args(), window=window)[:c.starts[-1]]
            c.tables = whole
            want, tol = c.want(window, 16 * wide)
            assert (np.abs(got.double().cpu().numpy() - want[:c.starts[-1]]) <= tol[:c.starts[-1]]).all()
    c.tables = np.zeros((len(reqs), 0), np.int32)
    assert (backend.attn_kv8(c.q, c.cache(), *c.args())[:c.starts[-1]] == 0).all()


@pytest.mark.parametrize("reqs,most", [([(2000, 12), (30, 3)], 5), ([(0, 70), (700, 90), (9, 1)], 33), ([(10, 300)], 43)])
def test_rows_past_max_new_stay(backend, reqs, most):
    """Rows within max_new are the request's own, the others left alone: in
    the same tile, with and without parts."""
    import torch
    c = Case(reqs, 16, 2, 3, 64, "float32", seed=18)
    out = torch.full(c.q.shape, 7.5, dtype=c.t, device="cuda")
    backend.attn_kv8(c.q, c.cache(), *c.args(max_new=most), out=out)
    want, tol = c.want()
    got = out.double().cpu().numpy()
    for b, m in enumerate(c.new):
        s = c.starts[b]
        assert (np.abs(got - want) <= tol)[s:s + min(m, most)].all() and (got[s + most:s + m] == 7.5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reqs", [[(100, 2), (90, 2)], [(100, 80), (3, 2)]])
def test_not_finite_pages(backend, dtype, reqs):
    """A page with a NaN scale makes NaN of the rows that see it and of no
    others: rows in front of it, behind a window, or of another head."""
    c = Case(reqs, 16, 2, 2, 64, dtype, seed=6)
    c.scales[0][c.tables[0, 2], 0] = np.nan   # positions 32..47, k, head 0
    c.scales[1][c.tables[1, 0], 1] = np.nan   # positions 0..15 of the second, v, head 1
    out = c.check(backend)
    assert out[:c.starts[1], :2].isnan().all() and not out[:c.starts[1], 2:].isnan().any()
    c.check(backend, window=30)
    # and a page's scale that only later rows see
    c = Case([(10, 60)], 16, 1, 2, 64, dtype, seed=7)
    c.scales[1][c.tables[0, 3], 0] = np.nan
    out = c.check(backend)
    assert not out[:38].isnan().any() and out[38:60].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_any_size(backend, dtype):
    """Very loud and very quiet rows, zeros, scores far apart."""
    for loud in (1e-4, 30.0):
        Case([(333, 2), (20, 40)], 32, 1, 3, 128, dtype, seed=8, loud=loud).check(backend)
    c = Case([(333, 2), (20, 40)], 32, 1, 3, 128, dtype, seed=9)
    c.q[1] = 0
    c.q[3, 1] = 0
    c.check(backend)


@pytest.mark.parametrize("reqs", [[(333, 2), (20, 1)], [(333, 100), (20, 1)]])
def test_not_finite_queries(backend, reqs):
    """A row with a NaN or an infinity is NaN, its neighbours are not."""
    import torch
    for bad in (float("nan"), float("inf")):
        c = Case(reqs, 32, 1, 4, 64, "float32", seed=10)
        c.q[1, 2, 5] = bad
        out = backend.attn_kv8(c.q, c.cache(), *c.args())[:c.starts[-1]]
        assert out[1, 2].isnan().all()
        out[1, 2] = 0
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_page_scales_far_apart(backend, dtype):
    """V scales from the smallest one up: no page's weight is lost or
    overflows, and pages of zeros count in the sum."""
    c = Case([(400, 3), (50, 50)], 16, 1, 4, 64, dtype, seed=11)
    c.scales[1][:] = np.float32(2.0) ** c.rng.integers(-60, 30, c.scales[1].shape)
    c.check(backend)
    c.scales[1][:] = 2.0**-60
    c.codes[1][:] = 0
    out = c.check(backend)
    assert (out[:c.starts[-1]] == 0).all()
    c.scales[1][c.tables[0, 3]] = 0.5
    c.codes[1][c.tables[0, 3]] = 100
    c.check(backend)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(backend, dtype):
    """q as part of a wider matrix, out as part of another."""
    import torch
    c = Case([(100, 2), (0, 33)], 16, 2, 2, 64, dtype, seed=12, gap=8)
    wide = torch.full((c.n, 4 * 64 + 16), 3.0, dtype=c.t, device="cuda")
    out = wide[:, :256].unflatten(1, (4, 64))
    backend.attn_kv8(c.q, c.cache(), *c.args(), out=out)
    ref = c.check(backend)
    assert torch.equal(out[:c.starts[-1]], ref[:c.starts[-1]]) and (wide[:, 256:] == 3).all() and (out[-2:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reqs", [[(5000, 1), (300, 1), (17, 1)], [(600, 4)], [(900, 200), (0, 1), (64, 17)]])
def test_same_bits_again(backend, dtype, reqs):
    """Again, with looser bounds, on other streams side by side, and beside
    other requests: a row's own result.  (Looser bounds may cut the keys
    otherwise, so those compare to the tolerance.)"""
    import torch
    c = Case(reqs, 16, 2, 4, 128, dtype, seed=13)
    cache, out = c.cache(), c.check(backend)
    mine = c.starts[-1]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        outs.append(backend.attn_kv8(c.q, cache, *c.args(), stream=s.cuda_stream))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[:mine], out[:mine])
    want, tol = c.want()
    loose = backend.attn_kv8(c.q, cache, *c.args(max_new=max(c.new) + 40, max_ctx=60000))[:mine].double().cpu().numpy()
    assert (np.abs(loose - want[:mine]) <= tol[:mine]).all()


@pytest.mark.parametrize("most", [1, 40])
def test_replayed(backend, most):
    """Two captured calls, replayed in turn and side by side for other
    requests and queries within their bounds, with eager calls between."""
    import torch
    rng = np.random.default_rng(14)
    nr, bound = 5, 1500
    graphs = []
    cases = [Case([(bound - most, most)] * nr, 16, 2, 4, 64, "float32", seed=s) for s in (20, 21)]
    for c in cases:
        c.dev = (c.q, c.cache(), *c.args())
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.out = backend.attn_kv8(*c.dev)
        graphs.append((g, s))
    for turn in range(3):
        for c in cases:
            c.new = rng.integers(0, most + 1, nr).tolist()
            c.ctx = [int(rng.integers(m, bound + 1)) for m in c.new]
            c.starts = np.concatenate([[0], np.cumsum(c.new)])
            c.dev[3].copy_(i32(c.starts))
            c.dev[4].copy_(i32(c.ctx))
            c.q.copy_(dev(rng.standard_normal(tuple(c.q.shape), np.float32)))
            c.out.fill_(7.5)
        torch.cuda.synchronize()
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c in cases:
            want, tol = c.want()
            mine = int(c.starts[-1])
            got = c.out.double().cpu().numpy()
            assert (np.abs(got - want)[:mine] <= tol[:mine]).all() and (got[mine:] == 7.5).all()
            eager = backend.attn_kv8(*c.dev)
            assert torch.equal(eager[:mine], c.out[:mine])
            float(eager[:mine].sum())


def test_far_offsets(backend):
    """A cache of more than 2^32 bytes of codes: its last pages."""
    import torch
    page, kvh, hd, n_pages = 256, 2, 128, 66000
    cache = gq.kv8_cache(n_pages, page, kvh, hd)
    assert cache.k.numel() > 2**32
    rng = np.random.default_rng(15)
    c = Case([(600, 30)], page, kvh, 2, hd, "float32", seed=15, spare=0)
    c.tables[0, :3] = [n_pages - 1, n_pages - 3, 65536]
    pos = np.arange(630)
    slots = c.tables[0, pos // page].astype(np.int64) * page + pos % page
    x = [rng.standard_normal((630, kvh, hd), np.float32) for _ in "kv"]
    backend.kv8_append(cache, dev(x[0]), dev(x[1]), i32(slots))
    got = backend.kv8_read(cache, i32(slots))
    for a, b in zip(got, x):
        # half a step of a scale (max / 127), and the f32 rounding of scale and product
        assert np.abs(a.cpu().numpy() - b).max() <= (0.5 + 1e-4) * 6 / 127
    out = backend.attn_kv8(c.q, cache, *c.args())
    small = gq.kv8_cache(3, page, kvh, hd)
    backend.kv8_append(small, dev(x[0]), dev(x[1]), i32(pos))
    c.tables[0, :3] = [0, 1, 2]
    assert torch.equal(backend.attn_kv8(c.q, small, *c.args())[:30], out[:30])


def test_whole_pass(backend):
    """Three passes of ragged requests as a server runs them (plan, rotary
    positions, append, attention), the last ones decoding, against the same
    computed request by request in 64 bits from the values that the cache
    holds."""
    import torch
    rng = np.random.default_rng(16)
    page, kvh, group, hd, nr = 16, 2, 3, 64, 4
    nh = kvh * group
    cache = gq.kv8_cache(40, page, kvh, hd)
    tables = torch.full((nr, 8), -1, dtype=torch.int32, device="cuda")
    free = i32(rng.permutation(40))
    inv, m = gq.rope_freqs(hd, 1e4, "yarn", 4.0, orig_ctx=64)
    cached, top = np.zeros(nr, int), 0.0
    for new in ([50, 3, 0, 33], [1, 20, 9, 1], [1, 1, 1, 1]):
        n = sum(new)
        plan = backend.page_plan(i32(cached), i32(new), page, free, tables, n)
        q, k, v = (dev(rng.standard_normal((n, h, hd), np.float32)) for h in (nh, kvh, kvh))
        qr, kr = backend.rope(q, k, plan.positions, dev(inv), mscale=m)
        backend.kv8_append(cache, kr, v, plan.slots)
        top = max(top, float(kr.abs().max()), float(v.abs().max()))
        ctx = cached + new
        out = backend.attn_kv8(qr, cache, tables, plan.q_start, plan.ctx_lens, max(new), int(ctx.max()))
        free = free[int(plan.counts[1]):].contiguous()
        at = 0
        for r in range(nr):
            pos = torch.arange(int(ctx[r]), dtype=torch.int32, device="cuda")
            slots = tables[r][(pos // page).long()] * page + pos % page
            ks, vs = (x.double().cpu().numpy() for x in backend.kv8_read(cache, slots.int().contiguous()))
            # what was appended, to half a scale: at most the largest value of any pass / 127
            if new[r]:
                back = backend.kv8_read(cache, plan.slots[at:at + new[r]].contiguous())
                for a, b in zip(back, (kr, v)):
                    assert (a - b[at:at + new[r]]).abs().max() <= 0.501 * top / 127
            for i in range(new[r]):
                p = cached[r] + i
                a = p * inv
                cs, sn = m * np.cos(a), m * np.sin(a)
                for h in range(nh):
                    x = q[at + i, h].double().cpu().numpy()
                    x = np.concatenate([x[:32] * cs - x[32:] * sn, x[:32] * sn + x[32:] * cs])
                    s = ks[:p + 1, h // group] @ x * hd ** -0.5
                    w = np.exp(s - s.max())
                    want = w @ vs[:p + 1, h // group] / w.sum()
                    # rotated q to 1e-6 of its size, scores of size 10 at most, sums of 60 values of size 5
                    assert np.abs(out[at + i, h].double().cpu().numpy() - want).max() <= 1e-4
            at += new[r]
        cached = ctx


def test_captured_pass(backend):
    """Plan, rotary positions, append and attention captured once, with room
    for 40 rows, replayed for passes of other lengths (padded, empty, a
    request that ends): the same bits as eager passes of exact size, in
    outputs and cache."""
    import torch
    rng = np.random.default_rng(19)
    page, kvh, group, hd, nr, room, most, bound = 16, 2, 3, 64, 4, 40, 20, 120
    nh = kvh * group
    inv, m = gq.rope_freqs(hd, 1e4)
    inv = dev(inv)
    order = rng.permutation(32).astype(np.int32)

    class Side:
        def __init__(self):
            self.cache = gq.kv8_cache(32, page, kvh, hd)
            for t in self.cache:
                t.zero_()
            self.tables = torch.full((nr, 8), -1, dtype=torch.int32, device="cuda")
            self.free, self.cached, self.new = i32(order), i32([0] * nr), i32([1] * nr)

        def run(self, q, k, v, rows):
            plan = backend.page_plan(self.cached, self.new, page, self.free, self.tables, rows)
            qr, kr = backend.rope(q, k, plan.positions, inv, mscale=m)
            backend.kv8_append(self.cache, kr, v, plan.slots)
            out = torch.full_like(q, 7.5)
            return plan, backend.attn_kv8(qr, self.cache, self.tables, plan.q_start, plan.ctx_lens, most, bound, out=out)

    a, b = Side(), Side()
    q, k, v = (torch.zeros((room, h, hd), device="cuda") for h in (nh, kvh, kvh))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan, out = a.run(q, k, v, room)
    cached, taken = np.zeros(nr, int), 0
    for new in ([20, 3, 0, 15], [1, 1, 1, 1], [0, 17, 20, 0], [0, 0, 0, 0], [1, 0, 1, 12], [1, 1, 1, 1]):
        n = sum(new)
        for t in (q, k, v):
            t.copy_(dev(rng.standard_normal(tuple(t.shape), np.float32)))
        for side in (a, b):
            side.cached.copy_(i32(cached))
            side.new.copy_(i32(new))
            side.free.copy_(i32(np.roll(order, -taken)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        exact, want = b.run(q[:n].contiguous(), k[:n].contiguous(), v[:n].contiguous(), n)
        assert torch.equal(out[:n], want) and (out[n:] == 7.5).all() and (plan.slots[n:] == -1).all()
        assert torch.equal(plan.slots[:n], exact.slots) and torch.equal(a.tables, b.tables)
        for x, y in zip(a.cache, b.cache):
            assert torch.equal(x, y)
        cached += new
        taken += int(exact.counts[1])
        float(want.sum())


def test_most_requests(backend):
    """65535 requests of one token that see one key, or none: its values."""
    import torch
    n, kvh, hd, page = 65535, 2, 64, 16
    cache = gq.kv8_cache(4, page, kvh, hd)
    x = [torch.randn((4, kvh, hd), device="cuda") for _ in "kv"]
    backend.kv8_append(cache, *x, i32([0, 16, 32, 48]))
    ids = torch.arange(n, device="cuda") % 5  # 4: not a page of the cache
    v = backend.kv8_read(cache, i32([0, 16, 32, 48, -1]))[1]
    out = backend.attn_kv8(torch.randn((n, 2 * kvh, hd), device="cuda"), cache, ids.int().view(n, 1), i32(np.arange(n + 1)),
                           torch.ones(n, dtype=torch.int32, device="cuda"), 1, 1)
    want = v[ids].repeat_interleave(2, 1)
    # one weight w: w c / (w / vs), with exp2's, the parts' and the reciprocal's roundings
    assert ((out - want).abs() <= 2.0**-18 * want.abs()).all() and (out[ids == 4] == 0).all()


def test_refuses_tensors(backend):
    import torch
    c = Case([(20, 2), (3, 1)], 16, 2, 2, 64, "float32")
    cache, (tables, starts, ctx, mn, mc) = c.cache(), c.args()
    good = dict(q=c.q, cache=cache, tables=tables, q_start=starts, ctx_lens=ctx, max_new=mn, max_ctx=mc)
    for bad in (dict(q=c.q.double()), dict(q=c.q[:, :3]), dict(q=c.q[..., :32]), dict(q=c.q.cpu()), dict(tables=tables[:1]),
                dict(tables=tables.long()), dict(tables=tables.t()), dict(q_start=starts[:2]), dict(ctx_lens=ctx.float()),
                dict(ctx_lens=ctx[:1]), dict(out=c.q.half()), dict(out=c.q[:1].clone()), dict(window=-1),
                dict(scale=float("inf")), dict(max_new=-1), dict(cache=cache._replace(k=cache.k[:1]))):
        with pytest.raises((ValueError, gq.GqError)):
            backend.attn_kv8(**{**good, **bad})
    need = gq.lib().gq_attn_kv8_workspace(gq.ctypes.byref(gq._cache(cache, 0)), 4, c.n, 2, 2, 5000)
    assert need
    for ws in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"), torch.empty(need, device="cuda"),
               torch.empty(need, dtype=torch.uint8)):
        with pytest.raises((ValueError, gq.GqError)):
            backend.attn_kv8(**{**good, "max_ctx": 5000}, workspace=ws)
    out = backend.attn_kv8(**{**good, "max_ctx": 5000}, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    want, tol = c.want()
    assert (np.abs(out[:3].double().cpu().numpy() - want[:3]) <= tol[:3]).all()
