"""The paged 8-bit cache's entry points without a GPU: what they refuse,
the rotary frequencies, and the index arithmetic that host and kernels share."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

import gq

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, EDTYPE = -1, -2
P = 1 << 20  # an address that is never read: every call here is refused


def refused(rc, code, text):
    assert rc == code, (rc, gq.lib().gq_last_error())
    msg = gq.lib().gq_last_error().decode()
    assert text in msg, msg


def kv8(n_pages=4, page=16, heads=2, hd=64, k=P, v=P, ks=P, vs=P):
    return ctypes.byref(gq._Kv8(n_pages, page, heads, hd, k, v, ks, vs))


PLAN = dict(cached=P, new=P, n=3, page=16, free=P, n_free=5, tables=P, wide=4, q_start=P, ctx=P, pos=P, slots=P, max_tokens=8,
            counts=P, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(page=8), "page_size 8"), (dict(page=24), "page_size 24"), (dict(page=0), "page_size 0"),
    (dict(page=272), "page_size 272"), (dict(n=-1), "-1 requests"), (dict(n=4097), "at most 4096"),
    (dict(n_free=-1), "negative size"), (dict(wide=-1), "negative size"), (dict(max_tokens=-1), "negative size"),
    (dict(cached=None), "null"), (dict(new=None), "null"), (dict(free=None), "null"), (dict(tables=None), "null"),
    (dict(q_start=None), "null"), (dict(ctx=None), "null"), (dict(pos=None), "null"), (dict(slots=None), "null"),
    (dict(counts=None), "null")])
def test_page_plan_refuses(change, text):
    refused(gq.lib().gq_page_plan(*dict(PLAN, **change).values()), EINVAL, text)


ROPE = dict(dtype=gq.F32, layout=0, n=2, hd=64, rot=64, freq=P, mscale=1.0, pos=P, q=P, qs=128, nq=2, qo=2 * P, qos=128,
            k=3 * P, ks=64, nk=1, ko=4 * P, kos=64, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=12), EDTYPE, "Q4_K"), (dict(dtype=7), EDTYPE, "unknown"), (dict(layout=2), EINVAL, "layout 2"),
    (dict(n=-1), EINVAL, "-1 tokens"), (dict(n=1 << 24), EINVAL, "less than 2^24"), (dict(rot=63), EINVAL, "63 of them"), (dict(rot=66), EINVAL, "66 of them"),
    (dict(rot=0), EINVAL, "0 of them"), (dict(hd=4098), EINVAL, "heads of 4098"), (dict(nq=0), EINVAL, "0 and 1 heads"),
    (dict(qs=127), EINVAL, "stride"), (dict(qos=127), EINVAL, "stride"), (dict(ks=63), EINVAL, "stride"),
    (dict(kos=0), EINVAL, "stride"), (dict(q=None), EINVAL, "null"), (dict(qo=None), EINVAL, "null"),
    (dict(ko=None), EINVAL, "null"), (dict(freq=None), EINVAL, "null"), (dict(pos=None), EINVAL, "null"),
    (dict(qo=P, qos=256), EINVAL, "in place"), (dict(ko=3 * P, kos=128), EINVAL, "in place")])
def test_rope_refuses(change, code, text):
    refused(gq.lib().gq_rope(*dict(ROPE, **change).values()), code, text)


def test_no_tokens_are_no_work():
    """Nothing to do needs no device either."""
    assert gq.lib().gq_rope(*dict(ROPE, n=0).values()) == 0
    assert gq.lib().gq_kv8_append(kv8(), gq.F32, P, 128, P, 128, P, 0, None) == 0
    assert gq.lib().gq_kv8_read(kv8(), P, 0, gq.F32, P, P, None) == 0
    for none in ("n", "nr", "max_new"):
        assert gq.lib().gq_attn_kv8(kv8(), *dict(ATTN, **{none: 0}).values()) == 0


CACHES = [(dict(page=20), "page_size 20"), (dict(page=512), "page_size 512"), (dict(hd=96), "head_dim 96"),
          (dict(heads=0), "0 KV heads"), (dict(heads=65536), "65536 KV heads"), (dict(n_pages=0), "0 pages"),
          (dict(n_pages=1 << 27), "slots"), (dict(n_pages=1 << 20, heads=2048), "scales"), (dict(k=None), "null cache"), (dict(v=None), "null cache"),
          (dict(ks=None), "null cache"), (dict(vs=None), "null cache"), (dict(k=P + 8), "multiple of 16"),
          (dict(v=P + 4), "multiple of 16")]


@pytest.mark.parametrize("change,text", CACHES)
def test_bad_caches_are_refused(change, text):
    c = kv8(**change)
    refused(gq.lib().gq_kv8_append(c, gq.F32, P, 4 << 20, P, 4 << 20, P, 2, None), EINVAL, text)
    refused(gq.lib().gq_kv8_read(c, P, 2, gq.F32, P, P, None), EINVAL, text)
    assert gq.lib().gq_attn_kv8_workspace(c, 4, 8, 2, 4, 64) == 0
    refused(gq.lib().gq_attn_kv8(c, *ATTN.values()), EINVAL, text)


ATTN = dict(dtype=gq.F32, q=P, qs=256, nh=4, n=8, tables=P, wide=4, q_start=P, ctx=P, nr=2, max_new=4, max_ctx=64, scale=0.1,
            window=0, out=2 * P, os=256, ws=P, wb=1 << 30, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=12), EDTYPE, "Q4_K"), (dict(nh=3), EINVAL, "3 heads"), (dict(nh=0), EINVAL, "0 heads"),
    (dict(n=-1), EINVAL, "-1 tokens"), (dict(nr=-1), EINVAL, "-1 requests"), (dict(nr=65536), EINVAL, "at most 65535"),
    (dict(max_new=-1), EINVAL, "max_new -1"), (dict(max_ctx=-1), EINVAL, "max_ctx -1"),
    (dict(max_ctx=2**30 + 1), EINVAL, "at most 2"), (dict(wide=-1), EINVAL, "max_pages -1"),
    (dict(window=-1), EINVAL, "window -1"), (dict(scale=math.inf), EINVAL, "scale"), (dict(scale=math.nan), EINVAL, "scale"),
    (dict(max_new=2**30), EINVAL, "too many rows"), (dict(max_new=2**22), EINVAL, "too many rows"),
    (dict(nr=65535, max_new=2**20), EINVAL, "by keys"), (dict(qs=255), EINVAL, "q: rows"), (dict(os=128), EINVAL, "out: rows"),
    (dict(qs=257), EINVAL, "multiples of 16"), (dict(os=258), EINVAL, "multiples of 16"), (dict(q=P + 4), EINVAL, "multiples of 16"),
    (dict(out=P + 8), EINVAL, "multiples of 16"), (dict(q=None), EINVAL, "null q"), (dict(out=None), EINVAL, "null out"),
    (dict(tables=None), EINVAL, "null"), (dict(q_start=None), EINVAL, "null"), (dict(ctx=None), EINVAL, "null"),
    (dict(max_ctx=9000, ws=None), -3, "have 0"), (dict(max_ctx=9000, wb=15), -3, "have 15"),
    (dict(ws=P + 8), EINVAL, "workspace must start")])
def test_attention_refuses(change, code, text):
    refused(gq.lib().gq_attn_kv8(kv8(), *dict(ATTN, **change).values()), code, text)


@pytest.mark.parametrize("dtype,k,ks,v,vs,slots,n,code,text", [
    (8, P, 128, P, 128, P, 2, EDTYPE, "Q8_0"), (gq.F32, P, 127, P, 128, P, 2, EINVAL, "k: rows"),
    (gq.F32, P, 128, P, 64, P, 2, EINVAL, "v: rows"), (gq.F32, P, 129, P, 128, P, 2, EINVAL, "multiples of 16"),
    (gq.BF16, P, 132, P, 128, P, 2, EINVAL, "multiples of 16"), (gq.F32, P + 4, 128, P, 128, P, 2, EINVAL, "multiples of 16"),
    (gq.F16, P, 128, P + 8, 128, P, 2, EINVAL, "multiples of 16"), (gq.F32, None, 128, P, 128, P, 2, EINVAL, "null k"),
    (gq.F32, P, 128, None, 128, P, 2, EINVAL, "null v"), (gq.F32, P, 128, P, 128, None, 2, EINVAL, "null slots"),
    (gq.F32, P, 128, P, 128, P, -1, EINVAL, "negative"), (gq.F32, P, 128, P, 128, P, 1 << 27, EINVAL, "in one call")])
def test_append_refuses(dtype, k, ks, v, vs, slots, n, code, text):
    refused(gq.lib().gq_kv8_append(kv8(), dtype, k, ks, v, vs, slots, n, None), code, text)


def test_read_refuses():
    refused(gq.lib().gq_kv8_read(kv8(), P, 2, 14, P, P, None), EDTYPE, "Q6_K")
    refused(gq.lib().gq_kv8_read(kv8(), P, -2, gq.F32, P, P, None), EINVAL, "-2 tokens")
    refused(gq.lib().gq_kv8_read(kv8(), None, 2, gq.F32, P, P, None), EINVAL, "null slots")
    refused(gq.lib().gq_kv8_read(kv8(), P, 2, gq.F32, P + 4, P, None), EINVAL, "multiples of 16")
    refused(gq.lib().gq_kv8_read(kv8(heads=65535, hd=128, n_pages=1), P, 1 << 30, gq.F32, P, P, None), EINVAL, "in one call")
    refused(gq.lib().gq_kv8_read(kv8(heads=2, hd=64), P, 1 << 27, gq.F32, P, P, None), EINVAL, "in one call")


# ------------------------------------------------------ rotary frequencies
def freqs(rot, theta, scaling="none", factor=1.0, orig=8192.0, fast=32.0, slow=1.0, low=1.0, high=4.0):
    """The definition, one pair at a time."""
    out = []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            turns = orig * f / (2 * math.pi)
            if turns < low:
                f /= factor
            elif turns < high:
                mix = (turns - low) / (high - low)
                f = (1 - mix) * f / factor + mix * f
        elif scaling == "yarn":
            a, b = (rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (fast, slow))
            a, b = max(math.floor(a), 0), min(math.ceil(b), rot - 1)
            r = min(1.0, max(0.0, (i - a) / max(b - a, 1e-3)))
            f = f / factor * r + f * (1 - r)
        out.append(f)
    return np.array(out)


@pytest.mark.parametrize("rot,theta", [(128, 1e6), (64, 1e4), (48, 5e5), (2, 1e4)])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("yarn", 4.0), ("yarn", 40.0), ("llama3", 8.0)])
def test_rope_freqs(rot, theta, scaling, factor):
    got, m = gq.rope_freqs(rot, theta, scaling, factor, orig_ctx=8192)
    np.testing.assert_allclose(got, freqs(rot, theta, scaling, factor), rtol=1e-13)
    assert m == np.float32(0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0)


def test_rope_freqs_factors_and_attn_factor():
    ff = np.linspace(1, 3, 32).astype(np.float32)
    got, m = gq.rope_freqs(64, 1e4, "linear", 2.0, freq_factors=ff, attn_factor=1.5)
    np.testing.assert_allclose(got, freqs(64, 1e4, "linear", 2.0) / ff.astype(np.float64), rtol=1e-13)
    assert m == 1.5


@pytest.mark.parametrize("kw,text", [
    (dict(rot_dim=63), "rot_dim 63"), (dict(rot_dim=0), "rot_dim 0"), (dict(theta=1.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(attn_factor=0.0), "attn_factor"),
    (dict(scaling="linear", factor=0.5), "factor 0.5"), (dict(scaling="yarn", factor=2.0), "orig_ctx"),
    (dict(scaling="yarn", factor=2.0, orig_ctx=4096, beta_fast=1.0), "betas"),
    (dict(scaling="llama3", factor=2.0, orig_ctx=4096, low_freq=4.0), "low_freq"),
    (dict(freq_factors=[1.0] * 31 + [0.0]), "factor 31")])
def test_rope_freqs_refuses(kw, text):
    with pytest.raises(gq.GqError, match=text):
        gq.rope_freqs(**{"rot_dim": 64, **kw})


def test_rope_freqs_refuses_in_python():
    with pytest.raises(ValueError, match="scaling"):
        gq.rope_freqs(64, scaling="ntk")
    with pytest.raises(ValueError, match="rot_dim / 2"):
        gq.rope_freqs(64, freq_factors=[1.0] * 31)


# --------------------------------------------------------- shared indexes
@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = tmp_path_factory.mktemp("paged") / "paged"
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-Xlinker", "--no-undefined",
                        "-I", os.path.join(ROOT, "agention-infer_amd", "csrc"),
                        os.path.join(ROOT, "tests", "cpp", "paged.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(lines):
        r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60)
        assert r.returncode == 0
        out = [[int(v) for v in line.split()] for line in r.stdout.splitlines()]
        assert len(out) == len(lines)
        return out
    return run


def test_counts_and_slots(ask):
    top = 2**31 - 1
    q = [(f"add {a} {b}", min(a + b, top)) for a in (0, 5, top - 1, top) for b in (0, 1, top)]
    q += [(f"pages {t} {p} {w}", min(-(-t // p), w)) for t in (0, 1, 16, 17, top) for p in (16, 48, 256) for w in (0, 1, top)]
    q += [(f"slot {i} {p} {o}", -1 if i < 0 or i * p + o > top else i * p + o)
          for i in (-2**31, -1, 0, 3, 2**23 - 1, 2**27 - 1, 2**27, top) for p in (16, 256) for o in (0, 15)]
    assert [r[0] for r in ask([a for a, _ in q])] == [b for _, b in q]


def test_owner(ask):
    """The request of every token, requests without tokens among them."""
    rng = np.random.default_rng(3)
    lines, want = [], []
    for n in (1, 2, 3, 7, 33):
        sizes = rng.integers(0, 4, n)
        sizes[rng.integers(0, n)] += 1
        at = np.concatenate([[0], np.cumsum(sizes)])
        for v in range(at[-1]):
            lines.append(f"owner {n} {v} " + " ".join(map(str, at)))
            want.append(int(np.searchsorted(at[1:], v, side="right")))
    assert [r[0] for r in ask(lines)] == want


def test_attention_rows_and_keys_stay_inside(ask):
    """Whatever the device's lengths hold: rows within the pass, keys within
    the table and the bound; sane lengths give the request's own."""
    rng = np.random.default_rng(2)
    wild = [-2**31, -5, 0, 3, 40, 2**31 - 1]
    cases = [(int(rng.choice(wild)), int(rng.choice(wild)), int(rng.choice(wild)), int(rng.choice([0, 1, 9, 2**31 - 1])),
              int(rng.choice([0, 1, 7, 2**23])), int(rng.choice([16, 48, 256])), int(rng.choice([0, 5, 700, 2**31 - 1])))
             for _ in range(400)]
    for (s, e, ctx, n, wide, page, most), (start, fresh, first, keys) in zip(
            cases, ask(["req " + " ".join(map(str, c)) for c in cases])):
        assert 0 <= start <= n and fresh >= 0 and start + fresh <= n
        assert 0 <= keys <= min(wide * page, most, max(ctx, 0)) and first == max(ctx, 0) - fresh
    assert ask(["req 4 9 30 20 9 16 64", "req 4 9 30 20 1 16 64", "req 4 9 30 20 9 16 25"]) == [
        [4, 5, 25, 30], [4, 5, 25, 16], [4, 5, 25, 25]]


def test_attention_keys(ask):
    """Against the definition: the keys of every row of a tile are within its
    [lo, hi), which holds no chunk in front of the first of them."""
    rng = np.random.default_rng(3)
    cases = []
    for _ in range(400):
        fresh, first = int(rng.integers(1, 40)), int(rng.integers(-20, 500))
        keys = int(rng.integers(0, max(1, first + fresh + 1)))
        i0 = int(rng.integers(0, fresh))
        cases.append((fresh, first, keys, i0, int(rng.integers(i0, fresh)), int(rng.choice([0, 1, 17, 64, 300])),
                      int(rng.choice([256, 512]))))
    for (fresh, first, keys, i0, i1, window, split), (lo, hi, parts) in zip(
            cases, ask(["keys " + " ".join(map(str, c)) for c in cases])):
        seen = [k for i in range(i0, i1 + 1) for k in range(max(0, first + i - window + 1 if window else 0),
                                                            min(keys, first + i + 1))]
        assert lo % 64 == 0 and lo >= 0 and hi <= keys
        assert parts == max(1, -(-(hi - lo) // split))
        if seen:
            assert lo <= min(seen) < lo + 64 and hi == max(seen) + 1
    big = 2**31 - 1
    assert ask([f"keys 1 {big - 1} {big} 0 0 0 {1 << 30}", f"keys 1 {big - 1} {big} 0 0 {big} 256",
                f"keys 3 -3 0 0 2 {big} 256"]) == [[0, big, 2], [0, big, 8388608], [0, 0, 1]]


def test_attention_cut(ask):
    """Every row has a tile and every key a part, whatever the sizes."""
    cases = [(n, r, kv, g, m, c) for n in (1, 700, 2**31 - 1) for r in (1, 3, 64, 65535) for kv in (1, 8) for g in (1, 7, 71)
             for m in (1, 5, 2048) for c in (0, 1, 255, 4097, 131072, 2**31 - 1)]
    for (n, r, kv, g, m, c), (most, rtiles, split, rparts, ttiles, tsplit, tparts, parts) in zip(
            cases, ask(["cut " + " ".join(map(str, x)) for x in cases])):
        few = min(m * g, most)
        assert (most == 64 or m * g > 64 and r == 1 and most == 0) and 16 * rtiles >= few > 16 * (rtiles - 1)
        if few:
            assert split % 64 == 0 and split > 0 and rparts >= 1 and rparts * split >= c and (rparts - 1) * split < max(c, 1)
        else:
            assert rparts == 0
        if m * g > 64:
            assert 256 * ttiles >= m * g > 256 * (ttiles - 1)
            assert tsplit % 64 == 0 and tsplit > 0 and tparts * tsplit >= c and (tparts - 1) * tsplit < max(c, 1)
        else:
            assert ttiles == tparts == 0
        assert parts == max(rparts, tparts)
        if few and c <= 2**30:  # and what parts add to the workspace and the grid is bounded
            blocks = r * kv * rtiles
            assert rparts <= max(1, 8192 // blocks, -(-512 // blocks))
