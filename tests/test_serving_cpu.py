"""The serving operators' refusals and host-only parts: no device call is made here."""
import ctypes as C
import math
import os

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "jasmine_amd", "libjasmine_hip.so")), reason="library not built")

P = 0x10000  # an aligned address that nothing here reads


@pytest.fixture(scope="module")
def capi():
    import jasmine_amd.capi as capi
    return capi


def refused(capi, rc, word, code=1):
    assert rc == code, (rc, capi.lib.jas_last_error())
    assert word in capi.lib.jas_last_error().decode(), capi.lib.jas_last_error()


def cache(capi, **kw):
    v = dict(d_k=P, d_v=P, d_k_scale=None, d_v_scale=None, d_table=P, page_stride=8 * 16 * 64, head_stride=16 * 64, tok_stride=64,
             table_stride=4, max_pages=4, dtype=capi.JAS_F32, n_pages=8, page_size=16, n_kv=8, dh=64)
    v.update(kw)
    return C.byref(capi.PagedKv(**v))


BAD_CACHES = [
    (dict(d_k=None), "null"), (dict(d_table=None), "null"), (dict(dtype=1), "holds"), (dict(dtype=9), "holds"),
    (dict(dtype=4), "scales"), (dict(dtype=5, d_k_scale=P), "scales"), (dict(dh=48), "dh"), (dict(dh=256), "dh"),
    (dict(n_pages=0), "positive"), (dict(page_size=0), "positive"), (dict(n_kv=-1), "positive"), (dict(max_pages=0), "positive"),
    (dict(table_stride=-1), "negative"), (dict(page_size=(1 << 20) + 1), "2^20"), (dict(tok_stride=32), "dh apart"),
    (dict(page_stride=-64), "negative"), (dict(d_v=P + 8), "16 bytes"), (dict(tok_stride=65), "16 bytes"),
    (dict(dtype=3, head_stride=68), "16 bytes"), (dict(d_table=P + 2), "4 bytes"),
]


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_cache_refused(capi, kw, word):
    lib, kv = capi.lib, cache(capi, **kw)
    refused(capi, lib.jas_kv_append(kv, P, P, 1, 512, 64, 1, P, P, 0, None), word)
    refused(capi, lib.jas_kv_read(kv, P, P, 1, 512, 64, 1, P, P, 0, None), word)
    refused(capi, lib.jas_attn_paged(P, P, kv, 1, 1, P, P, 8, 1, 16, 512, 64, 512, 64, 1.0, 1, 0, P, None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "negative"), (dict(B=-1), "negative"), (dict(cu=None), "null"), (dict(lens=None), "null"), (dict(cu=P + 1), "4 bytes"),
    (dict(dtype=1), "rows are"), (dict(dtype=4), "rows are"), (dict(k=P + 2), "aligned")])
def test_kv_rows_refused(capi, kw, word):
    v = dict(k=P, v=P, n=1, B=1, cu=P, lens=P, dtype=0)
    v.update(kw)
    for f in (capi.lib.jas_kv_append, capi.lib.jas_kv_read):
        refused(capi, f(cache(capi), v["k"], v["v"], v["n"], 512, 64, v["B"], v["cu"], v["lens"], v["dtype"], None), word)


def test_kv_null_rows(capi):
    refused(capi, capi.lib.jas_kv_append(cache(capi), P, None, 1, 512, 64, 1, P, P, 0, None), "null")
    # reading neither, and nothing to do, are no errors
    assert capi.lib.jas_kv_read(cache(capi), None, None, 1, 512, 64, 1, P, P, 0, None) == 0
    assert capi.lib.jas_kv_append(cache(capi), P, P, 0, 512, 64, 1, P, P, 0, None) == 0
    assert capi.lib.jas_kv_append(cache(capi), P, P, 4, 512, 64, 0, None, None, 0, None) == 0


@pytest.mark.parametrize("kw,word,code", [
    (dict(q=None), "null", 1), (dict(o=None), "null", 1), (dict(o=P), "overlap", 1), (dict(work=P + 8), "16 bytes", 1),
    (dict(work=None, max_len=100000), "workspace", 1), (dict(dtype=1), "rows are", 1), (dict(dtype=3), "over a JAS_F32 cache", 1),
    (dict(H=12), "multiple", 1), (dict(H=0), "multiple", 1), (dict(max_q=-1), "max_q", 1), (dict(max_len=-1), "max_q", 1),
    (dict(q=P + 2), "aligned", 1), (dict(n=1 << 28, H=16), "too many", 5)])
def test_attention_refused(capi, kw, word, code):
    v = dict(q=P, o=P + 4096, n=1, H=8, max_q=1, max_len=16, dtype=0, work=P)
    v.update(kw)
    refused(capi, capi.lib.jas_attn_paged(v["q"], v["o"], cache(capi), v["n"], 1, P, P, v["H"], v["max_q"], v["max_len"], 512, 64, 512, 64,
                                          1.0, 1, v["dtype"], v["work"], None), word, code)


def test_attention_nothing_to_do(capi):
    args = (8, 1, 16, 512, 64, 512, 64, 1.0, 1, 0, None, None)
    assert capi.lib.jas_attn_paged(P, P + 4096, cache(capi), 0, 1, P, P, *args) == 0
    assert capi.lib.jas_attn_paged(P, P + 4096, cache(capi), 3, 0, None, None, *args) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(x=None), "null"), (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(n=-1), "need n"), (dict(nh=0), "need n"),
    (dict(rot=3), "even rot"), (dict(rot=66), "even rot"), (dict(rot=-2), "even rot"), (dict(dtype=1), "dtype"), (dict(layout=2), "layout"),
    (dict(y=P, y_st=64), "same strides"), (dict(x=P + 2), "aligned"), (dict(freq=P + 4), "aligned")])
def test_rope_refused(capi, kw, word):
    v = dict(x=P, y=P + 4096, pos=P, freq=P, n=1, nh=2, dh=64, rot=64, x_st=128, x_sh=64, y_st=128, y_sh=64, layout=0, dtype=0)
    v.update(kw)
    refused(capi, capi.lib.jas_rope(v["x"], v["y"], v["pos"], v["freq"], v["n"], v["nh"], v["dh"], v["rot"], v["x_st"], v["x_sh"], v["y_st"],
                                    v["y_sh"], v["layout"], 1.0, v["dtype"], None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(x=None), "null"), (dict(u=None), "null"), (dict(ids=None), "null"), (dict(n=-1), "need n"), (dict(V=0), "need n"),
    (dict(V=(1 << 22) + 1), "need n"), (dict(ld=9), "need n"), (dict(dtype=1), "logits are"), (dict(x=P + 2), "aligned"),
    (dict(u=P + 2), "aligned"), (dict(n=65536), "65535"), (dict(work=None), "workspace"), (dict(work=P + 4), "workspace")])
def test_sample_refused(capi, kw, word):
    v = dict(x=P, n=1, V=10, ld=10, u=P, ids=P, dtype=0, work=P)
    v.update(kw)
    if v["V"] > 10:
        v["ld"] = v["V"]
    refused(capi, capi.lib.jas_sample(v["x"], v["n"], v["V"], v["ld"], P, P, P, P, v["u"], v["ids"], P, v["dtype"], v["work"], None), word)


def test_workspaces(capi):
    """0 for what the calls refuse or return from at once, and no less for larger bounds."""
    f, g = capi.lib.jas_attn_paged_workspace, capi.lib.jas_sample_workspace
    assert f(0, 1, 8, 8, 64, 1, 16) == f(4, 0, 8, 8, 64, 1, 16) == f(4, 1, 8, 3, 64, 1, 16) == f(4, 1, 8, 8, 64, -1, 16) == 0
    assert f(4, 4, 32, 8, 128, 1, 1 << 20) > 0 and g(0, 100) == g(1, 0) == g(1, (1 << 22) + 1) == 0
    assert all(g(n, V) >= n * 8 for n in (1, 7, 3000) for V in (1, 5000, 1 << 22))


def test_workspace_of_a_larger_call(capi):
    """Bytes for given numbers are enough for smaller ones: they never fall as a number grows."""
    rng = np.random.default_rng(3)
    upto = lambda hi: int(np.exp(rng.uniform(0, np.log(hi))))  # noqa: E731
    for _ in range(3000):
        n, B, max_q, max_len, V = upto(20000), upto(3000), upto(2000), upto(300000), upto(1 << 22)
        g, kv = int(rng.choice([1, 2, 4, 7, 16])), int(rng.choice([1, 2, 8, 12, 32]))
        less = [upto(v) for v in (n, B, max_q, max_len)]
        f = capi.lib.jas_attn_paged_workspace
        assert f(less[0], less[1], g * kv, kv, 64, less[2], less[3]) <= f(n, B, g * kv, kv, 64, max_q, max_len)
        assert capi.lib.jas_sample_workspace(less[0], upto(V)) <= capi.lib.jas_sample_workspace(n, V)


@pytest.mark.parametrize("n,B,H,n_kv,max_q", [(512, 512, 64, 8, 1), (4, 4, 32, 8, 1), (1 << 20, 1 << 20, 64, 64, 1), (5, 1, 8, 8, 5), (64, 2, 32, 8, 32)])
def test_workspace_of_any_bound(capi, n, B, H, n_kv, max_q):
    """max_len only bounds: the largest one is as good as another, and 63 parts of a row are the most."""
    for max_len in (0, 1, 4096, 1 << 24, 1 << 30, 2 ** 31 - 1):
        size = capi.lib.jas_attn_paged_workspace(n, B, H, n_kv, 64, max_q, max_len)
        assert 0 <= size <= (n * (H // n_kv) + 128 * B) * n_kv * 63 * (64 + 4) * 4


def test_launches_that_would_not_fit(capi):
    """2^32 threads or more in one launch are refused before it."""
    big = 2 ** 31 - 1
    refused(capi, capi.lib.jas_rope(P, P, P, P, big, 64, 64, 64, 4096, 64, 4096, 64, 0, 1.0, 0, None), "too many", 5)
    for f in (capi.lib.jas_kv_append, capi.lib.jas_kv_read):
        refused(capi, f(cache(capi), P, P, big, 512, 64, 1, P, P, 0, None), "too many", 5)
    refused(capi, capi.lib.jas_attn_paged(P, P + 4096, cache(capi), 1 << 20, 1 << 23, P, P, 8, 1, 16, 512, 64, 512, 64, 1.0, 1, 0, P, None), "too many", 5)


# ---------------------------------------------------------------- frequencies
def freqs(capi, *a, **kw):
    return capi.rope_freqs(*a, **kw)


@pytest.mark.parametrize("rot,theta", [(2, 10000.0), (64, 10000.0), (128, 500000.0)])
def test_freqs_plain_and_linear(capi, rot, theta):
    want = theta ** (-2.0 * np.arange(rot // 2) / rot)
    f, m = freqs(capi, rot, theta)
    # one power of two numbers that are exact: a few steps of 2^-53
    assert m == 1.0 and np.all(np.abs(f - want) <= 8 * 2.0 ** -53 * want)
    f, m = freqs(capi, rot, theta, capi.RopeScaling(capi.ROPE_SCALE_LINEAR, 0, 4.0, 0.0, 0.0))
    assert m == 1.0 and np.all(np.abs(f - want / 4) <= 8 * 2.0 ** -53 * want)


def test_freqs_yarn(capi):
    rot, theta, orig, factor, low, high = 64, 10000.0, 2048, 8.0, 1.0, 32.0
    f, m = freqs(capi, rot, theta, capi.RopeScaling(capi.ROPE_SCALE_YARN, orig, factor, low, high))
    base = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    turns = [orig * b / (2 * math.pi) for b in base]
    # pairs beyond either end of the ramp keep their frequency, or have it divided; between them it falls
    first = math.floor(rot * math.log(orig / (high * 2 * math.pi)) / (2 * math.log(theta)))
    last = math.ceil(rot * math.log(orig / (low * 2 * math.pi)) / (2 * math.log(theta)))
    assert turns[first] >= high > turns[first + 1] and turns[last - 1] > low >= turns[last]
    for i, b in enumerate(base):
        t = min(max((i - first) / (last - first), 0.0), 1.0)
        assert abs(f[i] - (b / factor * t + b * (1 - t))) <= 16 * 2.0 ** -53 * b
    assert f[0] == base[0] and m == np.float32(0.1 * math.log(factor) + 1.0)
    assert freqs(capi, rot, theta, capi.RopeScaling(capi.ROPE_SCALE_YARN, orig, 1.0, low, high))[1] == 1.0


def test_freqs_bands(capi):
    rot, theta, orig, factor, low, high = 128, 500000.0, 8192, 8.0, 1.0, 4.0
    f, m = freqs(capi, rot, theta, capi.RopeScaling(capi.ROPE_SCALE_BANDS, orig, factor, low, high))
    seen = set()
    for i in range(rot // 2):
        b = theta ** (-2.0 * i / rot)
        turns = orig * b / (2 * math.pi)
        kind = 0 if turns < low else 2 if turns > high else 1
        seen.add(kind)
        t = (turns - low) / (high - low)
        want = [b / factor, b * t + b / factor * (1 - t), b][kind]
        assert abs(f[i] - want) <= 32 * 2.0 ** -53 * b  # (t's own roundings count (1 - 1 / factor) / (high - low) times)
    assert seen == {0, 1, 2} and m == 1.0


@pytest.mark.parametrize("rot,theta,sc,word", [
    (3, 1e4, None, "even rot"), (0, 1e4, None, "even rot"), (4, 1.0, None, "theta"), (4, math.inf, None, "theta"),
    (4, 1e4, (7, 0, 1.0, 0.0, 0.0), "unknown scaling"), (4, 1e4, (1, 0, 0.0, 0.0, 0.0), "factor"), (4, 1e4, (1, 0, math.nan, 0.0, 0.0), "factor"),
    (4, 1e4, (2, 0, 2.0, 1.0, 32.0), "orig_ctx"), (4, 1e4, (3, 64, 2.0, 4.0, 4.0), "low < high"), (4, 1e4, (2, 64, 2.0, 0.0, 4.0), "low < high")])
def test_freqs_refused(capi, rot, theta, sc, word):
    out = (C.c_double * 8)()
    refused(capi, capi.lib.jas_rope_freqs(rot, theta, C.byref(capi.RopeScaling(*sc)) if sc else None, out, None), word)
    refused(capi, capi.lib.jas_rope_freqs(4, 1e4, None, None, None), "output")


# ---------------------------------------------------------------- the arithmetic behind the kernels
def test_page_division():
    """t / page_size by a product, as the kernels form it, over the ends of its range."""
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 8, 15, 16, 17, 20, 64, 100, 127, 128, 255, 256, 1000, 4095, 65535, 65537, (1 << 20) - 1, 1 << 20]:
        l = 0
        while (1 << l) < d:
            l += 1
        m = ((((1 << l) - d) << 32) // d + 1) & 0xFFFFFFFF
        t = np.unique(np.concatenate([np.arange(0, 3 * d, max(1, d // 7)), rng.integers(0, 2 ** 31, 5000),
                                      np.arange(1, 50) * d, np.arange(1, 50) * d - 1, [0, 2 ** 31 - 1, (2 ** 31 - 1) // d * d]])).astype(np.uint64)
        t = t[t < 2 ** 31]
        up = (t * np.uint64(m)) >> np.uint64(32)
        assert np.all(up + t < 2 ** 32) and np.all((up + t) >> np.uint64(l) == t // np.uint64(d)), d


def test_quotient_to_odd():
    """Rounding the quotient to odd in fp32 and then to the 8-bit type is rounding it once: rows of
    bf16 values, whose quotients by their largest often lie next to a tie."""
    from fractions import Fraction
    rng = np.random.default_rng(1)

    def fma(a, b, c):  # fp32, one rounding
        v = Fraction(float(a)) * Fraction(float(b)) + Fraction(float(c))
        d = np.float64(v.numerator / v.denominator)  # (to nearest in 53 bits; the cases here need fewer, or are far from a tie)
        return np.float32(d)

    for qmax in (127.0, 448.0):
        for _ in range(300):
            top = np.float32(rng.integers(128, 256) * 2.0 ** float(rng.integers(-8, 8)))
            x = np.float32(np.float64(rng.integers(128, 256)) * 2.0 ** float(np.floor(np.log2(top)) - 7 - rng.integers(0, 6)))
            x = np.float32(min(x, top) * (1 if rng.random() < .5 else -1))
            s = np.float32(top / np.float32(qmax))
            inv = np.float32(1) / s
            t0 = np.float32(x * inv)
            t = fma(fma(-t0, s, x), inv, t0)
            r = fma(-t, s, x)
            u = int(t.view(np.uint32))
            if r != 0:
                if (int(r.view(np.uint32)) ^ u) >> 31:
                    u -= 1
                u |= 1
            odd = float(np.uint32(u).view(np.float32))
            exact = Fraction(float(x)) / Fraction(float(s))
            if qmax == 127.0:
                assert np.rint(odd) == round(exact)
            else:
                e = max(math.frexp(odd)[1] - 4, -9)
                assert np.rint(odd / 2.0 ** e) == round(exact / Fraction(2) ** e)
