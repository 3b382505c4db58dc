"""Rotary positions, the paged cache, attention over it and sampling on the GPU, against plain
64-bit forms (serving_ref.py).

Tolerances.  A rounding is half a step: 2^-24 of the value in fp32, 2^-8 in bf16 (u below).
 rope       an angle's fp32 part (at most pi / 4, 2^-24 of it), two steps each of cos and sin, mscale's
            product, then two products and a sum: (|a| + |b|) mscale 2^-24 (0.8 + 4 + 1 + 2), and u |y|
 kv         exact: codes are rounded once, and the reference forms code * scale in fp32 as well
 attention  a score is off by ds = (D + 8) 2^-24 sum |q||k| scale (sums in any order; split products
            lose less than one step of each), a weight by 2 ds and exponentials' 2^-22, sums over L keys
            and at most 64 partial results by (L / 8 + 64) 2^-24 (matrix instructions add 32
            products at a time); bf16: weights rounded by 2^-8, and the result by 2^-8 |o|
 sample     ids equal; logp: 64-bit sums of weights rounded to 2^-shift, then 2^-24
"""
import math

import numpy as np
import pytest

import serving_ref as R
from serving_ref import BF16, F32, F8, I8
from split_model import ATTENTION_BOUND

pytestmark = pytest.mark.gpu


_held = []


@pytest.fixture(autouse=True)
def drop():
    """Buffers that a test names only in a call live until it ends, and the work on them."""
    yield
    if _held:
        import jasmine_amd
        jasmine_amd.check(jasmine_amd.lib.jas_synchronize(None))
    _held.clear()


def hold(a):
    _held.append(a)
    return a.p


def put(jas, x, dtype):
    return jas.to_device(R.to_bf16(x) if dtype == BF16 else np.ascontiguousarray(x, np.float32))


def rounded(x, dtype):
    return R.from_bf16(R.to_bf16(x)).astype(np.float32) if dtype == BF16 else np.ascontiguousarray(x, np.float32)


def got(a, dtype):
    return R.from_bf16(a.numpy()) if dtype == BF16 else a.numpy()


def empty(jas, shape, dtype, fill=7.0):
    return put(jas, np.full(shape, fill, np.float32), dtype)


def within(a, want, tol):
    a = a.astype(np.float64)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(a), nan)
    bad = ~nan & (np.abs(a - want) > tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], a[bad][:4], want[bad][:4], np.broadcast_to(tol, a.shape)[bad][:4])


# ---------------------------------------------------------------- rope
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("n,nh,dh,rot,pad", [(1, 1, 32, 32, 0), (5, 3, 64, 64, 0), (7, 9, 128, 64, 8), (3, 5, 128, 34, 0), (4, 6, 64, 32, 3),
                                             (2, 4, 32, 0, 0), (300, 5, 128, 128, 16), (3, 2, 10, 6, 0)])
def test_rope(jas, dtype, halves, n, nh, dh, rot, pad):
    rng = np.random.default_rng(n * 7 + rot)
    st, sh = nh * (dh + pad) + pad, dh + pad
    x = rounded(rng.standard_normal((n, st)), dtype)
    rows = np.lib.stride_tricks.as_strided(x, (n, nh, dh), (4 * st, 4 * sh, 4))
    pos = rng.integers(0, 200000, n).astype(np.int32)
    pos[0] = 0
    freq = 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    m = 1.25
    want = R.rope(rows, pos, freq, m, rot, halves)
    d_x, d_y = put(jas, x, dtype), empty(jas, (n, nh, dh), dtype)
    d_pos, d_f = jas.to_device(pos), jas.to_device(freq if rot else np.zeros(1))
    jas.check(jas.lib.jas_rope(d_x.p, d_y.p, d_pos.p, d_f.p, n, nh, dh, rot, st, sh, nh * dh, dh, halves, m, dtype, None))
    y = got(d_y, dtype)
    u = 2.0 ** -8 if dtype == BF16 else 0.0
    a = np.abs(rows).astype(np.float64)
    i = np.arange(rot // 2) if halves else np.arange(0, rot, 2)
    j = i + (rot // 2 if halves else 1)
    tol = np.zeros((n, nh, dh))
    tol[..., i] = tol[..., j] = (a[..., i] + a[..., j]) * m * 2.0 ** -24 * 7.8
    within(y, want, tol + u * np.abs(want))
    assert np.array_equal(y[..., rot:], rows[..., rot:])
    # in place, and what lies between the rows stays
    jas.check(jas.lib.jas_rope(d_x.p, d_x.p, d_pos.p, d_f.p, n, nh, dh, rot, st, sh, st, sh, halves, m, dtype, None))
    z = got(d_x, dtype)
    inner = np.lib.stride_tricks.as_strided(z, (n, nh, dh), (4 * st, 4 * sh, 4))
    assert np.array_equal(inner, y)
    mask = np.ones((n, st), bool)
    np.lib.stride_tricks.as_strided(mask, (n, nh, dh), (st, sh, 1))[:] = False
    assert np.array_equal(z[mask], x[mask])


def test_rope_far_positions(jas):
    """Angles of positions near 2^31 keep their places (formed in 64 bits: 2^31 turns, 2^-52 of them)."""
    dh = 64
    freq = 10000.0 ** (-2.0 * np.arange(dh // 2) / dh)
    pos = np.array([2 ** 31 - 1, 2 ** 30 + 12345, -5], np.int32)
    x = np.random.default_rng(0).standard_normal((3, 1, dh)).astype(np.float32)
    import decimal
    decimal.getcontext().prec = 60
    two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    turn = np.array([[float((decimal.Decimal(int(p)) * decimal.Decimal(float(f))) % two_pi) for f in freq] for p in pos])
    z = (x[:, 0, 0::2] + 1j * x[:, 0, 1::2]) * np.exp(1j * turn)
    d_y = empty(jas, x.shape, F32)
    jas.check(jas.lib.jas_rope(hold(jas.to_device(x)), d_y.p, hold(jas.to_device(pos)), hold(jas.to_device(freq)), 3, 1, dh, dh, dh, dh, dh, dh, 0, 1.0, F32, None))
    y = d_y.numpy()[:, 0]
    tol = (np.abs(x[:, 0, 0::2]) + np.abs(x[:, 0, 1::2])) * (2.0 ** -24 * 7.8 + 2.0 ** 31 * 2 * np.pi * 2.0 ** -51)
    within(y[:, 0::2], z.real, tol)
    within(y[:, 1::2], z.imag, tol)


def test_rope_equals_llama_entry(jas):
    """Pairs over the whole head, unscaled: what jas_rope_llama computes (its own roundings apart)."""
    n, nh, dh = 9, 4, 64
    x = np.random.default_rng(2).standard_normal((n, nh, dh)).astype(np.float32)
    pos = np.arange(n, dtype=np.int32) * 97
    f, _ = jas.rope_freqs(dh, 10000.0)
    a, y = jas.to_device(x), empty(jas, x.shape, F32)
    d_pos, d_f = jas.to_device(pos), jas.to_device(f)
    jas.check(jas.lib.jas_rope(a.p, y.p, d_pos.p, d_f.p, n, nh, dh, dh, nh * dh, dh, nh * dh, dh, 0, 1.0, F32, None))
    jas.check(jas.lib.jas_rope_llama(a.p, d_pos.p, n, nh, dh, nh * dh, 10000.0, None))
    s = np.abs(x[..., 0::2]) + np.abs(x[..., 1::2])
    within(y.numpy(), a.numpy().astype(np.float64), np.repeat(s, 2, -1) * 2.0 ** -24 * 9)


# ---------------------------------------------------------------- cache
def batch(rng, news, lens, page, spare=3, width=None, shuffle=True):
    """cu, lens and a table whose rows name pages of their own, in any order."""
    need = [-(-max(v, 0) // page) for v in lens]
    width = width or max(max(need), 1)
    pages = sum(need) + spare
    order = rng.permutation(pages) if shuffle else np.arange(pages)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32), np.array(lens, np.int32), table, pages


BATCHES = [
    ([1], [1], 16), ([1, 1, 1], [5, 1, 33], 16), ([3, 0, 5], [3, 7, 29], 8), ([2, 1, 17], [40, 1, 17], 20), ([7, 64], [100, 64], 1),
    ([33, 2, 1, 1], [64, 130, 65, 1], 64),
]


@pytest.mark.parametrize("news,lens,page", BATCHES)
@pytest.mark.parametrize("cache", [F32, BF16, I8, F8])
@pytest.mark.parametrize("dtype,dh,heads,token_major,pad", [(F32, 64, 3, False, 0), (BF16, 128, 2, True, 1), (F32, 32, 1, True, 0), (BF16, 32, 5, False, 2)])
def test_kv_append_read(jas, news, lens, page, cache, dtype, dh, heads, token_major, pad):
    rng = np.random.default_rng(len(news) + page)
    cu, lens, table, pages = batch(rng, news, lens, page)
    c = R.Cache(jas, cache, pages, heads, page, dh, table, token_major, pad)
    n = int(cu[-1])
    st, sh = heads * (dh + 3) + 1, dh + 3  # rows that do not start on 16 bytes
    if pad:
        st, sh = heads * dh, dh
    x = [rounded(rng.standard_normal((n + 2, st)) * np.exp(rng.uniform(-5, 5, (n + 2, 1))), dtype) for _ in range(2)]
    rows = [np.ascontiguousarray(np.lib.stride_tricks.as_strided(a, (n, heads, dh), (4 * st, 4 * sh, 4))) for a in x]
    d_cu, d_lens = jas.to_device(cu), jas.to_device(lens)
    d = [put(jas, a, dtype) for a in x]
    jas.check(jas.lib.jas_kv_append(c.ref, d[0].p, d[1].p, n + 2, st, sh, len(lens), d_cu.p, d_lens.p, dtype, None))
    c.put(rows[0], rows[1], cu, lens)
    for out in (F32, BF16):
        o = [empty(jas, (n + 2, heads, dh), out) for _ in range(2)]
        jas.check(jas.lib.jas_kv_read(c.ref, o[0].p, o[1].p, n + 2, heads * dh, dh, len(lens), d_cu.p, d_lens.p, out, None))
        for name, a in zip("kv", o):
            y = got(a, out)
            want = np.zeros((n, heads, dh))
            for i, pg, sl in c.slots(cu, lens):
                want[i] = c.plain[name][pg, :, sl]
            want = want.astype(np.float32)  # code * scale in fp32 (exact in 64 bits)
            assert np.array_equal(y[:n], rounded(want, out)), np.argwhere(y[:n] != rounded(want, out))[:4]
            assert np.all(y[n:] == 7.0)  # rows behind the last sequence stay
    # the whole sequences, by a cu that counts them: what was never written reads as it was (0)
    whole = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    o = empty(jas, (int(whole[-1]), heads, dh), F32)
    jas.check(jas.lib.jas_kv_read(c.ref, None, o.p, int(whole[-1]), heads * dh, dh, len(lens), hold(jas.to_device(whole)), d_lens.p, F32, None))
    want = np.concatenate([c.rows(b, lens[b])[1] for b in range(len(lens))])
    assert np.array_equal(o.numpy(), want.astype(np.float32))


def test_kv_many_sequences(jas):
    """More sequences than a workgroup keeps in LDS, some without new tokens."""
    rng = np.random.default_rng(5)
    news = rng.integers(0, 3, 1500)
    lens = news + rng.integers(0, 9, 1500)
    cu, lens, table, pages = batch(rng, news, list(lens), 4)
    c = R.Cache(jas, I8, pages, 1, 4, 32, table)
    n = int(cu[-1])
    x = [rng.standard_normal((n, 1, 32)).astype(np.float32) for _ in range(2)]
    d_cu, d_lens = jas.to_device(cu), jas.to_device(lens)
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, x[0], F32)), hold(put(jas, x[1], F32)), n, 32, 32, 1500, d_cu.p, d_lens.p, F32, None))
    c.put(x[0], x[1], cu, lens)
    o = [empty(jas, (n, 1, 32), F32) for _ in range(2)]
    jas.check(jas.lib.jas_kv_read(c.ref, o[0].p, o[1].p, n, 32, 32, 1500, d_cu.p, d_lens.p, F32, None))
    for name, a in zip("kv", o):
        want = np.zeros((n, 1, 32))
        for i, pg, sl in c.slots(cu, lens):
            want[i] = c.plain[name][pg, :, sl]
        assert np.array_equal(a.numpy(), want.astype(np.float32))


@pytest.mark.parametrize("cache", [I8, F8])
def test_kv_special_rows(jas, cache):
    """Zeros, one value, ties, tiny and huge magnitudes, infinities and NaN."""
    rng = np.random.default_rng(3)
    dh, rows = 64, 40
    x = rng.standard_normal((rows, 1, dh)).astype(np.float32)
    x[0] = 0
    x[1] = 0
    x[1, 0, 5] = -3.0
    x[2] *= np.float32(2.0 ** -120)  # a scale just above 2^-126, or none
    x[3] = np.float32(2.0 ** -149) * np.arange(dh)
    x[4] *= np.float32(2.0 ** 120)
    x[5, 0, 7] = np.inf
    x[6, 0, 9] = np.nan
    x[7] = np.float32(448.0)
    x[8] = np.linspace(-448, 448, dh)
    x[9, 0] = np.where(np.arange(dh) == 0, 127.0, np.arange(dh) - 31.5)  # ties of whole numbers, scale 1
    x[10, 0] = np.where(np.arange(dh) == 0, 448.0, (np.arange(dh) + 0.5) / 16 * 2.0 ** -6)  # ties of e4m3
    x[11] *= np.float32(2.0 ** -50)
    x[12] *= np.float32(2.0 ** 50)
    x[13] = np.float32(3.4e38)
    x[14, 0, 3] = -np.inf
    x[15:] = R.from_bf16(R.to_bf16(x[15:]))
    cu, lens, table, pages = batch(rng, [rows], [rows], 16)
    c = R.Cache(jas, cache, pages, 1, 16, dh, table)
    d_cu, d_lens = jas.to_device(cu), jas.to_device(lens)
    d = put(jas, x, F32)
    jas.check(jas.lib.jas_kv_append(c.ref, d.p, d.p, rows, dh, dh, 1, d_cu.p, d_lens.p, F32, None))
    o = empty(jas, x.shape, F32)
    jas.check(jas.lib.jas_kv_read(c.ref, o.p, None, rows, dh, dh, 1, d_cu.p, d_lens.p, F32, None))
    t, s = R.stored(x, cache)
    with np.errstate(all="ignore"):
        want = (t * s.astype(np.float64)[..., None]).astype(np.float32)
    assert np.array_equal(o.numpy(), want, equal_nan=True), np.argwhere(~((o.numpy() == want) | np.isnan(want)))[:5]
    assert np.isnan(want[5]).all() and np.isnan(want[6]).all() and (want[3] == 0).all()


def test_kv_bad_pages(jas):
    """Entries that are no pages, positions before the first and past the table's row: skipped, read as zeros."""
    rng = np.random.default_rng(4)
    dh, page = 32, 8
    table = np.array([[2, -1, 1], [5, 4, 3], [0, 99, -2 ** 31]], np.int32)
    cu, lens = np.array([0, 20, 26, 50], np.int32), np.array([20, 3, 30], np.int32)  # sequence 1: 6 new tokens of a length of 3; sequence 2 past its row
    c = R.Cache(jas, F32, 5, 2, page, dh, table)
    x = [rng.standard_normal((50, 2, dh)).astype(np.float32) for _ in range(2)]
    d_cu, d_lens = jas.to_device(cu), jas.to_device(lens)
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, x[0], F32)), hold(put(jas, x[1], F32)), 50, 2 * dh, dh, 3, d_cu.p, d_lens.p, F32, None))
    c.put(x[0], x[1], cu, lens)
    o = [empty(jas, (50, 2, dh), F32) for _ in range(2)]
    jas.check(jas.lib.jas_kv_read(c.ref, o[0].p, o[1].p, 50, 2 * dh, dh, 3, d_cu.p, d_lens.p, F32, None))
    for name, a in zip("kv", o):
        want = np.zeros((50, 2, dh))
        for i, pg, sl in c.slots(cu, lens):
            want[i] = c.plain[name][pg, :, sl]
        assert np.array_equal(a.numpy(), want.astype(np.float32))
    pool = c.k.numpy().view(np.float32).reshape(5, 2, page, dh)
    assert np.array_equal(pool, c.plain["k"].astype(np.float32))


# ---------------------------------------------------------------- attention
def attend(jas, c, q, cu, lens, scale, causal, dtype, max_q=None, max_len=None, n=None, pad=0, stream=None, within=None):
    n = n if n is not None else int(cu[-1])
    H, D = q.shape[1:]
    st, sh = H * (D + pad) + pad, D + pad
    x = np.full((n, st), 5.0, np.float32)
    np.lib.stride_tricks.as_strided(x, (n, H, D), (4 * st, 4 * sh, 4))[: len(q)] = q
    d_q, d_o = put(jas, x, dtype), empty(jas, (n, st), dtype)
    B = len(lens)
    max_q = max_q if max_q is not None else int(max(np.diff(cu)))
    max_len = max_len if max_len is not None else int(max(lens))
    size = jas.lib.jas_attn_paged_workspace(n, B, H, c.shape[1], D, max_q, max_len)
    if within is not None:  # the workspace of a larger call
        assert size <= within
        size = within
    work = jas.to_device(np.full(max(size, 1) + (1 << 20), 255, np.uint8))  # NaN partials, if one is read unwritten
    d_cu, d_lens = jas.to_device(cu), jas.to_device(lens)
    jas.check(jas.lib.jas_attn_paged(d_q.p, d_o.p, c.ref, n, B, d_cu.p, d_lens.p, H, max_q, max_len, st, sh, st, sh, scale, causal, dtype,
                                     work.p if size else None, stream))
    assert np.all(work.numpy()[max(size, 1):] == 255)
    y = got(d_o, dtype)
    inner = np.ascontiguousarray(np.lib.stride_tricks.as_strided(y, (n, H, D), (4 * st, 4 * sh, 4)))
    mask = np.ones((n, st), bool)
    np.lib.stride_tricks.as_strided(mask, (n, H, D), (st, sh, 1))[:] = False
    assert np.all(y[mask] == 7.0)  # what lies between the rows stays
    return inner


def tolerance(o, mag, big, D, L, dtype):
    ds = (D + 8) * 2.0 ** -24 * big
    t = (2 * ds + 2.0 ** -22 + (L / 8 + 64) * 2.0 ** -24) * mag
    return t + (2.0 ** -8 * mag + 2.0 ** -8 * np.abs(o) if dtype == BF16 else 0)


def filled(jas, rng, cache, news, lens, page, heads, dh, token_major=False, pad=0, std=1.0):
    """A cache that holds the whole sequences, written by jas_kv_append."""
    cu, lens, table, pages = batch(rng, news, lens, page)
    c = R.Cache(jas, cache, pages, heads, page, dh, table, token_major, pad, fill=np.nan if cache != I8 else 0.0)
    if cache == I8:  # scales of what was never written
        c.ks.upload(np.full((pages, heads, page), np.nan, np.float32))
        c.vs.upload(np.full((pages, heads, page), np.nan, np.float32))
    whole = np.concatenate([[0], np.cumsum(np.maximum(lens, 0))]).astype(np.int32)
    n = int(whole[-1])
    k, v = (rng.standard_normal((max(n, 1), heads, dh)).astype(np.float32) * np.float32(std) for _ in range(2))
    d_w, d_l = jas.to_device(whole), jas.to_device(lens)
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), n, heads * dh, dh, len(lens), d_w.p, d_l.p, F32, None))
    c.put(k, v, whole, lens)
    return c, cu, lens


TYPES = [(F32, F32), (F32, BF16), (F32, I8), (F32, F8), (BF16, BF16), (BF16, I8), (BF16, F8)]
ATTN = [  # new tokens, lengths, page, query heads per key head, key heads, dh
    ([1], [1], 16, 1, 1, 64),
    ([1, 1, 1], [5, 1, 200], 16, 4, 2, 128),
    ([1, 1], [333, 32], 20, 7, 1, 32),
    ([1, 1, 1, 1], [64, 65, 63, 31], 1, 1, 3, 64),
    ([2, 5, 1], [40, 5, 129], 8, 3, 2, 128),
    ([33, 1, 70], [33, 50, 150], 64, 2, 2, 64),
    ([130, 0, 7], [300, 12, 7], 256, 8, 1, 128),
    ([65, 3], [65, 257], 16, 1, 2, 32),
    ([16, 1], [700, 900], 20, 1, 1, 128),
]


@pytest.mark.parametrize("news,lens,page,g,heads,dh", ATTN)
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_attention(jas, news, lens, page, g, heads, dh, dtype, cache):
    rng = np.random.default_rng(sum(lens) + dh)
    c, cu, lens = filled(jas, rng, cache, news, lens, page, heads, dh, token_major=page == 16, pad=page == 8)
    q = rounded(rng.standard_normal((int(cu[-1]), g * heads, dh)), dtype)
    scale = np.float32(1 / math.sqrt(dh))
    for causal in (1, 0):
        rss = np.zeros(q.shape)
        o, mag, big = R.attention(c, q, cu, lens, float(scale), causal, len(q), rss)
        y = attend(jas, c, q, cu, lens, scale, causal, dtype, pad=page == 20)
        within(y, o, tolerance(o, mag, big, dh, max(lens), dtype))
        if dtype == F32:  # and closer on the whole than a lost product of split operands would leave it
            rms = np.sqrt(np.mean(((y - o) / np.where(rss > 0, rss, 1)) ** 2)) * 2.0 ** 24  # (no weight on anything but zeros: both 0)
            assert rms <= ATTENTION_BOUND * max(1.0, math.sqrt(max(lens) / 300)), rms


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("news,lens", [([1], [5000]), ([1, 1], [3000, 3]), ([20], [4001]), ([9, 1, 0], [2500, 2049, 0])])
def test_attention_long(jas, dtype, cache, news, lens):
    """Few rows over long sequences: keys split over workgroups and joined."""
    rng = np.random.default_rng(lens[0])
    c, cu, lens = filled(jas, rng, cache, news, lens, 16, 2, 64)
    q = rounded(rng.standard_normal((int(cu[-1]), 4, 64)) * 2, dtype)
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, len(q))
    y = attend(jas, c, q, cu, lens, 0.125, 1, dtype)
    within(y, o, tolerance(o, mag, big, 64, max(lens), dtype))
    if dtype == BF16 and max(news) <= 9 and cache != BF16:  # (weights of more than one bf16 part: the result's own rounding is left)
        within(y, o, tolerance(o, mag, big, 64, max(lens), F32) + 2.0 ** -15 * mag + 2.0 ** -8 * np.abs(o))
    # the hosts' numbers only bound: a larger max_len and max_q give the same result
    y2 = attend(jas, c, q, cu, lens, 0.125, 1, dtype, max_q=int(max(news)) + 100, max_len=20000)
    within(y2, o, tolerance(o, mag, big, 64, max(lens), dtype))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,news,lens", [(32, [100, 0, 217, 64, 3, 216], [150, 0, 217, 300, 3, 400]), (32, [129, 500, 400, 1], [129, 700, 401, 90])])
def test_attention_many_rows(jas, dtype, cache, heads, news, lens):
    """Enough rows that every unit has a tile of 64 of them, or of 128."""
    rng = np.random.default_rng(21)
    c, cu, lens = filled(jas, rng, cache, news, lens, 16, heads, 32)
    q = rounded(rng.standard_normal((int(cu[-1]), heads, 32)), dtype)
    o, mag, big = R.attention(c, q, cu, lens, 0.2, 1, len(q))
    within(attend(jas, c, q, cu, lens, 0.2, 1, dtype), o, tolerance(o, mag, big, 32, max(lens), dtype))


@pytest.mark.parametrize("dtype,cache", [(F32, F32), (BF16, BF16)])
def test_attention_steps_in_one_workspace(jas, dtype, cache):
    """Smaller steps, whose keys are split where the largest's are not, in the largest's workspace."""
    size = jas.lib.jas_attn_paged_workspace(600, 8, 32, 32, 32, 217, 900)
    for news, lens in [([1], [900]), ([1] * 8, [900] * 8), ([30, 1], [900, 20]), ([217], [900]), ([100, 0, 217, 64, 3, 216], [150, 0, 217, 300, 3, 900])]:
        rng = np.random.default_rng(22)
        c, cu, lens = filled(jas, rng, cache, news, lens, 16, 32, 32)
        q = rounded(rng.standard_normal((int(cu[-1]), 32, 32)), dtype)
        o, mag, big = R.attention(c, q, cu, lens, 0.2, 1, len(q))
        within(attend(jas, c, q, cu, lens, 0.2, 1, dtype, within=size), o, tolerance(o, mag, big, 32, max(lens), dtype))


@pytest.mark.parametrize("news,lens", [([1, 1], [700, 5]), ([20, 3], [300, 900]), ([40], [41])])
def test_attention_any_bound(jas, news, lens):
    """The largest max_len there is: the results are within the same tolerance."""
    rng = np.random.default_rng(20)
    c, cu, lens = filled(jas, rng, BF16, news, lens, 16, 2, 64)
    q = rng.standard_normal((int(cu[-1]), 6, 64)).astype(np.float32)
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, len(q))
    within(attend(jas, c, q, cu, lens, 0.125, 1, F32, max_len=2 ** 31 - 1), o, tolerance(o, mag, big, 64, max(lens), F32))


@pytest.mark.parametrize("dtype,cache", [(F32, F32), (BF16, BF16), (F32, F8)])
def test_attention_empty_and_outside(jas, dtype, cache):
    """Sequences of no token, lengths below the new tokens, above max_len and above the table's row,
    entries that are no page, rows behind the last sequence."""
    rng = np.random.default_rng(9)
    dh, page, heads, g = 64, 8, 2, 2
    c, _, lens = filled(jas, rng, cache, [1] * 6, [40, 24, 24, 40, 40, 17], page, heads, dh)
    cu = np.array([0, 1, 4, 4, 10, 12, 13], np.int32)
    lens = np.array([0, 2, 24, 60, 40, -7], np.int32)
    c.table_h[3, 1], c.table_h[4, 0], c.table_h[4, 3] = -1, c.shape[0], -2 ** 31
    c.table.upload(c.table_h)
    q = rounded(rng.standard_normal((13, g * heads, dh)), dtype)
    for max_len in (60, 33):
        cap = min(max_len, 40)
        o, mag, big = R.attention(c, q, cu, np.clip(lens, 0, cap), 0.125, 1, 16)
        y = attend(jas, c, q, cu, lens, 0.125, 1, dtype, max_len=max_len, n=16)
        assert np.all(y[13:] == 7.0) and np.all(y[0] == 0) and np.all(y[1] == 0) and np.all(y[12] == 0)
        within(y[:13], o[:13], tolerance(o, mag, big, dh, 64, dtype)[:13])
    # every page bad: zeros
    c.table.upload(np.full_like(c.table_h, -1))
    assert np.all(attend(jas, c, q, cu, lens, 0.125, 1, dtype)[:13] == 0)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attention_masked_values_do_not_reach(jas, dtype, cache, new, bad):
    """NaN and infinities in keys and values: rows that do not see them are as without, rows that do
    are NaN where a weight of them is not defined."""
    rng = np.random.default_rng(11)
    dh, L, at = 64, 90, 75
    c, cu, lens = filled(jas, rng, cache, [new], [L], 16, 1, dh)
    q = rounded(rng.standard_normal((new, 2, dh)), dtype)
    clean, _, _ = R.attention(c, q, cu, lens, 0.125, 1, new)
    # token `at` again, with one bad value in its value row
    k, v = rng.standard_normal((2, 1, 1, dh)).astype(np.float32)
    v[0, 0, 3] = bad
    one_cu, one_len = jas.to_device(np.array([0, 1], np.int32)), jas.to_device(np.array([at + 1], np.int32))
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), 1, dh, dh, 1, one_cu.p, one_len.p, F32, None))
    c.put(k, v, np.array([0, 1]), np.array([at + 1]))
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, new)
    y = attend(jas, c, q, cu, lens, 0.125, 1, dtype)
    sees = L - new + np.arange(new) >= at
    tol = tolerance(o, mag, big, dh, L, dtype)
    assert sees.any()
    within(y[~sees], o[~sees], tol[~sees])
    assert np.isfinite(o[~sees]).all()
    fine = np.isfinite(o[sees])
    assert np.array_equal(np.isfinite(y[sees]), fine) and not fine.all()
    assert np.all((np.abs(y[sees] - np.where(fine, o[sees], 0)) <= np.where(fine, tol[sees], np.inf)) | ~fine)
    if cache in (F32, BF16) and np.isinf(bad):
        assert np.all(y[sees][:, :, 3] == bad)
    # and in its key row: every row that sees it is NaN (an infinite score) or has no weight of it
    k[0, 0, 5] = bad
    v[0, 0, 3] = 0
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), 1, dh, dh, 1, one_cu.p, one_len.p, F32, None))
    c.put(k, v, np.array([0, 1]), np.array([at + 1]))
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, new)
    y = attend(jas, c, q, cu, lens, 0.125, 1, dtype)
    within(y, o, tolerance(o, mag, np.where(np.isfinite(big), big, 20.0), dh, L, dtype))


@pytest.mark.parametrize("dtype,cache", [(F32, F32), (F32, I8), (BF16, BF16), (BF16, F8)])
@pytest.mark.parametrize("new", [1, 24])
def test_attention_growing_scores(jas, dtype, cache, new):
    """Scores that grow along the keys by hundreds, and ones far below zero: the running maximum moves."""
    rng = np.random.default_rng(13)
    dh, L = 64, 500
    for sign in (1.0, -1.0):
        cu, lens, table, pages = batch(rng, [new], [L], 16)
        c = R.Cache(jas, cache, pages, 1, 16, dh, table)
        k = (rng.standard_normal((L, 1, dh)) * 0.1 + np.linspace(0, 6, L)[:, None, None] * sign).astype(np.float32)
        v = rng.standard_normal((L, 1, dh)).astype(np.float32)
        whole = np.array([0, L], np.int32)
        jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
        c.put(k, v, whole, lens)
        q = rounded(np.abs(rng.standard_normal((new, 3, dh))) + 1, dtype)
        o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, new)
        within(attend(jas, c, q, cu, lens, 0.125, 1, dtype), o, tolerance(o, mag, big, dh, L, dtype))
        within(attend(jas, c, -q, cu, lens, -0.125, 1, dtype), o, tolerance(o, mag, big, dh, L, dtype))


@pytest.mark.parametrize("mag", [2.0 ** -140, 2.0 ** -100, 2.0 ** 100, 2.0 ** 126])
def test_attention_fp32_magnitudes(jas, mag):
    """Values near both ends of fp32 keep its accuracy (subnormal ones their last bit)."""
    rng = np.random.default_rng(17)
    dh, L = 64, 70
    cu, lens, table, pages = batch(rng, [1], [L], 16)
    for new in (1, 20):
        cu = np.array([0, new], np.int32)
        c = R.Cache(jas, F32, pages, 1, 16, dh, table)
        k, v = rng.standard_normal((2, L, 1, dh)).astype(np.float32)
        v = np.clip(v, -1.9, 1.9) * np.float32(mag)
        whole = np.array([0, L], np.int32)
        jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
        c.put(k, v, whole, lens)
        q = rng.standard_normal((new, 2, dh)).astype(np.float32)
        o, m, big = R.attention(c, q, cu, lens, 0.125, 1, new)
        # (sums of subnormal products: half of the least number for each of the additions)
        within(attend(jas, c, q, cu, lens, 0.125, 1, F32), o, tolerance(o, m, big, dh, L, F32) + 2.0 ** -149 * (L + 8))


# ---------------------------------------------------------------- sampling
def draw(jas, x, dtype, temp=None, top_k=None, top_p=None, min_p=None, u=None, ld=None, logp=True):
    n, V = x.shape
    ld = ld or V
    a = np.full((n, ld), 1e30, np.float32)
    a[:, :V] = x
    arr = lambda v, t: None if v is None else jas.to_device(np.ascontiguousarray(v, t))  # noqa: E731
    d = [arr(temp, np.float32), arr(top_k, np.int32), arr(top_p, np.float32), arr(min_p, np.float32), arr(u, np.float32)]
    ids, lp = jas.to_device(np.full(n, -99, np.int32)), jas.to_device(np.full(n, 99, np.float32))
    size = jas.lib.jas_sample_workspace(n, V)
    work = jas.to_device(np.full(max(size, 1), 255, np.uint8))
    d_x = put(jas, a, dtype)
    jas.check(jas.lib.jas_sample(d_x.p, n, V, ld, *[v.p if v else None for v in d], ids.p, lp.p if logp else None, dtype, work.p if size else None, None))
    return ids.numpy(), lp.numpy()


def check_draw(jas, x, dtype, temp=None, top_k=None, top_p=None, min_p=None, u=None, ld=None):
    n, V = x.shape
    x = rounded(x, dtype)
    ids, lp = draw(jas, x, dtype, temp, top_k, top_p, min_p, u, ld)
    f = lambda v, i, d: d if v is None else float(np.float32(v[i]))  # noqa: E731
    for i in range(n):
        want = R.sample(x[i], f(temp, i, 1.0), 0 if top_k is None else int(top_k[i]), f(top_p, i, 1.0), f(min_p, i, 0.0), f(u, i, 0.0))
        assert ids[i] == want[0], (i, ids[i], want)
        if want[0] < 0:
            assert lp[i] == -np.inf
        else:
            bits = max(0, math.ceil(math.log2(V)))
            assert abs(lp[i] - want[1]) <= 2.0 ** -24 * abs(want[1]) + V * 2.0 ** -min(52, 62 - bits) + 1e-13, (i, lp[i], want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1025, 4099, 50257])
@pytest.mark.parametrize("k,p,mp", [(0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.1), (40, 0.9, 0.05), (1, 0.5, 0.5), (700, 0.3, 0.0)])
def test_sample(jas, dtype, V, k, p, mp):
    rng = np.random.default_rng(V + k)
    n = 6
    x = rng.standard_normal((n, V)) * 3
    x[1] = np.round(x[1])  # ties
    temp = rng.uniform(0.3, 1.5, n)
    check_draw(jas, x, dtype, temp, [k] * n, [p] * n, [mp] * n, rng.random(n), ld=V + 3 if V != 1000 else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,ld", [(1, 200003, None), (2, 1200000, 1200001), (600, 17000, 17003), (1100, 2500, None), (40, 33000, 33008)])
def test_sample_sizes(jas, dtype, n, V, ld):
    """Rows of many chunks and many rows of few; starts off 16 bytes."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((min(n, 24), V)).astype(np.float32) * 2.5
    x = x[np.arange(n) % len(x)]
    for k, p, mp in ((0, 0.95, 0.0), (30, 0.9, 0.0), (0, 1.0, 0.03)):
        rows = np.unique(np.concatenate([[0, n - 1], rng.integers(0, n, 8)]))
        u = rng.random(n).astype(np.float32)
        temp = rng.uniform(0.5, 1.2, n).astype(np.float32)
        ids, lp = draw(jas, x, dtype, temp, [k] * n, [p] * n, [mp] * n, u, ld)
        for i in rows:
            want = R.sample(rounded(x[i], dtype), float(temp[i]), k, float(np.float32(p)), float(np.float32(mp)), float(u[i]))
            assert ids[i] == want[0], (i, ids[i], want)
            assert abs(lp[i] - want[1]) <= 2.0 ** -24 * abs(want[1]) + V * 2.0 ** -41 + 1e-13


@pytest.mark.parametrize("V,k,p", [(50257, 2000, 1.0), (50257, 5000, 0.9), (6000, 5999, 0.5), (50257, 1024, 0.99), (50257, 1025, 0.99)])
def test_sample_large_top_k(jas, V, k, p):
    rng = np.random.default_rng(k)
    check_draw(jas, rng.standard_normal((3, V)) * 3, F32, [0.9, 1.0, 5.0], [k] * 3, [p] * 3, None, rng.random(3))


@pytest.mark.parametrize("spread", [1e-6, 1e-3, 100.0, 1e30])
def test_sample_spreads(jas, spread):
    """Logits all but equal, and ones whose weights are nearly all nothing; temperatures to match; a masked vocabulary."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((4, 30000)) * spread
    x[3, 10:] = np.finfo(np.float32).min
    for temp in (spread, spread * 0.01, 1.0, 1e-30):
        for k, p, mp in ((0, 0.9, 0.0), (50, 1.0, 0.0), (0, 1.0, 0.2), (20, 0.5, 0.5)):
            check_draw(jas, x, F32, [temp] * 4, [k] * 4, [p] * 4, [mp] * 4, rng.random(4))


@pytest.mark.parametrize("V", [37, 8200])
def test_sample_ties(jas, V):
    """All equal, and few levels: the lowest indexes are kept."""
    rng = np.random.default_rng(V)
    for x in (np.zeros((4, V)), rng.integers(0, 3, (4, V)).astype(float), np.where(np.arange(V) % 5 == 3, 2.0, -1e9)[None].repeat(4, 0)):
        for k, p in ((0, 1.0), (3, 1.0), (0, 0.5), (V - 2, 0.25), (V // 2, 0.9), (0, 0.0), (V + 5, -1.0)):
            check_draw(jas, x, F32, None, [k] * 4, [p] * 4, None, [0.0, 0.3, 0.999, 1.0 - 2.0 ** -24])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_special_rows(jas, dtype):
    V = 300
    rng = np.random.default_rng(8)
    x = rng.standard_normal((14, V)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, 5:] = -np.inf
    x[4, [7, 200]] = np.inf
    x[5] = np.finfo(np.float32).min
    x[6, 1:] = np.finfo(np.float32).min
    x[7] = -0.0
    x[7, 100:] = 0.0
    x[8] = 3e38
    x[9, :] = -np.inf
    x[9, 299] = -5
    temp = np.ones(14)
    temp[10:] = [0.0, -1.0, np.nan, np.inf]
    for k, p, mp in ((0, 1.0, 0.0), (4, 0.6, 0.0), (0, 0.4, 0.2), (0, 1.0, 5.0), (2, np.nan, np.nan)):
        for u in (0.0, 0.51, 0.9999999, 2.0, -3.0, np.nan):
            check_draw(jas, x, dtype, temp, [k] * 14, [p] * 14, [mp] * 14, [u] * 14)
    ids, _ = draw(jas, x[2:], dtype, u=[0.4] * 12, logp=False)
    assert ids[0] % 2 == 1


def test_sample_frequencies(jas):
    """A grid of uniform numbers draws each token as often as its share, to one draw."""
    V, n = 50, 1000
    x = np.random.default_rng(1).standard_normal(V)
    ids, _ = draw(jas, np.repeat(x[None], n, 0), F32, u=(np.arange(n) + 0.5) / n)
    share = np.exp(x - x.max())
    share /= share.sum()
    assert np.all(np.abs(np.bincount(ids, minlength=V) - share * n) <= 1.0)


def test_sample_greedy_is_argmax(jas):
    x = np.round(np.random.default_rng(2).standard_normal((9, 5000)) * 2).astype(np.float32)
    ids, lp = draw(jas, x, F32, temp=np.zeros(9), u=np.full(9, 0.7))
    d, out = jas.to_device(x), jas.to_device(np.zeros(9, np.int32))
    jas.check(jas.lib.jas_argmax(d.p, 9, 5000, 5000, out.p, None))
    assert np.array_equal(ids, out.numpy()) and np.all(lp == 0)


# ---------------------------------------------------------------- together
class Server:
    """Two layers' worth of a serving step on one stream: rotary, cache, attention, sampling."""

    def __init__(self, jas, dtype, cache, B, H, heads, dh, page, width, vocab, max_q, seed=0):
        rng = np.random.default_rng(seed)
        self.jas, self.dtype, self.B, self.H, self.heads, self.dh, self.vocab = jas, dtype, B, H, heads, dh, vocab
        table = rng.permutation(B * width).reshape(B, width).astype(np.int32)
        self.cache = R.Cache(jas, cache, B * width, heads, page, dh, table)
        self.freq_h, self.m = jas.rope_freqs(dh, 10000.0, jas.RopeScaling(2, 64, 4.0, 1.0, 8.0))
        self.freq = jas.to_device(self.freq_h)
        self.max_q, self.max_len, self.cap = max_q, width * page, B * max_q
        self.wide = (H + 2 * heads) * dh
        es = np.uint16 if dtype == BF16 else np.float32
        self.qkv, self.o = jas.DeviceArray((self.cap, self.wide), es), jas.DeviceArray((self.cap, H, dh), es)
        self.cu, self.lens, self.pos = (jas.DeviceArray(k, np.int32) for k in (B + 1, B, self.cap))
        self.work = jas.DeviceArray(max(1, jas.lib.jas_attn_paged_workspace(self.cap, B, H, heads, dh, max_q, self.max_len)), np.uint8)
        self.work2 = jas.DeviceArray(max(1, jas.lib.jas_sample_workspace(B, vocab)), np.uint8)
        self.logits, self.u = jas.DeviceArray((B, vocab), np.float32), jas.DeviceArray(B, np.float32)
        self.ids, self.logp = jas.DeviceArray(B, np.int32), jas.DeviceArray(B, np.float32)
        self.top_p = jas.to_device(np.full(B, 0.9, np.float32))
        self.qkv.zero(), self.o.zero(), self.pos.zero()

    def inputs(self, rng, news, lens):
        """A new batch: what the plain form needs of it."""
        cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        pos = np.zeros(self.cap, np.int32)
        for b in range(self.B):
            pos[cu[b]:cu[b + 1]] = lens[b] - news[b] + np.arange(news[b])
        x = rounded(rng.standard_normal((self.cap, self.wide)), self.dtype)
        u, lg = rng.random(self.B).astype(np.float32), rng.standard_normal((self.B, self.vocab)).astype(np.float32) * 3
        self.qkv.upload(R.to_bf16(x) if self.dtype == BF16 else x)
        self.cu.upload(cu), self.lens.upload(np.array(lens, np.int32)), self.pos.upload(pos), self.u.upload(u), self.logits.upload(lg)
        return cu, np.array(lens, np.int32), pos, x, u, lg

    def step(self, stream):
        j, lib = self.jas, self.jas.lib
        es = 2 if self.dtype == BF16 else 4
        at = lambda k: self.qkv.ptr + k * self.dh * es  # noqa: E731
        turn = self.H + self.heads
        j.check(lib.jas_rope(at(0), at(0), self.pos.p, self.freq.p, self.cap, turn, self.dh, self.dh, self.wide, self.dh, self.wide, self.dh, 1,
                             self.m, self.dtype, stream))
        j.check(lib.jas_kv_append(self.cache.ref, at(self.H), at(turn), self.cap, self.wide, self.dh, self.B, self.cu.p, self.lens.p, self.dtype, stream))
        j.check(lib.jas_attn_paged(at(0), self.o.p, self.cache.ref, self.cap, self.B, self.cu.p, self.lens.p, self.H, self.max_q, self.max_len,
                                   self.wide, self.dh, self.H * self.dh, self.dh, 1 / math.sqrt(self.dh), 1, self.dtype, self.work.p, stream))
        j.check(lib.jas_sample(self.logits.p, self.B, self.vocab, self.vocab, None, None, self.top_p.p, None, self.u.p, self.ids.p, self.logp.p,
                               F32, self.work2.p, stream))

    def check(self, cu, lens, pos, x, u, lg):
        n = int(cu[-1])
        rows = x.reshape(self.cap, -1, self.dh)
        turned = rounded(R.rope(rows[:, :self.H + self.heads], pos, self.freq_h, self.m, self.dh, 1), self.dtype)
        # the device's own turned rows, near the plain ones, go on from here: what is stored of them is exact
        got_rows = got(self.qkv, self.dtype).reshape(self.cap, -1, self.dh)
        dev = got_rows[:, :self.H + self.heads]
        assert np.all(np.abs(dev - turned) <= (2.0 ** -7 if self.dtype == BF16 else 2.0 ** -20) * (np.abs(turned) + 1.0) * 4)
        self.cache.put(dev[:n, self.H:], got_rows[:n, self.H + self.heads:], cu, lens)
        o, mag, big = R.attention(self.cache, dev[:n, :self.H], cu, lens, 1 / math.sqrt(self.dh), 1, n)
        within(got(self.o, self.dtype)[:n], o, tolerance(o, mag, big, self.dh, int(max(lens)), self.dtype))
        for b in range(self.B):
            assert self.ids.numpy()[b] == R.sample(lg[b], 1.0, 0, float(np.float32(0.9)), 0.0, float(u[b]))[0]


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_serving_steps(jas, dtype, cache):
    """Prompts in chunks, then decode steps beside a late prompt: every step against the plain form."""
    rng = np.random.default_rng(21)
    s = Server(jas, dtype, cache, 3, 4, 2, 64, 8, 12, 500, 20)
    lens = np.zeros(3, int)
    for news in ([20, 3, 0], [17, 1, 0], [1, 1, 9], [1, 1, 20], [1, 1, 1]):
        lens = lens + news
        case = s.inputs(rng, news, lens)
        s.step(None)
        jas.check(jas.lib.jas_synchronize(None))
        s.check(*case)


@pytest.mark.parametrize("dtype,cache", [(F32, F32), (BF16, BF16), (BF16, F8)])
def test_serving_graph(jas, dtype, cache):
    """A decode step captured once and replayed as lengths grow, with eager work between the replays."""
    hip, rng = R.Hip(), np.random.default_rng(23)
    s = Server(jas, dtype, cache, 3, 4, 2, 64, 8, 12, 500, 4)
    lens = np.array([4, 3, 2])
    case = s.inputs(rng, [4, 3, 2], lens)
    s.step(None)
    jas.check(jas.lib.jas_synchronize(None))
    s.check(*case)
    stream = hip.stream()
    graph = hip.capture(stream, lambda: s.step(stream))
    for k in range(6):
        news = [[1, 1, 1], [1, 0, 4], [2, 1, 1]][k % 3]
        lens = lens + news
        case = s.inputs(rng, news, lens)
        hip("hipGraphLaunch", graph, stream)
        hip("hipStreamSynchronize", stream)
        s.check(*case)
        jas.DeviceArray(1000).zero().numpy()  # the program's own work between the replays
    hip("hipGraphExecDestroy", graph)
    hip("hipStreamDestroy", stream)


def test_serving_two_streams(jas):
    """Two servers on two streams at once, each with its own workspace."""
    hip = R.Hip()
    a, b = (Server(jas, BF16, c, 3, 4, 2, 64, 8, 40, 3000, 4, k) for k, c in ((1, BF16), (2, I8)))
    streams = [hip.stream(), hip.stream()]
    rng = np.random.default_rng(29)
    lens = np.zeros(3, int)
    for news in ([4, 4, 4], [1, 1, 1], [1, 2, 1]):
        lens = lens + news
        cases = [x.inputs(rng, news, lens) for x in (a, b)]
        jas.check(jas.lib.jas_synchronize(None))
        for x, st in zip((a, b), streams):
            x.step(st)
        for st in streams:
            hip("hipStreamSynchronize", st)
        for x, case in zip((a, b), cases):
            x.check(*case)
    for st in streams:
        hip("hipStreamDestroy", st)


@pytest.mark.parametrize("B", [300, 700])
def test_attention_many_sequences(jas, B):
    """More sequences than a workgroup has threads: short ones, some without new tokens, some longer."""
    rng = np.random.default_rng(B)
    news = rng.integers(0, 2, B)
    news[[3, 7, B - 1]] = [40, 33, 20]
    lens = news + rng.integers(0, 40, B)
    c, cu, lens = filled(jas, rng, BF16, list(news), list(lens), 8, 1, 32)
    for dtype in (F32, BF16):
        q = rounded(rng.standard_normal((int(cu[-1]), 3, 32)), dtype)
        o, mag, big = R.attention(c, q, cu, lens, 0.2, 1, len(q))
        for max_q in (1, 40):
            within(attend(jas, c, q, cu, lens, 0.2, 1, dtype, max_q=max_q), o, tolerance(o, mag, big, 32, 80, dtype))


def test_far_slots(jas):
    """A pool whose last pages lie past 2^31 elements: offsets of 64 bits."""
    rng = np.random.default_rng(41)
    heads, page, dh = 2, 16, 128
    row = heads * page * dh
    pages = (1 << 31) // row + 8
    table = np.array([[pages - 1, 0, pages - 3, pages // 2 + 1, pages - 5]], np.int32)
    pools = [jas.DeviceArray(pages * row, np.uint8) for _ in range(2)]
    scales = [jas.DeviceArray(pages * heads * page, np.float32) for _ in range(2)]
    d_table = jas.to_device(table)
    kv = jas.PagedKv(pools[0].ptr, pools[1].ptr, scales[0].ptr, scales[1].ptr, d_table.ptr, row, page * dh, dh, 5, 5, F8, pages, page, heads, dh)
    small = R.Cache(jas, F8, 5, heads, page, dh, np.arange(5, dtype=np.int32)[None])  # the plain copy: the same pages, near
    L = 77
    k, v = rng.standard_normal((2, L, heads, dh)).astype(np.float32)
    whole, lens = np.array([0, L], np.int32), np.array([L], np.int32)
    d_w, d_l, d_k, d_v = (jas.to_device(a) for a in (whole, lens, k, v))
    jas.check(jas.lib.jas_kv_append(R.C.byref(kv), d_k.p, d_v.p, L, heads * dh, dh, 1, d_w.p, d_l.p, F32, None))
    small.put(k, v, whole, lens)
    for new in (1, 30):
        cu = np.array([0, new], np.int32)
        q = rounded(rng.standard_normal((new, 4, dh)), BF16)
        o, mag, big = R.attention(small, q, cu, lens, 0.09, 1, new)
        small.view, keep = kv, small.view
        y = attend(jas, small, q, cu, lens, 0.09, 1, BF16)
        small.view = keep
        within(y, o, tolerance(o, mag, big, dh, L, BF16))


def test_results_repeat(jas):
    """The same call twice gives the same bits."""
    rng = np.random.default_rng(31)
    c, cu, lens = filled(jas, rng, BF16, [1, 1], [3000, 700], 16, 2, 128)
    q = rounded(rng.standard_normal((2, 8, 128)), BF16)
    first = attend(jas, c, q, cu, lens, 0.09, 1, BF16)
    x, u = rng.standard_normal((3, 9000)), [0.2, 0.5, 0.8]
    ids = draw(jas, x, F32, top_p=[0.9] * 3, u=u)
    for _ in range(5):
        assert np.array_equal(attend(jas, c, q, cu, lens, 0.09, 1, BF16), first)
        again = draw(jas, x, F32, top_p=[0.9] * 3, u=u)
        assert np.array_equal(again[0], ids[0]) and np.array_equal(again[1], ids[1])


@pytest.mark.parametrize("dtype,cache,news,lens,heads,g,max_q", [
    (BF16, BF16, [32] * 8 + [137], [600, 14000, 64, 9000, 33, 2000, 500, 40, 14619], 1, 3, 156),  # tiles of 128 rows, tens of splits
    (BF16, I8, [3, 2, 1] * 11 + [1, 1, 15], [700, 7000, 90] * 11 + [60, 70, 7297], 1, 7, 2),  # of 16, max_q below the longest
    (F32, BF16, [1] * 412, [300, 5, 90, 2] * 102 + [640, 1, 17, 641], 1, 16, 1)])
def test_attention_splits_in_its_workspace(jas, dtype, cache, news, lens, heads, g, max_q):
    """Shares of the keys just above a multiple of 128: the last sequence's last splits end within the workspace."""
    rng = np.random.default_rng(len(lens))
    c, cu, lens = filled(jas, rng, cache, news, lens, 64, heads, 64)
    q = rounded(rng.standard_normal((int(cu[-1]), g * heads, 64)), dtype)
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, len(q))
    within(attend(jas, c, q, cu, lens, 0.125, 1, dtype, max_q=max_q), o, tolerance(o, mag, big, 64, max(lens), dtype))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attention_weightless_split_keeps_nan(jas, dtype, cache, new, bad):
    """A value that is not finite, of a key whose weight is nothing beside other splits' keys: 0 times it is NaN, as in one split."""
    rng = np.random.default_rng(51)
    dh, L = 64, 5000
    cu, lens, table, pages = batch(rng, [new], [L], 16)
    c = R.Cache(jas, cache, pages, 1, 16, dh, table)
    k, v = rng.standard_normal((2, L, 1, dh)).astype(np.float32)
    k[:600] -= 30  # (scores lower by some 300: no fp32 weight)
    v[10, 0, 3] = bad
    whole = np.array([0, L], np.int32)
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
    c.put(k, v, whole, lens)
    q = rounded(np.abs(rng.standard_normal((new, 2, dh))) + 0.5, dtype)
    o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, new)
    y = attend(jas, c, q, cu, lens, 0.125, 1, dtype)
    assert not np.isfinite(o[:, :, 3]).any() and not np.isfinite(y[:, :, 3]).any()
    fine = np.isfinite(o)
    within(np.where(fine, y, 0), np.where(fine, o, 0), np.where(fine, tolerance(o, mag, big, dh, L, dtype), 0))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new", [1, 24])
@pytest.mark.parametrize("level", [-60, -40, 30])
def test_attention_levels_and_magnitudes(jas, dtype, cache, new, level):
    """Rows whose scores all lie far from 0 (in powers of two), over small and large values: weights are relative to the row's own
    maximum, and numbers near the end of fp32 keep their accuracy."""
    rng = np.random.default_rng(53)
    dh, L = 64, 90
    cu, lens, table, pages = batch(rng, [new], [L], 16)
    q = rounded(rng.uniform(0.9, 1.1, (new, 2, dh)), dtype)
    k = (level / (dh * 0.125 * 1.4427) + 0.1 * rng.standard_normal((L, 1, dh))).astype(np.float32)
    unit = np.clip(rng.standard_normal((L, 1, dh)), -1.9, 1.9)
    for mag in (2.0 ** -100, 1.0, 2.0 ** 100):
        c = R.Cache(jas, cache, pages, 1, 16, dh, table)
        v = (unit * mag).astype(np.float32)
        whole = np.array([0, L], np.int32)
        jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
        c.put(k, v, whole, lens)
        o, m, big = R.attention(c, q, cu, lens, 0.125, 1, new)
        within(attend(jas, c, q, cu, lens, 0.125, 1, dtype), o, tolerance(o, m, big, dh, L, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", [BF16, I8, F8])
@pytest.mark.parametrize("new", [1, 24])
@pytest.mark.parametrize("mag", [2.0 ** -124, 2.0 ** -118, 2.0 ** -110, 2.0 ** 112, 2.0 ** 120])
def test_attention_small_cache_magnitudes(jas, dtype, cache, new, mag):
    """Caches of fewer bits that hold values near both ends of fp32 (8 bits: scales down to 2^-126): no part of a weight is lost."""
    rng = np.random.default_rng(57)
    dh, L = 64, 70
    cu, lens, table, pages = batch(rng, [new], [L], 16)
    c = R.Cache(jas, cache, pages, 1, 16, dh, table)
    k, v = rng.standard_normal((2, L, 1, dh)).astype(np.float32)
    v = (np.clip(v, -1.9, 1.9) * mag).astype(np.float32)
    whole = np.array([0, L], np.int32)
    jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
    c.put(k, v, whole, lens)
    q = rounded(rng.standard_normal((new, 2, dh)), dtype)
    o, m, big = R.attention(c, q, cu, lens, 0.125, 1, new)
    # (a bf16 result below 2^-126 is rounded to a multiple of 2^-133; sums of fp32 products to multiples of 2^-149)
    least = 2.0 ** -134 if dtype == BF16 else 0.0
    within(attend(jas, c, q, cu, lens, 0.125, 1, dtype), o, tolerance(o, m, big, dh, L, dtype) + least + 2.0 ** -149 * (L + 8))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("news,lens", [([1, 1], [70, 333]), ([40, 7], [90, 33]), ([70], [300]), ([20], [2500])])
def test_attention_scale_sign(jas, dtype, cache, news, lens):
    """Scales below zero, and of zero: the latter takes the same path as queries of zero, to the bit (a matrix instruction's sums are not
    the same bits with their signs changed)."""
    rng = np.random.default_rng(59)
    c, cu, lens = filled(jas, rng, cache, news, lens, 16, 2, 64)
    q = rounded(rng.standard_normal((int(cu[-1]), 6, 64)), dtype)
    for causal in (1, 0):
        o, mag, big = R.attention(c, q, cu, lens, -0.125, causal, len(q))
        within(attend(jas, c, q, cu, lens, -0.125, causal, dtype), o, tolerance(o, mag, big, 64, max(lens), dtype))
        zero = attend(jas, c, q, cu, lens, 0.0, causal, dtype)
        assert np.array_equal(zero, attend(jas, c, 0 * q, cu, lens, 0.125, causal, dtype))
        o, mag, big = R.attention(c, q, cu, lens, 0.0, causal, len(q))
        within(zero, o, tolerance(o, mag, big, 64, max(lens), dtype))


def test_kv_lengths_below_any_position(jas):
    """A length of -2^31: every position is below 0, however many rows the sequence has."""
    dh, page, n = 32, 1 << 20, 70000
    table = np.zeros((1, 2048), np.int32)  # a row that holds 2^31 positions, all of them in page 0
    cache = jas.DeviceArray(page * dh, np.uint8).zero()
    scales = jas.DeviceArray(page, np.float32).zero()
    d_table, d_cu, d_lens = jas.to_device(table), jas.to_device(np.array([0, n], np.int32)), jas.to_device(np.array([-2 ** 31], np.int32))
    kv = jas.PagedKv(cache.ptr, cache.ptr, scales.ptr, scales.ptr, d_table.ptr, page * dh, page * dh, dh, 2048, 2048, I8, 1, page, 1, dh)
    rows = jas.to_device(np.ones((n, dh), np.float32))
    jas.check(jas.lib.jas_kv_append(R.C.byref(kv), rows.p, rows.p, n, dh, dh, 1, d_cu.p, d_lens.p, F32, None))
    assert not cache.numpy().any() and not scales.numpy().any()
    scales.upload(np.ones(page, np.float32)), cache.upload(np.ones(page * dh, np.uint8))
    jas.check(jas.lib.jas_kv_read(R.C.byref(kv), rows.p, None, n, dh, dh, 1, d_cu.p, d_lens.p, F32, None))
    assert not rows.numpy().any()


@pytest.mark.parametrize("dtype,cache", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("new,L", [(1, 70), (24, 70), (1, 3000), (20, 3000)])
def test_attention_scores_of_minus_infinity(jas, dtype, cache, new, L):
    """Rows whose scores are all -inf are zeros, as rows that see no key are; beside finite scores, -inf ones have no weight."""
    rng = np.random.default_rng(61)
    dh = 64
    cu, lens, table, pages = batch(rng, [new], [L], 16)
    q = rounded(np.abs(rng.standard_normal((new, 2, dh))) + 0.5, dtype)
    for finite in (0, 3):
        c = R.Cache(jas, cache, pages, 1, 16, dh, table)
        k, v = rng.standard_normal((2, L, 1, dh)).astype(np.float32)
        k[:L - new + 1 - finite] = -np.inf
        k[L - new + 1:] = -np.inf
        whole = np.array([0, L], np.int32)
        jas.check(jas.lib.jas_kv_append(c.ref, hold(put(jas, k, F32)), hold(put(jas, v, F32)), L, dh, dh, 1, hold(jas.to_device(whole)), hold(jas.to_device(lens)), F32, None))
        c.put(k, v, whole, lens)
        y = attend(jas, c, q, cu, lens, 0.125, 1, dtype)
        if finite:
            o, mag, big = R.attention(c, q, cu, lens, 0.125, 1, new)
            big = (np.abs(q).max() * dh * 0.125 * 6) * np.ones_like(big)  # (of the finite scores: |k| < 6)
            within(y, o, tolerance(o, mag, big, dh, L, dtype))
        else:
            assert np.all(y == 0)
