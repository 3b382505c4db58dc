"""The serving operators of jasmine_amd as measurable cases: rotary positions, the paged
key/value cache (written, quantised and read back), attention of new tokens over it, and
sampling of the next token.  With `own` false, `run` computes the definition with elementary
torch operations in 32 bits (64 for rotary angles, quantisation steps and sampling's sums, where
32 lose what matters); with `own` true it makes the library's calls on its own stream."""
import ctypes as C
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8, "f8": torch.float8_e4m3fn}
CODES = {"f32": 0, "bf16": 3, "i8": 4, "f8": 5}  # JAS_F32, JAS_BF16, JAS_I8, JAS_F8E4M3
BYTES = {"f32": 4, "bf16": 2, "i8": 1, "f8": 1}
QMAX = {"i8": 127.0, "f8": 448.0}


# ------------------------------------------------------------------ the cases
def _rope(name, n, heads, dh, rot, layout, scaling, dtype, far):
    return {"name": name, "op": "rope", "n": n, "heads": heads, "dh": dh, "rot": rot, "layout": layout,
            "scaling": scaling, "dtype": dtype, "far": far}


def _kv(name, b, new, ctx, kv_heads, dh, page, cache, dtype, read, mixed=False):
    return {"name": name, "op": "kv", "b": b, "new": new, "ctx": ctx, "kv_heads": kv_heads, "dh": dh, "page": page,
            "cache": cache, "dtype": dtype, "read": read, "mixed": mixed}


def _attn(name, b, new, ctx, heads, kv_heads, dh, page, cache, dtype, mixed=False):
    return {"name": name, "op": "attn", "b": b, "new": new, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "dh": dh,
            "page": page, "cache": cache, "dtype": dtype, "mixed": mixed}


def _sample(name, n, vocab, dtype, top_k, top_p, min_p):
    return {"name": name, "op": "sample", "n": n, "vocab": vocab, "dtype": dtype, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # one decode step of 16 sequences: queries and keys of LLaMA-7B width with grouped
        # keys turned to their positions, interleaved pairs, fp32 as the runner holds them
        _rope("rope_decode", 16, 40, 128, 128, "pairs", "none", "f32", 4096),
        # a prompt batch in bf16: half of each head turns, halves layout, frequencies scaled for a
        # context far beyond the trained one
        _rope("rope_prompt", 8191, 40, 128, 64, "halves", "yarn", "bf16", 131072),
        # a decode step's keys and values of 61 sequences, written to an 8-bit float cache
        # and read back (latency counts)
        _kv("kv_decode_f8", 61, 1, 1000, 8, 128, 16, "f8", "bf16", "new"),
        # prompts of up to 2048 tokens written as 8-bit integers and read back in fp32
        _kv("kv_prompt_i8", 8, 2048, 2048, 8, 128, 64, "i8", "f32", "all"),
        # one sequence of GPT-2-small heads, fp32 cache, one new token: the smallest call
        _attn("attn_one_f32", 1, 1, 1000, 12, 12, 64, 16, "f32", "f32"),
        # a decode batch over bf16 caches of grouped heads, lengths spread from 1024 to 4096
        _attn("attn_decode_bf16", 32, 1, 4096, 32, 8, 128, 16, "bf16", "bf16"),
        # few sequences of a very long context in 8-bit integers: work split over the keys
        _attn("attn_long_i8", 3, 1, 65536, 32, 8, 128, 64, "i8", "bf16"),
        # chunks of a long prompt (up to 512 new tokens) over what is cached already, bf16
        _attn("attn_chunk_bf16", 4, 512, 4096, 32, 8, 128, 64, "bf16", "bf16"),
        # the framework's own arithmetic: fp32 queries over an fp32 cache, odd chunks
        _attn("attn_chunk_f32", 2, 333, 2001, 12, 12, 64, 16, "f32", "f32"),
        # a mixed batch: chunks of up to 256 tokens beside decoding sequences, 8-bit float cache
        _attn("attn_mixed_f8", 24, 256, 2048, 32, 8, 128, 32, "f8", "bf16", True),
        # one token for one sequence of GPT-2's vocabulary, every filter on
        _sample("sample_one", 1, 50257, "f32", 50, 0.9, 0.05),
        # a token for each of 128 sequences over a large vocabulary, nucleus only
        _sample("sample_batch", 128, 128000, "bf16", 0, 0.95, 0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "kv", "attn", "attn", "attn", "sample"])
    dh = rng.choice([32, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    if op == "rope":
        c = _rope("", _log(rng, 1, 8192), rng.choice([2, 5, 12, 24, 40]), dh, rng.choice([dh, dh, dh // 2, dh // 4 + 2]),
                  rng.choice(["pairs", "halves"]), rng.choice(["none", "linear", "yarn"]), rng.choice(["f32", "bf16"]),
                  _log(rng, 64, 131072))
    elif op == "kv":
        dtype = rng.choice(["f32", "bf16"])
        b, ctx = rng.randint(1, 64), _log(rng, 8, 4096)
        ctx = max(1, min(ctx, 16384 * 8 // (b * kv_heads)))
        new = rng.choice([1, _log(rng, 1, ctx), ctx])
        c = _kv("", b, new, ctx, kv_heads, dh, rng.choice([8, 16, 20, 64, 256]), rng.choice(["f32", "bf16", "i8", "f8"]), dtype,
                rng.choice(["new", "all"]), rng.random() < 0.3)
    elif op == "attn":
        dtype = rng.choice(["f32", "bf16"])
        cache = rng.choice(["f32", "bf16", "i8", "f8"] if dtype == "f32" else ["bf16", "i8", "f8"])
        group = rng.choice([1, 1, 2, 3, 4, 7, 8])
        if rng.random() < 0.55:
            b, new, ctx = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 65536)
        else:
            b, new, ctx = rng.randint(1, 16), _log(rng, 2, 512), _log(rng, 512, 8192)
        while b * kv_heads * ctx * dh * BYTES[cache] * 2 > (1 << 29) or b * kv_heads * group * new * ctx > (1 << 27):
            b, ctx = max(1, b * 3 // 4), max(1, ctx * 3 // 4)
        c = _attn("", b, min(new, ctx), ctx, kv_heads * group, kv_heads, dh, rng.choice([8, 16, 20, 64, 256]), cache, dtype,
                  rng.random() < 0.3)
    else:
        vocab = _log(rng, 256, 131072)
        c = _sample("", max(1, min(_log(rng, 1, 256), (1 << 24) // vocab)), vocab, rng.choice(["f32", "bf16"]),
                    rng.choice([0, 0, 1, 20, 64, 1000]), rng.choice([1.0, 0.5, 0.8, 0.95]), rng.choice([0.0, 0.0, 0.02, 0.1]))
    c.pop("name")
    return c


def _lens(c):
    """(new tokens, length with them) of each sequence: spread over the range by the case alone."""
    new, lens = [], []
    for i in range(c["b"]):
        t = (i * 0.6180339887498949) % 1.0
        n = max(1, c["new"] - int(t * c["new"] / 2))
        if c["mixed"] and i % 3:
            n = 1
        new.append(n)
        lens.append(max(n, c["ctx"] - int(t * c["ctx"] * 3 / 4)))
    return new, lens


# ------------------------------------------------------------------ inputs
def _gen(seed, k):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 64 + k)
    return g


def _normal(seed, k, shape, std=1.0):
    return torch.randn(shape, generator=_gen(seed, k), device=DEV, dtype=torch.float32).mul_(std)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _sums(v):
    return np.concatenate([[0], np.cumsum(v)]).astype(np.int32).tolist()


def _freqs(c):
    """Radians per position of each turning pair, in 64 bits, and the magnitude of cos and sin."""
    rot, theta, factor, orig = c["rot"], 10000.0, 16.0, 4096.0
    i = np.arange(rot // 2, dtype=np.float64)
    f = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "yarn":
        dim = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _pool(c, seed, k, pages):
    """One pool of the cache [pages, kv_heads, page, dh] and its scales, of normal values stored as the case's type."""
    x = _normal(seed, k, (pages, c["kv_heads"], c["page"], c["dh"]))
    if c["cache"] not in QMAX:
        return x.to(TYPES[c["cache"]]), None
    s = x.abs().amax(-1) / QMAX[c["cache"]]
    x /= s[..., None]
    return (x.round_().to(torch.int8) if c["cache"] == "i8" else x.to(torch.float8_e4m3fn)), s


def prepare(case, seed):
    c, op = dict(case), case["op"]
    s = {"case": c}
    if op == "rope":
        f, m = _freqs(c)
        s.update(x=_normal(seed, 0, (c["n"], c["heads"], c["dh"])).to(TYPES[c["dtype"]]), freq=torch.from_numpy(f).to(DEV), mscale=m,
                 pos=torch.randint(0, c["far"], (c["n"],), generator=_gen(seed, 1), device=DEV, dtype=torch.int32))
        s["y"] = torch.empty_like(s["x"])
    elif op == "sample":
        n = c["n"]
        uniform = lambda k: torch.rand(n, generator=_gen(seed, k), device=DEV)  # noqa: E731
        s.update(x=_normal(seed, 0, (n, c["vocab"]), 2.5).to(TYPES[c["dtype"]]), u=uniform(1), temp=uniform(2) * 0.8 + 0.4,
                 top_k=torch.full((n,), c["top_k"], dtype=torch.int32, device=DEV), top_p=torch.full((n,), c["top_p"], device=DEV),
                 min_p=torch.full((n,), c["min_p"], device=DEV), ids=torch.empty(n, dtype=torch.int32, device=DEV),
                 logp=torch.empty(n, device=DEV))
    else:
        new, lens = _lens(c)
        n, page = sum(new), c["page"]
        need = [-(-v // page) for v in lens]
        pages, width = sum(need) + 3, max(need)
        order = torch.randperm(pages, generator=_gen(seed, 0), device=DEV).to(torch.int32)
        at = torch.arange(width, device=DEV)[None] + _ints(_sums(need)[:-1])[:, None].long()
        s.update(table=order[at.clamp_max(pages - 1)].contiguous(), cu=_ints(_sums(new)), lens=_ints(lens), n=n, longest=max(lens),
                 most=max(new))
        s["k"], s["k_scale"] = _pool(c, seed, 1, pages)
        s["v"], s["v_scale"] = _pool(c, seed, 2, pages)
        if op == "kv":
            m = sum(lens) if c["read"] == "all" else n
            s.update(k_new=_normal(seed, 3, (n, c["kv_heads"], c["dh"])).to(TYPES[c["dtype"]]),
                     v_new=_normal(seed, 4, (n, c["kv_heads"], c["dh"])).to(TYPES[c["dtype"]]), cu_read=_ints(_sums(lens if c["read"] == "all" else new)))
            s.update(k_out=torch.empty(m, c["kv_heads"], c["dh"], dtype=TYPES[c["dtype"]], device=DEV))
            s["v_out"] = torch.empty_like(s["k_out"])
        else:
            s["q"] = _normal(seed, 3, (n, c["heads"], c["dh"]), 2.0).to(TYPES[c["dtype"]])
            s["o"] = torch.empty_like(s["q"])
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_rope(s):
    c, x = s["case"], s["x"].float()
    a = s["pos"].double()[:, None] * s["freq"]
    cs, sn = (torch.cos(a) * s["mscale"]).float()[:, None], (torch.sin(a) * s["mscale"]).float()[:, None]
    r, h = c["rot"], c["rot"] // 2
    p, q = (x[..., 0:r:2], x[..., 1:r:2]) if c["layout"] == "pairs" else (x[..., :h], x[..., h:r])
    y = (p * cs - q * sn, p * sn + q * cs)
    y = torch.stack(y, -1).flatten(-2) if c["layout"] == "pairs" else torch.cat(y, -1)
    return torch.cat((y, x[..., r:]), -1).to(s["x"].dtype)


def _slots(s, cu):
    """Page and slot of the tokens that cu counts: the last cu[b + 1] - cu[b] of each sequence."""
    n = s["k_out"].shape[0] if cu is s["cu_read"] else s["n"]
    i = torch.arange(n, device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), i.int(), right=True)
    pos = s["lens"][b].long() - cu[b + 1].long() + i
    return s["table"][b, pos // s["case"]["page"]].long(), pos % s["case"]["page"]


def _stored(x, kind):
    """fp32 rows as the cache holds them: (values in 64 bits before the type, scales)."""
    s = (x.abs().amax(-1).double() / QMAX[kind]).float()
    t = (x.double() / s.double()[..., None]).nan_to_num_(0.0)
    if kind == "i8":
        return t.round_(), s
    step = torch.exp2((torch.frexp(t)[1] - 4).clamp_min(-9).double())  # 2^-3 of the value's power of two
    return (t / step).round_() * step, s


def _write(s, name, page, slot):
    kind, pool, x = s["case"]["cache"], s[name], s[name + "_new"]
    if kind not in QMAX:
        pool[page, :, slot] = x.to(pool.dtype)
        return
    t, sc = _stored(x.float(), kind)
    t = t.float().to(pool.dtype)  # exact: whole numbers, or values of the 8-bit type
    pool.view(torch.uint8)[page, :, slot] = t.view(torch.uint8)
    s[name + "_scale"][page, :, slot] = sc


def _read(s, name, page, slot):
    t = s[name].view(torch.uint8)[page, :, slot].view(s[name].dtype).float() if s["case"]["cache"] == "f8" else s[name][page, :, slot].float()
    if s[name + "_scale"] is not None:
        t = t * s[name + "_scale"][page, :, slot][..., None]
    return t.to(s[name + "_new"].dtype)


def _plain_kv(s):
    at = _slots(s, s["cu"])
    _write(s, "k", *at)
    _write(s, "v", *at)
    at = _slots(s, s["cu_read"])
    got = {"k": _read(s, "k", *at), "v": _read(s, "v", *at)}
    return {**got, "k_scale": s["k_scale"], "v_scale": s["v_scale"]} if s["k_scale"] is not None else got


def _plain_attn(s):
    c = s["case"]
    b, hk, g, dh, page, m = c["b"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dh"], c["page"], s["most"]
    width = s["table"].shape[1]
    cu, lens = s["cu"].long(), s["lens"].long()

    def dense(pool, scale):  # [b, kv_heads, keys, dh]
        t = pool.view(torch.uint8)[s["table"].long()].view(pool.dtype).float() if c["cache"] == "f8" else pool[s["table"].long()].float()
        if scale is not None:
            t = t * scale[s["table"].long()][..., None]
        return t.transpose(1, 2).reshape(b, hk, width * page, dh)

    i, j = torch.arange(m, device=DEV), torch.arange(width * page, device=DEV)
    count = cu[1:] - cu[:-1]
    row = cu[:-1, None] + i  # [b, m]: rows of q, past the last where a sequence has fewer new tokens
    row = torch.where(i < count[:, None], row, s["n"])
    q = torch.cat((s["q"].float(), torch.zeros(1, c["heads"], dh, device=DEV)))[row]  # [b, m, heads, dh]
    q = q.reshape(b, m, hk, g, dh).permute(0, 2, 1, 3, 4).reshape(b, hk, m * g, dh)
    sc = torch.matmul(q, dense(s["k"], s["k_scale"]).transpose(-1, -2).contiguous()).view(b, hk, m, g, -1).mul_(1.0 / math.sqrt(dh))
    sees = j <= (lens - count)[:, None, None] + i[:, None]  # [b, m, keys]
    sc.masked_fill_(~sees[:, None, :, None], -math.inf)
    sc -= sc.amax(-1, keepdim=True)
    sc.exp_()
    total = sc.sum(-1, keepdim=True)
    v = dense(s["v"], s["v_scale"])
    v = torch.where((j < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(sc.view(b, hk, m * g, -1), v).view(b, hk, m, g, dh) / total
    out = torch.empty(s["n"] + 1, c["heads"], dh, device=DEV)
    out[row] = o.permute(0, 2, 1, 3, 4).reshape(b, m, c["heads"], dh)
    return out[: s["n"]].to(s["q"].dtype)


def _plain_sample(s):
    x = s["x"].double()
    top, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((top - top[:, :1]) / s["temp"].double()[:, None])
    rank = torch.arange(x.shape[1], device=DEV)
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = torch.cumsum(w, -1) - w
    keep = (before < s["top_p"].double()[:, None] * w.sum(-1, keepdim=True)) | (rank == 0)
    w = torch.where(keep & (w >= s["min_p"].double()[:, None]), w, 0.0)
    p = torch.zeros_like(w).scatter_(1, idx, w)
    run_ = torch.cumsum(p, -1)
    total = run_[:, -1:]
    ids = ((run_ > s["u"].double()[:, None] * total) & (p > 0)).int().argmax(-1)
    logp = torch.log(p.gather(1, ids[:, None]) / total)[:, 0]
    return {"ids": ids.int(), "logp": logp.float()}


# ------------------------------------------------------------------ the library's calls
def _workspace(size, kept=[]):  # (one for all calls: they follow each other on the library's stream)
    """Memory of the library's allocation: torch hands back blocks that its own stream's kernels may still use, and nothing
    orders those with the library's stream."""
    from jasmine_amd.capi import DeviceArray
    if not kept or kept[0].nbytes < size:
        kept[:] = [DeviceArray(max(1, size), np.uint8)]
    return kept[0]


def _own(s):
    from jasmine_amd.capi import PagedKv, check, lib
    c, op = s["case"], s["case"]["op"]
    p = lambda n: s[n].data_ptr()  # noqa: E731
    if op == "rope":
        h, d = c["heads"], c["dh"]
        check(lib.jas_rope(p("x"), p("y"), p("pos"), p("freq"), c["n"], h, d, c["rot"], h * d, d, h * d, d,
                           int(c["layout"] == "halves"), s["mscale"], CODES[c["dtype"]], None))
        return s["y"]
    if op == "sample":
        n, v = c["n"], c["vocab"]
        if "work" not in s:
            s["work"] = _workspace(lib.jas_sample_workspace(n, v))
        check(lib.jas_sample(p("x"), n, v, v, p("temp"), p("top_k"), p("top_p"), p("min_p"), p("u"), p("ids"), p("logp"),
                             CODES[c["dtype"]], s["work"].p, None))
        return {"ids": s["ids"], "logp": s["logp"]}
    hk, d, page, eight = c["kv_heads"], c["dh"], c["page"], c["cache"] in QMAX
    if "kv" not in s:
        s["kv"] = PagedKv(p("k"), p("v"), p("k_scale") if eight else None, p("v_scale") if eight else None, p("table"),
                          hk * page * d, page * d, d, s["table"].shape[1], s["table"].shape[1], CODES[c["cache"]],
                          s["k"].shape[0], page, hk, d)
    kv = C.byref(s["kv"])
    if op == "kv":
        t = CODES[c["dtype"]]
        check(lib.jas_kv_append(kv, p("k_new"), p("v_new"), s["n"], hk * d, d, c["b"], p("cu"), p("lens"), t, None))
        check(lib.jas_kv_read(kv, p("k_out"), p("v_out"), s["k_out"].shape[0], hk * d, d, c["b"], p("cu_read"), p("lens"), t, None))
        return {"k": s["k_out"], "v": s["v_out"], **({"k_scale": s["k_scale"], "v_scale": s["v_scale"]} if eight else {})}
    h = c["heads"]
    if "work" not in s:
        s["work"] = _workspace(lib.jas_attn_paged_workspace(s["n"], c["b"], h, hk, d, s["most"], s["longest"]))
    check(lib.jas_attn_paged(p("q"), p("o"), kv, s["n"], c["b"], p("cu"), p("lens"), h, s["most"], s["longest"], h * d, d, h * d, d,
                             1.0 / math.sqrt(d), 1, CODES[c["dtype"]], s["work"].p, None))
    return s["o"]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "kv": _plain_kv, "attn": _plain_attn, "sample": _plain_sample}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, op = case, case["op"]
    if op == "rope":
        n = c["n"] * c["heads"]
        return {"bytes": 2 * n * c["dh"] * BYTES[c["dtype"]] + 4 * c["n"], "flops": 3 * n * c["rot"]}
    if op == "sample":  # maximum, weight, sums and comparisons of each logit
        n = c["n"] * c["vocab"]
        return {"bytes": n * BYTES[c["dtype"]] + 28 * c["n"], "flops": 8 * n}
    new, lens = _lens(c)
    row = c["kv_heads"] * (c["dh"] * BYTES[c["cache"]] + (4 if c["cache"] in QMAX else 0))
    if op == "kv":
        m = sum(lens) if c["read"] == "all" else sum(new)
        io = c["kv_heads"] * c["dh"] * BYTES[c["dtype"]]
        return {"bytes": 2 * (sum(new) + m) * (row + io), "flops": 6 * (sum(new) + m) * c["kv_heads"] * c["dh"]}
    pairs = sum(n * (v - n) + n * (n + 1) // 2 for n, v in zip(new, lens))
    return {"bytes": 2 * sum(lens) * row + 2 * sum(new) * c["heads"] * c["dh"] * BYTES[c["dtype"]],
            "flops": 4 * pairs * c["heads"] * c["dh"]}


# ------------------------------------------------------------------ the same results in 64 bits
def _exact_rope(c, s):
    x = s["x"].double()
    out, r = x.clone(), c["rot"]
    z = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["freq"])[:, None]
    first = torch.arange(0, r, 2) if c["layout"] == "pairs" else torch.arange(r // 2)
    second = first + (1 if c["layout"] == "pairs" else r // 2)
    turned = torch.complex(x[..., first], x[..., second]) * z
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _exact_kv(c, s):
    """Host arithmetic on one sequence at a time."""
    new, lens = _lens(c)
    cu, table, page = _sums(new), s["table"].cpu().numpy(), c["page"]
    got = {}
    for name in ("k", "v"):
        pool = s[name].float().cpu().numpy().astype(np.float64)
        scale = s[name + "_scale"].cpu().numpy().copy() if c["cache"] in QMAX else None
        x = s[name + "_new"].float().cpu().numpy()
        rows = []
        for b in range(c["b"]):
            at = np.arange(lens[b])
            pg, sl = table[b, at // page], at % page
            y = x[cu[b]:cu[b + 1]]
            t = slice(lens[b] - new[b], lens[b])
            if c["cache"] in QMAX:
                sc = (np.abs(y).max(-1) / np.float32(QMAX[c["cache"]])).astype(np.float32)
                y = y.astype(np.float64) / sc.astype(np.float64)[..., None]
                if c["cache"] == "i8":
                    y = np.rint(y)
                else:
                    _, e = np.frexp(y)
                    step = np.ldexp(1.0, np.maximum(e - 4, -9))
                    y = np.rint(y / step) * step
                scale[pg[t], :, sl[t]] = sc
            elif c["cache"] == "bf16":
                y = torch.from_numpy(y).bfloat16().double().numpy()
            pool[pg[t], :, sl[t]] = y
            r = pool[pg, :, sl] * (scale[pg, :, sl].astype(np.float64)[..., None] if c["cache"] in QMAX else 1.0)
            rows.append(r if c["read"] == "all" else r[t])
        got[name] = np.concatenate(rows)
        if scale is not None:
            got[name + "_scale"] = scale.astype(np.float64)
    return got


def _exact_attn(c, s):
    new, lens = _lens(c)
    g, page, out = c["heads"] // c["kv_heads"], c["page"], []
    q, cu = s["q"].double(), _sums(new)
    for b in range(c["b"]):
        at = torch.arange(lens[b], device=DEV)
        pg, sl = s["table"][b].long()[at // page], at % page

        def rows(pool, scale):
            t = pool.float()[pg, :, sl].double()
            return t * scale[pg, :, sl].double()[..., None] if scale is not None else t

        k, v = rows(s["k"], s["k_scale"]), rows(s["v"], s["v_scale"])
        qb = q[cu[b]:cu[b + 1]]
        last = lens[b] - new[b] + torch.arange(new[b], device=DEV)
        ob = torch.empty_like(qb)
        for h in range(c["heads"]):
            sc = qb[:, h] @ k[:, h // g].T / math.sqrt(c["dh"])
            sc = sc.masked_fill(at[None] > last[:, None], -math.inf)
            ob[:, h] = torch.softmax(sc, -1) @ v[:, h // g]
        out.append(ob)
    return torch.cat(out)


def _exact_sample(c, s):
    """One row at a time, in the order of a sort by value (lowest index first among equals)."""
    n = c["n"]
    x = s["x"].double().cpu().numpy()
    temp, top_p, min_p, u = (s[k].double().cpu().numpy() for k in ("temp", "top_p", "min_p", "u"))
    ids, logp = np.zeros(n, np.int32), np.zeros(n)
    for r in range(n):
        order = np.argsort(-x[r], kind="stable")
        if c["top_k"] > 0:
            order = order[: c["top_k"]]
        w = np.exp((x[r][order] - x[r][order[0]]) / temp[r])
        upto = np.cumsum(w)
        count = 1 + int(np.searchsorted(upto, top_p[r] * upto[-1], side="left"))
        w, order = w[:count], order[:count]
        order, w = order[w >= min_p[r]], w[w >= min_p[r]]
        by = np.argsort(order)
        order, w = order[by], w[by]
        upto = np.cumsum(w)
        k = int(np.searchsorted(upto, u[r] * upto[-1], side="right"))
        ids[r], logp[r] = order[k], math.log(w[k] / upto[-1])
    return {"ids": ids, "logp": logp}


def exact(case, seed):
    c, s = dict(case), prepare(case, seed)
    return {"rope": _exact_rope, "kv": _exact_kv, "attn": _exact_attn, "sample": _exact_sample}[c["op"]](c, s)
