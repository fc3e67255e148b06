"""What is measured of the attention half of a decoder layer: the quantised key / value cache (write and
read back), attention over it, and the norms around a block.

`run` computes each in its plain form with elementary torch operations, or, where `own` is set, through
the package: `kvcache.KVCache.write / read / attend` and `mmvq.norm_block`.

The cache is paged; K and V are each Q4_0 or Q8_0, in blocks of 32 values along the head dimension with
one fp16 scale d (value = d * code):
    Q4_0   d = fp16(m / -8), m the value of largest magnitude (the first), code = clamp(rint(x / d), -8, 7)
    Q8_0   d = fp16(max |x| / 127), code = clamp(rint(x / d), -127, 127)
Bytes of a page of P tokens, J = dim / 32 blocks, b = 4 (Q4_0) or 8 (Q8_0) bytes per 8 values:
    k       [pages][heads][P][4][J][b]           values 8 t .. 8 t + 7 of block j at [t][j]
    v       [pages][heads][P / 2][8][J][b / 4][2][2]   tokens 2 i and 2 i + 1 side by side, values 4 g .. 4 g + 3
    scales  [pages][heads][P][2][J] fp16         K's scales, then V's
Codes are stored with 8 (Q4_0) or 128 (Q8_0) added.  Eight K values n0 .. n7 lie in their bytes as
(n0, n2), (n4, n6), (n1, n3), (n5, n7) for Q4_0 (low nibble first) and n0 n2 n1 n3 n4 n6 n5 n7 for Q8_0;
a token's four V values as (n0, n1), (n2, n3).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BITS = {"Q4_0": 4.5, "Q8_0": 8.5}


# ---- the cases -----------------------------------------------------------------------------------

def _attend(name, dtype, seqs, new, ctx, hq, hkv, dim, page, kf, vf, window=0):
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "new": new, "ctx": ctx, "hq": hq, "hkv": hkv,
            "dim": dim, "page": page, "kf": kf, "vf": vf, "window": window}


def _store(name, dtype, rows, hq, hkv, dim, page, kf, vf, rope):
    return {"name": name, "op": "store", "dtype": dtype, "rows": rows, "hq": hq, "hkv": hkv, "dim": dim, "page": page,
            "kf": kf, "vf": vf, "rope": rope}


def _norm(name, dtype, rows, n, gate, post):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "n": n, "gate": gate, "post": post}


def listed():
    return [
        # a chat's first answer tokens: one sequence, a short prompt behind it; latency alone
        _attend("token_short", "f32", 1, 1, 77, 32, 8, 128, 64, "Q4_0", "Q4_0"),
        # one user with a long document in the cache, fp32 queries as the matvecs give them
        _attend("token_long", "f32", 1, 1, 65519, 32, 8, 128, 64, "Q4_0", "Q4_0"),
        # a serving batch of unequal lengths
        _attend("token_batch", "bf16", 64, 1, 8191, 32, 8, 128, 64, "Q4_0", "Q4_0"),
        # a small model with 7 query heads a key head, a sliding window, keys kept in 8 bits, small pages
        _attend("token_window", "f16", 16, 1, 16385, 14, 2, 64, 16, "Q8_0", "Q4_0", 4096),
        # drafted tokens of several sequences checked at once, 8-bit cache
        _attend("draft", "bf16", 8, 5, 4099, 32, 4, 128, 32, "Q8_0", "Q8_0"),
        # an ordinary prompt
        _attend("prompt", "bf16", 1, 517, 517, 32, 8, 128, 64, "Q4_0", "Q4_0"),
        # prompts of several users behind what their caches hold already, wide heads, a window
        _attend("prompt_ragged", "bf16", 6, 1500, 6001, 16, 8, 256, 64, "Q8_0", "Q4_0", 1024),
        # a whole document
        _attend("prompt_long", "bf16", 1, 8192, 8192, 32, 8, 128, 64, "Q4_0", "Q4_0"),
        # the new token of each sequence of a batch, rotated and written, the queries rotated with it
        _store("store_token", "f32", 64, 32, 8, 128, 64, "Q4_0", "Q4_0", "half"),
        # a long prompt's keys and values
        _store("store_prompt", "bf16", 16381, 32, 8, 128, 64, "Q8_0", "Q4_0", "pairs"),
        # the norms around a block of a decode step
        _norm("norm_token", "f32", 1, 4096, False, True),
        # ... and of a long prompt, with a gate per channel and token
        _norm("norm_prompt", "bf16", 8192, 4096, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["token", "token", "draft", "prompt", "store", "norm"])
    dim = rng.choice([64, 96, 128, 128, 256])
    hkv, group = rng.choice([(8, 4), (4, 8), (2, 7), (1, 8), (16, 1), (4, 2), (2, 16), (5, 3)])
    page = rng.choice([16, 32, 64, 128, 256])
    kf, vf = rng.choice(["Q4_0", "Q8_0"]), rng.choice(["Q4_0", "Q8_0"])
    if kind in ("token", "draft"):
        seqs = _log(rng, 1, 64)
        most = min(65536, 64 * 8192 * 8 * 128 // (seqs * hkv * dim * (2 if "Q8_0" in (kf, vf) else 1)))
        ctx = _log(rng, 1, most)
        new = 1 if kind == "token" else rng.randint(2, 16)
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        return _attend("", rng.choice(list(DTYPES)), seqs, min(new, ctx), ctx, hkv * group, hkv, dim, page, kf, vf, window)
    if kind == "prompt":
        seqs = rng.randint(1, 4)
        new = _log(rng, 17, 8192 // seqs)
        ctx = min(8192, new + _log(rng, 1, 8192) - 1)
        while seqs * new * ctx * hkv * group * dim > 8192 * 8192 * 32 * 128 // 2:
            new, ctx = (new + 1) // 2, (ctx + 1) // 2
        dtype = "f32" if new <= 512 and rng.random() < 0.25 else "bf16"
        return _attend("", dtype, seqs, min(new, ctx), ctx, hkv * group, hkv, dim, page, kf, vf,
                       rng.choice([0, 0, _log(rng, 16, 8192)]))
    if kind == "store":
        rows = _log(rng, 1, min(16384, 16384 * 48 * 128 // (hkv * (group + 2) * dim)))
        return _store("", rng.choice(list(DTYPES)), rows, hkv * group, hkv, dim, page, kf, vf,
                      rng.choice(["none", "half", "pairs"]))
    n = _log(rng, 64, 16384)
    rows = _log(rng, 1, max(1, 8192 * 4096 // (2 * n)))
    return _norm("", rng.choice(list(DTYPES)), rows, n, rng.random() < 0.5, rng.random() < 0.7)


def _lengths(case):
    """(keys in the cache, new tokens among them) of each sequence: the first has the most, the others between
    a fifth and all of it."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"])
    keys = [case["ctx"]] + [r.randint((case["ctx"] + 4) // 5, case["ctx"]) for _ in range(case["seqs"] - 1)]
    if case["new"] <= 16:
        new = [min(case["new"], k) for k in keys]
    else:
        new = [case["new"]] + [min(k, r.randint((case["new"] + 4) // 5, case["new"])) for k in keys[1:]]
    return keys, new


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attend":
        row = case["hkv"] * case["dim"] * (BITS[case["kf"]] + BITS[case["vf"]]) / 8
        nbytes = pairs = 0
        for length, new in zip(*_lengths(case)):
            w = case["window"] or length
            first = max(0, length - new - w + 1)
            nbytes += (length - first) * row + 2 * new * case["hq"] * case["dim"] * e
            # query i sees min(w, length - new + i + 1) keys
            full = max(0, min(new, length - w + 1)) if length >= w else 0
            short = new - full
            pairs += full * w + short * (length - new + 1) + short * (short - 1) // 2
        return {"bytes": int(nbytes), "flops": int(4 * pairs * case["hq"] * case["dim"])}
    if case["op"] == "store":
        kv = 2 * case["hkv"] * case["dim"]
        held = case["hkv"] * case["dim"] * (BITS[case["kf"]] + BITS[case["vf"]]) / 8
        rope = case["rope"] != "none"
        q = 2 * case["hq"] * case["dim"] * e + case["dim"] * 4 if rope else 0
        # the values read, the codes written and read again, the values written back, the queries both ways
        return {"bytes": int(case["rows"] * (2 * kv * e + 2 * held + q)),
                "flops": int(case["rows"] * (kv * 6 + (3 * (kv // 2 + case["hq"] * case["dim"]) if rope else 0)))}
    one = case["rows"] * case["n"]
    return {"bytes": one * e * (5 if case["gate"] else 4) + case["n"] * (8 if case["post"] else 4), "flops": 12 * one}


# ---- the cache's values and bytes in plain operations ---------------------------------------------

def _quantise(x, fmt):
    """x (..., dim) fp32 -> (codes (..., J, 32) int32 without offset, d (..., J) fp16)."""
    b = torch.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    mag = b.abs()
    if fmt == "Q4_0":
        m = b.gather(-1, mag.argmax(-1, keepdim=True))[..., 0]
        d, lo, hi = (m * -0.125).half(), -8, 7
    else:
        amax = mag.amax(-1)
        d, lo, hi = (amax / torch.full_like(amax, 127.0)).half(), -127, 127
    df = d.float()[..., None]
    q = torch.where(df == 0, torch.zeros_like(b), b / torch.where(df == 0, torch.ones_like(df), df))
    return q.round().clamp(lo, hi).to(torch.int32), d


_K_NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]     # the value at each nibble, low nibble of byte 0 first
_K_BYTES = [0, 2, 1, 3, 4, 6, 5, 7]       # the value at each byte
_INV = {tuple(p): [p.index(i) for i in range(8)] for p in (_K_NIBBLES, _K_BYTES)}


def _nibbles(c):
    """(..., 2 n) values 0..15 -> (..., n) bytes, low nibble first."""
    p = c.unflatten(-1, (-1, 2))
    return (p[..., 0] | (p[..., 1] << 4)).to(torch.uint8)


def _split(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _pack_k(c, fmt):
    """codes (..., J, 32) -> bytes (..., 4, J, b)."""
    x = c.unflatten(-1, (4, 8)).transpose(-3, -2)
    return _nibbles((x + 8)[..., _K_NIBBLES]) if fmt == "Q4_0" else (x + 128)[..., _K_BYTES].to(torch.uint8)


def _unpack_k(b, fmt):
    """bytes (..., 4, J, b) -> values' codes (..., J, 32) fp32."""
    x = _split(b)[..., _INV[tuple(_K_NIBBLES)]] if fmt == "Q4_0" else b[..., _INV[tuple(_K_BYTES)]]
    return x.transpose(-3, -2).flatten(-2).float() - (8.0 if fmt == "Q4_0" else 128.0)


def _pack_v(c, fmt):
    """codes (..., J, 32) -> one token's bytes (..., 8, J, b / 4, 2)."""
    x = c.unflatten(-1, (8, 4)).transpose(-3, -2)
    return (_nibbles(x + 8) if fmt == "Q4_0" else (x + 128).to(torch.uint8)).unflatten(-1, (-1, 2))


def _unpack_v(b, fmt):
    """one token's bytes (..., 8, J, b / 4, 2) -> codes (..., J, 32) fp32."""
    x = b.flatten(-2)
    x = _split(x) if fmt == "Q4_0" else x
    return x.transpose(-3, -2).flatten(-2).float() - (8.0 if fmt == "Q4_0" else 128.0)


def _width(fmt):
    return 4 if fmt == "Q4_0" else 8


def _buffers(case, pages, device):
    """Empty cache tensors, in the shapes named above (codes flat behind the token)."""
    h, p, d = case["hkv"], case["page"], case["dim"]
    k = torch.zeros(pages, h, p, d * _width(case["kf"]) // 8, dtype=torch.uint8, device=device)
    v = torch.zeros(pages, h, p // 2, d * _width(case["vf"]) // 4, dtype=torch.uint8, device=device)
    return k, v, torch.zeros(pages, h, p, 2, d // 32, dtype=torch.float16, device=device)


def _k_view(st):
    return st["k_codes"].unflatten(-1, (4, st["dim"] // 32, _width(st["kf"])))


def _v_view(st):
    return st["v_codes"].unflatten(-1, (8, st["dim"] // 32, _width(st["vf"]) // 4, 2, 2))


def _put(st, k, v, slots):
    """Quantises k and v (rows, heads, dim) fp32 into the slots' places."""
    page, at = slots // st["page"], slots % st["page"]
    for name, x, fmt in (("k", k, st["kf"]), ("v", v, st["vf"])):
        c, d = _quantise(x, fmt)
        st["scales"][page, :, at, 0 if name == "k" else 1] = d
        if name == "k":
            _k_view(st)[page, :, at] = _pack_k(c, fmt)
        else:
            _v_view(st)[page, :, at // 2, :, :, :, at % 2] = _pack_v(c, fmt)


def _get(st, slots):
    """The values (rows, heads, dim) fp32 at the slots."""
    page, at = slots // st["page"], slots % st["page"]
    s = st["scales"][page, :, at].float()
    k = _unpack_k(_k_view(st)[page, :, at], st["kf"]) * s[:, :, 0, :, None]
    v = _unpack_v(_v_view(st)[page, :, at // 2, :, :, :, at % 2], st["vf"]) * s[:, :, 1, :, None]
    return k.flatten(-2), v.flatten(-2)


def _rotate(x, cos, sin, style):
    """x (rows, heads, dim) fp32, cos and sin (rows, dim / 2): the pairs (i, i + dim / 2) or (2 i, 2 i + 1)."""
    c, s = cos[:, None], sin[:, None]
    if style == "half":
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)


# ---- inputs -----------------------------------------------------------------------------------------

def _channels(g, dim, device):
    """Per-channel sizes of keys: mostly alike, a few channels far above, as trained keys have."""
    w = torch.exp(0.3 * torch.randn(dim, generator=g, device=device))
    w[torch.randint(0, dim, (3,), generator=g, device=device)] *= 4.0
    return w


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "norm":
        n, rows = case["n"], case["rows"]
        return {"op": "norm", "y": (3.0 * randn(rows, n)).to(dt), "h": (8.0 * randn(rows, n)).to(dt),
                "gate": torch.sigmoid(randn(rows, n)).to(dt) if case["gate"] else None,
                "w_post": 1.0 + 0.2 * randn(n) if case["post"] else None, "w_pre": 1.0 + 0.2 * randn(n),
                "eps": 1e-6, "rs": 0.7}

    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    st = {"op": case["op"], "page": page, "dim": dim, "kf": case["kf"], "vf": case["vf"]}
    wk = _channels(g, dim, dev)
    if case["op"] == "store":
        rows = case["rows"]
        pages = (2 * rows + page - 1) // page
        # rows of sequences that lie in pages of any order: whole runs, each at its own place
        run = min(page, rows)
        start = torch.randperm((pages * page) // run, generator=g, device=dev)[: (rows + run - 1) // run] * run
        st["slots"] = (start[:, None] + torch.arange(run, device=dev)).flatten()[:rows].contiguous()
        st["k"], st["v"] = (randn(rows, hkv, dim) * wk).to(dt), randn(rows, hkv, dim).to(dt)
        st["q"], st["rope"] = None, case["rope"]
        if case["rope"] != "none":
            st["q"] = randn(rows, hq, dim).to(dt)
            angle = torch.arange(32768, device=dev, dtype=torch.float64)[:, None] * torch.pow(
                torch.tensor(5e5, device=dev, dtype=torch.float64),
                -torch.arange(0, dim, 2, device=dev, dtype=torch.float64) / dim)
            st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
            st["positions"] = torch.randint(0, 32768, (rows,), generator=g, device=dev)
        st["k_codes"], st["v_codes"], st["scales"] = _buffers(case, pages, dev)
    else:
        keys, new = _lengths(case)
        per = [(k + page - 1) // page for k in keys]
        pages = sum(per) + 3
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        tables = torch.full((len(keys), max(per)), -1, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(per):
            tables[b, :n] = order[at:at + n]
            at += n
        st["k_codes"], st["v_codes"], st["scales"] = _buffers(case, pages, dev)
        step = max(1, (1 << 27) // (hkv * dim * page))
        for p0 in range(0, pages, step):                       # what the cache holds: quantised keys and values
            n = min(step, pages - p0) * page
            _put(st, (randn(n, hkv, dim) * wk).bfloat16().float(), randn(n, hkv, dim).bfloat16().float(),
                 torch.arange(p0 * page, p0 * page + n, device=dev))
        # queries that look at a part of the keys: logits of a standard deviation about 1.5
        st["q"] = (1.5 * randn(sum(new), hq, dim) / wk.square().mean().sqrt()).to(dt)
        st["tables"], st["window"], st["new"] = tables, case["window"], case["new"]
        st["lens"] = torch.tensor(keys, dtype=torch.int32, device=dev)
        st["starts"] = None
        if case["new"] > 1:
            st["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)
        st["news"] = torch.tensor(new, device=dev)
        st["row_seq"] = torch.repeat_interleave(torch.arange(len(new), device=dev), st["news"], output_size=sum(new))
        st["row_at"] = torch.arange(sum(new), device=dev) - (torch.cumsum(st["news"], 0) - st["news"])[st["row_seq"]]
    if own:
        from nemicli_terminal_b200 import kvcache
        st["cache"] = kvcache.KVCache(st["scales"].shape[0], hkv, dim, page, st["kf"], st["vf"],
                                      buffers=(st["k_codes"], st["v_codes"], st["scales"]))
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _plain_norm(st):
    y, h = st["y"].float(), st["h"].float()
    z = y
    if st["w_post"] is not None:
        z = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * st["w_post"]
    if st["gate"] is not None:
        z = z * st["gate"].float()
    new = h + st["rs"] * z
    x = new * torch.rsqrt(new.square().mean(-1, keepdim=True) + st["eps"]) * st["w_pre"]
    return {"x": x.to(st["y"].dtype), "h": new.to(st["h"].dtype)}


def _plain_store(st):
    k, v, q = st["k"].float(), st["v"].float(), st["q"]
    if st["rope"] != "none":
        cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
        k = _rotate(k, cos, sin, st["rope"])
        q = _rotate(q.float(), cos, sin, st["rope"]).to(st["q"].dtype)
    _put(st, k, v, st["slots"])
    k, v = _get(st, st["slots"])
    out = {"k": k.to(st["k"].dtype), "v": v.to(st["k"].dtype)}
    return out if q is None else {**out, "q": q}


def _plain_attend(st):
    """All sequences side by side, each filled up to the longest."""
    q, lens, page = st["q"], st["lens"], st["page"]
    _, hq, dim = q.shape
    seqs, width = st["tables"].shape
    hkv = st["scales"].shape[1]
    at = st["tables"].clamp(min=0).long()
    s = st["scales"][at].float()                                             # (seqs, width, hkv, page, 2, J)
    k = (_unpack_k(_k_view(st)[at], st["kf"]) * s[..., 0, :, None]).flatten(-2)
    v = _unpack_v(_v_view(st)[at].movedim(-2, 4).flatten(3, 4), st["vf"])     # pairs of tokens -> tokens
    v = (v * s[..., 1, :, None]).flatten(-2)
    k = k.transpose(1, 2).reshape(seqs, hkv, width * page, dim)
    v = v.transpose(1, 2).reshape(seqs, hkv, width * page, dim)
    x = torch.zeros(seqs, st["new"], hq, dim, device=q.device)
    x[st["row_seq"], st["row_at"]] = q.float()
    x = x.unflatten(2, (hkv, -1)).permute(0, 2, 1, 3, 4)                      # (seqs, hkv, new, group, dim)
    group = x.shape[3]
    logits = (x.reshape(seqs, hkv, -1, dim) @ k.transpose(-1, -2)).mul_(dim ** -0.5)
    logits = logits.unflatten(2, (-1, group))
    pos = (lens - st["news"])[:, None] + torch.arange(st["new"], device=q.device)         # (seqs, new)
    key = torch.arange(width * page, device=q.device)
    off = key > pos[..., None]
    if st["window"]:
        off = off | (key <= pos[..., None] - st["window"])
    logits = logits.masked_fill_(off[:, None, :, None, :], float("-inf"))
    top = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, group)) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 2, 1, 3, 4).flatten(2, 3)                                # (seqs, new, hq, dim)
    return {"o": o[st["row_seq"], st["row_at"]].to(q.dtype)}


def run(state):
    st = state
    if not own:
        return {"norm": _plain_norm, "store": _plain_store, "attend": _plain_attend}[st["op"]](st)
    if st["op"] == "norm":
        from nemicli_terminal_b200 import mmvq
        x, _, h = mmvq.norm_block(st["y"], st["h"], st["w_pre"], st["eps"], w_post=st["w_post"], gate=st["gate"],
                                  rs=st["rs"])
        return {"x": x, "h": h}
    cache = st["cache"]
    if st["op"] == "store":
        rope = None
        if st["rope"] != "none":
            rope = (st["cos"], st["sin"], st["positions"])
        q = cache.write(st["k"], st["v"], st["slots"], q=st["q"], rope=rope, paired=st["rope"] == "pairs")
        k, v = cache.read(st["slots"], st["k"].dtype)
        return {"k": k, "v": v} if q is None else {"k": k, "v": v, "q": q}
    return {"o": cache.attend(st["q"], st["tables"], st["lens"], starts=st["starts"], max_new=st["new"],
                              window=st["window"])}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _exact_values(raw, fmt, scale, value):
    """Cache bytes (..., bytes) as int64, scale (..., J) -> (..., dim) fp64; `value(i)` names the byte and the bit
    at which value i of a token starts."""
    dim = 32 * scale.shape[-1]
    where = [value(i) for i in range(dim)]
    byte = torch.tensor([w[0] for w in where], device=raw.device)
    bit = torch.tensor([w[1] for w in where], device=raw.device)
    mask, off = (15, 8) if fmt == "Q4_0" else (255, 128)
    code = ((raw[..., byte] >> bit) & mask) - off
    return code.double() * scale.double().repeat_interleave(32, -1)


def _exact_kv(st, pages, b_keys, head):
    """Keys and values of one sequence and head, (keys, dim) fp64."""
    J, dim = st["dim"] // 32, st["dim"]
    sc = st["scales"][pages, head].flatten(0, 1)
    kb = st["k_codes"][pages, head].flatten(0, 1).long()
    if st["kf"] == "Q4_0":
        def k_at(i):
            j, t, e = i // 32, (i % 32) // 8, i % 8
            pair, odd = e // 2, e % 2
            return t * 4 * J + 4 * j + 2 * odd + pair // 2, 4 * (pair % 2)
    else:
        def k_at(i):
            j, t, e = i // 32, (i % 32) // 8, i % 8
            return t * 8 * J + 8 * j + 4 * (e // 4) + 2 * (e % 2) + (e % 4) // 2, 0
    k = _exact_values(kb, st["kf"], sc[:, 0], k_at)
    vb = st["v_codes"][pages, head].flatten(0, 1).long()                      # (pairs, bytes of two tokens)
    halves = []
    for odd in (0, 1):
        if st["vf"] == "Q4_0":
            def v_at(i, odd=odd):
                j, g, e = i // 32, (i % 32) // 4, i % 4
                return (g * J + j) * 4 + 2 * odd + e // 2, 4 * (e % 2)
        else:
            def v_at(i, odd=odd):
                j, g, e = i // 32, (i % 32) // 4, i % 4
                return (g * J + j) * 8 + 4 * (e // 2) + 2 * odd + e % 2, 0
        halves.append(_exact_values(vb, st["vf"], sc[odd::2, 1], v_at))
    v = torch.stack(halves, 1).reshape(-1, dim)
    return k[:b_keys], v[:b_keys]


def _exact_attend(case, st):
    q = st["q"].double()
    hq, dim = q.shape[1:]
    hkv = st["scales"].shape[1]
    group, page = hq // hkv, st["page"]
    out = torch.zeros_like(q)
    row = 0
    for b, (keys, new) in enumerate(zip(*_lengths(case))):
        pages = st["tables"][b, : (keys + page - 1) // page].long()
        pos = torch.arange(keys - new, keys, device=q.device)[:, None, None]
        key = torch.arange(keys, device=q.device)
        for h in range(hkv):
            k, v = _exact_kv(st, pages, keys, h)
            step = max(1, (1 << 28) // (keys * group))
            for r0 in range(0, new, step):
                r1 = min(new, r0 + step)
                s = q[row + r0:row + r1, h * group:(h + 1) * group] @ k.T / math.sqrt(dim)
                p = pos[r0:r1]
                dead = key > p
                if st["window"]:
                    dead = dead | (p - key >= st["window"])
                s = torch.where(dead, torch.full_like(s, -math.inf), s)
                out[row + r0:row + r1, h * group:(h + 1) * group] = torch.softmax(s, -1) @ v
        row += new
    return {"o": out}


def _exact_store(case, st):
    out = {"k": None, "v": None}
    if case["dtype"] == "bf16":
        # in 8 bits of significand no quotient lies so near a border that its rounding to fp32 could move a code
        for name in ("k", "v") if case["rope"] == "none" else ("v",):
            x = st[name].double().unflatten(-1, (-1, 32))
            if case[name + "f"] == "Q4_0":
                top = torch.where(x.abs().amax(-1) == x.amax(-1), x.amax(-1), x.amin(-1))
                if bool((x.amax(-1) == -x.amin(-1)).any()):                   # the first of two as large: by its place
                    first = x.abs().argmax(-1, keepdim=True)
                    top = x.gather(-1, first)[..., 0]
                d, lo, hi = (top / -8).half().double(), -8, 7
            else:
                d, lo, hi = (x.abs().amax(-1) / 127).float().half().double(), -127, 127
            out[name] = ((x / d[..., None]).round().clamp(lo, hi) * d[..., None]).flatten(-2)
    if case["rope"] != "none":
        x = st["q"].double()
        c, s = st["cos"].double()[st["positions"]][:, None], st["sin"].double()[st["positions"]][:, None]
        y = torch.empty_like(x)
        half = x.shape[-1] // 2
        a, b = (slice(0, half), slice(half, None)) if case["rope"] == "half" else (slice(0, None, 2), slice(1, None, 2))
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
        out["q"] = y
    return out


def _exact_norm(st):
    z, h = st["y"].double(), st["h"].double()
    if st["w_post"] is not None:
        z = z / torch.sqrt((z ** 2).mean(-1, keepdim=True) + st["eps"]) * st["w_post"].double()
    if st["gate"] is not None:
        z = z * st["gate"].double()
    h = h + st["rs"] * z
    return {"x": h / torch.sqrt((h ** 2).mean(-1, keepdim=True) + st["eps"]) * st["w_pre"].double(), "h": h}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "store":
        return _exact_store(case, st)
    return _exact_attend(case, st)
