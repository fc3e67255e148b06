"""What is measured of a serving step around the quantised key / value cache: its page tables and slots, beam search
over them, attention over the pages that a query chooses, and positions of several axes.

`run` computes each in its plain form with elementary torch operations, or, where `own` is set, through the package:
`pages.plan / release / reorder`, `beams.select`, `KVCache.copy / summarise / choose / attend_chosen` and
`KVCache.write` with `axes`.

Pages come from a stack: `free` holds the free pages' numbers, `counts` how many of them count (the last is taken
first) and how many pages were asked for in vain.
    plan     sequence b holds lens[b] tokens and gets new[b]; tokens beyond its table's end are cut.  It needs the pages
             ceil(lens / P) .. ceil((lens + new) / P) - 1, taken in the order of sequences.  Row r of the step is
             token i of sequence b, at position lens[b] + i and slot page * P + position % P.
    release  the pages of sequences that are done go onto the stack, in the order of sequences.
    reorder  beam j of a request goes on from beam parents[j].  Pages that no chosen parent holds are free; of the
             beams that would write to the same last page the first keeps it, the others get a copy: in pages of their own
             request that became free, in order, then from the stack, where what is left over goes first.
    select   the n best of scores[k] + log_softmax(logits[k])[v] of a request's beams, the lowest k V + v first among
             equals.
    bounds   per page, key head and channel the least and largest key, rounded outwards to float16.
    choose   of the pages before a query's own those with the largest max over the group's heads of
             sum_c max(q_c lo_c, q_c hi_c), the first and the last ones always; in the order of the sequence.
The cache's bytes (pages of P tokens, J = dim / 32 blocks, b = 4 for Q4_0 or 8 for Q8_0 bytes of 8 values):
    k       [pages][heads][P][4][J][b]           values 8 t .. 8 t + 7 of block j at [t][j]
    v       [pages][heads][P / 2][8][J][b / 4][2][2]   tokens 2 i and 2 i + 1 side by side, values 4 g .. 4 g + 3
    scales  [pages][heads][P][2][J] fp16         K's scales, then V's; value = scale * (code - offset), offset 8 or 128
Eight K values n0 .. n7 lie in their bytes as (n0, n2), (n4, n6), (n1, n3), (n5, n7) for Q4_0 (low nibble first) and
n0 n2 n1 n3 n4 n6 n5 n7 for Q8_0; a token's four V values as (n0, n1), (n2, n3).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BITS = {"Q4_0": 4.5, "Q8_0": 8.5}
MOST = 3.4028234663852886e38               # the largest float32


# ---- the cases -----------------------------------------------------------------------------------

def _plan(name, seqs, ctx, width, page, prompts, prompt, rows):
    return {"name": name, "op": "plan", "seqs": seqs, "ctx": ctx, "width": width, "page": page, "prompts": prompts,
            "prompt": prompt, "rows": rows}


def _release(name, seqs, ctx, width, page, done):
    return {"name": name, "op": "release", "seqs": seqs, "ctx": ctx, "width": width, "page": page, "done": done}


def _select(name, dtype, reqs, beams, vocab, n):
    return {"name": name, "op": "select", "dtype": dtype, "reqs": reqs, "beams": beams, "vocab": vocab, "n": n}


def _fork(name, reqs, beams, prompt, made, hkv, dim, page, kf, vf):
    return {"name": name, "op": "fork", "reqs": reqs, "beams": beams, "prompt": prompt, "made": made, "hkv": hkv, "dim": dim,
            "page": page, "kf": kf, "vf": vf}


def _bounds(name, seqs, new, ctx, hkv, dim, page, kf):
    return {"name": name, "op": "bounds", "seqs": seqs, "new": new, "ctx": ctx, "hkv": hkv, "dim": dim, "page": page, "kf": kf,
            "vf": "Q4_0"}


def _sparse(name, dtype, seqs, new, ctx, hq, hkv, dim, page, kf, vf, keep, first, last):
    return {"name": name, "op": "sparse", "dtype": dtype, "seqs": seqs, "new": new, "ctx": ctx, "hq": hq, "hkv": hkv,
            "dim": dim, "page": page, "kf": kf, "vf": vf, "keep": keep, "first": first, "last": last}


def _axes(name, dtype, rows, hq, hkv, dim, page, kf, vf, sections, mixed, paired):
    """sections: the frequencies of each axis, as text "time,height,width"; mixed: the axes take turns."""
    return {"name": name, "op": "axes", "dtype": dtype, "rows": rows, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "kf": kf,
            "vf": vf, "sections": sections, "mixed": mixed, "paired": paired}


def listed():
    return [
        # one decode step of a serving batch: a token each, a page now and then
        _plan("plan_token", 64, 8191, 128, 64, 0, 0, 64),
        # a step of a large batch in small pages with new prompts among its sequences, rows filled up to a fixed number
        _plan("plan_mixed", 1021, 4099, 512, 16, 24, 1500, 16384),
        # requests that ended give their pages back
        _release("release", 1021, 8191, 512, 16, 0.25),
        # beam search for one user, fp32 logits as the vocabulary projection gives them
        _select("select_one", "f32", 1, 4, 128256, 8),
        # ... and for many, twice as many candidates as beams so that finished ones can leave
        _select("select_batch", "bf16", 64, 8, 128256, 16),
        # four beams of one answer part and join
        _fork("fork_one", 1, 4, 777, 90, 8, 128, 64, "Q4_0", "Q4_0"),
        # a batch of beams with an 8-bit cache of keys
        _fork("fork_batch", 32, 8, 1000, 160, 8, 128, 64, "Q8_0", "Q4_0"),
        # a long prompt's pages are looked over once, behind the cache's write
        _bounds("bounds_prompt", 1, 32001, 32001, 8, 128, 64, "Q4_0"),
        # one user with a whole book in the cache: 64 of 2048 pages are read
        _sparse("sparse_long", "f32", 1, 1, 131071, 32, 8, 128, 64, "Q4_0", "Q4_0", 64, 1, 2),
        # a serving batch of long, unequal sequences
        _sparse("sparse_batch", "bf16", 64, 1, 16383, 32, 8, 128, 64, "Q4_0", "Q4_0", 32, 1, 2),
        # a token each of sequences that hold pictures: time, height and width in blocks of frequencies
        _axes("axes_token", "f32", 64, 32, 8, 128, 64, "Q4_0", "Q4_0", "16,24,24", False, False),
        # a long prompt of pictures and text, the axes taking turns along the frequencies
        _axes("axes_prompt", "bf16", 16381, 32, 8, 128, 64, "Q8_0", "Q4_0", "24,20,20", True, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "release", "select", "select", "fork", "bounds", "sparse", "sparse", "axes"])
    page = rng.choice([16, 32, 64, 128, 256])
    dim = rng.choice([64, 96, 128, 128, 256])
    hkv, group = rng.choice([(8, 4), (4, 8), (2, 7), (1, 8), (16, 1), (4, 2), (2, 16), (5, 3)])
    kf, vf = rng.choice(["Q4_0", "Q8_0"]), rng.choice(["Q4_0", "Q8_0"])
    if kind in ("plan", "release"):
        seqs, ctx = _log(rng, 1, 1024), _log(rng, 1, 8192)
        width = (ctx + page - 1) // page + rng.randint(1, 128)
        if kind == "release":
            return _release("", seqs, ctx, width, page, rng.choice([0.05, 0.25, 1.0]))
        prompts = rng.choice([0, rng.randint(1, min(seqs, 32))])
        prompt = _log(rng, 1, min(4096, 16384 // max(1, prompts)))
        return _plan("", seqs, ctx, width, page, prompts, prompt, min(16384, seqs + prompts * prompt) + rng.choice([0, 0, 77]))
    if kind == "select":
        reqs, beams = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 5, 8, 16])
        dtype = rng.choice(list(DTYPES))
        vocab = min(_log(rng, 1000, 160000), 64 * 8 * 128256 // (reqs * beams * (2 if dtype == "f32" else 1)))
        return _select("", dtype, reqs, beams, vocab, rng.choice([beams, 2 * beams, 2 * beams]))
    if kind == "fork":
        page = min(page, 128)
        beams = rng.choice([2, 3, 4, 5, 8, 8, 16])
        return _fork("", _log(rng, 1, 256 // beams), beams, _log(rng, 1, 1024), _log(rng, 1, 160),
                     min(hkv, 8), min(dim, 128), page, kf, vf)
    if kind == "bounds":
        seqs = _log(rng, 1, 32)
        new = _log(rng, 1, 32768 // seqs)
        return _bounds("", seqs, new, min(32768 // seqs, new + rng.randint(0, 2000)), min(hkv, 8), min(dim, 128), page, kf)
    if kind == "sparse":
        seqs, new = _log(rng, 1, 64), rng.choice([1, 1, rng.randint(2, 8)])
        most = min(131072, 64 * 16384 * 8 * 128 // (seqs * hkv * dim * (2 if "Q8_0" in (kf, vf) else 1)))
        most = min(most, 64 * 16384 * 8 * page // (seqs * new * hkv * 64))
        ctx = _log(rng, new, most)
        first, last = rng.randint(0, 2), rng.randint(1, 3)
        keep = first + last + _log(rng, 1, max(1, 4096 // page))
        return _sparse("", rng.choice(list(DTYPES)), seqs, new, ctx, hkv * group, hkv, dim, page, kf, vf, keep, first, last)
    rows = _log(rng, 1, min(16384, 16384 * 48 * 128 // (hkv * (group + 2) * dim)))
    rot = rng.choice([dim, dim, dim // 2]) // 2
    a, b = rng.randint(1, rot // 2), rng.randint(1, rot // 4)
    return _axes("", rng.choice(list(DTYPES)), rows, hkv * group, hkv, dim, page, kf, vf, f"{rot - a - b},{a},{b}",
                 rng.random() < 0.5, rng.random() < 0.4)


def _held(case):
    """(tokens held, new ones) of each sequence of a plan; tokens held of each of the others."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"])
    held = [case["ctx"]] + [r.randint(0, case["ctx"]) for _ in range(case["seqs"] - 1)]
    new = [1] * case["seqs"]
    if case["op"] == "plan":
        for b in r.sample(range(case["seqs"]), case["prompts"]):
            new[b] = r.randint((case["prompt"] + 4) // 5, case["prompt"])
            held[b] = r.choice([0, held[b] // 2])
    return held, new


def _lengths(case):
    """(tokens in the cache, new ones among them) of each sequence: the first has the most."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"])
    held = [case["ctx"]] + [r.randint((case["ctx"] + 4) // 5, case["ctx"]) for _ in range(case["seqs"] - 1)]
    if case["op"] == "sparse":
        return held, [min(case["new"], k) for k in held]
    return held, [min(case["new"], held[0])] + [min(k, r.randint((case["new"] + 4) // 5, case["new"])) for k in held[1:]]


def _forks(case):
    """(tokens of each request, parents of its beams)"""
    r = random.Random(case["reqs"] * 1000003 + case["prompt"])
    made = [r.randint(1, case["made"]) for _ in range(case["reqs"])]
    parents = [[min(case["beams"] - 1, int(case["beams"] * r.random() ** 1.5)) for _ in range(case["beams"])] for _ in made]
    return [case["prompt"] + m for m in made], parents


def work(case):
    page = case.get("page")
    if case["op"] in ("plan", "release"):
        held, new = _held(case)
        if case["op"] == "release":
            pages = sum((h + page - 1) // page for h in held) * case["done"]
            return {"bytes": int(9 * case["seqs"] + 8 * pages), "flops": int(case["seqs"] + pages)}
        pages = sum((h + n + page - 1) // page - (h + page - 1) // page for h, n in zip(held, new))
        return {"bytes": int(16 * case["seqs"] + 16 * case["rows"] + 8 * pages), "flops": int(8 * case["rows"])}
    if case["op"] == "select":
        e, one = (4 if case["dtype"] == "f32" else 2), case["reqs"] * case["beams"]
        return {"bytes": int(one * (case["vocab"] * e + 4) + case["reqs"] * case["n"] * 12), "flops": int(3 * one * case["vocab"])}
    if case["op"] == "fork":
        nbytes = 0
        for t, parents in zip(*_forks(case)):
            nbytes += 3 * 4 * case["beams"] * ((t + page - 1) // page)
            if t % page:
                row = case["hkv"] * case["dim"] * (BITS[case["kf"]] + BITS[case["vf"]]) / 8
                nbytes += 2 * (case["beams"] - len(set(parents))) * (t % page) * row
        return {"bytes": int(nbytes), "flops": int(nbytes // 8)}
    if case["op"] == "bounds":
        full = sum(t // page - (t - n) // page for t, n in zip(*_lengths(case)))
        one = case["hkv"] * case["dim"]
        return {"bytes": int(full * one * (page * BITS[case["kf"]] / 8 + 4) + 4), "flops": int(3 * full * one * page + 1)}
    if case["op"] == "sparse":
        e = 4 if case["dtype"] == "f32" else 2
        nbytes = flops = 0
        for t, new in zip(*_lengths(case)):
            seen = set()
            for p in range(t - new, t):
                at = p // page                                          # pages before the query's own
                kept = min(at + 1, case["keep"])
                some = kept < at + 1
                tokens = (kept - 1) * page + p % page + 1
                flops += 4 * tokens * case["hq"] * case["dim"] + (3 * at * case["hq"] * case["dim"] if some else 0)
                seen.add((at if some else 0, tokens))
            bound, tokens = max(s[0] for s in seen), max(s[1] for s in seen)
            nbytes += bound * case["hkv"] * case["dim"] * 4
            nbytes += tokens * case["hkv"] * case["dim"] * (BITS[case["kf"]] + BITS[case["vf"]]) / 8
            nbytes += new * (2 * case["hq"] * case["dim"] * e + 4 * case["hkv"] * case["keep"])
        return {"bytes": int(nbytes), "flops": int(flops)}
    e = 4 if case["dtype"] == "f32" else 2
    kv = 2 * case["hkv"] * case["dim"]
    held = case["hkv"] * case["dim"] * (BITS[case["kf"]] + BITS[case["vf"]]) / 8
    # the values read, the codes written and read again, the values written back, the queries both ways, the angles
    return {"bytes": int(case["rows"] * (2 * kv * e + 2 * held + 2 * case["hq"] * case["dim"] * e + case["dim"] * 4 + 24)),
            "flops": int(case["rows"] * (kv * 6 + 3 * (kv // 2 + case["hq"] * case["dim"])))}


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


def _page_keys(st, pages):
    """The keys (..., heads, P, dim) fp32 of pages (...)."""
    s = st["scales"][pages].float()
    return (_unpack_k(_k_view(st)[pages], st["kf"]) * s[..., 0, :, None]).flatten(-2)


def _page_values(st, pages):
    s = st["scales"][pages].float()
    v = _unpack_v(_v_view(st)[pages].movedim(-2, -5).flatten(-6, -5), st["vf"])    # pairs of tokens -> tokens
    return (v * s[..., 1, :, None]).flatten(-2)


def _outwards(lo, hi):
    """fp32 or fp64 -> fp16, lo downwards and hi upwards, within fp16's finite range."""
    out = []
    for x, up in ((lo, False), (hi, True)):
        x = x.clamp(-65504.0, 65504.0)
        h = x.half()
        bits = h.view(torch.int16).to(torch.int32)
        back = h.to(x.dtype)
        off = back < x if up else back > x
        # the next value in the wanted direction: its bits are one up or down; zero goes to the smallest of that sign
        away = (bits >= 0) == up                                     # magnitude grows in that direction
        there = torch.where(back == 0, torch.full_like(bits, 1 if up else -32767), bits + torch.where(away, 1, -1))
        out.append(torch.where(off, there, bits).to(torch.int16).view(torch.float16).clamp(-65504.0, 65504.0))
    return torch.stack(out, -2)


def _rotate(x, cos, sin, paired):
    """x (rows, heads, dim) fp32, cos and sin (rows, rot / 2): the pairs (i, i + rot / 2) or (2 i, 2 i + 1)."""
    c, s = cos[:, None], sin[:, None]
    rot = 2 * cos.shape[-1]
    head, tail = x[..., :rot], x[..., rot:]
    if paired:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = head.chunk(2, -1)
        head = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((head, tail), -1)


def _axis_of(case):
    """The axis of each frequency: sections one behind the other, or in turns as long as each lasts."""
    sections = [int(n) for n in case["sections"].split(",")]
    if not case["mixed"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


# ---- inputs -----------------------------------------------------------------------------------------

def _fill(case, st, pages, g, dev):
    """What the cache holds: quantised keys whose pages differ in their mean, as the topics of a text do, and values.  A few
    hundred pages are made, and used again with other scales."""
    heads, dim, page = case["hkv"], case["dim"], case["page"]
    bank = min(pages, max(4, (1 << 24) // (heads * dim * page)))
    one = {**st, "page": page}
    one["k_codes"], one["v_codes"], one["scales"] = _buffers(case, bank, dev)
    mean = torch.randn(bank, 1, heads, dim, generator=g, device=dev)
    k = (0.7 * mean + torch.randn(bank, page, heads, dim, generator=g, device=dev)).flatten(0, 1)
    v = torch.randn(bank * page, heads, dim, generator=g, device=dev)
    _put(one, k.bfloat16().float(), v.bfloat16().float(), torch.arange(bank * page, device=dev))
    which = torch.randint(0, bank, (pages,), generator=g, device=dev)
    which[:bank] = torch.arange(bank, device=dev)
    st["k_codes"], st["v_codes"] = one["k_codes"][which], one["v_codes"][which]
    size = 0.75 + 0.5 * torch.rand(pages, 1, 1, 1, 1, generator=g, device=dev)
    st["scales"] = (one["scales"][which] * size.half())


def _tables(held, page, width, spare, g, dev):
    """(page tables with the sequences' pages in any order, -1 behind them, pages, the rest of them)"""
    per = [(h + page - 1) // page for h in held]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    n = torch.tensor(per, device=dev)
    at = (torch.cumsum(n, 0) - n)[:, None] + torch.arange(width, device=dev)
    there = torch.arange(width, device=dev) < n[:, None]
    tables = torch.where(there, order[at.clamp(max=pages - 1)], torch.full_like(at, -1, dtype=torch.int32)).to(torch.int32)
    return tables.contiguous(), pages, order[sum(per):]


def _int(x, dev, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


def _prepare_pages(case, st, g, dev):
    held, new = _held(case)
    page, width = case["page"], case["width"]
    spare = sum((h + n + page - 1) // page for h, n in zip(held, new)) - sum((h + page - 1) // page for h in held) + 5
    st["tables"], pages, rest = _tables(held, page, width, spare, g, dev)
    st["free"] = torch.zeros(pages, dtype=torch.int32, device=dev)
    st["free"][: len(rest)] = rest
    st["counts"], st["lens"], st["new"] = _int([len(rest), 0], dev), _int(held, dev), _int(new, dev)
    if case["op"] == "plan":
        st["rows"] = case["rows"]
    else:
        st["done"] = torch.rand(case["seqs"], generator=g, device=dev) < case["done"]


def _prepare_fork(case, st, g, dev):
    tokens, parents = _forks(case)
    page, beams = case["page"], case["beams"]
    width = (case["prompt"] + case["made"] + page - 1) // page + 2
    shared = case["prompt"] // page                                   # whole pages of the prompt: one for all beams
    rows, at = [], 0
    for t in tokens:
        need = (t + page - 1) // page
        base = list(range(at, at + shared))
        at += shared
        for _ in range(beams):
            own_pages = list(range(at, at + need - shared))
            at += need - shared
            rows.append(base + own_pages + [-1] * (width - need))
    pages = at + 3
    order = torch.cat((torch.randperm(pages, generator=g, device=dev), torch.tensor([-1], device=dev))).to(torch.int32)
    st["tables"] = order[_int(rows, dev, torch.int64)].contiguous()
    st["free"] = torch.zeros(pages, dtype=torch.int32, device=dev)
    st["free"][:3] = order[at:at + 3]
    st["counts"], st["beams"] = _int([3, 0], dev), beams
    st["lens"] = _int([t for t in tokens for _ in range(beams)], dev)
    st["parents"] = _int(parents, dev)
    _fill(case, st, pages, g, dev)


def _prepare_cache(case, st, g, dev):
    held, new = _lengths(case)
    page = case["page"]
    width = (max(held) + page - 1) // page + 1
    st["tables"], pages, _ = _tables(held, page, width, 3, g, dev)
    _fill(case, st, pages, g, dev)
    st["lens"], st["new"], st["news"] = _int(held, dev), case["new"], _int(new, dev, torch.int64)
    st["most"] = max(new)
    st["starts"] = None
    if case["new"] > 1:
        st["starts"] = _int([sum(new[:b]) for b in range(len(new) + 1)], dev)
    st["bounds"] = torch.zeros(pages, case["hkv"], 2, case["dim"], dtype=torch.float16, device=dev)
    if case["op"] == "bounds":
        return
    for p0 in range(0, pages, 1024):
        k = _page_keys(st, torch.arange(p0, min(pages, p0 + 1024), device=dev))
        st["bounds"][p0:p0 + 1024] = _outwards(k.amin(-2), k.amax(-2))
    rows = sum(new)
    st["row_seq"] = torch.repeat_interleave(torch.arange(len(new), device=dev), st["news"], output_size=rows)
    st["row_at"] = torch.arange(rows, device=dev) - (torch.cumsum(st["news"], 0) - st["news"])[st["row_seq"]]
    q = torch.randn(rows, case["hq"], case["dim"], generator=g, device=dev)
    st["q"] = (1.2 * q).to(DTYPES[case["dtype"]])
    st["keep"], st["first"], st["last"] = case["keep"], case["first"], case["last"]


def _prepare_axes(case, st, g, dev):
    rows, dim, page = case["rows"], case["dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    axis = _axis_of(case)
    pages = (2 * rows + page - 1) // page
    run = min(page, rows)
    start = torch.randperm((pages * page) // run, generator=g, device=dev)[: (rows + run - 1) // run] * run
    st["slots"] = (start[:, None] + torch.arange(run, device=dev)).flatten()[:rows].contiguous()
    st["k"], st["v"], st["q"] = (torch.randn(rows, h, dim, generator=g, device=dev).to(dt) for h in
                                 (case["hkv"], case["hkv"], case["hq"]))
    angle = torch.arange(32768, device=dev, dtype=torch.float64)[:, None] * torch.pow(
        torch.tensor(1e6, device=dev, dtype=torch.float64),
        -torch.arange(len(axis), device=dev, dtype=torch.float64) / len(axis))
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    # text, all axes alike, and pictures of 28 by 36 patches, one time step each
    n = torch.arange(rows, device=dev)
    base, patch = n // 2048 * 300 + n % 2048, n % 2048 - 256
    picture = (patch >= 0) & (patch < 1008)
    base = base + torch.randint(0, 16384 - 300 * 8 - 2048, (1,), generator=g, device=dev)
    t, h, w = (torch.where(picture, n // 2048 * 300 + x, base) for x in (torch.full_like(n, 256), 256 + patch // 36, 256 + patch % 36))
    st["positions"] = torch.stack((t, h, w)).contiguous()
    st["axes"], st["paired"] = axis, case["paired"]
    st["k_codes"], st["v_codes"], st["scales"] = _buffers(case, pages, dev)


def _prepare_select(case, st, g, dev):
    # logits of a model that is sure of a few dozen tokens, other ones for each beam; scores of a search under way
    reqs, beams, vocab = case["reqs"], case["beams"], case["vocab"]
    x = torch.empty(reqs, beams, vocab, dtype=DTYPES[case["dtype"]], device=dev)
    for r0 in range(0, reqs, 8):
        part = 2.5 * torch.randn(min(reqs, r0 + 8) - r0, beams, vocab, generator=g, device=dev)
        likely = torch.randint(0, vocab, (part.shape[0], 1, 40), generator=g, device=dev).expand(-1, beams, -1)
        part.scatter_add_(2, likely, 6.0 + 2.0 * torch.randn(part.shape[0], beams, 40, generator=g, device=dev))
        x[r0:r0 + 8] = part
    st["logits"] = x
    st["scores"] = -torch.rand(reqs, beams, generator=g, device=dev).mul(6.0).cumsum(1) - 12.0
    st["n"] = case["n"]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    st = {k: case[k] for k in ("op", "page", "dim", "kf", "vf", "hkv") if k in case}
    {"plan": _prepare_pages, "release": _prepare_pages, "fork": _prepare_fork, "bounds": _prepare_cache, "sparse": _prepare_cache,
     "axes": _prepare_axes, "select": _prepare_select}[case["op"]](case, st, g, dev)
    if own and "k_codes" in st:
        from nemicli_terminal_b200 import kvcache
        st["cache"] = kvcache.KVCache(st["scales"].shape[0], st["hkv"], st["dim"], st["page"], st["kf"], st["vf"],
                                      buffers=(st["k_codes"], st["v_codes"], st["scales"]))
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _plain_plan(st):
    page, tables, free, rows = st["page"], st["tables"], st["free"].long(), st["rows"]
    seqs, width = tables.shape
    n_free = st["counts"][0].long()
    held = st["lens"].long().clamp(0, width * page)
    take = torch.minimum(st["new"].long().clamp(min=0), width * page - held)
    ends = torch.cumsum(take, 0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    had, want = (held + page - 1) // page, (held + take + page - 1) // page
    need = want - had
    before = torch.cumsum(need, 0) - need

    def taken(k):
        return torch.where(k < n_free, free[(n_free - 1 - k).clamp(0, free.shape[0] - 1)], torch.full_like(k, -1))

    col = torch.arange(width, device=tables.device)
    new = (col >= had[:, None]) & (col < want[:, None])
    tables.copy_(torch.where(new, taken(before[:, None] + col - had[:, None]), tables.long()))
    r = torch.arange(rows, device=tables.device)
    b = torch.searchsorted(ends, r, right=True)
    live = b < seqs
    b = b.clamp(max=seqs - 1)
    pos = held[b] + r - starts[b]
    entry = tables[b, (pos // page).clamp(0, width - 1)].long()
    slots = torch.where(live & (entry >= 0), entry * page + pos % page, torch.full_like(pos, -1))
    total = need.sum()
    counts = torch.stack(((n_free - total).clamp(min=0), st["counts"][1].long() + (total - n_free).clamp(min=0)))
    return {"slots": slots, "positions": torch.where(live, pos, torch.zeros_like(pos)),
            "starts": starts.clamp(max=rows).to(torch.int32), "lens": (held + take).to(torch.int32),
            "counts": counts.to(torch.int32), "tables": tables}


def _plain_release(st):
    page, tables, free = st["page"], st["tables"], st["free"]
    seqs, width = tables.shape
    held = st["lens"].long().clamp(0, width * page)
    n = torch.where(st["done"], (held + page - 1) // page, torch.zeros_like(held))
    at = st["counts"][0].long() + torch.cumsum(n, 0) - n
    col = torch.arange(width, device=tables.device)
    gone = col < n[:, None]
    # what stays goes to one place more behind the stack
    spot = torch.where(gone, at[:, None] + col, torch.full_like(at, free.shape[0])[:, None]).clamp(max=free.shape[0])
    room = torch.cat((free, free[:1])).scatter_(0, spot.flatten(), tables.flatten())
    free.copy_(room[:-1])
    counts = torch.stack((st["counts"][0].long() + n.sum(), st["counts"][1].long()))
    return {"lens": torch.where(st["done"], torch.zeros_like(held), held).to(torch.int32), "free": free,
            "counts": counts.to(torch.int32)}


def _plain_select(st):
    x, scores, n = st["logits"], st["scores"], st["n"]
    reqs, beams, vocab = x.shape
    step = max(1, (1 << 27) // (beams * vocab))
    out = []
    for r0 in range(0, reqs, step):
        y = x[r0:r0 + step].double()
        y = torch.where(y.isnan(), torch.full_like(y, -math.inf), y).clamp_(max=MOST)
        top = y.amax(-1, keepdim=True).clamp(min=-MOST)
        total = (y - top).exp_().sum(-1, keepdim=True)
        y = (y - top) - total.clamp(min=1e-300).log() + scores[r0:r0 + step].double()[..., None]
        y = torch.where(y.isnan(), torch.full_like(y, -math.inf), y).flatten(1)
        best, index = torch.sort(y, dim=1, descending=True, stable=True)
        out.append((best[:, :n].float(), index[:, :n]))
    best, index = (torch.cat(o) for o in zip(*out))
    return {"scores": best, "parents": (index // vocab).to(torch.int32), "tokens": (index % vocab).to(torch.int32)}


def _plain_fork(st):
    page, beams, free = st["page"], st["beams"], st["free"]
    width = st["tables"].shape[1]
    old = st["tables"].long().unflatten(0, (-1, beams))                       # (requests, beams, width)
    reqs = old.shape[0]
    lens, parents = st["lens"].long().view(reqs, beams), st["parents"].long()
    col = torch.arange(width, device=old.device)
    n = (lens + page - 1) // page
    there = col < n[..., None]
    chosen = (parents[:, :, None] == torch.arange(beams, device=old.device)).any(1)       # (requests, beams)
    alike = (old[:, :, None] == old[:, None]) & there[:, :, None] & there[:, None]        # (requests, beams, other, width)
    first = torch.arange(beams, device=old.device)
    kept = (alike & chosen[:, None, :, None]).any(2) | (alike & (first[None] < first[:, None])[None, :, :, None]).any(2)
    gone = there & ~kept
    order = gone.transpose(1, 2).flatten(1)                                   # by place, then by beam
    pages = old.transpose(1, 2).flatten(1)
    rank = torch.cumsum(order, 1) - 1
    freed = order.sum(1)
    # the beams of the next step
    new_lens = torch.gather(lens, 1, parents)
    tables = torch.gather(old, 1, parents[..., None].expand(-1, -1, width))
    m = (new_lens + page - 1) // page
    tables = torch.where(col < m[..., None], tables, torch.full_like(tables, -1))
    end = torch.gather(tables, 2, (m - 1).clamp(min=0)[..., None])[..., 0]
    part = new_lens % page != 0
    earlier = (end[:, :, None] == end[:, None]) & part[:, None] & (first[None] < first[:, None])[None]
    copy = part & earlier.any(2)
    asked = torch.cumsum(copy, 1) - copy.long()
    wants = copy.sum(1)
    # freed pages of the request itself, what is left goes onto the stack, what is missing comes from there
    left, short = (freed - wants).clamp(min=0), (wants - freed).clamp(min=0)
    n_free = st["counts"][0].long()
    spot = (n_free + torch.cumsum(left, 0) - left)[:, None] + rank - wants[:, None]
    spot = torch.where(order & (rank >= wants[:, None]), spot, torch.full_like(spot, free.shape[0])).clamp(max=free.shape[0])
    free.copy_(torch.cat((free, free[:1])).scatter_(0, spot.flatten(), pages.flatten().to(torch.int32))[:-1])
    size = n_free + left.sum()
    mine = torch.full((reqs, beams + 1), -1, dtype=torch.int64, device=old.device)
    mine.scatter_(1, torch.where(order & (rank < wants[:, None]), rank, torch.full_like(rank, beams)), pages)
    k = size - 1 - ((torch.cumsum(short, 0) - short)[:, None] + asked - freed[:, None])
    pool = torch.where(k >= 0, free.long()[k.clamp(0, free.shape[0] - 1)], torch.full_like(k, -1))
    target = torch.where(asked < freed[:, None], torch.gather(mine[:, :beams], 1, asked.clamp(max=beams - 1)), pool)
    dst, src = (torch.where(copy, x, torch.full_like(x, -1)) for x in (target, end))
    tables = torch.where((col == (m - 1)[..., None]) & copy[..., None], target[..., None], tables)
    counts = torch.stack(((size - short.sum()).clamp(min=0), st["counts"][1].long() + (short.sum() - size).clamp(min=0)))
    # the copies: as many tokens as the page holds (values of two tokens lie side by side); the others stay
    used = torch.where(copy, new_lens % page, torch.zeros_like(new_lens)).flatten()
    s, d = src.flatten().clamp(min=0), dst.flatten()
    d = torch.where(d >= 0, d, torch.full_like(d, st["scales"].shape[0] - 1))
    at = torch.arange(page, device=old.device)
    go = (used[:, None] > at) & (dst.flatten() >= 0)[:, None]
    for name, mask in (("k_codes", go), ("v_codes", go[:, 0::2]), ("scales", go)):
        b = st[name]
        i, t = torch.nonzero(mask, as_tuple=True)
        b[d[i], :, t] = b[s[i], :, t]
    return {"tables": tables.flatten(0, 1).to(torch.int32), "lens": new_lens.flatten().to(torch.int32), "counts": counts.to(torch.int32),
            "src": src.flatten().to(torch.int32), "dst": dst.flatten().to(torch.int32), "free": free,
            "k_codes": st["k_codes"], "v_codes": st["v_codes"], "scales": st["scales"].view(torch.int16)}


def _plain_bounds(st):
    page, lens, bounds = st["page"], st["lens"].long(), st["bounds"]
    most = st["most"] // page + 1
    i = ((lens - st["news"]) // page)[:, None] + torch.arange(most, device=lens.device)
    b, at = torch.nonzero(i < (lens // page)[:, None], as_tuple=True)
    pages = st["tables"][b, i[b, at]].long()
    for p0 in range(0, pages.shape[0], 256):
        k = _page_keys(st, pages[p0:p0 + 256])
        bounds[pages[p0:p0 + 256]] = _outwards(k.amin(-2), k.amax(-2))
    return {"bounds": bounds}


def _plain_sparse(st):
    q, page, tables = st["q"], st["page"], st["tables"]
    rows, hq, dim = q.shape
    hkv, keep, first, last = st["hkv"], st["keep"], st["first"], st["last"]
    width = tables.shape[1]
    pos = (st["lens"].long() - st["news"])[st["row_seq"]] + st["row_at"]
    at = pos // page
    col = torch.arange(width, device=q.device)
    x = q.float().unflatten(1, (hkv, -1))
    score = torch.empty(rows, hkv, width, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 25) // (width * hkv * dim))
    for r0 in range(0, rows, step):                                           # in 64 bits: pages next to the border
        lo, hi = st["bounds"][tables[st["row_seq"][r0:r0 + step]].clamp(min=0).long()].double().unbind(-2)
        y = x[r0:r0 + step].double()                                          # (rows, hkv, group, dim); lo, hi (rows, width, hkv, dim)
        s = torch.full(lo.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
        for h in range(y.shape[2]):
            z = y[:, None, :, h]
            s = torch.maximum(s, torch.maximum(z * lo, z * hi).sum(-1))
        score[r0:r0 + step] = s.transpose(1, 2)
    must = (col < first) | (col > at[:, None] - last)
    score = torch.where(must[:, None], torch.full_like(score, math.inf), score)
    score = torch.where((col > at[:, None])[:, None], torch.full_like(score, -math.inf), score)
    count = (at + 1).clamp(max=keep)
    order = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :keep]
    here = torch.arange(order.shape[-1], device=q.device) < count[:, None]
    order = torch.sort(torch.where(here[:, None], order, torch.full_like(order, width)), -1)[0]
    entry = tables[st["row_seq"]][:, None].expand(-1, hkv, -1)
    chosen = torch.gather(entry, 2, order.clamp(max=width - 1))
    chosen = torch.where(here[:, None], chosen, torch.full_like(chosen, -1))
    chosen = torch.nn.functional.pad(chosen, (0, keep - chosen.shape[-1]), value=-1)
    held = (count - 1) * page + pos % page + 1
    o = torch.empty(rows, hkv, hq // hkv, dim, device=q.device)
    key = torch.arange(keep * page, device=q.device)
    head = torch.arange(hkv, device=q.device)[:, None]
    one = {**st}
    step = max(1, (1 << 26) // (keep * page * hkv * dim))
    for r0 in range(0, rows, step):
        c = chosen[r0:r0 + step].clamp(min=0).long()                          # (rows, hkv, keep)
        s = st["scales"][c, head].float()                                     # (rows, hkv, keep, P, 2, J)
        k = (_unpack_k(_k_view(one)[c, head], st["kf"]) * s[..., 0, :, None]).flatten(-2).flatten(2, 3)
        v = _unpack_v(_v_view(one)[c, head].movedim(-2, 4).flatten(3, 4), st["vf"])
        v = (v * s[..., 1, :, None]).flatten(-2).flatten(2, 3)
        logits = (x[r0:r0 + step] @ k.transpose(-1, -2)).mul_(dim ** -0.5)
        logits = torch.where((key < held[r0:r0 + step, None])[:, None, None], logits, torch.full_like(logits, -math.inf))
        p = (logits - logits.amax(-1, keepdim=True)).exp_()
        o[r0:r0 + step] = (p @ v) / p.sum(-1, keepdim=True)
    return {"chosen": chosen, "held": held.to(torch.int32), "o": o.flatten(1, 2).to(q.dtype)}


def _plain_axes(st):
    axis = torch.tensor(st["axes"], device=st["cos"].device)
    at = st["positions"][axis].T                                              # (rows, rot / 2)
    cos, sin = torch.gather(st["cos"], 0, at), torch.gather(st["sin"], 0, at)
    k = _rotate(st["k"].float(), cos, sin, st["paired"])
    q = _rotate(st["q"].float(), cos, sin, st["paired"]).to(st["q"].dtype)
    _put(st, k, st["v"].float(), st["slots"])
    k, v = _get(st, st["slots"])
    return {"k": k.to(st["k"].dtype), "v": v.to(st["k"].dtype), "q": q}


def run(state):
    st = state
    if not own:
        return {"plan": _plain_plan, "release": _plain_release, "select": _plain_select, "fork": _plain_fork, "bounds": _plain_bounds,
                "sparse": _plain_sparse, "axes": _plain_axes}[st["op"]](st)
    from nemicli_terminal_b200 import beams, pages
    if st["op"] == "plan":
        p = pages.plan(st["lens"], st["new"], st["tables"], st["free"], st["counts"], st["page"], st["rows"])
        return {"slots": p.slots, "positions": p.positions, "starts": p.starts, "lens": p.lens, "counts": p.counts,
                "tables": st["tables"]}
    if st["op"] == "release":
        lens, counts = pages.release(st["done"], st["lens"], st["tables"], st["free"], st["counts"], st["page"])
        return {"lens": lens, "free": st["free"], "counts": counts}
    if st["op"] == "select":
        scores, parents, tokens = beams.select(st["logits"], st["scores"], st["n"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    cache = st["cache"]
    if st["op"] == "fork":
        r = pages.reorder(st["parents"], st["lens"], st["tables"], st["free"], st["counts"], st["page"])
        cache.copy(r.src, r.dst, r.used)
        return {"tables": r.tables, "lens": r.lens, "counts": r.counts, "src": r.src, "dst": r.dst, "free": st["free"],
                "k_codes": cache.k_codes, "v_codes": cache.v_codes, "scales": cache.scales.view(torch.int16)}
    if st["op"] == "bounds":
        cache.summarise(st["bounds"], st["tables"], st["lens"], st["starts"], max_new=st["most"])
        return {"bounds": st["bounds"]}
    if st["op"] == "sparse":
        chosen, held = cache.choose(st["q"], st["bounds"], st["tables"], st["lens"], st["keep"], starts=st["starts"],
                                    first=st["first"], last=st["last"])
        return {"chosen": chosen, "held": held, "o": cache.attend_chosen(st["q"], chosen, held)}
    q = cache.write(st["k"], st["v"], st["slots"], q=st["q"], rope=(st["cos"], st["sin"], st["positions"]),
                    paired=st["paired"], axes=st["axes"])
    k, v = cache.read(st["slots"], st["k"].dtype)
    return {"k": k, "v": v, "q": q}


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


def _exact_keys(st, pages, head):
    """The keys of one head in pages (n,): (n, P, dim) fp64."""
    J = st["dim"] // 32

    def at(i):
        j, t, e = i // 32, (i % 32) // 8, i % 8
        if st["kf"] == "Q4_0":
            pair, odd = e // 2, e % 2
            return t * 4 * J + 4 * j + 2 * odd + pair // 2, 4 * (pair % 2)
        return t * 8 * J + 8 * j + 4 * (e // 4) + 2 * (e % 2) + (e % 4) // 2, 0

    return _exact_values(st["k_codes"][pages, head].long(), st["kf"], st["scales"][pages, head, :, 0], at)


def _exact_vals(st, pages, head):
    J, halves = st["dim"] // 32, []
    raw, sc = st["v_codes"][pages, head].long(), st["scales"][pages, head, :, 1]
    for odd in (0, 1):
        def at(i, odd=odd):
            j, g, e = i // 32, (i % 32) // 4, i % 4
            if st["vf"] == "Q4_0":
                return (g * J + j) * 4 + 2 * odd + e // 2, 4 * (e % 2)
            return (g * J + j) * 8 + 4 * (e // 2) + 2 * odd + e % 2, 0
        halves.append(_exact_values(raw, st["vf"], sc[:, odd::2], at))
    return torch.stack(halves, 2).flatten(1, 2)


def _exact_sparse(case, st):
    page, keep = st["page"], st["keep"]
    q = st["q"].double()
    group = case["hq"] // case["hkv"]
    out = torch.zeros_like(q)
    row = 0
    for b, (t, new) in enumerate(zip(*_lengths(case))):
        table = st["tables"][b].long()
        for p in range(t - new, t):
            own_page = p // page
            for h in range(case["hkv"]):
                mine = q[row, h * group:(h + 1) * group]
                pages = list(range(own_page + 1))
                if len(pages) > keep:
                    box = st["bounds"][table[:own_page + 1], h].double()
                    best = (mine.clamp(min=0) @ box[:, 1].T + mine.clamp(max=0) @ box[:, 0].T).amax(0)
                    must = set(pages[:st["first"]]) | set(pages[max(0, len(pages) - st["last"]):])
                    best = best.tolist()
                    rest = sorted((i for i in pages if i not in must), key=lambda i: (-best[i], i))
                    pages = sorted(must | set(rest[:keep - len(must)]))
                at = table[torch.tensor(pages, device=q.device)]
                n = (len(pages) - 1) * page + p % page + 1
                k, v = _exact_keys(st, at, h).flatten(0, 1)[:n], _exact_vals(st, at, h)[:, :].flatten(0, 1)[:n]
                out[row, h * group:(h + 1) * group] = torch.softmax(mine @ k.T / math.sqrt(case["dim"]), -1) @ v
            row += 1
    return {"chosen": None, "held": None, "o": out}


def _exact_bounds(case, st):
    out = st["bounds"].double()
    for b, (t, new) in enumerate(zip(*_lengths(case))):
        pages = st["tables"][b, (t - new) // case["page"]: t // case["page"]].long()
        for h in range(case["hkv"]):
            if len(pages):
                k = _exact_keys(st, pages, h)
                out[pages, h] = _outwards(k.amin(1), k.amax(1)).double()
    return {"bounds": out}


def _exact_select(case, st):
    best = []
    for r in range(case["reqs"]):
        x = torch.log_softmax(st["logits"][r].double(), -1) + st["scores"][r].double()[:, None]
        best.append(torch.topk(x.flatten(), case["n"]).values)
    return {"scores": torch.stack(best), "parents": None, "tokens": None}


def _exact_axes(case, st):
    out = {"k": None, "v": None}
    if case["dtype"] == "bf16":
        # in 8 bits of significand no quotient lies so near a border that its rounding to fp32 could move a code
        x = st["v"].double().unflatten(-1, (-1, 32))
        if case["vf"] == "Q4_0":
            first = x.abs().argmax(-1, keepdim=True)
            d, lo, hi = (x.gather(-1, first)[..., 0] / -8).half().double(), -8, 7
        else:
            d, lo, hi = (x.abs().amax(-1) / 127).float().half().double(), -127, 127
        out["v"] = ((x / d[..., None]).round().clamp(lo, hi) * d[..., None]).flatten(-2)
    x = st["q"].double()
    y = x.clone()
    half = len(st["axes"])
    for i, a in enumerate(st["axes"]):
        c, s = (t[st["positions"][a], i].double()[:, None] for t in (st["cos"], st["sin"]))
        m, n = (2 * i, 2 * i + 1) if st["paired"] else (i, i + half)
        y[..., m] = x[..., m] * c - x[..., n] * s
        y[..., n] = x[..., m] * s + x[..., n] * c
    out["q"] = y
    return out


def exact(case, seed):
    if case["op"] in ("plan", "release", "fork"):
        return None                                                           # whole numbers
    st = prepare(case, seed)
    if case["op"] == "sparse":
        return _exact_sparse(case, st) if sum(_lengths(case)[1]) * case["hkv"] <= 1024 else None
    return {"bounds": _exact_bounds, "select": _exact_select, "axes": _exact_axes}[case["op"]](case, st)
