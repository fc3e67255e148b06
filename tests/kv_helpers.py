"""Plain 64-bit forms of the quantised cache and of attention over it, for the tests (numpy / torch fp64, written from the
formulas and the byte layout in include/nemicli_qmv.h, sharing no arithmetic with the package)."""
from __future__ import annotations

import numpy as np
import torch

from nemicli_terminal_b200 import _lib

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, pos: np.ndarray, paired: bool) -> np.ndarray:
    """fp32 arithmetic, every product and sum rounded (numpy does not contract): x (rows, heads, dim) fp32."""
    x = x.astype(np.float32)
    half = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    y = x.copy()
    ia, ib = (np.arange(half) * 2, np.arange(half) * 2 + 1) if paired else (np.arange(half), np.arange(half) + half)
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def quantise(x: np.ndarray, fmt: str):
    """x (rows, heads, dim) fp32 -> codes (rows, heads, J, 32) with their offset, d (rows, heads, J) fp16."""
    b = np.where(np.isnan(x), np.float32(0), np.clip(x, -65504, 65504)).astype(np.float32)
    b = b.reshape(*x.shape[:-1], -1, 32)
    first = np.abs(b).argmax(-1)[..., None]
    m = np.take_along_axis(b, first, -1)[..., 0]
    with np.errstate(over="ignore", under="ignore", divide="ignore", invalid="ignore"):
        d = (m * np.float32(-0.125) if fmt == "Q4_0" else np.abs(m) / np.float32(127)).astype(np.float16)
        df = d.astype(np.float32)[..., None]
        q = np.where(df == 0, np.float32(0), np.rint(b / df))
    lo, hi, off = (-8, 7, 8) if fmt == "Q4_0" else (-127, 127, 128)
    return (np.clip(q, lo, hi) + off).astype(np.int64), d


def codes_of(cache, slots: np.ndarray):
    """(K codes, V codes (rows, heads, J, 32) with their offset, scales (rows, heads, 2, J)) read bit by bit out of
    the cache's buffers."""
    P, J = cache.page, cache.dim // 32
    page, at = slots // P, slots % P
    kc = cache.k_codes.cpu().numpy().astype(np.int64)[page, :, at]
    vc = cache.v_codes.cpu().numpy().astype(np.int64)[page, :, at // 2]
    rows, heads = kc.shape[:2]
    k = np.empty((rows, heads, J, 32), np.int64)
    v = np.empty_like(k)
    odd = (at % 2)[:, None]
    r, h = np.arange(rows)[:, None], np.arange(heads)[None]
    for j in range(J):
        for i in range(32):
            t, n = divmod(i, 8)
            if cache.k_fmt == "Q4_0":
                bit = 16 * (n & 1) + 4 * (n >> 1)
                k[..., j, i] = (kc[..., (t * J + j) * 4 + bit // 8] >> (bit % 8)) & 15
            else:
                k[..., j, i] = kc[..., (t * J + j) * 8 + 4 * (n >> 2) + 2 * (n & 1) + ((n & 3) >> 1)]
            g, n = divmod(i, 4)
            if cache.v_fmt == "Q4_0":
                bit = 4 * n
                v[..., j, i] = (vc[r, h, (g * J + j) * 4 + 2 * odd + bit // 8] >> (bit % 8)) & 15
            else:
                v[..., j, i] = vc[r, h, (g * J + j) * 8 + 4 * (n >> 1) + 2 * odd + (n & 1)]
    return k, v, cache.scales.cpu().numpy()[page, :, at]


def values(codes: np.ndarray, d: np.ndarray, fmt: str) -> np.ndarray:
    off = 8 if fmt == "Q4_0" else 128
    return ((codes - off) * d.astype(np.float64)[..., None]).reshape(*codes.shape[:-2], -1)


def attention(q, k, v, pos, scale, window):
    """One sequence: q (n, heads, dim), k, v (keys, n_kv, dim), pos (n,) in fp64 -> (out, sizes): sizes = (sum p |v|,
    sum p top(v), and over the keys the largest scale * sum |q k| and scale * sum |q| top(k)), where top is the
    largest magnitude of the value's 32-value block.  Rows that see no key: zeros."""
    n, heads, dim = q.shape
    keys, n_kv, _ = k.shape
    g = heads // n_kv
    o = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    mag, top = torch.zeros_like(o), torch.zeros_like(o)
    qk, qt = (torch.zeros(n, heads, dtype=torch.float64, device=q.device) for _ in range(2))
    key = torch.arange(keys, device=q.device)
    seen = key[None] <= pos[:, None]
    if window:
        seen &= key[None] > pos[:, None] - window
    some = seen.any(1)
    if keys == 0 or not bool(some.any()):
        return o, (mag, top, qk, qt)
    kt, vt = (x.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) for x in (k, v))
    for h in range(heads):
        s = (q[:, h] @ k[:, h // g].T) * scale
        s = s.masked_fill(~seen, -torch.inf)
        p = torch.where(some[:, None], torch.softmax(s, 1), torch.zeros_like(s))
        o[:, h] = p @ v[:, h // g]
        mag[:, h] = p @ v[:, h // g].abs()
        top[:, h] = p @ vt[:, h // g]
        for out, x in ((qk, k.abs()), (qt, kt)):
            out[:, h] = torch.where(seen, (q[:, h].abs() @ x[:, h // g].T) * scale, torch.zeros_like(s)).amax(1)
    return o, (mag, top, qk, qt)


def tiled(c, heads, n_seq, max_new, dtype, width, window=0):
    """Whether attend takes tiles of 128 rows for such a call: its workspace then has an odd number of bytes."""
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    return _lib.load().qmv_kv_attend_workspace_bytes(c._ref, heads, n_seq, max_new, code, width, window) % 2 == 1


def bound(sizes, o, dtype, keys, tiles):
    """How far an output may be off, from the kernels' roundings (first order, worst case).  The sums over code bits run
    before the codes' offset is taken off, so their partial sums are as large as the block's largest value times two
    (codes 0 .. 15 against an offset of 8, 1 .. 255 against 128; the largest value's code lies at the offset's distance),
    whatever the value itself is; a step of 16 products on the tensor cores is cut off at 2^-22 of them.
    - a score is off by ds: queries as two fp16 parts (2^-22; 16-bit types are exact), keys d * code exact or rounded
      to fp16 on the tile path (2^-11), and at most 16 such steps and block sums over the head's values;
    - a weight exp(s - m) / sum changes by 2 ds relatively, and by its own rounding: to fp16 (2^-11) or two fp16
      parts (2^-21); the value by 2^-11 on the tile path; exp2 and the final division: 2^-20;
    - the sums over the keys in steps of 16, and at most 16 joins of parts;
    - the output's own rounding: half a step."""
    mag, top, qk, qt = sizes
    exact = dtype == torch.float32
    ds = qk * ((2.0 ** -22 if exact else 0.0) + (2.0 ** -11 if tiles else 0.0)) + 2 * qt * 16 * 2.0 ** -22
    rel = 2 * ds[..., None] + (2.0 ** -21 if exact else 2.0 ** -11) + (2.0 ** -11 if tiles else 0.0) + 2.0 ** -20
    return mag * rel + 2 * top * (keys / 16 + 16) * 2.0 ** -22 + o.abs() * HALF_STEP[dtype] \
        + 2.0 ** -24 * (dtype == torch.float16) + 1e-30
