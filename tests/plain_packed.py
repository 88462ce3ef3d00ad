"""Plain 64-bit implementation of the packed cache: its format, rotation and quantisation, and attention over it.  Loops over
sequences and heads; nothing of the package is used."""
import math

import torch

F64 = torch.float64


def group_of(d):
    return 64 if d % 64 == 0 else 32 if d % 32 == 0 else 16


def page_bytes(bits, d, page):
    return page * 2 * (d * bits // 8) + page * 2 * 4 * (d // group_of(d))


def bf16_toward(x, up):
    """x (float64) to a bfloat16 number that is not below (above) it; a bfloat16 has eight significant bits."""
    m, e = torch.frexp(x)
    m = m * 256
    m = torch.ceil(m) if up else torch.floor(m)
    return torch.ldexp(m, e - 8)


def quantise(x, bits):
    """x [..., d] float64 -> codes [..., d] (float64), scale and offset [..., groups]."""
    d = x.shape[-1]
    y = x.reshape(*x.shape[:-1], d // group_of(d), group_of(d))
    bad = ~torch.isfinite(y).all(-1)
    off = bf16_toward(y.min(-1).values, False)
    scale = bf16_toward((y.max(-1).values - off) / (2 ** bits - 1), True)
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    code = ((y - off[..., None]) / safe[..., None]).round().clamp(0, 2 ** bits - 1)
    code = torch.where((scale > 0)[..., None] & ~bad[..., None], code, torch.zeros_like(code))
    nan = torch.full_like(scale, math.nan)
    return code.reshape(x.shape), torch.where(bad, nan, scale), torch.where(bad, nan, off)


def dequantise(code, scale, off):
    y = code.reshape(*scale.shape, code.shape[-1] // scale.shape[-1])
    return (y * scale[..., None] + off[..., None]).reshape(code.shape)


def through(x, bits):
    return dequantise(*quantise(x, bits))


def pack_row(x, bits):
    """The bytes of one token's row of d values (float64): codes, and (scale, offset) pairs."""
    code, scale, off = quantise(x, bits)
    code = code.to(torch.int64)
    if bits == 4:
        code = code[0::2] + 16 * code[1::2]
    pairs = torch.stack([scale, off], -1).reshape(-1).float().to(torch.bfloat16)
    return code.to(torch.uint8), pairs.view(torch.uint8)


def put(pages, slot, kvh, k, v, bits, page):
    """Write one token's key and value (float64 [d]) of one kv head into pages uint8 [n, nkv, bytes] (host)."""
    d = k.numel()
    row, par = d * bits // 8, 4 * (d // group_of(d))
    block, place = pages[slot // page, kvh], slot % page
    for which, x in enumerate((k, v)):
        code, pair = pack_row(x, bits)
        at = which * page * row + place * row
        block[at:at + row] = code
        at = 2 * page * row + which * page * par + place * par
        block[at:at + par] = pair


def get(pages, slot, kvh, d, bits, page):
    """(key, value) float64 [d] that the pages hold for one token and kv head."""
    row, par = d * bits // 8, 4 * (d // group_of(d))
    block, place = pages[slot // page, kvh], slot % page
    out = []
    for which in (0, 1):
        at = which * page * row + place * row
        code = block[at:at + row].to(torch.int64)
        if bits == 4:
            code = torch.stack([code % 16, code // 16], -1).reshape(-1)
        at = 2 * page * row + which * page * par + place * par
        pair = block[at:at + par].clone().view(torch.bfloat16).to(F64).reshape(-1, 2)
        out.append(dequantise(code.to(F64), pair[:, 0], pair[:, 1]))
    return out


def rotate(x, pos, inv_freq, interleaved=False, magnitude=1.0):
    """x [heads, d] float64 at position pos; the first 2 * len(inv_freq) channels turn."""
    half = inv_freq.numel()
    y = x.clone()
    c, s = torch.cos(pos * inv_freq) * magnitude, torch.sin(pos * inv_freq) * magnitude
    i0 = torch.arange(half) * (2 if interleaved else 1)
    i1 = i0 + (1 if interleaved else half)
    a, b = x[:, i0], x[:, i1]
    y[:, i0], y[:, i1] = a * c - b * s, a * s + b * c
    return y


def attend(q, keys, values, context, scale, window=0, softcap=0.0, sink=None, slopes=None, temperature=None):
    """q [a, nh, d] (the last a of ``context`` tokens), keys and values [context, nkv, d], float64."""
    a, nh, d = q.shape
    nkv = keys.shape[1]
    out = torch.zeros(a, nh, values.shape[2], dtype=F64)
    for i in range(a):
        p = context - a + i
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        factor = scale
        if temperature:
            factor = scale * (1.0 + temperature[0] * math.log(math.floor((p + 1) / temperature[1]) + 1.0))
        for h in range(nh):
            g = h // (nh // nkv)
            z = keys[lo:p + 1, g] @ q[i, h] * factor
            if softcap > 0:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                z = z - slopes[h].double() * (p - torch.arange(lo, p + 1, dtype=F64))
            if sink is not None:
                z = torch.cat([z, sink[h].double()[None]])
            w = torch.softmax(z, 0)[:p + 1 - lo]
            out[i, h] = w @ values[lo:p + 1, g]
    return out
