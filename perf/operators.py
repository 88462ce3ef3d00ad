"""What is measured of the packed cache: keys and values held in 4 or 8 bits.

Three operators: storing (rotate q and k, quantise k and v as they are written into their pages) with reading back (pages to
plain keys and values), attention of single tokens over such pages, and attention of prompt portions over them.

The format.  A page holds ``PAGE`` tokens of one kv head: the codes of its keys (a row of ``dim`` codes per token; in 4 bits,
channel 2i is the low half of byte i and 2i + 1 the high one), the codes of its values, then per token and group of 64 channels
(32, then 16, where 64 does not divide the head) a pair (scale, offset) in bfloat16 for the keys, and the same for the values.  A code c stands for
scale * c + offset.  offset is the group's smallest value rounded down to bfloat16, scale the smallest bfloat16 that is not
below (largest - offset) / (2^bits - 1), and c the whole number nearest to (x - offset) / scale, ties to even.
"""
import hashlib
import math

import torch

own = False

PAGE = 16
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# ---------------------------------------------------------------- the cases
def _case(path, bits, shape, **more):
    heads, kv, dim = shape
    return dict(path=path, bits=bits, heads=heads, kv=kv, dim=dim, dtype=more.pop("dtype", "bfloat16"), **more)


WIDE, SMALL, GQA, MQA, TINY, FULL = (32, 8, 128), (32, 8, 64), (16, 4, 128), (16, 1, 128), (32, 4, 64), (40, 40, 128)


def listed():
    return [
        # one request's next token is rotated and stored, and its page read back: the smallest call
        dict(name="store_token", **_case("store", 4, WIDE, seqs=1, new=1, context=14)),
        # the next tokens of a decoding batch in the float32 mode
        dict(name="store_batch_f32", **_case("store", 8, TINY, seqs=23, new=23, context=130, dtype="float32")),
        # a whole prompt in one step
        dict(name="store_prompt", **_case("store", 4, WIDE, seqs=1, new=2048, context=0)),
        # portions of three long prompts of odd lengths behind what earlier steps stored
        dict(name="store_portions", **_case("store", 8, SMALL, seqs=3, new=4099, context=6001)),
        # a single request with a short context: latency
        dict(name="decode_one", **_case("decode", 4, WIDE, seqs=1, context=700, sloped=False)),
        # eight requests at a 2048-token context, the batch of the serving benchmark
        dict(name="decode_batch", **_case("decode", 4, WIDE, seqs=8, context=2048, sloped=False)),
        # a busy server: 64 requests of different lengths
        dict(name="decode_server", **_case("decode", 4, WIDE, seqs=64, context=4096, sloped=False)),
        # one request far into a long context of odd length
        dict(name="decode_long", **_case("decode", 4, WIDE, seqs=1, context=100003, sloped=False)),
        # 8 bits, a window with a bias by distance and a sink (Rimidra's attention)
        dict(name="decode_sloped", **_case("decode", 8, GQA, seqs=48, context=3001, sloped=True)),
        # 8 bits, the heads of a 1B model
        dict(name="decode_8bit", **_case("decode", 8, SMALL, seqs=32, context=6000, sloped=False)),
        # a prompt attends to itself, stored in 4 bits
        dict(name="prompt", **_case("prompt", 4, WIDE, seqs=1, new=2048, context=0)),
        # portions of four prompts behind what earlier steps stored, in 8 bits
        dict(name="prompt_portions", **_case("prompt", 8, WIDE, seqs=4, new=1501, context=2900)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["store", "store", "decode", "decode", "decode", "prompt"])
    bits = rng.choice([4, 4, 8])
    shape = rng.choice([WIDE, WIDE, SMALL, GQA, MQA, TINY, FULL])
    dtype = "float32" if rng.random() < 0.12 else "bfloat16"
    if path == "store":
        new = _log(rng, 1, 4096 if shape is FULL or dtype == "float32" else 12000)
        seqs = min(new, _log(rng, 1, 40))
        return _case(path, bits, shape, seqs=seqs, new=new, context=rng.choice([0, _log(rng, 1, 12000 // seqs)]), dtype=dtype)
    if path == "decode":
        most = 24000 if dtype == "float32" or shape is FULL else 190000
        seqs = _log(rng, 1, 64)
        return _case(path, bits, shape, seqs=seqs, context=_log(rng, 1, min(131072, most // seqs)), sloped=rng.random() < 0.25, dtype=dtype)
    new = _log(rng, 5, 700 if dtype == "float32" or shape is FULL else 2048)
    seqs = min(max(1, new // 2), _log(rng, 1, 6))
    return _case(path, bits, shape, seqs=seqs, new=new, context=rng.choice([0, _log(rng, 1, 3000)]), dtype=dtype)


def _lens(total, n):
    """``total`` tokens over n sequences of different length, at least one each."""
    w = [3 + (5 * j + 2) % 7 for j in range(n)]
    lens = [max(1, total * x // sum(w)) for x in w]
    i = 0
    while sum(lens) != total:
        step = 1 if sum(lens) < total else -1
        if lens[i % n] + step >= 1:
            lens[i % n] += step
        i += 1
    return lens


def _lengths(c):
    """(new tokens, tokens held once those are stored) of every sequence."""
    n = c["seqs"]
    held = [c["context"] - (c["context"] * ((3 * j) % 8)) // 12 for j in range(n)]
    if c["path"] == "decode":
        return [1] * n, [max(1, h) for h in held]
    new = _lens(c["new"], n)
    return new, [a + b for a, b in zip(new, held)]


# ---------------------------------------------------------------- the format
def _group(dim):
    return 64 if dim % 64 == 0 else 32 if dim % 32 == 0 else 16


def _page_bytes(c):
    return 2 * PAGE * (c["dim"] * c["bits"] // 8 + 4 * (c["dim"] // _group(c["dim"])))


def _toward(x, up):
    """The nearest bfloat16 that is not below (above) x, by its bits."""
    r = x.to(F32).to(BF16)
    b = r.view(torch.int16)
    wrong = r.to(x.dtype) < x if up else r.to(x.dtype) > x
    shrink = (r > 0) if not up else (r < 0)
    moved = torch.where(r == 0, torch.full_like(b, 1 if up else -32767), torch.where(shrink, b - 1, b + 1))
    return torch.where(wrong, moved, b).view(BF16)


def _quantise(x, bits):
    """x [..., dim] -> codes uint8 [..., dim], scale and offset bfloat16 [..., groups]."""
    g = _group(x.shape[-1])
    y = x.unflatten(-1, (-1, g))
    offset = _toward(y.amin(-1), False)
    scale = _toward((y.amax(-1) - offset.to(x.dtype)) / (2 ** bits - 1), True)
    s = scale.to(x.dtype)[..., None]
    q = torch.round((y - offset.to(x.dtype)[..., None]) / torch.where(s > 0, s, 1)).clamp(0, 2 ** bits - 1)
    return q.flatten(-2).to(torch.uint8), scale, offset


def _rows(x, bits):
    """Bytes of the codes [..., dim * bits / 8] and of the pairs [..., groups * 4] of x."""
    q, scale, offset = _quantise(x, bits)
    if bits == 4:
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    return q, torch.stack([scale, offset], -1).flatten(-2).contiguous().view(torch.uint8)


def _put(pages, slots, k, v, bits):
    """Quantise k, v [T, kv, dim] into the pages at slots (page * PAGE + place)."""
    heads = torch.arange(pages.shape[1], device=pages.device)
    page, place = (slots // PAGE)[:, None, None], (slots % PAGE)[:, None, None]
    at = 0
    kq, kp = _rows(k, bits)
    vq, vp = _rows(v, bits)
    for r in (kq, vq, kp, vp):
        w = r.shape[-1]
        pages[page, heads[None, :, None], at + place * w + torch.arange(w, device=pages.device)] = r
        at += PAGE * w


def _take(pages, dim, bits, dtype):
    """The keys and values that pages [n, kv, bytes] stand for: two [n, kv, PAGE, dim]."""
    row, par = dim * bits // 8, 4 * (dim // _group(dim))
    q = pages[..., :2 * PAGE * row].unflatten(-1, (2, PAGE, row))
    p = pages[..., 2 * PAGE * row:].contiguous().view(BF16).unflatten(-1, (2, PAGE, par // 4, 2)).to(dtype)
    if bits == 4:
        q = torch.stack([q & 15, q >> 4], -1).flatten(-2)
    y = q.unflatten(-1, (par // 4, -1)).to(dtype)
    y = (y * p[..., 0, None] + p[..., 1, None]).flatten(-2)
    return y[:, :, 0], y[:, :, 1]


# ---------------------------------------------------------------- inputs
def _draws(seed, salt):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int.from_bytes(hashlib.sha256(f"{seed}/{salt}".encode()).digest()[:7], "little"))

    def normal(*shape, std=1.0, dtype=F32):
        return torch.empty(shape, dtype=F32, device="cuda").normal_(0.0, std, generator=gen).to(dtype)
    return gen, normal


def prepare(case, seed):
    c = case
    gen, normal = _draws(seed, "inputs")
    dtype = getattr(torch, c["dtype"])
    new, held = _lengths(c)
    n = c["seqs"]
    counts = [-(-h // PAGE) for h in held]
    total = sum(counts)
    stride = max(counts)
    order = torch.randperm(total + 3, generator=gen, device="cuda")[:total].to(torch.int32)
    tables = torch.full((n, stride), -1, dtype=torch.int32, device="cuda")
    first, at = [], 0
    for i, k in enumerate(counts):
        tables[i, :k] = order[at:at + k]
        first.append(at)
        at += k
    # a few channels of the keys are far larger than the others, as trained models have them
    loud = 1.0 + 3.0 * (torch.rand(c["kv"], c["dim"], generator=gen, device="cuda") < 0.04).float()
    pages = torch.zeros(total + 3, c["kv"], _page_bytes(c), dtype=torch.uint8, device="cuda")
    for lo in range(0, total, 1024):                     # what earlier steps left in the pages
        m = min(1024, total - lo)
        k = (normal(m * PAGE, c["kv"], c["dim"]) * loud).to(dtype).to(F32)
        v = normal(m * PAGE, c["kv"], c["dim"]).to(dtype).to(F32)
        slots = (order[lo:lo + m].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
        _put(pages, slots, k, v, c["bits"])
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    dev = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    s = dict(path=c["path"], bits=c["bits"], heads=c["heads"], kv=c["kv"], dim=c["dim"], pages=pages, tables=tables, new=new, held=held,
             cu=dev(cu), context=dev(held), first=dev(first), total_pages=total, scale=c["dim"] ** -0.5,
             window=0, slopes=None, sink=None)
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), dev(new, torch.long))
    pos = torch.arange(cu[-1], device="cuda") - dev(cu, torch.long)[seq] + (dev(held, torch.long) - dev(new, torch.long))[seq]
    s["positions"] = pos.to(torch.int32)
    s["slots"] = (tables[seq, pos // PAGE].long() * PAGE + pos % PAGE).to(torch.int32)
    s["seq"] = seq
    if c["path"] == "store":
        s["qkv"] = normal(cu[-1], (c["heads"] + 2 * c["kv"]) * c["dim"]).to(dtype)
        s["qkv"].view(cu[-1], -1, c["dim"])[:, c["heads"]:c["heads"] + c["kv"]] *= loud.to(dtype)
        s["inv_freq"] = 500000.0 ** (-torch.arange(0, c["dim"], 2, device="cuda", dtype=F64) / c["dim"])
    else:
        s["q"] = normal(cu[-1], c["heads"], c["dim"]).to(dtype)
    if c.get("sloped"):
        s["window"] = 1024
        s["slopes"] = dev([2.0 ** (-8.0 * (h + 1) / c["heads"]) for h in range(c["heads"])], F32)
        s["sink"] = normal(c["heads"])
    return s


# ---------------------------------------------------------------- the operators
def _rotate(x, positions, inv_freq):
    """x [T, heads, dim] float64, pairs (p, p + dim / 2)."""
    ang = positions.to(F64)[:, None, None] * inv_freq
    a, b = x.chunk(2, -1)
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)


def _store(s):
    T, H, K, D = s["qkv"].shape[0], s["heads"], s["kv"], s["dim"]
    x = s["qkv"].view(T, H + 2 * K, D).to(F64)
    qk = _rotate(x[:, :H + K], s["positions"], s["inv_freq"])
    _put(s["pages"], s["slots"].long(), qk[:, H:], x[:, H + K:], s["bits"])
    # the sequences' pages in order; what lies behind a sequence's last token reads as zero
    counts = (s["context"].long() + PAGE - 1) // PAGE
    seq = torch.repeat_interleave(torch.arange(len(s["held"]), device="cuda"), counts, output_size=s["total_pages"])
    place = torch.arange(s["total_pages"], device="cuda") - s["first"].long()[seq]
    k, v = _take(s["pages"][s["tables"][seq, place].long()], D, s["bits"], F32)
    there = (place[:, None] * PAGE + torch.arange(PAGE, device="cuda") < s["context"][seq][:, None])[:, None, :, None]
    dt = s["qkv"].dtype
    return {"q": qk[:, :H].to(dt), "k": torch.where(there, k, 0).to(dt), "v": torch.where(there, v, 0).to(dt)}


def _attend(s):
    """Attention of every new token over its sequence's pages: the sequences side by side, padded to the longest."""
    B, H, K, D = len(s["held"]), s["heads"], s["kv"], s["dim"]
    Q, L = max(s["new"]), s["tables"].shape[1] * PAGE
    k, v = _take(s["pages"][s["tables"].clamp(min=0).flatten().long()], D, s["bits"], F32)
    k, v = (x.view(B, -1, K, PAGE, D).transpose(1, 2).reshape(B, K, L, D) for x in (k, v))
    q = torch.zeros(B, Q, H, D, device="cuda")
    row = torch.arange(s["q"].shape[0], device="cuda") - s["cu"].long()[s["seq"]]
    q[s["seq"], row] = s["q"].to(F32)
    q = q.view(B, Q, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, -1, D)
    score = (q @ k.transpose(-1, -2)).view(B, H, Q, L) * s["scale"]
    at = (s["context"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None] + torch.arange(Q, device="cuda")
    dist = at[:, :, None] - torch.arange(L, device="cuda")
    seen = dist >= 0
    if s["window"]:
        seen = seen & (dist < s["window"])
    if s["slopes"] is not None:
        score = score - s["slopes"][:, None, None] * dist[:, None]
    score = torch.where(seen[:, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"][:, None, None])
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"][:, None, None] - top)
    out = weight.view(B, K, -1, L) @ torch.where(torch.arange(L, device="cuda")[:, None] < s["context"][:, None, None, None], v, 0)
    out = (out.view(B, H, Q, D) / total).transpose(1, 2)
    return out[s["seq"], row].to(s["q"].dtype)


def run(state):
    s = state
    if not own:
        return _store(s) if s["path"] == "store" else _attend(s)
    from gollmgo_b200.cache import PackedKV
    kv = PackedKV(s["pages"], s["dim"], PAGE, s["bits"])
    if s["path"] == "store":
        q = kv.write(s["qkv"], s["positions"], s["slots"], s["heads"], s["inv_freq"])
        k, v = kv.read(s["tables"], s["context"], s["first"], s["total_pages"], s["qkv"].dtype)
        return {"q": q, "k": k, "v": v}
    more = dict(window=s["window"], slopes=s["slopes"], sink=s["sink"])
    if s["path"] == "decode":
        return kv.decode(s["q"], s["tables"], s["context"], max(s["held"]), s["scale"], **more)
    return kv.prefill(s["q"], s["tables"], s["cu"], s["context"], s["new"], s["held"], s["scale"], **more)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    new, held = _lengths(c)
    esize = 2 if c["dtype"] == "bfloat16" else 4
    token = _page_bytes(c) // PAGE * c["kv"]              # bytes of a stored token
    T, H, K, D = sum(new), c["heads"], c["kv"], c["dim"]
    if c["path"] == "store":
        qkv = T * (H + 2 * K) * D * esize
        back = sum(-(-h // PAGE) * PAGE for h in held) * 2 * K * D * esize
        return {"bytes": qkv + T * H * D * esize + T * token + sum(held) * token + back,
                "flops": 6 * T * (H + K) * D // 2 + 6 * T * 2 * K * D + 2 * sum(held) * 2 * K * D}
    window = 1024 if c.get("sloped") else 1 << 40
    read = sum(min(h, window + a - 1) for a, h in zip(new, held))
    pairs = sum(sum(min(h - a + i + 1, window) for i in range(a)) for a, h in zip(new, held))
    return {"bytes": 2 * T * H * D * esize + read * token, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------- in 64 bits, sequence by sequence
def _bf16_bits(x, up):
    """Directed rounding to eight significant bits: x = m 2^e with |m| in [1/2, 1)."""
    m, e = torch.frexp(x)
    m = m * 256
    return torch.ldexp(torch.ceil(m) if up else torch.floor(m), e - 8)


def _through(x, bits):
    """What x [tokens, kv, dim] (float64) reads as once it has been stored."""
    g = _group(x.shape[2])
    out = torch.empty_like(x)
    for lo in range(0, x.shape[2], g):
        y = x[:, :, lo:lo + g]
        low = _bf16_bits(y.min(2, keepdim=True).values, False)
        step = _bf16_bits((y.max(2, keepdim=True).values - low) / (2 ** bits - 1), True)
        code = torch.where(step > 0, (y - low) / step, 0.0).round()
        out[:, :, lo:lo + g] = low + step * code.clamp(max=2 ** bits - 1)
    return out


def _held_rows(s, i):
    """Keys and values of sequence i as its pages hold them: two [tokens, kv, dim] float64."""
    n, D, bits = s["held"][i], s["dim"], s["bits"]
    row, pairs = D * bits // 8, D // _group(D)
    raw = s["pages"][s["tables"][i, :-(-n // PAGE)].long()].transpose(0, 1)           # [kv, pages, bytes]
    found = []
    for j in (0, 1):
        code = raw[:, :, j * PAGE * row:(j + 1) * PAGE * row].reshape(s["kv"], -1, row)[:, :n]
        if bits == 4:
            code = torch.stack((code % 16, code // 16), 3).reshape(s["kv"], n, D)
        at = 2 * PAGE * row + j * PAGE * pairs * 4
        pair = raw[:, :, at:at + PAGE * pairs * 4].contiguous().view(BF16).to(F64).reshape(s["kv"], -1, pairs, 2)[:, :n]
        pair = pair.repeat_interleave(D // pairs, 2)
        found.append((pair[..., 1] + pair[..., 0] * code.to(F64)).transpose(0, 1))
    return found


def exact(case, seed):
    s = prepare(case, seed)
    H, K, D = s["heads"], s["kv"], s["dim"]
    outs, ks, vs = [], [], []
    for i, (a, n) in enumerate(zip(s["new"], s["held"])):
        lo = int(s["cu"][i])
        k, v = _held_rows(s, i)
        if s["path"] == "store":
            x = s["qkv"][lo:lo + a].to(F64).view(a, H + 2 * K, D)
            turn = torch.polar(torch.ones(a, D // 2, dtype=F64, device="cuda"),
                               torch.arange(n - a, n, device="cuda", dtype=F64)[:, None] * s["inv_freq"])[:, None]
            z = torch.complex(x[:, :H + K, :D // 2], x[:, :H + K, D // 2:]) * turn
            qk = torch.cat([z.real, z.imag], 2)
            outs.append(qk[:, :H])
            k[n - a:], v[n - a:] = _through(qk[:, H:], s["bits"]), _through(x[:, H + K:], s["bits"])
            for kept, y in ((ks, k), (vs, v)):
                full = torch.zeros(-(-n // PAGE) * PAGE, K, D, dtype=F64, device="cuda")
                full[:n] = y
                kept.append(full.view(-1, PAGE, K, D).transpose(1, 2))
            continue
        q = s["q"][lo:lo + a].to(F64)
        where = torch.arange(n - a, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None]
        out = torch.empty(a, H, D, dtype=F64, device="cuda")
        for h in range(H):
            z = q[:, h] @ k[:, h * K // H].T * s["scale"]
            if s["slopes"] is not None:
                z = z - s["slopes"][h].to(F64) * where
            z = z.masked_fill(where < 0, -math.inf)
            if s["window"]:
                z = z.masked_fill(where >= s["window"], -math.inf)
            if s["sink"] is not None:
                z = torch.cat([z, s["sink"][h].to(F64).expand(a, 1)], 1)
            out[:, h] = torch.softmax(z, 1)[:, :n] @ v[:, h * K // H]
        outs.append(out)
    if s["path"] == "store":
        return {"q": torch.cat(outs), "k": torch.cat(ks), "v": torch.cat(vs)}
    return torch.cat(outs)
