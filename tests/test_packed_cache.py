"""The packed cache on the device against its plain 64-bit implementation (tests/plain_packed.py): what a write leaves in the
pages, what reads back, and attention over them, with the sizes, masks and layouts where it can go wrong."""
import math

import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def kit():
    from gollmgo_b200.cache import PackedKV
    from gollmgo_b200.csrc import ops
    return PackedKV, ops


def freqs(rot, theta=500000.0):
    return theta ** (-torch.arange(0, rot, 2, dtype=F64) / rot)


class Pool:
    """Packed pages of several sequences in a shuffled pool, with random codes where nothing was written, and the float64
    keys and values that the pages stand for (host)."""

    def __init__(self, lens, nkv, d, page, bits, seed, dtype=BF16, spare=3):
        PackedKV, _ = kit()
        g = torch.Generator().manual_seed(seed)
        self.lens, self.nkv, self.d, self.page, self.bits = list(lens), nkv, d, page, bits
        counts = [-(-n // page) for n in lens]
        total = sum(counts) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.width = max(counts + [1]) + 1
        self.tables = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        host = torch.randint(0, 256, (total, nkv, plain.page_bytes(bits, d, page)), dtype=torch.uint8, generator=g)
        # whatever was there before: every pair a NaN, so that a key that is not in sight shows where it is used
        pairs = 2 * page * (d * bits // 8)
        host[..., pairs:] = 0xff
        self.keys, self.values = [], []
        at = 0
        for b, (n, c) in enumerate(zip(lens, counts)):
            self.tables[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
            x = torch.randn(2, n, nkv, d, generator=g).to(dtype).double()
            code, scale, off = plain.quantise(x, bits)
            y = plain.dequantise(code, scale, off)
            self.keys.append(y[0])
            self.values.append(y[1])
            if n == 0:
                continue
            row, par = d * bits // 8, 4 * (d // plain.group_of(d))
            c8 = code.to(torch.int64)
            if bits == 4:
                c8 = c8[..., 0::2] + 16 * c8[..., 1::2]
            c8 = c8.to(torch.uint8)
            pr = torch.stack([scale, off], -1).flatten(-2).float().to(BF16).contiguous().view(torch.uint8)
            tok = torch.arange(n)
            pg, pl = self.tables[b][tok // page].long(), tok % page
            for which in (0, 1):
                for h in range(nkv):
                    cols = which * page * row + pl[:, None] * row + torch.arange(row)
                    host[pg[:, None], h, cols] = c8[which, :, h]
                    cols = 2 * page * row + which * page * par + pl[:, None] * par + torch.arange(par)
                    host[pg[:, None], h, cols] = pr[which, :, h]
        self.host = host
        self.kv = PackedKV(host.cuda(), d, page, bits)

    def slots(self, b, lo, hi):
        t = torch.arange(lo, hi)
        return (self.tables[b][t // self.page].long() * self.page + t % self.page).to(torch.int32)


# ---------------------------------------------------------------- the write
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh,nkv,d,rot,interleaved,page", [
    (4, 2, 64, 64, False, 16), (32, 8, 128, 128, False, 16), (5, 5, 96, 64, False, 8), (3, 1, 256, 256, True, 32),
    (2, 2, 16, 8, True, 4), (6, 3, 80, 0, False, 16), (8, 1, 128, 128, False, 64), (16, 4, 128, 64, False, 16)])
def test_write_leaves_the_codes_of_the_formula(bits, dtype, nh, nkv, d, rot, interleaved, page):
    PackedKV, _ = kit()
    T, pages_n = 21, 7
    g = torch.Generator().manual_seed(bits * 1000 + d + nh)
    qkv = (torch.randn(T, (nh + 2 * nkv) * d, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(dtype)
    pos = torch.randint(0, 100000, (T,), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages_n * page, generator=g)[:T].to(torch.int32)
    slots[3], slots[7], slots[8] = -1, pages_n * page, 2 ** 31 - 1          # not stored
    before = torch.randint(0, 256, (pages_n, nkv, plain.page_bytes(bits, d, page)), dtype=torch.uint8, generator=g)
    kv = PackedKV(before.clone().cuda(), d, page, bits)
    inv = freqs(rot) if rot else None
    q = kv.write(qkv.cuda(), pos.cuda(), slots.cuda(), nh, inv.cuda() if rot else None, interleaved, 1.25 if rot else 1.0)
    want = before.clone()
    eps = torch.finfo(dtype).eps / 2
    for t in range(T):
        x = qkv[t].double().view(nh + 2 * nkv, d)
        y = plain.rotate(x[:nh + nkv], float(pos[t]), inv, interleaved, 1.25) if rot else x[:nh + nkv]
        # one rounding of the result, and (bfloat16 mode) a float32 rotation: a few float32 steps of the two products
        big = torch.maximum(x[:nh].abs().amax(-1, keepdim=True), y[:nh].abs())
        assert ((q[t].cpu().double() - y[:nh]).abs() <= eps * y[:nh].abs() + (8 * 2.0 ** -24 if dtype == BF16 else 2.0 ** -50) * 2 * big).all()
        s = int(slots[t])
        if s < 0 or s >= pages_n * page:
            continue
        for h in range(nkv):
            plain.put(want, s, h, y[nh + h], x[nh + nkv + h], bits, page)
    assert torch.equal(kv.pages.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nh,nkv,d", [(4, 8, 128), (2, 8, 64), (1, 2, 96)])
def test_many_rotated_keys_take_the_codes_of_the_formula(bits, nh, nkv, d):
    """Far positions, a million keys' channels: none on the wrong side of a border between two codes, or of a bfloat16 scale or offset."""
    PackedKV, _ = kit()
    T, page = 1100, 16
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(T, (nh + 2 * nkv) * d, generator=g).to(BF16).cuda()
    pos = torch.randint(0, 131072, (T,), generator=g, dtype=torch.int32).cuda()
    kv = PackedKV.empty(-(-T // page), nkv, d, page, bits)
    kv.write(qkv, pos, torch.arange(T, dtype=torch.int32).cuda(), nh, freqs(d).cuda())
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    n = kv.pages.shape[0]
    k, v = kv.read(torch.arange(n, dtype=torch.int32).view(1, n).cuda(), dev([T]), dev([0]), n, F32)
    x = qkv.view(T, -1, d)[:, nh:].double()
    ang = pos.double()[:, None, None] * freqs(d).cuda()
    a, b = x[:, :nkv].chunk(2, -1)
    keys = torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    for got, want in ((k, keys), (v, x[:, nkv:])):
        got = got.transpose(1, 2).reshape(-1, nkv, d)[:T].double()
        want = plain.through(want.cpu(), bits)
        assert ((got.cpu() - want).abs() <= 2.0 ** -22 * want.abs().clamp(min=1e-3)).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_write_of_hard_rows(bits, dtype):
    """Constant rows, zeros, one huge value, the largest range, subnormals, exact ties, infinities and NaN."""
    PackedKV, _ = kit()
    d, page = 64, 16
    big = torch.finfo(BF16).max
    rows = [torch.zeros(d), torch.full((d,), -3.0), torch.full((d,), 0.1), torch.arange(d).float(), torch.arange(d) * 0.5 - 7,
            torch.cat([torch.tensor([1e4]), torch.linspace(-1, 1, d - 1)]), torch.linspace(-big, big, d), torch.full((d,), 2.0 ** -130),
            torch.linspace(-2.0 ** -120, 2.0 ** -121, d), torch.cat([torch.tensor([math.inf]), torch.ones(d - 1)]),
            torch.cat([torch.ones(d - 1), torch.tensor([math.nan])]), torch.cat([torch.tensor([-math.inf]), torch.zeros(d - 1)]),
            torch.cat([torch.tensor([0.0, 15.0]), torch.arange(d - 2) % 30 * 0.5]), torch.cat([torch.tensor([0.0, 255.0]), torch.arange(d - 2) % 510 * 0.5])]
    T = len(rows)
    v = torch.stack(rows).to(dtype)
    qkv = torch.cat([v.flip(0), v], 1)                        # no q heads: keys and values alone
    kv = PackedKV.empty(2, 1, d, page, bits)
    slots = torch.arange(T, dtype=torch.int32)
    q = kv.write(qkv.cuda(), None, slots.cuda(), 0)
    assert q.shape == (T, 0, d)
    got = kv.pages.cpu()
    for t in range(T):
        k1, v1 = plain.get(got, t, 0, d, bits, page)
        for y, x in ((k1, v.flip(0)[t].double()), (v1, v[t].double())):
            if not torch.isfinite(x).all():
                assert torch.isnan(y).all()
                continue
            code, scale, off = plain.quantise(x, bits)
            tiny = 2.0 ** -132                                 # a scale below the smallest normal bfloat16 is one of the subnormal ones
            assert ((y - x).abs() <= scale.max() * 0.5 + tiny).all()
            if scale.max() > 2.0 ** -126 or scale.max() == 0:
                assert torch.equal(y, plain.dequantise(code, scale, off))


def test_write_takes_strided_rows_and_rotates_in_place():
    PackedKV, _ = kit()
    nh, nkv, d, T = 4, 2, 64, 9
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(T, (nh + 2 * nkv) * d + 40, generator=g).to(BF16).cuda()
    pos, slots, inv = torch.arange(T, dtype=torch.int32).cuda() + 50, torch.arange(T, dtype=torch.int32).cuda(), freqs(d).cuda()
    a, b = PackedKV.empty(1, nkv, d, 16, 4), PackedKV.empty(1, nkv, d, 16, 4)
    q1 = a.write(wide[:, :(nh + 2 * nkv) * d].contiguous(), pos, slots, nh, inv)
    rest = wide[:, nh * d:].clone()
    view = wide[:, :nh * d].unflatten(1, (nh, d))
    q2 = b.write(wide[:, :(nh + 2 * nkv) * d], pos, slots, nh, inv, q_out=view)
    assert torch.equal(q1, q2) and q2.data_ptr() == wide.data_ptr()
    assert torch.equal(a.pages, b.pages)
    assert torch.equal(wide[:, nh * d:], rest)               # only the q columns were written


# ---------------------------------------------------------------- reading back
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nkv,d,page", [(2, 64, 16), (8, 128, 16), (1, 96, 8), (3, 256, 4), (2, 16, 32), (5, 80, 16)])
def test_read_gives_what_the_pages_stand_for(bits, dtype, nkv, d, page):
    lens = [1, page, page + 1, 3 * page - 1, 0, 2 * page]
    pool = Pool(lens, nkv, d, page, bits, seed=d + bits)
    pool.tables[5, 0] = -1                                    # given back: reads as zero
    counts = [-(-n // page) for n in lens]
    first, at = [], 2
    for c in counts:
        first.append(at)
        at += c
    mark = 7.0
    out = tuple(torch.full((at + 1, nkv, page, d), mark, dtype=dtype, device="cuda") for _ in range(2))
    k, v = pool.kv.read(pool.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(first, dtype=torch.int32).cuda(),
                        at + 1, dtype, out)
    eps = torch.finfo(dtype).eps / 2
    for got, held in ((k, pool.keys), (v, pool.values)):
        got = got.cpu().double()
        assert (got[:2] == mark).all() and (got[at:] == mark).all()
        for b, n in enumerate(lens):
            rows = got[first[b]:first[b] + counts[b]].transpose(1, 2).reshape(-1, nkv, d)
            want = held[b].clone()
            if b == 5:
                want[:page] = 0
            # the result rounds once; scale * code + offset in float32 before that is off by its own rounding
            assert ((rows[:n] - want).abs() <= (eps + 2.0 ** -23) * want.abs() + 1e-30).all()
            assert (rows[n:] == 0).all()


# ---------------------------------------------------------------- attention
def bound(ref, values, dtype, score_err, weight_err):
    """|out - ref| at most: the result's own rounding, and weights off by score_err (relative, twice: numerator and sum) and weight_err."""
    top = max(float(v.abs().max()) if v.numel() else 0.0 for v in values)
    return torch.finfo(dtype).eps / 2 * ref.abs() + (2 * score_err + weight_err) * top + 1e-30


OPTIONS = [dict(), dict(window=20), dict(softcap=5.0), dict(sink=True), dict(slopes=True, window=33, sink=True, temperature=(0.1, 16))]


def options_of(o, nh, seed):
    g = torch.Generator().manual_seed(seed)
    o = dict(o)
    if o.get("sink"):
        o["sink"] = torch.randn(nh, generator=g)
    if o.get("slopes"):
        o["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)])
    return o, {k: v.cuda() if torch.is_tensor(v) else v for k, v in o.items()}


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("option", range(len(OPTIONS)))
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 16), (32, 8, 128, 16), (5, 5, 128, 32), (16, 1, 128, 16), (40, 2, 64, 64), (6, 2, 96, 16),
                                           (4, 1, 256, 16), (4, 2, 128, 8), (3, 1, 16, 4)])
def test_decode(bits, dtype, option, nh, nkv, d, page):
    lens = [1, 15, 16, 17, 64, 65, 200, 0, 131]
    pool = Pool(lens, nkv, d, page, bits, seed=d + option, dtype=dtype)
    o, oc = options_of(OPTIONS[option], nh, 5)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(len(lens), nh, d, generator=g).to(dtype)
    scale = d ** -0.5
    out = pool.kv.decode(q.cuda(), pool.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), max(lens), scale, **oc).cpu().double()
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        ref = plain.attend(q[b:b + 1].double(), pool.keys[b], pool.values[b], n, scale, **o)[0]
        assert ((out[b] - ref).abs() <= bound(ref, [pool.values[b]], dtype, *errors_of(dtype, q[b], pool.keys[b], scale))).all(), (b, n)


def errors_of(dtype, q, keys, scale):
    """Scores: d products summed in float32, relative to sum |q k| <= |q| |k|: a few steps of 2^-24 of it (the sum may be
    truncated where a tensor core adds: 2^-21).  Weights: 2^-11 in bfloat16 mode (they are rounded to half precision), 2^-20 in float32."""
    size = float(q.double().norm(dim=-1).max() * keys.norm(dim=-1).max()) * scale * 1.2
    return size * 2.0 ** -20 + 2.0 ** -20, 2.0 ** -11 if dtype == BF16 else 2.0 ** -20


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("page", [16, 8])
def test_decode_of_listed_sequences(bits, page):
    """Tokens of some of a step's sequences: seqs with padding, rows through cu_q_lens, the other rows left as they were (pages of 16:
    on the tensor cores, of 8: the general kernel).  A context longer than its block table is cut there."""
    nh, nkv, d = 8, 2, 128
    lens = [40, 7, 90, 33]
    pool = Pool(lens, nkv, d, page, bits, seed=1)
    g = torch.Generator().manual_seed(2)
    cu = torch.tensor([0, 3, 4, 9, 10], dtype=torch.int32)                 # sequences 1 and 3 bring one token
    wide = torch.randn(10, (nh + 2 * nkv) * d, generator=g).to(BF16).cuda()
    q = wide[:, :nh * d].unflatten(1, (nh, d))
    out = torch.full((10, nh, d), 3.0, dtype=BF16, device="cuda")
    seqs = torch.tensor([3, -1, 1, 4], dtype=torch.int32).cuda()           # below 0 and beyond the tables: padding
    pool.kv.decode(q, pool.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 90, d ** -0.5, cu_q_lens=cu.cuda(), seqs=seqs, out=out)
    for b in (1, 3):
        row = int(cu[b])
        ref = plain.attend(q[row:row + 1].cpu().double(), pool.keys[b], pool.values[b], lens[b], d ** -0.5)[0]
        e = errors_of(BF16, q[row].cpu(), pool.keys[b], d ** -0.5)
        assert ((out[row].cpu().double() - ref).abs() <= bound(ref, [pool.values[b]], BF16, *e)).all()
    others = [r for r in range(10) if r not in (3, 9)]
    assert (out[others] == 3.0).all()
    held = -(-90 // page) * page                       # sequence 2 with a table of just its pages and a context that says more
    far = pool.kv.decode(q[4:5], pool.tables[2:3, :held // page].contiguous().cuda(), torch.tensor([10 ** 6], dtype=torch.int32).cuda(), 90, d ** -0.5)
    same = pool.kv.decode(q[4:5], pool.tables[2:3].cuda(), torch.tensor([held], dtype=torch.int32).cuda(), 90, d ** -0.5)
    assert torch.equal(far.isnan(), same.isnan()) and torch.equal(far.nan_to_num(), same.nan_to_num())


def prompt_errors(dtype, q, keys, scale):
    """Prompt portions may read the cache back in the type of the activations: keys, values and weights round once each."""
    s, w = errors_of(dtype, q, keys, scale)
    if dtype == BF16:
        s += float(q.double().norm(dim=-1).max() * keys.norm(dim=-1).max()) * scale * 2.0 ** -8
        w += 2 * 2.0 ** -8
    return s, w


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("option", range(len(OPTIONS)))
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 16), (8, 4, 128, 16), (5, 5, 128, 32), (6, 2, 96, 16), (2, 1, 256, 8), (3, 1, 16, 4)])
def test_prefill(bits, dtype, option, nh, nkv, d, page):
    q_lens, lens = [5, 1, 33, 16, 2, 70], [5, 40, 90, 16, 65, 140]
    pool = Pool(lens, nkv, d, page, bits, seed=d + option, dtype=dtype)
    o, oc = options_of(OPTIONS[option], nh, 5)
    cu = [0]
    for a in q_lens:
        cu.append(cu[-1] + a)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(cu[-1], nh, d, generator=g).to(dtype)
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    out = pool.kv.prefill(q.cuda(), pool.tables.cuda(), dev(cu), dev(lens), q_lens, lens, d ** -0.5, **oc).cpu().double()
    for b, (a, n) in enumerate(zip(q_lens, lens)):
        x = q[cu[b]:cu[b + 1]]
        ref = plain.attend(x.double(), pool.keys[b], pool.values[b], n, d ** -0.5, **o)
        e = prompt_errors(dtype, x, pool.keys[b], d ** -0.5)
        assert ((out[cu[b]:cu[b + 1]] - ref).abs() <= bound(ref, [pool.values[b]], dtype, *e)).all(), (b, a, n)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (3, 1), (7, 1), (9, 1), (24, 1), (17, 1), (32, 1), (66, 2)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_groups_of_any_size(bits, nh, nkv, d, dtype):
    lens = [33, 5, 260]
    pool = Pool(lens, nkv, d, 16, bits, seed=nh)
    g = torch.Generator().manual_seed(nh)
    q = torch.randn(3, nh, d, generator=g).to(dtype)
    out = pool.kv.decode(q.cuda(), pool.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 260, d ** -0.5).cpu().double()
    for b, n in enumerate(lens):
        ref = plain.attend(q[b:b + 1].double(), pool.keys[b], pool.values[b], n, d ** -0.5)[0]
        assert ((out[b] - ref).abs() <= bound(ref, [pool.values[b]], dtype, *errors_of(dtype, q[b], pool.keys[b], d ** -0.5))).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nh,nkv", [(1, 1), (4, 2), (3, 1), (8, 2), (5, 1), (8, 1), (16, 1), (9, 1)])
@pytest.mark.parametrize("d,window,option", [(64, 0, 0), (128, 7, 1), (128, 40, 0), (64, 100, 1)])
def test_prompts_in_float32_of_groups_of_any_size(bits, nh, nkv, d, window, option):
    """Rows of a portion share the columns of a product where a kv head has few heads: portions that end inside such a group, windows
    and contexts that end between its rows; the rows of short sequences and behind the last one stay as they were."""
    q_lens, lens = [13, 1, 0, 64, 3, 7], [13, 50, 9, 200, 65, 300]
    pool = Pool(lens, nkv, d, 16, bits, seed=nh + window, dtype=F32)
    o, oc = options_of(dict(softcap=20.0, slopes=True, sink=True, temperature=(0.1, 8.0)) if option else {}, nh, 3)
    cu = [0]
    for a in q_lens:
        cu.append(cu[-1] + a)
    q = torch.randn(cu[-1] + 2, nh, d, generator=torch.Generator().manual_seed(nh))
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    out = torch.full((cu[-1] + 2, nh, d), 3.0, device="cuda")
    pool.kv.prefill(q.cuda(), pool.tables.cuda(), dev(cu), dev(lens), q_lens, lens, d ** -0.5, window=window, least=3, out=out, **oc)
    out = out.cpu().double()
    for b, (a, n) in enumerate(zip(q_lens, lens)):
        x = q[cu[b]:cu[b + 1]]
        if a < 3:
            assert (out[cu[b]:cu[b + 1]] == 3.0).all()
            continue
        ref = plain.attend(x.double(), pool.keys[b], pool.values[b], n, d ** -0.5, window=window, **o)
        e = errors_of(F32, x, pool.keys[b], d ** -0.5)
        e = (e[0] * (1.0 + 0.1 * math.log(1 + n / 8.0) if option else 1.0), e[1])
        assert ((out[cu[b]:cu[b + 1]] - ref).abs() <= bound(ref, [pool.values[b]], F32, *e)).all(), (b, a, n)
    assert (out[cu[-1]:] == 3.0).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (8, 2), (10, 1)])
def test_prompts_in_float32_see_bad_tokens_of_their_own_past_only(bits, nh, nkv):
    d, n, page = 64, 37, 16
    g = torch.Generator().manual_seed(nh)
    x = torch.randn(n, (nh + 2 * nkv) * d, generator=g)
    x[17, nh * d + 3] = math.nan                              # a key of kv head 0
    x[6, (nh + 2 * nkv) * d - 1] = math.inf                   # a value of the last kv head
    kv = PackedKV_of(4, nkv, d, page, bits)
    tables = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    t = torch.arange(n)
    q = kv.write(x.cuda(), None, (tables[0][t // page] * page + t % page).to(torch.int32).cuda(), nh)
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()
    out = kv.prefill(q, tables.cuda(), dev([0, n]), dev([n]), [n], [n], 0.125, window=9)
    for row in range(n):
        for h in range(nh):
            kvh = h * nkv // nh
            past = range(max(0, row - 8), row + 1)
            bad = (kvh == 0 and 17 in past) or (kvh == nkv - 1 and 6 in past)
            assert bool(out[row, h].isnan().any()) == bad, (row, h)


@pytest.mark.parametrize("bits", [4, 8])
def test_prompts_in_float32_of_more_items_than_a_launch_takes(bits):
    PackedKV, ops = kit()
    nh, nkv, d, page = 8, 1, 64, 16
    a, n = ops.PACKED_DECODE_TOKENS + 90, ops.PACKED_DECODE_TOKENS + 90
    pool = Pool([40, n], nkv, d, page, bits, seed=1, dtype=F32)
    q = torch.randn(3 + a, nh, d, generator=torch.Generator().manual_seed(2))
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()
    out = pool.kv.prefill(q.cuda(), pool.tables.cuda(), dev([0, 3, 3 + a]), dev([40, n]), [3, a], [40, n], 0.125).cpu().double()
    for b, lo, hi, c in ((0, 0, 3, 40), (1, 3, 3 + a, n)):
        ref = plain.attend(q[lo:hi].double(), pool.keys[b], pool.values[b], c, 0.125)
        assert ((out[lo:hi] - ref).abs() <= bound(ref, [pool.values[b]], F32, *errors_of(F32, q[lo:hi], pool.keys[b], 0.125))).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("window", [0, 1, 16, 31, 1000])
def test_decode_of_contexts_longer_than_said_and_of_every_split(bits, window):
    """max_context only spreads the work: any value gives the same attention.  Long contexts are cut between blocks."""
    nh, nkv, d, page = 4, 1, 128, 16
    lens = [900, 1, 31, 2500]
    pool = Pool(lens, nkv, d, page, bits, seed=window)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(4, nh, d, generator=g).to(BF16)
    args = (q.cuda(), pool.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    for said in (1, 40, 600, 2500, 100000):
        out = pool.kv.decode(*args, said, d ** -0.5, window=window).cpu().double()
        for b, n in enumerate(lens):
            ref = plain.attend(q[b:b + 1].double(), pool.keys[b], pool.values[b], n, d ** -0.5, window=window)[0]
            assert ((out[b] - ref).abs() <= bound(ref, [pool.values[b]], BF16, *errors_of(BF16, q[b], pool.keys[b], d ** -0.5))).all(), (said, n)
    alone = pool.kv.decode(args[0][3:], args[1][3:], args[2][3:], 2500, d ** -0.5, window=window).cpu().double()
    ref = plain.attend(q[3:].double(), pool.keys[3], pool.values[3], 2500, d ** -0.5, window=window)[0]
    assert ((alone[0] - ref).abs() <= bound(ref, [pool.values[3]], BF16, *errors_of(BF16, q[3], pool.keys[3], d ** -0.5))).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_of_bad_values_and_far_scales(bits, dtype):
    """Infinities and NaN reach the heads (keys) or channels (values) that see them and nothing else; values of 2^100 beside values of
    2^-100, and a loud token that is hardly attended to, cost the others nothing."""
    nh, nkv, d, page, n = 4, 2, 128, 16, 100
    g = torch.Generator().manual_seed(7)
    x = torch.randn(4, n, (nh + 2 * nkv) * d, generator=g)
    k0 = nh * d
    v0 = k0 + nkv * d
    x[0, 3, k0 + 5] = math.nan                      # sequence 0: a key of kv head 0, behind the window
    x[0, 2, v0 + d + 70] = math.inf                 # ... and a value of kv head 1
    x[1, 90, k0 + 5] = -math.inf                    # sequence 1: a key of kv head 0 in sight
    x[1, 91, v0 + d + 70] = math.nan                # ... a value of kv head 1, second group of channels
    x[2, :, v0:v0 + d] *= 2.0 ** 100                # sequence 2: huge and tiny values
    x[2, :, v0 + d:] *= 2.0 ** -100
    x[3, 80, v0:] *= 2.0 ** 20                      # sequence 3: one loud value, whose key points away
    x[3, 80, k0:v0] *= -4.0
    x = x.to(dtype)
    kv = PackedKV_of(4 * 8, nkv, d, page, bits)
    tables = torch.arange(32, dtype=torch.int32).view(4, 8)
    slots = (tables.repeat_interleave(page, 1)[:, :n] * page + torch.arange(n) % page).to(torch.int32)
    q = x[:, -1, :k0].view(4, nh, d) * 1.0
    q[3] = -8 * x[3, 80, k0:v0].view(nkv, 1, d).expand(nkv, nh // nkv, d).reshape(nh, d) / x[3, 80, k0:v0].abs().max()
    kv.write(x.reshape(4 * n, -1).cuda(), None, slots.reshape(-1).cuda(), nh)
    out = kv.decode(q.cuda(), tables.cuda(), torch.full((4,), n, dtype=torch.int32).cuda(), n, d ** -0.5, window=90).cpu().double()
    grp = nh // nkv
    for b in range(4):
        held = [torch.stack([torch.stack([plain.get(kv.pages[b * 8:b * 8 + 8].cpu(), t, h, d, bits, page)[w] for h in range(nkv)]) for t in range(n)])
                for w in (0, 1)]
        for h in range(nh):
            kvh = h // grp
            ref = plain.attend(q[b:b + 1, h:h + 1].double(), held[0][:, kvh:kvh + 1], held[1][:, kvh:kvh + 1], n, d ** -0.5, window=90)[0, 0]
            if b == 1 and kvh == 0:
                assert torch.isnan(out[b, h]).all()
                continue
            if b == 1:
                bad = torch.isnan(ref)
                assert bad[64:].all() and not bad[:64].any()
                assert torch.equal(torch.isnan(out[b, h]), bad)
                continue
            seen = held[1][n - 90:, kvh]
            p = torch.softmax(held[0][n - 90:, kvh] @ q[b, h].double() * d ** -0.5, 0)
            size = (p[:, None] * seen.abs()).sum(0).max()          # what the weights' roundings are relative to
            e, wt = errors_of(dtype, q[b, h:h + 1], held[0][n - 90:, kvh:kvh + 1], d ** -0.5)
            assert ((out[b, h] - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (2 * e + 2 * wt) * size).all(), (b, h)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("loud", [2.0 ** 25, 2.0 ** 60])
def test_loud_values_that_another_head_or_an_earlier_key_attends_to(bits, dtype, d, loud):
    """Head 0 attends to one loud value, head 1 of the same kv head does not: what it sums is held relative to its own.  Head 2 attends to
    another loud value in an early tile, but far more to what comes later."""
    n, page, nh = 400, 16, 3
    g = torch.Generator().manual_seed(11)
    x = torch.randn(n, (nh + 2) * d, generator=g)
    k, v = x[:, nh * d:(nh + 1) * d], x[:, (nh + 1) * d:]
    k[:, :2] = 0.0
    k[[150, 5], 0] = torch.tensor([30.0, -30.0])
    k[300:, 1] = 30.0
    v[[150, 5]] *= loud
    x = x.to(dtype)
    q = torch.randn(1, nh, d, generator=g) * 0.3
    q[0, 0, :2] = torch.tensor([8.0, 0.0])                     # towards key 150
    q[0, 1, :2] = torch.tensor([0.0, 50.0])                    # to the keys from 300 on alone
    q[0, 2, :2] = torch.tensor([-8.0, 60.0])                   # towards key 5, and more to those
    q = q.to(dtype)
    kv = PackedKV_of(n // page, 1, d, page, bits)
    kv.write(x.cuda(), None, torch.arange(n, dtype=torch.int32).cuda(), nh)
    out = kv.decode(q.cuda(), torch.arange(n // page, dtype=torch.int32).view(1, -1).cuda(), torch.tensor([n], dtype=torch.int32).cuda(), n, 0.5).cpu().double()
    held = [torch.stack([torch.stack([plain.get(kv.pages.cpu(), t, 0, d, bits, page)[w]]) for t in range(n)]) for w in (0, 1)]
    for h in range(nh):
        ref = plain.attend(q[:, h:h + 1].double(), held[0], held[1], n, 0.5)[0, 0]
        p = torch.softmax(held[0][:, 0] @ q[0, h].double() * 0.5, 0)
        size = (p[:, None] * held[1][:, 0].abs()).sum(0).max()
        e, w = errors_of(dtype, q[0, h:h + 1], held[0], 0.5)
        assert ((out[0, h] - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (2 * e + 2 * w) * size).all(), h


def PackedKV_of(*a):
    return kit()[0].empty(*a)


@pytest.mark.parametrize("bits", [4, 8])
def test_more_tokens_than_a_launch_takes(bits):
    PackedKV, ops = kit()
    n, nh, nkv, d, page = ops.PACKED_DECODE_TOKENS + 77, 2, 1, 64, 16
    kv = PackedKV.empty(n, nkv, d, page, bits)
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(n * page, (nh + 2 * nkv) * d, generator=g).to(BF16).cuda()
    kv.write(rows, None, torch.arange(n * page, dtype=torch.int32).cuda(), nh)
    tables = torch.randperm(n, generator=g).to(torch.int32).view(n, 1).cuda()
    ctx = torch.randint(0, page + 1, (n,), generator=g).to(torch.int32).cuda()
    q = torch.randn(n, nh, d, generator=g).to(BF16).cuda()
    out = kv.decode(q, tables, ctx, page, 0.125)
    k, v = kv.read(tables, torch.full_like(ctx, page), torch.arange(n, dtype=torch.int32).cuda(), n, F32)
    z = torch.einsum("bhd,bpd->bhp", q.float(), k[:, 0]) * 0.125
    z = z.masked_fill(torch.arange(page, device="cuda") >= ctx[:, None, None], -math.inf)
    w = torch.where(ctx[:, None, None] > 0, torch.softmax(z, -1), 0).nan_to_num()
    ref = torch.einsum("bhp,bpd->bhd", w, v[:, 0])
    assert ((out.float() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -10 * float(v.abs().max())).all()
    order = torch.randperm(n, generator=g).to(torch.int32).cuda()
    cu = torch.arange(n + 1, dtype=torch.int32).cuda()
    assert torch.equal(kv.decode(q, tables, ctx, page, 0.125, seqs=order, cu_q_lens=cu), out)
    assert torch.equal(kv.decode(q, tables, ctx, page, 0.125, cu_q_lens=cu), out)


@pytest.mark.parametrize("bits", [4, 8])
def test_offsets_past_32_bits(bits):
    """Pages that lie more than 2^31 and 2^32 bytes into the pool."""
    PackedKV, ops = kit()
    nh, nkv, d, page = 8, 8, 128, 16
    block = nkv * ops.packed_page_bytes(bits, d, page)
    pages_n = 2 ** 32 // block + 40
    kv = PackedKV.empty(pages_n, nkv, d, page, bits)
    small = PackedKV.empty(8, nkv, d, page, bits)
    n = 100
    high = torch.tensor([pages_n - 1, 2 ** 31 // block + 1, 3, pages_n - 7, 2 ** 32 // block + 1, 2 ** 31 // block, 0], dtype=torch.int32)
    low = torch.tensor([6, 1, 3, 2, 4, 5, 0], dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(n, (nh + 2 * nkv) * d, generator=g).to(BF16).cuda()
    q = torch.randn(1, nh, d, generator=g).to(BF16).cuda()
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    got = []
    for c, table in ((kv, high), (small, low)):
        t = torch.arange(n)
        slots = (table[t // page].long() * page + t % page).to(torch.int32).cuda()
        tables = table.view(1, -1).cuda()
        c.write(rows, dev(list(range(n))), slots, nh, freqs(d).cuda())
        got.append((*c.read(tables, dev([n]), dev([0]), 7), c.decode(q, tables, dev([n]), n, 0.1),
                    c.prefill(rows[:, :nh * d].unflatten(1, (nh, d)), tables, dev([0, n]), dev([n]), [n], [n], 0.1)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_calls_that_are_refused():
    PackedKV, ops = kit()
    pool = Pool([20], 2, 64, 16, 4, seed=0)
    kv, tables, ctx = pool.kv, pool.tables.cuda(), torch.tensor([20], dtype=torch.int32).cuda()
    q = torch.zeros(1, 4, 64, dtype=BF16, device="cuda")
    E = ops.KernelError
    for bad in (dict(tables=tables.cpu()), dict(tables=tables.long()), dict(tables=tables[0]), dict(context_lens=ctx.long()), dict(context_lens=ctx.cpu()),
                dict(q=q.half()), dict(q=q.cpu()), dict(q=torch.zeros(2, 4, 64, dtype=BF16, device="cuda")), dict(window=-1),
                dict(sink=torch.zeros(3, device="cuda")), dict(slopes=torch.zeros(4, device="cuda", dtype=BF16)), dict(out=torch.zeros(1, 4, 64, device="cuda")),
                dict(seqs=torch.zeros(1, device="cuda", dtype=torch.int64)), dict(cu_q_lens=torch.zeros(1, device="cuda", dtype=torch.int32))):
        args = dict(dict(q=q, tables=tables, context_lens=ctx, max_context=20, scale=0.1), **bad)
        with pytest.raises(E):
            kv.decode(**args)
    row = torch.zeros(1, 8 * 64, dtype=BF16, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for a in ((row[:, :100], pos, pos, 4), (row, pos.long(), pos, 4), (row, pos, pos[:0], 4), (row.half(), pos, pos, 4), (row, pos, pos, 3),
              (row, pos, pos, 4, torch.ones(32, device="cuda")), (row, None, pos, 4, torch.ones(32, device="cuda", dtype=F64)),
              (row, pos, pos, 4, torch.ones(33, device="cuda", dtype=F64))):
        with pytest.raises(E):
            kv.write(*a)
    with pytest.raises(E):
        kv.read(tables, ctx, pos, 2, out=(torch.zeros(2, 2, 16, 64, device="cuda"), torch.zeros(2, 2, 16, 64, device="cuda", dtype=BF16)))
    with pytest.raises(E):
        kv.read(tables, ctx.long(), pos, 2)
    two, cu = torch.zeros(2, 4, 64, dtype=BF16, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(q=two.half()), dict(q=two.cpu()), dict(q=torch.zeros(4, 2, 64, dtype=BF16, device="cuda").transpose(0, 1)), dict(tables=tables.cpu()),
                dict(cu_q_lens=cu[:1]), dict(cu_q_lens=cu.long()), dict(context_lens=ctx.cpu()), dict(window=-1), dict(out=torch.zeros(2, 4, 64, device="cuda")),
                dict(out=torch.zeros(3, 4, 64, dtype=BF16, device="cuda")), dict(sink=torch.zeros(4)), dict(sink=torch.zeros(3, device="cuda")),
                dict(q_lens=[2, 2]), dict(contexts=[1]), dict(contexts=[10 ** 6])):
        args = dict(dict(q=two, tables=tables, cu_q_lens=cu, context_lens=ctx, q_lens=[2], contexts=[20], scale=0.1), **bad)
        with pytest.raises(E):
            kv.prefill(**args)
    assert kv.decode(q[:0], tables[:0], ctx[:0], 20, 0.1).shape == (0, 4, 64)
    assert kv.write(row[:0], pos[:0], pos[:0], 4).shape == (0, 4, 64)
    assert kv.prefill(q[:0], tables, torch.zeros(2, dtype=torch.int32, device="cuda"), ctx, [0], [20], 0.1).shape == (0, 4, 64)


@pytest.mark.parametrize("bits", [4, 8])
def test_prefill_in_several_runs(bits, monkeypatch):
    """More tokens than are read back at a time: the same result in runs of sequences."""
    from gollmgo_b200.cache import packed
    nh, nkv, d, page = 8, 2, 64, 16
    q_lens, lens = [5, 0, 33, 16, 2, 70], [5, 9, 90, 16, 65, 140]
    pool = Pool(lens, nkv, d, page, bits, seed=4)
    cu = [0]
    for a in q_lens:
        cu.append(cu[-1] + a)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(cu[-1], nh, d, generator=g).to(BF16).cuda()
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    args = (q, pool.tables.cuda(), dev(cu), dev(lens), q_lens, lens, 0.125)
    want = pool.kv.prefill(*args)
    for most in (1, 100, 200):
        monkeypatch.setattr(packed, "SCRATCH_TOKENS", most)
        got = pool.kv.prefill(*args)
        # (runs of few keys may go to another of the prompt kernels)
        assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    monkeypatch.setattr(packed, "MOST_SEQUENCES", 2)
    assert float((pool.kv.prefill(*args).float() - want.float()).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    mark = torch.full_like(want, 9.0)
    pool.kv.prefill(*args, least=10, out=mark)
    kept = [r for b in (0, 4) for r in range(cu[b], cu[b + 1])]
    assert (mark[kept] == 9.0).all() and (mark != 9.0).any(-1).any(-1).sum() == cu[-1] - len(kept)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("scale", [0.09, -0.05, 0.0])
def test_decode_of_loud_quiet_and_bad_queries(bits, scale):
    """Heads that share a kv head and differ by 2^60, a head with an infinity, one with a NaN, one of zeros: each its own result."""
    nh, nkv, d, n = 6, 1, 128, 70
    pool = Pool([n], nkv, d, 16, bits, seed=1)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(1, nh, d, generator=g)
    q[0, 1] *= 2.0 ** 30 * 1e-10 if scale else 1.0
    q[0, 2] *= 2.0 ** -60
    q[0, 3] = 0
    q[0, 4, 77] = math.inf
    q[0, 5, 3] = math.nan
    q = q.to(BF16)
    out = pool.kv.decode(q.cuda(), pool.tables.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), n, scale).cpu().double()[0]
    ref = plain.attend(q.double(), pool.keys[0], pool.values[0], n, scale)[0]
    assert torch.isnan(out[4:]).all()
    for h in range(4):
        e = errors_of(BF16, q[0, h:h + 1], pool.keys[0], abs(scale))
        assert ((out[h] - ref[h]).abs() <= bound(ref[h], [pool.values[0]], BF16, *e)).all(), h
