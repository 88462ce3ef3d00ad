"""Prompt portions over a packed cache: the runs of sequences that a step is cut into (host), and steps with many decoding
sequences around their portions against the plain 64-bit implementation (device)."""
import pytest
import torch

import plain_packed as plain
from gollmgo_b200.cache import PackedKV


def runs_of(monkeypatch, q_lens, contexts, least=1, window=0, page=16, most=None, tokens=None):
    """The runs of sequences that prefill() of bfloat16 rows is cut into: (lo, hi, pages, longest table, tiles, longest context)."""
    from gollmgo_b200.cache import packed
    for name, value in (("MOST_SEQUENCES", most), ("SCRATCH_TOKENS", tokens)):
        if value is not None:
            monkeypatch.setattr(packed, name, value)

    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, page, 4, 1, 148
            self.runs = []

        def _portions(self, q, out, tables, cu_q_lens, context_lens, lo, hi, pages, most, counts, longest, *more):
            self.runs.append((lo, hi, pages, most, list(counts), longest))
    kv = NoDevice()
    B, rows = len(q_lens), sum(q_lens)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    kv.prefill(torch.zeros(rows, 2, 64, dtype=torch.bfloat16), torch.zeros(B, -(-max(contexts) // page), dtype=torch.int32), cu,
               torch.tensor(contexts, dtype=torch.int32), q_lens, contexts, 1.0, window=window, least=least)
    return kv.runs


@pytest.mark.parametrize("q_lens,least", [([1] * 9 + [40], 2), ([40] + [1] * 9 + [40], 2), ([1] * 9 + [40, 40], 2), ([1] * 3 + [5] * 7 + [1] * 5, 2),
                                          ([5, 1, 1, 6, 1, 7, 1, 1, 1, 1, 8, 1], 2), ([1] * 12, 1), ([0, 0, 0, 0, 0, 3], 1), ([1] * 7, 2), ([70, 1, 70], 2)])
@pytest.mark.parametrize("most", [1, 2, 4, 1024])
@pytest.mark.parametrize("window", [0, 20])
def test_every_portion_lies_in_one_run(monkeypatch, q_lens, least, most, window):
    contexts = [a + 3 * i for i, a in enumerate(q_lens)]
    contexts = [max(1, c) for c in contexts]
    runs = runs_of(monkeypatch, q_lens, contexts, least, window, most=most, tokens=160)
    portions = [b for b, a in enumerate(q_lens) if a >= least and a > 0]
    assert [b for lo, hi, *_ in runs for b in range(lo, hi) if b in portions] == portions
    for lo, hi, pages, longest_table, counts, longest in runs:
        mine = [b for b in portions if lo <= b < hi]
        assert mine and hi - lo <= most
        seen = [-(-contexts[b] // 16) - (max(0, contexts[b] - q_lens[b] - window + 1) // 16 if window else 0) for b in mine]
        assert pages == sum(seen) and (pages * 16 <= 160 or len(mine) == 1)
        assert longest_table == max(-(-contexts[b] // 16) for b in mine) and longest == max(contexts[b] for b in mine)
        assert counts == [sum(-(-q_lens[b] // h) for b in mine) for h in (16, 64, 128)]


def test_runs_of_more_sequences_than_a_launch_takes(monkeypatch):
    """A step of a busy server: more decoding sequences than a launch takes before, between and behind its portions."""
    for q_lens, want in (([1] * 1200 + [40], [(1200, 1201)]), ([40] + [1] * 1200 + [40], [(0, 1), (1201, 1202)]), ([1] * 1200 + [40, 40] + [1] * 1100, [(1200, 1202)]),
                         ([40] + [1] * 1022 + [40, 40], [(0, 1024), (1024, 1025)])):
        runs = runs_of(monkeypatch, q_lens, [a + 9 for a in q_lens], least=2)
        assert [r[:2] for r in runs] == want


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 96])
@pytest.mark.parametrize("counts", [(1200, 0, 0), (3, 1200, 2), (1100, 5, 1100)])
def test_portions_among_many_decoding_sequences(bits, dtype, d, counts):
    """More decoding sequences than a launch takes before, between and behind two portions: those are right, and no other row is touched."""
    nh, nkv, page = 4, 2, 16
    g = torch.Generator().manual_seed(d + bits)
    before, between, behind = counts
    q_lens = [1] * before + [37] + [1] * between + [19] + [1] * behind
    contexts = [3] * before + [90] + [5] * between + [19] + [2] * behind
    B, width = len(q_lens), 6
    at = [before, before + 1 + between]
    kv = PackedKV.empty(64, nkv, d, page, bits)
    kv.pages.copy_(torch.randint(0, 256, kv.pages.shape, dtype=torch.uint8, generator=g))        # what a stray read would find
    kv.pages[..., 2 * page * (d * bits // 8):] = 255                                            # ... and every scale of it a NaN
    tables = torch.full((B, width), 63, dtype=torch.int32)
    order = torch.randperm(63, generator=g).to(torch.int32)
    refs, lo = {}, 0
    for b in at:
        n = -(-contexts[b] // page)
        tables[b, :n] = order[lo:lo + n]
        lo += n
        rows = torch.randn(contexts[b], (nh + 2 * nkv) * d, generator=g).to(dtype)
        t = torch.arange(contexts[b])
        slots = (tables[b][t // page].long() * page + t % page).to(torch.int32)
        kv.write(rows.cuda(), None, slots.cuda(), nh)
        held = [plain.through(x.double().view(-1, nkv, d), bits) for x in rows[:, nh * d:].chunk(2, 1)]
        refs[b] = (rows[-q_lens[b]:, :nh * d].reshape(-1, nh, d), held)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    q = torch.zeros(int(cu[-1]), nh, d, dtype=dtype)
    for b in at:
        q[cu[b]:cu[b + 1]] = refs[b][0]
    out = torch.full(q.shape, 9.0, dtype=dtype, device="cuda")
    kv.prefill(q.cuda(), tables.cuda(), cu.cuda(), torch.tensor(contexts, dtype=torch.int32).cuda(), q_lens, contexts, d ** -0.5, least=2, out=out)
    out = out.cpu().double()
    mark = torch.ones(q.shape[0], dtype=torch.bool)
    for b in at:
        x, (k, v) = refs[b]
        mark[cu[b]:cu[b + 1]] = False
        got = out[cu[b]:cu[b + 1]]
        ref = plain.attend(x.double(), k, v, contexts[b], d ** -0.5)
        assert bool((got != 9.0).any(-1).all())
        assert ((got - ref).abs() <= tolerance(x, k, v, contexts[b], d ** -0.5, dtype, d in (64, 128))).all()
    assert bool((out[mark] == 9.0).all())


def tolerance(q, keys, values, context, scale, dtype, tensor_cores, window=0, softcap=0.0, sink=None, slopes=None, temperature=None):
    """How far a row may be from attend(): S(j) = sum over channels of |q k| scale, P = the weights.  A score that moves by m(j) moves the
    output by sum P m |v - out|.
    float32: products of d terms, d roundings of 2^-24 of S at most, and those of the exponential, of the sum over the context and of the output.
    On the tensor cores a key is not one number there but s (c - M) + (o + M s) with the middle code M, two sums that are made apart and may cancel.
    Of a group whose largest value is G, |o + M s| <= 1.01 G (it lies inside the codes' range, whose end is at most a bfloat16 step of the scale
    beyond the largest value) and |s (c - M)| <= 1.01 x 8 / 15 x 2 G, so roundings are relative to 2.1 G in the place of |k|, and of |v| alike.
    bfloat16 on the tensor cores: a key rounds to half precision as it is read back, so a score moves by 2^-11 S, and a weight and a value round
    once (2^-11 each, relative to sum P |v|).  A weight is held times 2^7 or 2^15 relative to the row's largest, which is 1 at least, and below 2^-14
    as held off by 2^-25 at most: of each key 2^-32 of the largest value.  (Keys and values below 2^-26 of their kv head's largest lose bits too, which tests of that
    allow for.)  A cap is a tanh of the special-function unit there: 2^-11 of the capped score.  The general kernel computes in float32 whatever the type.
    A bias by distance rounds in float32, and the result rounds once."""
    a, nh, d = q.shape
    group = nh // keys.shape[1]
    tol = torch.zeros(a, nh, d, dtype=torch.float64)
    fast = dtype == torch.bfloat16 and tensor_cores
    half = 2.0 ** -11 if fast else 0.0
    at, j = torch.arange(context - a, context)[:, None], torch.arange(context)[None]
    seen = (j <= at) & ((at - j < window) if window else True)
    factor = torch.full((a, 1), float(scale), dtype=torch.float64)
    if temperature:
        factor = factor * (1.0 + temperature[0] * torch.log(torch.floor((at + 1).double() / temperature[1]) + 1.0))
    for h in range(nh):
        k, v, x = keys[:, h // group], values[:, h // group], q[:, h].double()
        size_k, size_v = k.abs(), v.abs()
        if dtype == torch.float32 and tensor_cores:
            size_k, size_v = ((2.1 * y.abs().view(context, d // 64, 64).amax(2, keepdim=True)).expand(-1, -1, 64).reshape(context, d) for y in (k, v))
        z, move = x @ k.T * factor, x.abs() @ size_k.T * factor.abs() * (half + (d + 8) * 2.0 ** -24)
        if softcap > 0:
            z = softcap * torch.tanh(z / softcap)
            move = move + z.abs() * (1.1 * 2.0 ** -11 if fast else 2.0 ** -21)
        if slopes is not None:
            z = z - slopes[h].double() * (at - j)
            move = move + (z.abs() + slopes[h].double() * (at - j).abs()) * 2.0 ** -22
        move = move + (z.abs() + 1.0) * 2.0 ** -22                     # the exponential and its argument
        z = z.masked_fill(~seen, -float("inf"))
        if sink is not None:
            z = torch.cat([z, sink[h].double().expand(a, 1)], 1)
        w = torch.softmax(z, 1)[:, :context]
        out = w @ v
        spread = torch.einsum("ij,ijc->ic", w * move.masked_fill(~seen, 0.0), (v[None] - out[:, None]).abs()) + 2.0 ** -21 * out.abs()
        rounds = (2 * half + (context + 8) * 2.0 ** -24) * (w @ size_v)
        if fast:
            rounds = rounds + context * 2.0 ** -32 * v.abs().max()
        tol[:, h] = 1.05 * (spread + rounds) + torch.finfo(dtype).eps / 2 * out.abs() + 1e-30
    return tol


OPTIONS = [dict(), dict(window=20), dict(softcap=5.0), dict(sink=True), dict(slopes=True, window=33, sink=True, temperature=(0.1, 16)), dict(slopes=True, window=130)]


Q_LENS, LENS = [5, 1, 33, 16, 2, 70, 150], [5, 40, 90, 16, 65, 140, 301]


def pointed_portions(bits, dtype, option, nh, nkv, d, seed):
    """Queries, keys and values as they come, what the cache holds of them, and the options.  Every second row attends to one key nearly alone:
    its own, the first in sight or one between, so that a key that is left out, doubled or taken for another shows."""
    g = torch.Generator().manual_seed(seed)
    o = dict(OPTIONS[option])
    if o.get("sink"):
        o["sink"] = torch.randn(nh, generator=g)
    if o.get("slopes"):
        o["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)])
    cu = torch.tensor([0] + Q_LENS).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), nh, d, generator=g)
    rows, held = [], []
    for b, n in enumerate(LENS):
        rows.append(torch.randn(n, 2 * nkv * d, generator=g).to(dtype))
        held.append([plain.through(y.double().view(n, nkv, d), bits) for y in rows[b].chunk(2, 1)])
        for i in range(0, Q_LENS[b], 2):
            p = n - Q_LENS[b] + i
            lo = max(0, p - o["window"] + 1) if o.get("window") else 0
            to = (p, lo, (p + lo) // 2)[i // 2 % 3]
            q[cu[b] + i] = held[b][0][to].float().repeat_interleave(nh // nkv, 0) * (200.0 / d) ** 0.5
    return q.to(dtype), cu, rows, held, o


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,policy", [(torch.bfloat16, "auto"), (torch.bfloat16, "mma"), (torch.bfloat16, "general"), (torch.float32, "auto")])
@pytest.mark.parametrize("option", range(len(OPTIONS)))
@pytest.mark.parametrize("nh,nkv,d,page", [(4, 1, 64, 16), (4, 2, 128, 16), (3, 3, 128, 32), (4, 2, 128, 8), (2, 1, 64, 128), (2, 1, 64, 4), (2, 1, 128, 256), (4, 2, 96, 16), (3, 1, 16, 4)])
def test_portions_are_as_near_as_their_roundings(monkeypatch, bits, dtype, policy, option, nh, nkv, d, page):
    from gollmgo_b200.cache import packed
    monkeypatch.setattr(packed, "ATTN_POLICY", policy)
    q, cu, rows, held, o = pointed_portions(bits, dtype, option, nh, nkv, d, d + option)
    counts = [-(-n // page) for n in LENS]
    tables = torch.full((len(LENS), max(counts) + 1), -1, dtype=torch.int32)
    order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(d)).to(torch.int32).split(counts)
    kv = PackedKV.empty(sum(counts), nkv, d, page, bits)
    kv.pages.fill_(255)                                                        # (NaN where nothing is written)
    for b, n in enumerate(LENS):
        tables[b, :counts[b]] = order[b]
        t = torch.arange(n)
        kv.write(rows[b].cuda(), None, (tables[b][t // page].long() * page + t % page).to(torch.int32).cuda(), 0)
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    on_device = {k: v.cuda() if torch.is_tensor(v) else v for k, v in o.items()}
    out = kv.prefill(q.cuda(), tables.cuda(), cu.cuda(), dev(LENS), Q_LENS, LENS, d ** -0.5, **on_device).cpu().double()
    for b, n in enumerate(LENS):
        x = q[cu[b]:cu[b + 1]]
        ref = plain.attend(x.double(), *held[b], n, d ** -0.5, **o)
        tol = tolerance(x, *held[b], n, d ** -0.5, dtype, d in (64, 128) and policy != "general", **o)
        assert ((out[cu[b]:cu[b + 1]] - ref).abs() <= tol).all(), (b, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("option", range(len(OPTIONS)))
@pytest.mark.parametrize("mistake", ["zeros", "scale", "last key", "first key", "next head", "window"])
def test_the_tolerance_of_portions_tells_mistakes(dtype, option, mistake):
    """What test_portions_are_as_near_as_their_roundings allows, against attention with a mistake in it: in every portion of some rows it shows."""
    nh, nkv, d = 2, 2, 64
    q, cu, _, held, o = pointed_portions(4, dtype, option, nh, nkv, d, 5)
    if mistake == "window" and not o.get("window"):
        return
    for b, n in enumerate(LENS):
        x, (k, v) = q[cu[b]:cu[b + 1]], held[b]
        if x.shape[0] < 5 or n > 140:
            continue
        ref = plain.attend(x.double(), k, v, n, d ** -0.5, **o)
        tol = tolerance(x, k, v, n, d ** -0.5, dtype, True, **o)
        scale, wrong = d ** -0.5, dict(o)
        if mistake == "scale":
            scale *= 0.7
        if mistake == "window":
            wrong["window"] -= 1
            if n <= o["window"]:
                continue
        if mistake == "next head":
            k, v = k.flip(1), v.flip(1)
        got = plain.attend(x.double(), k, v, n, scale, **wrong)
        if mistake == "zeros":
            got = torch.zeros_like(ref)
        if mistake in ("last key", "first key"):        # of each row: as if it stood at its neighbour's place
            k2, v2 = k.clone(), v.clone()
            i = x.shape[0] - 1 - (x.shape[0] - 1) % 6 if mistake == "last key" else None
            if mistake == "last key":                   # a row that points to its own key sees the one before instead
                at = n - x.shape[0] + i
            else:                                       # the last row but some that points to the first key in sight
                i = max(j for j in range(0, x.shape[0], 2) if j // 2 % 3 == 1)
                at = max(0, n - x.shape[0] + i - o["window"] + 1) if o.get("window") else 0
            k2[at], v2[at] = k[at + (1 if at + 1 < n else -1)], v[at + (1 if at + 1 < n else -1)]
            got = plain.attend(x.double(), k2, v2, n, scale, **o)
        bad = ((got - ref).abs() > tol).any(-1).any(-1)
        assert bad.any(), (b, n)


@pytest.mark.parametrize("rows,q_lens", [(3, [4]), (0, [1]), (9, [5, 5]), (9, [1, 9]), (9, [0, 10, -3])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_of_more_rows_than_q_has_are_refused(rows, q_lens, dtype):
    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 1, 148

        def _portions(self, *a):
            raise AssertionError("rows behind the end of q")
    from gollmgo_b200.csrc import ops
    B = len(q_lens)
    lists = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="rows in q"):
        NoDevice().prefill(torch.zeros(rows, 2, 64, dtype=dtype), torch.zeros(B, 4, dtype=torch.int32), *lists, q_lens, [20] * B, 1.0)


# ---------------------------------------------------------------- which prompt kernel
SHAPES = [([3], [0]), ([40], [0]), ([100], [40]), ([144], [0]), ([145], [0]), ([256], [0]), ([257], [0]), ([64], [193]), ([700], [0]), ([20] * 30, [0] * 30),
          ([100] * 12, [0] * 12), ([200] * 12, [0] * 12), ([30, 90], [3000, 0]), ([2048], [0])]


@pytest.mark.parametrize("nh", [2, 8, 16, 32])
@pytest.mark.parametrize("window", [None, 64, 127, 128, 200, 256, 1000])
@pytest.mark.parametrize("options", [False, True])
def test_the_line_between_the_prompt_kernels_is_the_attention_layers(nh, window, options):
    from types import SimpleNamespace

    from gollmgo_b200.cache import packed
    from gollmgo_b200.parts import BuildContext, PartSpec, build_mixer
    from gollmgo_b200.parts.attention import TILES_TC_X
    spec = PartSpec("attention", dict(hidden_size=64, num_heads=nh, num_kv_heads=nh // 2, head_dim=64, window=window, position=PartSpec("none"), sink=options))
    plain_layer = build_mixer(spec, BuildContext(torch.bfloat16, "cpu", 64, 4, 16))
    for q_lens, q_starts in SHAPES:
        tiles = sum(-(-a // 128) for a in q_lens)
        batch = SimpleNamespace(q_lens=q_lens, q_starts=q_starts, tiles={})
        if options:
            chosen = TILES_TC_X.chosen(range(len(q_lens)), q_lens, q_starts)
            batch.tiles[TILES_TC_X] = SimpleNamespace(count=tiles if chosen else 0, seq=None, q0=None)
            want = bool(plain_layer.long_tiles(batch))
        else:
            want = not plain_layer._few_short_tiles(tiles, batch)
        longest = max(a + s for a, s in zip(q_lens, q_starts))
        assert packed.long_tiles(options, tiles, nh, window or 0, longest, plain_layer.num_sms) == want, (q_lens, q_starts)


@pytest.mark.parametrize("policy,lists", [("auto", [64, 128]), ("mma", [64]), ("general", [16])])
@pytest.mark.parametrize("options", [False, True])
def test_the_switch_of_the_prompt_kernels_holds_for_portions(monkeypatch, policy, lists, options):
    from gollmgo_b200.cache import packed
    from gollmgo_b200.csrc import ops
    seen = {}
    monkeypatch.setattr(packed, "ATTN_POLICY", policy)
    monkeypatch.setattr(ops, "packed_prefill_rows", lambda *a: None)
    monkeypatch.setattr(ops, "packed_unfold", lambda *a: seen.update(lists=[h for h, *_ in a[8]]))
    monkeypatch.setattr(ops, "attn_prefill_half", lambda *a: seen.update(kernel="options" if a[17] else "plain", tile128=a[9]))
    monkeypatch.setattr(ops, "packed_prefill", lambda *a, **k: seen.update(kernel="general"))

    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 1, 148
            self.pages = None
    NoDevice().prefill(torch.zeros(400, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 25, dtype=torch.int32), torch.tensor([0, 400], dtype=torch.int32),
                       torch.tensor([400], dtype=torch.int32), [400], [400], 0.1, sink=torch.zeros(2) if options else None)
    assert seen["lists"] == lists and seen["kernel"] == ("general" if policy == "general" else "options" if options else "plain")
    assert (seen.get("tile128") is not None) == (128 in lists)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 1, 128), (3, 3, 128), (2, 1, 96)])
def test_portions_with_a_scale_that_is_not_positive(bits, dtype, scale, nh, nkv, d):
    q_lens, lens, page = [5, 40, 290], [5, 90, 300], 16
    g = torch.Generator().manual_seed(d)
    counts = [-(-n // page) for n in lens]
    tables = torch.zeros(len(lens), max(counts), dtype=torch.int32)
    for b, order in enumerate(torch.randperm(sum(counts), generator=g).to(torch.int32).split(counts)):
        tables[b, :counts[b]] = order
    kv = PackedKV.empty(sum(counts), nkv, d, page, bits)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), nh, d, generator=g).to(dtype)
    held = []
    for b, n in enumerate(lens):
        x = torch.randn(n, 2 * nkv * d, generator=g).to(dtype)
        t = torch.arange(n)
        kv.write(x.cuda(), None, (tables[b][t // page].long() * page + t % page).to(torch.int32).cuda(), 0)
        held.append([plain.through(y.double().view(n, nkv, d), bits) for y in x.chunk(2, 1)])
    out = kv.prefill(q.cuda(), tables.cuda(), cu.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q_lens, lens, scale).cpu().double()
    for b, n in enumerate(lens):
        x = q[cu[b]:cu[b + 1]]
        ref = plain.attend(x.double(), *held[b], n, scale)
        assert ((out[cu[b]:cu[b + 1]] - ref).abs() <= tolerance(x, *held[b], n, scale, dtype, d in (64, 128))).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,page", [(96, 16), (128, 8), (16, 4)])
@pytest.mark.parametrize("sink", [False, True])
def test_portions_on_the_general_kernel_do_not_attend_to_missing_pages(monkeypatch, bits, dtype, d, page, sink):
    from gollmgo_b200.cache import packed
    monkeypatch.setattr(packed, "ATTN_POLICY", "general")
    nh, nkv, n, a = 2, 1, 70, 30
    if dtype == torch.float32 and d == 128 and page >= 16:
        return
    g = torch.Generator().manual_seed(d)
    width = -(-n // page)
    kv = PackedKV.empty(width, nkv, d, page, bits)
    table = torch.randperm(width, generator=g).to(torch.int32)
    x = torch.randn(n, 2 * nkv * d, generator=g).to(dtype)
    t = torch.arange(n)
    kv.write(x.cuda(), None, (table[t // page].long() * page + t % page).to(torch.int32).cuda(), 0)
    k, v = (plain.through(y.double().view(n, nkv, d), bits) for y in x.chunk(2, 1))
    missing = table.clone()
    missing[0], missing[-1] = -1, width
    there = ((missing >= 0) & (missing < width))[t // page]
    q = torch.randn(a, nh, d, generator=g).to(dtype)
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    s = torch.randn(nh, generator=g) if sink else None
    for gone in (False, True):
        if gone:
            missing[:] = -1
        out = kv.prefill(q.cuda(), missing.view(1, -1).cuda(), dev([0, a]), dev([n]), [a], [n], d ** -0.5, sink=None if s is None else s.cuda()).cpu().double()
        if gone:
            assert (out == 0).all()
            continue
        for i in range(a):
            seen = there & (t <= n - a + i)
            for h in range(nh):
                z = k[seen, 0] @ q[i, h].double() * d ** -0.5
                z = torch.cat([z, s[h].double()[None]]) if sink else z
                w = torch.softmax(z, 0)[:int(seen.sum())]
                # float32 arithmetic: d products a score (relative to |q| |k|), twice, and a sum over the context; the result's rounding
                e = float(q[i, h].double().norm() * k.norm(dim=-1).max()) * d ** -0.5 * (d + 8) * 2.0 ** -24 + 2.0 ** -20
                ref = w @ v[seen, 0]
                assert ((out[i, h] - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (2 * e + (n + 8) * 2.0 ** -24) * (w @ v[seen, 0].abs()).max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 96, 16), (torch.float32, 96, 16), (torch.float32, 128, 8), (torch.float32, 64, 16)])
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_tokens_reach_the_rows_that_see_them(bits, dtype, d, page, window, bad, whole=False):
    """A bad key makes the rows of its kv head from its token on NaN, a bad value its group of channels (``whole``: all of them); rows before it,
    and behind the window, are as without it."""
    nh, nkv, n = 4, 2, 200
    g = torch.Generator().manual_seed(d)
    x = torch.randn(n, (nh + 2 * nkv) * d, generator=g).to(dtype)
    width = -(-n // page)
    table = torch.randperm(width, generator=g).to(torch.int32)
    t = torch.arange(n)
    slots = (table[t // page].long() * page + t % page).to(torch.int32).cuda()
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    outs = []
    key, value = 150, 37
    for spoilt in (False, True):
        y = x.clone()
        if spoilt:
            y[key, nh * d + 3] = bad                              # a key of kv head 0
            y[value, (nh + 2 * nkv) * d - 1] = -bad               # the last channel of a value of kv head 1
        kv = PackedKV.empty(width, nkv, d, page, bits)
        q = kv.write(y.cuda(), None, slots, nh)
        outs.append(kv.prefill(q, table.view(1, -1).cuda(), dev([0, n]), dev([n]), [n], [n], d ** -0.5, window=window).cpu())
    good, got = outs
    sees = lambda at: (t >= at) & (t < at + window if window else True)  # noqa: E731
    group = plain.group_of(d)
    hidden = torch.zeros(n, nh, d, dtype=torch.bool)
    hidden[sees(key), :2] = True
    hidden[sees(value), 2:, 0 if whole else d - group:] = True
    assert torch.equal(got.isnan(), hidden)
    assert torch.equal(got[~hidden], good[~hidden])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("policy", ["auto", "mma"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 32)])
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_tokens_of_bfloat16_portions(monkeypatch, bits, policy, d, page, window, bad):
    from gollmgo_b200.cache import packed
    monkeypatch.setattr(packed, "ATTN_POLICY", policy)
    monkeypatch.setattr(packed, "SHORT_PROMPT_KEYS", 100)            # (200 keys: on tcgen05 where it may)
    test_bad_tokens_reach_the_rows_that_see_them(bits, torch.bfloat16, d, page, window, bad, whole=True)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("policy", ["auto", "mma", "general"])
@pytest.mark.parametrize("options", [False, True])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (2, 2, 128)])
@pytest.mark.parametrize("key,value", [(0, 0), (40, 100), (-40, -100), (100, 60), (-100, 126)])
def test_portions_of_loud_and_quiet_heads(monkeypatch, bits, policy, options, nh, nkv, d, key, value):
    """Keys of one kv head times 2^key, its queries times 2^-key, values times 2^value; the other kv head's the other way round; rows of q that differ
    by 2^20 beside one another, and a value 2^20 times the others that hardly any row attends to."""
    from gollmgo_b200.cache import packed
    if policy == "general" and value == 126:
        return      # its float32 sums are divided at the end: 300 weights of 1 and values of 2^126 make 2^134, a float ends at 2^128
    monkeypatch.setattr(packed, "ATTN_POLICY", policy)
    page, q_lens, lens = 16, [40, 290], [90, 300]
    g = torch.Generator().manual_seed(d + key)
    counts = [-(-n // page) for n in lens]
    tables = torch.zeros(len(lens), max(counts), dtype=torch.int32)
    for b, order in enumerate(torch.randperm(sum(counts), generator=g).to(torch.int32).split(counts)):
        tables[b, :counts[b]] = order
    kv = PackedKV.empty(sum(counts), nkv, d, page, bits)
    kv.pages.fill_(255)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    sign = torch.tensor([1.0, -1.0])
    up_k, up_v = 2.0 ** (key * sign)[:, None], 2.0 ** (value * sign)[:, None]
    q = torch.randn(int(cu[-1]), nkv, nh // nkv, d, generator=g)
    q[1::2] *= 2.0 ** -20
    q = (q / up_k[:, None]).view(-1, nh, d).to(torch.bfloat16)
    held = []
    for b, n in enumerate(lens):
        x = torch.randn(n, 2, nkv, d, generator=g)
        x[:, 0, :, 0] = 0.0
        x[7, 1] *= 2.0 ** 20 if value < 100 else 1.0
        x[7, 0, :, 0] = -400.0                                   # (no row attends to it but those whose first channel says so)
        x[:, 0] *= up_k
        x[:, 1] *= up_v
        x = x.flatten(1).to(torch.bfloat16)
        t = torch.arange(n)
        kv.write(x.cuda(), None, (tables[b][t // page].long() * page + t % page).to(torch.int32).cuda(), 0)
        held.append([plain.through(y.double().view(n, nkv, d), bits) for y in x.chunk(2, 1)])
    q.view(-1, nh, d)[..., 0] = q[..., 0].abs()
    o = dict(sink=torch.zeros(nh), window=280) if options else {}
    out = kv.prefill(q.cuda(), tables.cuda(), cu.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q_lens, lens, d ** -0.5,
                     **{k: v.cuda() if torch.is_tensor(v) else v for k, v in o.items()}).cpu().double()
    for b, n in enumerate(lens):
        x, (k, v) = q[cu[b]:cu[b + 1]], held[b]
        ref = plain.attend(x.double(), k, v, n, d ** -0.5, **o)
        for h in range(nh):
            one = h * nkv // nh
            # (keys and values below 2^-26 of their kv head's largest are off by 2^-37 of it)
            there = v[:, one:one + 1].nan_to_num()                   # (rows that are kept see none of the others)
            more = dict(o, sink=o["sink"][h:h + 1]) if options else {}
            tol = tolerance(x[:, h:h + 1], k[:, one:one + 1], there, n, d ** -0.5, torch.bfloat16, policy != "general", **more)
            got, gone = out[cu[b]:cu[b + 1], h], ref[:, h].isnan()       # (2^126 times what is above 4 is an infinity: rows that see it are NaN)
            assert got[gone].isnan().all()
            tol = tol[:, 0] + 2.0 ** -36 * there.abs().max()
            kept = ~gone.any(-1)
            assert kept.any() or value == 126
            assert ((got[kept] - ref[kept, h]).abs() <= tol[kept]).all(), (b, h)


def test_the_launchers_of_portions_refuse_sizes_and_missing_lists():
    from gollmgo_b200.csrc import ops
    ops.lib()

    def refused(name, args, cases):
        f = ops._packed(name)
        for at, v, message in cases:
            bad = list(args)
            bad[at] = v
            assert f(*bad) != 0
            assert message in ops.lib().gg_last_error().decode(), (name, at, v)
    one = 16                                          # (any address that is not looked at)
    refused("gg_packed_unfold", [None, 4, one, 8, one, one, 2, one, one, 3, 2, one, one, 64, 1, one, one, 0, 0, None, None, 1, 2, 64, 16, 4, 0, None],
            [(6, 0, "bad sizes"), (6, 1025, "bad sizes"), (10, 9, "bad sizes"), (26, -1, "bad sizes"), (7, 8, "16 bytes"), (0, 8, "16 bytes"), (8, None, "missing"),
             (11, None, "missing"), (12, None, "missing"), (7, None, "missing"), (22, 1025, "missing"), (23, 96, "missing"), (25, 5, "packed cache")])
    refused("gg_packed_prefill", [one, 128, 1, None, 4, one, 8, one, one, one, one, 1, one, 4, 2, 64, 16, 4, 0, 1.0, 0.0, None, None, 0.0, 0.0, None],
            [(2, 7, "dtype"), (13, 3, "multiple"), (14, 0, "bad sizes"), (11, -1, "bad lists"), (9, None, "bad lists"), (7, None, "bad lists"), (18, -1, "window"),
             (17, 3, "packed cache")])
    refused("gg_attn_prefill_half", [one, 256, one, one, one, one, 8, one, one, one, one, 1, None, None, 0, one, 3, 4, 4, 2, 64, 16, 0, 0, 1.0, 0.0, None, None, 0.0, 0.0,
                                     None, None],
            [(20, 96, "head size"), (21, 24, "pages"), (4, None, "no lists"), (9, None, "no lists"), (0, 8, "aligned"), (1, 100, "aligned"), (15, 18, "aligned"), (24, -1.0, "options"),
             (25, 3.0, "options"), (26, one, "options"), (27, one, "options"), (29, 2.0, "options"), (18, 3, "multiple")])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 96])
def test_portions_on_two_streams_and_in_two_graphs(bits, d):
    """Two prefills at once, eager and captured, behind writes of their own: each as alone, also with other keys in the pages at a replay."""
    nh, nkv, page, lens = 4, 2, 16, [300, 70]
    g = torch.Generator().manual_seed(d)
    counts = [-(-n // page) for n in lens]
    table = torch.zeros(2, max(counts), dtype=torch.int32)
    for b, order in enumerate(torch.randperm(sum(counts), generator=g).to(torch.int32).split(counts)):
        table[b, :counts[b]] = order
    rows = [torch.randn(sum(lens), (nh + 2 * nkv) * d, generator=g).to(torch.bfloat16).cuda() for _ in range(3)]
    slots = torch.cat([table[b][torch.arange(n) // page].long() * page + torch.arange(n) % page for b, n in enumerate(lens)]).to(torch.int32).cuda()
    cu, ctx, table = torch.tensor([0, 300, 370], dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda()

    def step(kv, x):
        q = kv.write(x, None, slots, nh)
        return kv.prefill(q, table, cu, ctx, lens, lens, d ** -0.5)
    caches = [PackedKV.empty(sum(counts), nkv, d, page, bits) for _ in range(2)]
    want = [step(caches[0], x).clone() for x in rows]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, kv, x in zip(streams, caches, rows):
            with torch.cuda.stream(s):
                got.append(step(kv, x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    live, graphs, outs = [rows[0].clone(), rows[1].clone()], [], []
    for kv, x in zip(caches, live):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(kv, x))
        graphs.append(graph)
    for a, b in ((0, 1), (2, 0), (1, 2)):
        live[0].copy_(rows[a])
        live[1].copy_(rows[b])
        torch.cuda.synchronize()
        for _ in range(4):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b])


def test_a_result_that_starts_anywhere_takes_the_kernel_that_stores_it(monkeypatch):
    """The tensor-core kernels store 4 and 16 bytes at a time."""
    from gollmgo_b200.csrc import ops
    seen = []
    monkeypatch.setattr(ops, "packed_prefill_rows", lambda *a: None)
    monkeypatch.setattr(ops, "packed_unfold", lambda *a: None)
    monkeypatch.setattr(ops, "attn_prefill_half", lambda *a: seen.append("half"))
    monkeypatch.setattr(ops, "packed_prefill", lambda *a, **k: seen.append("general"))

    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 1, 148
            self.pages = None
    room = torch.zeros(40 * 2 * 64 + 16, dtype=torch.bfloat16)
    first = -room.data_ptr() % 16 // 2
    for at, want in ((0, "half"), (1, "general"), (2, "general"), (4, "general"), (8, "half")):
        out = room[first + at:first + at + 40 * 2 * 64].view(40, 2, 64)
        NoDevice().prefill(torch.zeros(40, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.tensor([0, 40], dtype=torch.int32),
                           torch.tensor([40], dtype=torch.int32), [40], [40], 0.1, out=out)
        assert seen.pop() == want, at


@pytest.mark.gpu
@pytest.mark.parametrize("at", [1, 2, 4, 8])
@pytest.mark.parametrize("nh,nkv", [(4, 2), (3, 3)])
def test_results_that_start_anywhere(at, nh, nkv):
    d, n, page = 64, 300, 16
    g = torch.Generator().manual_seed(at)
    kv = PackedKV.empty(20, nkv, d, page, 4)
    x = torch.randn(n, (nh + 2 * nkv) * d, generator=g).to(torch.bfloat16)
    q = kv.write(x.cuda(), None, torch.arange(n, dtype=torch.int32).cuda(), nh)
    table = torch.arange(20, dtype=torch.int32).view(1, -1).cuda()
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    room = torch.full((n * nh * d + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[at:at + n * nh * d].view(n, nh, d)
    kv.prefill(q, table, dev([0, n]), dev([n]), [n], [n], 0.125, out=out)
    held = [plain.through(y.double().view(n, nkv, d), 4) for y in x[:, nh * d:].chunk(2, 1)]
    rows = x[:, :nh * d].view(n, nh, d)
    ref = plain.attend(rows.double(), *held, n, 0.125)
    assert ((out.cpu().double() - ref).abs() <= tolerance(rows, *held, n, 0.125, torch.bfloat16, True)).all()
    assert (room[:at] == 7.0).all() and (room[at + n * nh * d:] == 7.0).all()
