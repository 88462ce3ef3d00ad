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


def tolerance(q, keys, values, context, scale, dtype, tensor_cores):
    """How far a row may be from attend(): S(j) = sum over channels of |q k| scale, P = the weights.
    float32: products of d terms, d roundings of 2^-24 of S at most, and those of the exponential, of the sum over the context and of the output.
    bfloat16: a key rounds as it is read back, so a score moves by 2^-8 S (and weights move by
    as much relative to themselves), a weight and a value round once (2^-8 each, relative to sum P |v|), and the result rounds once.  On the
    general kernel weights stay float32."""
    a, nh, d = q.shape
    group = nh // keys.shape[1]
    tol = torch.zeros(a, nh, d, dtype=torch.float64)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for i in range(a):
        p = context - a + i
        for h in range(nh):
            k, v = keys[:p + 1, h // group], values[:p + 1, h // group]
            z = k @ q[i, h].double() * scale
            size = (k.abs() @ q[i, h].double().abs()) * abs(scale)
            w = torch.softmax(z, 0)
            move = size * (half + (d + 4) * 2.0 ** -24)                # of each score
            mean = (w @ v).abs()
            # d out = sum_j P_j dz_j (v_j - out): each term apart
            spread = (w * move) @ (v - (w @ v)).abs()
            rounds = (half * (2 if tensor_cores else 1) + (p + 8) * 2.0 ** -24) * (w @ v.abs())
            tol[i, h] = 1.05 * (spread + rounds) + torch.finfo(dtype).eps / 2 * mean + 1e-30
    return tol


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


@pytest.mark.parametrize("policy,lists,mma", [("auto", [64, 128], True), ("mma", [64], True), ("general", [16], False)])
@pytest.mark.parametrize("options", [False, True])
def test_the_switch_of_the_prompt_kernels_holds_for_portions(monkeypatch, policy, lists, mma, options):
    from gollmgo_b200.cache import packed
    from gollmgo_b200.csrc import ops
    seen = {}
    monkeypatch.setattr(packed, "ATTN_POLICY", policy)
    monkeypatch.setattr(ops, "packed_prefill_rows", lambda *a: None)
    monkeypatch.setattr(ops, "packed_unfold", lambda *a, **k: seen.update(lists=[h for h, *_ in a[8]]))
    monkeypatch.setattr(ops, "attn_prefill", lambda *a, **k: seen.update(kernel=False, **k))
    monkeypatch.setattr(ops, "attn_prefill_x", lambda *a, **k: seen.update(kernel=True, **k))

    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 1, 148
            self.pages = None
    NoDevice().prefill(torch.zeros(400, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 25, dtype=torch.int32), torch.tensor([0, 400], dtype=torch.int32),
                       torch.tensor([400], dtype=torch.int32), [400], [400], 0.1, sink=torch.zeros(2) if options else None)
    assert seen["lists"] == lists and seen["kernel"] == options and seen["allow_mma"] == mma and ("tile128_seq" in seen) == (128 in lists)
