"""Captured decode steps over a packed cache: a step is replayed for every context of its tag, so its launches have to be those that the
context at hand wants."""
import pytest
import torch

from gollmgo_b200.csrc import ops
from gollmgo_b200.parts import BuildContext, PartSpec, StepFacts, build_mixer
from gollmgo_b200.parts.attention import TILE_KEYS, context_tiles

CONTEXTS = [1, 60, 64, 65, 100, 200, 512, 900, 1024, 1100, 2000, 2048, 3000, 4096, 7000, 8192, 16384, 20000, 32768, 65536, 131072]


def layer(nh, nkv, d, page, bits, dtype=torch.bfloat16, window=None):
    spec = PartSpec("attention", dict(hidden_size=64, num_heads=nh, num_kv_heads=nkv, head_dim=d, window=window, position=PartSpec("none")))
    return build_mixer(spec, BuildContext(dtype, "cpu", 64, 64, page, cache_bits=bits))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,d", [(1, 1, 64), (32, 8, 128), (16, 16, 64), (40, 40, 128), (32, 32, 128), (64, 2, 128)])
@pytest.mark.parametrize("window", [None, 1000])
def test_a_captured_step_has_the_blocks_of_every_context_of_its_tag(bits, dtype, nh, nkv, d, window):
    mixer = layer(nh, nkv, d, 16, bits, dtype, window)
    for n in (1, 2, 4, 8, 16, 24, 32, 64):
        first = {}
        for c in CONTEXTS:
            first.setdefault(mixer.step_tags(StepFacts(n, n, True, c)), c)
        assert len(first) <= 11
        # (scratch is so many floats a block; a step is spread for the context that decode() is given)
        size = {c: ops.packed_decode_scratch(dtype, n, nh, nkv, d, bits, context_tiles(c) * TILE_KEYS, window or 0) for c in CONTEXTS}
        for c in CONTEXTS:
            assert size[first[mixer.step_tags(StepFacts(n, n, True, c))]] == size[c], (n, c)


@pytest.mark.parametrize("n,nkv,d,page", [(1, 2, 96, 16), (4, 1, 128, 8), (30, 8, 256, 16)])
def test_steps_on_the_general_kernel_have_the_slices_of_every_context_of_their_tag(n, nkv, d, page):
    from gollmgo_b200.cache import PackedKV
    mixer = layer(2 * nkv, nkv, d, page, 4)
    first = {}
    for c in CONTEXTS:
        first.setdefault(mixer.step_tags(StepFacts(n, n, True, c)), c)
    longest = max(CONTEXTS)
    found = first[mixer.step_tags(StepFacts(n, n, True, longest))]
    assert PackedKV._splits(n, nkv, context_tiles(found) * TILE_KEYS, 0) == PackedKV._splits(n, nkv, longest, 0)


@pytest.mark.parametrize("given", [True, False])
def test_a_list_made_by_the_call_itself_is_not_read_early(monkeypatch, given):
    """Rows through cu_q_lens, more tokens than a launch takes: without seqs the call makes that list on the stream, so the launches wait for it."""
    from gollmgo_b200.cache import PackedKV

    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 1, 148
            self.pages = None
    seen = []
    monkeypatch.setattr(ops, "packed_decode_mma", lambda q, pages, tables, cu, ctx, seqs, n, *more: seen.append((seqs.tolist(), more[-1])))
    n = ops.PACKED_DECODE_TOKENS + 3
    lists = torch.arange(n + 1, dtype=torch.int32)
    NoDevice().decode(torch.zeros(n, 2, 64, dtype=torch.bfloat16), torch.zeros(n, 4, dtype=torch.int32), lists[:n], 40, 0.1, cu_q_lens=lists,
                      seqs=lists[:n] if given else None, early=True)
    assert [b for part, _ in seen for b in part] == list(range(n))
    assert [early for _, early in seen] == [given, given]


def test_more_than_eight_heads_of_a_kv_head_are_a_shape_of_their_own():
    """Sixteen columns at a time from so many keys on: steps of either side have tags of their own, and scratch for what they run."""
    mixer = layer(32, 2, 128, 16, 4)
    below, above = (StepFacts(64, 64, True, c) for c in (4096, 8192))            # 64 x 2 x 4096 keys, and twice as many
    assert mixer.step_tags(below) != mixer.step_tags(above)
    few, many = (ops.packed_decode_scratch(torch.bfloat16, 64, 32, 2, 128, 4, c, 0) for c in (4096, 8192))
    assert few == 148 * (18 * (8 * 128 + 16) + 4) and many == 148 * (10 * (16 * 128 + 32) + 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nh,nkv", [(9, 1), (16, 1), (24, 1), (33, 1), (66, 2)])
@pytest.mark.parametrize("d,option", [(64, 0), (128, 0), (128, 1)])
def test_many_heads_of_a_kv_head_in_either_shape(bits, nh, nkv, d, option):
    import plain_packed as plain
    from gollmgo_b200.cache import PackedKV
    lens, page = [33, 5, 260, 700], 16
    g = torch.Generator().manual_seed(nh)
    counts = [-(-n // page) for n in lens]
    kv = PackedKV.empty(sum(counts), nkv, d, page, bits)
    tables = torch.zeros(4, max(counts), dtype=torch.int32)
    held = []
    for b, order in enumerate(torch.randperm(sum(counts), generator=g).to(torch.int32).split(counts)):
        tables[b, :counts[b]] = order
        x = torch.randn(lens[b], 2 * nkv * d, generator=g).to(torch.bfloat16)
        t = torch.arange(lens[b])
        kv.write(x.cuda(), None, (order[t // page].long() * page + t % page).to(torch.int32).cuda(), 0)
        held.append([plain.through(y.double().view(lens[b], nkv, d), bits) for y in x.chunk(2, 1)])
    q = torch.randn(4, nh, d, generator=g).to(torch.bfloat16)
    o = dict(sink=torch.randn(nh, generator=g), slopes=torch.rand(nh, generator=g) * 0.1, window=300) if option else {}
    more = {k: v.cuda() if torch.is_tensor(v) else v for k, v in o.items()}
    for said in (700, 10 ** 6):                      # (the work is spread for so long contexts; a window is counted instead)
        out = kv.decode(q.cuda(), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), said, d ** -0.5, **more).cpu().double()
        for b, n in enumerate(lens):
            k, v = held[b]
            ref = plain.attend(q[b:b + 1].double(), k, v, n, d ** -0.5, **o)[0]
            # scores: |q| |k| scale in steps of 2^-20 at most where a tensor core truncates, twice, and a bias of up to 30; weights as halves; the result's rounding
            e = float(q[b].double().norm(dim=-1).max() * k.norm(dim=-1).max()) * d ** -0.5 * 2.0 ** -20 + 2.0 ** -18
            assert ((out[b] - ref).abs() <= 2.0 ** -8 * ref.abs() + (2 * e + 2.0 ** -11) * float(v.abs().max())).all(), (said, b)
