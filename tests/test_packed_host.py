"""The packed cache without a device: sizes, refusals, the cache manager's accounting, options."""
import pytest
import torch

import plain_packed as plain
from gollmgo_b200.cache import CacheManager, FixedStateNeed, PackedKV, PagedKVNeed
from gollmgo_b200.config import EngineConfig
from gollmgo_b200.csrc import ops
from gollmgo_b200.parts import BuildContext, PartSpec, build_mixer


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [4, 16, 64])
def test_page_bytes(bits, d, page):
    assert ops.packed_page_bytes(bits, d, page) == plain.page_bytes(bits, d, page)
    assert ops.packed_group(d) == plain.group_of(d)
    assert ops.packed_page_bytes(bits, d, page) % 16 == 0        # bulk copies start and end on 16 bytes


@pytest.mark.parametrize("bits,d,page", [(2, 64, 16), (16, 64, 16), (4, 8, 16), (4, 72, 16), (8, 272, 16), (4, 0, 16), (4, 64, 2), (4, 64, 24), (8, 64, 512)])
def test_sizes_that_are_refused(bits, d, page):
    with pytest.raises(ops.KernelError, match="packed cache"):
        ops.packed_page_bytes(bits, d, page)


def test_pages_that_are_refused():
    size = ops.packed_page_bytes(4, 64, 16)
    for pages in (torch.zeros(3, 2, size, dtype=torch.uint8),                  # not on a device
                  torch.zeros(3, 2, size + 16, dtype=torch.uint8), torch.zeros(3, 2 * size, dtype=torch.uint8),
                  torch.zeros(3, 2, size, dtype=torch.int8)):
        with pytest.raises(ops.KernelError, match="packed pages"):
            PackedKV(pages, 64, 16, 4)


def test_the_launchers_refuse_sizes_and_missing_lists():
    """The library's own checks, which come before anything touches a device."""
    ops.lib()
    f = ops._packed("gg_packed_write")
    base = [None, 64, 1, None, None, None, 1.0, None, 4, None, 0, 2, 0, 1, 64, 0, 16, 4, 0, 0, None]

    def refused(message, **at):
        args = list(base)
        for k, v in at.items():
            args[int(k[1:])] = v
        assert f(*args) != 0
        assert message in ops.lib().gg_last_error().decode()
    refused("packed cache", _17=3)
    refused("packed cache", _14=24)
    refused("packed cache", _16=12)
    refused("16 bytes", _7=8)
    refused("rotary width", _15=66)
    refused("rotary width", _15=3)
    refused("without frequencies", _15=64)
    refused("bad sizes", _11=-1)
    refused("bad sizes", _13=0)
    g = ops._packed("gg_packed_decode_mma")
    args = [None, 64, 1, None, 4, None, 8, 4, None, None, None, 1, 64, None, 0, None, 8, 2, 64, 16, 4, 0, 1.0, 0.0, None, None, 0.0, 0.0, 0, None]
    for at, v, message in ((18, 96, "not taken"), (19, 8, "not taken"), (20, 5, "not taken"), (16, 7, "multiple"), (11, 2000, "too many"),
                           (21, -1, "bad sizes"), (7, 0, "sequences"), (6, 2 ** 29, "too large"), (1, 4, "16 bytes"), (0, 8, "16 bytes"), (0, None, "scratch"),
                           (2, 7, "not taken"), (11, -1, "bad sizes"), (12, -1, "too many")):
        bad = list(args)
        bad[at] = v
        assert g(*bad) != 0
        assert message in ops.lib().gg_last_error().decode(), (at, v)
    p = ops._packed("gg_packed_prompt_f32")
    args = [None, 64, None, 4, None, 8, 4, 16, None, 1, 5, 16, 64, None, 0, None, 8, 2, 64, 16, 4, 0, 1.0, 0.0, None, None, 0.0, 0.0, None]
    for at, v, message in ((18, 96, "not taken"), (19, 8, "not taken"), (20, 5, "not taken"), (16, 7, "multiple"), (10, -1, "bad sizes"), (6, -1, "bad sizes"),
                           (21, -1, "bad sizes"), (1, 2, "16 bytes"), (0, 4, "16 bytes"), (15, 8, "16 bytes"), (7, None, "lists"), (11, None, "lists"),
                           (12, -1, "lists"), (5, 2 ** 29, "too large"), (0, None, "scratch")):
        bad = list(args)
        bad[at] = v
        assert p(*bad) != 0
        assert message in ops.lib().gg_last_error().decode(), (at, v)
    assert [ops.packed_prompt_fold(h, 1) for h in (1, 2, 3, 4, 5, 8, 16)] == [8, 4, 2, 2, 1, 1, 1]


def test_rows_and_lists_that_are_refused():
    x = torch.zeros(6, 256)
    assert ops._rows_of(x, 256, "x") == 256
    assert ops._rows_of(x[:, :128], 128, "x") == 256
    assert ops._rows_of(x[:, :128].unflatten(1, (2, 64)), 128, "x") == 256
    for bad in (x[:, :100], x.T, x.unflatten(1, (4, 64)).transpose(1, 2), x[:, ::2], x[:, :128].unflatten(1, (2, 64)).expand(6, 2, 64).transpose(0, 1),
                x[:1, :128].expand(6, 128)):
        with pytest.raises(ops.KernelError, match="rows of"):
            ops._rows_of(bad, 128, "x")
    ops._ints("x", 3, torch.zeros(3, dtype=torch.int32), None)
    for bad in (torch.zeros(3), torch.zeros(2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2], torch.zeros(3, dtype=torch.int64)):
        with pytest.raises(ops.KernelError, match="index lists"):
            ops._ints("x", 3, bad)
    for bad in (torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2), torch.zeros(2, 4, dtype=torch.int32)[:, :2]):
        with pytest.raises(ops.KernelError, match="block tables"):
            ops._tables("x", bad)


# ---------------------------------------------------------------- the cache manager and the options
def test_manager_holds_packed_groups_beside_others():
    needs = [PagedKVNeed(2, 64, None, bits=4), PagedKVNeed(2, 64, None), PagedKVNeed(2, 64, None, bits=4), FixedStateNeed((3,)),
             (PagedKVNeed(1, 128, 20, bits=8), None)]
    cm = CacheManager(needs, 16, 6, 4, dtype=torch.bfloat16, device="cpu")
    assert [len(g.cache_ids) for g in cm.groups] == [2, 1, 1]
    assert cm.groups[0].kv.shape == (2, 6, 2, plain.page_bytes(4, 64, 16)) and cm.groups[0].kv.dtype == torch.uint8
    assert cm.groups[1].kv.shape == (1, 2, 6, 2, 16, 64)
    assert cm.groups[2].kv.shape == (1, 6, 1, plain.page_bytes(8, 128, 16))
    want = 2 * 2 * plain.page_bytes(4, 64, 16) + 2 * 2 * 64 * 16 * 2 + plain.page_bytes(8, 128, 16)
    assert CacheManager.bytes_per_page(needs, 16, 2) == want
    cm.poison_freed = True
    cm.admit("a")
    cm.append("a", 40)
    page = cm.block_table("a", 0)[0]
    cm.free("a")
    cm.audit()
    assert (cm.groups[0].kv[:, page] == 255).all()
    pairs = cm.groups[0].kv[0, page, 0, -4:].view(torch.bfloat16)
    assert torch.isnan(pairs).all()


def test_a_packed_page_is_a_fraction_of_a_plain_one():
    plain_page = CacheManager.bytes_per_page([PagedKVNeed(8, 128, None)], 16, 2)
    assert plain_page / CacheManager.bytes_per_page([PagedKVNeed(8, 128, None, bits=4)], 16, 2) == 65536 / 18432
    assert plain_page / CacheManager.bytes_per_page([PagedKVNeed(8, 128, None, bits=8)], 16, 2) == 65536 / 34816


def test_scratch_is_bounded_by_the_longest_sequence_or_the_run():
    need = PagedKVNeed(8, 128, None, bits=4)
    assert PackedKV.scratch_bytes([need, None, (need, FixedStateNeed((2,)))], 100, torch.bfloat16) == 65536 * 8 * 128 * 2 * 2
    assert PackedKV.scratch_bytes([need], 131072, torch.float32) == 131072 * 8 * 128 * 2 * 4
    assert PackedKV.scratch_bytes([PagedKVNeed(8, 128, None)], 100, torch.bfloat16) == 0


def test_engine_option():
    for bits in (None, 4, 8):
        EngineConfig(cache_bits=bits).validate()
    for bits in (0, 2, 16, "4"):
        with pytest.raises(ValueError, match="cache_bits"):
            EngineConfig(cache_bits=bits).validate()
    with pytest.raises(ValueError, match="pages of 4"):
        EngineConfig(cache_bits=4, block_size=2).validate()


def spec(**more):
    p = dict(hidden_size=64, num_heads=4, num_kv_heads=2, head_dim=32, window=None, position=PartSpec("none"))
    p.update(more)
    return PartSpec("attention", p)


def test_layers_that_take_a_packed_cache_and_layers_that_refuse_it():
    ctx = BuildContext(torch.float32, "cpu", 64, 4, 16, cache_bits=4)
    need = build_mixer(spec(window=30, softcap=5.0, sink=True, distance_bias=True, temperature=(0.1, 8)), ctx).cache_need()
    assert need == PagedKVNeed(2, 32, 30, bits=4)
    for bad in (dict(v_head_dim=16), dict(row_norm=1e-6), dict(head_dim=24)):
        with pytest.raises((ValueError, ops.KernelError), match="cache"):
            build_mixer(spec(**bad), ctx)
    plain_need = build_mixer(spec(), BuildContext(torch.float32, "cpu", 64, 4, 16)).cache_need()
    assert plain_need == PagedKVNeed(2, 32, None)


def test_portions_that_are_refused():
    class NoDevice(PackedKV):
        def __init__(self):
            self.head_dim, self.page_size, self.bits, self.kv_heads, self._sms = 64, 16, 4, 2, 148
    kv = NoDevice()
    q, cu = torch.zeros(3, 4, 64), torch.zeros(2, dtype=torch.int32)
    tables, ctx = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for lens, held, message in (([3], [2], "brings"), ([3], [33], "block table"), ([3, 1], [3], "contexts")):
        with pytest.raises(ops.KernelError, match=message):
            kv.prefill(q, tables, cu, ctx, lens, held, 1.0)
    for bad in (torch.zeros(3, 3, 64), torch.zeros(3, 4, 32), torch.zeros(3, 256), torch.zeros(3, 0, 64)):
        with pytest.raises(ops.KernelError, match="q is"):
            kv.prefill(bad, tables, cu, ctx, [3], [3], 1.0)
        with pytest.raises(ops.KernelError, match="q is"):
            kv.decode(bad, tables, ctx, 3, 1.0)


@pytest.mark.parametrize("name,taken", [("llama_3_1_8b", True), ("llama_3_2_1b", True), ("llama_2_13b", True), ("rimidra_w2048", True),
                                        ("tekenex_w2048", False), ("bevuvik_w2048", False), ("fapudra_w2048", False), ("fivesun_w2048", False),
                                        ("matusun_w2048", False)])
def test_designs_that_take_a_packed_cache(name, taken):
    import json
    import os

    import gollmgo_b200
    from gollmgo_b200.parts import build_model
    with open(os.path.join(os.path.dirname(gollmgo_b200.__file__), "bench_shapes", name + ".json")) as f:
        config = json.load(f)
    ctx = BuildContext(torch.bfloat16, "cpu", 64, 4, 16, cache_bits=4)
    if not taken:
        with pytest.raises(ValueError, match="cache_bits"):
            build_model(config, ctx)
        return
    needs = build_model(config, ctx)[2].cache_needs()
    paged = [n for need in needs for n in (need if isinstance(need, tuple) else (need,)) if isinstance(n, PagedKVNeed)]
    assert paged and all(n.bits == 4 for n in paged)
