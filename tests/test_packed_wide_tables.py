"""Block tables so wide that a launch takes few tokens: more go in several launches."""
import pytest
import torch

import plain_packed as plain
from gollmgo_b200.csrc import ops


def test_tokens_of_a_launch_and_their_scratch():
    most = ops.PACKED_DECODE_TOKENS
    assert ops.packed_decode_tokens(32, 8192, 16) == most
    assert ops.packed_decode_tokens(128, 2 ** 16, 16) == 255 and ops.packed_decode_tokens(8, 2 ** 24, 16) == 15
    assert ops.packed_decode_tokens(8, 2 ** 29, 16) == 1
    f = ops._packed("gg_packed_decode_mma")
    for n, message in ((255, "scratch"), (256, "too large")):
        args = [None, 64, 1, None, 4, None, 2 ** 16, 512, None, None, None, n, 64, None, 0, None, 128, 8, 64, 16, 4, 0, 1.0, 0.0, None, None, 0.0, 0.0, 0, None]
        assert f(*args) != 0 and message in ops.lib().gg_last_error().decode()
    p = ops._packed("gg_packed_prompt_f32")
    args = [None, 64, None, 4, None, 2 ** 16, 4, 16, None, 1, 600, 16, 64, None, 0, None, 128, 8, 64, 16, 4, 0, 1.0, 0.0, None, None, 0.0, 0.0, None]
    assert p(*args) != 0 and "scratch" in ops.lib().gg_last_error().decode()
    # a single token of a short context has a block for each pair (8 here); three have one for four tiles: 12 where a context has two, 6 where it has one
    for context, larger in ((40, 3), (20, 1)):
        sizes = (8, 8, 64, 4, context, 0)
        size = {n: ops.packed_decode_scratch(torch.bfloat16, n, *sizes) for n in (1, 3)}
        assert size[larger] > size[4 - larger]
        assert ops.packed_launches_scratch(torch.bfloat16, 7, 3, *sizes) == size[larger] and ops.packed_launches_scratch(torch.bfloat16, 6, 3, *sizes) == size[3]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_and_portions_over_very_wide_tables(bits, dtype):
    from gollmgo_b200.cache import PackedKV
    nh, nkv, d, page, n = 8, 8, 64, 256, 7
    width = 2 ** 31 // (nh * 16 * 3) - 1
    assert ops.packed_decode_tokens(nh, width, page) == 3
    kv = PackedKV.empty(n, nkv, d, page, bits)
    g = torch.Generator().manual_seed(bits)
    lens = [40, 1, 33, 17, 256, 64, 39]
    x = torch.randn(n, page, (nh + 2 * nkv) * d, generator=g).to(dtype)
    kv.write(x.view(n * page, -1).cuda(), None, torch.arange(n * page, dtype=torch.int32).cuda(), nh)
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    tables[:, 0] = torch.arange(n, dtype=torch.int32)
    ctx = torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.randn(n, nh, d, generator=g).to(dtype)
    held = [[plain.through(y.double().view(page, nkv, d), bits) for y in x[b, :, nh * d:].chunk(2, 1)] for b in range(n)]

    def check(out, rows, b, context):
        ref = plain.attend(rows.double(), held[b][0][:context], held[b][1][:context], context, d ** -0.5)
        # scores in float32: |q| |k| in steps of 2^-20 at most, twice; weights rounded to half precision in bfloat16; the result's rounding
        e = float(rows.double().norm(dim=-1).max() * held[b][0].norm(dim=-1).max()) * d ** -0.5 * 2.0 ** -20 + 2.0 ** -20
        w = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -20
        top = float(held[b][1][:context].abs().max())
        assert ((out.cpu().double() - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (2 * e + 2 * w) * top).all(), b
    order = torch.randperm(n, generator=g).to(torch.int32).cuda()
    cu = torch.arange(n + 1, dtype=torch.int32).cuda()
    for said, more in ((40, dict()), (40, dict(cu_q_lens=cu)), (40, dict(seqs=order, cu_q_lens=cu)), (20, dict()), (20, dict(cu_q_lens=cu))):
        out = kv.decode(q.cuda(), tables, ctx, said, d ** -0.5, **more)
        for b in range(n):
            check(out[b:b + 1], q[b:b + 1], b, lens[b])
    if dtype == torch.float32:                       # (portions of 7 rows: 8 rows share an item, so an item each)
        q = torch.randn(n * 7, nh, d, generator=g)
        held_lens = [max(7, c) for c in lens]
        out = kv.prefill(q.cuda(), tables, cu * 7, torch.tensor(held_lens, dtype=torch.int32).cuda(), [7] * n, held_lens, d ** -0.5)
        for b in range(n):
            check(out[7 * b:7 * b + 7], q[7 * b:7 * b + 7], b, held_lens[b])
