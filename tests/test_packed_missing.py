"""Pages that are in sight but not in the pool (given back, or an id outside it): their keys are not attended to by single tokens,
whichever kernel runs."""
import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (96, 16), (128, 8), (64, 4)])
@pytest.mark.parametrize("option", [0, 1, 2])
def test_single_tokens_do_not_attend_to_missing_pages(bits, dtype, d, page, option):
    from gollmgo_b200.cache import PackedKV
    nh, nkv, n, width = 6, 2, 150, -(-150 // page)
    g = torch.Generator().manual_seed(d + page)
    kv = PackedKV.empty(4 * width, nkv, d, page, bits)
    x = torch.randn(4, n, (nh + 2 * nkv) * d, generator=g).to(dtype)
    tables = torch.randperm(4 * width, generator=g).to(torch.int32).view(4, width)
    t = torch.arange(n)
    slots = torch.cat([tables[b][t // page].long() * page + t % page for b in range(4)]).to(torch.int32)
    kv.write(x.view(4 * n, -1).cuda(), None, slots.cuda(), nh)
    missing = tables.clone()
    missing[0, 0] = -1
    missing[0, -1] = 4 * width                       # (the newest keys: the first id outside the pool)
    missing[1, 1::2] = 2 ** 30
    missing[2] = -1                                  # nothing is left
    q = torch.randn(4, nh, d, generator=g).to(dtype)
    more = [dict(), dict(window=70), dict(slopes=True, sink=True, softcap=4.0)][option]
    if option == 2:
        more["sink"], more["slopes"] = torch.randn(nh, generator=g), torch.tensor([2.0 ** -(h + 2) for h in range(nh)])
    ctx = torch.full((4,), n, dtype=torch.int32).cuda()
    out = kv.decode(q.cuda(), missing.cuda(), ctx, n, d ** -0.5, **{k: v.cuda() if torch.is_tensor(v) else v for k, v in more.items()}).cpu().double()
    for b in range(4):
        k, v = (plain.through(y.double().view(n, nkv, d), bits) for y in x[b, :, nh * d:].chunk(2, 1))
        there = ((missing[b] >= 0) & (missing[b] < 4 * width))[t // page]
        if more.get("window"):
            there &= t >= n - more["window"]
        for h in range(nh):
            z = k[there, h // 3] @ q[b, h].double() * d ** -0.5
            if option == 2:
                z = more["softcap"] * torch.tanh(z / more["softcap"]) - more["slopes"][h].double() * (n - 1 - t[there])
                z = torch.cat([z, more["sink"][h].double()[None]])
            if not there.any():
                assert (out[b, h] == 0).all()
                continue
            w = torch.softmax(z, 0)[:int(there.sum())]
            ref, size = w @ v[there, h // 3], w @ v[there, h // 3].abs()
            # scores: products of d terms (|q| |k| scale of them, in steps of 2^-20 at most where a tensor core truncates), twice; weights as halves
            # in bfloat16 (2^-11); the result's rounding
            e = float(q[b, h].double().norm() * k.norm(dim=-1).max()) * d ** -0.5 * 2.0 ** -20 + 2.0 ** -20
            wt = 2.0 ** -11 if dtype == BF16 else 2.0 ** -20
            assert ((out[b, h] - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (2 * e + 2 * wt) * size.max()).all(), (b, h)
