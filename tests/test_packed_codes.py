"""Codes of the packed cache where a value lies on the border between two of them, or next to one: the bytes of the pages are the
formula's (tests/plain_packed.py), whichever kernel writes them."""
import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def page_bytes_of(k, v, bits, page):
    """Pages uint8 [pages, kv heads, bytes] that hold k, v [T, kv heads, d] (float64, host) in slots 0 .. T - 1; zeros behind them."""
    T, nkv, d = k.shape
    row, par = d * bits // 8, 4 * (d // plain.group_of(d))
    out = torch.zeros(-(-T // page), nkv, plain.page_bytes(bits, d, page), dtype=torch.uint8)
    pg, pl = torch.arange(T) // page, torch.arange(T) % page
    for which, x in enumerate((k, v)):
        code, scale, off = plain.quantise(x, bits)
        c = code.to(torch.int64)
        if bits == 4:
            c = c[..., 0::2] + 16 * c[..., 1::2]
        pairs = torch.stack([scale, off], -1).flatten(-2).float().to(BF16).contiguous().view(torch.uint8)
        for h in range(nkv):
            out[pg[:, None], h, (which * page + pl[:, None]) * row + torch.arange(row)] = c[:, h].to(torch.uint8)
            out[pg[:, None], h, 2 * page * row + (which * page + pl[:, None]) * par + torch.arange(par)] = pairs[:, h]
    return out


def stored(qkv, nh, nkv, d, bits, page, pos=None, inv=None, magnitude=1.0):
    from gollmgo_b200.cache import PackedKV
    T = qkv.shape[0]
    kv = PackedKV.empty(-(-T // page), nkv, d, page, bits)
    kv.write(qkv.cuda(), None if pos is None else pos.cuda(), torch.arange(T, dtype=torch.int32).cuda(), nh, None if inv is None else inv.cuda(), False, magnitude)
    return kv.pages.cpu()


def rows_on_borders(T, nkv, d, g):
    """bfloat16 rows with many values half-way between two codes of 4 and of 8 bits: whole and half numbers, some of other scales and offsets."""
    x = torch.randint(0, 31, (T, nkv, d), generator=g) * 0.5
    x[..., 0::16], x[..., 1::16] = 0.0, 15.0
    wide = torch.randint(0, 511, (T, nkv, d), generator=g) * 0.5
    wide = torch.where(wide > 128, wide.round(), wide)                # (eight bits of a number)
    wide[..., 0::16], wide[..., 1::16] = 0.0, 255.0
    x = torch.where((torch.arange(T) % 2 == 0)[:, None, None], x, wide)
    scale = 2.0 ** torch.randint(-30, 30, (T, nkv, 1), generator=g)
    return (x * scale).to(BF16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("rows", ["normal", "borders"])
@pytest.mark.parametrize("turn", ["position 0", "frequency 0", "none"])
def test_values_between_two_codes(bits, d, rows, turn):
    """A rotation by nothing leaves bfloat16 values, which lie exactly between two codes often: ties go to the even one."""
    T, nh, nkv, page = 400, 1, 4, 16
    g = torch.Generator().manual_seed(bits * d)
    if rows == "normal":
        qkv = torch.randn(T, (nh + 2 * nkv) * d, generator=g).to(BF16)
    else:
        qkv = torch.cat([torch.zeros(T, nh, d, dtype=BF16), rows_on_borders(T, 2 * nkv, d, g)], 1).view(T, -1)
    inv = 500000.0 ** (-torch.arange(0, d, 2, dtype=F64) / d)
    pos = torch.zeros(T, dtype=torch.int32)
    if turn == "frequency 0":
        inv, pos = torch.zeros_like(inv), torch.arange(T, dtype=torch.int32) + 7
    got = stored(qkv, nh, nkv, d, bits, page, None if turn == "none" else pos, None if turn == "none" else inv)
    k, v = qkv.view(T, -1, d)[:, nh:].double().split(nkv, 1)
    assert torch.equal(got, page_bytes_of(k, v, bits, page))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tiny_values_beside_a_border(bits, d, dtype):
    """-9 + 2 x 4.5 is 0: a value of 2^-30 lies above the border and one of -2^-30 below it, though both vanish beside the offset in float32.
    (-11: the border between 5 and 6.  2^-60 vanishes in float64 too, and counts as the border.)"""
    nkv, page = 2, 16
    g = torch.Generator().manual_seed(d)
    rows = []
    for off, top in ((-9.0, 21.0 if bits == 4 else 500.0), (-11.0, 19.0 if bits == 4 else 498.0)):
        for up in (0, -20, 40):
            x = torch.randint(-4, 10, (2, nkv, d), generator=g).double()
            x[..., 0::16], x[..., 1::16] = off, top
            for i, tiny in enumerate((2.0 ** -30, -2.0 ** -30, 0.0, 2.0 ** -60, -2.0 ** -60, 2.0 ** -14, -2.0 ** -14)):
                x[..., 2 + i::16] = tiny
            rows.append(x * 2.0 ** up)
    x = torch.cat(rows)
    assert torch.equal(x.to(BF16).double(), x)
    k, v = x[0::2], x[1::2]
    got = stored(torch.cat([k, v], 1).flatten(1).to(dtype), 0, nkv, d, bits, page)
    code, scale, off = plain.quantise(k[:1], bits)
    assert float(scale[0, 0, 0]) == 2.0 and [int(c) for c in code[0, 0, 2:7]] == [5, 4, 4, 4, 4]
    assert torch.equal(got, page_bytes_of(k, v, bits, page))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_equal_values_have_code_0(bits, d, dtype):
    """A group of equal values has scale 0 and code 0, however large they are."""
    values = [0.0, 1.0, -3.0, 2.0 ** -100, 2.0 ** 62, -2.0 ** 64, 2.0 ** 65, 2.0 ** 100, -3e38, 3.3e38]
    x = torch.tensor(values, dtype=F64).to(BF16).double()[:, None, None].expand(-1, 2, d)
    got = stored(torch.cat([x, -x], 1).flatten(1).to(dtype), 0, 2, d, bits, 16)
    want = page_bytes_of(x, -x, bits, 16)
    assert torch.equal(got[0, :, :2 * 16 * (d * bits // 8)], torch.zeros_like(got[0, :, :2 * 16 * (d * bits // 8)]))
    # (the sign of a zero may be either)
    assert torch.equal(got[..., 2 * 16 * (d * bits // 8):].contiguous().view(BF16).double(), want[..., 2 * 16 * (d * bits // 8):].contiguous().view(BF16).double())
