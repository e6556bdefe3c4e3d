"""The 4-bit paged KV cache against its definition in 64 bits: storing, reading, decode attention, eviction.  Every
test runs on the CPU references and, marked ``gpu``, on the kernels."""

import math

import pytest
import torch

from rl_project_b200.ops.paged_q4 import (paged_decode_q4, paged_evict_q4, paged_gather_q4, paged_read_q4,
                                          paged_write_q4, q4_block_bytes)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF = torch.bfloat16
F64 = torch.float64


@pytest.fixture(params=DEVICES)
def dev(request):
    yield request.param
    if request.param == "cuda":  # no test leaves an index error behind
        from rl_project_b200.ops._ext import check_bounds

        check_bounds(torch.device("cuda", 0))


def index_error(dev, call):
    """The call's index error: raised by the CPU references, left in the device's word by the kernels."""
    if dev == "cpu":
        with pytest.raises(IndexError):
            call()
        return None
    from rl_project_b200.core.errors import KernelError
    from rl_project_b200.ops._ext import check_bounds

    out = call()
    with pytest.raises(KernelError):
        check_bounds(torch.device("cuda", 0))
    return out


# ---------------------------------------------------------------- the definition, on the CPU in 64 bits
def stored(x):
    """Codes, scales and minima of bf16 rows [..., D], and the values they stand for."""
    g = min(x.shape[-1], 64)
    y = x.cpu().to(F64).unflatten(-1, (-1, g))
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).to(BF).to(F64)
    code = torch.where(scale > 0, (y - lo) / scale.clamp_min(1e-300), torch.zeros_like(y)).round().clamp(0, 15)
    return code.flatten(-2), scale, lo, (code * scale + lo).flatten(-2)


def rows(*shape):
    spread = 0.2 + 3 * torch.rand(shape[-1]) ** 3
    return (torch.randn(*shape) * spread + torch.randn(shape[-1])).to(BF)


def cache(lens, Hkv, D, dev, extra=0, spare=3):
    """Pools holding random rows for sequences of `lens`, in shuffled blocks, the unused bytes all 0xff (scales that
    are NaN); returns (k, v) values as lists of [n, Hkv, D] fp64, the pools, tables and lens."""
    width = max(1, max(-(-n // 16) for n in lens))
    ids = torch.randperm(len(lens) * width + extra + spare)
    tables = ids[:len(lens) * width].view(len(lens), width).int()
    pools = [torch.full((len(ids), Hkv, q4_block_bytes(D)), 255, dtype=torch.uint8, device=dev) for _ in range(2)]
    blocks, offs, ks, vs = [], [], [], []
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        blocks.append(tables[b][pos // 16])
        offs.append((pos % 16).int())
        ks.append(rows(n, Hkv, D))
        vs.append(rows(n, Hkv, D))
    paged_write_q4(torch.cat(ks).to(dev), torch.cat(vs).to(dev), *pools, torch.cat(blocks).int().to(dev),
                   torch.cat(offs).to(dev))
    vals = [[stored(x)[3] for x in xs] for xs in (ks, vs)]
    return vals[0], vals[1], pools, tables.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), ids


def attention(q, k, v, scale, softcap, window):
    """fp64 output [Hq, D], weights [Hkv, n] summed over each group, and what errors are measured by (check_decode),
    of one sequence."""
    n, Hkv, D = k.shape
    if n == 0:
        z = torch.zeros(q.shape, dtype=F64)
        return z, torch.zeros(Hkv, 0, dtype=F64), z
    s = torch.einsum("hgd,thd->hgt", q.cpu().to(F64).view(Hkv, -1, D), k) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if window and n > window:
        s[..., :n - window] = -math.inf
    p = torch.softmax(s, -1)
    groups = v.unflatten(-1, (-1, min(D, 64)))
    eight = (groups.amax(-1, keepdim=True) - groups.amin(-1, keepdim=True)).expand_as(groups).flatten(-2) * 8 / 15
    o, a = (torch.einsum("hgt,thd->hgd", p, x).reshape(q.shape) for x in (v, v.abs() + 8 * eight))
    return o, p.sum(1), a


# Decode's error: rounding the output to bf16 is 2^-8 of the value.  Before it, a weight's relative error is that of its
# exponent (|s| below 2^5 here, held in fp32 with a few roundings: 2^5 * 2^-23 * 4 = 2^-16), and the sums are fp32:
# together below 2^-14 of sum p |v|.  The kernel also rounds each p * scale to fp16, 2^-11 of it, which multiplies a
# centred code (code - 8, at most 8): 2^-11 sum p 8 scale, with scale a 15th of the spread of the token's group (both
# ends of which are stored values).  attention() returns sum p |v| + 2^3 sum p 8 scale.
def check_decode(out, o, a):
    err = (out.cpu().to(F64) - o).abs()
    assert (err <= 2 ** -8 * o.abs() + 2 ** -14 * a + 1e-30).all(), (err - 2 ** -8 * o.abs() - 2 ** -14 * a).max()


# ---------------------------------------------------------------- storing and reading
@pytest.mark.parametrize("N,Hkv,D", [(1, 1, 64), (5, 3, 128), (37, 2, 32), (300, 8, 64), (0, 2, 64), (1000, 4, 128)])
def test_write_and_read(dev, N, Hkv, D):
    blocks = N // 16 + 3
    place = torch.randperm(blocks * 16)
    used, free = place[:N], place[N:]
    pools = [torch.full((blocks, Hkv, q4_block_bytes(D)), 37, dtype=torch.uint8, device=dev) for _ in range(2)]
    before = [x.cpu() for x in paged_read_q4(*pools, (free // 16).int().to(dev), (free % 16).int().to(dev), D)]
    blk, off = (used // 16).int().to(dev), (used % 16).int().to(dev)
    k, v = rows(N, Hkv, D), rows(N, Hkv, D)
    paged_write_q4(k.to(dev), v.to(dev), *pools, blk, off)
    got = paged_read_q4(*pools, blk, off, D)
    for x, y in zip((k, v), got):
        assert y.shape == (N, Hkv, D) and y.dtype == BF
        want = stored(x)[3]
        assert ((y.cpu().to(F64) - want).abs() <= 2 ** -8 * want.abs()).all()  # one rounding to bf16
    after = paged_read_q4(*pools, (free // 16).int().to(dev), (free % 16).int().to(dev), D)
    for x, y in zip(before, after):  # the other slots are as they were
        assert torch.equal(x, y.cpu())


@pytest.mark.parametrize("D", [32, 64, 128])
def test_stored_bytes(dev, D):
    """The documented layout, byte by byte."""
    k, v = rows(16, 2, D), rows(16, 2, D)
    pools = [torch.zeros(1, 2, q4_block_bytes(D), dtype=torch.uint8, device=dev) for _ in range(2)]
    paged_write_q4(k.to(dev), v.to(dev), *pools, torch.zeros(16, dtype=torch.int32, device=dev),
                   torch.arange(16, dtype=torch.int32, device=dev))
    g = min(D, 64)
    for x, pool in zip((k, v), pools):
        code, scale, lo, _ = stored(x)
        for h in range(2):
            b = pool[0, h].cpu()
            want = code[:, h].view(16, D // g, g // 2, 2).transpose(0, 1).to(torch.uint8)
            assert torch.equal(b[:8 * D].view(D // g, 16, g // 2), want[..., 0] | (want[..., 1] << 4))
            meta = b[8 * D:].view(BF).view(D // g, 16, 2).transpose(0, 1).to(F64)
            assert torch.equal(meta[..., 0], scale[:, h, :, 0]) and torch.equal(meta[..., 1], lo[:, h, :, 0])


def test_write_strided_and_special_rows(dev):
    """Rows inside a wider projection; groups without spread, of the lowest value, with NaN and with infinities."""
    D, Hkv = 64, 2
    wide = rows(9, 6, D)
    wide[1, 2] = 0.75
    wide[2, 2] = torch.finfo(BF).min
    wide[3, 2, 5] = math.nan
    wide[4, 2, 7] = math.inf
    wide[5, 2, 7] = -math.inf
    wide[6, 2, :] = 0.0
    wide[6, 2, 3] = 1e-40
    wide = wide.to(dev)
    odd = torch.empty(9, 2, D + 1, dtype=BF, device=dev)[..., 1:]  # rows that do not start on 16 bytes
    odd.copy_(wide[:, 4:])
    pools = [torch.zeros(1, Hkv, q4_block_bytes(D), dtype=torch.uint8, device=dev) for _ in range(2)]
    blk, off = torch.zeros(9, dtype=torch.int32, device=dev), torch.arange(9, dtype=torch.int32, device=dev)
    paged_write_q4(wide[:, 2:4], odd, *pools, blk, off)
    k, v = (t.cpu().to(F64) for t in paged_read_q4(*pools, blk, off, D))
    x = wide[:, 2:4].cpu()
    bad = torch.zeros(9, 2, dtype=torch.bool)
    bad[3:6, 0] = True
    assert torch.isnan(k[bad]).all()
    want = stored(torch.where(bad[..., None], torch.zeros_like(x), x))[3]
    assert ((k - want).abs()[~bad] <= (2 ** -8 * want.abs())[~bad] + 1e-41).all()
    want = stored(wide[:, 4:])[3]
    assert ((v - want).abs() <= 2 ** -8 * want.abs()).all()
    assert torch.equal(k[1, 0], torch.full((D,), 0.75, dtype=F64))


def test_bad_slots(dev):
    D = 64
    pools = [torch.zeros(2, 1, q4_block_bytes(D), dtype=torch.uint8, device=dev) for _ in range(2)]
    x = rows(3, 1, D).to(dev)
    for blk, off in (([0, 2, 1], [0, 0, 0]), ([0, -1, 1], [0, 0, 0]), ([0, 0, 1], [0, 16, 0]), ([0, 0, 1], [0, -1, 0])):
        blk = torch.tensor(blk, dtype=torch.int32, device=dev)
        off = torch.tensor(off, dtype=torch.int32, device=dev)
        index_error(dev, lambda: paged_write_q4(x, x, *pools, blk, off))
        out = index_error(dev, lambda: paged_read_q4(*pools, blk, off, D))
        if out is not None:  # the good rows are there, the bad one reads as zeros
            want = stored(x)[3]
            for i in (0, 2):
                assert ((out[0][i].cpu().to(F64) - want[i]).abs() <= 2 ** -8 * want[i].abs()).all()
            assert not out[0][1].any()


@pytest.mark.parametrize("max_len", [1, 20, 64])
def test_gather(dev, max_len):
    lens = [17, 0, 64, 1]
    ks, vs, pools, tables, n, _ = cache(lens, 2, 64, dev)
    k, v = paged_gather_q4(*pools, tables, n, 64, max_len)
    assert k.shape == (4, max_len, 2, 64)
    for b, m in enumerate(lens):
        m = min(m, max_len)
        for got, want in ((k, ks[b][:m]), (v, vs[b][:m])):
            assert ((got[b, :m].cpu().to(F64) - want).abs() <= 2 ** -8 * want.abs()).all()
            assert not got[b, m:].any()


# ---------------------------------------------------------------- decode attention
@pytest.mark.parametrize("lens,Hkv,G,D,window,softcap", [
    ([1], 1, 1, 64, 0, 0.0),
    ([16, 15, 17, 1, 0, 33], 2, 4, 64, 0, 0.0),
    ([500, 3, 0, 129], 3, 1, 128, 0, 0.0),
    ([257, 256], 2, 8, 128, 0, 0.0),
    ([70, 31, 200], 1, 16, 64, 0, 0.0),
    ([70, 31, 200], 2, 11, 128, 0, 0.0),
    ([90, 5], 2, 3, 32, 0, 0.0),
    ([300, 40, 41, 39], 2, 4, 64, 40, 0.0),
    ([300, 40, 41, 39], 2, 5, 128, 1, 0.0),
    ([150, 64], 2, 2, 128, 100, 5.0),
    ([1000] * 3, 2, 7, 64, 0, 20.0),
    ([5000, 1], 1, 4, 128, 0, 0.0),
    ([4097, 20, 800], 2, 4, 32, 3000, 0.0),
    ([20011], 1, 2, 64, 0, 0.0),
])
@pytest.mark.parametrize("weighted", [False, True])
def test_decode(dev, lens, Hkv, G, D, window, softcap, weighted):
    if dev == "cpu" and max(lens) > 10000:
        pytest.skip("long contexts are for the kernels")
    ks, vs, pools, tables, n, _ = cache(lens, Hkv, D, dev)
    q = torch.randn(len(lens), Hkv * G, D).to(BF).to(dev)
    scale = 1 / math.sqrt(D)
    w = w_rows = w0 = None
    if weighted:
        w = torch.rand(len(lens) + 2, Hkv, tables.shape[1] * 16 + 5).to(dev)
        w0 = w.cpu().to(F64)
        w_rows = torch.randperm(len(lens) + 2)[:len(lens)].int()
        w_rows[-1] = w_rows[-1] if len(lens) == 1 else -1  # the last sequence accumulates nothing
    out = paged_decode_q4(q, *pools, tables, n, scale, softcap, window, w,
                          None if w_rows is None else w_rows.to(dev))
    assert out.shape == q.shape and out.dtype == BF
    add = None if w0 is None else torch.zeros_like(w0)
    for b, m in enumerate(lens):
        o, p, a = attention(q[b], ks[b], vs[b], scale, softcap, window)
        check_decode(out[b], o, a)
        if weighted and w_rows[b] >= 0:
            add[w_rows[b], :, :m] += p
    if weighted:  # a weight is off like decode's (2^-15 of it), the sum by one rounding
        err = (w.cpu().to(F64) - (w0 + add)).abs()
        assert (err <= 2 ** -15 * add + 2 ** -23 * (w0 + add)).all(), err.max()
        assert torch.equal(w.cpu().to(F64)[add == 0], w0[add == 0])


def test_decode_large_scores(dev):
    """Scores far apart: the largest takes all, early or late in the cache, and nothing overflows."""
    lens, D = [700, 700], 64
    ks, vs, pools, tables, n, _ = cache(lens, 1, D, dev)
    q = torch.stack([ks[0][3, 0], ks[1][690, 0]]).to(BF)[:, None].to(dev) * 8
    out = paged_decode_q4(q, *pools, tables, n, 1.0)
    for b in range(2):
        # scores up to 2^12: their exponents are off by 2^12 * 2^-23 * 4, so weights by 2^-9 of sum p |v|
        o, _, a = attention(q[b], ks[b], vs[b], 1.0, 0.0, 0)
        assert ((out[b].cpu().to(F64) - o).abs() <= 2 ** -8 * o.abs() + 2 ** -9 * a).all()


def test_decode_offset_channels(dev):
    """Values with a common offset far above their spread (the codes' own rounding is tested against the stored
    values): the output keeps the offset's precision."""
    lens, D = [300], 128
    ks, vs, pools, tables, n, _ = cache(lens, 2, D, dev)
    v = (torch.randn(300, 2, D) * 0.05 + 30).to(BF)
    k = rows(300, 2, D)
    pos = torch.arange(300)
    paged_write_q4(k.to(dev), v.to(dev), *pools, tables[0][(pos // 16).to(dev)].contiguous(), (pos % 16).int().to(dev))
    q = torch.randn(1, 8, D).to(BF).to(dev)
    out = paged_decode_q4(q, *pools, tables, n, 1 / math.sqrt(D))
    o, _, a = attention(q[0], stored(k)[3], stored(v)[3], 1 / math.sqrt(D), 0.0, 0)
    check_decode(out[0], o, a)


@pytest.mark.parametrize("size", [1e-12, 1e-4, 1e15, 1e19, 1e22, 1e30])
def test_decode_value_sizes(dev, size):
    """Values of any size, alone and behind ordinary ones; the weights do not depend on them."""
    lens, D = [300, 2000], 64
    ks, vs, pools, tables, n, _ = cache(lens, 1, D, dev)
    k, v = (torch.cat(x) for x in (ks, vs))
    big = v * size
    big[300:1700] = v[300:1700]  # the second sequence's last values only
    pos = torch.cat([torch.arange(m) for m in lens])
    seq = torch.arange(2).repeat_interleave(torch.tensor(lens))
    big = big.to(BF)
    paged_write_q4(k.to(BF).to(dev), big.to(dev), *pools, tables[seq.to(dev), (pos // 16).to(dev)].contiguous(),
                   (pos % 16).int().to(dev))
    ks, vs = (stored(x.to(BF))[3].split(lens) for x in (k, big))
    q = torch.randn(2, 4, D).to(BF).to(dev)
    w = torch.zeros(2, 1, tables.shape[1] * 16, device=dev)
    out = paged_decode_q4(q, *pools, tables, n, 0.125, weights=w, weight_rows=torch.tensor([0, 1], dtype=torch.int32, device=dev))
    for b in range(2):
        o, p, a = attention(q[b], ks[b], vs[b], 0.125, 0.0, 0)
        check_decode(out[b], o, a)
        assert ((w[b, 0, :lens[b]].cpu().to(F64) - p.sum(0).flatten()).abs() <= 2 ** -15 * p.sum(0).flatten()).all()


@pytest.mark.parametrize("D,G", [(32, 3), (64, 4), (128, 1), (128, 11)])
@pytest.mark.parametrize("lens", [[1, 5], [40, 700]])
def test_decode_weights_keep_their_bits(dev, D, G, lens):
    """Dimensions that are zero in every value, while their groups' scales are not, come out as zero: the minimum's part
    and the codes' part cancel up to the weights' own rounding."""
    ks, vs, pools, tables, n, _ = cache(lens, 1, D, dev)
    q = torch.randn(len(lens), G, D).to(BF).to(dev)
    for b, m in enumerate(lens):
        v = torch.rand(m, 1, D).to(BF) + 1
        v[..., ::5] = 0
        pos = torch.arange(m)
        paged_write_q4(ks[b].to(BF).to(dev), v.to(dev), *pools, tables[b][(pos // 16).to(dev)].contiguous(),
                       (pos % 16).int().to(dev))
        vs[b] = v
    out = paged_decode_q4(q, *pools, tables, n, 1 / math.sqrt(D)).cpu().to(F64)
    # a weight is held in two bf16 parts, 2^-16 of it; it multiplies 8 scales, a scale being 2 / 15 at most
    # (bf16's rounding included: 0.14); the fp32 sums add 700 * 2^-24 of the same
    assert out[..., ::5].abs().max() <= (2 ** -16 + 2 ** -14) * 8 * 0.14
    assert (out[..., 1::5] > 0.9).all()


@pytest.mark.parametrize("D,G", [(32, 2), (64, 4), (128, 9)])
@pytest.mark.parametrize("ratio", [10, 20, 28, 60])
def test_decode_values_far_apart(dev, ratio, D, G):
    """Tokens whose values are 2^ratio times the others', but whose weight makes them count for nothing, take no bits
    from the others."""
    lens = [2000, 37]
    ks, vs, pools, tables, n, _ = cache(lens, 1, D, dev)
    q = torch.randn(2, G, D).to(BF)
    q[..., 0] = 8
    gap = (ratio + 12) * math.log(2) + 12  # in scores; the others lie within 4 of 0 or so
    for b, m in enumerate(lens):
        k, v = torch.randn(m, 1, D) * 0.3, torch.randn(m, 1, D)
        far = torch.arange(m) % 29 == 20
        k[far] *= 0.1
        k[far, :, 0] = -gap
        v[far] *= 2.0 ** ratio
        pos = torch.arange(m)
        paged_write_q4(k.to(BF).to(dev), v.to(BF).to(dev), *pools, tables[b][(pos // 16).to(dev)].contiguous(),
                       (pos % 16).int().to(dev))
        ks[b], vs[b] = stored(k.to(BF))[3], stored(v.to(BF))[3]
    out = paged_decode_q4(q.to(dev), *pools, tables, n, 0.125).cpu().to(F64)
    for b in range(2):
        o, _, a = attention(q[b], ks[b], vs[b], 0.125, 0.0, 0)
        near = torch.arange(lens[b]) % 29 != 20
        # without the far tokens: theirs is 2^-12 of a value or less, which `a` holds
        _, _, rest = attention(q[b], ks[b][near], vs[b][near], 0.125, 0.0, 0)
        assert (a <= 2 * rest).all()
        # check_decode's bound, on a measure without the 8 times 8 scales of a single fp16 weight
        p = torch.softmax(torch.einsum("hd,td->ht", q[b].to(F64), ks[b][:, 0]) * 0.125, -1)
        groups = vs[b][:, 0].unflatten(-1, (-1, min(D, 64)))
        eight = ((groups.amax(-1) - groups.amin(-1)) * 8 / 15)[..., None].expand_as(groups).flatten(-2)
        bound = torch.einsum("ht,td->hd", p, vs[b][:, 0].abs() + eight)
        err = (out[b] - o).abs() - 2 ** -8 * o.abs()
        assert (err <= 2 ** -14 * bound).all(), (err / bound).max()


def test_decode_not_a_number(dev):
    """A key or a value that holds NaN: its head's output is NaN (with a NaN key its weights too), others are as ever."""
    lens, D = [50, 700], 64
    ks, vs, pools, tables, n, _ = cache(lens, 2, D, dev)
    # a row's weights sum up to its 2 query heads, off by 700 roundings and exponents of 2^-24 to 2^-22 each
    bad = torch.full((1, 2, D), math.nan, dtype=BF, device=dev)
    for b, h, pos, pool in ((0, 1, 3, 0), (1, 0, 650, 0), (1, 1, 699, 1)):
        both = [p.clone() for p in pools]
        i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)
        paged_write_q4(bad, bad, *both, i32(int(tables[b, pos // 16])), i32(pos % 16))
        blk, other = int(tables[b, pos // 16]), 1 - h
        pools_b = [p.clone() for p in pools]
        pools_b[pool][blk, h] = both[pool][blk, h]
        q = torch.randn(2, 4, D).to(BF).to(dev)
        w = torch.zeros(2, 2, tables.shape[1] * 16, device=dev)
        rows_ = torch.tensor([1, 0], dtype=torch.int32, device=dev)
        out = paged_decode_q4(q, *pools_b, tables, n, 0.125, weights=w, weight_rows=rows_).view(2, 2, 2, D)
        assert out[b, h].isnan().all()
        if pool == 0:
            assert w[rows_[b], h, :lens[b]].isnan().all()
        else:
            assert abs(float(w[rows_[b], h].sum()) - 2) < 1e-4
        for s, head in ((b, other), (1 - b, 0), (1 - b, 1)):
            o, p, a = attention(q[s].view(2, 2, D)[head], ks[s][:, head:head + 1], vs[s][:, head:head + 1], 0.125, 0.0, 0)
            check_decode(out[s, head], o, a)
            assert abs(float(w[rows_[s], head].sum()) - 2) < 1e-4 and not w[rows_[s], head, lens[s]:].any()


def test_decode_bad_index(dev):
    """A block outside the pool, a context longer than its table, an accumulator row that is not there."""
    lens, D = [40, 40], 64
    ks, vs, pools, tables, n, _ = cache(lens, 1, D, dev)
    q = torch.randn(2, 2, D).to(BF).to(dev)
    for bad in (-1, 10 ** 6):
        t = tables.clone()
        t[0, 1] = bad
        out = index_error(dev, lambda: paged_decode_q4(q, *pools, t, n, 0.125))
        if out is not None:  # the other sequence is right, and the bad block's tokens are left out
            o, _, a = attention(q[1], ks[1], vs[1], 0.125, 0.0, 0)
            check_decode(out[1], o, a)
            left = torch.cat([torch.arange(16), torch.arange(32, 40)])
            o, _, a = attention(q[0], ks[0][left], vs[0][left], 0.125, 0.0, 0)
            check_decode(out[0], o, a)
    index_error(dev, lambda: paged_decode_q4(q, *pools, tables, n + 30, 0.125))
    short = torch.zeros(2, 1, 39, device=dev)  # (tokens that have a place are accumulated all the same)
    index_error(dev, lambda: paged_decode_q4(q, *pools, tables, n, 0.125, 0.0, 0, short,
                                             torch.tensor([0, 1], dtype=torch.int32, device=dev)))
    w = torch.zeros(2, 1, 48, device=dev)
    index_error(dev, lambda: paged_decode_q4(q, *pools, tables, n, 0.125, 0.0, 0, w,
                                             torch.tensor([0, 2], dtype=torch.int32, device=dev)))


def test_decode_without_any_block(dev):
    """A sequence none of whose blocks exist: reported, its output zero, its weights as they were, the others' right."""
    lens, D = [40, 700], 64
    ks, vs, pools, tables, n, _ = cache(lens, 2, D, dev)
    q = torch.randn(2, 4, D).to(BF).to(dev)
    for b in range(2):
        t = tables.clone()
        t[b] = -1
        w = torch.ones(2, 2, tables.shape[1] * 16, device=dev)
        out = index_error(dev, lambda: paged_decode_q4(q, *pools, t, n, 0.125, 0.0, 0, w,
                                                       torch.tensor([0, 1], dtype=torch.int32, device=dev)))
        if out is not None:
            o, p, a = attention(q[1 - b], ks[1 - b], vs[1 - b], 0.125, 0.0, 0)
            check_decode(out[1 - b], o, a)
            assert not out[b].any() and (w[b] == 1).all()
            assert ((w[1 - b, :, :lens[1 - b]].cpu() - 1 - p).abs() <= 2 ** -15 * p + 2 ** -23 * (1 + p)).all()


# ---------------------------------------------------------------- eviction
def chosen(w, n, keep, sink, recent):
    """Positions kept of one head's weights (a list of floats), by definition."""
    if n <= keep:
        return list(range(n))
    fixed = [t for t in range(n) if t < sink or t >= n - recent]
    rest = [t for t in range(n) if sink <= t < n - recent]
    rank = sorted(rest, key=lambda t: (-math.inf if math.isnan(w[t]) else w[t], -t), reverse=True)
    return sorted(fixed + rank[:keep - len(fixed)])


@pytest.mark.parametrize("lens,Hkv,D,keep,sink,recent,kind", [
    ([100, 16, 37, 0, 1], 2, 64, 20, 2, 5, "random"),
    ([300, 299], 3, 128, 256, 0, 0, "random"),
    ([50, 80], 1, 32, 17, 17, 0, "random"),
    ([50, 80], 1, 64, 17, 0, 17, "random"),
    ([50, 80], 2, 128, 1, 0, 0, "random"),
    ([2500, 1025, 1024, 1023], 2, 64, 1000, 4, 64, "ties"),
    ([5000], 1, 64, 4100, 1, 10, "zeros"),
    ([9000, 4097, 8999], 1, 32, 4096, 3, 100, "ties"),
    ([17000], 2, 32, 3001, 0, 1, "random"),
    ([41000, 40960], 1, 32, 2000, 2, 9, "random"),
    ([41000], 1, 32, 40000, 2, 9, "odd"),
    ([16384], 1, 32, 16000, 0, 0, "ties"),
    ([132000, 131073], 1, 32, 3000, 2, 9, "random"),
    ([132000], 1, 32, 131000, 2, 9, "odd"),
    ([20000, 17, 9000, 5001], 2, 64, 5000, 4, 30, "ties"),
    ([40000, 16385], 2, 32, 3000, 0, 2900, "odd"),
    ([131072, 70000], 1, 32, 100, 0, 0, "zeros"),
    ([131072], 1, 32, 77, 70, 7, "random"),
    ([17000, 30, 400], 12, 32, 300, 3, 50, "ties"),
    ([40960, 16500, 90], 11, 32, 16500, 1, 0, "odd"),
    ([90, 33], 2, 64, 30, 1, 1, "odd"),
    ([70], 2, 64, 90, 1, 1, "random"),
])
def test_evict(dev, lens, Hkv, D, keep, sink, recent, kind):
    if dev == "cpu" and max(lens) > 50000:
        pytest.skip("long sequences are for the kernels")
    new_w = -(-keep // 16)
    ks, vs, pools, tables, n, ids = cache(lens, Hkv, D, dev, extra=len(lens) * new_w)
    new = ids[-len(lens) * new_w:].view(len(lens), new_w).int().to(dev)
    old = [p.clone().cpu() for p in pools]
    w = torch.rand(len(lens) + 1, Hkv, tables.shape[1] * 16 + 3)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "zeros":
        w = torch.zeros_like(w)
    elif kind == "odd":
        w = w - 0.5
        w[..., ::5], w[..., 1::7], w[..., 2::9], w[..., 3::11] = math.nan, -0.0, 0.0, math.inf
    w_rows = torch.randperm(len(lens) + 1)[:len(lens)].int()
    wd = w.clone().to(dev)
    kept, new_lens = paged_evict_q4(*pools, tables, n, new, wd, w_rows.to(dev), keep, D, recent=recent, sink=sink)
    assert kept.shape == (len(lens), Hkv, keep) and kept.dtype == torch.int32 and new_lens.dtype == torch.int32
    assert new_lens.tolist() == [min(m, keep) for m in lens]
    k, v = paged_gather_q4(*pools, new, new_lens, D, keep)
    want_w = w.clone()
    for b, m in enumerate(lens):
        for h in range(Hkv):
            row = w[w_rows[b], h]
            pos = chosen(row[:m].tolist(), m, keep, sink, recent)
            assert kept[b, h].tolist() == pos + [-1] * (keep - len(pos))
            if m > keep:
                want_w[w_rows[b], h, :m] = 0
                want_w[w_rows[b], h, :len(pos)] = row[pos]
            for got, xs in ((k, ks), (v, vs)):
                want = xs[b][pos, h]
                assert ((got[b, :len(pos), h].cpu().to(F64) - want).abs() <= 2 ** -8 * want.abs()).all()
    assert torch.equal(wd.cpu().view(torch.int32), want_w.view(torch.int32))
    rest = torch.ones(len(old[0]), dtype=torch.bool)
    rest[new.cpu().long().flatten()] = False
    for p, q in zip(old, pools):  # no other block changes
        assert torch.equal(p[rest], q.cpu()[rest])


def test_evict_many_long_rows(dev):
    """More long rows than clusters take: one CTA a row."""
    test_evict(dev, [41000, 40970, 500], 22, 32, 700, 3, 60, "ties")


def test_empty_calls(dev):
    """No rows, no sequences, tables without blocks, and a batch of nothing but padding."""
    D = 64
    pools = [torch.zeros(2, 2, q4_block_bytes(D), dtype=torch.uint8, device=dev) for _ in range(2)]
    i0, t0 = (torch.zeros(*s, dtype=torch.int32, device=dev) for s in ((0,), (0, 3)))
    assert paged_decode_q4(torch.zeros(0, 4, D, dtype=BF, device=dev), *pools, t0, i0, 1.0).shape == (0, 4, D)
    kept, lens = paged_evict_q4(*pools, t0, i0, t0, torch.zeros(1, 2, 48, device=dev), i0, 8, D)
    assert kept.shape == (0, 2, 8) and lens.shape == (0,)
    assert paged_gather_q4(*pools, t0, i0, D, 5)[0].shape == (0, 5, 2, D)
    n, none = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, 0, dtype=torch.int32, device=dev)
    out = paged_decode_q4(torch.ones(3, 4, D, dtype=BF, device=dev), *pools, none, n, 1.0)
    assert not out.any()
    assert paged_gather_q4(*pools, none, n, D, 0)[0].shape == (3, 0, 2, D)
    w = torch.ones(3, 2, 16, device=dev)
    kept, lens = paged_evict_q4(*pools, none, n, torch.zeros(3, 1, dtype=torch.int32, device=dev), w, n - 1, 4, D)
    assert (kept == -1).all() and not lens.any() and (w == 1).all()


def test_evict_shared_source(dev):
    """Two sequences over the same blocks (a shared prompt) are cut by their own weights."""
    ks, vs, pools, tables, n, ids = cache([80], 1, 64, dev, extra=4)
    new = ids[-4:].view(2, 2).int().to(dev)
    w = torch.rand(2, 1, 80)
    kept, lens = paged_evict_q4(*pools, tables.repeat(2, 1), n.repeat(2), new, w.clone().to(dev),
                                torch.tensor([1, 0], dtype=torch.int32, device=dev), 32, 64)
    for b in range(2):
        assert kept[b, 0].tolist() == chosen(w[1 - b, 0].tolist(), 80, 32, 0, 0)


def test_evict_bad_index(dev):
    _, _, pools, tables, n, ids = cache([40], 1, 64, dev, extra=2)
    new, row = ids[-2:].view(1, 2).int().to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    w = torch.rand(1, 1, 48, device=dev)
    index_error(dev, lambda: paged_evict_q4(*pools, tables, n, new, w, row + 1, 20, 64))
    index_error(dev, lambda: paged_evict_q4(*pools, tables, n, new, w, row - 1, 20, 64))
    index_error(dev, lambda: paged_evict_q4(*pools, tables, n, new + 100, w, row, 20, 64))
    index_error(dev, lambda: paged_evict_q4(*pools, tables + 100, n, new, w, row, 20, 64))


# ---------------------------------------------------------------- refusals
def test_refusals(dev):
    D = 64
    pools = [torch.zeros(4, 2, q4_block_bytes(D), dtype=torch.uint8, device=dev) for _ in range(2)]
    x = torch.zeros(3, 2, D, dtype=BF, device=dev)
    i3, t, n = (torch.zeros(*s, dtype=torch.int32, device=dev) for s in ((3,), (3, 1), (3,)))
    q = torch.zeros(3, 4, D, dtype=BF, device=dev)
    w = torch.zeros(3, 2, 16, device=dev)
    for call in (
        lambda: q4_block_bytes(96),
        lambda: paged_write_q4(x[..., :48].contiguous(), x[..., :48].contiguous(), *pools, i3, i3),
        lambda: paged_write_q4(x[:, :1], x[:, :1], *pools, i3, i3),
        lambda: paged_write_q4(x, x[:2], *pools, i3, i3),
        lambda: paged_write_q4(x, x, *pools, i3.long(), i3),
        lambda: paged_write_q4(x, x, *pools, i3[:2], i3),
        lambda: paged_write_q4(x, x, pools[0].float(), pools[1], i3, i3),
        lambda: paged_write_q4(x, x, pools[0][:2], pools[1], i3, i3),
        lambda: paged_read_q4(*pools, i3, i3, 128),
        lambda: paged_gather_q4(*pools, t, n[:2], D, 16),
        lambda: paged_decode_q4(q[:, :3], *pools, t, n, 1.0),
        lambda: paged_decode_q4(torch.zeros(3, 34, D, dtype=BF, device=dev), *pools, t, n, 1.0),
        lambda: paged_decode_q4(q, *pools, t, n[:2], 1.0),
        lambda: paged_decode_q4(q, *pools, t.long(), n, 1.0),
        lambda: paged_decode_q4(q, *pools, t, n, 1.0, 0.0, 0, w),
        lambda: paged_decode_q4(q, *pools, t, n, 1.0, 0.0, 0, w.double(), i3),
        lambda: paged_decode_q4(q, *pools, t, n, 1.0, 0.0, 0, w[:, :1].contiguous(), i3),
        lambda: paged_evict_q4(*pools, t, n, t, w, i3, 0, D),
        lambda: paged_evict_q4(*pools, t, n, t, w, i3, 4, D, recent=3, sink=2),
        lambda: paged_evict_q4(*pools, t, n, t, w, i3, 4, D, recent=-1),
        lambda: paged_evict_q4(*pools, t, n, t, w, i3, 17, D),
        lambda: paged_evict_q4(*pools, t, n, t[:2], w, i3, 16, D),
    ):
        with pytest.raises(ValueError if dev == "cpu" else (ValueError, RuntimeError)):
            call()


@pytest.mark.gpu
def test_refuses_other_devices():
    D = 64
    pools = [torch.zeros(4, 2, q4_block_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    t, n = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 4, D, dtype=BF, device="cuda")
    for call in (lambda: paged_decode_q4(q, *pools, t, n.cpu(), 1.0), lambda: paged_decode_q4(q.cpu(), *pools, t, n, 1.0),
                 lambda: paged_decode_q4(q, pools[0], pools[1].cpu(), t, n, 1.0),
                 lambda: paged_decode_q4(q, *pools, t, n, 1.0, window=1 << 32)):
        with pytest.raises(RuntimeError):
            call()


# ---------------------------------------------------------------- together, streams, graphs
def test_serving_run(dev):
    """Prompt rows stored, steps decoded with accumulated weights, the caches cut, and decoded again."""
    torch.manual_seed(3)
    lens, Hkv, G, D, keep, steps = [50, 23], 2, 4, 64, 32, 12
    ks, vs, pools, tables, n, ids = cache([m + steps for m in lens], Hkv, D, dev, extra=2 * 3)
    new = torch.cat([ids[-4:].view(2, 2), ids[-6:-4].view(2, 1)], 1).int().to(dev)
    w = torch.zeros(2, Hkv, 64, device=dev)
    w_rows = torch.tensor([1, 0], dtype=torch.int32, device=dev)
    acc = [torch.zeros(Hkv, m + steps, dtype=F64) for m in lens]
    for s in range(steps):
        ctx = torch.tensor([m + s + 1 for m in lens], dtype=torch.int32, device=dev)
        k, v = rows(2, Hkv, D), rows(2, Hkv, D)
        at = ctx - 1
        paged_write_q4(k.to(dev), v.to(dev), *pools, tables.gather(1, (at // 16).long()[:, None])[:, 0].contiguous(),
                       at % 16)
        q = torch.randn(2, Hkv * G, D).to(BF).to(dev)
        out = paged_decode_q4(q, *pools, tables, ctx, 0.125, 0.0, 0, w, w_rows)
        for b, m in enumerate(lens):
            ks[b][m + s], vs[b][m + s] = stored(k[b])[3], stored(v[b])[3]
            o, p, a = attention(q[b], ks[b][:m + s + 1], vs[b][:m + s + 1], 0.125, 0.0, 0)
            check_decode(out[b], o, a)
            acc[b][:, :m + s + 1] += p
    for b in range(2):
        assert ((w[w_rows[b], :, :lens[b] + steps].cpu().to(F64) - acc[b]).abs() <= 2 ** -14 * acc[b] + 1e-12).all()
    before = w.clone().cpu()
    kept, left = paged_evict_q4(*pools, tables, ctx, new, w, w_rows, keep, D, recent=8, sink=1)
    assert left.tolist() == [keep, keep]
    q = torch.randn(2, Hkv * G, D).to(BF).to(dev)
    out = paged_decode_q4(q, *pools, new, left, 0.125, 0.0, 0, w, w_rows)
    for b, m in enumerate(lens):
        cut = [[x[b][chosen(before[w_rows[b], h].tolist(), m + steps, keep, 1, 8), h] for h in range(Hkv)]
               for x in (ks, vs)]
        o, _, a = attention(q[b], torch.stack(cut[0], 1), torch.stack(cut[1], 1), 0.125, 0.0, 0)
        check_decode(out[b], o, a)


@pytest.mark.gpu
def test_captured_and_replayed():
    """One graph holds write, decode with weights and eviction; replays follow the inputs' new contents, two graphs
    do not disturb each other, and an eager call between them changes nothing."""
    dev, Hkv, G, D = "cuda", 2, 4, 128
    ks, vs, pools, tables, n, ids = cache([700, 90], Hkv, D, dev, extra=8)
    new = ids[-8:].view(2, 4).int().to(dev)
    q = torch.randn(2, Hkv * G, D, device=dev).to(BF)
    k_new, v_new = torch.randn(2, Hkv, D, device=dev).to(BF), torch.randn(2, Hkv, D, device=dev).to(BF)
    at = n - 1
    slot, off = tables.gather(1, (at // 16).long()[:, None])[:, 0].contiguous(), at % 16
    w, w_rows = torch.zeros(2, Hkv, 720, device=dev), torch.arange(2, dtype=torch.int32, device=dev)

    def step():
        paged_write_q4(k_new, v_new, *pools, slot, off)
        return paged_decode_q4(q, *pools, tables, n, 0.1, 0.0, 0, w, w_rows)

    def cut():
        return paged_evict_q4(*pools, tables, n, new, w, w_rows, 64, D, recent=4)

    step()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = step()
    with torch.cuda.graph(g2):
        out2 = step()
        kept, left = cut()
    for trial in range(3):
        for t in (q, k_new, v_new):
            t.copy_(torch.randn_like(t.float()))
        w.zero_()
        g1.replay()
        g2.replay()
        eager = paged_decode_q4(q, *pools, tables, n, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(out1, out2) and torch.equal(out1, eager)
        for b, m in enumerate((700, 90)):
            ks[b][m - 1], vs[b][m - 1] = stored(k_new[b])[3], stored(v_new[b])[3]
            o, p, a = attention(q[b], ks[b], vs[b], 0.1, 0.0, 0)
            check_decode(out1[b], o, a)
            for h in range(Hkv):
                assert sorted(kept[b, h].tolist()) == kept[b, h].tolist() and left[b] == 64
                # what was dropped weighed no more than what was kept (twice the weight: two replays)
                dropped = torch.ones(m, dtype=torch.bool)
                dropped[kept[b, h].long().cpu()] = False
                mine = [t for t in kept[b, h].tolist() if t < m - 4]
                assert 2 * p[h][dropped].max() <= w[b, h, :64][:len(mine)].min() * (1 + 2 ** -12)


@pytest.mark.gpu
def test_other_stream():
    ks, vs, pools, tables, n, _ = cache([400, 33], 2, 64, "cuda")
    q = torch.randn(2, 8, 64).to(BF).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = paged_decode_q4(q, *pools, tables, n, 0.125)
    side.synchronize()
    assert torch.equal(out, paged_decode_q4(q, *pools, tables, n, 0.125))


@pytest.mark.gpu
def test_same_result_every_time():
    _, _, pools, tables, n, _ = cache([3000, 100, 1700], 2, 128, "cuda")
    q = torch.randn(3, 8, 128).to(BF).cuda()
    w_rows = torch.arange(3, dtype=torch.int32, device="cuda")

    def once():
        w = torch.zeros(3, 2, tables.shape[1] * 16, device="cuda")
        return paged_decode_q4(q, *pools, tables, n, 0.1, 0.0, 0, w, w_rows), w

    first = once()
    for _ in range(5):
        again = once()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
