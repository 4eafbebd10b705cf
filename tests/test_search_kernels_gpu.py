"""The kernels of a search over beams and of forked sequences against plain 64-bit forms: the choice of continuations, the copies of pages and
states, attention behind shared pages."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOWEST = -3.4028234663852886e38


def ops():
    from ithaca_b200.csrc import ops as o
    return o


def gen(seed):
    return torch.Generator().manual_seed(seed)


# -- the choice of continuations -------------------------------------------------------------------------------------------
def plain_scores(logits, sums):
    """Scores [R, K * V] in 64 bits; -inf where there is no candidate."""
    R, K = sums.shape
    l = logits.double().view(R, K, -1)
    l = torch.where(torch.isnan(l), -math.inf, l)
    infinite = l == math.inf
    share = infinite.any(-1, keepdim=True)
    l = torch.where(share, torch.where(infinite, 0.0, -math.inf), l)
    top = l.amax(-1, keepdim=True)
    lse = torch.where(top > -math.inf, top + (l - torch.where(top > -math.inf, top, 0.0)).exp().sum(-1, keepdim=True).log(), 0.0)
    c = sums.double()[..., None]
    s = torch.where((c > -math.inf) & (l > -math.inf), c + (l - lse), -math.inf)
    return s.flatten(1)


# A float exponential is off by up to 2 units in the last place (2^-22), a thread adds 32 of them in float (32 x 2^-24), and the argument's
# rounding is 2^-24 of it, weighted by the exponential: below 20 x 2^-24 on average.  All relative to the sum, so absolute in its logarithm.
LSE = 2 ** -22 + 32 * 2 ** -24 + 20 * 2 ** -24


def check_select(logits, sums, n):
    got_s, got_b, got_v = (t.cpu() for t in ops().beam_select(logits.to(DEV), sums.to(DEV), n))
    (R, K), V = sums.shape, logits.shape[1]
    want = plain_scores(logits, sums)
    assert got_s.shape == got_b.shape == got_v.shape == (R, n) and got_b.dtype == got_v.dtype == torch.int32
    for r in range(R):
        order = torch.sort(want[r], descending=True, stable=True)
        best = [float(x) for x in order.values[:n] if x > -math.inf]
        at = [int(b) * V + int(v) for b, v in zip(got_b[r], got_v[r])]
        assert len(set(at[:len(best)])) == len(best)
        for i in range(n):
            if i >= len(best):
                assert got_s[r, i] == -math.inf and got_b[r, i] == -1 and got_v[r, i] == -1
                continue
            assert 0 <= got_b[r, i] < K and 0 <= got_v[r, i] < V
            # what was chosen at this rank is as good as the best there, to the errors of two sums
            assert abs(float(want[r, at[i]]) - best[i]) <= 2 * LSE, (r, i, at[i], int(order.indices[i]))
            assert abs(float(got_s[r, i]) - float(want[r, at[i]])) <= LSE + abs(best[i]) * 2 ** -24 + 1e-30
            if i and got_b[r, i] == got_b[r, i - 1]:                        # within a beam the order is the logits' own
                x, y = logits[r * K + got_b[r, i], got_v[r, i - 1]], logits[r * K + got_b[r, i], got_v[r, i]]
                assert x > y or (x == y and got_v[r, i - 1] < got_v[r, i])
    return got_s, got_b, got_v


SIZES = [(1, 1, 1, 1), (1, 1, 5, 3), (1, 2, 3, 8), (2, 3, 17, 6), (3, 4, 1000, 8), (5, 5, 8192, 10), (1, 16, 8193, 32), (2, 2, 50257, 4), (1, 4, 128256, 8), (7, 1, 32000, 1),
         (1, 16, 300001, 32), (33, 2, 256, 5)]


@pytest.mark.parametrize("R,K,V,n", SIZES)
def test_select_on_logits(R, K, V, n):
    g = gen(V + n)
    check_select(torch.randn((R * K, V), generator=g) * 3, torch.rand((R, K), generator=g) * -20, n)


@pytest.mark.parametrize("kind", ["constant", "few values", "masked", "lowest", "one left", "none left", "nan", "infinite", "rising", "falling", "peaked"])
@pytest.mark.parametrize("R,K,V,n", [(2, 3, 1001, 6), (1, 5, 20000, 32)])
def test_select_on_rows_that_are_not_ordinary(kind, R, K, V, n):
    g = gen(V)
    l = torch.randn((R * K, V), generator=g) * 3
    sums = torch.rand((R, K), generator=g) * -20
    if kind == "constant":
        l = torch.full_like(l, 0.25)
    elif kind == "few values":
        l = (l / 2).round() * 2
    elif kind == "masked":
        l[:, torch.rand(V, generator=g) < 0.995] = -math.inf
    elif kind == "lowest":
        l[:, torch.rand(V, generator=g) < 0.999] = LOWEST
    elif kind in ("one left", "none left"):
        l[0] = -math.inf
        l[1] = -math.inf
        if kind == "one left":
            l[1, V - 1] = -5.0
    elif kind == "nan":
        l[torch.rand((R * K, V), generator=g) < 0.01] = math.nan
        l[1] = math.nan
    elif kind == "infinite":
        l[0, 7] = l[0, 500] = l[1, V - 1] = math.inf
    elif kind == "rising":
        l = l.sort(1).values
    elif kind == "falling":
        l = l.sort(1, descending=True).values
    else:
        l[:, 321] += 60.0
    check_select(l, sums, n)


@pytest.mark.parametrize("kind", ["random", "few values", "rising", "signed zeros"])
@pytest.mark.parametrize("R,K,V,n", [(1, 16, 1000, 32), (3, 8, 1001, 16), (2, 16, 1024, 32), (2, 10, 4096, 32), (1, 1, 1000, 32), (5, 2, 33, 32), (2, 16, 2, 32)])
def test_select_from_few_tiles(kind, R, K, V, n):
    """Fewer stretches of 1,024 logits than results, or hardly more: many of each one's logits are candidates."""
    l = torch.randn((R * K, V), generator=gen(V + n)) * 3
    if kind == "few values":
        l = (l / 2).round() * 2
    elif kind == "rising":
        l = l.sort(1).values
    elif kind == "signed zeros":
        l = torch.where(l > 0, 0.0, -0.0)
    check_select(l, torch.rand((R, K), generator=gen(n)) * -2, n)


def test_equal_candidates_come_by_beam_and_token():
    """Equal beams (odd vocabularies: their rows start on different alignments) with equal sums: every rank has an exact tie."""
    for V, n in ((1001, 8), (20003, 32), (128256, 16)):
        row = torch.randn((1, V), generator=gen(V)).repeat(4, 1)
        s, b, v = ops().beam_select(row.to(DEV), torch.full((1, 4), -3.0, device=DEV), n)
        top = torch.sort(row[0], descending=True, stable=True).indices
        assert b[0].tolist() == [i % 4 for i in range(n)]
        assert v[0].tolist() == [int(top[i // 4]) for i in range(n)]
    flat = torch.zeros((3, 70000), device=DEV)
    s, b, v = ops().beam_select(flat, torch.zeros((1, 3), device=DEV), 20)
    assert b[0].tolist() == [0] * 20 and v[0].tolist() == list(range(20))


def test_scores_below_the_range_of_a_float_are_no_candidates():
    """Tokens masked by the type's lowest value, of beams whose sums are such values already."""
    l = torch.full((4, 2000), LOWEST)
    l[0, 5] = l[1, 7] = l[2, 1999] = 1.0
    s, b, v = (t.cpu() for t in ops().beam_select(l.to(DEV), torch.tensor([[-1.0, -2.0], [LOWEST, LOWEST]], device=DEV), 4))
    # beam 0's and 1's own tokens, then beam 0's first masked ones; the second request: one token costs nothing, all others two lowest values
    assert b.tolist() == [[0, 1, 0, 0], [0, 1, 1, 1]] and v.tolist() == [[5, 7, 0, 1], [1999, 0, 1, 2]]
    # (a row of nothing but the lowest value is an even distribution)
    assert s[0].tolist() == pytest.approx([-1.0, -2.0, LOWEST, LOWEST]) and s[1].tolist() == pytest.approx([LOWEST] * 4)
    s, b, v = (t.cpu() for t in ops().beam_select(l[:3].to(DEV), torch.tensor([[LOWEST, LOWEST, LOWEST]], device=DEV), 5))
    assert b.tolist() == [[0, 1, 2, -1, -1]] and v.tolist() == [[5, 7, 1999, -1, -1]] and s[0, 3:].tolist() == [-math.inf] * 2


@pytest.mark.parametrize("V", [1500, 1501, 5000])
def test_sums_beside_which_logits_do_not_count(V):
    """Beams that all have the type's lowest value, or something as large, as their sum: in 64 bits every score is the same, and the first tokens are chosen."""
    l = torch.randn((2, V), generator=gen(V))
    for c in (LOWEST, -1e30):
        s, b, v = (t.cpu() for t in ops().beam_select(l.to(DEV), torch.full((1, 2), c, device=DEV), 8))
        assert s[0].tolist() == pytest.approx([c] * 8) and b[0].tolist() == [0] * 8 and v[0].tolist() == list(range(8))
    s, b, v = (t.cpu() for t in ops().beam_select(l.to(DEV), torch.tensor([[LOWEST, -1.0]], device=DEV), 8))
    assert b[0].tolist() == [1] * 8 and v[0].tolist() == torch.sort(l[1], descending=True).indices[:8].tolist()


def test_dead_beams_are_left_alone():
    g = gen(3)
    l = torch.randn((8, 501), generator=g)
    sums = torch.tensor([[-math.inf, -2.0, -math.inf, -1.0], [-math.inf] * 4])
    sums[0, 2] = math.nan
    l[0], l[2] = math.nan, math.inf
    check = torch.where(torch.isnan(sums), -math.inf, sums)
    s, b, v = ops().beam_select(l.to(DEV), sums.to(DEV), 8)
    assert set(b[0].tolist()) <= {1, 3} and b[1].tolist() == [-1] * 8 and v[1].tolist() == [-1] * 8
    check_select(torch.where(torch.isnan(l) | (l == math.inf), 0.0, l), check, 8)


def test_select_reads_rows_with_a_stride_and_writes_where_it_is_told():
    g = gen(5)
    wide = torch.randn((6, 900), generator=g)
    sums = torch.rand((2, 3), generator=g) * -4
    for lo, hi in ((0, 800), (1, 800), (3, 64), (7, 900)):
        view = wide.to(DEV)[:, lo:hi]
        assert not view.is_contiguous()
        out = torch.full((3, 2, 6), 77, dtype=torch.int32, device=DEV)
        got = ops().beam_select(view, sums.to(DEV), 6, out=out)
        want = ops().beam_select(wide[:, lo:hi].contiguous().to(DEV), sums.to(DEV), 6)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(out[1], want[1]) and torch.equal(out[0].view(torch.float32), want[0])


def test_select_on_another_stream_and_replayed():
    g = gen(6)
    l, sums = (torch.randn((8, 33000), generator=g)).to(DEV), (torch.rand((2, 4), generator=g) * -9).to(DEV)
    want = [t.clone() for t in ops().beam_select(l, sums, 8)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in ops().beam_select(l, sums, 8)]
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.zeros((3, 2, 8), dtype=torch.int32, device=DEV)
    with torch.cuda.graph(graph):
        ops().beam_select(l, sums, 8, out=out)
    for shift in (0, 1):
        rolled = l.roll(shift * 4, 0).clone()
        other = [t.clone() for t in ops().beam_select(rolled, sums, 8)]
        l.copy_(rolled)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0].view(torch.float32), other[0]) and torch.equal(out[1], other[1]) and torch.equal(out[2], other[2])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_select_refuses():
    o = ops()
    l, s = torch.zeros((4, 10), device=DEV), torch.zeros((2, 2), device=DEV)
    for bad in (lambda: o.beam_select(l.double(), s, 2), lambda: o.beam_select(l, s.half(), 2), lambda: o.beam_select(l.cpu(), s, 2), lambda: o.beam_select(l, s.cpu(), 2),
                lambda: o.beam_select(l, s, 0), lambda: o.beam_select(l, s, 33), lambda: o.beam_select(l[:3], s, 2), lambda: o.beam_select(l.t(), s, 2),
                lambda: o.beam_select(torch.zeros((17, 10), device=DEV), torch.zeros((1, 17), device=DEV), 2), lambda: o.beam_select(l[:, :0], s, 2),
                lambda: o.beam_select(l[:0], s[:0], 2), lambda: o.beam_select(l, s, 2, out=torch.zeros((3, 2, 3), dtype=torch.int32, device=DEV)),
                lambda: o.beam_select(l[:1].expand(4, 10), s, 2)):
        with pytest.raises(o.KernelError):
            bad()
    both = torch.zeros(200, device=DEV)                             # results may not be written where the inputs are read
    for logits, scores, at in ((both[:40].view(4, 10), s, 30), (l, both[40:44].view(2, 2), 36), (l, both[40:44].view(2, 2), 40)):
        out = both[at:at + 12].view(torch.int32).view(3, 2, 2)
        with pytest.raises(o.KernelError, match="overlap"):
            o.beam_select(logits, scores, 2, out=out)
    o.beam_select(both[:40].view(4, 10), both[40:44].view(2, 2), 2, out=both[44:56].view(torch.int32).view(3, 2, 2))


# -- copies ----------------------------------------------------------------------------------------------------------------
def plain_copy(t, src, dst, positions):
    t = t.clone()
    old = t.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        if positions is None:
            t[:, d] = old[:, s]
        else:
            t[:, d, :, :positions[i]] = old[:, s, :, :positions[i]]
    return t


@pytest.mark.parametrize("shape,dtype,whole", [((2, 9, 3, 64, 16), torch.bfloat16, False), ((3, 9, 2, 64, 33), torch.bfloat16, False), ((1, 9, 1, 64, 5), torch.float32, False),
                                               ((5, 9, 4, 64), torch.float32, False), ((2, 9, 8, 64, 128), torch.bfloat16, False), ((3, 9, 7), torch.float32, True),
                                               ((2, 9, 2, 4099), torch.float32, True), ((2, 9, 3), torch.bfloat16, True), ((4, 9, 2, 16, 64, 64), torch.float32, True),
                                               ((2, 9, 5), torch.int32, True)])
def test_copies_of_pages_and_states(shape, dtype, whole):
    g = gen(sum(shape))
    t = (torch.randn(shape, generator=g) * 100).to(dtype)
    src, dst = [4, 4, 4, 0, 7, 7], [1, 8, 2, 3, 5, 6]
    for positions in ([None] if whole else [[64] * 6, [1] * 6, [0, 5, 5, 63, 64, 17]]):
        d = t.to(DEV)
        ops().copy_rows([(d, src, dst, positions)])
        assert torch.equal(d.cpu(), plain_copy(t, src, dst, positions))


def test_copies_in_several_tensors_and_long_lists():
    """Lists beyond what one launch carries, several tensors with lists of their own, a fan of destinations wider than a move carries."""
    g = gen(1)
    k, v = torch.randn((2, 500, 2, 64, 16), generator=g).to(torch.bfloat16), torch.randn((2, 500, 2, 64, 24), generator=g).to(torch.bfloat16)
    st = [torch.randn((3, 40, 11), generator=g) for _ in range(20)]
    order = torch.randperm(500, generator=g).tolist()
    src, dst = [order[0]] * 30 + order[1:220], order[220:469]
    rows = torch.randint(0, 65, (249,), generator=g).tolist()
    slots = torch.randperm(40, generator=g).tolist()
    gpu = [t.to(DEV) for t in (k, v, *st)]
    ops().copy_rows([(gpu[0], src, dst, rows), (gpu[1], src, dst, rows)] + [(t, slots[:i], slots[20:20 + i], None) for i, t in enumerate(gpu[2:])])
    want = [plain_copy(k, src, dst, rows), plain_copy(v, src, dst, rows)] + [plain_copy(t, slots[:i], slots[20:20 + i], None) for i, t in enumerate(st)]
    for a, b in zip(gpu, want):
        assert torch.equal(a.cpu(), b)
    ops().copy_rows([])
    ops().copy_rows([(gpu[0], [], [], [])])
    assert torch.equal(gpu[0].cpu(), want[0])


def test_copies_within_views():
    """A layer's own part of a cache, rows with a stride, one entry of many."""
    base = torch.randn((4, 10, 2, 64, 8), generator=gen(2))
    d = base.to(DEV)
    ops().copy_rows([(d[1:2], [3], [5], [9]), (d[2:, 1::2], [0, 0], [1, 4], [64, 64])])
    want = base.clone()
    want[1:2] = plain_copy(base[1:2], [3], [5], [9])
    want[2:, 1::2] = plain_copy(base[2:, 1::2], [0, 0], [1, 4], [64, 64])
    assert torch.equal(d.cpu(), want)


def test_a_captured_copy_keeps_its_lists():
    d = torch.arange(60, dtype=torch.float32, device=DEV).view(1, 20, 3).clone()
    ops().copy_rows([(d, [0], [1], None)])
    graph, src, dst = torch.cuda.CUDAGraph(), [2, 2], [3, 4]
    with torch.cuda.graph(graph):
        ops().copy_rows([(d, src, dst, None)])
    src[:], dst[:] = [9, 9], [0, 1]
    d[0, 2] = 5.0
    graph.replay()
    torch.cuda.synchronize()
    assert d[0, 3].tolist() == d[0, 4].tolist() == [5.0] * 3 and d[0, 0].tolist() == [0.0, 1.0, 2.0]


def test_copies_are_refused_whole():
    o = ops()
    t = torch.arange(2 * 6 * 2 * 64 * 4, dtype=torch.float32, device=DEV).view(2, 6, 2, 64, 4)
    keep = t.clone()
    for bad in ([(t, [0], [6], None)], [(t, [-1], [2], None)], [(t, [0, 1], [2, 2], None)], [(t, [0, 1], [1, 2], None)], [(t, [0], [0], None)], [(t, [0], [1], [65])],
                [(t, [0], [1], [-1])], [(t, [0, 1], [2], None)], [(t, [0], [1], [])], [(t.cpu(), [0], [1], None)], [(t.transpose(3, 4), [0], [1], None)],
                [(t[0, 0, 0], [0], [1], [3])], [(t, [1], [2], None), (t, [3], [4], None)], [(t, [1], [2], None), (t[1:], [3], [4], None)],
                [(t, [1], [2], None), (torch.zeros((1, 3), dtype=torch.int8, device=DEV), [0], [1], None)]):
        with pytest.raises(o.KernelError):
            o.copy_rows(bad)
    assert torch.equal(t, keep)


# -- attention behind shared pages -----------------------------------------------------------------------------------------
def layout(members, shared, lens, seed, extra=3):
    """A block table in which every group's members name the same first pages, all pages in random order."""
    owns = [-(-n // 64) for n in lens]
    total = sum(shared) + sum(owns) + extra
    order = torch.randperm(total, generator=gen(seed)).tolist()
    table, b = torch.full((len(lens), max(1, max(owns))), -1, dtype=torch.int32), 0
    for m, s in zip(members, shared):
        first, order = order[:s], order[s:]
        for _ in range(m):
            rest, order = order[:max(0, owns[b] - s)], order[max(0, owns[b] - s):]
            table[b, :owns[b]] = torch.tensor((first + rest)[:owns[b]], dtype=torch.int32)
            b += 1
    return table, total


def run_shared(nh, nkv, hd, members, shared, lens, seed=0, softcap=0.0, sink=False, scale=None, garbage=True, bounds=None):
    from ithaca_b200.csrc import attention_bf16
    g = gen(seed + hd)
    table, total = layout(members, shared, lens, seed)
    B, scale = len(lens), scale or hd ** -0.5
    q = torch.randn((B, nh * hd), generator=g).to(torch.bfloat16)
    k, v = ((torch.randn((total, nkv, 64, hd), generator=g) * f).to(torch.bfloat16) for f in (1.5, 1.0))
    if garbage:                                                     # behind a sequence's last key anything may lie
        for b, n in enumerate(lens):
            if n % 64:
                k[table[b, n // 64], :, n % 64:] = math.nan
                v[table[b, n // 64], :, n % 64:] = math.inf
    per = [s for m, s in zip(members, shared) for _ in range(m)]
    starts = torch.tensor([0] + torch.tensor(members).cumsum(0).tolist(), dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    owns = [-(-n // 64) - s for n, s in zip(lens, per)]
    got = attention_bf16.decode_shared(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV), starts.to(DEV),
                                       torch.tensor(per, dtype=torch.int32, device=DEV), len(members), max(members), *(bounds or (max(shared), max(owns))), nh, scale, status,
                                       softcap=softcap, sink=sink.to(DEV) if torch.is_tensor(sink) else sink).cpu().double().view(B, nh, hd)
    assert status.item() == 0
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        pages = table[b, :-(-n // 64)].long()
        kb, vb = (t[pages].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :n].repeat_interleave(nh // nkv, 0) for t in (k, v))
        s = torch.einsum("hd,hjd->hj", q[b].double().view(nh, hd), kb) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        top = s.amax(-1, keepdim=True)
        sinks = sink.double()[:, None] if torch.is_tensor(sink) else torch.zeros((nh, 1), dtype=torch.float64)
        if torch.is_tensor(sink) or sink:
            top = torch.maximum(top, sinks)
        p = (s - top).exp()
        total_p = p.sum(-1, keepdim=True) + ((sinks - top).exp() if torch.is_tensor(sink) or sink else 0.0)
        want = torch.einsum("hj,hjd->hd", p, vb) / total_p
        size = torch.einsum("hj,hjd->hd", p, vb.abs()) / total_p
        # a probability and the result are rounded to bfloat16 (2^-8 each); a score is a float sum of hd products (about hd 2^-24 of their sizes, below
        # 2^-14 here), which the exponential passes on; the cap's tanh is off by up to 2^-11 of the cap
        tol = 2 ** -8 * (size + want.abs()) + 2 ** -14 * size + (softcap * 2 ** -10 * size if softcap else 0.0)
        assert torch.isfinite(got[b]).all()
        assert ((got[b] - want).abs() <= tol).all(), (b, ((got[b] - want).abs() / tol).max())


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (32, 8, 64), (8, 8, 16), (6, 2, 48), (40, 40, 128), (20, 1, 64), (6, 3, 80), (4, 2, 256), (64, 8, 128)])
@pytest.mark.parametrize("members,shared,lens", [
    ([4], [2], [129, 129, 129, 129]),                               # a tail of one key
    ([1], [0], [1]),                                                 # one sequence, one key
    ([3, 1, 2], [5, 0, 1], [321, 330, 450, 70, 65, 128]),            # unequal groups, one alone, a tail that fills its page
    ([2, 2], [0, 3], [5, 64, 200, 256]),                             # a group that shares nothing yet
    ([16], [1], [65 + 3 * i for i in range(16)]),
    ([2, 3], [1, 0], [64, 100, 0, 1, 63]),                           # nothing behind the shared page; a sequence without keys
])
def test_attention_behind_shared_pages(nh, nkv, hd, members, shared, lens):
    run_shared(nh, nkv, hd, members, shared, lens, seed=len(lens))


@pytest.mark.parametrize("nh,nkv,hd", [(40, 40, 128), (64, 64, 64), (80, 1, 64), (40, 1, 128), (20, 1, 64), (4, 4, 16), (24, 2, 96), (148, 148, 32)])
@pytest.mark.parametrize("seed", range(4))
def test_many_groups_of_all_sizes(nh, nkv, hd, seed):
    """Runs of pages that end inside tiles, cover several, begin among shared pages or among a member's own; more heads per kv head than a tile has rows; groups
    of more members than fit one."""
    r = random.Random(seed)
    members = [r.choice([1, 1, 2, 3, 7, 20]) for _ in range(r.choice([1, 5, 14]))]
    shared = [r.choice([0, 1, 2, 9]) if m > 1 else r.choice([0, 0, 3]) for m in members]
    lens = [s * 64 + r.choice([0, 1, 3, 64, 65, 200, r.randint(0, 700)]) for m, s in zip(members, shared) for _ in range(m)]
    run_shared(nh, nkv, hd, members, shared, lens, seed=seed)


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,members", [(64, 8, 16, [3] * 14), (40, 40, 64, [2, 1, 3] * 11), (20, 1, 256, [8] * 17), (6, 3, 80, [5, 1, 2] * 56), (50, 10, 48, [17] * 3), (32, 8, 128, [1] * 80)])
def test_more_sequences_and_heads_than_blocks_at_a_time(nh, nkv, hd, members, sink):
    """The join by groups of a block: its last block of heads is not always full."""
    r = random.Random(nh)
    shared = [r.randint(0, 3) if m > 1 else 0 for m in members]
    lens = [64 * s + r.choice([0, 1, 40, 64, 65, 150]) for m, s in zip(members, shared) for _ in range(m)]
    assert len(lens) * nh > 17 * 148
    run_shared(nh, nkv, hd, members, shared, lens, seed=nh + hd, sink=torch.randn(nh, generator=gen(nh)) if sink else False)


def test_bounds_that_are_too_small_cost_time_only():
    for bounds in ((1, 1), (0, 0), (3, 2), (100, 100)):
        run_shared(8, 2, 64, [3, 2], [7, 4], [449, 500, 700, 257, 300], seed=4, bounds=bounds)


def test_cap_sink_and_scale():
    run_shared(8, 2, 64, [3, 2], [3, 4], [200, 211, 340, 257, 300], seed=6, softcap=20.0, scale=0.3)
    run_shared(8, 2, 64, [3, 2], [3, 4], [200, 211, 340, 257, 300], seed=7, sink=True)
    run_shared(8, 2, 64, [3, 2], [3, 4], [200, 211, 340, 257, 0], seed=8, sink=torch.randn(8, generator=gen(9)) * 3)


def test_a_group_of_everything_and_long_prompts():
    run_shared(32, 8, 128, [8, 8], [130, 33], [130 * 64 + 70 + i for i in range(8)] + [33 * 64 + 1] * 8, seed=10)


@pytest.mark.parametrize("hd", [48, 64, 128])
def test_a_value_that_one_of_a_group_has_stays_with_it(hd):
    """Infinite and undefined keys and values in a member's own pages: the others' results are those of a call without them, to the last bit."""
    from ithaca_b200.csrc import attention_bf16
    g = gen(hd)
    lens, shared = [200, 260, 130, 64 * 5], 2
    table, total = layout([4], [shared], lens, 3)
    q = torch.randn((4, 4 * hd), generator=g).to(torch.bfloat16).to(DEV)
    k, v = (torch.randn((total, 2, 64, hd), generator=g).to(torch.bfloat16) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    run = lambda k, v: attention_bf16.decode_shared(q, k.to(DEV), v.to(DEV), ints(lens), table.to(DEV), ints([0, 4]), ints([shared] * 4), 1, 4, 2, 3, 4, hd ** -0.5, None)
    want = run(k, v)
    for t, x in ((v, math.inf), (v, math.nan), (k, math.nan), (k, -math.inf)):
        spoilt = t.clone()
        spoilt[int(table[1, 3]), :, 5] = x
        got = run(*((k, spoilt) if t is v else (spoilt, v)))
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
        assert not torch.equal(got[1], want[1])


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("hd", [64, 48])
def test_a_sequence_without_keys_takes_nothing_from_its_neighbours(hd, sink):
    """A place of a padded batch stands in a group whose shared pages hold infinite values: zeros."""
    from ithaca_b200.csrc import attention_bf16
    g = gen(hd)
    lens = [200, 0, 130]
    table, total = layout([3], [2], [200, 130, 130], 3)
    q = torch.randn((3, 4 * hd), generator=g).to(torch.bfloat16).to(DEV)
    k, v = (torch.randn((total, 2, 64, hd), generator=g).to(torch.bfloat16) for _ in range(2))
    v[int(table[0, 0]), :, 5, 3], v[int(table[0, 1]), :, 7, 4] = math.inf, math.nan
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    got = attention_bf16.decode_shared(q, k.to(DEV), v.to(DEV), ints(lens), table.to(DEV), ints([0, 3]), ints([2, 2, 2]), 1, 3, 2, 2, 4, hd ** -0.5, None, sink=sink).view(3, 4, hd)
    assert (got[1] == 0).all() and (got[[0, 2]][..., 3] == math.inf).all() and torch.isnan(got[[0, 2]][..., 4]).all()
    assert torch.isfinite(got[[0, 2]][..., 5:]).all()


def test_pages_outside_the_pool_are_not_followed():
    from ithaca_b200.csrc import attention_bf16
    k = torch.randn((6, 2, 64, 64), device=DEV).to(torch.bfloat16)
    q = torch.randn((4, 256), device=DEV).to(torch.bfloat16)
    args = (torch.tensor([130] * 4, dtype=torch.int32, device=DEV),)
    for table in ([[0, 99, 1]] * 4, [[0, 1, -1]] * 4):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        attention_bf16.decode_shared(q, k, k, *args, torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV),
                                     torch.tensor([2] * 4, dtype=torch.int32, device=DEV), 1, 4, 2, 1, 4, 0.125, status)
        assert status.item() == 1 << 2


def test_groups_that_are_not_what_was_said_are_reported():
    """A group of more members than the launch was made for, or bounds out of order: a status, no access elsewhere, and the others as ever."""
    from ithaca_b200.csrc import attention_bf16
    from ithaca_b200.engine.step import describe_status
    g = gen(3)
    lens = [200] * 6
    table, total = layout([4, 2], [2, 2], lens, 3)
    q = torch.randn((6, 4 * 64), generator=g).to(torch.bfloat16).to(DEV)
    k, v = (torch.randn((total, 2, 64, 64), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    def run(starts, most):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = attention_bf16.decode_shared(q, k, v, ints(lens), table.to(DEV), ints(starts), ints([2] * 6), len(starts) - 1, most, 2, 2, 4, 64 ** -0.5, status)
        return out, int(status.item())
    want, status = run([0, 4, 6], 4)
    assert status == 0 and run([0, 4, 6, 6], 4)[1] == 0             # an empty group is none
    for starts, most in (([0, 4, 6], 3), ([0, 4, 7], 4), ([-1, 4, 6], 4), ([0, 4, 2], 4), ([0, 2147483647, 6], 4)):
        got, status = run(starts, most)
        assert "groups of sequences" in describe_status(status), (starts, most)
        assert torch.isfinite(got).all()
    assert torch.equal(run([0, 4, 6], 3)[0][4:], want[4:])           # (a page to a run in both calls)


def test_shared_attention_replayed_for_other_lengths():
    from ithaca_b200.csrc import attention_bf16
    g = gen(11)
    k, v = (torch.randn((40, 2, 64, 64), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn((4, 512), generator=g).to(torch.bfloat16).to(DEV)
    table = torch.stack([torch.cat((torch.arange(6), 6 + 6 * i + torch.arange(6))) for i in range(4)]).to(torch.int32).to(DEV)
    lens, starts, shared = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([400] * 4, [0, 2, 4], [6] * 4))
    status, out = torch.zeros(1, dtype=torch.int32, device=DEV), torch.empty_like(q)
    call = lambda o=None: attention_bf16.decode_shared(q, k, v, lens, table, starts, shared, 2, 2, 6, 6, 8, 0.125, status, out=o)
    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for n, s in (([400, 401, 600, 768], [6] * 4), ([700, 390, 450, 500], [3, 3, 6, 6]), ([1, 2, 3, 4], [0] * 4)):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        shared.copy_(torch.tensor(s, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, call())
    assert status.item() == 0


def test_shared_attention_refuses():
    from ithaca_b200.csrc import attention_bf16
    o = ops()
    k = torch.zeros((6, 2, 64, 64), dtype=torch.bfloat16, device=DEV)
    q = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = dict(q=q, k_pages=k, v_pages=k, kv_lens=ints(70, 70, 70, 70), table=torch.zeros((4, 2), dtype=torch.int32, device=DEV), starts=ints(0, 4), shared=ints(1, 1, 1, 1),
                n_groups=1, max_members=4, shared_bound=1, own_bound=1, n_heads=4, scale=0.125, status=None)
    attention_bf16.decode_shared(**good)
    for bad in (dict(q=q.float()), dict(k_pages=k.float()), dict(v_pages=k[:5]), dict(n_heads=3), dict(q=q[:3]), dict(starts=ints(0, 2, 4)), dict(shared=ints(1, 1)), dict(max_members=0),
                dict(max_members=5), dict(n_groups=0, starts=ints(0)), dict(table=good["table"][:3]), dict(table=good["table"].long()), dict(kv_lens=good["kv_lens"].cpu()), dict(k_pages=k[:, :, :32], v_pages=k[:, :, :32]),
                dict(sink=torch.zeros(3, device=DEV)), dict(k_pages=k[..., :24], v_pages=k[..., :24]), dict(out=q.float()), dict(out=q[:3]), dict(shared_bound=-1)):
        with pytest.raises(o.KernelError):
            attention_bf16.decode_shared(**{**good, **bad})


def test_calls_on_two_streams_at_once():
    """Each of the three on two streams side by side, many times, with other inputs: none has anything in common with a call beside it."""
    from ithaca_b200.csrc import attention_bf16
    g = gen(12)
    logits = [torch.randn((16, 30011), generator=g).to(DEV) for _ in range(2)]
    sums = [(torch.rand((4, 4), generator=g) * -5).to(DEV) for _ in range(2)]
    pages = [torch.randn((3, 40, 2, 64, 32), generator=g).to(DEV) for _ in range(2)]
    k, v = (torch.randn((60, 2, 64, 128), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    q = [torch.randn((6, 8 * 128), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    table = [ints([[i + 7 * j for i in range(4)] + [30 + 4 * b + i for i in range(4)] for b in range(6)]) for j in range(2)]
    lens, starts, shared = [ints([400 + 9 * b for b in range(6)]), ints([300, 290, 512, 257, 400, 333])], ints([0, 3, 6]), ints([4] * 6)
    moves = [([1, 2, 3], [21, 22, 23], [64, 5, 33]), ([7, 7, 9], [30, 31, 32], [12, 12, 64])]

    def run(i):
        s, b, t = ops().beam_select(logits[i], sums[i], 8)
        p = pages[i].clone()
        ops().copy_rows([(p, *moves[i])])
        a = attention_bf16.decode_shared(q[i], k, v, lens[i], table[i], starts, shared, 2, 3, 4, 4, 8, 0.09, None)
        return s, b, t, p, a

    want = [[t.clone() for t in run(i)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_two_captured_steps_replayed_in_turn_share_nothing():
    """Selection and attention captured twice for other inputs; the graphs replayed one after the other, in either order, on two streams."""
    from ithaca_b200.csrc import attention_bf16
    g = gen(13)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    k = torch.randn((40, 2, 64, 64), generator=g).to(torch.bfloat16).to(DEV)
    cases, graphs = [], []
    for i in range(2):
        l, s = torch.randn((8, 5003), generator=g).to(DEV), (torch.rand((2, 4), generator=g) * -4).to(DEV)
        q = torch.randn((4, 256), generator=g).to(torch.bfloat16).to(DEV)
        args = (q, k, k, ints([500 - 70 * i] * 4), ints([[j + i for j in range(5)] + [20 + 3 * b + j for j in range(3)] for b in range(4)]), ints([0, 4]), ints([5] * 4), 1, 4, 5, 3, 4, 0.125, None)
        out, att = torch.zeros((3, 2, 8), dtype=torch.int32, device=DEV), torch.zeros_like(q)
        want = [t.clone() for t in ops().beam_select(l, s, 8)] + [attention_bf16.decode_shared(*args).clone()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops().beam_select(l, s, 8, out=out)
            attention_bf16.decode_shared(*args, out=att)
        cases.append((l, s, args, out, att, want))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for c in cases:
            c[3].zero_()
            c[4].zero_()
        torch.cuda.synchronize()
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for l, s, args, out, att, want in cases:
            assert torch.equal(out[0].view(torch.float32), want[0]) and torch.equal(out[1], want[1]) and torch.equal(out[2], want[2]) and torch.equal(att, want[3])


def test_a_vocabulary_of_the_largest_size_and_many_requests():
    g = gen(14)
    check_select(torch.randn((2, 1 << 20), generator=g), torch.tensor([[-1.0, -1.5]]), 32)
    check_select(torch.randn((700 * 3, 37), generator=g), torch.rand((700, 3), generator=g) * -3, 6)
    with pytest.raises(ops().KernelError):
        ops().beam_select(torch.zeros((1, (1 << 20) + 1), device=DEV), torch.zeros((1, 1), device=DEV), 2)
