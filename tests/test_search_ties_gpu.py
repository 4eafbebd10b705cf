"""The choice of continuations where more tiles reach the bound than are taken as they come: the number of them is counted twice, and every
thread has to have read the first count before the second begins."""
import math

import pytest
import torch

from test_search_kernels_gpu import check_select, gen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from ithaca_b200.csrc import ops as o
    return o


@pytest.mark.parametrize("R,K,V,n", [(300, 4, 20000, 8), (40, 16, 50257, 32), (150, 1, 128256, 1), (2, 2, 1 << 20, 16)])
def test_equal_logits_of_many_tiles(R, K, V, n):
    """Every tile of every beam is as good as the bound, in more requests than run at a time, again and again: the first tokens of the first beam."""
    l = torch.full((R * K, V), 0.5, device=DEV)
    sums = torch.full((R, K), -3.0, device=DEV)
    for _ in range(20):
        s, b, v = ops().beam_select(l, sums, n)
        assert (b == 0).all() and (v == torch.arange(n, device=DEV, dtype=torch.int32)).all()
        # every tile's sum is a whole number: what is left is the result's rounding (and that of 64 bits)
        assert (s.double() - (-3.0 - math.log(V))).abs().max().item() <= 2 ** -24 * (3 + math.log(V)) + 1e-12


@pytest.mark.parametrize("R,K,V,n", [(6, 4, 50257, 8), (2, 16, 128256, 32), (3, 1, 128256, 32)])
@pytest.mark.parametrize("bits", [1, 2, 3])
def test_logits_of_few_bits(R, K, V, n, bits):
    """Coarse logits: the largest value stands in nearly every tile, at places that differ from tile to tile; beams with equal and with other sums."""
    l = torch.randint(0, 1 << bits, (R * K, V), generator=gen(V + bits)).float()
    sums = torch.where(torch.rand((R, K), generator=gen(n)) < 0.5, -1.0, -1.5)
    first = check_select(l, sums, n)
    l, sums = l.to(DEV), sums.to(DEV)
    for _ in range(50):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(ops().beam_select(l, sums, n), first))


def test_ordinary_and_tied_requests_side_by_side():
    """Blocks that count twice beside blocks that do not, and a request of which few threads have any candidate."""
    R, K, V, n = 64, 4, 40000, 16
    l = torch.randn((R * K, V), generator=gen(1)) * 3
    l[::3] = l[::3].round() / 4
    l[K * 5:K * 6] = -math.inf
    l[K * 5, 39990:] = 1.0
    sums = torch.rand((R, K), generator=gen(2)) * -2
    first = check_select(l, sums, n)
    l, sums = l.to(DEV), sums.to(DEV)
    for _ in range(50):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(ops().beam_select(l, sums, n), first))
