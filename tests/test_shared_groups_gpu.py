"""Attention behind shared pages: groups that are larger than the call says."""
import pytest
import torch

from test_search_kernels_gpu import gen, layout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 48), (2, 2, 128), (20, 1, 64)])
@pytest.mark.parametrize("most", [1, 3, 17, 33])
def test_members_beyond_the_bound_get_zeros(nh, nkv, hd, most):
    """Also those for whom there would be room in a tile's rows; the members before them and the other groups have what they have in a call that fits."""
    from ithaca_b200.csrc import attention_bf16
    members = [40, min(most, 5)]
    g, B = gen(hd + most), sum(members)
    lens = [64 * 3 + 1 + 7 * i for i in range(B)]
    table, total = layout(members, [2, 1], lens, 3)
    q = torch.randn((B, nh * hd), generator=g).to(torch.bfloat16)
    k, v = (torch.randn((total, nkv, 64, hd), generator=g).to(torch.bfloat16) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = attention_bf16.decode_shared(q.to(DEV), k.to(DEV), v.to(DEV), ints(lens), table.to(DEV), ints([0, 40, B]), ints([2] * 40 + [1] * members[1]), 2, most, 2, 4, nh, hd ** -0.5,
                                       status).cpu().double().view(B, nh, hd)
    assert status.item() == 1 << 5
    assert (got[most:40] == 0).all()
    for b in [*range(most), *range(40, B)]:
        pages = table[b, :-(-lens[b] // 64)].long()
        kb, vb = (t[pages].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :lens[b]].repeat_interleave(nh // nkv, 0) for t in (k, v))
        p = torch.softmax(torch.einsum("hd,hjd->hj", q[b].double().view(nh, hd), kb) * hd ** -0.5, -1)
        want, size = torch.einsum("hj,hjd->hd", p, vb), torch.einsum("hj,hjd->hd", p, vb.abs())
        # probabilities and the result are rounded to bfloat16 (2^-8 each), scores are float sums (below 2^-14 at these sizes)
        assert ((got[b] - want).abs() <= 2 ** -8 * (size + want.abs()) + 2 ** -14 * size).all()
