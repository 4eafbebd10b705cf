"""Attention behind shared pages refuses whatever it would hand to the kernel from elsewhere than the current device, before anything is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_status_and_sink_of_the_host_are_refused():
    from ithaca_b200.csrc import attention_bf16
    from ithaca_b200.csrc.ops import KernelError, launch_count
    k = torch.zeros((6, 2, 64, 64), dtype=torch.bfloat16, device=DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = dict(q=torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV), k_pages=k, v_pages=k, kv_lens=ints(70, 70, 70, 70), table=torch.zeros((4, 2), dtype=torch.int32, device=DEV),
                starts=ints(0, 4), shared=ints(1, 1, 1, 1), n_groups=1, max_members=4, shared_bound=1, own_bound=1, n_heads=4, scale=0.125, status=ints(0))
    n = launch_count()
    for bad in (dict(status=torch.zeros(1, dtype=torch.int32)), dict(status=torch.zeros(1, device=DEV)), dict(sink=torch.zeros(4)), dict(sink=torch.zeros(4, device=DEV).double()),
                dict(sink=torch.zeros(8, device=DEV)[::2])):
        with pytest.raises(KernelError):
            attention_bf16.decode_shared(**{**good, **bad})
    assert launch_count() == n
    for fine in (dict(), dict(status=None), dict(sink=True), dict(sink=torch.zeros(4, device=DEV))):
        assert torch.equal(attention_bf16.decode_shared(**{**good, **fine}), torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV))
    assert good["status"].item() == 0
