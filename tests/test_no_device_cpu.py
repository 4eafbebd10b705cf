"""What a host without a device, or a torch built without CUDA, sees of the package."""
import subprocess
import sys

import pytest
import torch

from ithaca_b200.csrc import attention_bf16, ops


def test_the_package_is_imported_by_a_torch_without_cuda():
    """Such a torch lacks the functions that ask for the current device and stream."""
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_get')]:\n"
            "    delattr(torch._C, name)\n"
            "import ithaca_b200, ithaca_b200.csrc.ops, ithaca_b200.csrc.attention_bf16, ithaca_b200.engine.beam\n"
            "try:\n"
            "    ithaca_b200.csrc.ops._stream()\n"
            "except ithaca_b200.csrc.ops.KernelError as e:\n"
            "    assert 'without CUDA' in str(e)\n"
            "    print('imported')\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and run.stdout.split() == ["imported"], run.stderr[-2000:]


def test_tensors_of_the_host_are_refused_without_a_device():
    """The library's own error, whether there is a device or not."""
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    pages = torch.zeros((2, 1, 64, 64), dtype=torch.bfloat16)
    calls = [lambda: ops.beam_select(torch.zeros((2, 5)), torch.zeros((1, 2)), 2),
             lambda: ops.copy_rows([(torch.zeros((1, 3, 2)), [0], [1], None)]),
             lambda: attention_bf16.decode_shared(torch.zeros((2, 64), dtype=torch.bfloat16), pages, pages, ints(3, 4), torch.zeros((2, 1), dtype=torch.int32), ints(0, 2), ints(0, 0),
                                                  1, 2, 0, 1, 1, 0.125, None)]
    for call in calls:
        with pytest.raises(ops.KernelError, match="CUDA tensor"):
            call()
    ops.copy_rows([])                              # nothing to do needs no device
