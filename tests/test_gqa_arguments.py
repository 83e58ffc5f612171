"""CPU: checks of the grouped-query entry points' Python arguments that need
no GPU."""
import pytest
import torch

import deepseek_v4_kernel as dk


def test_status_refuses_other_devices():
    for device in ("cpu", torch.device("cpu"), torch.device("meta")):
        with pytest.raises(RuntimeError, match="not a CUDA device"):
            dk.gqa_status(device)
