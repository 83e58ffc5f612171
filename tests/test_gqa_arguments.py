"""CPU: checks of the grouped-query entry points' Python arguments that need
no GPU."""
import pytest
import torch

import deepseek_v4_kernel as dk


def test_status_refuses_other_devices():
    for device in ("cpu", torch.device("cpu"), torch.device("meta")):
        with pytest.raises(RuntimeError, match="not a CUDA device"):
            dk.gqa_status(device)


def test_tensors_apart():
    """Whether weights and new_weights share an element, against the elements' addresses."""
    from deepseek_v4_kernel.gqa import _apart
    pool = torch.zeros(40, 6, 64)
    flat = pool.view(-1)
    views = [pool[:2, :3, :20], pool[:2, :3, 20:50], pool[:2, :3, 19:50], pool[:2, :3, 44:], pool[2:4, :3, :20], pool[1:3, :3, :20],
             pool[:2, 3:, :20], pool[:2, 2:5, :20], pool[:2, 2:5, 20:30], pool[0:4:2, :3, :20], pool[1:5:2, :3, :20], pool[:2, :, :64],
             pool[:2, :1, :20], pool[:2, 1:2, 10:30], pool[:1, :3, :20], pool[:1, 1:4, 20:], pool[:1, :1, :8], pool[:1, :1, 8:16],
             pool[:1, :1, 7:16], pool[:2, :1, :16].expand(2, 3, 16), pool[4:6, :1, :16].expand(2, 3, 16), pool[30:32, :3, 4:24],
             flat[5:5 + 2 * 3 * 20].view(2, 3, 20), flat[2000:2000 + 120].view(2, 3, 20)]

    def elements(t):
        at = t.storage_offset() + sum(torch.arange(n).view([-1 if i == j else 1 for j in range(3)]) * x
                                      for i, (n, x) in enumerate(zip(t.shape, t.stride())))
        return set(at.flatten().tolist())

    sets = [elements(v) for v in views]
    for a, x in zip(views, sets):
        for b, y in zip(views, sets):
            assert _apart(a, b) == (not x & y), (a.shape, a.stride(), b.shape, b.stride())


@pytest.mark.parametrize("shape,strides", [((2, 3, 8), (24, 8, 1)), ((2, 3, 8), (8, 16, 1)), ((2, 3, 8), (8, 8, 1)), ((2, 3, 8), (7, 40, 1)),
                                           ((2, 3, 8), (40, 4, 1)), ((1, 3, 8), (0, 8, 1)), ((2, 1, 8), (8, 3, 1)), ((2, 3, 8), (0, 8, 1)),
                                           ((2, 2, 8), (24, 32, 1)), ((2, 2, 8), (24, 30, 1)), ((2, 2, 8), (8, 15, 1)), ((4, 3, 8), (48, 16, 1)),
                                           ((4, 3, 8), (40, 16, 1)), ((2, 3, 4, 8), (96, 8, 24, 1)), ((2, 3, 4, 8), (88, 8, 24, 1)), ((3, 2, 2, 8), (8, 24, 48, 1))])
def test_written_rows_must_not_overlap(shape, strides):
    from deepseek_v4_kernel.gqa import _own_rows
    t = torch.zeros(4096).as_strided(shape, strides)
    at = sum(torch.arange(n).view([-1 if i == j else 1 for j in range(len(shape))]) * x for i, (n, x) in enumerate(zip(shape, strides)))
    if at.unique().numel() == at.numel():
        _own_rows(t, "out")
    else:
        with pytest.raises(RuntimeError, match="overlap"):
            _own_rows(t, "out")
