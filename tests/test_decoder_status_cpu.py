"""Which device ``check_operators`` asks, and what it makes of the answer, with a fake of the native call."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from configurable_hierarchical_allreduce_algorithms_b200.ops import decoder


@pytest.mark.parametrize("asked,index", [(None, 3), ("cuda", 3), (torch.device("cuda"), 3), ("cuda:0", 0), (2, 2), (torch.device("cuda", 1), 1)])
@pytest.mark.parametrize("expired", [0, 1])
def test_the_device_that_is_asked(monkeypatch, asked, index, expired):
    seen = []

    def call(name, device, word):
        seen.append((name, device))
        word._obj.value = expired

    monkeypatch.setattr(decoder, "_call", call)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    if expired:
        with pytest.raises(chb.OperatorError, match="ran out"):
            chb.check_operators(asked)
    else:
        chb.check_operators(asked)
    assert seen == [("chb_matrix_status", torch.device("cuda", index))]


def test_other_devices_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        chb.check_operators("cpu")
