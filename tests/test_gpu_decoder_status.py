"""The status of the waits inside the matrix kernels: told once, and never lost.  The fault is a count that a kernel raises."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from configurable_hierarchical_allreduce_algorithms_b200.ops import decoder

pytestmark = pytest.mark.gpu


def raise_status():
    decoder._call("chb_matrix_status_raise", torch.device("cuda", torch.cuda.current_device()))


def test_told_once(cuda):
    chb.check_operators()
    raise_status()
    raise_status()
    with pytest.raises(chb.OperatorError, match="ran out"):
        chb.check_operators("cuda")
    chb.check_operators()


def test_none_is_lost_to_a_check_at_the_same_time(cuda):
    side = torch.cuda.Stream()
    chb.check_operators()
    for _ in range(300):
        told = 0
        with torch.cuda.stream(side):
            raise_status()
        for wait in (False, True):
            if wait:
                side.synchronize()
            try:
                chb.check_operators()
            except chb.OperatorError:
                told += 1
        assert told == 1


@pytest.mark.parametrize("mode", ["dp", "zero"])
def test_the_training_command_asks(cuda, mode, capsys):
    from configurable_hierarchical_allreduce_algorithms_b200.bench import train

    argv = ["--mode", mode, "--tiny", "--steps", "1", "--warmup", "1"]
    raise_status()
    with pytest.raises(chb.OperatorError, match="ran out"):
        train.main([*argv, "--native"])
    assert "tokens_per_s" not in capsys.readouterr().out
    train.main([*argv, "--native"])                               # (and the next run is not blamed)
    assert "tokens_per_s" in capsys.readouterr().out


def test_smoke_runs_the_operators(cuda, monkeypatch):
    import __graft_entry__

    called = []
    call = decoder._call
    monkeypatch.setattr(decoder, "_call", lambda name, *a: (called.append(name), call(name, *a))[1])
    __graft_entry__.smoke()
    assert {"chb_head_rope", "chb_attention_forward", "chb_attention_backward", "chb_linear_ce_forward", "chb_linear_ce_backward",
            "chb_matrix_status"} <= set(called)
