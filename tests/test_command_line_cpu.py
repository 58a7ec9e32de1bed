"""Flags of train.py that say nothing alone, on the CPU."""
import pytest

import train
from gpt_from_scratch_b200.ops import RopeScaling


@pytest.mark.parametrize("argv", [["--rope-scaling", "linear"], ["--rope-scaling", "by_parts", "--rope-original-length", "1024"],
                                  ["--rope-scaling-factor", "2"], ["--rope-original-length", "1024"],
                                  ["--rope-scaling", "ntk", "--rope-scaling-factor", "2", "--rope-original-length", "1024"]])
def test_scaling_flags_that_would_change_nothing_are_refused(argv, capsys):
    with pytest.raises(SystemExit):
        train.parse_args(argv)
    assert "--rope" in capsys.readouterr().err


def test_scaling_flags():
    for kind in ("linear", "ntk"):
        cfg = train.build_config(train.parse_args(["--rope-scaling", kind, "--rope-scaling-factor", "2"]))
        assert cfg.rope_scaling == RopeScaling(kind, 2.0)
    assert train.build_config(train.parse_args([])).rope_scaling is None
