"""The command that runs one operator on a seeded case."""
import json

import pytest

from auto_gpu_kernel_b200 import run_case


def test_usage_without_a_device_or_case(capsys):
    with pytest.raises(SystemExit):
        run_case.main(["no-such-case"])
    assert "paged" in capsys.readouterr().err


@pytest.mark.gpu
@pytest.mark.parametrize("argv", [["paged", "--batch", "3", "--context", "700"],
                                  ["paged", "--batch", "2", "--context", "300", "--heads", "40", "--new-tokens", "2", "--weights"],
                                  ["evict", "--batch", "3", "--context", "700", "--budget", "100"],
                                  ["rotary", "--batch", "100"]])
def test_new_operators(argv, capsys):
    assert run_case.main([*argv, "--iters", "2", "--warmup", "1"]) == 0
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["case"] == argv[0] and line["status"] == 0 and line["us_per_iter"] > 0
