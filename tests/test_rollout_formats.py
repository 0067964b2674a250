"""Every command that names the rollout engine's weight formats names the same ones."""
import os
import re
import subprocess
import sys

import pytest

from miles_b200.utils.arguments import TRAINER_FLAGS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("command,flag", [(["bench.py"], "--rollout-quantization"), (["benchmarks/bench_decode.py"], "--quantization"),
                                          (["-m", "miles_b200.engine.server"], "--quantization")])
def test_formats(command, flag):
    want = {f[0]: f[3].get("choices") for f in TRAINER_FLAGS}["--rollout-quantization"]
    out = subprocess.run([sys.executable, *command, "--help"], cwd=ROOT, capture_output=True, text=True, timeout=300, env={**os.environ, "COLUMNS": "200"})
    assert out.returncode == 0, out.stderr
    assert re.search(rf"{flag} {{([a-z0-9_,]+)}}", out.stdout).group(1).split(",") == want
