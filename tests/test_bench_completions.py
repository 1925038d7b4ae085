"""`bench.py --completions`: one JSON line with both ways of asking for several completions."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_completions_beside_prompts():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--completions", "3", "--prompt-len", "100", "--layers", "1",
                        "--shape", "llama-3.2-1b"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout.splitlines()[-1])
    assert line["layers"] == 1 and line["prompt_len"] == 100 and line["steps"] == 64
    for way in ("completions", "prompts"):
        assert line[way]["first_ms"] > 0 and line[way]["ms_per_step"] > 0
