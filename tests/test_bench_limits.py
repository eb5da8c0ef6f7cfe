"""What bench.py asks of the machine, checked without one (CPU)."""
import os
import re
import subprocess
import sys

from conftest import ROOT


def test_the_long_read_leg_and_the_bench_itself_are_at_most_16_processes_on_a_card():
    with open(os.path.join(ROOT, "bench.py")) as f:
        n = int(re.search(r'"--lgs-workers", type=int, default=(\d+)', f.read()).group(1))
    assert n + 1 <= 16


def test_progress_goes_to_stderr_of_rank_0_only():
    for rank, lines in (("0", 1), ("1", 0)):
        p = subprocess.run([sys.executable, "-c", "import bench; bench.step('a part has ended')"], cwd=ROOT, capture_output=True, text=True, env=dict(os.environ, RANK=rank))
        assert p.returncode == 0 and p.stdout == "" and p.stderr.count("a part has ended") == lines, (rank, p.stdout, p.stderr)
