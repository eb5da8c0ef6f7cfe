"""The watchdog of tests/conftest.py: a test that runs past the limit ends the process with SIGABRT and leaves the threads' states and Python's
frames behind.  It reads only its own process: no other program is started.  (CPU; the stopped test sleeps in a child process.)"""
import os
import signal
import subprocess
import sys

from conftest import ROOT

CHILD = '''
import subprocess
import time


def refuse(*a, **k):
    print("a program was started: %r" % (a,), flush=True)
    raise OSError("no program may be started here")


def test_that_does_not_end():
    subprocess.Popen.__init__ = refuse
    time.sleep(120)
'''


def test_a_stopped_test_is_reported_and_ended_from_inside_the_process(tmp_path):
    (tmp_path / "test_child.py").write_text(CHILD)
    env = dict(os.environ, NP_TEST_WATCHDOG_S="3", PYTHONPATH=os.path.join(ROOT, "tests"))
    env.pop("NP_ABORT_TRACE", None)
    p = subprocess.Popen([sys.executable, "-m", "pytest", "-p", "conftest", "-p", "no:cacheprovider", "-s", "--rootdir", str(tmp_path), str(tmp_path / "test_child.py")],
                         cwd=str(tmp_path), env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    out = p.communicate(timeout=110)[0].decode("utf-8", "replace")
    made = [os.path.join(ROOT, "gpurun_out", n % p.pid) for n in ("hang_%d.txt", "hang_%d.txt.streams", "abort_%d.txt")]
    try:
        report = open(made[0]).read()
    finally:
        for f in made:
            if os.path.exists(f):
                os.remove(f)
    assert p.returncode == -signal.SIGABRT, out[-2000:]
    assert "test_that_does_not_end has been running for" in report
    assert "[np watchdog] threads (tid comm wchan state syscall):" in report and "state=S" in report
    assert "[np watchdog] Python frames:" in report and "in test_that_does_not_end" in report
    assert "a program was started" not in out, out[-2000:]
    assert "debugger" not in report and "debugger" not in out
