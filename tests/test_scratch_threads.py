"""The scratch that the calls of a stream share, with several threads calling
(tests/host_check/scratch_check.cpp).  CPU only."""
import json
import os
import subprocess

DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_check")


def test_a_call_s_launches_have_the_scratch_to_themselves():
    subprocess.run(["make", "-C", DIR, "-s", "scratch_check"], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([os.path.join(DIR, "scratch_check")], capture_output=True, text=True, timeout=300, env=env)
    assert "Sanitizer" not in r.stderr and "runtime error" not in r.stderr, r.stderr[-4000:]
    found = json.loads(r.stdout.splitlines()[-1])
    # (Calls on the two streams do go on side by side.)
    assert found["failures"] == 0 and found["launches"] > 700 and found["side_by_side"] > 0, r.stdout
