"""The package can be imported from the repository's root alone."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import_from_the_root():
    code = ("import q4rdna; from q4rdna import api, _lib; "
            "assert q4rdna.load() is _lib.load() and q4rdna.api is api and api.add_norm; print(q4rdna.__file__)")
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip().endswith(os.path.join("rdna-gfx1201-v0.1_amd", "q4rdna", "__init__.py"))
