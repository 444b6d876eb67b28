"""What importing the package brings along."""
import os
import subprocess
import sys

import appy_b200 as appy

WITHOUT_TORCH = """
import sys
class NoTorch:
    def find_spec(self, name, path=None, target=None):
        if name.split(".")[0] == "torch":
            raise ModuleNotFoundError("no torch here", name=name)
sys.meta_path.insert(0, NoTorch())
"""


def run(code):
    root = os.path.dirname(os.path.dirname(os.path.abspath(appy.__file__)))
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=root)


def test_a_star_import_needs_no_torch():
    r = run(WITHOUT_TORCH + "from appy_b200 import *\nassert callable(jit) and callable(prange) and not any(m.startswith('torch') for m in sys.modules)")
    assert r.returncode == 0, r.stderr


def test_operators_are_listed_and_come_when_asked_for():
    names = ["embedding", "embedding_grad", "gated_scan", "gated_scan_grad", "token_logprobs", "token_logprobs_grad"]
    assert set(names) <= set(dir(appy)) and all(callable(getattr(appy, n)) for n in names)
    r = run("import sys, appy_b200\ndir(appy_b200)\nassert 'torch' not in sys.modules\nfrom appy_b200 import embedding\nassert 'torch' in sys.modules")
    assert r.returncode == 0, r.stderr
