"""The build without torch, which only the operators' binding needs."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys, types
sys.modules["torch"] = {torch}
sys.path.insert(0, {package!r})
import build_ext
built = []
build_ext._build_engine = lambda *a: built.append("engine")
assert build_ext.build(force=True) == build_ext.OUT and built == ["engine"]
"""


@pytest.mark.parametrize("torch", ["None", "types.SimpleNamespace(version=types.SimpleNamespace(cuda=None), "
                                           "__version__='2', __file__='/nowhere/torch/__init__.py')"],
                         ids=["none", "without CUDA"])
def test_the_engine_builds_without_torch(torch):
    r = subprocess.run([sys.executable, "-c", CHILD.format(torch=torch, package=os.path.join(ROOT, "alphazero-go_b200"))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "_azb_torch.so is not built" in r.stderr, r.stderr
