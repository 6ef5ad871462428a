"""The package without the shared objects of its C++ op layers: refused, with what to do; but the switches that keep every other op on its Python
implementation need libb2q.so alone, and then only the 8-bit integer operators fail, each when it is called.  No GPU needed."""
import os
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "custom_esimd_kernels_vllm")
CALL = """
import custom_esimd_kernels_vllm as e
print("imported", e._lib.lib.b2q_version() >= 100)
try:
    e.quantize_int8(None)
except ImportError as x:
    print("refused", "libb2q_int8.so" in str(x))
"""


@pytest.fixture(scope="module")
def tree(lib_built, tmp_path_factory):
    d = tmp_path_factory.mktemp("tree")
    shutil.copytree(PKG, d / "custom_esimd_kernels_vllm", ignore=shutil.ignore_patterns("__pycache__", "libb2q_torch.so", "libb2q_int8.so"))
    return str(d)


def _run(tree, **env):
    return subprocess.run([sys.executable, "-c", CALL], cwd=tree, env=dict(os.environ, PYTHONPATH=tree, **env), capture_output=True, text=True)


@pytest.mark.parametrize("switch", ["B2Q_PYTHON_DISPATCH", "B2Q_CHECK_STATUS"])
def test_python_dispatch_needs_the_kernels_alone(tree, switch):
    r = _run(tree, **{switch: "1"})
    assert r.returncode == 0 and r.stdout.split("\n")[:2] == ["imported True", "refused True"], r.stderr[-500:]


def test_otherwise_the_import_is_refused(tree):
    r = _run(tree)
    assert r.returncode != 0 and "llm-scaler_b200/build.py" in r.stderr
