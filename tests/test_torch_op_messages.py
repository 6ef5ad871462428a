"""A refusal of the C++ torch ops is an exception, whatever its message holds and however the compiler comes by its libstdc++."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "llm-scaler_b200")
OP = """
#include <ATen/ATen.h>
#include <torch/library.h>
namespace {
at::Tensor refuse(const at::Tensor& a) { TORCH_CHECK(false, "shape [", a.size(0), ", ", a.size(1), "] of ", 0.5, " ", a.scalar_type()); return a; }
}
TORCH_LIBRARY(b2q_message_test, m) { m.def("refuse(Tensor a) -> Tensor"); }
TORCH_LIBRARY_IMPL(b2q_message_test, CPU, m) { m.impl("refuse", &refuse); }
"""
CALL = """
import sys, torch
torch.ops.load_library(sys.argv[1])
try:
    torch.ops.b2q_message_test.refuse(torch.zeros(3, 4))
except RuntimeError as x:
    print(str(x).split("\\n")[0])
"""


def test_numbers_in_a_message(lib_built, tmp_path):
    """An op built as the package's own are: its message holds numbers, which ended the process while a second libstdc++ was linked in."""
    spec = importlib.util.spec_from_file_location("b2q_build_for_messages", os.path.join(PKG, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    (tmp_path / "op.cpp").write_text(OP)
    out = build.build_torch_ops(True, str(tmp_path / "libop.so"), str(tmp_path / "op.cpp"))
    r = subprocess.run([sys.executable, "-c", CALL, out], capture_output=True, text=True, env=dict(os.environ, LD_LIBRARY_PATH=os.path.join(PKG, "custom_esimd_kernels_vllm")))
    assert r.returncode == 0 and r.stdout.startswith("shape [3, 4] of 0.5 Float"), (r.returncode, r.stdout, r.stderr[-500:])


REFUSALS = """
import torch, custom_esimd_kernels_vllm as e
x, w, out = torch.zeros(2, 256, device="cuda").half(), torch.zeros(64, 128, dtype=torch.uint8, device="cuda"), torch.zeros(2, 64, device="cuda").half()
for scale in ((64, 3), (3, 64), (2, 2)):
    try:
        torch.ops.custom_esimd_kernels_vllm.esimd_gemm_int4_pgrp(x, w, torch.zeros(scale, device="cuda").half(), out)
    except RuntimeError as error:
        print("refused", "scale" in str(error))
"""


@pytest.mark.gpu
def test_an_int4_scale_of_the_wrong_shape_is_refused():
    r = subprocess.run([sys.executable, "-c", REFUSALS], capture_output=True, text=True, env=dict(os.environ, PYTHONPATH=PKG))
    assert r.returncode == 0 and r.stdout.split() == ["refused", "True"] * 3, (r.returncode, r.stdout, r.stderr[-500:])
