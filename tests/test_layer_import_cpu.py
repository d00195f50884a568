"""The package without the torch binding of the decoder-layer operators (another torch, or only the C library built)."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "onnxruntime-ep-mlx_b200")

WITHOUT = """
import sys
sys.modules["onnxruntime_ep_b200._layer"] = None  # what cannot be loaded
import onnxruntime_ep_b200 as b200
from onnxruntime_ep_b200 import ep, paged
assert callable(b200.paged_attention) and callable(b200.kv_append) and b200.kernel_library_path().endswith(".so")
for call in (lambda: b200.skip_rms_norm(None, None, None),
             lambda: b200.rotary_append(*[None] * 9, num_heads=1, kv_num_heads=1),
             lambda: b200.shared_prefix_attention(*[None] * 7, prefix_length=0, num_heads=1, kv_num_heads=1)):
    try:
        call()
    except ImportError as e:
        assert "_layer.so" in str(e) and "make" in str(e), e
    else:
        raise AssertionError("no error without the binding")
print("fine")
"""


def test_the_rest_of_the_package_needs_no_binding():
    env = dict(os.environ, PYTHONPATH=PKG)
    done = subprocess.run([sys.executable, "-c", WITHOUT], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine", done.stderr


def test_the_library_builds_without_torch():
    """A python without torch: make plans the library, and not the binding."""
    done = subprocess.run(["make", "-n", "-B", "-C", os.path.join(PKG, "csrc"), "PYTHON=false"], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr
    assert "libb200_paged.so" in done.stdout and "layer_binding.cpp" not in done.stdout


def test_the_binding_loads_and_knows_the_error_class():
    from onnxruntime_ep_b200 import B200Error, skip_rms_norm

    try:
        skip_rms_norm(None, None, None)
    except B200Error as e:
        assert "x must be a tensor" in str(e)
    else:
        raise AssertionError("no error")
