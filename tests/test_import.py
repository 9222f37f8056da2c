"""CPU: importing the package."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_package_imports_without_torch():
    """Calls that take tensors import torch; the package itself, its C ABI and its tables do without."""
    code = ("import sys; sys.modules['torch'] = None; import animaxs_b200; "
            "assert animaxs_b200.qwen_rope(4).shape == (4 * 64 * 4,); assert animaxs_b200.QuantizedKVCache")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=120)


def test_the_package_does_not_import_torch():
    code = "import sys, animaxs_b200; assert 'torch' not in sys.modules"
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=120)
