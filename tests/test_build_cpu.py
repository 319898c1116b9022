"""The C library is built with nvcc alone; the torch extension only where there is a torch with CUDA."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

NO_TORCH = "sys.modules['torch'] = None"  # `import torch` raises ImportError
CPU_TORCH = ("t = types.ModuleType('torch'); t.version = types.SimpleNamespace(cuda=None); t.__version__ = '0'; "
             "t.__file__ = '/nowhere/__init__.py'; sys.modules['torch'] = t")


@pytest.mark.parametrize("torch", [NO_TORCH, CPU_TORCH], ids=["none", "cpu"])
def test_library_builds_without_cuda_torch(built_lib, torch):
    code = (f"import sys, types; sys.path.insert(0, {str(ROOT)!r}); {torch}; from aethermind_b200 import build; "
            "assert build.build() == build.LIB and build.LIB.exists(); assert build.build_native() is None; "
            "from aethermind_b200 import _lib; _lib.lib(); print('built')")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip() == "built", r.stderr
