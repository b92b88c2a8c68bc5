"""Without the C++ binding (not built, or built against another torch) only the functions that it
holds are missing, and those say so."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpt-oss-tvm_amd")

SCRIPT = """
import sys
sys.modules["attn_binding"] = None            # `import attn_binding` raises ImportError
import torch
import attn_native as A
from engine import Engine
assert A.decode_workspace_bytes(1, 1000) > 0 and Engine is not None
i = torch.zeros(2, dtype=torch.int32)
for call in (lambda: A.beam_top_k(i, i, 1), lambda: A.kv_copy_pages(i, i, i),
             lambda: A.tree_commit(i, i, i, i, i, 1, i, i, i),
             lambda: A.tree(i, i, 1, i, i, i, i, i, i, 0, 1.0, i, i),
             lambda: A.tree_fp8(i, i, 1, i, i, i, i, i, i, 0, 1.0, i, i)):
    try:
        call()
    except ImportError as e:
        assert "build_native" in str(e) and isinstance(e.__cause__, ImportError)
    else:
        raise SystemExit("no error")
print("fine")
"""


def test_only_its_functions_are_missing():
    run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=PKG, text=True, timeout=300,
                         capture_output=True)
    assert run.returncode == 0 and run.stdout.endswith("fine\n"), run.stdout + run.stderr
