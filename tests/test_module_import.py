"""What importing the package loads."""
from __future__ import annotations

import subprocess
import sys

from conftest import ROOT

BLOCK = """
import sys
class NoTorch:
    def find_spec(self, name, path=None, target=None):
        if name == "torch" or name.startswith("torch."):
            raise ModuleNotFoundError(f"No module named {name!r}", name=name)
sys.meta_path.insert(0, NoTorch())
"""


def run(code):
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)


def test_star_import_without_torch():
    run(BLOCK + """
from flash_attn_metal_cpp_b200 import *
assert callable(forward) and callable(metal_attention)
try:
    import flash_attn_metal_cpp_b200 as p
    p.paged_forward
    raise SystemExit("no error")
except ModuleNotFoundError as e:
    assert e.name == "torch"
""")


def test_star_import_loads_no_torch():
    run("""
import sys
from flash_attn_metal_cpp_b200 import *
from _flash_attn_metal import *
assert callable(forward) and "torch" not in sys.modules
import flash_attn_metal_cpp_b200 as p
assert {"plan_pages", "store_kv", "paged_forward", "shared_prefix_forward"} <= set(dir(p)) and "torch" not in sys.modules
""")
