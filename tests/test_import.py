"""What the package needs at import: the HIP library alone; the attention block's
modules bring their compiled binding when they are first used."""
import subprocess
import sys

from conftest import ROOT

WITHOUT_BINDING = """
import sys
sys.modules["ubridge_amd._native"] = None  # not built, or built for another torch
import ubridge_amd
from ubridge_amd import QMatMul, dequantize_block, fp8, get_function, moe
from ubridge_amd.ops import gemm_dense
for name in ("attention", "int8", "kvcache", "rope"):
    assert name in dir(ubridge_amd)
    try:
        getattr(ubridge_amd, name)
    except ImportError as e:
        assert "build.py" in str(e), e
    else:
        raise AssertionError(name)
try:
    ubridge_amd.nothing
except AttributeError as e:
    assert "nothing" in str(e)
"""

WITH_BINDING = """
import ubridge_amd
assert ubridge_amd.int8.Linear and ubridge_amd.kvcache.PagedCache
from ubridge_amd import attention, rope
import ubridge_amd.rope as again
assert rope is again is ubridge_amd.rope and attention.paged_decode
"""


def run(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_without_the_binding():
    run(WITHOUT_BINDING)


def test_with_the_binding():
    run(WITH_BINDING)
