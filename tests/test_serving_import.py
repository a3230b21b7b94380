"""The compiled module behind kvcache and speculative is needed by them alone: where it cannot be loaded, the rest of
the package works and they say so."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)


def test_the_package_works_without_the_serving_module():
    p = _run("""
import sys
sys.modules["tallax_amd._build.serving_ext"] = None  # its import fails
import tallax_amd
from tallax_amd import _lib, kvcache, prefill, sampling, speculative, tax, tumpy
assert _lib.select_plan(8, 32000, _lib.BF16)["threads"] > 0
for call in (lambda: kvcache.append(*[None] * 6), lambda: kvcache.decode(*[None] * 5),
             lambda: kvcache.evict(*[None] * 7, budget=1), lambda: speculative.verify(*[None] * 4)):
    try:
        call()
    except ImportError as e:
        assert "serving_ext" in str(e)
    else:
        raise AssertionError("no ImportError")
print("fine")
""")
    assert p.returncode == 0 and p.stdout.strip() == "fine", p.stderr


def test_the_serving_module_is_loaded_on_first_use():
    p = _run("""
import importlib, sys
import tallax_amd
from tallax_amd import _lib, kvcache
assert "tallax_amd._build.serving_ext" not in sys.modules
for _ in range(2):
    try:
        kvcache.append(*[None] * 6)
    except ValueError as e:
        assert "must be torch tensors" in str(e)
    else:
        raise AssertionError("no ValueError")
    assert _lib.SERVING is sys.modules["tallax_amd._build.serving_ext"]
    importlib.reload(_lib)
assert not hasattr(_lib, "NOTHING")
print("fine")
""")
    assert p.returncode == 0 and p.stdout.strip() == "fine", p.stderr
