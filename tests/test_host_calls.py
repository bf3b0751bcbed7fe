"""CPU checks of how the Python operators pass streams to the library."""

import subprocess
import sys

from conftest import ROOT

_WITHOUT_RAW_STREAM = """
import types, torch
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    del torch._C._cuda_getCurrentRawStream
import heteromega_amd.ffn as ffn
torch.cuda.current_stream = lambda device=None: types.SimpleNamespace(cuda_stream=4096 + device.index)
assert ffn._stream(None, torch.device("cuda", 3)) == 4099
assert ffn._stream(17, torch.device("cuda", 3)) == 17
"""


def test_current_stream_without_torchs_private_handle():
    # The raw handle comes from a private function of torch; without it the public call serves.
    res = subprocess.run([sys.executable, "-c", _WITHOUT_RAW_STREAM], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


_WITHOUT_THE_ATTENTION_MODULE = """
import sys
import importlib.abc

class Missing(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path=None, target=None):
        if name == "heteromega_amd._attention_host":
            raise ImportError("no such module here")

sys.meta_path.insert(0, Missing())
import torch
import heteromega_amd as hm
assert hm.packed_bytes(256, 128) > 0 and hm.rope_frequencies(64).numel() == 32
i, q = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 12 * 64), dtype=torch.float16)
for call in (lambda: hm.page_plan(hm.PagePlan(2, 4, 16, "cpu"), i, i, i[:, None], i, torch.zeros(4, dtype=torch.int64)),
             lambda: hm.qk_norm_rope(q[:, :512], q, hm.rope_frequencies(64), i, k_out=q[:, 512:640], kv_heads=2, head_dim=64)):
    try:
        call()
    except ImportError as e:
        assert "heteromega_amd/build.py" in str(e) and "no such module here" in str(e.__cause__), e
    else:
        raise AssertionError("a call without its compiled module")
"""


def test_the_package_needs_the_attention_module_for_attention_alone():
    res = subprocess.run([sys.executable, "-c", _WITHOUT_THE_ATTENTION_MODULE], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def test_the_library_alone_is_built_without_torchs_headers():
    # what was built without them before: the build script's option leaves every module out that is compiled against torch
    probe = """
import sys
sys.argv = ["build.py", "--no-shim"]
import runpy, subprocess
real = subprocess.run
def run(cmd, **kw):
    assert cmd[0] != "g++", cmd
    return subprocess.CompletedProcess(cmd, 0, "", "")
subprocess.run = run
import os
os.replace = lambda a, b: None
runpy.run_path("heteromega_amd/build.py", run_name="__main__")
"""
    res = subprocess.run([sys.executable, "-c", probe], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
