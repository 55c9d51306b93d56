"""CPU: without libvoltattn_torch.so, with one that does not load, or with one that was built for another PyTorch,
importing the ops warns where there is a GPU and leaves every op as it is (append_rope's and attend_paged's plain
calls then go through Python, as the calls that are not plain always do)."""
import re
import shutil
import subprocess
import sys
import warnings
from pathlib import Path

import pytest
import torch

import voltattn_amd
from voltattn_amd import torch_ops

PKG = Path(voltattn_amd.__file__).parent
CHILD = """
import warnings
import torch
torch.cuda.device_count = lambda: 1
with warnings.catch_warnings(record=True) as w:
    warnings.simplefilter("always")
    import voltattn_amd.torch_ops
print(*(str(x.message) for x in w if "voltattn" in str(x.message)))
h = lambda *s: torch.empty(s, dtype=torch.float16, device="meta")
i = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")
ops = torch.ops.voltattn
assert ops.prefill(h(5, 4, 64), h(5, 2, 64), h(5, 2, 64), i(2)).shape == (5, 4, 64)
assert ops.decode(h(4, 64), h(4, 7, 64), h(4, 7, 64), None, None, "f16+").shape == (4, 64)
pool = torch.empty((2, 2, 64, 64), dtype=torch.float8_e4m3fn, device="meta")
assert ops.attend_paged(h(5, 4, 64), pool, pool, h(2, 2, 2), h(2, 2, 2), i(1, 2), i(2), i(1), "b8+", 128, 32).shape == (5, 4, 64)
for op in (ops.attend_paged, ops.append_rope):
    assert torch._C._dispatch_has_computed_kernel_for_dispatch_key(op._qualified_op_name, "CUDA")
"""


@pytest.mark.parametrize("what", ["none", "junk", "of another PyTorch", "broken"])
def test_import_without_it(tmp_path, what):
    pkg = tmp_path / "voltattn_amd"
    pkg.mkdir()
    for p in PKG.glob("*.py"):
        shutil.copy(p, pkg / p.name)
    (pkg / "libvoltattn_hip.so").symlink_to(PKG / "libvoltattn_hip.so")
    out = pkg / "libvoltattn_torch.so"
    built = (PKG / "libvoltattn_torch.so").read_bytes()
    mark = b"voltattn calls for PyTorch " + re.match(r"\d+\.\d+\.\d+", torch.__version__)[0].encode() + b"\0"
    assert built.count(mark) == 1
    if what == "junk":
        out.write_bytes(b"\0" * 64)
    elif what == "of another PyTorch":
        out.write_bytes(built.replace(mark, mark.replace(b"PyTorch 2", b"PyTorch 1")))
    elif what == "broken":
        out.write_bytes(b"\x7fELF" + mark)
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=tmp_path, env={"PATH": "/usr/bin:/bin", "PYTHONPATH": str(tmp_path), "HOME": str(tmp_path)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert {"none": "is not built", "broken": "does not load"}.get(what, "was built for another PyTorch") in r.stdout


def test_without_a_gpu_nothing_is_said(tmp_path, monkeypatch):
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 0)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        torch_ops._load_calls(tmp_path / "none.so")
