"""Host side of the drafted-token step at its edges (no GPU needed)."""

import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT


def test_tree_work_list_refuses_batches_whose_last_tile_passes_32_bits():
    """A key's number in an item, its drafted tokens and the tile's end included, is an int32."""
    from akv_b200.context_tree import tree_work_list

    for keys, new in ((2**31 - 1, 1), (2**31 - 64, 64), (2**31 - 150, 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            tree_work_list([0, keys], [0, new], 8, 1, True, 1)
    items, *_ = tree_work_list([0, 2**31 - 400], [0, 64], 8, 1, True, 1)
    assert items.dtype == np.int32 and (items[:, 4] >= 0).all() and (items[:, 5] > items[:, 4]).all()
    assert items[:, 5].max() == 2**31 - 336


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                          timeout=300)


BLOCK = """
import sys, importlib.abc
class No(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path=None, target=None):
        if name.endswith("._tensor_fields"):
            raise ImportError("not here")
sys.meta_path.insert(0, No())
"""


def test_the_package_works_without_the_module_that_torch_is_compiled_into():
    """Everything that needs the kernels' library alone imports and runs; the
    drafted-token step says what to build."""
    got = run(BLOCK + """
import torch
from akv_b200 import (_native, context_attention, context_drop, context_occurrence,
                      context_page_table, context_prefill, context_reposition, context_rope,
                      context_slots, context_tree)
assert _native.lib.akv_map_slots(None, None) == _native.AKV_ERR_INVALID
assert len(context_tree.tree_work_list([0, 500], [0, 4], 8, 8, True, 148)[0])
x = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
try:
    context_rope.qk_norm_rope(x, x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))
except ImportError as e:
    assert "akv_b200.build" in str(e) and "not here" in str(e), e
    print("refused")
""")
    assert got.returncode == 0 and got.stdout.strip() == "refused", got.stderr[-2000:]


def test_a_module_built_for_another_torch_is_not_used():
    got = run("""
import torch
torch.__version__ = torch.__version__ + ".other"
from akv_b200 import _native
try:
    _native.fields(1)
except ImportError as e:
    assert "another torch" in str(e), e
    print("refused")
""")
    assert got.returncode == 0 and got.stdout.strip() == "refused", got.stderr[-2000:]


def test_the_module_is_rebuilt_for_another_torch_or_python(tmp_path, monkeypatch):
    import sysconfig

    import torch

    from akv_b200 import build

    assert build.FIELDS.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    calls = []
    monkeypatch.setattr(build, "FIELDS", str(tmp_path / "_tensor_fields.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))

    def compile_(cmd, check):
        calls.append(cmd)
        open(build.FIELDS, "w").close()

    monkeypatch.setattr(build.subprocess, "run", compile_)
    build.build_fields()
    build.build_fields()
    assert len(calls) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_fields()
    build.build_fields()
    assert len(calls) == 2 and any("9.9.9" in part for part in calls[1])
    build.build_fields(force=True)
    assert len(calls) == 3


def test_the_polynomial_exponential_is_as_good_as_its_comment_says():
    """2^f on [-1/2, 1/2] by the kernel's constants: as a real polynomial, and in
    fp32 with one rounding per step, as the kernel's fused multiply-adds."""
    import os
    import re

    text = open(os.path.join(ROOT, "akv_b200", "csrc", "tree_attention.cu")).read()
    body = text[text.index("void exp2_pair"):]
    body = body[: body.index("\n}\n")]
    c = [float.fromhex(x) for x in re.findall(r"f2_pack\((0x[0-9a-fp.+-]+)f, ", body)] + [1.0]
    assert len(c) == 6
    f = np.linspace(-0.5, 0.5, 400001).astype(np.float32)
    want = np.exp2(f.astype(np.longdouble))
    real, rounded = np.longdouble(c[0]), np.full_like(f, c[0])
    for k in c[1:]:
        real = real * f + np.longdouble(k)
        # The product of two fp32 numbers is exact in 64 bits; the sum's own rounding there is
        # 2^-29 of one in fp32.
        rounded = (rounded.astype(np.float64) * f + k).astype(np.float32)
    assert np.abs(real / want - 1).max() < 1.1e-7
    assert np.abs(rounded / want - 1).max() < 1.7e-7 < 2 * 2.0**-23
