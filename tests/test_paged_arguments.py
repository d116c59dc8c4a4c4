"""Arguments of the paged-serving entry points that would fault on the device, refused before any launch (no GPU)."""
import os
import re

import pytest
import torch

from sunshape_b200 import _lib, paged


def _expect(rc, code, text):
    assert rc == code
    assert text in _lib.load_library().sunshape_last_error().decode()


def _rows(heads=2, data=16):
    return _lib.RowsDesc(data, 64, 64, 64, heads)


def test_attention_output_alignment():
    """Results are stored eight bytes at a time: a 16-bit view that begins at an odd element is refused."""
    f = _lib.load_library().sunshape_paged_attention
    cd = _lib.CodecDesc(16, 16, None, 1, 64, 8, 256, 0, None)
    pg = _lib.PagesDesc(16, None, 16, 4, 2, 16, 64, _lib.BF16)
    for out in (16 + 2, 16 + 4, 16 + 6):
        _expect(f(cd, 256, pg, _rows(4), 1, 1, 16, 2, 2, 16, None, 0, 1.0, 1, out, 256, 1 << 24, None), -1, "8-byte aligned")


def test_rotation_table_without_rows():
    """A position outside the table reads row 0 in its place: a table has one."""
    lib = _lib.load_library()
    rot = _lib.RotationDesc(16, 16, 16, 1, 1, 0, _lib.I64, 64, 0)
    _expect(lib.sunshape_norm_rotate(_rows(), _rows(), None, None, None, None, _lib.BF16, _lib.BF16, 1, 1, 64, 1e-6, rot, None),
            -1, "table has no rows")
    cd = _lib.CodecDesc(16, 16, None, 1, 64, 8, 256, 0, None)
    pg = _lib.PagesDesc(16, None, 16, 4, 2, 16, 64, _lib.BF16)
    _expect(lib.sunshape_paged_append(cd, 256, pg, _rows(), _rows(), 1, 1, 16, 1, 1, rot, None), -1, "table has no rows")
    # nothing to rotate: nothing is read
    assert lib.sunshape_norm_rotate(_rows(), _rows(), None, None, None, None, _lib.BF16, _lib.BF16, 0, 1, 64, 1e-6, rot, None) == 0


def test_no_launch_status_is_dropped():
    """A kernel that reads what another one wrote must not be launched where that one was refused: each launch of the paged
    entry points is checked before the next."""
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    for name in ("paged_append.cu", "paged_attention.cu", "paged_attention_kernel.cuh", "paged_prefix.cuh"):
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        assert not re.findall(r"^\s*(?:cudaLaunchKernelEx|ready_kernel|launch<.*>)\(.*", text, re.M), name
        after = re.findall(r"<<<[^;]*;\s*(.*)", text)
        assert all("launch_status" in line or line.startswith("SUNSHAPE_TABLES_CASE") for line in after), (name, after)


def test_gradients_are_not_dropped_silently():
    """No paged call has a backward pass: an input that wants gradients is refused where they are recorded."""
    x, w = torch.zeros(1, 2, 1, 64), torch.ones(64)
    cases = [lambda g: paged.norm_rotate(g(x)), lambda g: paged.norm_rotate(x, g(x)), lambda g: paged.norm_rotate(x, q_weight=g(w)),
             lambda g: paged.norm_rotate(x, x, k_weight=g(w)), lambda g: paged.append_paged(None, g(x), x, None),
             lambda g: paged.append_paged(None, x, g(x), None), lambda g: paged.paged_attention(None, g(x), None, None)]
    for call in cases:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call(lambda t: t.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(Exception) as other:      # CPU tensors, or no cache
            call(lambda t: t.clone().requires_grad_())
        assert "no backward pass" not in str(other.value)
