"""Arguments of the paged-serving entry points that would fault on the device, refused before any launch (no GPU)."""
from sunshape_b200 import _lib


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
