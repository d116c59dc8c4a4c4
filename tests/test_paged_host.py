"""Paged-serving entry points: what is refused before any launch (no GPU)."""
import ctypes

import pytest
import torch

from sunshape_b200 import _lib, paged


def _expect(rc, code, text):
    assert rc == code
    assert text in _lib.load_library().sunshape_last_error().decode()


def _rows(heads=2, data=16):
    return _lib.RowsDesc(data, 64, 64, 64, heads)


def test_norm_rotate_refusals():
    f = _lib.load_library().sunshape_norm_rotate
    rot = _lib.RotationDesc(16, 16, 16, 1, 1, 10, _lib.I64, 64, 0)
    _expect(f(None, None, None, None, None, None, 1, 1, 1, 1, 64, 1e-6, None, None), -1, "descriptor is NULL")
    _expect(f(_rows(), _rows(3), None, None, None, None, 1, 1, 1, 1, 64, 1e-6, None, None), -1, "same number of heads")
    _expect(f(_rows(), _rows(), None, _rows(), None, None, 1, 1, 1, 1, 64, 1e-6, None, None), -1, "an input and an output")
    _expect(f(_rows(), _rows(), None, None, None, None, 4, 1, 1, 1, 64, 1e-6, None, None), -1, "row dtype")
    _expect(f(_rows(), _rows(), 16, None, None, None, 1, 5, 1, 1, 64, 1e-6, None, None), -1, "weight dtype")
    _expect(f(_rows(), _rows(), None, None, None, None, 1, 1, -1, 1, 64, 1e-6, None, None), -1, "batch and length")
    _expect(f(_rows(), _rows(), None, None, None, None, 1, 1, 1, 1, 32, 1e-6, rot, None), -1, "rot_dim")
    rot.rot_dim, rot.position_dtype = 32, _lib.F32
    _expect(f(_rows(), _rows(), None, None, None, None, 1, 1, 1, 1, 32, 1e-6, rot, None), -1, "I32 or I64")
    rot.position_dtype, rot.cos = _lib.I32, None
    _expect(f(_rows(), _rows(), None, None, None, None, 1, 1, 1, 1, 32, 1e-6, rot, None), -1, "rotation pointer is NULL")
    assert f(_rows(), _rows(), None, None, None, None, 1, 1, 0, 1, 64, 1e-6, None, None) == 0


def test_append_refusals():
    f = _lib.load_library().sunshape_paged_append
    cd = _lib.CodecDesc(16, 16, None, 1, 64, 8, 256, 0, None)
    pg = _lib.PagesDesc(16, None, 16, 4, 2, 16, 64, _lib.BF16)
    assert f(cd, 256, pg, _rows(), _rows(), 0, 1, 16, 1, 1, None, None) == 0
    _expect(f(cd, 256, None, _rows(), _rows(), 1, 1, 16, 1, 1, None, None), -1, "page pool descriptor")
    _expect(f(cd, 256, pg, _rows(3), _rows(), 1, 1, 16, 1, 1, None, None), -1, "kv_heads")
    _expect(f(cd, 256, pg, _rows(), _rows(), 1, 1, None, 1, 1, None, None), -1, "slots pointer")
    for change, code, text in ((dict(page_size=8), -1, "page_size"), (dict(dtype=_lib.F32), -2, "BF16 or F16"),
                               (dict(value=24), -1, "16-byte aligned"), (dict(indices=None), -1, "pool pointer")):
        bad = _lib.PagesDesc(16, None, 16, 4, 2, 16, 64, _lib.BF16)
        for k, v in change.items():
            setattr(bad, k, v)
        _expect(f(cd, 256, bad, _rows(), _rows(), 1, 1, 16, 1, 1, None, None), code, text)
    _expect(f(_lib.CodecDesc(16, 16, None, 1, 64, 16, 256, 0, None), 256, pg, _rows(), _rows(), 1, 1, 16, 1, 1, None, None), -2,
            "block_dim 2, 4 or 8")
    _expect(f(_lib.CodecDesc(16, 16, None, 1, 64, 8, 300, 0, None), 256, pg, _rows(), _rows(), 1, 1, 16, 1, 1, None, None), -2,
            "256 codewords")
    _expect(f(_lib.CodecDesc(16, 16, 16, 1, 64, 8, 256, 2, None), 256, pg, _rows(), _rows(), 1, 1, 16, 1, 1, None, None), -1,
            "heavy pool")


def test_attention_refusals():
    lib = _lib.load_library()
    f = lib.sunshape_paged_attention
    cd = _lib.CodecDesc(16, 16, None, 1, 64, 8, 256, 0, None)
    pg = _lib.PagesDesc(16, None, 16, 4, 2, 16, 64, _lib.BF16)

    def call(codec=cd, pages=pg, query=None, batch=1, query_len=1, table=16, cols=2, lens=16, prefix=None, prefix_len=0,
             ws=256, size=1 << 24):
        return f(codec, 256, pages, query or _rows(4), batch, query_len, table, 2, cols, lens, prefix, prefix_len, 1.0, 1, 16,
                 ws, size, None)

    assert call(batch=0) == 0 and call(query_len=0) == 0
    _expect(call(query=_rows(3)), -1, "divisible by kv-head")
    _expect(call(batch=-1), -1, "negative size")
    _expect(call(lens=None), -1, "pointer is NULL")
    _expect(call(prefix_len=5), -1, "pointer is NULL")
    _expect(call(ws=128), -4, "workspace")
    _expect(call(size=16), -4, "workspace")
    _expect(call(cols=1 << 29), -2, "2^30 tokens")
    _expect(call(codec=_lib.CodecDesc(16, 16, None, 1, 96, 8, 256, 0, None)), -2, "head_dim 64 or 128")
    _expect(call(pages=_lib.PagesDesc(16, None, 16, 4, 2, 16, 72, _lib.BF16)), -2, "value_dim 64 or 128")
    assert lib.sunshape_paged_attention_workspace_bytes(4, 8, 2, 1, 64, 100, 16, 0) > 0


def test_tables_refusals():
    lib = _lib.load_library()
    cd = _lib.CodecDesc(16, 16, None, 2, 64, 8, 256, 0, None)
    n = lib.sunshape_paged_tables_bytes(cd)
    assert n > 0
    _expect(lib.sunshape_paged_tables(cd, None, n, None), -1, "tables buffer")
    _expect(lib.sunshape_paged_tables(cd, 256, n - 1, None), -1, "tables buffer")
    _expect(lib.sunshape_paged_tables(cd, 128, n, None), -1, "tables buffer")
    assert lib.sunshape_paged_tables_bytes(_lib.CodecDesc(16, 16, None, 2, 64, 8, 300, 0, None)) == -2


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.norm_rotate(torch.zeros(1, 2, 3, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.SunShapePagedCache(None, torch.zeros(1, 1, 16, 8, dtype=torch.uint8), torch.zeros(1, 1, 16, 64))


def test_rotary_table_is_exact_at_far_positions():
    import math

    cos, sin = paged.rotary_table(200001, 64)
    assert cos.shape == (200001, 32) and cos.dtype == torch.float32
    for p, i in ((200000, 0), (131071, 3), (99999, 31)):
        a = p * 10000.0 ** (-2 * i / 64)
        assert abs(float(cos[p, i]) - math.cos(a)) <= 2.0 ** -24 and abs(float(sin[p, i]) - math.sin(a)) <= 2.0 ** -24


def test_slots_of_positions():
    cache = object.__new__(paged.SunShapePagedCache)
    cache.indices = torch.zeros(1, 1, 16, 8)
    table = torch.tensor([[5, 2], [7, 0]], dtype=torch.int32)
    got = paged.SunShapePagedCache.slots(cache, table, torch.tensor([[0, 17, -1], [15, 16, 31]]))
    assert got.tolist() == [[80, 33, -1], [127, 0, 15]]
    # beyond the table: a slot outside the pool of one page, for the append to record
    got = paged.SunShapePagedCache.slots(cache, table, torch.tensor([[32, 5], [10 ** 9, -1]]))
    assert got.tolist() == [[16, 85], [16, -1]]
    assert paged.SunShapePagedCache.slots(cache, table[:, :0], torch.tensor([[0, -1], [3, 4]])).tolist() == [[16, -1], [16, 16]]
