"""The tables that the paged kernels read of a codec: when they are derived, what waits for what, where they lie."""
import pytest
import torch

from sunshape_b200 import _lib, paged


class _Codec:
    """A codec's side of the tables, on the CPU."""

    mode = "profileperm_mixed_precision"
    _desc_cache = None
    _paged_tables = None
    _paged_retired = ()
    heavy = 2

    def __init__(self):
        self.centroids = torch.zeros(2, 8, 256, 8)

    n_codebooks = property(lambda self: self.centroids.shape[0])

    def kernel_desc(self):
        if self._desc_cache is None:
            self.log.append("read the codec")
            perm, mask = torch.arange(64), torch.zeros(8, dtype=torch.uint8)
            mask[:self.heavy] = 1
            desc = _lib.codec_desc(self.centroids, perm, mask, self.heavy, 64, 8)
            self._desc_cache = (desc, (self.centroids, perm, mask, None), self.heavy)
        return self._desc_cache

    def invalidate(self):
        self._desc_cache = None
        paged.renew_after_edit(self)


@pytest.fixture
def codec(monkeypatch):
    c = _Codec()
    c.log, c.capturing = [], False
    monkeypatch.setattr(_lib, "require_cuda", lambda t: t.device)
    monkeypatch.setattr(_lib, "paged_tables_bytes", lambda desc: 4096)
    monkeypatch.setattr(_lib, "paged_tables", lambda desc, out: c.log.append("fill"))
    monkeypatch.setattr(torch.cuda, "device", lambda d: __import__("contextlib").nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: c.log.append("wait"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: c.capturing)
    return c


def test_waits_before_and_after(codec):
    """Edits of the codec and readers of the old tables come before the fill, every reader of the new ones after it."""
    paged.renew_tables(codec)
    assert codec.log == ["wait", "read the codec", "fill", "wait"]
    codec.log.clear()
    codec.invalidate()
    assert codec.log == ["wait", "read the codec", "fill", "wait"]


def test_addresses_stay(codec):
    tables = paged.renew_tables(codec)
    at = [t.data_ptr() for t in (tables.buffer, tables.perm, tables.mask)]
    codec.centroids = codec.centroids + 1
    codec.invalidate()
    assert codec._paged_tables is tables
    assert at == [t.data_ptr() for t in (tables.buffer, tables.perm, tables.mask)]
    assert [tables.desc.permutation, tables.desc.heavy_mask] == at[1:]
    # another number of dense blocks: graphs captured with the old number keep a mask that has it
    codec.heavy = 3
    codec.invalidate()
    assert codec._paged_tables is not tables and tables in codec._paged_retired
    assert tables.mask.tolist() == [1, 1, 0, 0, 0, 0, 0, 0]
    assert codec._paged_tables.mask.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]


def test_not_during_a_capture(codec):
    codec.capturing = True
    with pytest.raises(RuntimeError, match="captured"):
        paged.renew_tables(codec)
    assert codec.log == []
    codec.capturing = False
    tables = paged.renew_tables(codec)
    codec.log.clear()
    codec.capturing = True
    codec.invalidate()                       # left to the next call, which a capture refuses
    assert codec.log == [] and tables.made is not codec._desc_cache


def test_another_shape_waits_for_the_next_call(codec):
    paged.renew_tables(codec)
    codec.log.clear()
    codec.centroids = torch.zeros(2, 8, 300, 8)
    codec.invalidate()
    assert codec.log == []


def test_slots_of_table_entries_that_name_no_page():
    """An entry of -1 (no page yet) is no padding, not even in a page's last row, where it would come out as -1."""
    cache = object.__new__(paged.SunShapePagedCache)
    cache.indices = torch.zeros(4, 1, 16, 8)
    table = torch.tensor([[2, -1], [-3, 3]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([[15, 16, 31, -1], [0, 15, 31, 47]]))
    assert got.tolist() == [[47, 64, 64, -1], [64, 64, 63, 64]]
