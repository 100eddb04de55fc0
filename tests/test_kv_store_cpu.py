"""The paged cache's 8-bit store, chunks and rollback as a Python object (no GPU; a recorder stands where the binding is called):
bookkeeping and refusals, which change nothing."""
import copy

import pytest
import torch

from pope_pytorch_b200 import PagedKVCache, kv_cache


class Recorder:
    def __init__(self):
        self.maps, self.appends, self.attended, self.reads = [], [], [], []

    def Pages(self, *tensors):
        return tensors

    def kv_map(self, pages, index, value):
        self.maps.append((list(index), list(value)))

    def kv_append(self, pages, k, v, row):
        self.appends.append(row)

    def kv_read(self, pages, row, first, n, bf16):
        self.reads.append((row, first, n, bf16))

    def kv_attend(self, pages, q, freqs, bias, counts, scale, nk, want_lse):
        self.attended.append((counts, scale, nk))
        return q, q[..., 0]


@pytest.fixture
def ops(monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(kv_cache.N, "_ops", lambda: recorder)
    return recorder


def make(store=None, **over):
    return PagedKVCache(3, 2, 64, **{**dict(num_pages=8, page_size=64, max_seq_len=256, device="cpu", store=store), **over})


def rows(n, dtype=torch.bfloat16):
    return torch.randn(2, n, 64).to(dtype)


@pytest.mark.parametrize("store", [torch.int8, torch.float8_e4m3fn])
def test_the_pages_hold_codes_and_scales(ops, store):
    cache = make(store)
    assert cache.k_pages.dtype == cache.v_pages.dtype == store and cache.dtype == torch.bfloat16
    assert cache.k_scales.shape == cache.v_scales.shape == (8, 2, 64) and cache.k_scales.dtype == torch.float32
    assert len(cache._pages()) == 6
    twin = copy.deepcopy(cache)
    assert twin.store == store and twin.k_scales.data_ptr() != cache.k_scales.data_ptr()
    assert len(make()._pages()) == 4 and make().k_scales is None and make(torch.bfloat16).store is None


@pytest.mark.parametrize("store", [torch.float16, torch.uint8, torch.float32, torch.float8_e5m2])
def test_other_stores_are_refused(store):
    with pytest.raises(TypeError):
        make(store)


def test_rollback_returns_pages_and_lengths(ops):
    cache = make()
    cache.append_to(0, rows(130), rows(130))
    cache.append_to(2, rows(64), rows(64))
    held = list(cache.alloc.table[0])
    del ops.maps[:]
    cache.rollback([2, 0, 1])
    assert cache.lens == [128, 0, 63] and cache.alloc.table[0] == held[:2] and len(cache.alloc.table[2]) == 1
    assert ops.maps == [([-1, -3], [128, 63])]
    cache.append_to(0, rows(1), rows(1))
    assert cache.alloc.table[0] == held           # the page that was given back comes again
    cache.rollback([129, 0, 63])
    assert cache.lens == [0, 0, 0] and len(cache.alloc.free) == 8
    cache.rollback(0)
    assert len(ops.maps) == 3                     # (two rollbacks and the page of the append)


@pytest.mark.parametrize("counts", [[1, 0], [0, 1, 0], -1, 71, [0, 0, 71]])
def test_rollbacks_that_are_refused(ops, counts):
    cache = make()
    cache.append_to(0, rows(70), rows(70))
    cache.append_to(2, rows(70), rows(70))
    before = (cache.lens, copy.deepcopy(cache.alloc.table), list(cache.alloc.free), list(ops.maps))
    with pytest.raises(ValueError):
        cache.rollback(counts)
    assert before == (cache.lens, cache.alloc.table, cache.alloc.free, ops.maps)


def test_reads(ops):
    cache = make(torch.int8)
    cache.append_to(1, rows(70), rows(70))
    cache.read(1), cache.read(-2, 3, 9), cache.read(1, 70), cache.read(0)
    assert ops.reads == [(1, 0, 70, True), (1, 3, 6, True), (1, 70, 0, True), (0, 0, 0, True)]
    for b, lo, hi in ((1, 0, 71), (1, 9, 3), (1, -1, 5), (3, 0, 0), (0, 0, 1)):
        with pytest.raises(IndexError):
            cache.read(b, lo, hi)
    assert len(ops.reads) == 4


def test_chunks(ops):
    cache = make()
    cache.append_to(1, rows(70), rows(70))
    emb, q = (torch.zeros(80, 32), torch.zeros(2, 32)), torch.zeros(3, 4, 5, 64).bfloat16()
    counts = torch.tensor([1, 2, 3], dtype=torch.int32)
    cache.attend(q, emb)
    cache.attend(q, emb, counts=counts, softmax_scale=0.5)
    assert ops.attended[0] == (None, 64 ** -0.5, 70) and ops.attended[1][0] is counts and ops.attended[1][1:] == (0.5, 70)
    for bad, err in ((dict(q=q[:2]), ValueError), (dict(q=q[..., :32]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(q=q[:, :0]), ValueError), (dict(q=q[0]), ValueError),
                     (dict(q=q.half()), TypeError), (dict(pos_emb=(emb[0][:69], emb[1])), ValueError),
                     (dict(pos_emb=(emb[0][None], emb[1])), ValueError), (dict(counts=counts.long()), TypeError),
                     (dict(counts=counts[:2]), ValueError), (dict(counts=counts[:, None]), ValueError)):
        with pytest.raises(err):
            cache.attend(**{**dict(q=q, pos_emb=emb), **bad})
    assert len(ops.attended) == 2
    cache = make(torch.int8)
    cache.decode(q[:, :, :1], emb)
    assert ops.attended[2] == (None, 64 ** -0.5, 1)
