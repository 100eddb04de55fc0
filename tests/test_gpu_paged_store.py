"""A paged cache that holds 8 bits: what is written, what is read back, and the decode over it."""
import math

import pytest
import torch

import paged_reference as R
from pope_pytorch_b200 import PagedKVCache, PoPE, _native

pytestmark = pytest.mark.gpu
DEV = "cuda"
STORES = [torch.int8, torch.float8_e4m3fn]


def make(b, hk, d, dtype, store, longest, page=64, seed=0):
    width = -(-longest // page)
    cache = PagedKVCache(b, hk, d, num_pages=b * width + 3, page_size=page, max_seq_len=longest, dtype=dtype, device=DEV, store=store)
    cache.alloc.free = torch.randperm(b * width + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    return cache


def stored(cache, b):
    """(codes, scales) of k and v of sequence b, through the page table with torch."""
    pages, n = cache.alloc.table[b], cache.lens[b]
    got = []
    for codes, scales in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)):
        c = codes.view(torch.uint8)[pages].view(codes.dtype).float().permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
        got.append((c, scales[pages].permute(1, 0, 2).flatten(1, 2)[:, :n]))
    return got


def check_codes(x, codes, scales, store):
    """Nearest codes of x (hk, n, d): x * (M / A) carries two roundings of fp32, so a code may be off by that much more than half a step."""
    x, top = x.double(), R.TOP[store]
    amax = x.abs().amax(-1)
    # (the division in 64 bits: PyTorch divides a CUDA tensor by a number through the number's reciprocal)
    assert torch.equal(scales, (amax / top).float())
    y = x * (top / amax)[..., None]
    if store == torch.int8:
        half = torch.full_like(y, 0.5)
    else:
        half = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 4)
    assert ((codes.double() - y).abs() <= half + y.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("d,dtype,n", [(64, torch.float16, 1), (96, torch.bfloat16, 37), (128, torch.bfloat16, 200), (128, torch.float16, 1001), (64, torch.bfloat16, 2000)])
def test_rows_are_written_and_read_back(store, d, dtype, n):
    g = torch.Generator(device=DEV).manual_seed(n + d)
    b, hk = 2, 3
    cache = make(b, hk, d, dtype, store, n + 130)
    # (b, n, h, d) memory, seen as (b, h, n, d)
    k, v = (torch.randn(b, n, hk, d, device=DEV, generator=g).mul(torch.rand(b, n, hk, 1, device=DEV, generator=g) * 5).to(dtype).transpose(1, 2) for _ in range(2))
    one = torch.randn(hk, 5, d, device=DEV, generator=g).to(dtype)
    cache.append_to(1, one, one)       # the rows that follow start inside a page
    cache.append(k, v)
    assert _native.last_path() == "kv_write" and cache.seq_lens.tolist() == cache.lens == [n, n + 5]
    for i, first in ((0, 0), (1, 5)):
        for (codes, scales), x, got in zip(stored(cache, i), (k, v), cache.read(i)):
            check_codes(x[i], codes[:, first:], scales[:, first:], store)
            assert got.dtype == dtype and got.is_contiguous()
            assert torch.equal(got, (codes * scales[..., None]).to(dtype))
    part = cache.read(1, 3, n + 4)
    whole = cache.read(1)
    assert all(torch.equal(p, w[:, 3:n + 4]) for p, w in zip(part, whole))
    assert cache.read(0, n, n)[0].shape == (hk, 0, d)
    assert all(torch.equal(a, b_) for a, b_ in zip(cache.gather(0), cache.read(0)))
    assert _native.device_status() == 0


@pytest.mark.parametrize("page", [64, 192])
def test_a_16_bit_cache_reads_back_what_was_written(page):
    cache = make(2, 2, 96, torch.bfloat16, None, 500, page)
    k, v = (torch.randn(2, 2, 413, 96, device=DEV).bfloat16() for _ in range(2))
    cache.append(k, v)
    for i in range(2):
        assert torch.equal(cache.read(i)[0], k[i]) and torch.equal(cache.read(i, 60, 300)[1], v[i, :, 60:300])


@pytest.mark.parametrize("store", STORES)
def test_rows_out_of_the_ordinary(store):
    """Zeros, values next to the type's smallest, infinities and NaN: a row never touches its neighbours."""
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(1, 1, 8, 64, device=DEV, generator=g).bfloat16()
    x[0, 0, 0] = 0
    x[0, 0, 1] *= 1e-38          # below 2^-119
    x[0, 0, 2] *= 1e-34
    x[0, 0, 3, 7] = math.inf
    x[0, 0, 4, 0] = math.nan
    x[0, 0, 5] *= 1e37
    x[0, 0, 6] = -0.0
    x[0, 0, 6, 3] = -3e38
    cache = make(1, 1, 64, torch.bfloat16, store, 100)
    cache.append(x, x.neg())
    k, v = cache.read(0)
    assert not k[0, :2].any() and not v[0, :2].any()
    assert k[0, 3:5].isnan().all() and v[0, 3:5].isnan().all()
    for (codes, scales), want in zip(stored(cache, 0), (x, -x)):
        assert torch.isfinite(codes).all()
        keep = [2, 5, 6, 7]
        check_codes(want[0][:, keep], codes[:, keep], scales[:, keep], store)
    assert torch.isfinite(k[0, [0, 1, 2, 5, 6, 7]]).all()


CASES = [
    # lens, heads, key heads, d, r, dtype, store, page
    ([130, 1, 64], 4, 2, 64, 32, torch.float16, torch.int8, 64),
    ([63, 500], 4, 4, 128, 128, torch.bfloat16, torch.float8_e4m3fn, 128),
    ([300, 0, 129], 12, 2, 96, 48, torch.bfloat16, torch.int8, 192),
    ([1500], 17, 1, 128, 64, torch.float16, torch.float8_e4m3fn, 256),
    ([700], 8, 1, 128, 0, torch.bfloat16, torch.int8, 256),
    ([90, 400], 2, 2, 96, 8, torch.float16, torch.int8, 64),
    ([257], 40, 1, 64, 24, torch.bfloat16, torch.float8_e4m3fn, 64),
]


@pytest.mark.parametrize("lens,h,hk,d,r,dtype,store,page", CASES)
def test_decode(lens, h, hk, d, r, dtype, store, page):
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + h)
    cache = make(len(lens), hk, d, dtype, store, max(lens) + 9, page)
    for i, n in enumerate(lens):
        cache.append_to(i, *(torch.randn(hk, n, d, device=DEV, generator=g).to(dtype) for _ in range(2)))
    q = torch.randn(len(lens), h, 1, d, device=DEV, generator=g).to(dtype)
    nmax = max(lens)
    freqs = PoPE(r, heads=hk)(nmax).freqs.to(DEV) if r else torch.empty(nmax, 0, device=DEV)
    bias = -6 * torch.rand(hk, r, device=DEV, generator=g)
    out, lse = cache.decode(q, (freqs, bias), return_lse=True)
    assert out.shape == q.shape and lse.shape == q.shape[:2]
    held = [stored(cache, i) for i in range(len(lens))]
    values = [[c * s[..., None] for c, s in one] for one in held]
    want = R.attend(q, [x[0] for x in values], [x[1] for x in values], freqs, bias, lens, [1] * len(lens), d ** -0.5, store)
    R.check(out, want[0], want[2], want[3], lse[..., None], want[1])
    assert _native.device_status() == 0
