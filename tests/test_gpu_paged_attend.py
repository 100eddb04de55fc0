"""Attention of a chunk of new tokens over the paged cache, 16-bit and 8-bit, against the definition in 64 bits."""
import math

import pytest
import torch

import paged_reference as R
from pope_pytorch_b200 import PagedKVCache, PoPE, _native, flash_attn_with_pope
from test_gpu_paged_store import make, stored

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, F8, BF, HF = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16


def fill(cache, lens, g):
    for i, n in enumerate(lens):
        cache.append_to(i, *(torch.randn(cache.kv_heads, n, cache.head_dim, device=DEV, generator=g).to(cache.dtype) for _ in range(2)))


def held(cache):
    if cache.store is None:
        return [[t.float() for t in cache.gather(i)] for i in range(cache.batch)]
    return [[c * s[..., None] for c, s in stored(cache, i)] for i in range(cache.batch)]


def table(r, hk, n, g):
    freqs = PoPE(r, heads=hk)(n).freqs.to(DEV) if r else torch.empty(n, 0, device=DEV)
    return freqs, -6 * torch.rand(hk, r, device=DEV, generator=g)


CASES = [
    # lens, new, counts, heads, key heads, d, r, dtype, store, page
    ([200, 70], 5, None, 4, 2, 64, 32, BF, None, 64),                 # a few tokens of each
    ([131, 64, 300], 7, [7, 1, 3], 4, 4, 128, 64, HF, None, 128),     # ragged
    ([3, 0, 40], 9, None, 2, 1, 96, 48, BF, None, 64),                # shorter than the chunk, and empty
    ([150, 99], 33, [0, 33], 8, 2, 128, 128, BF, None, 64),           # a sequence without new tokens
    ([260], 130, None, 4, 1, 128, 64, HF, None, 256),                 # several row blocks of one key head
    ([129], 129, None, 4, 2, 64, 64, BF, None, 64),                   # the whole sequence is new
    ([385, 200], 70, [70, 41], 6, 2, 96, 96, HF, None, 192),
    ([500], 1, None, 4, 4, 128, 64, BF, None, 64),                    # one token
    ([100], 20, None, 3, 3, 64, 0, BF, None, 64),                     # nothing rotated
    ([100], 40, None, 5, 1, 128, 24, HF, None, 64),                   # widths that are no multiple of 16
    ([90, 30], 50, [50, 30], 2, 2, 96, 8, BF, None, 64),
    ([200, 70], 5, None, 4, 2, 64, 32, BF, I8, 64),
    ([131, 64, 300], 7, [7, 1, 3], 4, 4, 128, 64, HF, F8, 128),
    ([3, 0, 40], 9, None, 2, 1, 96, 48, BF, I8, 64),
    ([260], 130, None, 4, 1, 128, 64, HF, I8, 256),
    ([385, 200], 70, [70, 41], 6, 2, 96, 96, BF, F8, 192),
    ([100], 40, None, 5, 1, 128, 24, HF, I8, 64),
    ([129], 129, None, 4, 2, 64, 64, BF, F8, 64),
    # more than 256 rows of a key head
    ([300, 150], 100, [100, 60], 8, 2, 96, 48, HF, None, 64),
    ([400], 300, None, 1, 1, 64, 0, BF, None, 64),
    ([310, 129], 150, [1, 150], 4, 2, 128, 128, BF, None, 128),
    ([290, 64], 290, None, 2, 2, 64, 24, BF, F8, 64),
    ([200], 90, None, 6, 2, 96, 8, HF, I8, 192),
    ([333], 100, None, 4, 1, 128, 64, BF, I8, 256),
    # 17 to 256 of them
    ([200, 100], 20, [20, 9], 4, 4, 96, 96, BF, F8, 64),
    ([500], 64, None, 4, 1, 128, 128, HF, I8, 128),
    ([70, 65, 64], 18, None, 1, 1, 64, 0, HF, F8, 64),
]


@pytest.mark.parametrize("lens,new,counts,h,hk,d,r,dtype,store,page", CASES)
def test_attend(lens, new, counts, h, hk, d, r, dtype, store, page):
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + new)
    cache = make(len(lens), hk, d, dtype, store, max(lens) + 70, page, seed=new)
    fill(cache, lens, g)
    q = torch.randn(len(lens), h, new, d, device=DEV, generator=g).to(dtype)
    emb = table(r, hk, max(lens) + 3, g)
    given = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, emb, counts=given, return_lse=True)
    assert _native.device_status() == 0
    vals = held(cache)
    want = R.attend(q, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], lens, counts or [new] * len(lens), d ** -0.5, store)
    R.check(out, want[0], want[2], want[3], lse, want[1])
    for i, c in enumerate(counts or []):
        assert not out[i, :, c:].any()


@pytest.mark.parametrize("store", [None, I8])
def test_chunks_give_what_one_call_over_the_whole_prompt_gives(store):
    """A prompt in chunks, then tokens one by one: append and attend / decode as a serving loop uses them."""
    b, h, hk, d, r = 2, 4, 2, 64, 32
    g = torch.Generator(device=DEV).manual_seed(9)
    n = 230
    k, v, q = (torch.randn(b, x, n, d, device=DEV, generator=g).half() for x in (hk, hk, h))
    emb = table(r, hk, n, g)
    cache = make(b, hk, d, HF, store, n)
    outs, at = [], 0
    for m in (100, 1, 64, 37, 20):
        cache.append(k[:, :, at:at + m], v[:, :, at:at + m])
        outs.append(cache.attend(q[:, :, at:at + m], emb))
        at += m
    while at < n:
        cache.append(k[:, :, at:at + 1], v[:, :, at:at + 1])
        outs.append(cache.decode(q[:, :, at:at + 1], emb))
        at += 1
    vals = held(cache)
    want = R.attend(q, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], [n] * b, [n] * b, d ** -0.5, store)
    R.check(torch.cat(outs, 2), want[0], want[2], want[3])


@pytest.mark.parametrize("store", [None, I8, F8])
def test_what_is_not_a_key_never_counts(store):
    """Pages whose unused rows hold infinities and NaN from somebody before, and a rollback that leaves such rows behind."""
    g = torch.Generator(device=DEV).manual_seed(4)
    lens, new, h, hk, d, r = [70, 129], 6, 4, 2, 128, 64
    cache, clean = (make(2, hk, d, BF, store, 400, seed=2) for _ in range(2))
    bad = torch.full((2, hk, 300, d), math.nan, device=DEV).bfloat16()
    bad[:, :, ::2] = math.inf
    cache.append(bad, bad)
    cache.rollback(300)
    for c in (cache, clean):
        fill(c, lens, torch.Generator(device=DEV).manual_seed(8))
    q = torch.randn(2, h, new, d, device=DEV, generator=g).bfloat16()
    emb = table(r, hk, 200, g)
    for rows in (q, q[:, :, :1], q.repeat(1, 1, 6, 1), q.repeat(1, 1, 25, 1)):
        got, want = cache.attend(rows, emb), clean.attend(rows, emb)
        assert torch.isfinite(got).all() and torch.equal(got, want)
    cache.append(bad[:, :, :3], bad[:, :, :3])
    assert cache.attend(q, emb)[:, :, -3:].isnan().any()
    cache.rollback([3, 3])
    assert cache.lens == lens and cache.seq_lens.tolist() == lens
    assert torch.equal(cache.attend(q, emb), clean.attend(q, emb))


@pytest.mark.parametrize("store", [None, I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new", [3, 30, 200])
def test_later_tokens_do_not_reach_earlier_rows(store, dtype, new):
    """Infinities and NaN in k and v of a token: the rows before it are untouched, to the bit; it and the rows behind it are not finite."""
    g = torch.Generator(device=DEV).manual_seed(new)
    h, hk, d, r, n = 4, 2, 128, 64, 333
    k, v = (torch.randn(1, hk, n, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(1, h, new, d, device=DEV, generator=g).to(dtype)
    emb = table(r, hk, n, g)

    def run(k, v):
        cache = make(1, hk, d, dtype, store, n, seed=1)
        cache.append(k, v)
        return cache.attend(q, emb)

    want = run(k, v)
    bad = n - 1 - new // 3          # seen by the last rows alone
    first = new - 1 - new // 3
    for what, value in (("k", math.nan), ("v", math.nan), ("v", math.inf), ("v", -math.inf)):
        kk, vv = k.clone(), v.clone()
        (kk if what == "k" else vv)[:, 1, bad, 5 if what == "v" else slice(None)] = value
        got = run(kk, vv)
        assert torch.equal(got[:, :, :first], want[:, :, :first])
        assert torch.equal(got[:, 0::2], want[:, 0::2])                 # the other key head's
        hit = got[:, 1::2, first:]
        if store is not None or what == "k":                            # an 8-bit row with such a value is NaN as a whole
            assert hit.isnan().all()
        else:
            assert (hit[..., 5].isnan().all() if math.isnan(value) else (hit[..., 5] == value).all())
            rest = torch.arange(d, device=DEV) != 5
            assert torch.equal(hit[..., rest], want[:, 1::2, first:][..., rest])


@pytest.mark.parametrize("store", [None, I8])
@pytest.mark.parametrize("new", [4, 40, 150])
def test_layouts_and_scales(store, new):
    g = torch.Generator(device=DEV).manual_seed(new)
    h, hk, d, r = 4, 2, 64, 32
    cache = make(2, hk, d, HF, store, 300)
    fill(cache, [200, 260], g)
    emb = table(r, hk, 300, g)
    wide = torch.randn(2, new, h, d + 3, device=DEV, generator=g).half()
    q = wide[..., 1:1 + d].transpose(1, 2)          # rows that start on no 16-byte boundary, (b, n, h, d) memory
    want = cache.attend(q.contiguous(), emb)
    assert torch.equal(cache.attend(q, emb), want)
    shared = q[:1, :1].expand(2, h, new, d)
    assert torch.equal(cache.attend(shared, emb), cache.attend(shared.contiguous(), emb))
    vals = held(cache)
    for scale in (0.02, 1.0, 0.0, -0.1):
        ref = R.attend(q[:, :, -3:], [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], [200, 260], [3, 3], scale, store)
        R.check(cache.attend(q, emb, softmax_scale=scale)[:, :, -3:], ref[0], ref[2], ref[3])


@pytest.mark.parametrize("store", [None, I8, F8])
@pytest.mark.parametrize("new", [2, 40, 135])
def test_magnitudes_beyond_fp16(store, new):
    """bf16 keys up to 3e5 against small queries, queries up to 3e5 against small keys, values from 1e-30 to 1e30."""
    g = torch.Generator(device=DEV).manual_seed(new)
    hk, d, r, n = 2, 64, 32, 150
    k = torch.randn(1, hk, n, d, device=DEV, generator=g)
    v = torch.randn(1, hk, n, d, device=DEV, generator=g)
    q = torch.randn(1, 4, new, d, device=DEV, generator=g)
    emb = table(r, hk, n, g)
    rows = torch.arange(n, device=DEV)
    for dk, dq, dv in ((1e5, 1e-5, 1.0), (1e-5, 1e5, 1e30), (1.0, 1.0, 1e-30), (1.0, 1.0, 1e30)):
        cache = make(1, hk, d, BF, store, n)
        many = (rows % 3 == 1)[:, None]
        cache.append((torch.where(many, k * dk, k)).bfloat16(), (v * dv).bfloat16())
        qq = (q * dq).bfloat16()
        vals = held(cache)
        ref = R.attend(qq, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], [n], [new], 0.125, store)
        got = cache.attend(qq, emb).double() / dv
        R.check(got, ref[0] / dv, ref[2] / dv, ref[3] / dv)


def test_counts_out_of_range_are_clamped_and_no_rows_are_none():
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = make(2, 1, 64, BF, None, 200)
    fill(cache, [100, 50], g)
    emb = table(32, 1, 200, g)
    q = torch.randn(2, 2, 8, 64, device=DEV, generator=g).bfloat16()
    got = cache.attend(q, emb, counts=torch.tensor([1 << 30, -5], dtype=torch.int32, device=DEV))
    assert torch.equal(got[0], cache.attend(q, emb)[0]) and not got[1].any()
    assert cache.attend(q[:, :, :0], emb).shape == (2, 2, 0, 64)


@pytest.mark.parametrize("new", [3, 40, 150])
def test_a_page_outside_the_pool_is_reported_not_read(new):
    g = torch.Generator(device=DEV).manual_seed(2)
    for store in (None, I8):
        cache = make(2, 2, 64, BF, store, 300)
        fill(cache, [200, 250], g)
        emb = table(32, 2, 300, g)
        q = torch.randn(2, 4, new, 64, device=DEV, generator=g).bfloat16()
        want = cache.attend(q, emb)
        good = int(cache.page_table[0, 1])
        for wrong in (1 << 30, -1):
            cache.page_table[0, 1] = wrong
            assert torch.equal(cache.attend(q, emb)[1], want[1])
            assert _native.device_status() & 2
            _native.clear_device_status()
        cache.page_table[0, 1] = good
        assert torch.equal(cache.attend(q, emb), want) and _native.device_status() == 0


@pytest.mark.parametrize("new,store", [(1, I8), (5, None), (90, None), (90, F8), (140, None), (140, I8)])
def test_captured_calls_follow_the_cache(new, store):
    """Append and attend in a graph: replays see the lengths and the rows of the moment."""
    g = torch.Generator(device=DEV).manual_seed(3)
    h, hk, d, r = 4, 2, 128, 64
    cache, twin = (make(2, hk, d, BF, store, 700, 256, seed=6) for _ in range(2))
    for c in (cache, twin):
        fill(c, [120, 180], torch.Generator(device=DEV).manual_seed(11))
    emb = table(r, hk, 700, g)
    q, k, v = (torch.randn(2, x, new, d, device=DEV, generator=g).bfloat16() for x in (h, hk, hk))
    twin.append(k, v)
    want = twin.attend(q, emb)

    def turn():
        cache.append(k, v)
        out = cache.attend(q, emb)
        cache.rollback(new)
        return out

    assert torch.equal(turn(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = turn()
    for _ in range(2):
        q.normal_(generator=g), k.normal_(generator=g), v.normal_(generator=g)
        twin.rollback(new)
        twin.append(k, v)
        want = twin.attend(q, emb)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert _native.device_status() == 0


def test_calls_in_a_row_and_on_another_stream_give_the_same():
    g = torch.Generator(device=DEV).manual_seed(13)
    cache = make(3, 4, 128, BF, I8, 3000, 256)
    fill(cache, [2900, 1000, 300], g)
    emb = table(64, 4, 3000, g)
    qs = [torch.randn(3, 8, n, 128, device=DEV, generator=g).bfloat16() for n in (1, 6, 64, 200)]   # every kernel, with parts to merge
    want = [cache.attend(q, emb).clone() for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        assert all(torch.equal(cache.attend(q, emb), w) for q, w in zip(qs, want))
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(10):
        got = []
        for s, q in zip(streams, qs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(cache.attend(q, emb))
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


@pytest.mark.parametrize("store", [I8, None])
def test_a_pool_whose_offsets_pass_32_bits(store):
    """Pages at the far end of a pool of more than 2^32 bytes (and 2^31 values)."""
    size = 1 if store else 2
    pages = (1 << 32) // (8 * 256 * 128 * size) + 40
    cache = PagedKVCache(1, 8, 128, num_pages=pages, page_size=256, max_seq_len=1024, dtype=BF, device=DEV, store=store)
    small = PagedKVCache(1, 8, 128, num_pages=4, page_size=256, max_seq_len=1024, dtype=BF, device=DEV, store=store)
    cache.alloc.free = [3, pages - 1, pages - 17, pages - 2]
    for c in (cache, small):
        fill(c, [900], torch.Generator(device=DEV).manual_seed(21))
    g = torch.Generator(device=DEV).manual_seed(22)
    emb = table(64, 8, 900, g)
    for n in (1, 4, 64, 300):
        q = torch.randn(1, 16, n, 128, device=DEV, generator=g).bfloat16()
        assert torch.equal(cache.attend(q, emb), small.attend(q, emb))
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0), small.read(0)))


@pytest.mark.parametrize("store", [None, I8])
def test_transposed_vectors(store):
    """One token whose features were the last axis but one: the strides of axes of one element say nothing."""
    g = torch.Generator(device=DEV).manual_seed(4)
    cache, other = make(1, 2, 64, BF, store, 100), make(1, 2, 64, BF, store, 100)
    col = lambda h: torch.randn(1, h, 64, 1, device=DEV, generator=g).bfloat16().transpose(2, 3)
    for _ in range(3):
        k, v = col(2), col(2)
        assert k.stride(2) == 1
        cache.append(k, v)
        other.append_to(0, k[0].clone(memory_format=torch.contiguous_format), v[0].clone(memory_format=torch.contiguous_format))
    for a, b in zip(cache.gather(0), other.gather(0)):
        assert torch.equal(a, b)
    emb, q = table(32, 2, 100, g), col(4)
    want = other.attend(q.clone(memory_format=torch.contiguous_format), emb)
    assert torch.equal(cache.attend(q, emb), want)
    vals = held(cache)
    ref = R.attend(q, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], [3], [1], 0.125, store)
    R.check(want, ref[0], ref[2], ref[3])


@pytest.mark.parametrize("store", [None, F8])
def test_refusals(store):
    g = torch.Generator(device=DEV).manual_seed(2)
    cache = make(2, 2, 64, BF, store, 100)
    fill(cache, [40, 60], g)
    q = torch.randn(2, 4, 3, 64, device=DEV, generator=g).bfloat16()
    freqs, bias = table(32, 2, 100, g)
    before = [cache.lens, cache.page_table.clone(), cache.seq_lens.clone()]
    for err, qq, emb, more in (
            (TypeError, q.half(), (freqs, bias), {}),
            (TypeError, q.cpu(), (freqs, bias), {}),
            (ValueError, q[:, :3], (freqs, bias), {}),
            (ValueError, q[:1], (freqs, bias), {}),
            (ValueError, q, (freqs[None], bias), {}),
            (ValueError, q, (freqs[:59], bias), {}),
            (ValueError, q, (freqs, bias[:1]), {}),
            (ValueError, q, (freqs[:, :12], bias), {}),          # not a multiple of eight
            (ValueError, q, (torch.cat([freqs] * 3, -1), bias), {}),
            ((TypeError, ValueError, RuntimeError), q, (freqs.cpu(), bias), {}),
            ((TypeError, ValueError, RuntimeError), q, (freqs, bias.cpu()), {}),
            (TypeError, q, (freqs, bias), dict(counts=torch.zeros(2, dtype=torch.int64, device=DEV))),
            (TypeError, q, (freqs, bias), dict(counts=torch.zeros(2, dtype=torch.int32))),
            (ValueError, q, (freqs, bias), dict(counts=torch.zeros(3, dtype=torch.int32, device=DEV)))):
        with pytest.raises(err):
            cache.attend(qq, emb, **more)
    with pytest.raises(TypeError):
        cache.append(q[:, :2], q[:, :2].float())
    with pytest.raises(IndexError):
        cache.read(0, 0, 41)
    assert cache.lens == before[0] and torch.equal(cache.page_table, before[1]) and torch.equal(cache.seq_lens, before[2])
    assert _native.device_status() == 0


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("store", [None, I8, F8])
def test_every_width_of_rotation_and_number_of_heads(d, store):
    """Every r, with numbers of key heads and rows that give every split of work over warps, CTAs and kernels: each has to fit the SM."""
    g = torch.Generator(device=DEV).manual_seed(d)
    for at, r in enumerate(range(0, d + 1, 8)):
        dtype = (BF, HF)[at % 2]
        for hk, h, new in ((1, 1, 1), (2, 2, 8), (4, 16, 1), (3, 3, 11), (4, 8, 8), (2, 4, 19), (1, 2, 131)):
            lens = [70, 131 + new]
            cache = make(2, hk, d, dtype, store, 280, 64, seed=r)
            fill(cache, lens, g)
            q = torch.randn(2, h, new, d, device=DEV, generator=g).to(dtype)
            emb = table(r, hk, 280, g)
            vals = held(cache)
            want = R.attend(q, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], lens, [new] * 2, d ** -0.5, store)
            R.check(cache.attend(q, emb), want[0], want[2], want[3])
    assert _native.device_status() == 0


@pytest.mark.parametrize("seed", range(12))
def test_drawn_shapes(seed):
    """Sizes of all kinds: long and ragged caches, chunks from one token to hundreds, every kernel and every cut along the keys."""
    import random
    rng = random.Random(seed)
    d = rng.choice([64, 96, 128])
    r = rng.choice([d, d // 2, d // 4 // 8 * 8])
    hk = rng.choice([1, 2, 3, 4, 8])
    h = hk * rng.choice([1, 2, 4, 5])
    b, dtype, store, page = rng.choice([1, 2, 5]), rng.choice([BF, HF]), rng.choice([None, I8, F8]), rng.choice([64, 128, 192, 256])
    lens = [round(math.exp(rng.uniform(0, math.log(9000)))) for _ in range(b)]
    new = min(max(lens), rng.choice([1, 2, 3, 7, 16, 33, 64, 100, 257]))
    counts = [rng.randint(0, new) for _ in lens] if rng.random() < 0.5 else None
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = make(b, hk, d, dtype, store, max(lens) + 5, page, seed)
    fill(cache, lens, g)
    q = torch.randn(b, h, new, d, device=DEV, generator=g).to(dtype)
    emb = table(r, hk, max(lens), g)
    given = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, emb, counts=given, return_lse=True)
    vals = held(cache)
    want = R.attend(q, [x[0] for x in vals], [x[1] for x in vals], emb[0], emb[1], lens, counts or [new] * b, d ** -0.5, store)
    R.check(out, want[0], want[2], want[3], lse, want[1])
    assert _native.device_status() == 0


@pytest.mark.parametrize("store", [None, I8])
def test_one_long_sequence_among_many(store):
    """Forty sequences, one of 110000 keys: more than 8 GB of expanded keys, were each given the room of the longest."""
    g = torch.Generator(device=DEV).manual_seed(9)
    b, hk, d, r, new, n = 40, 8, 64, 64, 300, 110000
    lens = [n if i == 7 else 305 + i for i in range(b)]
    cache = PagedKVCache(b, hk, d, num_pages=-(-n // 256) + 2 * b, page_size=256, max_seq_len=n, dtype=BF, store=store)
    fill(cache, lens, g)
    q = torch.randn(b, hk, new, d, device=DEV, generator=g).bfloat16()
    emb = table(r, hk, n, g)
    got = cache.attend(q, emb)
    for i in (0, 7, 39):
        k, v = (x.float() for x in cache.gather(i)) if store is None else (c * s[..., None] for c, s in stored(cache, i))
        want = R.attend(q[i:i + 1, :, -40:], [k], [v], emb[0], emb[1], [lens[i]], [40], d ** -0.5)
        R.check(got[i:i + 1, :, -40:], want[0], want[2], want[3])
    assert _native.device_status() == 0


def test_against_the_attention_over_contiguous_keys():
    """Every position of a prompt at once: the causal forward over the same keys."""
    g = torch.Generator(device=DEV).manual_seed(31)
    k, v, q = (torch.randn(2, x, 640, 128, device=DEV, generator=g).half() for x in (2, 2, 8))
    emb = table(64, 2, 640, g)
    cache = make(2, 2, 128, HF, None, 640)
    cache.append(k, v)
    a, b = cache.attend(q, emb).float(), flash_attn_with_pope(q, k, v, pos_emb=emb, causal=True).float()
    # both are within the roundings of fp16 operands of the exact result
    assert (a - b).norm() <= 4e-3 * b.norm()
