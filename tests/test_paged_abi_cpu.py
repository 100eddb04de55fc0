"""The C entry points of the paged cache's 8-bit store and of its chunks, without a GPU: layouts of the structs, refusals, workspace."""
import ctypes as C
import os
import subprocess

import pytest

from pope_pytorch_b200 import _native as N
from pope_pytorch_b200 import build as B

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "pope_b200.h")
BAD, UNSUPPORTED, MISALIGNED, WORKSPACE = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    B.build()
    return N.load_library()


@pytest.fixture(scope="module")
def ptr():
    """An address on 256 bytes; nothing here is read (every call is refused before)."""
    buf = (C.c_char * 4096)()
    yield (C.addressof(buf) + 255) & ~255
    del buf


def test_struct_layouts(tmp_path):
    structs = {"PopePagedStore": N.PagedStore, "PopeKvWriteArgs": N.KvWriteArgs, "PopeKvReadArgs": N.KvReadArgs, "PopePagedAttnArgs": N.PagedAttnArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for name, ct in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in ct._fields_]
    lines.append('printf("enums %d\\n", POPE_OP_ATTN_PAGED * 1000 + POPE_STORE_16 * 100 + POPE_STORE_INT8 * 10 + POPE_STORE_E4M3); return 0;}')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, ct in structs.items():
        assert int(got[name]) == C.sizeof(ct), name
        for f, _ in ct._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(ct, f).offset, (name, f)
    assert int(got["enums"]) == N.OP_ATTN_PAGED * 1000 + N.STORE_16 * 100 + N.STORE_INT8 * 10 + N.STORE_E4M3


def store(ptr, **over):
    f = {**dict(k=ptr, v=ptr, table=ptr, lens=ptr, pages=64, size=256, most=16, ks=ptr, vs=ptr, store=N.STORE_INT8), **over}
    return N.PagedStore(N.PagedKV(f["k"], f["v"], f["table"], f["lens"], f["pages"], f["size"], f["most"], 0), f["ks"], f["vs"], f["store"], 0)


STORES = [(BAD, dict(k=None)), (BAD, dict(v=None)), (BAD, dict(table=None)), (BAD, dict(lens=None)), (BAD, dict(pages=0)), (BAD, dict(most=0)), (BAD, dict(size=0)),
          (UNSUPPORTED, dict(size=100)), (BAD, dict(store=3)), (BAD, dict(store=-1)), (BAD, dict(ks=None)), (BAD, dict(vs=None))]


def call(lib, name, a):
    return getattr(lib, name)(C.addressof(a), None)


def make_write(ptr, **over):
    a = N.KvWriteArgs()
    a.struct_bytes, a.dtype, a.B, a.Hk, a.d, a.n_new, a.cache, a.k, a.v = C.sizeof(a), 1, 2, 2, 64, 4, store(ptr), ptr, ptr
    a.sk = a.sv = N.Stride3(512, 256, 64)
    for f, x in over.items():
        setattr(a, f, x)
    return a


def test_writes(lib, ptr):
    assert lib.pope_b200_kv_write(None, None) == BAD
    for want, over in [(BAD, dict(struct_bytes=8)), (BAD, dict(B=0)), (BAD, dict(Hk=0)), (BAD, dict(d=0)), (BAD, dict(n_new=-1)), (BAD, dict(k=None)),
                       (BAD, dict(v=None)), (UNSUPPORTED, dict(dtype=0)), (UNSUPPORTED, dict(d=80)), (UNSUPPORTED, dict(Hk=65536)), (UNSUPPORTED, dict(B=65536)),
                       (MISALIGNED, dict(k=ptr + 2)), (MISALIGNED, dict(sv=N.Stride3(512, 256, 60))), (0, dict(n_new=0))]:
        assert call(lib, "pope_b200_kv_write", make_write(ptr, **over)) == want, over
    for want, over in STORES + [(UNSUPPORTED, dict(store=N.STORE_16)), (MISALIGNED, dict(k=ptr + 8)), (MISALIGNED, dict(vs=ptr + 4))]:
        assert call(lib, "pope_b200_kv_write", make_write(ptr, cache=store(ptr, **over))) == want, over


def make_read(ptr, **over):
    a = N.KvReadArgs()
    a.struct_bytes, a.dtype, a.Hk, a.d, a.first, a.n, a.cache, a.k, a.v = C.sizeof(a), 2, 2, 96, 0, 4, store(ptr), ptr, ptr
    a.sk_h, a.sk_n, a.sv_h, a.sv_n = 384, 96, 384, 96
    for f, x in over.items():
        setattr(a, f, x)
    return a


def test_reads(lib, ptr):
    assert lib.pope_b200_kv_read(None, None) == BAD
    for want, over in [(BAD, dict(struct_bytes=8)), (BAD, dict(Hk=0)), (BAD, dict(d=0)), (BAD, dict(n=-1)), (BAD, dict(first=-1)), (BAD, dict(first=2 ** 31 - 2)),
                       (BAD, dict(k=None)), (BAD, dict(v=None)), (UNSUPPORTED, dict(dtype=0)), (UNSUPPORTED, dict(d=32)), (UNSUPPORTED, dict(Hk=65536)),
                       (MISALIGNED, dict(v=ptr + 4)), (MISALIGNED, dict(sk_n=97)), (0, dict(n=0))]:
        assert call(lib, "pope_b200_kv_read", make_read(ptr, **over)) == want, over
    for want, over in STORES:
        assert call(lib, "pope_b200_kv_read", make_read(ptr, cache=store(ptr, **over))) == want, over


def make_attn(ptr, shape=(), **over):
    a = N.PagedAttnArgs()
    s = {**dict(B=2, H=4, Hk=2, Nq=5, Nk=4096, d=128, r=64, dtype=1), **dict(shape)}
    a.struct_bytes, a.softmax_scale, a.shape = C.sizeof(a), 0.1, N.Shape(*[s[k] for k in ("B", "H", "Hk", "Nq", "Nk", "d", "r", "dtype")])
    a.embed.freqs, a.embed.bias, a.embed.sf, a.embed.bias_stride_h = ptr, ptr, N.Stride3(0, 0, 64), 64
    a.cache, a.q, a.out = store(ptr), ptr, ptr
    a.sq = a.so = N.Stride3(4 * 5 * 128, 5 * 128, 128)
    for f, x in over.items():
        setattr(a, f, x)
    return a


def test_attention(lib, ptr):
    name = "pope_b200_attn_paged"
    assert lib.pope_b200_attn_paged(None, None) == BAD
    for want, shape in [(BAD, dict(B=0)), (BAD, dict(H=3)), (BAD, dict(Nq=0)), (BAD, dict(Nk=0)), (BAD, dict(r=136)), (BAD, dict(dtype=7)),
                        (UNSUPPORTED, dict(dtype=0)), (UNSUPPORTED, dict(d=80, r=64)), (UNSUPPORTED, dict(r=12)), (UNSUPPORTED, dict(Nk=(1 << 24) + 1)),
                        (UNSUPPORTED, dict(B=65536)), (WORKSPACE, dict(Nq=5000))]:
        assert call(lib, name, make_attn(ptr, shape)) == want, shape
    for want, over in [(BAD, dict(struct_bytes=8)), (BAD, dict(embed=N.Embed())), (BAD, dict(q=None)), (BAD, dict(out=None)),
                       (MISALIGNED, dict(out=ptr + 2)), (MISALIGNED, dict(so=N.Stride3(2560, 640, 124))), (WORKSPACE, {})]:
        assert call(lib, name, make_attn(ptr, **over)) == want, over
    for want, over in STORES:
        assert call(lib, name, make_attn(ptr, cache=store(ptr, **over))) == want, over
    for new in (1, 8, 20, 300):       # one size of workspace for every kernel
        a = make_attn(ptr, dict(Nq=new))
        need = lib.pope_b200_workspace_bytes(N.OP_ATTN_PAGED, C.addressof(a))
        assert need > 0
        a.workspace, a.workspace_bytes = ptr, need - 1
        assert call(lib, name, a) == WORKSPACE
        a.workspace, a.workspace_bytes = ptr + 16, need
        assert call(lib, name, a) == MISALIGNED
    a = make_attn(ptr, dict(d=80))
    assert lib.pope_b200_workspace_bytes(N.OP_ATTN_PAGED, C.addressof(a)) == 0


def test_images_of_a_large_cache_stay_out_of_the_workspace(lib, ptr):
    """Sixty-four sequences of up to 131072 keys: expanded keys of all of them would be 27 GB and more."""
    for kind in (N.STORE_16, N.STORE_INT8):
        a = make_attn(ptr, dict(B=64, H=8, Hk=8, Nq=2048, Nk=131072), cache=store(ptr, store=kind, most=512))
        assert 0 < lib.pope_b200_workspace_bytes(N.OP_ATTN_PAGED, C.addressof(a)) < 1 << 30
