"""The 8-bit paged cache without a GPU: refusals at the C boundary and in the
Python class, the struct's layout, and the byte order of a page."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from draftkv import _lib
from tests.q8_reference import exponent_of, page_index, round_e4m3

torch = pytest.importorskip("torch")
HEADER = Path(__file__).resolve().parent.parent / "include" / "draftkv_b200.h"


@pytest.fixture(scope="module")
def lib():
    return _lib.load(require_device=False)


def cache(**kw):
    f = dict(codes=1024, scale=1024, page_table=1024, n_pages=8, page_size=16, max_pages=4)
    f.update(kw)
    return _lib.Q8CacheS(*f.values())


def dims(n_layers=2, n_kv=2, d=64, batch=2):
    return _lib.DimsS(n_layers, n_kv, d, batch)


P = 4096          # a 16-byte aligned address that is never followed


def append(lib, c=None, dm=None, layer=0, k=P, v=P, dt=_lib.BF16, rows=1, e0=P):
    return lib.dkv_q8_append(C.byref(c or cache()), dm or dims(), layer, k, v, dt, rows, 128, 128, 64, e0, None, None, None,
                             None, None)


def attn(lib, c=None, dm=None, layer=0, group=1, T=1, q=P, e0=P, out=P, dt=_lib.BF16, split=0, mass=None, work=P,
         nbytes=1 << 40):
    return lib.dkv_q8_attn(C.byref(c or cache()), dm or dims(), layer, group, T, q, e0, None, out, dt, split, mass, work,
                           nbytes, None)


def evict(lib, c=None, n=P, sink=0, recent=0, mass=P, pos=None, table=P, pages=2, mass_out=2 * P, pos_out=None, kept=P):
    return lib.dkv_q8_evict(C.byref(c or cache()), dims(), 0, n, P, sink, recent, mass, pos, table, pages, mass_out, pos_out,
                            kept, None)


CACHE_FAULTS = [
    (dict(codes=None), _lib.EINVAL), (dict(scale=None), _lib.EINVAL), (dict(page_table=None), _lib.EINVAL),
    (dict(codes=1032), _lib.EINVAL), (dict(page_size=8), _lib.EUNSUPPORTED), (dict(page_size=24), _lib.EUNSUPPORTED),
    (dict(page_size=256), _lib.EUNSUPPORTED), (dict(n_pages=0), _lib.EINVAL), (dict(max_pages=0), _lib.EINVAL),
    (dict(max_pages=1 << 30), _lib.EINVAL),
]


@pytest.mark.parametrize("fields,status", CACHE_FAULTS)
def test_bad_caches_are_refused(lib, fields, status):
    for call in (append, attn, evict):
        assert call(lib, c=cache(**fields)) == status, call.__name__
        assert call.__name__.replace("attn", "q8_attn") in lib.dkv_last_error().decode()


@pytest.mark.parametrize("dm,status", [(dims(d=96), _lib.EUNSUPPORTED), (dims(d=256), _lib.EUNSUPPORTED),
                                       (dims(batch=0), _lib.EINVAL), (dims(n_kv=0), _lib.EINVAL)])
def test_bad_dims_are_refused(lib, dm, status):
    assert append(lib, dm=dm) == status
    assert attn(lib, dm=dm) == status


def test_bad_arguments_are_refused(lib):
    bad = [append(lib, layer=2), append(lib, layer=-1), append(lib, k=None), append(lib, v=None), append(lib, e0=None),
           append(lib, dt=7), append(lib, rows=-1), append(lib, rows=65),
           attn(lib, layer=2), attn(lib, q=None), attn(lib, e0=None), attn(lib, out=None), attn(lib, dt=7),
           attn(lib, group=0), attn(lib, T=0), attn(lib, q=P + 4), attn(lib, out=P + 2), attn(lib, split=100),
           attn(lib, work=None), attn(lib, nbytes=64),
           evict(lib, n=None), evict(lib, mass=None), evict(lib, mass_out=None), evict(lib, mass_out=P),
           evict(lib, table=None), evict(lib, kept=None), evict(lib, sink=-1), evict(lib, recent=-1), evict(lib, pages=0),
           evict(lib, pages=5), evict(lib, pos=P), evict(lib, pos=P, pos_out=P),
           lib.dkv_q8_read(C.byref(cache()), dims(), 2, 0, 1, P, None),
           lib.dkv_q8_read(C.byref(cache()), dims(), 0, 0, 65, P, None),
           lib.dkv_q8_read(C.byref(cache()), dims(), 0, 0, 1, None, None)]
    assert bad == [_lib.EINVAL] * len(bad)
    assert attn(lib, group=4, T=17, mass=P) == _lib.EUNSUPPORTED      # the mass of more than 64 rows


def test_empty_calls_do_nothing(lib):
    assert append(lib, rows=0, k=None, v=None, e0=None) == _lib.OK
    assert lib.dkv_q8_read(C.byref(cache()), dims(), 0, 0, 0, None, None) == _lib.OK
    assert lib.dkv_q8_attn_work_bytes(dims(), 0, 1, 64, 0, 0) == 0


def test_struct_layout_matches_the_header(tmp_path):
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
            'printf("%zu\\n", sizeof(dkv_q8_cache));']
    prog += [f'printf("%zu\\n", offsetof(dkv_q8_cache, {n}));' for n, _ in _lib.Q8CacheS._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(prog + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(_lib.Q8CacheS)] + [getattr(_lib.Q8CacheS, n).offset for n, _ in _lib.Q8CacheS._fields_]


@pytest.mark.parametrize("d", [64, 128])
def test_tile_tables_match_the_stated_words(d):
    from draftkv.q8 import tile_bytes
    k, v = tile_bytes(d)
    at = page_index(16, d)
    assert np.array_equal(k, at[0]) and np.array_equal(v + 16 * d, at[1])


def test_reference_rounding_is_e4m3():
    """The tests' rounding against torch's conversion, over every code's neighbourhood."""
    b = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    b = b[torch.isfinite(b)].unique()
    mid = (b[1:] + b[:-1]) / 2
    x = torch.cat([b, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    assert np.array_equal(round_e4m3(x.numpy()), x.float().to(torch.float8_e4m3fn).double().numpy())
    assert [exponent_of(a) for a in (0.0, 448.0, 449.0, 1.0, 1.75, 1.76, 1e-44, 3.4e38)] == \
        [-120, 0, 1, -8, -8, -7, -120, 119]


def test_class_refuses_shapes_before_the_device():
    from draftkv import Q8KVCache
    for kw in (dict(d_head=96), dict(block_size=24), dict(d_head=256)):
        with pytest.raises(ValueError):
            Q8KVCache(**{**dict(n_layers=1, n_heads=1, d_head=64), **kw})
    codes = torch.zeros((2, 1, 2, 16 * 64), dtype=torch.uint8)
    scale, table = torch.ones((2, 1, 2)), torch.zeros((1, 1, 2), dtype=torch.int32)
    for args in ((codes.float(), scale, table), (codes, scale.double(), table), (codes, scale[:1], table),
                 (codes, scale, table.long()), (codes, scale, table[0]), (codes[:, :, :, :1000], scale, table),
                 (codes, scale, table)):             # the last: not on a CUDA device
        with pytest.raises(ValueError):
            Q8KVCache.from_storage(*args)
