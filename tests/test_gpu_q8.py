"""The 8-bit paged cache on the GPU against its 64-bit restatement
(tests/q8_reference.py): append and eviction exactly, attention and mass within
derived bounds."""
import ctypes as C

import numpy as np
import pytest

from tests import q8_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def lib():
    from draftkv import _lib
    _lib.load()
    return _lib


def device_error():
    e = C.c_uint32(0)
    lib().call("dkv_device_error", C.byref(e), lib().stream_ptr())
    return e.value


@pytest.fixture(autouse=True)
def clean_error_word():
    device_error()
    yield
    assert device_error() == 0, "a test left the device error word set"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Made:
    """A cache over its own storage with shuffled pages: the unused ones hold
    bytes and scales that must never be read (NaN)."""

    def __init__(self, batch=2, layers=2, kv=2, d=64, page=16, pages=4, seed=0, spare=3):
        from draftkv import Q8KVCache
        self.batch, self.layers, self.kv, self.d, self.page, self.pages = batch, layers, kv, d, page, pages
        rng = np.random.default_rng(seed)
        n = batch * layers * pages + spare
        self.codes = torch.full((n, kv, 2, page * d), 0x7F, dtype=torch.uint8, device="cuda")
        self.scale = torch.full((n, kv, 2), float("nan"), device="cuda")
        self.table_np = rng.permutation(n)[: batch * layers * pages].reshape(batch, layers, pages).astype(np.int32)
        self.table = torch.from_numpy(self.table_np).cuda()
        self.cache = Q8KVCache.from_storage(self.codes, self.scale, self.table, block_size=page)
        self.cap = pages * page

    def reference(self):
        sc = np.nan_to_num(self.scale.cpu().numpy(), nan=1.0)
        r = ref.RefCache(self.codes.cpu().numpy(), sc, self.table_np, self.page, self.d)
        return r

    def fill(self, n, rng, layer=0, spread=1.0, dtype=torch.bfloat16):
        """Appends n[b] random rows to each sequence from its start; returns the reference."""
        rows = max(n)
        r = self.reference()
        k = rng.standard_normal((self.batch, rows, self.kv, self.d)) * np.exp(spread * rng.standard_normal((self.batch, rows, 1, 1)))
        v = rng.standard_normal(k.shape) * np.exp(spread * rng.standard_normal((self.batch, rows, self.kv, 1)))
        k, v = (torch.from_numpy(x.astype(np.float32)).cuda().to(dtype) for x in (k, v))
        self.cache.write(layer, k, v, i32([0] * self.batch), n_rows=i32(n))
        r.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), [0] * self.batch, n)
        return r

    def same_as(self, r, layer, n):
        """Codes and scales of the first n[b] entries equal the reference's exactly."""
        got = ref.decode(self.codes.cpu().numpy(), self.page, self.d, r.index)
        sc = self.scale.cpu().numpy().astype(np.float64)
        for b in range(self.batch):
            for e in range(0, n[b], self.page):
                pid = self.table_np[b, layer, e // self.page]
                cnt = min(self.page, n[b] - e)
                assert np.array_equal(sc[pid], np.ldexp(1.0, r.exp[pid])), (b, e)
                assert np.array_equal(got[pid][:, :, :cnt], r.vals[pid][:, :, :cnt]), (b, e)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_matches_the_definition(d, page, dtype):
    """A ragged prompt from the start, then ragged runs that begin inside a
    page (and one sequence that gets nothing), scales growing on the way."""
    mk = Made(batch=3, d=d, page=page, pages=max(3, 160 // page), seed=page + d)
    rng = np.random.default_rng(d + page)
    n = [37, 1, 70]
    r = mk.fill(n, rng, layer=1, dtype=dtype)
    mk.same_as(r, 1, n)
    for step, add in enumerate(([1, 0, 9], [1, 17, 1], [0, 1, 5])):
        rows = max(add)
        k = rng.standard_normal((3, rows, mk.kv, d)) * 3.0 ** step
        v = rng.standard_normal(k.shape) * 0.3 ** step
        k, v = (torch.from_numpy(x.astype(np.float32)).cuda().to(dtype) for x in (k, v))
        mk.cache.write(1, k, v, i32(n), n_rows=i32(add))
        r.append(1, k.float().cpu().numpy(), v.float().cpu().numpy(), n, add)
        n = [x + y for x, y in zip(n, add)]
        mk.same_as(r, 1, n)


def test_append_leaves_other_bytes_alone():
    """Rows behind the last one, other layers' pages and spare pages keep their bytes."""
    mk = Made(batch=2, d=64, page=32, pages=2)
    before, sc = mk.codes.clone(), mk.scale.clone()
    x = torch.randn((2, 21, 2, 64), device="cuda")
    mk.cache.write(0, x, x, i32([0, 0]), n_rows=i32([21, 5]))
    idx = ref.page_index(32, 64)
    written = torch.zeros_like(mk.codes, dtype=torch.bool)
    for b, n in ((0, 21), (1, 5)):
        for i in (0, 1):
            at = torch.from_numpy((idx[i] - i * 32 * 64)[:n].reshape(-1)).cuda()
            written[int(mk.table_np[b, 0, 0]), :, i, at] = True
    assert torch.equal(mk.codes[~written], before[~written])
    assert not torch.isnan(mk.scale[mk.table_np[:, 0, 0]]).any()
    other = [p for p in range(mk.codes.shape[0]) if p not in mk.table_np[:, 0, 0]]
    assert torch.isnan(mk.scale[other]).all() and torch.isnan(sc).all()


def test_append_takes_strided_and_unaligned_sources():
    """K and V as slices of one fused projection [b, r, n_kv, 2, d], with a padded
    row, and from an address that 16-byte loads cannot take."""
    for offset in (0, 1):
        mk = Made(batch=2, kv=3, d=64, page=16, pages=3)
        buf = torch.randn(2 * 20 * 3 * 2 * 64 + offset + 3, device="cuda").to(torch.bfloat16)[offset:]
        fused = buf.as_strided((2, 20, 3, 2, 64), (20 * 384, 384, 128, 64, 1))
        k, v = fused[:, :, :, 0], fused[:, :, :, 1]
        r = mk.reference()
        mk.cache.write(0, k, v, i32([0, 0]), n_rows=i32([20, 11]))
        r.append(0, k.float().cpu().numpy(), v.float().cpu().numpy(), [0, 0], [20, 11])
        mk.same_as(r, 0, [20, 11])


def test_append_values_at_the_type_s_ends():
    """Zeros, subnormals, the largest values, and a page whose range is wide."""
    mk = Made(batch=1, kv=1, d=64, page=16, pages=8)
    x = np.zeros((1, 128, 1, 64), np.float32)
    x[0, 16:32] = 1e-40
    x[0, 32:48] = 3.4e38
    x[0, 48:64] = np.float32(448.0) * np.linspace(-1, 1, 64, dtype=np.float32)
    x[0, 64:80] = 2.0 ** -np.arange(64, dtype=np.float32)
    x[0, 80:96] = np.nextafter(np.float32(1.75), np.float32(2.0))
    x[0, 96:112] = -1.75
    x[0, 112:128] = (17.0 + np.arange(64)) / 16        # ties of the rounding
    t = torch.from_numpy(x).cuda()
    r = mk.reference()
    mk.cache.write(0, t, -t, i32([0]))
    r.append(0, x, -x, [0], [128])
    mk.same_as(r, 0, [128])
    got = mk.cache.read_rows(0, 128).cpu().numpy()
    k, v = r.entries(0, 0, 0, 128)
    assert np.array_equal(got[:, 0, 0], k.astype(np.float32)) and np.array_equal(got[:, 0, 1], v.astype(np.float32))


def test_append_reports_what_it_cannot_store():
    mk = Made(batch=2, kv=1, d=64, page=16, pages=2)
    x = torch.ones((2, 3, 1, 64), device="cuda")
    x[0, 1, 0, 5], x[1, 0, 0, 0], x[1, 2, 0, 63] = float("nan"), float("inf"), float("-inf")
    mk.cache.write(0, x, x, i32([0, 0]))
    assert device_error() == 0x800
    got = mk.cache.read_rows(0, 3, 0)[:, 0, 0]
    assert got[1, 5] == 0 and (got[0] == 1).all()
    got = mk.cache.read_rows(0, 3, 1)[:, 0, 0]
    # the largest stored value is 448 * 2^119 = 1.75 * 2^127 = 2.98e38
    assert got[0, 0] == 448 * 2.0 ** 119 and got[2, 63] == -448 * 2.0 ** 119
    # entries outside the capacity, a negative one, a bad page: nothing is written
    before = mk.codes.clone()
    mk.cache.write(0, x[:, :1] * 0, x[:, :1] * 0, i32([32, -1]))
    assert device_error() & 0x400
    mk.table[0, 1, 0], mk.table[1, 1, 0] = mk.codes.shape[0], -1
    mk.cache.write(1, torch.ones_like(x), torch.ones_like(x), i32([0, 0]))
    assert device_error() == 0x400
    assert torch.equal(mk.codes, before)


def test_append_resets_mass_and_positions_of_new_entries_only():
    mk = Made(batch=2, kv=2, d=64, page=16, pages=4)
    mass = torch.full((2, 2, 64), 7.0, device="cuda")
    pos = torch.full((2, 2, 64), -5, dtype=torch.int32, device="cuda")
    x = torch.randn((2, 20, 2, 64), device="cuda")
    mk.cache.write(0, x, x, i32([10, 30]), n_rows=i32([20, 1]), pos0=i32([100, 30]), mass=mass, pos=pos)
    want_m, want_p = torch.full((2, 64), 7.0), torch.full((2, 64), -5, dtype=torch.int32)
    want_m[0, 10:30], want_p[0, 10:30] = 0, torch.arange(100, 120, dtype=torch.int32)
    want_m[1, 30], want_p[1, 30] = 0, 30
    for h in range(2):
        assert torch.equal(mass[:, h].cpu(), want_m) and torch.equal(pos[:, h].cpu(), want_p)


def test_rollback_then_append_restarts_an_emptied_page():
    """A rolled-back page written from its start again forgets the old scale; one
    cut in the middle keeps the larger."""
    mk = Made(batch=1, kv=1, d=64, page=16, pages=2)
    r = mk.reference()
    for size, e0, n in ((0.3, 0, 16), (1e6, 16, 4), (0.3, 16, 4), (1e6, 20, 4), (0.3, 18, 4)):
        x = np.full((1, n, 1, 64), size, np.float32)
        t = torch.from_numpy(x).cuda()
        mk.cache.write(0, t, t, i32([e0]))
        r.append(0, x, x, [e0], [n])
        mk.same_as(r, 0, [e0 + n])


# --------------------------------------------------------------- attention
def check_attention(mk, r, q, entry0, layer=0, n_rows=None, out_dtype=torch.bfloat16, with_mass=False, **kw):
    mass = torch.rand((mk.batch, mk.kv, mk.cap), device="cuda") if with_mass else None
    start = mass.clone() if with_mass else None
    out = mk.cache.attention(layer, torch.from_numpy(q).cuda(), i32(entry0), n_rows=None if n_rows is None else i32(n_rows),
                             out_dtype=out_dtype, mass=mass, **kw)
    want, add, bound = r.attention(layer, q, entry0, n_rows)
    n = max(max(entry0) + q.shape[1], 1)
    vmax = max([1e-30] + [np.abs(r.entries(b, layer, h, entry0[b] + q.shape[1])[1]).max() for b in range(mk.batch)
                          for h in range(mk.kv) if entry0[b] + q.shape[1] > 0])
    rows = q.shape[1] * q.shape[2] // mk.kv
    rel, ab = (ref.attention_tolerance if rows <= 64 else ref.prompt_tolerance)(mk.d, n, bound, vmax,
                                                                              torch.finfo(out_dtype).eps)
    got = out.double().cpu().numpy()
    live = ~np.isnan(want)
    assert np.isfinite(got[live]).all()
    err = np.abs(got - want)[live] - rel * np.abs(want[live])
    assert err.max() <= ab, (err.max(), ab)
    if with_mass:
        # a weight is off by the factor 1 +- 2 (delta + roundings) (see attention_tolerance with vmax 1)
        _, one = ref.attention_tolerance(mk.d, n, bound, 1.0, 0.0)
        got_m = mass.double().cpu().numpy() - start.double().cpu().numpy()
        assert (np.abs(got_m - add) <= one * add + 2.0 ** -23 * (q.shape[1] * q.shape[2] // mk.kv + 2)).all()
        assert np.array_equal(got_m[add == 0], np.zeros((add == 0).sum()))
    return out


SHAPES = [   # batch, kv, group, d, page, pages, T, entries before the call
    (1, 1, 1, 64, 16, 1, 1, [0]), (1, 3, 3, 64, 16, 3, 1, [36]), (2, 2, 4, 128, 16, 24, 1, [15, 370]),
    (2, 2, 4, 128, 32, 12, 2, [300, 16]), (3, 1, 8, 128, 64, 5, 1, [1, 64, 300]), (2, 2, 1, 64, 128, 3, 9, [0, 350]),
    (2, 1, 5, 64, 32, 8, 3, [5, 240]), (1, 2, 7, 128, 16, 40, 9, [600]), (2, 2, 16, 64, 64, 4, 4, [200, 3]),
    (1, 1, 1, 128, 128, 9, 64, [1000]), (1, 2, 2, 64, 16, 70, 17, [1088]), (1, 1, 3, 128, 16, 20, 21, [0]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"b{s[0]}kv{s[1]}g{s[2]}d{s[3]}p{s[4]}T{s[6]}")
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_attention_matches_the_definition(shape, out_dtype):
    batch, kv, group, d, page, pages, T, e0 = shape
    mk = Made(batch, 2, kv, d, page, pages, seed=T)
    rng = np.random.default_rng(d + T)
    r = mk.fill([x + T for x in e0], rng, layer=1, spread=0.7)
    q = (rng.standard_normal((batch, T, kv * group, d)) * 1.5).astype(np.float32)
    check_attention(mk, r, q, e0, layer=1, out_dtype=out_dtype, with_mass=T * group <= 64)


@pytest.mark.parametrize("split", [128, 256, 1024])
@pytest.mark.parametrize("T,group", [(1, 4), (5, 4), (40, 1)])
def test_attention_split_over_keys(split, T, group):
    mk = Made(2, 1, 1, 128, 16, 90, seed=3)
    rng = np.random.default_rng(split + T)
    e0 = [1400 - T, 515]
    r = mk.fill([x + T for x in e0], rng, spread=0.5)
    q = rng.standard_normal((2, T, group, 128)).astype(np.float32)
    check_attention(mk, r, q, e0, out_dtype=torch.float32, split_keys=split, with_mass=True)


def test_mass_behind_several_waves():
    """32 splits x 2 heads x 2 sequences x 3 row blocks are more CTAs than the GPU holds."""
    mk = Made(2, 1, 2, 64, 16, 256, seed=8)
    rng = np.random.default_rng(6)
    r = mk.fill([4000, 2100], rng, spread=0.5)
    q = rng.standard_normal((2, 11, 6, 64)).astype(np.float32)
    check_attention(mk, r, q, [3989, 2089], with_mass=True, split_keys=128, out_dtype=torch.float32)


@pytest.mark.parametrize("d,group", [(64, 3), (128, 4), (128, 1)])
def test_verify_rows_equal_decode_rows_bit_for_bit(d, group):
    mk = Made(2, 1, 2, d, 16, 80, seed=5)
    rng = np.random.default_rng(d)
    T = 9
    e0 = [1200, 251]
    mk.fill([x + T for x in e0], rng, spread=1.0)
    q = torch.from_numpy((rng.standard_normal((2, T, 2 * group, d)) * 2).astype(np.float32)).cuda()
    for dt in (torch.bfloat16, torch.float32):
        whole = mk.cache.attention(0, q, i32(e0), out_dtype=dt)
        for t in range(T):
            one = mk.cache.attention(0, q[:, t:t + 1].contiguous(), i32([x + t for x in e0]), out_dtype=dt)
            assert torch.equal(one[:, 0], whole[:, t]), t
        few = mk.cache.attention(0, q[:, 2:5].contiguous(), i32([x + 2 for x in e0]), out_dtype=dt)
        assert torch.equal(few, whole[:, 2:5])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,group", [(5, 4), (9, 4), (11, 5)])
def test_row_blocks_of_either_size(d, T, group):
    """20, 36 and 55 rows come in blocks of 8 or of 16: against the definition, and row by row as one-token calls."""
    mk = Made(2, 1, 2, d, 32, 20, seed=T)
    rng = np.random.default_rng(T * d)
    e0 = [500, 90]
    r = mk.fill([x + T for x in e0], rng, spread=0.5)
    q = rng.standard_normal((2, T, 2 * group, d)).astype(np.float32)
    out = check_attention(mk, r, q, e0, out_dtype=torch.float32, with_mass=True)
    for t in range(T):
        one = mk.cache.attention(0, torch.from_numpy(q[:, t:t + 1].copy()).cuda(), i32([x + t for x in e0]),
                                 out_dtype=torch.float32)
        assert torch.equal(one[:, 0], out[:, t])


def test_rows_that_see_nothing_and_rows_that_are_not_there():
    """entry0 below zero empties rows (zeros); tokens past n_rows keep their output."""
    mk = Made(3, 1, 2, 64, 16, 4, seed=9)
    rng = np.random.default_rng(2)
    r = mk.fill([4, 33, 20], rng)
    q = rng.standard_normal((3, 4, 4, 64)).astype(np.float32)
    check_attention(mk, r, q, [-2, 29, 16], with_mass=True)
    out = torch.full((3, 4, 4, 64), 5.0, dtype=torch.float32, device="cuda")
    mass = torch.zeros((3, 2, 64), device="cuda")
    got = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([-4, 29, 16]), n_rows=i32([4, 0, 2]), out=out, mass=mass)
    assert got.data_ptr() == out.data_ptr()
    assert (out[0] == 0).all() and (out[1] == 5).all() and (out[2, 2:] == 5).all()
    want, add, _ = r.attention(0, q, [-4, 29, 16], [4, 0, 2])
    assert np.abs(out[2, :2].cpu().numpy() - want[2, :2]).max() < 1e-3       # bound checked above
    assert (mass[0] == 0).all() and (mass[1] == 0).all() and (mass[2, :, 18:] == 0).all()
    assert np.abs(mass[2].cpu().numpy().sum(-1) - 4).max() < 1e-4           # 2 tokens x 2 heads of weight 1


def test_values_of_very_different_size():
    """Blocks whose V differ by 2^16 and a block of zeros: what the weights select
    keeps its precision; K blocks of different scale too."""
    for d in (64, 128):
        mk = Made(1, 1, 1, d, 16, 8, seed=1)
        rng = np.random.default_rng(d)
        k = rng.standard_normal((1, 128, 1, d)).astype(np.float32)
        v = rng.standard_normal((1, 128, 1, d)).astype(np.float32)
        size = np.repeat(2.0 ** np.array([0, -16, 3, -9, 0, -16, 8, -3]), 16).astype(np.float32)[None, :, None, None]
        v *= size
        v[:, 64:80] = 0
        k[:, 32:48] *= 40
        r = mk.reference()
        mk.cache.write(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0]))
        r.append(0, k, v, [0], [128])
        for target in (20, 70, 90, 100):       # a query that picks one entry almost alone
            kk, vv = r.entries(0, 0, 0, 128)
            q = (kk[target] / np.linalg.norm(kk[target]) ** 2 * 40 * np.sqrt(d)).astype(np.float32).reshape(1, 1, 1, d)
            out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([127]), out_dtype=torch.float32).cpu().numpy()
            want, _, bound = r.attention(0, q, [127])
            s = kk @ q.reshape(-1).astype(np.float64) / np.sqrt(d)
            p = np.exp(s - s.max())
            p /= p.sum()
            # each weight is off by 2 delta: the error is that much of sum p |v|, and f16 keeps 2^-30 of the largest
            delta = ref.attention_tolerance(d, 128, bound, 1.0, 0.0)[1]
            ab = delta * (p @ np.abs(vv)) + 2.0 ** -30 * np.abs(vv).max(0)
            assert (np.abs(out.reshape(-1) - want.reshape(-1)) <= ab).all(), target


def test_large_queries_and_peaked_scores():
    mk = Made(1, 1, 2, 128, 16, 20, seed=4)
    rng = np.random.default_rng(8)
    r = mk.fill([300], rng, spread=0.2)
    for size in (1e-30, 1e-3, 30.0):
        q = (rng.standard_normal((1, 1, 4, 128)) * size).astype(np.float32)
        check_attention(mk, r, q, [299], out_dtype=torch.float32, with_mass=True)
    q = np.zeros((1, 2, 4, 128), np.float32)
    check_attention(mk, r, q, [298], out_dtype=torch.float32)
    # a NaN query poisons its own row alone
    q = rng.standard_normal((1, 2, 4, 128)).astype(np.float32)
    clean = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([298]), out_dtype=torch.float32)
    q[0, 1, 2, 7] = np.nan
    out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([298]), out_dtype=torch.float32)
    assert torch.isnan(out[0, 1, 2]).all()
    keep = torch.ones((1, 2, 4), dtype=torch.bool)
    keep[0, 1, 2] = False
    assert torch.equal(out[keep], clean[keep])


def test_bad_pages_and_entries_beyond_the_capacity():
    """Keys on a bad page are not seen; entries past the capacity neither; both are recorded."""
    mk = Made(1, 1, 1, 64, 16, 6, seed=6)
    rng = np.random.default_rng(0)
    r = mk.fill([90], rng)
    q = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    kk, vv = r.entries(0, 0, 0, 90)
    for bad in (mk.codes.shape[0], -1, 2 ** 31 - 1):
        keep = mk.table[0, 0, 2].item()
        mk.table[0, 0, 2] = bad
        out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([89]), out_dtype=torch.float32).cpu().numpy()
        assert device_error() == 0x400
        mk.table[0, 0, 2] = keep
        see = np.r_[0:32, 48:90]
        s = q[0, 0].astype(np.float64) @ kk[see].T / 8
        p = np.exp(s - s.max(-1, keepdims=True))
        want = p / p.sum(-1, keepdims=True) @ vv[see]
        assert np.abs(out[0, 0] - want).max() < 1e-4 * np.abs(vv).max()
    mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([96]))
    assert device_error() == 0x400
    mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([2 ** 31 - 1]))
    assert device_error() == 0x400


# ------------------------------------------------------------ prompt chunks
PROMPTS = [   # batch, kv, group, d, page, pages, T, entries before the call
    (1, 1, 1, 64, 16, 5, 65, [0]), (2, 2, 4, 128, 16, 20, 17, [300, 0]), (1, 2, 1, 64, 32, 10, 301, [3]),
    (2, 1, 3, 128, 64, 6, 100, [250, 7]), (1, 1, 8, 128, 128, 4, 70, [400]), (3, 1, 2, 64, 16, 40, 129, [500, 128, 1]),
    (1, 1, 5, 64, 16, 9, 13, [127]),
]


@pytest.mark.parametrize("shape", PROMPTS, ids=lambda s: f"b{s[0]}kv{s[1]}g{s[2]}d{s[3]}p{s[4]}T{s[6]}")
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_prompt_attention_matches_the_definition(shape, out_dtype):
    batch, kv, group, d, page, pages, T, e0 = shape
    mk = Made(batch, 2, kv, d, page, pages, seed=T)
    rng = np.random.default_rng(d + T)
    r = mk.fill([x + T for x in e0], rng, layer=1, spread=0.7)
    q = (rng.standard_normal((batch, T, kv * group, d)) * 1.5).astype(np.float32)
    check_attention(mk, r, q, e0, layer=1, out_dtype=out_dtype)


@pytest.mark.parametrize("d,page", [(128, 16), (64, 128)])
def test_prompt_attention_over_key_splits(d, page):
    """A capacity of several splits, of which the sequence fills the first two and a bit."""
    mk = Made(1, 1, 1, d, page, 40960 // page, seed=2)
    rng = np.random.default_rng(d)
    T, e0 = 70, 5000
    r = mk.fill([e0 + T], rng, spread=0.5)
    q = rng.standard_normal((1, T, 2, d)).astype(np.float32)
    check_attention(mk, r, q, [e0])
    r0 = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([-T]))
    assert (r0 == 0).all()


@pytest.mark.parametrize("d,out_dtype", [(64, torch.float32), (128, torch.bfloat16)])
def test_prompt_row_blocks_over_key_splits(d, out_dtype):
    """Two row blocks, four key splits of which the short sequence reaches one, tokens that are not there."""
    mk = Made(2, 1, 2, d, 32, 64, seed=3)
    rng = np.random.default_rng(d)
    T, e0 = 130, [1500, 3]
    r = mk.fill([x + T for x in e0], rng, spread=0.5)
    q = rng.standard_normal((2, T, 6, d)).astype(np.float32)
    check_attention(mk, r, q, e0, n_rows=[130, 77], out_dtype=out_dtype)


def test_prompt_rows_that_see_nothing_or_are_not_there():
    mk = Made(2, 1, 1, 64, 16, 30, seed=9)
    rng = np.random.default_rng(5)
    r = mk.fill([150, 200], rng)
    q = rng.standard_normal((2, 90, 2, 64)).astype(np.float32)
    check_attention(mk, r, q, [-30, 100], n_rows=[90, 41])
    out = torch.full((2, 90, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([-30, 100]), n_rows=i32([0, 41]), out=out)
    assert (out[0] == 5).all() and (out[1, 41:] == 5).all() and not (out[1, :41] == 5).all()
    # a NaN query poisons its own row alone
    clean = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([10, 100]))
    q[1, 3, 1, 0] = np.nan
    got = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([10, 100]))
    assert torch.isnan(got[1, 3, 1]).all()
    keep = torch.ones((2, 90, 2), dtype=torch.bool)
    keep[1, 3, 1] = False
    assert torch.equal(got[keep], clean[keep])


def test_prompt_attention_with_bad_pages():
    mk = Made(1, 1, 1, 64, 32, 8, seed=6)
    rng = np.random.default_rng(0)
    r = mk.fill([240], rng)
    q = rng.standard_normal((1, 80, 1, 64)).astype(np.float32)
    kk, vv = r.entries(0, 0, 0, 240)
    mk.table[0, 0, 4] = mk.codes.shape[0] + 7
    out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([160]), out_dtype=torch.float32).cpu().numpy()
    assert device_error() == 0x400
    for t in (0, 5, 79):
        see = np.r_[0:128, 160:161 + t]
        s = q[0, t, 0].astype(np.float64) @ kk[see].T / 8
        p = np.exp(s - s.max())
        assert np.abs(out[0, t, 0] - p / p.sum() @ vv[see]).max() < 1e-2 * np.abs(vv).max()
    mk.table[0, 0, 4] = int(mk.table_np[0, 0, 4])
    mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([200]))
    assert device_error() == 0x400                           # entries past the capacity


def test_prompt_values_of_very_different_size():
    mk = Made(1, 1, 1, 128, 16, 8, seed=1)
    rng = np.random.default_rng(3)
    k = rng.standard_normal((1, 128, 1, 128)).astype(np.float32)
    v = rng.standard_normal((1, 128, 1, 128)).astype(np.float32)
    v *= np.repeat(2.0 ** np.array([0, -12, 3, -9, 0, -14, 6, -3]), 16).astype(np.float32)[None, :, None, None]
    v[:, 64:80] = 0
    k[:, 32:48] *= 20
    r = mk.reference()
    mk.cache.write(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0]))
    r.append(0, k, v, [0], [128])
    kk, vv = r.entries(0, 0, 0, 128)
    q = (kk / (kk ** 2).sum(-1, keepdims=True) * 40 * np.sqrt(128)).astype(np.float32).reshape(1, 128, 1, 128)
    out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([0]), out_dtype=torch.float32).cpu().numpy()
    want, _, bound = r.attention(0, q, [0])
    for t in range(127):
        s = kk[:t + 1] @ q[0, t, 0].astype(np.float64) / np.sqrt(128)
        p = np.exp(s - s.max())
        p /= p.sum()
        # weights off by 2 delta + 2^-11; f16 values keep 2^-30 of the largest block's
        delta = ref.prompt_tolerance(128, 128, bound, 1.0, 0.0)[1]
        ab = delta * (p @ np.abs(vv[:t + 1])) + 2.0 ** -30 * np.abs(vv).max()
        assert (np.abs(out[0, t, 0] - want[0, t, 0]) <= ab).all(), t


# ---------------------------------------------------------------- eviction
def run_evict(mk, r, n, budget, sink, recent, mass, layer=0, pages=None):
    m = [min(x, max(y, sink + recent)) for x, y in zip(n, budget)]
    pages = pages or max(1, max(-(-x // mk.page) for x in m))
    used = set(mk.table_np.reshape(-1).tolist())
    free = [p for p in range(mk.codes.shape[0]) if p not in used]
    out = np.array(free[: mk.batch * pages], np.int32).reshape(mk.batch, pages)
    pos = torch.arange(mk.cap, dtype=torch.int32, device="cuda").expand(mk.batch, mk.kv, -1).contiguous() * 3
    before = mk.codes[torch.from_numpy(mk.table_np.reshape(-1)).cuda().long()].clone()
    kept, mass2, pos2 = mk.cache.evict_rows(layer, i32(n), i32(budget), torch.from_numpy(out).cuda(),
                                            torch.from_numpy(mass).cuda(), pos, sink, recent)
    assert torch.equal(mk.codes[torch.from_numpy(mk.table_np.reshape(-1)).cuda().long()], before)
    kept, mass2, pos2 = kept.cpu().numpy(), mass2.cpu().numpy(), pos2.cpu().numpy()
    want = mk.reference()
    got = mk.reference()
    want.vals[out.reshape(-1)] = 0
    for b in range(mk.batch):
        for h in range(mk.kv):
            ks = ref.evict(mass[b, h], n[b], budget[b], sink, recent)
            assert kept[b, h, :len(ks)].tolist() == ks.tolist(), (b, h)
            assert (kept[b, h, len(ks):] == -1).all()
            assert np.array_equal(mass2[b, h, :len(ks)], mass[b, h, ks]) and (mass2[b, h, len(ks):] == 0).all()
            assert np.array_equal(pos2[b, h, :len(ks)], 3 * ks) and (pos2[b, h, len(ks):] == -1).all()
            if not len(ks):
                continue
            k, v = r.entries(b, layer, h, n[b])
            for p in range(0, len(ks), mk.page):
                rows = ks[p:p + mk.page]
                for i, x in ((0, k), (1, v)):
                    want._put(out[b, p // mk.page], h, i, 0, x[rows])
                pid = out[b, p // mk.page]
                assert np.array_equal(got.exp[pid, h], want.exp[pid, h])
                assert np.array_equal(got.vals[pid, h, :, :len(rows)], want.vals[pid, h, :, :len(rows)])
    return out, kept


EVICTS = [   # batch, kv, d, page, pages, n, budget, sink, recent
    (1, 1, 64, 16, 2, [1], [1], 0, 0), (1, 1, 64, 16, 2, [30], [1], 0, 0), (2, 2, 64, 16, 6, [90, 41], [40, 41], 4, 8),
    (2, 3, 128, 32, 5, [150, 0], [60, 9], 1, 16), (1, 2, 128, 64, 4, [256], [255], 0, 1), (2, 1, 64, 128, 2, [200, 129], [30, 500], 4, 64),
    (1, 2, 64, 16, 200, [3150], [1000], 4, 32), (1, 1, 128, 16, 4, [50], [3], 20, 30), (1, 1, 64, 16, 4, [64], [10], 40, 40),
]


@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"b{c[0]}kv{c[1]}d{c[2]}p{c[3]}n{c[5][0]}m{c[6][0]}")
def test_evict_matches_the_definition(case):
    batch, kv, d, page, pages, n, budget, sink, recent = case
    mk = Made(batch, 1, kv, d, page, pages, seed=page, spare=batch * pages)
    rng = np.random.default_rng(page + n[0])
    r = mk.fill(n, rng, spread=1.5)
    mass = np.exp(2 * rng.standard_normal((batch, kv, mk.cap))).astype(np.float32)
    mass[rng.random(mass.shape) < 0.3] = 0.0
    run_evict(mk, r, n, budget, sink, recent, mass)


@pytest.mark.parametrize("kind", ["all equal", "two values", "negative zero", "descending", "tiny and huge", "infinite"])
def test_evict_order_of_hard_masses(kind):
    mk = Made(1, 1, 2, 64, 16, 80, seed=2, spare=80)
    rng = np.random.default_rng(3)
    r = mk.fill([1270], rng)
    mass = np.zeros((1, 2, mk.cap), np.float32)
    if kind == "all equal":
        mass[:] = 0.25
    elif kind == "two values":
        mass[:] = rng.integers(0, 2, mass.shape)
    elif kind == "negative zero":
        mass[:] = np.where(rng.random(mass.shape) < 0.5, -0.0, 0.0)
    elif kind == "descending":
        mass[:] = np.arange(mk.cap, 0, -1)
    elif kind == "tiny and huge":
        mass[:] = 10.0 ** rng.uniform(-44, 38, mass.shape)
    else:
        mass[:] = np.where(rng.random(mass.shape) < 0.5, np.inf, rng.random(mass.shape))
    run_evict(mk, r, [1270], [511], 3, 70, mass)


@pytest.mark.parametrize("kv,pages,n,budget,kind", [
    (1, 72, [9001], [2300], "lognormal"), (2, 160, [20000], [5000], "ties"), (1, 330, [42000], [40001], "lognormal"),
    (1, 330, [700], [333], "ties"), (1, 3136, [401000], [2000], "ties"), (3, 330, [42240], [1], "equal")])
def test_evict_from_long_sequences(kv, pages, n, budget, kind):
    """Selections over several CTAs (clusters of 2, 4 and 8), a short sequence in a
    long capacity, and slices that shared memory does not hold."""
    mk = Made(1, 1, kv, 64, 128, pages, seed=4, spare=pages)
    rng = np.random.default_rng(n[0])
    mk.codes.copy_(torch.randint(0, 127, mk.codes.shape, dtype=torch.uint8, device="cuda"))      # any finite codes
    mk.scale.copy_(torch.ldexp(torch.ones(mk.scale.shape, device="cuda"), torch.randint(-9, 3, mk.scale.shape, device="cuda")))
    mass = np.exp(2 * rng.standard_normal((1, kv, mk.cap))).astype(np.float32)
    if kind == "ties":
        mass = np.round(mass * 2).astype(np.float32)
    elif kind == "equal":
        mass[:] = 1.5
    run_evict(mk, mk.reference(), n, budget, 4, 64, mass)


def test_evict_into_too_small_a_table_is_reported():
    mk = Made(1, 1, 1, 64, 16, 4, seed=2, spare=8)
    rng = np.random.default_rng(1)
    mk.fill([60], rng)
    mass = torch.rand((1, 1, 64), device="cuda")
    kept, m2, _ = mk.cache.evict_rows(0, i32([60]), i32([40]), i32([[64 // 16]]) * 0 + int(mk.codes.shape[0] - 1), mass)
    assert device_error() == 0x400
    assert (kept[0, 0] >= 0).all() and kept.shape == (1, 1, 16)


# ------------------------------------------------------------ run together
def test_append_attend_evict_and_go_on():
    """As a bounded cache is used: prompt, decode steps that add up the mass,
    eviction, more steps, a rollback; every state against the reference."""
    from draftkv import Q8KVCache
    d, kv, group, page = 64, 2, 2, 16
    cache = Q8KVCache(1, kv, d, block_size=page, n_blocks=40, max_blocks_per_seq=16, track_mass=True)
    rng = np.random.default_rng(0)
    K = np.zeros((kv, 0, d))
    V = np.zeros((kv, 0, d))
    mass = np.zeros((kv, 0))
    where = np.zeros((kv, 0), np.int64)

    def sync():
        """The dequantized cache is the truth for the next attention."""
        n = cache.length
        o = cache.read_rows(0, n).double().cpu().numpy()
        return o[:, :, 0].transpose(1, 0, 2), o[:, :, 1].transpose(1, 0, 2)

    def put(n, pos):
        nonlocal mass, where
        x = rng.standard_normal((2, n, kv, d)).astype(np.float32)
        cache.append(0, x[0], x[1], np.arange(pos, pos + n))
        mass = np.concatenate([mass, np.zeros((kv, n))], 1)
        where = np.concatenate([where, np.tile(np.arange(pos, pos + n), (kv, 1))], 1)
        k, v = sync()
        # 3 fraction bits of e4m3: at most 2^-4 of the value, or of the block's smallest normal
        assert np.abs(k[:, -n:] - x[0].transpose(1, 0, 2)).max() <= 2.0 ** -4 * np.abs(x).max()

    def step():
        nonlocal mass
        n = cache.length
        q = rng.standard_normal((1, 1, kv * group, d)).astype(np.float32)
        k, v = sync()
        got = cache.attention(0, torch.from_numpy(q).cuda(), i32([n - 1]), mass=cache.mass[0], out_dtype=torch.float32)
        for h in range(kv):
            s = q[0, 0, h * group:(h + 1) * group].astype(np.float64) @ k[h].T / np.sqrt(d)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            assert np.abs(got[0, 0, h * group:(h + 1) * group].cpu().numpy() - p @ v[h]).max() < 1e-4
            mass[h] += p.sum(0)

    pos = 0
    put(50, pos)
    pos = 50
    for _ in range(14):
        put(1, pos)
        pos += 1
        step()
    for _ in range(2):
        n = cache.length
        dev_mass = cache.mass[0][0, :, :n].cpu().numpy()
        assert np.abs(dev_mass - mass).max() < 1e-4
        kept = cache.evict(32, sink=2, recent=8)[0].cpu().numpy()[0]
        for h in range(kv):
            ks = ref.evict(dev_mass[h], n, 32, 2, 8)
            assert kept[h, :32].tolist() == ks.tolist()
        mass = np.stack([mass[h, kept[h, :32]] for h in range(kv)])
        where = np.stack([where[h, kept[h, :32]] for h in range(kv)])
        assert cache.length == 32 and cache.blocks_in_use == 2
        assert np.array_equal(cache.positions(0), where)
        for _ in range(20):
            put(1, pos)
            pos += 1
            step()
        assert np.array_equal(cache.positions(0), where)
    cache.truncate(45)
    assert cache.length == 45 and cache.blocks_in_use == 3
    cache.pool.check_invariants()
    mass, where, pos = mass[:, :45], where[:, :45], pos - 7
    put(3, pos)
    step()


def test_side_streams_and_a_replayed_graph():
    """Two streams at once over one cache, and a captured decode step replayed on new inputs."""
    mk = Made(2, 1, 2, 128, 16, 70, seed=7)
    rng = np.random.default_rng(1)
    mk.fill([1100, 700], rng)
    q = torch.randn((2, 1, 8, 128), device="cuda")
    e0 = i32([1099, 699])
    want = mk.cache.attention(0, q, e0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([mk.cache.attention(0, q, e0) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for run in outs for o in run)
    # capture: append one token, attend to it with the mass
    k, v = (torch.randn((2, 1, 2, 128), device="cuda") for _ in range(2))
    n = e0 + 1
    mass = torch.zeros((2, 2, mk.cap), device="cuda")
    out = torch.empty((2, 1, 8, 128), dtype=torch.bfloat16, device="cuda")

    def body():
        mk.cache.write(0, k, v, n)
        mk.cache.attention(0, q, n, out=out, mass=mass)

    body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body()
    for i in range(3):
        n += 1
        k.copy_(torch.randn_like(k))
        q.copy_(torch.randn_like(q))
        mass.zero_()
        g.replay()
        got, got_m = out.clone(), mass.clone()
        mass.zero_()
        body()
        assert torch.equal(out, got) and torch.equal(mass, got_m)


def test_class_refuses_wrong_tensors():
    mk = Made(2, 1, 2, 64, 16, 4)
    c = mk.cache
    x = torch.zeros((2, 3, 2, 64), device="cuda")
    q = torch.zeros((2, 1, 4, 64), device="cuda")
    e0, m = i32([0, 0]), torch.zeros((2, 2, 64), device="cuda")
    for args, kw in (((0, x[:1], x[:1], e0), {}), ((0, x, x[..., :32], e0), {}), ((0, x.double(), x.double(), e0), {}),
                     ((0, x, x.to(torch.bfloat16), e0), {}), ((0, x.cpu(), x.cpu(), e0), {}),
                     ((0, x, x, e0.long()), {}), ((0, x, x, e0[:1]), {}), ((0, x, x, e0), dict(n_rows=e0.float())),
                     ((0, x, x, e0), dict(mass=m[:, :, :32])), ((0, x, x, e0), dict(pos=m)),
                     ((0, x[:, :2], x[:, ::2], e0), {})):
        with pytest.raises(ValueError):
            c.write(*args, **kw)
    for args, kw in (((0, q[:1], e0), {}), ((0, q[:, :, :3], e0), {}), ((0, q.to(torch.bfloat16), e0), {}),
                     ((0, q.cpu(), e0), {}), ((0, q, e0.cpu()), {}), ((0, q, e0), dict(out_dtype=torch.float16)),
                     ((0, q, e0), dict(out=q[:1])), ((0, q, e0), dict(mass=m.double())),
                     ((0, q[..., :32], e0), {}), ((0, q.transpose(1, 2), e0), {})):
        with pytest.raises(ValueError):
            c.attention(*args, **kw)
    from draftkv import DraftKVError
    with pytest.raises(DraftKVError):
        c.attention(0, torch.zeros((2, 17, 8, 64), device="cuda"), e0, mass=m)     # 68 rows a head
    with pytest.raises(DraftKVError):
        c.attention(1, q, e0)
    with pytest.raises(DraftKVError):
        c.attention(0, q, e0, split_keys=100)
    with pytest.raises(ValueError):
        c.evict_rows(0, e0, e0, i32([0, 1]), m)
    with pytest.raises(ValueError):
        c.evict_rows(0, e0, e0, i32([[0], [1]]), None)


def test_captured_calls_have_scratch_of_their_own():
    """Two graphs captured on one stream that has run the call before (so that the
    cache holds scratch for it) are replayed side by side; one eviction inside."""
    mk = Made(1, 1, 2, 128, 16, 130, seed=7, spare=8)
    rng = np.random.default_rng(1)
    mk.fill([2000], rng)
    e0, n, m, mass = i32([1997]), i32([2000]), i32([64]), torch.rand((1, 2, mk.cap), device="cuda")
    used = set(mk.table_np.reshape(-1).tolist())
    table = i32([[p for p in range(mk.codes.shape[0]) if p not in used][:4]])
    s, side = torch.cuda.Stream(), torch.cuda.Stream()
    qs = [torch.randn((1, 3, 8, 128), device="cuda") for _ in range(2)]
    outs = [torch.empty((1, 3, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        want = [mk.cache.attention(0, q, e0) for q in qs]
        gone = mk.cache.evict_rows(0, n, m, table, mass, None, 2, 16)
        eager = mk.cache._workspace(3, 4, 0, False, s.cuda_stream)
    torch.cuda.synchronize()
    graphs, kept = [], None
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert mk.cache._workspace(3, 4, 0, False, s.cuda_stream).data_ptr() != eager.data_ptr()
            for _ in range(4):
                mk.cache.attention(0, qs[i], e0, out=outs[i])
            if i == 0:
                kept = mk.cache.evict_rows(0, n, m, table, mass, None, 2, 16)
        graphs.append(g)
    for _ in range(10):
        for g, st in zip(graphs, (s, side)):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert mk.cache._workspace(3, 4, 0, False, s.cuda_stream) is eager
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    assert torch.equal(kept[0], gone[0]) and torch.equal(kept[1], gone[1])


def test_one_scratch_serves_calls_of_any_size():
    """Decode, verify, mass and prompt calls of one stream in turn, each over what the others left."""
    mk = Made(1, 1, 2, 64, 16, 1280, seed=3)
    rng = np.random.default_rng(2)
    mk.fill([20000], rng, spread=0.5)
    mass = torch.zeros((1, 2, mk.cap), device="cuda")
    calls = [(1, False, 0), (40, False, 0), (6, True, 0), (200, False, 0), (8, True, 256), (1, False, 512), (30, True, 0)]
    q = [torch.randn((1, T, 4, 64), device="cuda") for T, _, _ in calls]

    def run(i, **kw):
        T, noted, split = calls[i]
        return mk.cache.attention(0, q[i], i32([20000 - T]), mass=mass if noted else None, split_keys=split, **kw)

    want = []
    for i, (T, noted, split) in enumerate(calls):      # scratch of its own, cleared as the header asks
        nb = lib().load().dkv_q8_attn_work_bytes(mk.cache._dims, 2, T, mk.cap, split, int(noted))
        w = torch.full((nb,), 0xA5, dtype=torch.uint8, device="cuda")
        w[:65536] = 0
        want.append(run(i, work=w))
        assert (w[:65536] == 0).all()
    for order in (range(len(calls)), reversed(range(len(calls)))):
        for i in order:
            assert torch.equal(run(i), want[i]), calls[i]
    assert len({w.data_ptr() for w in mk.cache._work.values()}) == 1


def test_prompt_values_near_the_smallest_scale():
    """Thousands of entries whose scores stay just below the growth that raises the
    max, over V at the smallest scale: 2^-120 over the sum (2^26) is far below fp32's
    normal numbers, the outputs (2^-115) are not."""
    d, n, T = 64, 8192, 70
    mk = Made(1, 1, 1, d, 16, n // 16, seed=5)
    rng = np.random.default_rng(4)
    k = np.zeros((1, n, 1, d), np.float32)
    k[:, 128:] = 7.5 * np.log(2) * np.sqrt(d) / d
    v = np.ldexp(1 + rng.random((1, n, 1, d)), -115).astype(np.float32)
    r = mk.reference()
    mk.cache.write(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0]))
    r.append(0, k, v, [0], [n])
    kk, vv = r.entries(0, 0, 0, n)
    assert 7 < (kk[-1].sum() / np.sqrt(d)) / np.log(2) < 8
    q = np.ones((1, T, 1, d), np.float32)
    out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([n - T]), out_dtype=torch.float32).double().cpu().numpy()
    want, _, bound = r.attention(0, q, [n - T])
    # 2^-115 <= v <= 2^-114 (rounded to e4m3 too), so an error of delta x the largest v is 2 delta of the output
    delta = ref.prompt_tolerance(d, n, bound, 1.0, 0.0)[1]
    assert (np.abs(out - want) <= 2 * delta * want).all()


def test_more_rows_than_tickets_where_the_keys_are_not_split():
    mk = Made(600, 1, 32, 64, 16, 1, seed=8)
    rng = np.random.default_rng(3)
    mk.fill([int(x) for x in rng.integers(1, 17, 600)], rng)
    q = torch.randn((600, 1, 32, 64), device="cuda")
    e0 = torch.from_numpy(rng.integers(0, 16, 600).astype(np.int32)).cuda()
    from draftkv import Q8KVCache
    out = torch.zeros((600, 1, 32, 64), dtype=torch.bfloat16, device="cuda")
    n = torch.from_numpy(np.random.default_rng(3).integers(1, 17, 600).astype(np.int32)).cuda()
    e0 = torch.minimum(e0, n - 1)
    mk.cache.attention(0, q, e0, out=out)
    for a in (0, 300):
        half = Q8KVCache.from_storage(mk.codes, mk.scale, mk.table[a:a + 300].contiguous())
        assert torch.equal(half.attention(0, q[a:a + 300], e0[a:a + 300]), out[a:a + 300])


def test_extreme_entries_and_split_lengths():
    mk = Made(1, 1, 1, 64, 16, 6, seed=6)
    mk.fill([96], np.random.default_rng(0))
    for T in (1, 4, 80):
        q = torch.randn((1, T, 2, 64), device="cuda")
        last = mk.cache.attention(0, q, i32([96]))              # every token sees all 96
        assert device_error() == 0x400
        for e0 in (97, 2 ** 30, 2 ** 31 - 1):
            assert torch.equal(mk.cache.attention(0, q, i32([e0])), last)
            assert device_error() == 0x400
        assert (mk.cache.attention(0, q, i32([-2 ** 31])) == 0).all()
        whole = mk.cache.attention(0, q, i32([96 - T]))
        for split in (128, 2 ** 31 - 128):
            assert torch.equal(mk.cache.attention(0, q, i32([96 - T]), split_keys=split), whole)


def test_evict_plans_all_layers_first():
    """Too few free blocks, a layer named twice, a layer that is not there, and how
    far back a sequence can go after an eviction."""
    from draftkv import BlockPoolExhausted, Q8KVCache
    c = Q8KVCache(2, 1, 64, block_size=16, n_blocks=10, max_blocks_per_seq=8, track_mass=True)
    x = np.random.default_rng(0).standard_normal((80, 1, 64)).astype(np.float32)
    c.append(0, x[:17], x[:17], np.arange(17))
    c.append(1, x, x, np.arange(80))
    for m in c.mass:
        m.copy_(torch.rand_like(m))

    def state():
        return [c.counts, c.block_tables, c.pool.n_free, c._floor]

    import copy
    before = copy.deepcopy(state())
    with pytest.raises(BlockPoolExhausted):        # 4 blocks for layer 1, 3 are free
        c.evict(64, sink=0, recent=0)
    with pytest.raises(ValueError):
        c.evict(8, sink=0, recent=4, layers=[1, -1])
    with pytest.raises(ValueError):
        c.evict(8, sink=0, recent=4, layers=[2])
    assert state() == before
    c.pool.check_invariants()
    out = c.evict(8, sink=0, recent=4, layers=[0, 0, 1])
    assert set(out) == {0, 1} and c.counts == [[8, 8]]
    c.pool.check_invariants()
    assert all(p[-4:] == list(range(n - 4, n)) for p, n in zip(c.pos, (17, 80)))
    c.next_pos[0] = 80
    with pytest.raises(ValueError):
        c.truncate(3)
    c.truncate(5)
    assert c.length == 5 and c.next_pos == [77]
    c.truncate(0)
    assert c.length == 0 and c.next_pos == [0] and c.blocks_in_use == 0
    c.append(0, x[:3], x[:3], np.arange(3))
    c.truncate(1)


def test_class_refuses_foreign_scratch():
    mk = Made(1, 1, 1, 64, 16, 4)
    mk.fill([3], np.random.default_rng(0))
    q, e0 = torch.zeros((1, 1, 1, 64), device="cuda"), i32([2])
    for w in (torch.zeros(1 << 20, device="cuda"), torch.zeros(1 << 20, dtype=torch.uint8),
              torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError):
            mk.cache.attention(0, q, e0, work=w)
