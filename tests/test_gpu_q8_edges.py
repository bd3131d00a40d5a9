"""The 8-bit paged cache on the GPU where its blocks, tiles and scales are
least even: what a row of attention may depend on, values of any size, rows and
blocks of zeros.  Against the 64-bit restatement (tests/q8_reference.py)."""
import numpy as np
import pytest

from tests import q8_reference as ref
from tests.test_gpu_q8 import Made, clean_error_word, device_error, i32  # noqa: F401 (clean_error_word: a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def fill(mk, k, v, n):
    """Writes k, v [batch, rows, kv, d] (fp32) from the start, n[b] rows; returns the reference."""
    r = mk.reference()
    mk.cache.write(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0] * mk.batch), n_rows=i32(n))
    r.append(0, k, v, [0] * mk.batch, n)
    return r


def row_error(mk, r, b, h, n, q, got, out_dtype, see=None, prompt=False):
    """Largest error of output rows got [rows, d] of queries q [rows, d] over entries
    `see` (all n) of one head, in units of the bound.

    An output is sum p v.  Weights are off by the factor 1 +- 2 delta (scores,
    sums and merges: attention_tolerance with vmax 1), so the sum by 2 delta
    sum p |v|.  What enters the product is p 2^(e - E) in f16 beside codes of at
    most 448, e the block's exponent and E the largest of the blocks in sight:
    one f16 number for bf16 outputs (half a step, 2^-11 of it), two for fp32
    (2^-22), and below f16's normal numbers half a step of 2^-24 beside weights
    that enter times 2^6: 2^-31 of 448 2^E for each key.  Then one rounding to
    the output's type.  Prompt calls with bf16 outputs: queries are one f16
    number too, see prompt_tolerance."""
    see = np.arange(n) if see is None else see
    kk, vv = (x[see] for x in r.entries(b, 0, h, n))
    s = q.astype(np.float64) @ kk.T / np.sqrt(mk.d)
    bound = (np.abs(q.astype(np.float64)) @ np.abs(kk).T).max() / np.sqrt(mk.d)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = p @ vv
    top = 448 * 2.0 ** max(int(r.exp[mk.table_np[b, 0, e // mk.page], h, 1]) for e in see)
    delta = ref.attention_tolerance(mk.d, n, bound, 1.0, 0.0)[1] + (2.0 ** -11 if out_dtype is BF16 else 2.0 ** -22)
    if prompt and out_dtype is BF16:
        delta += 2 * 2.0 ** -11 * bound
    tol = delta * (p @ np.abs(vv)) + len(see) * 2.0 ** -31 * top + torch.finfo(out_dtype).eps / 2 * np.abs(want) \
        + torch.finfo(out_dtype).smallest_normal
    return float((np.abs(got.double().cpu().numpy() - want) / tol).max())


# ----------------------------------------------- up to 64 rows: tiles of a unit
@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 16)])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e-6, 2.0 ** -30, 2.0 ** -100])
def test_small_values_in_a_half_filled_unit(d, page, size):
    """Lengths whose last 32 entries hold one tile of 16, or a part of it."""
    lengths = [1, 5, 12, 16, 33, 37, 48, 64]
    mk = Made(len(lengths), 1, 2, d, page, 128 // page, seed=d)
    rng = np.random.default_rng(page)
    k, v = (rng.standard_normal((len(lengths), 64, 2, d)).astype(np.float32) for _ in range(2))
    r = fill(mk, k, (v * np.float32(size)).astype(np.float32), lengths)
    for group in (1, 3, 6):
        q = rng.standard_normal((len(lengths), 1, 2 * group, d)).astype(np.float32)
        for dt in (BF16, F32):
            out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([n - 1 for n in lengths]), out_dtype=dt)
            for b, n in enumerate(lengths):
                for h in range(2):
                    at = slice(h * group, (h + 1) * group)
                    err = row_error(mk, r, b, h, n, q[b, 0, at], out[b, 0, at], dt)
                    assert err <= 1, (n, group, dt, err)


def test_small_values_beside_a_bad_page():
    mk = Made(1, 1, 1, 64, 16, 6, seed=6)
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((1, 90, 1, 64)).astype(np.float32) for _ in range(2))
    r = fill(mk, k, (v * 1e-8).astype(np.float32), [90])
    q = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    for page in (2, 3):
        mk.table[0, 0, page] = -1
        for dt in (BF16, F32):
            out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([89]), out_dtype=dt)
            assert device_error() == 0x400
            see = np.r_[0:16 * page, 16 * page + 16:90]
            assert row_error(mk, r, 0, 0, 90, q[0, 0], out[0, 0], dt, see) <= 1
        mk.table[0, 0, page] = int(mk.table_np[0, 0, page])


@pytest.mark.parametrize("d,page", [(64, 16), (64, 32), (128, 16)])
@pytest.mark.parametrize("step", [0, 10, -10, 40, 200, -200])
def test_rows_do_not_depend_on_tiles_they_do_not_see(d, page, step):
    """Verify calls from a unit's first tile into its second and beyond, V of
    neighbouring tiles 2^step apart (at 200 from one end of the scales to the
    other): every row equals the one-token call at its entry bit for bit."""
    mk = Made(2, 1, 1, d, page, 1280 // page, seed=5)
    rng = np.random.default_rng(d + page)
    k, v = (rng.standard_normal((2, 1280, 1, d)).astype(np.float32) for _ in range(2))
    size = np.ldexp(1.0, (np.arange(1280) // 16 % 2) * step - (step // 2 if step > 100 else 0)
                    + (-step // 2 if step < -100 else 0))
    fill(mk, k, (v * size[None, :, None, None]).astype(np.float32), [1280, 1280])
    for e0, T, group in (([10, 1194], 9, 1), ([1194, 26], 9, 3), ([10, 1178], 17, 1), ([15, 31], 2, 2), ([8, 1000], 21, 3)):
        q = torch.from_numpy((rng.standard_normal((2, T, group, d)) * 2).astype(np.float32)).cuda()
        for dt in (BF16, F32):
            whole = mk.cache.attention(0, q, i32(e0), out_dtype=dt)
            assert torch.isfinite(whole).all()
            for t in range(T):
                one = mk.cache.attention(0, q[:, t:t + 1].contiguous(), i32([x + t for x in e0]), out_dtype=dt)
                assert torch.equal(one[:, 0], whole[:, t]), (e0, T, group, dt, t)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group,T", [(1, 64), (4, 16), (1, 8)])
def test_rows_do_not_depend_on_far_larger_values_behind_them(d, group, T):
    """From entry 256 on V is 2^200 larger: the rows before it, in one call with
    rows behind it, give what they give alone."""
    mk = Made(1, 1, 1, d, 16, 80, seed=5)
    rng = np.random.default_rng(d)
    k, v = (rng.standard_normal((1, 320, 1, d)).astype(np.float32) for _ in range(2))
    v = np.ldexp(v, np.where(np.arange(320) < 256, -100, 100)[None, :, None, None]).astype(np.float32)
    r = fill(mk, k, v, [320])
    q = rng.standard_normal((1, T, group, d)).astype(np.float32)
    e0 = 259 - T
    for dt in (BF16, F32):
        whole = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([e0]), out_dtype=dt)
        for t in range(T):
            one = mk.cache.attention(0, torch.from_numpy(q[:, t:t + 1].copy()).cuda(), i32([e0 + t]), out_dtype=dt)
            assert torch.equal(one[:, 0], whole[:, t]), (dt, t)
            assert row_error(mk, r, 0, 0, e0 + t + 1, q[0, t], whole[0, t], dt) <= 1, (dt, t)


# ------------------------------------------------------------- prompt chunks
def check_rows(mk, r, q, e0, out, out_dtype, prompt=True):
    for b in range(mk.batch):
        for h in range(mk.kv):
            G = q.shape[2] // mk.kv
            for t in range(q.shape[1]):
                at = slice(h * G, (h + 1) * G)
                err = row_error(mk, r, b, h, e0[b] + t + 1, q[b, t, at], out[b, t, at], out_dtype, prompt=prompt)
                assert err <= 1, (b, h, t, err)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [3, 100])
def test_rows_and_blocks_of_zeros(d, T):
    """Queries of zero, tiny ones, keys of zero: equal weights over what is seen,
    also where 2^-100 (a zero query's exponent) meets 2^-120 (a zero block's)."""
    mk = Made(1, 1, 1, d, 16, 16, seed=2)
    rng = np.random.default_rng(d)
    k, v = (rng.standard_normal((1, 200, 1, d)).astype(np.float32) for _ in range(2))
    k[:, :48] = 0
    k[:, 64:96] *= np.float32(2.0 ** -110)
    v[:, 16:32] = 0
    r = fill(mk, k, v, [200])
    q = rng.standard_normal((1, T, 2, d)).astype(np.float32)
    q[:, ::3] = 0
    q[:, 1::3] *= np.float32(2.0 ** -90)
    for e0 in (0, 30, 200 - T):
        out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([e0]), out_dtype=BF16)
        check_rows(mk, r, q, [e0], out, BF16)
    # keys near fp32's largest under queries near its smallest
    k = (rng.standard_normal((1, 200, 1, d)) * 2.0 ** 120).astype(np.float32)
    r = fill(mk, k, v, [200])
    q = (rng.standard_normal((1, T, 2, d)) * 2.0 ** -120).astype(np.float32)
    out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([200 - T]), out_dtype=BF16)
    check_rows(mk, r, q, [200 - T], out, BF16)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 64)])
@pytest.mark.parametrize("step", [24, 60, 200])
def test_prompt_rows_before_far_larger_values(d, page, step):
    """V grows by 2^step at entry 48 (inside the first tile of 128 keys), or at
    200: rows before it keep the precision of what they see."""
    T = 280
    rng = np.random.default_rng(d + step)
    for at in (48, 200):
        mk = Made(1, 1, 1, d, page, 320 // page, seed=2)
        k, v = (rng.standard_normal((1, T, 1, d)).astype(np.float32) for _ in range(2))
        at -= at % page
        v = np.ldexp(v, np.where(np.arange(T) < at, -step // 2, step - step // 2)[None, :, None, None]).astype(np.float32)
        r = fill(mk, k, v, [T])
        q = rng.standard_normal((1, T, 1, d)).astype(np.float32)
        out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([0]), out_dtype=BF16)
        check_rows(mk, r, q, [0], out, BF16)


def test_prompt_rows_before_far_larger_values_over_key_splits():
    """The same where the keys are split (512 a split) and where a bad page lies between."""
    T, e0, d = 100, 1000, 128
    rng = np.random.default_rng(1)
    for at, bad in ((1056, None), (992, 30), (512, None), (96, 61)):
        mk = Made(1, 1, 1, d, 16, 80, seed=2)
        k, v = (rng.standard_normal((1, e0 + T, 1, d)).astype(np.float32) for _ in range(2))
        v = np.ldexp(v, np.where(np.arange(e0 + T) < at, -60, 40)[None, :, None, None]).astype(np.float32)
        r = fill(mk, k, v, [e0 + T])
        if bad is not None:
            mk.table[0, 0, bad] = -1
        q = rng.standard_normal((1, T, 2, d)).astype(np.float32)
        out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([e0]), out_dtype=BF16)
        assert device_error() == (0 if bad is None else 0x400)
        for t in range(0, T, 7):
            see = np.arange(e0 + t + 1)
            see = see if bad is None else see[see // 16 != bad]
            assert row_error(mk, r, 0, 0, e0 + t + 1, q[0, t], out[0, t], BF16, see, prompt=True) <= 1, (at, t)


WIDE = [   # batch, kv, group, d, page, pages, T, entries before the call, n_rows
    (1, 1, 1, 64, 16, 5, 65, [0], None), (2, 2, 4, 128, 16, 20, 17, [300, 0], None), (1, 1, 1, 64, 32, 10, 301, [3], None),
    (2, 1, 3, 128, 64, 6, 100, [250, 7], [100, 31]), (3, 1, 2, 64, 16, 40, 129, [500, 128, -20], None),
    (1, 1, 2, 128, 16, 80, 70, [1200], None), (2, 1, 4, 64, 16, 320, 40, [5000, 17], [40, 0]),
]


@pytest.mark.parametrize("shape", WIDE, ids=lambda s: f"b{s[0]}kv{s[1]}g{s[2]}d{s[3]}p{s[4]}T{s[6]}")
@pytest.mark.parametrize("size", [1.0, 1e-20])
def test_prompt_calls_with_fp32_outputs_hold_their_bits(shape, size):
    """More than 64 rows a head, fp32 outputs: queries and weights as two f16
    numbers each, as calls of up to 64 rows hold them."""
    batch, kv, group, d, page, pages, T, e0, n_rows = shape
    mk = Made(batch, 1, kv, d, page, pages, seed=T)
    rng = np.random.default_rng(d + T)
    n = [max(x + T, 1) for x in e0]
    k, v = (rng.standard_normal((batch, max(n), kv, d)).astype(np.float32) for _ in range(2))
    v *= np.exp(rng.standard_normal((batch, max(n), kv, 1))).astype(np.float32)
    r = fill(mk, k, (v * np.float32(size)).astype(np.float32), n)
    q = (rng.standard_normal((batch, T, kv * group, d)) * 1.5).astype(np.float32)
    out = torch.full(q.shape, 5.0, device="cuda")
    mk.cache.attention(0, torch.from_numpy(q).cuda(), i32(e0), n_rows=None if n_rows is None else i32(n_rows), out=out)
    for b in range(batch):
        live = T if n_rows is None else n_rows[b]
        assert (out[b, live:] == 5).all()
        for t in range(0, live, 3):
            if e0[b] + t < 0:
                assert (out[b, t] == 0).all()
                continue
            for h in range(kv):
                at = slice(h * group, (h + 1) * group)
                err = row_error(mk, r, b, h, e0[b] + t + 1, q[b, t, at], out[b, t, at], F32, prompt=True)
                assert err <= 1, (b, t, h, err)


def test_prompt_calls_with_fp32_outputs_where_scales_differ():
    """fp32 outputs over blocks 2^24 and 2^60 apart, zeros and a bad page."""
    T, d = 200, 64
    rng = np.random.default_rng(6)
    mk = Made(1, 1, 1, d, 16, 16, seed=2)
    k, v = (rng.standard_normal((1, T, 1, d)).astype(np.float32) for _ in range(2))
    v = np.ldexp(v, np.array([-60, -36, 0, -3, 24, 0, 8, -50, 3, 30, 0, 0, 0])[np.arange(T) // 16][None, :, None, None])
    k[:, 32:48], v[:, 64:80] = 0, 0
    r = fill(mk, k.astype(np.float32), v.astype(np.float32), [T])
    q = rng.standard_normal((1, T, 2, d)).astype(np.float32)
    q[:, ::9] = 0
    for bad in (None, 3):
        if bad is not None:
            mk.table[0, 0, bad] = -1
        out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([0]), out_dtype=F32)
        assert device_error() == (0 if bad is None else 0x400)
        for t in range(T):
            see = np.arange(t + 1)
            see = see if bad is None else see[see // 16 != bad]
            assert row_error(mk, r, 0, 0, t + 1, q[0, t], out[0, t], F32, see, prompt=True) <= 1, t


# ------------------------------------------------------------------- scratch
def test_threads_with_streams_of_their_own_share_a_cache():
    """Several threads, a stream each, call one cache with sizes it has not seen:
    the scratch of one must not be in another's way."""
    import sys
    import threading
    mk = Made(1, 1, 1, 64, 16, 70, seed=4)
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((1, 1100, 1, 64)).astype(np.float32) for _ in range(2))
    fill(mk, k, v, [1100])
    calls = [(T, split) for T in range(1, 60) for split in (0, 128, 256)]
    q = {T: torch.randn((1, T, 1, 64), device="cuda") for T in range(1, 60)}
    e0 = {T: i32([1100 - T]) for T in q}
    want = {c: mk.cache.attention(0, q[c[0]], e0[c[0]], split_keys=c[1]) for c in calls}
    from draftkv import Q8KVCache
    shared = Q8KVCache.from_storage(mk.codes, mk.scale, mk.table)
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(4)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for c in calls[i::2] + calls[::2]:
                    got = shared.attention(0, q[c[0]], e0[c[0]], split_keys=c[1])
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(got, want[c]):
                        wrong.append(c)
        except Exception as e:
            wrong.append(e)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert not wrong, wrong[:3]


# -------------------------------------------------- values near fp32's largest
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32)])
@pytest.mark.parametrize("T,n", [(1, 1), (1, 700), (9, 300), (20, 1200), (80, 80), (100, 1200), (70, 40)])
def test_values_near_fp32_s_largest(d, page, T, n):
    """V up to 448 2^119, over one warp, several, key splits and prompt chunks:
    averages of finite values are finite."""
    mk = Made(1, 1, 1, d, page, 1280 // page, seed=3)
    rng = np.random.default_rng(T + n)
    n = max(n, T)
    k = (rng.standard_normal((1, n, 1, d)) * 0.3).astype(np.float32)
    v = np.ldexp(1 + rng.random((1, n, 1, d)) * 0.7, 127).astype(np.float32) * np.sign(rng.standard_normal((1, n, 1, 1))).astype(np.float32)
    r = fill(mk, k, v, [n])
    q = rng.standard_normal((1, T, 2, d)).astype(np.float32)
    mass = torch.zeros((1, 1, mk.cap), device="cuda") if T * 2 <= 64 else None
    for dt in (BF16, F32):
        for split in (0, 128) if T * 2 <= 64 else (0,):
            out = mk.cache.attention(0, torch.from_numpy(q).cuda(), i32([n - T]), out_dtype=dt, split_keys=split, mass=mass)
            assert torch.isfinite(out).all()
            check_rows(mk, r, q, [n - T], out, dt, prompt=T * 2 > 64)
