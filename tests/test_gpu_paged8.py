"""8-bit paged cache, append with rotation, and windowed attention on the GPU, against plain
64-bit implementations.

Tolerances.  A code is the nearest of the block's values: at most half a step away, 2^-4 of the
value (e4m3: 4 significant bits) or half the smallest step, s * 2^-10; rotated keys carry a few
fp32 roundings besides.  Attention: the output is rounded once (eps / 2 of its type), the
probabilities once (fp16 2^-11 in narrow tiles over an 8-bit cache, eps / 2 of the query's type
otherwise; so
the output moves by at most that times A = sum p |v|), and scores in fp32 move each
probability by a relative 2.4e-4 at the sizes here: D + 4 = 132 roundings of 2^-24 of sums whose terms
come to sum |q k| sm_scale <= 30, 132 * 2^-24 * 30 = 2.36e-4 (the hardware exponential's 2^-22 besides).
Below 2^-14 fp16 has steps of 2^-24: a probability there is off by up to 2^-25 of the row's
largest, the output by 2^-25 B, B = sum |v| (a dim in which the heavy tokens have values near 0).
(One token of weight near 1 whose probability and output round the same way takes the two half steps
in full, so this term has to hold the scores' error alone.)"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from beam_engine_b200 import _lib
from beam_engine_b200._lib import check, lib

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def clean_status():
    check(lib().be_device_status_clear(None))
    yield
    check(lib().be_device_status_clear(None))


def status():
    out = C.c_int32()
    check(lib().be_device_status(C.byref(out), None))
    return out.value


def pow2_scale(amax):
    m, e = np.frexp(np.asarray(amax, np.float64))
    e = np.where(amax == 0, -40, e - np.where(m <= 0.875, 9, 8))
    return np.ldexp(1.0, np.clip(e, -40, 40))


def to_codes(x):
    """float64 -> e4m3 codes (as values): nearest, ties to even, saturating, NaN kept."""
    x = np.asarray(x, np.float64)
    safe = np.where(np.isfinite(x), x, 0.0)
    e = np.maximum(np.frexp(safe)[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    out = np.clip(np.round(safe / step) * step, -448, 448)
    return np.where(np.isnan(x), np.nan, np.where(np.isinf(x), np.sign(x) * 448, out))


class Pool:
    """The definition, sequentially, in 64 bits: codes as values and scales."""

    def __init__(self, pool, scale):
        self.c = pool.float().cpu().numpy().astype(np.float64)
        self.s = scale.cpu().numpy().astype(np.float64)

    def append(self, k, v, pages, slots):
        rows = np.stack([k, v], 1)                      # [n, 2, H, D]
        for p in sorted(set(pages)):
            at = {}
            for i, (pp, ss) in enumerate(zip(pages, slots)):
                if pp == p:
                    at[ss] = i                          # the later row of a slot is kept
            x = rows[list(at.values())]
            amax = np.where(np.isfinite(x), np.abs(x), 0).max((0, 3))
            new = pow2_scale(amax)
            if 0 in at:
                s = new
            else:
                s = np.maximum(new, self.s[p])
                keep = [t for t in range(self.c.shape[2]) if t not in at]
                f = (self.s[p] / s)[:, None, :, None]
                grew = f != 1
                self.c[p][:, keep] = np.where(grew, to_codes(self.c[p][:, keep] * f), self.c[p][:, keep])
            self.s[p] = s
            for t, i in at.items():
                self.c[p][:, t] = to_codes(rows[i] / s[:, :, None])


def rotate(k, pos, inv_freq):
    ang = np.asarray(pos, np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    h = k.shape[-1] // 2
    return np.concatenate([k[..., :h] * c - k[..., h:] * s, k[..., h:] * c + k[..., :h] * s], -1)


def check_pool(pool, scale, ref, exact_planes=(1,)):
    """Codes and scales against the definition; planes not listed may differ by the rotation's
    fp32 roundings next to a border: a neighbouring code, in few places."""
    got = pool.float().cpu().numpy().astype(np.float64)
    np.testing.assert_array_equal(scale.cpu().numpy().astype(np.float64), ref.s)
    for plane in (0, 1):
        g, e = got[:, plane], ref.c[:, plane]
        if plane in exact_planes:
            np.testing.assert_array_equal(g, e)
        else:
            assert (np.isnan(g) == np.isnan(e)).all()
            d = np.abs(np.nan_to_num(g) - np.nan_to_num(e))
            assert (d <= np.maximum(np.abs(np.nan_to_num(e)) * 0.125, 2.0 ** -9) * (1 + 1e-9)).all()
            assert (d > 0).sum() <= 1 + 1e-5 * d.size


def inv_freq_of(d):
    return (1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.int64).float() / d))).cuda()


def make_rows(n, h, d, dt, seed, big=1.0, strided=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, 3 * h * d + 8 * strided), generator=g, device="cuda") * big
    x = x.to(dt)
    return x, x[:, :h * d].view(n, h, d) if not strided else x[:, :h * d].unflatten(1, (h, d)), \
        x[:, h * d:2 * h * d].unflatten(1, (h, d))


def n64(t):
    return t.double().cpu().numpy()


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,d,ps", [(2, 64, 16), (8, 128, 16), (1, 32, 8), (3, 256, 5), (4, 128, 1),
                                    (2, 64, 100), (2, 128, 256)])
@pytest.mark.parametrize("rope", [False, True])
def test_append8_sequence_of_calls(dt, h, d, ps, rope):
    """A sequence grows by calls of many sizes, far positions included; after each the codes and
    scales are the definition's."""
    from beam_engine_b200.page import append_paged_kv_cache
    P, f = 12, inv_freq_of(d)
    pool = torch.randn((P, 2, ps, h, d), device="cuda").to(F8)
    scale = torch.zeros((P, 2, h), device="cuda")
    ref = Pool(pool, scale)
    pages = np.random.default_rng(ps).permutation(P)[:10]
    at = 0
    for step, n in enumerate((1, 2, ps, 1, 3 * ps + 1, 1)):
        n = min(n, 10 * ps - at)
        if n <= 0:
            break
        _, k, v = make_rows(n, h, d, dt, step, big=[1.0, 30.0, 0.01, 1000.0, 1.0, 5.0][step])
        pos = np.arange(at, at + n)
        far = pos * 1009 + 100003
        append_paged_kv_cache(k, v, i32(np.zeros(n)), i32(pos), pool, i32(pages), i32([0, 10]),
                              kv_scale=scale, rope_inv_freq=f if rope else None,
                              rope_positions=i32(far) if rope else None)
        kr = rotate(n64(k), far, f.cpu().numpy()) if rope else n64(k)
        ref.append(kr, n64(v), pages[pos // ps].tolist(), (pos % ps).tolist())
        check_pool(pool, scale, ref, exact_planes=(1,) if rope else (0, 1))
        # differences that a border let through must not build up in the comparison
        ref.c = pool.float().cpu().numpy().astype(np.float64)
        at += n
    assert status() == 0


@pytest.mark.parametrize("n", [40, 700])
def test_append8_any_order_and_repeated_slots(n):
    """Rows in any order, some slots twice: the later row of the call is kept, and pages whose rows
    lie apart in the call get one scale."""
    from beam_engine_b200.page import append_paged_kv_cache
    h, d, ps, P = 2, 64, 16, 64
    rng = np.random.default_rng(n)
    pool = torch.randn((P, 2, ps, h, d), device="cuda").to(F8)
    scale = torch.full((P, 2, h), 2.0 ** -9, device="cuda")
    ref = Pool(pool, scale)
    _, k, v = make_rows(n, h, d, torch.bfloat16, 5, big=3.0)
    batch = rng.integers(0, 3, n)
    pos = rng.integers(0, 20 * ps, n)
    indices = rng.permutation(P)[:60]
    append_paged_kv_cache(k, v, i32(batch), i32(pos), pool, i32(indices), i32([0, 20, 40, 60]),
                          kv_scale=scale)
    pages = indices[batch * 20 + pos // ps]
    ref.append(n64(k), n64(v), pages.tolist(), (pos % ps).tolist())
    check_pool(pool, scale, ref, (0, 1))


@pytest.mark.parametrize("n", [5, 600])
def test_append8_skips_bad_pages_and_flags_them(n):
    from beam_engine_b200.page import append_paged_kv_cache
    h, d, ps, P = 2, 64, 16, 80
    pool, scale = torch.zeros((P, 2, ps, h, d), device="cuda").to(F8), torch.zeros((P, 2, h), device="cuda")
    ref = Pool(pool, scale)
    _, k, v = make_rows(n, h, d, torch.float16, 1)
    pos = np.arange(n)
    indices = np.arange(n // ps + 1) + 3
    indices[0] = P
    if len(indices) > 4:
        indices[4] = -1
    append_paged_kv_cache(k, v, i32(np.zeros(n)), i32(pos), pool, i32(indices), i32([0, len(indices)]),
                          kv_scale=scale)
    pages = indices[pos // ps]
    ok = (pages >= 0) & (pages < P)
    ref.append(n64(k)[ok], n64(v)[ok], pages[ok].tolist(), (pos % ps)[ok].tolist())
    check_pool(pool, scale, ref, (0, 1))
    assert status() == _lib.BE_EDEVICE_RANGE


def test_append8_values_that_are_not_finite_and_the_ends_of_the_range():
    from beam_engine_b200.page import append_paged_kv_cache
    h, d, ps = 2, 64, 16
    pool, scale = torch.zeros((2, 2, ps, h, d), device="cuda").to(F8), torch.zeros((2, 2, h), device="cuda")
    ref = Pool(pool, scale)
    _, k, v = make_rows(4, h, d, torch.float32, 1)
    k[0, 0, 3], k[1, 0, 4], k[2, 0, 5], k[0, 1] = math.inf, -math.inf, math.nan, 0.0
    k[1:, 1] = 0.0
    v[0, 0, 0], v[1, 1, 1] = 3e20, 448.0
    v[:, 1] = v[:, 1].clamp(-448, 448)
    v[2, 0, 5] = 1e-30
    z = i32(np.zeros(4))
    append_paged_kv_cache(k, v, z, i32([0, 1, 2, 3]), pool, i32([1]), i32([0, 1]), kv_scale=scale)
    ref.append(n64(k), n64(v), [1] * 4, [0, 1, 2, 3])
    check_pool(pool, scale, ref, (0, 1))
    assert scale[1, 1, 1].item() == 1.0 and scale[1, 0, 1].item() == 2.0 ** -40
    assert scale[1, 1, 0].item() == 2.0 ** 40


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [3, 700])
def test_append_with_rotation_into_the_rows_type(dt, n):
    from beam_engine_b200.page import append_paged_kv_cache
    h, d, ps, P = 2, 128, 16, 60
    f = inv_freq_of(d)
    pool = torch.randn((P, 2, ps, h, d), device="cuda").to(dt)
    before = pool.clone()
    _, k, v = make_rows(n, h, d, dt, 3)
    pos = np.arange(n) + 5
    pages = np.random.default_rng(1).permutation(P)[:(n + 5) // ps + 1]
    append_paged_kv_cache(k, v, i32(np.zeros(n)), i32(pos), pool, i32(pages), i32([0, len(pages)]),
                          rope_inv_freq=f)
    at = pages[pos // ps], pos % ps
    want = rotate(n64(k), pos, f.cpu().numpy())
    got = n64(pool)
    # one rounding to the type and a few of fp32 on sums of two products
    size = np.abs(n64(k)).max() * 2
    tol = np.abs(want) * torch.finfo(dt).eps / 2 * 1.01 + 8 * 2.0 ** -24 * size
    assert (np.abs(got[at[0], 0, at[1]] - want) <= tol).all()
    np.testing.assert_array_equal(got[at[0], 1, at[1]], n64(v))
    mask = np.ones((P, ps), bool)
    mask[at] = False
    np.testing.assert_array_equal(got.transpose(0, 2, 1, 3, 4)[mask],
                                  n64(before).transpose(0, 2, 1, 3, 4)[mask])


def test_append_and_read_refusals():
    from beam_engine_b200.page import append_paged_kv_cache, read_paged_kv_cache
    pool = torch.zeros((4, 2, 16, 2, 64), device="cuda").to(F8)
    scale = torch.zeros((4, 2, 2), device="cuda")
    _, k, v = make_rows(2, 2, 64, torch.bfloat16, 0)
    idx = (i32([0, 0]), i32([0, 1]))
    tail = (i32([1]), i32([0, 1]))

    def go(kk=k, vv=v, a=idx, p=pool, s=scale, **kw):
        append_paged_kv_cache(kk, vv, *a, p, *tail, kv_scale=s, **kw)
    for kw in (dict(s=None), dict(s=scale.double()), dict(s=scale[:3]), dict(kk=k[:, :1]),
               dict(vv=v.float()), dict(a=(idx[0][:1], idx[1])), dict(rope_inv_freq=inv_freq_of(128)),
               dict(p=pool.float()), dict(p=pool.transpose(0, 2)),
               dict(rope_inv_freq=inv_freq_of(64), rope_positions=i32([1]))):
        with pytest.raises(ValueError):
            go(**kw)
    for args in ((pool, i32([[0]]), scale), (pool, i32([0]), scale, torch.int8),
                 (pool[:, :1], i32([0]), scale)):
        with pytest.raises(ValueError):
            read_paged_kv_cache(*args)
    with pytest.raises(RuntimeError):
        read_paged_kv_cache(pool, torch.zeros(1, dtype=torch.int32), scale)
    go(kk=k[:0], vv=v[:0], a=(idx[0][:0], idx[1][:0]))     # no rows: nothing to do
    assert not scale.any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_read_pages(dt):
    from beam_engine_b200.page import read_paged_kv_cache
    pool = (torch.randn((9, 2, 7, 3, 64), device="cuda") * 50).to(F8)
    scale = torch.ldexp(torch.ones(9, 2, 3), torch.randint(-6, 3, (9, 2, 3))).cuda()
    ids = i32([8, 0, 8, 9, -1, 3])
    got = read_paged_kv_cache(pool, ids, scale, dt)
    want = (pool.float() * scale[:, :, None, :, None])
    for j, p in enumerate(ids.tolist()):
        e = want[p] if 0 <= p < 9 else torch.zeros_like(want[0])
        assert torch.equal(got[j], e.to(dt))
    assert status() == _lib.BE_EDEVICE_RANGE


def test_page_table_in_8_bits_copies_scales_with_tokens():
    """write_block / write_blocks_vectorized / copy_block of an 8-bit PageTable."""
    from beam_engine_b200.page_table import PageTable
    pt = PageTable(2, page_size=16, max_num_pages=8, head_num=2, head_dim=64, store_dtype=F8)
    _, k, v = make_rows(9, 2, 64, torch.bfloat16, 0, strided=False)
    a = pt.allocate_block()
    for layer in (0, 1):
        pt.write_block(layer, a, k * (layer + 1) * 7, v, 0)
    b = pt.copy_block(a, 5)
    for layer in (0, 1):
        got = pt.read_pages(layer, [a, b])
        for plane, x in ((0, k * (layer + 1) * 7), (1, v)):
            x = n64(x)
            tol = np.abs(x) * 2.0 ** -4 + pt.kv_scale[layer, a, plane].double().cpu().numpy()[:, None] * 2.0 ** -10
            assert (np.abs(n64(got[0, plane, :9]) - x) <= tol).all()
            assert torch.equal(got[1, plane, :5], got[0, plane, :5])
    # the copy goes on by itself: a larger value raises its scale, not the source's
    old = pt.read_pages(0, [a])
    pt.write_block(0, b, k[:1] * 1000, v[:1], 5)
    assert torch.equal(pt.read_pages(0, [a]), old)
    assert (pt.kv_scale[0, b, 0] > pt.kv_scale[0, a, 0]).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def reference(q, pool, scale, ptr, pages, kv, qo, causal, window, sinks, sm):
    """(out, lse, A, B) per query in 64 bits; A = sum p |v|, B = sum |v|.  Tokens a query does not see do not
    enter, whatever their cache slots hold."""
    val = pool.double() if scale is None else pool.double() * scale.double()[:, :, None, :, None]
    n, hq, d = q.shape
    hkv = pool.shape[3]
    g = hq // hkv
    out = torch.zeros((n, hq, d), dtype=torch.float64, device="cuda")
    size, whole = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    for r in range(len(kv)):
        m = qo[r + 1] - qo[r]
        if not m:
            continue
        blk = val[torch.tensor(pages[ptr[r]:ptr[r + 1]], device="cuda", dtype=torch.long)]
        blk = blk.transpose(0, 1).reshape(2, -1, hkv, d)[:, :kv[r]]
        for i in range(m):
            p = kv[r] - m + i
            see = [t for t in range(kv[r]) if (not causal or t <= p)
                   and (window < 0 or t >= p - window or t < sinks)]
            if not see:
                continue
            k, v = blk[:, torch.tensor(see, device="cuda")]
            x = torch.einsum("hgd,thd->hgt", q[qo[r] + i].double().view(hkv, g, d), k) * sm
            e = torch.logsumexp(x, -1)
            pr = torch.exp(x - e[..., None])
            out[qo[r] + i] = torch.einsum("hgt,thd->hgd", pr, v).reshape(hq, d)
            size[qo[r] + i] = torch.einsum("hgt,thd->hgd", pr, v.abs()).reshape(hq, d)
            whole[qo[r] + i] = v.abs().sum(0).repeat_interleave(g, 0)
            lse[qo[r] + i] = e.reshape(hq)
    return out, lse, size, whole


def make_pool(P, ps, hkv, d, dt, cache8, seed, spread=4, clean=True):
    """clean False: about one code in 3000 of an 8-bit pool is NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randn((P, 2, ps, hkv, d), generator=g, device="cuda")
    if not cache8:
        return pool.to(dt), None
    scale = torch.ldexp(torch.ones((P, 2, hkv), device="cuda"),
                        torch.randint(-8 - spread, -8 + spread, (P, 2, hkv), generator=g, device="cuda"))
    pool = pool / 2.0 ** -7
    return (pool.clamp(-448, 448) if clean else pool).to(F8), scale


def compare(out, lse, ref, dt, u):
    o, e, a, b = ref
    eps = torch.finfo(dt).eps / 2
    got = out.double()
    bad = torch.isnan(o)
    assert torch.equal(torch.isnan(got), bad)
    tol = eps * o.abs() + (u + 2.4e-4) * a + 2.0 ** -24 + (2.0 ** -25 * b if u == 2.0 ** -11 else 0)
    assert ((got - o).abs()[~bad] <= tol[~bad]).all(), ((got - o).abs() / tol)[~bad].max()
    live = torch.isfinite(e)
    assert torch.equal(torch.isfinite(lse), live) and torch.equal(torch.isnan(lse), torch.isnan(e))
    assert ((lse.double() - e)[live].abs() <= 2e-5).all()


def u_of(dt, cache8, rows=1):
    """Half a step of the type that P is rounded to: narrow tiles (16 rows) of an 8-bit cache use fp16,
    wide ones the query's type."""
    return 2.0 ** -11 if cache8 and rows <= 16 else torch.finfo(dt).eps / 2


def single(dt, cache8, hq, hkv, d, ps, qlen, kv, causal, window, sinks, seed, qmul=1.5, poison=None,
           sm=None, clean=True):
    """One BatchPrefill call against the reference; ``poison(pool, pages, ptr)`` may spoil slots."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    rng = np.random.default_rng(seed)
    np_ = [-(-k // ps) for k in kv]
    P = sum(np_) + 3
    pages = rng.permutation(P)[:sum(np_)].tolist()
    ptr = np.concatenate([[0], np.cumsum(np_)]).tolist()
    qo = np.concatenate([[0], np.cumsum(qlen)]).tolist()
    pool, scale = make_pool(P, ps, hkv, d, dt, cache8, seed, clean=clean)
    n = qo[-1]
    q = (torch.randn((n, (hq + 2) * d), device="cuda",
                     generator=torch.Generator(device="cuda").manual_seed(seed + 1)) * qmul).to(dt)
    q = q[:, :hq * d].unflatten(1, (hq, d))
    if poison:
        poison(pool, pages, ptr)
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan(qo, ptr, pages, [(k - 1) % ps + 1 if k else 0 for k in kv], hq, hkv, d, ps, causal=causal,
           window_left=window, num_sinks=sinks, kv_data_type=F8 if cache8 else dt, sm_scale=sm)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    ref = reference(q, pool, scale, ptr, pages, kv, qo, causal, window, sinks,
                    d ** -0.5 if sm is None else sm)
    compare(out, lse, ref, dt, u_of(dt, cache8, max(qlen) * (hq // hkv)))
    return w, q, pool, scale, out, lse


SHAPES = [([1, 1, 1], [1, 17, 64]), ([1, 0, 1], [0, 5, 33]), ([3, 1, 5], [3, 40, 90]),
          ([17, 9], [17, 130]), ([4], [2]), ([70], [300])]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache8,window,sinks", [(True, -1, 0), (True, 7, 3), (False, 20, 0), (False, 0, 5)])
@pytest.mark.parametrize("hq,hkv,d,ps", [(4, 2, 64, 16), (8, 8, 128, 8), (6, 2, 128, 16), (16, 1, 64, 5)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("clean", [True, False])
def test_paged_attention(dt, cache8, window, sinks, hq, hkv, d, ps, shape, clean):
    qlen, kv = SHAPES[shape]
    single(dt, cache8, hq, hkv, d, ps, qlen, kv, True, window, sinks, shape, clean=clean)
    assert status() == 0


@pytest.mark.parametrize("cache8", [True, False])
@pytest.mark.parametrize("window,sinks", [(100, 4), (2000, 0), (10 ** 9, 0)])
def test_long_contexts_are_split_and_merged(cache8, window, sinks):
    single(torch.bfloat16, cache8, 8, 2, 128, 16, [1, 2], [5003, 2500], True, window, sinks, 3)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache8,window,sinks", [(True, -1, 0), (True, 300, 130), (False, 77, 5),
                                                 (False, 10 ** 6, 0)])
@pytest.mark.parametrize("hq,hkv,d,ps,qlen,kv", [
    (8, 2, 128, 16, [300, 64], [1100, 64]), (4, 4, 64, 8, [257], [700]), (10, 2, 128, 16, [129], [129]),
    (64, 1, 64, 16, [1, 5], [400, 333]), (128, 1, 128, 32, [3], [200]), (34, 2, 128, 16, [1], [3000])])
def test_wide_tiles(dt, cache8, window, sinks, hq, hkv, d, ps, qlen, kv):
    """More than 16 rows per KV head: prompts, chunks after a context, many heads per KV head."""
    single(dt, cache8, hq, hkv, d, ps, qlen, kv, True, window, sinks, 7)
    assert status() == 0


def test_wide_tiles_split_over_tokens():
    """One chunk after a long context: its tiles are cut and merged."""
    w, *_ = single(torch.bfloat16, True, 8, 2, 128, 16, [40], [9000], True, -1, 0, 8)
    assert w._inner._plan.info.n_parts > 40


@pytest.mark.parametrize("qlen", [1, 40])
def test_pages_that_do_not_exist_inside_a_tile(qlen):
    """A bad page id in the middle of a sequence: its tokens drop out, the call is flagged."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(40, 16, 2, 64, torch.bfloat16, True, 1)
    q = torch.randn((qlen, 8, 64), device="cuda").bfloat16()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    pages = list(range(30))
    w.plan([0, qlen], [0, 30], pages[:7] + [-3] + pages[8:20] + [40] + pages[21:], [16], 8, 2, 64, 16,
           causal=False, kv_data_type=F8)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    keep = pages[:7] + pages[8:20] + pages[21:]
    ref = reference(q, pool, scale, [0, 28], keep, [448], [0, qlen], False, -1, 0, 0.125)
    compare(out, lse, ref, torch.bfloat16, 2.0 ** -11 if qlen == 1 else 2.0 ** -8)
    assert status() == _lib.BE_EDEVICE_RANGE


@pytest.mark.parametrize("window,sinks", [(-1, 0), (10, 2)])
def test_without_the_causal_limit(window, sinks):
    single(torch.float16, True, 4, 2, 64, 16, [3, 40], [50, 90], False, window, sinks, 4)


@pytest.mark.parametrize("cache8", [True, False])
@pytest.mark.parametrize("sm", [0.0, 0.02, 3.0])
def test_scale_of_the_scores(cache8, sm):
    """Scores of 0 (a mean), and sharp ones (one token has nearly all the weight)."""
    single(torch.float16, cache8, 4, 2, 64, 16, [2, 1], [200, 70], True, 64, 2, 5, qmul=0.2, sm=sm)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache8", [True, False])
def test_slots_that_no_query_sees_may_hold_anything(dt, cache8):
    """NaN behind the last token, in pages of no request and in tokens between sinks and window."""
    ps, kv, window, sinks = 16, [37, 90, 16], 20, 3

    def poison(pool, pages, ptr):
        raw = pool.view(torch.uint8 if cache8 else torch.int16)
        bad = 0x7f if cache8 else 0x7fff
        raw[sorted(set(range(pool.shape[0])) - set(pages))] = bad
        for r, k in enumerate(kv):
            for t in range(((k - 1) // ps + 1) * ps):
                if t >= k or (sinks <= t < k - 1 - window):
                    raw[pages[ptr[r] + t // ps], :, t % ps] = bad
    single(dt, cache8, 8, 2, 128, ps, [1, 1, 1], kv, True, window, sinks, 6, poison=poison)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache8", [True, False])
@pytest.mark.parametrize("qlen,kv", [(7, 30), (40, 50), (150, 150)])
def test_a_value_that_is_not_finite_reaches_only_the_queries_that_see_it(dt, cache8, qlen, kv):
    """A NaN key and value (and an infinity in 16 bits) late in a prompt: earlier queries of the
    same tile stay as they were; windows let later ones forget it."""
    ps = 16

    def poison(pool, pages, ptr):
        raw = pool.view(torch.uint8 if cache8 else torch.int16)
        t = kv - qlen + qlen // 2
        raw[pages[t // ps], 1, t % ps, :, 5] = 0x7f if cache8 else 0x7fff
        t = kv - 2
        raw[pages[t // ps], 0, t % ps, 0, 1] = 0x7f if cache8 else 0x7fff
        if not cache8:
            t = kv - qlen + qlen // 3
            pool[pages[t // ps], 1, t % ps, 1, 9] = math.inf

    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    for window in (-1, qlen // 4) if cache8 else (10 ** 6, qlen // 4):
        rng = np.random.default_rng(9)
        n_p = -(-kv // ps)
        pages = rng.permutation(n_p + 2)[:n_p].tolist()
        pool, scale = make_pool(n_p + 2, ps, 2, 64, dt, cache8, 1)
        poison(pool, pages, [0])
        q = torch.randn((qlen, 8, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dt)
        w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
        w.plan([0, qlen], [0, n_p], pages, [(kv - 1) % ps + 1], 8, 2, 64, ps, causal=True,
               window_left=window, num_sinks=2, kv_data_type=F8 if cache8 else dt)
        out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
        o, e, a, _ = reference(q, pool, scale, [0, n_p], pages, [kv], [0, qlen], True, window, 2, 0.125)
        fin = torch.isfinite(o)
        assert torch.equal(torch.isnan(out), torch.isnan(o))
        assert torch.equal(out.double()[~fin & ~torch.isnan(o)], o[~fin & ~torch.isnan(o)])
        a = torch.where(torch.isfinite(a), a, torch.zeros_like(a))
        tol = torch.finfo(dt).eps / 2 * o.abs() + (u_of(dt, cache8, qlen * 4) + 2.4e-4) * a + 2.0 ** -24
        assert ((out.double() - o).abs()[fin] <= tol[fin]).all()
        assert torch.equal(torch.isnan(lse), torch.isnan(e))


def test_scales_far_apart():
    """Blocks whose scales differ by 2^60 in either plane: no overflow, nothing lost."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    ps, hkv, d, kv = 16, 2, 64, 64
    pool, scale = make_pool(4, ps, hkv, d, torch.bfloat16, True, 1)
    for k_exp, v_exp in (([-30, 0, -8, 5], [30, -30, 0, -8]), ([-8] * 4, [-40, -40, -40, 20])):
        scale[:, 0] = torch.tensor([2.0 ** e for e in k_exp], device="cuda")[:, None]
        scale[:, 1] = torch.tensor([2.0 ** e for e in v_exp], device="cuda")[:, None]
        q = torch.randn((1, 4, d), device="cuda").bfloat16() * 1e-3
        w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
        w.plan([0, 1], [0, 4], [2, 0, 1, 3], [16], 4, hkv, d, ps, causal=True, kv_data_type=F8)
        out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
        ref = reference(q, pool, scale, [0, 4], [2, 0, 1, 3], [kv], [0, 1], True, -1, 0, 0.125)
        compare(out, lse, ref, torch.bfloat16, 2.0 ** -11)


def test_bad_pages_are_skipped_and_flagged():
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(5, 16, 2, 64, torch.bfloat16, True, 1)
    q = torch.randn((1, 4, 64), device="cuda").bfloat16()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, 1], [0, 3], [1, 5, 3], [16], 4, 2, 64, 16, causal=True, kv_data_type=F8)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    ref = reference(q, pool, scale, [0, 2], [1, 3], [32], [0, 1], True, -1, 0, 0.125)
    compare(out, lse, ref, torch.bfloat16, 2.0 ** -11)
    assert status() == _lib.BE_EDEVICE_RANGE


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache8,window,sinks", [(True, -1, 0), (True, 30, 2), (False, 30, 40)])
@pytest.mark.parametrize("beams,g", [(3, 4), (16, 4), (40, 1)])
def test_cascade_levels(dt, cache8, window, sinks, beams, g):
    """Beams with a shared prefix in two levels give what each alone gives over all its pages."""
    from beam_engine_b200.cascade import MultiLevelCascadeAttentionWrapper
    ps, hkv, d, prompts = 16, 2, 128, 2
    hq, n = g * hkv, beams * prompts
    rng = np.random.default_rng(beams)
    pre = [5, 2]
    own = rng.integers(1, 40, n)
    own_p = [-(-int(k) // ps) for k in own]
    P = sum(pre) + sum(own_p)
    ids = rng.permutation(P).tolist()
    pool, scale = make_pool(P, ps, hkv, d, dt, cache8, beams)
    heads = [ids[:5], ids[5:7]]
    tails, at = [], 7
    for k in own_p:
        tails.append(ids[at:at + k])
        at += k
    q = torch.randn((n, hq, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(dt)
    w = MultiLevelCascadeAttentionWrapper(2, torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([[0, beams, n], list(range(n + 1))], [[0, 5, 7], np.concatenate([[0], np.cumsum(own_p)])],
           [heads[0] + heads[1], [p for t in tails for p in t]],
           [[ps, ps], [(int(k) - 1) % ps + 1 for k in own]], hq, hkv, d, ps, causal=True,
           window_left=window, num_sinks=sinks, kv_data_type=F8 if cache8 else dt)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    lists = [heads[i // beams] + tails[i] for i in range(n)]
    kv = [pre[i // beams] * ps + int(own[i]) for i in range(n)]
    ref = reference(q, pool, scale, np.concatenate([[0], np.cumsum([len(x) for x in lists])]).tolist(),
                    [p for x in lists for p in x], kv, list(range(n + 1)), True, window, sinks, d ** -0.5)
    compare(out, lse, ref, dt, u_of(dt, cache8, beams * g))


def test_a_cache_in_8_bits_is_planned_again_when_the_plan_did_not_know():
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(4, 16, 2, 128, torch.bfloat16, True, 1)
    q = torch.randn((1, 8, 128), device="cuda").bfloat16()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, 1], [0, 3], [1, 0, 3], [9], 8, 2, 128, 16, causal=True)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    ref = reference(q, pool, scale, [0, 3], [1, 0, 3], [41], [0, 1], True, -1, 0, 128 ** -0.5)
    compare(out, lse, ref, torch.bfloat16, 2.0 ** -11)


def test_attention_refusals():
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(4, 16, 2, 128, torch.bfloat16, True, 1)
    q = torch.randn((1, 8, 128), device="cuda").bfloat16()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    w = BatchPrefillWithPagedKVCacheWrapper(ws)
    base = ([0, 1], [0, 3], [1, 0, 3], [9], 8, 2)
    with pytest.raises(ValueError):
        w.plan(*base, 96, 16, causal=True, window_left=4)
    with pytest.raises(ValueError):
        w.plan(*base, 128, 16, causal=True, window_left=4, num_sinks=-1)
    with pytest.raises(ValueError):
        w.plan([0, 1], [0, 3], [1, 0, 3], [17], 8, 2, 128, 16, causal=True, window_left=4)
    with pytest.raises(ValueError, match="workspace"):
        BatchPrefillWithPagedKVCacheWrapper(ws[:100]).plan(*base, 128, 16, causal=True, window_left=4)
    w.plan(*base, 128, 16, causal=True, window_left=4)
    half = torch.zeros((4, 2, 16, 2, 128), dtype=torch.bfloat16, device="cuda")
    for args, kw in (((q, pool), {}), ((q, pool), dict(kv_scale=scale[:2])), ((q.half(), half), {}),
                     ((q.float(), half.float()), {}), ((q, half), dict(kv_scale=scale)),
                     ((q[:, :4], half), {}), ((q, half[:, :, :8]), {}),
                     ((q, half), dict(out=torch.empty_like(q).float())), ((q[:0], half), {})):
        with pytest.raises(ValueError):
            w.run(*args, **kw)
    w.plan(*base, 128, 16, causal=True)
    with pytest.raises(ValueError):
        w.run(q, half, kv_scale=scale)


@pytest.mark.parametrize("cache8", [True, False])
def test_captured_and_replayed_on_another_stream(cache8):
    """One recorded launch on a side stream, replayed with other queries, another cache and another
    plan of the same size; the eager call beside it is not disturbed."""
    dt = torch.bfloat16
    w, q, pool, scale, out, lse = single(dt, cache8, 8, 2, 128, 16, [1, 1, 2], [700, 90, 1800], True,
                                         400, 4, 11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    res = torch.empty_like(out)
    with torch.cuda.stream(side):
        w.run(q, pool, out=res, kv_scale=scale)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            w.run(q, pool, out=res, kv_scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    q2 = torch.randn_like(q)
    for new in (q2, q.clone()):
        q.copy_(new)
        res.zero_()
        g.replay()
        assert torch.equal(res, w.run(q, pool, kv_scale=scale))
    assert torch.equal(res, out)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_append_then_attend_as_a_decode_loop_does(dt):
    """Prompt, then single tokens: append (with the rotation) and attend, under a window with
    sinks, against 64-bit attention over the cache's values as read back."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    from beam_engine_b200.page import append_paged_kv_cache, read_paged_kv_cache
    hq, hkv, d, ps, P = 8, 2, 128, 16, 12
    pool, scale = torch.zeros((P, 2, ps, hkv, d), device="cuda").to(F8), torch.zeros((P, 2, hkv), device="cuda")
    f, at = inv_freq_of(d), 0
    pages = np.random.default_rng(0).permutation(P).tolist()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    for step, n in enumerate([90, 1, 1, 7, 1]):
        _, k, v = make_rows(n, hkv, d, dt, step, big=1 + step)
        q = torch.randn((n, hq, d), device="cuda").to(dt)
        used = -(-(at + n) // ps)
        append_paged_kv_cache(k, v, i32(np.zeros(n)), i32(np.arange(at, at + n)), pool, i32(pages[:used]),
                              i32([0, used]), kv_scale=scale, rope_inv_freq=f)
        at += n
        w.plan([0, n], [0, used], pages[:used], [(at - 1) % ps + 1], hq, hkv, d, ps, causal=True,
               window_left=40, num_sinks=4, kv_data_type=F8)
        out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
        values = read_paged_kv_cache(pool, i32(np.arange(P)), scale, torch.float32)
        ref = reference(q, values, None, [0, used], pages[:used], [at], [0, n], True, 40, 4, d ** -0.5)
        compare(out, lse, ref, dt, u_of(dt, True, n * 4))


def test_windows_beyond_int32_see_everything():
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    outs = []
    pool, _ = make_pool(8, 16, 2, 64, torch.bfloat16, False, 1)
    q = torch.randn((6, 4, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    for window, sinks in ((10 ** 6, 0), (2 ** 32 + 5, 0), (0, 2 ** 32 + 1)):
        w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
        w.plan([0, 6], [0, 6], [5, 1, 2, 7, 0, 3], [9], 4, 2, 64, 16, causal=True, window_left=window,
               num_sinks=sinks)
        outs.append(w.run(q, pool))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_capture_needs_a_plan_for_the_cache():
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(4, 16, 2, 64, torch.bfloat16, True, 1)
    q = torch.zeros((2, 4, 64), device="cuda", dtype=torch.bfloat16)
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, 2], [0, 2], [1, 2], [9], 4, 2, 64, 16, causal=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="kv_data_type"):
            w.run(q, pool, kv_scale=scale)


def test_two_graphs_with_workspaces_of_their_own_replayed_together():
    """Two captured calls on two streams, replayed at once, give what each gives alone."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    calls = []
    for seed, (qo, kv) in enumerate((([0, 1, 2], [3000, 2000]), ([0, 40, 41], [700, 2500]))):
        ptr = np.concatenate([[0], np.cumsum([-(-k // 16) for k in kv])]).tolist()
        pool, scale = make_pool(ptr[-1], 16, 2, 128, torch.bfloat16, True, seed)
        pages = np.random.default_rng(seed).permutation(ptr[-1]).tolist()
        q = torch.randn((qo[-1], 8, 128), device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()
        w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
        w.plan(qo, ptr, pages, [(k - 1) % 16 + 1 for k in kv], 8, 2, 128, 16, causal=True, kv_data_type=F8)
        want = w.run(q, pool, kv_scale=scale)
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            w.run(q, pool, kv_scale=scale, out=out)
        calls.append((g, out, want, torch.cuda.Stream(), (w, q, pool, scale)))
    for _ in range(5):
        for g, out, _, st, _ in calls:
            with torch.cuda.stream(st):
                out.zero_()
                for _ in range(3):
                    g.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in calls:
        assert torch.equal(out, want)
    assert status() == 0
