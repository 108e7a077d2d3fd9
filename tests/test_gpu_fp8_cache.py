"""The 8-bit cache's writers and its read-back against the 64-bit oracle (oracle/fp8_ref.py).

Codes and scale bytes are compared bit for bit over the whole pool, whose other slots hold a pattern that has to
stay.  A key that the norm and the rotation made in fp32 may round to e4m3 the other way where its 64-bit value lies
next to a tie, so those are held to half a step plus the fp32 error.
"""
import numpy as np
import pytest
import torch

from ecahlang_amd import ops
from oracle import fp8_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}  # half the smallest subnormal


def table(kv, new, ps, pool_extra=3, seed=0):
    """Page table of sequences of kv tokens, and where their last `new` tokens go."""
    rng = np.random.default_rng(seed)
    npages = [-(-n // ps) for n in kv]
    pool = sum(npages) + pool_extra
    indices = rng.permutation(pool)[: sum(npages)].astype(np.int32)
    indptr = np.concatenate([[0], np.cumsum(npages)]).astype(np.int32)
    b = np.repeat(np.arange(len(kv)), new).astype(np.int32)
    pos = np.concatenate([np.arange(n - c, n) for n, c in zip(kv, new)] or [[]]).astype(np.int32)
    last = np.array([(n - 1) % ps + 1 if n else 0 for n in kv], dtype=np.int32)
    page = indices[indptr[b] + pos // ps] if len(pos) else pos
    return dict(indptr=indptr, indices=indices, last=last, b=b, pos=pos, page=page, slot=pos % ps, pool=pool)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def pool8(pool, ps, hkv, d, seed=1):
    """A pool of patterns (NaN codes among them) and its scale bytes, on the host."""
    rng = np.random.default_rng(seed)
    return rng.integers(0, 256, (pool, 2, ps, hkv, d), dtype=np.uint8), rng.integers(0, 256, (pool, 2, hkv, ps), dtype=np.uint8)


def on_dev(codes, scales):
    return dev(codes).view(F8), dev(scales).view(E8)


def f64(t):
    return t.detach().cpu().double().numpy()


def expected(codes, scales, t, k, v):
    codes, scales = codes.copy(), scales.copy()
    for j, x in enumerate((k, v)):
        c, s = fp8_ref.quantise(f64(x))
        codes[t["page"], j, t["slot"]] = c
        scales[t["page"], j, :, t["slot"]] = s
    return codes, scales


def same(cache, scales, codes, bytes_):
    np.testing.assert_array_equal(scales.view(torch.uint8).cpu().numpy(), bytes_)
    got, nan = cache.view(torch.uint8).cpu().numpy(), np.isnan(fp8_ref.E4M3)
    ok = (got == codes) | (nan[got] & nan[codes])  # (the sign of a NaN is not kept)
    assert ok.all(), f"{(~ok).sum()} codes differ"


def rows(n, hkv, d, dtype, seed, scale=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, hkv, d), generator=g)
    if scale is None:
        x = x * torch.exp2(torch.randint(-12, 8, (n, hkv, 1), generator=g).float())
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,ps", [(2, 128, 16), (8, 64, 16), (1, 16, 1), (3, 80, 5), (4, 256, 64), (2, 512, 16), (16, 48, 8)])
def test_append_is_bit_exact(dtype, hkv, d, ps):
    t = table([1, 17, 64, 33], [1, 5, 64, 2], ps, seed=d)
    n = len(t["pos"])
    codes, scales = pool8(t["pool"], ps, hkv, d)
    k, v = rows(n, hkv, d, dtype, 5), rows(n, hkv, d, dtype, 6)
    cache, sc = on_dev(codes, scales)
    ops.append_paged_kv_cache(k, v, dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]), kv_scales=sc)
    same(cache, sc, *expected(codes, scales, t, k, v))
    # by slots: the same bytes
    cache2, sc2 = on_dev(codes, scales)
    ops.append_paged_kv_cache_slots(k, v, dev((t["page"] * ps + t["slot"]).astype(np.int32)), cache2, kv_scales=sc2)
    assert torch.equal(cache2.view(torch.uint8), cache.view(torch.uint8)) and torch.equal(sc2.view(torch.uint8), sc.view(torch.uint8))


def test_every_16_bit_value_rounds_to_the_nearest_code():
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
        x = x[x.isfinite() & (x.abs() <= 448)]
        x = torch.cat([x, x.new_zeros(-len(x) % 127)]).view(-1, 1, 127)
        k = torch.cat([torch.full_like(x[..., :1], 448.0), x], dim=-1).to(DEV)
        n = len(k)
        t = table([n], [n], 16)
        codes, scales = pool8(t["pool"], 16, 1, 128)
        cache, sc = on_dev(codes, scales)
        ops.append_paged_kv_cache(k, k.flip(0), dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]), kv_scales=sc)
        same(cache, sc, *expected(codes, scales, t, k, k.flip(0)))


def test_rows_of_unusual_values():
    f = torch.finfo(torch.float32)
    d = 32
    special = [[0.0] * d, [-0.0] * d, [f.tiny] * d, [2.0 ** -149] + [0.0] * (d - 1), [f.max] * d, [f.max, f.tiny] * (d // 2),
               [float("inf")] + [1.0] * (d - 1), [float("nan")] * d, [float("nan"), -3.0] * (d // 2), [448.0] * d,
               [float(np.nextafter(np.float32(448), np.float32(500)))] * d, [2.0 ** -126] * d, [2.0 ** -118 * 1.75] * d,
               [1e-3, 1e3] * (d // 2), [17.0, 28.0] * (d // 2), [2.0 ** -9, 448.0] * (d // 2), [2.0 ** -10, 448.0] * (d // 2),
               [3 * 2.0 ** -11, 448.0] * (d // 2), [float("-inf")] * d]
    k = torch.tensor(special, dtype=torch.float32, device=DEV)[:, None]
    n = len(special)
    t = table([n], [n], 4)
    codes, scales = pool8(t["pool"], 4, 1, d)
    cache, sc = on_dev(codes, scales)
    ops.append_paged_kv_cache(k, k * 2, dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]), kv_scales=sc)
    same(cache, sc, *expected(codes, scales, t, k, k * 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_takes_strided_and_unaligned_rows_and_split_caches(dtype):
    hkv, d, ps = 2, 64, 16
    t = table([40, 9], [33, 9], ps)
    n = len(t["pos"])
    big = rows(n, 3 * hkv, d + 1, dtype, 9)
    k, v = big[:, :hkv, 1:], big[:, 2 * hkv:, :d]                  # rows at odd addresses
    kt = rows(hkv, n, d, dtype, 10).transpose(0, 1)                # heads outermost
    codes, scales = pool8(t["pool"], ps, hkv, d)
    args = (dev(t["b"]), dev(t["pos"]))
    tab = (dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    for a, b in ((k, v), (kt, v), (kt, kt)):
        cache, sc = on_dev(codes, scales)
        ops.append_paged_kv_cache(a, b, *args, cache, *tab, kv_scales=sc)
        same(cache, sc, *expected(codes, scales, t, a, b))
        pair = (cache[:, 0].contiguous(), cache[:, 1].contiguous())
        spair = (sc[:, 0].contiguous(), sc[:, 1].contiguous())
        ops.append_paged_kv_cache(b, a, *args, pair, *tab, kv_scales=spair)
        c2, s2 = expected(codes, scales, t, b, a)
        same(torch.stack([p.view(torch.uint8) for p in pair], 1).view(F8), torch.stack([p.view(torch.uint8) for p in spair], 1).view(E8), c2, s2)


def test_bad_metadata_is_skipped_and_counted():
    hkv, d, ps = 2, 64, 16
    t = table([20, 20], [20, 20], ps)
    n = len(t["pos"])
    b, pos, idx = t["b"].copy(), t["pos"].copy(), t["indices"].copy()
    bad = np.zeros(n, bool)
    for i, (bb, pp) in {0: (2, 0), 1: (-1, 0), 2: (0, 32), 3: (0, -1), 4: (1, 2 ** 31 - 1)}.items():
        b[i], pos[i], bad[i] = bb, pp, True
    idx[3] = t["pool"]                       # sequence 1's second page: outside the pool
    bad |= (t["b"] == 1) & (t["pos"] >= 16)
    k, v = rows(n, hkv, d, torch.float16, 1), rows(n, hkv, d, torch.float16, 2)
    codes, scales = pool8(t["pool"], ps, hkv, d)
    good = {x: t[x][~bad] for x in ("page", "slot")}
    keep = torch.from_numpy(~bad).to(DEV)
    want = expected(codes, scales, good, k[keep], v[keep])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache, sc = on_dev(codes, scales)
    ops.append_paged_kv_cache(k, v, dev(b), dev(pos), cache, dev(idx), dev(t["indptr"]), dev(t["last"]), err_count=err, kv_scales=sc)
    same(cache, sc, *want)
    assert err.item() == bad.sum() * 2 * hkv
    slots = (t["page"] * ps + t["slot"]).astype(np.int32)
    slots[bad] = -1
    slots[np.flatnonzero(bad)[:2]] = t["pool"] * ps
    err.zero_()
    cache, sc = on_dev(codes, scales)
    ops.append_paged_kv_cache_slots(k, v, dev(slots), cache, err_count=err, kv_scales=sc)
    same(cache, sc, *want)
    assert err.item() == bad.sum() * 2 * hkv
    # the norm and rotation: counted once a token, and its queries are written
    q = rows(n, 4, d, torch.float16, 3)
    one, zero = torch.ones((n, d), dtype=torch.float16, device=DEV), torch.zeros((n, d), dtype=torch.float16, device=DEV)
    err.zero_()
    cache, sc = on_dev(codes, scales)
    out = ops.append_paged_kv_cache_with_norm_rope(q, k, v, None, None, one, zero, dev(b), dev(pos), cache, dev(idx), dev(t["indptr"]),
                                                   dev(t["last"]), err_count=err, kv_scales=sc)
    same(cache, sc, *want)                   # (turned by nothing: as it was)
    assert err.item() == bad.sum() and torch.equal(out, q)


def _norm_case(dtype, hq, hkv, d, ps, seed, wdt=None, cdt=None, kv=(40, 1, 129, 16), new=(33, 1, 17, 16)):
    t = table(list(kv), list(new), ps, seed=seed)
    n = len(t["pos"])
    g = torch.Generator().manual_seed(seed)
    ang = torch.from_numpy(t["pos"]).double()[:, None] / (10000.0 ** (torch.arange(0, d, 2).double() / d))[None]
    ang = torch.cat([ang, ang], 1)
    cos, sin = (f(ang).to(cdt or dtype).to(DEV) for f in (torch.cos, torch.sin))
    w = (1 + 0.3 * torch.randn((2, d), generator=g)).to(wdt or dtype).to(DEV)
    return t, rows(n, hq, d, dtype, seed + 1), rows(n, hkv, d, dtype, seed + 2), rows(n, hkv, d, dtype, seed + 3), w[0], w[1], cos, sin


def _fp32_error(x, w, cos, sin, eps, d):
    """What fp32 arithmetic may be off: the norm's factor by (d / 2 + 8) half steps of 2^-24 (a sum of d squares, all
    positive, in any order: at most d half steps, half that after the root; then eps, the root, the division), each
    product by two more, the rotation's sum by two."""
    z = np.abs(x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w) if w is not None else np.abs(x)
    h = d // 2
    y = z * np.abs(cos)[:, None] + np.concatenate([z[..., h:], z[..., :h]], -1) * np.abs(sin)[:, None]
    return y * (d / 2 + 16) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,ps", [(16, 2, 128, 16), (32, 8, 64, 16), (8, 4, 256, 8), (5, 5, 80, 3), (3, 1, 512, 16), (1, 1, 16, 16)])
@pytest.mark.parametrize("cache8", [True, False])
def test_norm_rope_append(dtype, hq, hkv, d, ps, cache8):
    eps = 1e-5
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, d + hq)
    c, s = f64(cos), f64(sin)
    want_q, want_k = fp8_ref.norm_rotate(f64(q), f64(qw), c, s, eps), fp8_ref.norm_rotate(f64(k), f64(kw), c, s, eps)
    err_q, err_k = _fp32_error(f64(q), f64(qw), c, s, eps, d), _fp32_error(f64(k), f64(kw), c, s, eps, d)
    args = (qw, kw, cos, sin, dev(t["b"]), dev(t["pos"]))
    tab = (dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    if cache8:
        codes, scales = pool8(t["pool"], ps, hkv, d)
        cache, sc = on_dev(codes, scales)
    else:
        cache, sc = torch.full((t["pool"], 2, ps, hkv, d), float("nan"), dtype=dtype, device=DEV), None
    out = ops.append_paged_kv_cache_with_norm_rope(q, k, v, *args, cache, *tab, eps=eps, kv_scales=sc)
    assert (np.abs(f64(out) - want_q) <= HALF[dtype] * (np.abs(want_q) + err_q) + TINY[dtype] + err_q).all()
    page, slot = t["page"], t["slot"]
    if not cache8:
        got = f64(cache)[page, 0, slot]
        assert (np.abs(got - want_k) <= HALF[dtype] * (np.abs(want_k) + err_k) + TINY[dtype] + err_k).all()
        assert torch.equal(cache[torch.from_numpy(page).long(), 1, torch.from_numpy(slot).long()], v)
        mine = torch.zeros(cache.shape[:3], dtype=torch.bool, device=DEV)
        mine[torch.from_numpy(page).long(), :, torch.from_numpy(slot).long()] = True
        assert cache[~mine].isnan().all()
        return
    want_c, want_s = expected(codes, scales, t, torch.from_numpy(want_k), v)
    gc, gs = cache.view(torch.uint8).cpu().numpy(), sc.view(torch.uint8).cpu().numpy()
    # values, and everything that is not a new key: bit for bit
    at = np.zeros(gc.shape[:3], bool)
    at[page, 0, slot] = True
    nan = np.isnan(fp8_ref.E4M3)
    assert ((gc == want_c) | (nan[gc] & nan[want_c]))[~at].all()
    assert (gs == want_s)[~np.swapaxes(np.broadcast_to(at[..., None], at.shape + (hkv,)), 2, 3)].all()
    # keys: the scale is that of the 64-bit row or, next to a border, of one half as large or twice; half a step then
    got_s = 2.0 ** (gs[page, 0, :, slot].astype(float) - 127)
    amax, off = np.abs(want_k).max(-1), err_k.max(-1)
    assert (amax - off <= 448 * got_s).all() and ((amax + off >= 224 * got_s) | (got_s == 2.0 ** -126)).all()
    got = fp8_ref.E4M3[gc[page, 0, slot]] * got_s[..., None]
    assert (np.abs(got - want_k) <= np.maximum(2.0 ** -4 * np.abs(want_k), 2.0 ** -10 * got_s[..., None]) + 1.1 * err_k).all()


@pytest.mark.parametrize("wdt,cdt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_norm_rope_takes_fp32_weights_and_angles_in_place_and_strided(wdt, cdt):
    dtype, hq, hkv, d, ps = torch.bfloat16, 6, 2, 128, 16
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, 77, wdt, cdt)
    n = len(t["pos"])
    wide = torch.empty((n, hq + 2 * hkv, d), dtype=dtype, device=DEV)      # one projection's output
    wide[:, :hq], wide[:, hq:hq + hkv], wide[:, hq + hkv:] = q, k, v
    c, s = f64(cos), f64(sin)
    want = fp8_ref.norm_rotate(f64(q), f64(qw), c, s, 1e-6)
    err = _fp32_error(f64(q), f64(qw), c, s, 1e-6, d)
    cache = torch.zeros((t["pool"], 2, ps, hkv, d), dtype=dtype, device=DEV)
    args = (dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    qv = wide[:, :hq]
    out = ops.append_paged_kv_cache_with_norm_rope(qv, wide[:, hq:hq + hkv], wide[:, hq + hkv:], qw, kw, cos, sin, *args, q_out=qv)
    assert out.data_ptr() == wide.data_ptr()
    assert (np.abs(f64(out) - want) <= HALF[dtype] * (np.abs(want) + err) + err).all()
    assert torch.equal(wide[:, hq:hq + hkv], k) and torch.equal(wide[:, hq + hkv:], v)
    # rows at odd addresses, weights and angles too: the same values
    odd = torch.empty((n, hq, d + 1), dtype=dtype, device=DEV)[..., 1:].copy_(q)
    shift = lambda x: torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)  # noqa: E731
    out2 = ops.append_paged_kv_cache_with_norm_rope(odd, k, v, shift(qw), shift(kw), shift(cos), shift(sin), *args)
    assert torch.equal(out2, out)


def test_norm_rope_without_weights_rotates_only():
    dtype, hq, hkv, d, ps = torch.float32, 4, 2, 64, 16
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, 3)
    c, s = f64(cos), f64(sin)
    cache = torch.zeros((t["pool"], 2, ps, hkv, d), dtype=dtype, device=DEV)
    args = (cos, sin, dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    for wq, wk in ((None, kw), (qw, None), (None, None)):
        out = ops.append_paged_kv_cache_with_norm_rope(q, k, v, wq, wk, *args)
        for got, x, w in ((f64(out), q, wq), (f64(cache)[t["page"], 0, t["slot"]], k, wk)):
            w = f64(w) if w is not None else None
            want = fp8_ref.norm_rotate(f64(x), w, c, s, 1e-6)
            assert (np.abs(got - want) <= 1.01 * _fp32_error(f64(x), w, c, s, 1e-6, d) + HALF[dtype] * np.abs(want)).all()


def test_a_row_of_zeros_and_one_of_what_is_not_finite():
    d, hkv, ps = 64, 1, 16
    t = table([3], [3], ps)
    k = torch.randn((3, 1, d), device=DEV, dtype=torch.float32)
    k[0], k[1, 0, 5] = 0.0, float("nan")
    one, zero = torch.ones((3, d), device=DEV), torch.zeros((3, d), device=DEV)
    codes, scales = pool8(t["pool"], ps, hkv, d)
    cache, sc = on_dev(codes, scales)
    out = ops.append_paged_kv_cache_with_norm_rope(k.clone(), k, k, one[0], one[0], one, zero, dev(t["b"]), dev(t["pos"]), cache,
                                                   dev(t["indices"]), dev(t["indptr"]), dev(t["last"]), eps=1e-6, kv_scales=sc)
    assert (out[0] == 0).all() and out[1].isnan().all() and out[2].isfinite().all()
    got = fp8_ref.E4M3[cache.view(torch.uint8).cpu().numpy()[t["page"], 0, t["slot"]]]
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isfinite(got[2]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,ps", [(2, 128, 16), (8, 64, 16), (1, 16, 1), (3, 80, 5), (4, 256, 64), (1, 512, 16)])
def test_read_back_holds_the_values(dtype, hkv, d, ps):
    t = table([1, 17, 64, 33], [0] * 4, ps, seed=d)
    rng = np.random.default_rng(2)
    codes, scales = pool8(t["pool"], ps, hkv, d)
    scales = rng.integers(100, 131, scales.shape, dtype=np.uint8) if dtype != torch.float32 else np.maximum(np.minimum(scales, 246), 10)
    cache, sc = on_dev(codes, scales)
    idx = np.concatenate([t["indices"], [0, 0]]).astype(np.int32)  # a list longer than its sequences need
    idx[1], idx[2] = t["pool"], -1
    n = len(t["indices"])
    out = torch.full((n + 2, 2, ps, hkv, d), 7.0, dtype=dtype, device=DEV)
    got = ops.read_paged_kv_cache(cache, sc, dev(idx), dev(t["indptr"]), dtype, out=out)
    assert got is out and (out[n:] == 7).all() and (out[1:3] == 0).all()
    want = fp8_ref.values(codes, scales)[np.clip(idx, 0, t["pool"] - 1)][:n]
    want[1:3] = 0
    want = torch.from_numpy(want).to(dtype).to(DEV)  # (bf16, fp32: exact; fp16: nearest)
    assert torch.equal(torch.nan_to_num(out[:n], nan=3.0), torch.nan_to_num(want, nan=3.0))
    pair = (cache[:, 0].contiguous(), cache[:, 1].contiguous()), (sc[:, 0].contiguous(), sc[:, 1].contiguous())
    assert torch.equal(torch.nan_to_num(ops.read_paged_kv_cache(*pair, dev(t["indices"]), dev(t["indptr"]), dtype)[3:], nan=3.0),
                       torch.nan_to_num(want[3:], nan=3.0))


def test_read_back_of_the_extreme_scales():
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 1, 1, 1, 256), (1, 2, 3, 1, 1))
    scales = np.array([0, 1, 254, 247, 120, 255], dtype=np.uint8).reshape(1, 2, 1, 3)
    cache, sc = on_dev(codes, scales)
    got = ops.read_paged_kv_cache(cache, sc, dev(np.zeros(1, np.int32)), dev(np.array([0, 1], np.int32)), torch.float32)
    with np.errstate(over="ignore"):
        want = fp8_ref.values(codes, scales).astype(np.float32)
    want[0, 1, 2] = np.nan  # (255 is E8M0's NaN)
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_nothing_to_do():
    cache, sc = on_dev(*pool8(4, 16, 2, 64))
    before = cache.view(torch.uint8).clone()
    none = torch.empty((0, 2, 64), dtype=torch.float16, device=DEV)
    i0, p1 = torch.empty(0, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.append_paged_kv_cache(none, none, i0, i0, cache, i0, p1, p1[:1], kv_scales=sc)
    ops.append_paged_kv_cache_slots(none, none, i0, cache, kv_scales=sc)
    cs = torch.empty((0, 64), dtype=torch.float16, device=DEV)
    assert ops.append_paged_kv_cache_with_norm_rope(none, none, none, None, None, cs, cs, i0, i0, cache, i0, p1, p1[:1], kv_scales=sc).shape == none.shape
    assert ops.read_paged_kv_cache(cache, sc, i0, p1, torch.float16).shape == (0, 2, 16, 2, 64)
    torch.cuda.synchronize()
    assert torch.equal(before, cache.view(torch.uint8))


def test_new_scales_are_ones():
    cache = torch.zeros((3, 5, 2, 16, 4, 64), dtype=F8, device=DEV)
    sc = ops.new_kv_scales(cache)
    assert sc.shape == (3, 5, 2, 4, 16) and sc.dtype == E8 and (sc.float() == 1).all()


def test_refusals():
    hkv, d, ps = 2, 64, 16
    cache, sc = on_dev(*pool8(4, ps, hkv, d))
    k = torch.zeros((3, hkv, d), dtype=torch.float16, device=DEV)
    i = torch.zeros(3, dtype=torch.int32, device=DEV)
    p = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    ap = lambda kk=k, vv=k, b=i, c=cache, s=sc: ops.append_paged_kv_cache(kk, vv, b, i, c, i, p, i[:1], kv_scales=s)  # noqa: E731
    ap()
    bad = [dict(s=None), dict(s=sc.view(torch.uint8)), dict(s=sc[:3]), dict(s=sc.transpose(2, 3)), dict(s=sc.cpu()), dict(s=(sc,)),
           dict(kk=k.float()), dict(kk=k.double(), vv=k.double()), dict(kk=k[:2]), dict(kk=k[..., :32]), dict(kk=k.cpu()), dict(b=i[:2]),
           dict(b=i.long()), dict(c=torch.zeros((4, 2, ps, hkv, d), dtype=torch.float16, device=DEV)),
           dict(c=torch.zeros((4, 2, ps, hkv, 72), dtype=F8, device=DEV), kk=k.new_zeros((3, hkv, 72)), vv=k.new_zeros((3, hkv, 72)))]
    for kw in bad:
        with pytest.raises(ValueError):
            ap(**kw)
    cs, w = torch.zeros((3, d), dtype=torch.float16, device=DEV), torch.ones(d, dtype=torch.float16, device=DEV)
    nr = lambda q=k, qw=w, kw_=w, c=cs, s=cs, ca=cache, sc_=sc, **kw: ops.append_paged_kv_cache_with_norm_rope(  # noqa: E731
        q, k, k, qw, kw_, c, s, i, i, ca, i, p, i[:1], kv_scales=sc_, **kw)
    nr()
    for kw in [dict(q=k[:2]), dict(q=k.float()), dict(qw=w[:32]), dict(qw=w.bfloat16()), dict(qw=w.float()), dict(c=cs[:, :32]), dict(c=cs.float()),
               dict(eps=-1.0), dict(eps=float("nan")), dict(q_out=k[:2]), dict(sc_=None), dict(qw=w.cpu(), kw_=w.cpu()),
               dict(ca=torch.zeros((4, 2, ps, hkv, d), dtype=torch.float16, device=DEV)),
               dict(ca=torch.zeros((4, 2, ps, hkv, d), dtype=torch.bfloat16, device=DEV), sc_=None)]:
        with pytest.raises(ValueError):
            nr(**kw)
    rd = lambda c=cache, s=sc, ii=i, pp=p, dt=torch.float16, **kw: ops.read_paged_kv_cache(c, s, ii, pp, dt, **kw)  # noqa: E731
    rd()
    for kw in [dict(s=None), dict(ii=i.long()), dict(pp=p.cpu()), dict(dt=F8), dict(out=torch.empty(3, device=DEV)), dict(pp=p[:0])]:
        with pytest.raises(ValueError):
            rd(**kw)
