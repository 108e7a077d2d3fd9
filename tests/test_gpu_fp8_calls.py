"""Ways to call the 8-bit cache's operators: wrappers that take turns on one workspace, captured and replayed calls, two
streams at once, caches past 32-bit offsets, bytes that no append writes.
"""
import numpy as np
import pytest
import torch

from ecahlang_amd import ops
from ecahlang_amd.wrappers import BatchDecodeWithPagedKVCacheWrapper, BatchPrefillWithPagedKVCacheWrapper
from oracle import fp8_ref
from test_gpu_fp8_cache import F8, _norm_case, dev, f64, on_dev, pool8, rows, same, expected, table
from test_gpu_fp8_decode import batch, check, planned, workspace

pytestmark = pytest.mark.gpu
DEV = "cuda"


def u8(t):
    return t.view(torch.uint8)


def test_wrappers_take_turns_on_one_workspace():
    # each lays its partials behind counters that are its own and the others' alike
    ws = workspace()
    turns = []
    for i, (kv, hq, hkv, dtype) in enumerate([([5000, 3], 8, 2, torch.float16), ([3000] + [200] * 69, 16, 8, torch.bfloat16),
                                              ([60] * 399 + [1500], 40, 8, torch.float16), ([2500, 1, 4000], 28, 4, torch.bfloat16)]):
        t, codes, scales, q = batch(kv, 16, hq, hkv, 128, dtype, seed=i)
        w = BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
        turns.append((w, t, codes, scales, q, *on_dev(codes, scales), kv, hq, hkv, dtype))
    w16 = BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
    first = [None] * len(turns)
    for r in range(3):
        for i, (w, t, codes, scales, q, cache, sc, kv, hq, hkv, dtype) in enumerate(turns[::-1] if r == 1 else turns):
            at = len(turns) - 1 - i if r == 1 else i
            tab = (dev(t["indptr"]), dev(t["indices"]), dev(t["last"]))
            w.plan(*tab, hq, hkv, 128, 16, q_data_type=dtype, kv_data_type=F8)
            out = w.run(q, cache, kv_scales=sc)
            if r == 0:
                first[at] = out
                check(out, q, t, codes, scales, kv, 16, rows=[0, len(kv) - 1])
            assert torch.equal(out, first[at])
            if r == 2:  # a 16-bit decode between
                c16 = ops.read_paged_kv_cache(cache, sc, torch.arange(t["pool"], dtype=torch.int32, device=DEV),
                                              torch.tensor([0, t["pool"]], dtype=torch.int32, device=DEV), dtype)
                w16.plan(*tab, hq, hkv, 128, 16, q_data_type=dtype)
                assert w16.run(q, c16).isfinite().all()


@pytest.mark.parametrize("ps", [16, 8])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (8, 1, 128)])
def test_scale_bytes_that_no_append_writes(ps, hq, hkv, d):
    # 0 is 2^-127, 255 NaN: a key's or a value's makes its head's output NaN, unless the slot is past the end
    kv = [40, 37, 20]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.bfloat16, seed=3)
    at = lambda b, pos: (t["indices"][t["indptr"][b] + pos // ps], pos % ps)  # noqa: E731
    for pos in range(40):
        p, s = at(0, pos)
        scales[p, 1, 0, s] = 0  # values of 2^-127 times a code
        scales[p, 0, 0, s] = 0
    g = hq // hkv
    p, s = at(1, 33)
    scales[p, 0, hkv - 1, s] = 255
    p, s = at(2, 7)
    scales[p, 1, 0, s] = 255
    cache, sc = on_dev(codes, scales)
    out = planned(t, hq, hkv, d, ps, torch.bfloat16).run(q, cache, kv_scales=sc)
    assert out[1, -g:].isnan().all() and out[1, :-g].isfinite().all()
    assert out[2, :g].isnan().all() and out[2, g:].isfinite().all()
    own = t["indices"][t["indptr"][0]:t["indptr"][1]]
    vals = fp8_ref.values(codes, np.minimum(scales, 254))
    k, v = (vals[own, j].reshape(-1, hkv, d)[:40] for j in (0, 1))
    want, mag, _ = fp8_ref.attend(f64(q)[0], k, v, d ** -0.5)
    # (scores are near 0: bf16's half step, the weights' 17 bits, and as weights of 2^-127 are subnormal in bf16 too, half its
    # smallest one, 2^-133, of each, times codes of at most 448)
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -13 * mag + 448 * 2.0 ** -134
    assert (np.abs(f64(out)[0, :g] - want[:g]) <= tol[:g]).all() and (want[:g] != 0).any()


def test_a_refused_plan_leaves_none():
    kv, ps, hq, hkv, d = [20, 5, 90], 16, 8, 2, 64
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.float16)
    cache, sc = on_dev(codes, scales)
    w = planned(t, hq, hkv, d, ps, torch.float16)
    w.run(q, cache, kv_scales=sc)
    one = (dev(t["indptr"][:2]), dev(t["indices"]), dev(t["last"][:1]))
    with pytest.raises(ValueError):
        w.plan(*one, hq, hkv, 512, ps, q_data_type=torch.float16, kv_data_type=F8)
    with pytest.raises(RuntimeError):
        w.run(q[:1], cache, kv_scales=sc)


def test_appends_and_reads_captured_and_replayed():
    ps, hq, hkv, d, dtype = 16, 8, 2, 128, torch.bfloat16
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, 5)
    codes, scales = pool8(t["pool"], ps, hkv, d)
    caches = [on_dev(codes, scales) for _ in range(2)]
    tab = (dev(t["b"]), dev(t["pos"]))
    pages = (dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(x, cache, sc, out, read):
        ops.append_paged_kv_cache(x[1], x[2], *tab, cache, *pages, kv_scales=sc, err_count=err)
        ops.append_paged_kv_cache_with_norm_rope(*x, qw, kw, cos, sin, *tab, cache, *pages, kv_scales=sc, q_out=out)
        ops.read_paged_kv_cache(cache, sc, pages[0], pages[1], torch.float32, out=read)

    x = [torch.zeros_like(a) for a in (q, k, v)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    reads = [torch.zeros((len(t["indices"]), 2, ps, hkv, d), device=DEV) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, *caches[0], outs[0], reads[0])
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(x, *caches[0], outs[0], reads[0])
    for i in range(4):
        for a, b in zip(x, (q, k, v)):
            a.copy_(b.roll(i, 0) * 2.0 ** i)
        for c, raw in zip(caches[0], (codes, scales)):
            u8(c).copy_(dev(raw))
        for c, raw in zip(caches[1], (codes, scales)):
            u8(c).copy_(dev(raw))
        g.replay()
        torch.cuda.synchronize()
        step(x, *caches[1], outs[1], reads[1])
        (q.float() @ q.float().transpose(1, 2).contiguous()).sum().item()  # (the program's own work between replays)
        assert all(torch.equal(u8(a), u8(b)) for a, b in zip(*caches)) and torch.equal(outs[0], outs[1])
        assert torch.equal(reads[0].view(torch.int32), reads[1].view(torch.int32))
    assert err.item() == 0


@pytest.mark.parametrize("dtype,hq,hkv,d,wdt,cdt", [
    (torch.bfloat16, 16, 8, 128, None, None), (torch.float16, 3, 4, 64, None, None), (torch.bfloat16, 1, 4, 256, None, torch.float32),
    (torch.float16, 2, 3, 80, torch.float32, None), (torch.float32, 4, 2, 512, None, None), (torch.bfloat16, 5, 5, 16, torch.float32, torch.float32)])
@pytest.mark.parametrize("weights", [True, False])
def test_quantised_keys_are_those_of_64_bits(dtype, hq, hkv, d, wdt, cdt, weights):
    # bit for bit: next to a tie of e4m3 an fp32 key would round to the other side now and then
    eps = 2.0 ** -17  # (the same in any type)
    kv = [1500, 900, 7]
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, 16, 21 + d, wdt=wdt, cdt=cdt, kv=kv, new=kv)
    qw, kw = (qw, kw) if weights else (None, None)
    codes, scales = pool8(t["pool"], 16, hkv, d)
    cache, sc = on_dev(codes, scales)
    ops.append_paged_kv_cache_with_norm_rope(q, k, v, qw, kw, cos, sin, dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]),
                                             dev(t["indptr"]), dev(t["last"]), eps=eps, kv_scales=sc)
    want = fp8_ref.norm_rotate(f64(k), f64(kw) if weights else None, f64(cos), f64(sin), eps)
    same(cache, sc, *expected(codes, scales, t, torch.from_numpy(want), v))


def test_two_streams_at_once():
    ps, hq, hkv, d, dtype = 16, 16, 2, 128, torch.float16
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, 6, kv=(3000, 500, 77), new=(300, 9, 77))
    codes, scales = pool8(t["pool"], ps, hkv, d)
    scales[:] = 127
    codes[:] = codes % 0x70
    tab, pages = (dev(t["b"]), dev(t["pos"])), (dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    qd = q[[299, 308, 385]].contiguous()

    def turn():
        cache, sc = on_dev(codes, scales)
        w = planned(t, hq, hkv, d, ps, dtype)
        outs = []
        for _ in range(5):
            ops.append_paged_kv_cache_with_norm_rope(q, k, v, qw, kw, cos, sin, *tab, cache, *pages, kv_scales=sc)
            outs.append(w.run(qd, cache, kv_scales=sc))
        return outs + [u8(cache), u8(sc)]

    want = turn()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append(turn())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))


def test_prefill_captured_after_its_plan_and_replayed_after_another():
    # the replay keeps the page numbers it was captured with
    ps, hq, hkv, d, dtype = 16, 16, 2, 128, torch.float16
    kv = [300, 40]
    t, codes, scales, _ = batch(kv, ps, hq, hkv, d, dtype, seed=2)
    cache, sc = on_dev(codes, scales)
    q = torch.randn((60, hq, d), device=DEV).to(dtype)
    tab = (dev(t["indptr"]), dev(t["indices"]), dev(t["last"]))
    qo = dev(np.array([0, 30, 60], np.int32))
    w = BatchPrefillWithPagedKVCacheWrapper(workspace(), "NHD")
    w.plan(qo, *tab, hq, hkv, d, ps, causal=True, q_data_type=dtype, kv_data_type=F8)
    want = w.run(q, cache, kv_scales=sc)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.run(q, cache, kv_scales=sc, out=out)
    # (another wrapper's plan takes the memory that this one's would have given back)
    w._plan_read()
    filler = [torch.full((len(t["indices"]),), 7, dtype=torch.int32, device=DEV) for _ in range(64)]
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        filler[0].sum().item()


@pytest.mark.parametrize("cache8", [True, False])
def test_caches_past_32_bit_offsets(cache8):
    ps, hq, hkv, d, dtype = 16, 16, 8, 128, torch.bfloat16
    kv, new = [150, 33], [150, 33]
    t, q, k, v, qw, kw, cos, sin = _norm_case(dtype, hq, hkv, d, ps, 8, kv=kv, new=new)
    near = t["pool"]
    pool = ((1 << 32) // (2 * ps * hkv * d * (1 if cache8 else 2)) + 1000)  # the last 1000 pages lie past 4 GiB
    far = t["indices"] + (pool - near)
    tab, last = (dev(t["b"]), dev(t["pos"])), dev(t["last"])

    def store(pages, indices):
        cache = torch.zeros((pages, 2, ps, hkv, d), dtype=torch.uint8 if cache8 else dtype, device=DEV)
        sc = None
        if cache8:
            cache = cache.view(F8)
            sc = ops.new_kv_scales(cache)
        tb = (dev(indices), dev(t["indptr"]), last)
        out = ops.append_paged_kv_cache_with_norm_rope(q, k, v, qw, kw, cos, sin, *tab, cache, *tb, kv_scales=sc)
        if cache8:  # (the last tokens again, by their slots and by the plain append: the same bytes)
            n = 33
            slots = dev((indices[t["indptr"][t["b"]] + t["pos"] // ps] * ps + t["pos"] % ps)[-n:].astype(np.int32))
            ops.append_paged_kv_cache_slots(k[-n:], v[-n:], slots, cache, kv_scales=sc)
            ops.append_paged_kv_cache(k[:n], v[:n], tab[0][:n], tab[1][:n], cache, *tb, kv_scales=sc)
        return cache, sc, tb, out

    a, b = store(near, t["indices"]), store(pool, far)
    assert torch.equal(a[3], b[3])
    assert torch.equal(u8(a[0]), u8(b[0][-near:])) and not u8(b[0][:5000]).any()
    if not cache8:
        return
    assert torch.equal(u8(a[1]), u8(b[1][-near:]))
    ro = [ops.read_paged_kv_cache(c, s, tb[0], tb[1], dtype) for c, s, tb, _ in (a, b)]
    assert torch.equal(ro[0], ro[1])
    outs = []
    for c, s, tb, _ in (a, b):
        w = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
        w.plan(tb[1], tb[0], tb[2], hq, hkv, d, ps, q_data_type=dtype, kv_data_type=F8)
        outs.append(w.run(q[:2].contiguous(), c, kv_scales=s))
    assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all()
    # and a result past 4 GiB: the far pages of a list of 33,000 in fp32
    n = 33000
    listed = torch.zeros(n, dtype=torch.int32, device=DEV)
    listed[-len(far):] = dev(far)
    big = ops.read_paged_kv_cache(b[0], b[1], listed, torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.float32)
    assert torch.equal(big[-len(far):], ro[0].float()) and not big[n - len(far) - 1].any()


def test_one_token_and_the_largest_heads():
    # the smallest call and the widest row each operator takes
    for hkv, d, ps in ((1, 16, 1), (1, 512, 16)):
        t = table([1], [1], ps)
        k, v = rows(1, hkv, d, torch.float16, 1), rows(1, hkv, d, torch.float16, 2)
        codes, scales = pool8(t["pool"], ps, hkv, d)
        cache, sc = on_dev(codes, scales)
        ops.append_paged_kv_cache(k, v, dev(t["b"]), dev(t["pos"]), cache, dev(t["indices"]), dev(t["indptr"]), dev(t["last"]), kv_scales=sc)
        same(cache, sc, *expected(codes, scales, t, k, v))
        got = ops.read_paged_kv_cache(cache, sc, dev(t["indices"]), dev(t["indptr"]), torch.float32)
        vals = fp8_ref.values(*expected(codes, scales, t, k, v))[t["indices"][0]]
        np.testing.assert_array_equal(f64(got)[0, :, 0], vals[:, 0])


@pytest.mark.parametrize("ps", [16, 8])
def test_batches_without_a_token(ps):
    # zero rows, and rows of a batch's empty sequences, wherever they stand
    hq, hkv, d, dtype = 16, 2, 128, torch.float16
    cache = torch.zeros((3, 2, ps, hkv, d), dtype=torch.uint8, device=DEV).view(F8)
    sc = ops.new_kv_scales(cache)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for indptr, indices, last in ((i32(0, 0, 0), i32(), i32(0, 0)), (i32(0, 0), i32(1, 2), i32(7))):
        w = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
        w.plan(indptr, indices, last, hq, hkv, d, ps, q_data_type=dtype, kv_data_type=F8)
        out = torch.full((last.numel(), hq, d), float("nan"), dtype=dtype, device=DEV)
        w.run(torch.randn_like(out.float()).to(dtype), cache, kv_scales=sc, out=out)
        assert not out.any()
    kv = [0, 70, 0, 0, 3000, 1, 0]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=9)
    out = planned(t, hq, hkv, d, ps, dtype).run(q, on_dev(codes, scales)[0], kv_scales=on_dev(codes, scales)[1])
    check(out, q, t, codes, scales, kv, ps)


def test_more_sequences_than_a_plan_looks_at():
    kv = [1 + i % 5 for i in range(4500)]
    kv[7], kv[4400] = 2000, 900
    t, codes, scales, q = batch(kv, 16, 4, 2, 64, torch.bfloat16, seed=10)
    out = planned(t, 4, 2, 64, 16, torch.bfloat16).run(q, on_dev(codes, scales)[0], kv_scales=on_dev(codes, scales)[1])
    check(out, q, t, codes, scales, kv, 16, rows=[0, 7, 8, 4095, 4096, 4400, 4499])


def test_pages_shared_by_sequences():
    kv, ps, hq, hkv, d, dtype = [600, 50], 16, 16, 2, 128, torch.bfloat16
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=11)
    n = t["indptr"][1]
    shared = dict(indptr=np.array([0, n, 2 * n, 3 * n], np.int32), indices=np.tile(t["indices"][:n], 3), last=np.array([8, 8, 1], np.int32))
    cache, sc = on_dev(codes, scales)
    q3 = q[[0, 0, 0]].contiguous()
    out = planned(shared, hq, hkv, d, ps, dtype).run(q3, cache, kv_scales=sc)
    check(out, q3, shared, codes, scales, [600, 600, 593], ps)
    pages = ops.read_paged_kv_cache(cache, sc, dev(shared["indices"]), dev(shared["indptr"]), dtype)
    assert torch.equal(pages[:n].view(torch.int16), pages[n:2 * n].view(torch.int16))


def test_rotation_without_query_heads():
    t, q, k, v, qw, kw, cos, sin = _norm_case(torch.float16, 1, 3, 64, 16, 12)
    args = (qw, kw, cos, sin, dev(t["b"]), dev(t["pos"]))
    tab = (dev(t["indices"]), dev(t["indptr"]), dev(t["last"]))
    both = [torch.zeros((t["pool"], 2, 16, 3, 64), dtype=torch.float16, device=DEV) for _ in range(2)]
    out = ops.append_paged_kv_cache_with_norm_rope(q[:, :0], k, v, *args, both[0], *tab)
    assert out.shape == (len(t["pos"]), 0, 64)
    ops.append_paged_kv_cache_with_norm_rope(q, k, v, *args, both[1], *tab)
    assert torch.equal(both[0], both[1]) and both[0].any()
