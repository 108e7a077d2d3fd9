"""Attention over an 8-bit cache against the 64-bit oracle (oracle/fp8_ref.py).

Tolerance, for each output: half a step of its type, and what fp32 sums and the weights' 17 bits may be off:
sum_t p_t |v_t| times 2 ds + 2^-15, where a score is off by ds <= (D + 8) 2^-24 max_t sum_d |q_d k_d| (any order of
a sum of D products, and the products with scale and log2 e; the exponential's argument in base 2 loses as much
again, within the same bound), twice for numerator and denominator, and 2^-15 covers 2^-17 of the weights, the
exponential's 2^-22 and the sums of weights (all positive: 2^-24 a tile, over at most some hundred rounds).
"""
import numpy as np
import pytest
import torch

from ecahlang_amd import ops
from ecahlang_amd.wrappers import BatchDecodeWithPagedKVCacheWrapper, BatchPrefillWithPagedKVCacheWrapper
from oracle import fp8_ref
from test_gpu_fp8_cache import E8, F8, HALF, dev, f64, on_dev, table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def workspace(mb=64):
    return torch.empty(mb << 20, dtype=torch.uint8, device=DEV)


def batch(kv, ps, hq, hkv, d, dtype, seed=0, spread=3):
    """Sequences of kv tokens: slots nobody owns hold NaN codes and NaN scales."""
    rng = np.random.default_rng(seed)
    t = table(kv, [0] * len(kv), ps, seed=seed)
    codes = np.full((t["pool"], 2, ps, hkv, d), 0x7F, np.uint8)
    scales = np.full((t["pool"], 2, hkv, ps), 255, np.uint8)
    for b, n in enumerate(kv):
        pos = np.arange(n)
        page, slot = t["indices"][t["indptr"][b] + pos // ps], pos % ps
        for j in range(2):
            x = rng.standard_normal((n, hkv, d)) * 2.0 ** rng.integers(-spread, spread + 1, (n, hkv, 1) if j else (1, hkv, 1))
            c, s = fp8_ref.quantise(x)
            codes[page, j, slot], scales[page, j, :, slot] = c, s
    q = torch.from_numpy(rng.standard_normal((len(kv), hq, d))).to(dtype).to(DEV)
    return t, codes, scales, q


def check(out, q, t, codes, scales, kv, ps, sm_scale=None, rows=None):
    vals, got, qd = fp8_ref.values(codes, np.minimum(scales, 254)), f64(out), f64(q)
    d = qd.shape[-1]
    sm_scale = d ** -0.5 if sm_scale is None else sm_scale
    for b in range(len(kv)) if rows is None else rows:
        n = kv[b]
        own = t["indices"][t["indptr"][b]:t["indptr"][b + 1]]
        k, v = (vals[own, j].reshape(-1, *vals.shape[3:])[:n] for j in (0, 1))
        want, mag, big = fp8_ref.attend(qd[b], k, v, sm_scale)
        ds = (d + 8) * 2.0 ** -24 * big
        tol = HALF[out.dtype] * np.abs(want) + (1 + HALF[out.dtype]) * mag * (2 * ds + 2.0 ** -15) + 2.0 ** -24
        bad = np.abs(got[b] - want) > tol
        assert not bad.any(), f"sequence {b} of {n}: {bad.sum()} off, by up to {np.nanmax(np.abs(got[b] - want) / tol):.2f} of the tolerance"


def planned(t, hq, hkv, d, ps, dtype, ws=None, **kw):
    w = BatchDecodeWithPagedKVCacheWrapper(workspace() if ws is None else ws, "NHD")
    w.plan(dev(t["indptr"]), dev(t["indices"]), dev(t["last"]), hq, hkv, d, ps, q_data_type=dtype, kv_data_type=F8, **kw)
    return w


SHAPES = [(16, 2, 128), (32, 8, 64), (28, 4, 128), (8, 4, 256), (5, 5, 64), (24, 1, 128), (33, 1, 64), (40, 2, 256), (1, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("ps", [16, 64, 5])
def test_decode(dtype, hq, hkv, d, ps):
    kv = [1, 15, 16, 17, 100, 333, 2, 64, 129]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=hq + d + ps)
    out = planned(t, hq, hkv, d, ps, dtype).run(q, on_dev(codes, scales)[0], kv_scales=on_dev(codes, scales)[1])
    check(out, q, t, codes, scales, kv, ps)


@pytest.mark.parametrize("ps", [1, 2, 3, 8, 16, 32, 48, 128])
def test_page_sizes(ps):
    kv = [ps, ps + 1, 2 * ps - 1, 3, 200]
    t, codes, scales, q = batch(kv, ps, 8, 2, 64, torch.float16, seed=ps)
    cache, sc = on_dev(codes, scales)
    check(planned(t, 8, 2, 64, ps, torch.float16).run(q, cache, kv_scales=sc), q, t, codes, scales, kv, ps)


@pytest.mark.parametrize("ps", [16, 7, 64])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (14, 2, 64), (40, 2, 128)])
def test_long_sequences_are_split_and_joined(ps, hq, hkv, d):
    kv = [5000, 1, 2311, 40]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.float16, seed=ps + d)
    cache, sc = on_dev(codes, scales)
    for ctas in (None, 3, 64, 2000):
        w = planned(t, hq, hkv, d, ps, torch.float16, num_ctas=ctas)
        a = w.run(q, cache, kv_scales=sc)
        check(a, q, t, codes, scales, kv, ps)
        b = w.run(q, cache, kv_scales=sc)
        assert torch.equal(a, b)  # (the same bits: parts are joined in their order)


def test_many_sequences():
    rng = np.random.default_rng(0)
    kv = [int(x) for x in rng.integers(0, 70, 300)]
    kv[17], kv[255] = 3000, 1500
    t, codes, scales, q = batch(kv, 16, 4, 2, 64, torch.bfloat16, seed=8)
    cache, sc = on_dev(codes, scales)
    out = planned(t, 4, 2, 64, 16, torch.bfloat16).run(q, cache, kv_scales=sc)
    check(out, q, t, codes, scales, kv, 16)
    assert all((out[b] == 0).all() for b, n in enumerate(kv) if n == 0)


def test_values_of_very_unlike_scales():
    # a token of small weight may hold the largest values, and rows of zeros have the smallest scale there is
    kv, ps, hq, hkv, d = [400], 16, 8, 2, 128
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.bfloat16, seed=4, spread=0)
    rng = np.random.default_rng(9)
    pos = np.arange(400)
    page, slot = t["indices"][pos // ps], pos % ps
    v = rng.standard_normal((400, hkv, d)) * 2.0 ** rng.integers(-60, 61, (400, hkv, 1))
    v[::7] = 0.0
    codes[page, 1, slot], scales[page, 1, :, slot] = fp8_ref.quantise(v)
    cache, sc = on_dev(codes, scales)
    check(planned(t, hq, hkv, d, ps, torch.bfloat16).run(q, cache, kv_scales=sc), q, t, codes, scales, kv, ps)
    v[:] = 0.0
    v[:3] = 1.0
    codes[page, 1, slot], scales[page, 1, :, slot] = fp8_ref.quantise(v)
    cache, sc = on_dev(codes, scales)
    check(planned(t, hq, hkv, d, ps, torch.bfloat16).run(q, cache, kv_scales=sc), q, t, codes, scales, kv, ps)


def test_a_nan_in_a_row_reaches_its_head_alone():
    kv, ps, hq, hkv, d = [50, 20], 16, 4, 2, 64
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.float16, seed=4)
    codes[t["indices"][1], 0, 3, 1, 7] = 0x7F       # sequence 0, a key of KV head 1
    codes[t["indices"][0], 1, 2, 0, 9] = 0xFF       # and a value of KV head 0, dim 9
    out = planned(t, hq, hkv, d, ps, torch.float16).run(q, on_dev(codes, scales)[0], kv_scales=on_dev(codes, scales)[1])
    assert out[0, 2:].isnan().all() and out[0, :2, 9].isnan().all() and out[0, :2, :9].isfinite().all() and out[1].isfinite().all()


def test_scores_of_any_size():
    kv, ps, hq, hkv, d = [100], 16, 4, 2, 128
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, torch.float16, seed=6)
    cache, sc = on_dev(codes, scales)
    for sm in (1e-6, 1.0, 30.0):
        out = planned(t, hq, hkv, d, ps, torch.float16, sm_scale=sm).run(q, cache, kv_scales=sc)
        assert out.isfinite().all()
        if sm < 2:
            check(out, q, t, codes, scales, kv, ps, sm)
    # one token far above the rest: its value
    q[:] = 0
    codes[t["indices"][2], 0, 5], scales[t["indices"][2], 0, :, 5] = 0x38, 127 + 20
    q[..., 0] = 1.0
    cache, sc = on_dev(codes, scales)
    out = planned(t, hq, hkv, d, ps, torch.float16, sm_scale=1.0).run(q, cache, kv_scales=sc)
    want = fp8_ref.values(codes, np.minimum(scales, 254))[t["indices"][2], 1, 5]
    np.testing.assert_allclose(f64(out)[0], np.repeat(want, 2, axis=0), rtol=2.0 ** -10)


def test_pages_outside_the_pool_and_a_list_cut_short_have_no_mass():
    ps, hq, hkv, d, dtype = 16, 8, 2, 64, torch.float16
    for size in (16, 8):
        kv = [100, 100]
        t, codes, scales, q = batch(kv, size, hq, hkv, d, dtype, seed=6)
        cache, sc = on_dev(codes, scales)
        idx = t["indices"].copy()
        idx[1], idx[2] = t["pool"], -5
        t2 = dict(t, indices=idx)
        out = planned(t2, hq, hkv, d, size, dtype).run(q, cache, kv_scales=sc)
        check(out, q, t, codes, scales, kv, size, rows=[1])
        vals = fp8_ref.values(codes, np.minimum(scales, 254))
        own = t["indices"][:t["indptr"][1]]
        k, v = (vals[own, j].reshape(-1, hkv, d)[:100] for j in (0, 1))
        keep = np.r_[0:size, 3 * size:100]
        want, mag, big = fp8_ref.attend(f64(q)[0], k[keep], v[keep], d ** -0.5)
        assert (np.abs(f64(out)[0] - want) <= HALF[dtype] * np.abs(want) + 1.01 * mag * (2 * (d + 8) * 2.0 ** -24 * big + 2.0 ** -15) + 2.0 ** -24).all()
        # a list that ends early: the second sequence keeps the tokens of the pages that are there
        cut = t["indptr"][1] + 2
        w = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
        w.plan(dev(t["indptr"]), dev(t["indices"][:cut]), dev(t["last"]), hq, hkv, d, size, q_data_type=dtype, kv_data_type=F8)
        out = w.run(q, cache, kv_scales=sc)
        check(out, q, t, codes, scales, [100, 2 * size], size)
        # nothing but ids outside the pool
        out = planned(dict(t, indices=np.full_like(idx, -1)), hq, hkv, d, size, dtype).run(q, cache, kv_scales=sc)
        assert (out == 0).all()


def test_an_empty_last_page():
    # the pool may give a sequence an empty page (kv_last_page_len 0) when its last one has filled
    for ps in (16, 8, 32):
        kv = [2 * ps, ps, 5]
        t, codes, scales, q = batch([2 * ps + 1, ps + 1, 5], ps, 4, 2, 64, torch.float16, seed=3)
        last = np.array([0, 0, 5], np.int32)
        cache, sc = on_dev(codes, scales)
        out = planned(dict(t, last=last), 4, 2, 64, ps, torch.float16).run(q, cache, kv_scales=sc)
        check(out, q, t, codes, scales, kv, ps)


def test_strided_queries_and_outputs_and_split_caches():
    kv, ps, hq, hkv, d, dtype = [37, 300], 16, 6, 2, 128, torch.bfloat16
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=5)
    cache, sc = on_dev(codes, scales)
    w = planned(t, hq, hkv, d, ps, dtype)
    want = w.run(q, cache, kv_scales=sc)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((2, hq + 3, d + 8), dtype=dtype, device=DEV)
    wide[:, 1:hq + 1, 8:] = q
    odd = torch.zeros((2, hq, d + 1), dtype=dtype, device=DEV)
    odd[..., 1:] = q
    for x in (qt, wide[:, 1:hq + 1, 8:], odd[..., 1:]):
        assert torch.equal(w.run(x, cache, kv_scales=sc), want)
    frame = torch.full((2, hq + 2, d + 1), 9.0, dtype=dtype, device=DEV)
    out = w.run(q, cache, kv_scales=sc, out=frame[:, 1:hq + 1, 1:])
    assert torch.equal(out, want) and (frame[:, 0] == 9).all() and (frame[:, -1] == 9).all() and (frame[..., 0] == 9).all()
    pair = (cache[:, 0].contiguous(), cache[:, 1].contiguous())
    assert torch.equal(w.run(q, pair, kv_scales=(sc[:, 0].contiguous(), sc[:, 1].contiguous())), want)


def test_workspace_is_left_as_found_and_shared_with_other_plans():
    # the counters are back at zero after each run, whatever ran on the workspace before
    ws = workspace()
    ps, hq, hkv, d, dtype = 16, 8, 2, 64, torch.float16
    w = BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
    for kv in ([4000, 3, 900], [7] * 500, [2500], [100] * 40):
        t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=len(kv))
        cache, sc = on_dev(codes, scales)
        w.plan(dev(t["indptr"]), dev(t["indices"]), dev(t["last"]), hq, hkv, d, ps, q_data_type=dtype, kv_data_type=F8)
        check(w.run(q, cache, kv_scales=sc), q, t, codes, scales, kv, ps)
        # a 16-bit decode with its schedule in between
        c16 = ops.read_paged_kv_cache(cache, sc, torch.arange(t["pool"], dtype=torch.int32, device=DEV),
                                      torch.tensor([0, t["pool"]], dtype=torch.int32, device=DEV), dtype)
        w.plan(dev(t["indptr"]), dev(t["indices"]), dev(t["last"]), hq, hkv, d, ps, q_data_type=dtype)
        assert w.run(q, c16).isfinite().all()


def test_captured_and_replayed():
    ps, hq, hkv, d, dtype = 16, 16, 2, 128, torch.float16
    kv = [3000, 77, 500, 1]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=1)
    cache, sc = on_dev(codes, scales)
    w = planned(t, hq, hkv, d, ps, dtype)
    want = w.run(q, cache, kv_scales=sc)
    out, static_q = torch.zeros_like(q), torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.plan(w._indptr, w._indices, w._last, hq, hkv, d, ps, q_data_type=dtype, kv_data_type=F8)
        w.run(static_q, cache, kv_scales=sc, out=out)
        w.run(static_q, cache, kv_scales=sc, out=out)
    for i in range(4):
        static_q.copy_(q.roll(i, 0))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w.run(static_q, cache, kv_scales=sc))
        if i == 0:
            assert torch.equal(out, want)
        (q @ q.transpose(1, 2)).sum().item()  # (the program's own work between replays)
    # the page table changes in place: the run reads it when it runs
    w._last.copy_(dev(np.array([t["last"][0], 3, 2, 1], np.int32)))
    g.replay()
    kv2 = [3000, 67, 498, 1]
    check(out, static_q, t, codes, scales, kv2, ps)


def test_on_a_stream_of_its_own():
    ps, hq, hkv, d, dtype = 16, 16, 2, 128, torch.bfloat16
    kv = [3000, 77, 500, 1]
    t, codes, scales, q = batch(kv, ps, hq, hkv, d, dtype, seed=1)
    cache, sc = on_dev(codes, scales)
    want = planned(t, hq, hkv, d, ps, dtype).run(q, cache, kv_scales=sc)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:
        with torch.cuda.stream(s):
            outs.append([planned(t, hq, hkv, d, ps, dtype).run(q, cache, kv_scales=sc) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for x in outs for o in x)


@pytest.mark.parametrize("dtype,hq,hkv,d,ps", [(torch.float16, 16, 2, 128, 16), (torch.bfloat16, 28, 4, 128, 16), (torch.bfloat16, 4, 2, 64, 8)])
def test_prefill_reads_the_cache_back(dtype, hq, hkv, d, ps):
    kv, new = [70, 16, 301], [70, 5, 33]
    t, codes, scales, _ = batch(kv, ps, hq, hkv, d, dtype, seed=2)
    q = torch.randn((sum(new), hq, d), device=DEV).to(dtype)
    cache, sc = on_dev(codes, scales)
    qo = dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    tab = (dev(t["indptr"]), dev(np.concatenate([t["indices"], [-1] * 9]).astype(np.int32)), dev(t["last"]))  # a longer list
    w8, w16 = (BatchPrefillWithPagedKVCacheWrapper(workspace(), "NHD") for _ in range(2))
    w8.plan(qo, *tab, hq, hkv, d, ps, causal=True, q_data_type=dtype, kv_data_type=F8)
    out = w8.run(q, cache, kv_scales=sc)
    every = torch.arange(t["pool"], dtype=torch.int32, device=DEV)
    c16 = ops.read_paged_kv_cache(cache, sc, every, torch.tensor([0, t["pool"]], dtype=torch.int32, device=DEV), dtype)
    w16.plan(qo, *tab, hq, hkv, d, ps, causal=True, q_data_type=dtype)
    assert torch.equal(out, w16.run(q, c16)) and out.isfinite().all()
    for bad in (dict(kv_scales=None), dict(kv_scales=sc.view(torch.uint8))):
        with pytest.raises(ValueError):
            w8.run(q, cache, **bad)
    with pytest.raises(ValueError):
        w8.run(q, c16)
    with pytest.raises(ValueError):
        w16.run(q, c16, kv_scales=sc)


def test_a_layers_steps_together():
    """Norm, rotation and append of a prompt, its prefill, then steps of one token: norm, rotation, append, decode,
    each against 64 bits over the values that the cache then holds."""
    ps, hq, hkv, d, dtype, eps = 16, 8, 2, 128, torch.bfloat16, 1e-6
    prompt, steps = [30, 1, 16], 20
    t = table([n + steps for n in prompt], prompt, ps)
    cache = torch.zeros((t["pool"], 2, ps, hkv, d), dtype=torch.uint8, device=DEV).view(F8)
    sc = ops.new_kv_scales(cache)
    indptr, indices = dev(t["indptr"]), dev(t["indices"])
    g = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    qw, kw = 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d)

    def angles(pos):
        a = pos.double()[:, None] / (10000.0 ** (torch.arange(0, d, 2, device=DEV).double() / d))
        a = torch.cat([a, a], 1)
        return a.cos().to(dtype), a.sin().to(dtype)

    def write(q, k, v, b, pos, last):
        return ops.append_paged_kv_cache_with_norm_rope(q, k, v, qw, kw, *angles(pos), b, pos, cache, indices, indptr, last, eps=eps, kv_scales=sc)

    n = sum(prompt)
    b = torch.repeat_interleave(torch.arange(3), torch.tensor(prompt)).int().to(DEV)
    pos = torch.cat([torch.arange(c) for c in prompt]).int().to(DEV)
    q = write(rnd(n, hq, d), rnd(n, hkv, d), rnd(n, hkv, d), b, pos, dev(t["last"]))
    # the prompt's pages only
    used = [-(-c // ps) for c in prompt]
    pp = np.concatenate([[0], np.cumsum(used)]).astype(np.int32)
    pi = np.concatenate([t["indices"][t["indptr"][i]:t["indptr"][i] + u] for i, u in enumerate(used)])
    pl = dev(np.array([(c - 1) % ps + 1 for c in prompt], np.int32))
    w = BatchPrefillWithPagedKVCacheWrapper(workspace(), "NHD")
    qo = np.concatenate([[0], np.cumsum(prompt)])
    w.plan(dev(qo.astype(np.int32)), dev(pp), dev(pi), pl, hq, hkv, d, ps, causal=True, q_data_type=dtype, kv_data_type=F8)
    o = f64(w.run(q, cache, kv_scales=sc))
    vals = lambda: fp8_ref.values(cache.view(torch.uint8).cpu().numpy(), sc.view(torch.uint8).cpu().numpy())  # noqa: E731
    held = vals()
    for i, c in enumerate(prompt):
        own = t["indices"][t["indptr"][i]:t["indptr"][i + 1]]
        k, v = (held[own, j].reshape(-1, hkv, d) for j in (0, 1))
        for r in range(c):
            want, mag, _ = fp8_ref.attend(f64(q)[qo[i] + r], k[:r + 1], v[:r + 1], d ** -0.5)
            # (the prefill kernel rounds its weights to bf16: 2^-8 each)
            assert (np.abs(o[qo[i] + r] - want) <= 2.0 ** -8 * np.abs(want) + mag * 2.0 ** -7 + 1e-5).all()
    dw = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
    bi = torch.arange(3, dtype=torch.int32, device=DEV)
    for s in range(steps):
        kv = [c + s + 1 for c in prompt]
        pos = torch.tensor([n - 1 for n in kv], dtype=torch.int32, device=DEV)
        used = [-(-c // ps) for c in kv]
        pp = dev(np.concatenate([[0], np.cumsum(used)]).astype(np.int32))
        own = np.concatenate([t["indices"][t["indptr"][i]:t["indptr"][i] + u] for i, u in enumerate(used)])
        last = dev(np.array([(n - 1) % ps + 1 for n in kv], np.int32))
        q = write(rnd(3, hq, d), rnd(3, hkv, d), rnd(3, hkv, d), bi, pos, last)
        dw.plan(pp, dev(own), last, hq, hkv, d, ps, q_data_type=dtype, kv_data_type="float8_e4m3fn")
        out = dw.run(q, cache, kv_scales=sc)
        codes, scales = cache.view(torch.uint8).cpu().numpy(), sc.view(torch.uint8).cpu().numpy()
        check(out, q, dict(t, indptr=f64(pp).astype(int), indices=own), codes, scales, kv, ps)


def test_refusals():
    ps, hq, hkv, d = 16, 8, 2, 64
    t, codes, scales, q = batch([20, 5], ps, hq, hkv, d, torch.float16)
    cache, sc = on_dev(codes, scales)
    tab = (dev(t["indptr"]), dev(t["indices"]), dev(t["last"]))
    w = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
    plan = lambda **kw: w.plan(*tab, *(kw.pop("geo", (hq, hkv, d, ps))), **{"q_data_type": torch.float16, "kv_data_type": F8, **kw})  # noqa: E731
    plan()
    w.run(q, cache, kv_scales=sc)
    for kw in (dict(), dict(kv_scales=sc.view(torch.uint8)), dict(kv_scales=sc[:1]), dict(kv_scales=(sc,))):
        with pytest.raises(ValueError):
            w.run(q, cache, **kw)
    with pytest.raises(NotImplementedError):
        w.run(q, cache, kv_scales=sc, append_kv=(q[:, :hkv], q[:, :hkv]))
    with pytest.raises(NotImplementedError):
        w.run(q, cache, kv_scales=sc, force_valu=True)
    with pytest.raises(ValueError):
        w.run(q.bfloat16(), cache, kv_scales=sc)
    with pytest.raises(ValueError):
        w.run(q, torch.zeros(cache.shape, dtype=torch.float16, device=DEV), kv_scales=sc)
    for kw in (dict(q_data_type=torch.float32), dict(kv_data_type=torch.bfloat16)):
        with pytest.raises(NotImplementedError):
            plan(**kw)
    for geo in ((hq, hkv, 80, ps), (hq, hkv, 512, ps)):
        with pytest.raises(ValueError):
            plan(geo=geo)
    with pytest.raises(ValueError):
        plan(num_ctas=0)
    small = BatchDecodeWithPagedKVCacheWrapper(torch.empty(4096, dtype=torch.uint8, device=DEV), "NHD")
    with pytest.raises(RuntimeError, match="too small"):
        small.plan(*tab, hq, hkv, d, ps, q_data_type=torch.float16, kv_data_type=F8)
    w.plan(*tab, hq, hkv, d, ps, q_data_type=torch.float16)
    with pytest.raises(ValueError):
        w.run(q, torch.zeros(cache.shape, dtype=torch.float16, device=DEV), kv_scales=sc)
