"""The serving path over an 8-bit cache: the page pool's appends, its copies on write, the attention hook, eager
and captured, each against the plain operators or 64 bits over the values that the cache holds."""
import numpy as np
import pytest
import torch

from ecahlang_amd import hook, ops
from ecahlang_amd.manager import AutoKVCacheManager
from ecahlang_amd.wrappers import BatchDecodeWithPagedKVCacheWrapper, BatchPrefillWithPagedKVCacheWrapper
from test_gpu_fp8_cache import E8, F8, dev, f64
from test_gpu_fp8_decode import check, workspace
from oracle import fp8_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
L, HQ, HKV, D = 2, 8, 2, 64


def pool(pages, dtype=torch.float16, **kw):
    return AutoKVCacheManager(L, HKV, D, vocab_size=64, dtype=dtype, device=DEV, kv_dtype="float8_e4m3fn",
                              total_gpu_mem_bytes=pages * 16 * HKV * (D + 1) * 2 * L, mem_utilization=1.0, **kw)


def bytes_of(m):
    return m.kv_cache.view(torch.uint8), m.kv_scales.view(torch.uint8)


def test_the_pool_counts_pages_with_their_scales():
    m = pool(40)
    assert m.max_blocks == 40 and m.kv_cache.dtype == F8 and m.kv_scales.dtype == E8
    assert m.kv_cache.shape == (L, 40, 2, 16, HKV, D) and m.kv_scales.shape == (L, 40, 2, HKV, 16)
    assert m.dtype == torch.float16 and (m.kv_scales.float() == 1).all() and (m.kv_cache.float() == 0).all()
    plain = AutoKVCacheManager(L, HKV, D, vocab_size=64, device=DEV, total_gpu_mem_bytes=40 * 16 * HKV * D * 4 * L, mem_utilization=1.0)
    assert plain.kv_scales is None and plain.layer_scales(0) is None and plain.max_blocks == 40
    for kw in (dict(kv_dtype=torch.bfloat16), dict(kv_dtype=torch.float8_e5m2), dict(kv_dtype="float8_e4m3fn", block_size=3)):
        with pytest.raises(ValueError):
            AutoKVCacheManager(L, HKV, D, vocab_size=64, device=DEV, total_gpu_mem_bytes=1 << 24, **kw)


def test_appends_of_the_pool_are_the_operators():
    m = pool(60)
    m.init_cuda_graph_buffers([4])
    lens, ids = [20, 3, 33], ["a", "b", "c"]
    for i, n in zip(ids, lens):
        m.allocate(i, n)
    ptr = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    n = sum(lens)
    k, v = torch.randn((2, n, HKV, D), device=DEV).half()
    m.prepare_append_metadata(ids, ptr)
    m.append_paged_kv_cache_cached(k, v, 1)
    want, ws = (torch.zeros_like(x[1]) for x in bytes_of(m))
    ws.fill_(127)
    args = (m._cached_batch_indices, m._cached_positions, want.view(F8), m._cached_kv_indices, m._cached_kv_indptr, m._cached_kv_last_page_len)
    ops.append_paged_kv_cache(k, v, *args, kv_scales=ws.view(E8))
    c, s = bytes_of(m)
    assert torch.equal(c[1], want) and torch.equal(s[1], ws) and (c[0] == 0).all()
    m.append_paged_kv_cache(ids, k, v, ptr, 0)
    assert torch.equal(c[0], want) and torch.equal(s[0], ws)
    # a step's rows through the bucket, a padding row among them
    for i in ids:
        m.append_tokens(i, 1)
    m.fill_cuda_graph_metadata(4, ids)
    k1, v1 = torch.randn((2, 4, HKV, D), device=DEV).half()
    m.append_paged_kv_cache_cuda_graph(k1, v1, 4, 0)
    pages = {i: m.batch_to_blocks[i] for i in ids}
    for r, (i, n) in enumerate(zip(ids, lens)):
        pg, sl = pages[i][n // 16], n % 16
        qc, qs = fp8_ref.quantise(f64(k1[r]))
        assert np.array_equal(c[0, pg, 0, sl].cpu().numpy(), qc) and np.array_equal(s[0, pg, 0, :, sl].cpu().numpy(), qs)
    assert m.pool_errors() == 0


def test_copies_on_write_take_the_scales_along():
    m = pool(40)
    c, s = bytes_of(m)
    c.copy_(torch.randint(0, 256, c.shape, dtype=torch.uint8, device=DEV))
    s.copy_(torch.randint(1, 255, s.shape, dtype=torch.uint8, device=DEV))
    c0, s0 = c.clone(), s.clone()
    m.allocate("p", 40)
    m.allocate("a", 40, prefix="p")
    m.append_tokens("a", 1)  # into the shared page: copied first
    pa, pp = m.batch_to_blocks["a"], m.batch_to_blocks["p"]
    torch.cuda.synchronize()
    assert pa[:2] == pp[:2] and pa[2] != pp[2]
    for x, x0 in ((c, c0), (s, s0)):
        assert torch.equal(x[:, pa[2]], x0[:, pp[2]])
        others = [y for y in range(40) if y != pa[2]]
        assert torch.equal(x[:, others], x0[:, others])
    assert m.pool_errors() == 0


def held(m, layer):
    c, s = bytes_of(m)
    return c[layer].cpu().numpy(), s[layer].cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("model_dtype", [None, torch.float32])
def test_the_hook_over_an_8_bit_cache(dtype, model_dtype):
    m = pool(80, dtype)
    lens, ids = [5, 17, 32], ["a", "b", "c"]
    for i, n in zip(ids, lens):
        m.allocate(i, n)
    ptr = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    m.prepare_append_metadata(ids, ptr)
    rnd = lambda h, n: torch.randn((1, h, n, D), device=DEV).to(dtype).to(model_dtype or dtype)  # noqa: E731
    pw = BatchPrefillWithPagedKVCacheWrapper(workspace(), "NHD")
    pw.plan(ptr, m._cached_kv_indptr, m._cached_kv_indices, m._cached_kv_last_page_len, HQ, HKV, D, 16, causal=True,
            q_data_type=dtype, kv_data_type=m.kv_dtype)
    m.prefill_layer_idx = 0
    n = sum(lens)
    for layer in range(L):
        q, k, v = rnd(HQ, n), rnd(HKV, n), rnd(HKV, n)
        o, _ = hook.ecah_attention(None, q, k, v, None, wrapper=pw, manager=m, prefill=True)
        assert o.shape == (1, n, HQ, D) and o.dtype == q.dtype and o.isfinite().all()
        # a prompt's first token sees itself alone: its value, as the cache holds it
        codes, scales = held(m, layer)
        vals = fp8_ref.values(codes, scales)
        for b, i in enumerate(ids):
            first = vals[m.batch_to_blocks[i][0], 1, 0]
            np.testing.assert_allclose(f64(o)[0, int(ptr[b])], np.repeat(first, HQ // HKV, axis=0), rtol=2.0 ** -7, atol=2.0 ** -14)
    assert m.prefill_layer_idx == L
    dw = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
    steps = torch.arange(len(ids) + 1, dtype=torch.int32, device=DEV)
    for _ in range(3):
        for i in ids:
            m.append_tokens(i, 1)
        lens = [n + 1 for n in lens]
        m.prepare_append_metadata(ids, steps)
        dw.plan(m._cached_kv_indptr, m._cached_kv_indices, m._cached_kv_last_page_len, HQ, HKV, D, 16, q_data_type=dtype,
                kv_data_type=m.kv_dtype)
        m.decode_layer_idx = 0
        for layer in range(L):
            q, k, v = rnd(HQ, 3), rnd(HKV, 3), rnd(HKV, 3)
            o, _ = hook.ecah_attention(None, q, k, v, None, wrapper=dw, manager=m, prefill=False)
            t = dict(indptr=f64(m._cached_kv_indptr).astype(int), indices=f64(m._cached_kv_indices).astype(int))
            check(o[0].to(dtype), q[0].transpose(0, 1).to(dtype), t, *held(m, layer), lens, 16)
    assert m.pool_errors() == 0


def test_the_hook_captured_with_a_padding_row():
    m = pool(80)
    m.init_cuda_graph_buffers([4])
    m.cuda_graph_mode = True
    ids, lens = ["a", "b", "c"], [15, 40, 3]
    for i, n in zip(ids, lens):
        m.allocate(i, n)
    ptr = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    m.prepare_append_metadata(ids, ptr)
    n = sum(lens)
    kv = torch.randn((2, n, HKV, D), device=DEV).half()
    for layer in range(L):
        m.append_paged_kv_cache_cached(kv[0], kv[1], layer)
    dw = BatchDecodeWithPagedKVCacheWrapper(workspace(), "NHD")
    q = torch.zeros((L, 1, HQ, 4, D), device=DEV, dtype=torch.float16)
    k, v = torch.zeros((2, L, 1, HKV, 4, D), device=DEV, dtype=torch.float16)
    out = torch.zeros((L, 4, HQ, D), device=DEV, dtype=torch.float16)

    def step():
        dw.plan(m._cg_kv_indptr[4], m._cg_kv_indices[4], m._cg_kv_last_page_len[4], HQ, HKV, D, 16, q_data_type=torch.float16,
                kv_data_type=m.kv_dtype)
        m.decode_layer_idx = 0
        for layer in range(L):
            out[layer].copy_(hook.ecah_attention(None, q[layer], k[layer], v[layer], None, wrapper=dw, manager=m, prefill=False)[0][0])

    def advance():
        for i in ids:
            m.append_tokens(i, 1)
        m.fill_cuda_graph_metadata(4, ids)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV))

    advance()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for s in range(4):
        if s:
            advance()
        g.replay()
        now = [x + s + 1 for x in lens]
        idx = [m.batch_to_blocks[i] for i in ids]
        t = dict(indptr=np.concatenate([[0], np.cumsum([len(x) for x in idx])]), indices=np.concatenate(idx))
        for layer in range(L):
            check(out[layer][:3], q[layer, 0].transpose(0, 1)[:3], t, *held(m, layer), now, 16)
    assert m.pool_errors() == 0
