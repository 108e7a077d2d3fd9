"""What the 8-bit cache's C entry points refuse, on the CPU: a refused call launches nothing, so the addresses
here are never read."""
import ctypes as C

import pytest

from ecahlang_amd import _lib

DTYPE, HEAD, GROUP, ALIGN, ARG, WS, PAGE = -1, -2, -3, -4, -5, -6, -7
F16, BF16, F32 = 0, 1, 2
P = 1 << 20  # an address, aligned and never read


def codes():
    import torch

    return {_lib.DTYPE_CODE[torch.float16], _lib.DTYPE_CODE[torch.bfloat16], _lib.DTYPE_CODE[torch.float32]}


def test_type_codes():
    assert codes() == {F16, BF16, F32}


APPEND = dict(k=P, ksn=256, ksh=128, v=P, vsn=256, vsh=128, bi=P, pos=P, slots=0, nnz=4, kc=P, vc=P, stride=8192, pages=10,
              ks=P, vs=P, sstride=64, idx=P, nidx=10, ptr=P, batch=2, hkv=2, d=128, ps=16, dtype=F16, err=0, stream=0)
NORM = dict(q=P, qsn=2048, qsh=128, qo=P, osn=2048, osh=128, hq=16, k=P, ksn=256, ksh=128, v=P, vsn=256, vsh=128, qw=P, kw=P,
            wdt=F16, eps=1e-6, cos=P, sin=P, csn=128, cdt=F16, bi=P, pos=P, nnz=4, kc=P, vc=P, stride=8192, pages=10, ks=P,
            vs=P, sstride=64, idx=P, nidx=10, ptr=P, batch=2, hkv=2, d=128, ps=16, dtype=F16, err=0, stream=0)
READ = dict(kc=P, vc=P, stride=8192, pages=10, ks=P, vs=P, sstride=64, idx=P, nidx=10, ptr=P, batch=2, hkv=2, d=128, ps=16,
            out=P, dtype=F16, stream=0)
DECODE = dict(q=P, qsn=2048, qsh=128, kc=P, vc=P, stride=8192, pages=10, ks=P, vs=P, sstride=64, ptr=P, idx=P, nidx=10, last=P,
              batch=2, hq=16, hkv=2, d=128, ps=16, scale=0.1, ctas=512, ws=P, wsb=1 << 30, out=P, osn=2048, osh=128,
              dtype=F16, flags=0, stream=0)
PLAN = dict(ptr=P, nidx=10, last=P, batch=2, hq=16, hkv=2, d=128, ps=16, ctas=512, ws=P, wsb=1 << 30, stream=0)
ENTRIES = {"pkv_append_paged_kv_cache_fp8": (APPEND, _lib.CALL_APPEND_FP8),
           "pkv_append_paged_kv_cache_norm_rope": (NORM, _lib.CALL_NORM_ROPE),
           "pkv_read_paged_kv_cache_fp8": (READ, _lib.CALL_READ_FP8),
           "pkv_batch_decode_fp8": (DECODE, _lib.CALL_DECODE_FP8),
           "pkv_decode_fp8_plan": (PLAN, None)}

REFUSED = [("pkv_append_paged_kv_cache_fp8", kw, rc) for kw, rc in [
    (dict(dtype=3), DTYPE), (dict(dtype=-1), DTYPE), (dict(d=0), HEAD), (dict(d=24), HEAD), (dict(d=528), HEAD),
    (dict(nnz=-1), ARG), (dict(hkv=0), ARG), (dict(ps=0), ARG), (dict(batch=-1), ARG), (dict(nidx=-1), ARG),
    (dict(k=0), ARG), (dict(v=0), ARG), (dict(kc=0), ARG), (dict(vc=0), ARG), (dict(ks=0), ARG), (dict(vs=0), ARG),
    (dict(bi=0), ARG), (dict(pos=0), ARG), (dict(ptr=0), ARG), (dict(ksn=-256), ARG), (dict(vsh=-1), ARG),
    (dict(ksn=1 << 31), ARG), (dict(nnz=1 << 30), ARG), (dict(ps=1 << 21, hkv=8), ARG), (dict(k=P + 1), ALIGN),
]] + [("pkv_append_paged_kv_cache_norm_rope", kw, rc) for kw, rc in [
    (dict(dtype=3), DTYPE), (dict(wdt=BF16), DTYPE), (dict(cdt=BF16), DTYPE), (dict(dtype=F32), DTYPE), (dict(d=40), HEAD),
    (dict(nnz=-1), ARG), (dict(hq=-1), ARG), (dict(hkv=0), ARG), (dict(ps=0), ARG), (dict(ks=0), ARG), (dict(vs=0), ARG),
    (dict(cos=0), ARG), (dict(sin=0), ARG), (dict(bi=0), ARG), (dict(pos=0), ARG), (dict(ptr=0), ARG), (dict(q=0), ARG),
    (dict(qo=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG), (dict(kc=0), ARG), (dict(vc=0), ARG), (dict(csn=-1), ARG),
    (dict(qsn=-1), ARG), (dict(osh=1 << 31), ARG), (dict(nnz=1 << 27), ARG), (dict(q=P + 1), ALIGN), (dict(cos=P + 1), ALIGN),
    (dict(kw=P + 1), ALIGN), (dict(ks=0, vs=0, kc=P + 1), ALIGN),
]] + [("pkv_read_paged_kv_cache_fp8", kw, rc) for kw, rc in [
    (dict(dtype=5), DTYPE), (dict(d=8), HEAD), (dict(hkv=0), ARG), (dict(ps=-1), ARG), (dict(batch=-1), ARG), (dict(nidx=-1), ARG),
    (dict(pages=-1), ARG), (dict(ptr=0), ARG), (dict(idx=0), ARG), (dict(out=0), ARG), (dict(kc=0), ARG), (dict(vs=0), ARG),
    (dict(ps=1 << 22), ARG), (dict(kc=P + 4), ALIGN), (dict(stride=8196), ALIGN), (dict(out=P + 8), ALIGN),
]] + [("pkv_batch_decode_fp8", kw, rc) for kw, rc in [
    (dict(dtype=F32), DTYPE), (dict(hq=15), GROUP), (dict(hkv=0), GROUP), (dict(hq=0), GROUP), (dict(ps=0), PAGE), (dict(d=80), HEAD),
    (dict(d=512), HEAD), (dict(pages=-1), ARG), (dict(batch=0), ARG), (dict(nidx=-1), ARG), (dict(ctas=0), ARG),
    (dict(nidx=1 << 28), ARG), (dict(batch=1 << 24), ARG), (dict(q=0), ARG), (dict(out=0), ARG), (dict(ptr=0), ARG), (dict(last=0), ARG),
    (dict(idx=0), ARG), (dict(kc=0), ARG), (dict(ks=0), ARG), (dict(ws=0), ARG), (dict(wsb=40000), WS), (dict(q=P + 8), ALIGN),
    (dict(qsn=2052), ALIGN), (dict(vc=P + 8), ALIGN), (dict(stride=8200), ALIGN), (dict(ks=P + 2), ALIGN), (dict(sstride=66), ALIGN),
]] + [("pkv_decode_fp8_plan", kw, rc) for kw, rc in [
    (dict(batch=0), ARG), (dict(batch=4097), ARG), (dict(hq=15), ARG), (dict(d=80), HEAD), (dict(ps=0), ARG), (dict(ptr=0), ARG),
    (dict(last=0), ARG), (dict(ws=0), ARG), (dict(wsb=40000), WS),
]]


@pytest.mark.parametrize("name,kw,rc", REFUSED)
def test_refused(name, kw, rc):
    args, entry = ENTRIES[name]
    assert set(kw) <= set(args)
    values = list({**args, **kw}.values())
    assert getattr(_lib.lib(), name)(*values) == rc
    if entry is not None:
        assert _lib.call(entry, *values) == rc


@pytest.mark.parametrize("name,kw", [("pkv_append_paged_kv_cache_fp8", dict(nnz=0)), ("pkv_append_paged_kv_cache_norm_rope", dict(nnz=0)),
                                     ("pkv_read_paged_kv_cache_fp8", dict(nidx=0)), ("pkv_read_paged_kv_cache_fp8", dict(batch=0))])
def test_nothing_to_do_launches_nothing(name, kw):
    args, entry = ENTRIES[name]
    assert _lib.call(entry, *{**args, **kw}.values()) == 0


def test_packed_calls_count_their_arguments():
    h = _lib.lib()
    buf = bytes(8 * 64)
    for name, (args, entry) in ENTRIES.items():
        if entry is None:
            continue
        assert len(args) == len(_lib.SIGNATURES[name][1])
        for n in (0, len(args) - 1, len(args) + 1, -1):
            assert h.pkv_call(entry, buf, n) == ARG
    for entry in (-1, 4, 1 << 30):
        assert h.pkv_call(entry, buf, 0) == ARG
    assert h.pkv_call(0, None, len(APPEND)) == ARG


def test_a_packed_call_passes_every_argument():
    # each argument changed alone is told apart where the plain call tells it apart
    for name, (args, entry) in ENTRIES.items():
        if entry is None:
            continue
        f = getattr(_lib.lib(), name)
        for key in args:
            values = list({**args, "dtype": 9, key: 9 if key == "dtype" else -7}.values())
            if any(v < 0 and t is C.c_void_p for v, t in zip(values, _lib.SIGNATURES[name][1])):
                continue
            assert _lib.call(entry, *values) == f(*values) != 0


def test_workspace_sizes():
    ws = _lib.lib().pkv_decode_fp8_workspace_bytes
    base = ws(2, 16, 2, 128, 16, 512, 10)
    assert base > 4 * 8192
    assert ws(64, 16, 2, 128, 16, 512, 10000) > base
    for bad in ((0, 16, 2, 128, 16, 512, 10), (2, 15, 2, 128, 16, 512, 10), (2, 16, 2, 128, 0, 512, 10), (2, 16, 2, 128, 16, 0, 10),
                (2, 16, 2, 128, 16, 512, -1), (2, 16, 2, 128, 16, 512, 1 << 28), (1 << 26, 16, 2, 128, 16, 512, 10)):
        assert ws(*bad) == ARG
    # (the launch's limit on partial rows: 2^31 bytes)
    assert ws(200000, 16, 2, 128, 16, 512, 10) > 0 and ws(300000, 16, 2, 128, 16, 512, 10) == ARG
