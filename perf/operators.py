"""The 8-bit paged cache's operators as a serving program calls them, and the same in plain tensor operations.

A server that keeps its K/V cache in 8 bits writes each new token's rows as e4m3 values with one power-of-two
scale a token and head (E8M0), attends single tokens to such pages, and reads pages back to 16 bits where a
prompt's chunk is attended by the prefill kernels.  Models that normalise queries and keys per head do that,
and the rotation, on the way into the cache, of 8 bits or of the model's own type.

Four kinds of call:
  rope    RMS norm of every query and key head, rotary embedding, append (cache in the model's type or 8 bits)
  append  K/V rows into an 8-bit cache
  decode  one query token a sequence over an 8-bit cache
  read    listed pages of an 8-bit cache back as 16-bit pages

A case holds plain values; the lengths of its sequences come from the case alone (``lengths`` seeds them), its
tensors' values from the seed given to ``prepare``.  Pages are a random permutation of the pool and slots that no
sequence owns hold stale values, as in a pool that has served for a while.

The 8-bit format: a row x[0 .. D) of one token and head has the smallest power of two s >= 2^-126 with
max|x| <= 448 s; it is stored as s and the e4m3 values nearest to x[d] / s (ties to even).
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1}
EPS = 1e-6


def _heads(hq, hkv, d, dtype):
    return {"hq": hq, "hkv": hkv, "d": d, "dtype": dtype}


QWEN3B = _heads(16, 2, 128, "fp16")   # the headline configuration's attention
LLAMA8B = _heads(32, 8, 128, "bf16")  # the long-context configuration's
LLAMA1B = _heads(32, 8, 64, "fp32")   # the fp32 configuration's
GQA7 = _heads(28, 4, 128, "bf16")     # seven query heads a KV head


def listed():
    return [
        # The smallest step: four chats' new tokens, normalised, rotated and appended to a cache of the model's type.
        {"name": "rope_b4_fp16", "kind": "rope", **QWEN3B, "cache": "fp16", "ps": 16, "tokens": 4, "requests": 4, "lengths": 51},
        # A decode step of 128 sequences into the 8-bit cache.
        {"name": "rope_b128_bf16_fp8", "kind": "rope", **LLAMA8B, "cache": "fp8", "ps": 16, "tokens": 128, "requests": 128, "lengths": 52},
        # A large prefill batch, an odd number of tokens, into the 8-bit cache.
        {"name": "rope_bulk_bf16_fp8", "kind": "rope", **LLAMA8B, "cache": "fp8", "ps": 16, "tokens": 16003, "requests": 9, "lengths": 53},
        # The appends of a decode step whose rotation ran elsewhere.
        {"name": "append_b64_fp16", "kind": "append", **QWEN3B, "ps": 16, "tokens": 64, "requests": 64, "lengths": 54},
        # A full-precision model's prompts into the 8-bit cache, 64 dimensions a head.
        {"name": "append_prompts_fp32", "kind": "append", **LLAMA1B, "ps": 16, "tokens": 2001, "requests": 6, "lengths": 55},
        # The append of a large prefill batch: 65,536 tokens into scattered pages.
        {"name": "append_bulk_fp16", "kind": "append", **QWEN3B, "ps": 16, "tokens": 65536, "requests": 128, "lengths": 56},
        # Four short chats: plan, then one layer's attention, called eagerly.
        {"name": "decode_b4_short_fp16", "kind": "decode", **QWEN3B, "ps": 16, "batch": 4, "lo": 16, "hi": 300, "dist": "uniform",
         "lengths": 57, "plan": True},
        # One layer of the headline decode step: 64 sequences of 512 to 4096 tokens, the plan shared by its layers.
        {"name": "decode_b64_fp16", "kind": "decode", **QWEN3B, "ps": 16, "batch": 64, "lo": 512, "hi": 4096, "dist": "uniform",
         "lengths": 1002, "plan": False},
        # One conversation of 100,003 tokens over pages of 64: the length has to be split to fill the card.
        {"name": "decode_b1_long_bf16", "kind": "decode", **GQA7, "ps": 64, "batch": 1, "lo": 100002, "hi": 100002, "dist": "uniform",
         "lengths": 58, "plan": False},
        # One layer of a long-context step: 32 sequences, log-uniform 1k to 32k tokens.
        {"name": "decode_b32_long_bf16", "kind": "decode", **LLAMA8B, "ps": 16, "batch": 32, "lo": 1024, "hi": 32768, "dist": "log",
         "lengths": 1004, "plan": False},
        # A short prompt's cached prefix, read back for its next chunk.
        {"name": "read_b1_short_fp16", "kind": "read", **QWEN3B, "ps": 16, "batch": 1, "lo": 300, "hi": 300, "dist": "uniform", "lengths": 59},
        # Eight requests' prefixes of up to 8192 tokens and their 512-token chunks, read back for the chunks' attention.
        {"name": "read_chunks_bf16", "kind": "read", **LLAMA8B, "ps": 16, "batch": 8, "lo": 512, "hi": 8704, "dist": "uniform",
         "lengths": 1003},
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "decode", "decode", "decode", "read"])
    heads = rng.choice([QWEN3B, LLAMA8B, GQA7, _heads(12, 2, 128, "fp16"), _heads(14, 2, 64, "bf16"), _heads(40, 8, 128, "fp16"),
                        _heads(32, 8, 64, "bf16"), _heads(16, 16, 64, "fp16"), _heads(24, 1, 128, "bf16"), _heads(8, 4, 256, "bf16")])
    if kind in ("rope", "append") and rng.random() < 0.2:
        heads = dict(heads, dtype="fp32")
    case = {"kind": kind, **heads, "ps": rng.choice([16, 16, 16, 32, 64, 8]), "lengths": rng.randrange(1 << 20)}
    if kind in ("rope", "append"):
        row = (heads["hq"] + 2 * heads["hkv"]) * heads["d"] * SIZE[heads["dtype"]]
        tokens = _logint(rng, 1, max(64, min(65536 if kind == "append" else 16384, 100_000_000 // row)))
        case |= {"tokens": tokens, "requests": max(1, min(tokens, _logint(rng, 1, 128)))}
        if kind == "rope":
            case["cache"] = rng.choice(["fp8", "fp8", heads["dtype"]])
        return case
    batch = _logint(rng, 1, 256 if kind == "decode" else 16)
    most = (400_000_000 if kind == "decode" else 60_000_000) // (batch * 2 * heads["hkv"] * heads["d"])
    hi = max(32, min(_logint(rng, 32, 65536 if kind == "decode" else 16384), most))
    case |= {"batch": batch, "lo": max(1, hi // rng.choice([1, 4, 16, 32])), "hi": hi, "dist": rng.choice(["uniform", "log"])}
    if kind == "decode":
        case["plan"] = rng.random() < 0.3
    return case


# ---------------------------------------------------------------- lengths and page tables

def _lengths(case):
    """(tokens per sequence, new tokens per sequence), from the case alone."""
    rng = random.Random(case["lengths"])
    if case["kind"] in ("decode", "read"):
        spread = _logint if case["dist"] == "log" else lambda r, lo, hi: r.randint(lo, hi)
        kv = [spread(rng, case["lo"], case["hi"]) + (case["kind"] == "decode") for _ in range(case["batch"])]
        return kv, [0] * len(kv)
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["requests"] - 1))
    new = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return [n + rng.randint(0, 100) for n in new], new


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cumsum(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


# ---------------------------------------------------------------- the 8-bit format in plain operations

def _quantise(x):
    """x [..., D] -> (e4m3 values, E8M0 scales [...])."""
    bits = x.float().abs().amax(-1).view(torch.int32)
    # amax = m 2^E with 1 <= m < 2: the scale's exponent is E - 8, or E - 7 where m > 1.75 (448 = 1.75 * 2^8)
    e = (((bits + 0x1FFFFF) >> 23) - 8).clamp_(min=1)
    codes = (x.float() * ((254 - e) << 23).view(torch.float32)[..., None]).to(torch.float8_e4m3fn)
    return codes, e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _put(dst, at, rows):
    """dst[at] = rows, as bytes where the type is of 8 bits."""
    if dst.element_size() == 1:
        dst, rows = dst.view(torch.uint8), rows.view(torch.uint8)
    dst[at] = rows.to(dst.dtype)


# ---------------------------------------------------------------- states

def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, ps, hq, hkv, d = DTYPES[case["dtype"]], case["ps"], case["hq"], case["hkv"], case["d"]
    kv, new = _lengths(case)
    npages = [-(-n // ps) for n in kv]
    used = sum(npages)
    pool = used + used // 4 + 1
    # keys have channels of very unlike sizes, the same ones for every token
    gain = torch.exp(0.5 * torch.randn((2, 1, hkv, d), generator=gen, device=DEV))
    st = {"case": case, "kv": kv, "new": new, "most": max(npages), "pages": used,
          "indptr": _i32(_cumsum(npages)), "last": _i32([(n - 1) % ps + 1 for n in kv]),
          "indices": torch.randperm(pool, generator=gen, device=DEV)[:used].to(torch.int32)}
    kept = case.get("cache", "fp8")
    cache = torch.empty((pool, 2, ps, hkv, d), dtype=DTYPES[kept], device=DEV)
    if kept == "fp8":
        scales = torch.empty((pool, 2, hkv, ps), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 27) // (2 * ps * hkv * d))
        for a in range(0, pool, step):
            x = torch.randn((min(step, pool - a), 2, ps, hkv, d), generator=gen, device=DEV) * gain
            codes, e = _quantise(x)
            cache[a:a + step] = codes
            scales[a:a + step] = e.view(torch.uint8).transpose(2, 3)
        st["scales"] = scales.view(torch.float8_e8m0fnu)
    else:
        cache.normal_(generator=gen)
    st["cache"] = cache
    nnz = len(kv) if case["kind"] == "decode" else sum(new)
    if nnz:
        st["q"] = torch.randn((nnz, hq, d), generator=gen, device=DEV).to(dtype)
        rows = torch.randn((2, nnz, hkv, d), generator=gen, device=DEV) * gain
        st["k"], st["v"] = rows[0].to(dtype), rows[1].to(dtype)
    if case["kind"] in ("rope", "append"):
        st["positions"] = torch.cat([torch.arange(n - c, n, dtype=torch.int32) for n, c in zip(kv, new)]).to(DEV)
        st["batch_indices"] = torch.repeat_interleave(torch.arange(len(new), dtype=torch.int32), torch.tensor(new)).to(DEV)
    if case["kind"] == "rope":
        st["qw"], st["kw"] = (1 + 0.2 * torch.randn((2, d), generator=gen, device=DEV)).to(dtype)
        # the model's position embeddings of these tokens
        inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))
        ang = st["positions"].double()[:, None] * inv[None, :]
        ang = torch.cat([ang, ang], dim=1)
        st["cos"], st["sin"] = ang.cos().to(dtype), ang.sin().to(dtype)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["kind"] == "decode":
        from ecahlang_amd.wrappers import BatchDecodeWithPagedKVCacheWrapper
        st["wrapper"] = BatchDecodeWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device=DEV), "NHD")
        _plan(st)
    return st


def _plan(st):
    case = st["case"]
    st["wrapper"].plan(st["indptr"], st["indices"], st["last"], case["hq"], case["hkv"], case["d"], case["ps"],
                       pos_encoding_mode="NONE", q_data_type=DTYPES[case["dtype"]], kv_data_type=torch.float8_e4m3fn)


# ---------------------------------------------------------------- one pass

def run(st):
    if own:
        return _run_own(st)
    return {"rope": _rope, "append": _append, "decode": _decode, "read": _read}[st["case"]["kind"]](st)


def _run_own(st):
    from ecahlang_amd import ops
    case = st["case"]
    if case["kind"] == "rope":
        q = ops.append_paged_kv_cache_with_norm_rope(
            st["q"], st["k"], st["v"], st["qw"], st["kw"], st["cos"], st["sin"], st["batch_indices"], st["positions"],
            st["cache"], st["indices"], st["indptr"], st["last"], eps=EPS, kv_scales=st.get("scales"))
        return (q, st["cache"], st["scales"]) if "scales" in st else (q, st["cache"])
    if case["kind"] == "append":
        ops.append_paged_kv_cache(st["k"], st["v"], st["batch_indices"], st["positions"], st["cache"], st["indices"],
                                  st["indptr"], st["last"], kv_scales=st["scales"])
        return st["cache"], st["scales"]
    if case["kind"] == "decode":
        if case["plan"]:
            _plan(st)
        return st["wrapper"].run(st["q"], st["cache"], kv_scales=st["scales"])
    return ops.read_paged_kv_cache(st["cache"], st["scales"], st["indices"], st["indptr"], DTYPES[case["dtype"]])


def _slots(st):
    """Page and slot of every new token."""
    pos, ps = st["positions"].long(), st["case"]["ps"]
    return st["indices"].long()[st["indptr"].long()[st["batch_indices"].long()] + pos // ps], pos % ps


def _write(st, k, v):
    page, slot = _slots(st)
    for j, x in enumerate((k, v)):
        if "scales" in st:
            codes, e = _quantise(x)
            _put(st["cache"][:, j], (page, slot), codes)
            _put(st["scales"][:, j].transpose(1, 2), (page, slot), e)
        else:
            _put(st["cache"][:, j], (page, slot), x)


def _norm_turn(x, w, cos, sin):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    h = x.shape[-1] // 2
    return x * cos.float()[:, None] + torch.cat([-x[..., h:], x[..., :h]], dim=-1) * sin.float()[:, None]


def _rope(st):
    q = _norm_turn(st["q"], st["qw"], st["cos"], st["sin"]).to(st["q"].dtype)
    _write(st, _norm_turn(st["k"], st["kw"], st["cos"], st["sin"]), st["v"])
    return (q, st["cache"], st["scales"]) if "scales" in st else (q, st["cache"])


def _append(st):
    _write(st, st["k"], st["v"])
    return st["cache"], st["scales"]


def _values(st, pages):
    """The values that pages [...] hold, in 32 bits: [..., 2, ps, hkv, d]."""
    codes = st["cache"].view(torch.uint8)[pages].view(torch.float8_e4m3fn)
    scales = st["scales"].view(torch.uint8)[pages].view(torch.float8_e8m0fnu)
    return codes.float() * scales.float().transpose(-1, -2)[..., None]


def _decode(st):
    case, most = st["case"], st["most"]
    hkv, d, ps = case["hkv"], case["d"], case["ps"]
    n = st["indptr"][1:] - st["indptr"][:-1]
    at = torch.arange(most, device=DEV)
    pages = st["indices"].long()[(st["indptr"][:-1, None] + at).clamp(max=st["pages"] - 1).long()]
    kv = _values(st, pages).permute(2, 0, 4, 1, 3, 5)  # [2, B, hkv, pages, ps, d]
    k, v = (x.reshape(len(n), hkv, most * ps, d) for x in kv)
    q = st["q"].float().view(len(n), hkv, -1, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    length = (n - 1) * ps + st["last"]
    s = s.masked_fill(torch.arange(most * ps, device=DEV) >= length[:, None, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(st["q"].shape).to(st["q"].dtype)


def _read(st):
    return _values(st, st["indices"].long()).to(DTYPES[st["case"]["dtype"]])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    es, hq, hkv, d, ps = SIZE[case["dtype"]], case["hq"], case["hkv"], case["d"], case["ps"]
    kv, new = _lengths(case)
    pages = sum(-(-n // ps) for n in kv)
    table = 4 * (pages + 2 * len(kv) + 1)
    row8 = 2 * hkv * (d + 1)  # a token's K and V in 8 bits, with their scales
    if case["kind"] == "decode":
        return {"bytes": sum(kv) * row8 + 2 * len(kv) * hq * d * es + table, "flops": 4 * hq * d * sum(kv)}
    if case["kind"] == "read":
        return {"bytes": pages * ps * (row8 + 2 * hkv * d * es) + 4 * pages, "flops": 2 * pages * ps * hkv * d}
    nnz = sum(new)
    kept = row8 if case.get("cache", "fp8") == "fp8" else 2 * hkv * d * es
    each = 2 * hkv * d * es + kept + 8
    if case["kind"] == "append":
        return {"bytes": nnz * each + table, "flops": 4 * nnz * hkv * d}
    return {"bytes": nnz * (each + (2 * hq + 2) * d * es) + table + 2 * d * es, "flops": 8 * nnz * (hq + hkv) * d + 2 * nnz * hkv * d}


# ---------------------------------------------------------------- the same results in 64 bits

def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3_64(x):
    """(nearest e4m3 values of each row over its scale, the scales), in 64 bits by arithmetic alone."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(torch.where(amax > 0, amax, torch.ones_like(amax)) / 448)  # in [1/2, 1) * 2^e
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    y = x * _pow2_64(-e)[..., None]
    quantum = _pow2_64((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return torch.round(y / quantum) * quantum, _pow2_64(e)


def _held64(st, page):
    """The values of one page, [2, ps, hkv, d]."""
    return st["cache"][page].double() * st["scales"][page].double().transpose(-1, -2)[..., None]


def exact(case, seed):
    st = _inputs(case, seed)
    hkv, d, ps = case["hkv"], case["d"], case["ps"]
    ptr = _cumsum([-(-n // ps) for n in st["kv"]])
    idx = st["indices"].tolist()
    if case["kind"] == "read":
        out = torch.empty((len(idx), 2, ps, hkv, d), dtype=torch.float64, device=DEV)
        for i, page in enumerate(idx):
            out[i] = _held64(st, page)
        return out
    if case["kind"] == "decode":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
        g = case["hq"] // hkv
        for b, n in enumerate(st["kv"]):
            mine = st["indices"][ptr[b]:ptr[b + 1]].long()
            for h in range(hkv):
                k, v = ((st["cache"].view(torch.uint8)[mine, j, :, h].view(torch.float8_e4m3fn).double()
                         * st["scales"].view(torch.uint8)[mine, j, h].view(torch.float8_e8m0fnu).double()[..., None]
                         ).reshape(-1, d)[:n] for j in (0, 1))
                s = st["q"][b, h * g:(h + 1) * g].double() @ k.t() * d ** -0.5
                out[b, h * g:(h + 1) * g] = torch.softmax(s, dim=-1) @ v
        return out
    # every new token's page and slot, counted off sequence by sequence
    page, slot = [], []
    for b, (n, c) in enumerate(zip(st["kv"], st["new"])):
        page += [idx[ptr[b] + p // ps] for p in range(n - c, n)]
        slot += [p % ps for p in range(n - c, n)]
    page, slot = torch.tensor(page, device=DEV), torch.tensor(slot, device=DEV)
    k, v, q = st["k"].double(), st["v"].double(), None
    if case["kind"] == "rope":
        c, s, h = st["cos"].double()[:, None], st["sin"].double()[:, None], d // 2

        def turned(x, w):
            x = x.double()
            y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
            return torch.cat([y[..., :h] * c[..., :h] - y[..., h:] * s[..., :h], y[..., h:] * c[..., h:] + y[..., :h] * s[..., h:]], dim=-1)
        q, k = turned(st["q"], st["qw"]), turned(k, st["kw"])
    cache = st["cache"].double()
    if "scales" not in st:
        cache[page, 0, slot], cache[page, 1, slot] = k, v
        return q, cache
    scales = st["scales"].double()
    for j, x in enumerate((k, v)):
        codes, e = _e4m3_64(x)
        cache[page, j, slot] = codes
        scales[:, j].transpose(1, 2)[page, slot] = e
    return (q, cache, scales) if q is not None else (cache, scales)
