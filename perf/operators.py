"""What the 8-bit product and the quantised key/value cache are measured on.

Operators (the package's names):

* ``quantize_int8`` / ``dequantize_int8`` -- rows of activations or weights to
  8-bit codes with one scale a row, and back;
* ``int8_matmul`` -- y = x W^T for x quantised a token at a time inside the
  call and W held as 8-bit codes with a scale for each output channel;
* ``cache_write`` / ``cache_read`` -- keys and values quantised to 8 or 4 bits
  as they are written into a paged cache, and read back;
* ``cache_attention`` -- one query token a sequence over that cache.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes a case's inputs on the GPU, ``run`` is one call as a user
makes it (or, with ``own`` false, the same in elementary torch operations),
``work`` what the call cannot do without and ``exact`` its result in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
GROUP4 = 32  # channels that share a 4-bit scale and minimum


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rows(rows, K, dtype, name=None):
    c = {"op": "rows", "rows": rows, "K": K, "dtype": dtype}
    return dict(c, name=name) if name else c


def _matmul(M, N, K, dtype, bias, name=None):
    c = {"op": "matmul", "M": M, "N": N, "K": K, "dtype": dtype, "bias": bias}
    return dict(c, name=name) if name else c


def _cache(new, context, heads, dim, bits, page, dtype, name=None):
    c = {"op": "cache", "new": new, "context": context, "kv_heads": heads, "dim": dim,
         "bits": bits, "page": page, "dtype": dtype}
    return dict(c, name=name) if name else c


def _attention(batch, heads, kv_heads, dim, longest, bits, page, empty, dtype, name=None):
    c = {"op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "longest": longest, "bits": bits, "page": page, "empty": empty, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the hidden states of a few sequences' single tokens: a latency
        _rows(8, 4096, "float16", "rows 8x4096"),
        # a long prompt's MLP activations (or a weight matrix, an output channel a row)
        _rows(8192, 11008, "bfloat16", "rows 8192x11008"),
        # one token through a 4096 x 4096 projection
        _matmul(1, 4096, 4096, "float16", False, "matmul 1 token"),
        # a serving batch of single tokens through the MLP's wide projection
        _matmul(48, 11008, 4096, "bfloat16", False, "matmul 48 tokens"),
        # a short prompt and sizes that no tile divides, with a bias
        _matmul(515, 4100, 1001, "float16", True, "matmul ragged"),
        # four 2048-token prompts through the MLP's wide projection
        _matmul(8192, 11008, 4096, "bfloat16", False, "matmul prompts"),
        # single tokens of a batch stored, and read back
        _cache(24, 24, 32, 128, 8, 16, "float16", "cache 24 tokens"),
        # a chunk of a prompt stored in 4 bits, the context so far read back
        _cache(2048, 8000, 8, 128, 4, 64, "bfloat16", "cache chunk"),
        # one short sequence: a latency
        _attention(1, 32, 32, 128, 300, 8, 16, False, "float16", "attend 1x300"),
        # a serving batch, a key/value head for each query head, one padded row
        _attention(16, 32, 32, 128, 2048, 8, 16, True, "float16", "attend 16x2048"),
        # a larger batch with eight query heads to a key/value head, 4 bits
        _attention(48, 64, 8, 128, 8192, 4, 64, False, "bfloat16", "attend 48x8192"),
        # two long documents
        _attention(2, 32, 8, 128, 100001, 8, 128, False, "bfloat16", "attend 2x100001"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "matmul", "matmul", "cache", "attention", "attention"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "rows":
        K = _log(rng, 17, 30000)
        rows = _log(rng, 1, max(2, min(60000, 90000000 // K)))
        return _rows(rows, K, rng.choice(["float16", "bfloat16", "float32"]))
    if op == "matmul":
        N, K = _log(rng, 40, 16384), _log(rng, 40, 16384)
        M = _log(rng, 1, max(2, min(8192, 8192 * 11008 * 4096 // (N * K))))
        return _matmul(M, N, K, dtype, rng.random() < 0.5)
    bits = rng.choice([8, 4])
    dim = rng.choice([64, 80, 128, 192, 256] if bits == 8 else [64, 96, 128, 256])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16, 32])
    if op == "cache":
        context = _log(rng, 1, max(2, min(65536, 8388608 // (kv_heads * dim // 2))))
        return _cache(_log(rng, 1, context) if context > 1 else 1, context, kv_heads, dim, bits,
                      page, dtype)
    group = rng.choice([1, 2, 4, 7, 8, 12, 16])
    batch = _log(rng, 1, 96)
    longest = _log(rng, 1, max(2, min(100000, 100000000 // (batch * kv_heads * dim))))
    return _attention(batch, group * kv_heads, kv_heads, dim, longest, bits, page,
                      batch > 1 and rng.random() < 0.3, dtype)


def _lengths(case):
    """The first sequence has the longest length, the others are spread over
    1 .. longest; with "empty" the last row of the batch is padding."""
    n = [1 + int((case["longest"] - 1) * ((i * 0.6180339887) % 1.0)) for i in range(case["batch"])]
    n[0] = case["longest"]
    if case["empty"]:
        n[-1] = 0
    return n


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(shape, g, dtype):
    """Gaussian rows, one channel in about a hundred 20 times larger."""
    x = torch.randn(shape, generator=g, device="cuda")
    big = torch.rand(shape[-1:], generator=g, device="cuda") < 0.01
    return torch.where(big, x * 20, x).to(DTYPES[dtype])


def _keys_values(shape, g, dtype):
    """Gaussian keys with a few large channels; values of differing size from
    token to token."""
    k, v = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
    big = torch.rand(shape[-1:], generator=g, device="cuda") < 0.03
    size = 0.25 + torch.rand(shape[:-1] + (1,), generator=g, device="cuda")
    return torch.where(big, k * 6, k).to(DTYPES[dtype]), (v * size).to(DTYPES[dtype])


def _per_row(x, dtype):
    return torch.full((), x, dtype=dtype, device="cuda")


def _encode8(x):
    """int8 codes and fp32 scales of the rows of x: scale = max|x| / 127, code
    = x / scale to the nearest, ties to even (the quotient in 64 bits: the
    codes next to a border depend on it)."""
    scale = x.float().abs().amax(-1) / _per_row(127.0, torch.float32)
    s = scale.double().unsqueeze(-1)
    q = torch.round(x.double() / s).clamp(-127, 127)
    return torch.where(s > 0, q, torch.zeros_like(q)).to(torch.int8), scale


def _encode4(x):
    """uint8 bytes of two 4-bit codes (even channel low) and fp16 (scale,
    minimum) of each 32 channels of x: code = (x - minimum) / scale to the
    nearest, ties to even."""
    g = x.double().unflatten(-1, (-1, GROUP4))
    lo, hi = g.amin(-1), g.amax(-1)
    m = lo.float().half()
    s = ((hi - lo) / _per_row(15.0, torch.float64)).float().half()
    s64 = s.double().unsqueeze(-1)
    q = torch.round((g - m.double().unsqueeze(-1)) / s64).clamp(0, 15)
    q = torch.where(s64 > 0, q, torch.zeros_like(q)).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack((s, m), -1)


def _encode(x, bits):
    return _encode8(x) if bits == 8 else _encode4(x)


def _decode(codes, scales, bits):
    """The fp32 values that codes stand for."""
    if bits == 8:
        return codes.float() * scales.unsqueeze(-1)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP4))
    return (scales[..., 1:].float() + scales[..., :1].float() * q).flatten(-2)


def _empty_cache(pages, case):
    bits, dim = case["bits"], case["dim"]
    shape = (pages, case["kv_heads"], case["page"])
    out = {}
    for n in ("k", "v"):
        if bits == 8:
            out[n + "_codes"] = torch.zeros(shape + (dim,), dtype=torch.int8, device="cuda")
            out[n + "_scales"] = torch.zeros(shape, dtype=torch.float32, device="cuda")
        else:
            out[n + "_codes"] = torch.zeros(shape + (dim // 2,), dtype=torch.uint8, device="cuda")
            out[n + "_scales"] = torch.zeros(shape + (dim // GROUP4, 2), dtype=torch.float16,
                                             device="cuda")
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 9176 + 11)
    state = {"case": case}
    if case["op"] == "rows":
        x = _activations((case["rows"], case["K"]), g, case["dtype"])
        if case["rows"] > 4:
            x[2] = 0  # a padding token
        return dict(state, x=x)
    if case["op"] == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        w = torch.randn((N, K), generator=g, device="cuda") * 0.02
        codes, scales = _encode8(w)
        held = torch.zeros((N, -(-K // 16) * 16), dtype=torch.int8, device="cuda")[:, :K]
        held.copy_(codes)  # rows begin on 16-byte boundaries
        bias = None
        if case["bias"]:
            bias = torch.randn((N,), generator=g, device="cuda").to(DTYPES[case["dtype"]])
        return dict(state, x=_activations((M, K), g, case["dtype"]), w_codes=held,
                    w_scales=scales, bias=bias)
    page = case["page"]
    if case["op"] == "cache":
        context, new = case["context"], case["new"]
        pages = -(-context // page) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(context, device="cuda")
        slots = order[t // page] * page + t % page
        cache = _empty_cache(pages, case)
        if context > new:  # what is there before the new tokens
            k, v = _keys_values((pages, case["kv_heads"], page, case["dim"]), g, case["dtype"])
            for n, x in (("k", k), ("v", v)):
                cache[n + "_codes"], cache[n + "_scales"] = _encode(x, case["bits"])
        k, v = _keys_values((new, case["kv_heads"], case["dim"]), g, case["dtype"])
        return dict(state, cache=cache, k=k, v=v, slots=slots,
                    new_slots=slots[context - new:].contiguous())
    lengths = _lengths(case)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = _keys_values((pages, case["kv_heads"], page, case["dim"]), g, case["dtype"])
    cache = {}
    cache["k_codes"], cache["k_scales"] = _encode(k, case["bits"])
    cache["v_codes"], cache["v_scales"] = _encode(v, case["bits"])
    q = torch.randn((case["batch"], case["heads"], case["dim"]), generator=g, device="cuda")
    return dict(state, cache=cache, q=q.to(DTYPES[case["dtype"]]), table=table,
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        codes, scales = _encode8(state["x"])
        return {"values": _decode(codes, scales, 8).to(dtype), "scales": scales}
    if case["op"] == "matmul":
        codes, scales = _encode8(state["x"])
        y = codes.double() @ state["w_codes"].double().T
        y = y * scales.double().unsqueeze(1) * state["w_scales"].double()
        if state["bias"] is not None:
            y = y + state["bias"].double()
        return y.to(dtype)
    cache, bits, page = state["cache"], case["bits"], case["page"]
    if case["op"] == "cache":
        out = []
        at, slots = state["new_slots"], state["slots"]
        for n in ("k", "v"):
            codes, scales = _encode(state[n], bits)
            cache[n + "_codes"][at // page, :, at % page] = codes
            cache[n + "_scales"][at // page, :, at % page] = scales
            out.append(_decode(cache[n + "_codes"][slots // page, :, slots % page],
                               cache[n + "_scales"][slots // page, :, slots % page],
                               bits).to(dtype))
        return out
    q, table = state["q"], state["table"].clamp(min=0)
    B, H, D = q.shape
    Hkv = case["kv_heads"]

    def gather(n):  # [B, Hkv, positions, D]
        x = _decode(cache[n + "_codes"][table], cache[n + "_scales"][table], bits)
        return x.transpose(1, 2).reshape(B, Hkv, -1, D)

    k = gather("k")
    s = (q.float().view(B, Hkv, H // Hkv, D) @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    del k
    seen = torch.arange(s.shape[-1], device="cuda") < state["lengths"].view(B, 1, 1, 1)
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    o = (p @ gather("v")) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(B, H, D).to(dtype)


def _run_own(state):
    import memboost_b200 as mb
    case = state["case"]
    if case["op"] == "rows":
        t = mb.quantize_int8(state["x"])
        return {"values": mb.dequantize_int8(t, dtype=state["x"].dtype), "scales": t.scales}
    if case["op"] == "matmul":
        w = mb.Int8Tensor(state["w_codes"], state["w_scales"])
        return mb.int8_matmul(state["x"], w, bias=state["bias"])
    cache = mb.QuantizedCache(**state["cache"])
    if case["op"] == "cache":
        mb.cache_write(cache, state["k"], state["v"], state["new_slots"])
        return list(mb.cache_read(cache, state["slots"], dtype=state["k"].dtype))
    return mb.cache_attention(state["q"], cache, state["table"], state["lengths"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _row_bytes(case):
    """Codes and scales of one token's key (or value) of one head."""
    return case["dim"] + 4 if case["bits"] == 8 else case["dim"] // 2 + case["dim"] // GROUP4 * 4


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rows":
        # x in, codes and scales out; codes and scales in, values out
        n = case["rows"] * case["K"]
        return {"bytes": n * (2 * size + 2) + 8 * case["rows"], "flops": 4 * n}
    if case["op"] == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        bytes_ = M * K * size + N * K + 4 * N + M * N * size + (N * size if case["bias"] else 0)
        return {"bytes": bytes_, "flops": 2 * M * N * K}
    if case["op"] == "cache":
        values = 2 * case["kv_heads"] * case["dim"] * size
        held = 2 * case["kv_heads"] * _row_bytes(case)
        n = case["new"] + case["context"]
        return {"bytes": n * (values + held + 8), "flops": n * values}
    tokens = sum(_lengths(case))
    rows = 2 * case["batch"] * case["heads"] * case["dim"] * size
    return {"bytes": tokens * 2 * case["kv_heads"] * _row_bytes(case) + rows
            + 4 * tokens // case["page"],
            "flops": 4 * tokens * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _nearest_even(x):
    low = torch.floor(x)
    part = x - low
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(low, 2) == 1))
    return low + up.to(x.dtype)


def _values64(x, bits):
    """The values that rows of x stand for once held in `bits` bits, in 64
    bits; the scales are those the format stores (fp32 for 8 bits, fp16 for
    4), since they define the codes."""
    x = x.to(torch.float64)
    if bits == 8:
        s = (x.abs().max(dim=-1, keepdim=True).values / 127.0).to(torch.float32).to(torch.float64)
        q = _nearest_even(x / torch.where(s == 0, torch.ones_like(s), s))
        return torch.minimum(torch.maximum(q, -127.0 + 0 * q), 127.0 + 0 * q) * s, s[..., 0]
    shape = x.shape
    x = x.reshape(shape[:-1] + (shape[-1] // GROUP4, GROUP4))
    low = x.min(dim=-1, keepdim=True).values
    high = x.max(dim=-1, keepdim=True).values
    m = low.to(torch.float16).to(torch.float64)
    s = ((high - low) / 15.0).to(torch.float32).to(torch.float16).to(torch.float64)
    q = _nearest_even((x - m) / torch.where(s == 0, torch.ones_like(s), s))
    q = torch.where(q < 0, torch.zeros_like(q), torch.where(q > 15, 15 + 0 * q, q))
    return (m + torch.where(s == 0, torch.zeros_like(q), q) * s).reshape(shape), None


def _held64(codes, scales, bits):
    """The values of held codes, in 64 bits."""
    if bits == 8:
        return codes.to(torch.float64) * scales.to(torch.float64)[..., None]
    byte = codes.to(torch.int64)
    q = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device="cuda")
    q[..., 0::2] = (byte % 16).to(torch.float64)
    q[..., 1::2] = torch.div(byte, 16, rounding_mode="floor").to(torch.float64)
    s = scales.to(torch.float64).repeat_interleave(GROUP4, dim=-2)
    return s[..., 1] + s[..., 0] * q


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rows":
        values, scales = _values64(state["x"], 8)
        return {"values": values, "scales": scales}
    if case["op"] == "matmul":
        x, _ = _values64(state["x"], 8)
        y = torch.empty((case["M"], case["N"]), dtype=torch.float64, device="cuda")
        for n0 in range(0, case["N"], 2048):
            w = _held64(state["w_codes"][n0:n0 + 2048], state["w_scales"][n0:n0 + 2048], 8)
            y[:, n0:n0 + 2048] = torch.einsum("mk,nk->mn", x, w)
        return y if state["bias"] is None else y + state["bias"].to(torch.float64)
    bits, page, cache = case["bits"], case["page"], state["cache"]
    if case["op"] == "cache":
        out = []
        old = case["context"] - case["new"]
        slots = state["slots"]
        pages, rows = torch.div(slots, page, rounding_mode="floor"), torch.remainder(slots, page)
        for n in ("k", "v"):
            was = _held64(cache[n + "_codes"][pages[:old], :, rows[:old]],
                          cache[n + "_scales"][pages[:old], :, rows[:old]], bits)
            out.append(torch.cat((was, _values64(state[n], bits)[0])))
        return out
    q = state["q"].to(torch.float64)
    B, H, D = q.shape
    group = H // case["kv_heads"]
    out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        used = state["table"][b, :-(-n // page)].long()
        k, v = (_held64(cache[x + "_codes"][used], cache[x + "_scales"][used], bits)
                for x in ("k", "v"))  # [pages, Hkv, page, D]
        for h in range(case["kv_heads"]):
            kh, vh = k[:, h].reshape(-1, D)[:n], v[:, h].reshape(-1, D)[:n]
            mine = slice(h * group, (h + 1) * group)
            s = q[b, mine] @ kh.T / math.sqrt(D)
            out[b, mine] = torch.softmax(s, dim=-1) @ vh
    return out
