"""8-bit rows, their product and the quantised cache without a GPU: what the
functions refuse, and the 64-bit oracle against definitions worked out by
hand."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import serving


def test_public_surface(mb):
    for n in ("Int8Tensor", "quantize_int8", "dequantize_int8", "int8_matmul", "QuantizedCache",
              "cache_write", "cache_read", "cache_attention"):
        assert hasattr(mb, n) and n in mb.__all__


def test_rows_oracle_by_hand():
    codes, scales = serving.quantize_rows(np.array([[127.0, 0.5, 1.5, -2.5, -127.0],
                                                    [0, 0, 0, 0, 0], [1, np.nan, 2, 3, 4],
                                                    [1, -np.inf, 2, 3, 4]]))
    assert scales[0] == 1 and codes[0].tolist() == [127, 0, 2, -2, -127]
    assert scales[1] == 0 and not codes[1].any()
    assert np.isnan(scales[2:]).all() and not codes[2:].any()


def test_groups_oracle_by_hand():
    x = np.zeros(64)
    x[:32] = np.arange(32) / 2  # min 0, max 15.5
    x[32:] = -3.0               # one value: scale 0
    codes, groups = serving.quantize_groups(x)
    s = np.float16(15.5 / 15)
    assert groups[0].tolist() == [s, 0] and groups[1].tolist() == [0, -3]
    assert codes[16:].sum() == 0 and codes[15] >> 4 == 15
    assert (serving.dequantize_groups(codes, groups)[32:] == -3).all()


def test_oracle_attention_uniform(mb):
    cache = mb.QuantizedCache.allocate(3, 16, 1, 16, device="cpu")
    c = serving.Cache(cache)
    k = np.zeros((2, 1, 16))
    v = np.stack([np.full((1, 16), 1.27), np.full((1, 16), 2.54)])
    c.write(k, v, [32, 33])
    out, *_ = serving.attention(np.ones((1, 1, 16)), c, np.array([[2]]), [2], 1.0)
    assert np.allclose(out, 1.905, atol=1e-6)
    assert (serving.attention(np.ones((1, 1, 16)), c, np.array([[2]]), [0], 1.0)[0] == 0).all()


@pytest.mark.parametrize("bits,dim", [(8, 80), (4, 96)])
def test_cache_fields(mb, bits, dim):
    c = mb.QuantizedCache.allocate(5, 32, 3, dim, bits=bits, device="cpu")
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim, c.bits) == (5, 32, 3, dim, bits)
    per_row = dim + 4 if bits == 8 else dim // 2 + dim // 32 * 4
    assert c.nbytes == 2 * 5 * 32 * 3 * per_row


@pytest.mark.parametrize("args,msg", [
    ((5, 32, 3, 64, 2), "bits must be 8 or 4"), ((5, 24, 3, 64, 8), "multiple of 16"),
    ((5, 0, 3, 64, 8), "multiple of 16"), ((5, 16, 3, 72, 8), "head_dim must be a multiple of 16"),
    ((5, 16, 3, 80, 4), "head_dim must be a multiple of 32"),
    ((5, 16, 3, 288, 8), "up to 256"), ((0, 16, 3, 64, 8), "pages and kv_heads"),
    ((5, 16, 0, 64, 8), "pages and kv_heads"),
])
def test_cache_allocation_refusals(mb, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        mb.QuantizedCache.allocate(*args, device="cpu")


def test_rows_begin_on_16_bytes():
    from memboost_b200.formats import int8_rows
    t = int8_rows(3, 33, "cpu")
    assert tuple(t.shape) == (3, 33) and t.stride() == (48, 1)


def test_refused_without_cuda(mb):
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        mb.quantize_int8(torch.zeros(2, 16))
    with pytest.raises(RuntimeError, match="x must be float16 or bfloat16 or float32"):
        mb.quantize_int8(torch.zeros(2, 16, dtype=torch.float64))
    t = mb.Int8Tensor(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2))
    with pytest.raises(RuntimeError, match="codes must be on CUDA"):
        mb.dequantize_int8(t)
    with pytest.raises(RuntimeError, match="w.codes must be on CUDA"):
        mb.int8_matmul(torch.zeros(2, 16), t)
    with pytest.raises(RuntimeError, match="2D int8"):
        mb.dequantize_int8(mb.Int8Tensor(torch.zeros(2, 16), torch.zeros(2)))
    cache = mb.QuantizedCache.allocate(1, 16, 1, 64, device="cpu")
    slots = torch.zeros(1, dtype=torch.int64)
    kv = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="k_codes must be on CUDA"):
        mb.cache_write(cache, kv, kv, slots)
    with pytest.raises(RuntimeError, match="k_codes must be on CUDA"):
        mb.cache_read(cache, slots)
    with pytest.raises(RuntimeError, match="k_codes must be on CUDA"):
        mb.cache_attention(kv, cache, torch.zeros(1, 1, dtype=torch.int32),
                           torch.zeros(1, dtype=torch.int32))


def _c():
    from memboost_b200 import _C
    return _C


P = 1 << 20  # a pointer that no refused call touches


def _refused(status, words):
    C = _c()
    assert status in (1, 3), C._lib.mb_last_error()
    assert words.encode() in C._lib.mb_last_error(), C._lib.mb_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(x=None), "null"), (dict(t=3), "unknown type"), (dict(rows=0), "positive"),
    (dict(K=-1), "positive"), (dict(cs=31), "codes_stride must be at least"),
    (dict(cs=40), "16-byte"), (dict(codes=P + 8), "16-byte"), (dict(x=P + 1), "misaligned"),
    (dict(rows=1 << 31), "too many rows"), (dict(xs=-32), "x_stride must not be negative"),
])
def test_quantize_entry_refusals(change, words):
    a = dict(x=P, t=0, rows=2, K=32, xs=32, codes=P, cs=32, scales=P)
    a.update(change)
    _refused(_c()._lib.mb_int8_quantize(a["x"], a["t"], a["rows"], a["K"], a["xs"], a["codes"],
                                        a["cs"], a["scales"], None), words)


@pytest.mark.parametrize("change,words", [
    (dict(out=None), "null"), (dict(t=-1), "unknown type"), (dict(K=0), "positive"),
    (dict(os=16), "strides"), (dict(codes=P + 1), "16-byte"), (dict(out=P + 1), "misaligned"),
])
def test_dequantize_entry_refusals(change, words):
    a = dict(codes=P, cs=32, scales=P, rows=2, K=32, out=P, t=1, os=32)
    a.update(change)
    _refused(_c()._lib.mb_int8_dequantize(a["codes"], a["cs"], a["scales"], a["rows"], a["K"],
                                          a["out"], a["t"], a["os"], None), words)


@pytest.mark.parametrize("change,words", [
    (dict(a=None), "null"), (dict(ot=7), "unknown type"), (dict(bias=P, bt=7), "unknown type"),
    (dict(M=0), "positive"), (dict(K=131073, cs=131088), "exact"), (dict(cs=16), "strides"),
    (dict(cs=40), "16-byte"), (dict(b=P + 4), "16-byte"), (dict(os=3), "strides"),
    (dict(out=P + 1), "misaligned"), (dict(N=1 << 31, os=1 << 31), "too large"),
])
def test_matmul_entry_refusals(change, words):
    a = dict(a=P, cs=32, M=2, b=P, N=4, K=32, bias=None, bt=0, out=P, ot=0, os=4)
    a.update(change)
    _refused(_c()._lib.mb_int8_matmul(a["a"], a["cs"], P, a["M"], a["b"], a["cs"], P, a["N"],
                                      a["K"], a["bias"], a["bt"], a["out"], a["ot"], a["os"],
                                      None), words)


def test_linear_entry_refusals():
    lib = _c()._lib
    n = lib.mb_int8_linear_workspace_size(3, 33)
    assert n == 3 * (48 + 4) and lib.mb_int8_linear_workspace_size(0, 33) == 0

    def call(x=P, t=0, M=3, K=33, b=P, ws=P, nbytes=n, out=P):
        return lib.mb_int8_linear(x, t, 33, M, b, 48, P, 4, K, None, 0, out, 0, 4, ws, nbytes, None)

    _refused(call(M=0), "positive")
    _refused(call(K=131073), "exact")
    _refused(call(nbytes=n - 1), "workspace")
    _refused(call(ws=None), "workspace")
    _refused(call(ws=P + 8), "workspace")
    _refused(call(x=None), "null")
    _refused(call(t=5), "unknown type")


CACHE = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, pages=4, page_size=16, kv_heads=2,
             head_dim=64, bits=8)


@pytest.mark.parametrize("change,words", [
    (dict(k_codes=None), "null"), (dict(v_scales=P + 4), "16-byte"), (dict(bits=3), "bits"),
    (dict(pages=0), "positive"), (dict(page_size=24), "multiple of 16"),
    (dict(head_dim=72), "multiple of 16"), (dict(bits=4, head_dim=80), "multiple of 32"),
    (dict(head_dim=272), "up to 256"), (dict(pages=1 << 28), "too many slots"),
])
def test_cache_refused_by_every_entry(change, words):
    C = _c()
    c = C.KVCache(**dict(CACHE, **change))
    r = ctypes.byref(c)
    _refused(C._lib.mb_cache_write(r, P, 128, 64, P, 128, 64, 0, 1, P, None, 0, None), words)
    _refused(C._lib.mb_cache_read(r, P, 1, P, P, 0, None), words)
    _refused(C._lib.mb_cache_attention(r, P, 128, 64, 0, 1, 2, P, 1, 1, P, 1.0, P, None, 0, None),
             words)


def test_cache_entry_refusals():
    C = _c()
    r = ctypes.byref(C.KVCache(**CACHE))
    w, rd, at = C._lib.mb_cache_write, C._lib.mb_cache_read, C._lib.mb_cache_attention
    _refused(w(r, None, 128, 64, P, 128, 64, 0, 1, P, None, 0, None), "null")
    _refused(w(r, P, 128, 64, P, 128, 64, 2, 1, P, None, 0, None), "fp16 or bf16")
    _refused(w(r, P, 128, 64, P, 128, 64, 0, 0, P, None, 0, None), "positive")
    _refused(w(r, P, 128, 64, P, 128, 64, 0, 1 << 40, P, None, 0, None), "too many tokens")
    _refused(w(r, P, 128, 64, P, 128, 64, 0, 50000, P, None, 0, None), "workspace")
    n = C._lib.mb_cache_write_workspace_size(50000)
    _refused(w(r, P, 128, 64, P, 128, 64, 0, 50000, P, P, n - 1, None), "workspace")
    _refused(rd(r, P, 1, P + 2, P, 0, None), "aligned")
    _refused(rd(r, P, 1, P, P, 9, None), "unknown type")
    _refused(at(r, P, 128, 64, 2, 1, 2, P, 1, 1, P, 1.0, P, None, 0, None), "fp16 or bf16")
    _refused(at(r, P, 128, 64, 0, 1, 3, P, 1, 1, P, 1.0, P, None, 0, None), "multiple of kv_heads")
    _refused(at(r, P, 128, 64, 0, 0, 2, P, 1, 1, P, 1.0, P, None, 0, None), "batch")
    _refused(at(r, P, 128, 64, 0, 1, 2, P, 1, -1, P, 1.0, P, None, 0, None), "table_width")
    _refused(at(r, P, 128, 64, 0, 1, 2, None, 1, 1, P, 1.0, P, None, 0, None), "null")
    _refused(at(r, P, 128, 64, 0, 1, 2, P, 1, 1, P, float("inf"), P, None, 0, None), "finite")


def test_calls_leave_the_unusual_alone(mb):
    """The native form of the calls takes ordinary CUDA tensors only; it
    returns None, and does nothing, for all else."""
    from memboost_b200 import _calls
    x = torch.zeros(2, 16)
    codes, scales = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    cache = mb.QuantizedCache.allocate(1, 16, 1, 64, device="cpu")
    parts = (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)
    slots = torch.zeros(1, dtype=torch.int64)
    kv = torch.zeros(1, 1, 64, dtype=torch.float16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for fn, args in ((_calls.quantize_int8, (x,)),
                     (_calls.dequantize_int8, (codes, scales, torch.float16)),
                     (_calls.int8_matmul, (x, None, codes, scales, None, None)),
                     (_calls.int8_matmul, (codes, scales, codes, scales, None, None)),
                     (_calls.cache_write, parts + (kv, kv, slots)),
                     (_calls.cache_read, parts + (slots, torch.float16)),
                     (_calls.cache_attention, parts + (kv, table, lengths, 1.0))):
        assert fn(*args) is None
        assert fn() is None and fn(*args[:-1]) is None and fn(*args, None) is None
        for i in range(len(args)):
            for other in (None, 1, "x", torch.float64, torch.zeros(0)):
                assert fn(*args[:i], other, *args[i + 1:]) is None


def test_int8_linear_refuses_an_input_that_wants_a_gradient(mb):
    from memboost_b200 import gptq
    lin = gptq.Int8Linear(mb.Int8Tensor(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)))
    x = torch.zeros(2, 16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        lin(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        lin(x * 2)
    with torch.no_grad(), pytest.raises(RuntimeError, match="w.codes must be on CUDA"):
        lin(x)
    with pytest.raises(RuntimeError, match="w.codes must be on CUDA"):
        lin(x.detach())
