"""cache_attention where sizes differ widely within a sequence: scales of values
that tokens without weight carry, one token with nearly all the weight, query
channels far above the others, keys far from 0.

The bound, against 64 bits.  A query is held to 2^-22 of its largest channel
(8-bit keys; as it is with 4-bit ones), keys and sums as they are: a score is
off by
  d <= 2^-22 scale max |q| sum |k| + 2^-20 sum |scale q k| + 2^-18 (1 + sum |scale q k|)
(fp32 sums of at most 256 products, the exponent's scaling and exp2 with it),
which changes p by a factor within e^(2d).  Probabilities (with 8 bits: times
the value's scale) and 4-bit values are rounded to fp16, u = 2^-11 each, the
former above fp16's normal numbers: below them each is off by at most 2^-32 of
the largest that the sequence has (8 bits), or 2^-32 of the largest probability
times the largest value (4 bits)."""
import math

import numpy as np
import pytest
import torch

import memboost_b200 as mb
from oracle import serving
from test_gpu_cache import _np

pytestmark = pytest.mark.gpu


def _check(got, q, cache, table, lengths, scale):
    q, mirror = _np(q), serving.Cache(cache)
    heads, bits = cache.kv_heads, cache.bits
    group = q.shape[1] // heads
    u, f = 2.0 ** -11, torch.finfo(got.dtype)
    for b in range(q.shape[0]):
        for h in range(heads):
            k, v = (mirror.tokens(w, table[b], int(lengths[b]), h) for w in (0, 1))
            big = np.abs(v).max(-1)
            for j in range(h * group, (h + 1) * group):
                s = (k @ q[b, j]) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                want, weight = p @ v, p @ np.abs(v)
                reach = (np.abs(k) @ np.abs(q[b, j])).max() * abs(scale)
                d = 2.0 ** -20 * reach + 2.0 ** -18 * (1 + reach)
                if bits == 8:
                    d += 2.0 ** -22 * np.abs(k).sum(-1).max() * np.abs(q[b, j]).max() * abs(scale)
                lost = 2.0 ** -32 * len(k) * ((p * big).max() if bits == 8 else p.max() * big.max())
                work = weight * (np.exp(2 * d) * (1 + 2 * u) * (1 + 2.0 ** -16) - 1) + lost
                tol = work + f.eps / 2 * (np.abs(want) + work) + f.tiny * f.eps / 2
                err = np.abs(_np(got[b, j]) - want)
                assert np.all(err <= tol), (b, j, (err / tol).max(), err.max())


def _cache(k, v, bits, page=16):
    """One sequence's tokens in pages 0, 1, ..., and the table."""
    pages = -(-k.shape[0] // page)
    cache = mb.QuantizedCache.allocate(pages, page, k.shape[1], k.shape[2], bits=bits)
    mb.cache_write(cache, k.cuda(), v.cuda(), torch.arange(k.shape[0], device="cuda"))
    return cache, torch.arange(pages, dtype=torch.int32).unsqueeze(0)


def _attend(q, k, v, bits, scale):
    cache, table = _cache(k, v, bits)
    n = torch.tensor([k.shape[0]], dtype=torch.int32)
    got = mb.cache_attention(q.cuda(), cache, table.cuda(), n.cuda(), scale=scale)
    assert torch.isfinite(got).all()
    _check(got, q, cache, table.numpy(), n.tolist(), scale)


def _inputs(n, heads, group, dim, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((n, heads, dim), generator=g) for _ in range(2))
    return torch.randn((1, heads * group, dim), generator=g), k, v


LENGTHS = [40, 300, 3000]


@pytest.mark.parametrize("dtype,size", [(torch.float16, 15000.0), (torch.bfloat16, 1e12),
                                        (torch.bfloat16, 1e30)])
@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 12), (192, 3)])
def test_large_values_without_weight(n, dim, group, dtype, size):
    """Tokens whose probability is 0 carry values far above the others'."""
    q, k, v = _inputs(n, 2, group, dim, seed=n)
    q[..., 0], k[..., 0] = 8, 0
    some = torch.arange(n) % 7 == 3
    k[some, :, 0] = -100  # scores about -100 and -70: no weight
    v[some] *= size
    v.clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    _attend(q.to(dtype), k.to(dtype), v.to(dtype), 8, 1 / math.sqrt(dim))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("bits_ahead", [20, 27])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 12), (256, 3)])
def test_one_token_with_nearly_all_weight(n, dim, group, bits_ahead, dtype, bits):
    """The first token has 2^20 or 2^27 times the others' weight and values of
    0: the output is what the others add."""
    q, k, v = _inputs(n, 2, group, dim, seed=n)
    scale = 1 / math.sqrt(dim)
    q, k = q * 0.2, k * 0.5
    q[..., 0], k[..., 0] = 8, 0
    k[0] = 0
    k[0, :, 0] = bits_ahead * math.log(2) / (8 * scale)
    v = 1 + 0.1 * v
    v[0] = 0
    _attend(q.to(dtype), k.to(dtype), v.to(dtype), bits, scale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("n", [2, 5, 300, 3000])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 12), (192, 3)])
def test_query_channels_far_above_the_others(n, dim, group, dtype, bits):
    """One channel of the query a thousand times the others, where the keys
    have nothing."""
    if bits == 4 and dim == 192:
        dim = 160
    q, k, v = _inputs(n, 2, group, dim, seed=n)
    q[..., 5] = 1000
    k[..., 5] = 0
    if bits == 4:  # a group of its own, so that its code 0 stands for 0
        k[..., :32] = 0
    _attend(q.to(dtype), k.to(dtype), v.to(dtype), bits, 1 / math.sqrt(dim))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("n", [2, 5, 300, 3000])
@pytest.mark.parametrize("dim,group", [(32, 1), (96, 5), (128, 12), (256, 3)])
def test_keys_far_from_zero(n, dim, group, dtype, bits):
    """Each group of channels lies around 500 or -500, a few steps wide."""
    q, k, v = _inputs(n, 2, group, dim, seed=n)
    side = torch.where(torch.arange(dim) // 32 % 2 == 0, 500.0, -500.0)
    _attend(q.to(dtype), (k + side).to(dtype), v.to(dtype), bits, 1 / math.sqrt(dim))


def test_values_of_a_4_bit_cache_beyond_fp16():
    """Read back they are finite; the attention takes them as infinite.  Keys may
    be as large as the cache holds."""
    q, k, v = _inputs(70, 1, 2, 64, seed=1)
    v[33, 0, 40] = 1e5
    cache, table = _cache(k.bfloat16(), v.bfloat16(), 4)
    read = mb.cache_read(cache, torch.arange(70, device="cuda"), torch.float32)[1]
    assert torch.isfinite(read).all() and read[33, 0, 40] > 65504
    n = torch.tensor([70], dtype=torch.int32).cuda()
    got = mb.cache_attention(q.bfloat16().cuda(), cache, table.cuda(), n)
    where = ~torch.isfinite(got)
    assert where[..., 40].all() and not where[..., :32].any()
    k[..., 3] = 1e5
    _attend((q * 1e-4).bfloat16(), k.bfloat16(), torch.ones_like(v).bfloat16(), 4, 1.0)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("sign", [1, -1])
def test_queries_and_scales_near_the_end_of_fp32(sign, bits):
    """The query times the scale alone is beyond fp32: keys that make scores of a
    few, and keys of zero."""
    q, k, v = _inputs(100, 1, 2, 64, seed=2)
    q = (q / q.abs().max() * 1.9).double() * 2.0 ** 126
    small = (k.double() * 2.0 ** -137) if bits == 8 else k.double() * 0
    for keys in (small, k.double() * 0):
        _attend(q.bfloat16(), keys.bfloat16(), v.bfloat16(), bits, sign * 2.0 ** 9)


@pytest.mark.parametrize("n", [40, 3000])
def test_values_near_the_end_of_bf16(n):
    """Outputs of a size next to fp32's largest are not infinite on their way."""
    q, k, v = _inputs(n, 2, 12, 128, seed=n + 1)
    for size in (2.0 ** 105, 2.0 ** 124, 2.0 ** -66):
        _attend(q.bfloat16(), k.bfloat16(), (v.clamp(-3, 3) * size).bfloat16(), 8, 128 ** -0.5)
