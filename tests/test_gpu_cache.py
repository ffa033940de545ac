"""The quantised key/value cache on sm_100a against the 64-bit oracle.

What is written is exact (codes and scales equal the oracle's), what is read
back one rounding to fp32 and one to the output's type.  The attention's
bound: see _check_attention."""
import math

import numpy as np
import pytest
import torch

import memboost_b200 as mb
from oracle import serving

pytestmark = pytest.mark.gpu

KINDS = [(8, 16), (8, 64), (8, 80), (8, 128), (8, 192), (8, 256), (4, 32), (4, 64), (4, 96),
         (4, 128), (4, 256)]
KIND_IDS = [f"{b}bit{d}" for b, d in KINDS]


def _kv(tokens, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((tokens, heads, dim), generator=g) for _ in range(2))
    k[..., dim // 3] *= 8
    v = v * torch.exp2(torch.randint(-6, 4, (tokens, heads, 1), generator=g).float())
    return k.to(dtype).cuda(), v.to(dtype).cuda()


def _np(t):
    return t.detach().cpu().double().numpy()


def _check_fields(cache, mirror):
    for w, n in ((0, "k"), (1, "v")):
        got = getattr(cache, n + "_codes").cpu().numpy()
        assert np.array_equal(got, mirror.codes[w]), n
        assert np.array_equal(getattr(cache, n + "_scales").cpu().numpy(), mirror.scales[w],
                              equal_nan=True), n


def _check_values(got, want64):
    """One rounding to fp32 and one to the type: equal to torch's."""
    want = torch.from_numpy(want64.astype(np.float32)).to(got.dtype)
    assert torch.equal(got.cpu().nan_to_num(12345.0), want.nan_to_num(12345.0))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("bits,dim", KINDS, ids=KIND_IDS)
def test_write_and_read(bits, dim, dtype):
    heads, page = 3, 48
    cache = mb.QuantizedCache.allocate(6, page, heads, dim, bits=bits)
    mirror = serving.Cache(cache)
    k, v = _kv(37, heads, dim, dtype, seed=dim + bits)
    slots = torch.randperm(6 * page, generator=torch.Generator().manual_seed(1))[:37].cuda()
    mb.cache_write(cache, k, v, slots)
    mirror.write(_np(k), _np(v), slots.tolist())
    _check_fields(cache, mirror)
    ask = torch.cat((slots, torch.tensor([-1, 0, 6 * page, 6 * page - 1], device="cuda")))
    for out in (torch.float16, torch.bfloat16, torch.float32):
        got = mb.cache_read(cache, ask, out)
        for w in range(2):
            _check_values(got[w], mirror.read(w, ask.tolist()))


@pytest.mark.parametrize("tokens", [1, 40, 2048, 2049, 16384, 16385])
@pytest.mark.parametrize("bits", [8, 4])
def test_write_same_slot_and_outside(tokens, bits):
    """The last token of a slot stays, whatever their number; slots outside
    the cache are left out; other places stay as they were."""
    cache = mb.QuantizedCache.allocate(20, 16, 2, 64, bits=bits)
    k0, v0 = _kv(320, 2, 64, torch.float16, seed=4)
    mb.cache_write(cache, k0, v0, torch.arange(320, device="cuda"))
    mirror = serving.Cache(cache)
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randint(-20, 340, (tokens,), generator=g)
    slots[0] = 2 ** 40
    slots[-1] = 7
    k, v = _kv(tokens, 2, 64, torch.float16, seed=5)
    mb.cache_write(cache, k, v, slots.cuda())
    mirror.write(_np(k), _np(v), slots.tolist())
    _check_fields(cache, mirror)


def test_write_not_finite_and_constant():
    for bits in (8, 4):
        cache = mb.QuantizedCache.allocate(2, 16, 1, 64, bits=bits)
        mirror = serving.Cache(cache)
        k, v = _kv(8, 1, 64, torch.bfloat16, seed=6)
        k[0, 0, 5] = float("nan")
        k[1, 0, 63] = float("inf")
        k[2, 0, 0] = -float("inf")
        k[3] = 0
        k[4] = 2.5
        k[5] *= 1e5       # beyond fp16
        k[6] *= 1e-7      # below fp16's normal numbers
        v[7, 0, :32] = 100 + v[7, 0, :32] * 1e-3
        slots = torch.arange(3, 11, device="cuda")
        mb.cache_write(cache, k, v, slots)
        mirror.write(_np(k), _np(v), slots.tolist())
        _check_fields(cache, mirror)
        got = mb.cache_read(cache, slots, torch.float32)
        for w in range(2):
            _check_values(got[w], mirror.read(w, slots.tolist()))
        assert torch.isnan(got[0][0]).any() and (got[0][3] == 0).all()


def test_write_codes_next_to_borders():
    """Values half-way between codes, and an fp32 rounding away from it."""
    g = torch.Generator().manual_seed(8)
    k = torch.randint(0, 31, (200, 2, 64), generator=g).half() / 2   # halves: min 0, max 15
    k[..., 0], k[..., 1], k[..., 32], k[..., 33] = 0, 15, 0, 15
    v = torch.randint(-254, 255, (200, 2, 64), generator=g).half() / 2
    v[..., 7] = 127
    for bits in (8, 4):
        cache = mb.QuantizedCache.allocate(13, 16, 2, 64, bits=bits)
        mirror = serving.Cache(cache)
        slots = torch.arange(200, device="cuda")
        mb.cache_write(cache, k.cuda(), v.cuda(), slots)
        mirror.write(_np(k), _np(v), slots.tolist())
        _check_fields(cache, mirror)


def test_write_strided():
    """Keys and values as parts of one projection's output."""
    for bits in (8, 4):
        cache = mb.QuantizedCache.allocate(3, 16, 4, 64, bits=bits)
        mirror = serving.Cache(cache)
        g = torch.Generator().manual_seed(9)
        for width, off in ((12 * 64, 4 * 64), (12 * 64 + 5, 4 * 64 + 3)):
            qkv = torch.randn((10, width), generator=g).half().cuda()
            k = qkv[:, off:off + 256].unflatten(1, (4, 64))
            v = qkv[:, off + 256:off + 512].unflatten(1, (4, 64))
            slots = torch.arange(20, 30, device="cuda")
            mb.cache_write(cache, k, v, slots)
            mirror.write(_np(k), _np(v), slots.tolist())
            _check_fields(cache, mirror)
        kt = torch.randn((4, 10, 64), generator=g).half().cuda().transpose(0, 1)  # heads first
        kn = torch.randn((10, 64, 4), generator=g).half().cuda().transpose(1, 2)  # channels last
        mb.cache_write(cache, kt, kn, slots)
        mirror.write(_np(kt), _np(kn), slots.tolist())
        _check_fields(cache, mirror)


def test_cache_refusals():
    cache = mb.QuantizedCache.allocate(3, 16, 2, 64)
    k, v = _kv(4, 2, 64, torch.float16)
    s = torch.arange(4, device="cuda")
    q = k
    table = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    n = torch.ones(4, dtype=torch.int32, device="cuda")
    W, A = mb.cache_write, mb.cache_attention
    other = mb.QuantizedCache(cache.k_codes, cache.v_codes[:2], cache.k_scales, cache.v_scales)
    half = mb.QuantizedCache(cache.k_codes, cache.v_codes, cache.k_scales.half(), cache.v_scales)
    bent = mb.QuantizedCache(cache.k_codes.transpose(1, 2).contiguous().transpose(1, 2),
                             cache.v_codes, cache.k_scales, cache.v_scales)
    for fn, args, msg in [
        (W, (cache, k[:, :1], v, s), "k must be"), (W, (cache, k, v[:3], s), "same number"),
        (W, (cache, k, v.bfloat16(), s), "k's dtype"), (W, (cache, k.float(), v.float(), s), "k must be float16"),
        (W, (cache, k, v, s.int()), "int64"), (W, (cache, k, v, s[:3]), "slot for each token"),
        (W, (cache, k, v, s.cpu()), "device of the cache"), (W, (other, k, v, s), "v_codes must be"),
        (W, (half, k, v, s), "k_scales must be"), (W, (bent, k, v, s), "contiguous"),
        (mb.cache_read, (cache, s, torch.int8), "dtype must be"),
        (A, (q[:, :, :32], cache, table, n), "q must be"),
        (A, (q[:, :1], cache, table, n), "multiple of the cache's"),
        (A, (q.float(), cache, table, n), "q must be float16 or bfloat16"),
        (A, (q, cache, table.long(), n), "page_table must be"),
        (A, (q, cache, table[:2], n), "page_table must be"),
        (A, (q, cache, table, n.long()), "lengths must be"),
        (A, (q, cache, table, n, float("nan")), "finite"),
        (A, (q, cache, table, n, None, q.bfloat16()), "out must be"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            fn(*args)


def _filled(pages, page, heads, dim, bits, dtype=torch.float16, seed=0):
    cache = mb.QuantizedCache.allocate(pages, page, heads, dim, bits=bits)
    k, v = _kv(pages * page, heads, dim, dtype, seed)
    mb.cache_write(cache, k, v, torch.arange(pages * page, device="cuda"))
    return cache


def _check_attention(got, q, cache, table, lengths, scale):
    """The kernel may round, each to fp16 at half a step (u = 2^-11): a 4-bit
    key and value as they are read, the probabilities (and with 8 bits their
    product with the value's scale); sums, maximum and exponentials are fp32.
    A query is rounded to fp16 relative to its largest channel, or with 8-bit
    keys to 2^-14 of it.  A score s is then off by
    d <= (2 u + 2^-20) sum |scale q k| + 2^-18 (1 + |s|) (u for the key and u
    for the query; fp32 sums of at most 256 products, the exponent's scaling
    and exp2 with it), with 8 bits also by 2^-14 scale max |q| sum |k|, which
    changes p by a factor within e^(2d); p, v and p times the scale add 3 u.
    Probabilities below fp16's normal numbers are off by at most 2^-24 of the
    largest value each."""
    want, weight, reach, spread, coarse = serving.attention(
        _np(q), serving.Cache(cache), table, lengths, scale)
    u = 2.0 ** -11
    d = (2 * u + 2.0 ** -20) * reach + 2.0 ** -18 * (1 + reach)
    if cache.bits == 8:
        d = d + 2.0 ** -14 * coarse
    f = torch.finfo(got.dtype)
    work = weight * (np.exp(2 * d) * (1 + 3 * u) * (1 + 2.0 ** -16) - 1) + 2.0 ** -24 * spread
    tol = work + (f.eps / 2) * (np.abs(want) + work) + f.tiny * f.eps / 2
    err = np.abs(_np(got) - want)
    assert np.all(err <= tol), ((err - tol).max(), err.max())


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 128, 129, 200, 500, 611]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("bits,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("group", [1, 8])
def test_attention(bits, dim, group, dtype):
    _attend(bits, dim, 2, group, 48, dtype)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,group,page", [(1, 3, 16), (3, 5, 32), (1, 12, 128), (2, 16, 16),
                                              (1, 17, 64), (1, 40, 256), (5, 7, 16)])
def test_attention_head_layouts(heads, group, page, bits):
    _attend(bits, 64, heads, group, page, torch.float16)


def _attend(bits, dim, heads, group, page, dtype):
    need = [-(-n // page) for n in LENGTHS]
    pages = sum(need) + 2
    cache = _filled(pages, page, heads, dim, bits, seed=dim + group)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table = torch.full((len(LENGTHS), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    g = torch.Generator().manual_seed(3)
    q = (torch.randn((len(LENGTHS), heads * group, dim), generator=g)).to(dtype).cuda()
    n = torch.tensor(LENGTHS, dtype=torch.int32)
    got = mb.cache_attention(q, cache, table.cuda(), n.cuda())
    _check_attention(got, q, cache, table.numpy(), LENGTHS, 1 / math.sqrt(dim))
    assert (got[0] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("batch,longest", [(1, 5000), (3, 20000), (40, 900)])
def test_attention_long(batch, longest, bits):
    page, heads, dim, group = 64, 2, 128, 4
    lengths = [max(1, longest - 37 * b * b) for b in range(batch)]
    need = [-(-n // page) for n in lengths]
    cache = _filled(sum(need), page, heads, dim, bits, seed=1)
    table = torch.zeros((batch, max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randn((batch, heads * group, dim), generator=torch.Generator().manual_seed(1))
    q = (q * 3).half().cuda()  # a few tokens carry most of the weight
    got = mb.cache_attention(q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    _check_attention(got, q, cache, table.numpy(), lengths, 1 / math.sqrt(dim))


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_bad_pages_lengths_and_stale_places(bits):
    """Pages outside the cache are left out, lengths beyond the table count as
    the table's, negative ones as none, and what lies behind a sequence's end
    is never used."""
    cache = _filled(12, 16, 2, 64, bits, seed=5)
    table = torch.tensor([[3, -1, 5, 99], [-7, 2 ** 30, -1, 12], [0, 1, 2, 3], [4, 5, 6, 7],
                          [8, 8, 8, 8], [9, 10, 11, 0]], dtype=torch.int32)
    lengths = [60, 64, 10 ** 6, -5, 50, 41]
    last = mb.QuantizedCache(*(t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales,
                                                    cache.v_scales)))
    for t in (last.k_scales, last.v_scales):
        t[11, :, 9:] = float("nan")  # behind the last sequence's 41 tokens
        t[0] = float("nan")
    table[2, 0] = 7
    q = torch.randn((6, 6, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    got = mb.cache_attention(q, last, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    _check_attention(got, q, cache, table.numpy(), lengths, 0.125)
    assert (got[1] == 0).all() and (got[3] == 0).all()
    # a NaN that is seen is not lost
    seen = mb.cache_attention(q, last, table.cuda(),
                              torch.tensor([60, 64, 64, 0, 50, 42], dtype=torch.int32).cuda())
    assert torch.isnan(seen[5]).all() and torch.isfinite(seen[:5]).all()


def test_attention_extreme_sizes_of_values():
    """Value scales from tiny to large in one sequence, scores of hundreds,
    zero keys, zero queries, a scale of zero."""
    for bits in (8, 4):
        cache = mb.QuantizedCache.allocate(8, 16, 1, 64, bits=bits)
        k, v = _kv(128, 1, 64, torch.bfloat16, seed=7)
        e = torch.randint(-14, 12, (128, 1, 1), generator=torch.Generator().manual_seed(2))
        v = (v * torch.exp2(e.float()).cuda()).bfloat16()
        k[3] = 0
        v[4] = 0
        mb.cache_write(cache, k, v, torch.arange(128, device="cuda"))
        table = torch.arange(8, dtype=torch.int32).unsqueeze(0).repeat(4, 1)
        q = torch.randn((4, 3, 64), generator=torch.Generator().manual_seed(1)).bfloat16()
        q[1] *= 100
        q[2] = 0
        q[3] *= 1e-30
        q = q.cuda()
        n = torch.full((4,), 125, dtype=torch.int32)
        for scale in (0.125, 0.0, -0.5):
            got = mb.cache_attention(q, cache, table.cuda(), n.cuda(), scale=scale)
            _check_attention(got, q, cache, table.numpy(), n.tolist(), scale)


def test_attention_queries_at_the_ends_of_bf16():
    """Queries up to the largest bf16 numbers and down to the smallest, with a
    scale that makes scores of ordinary size; one that is not finite."""
    for bits in (8, 4):
        cache = _filled(4, 16, 1, 64, bits, seed=9)
        table = torch.arange(4, dtype=torch.int32).unsqueeze(0).repeat(6, 1)
        g = torch.Generator().manual_seed(4)
        base = torch.randn((6, 2, 64), generator=g)
        n = torch.full((6,), 60, dtype=torch.int32)
        for exponent in (127, 126, 125, 100, -100, -115, -125, -132):
            q = (base / base.abs().amax(-1, keepdim=True) * 1.9).double() * 2.0 ** exponent
            q = q.bfloat16().cuda()
            scale = float(np.float32(2.0 ** min(-exponent, 127)))
            got = mb.cache_attention(q, cache, table.cuda(), n.cuda(), scale=scale)
            if exponent >= -118:  # below, the query's rounding is not relative to itself
                _check_attention(got, q, cache, table.numpy(), n.tolist(), scale)
            assert torch.isfinite(got).all()
        q[1, 1, 5], q[2, 0, 7] = float("nan"), float("inf")
        got = mb.cache_attention(q, cache, table.cuda(), n.cuda())
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[1, 1], bad[2, 0] = True, True
        assert torch.equal(torch.isnan(got), bad)


def test_attention_values_that_are_all_zero():
    for bits in (8, 4):
        cache = mb.QuantizedCache.allocate(4, 16, 1, 64, bits=bits)
        q = torch.ones((1, 1, 64), dtype=torch.float16, device="cuda")
        table = torch.arange(4, dtype=torch.int32, device="cuda").unsqueeze(0)
        got = mb.cache_attention(q, cache, table, torch.tensor([50], dtype=torch.int32).cuda())
        assert (got == 0).all()


def test_attention_strided_and_out():
    cache = _filled(6, 16, 2, 64, 8, seed=5)
    wide = torch.randn((3, 9, 64), generator=torch.Generator().manual_seed(1)).half().cuda()
    q = wide[:, 2:8]
    table = torch.arange(12, dtype=torch.int32).view(3, 4).cuda() % 6
    n = torch.tensor([20, 31, 32], dtype=torch.int32, device="cuda")
    want = mb.cache_attention(q.contiguous(), cache, table[:, :2].contiguous(), n)
    assert torch.equal(mb.cache_attention(q, cache, table[:, :2], n), want)
    assert torch.equal(mb.cache_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache,
                                          table, n), want)
    out = torch.full((5, 6, 64), 7.0, dtype=torch.float16, device="cuda")
    mb.cache_attention(q, cache, table, n, out=out[1:4])
    assert torch.equal(out[1:4], want) and (out[0] == 7).all() and (out[4] == 7).all()
    assert mb.cache_attention(q[:0], cache, table[:0], n[:0]).shape == (0, 6, 64)
    empty = mb.cache_attention(q, cache, table[:, :0], n)
    assert (empty == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_same_result_every_time(bits):
    cache = _filled(64, 64, 2, 128, bits, seed=5)
    q = torch.randn((2, 16, 128), generator=torch.Generator().manual_seed(1)).half().cuda()
    table = torch.arange(64, dtype=torch.int32).view(2, 32).cuda()
    n = torch.tensor([2048, 1777], dtype=torch.int32, device="cuda")
    first = mb.cache_attention(q, cache, table, n)
    for _ in range(20):
        assert torch.equal(mb.cache_attention(q, cache, table, n), first)


@pytest.mark.parametrize("bits", [8, 4])
def test_two_graphs_and_streams(bits):
    """Writing a token and attending to it, captured twice over one cache,
    replayed with new tokens and lengths, and on two streams at once."""
    page, heads, dim, group, pages = 16, 2, 64, 4, 80
    cache = _filled(pages, page, heads, dim, bits, seed=5)
    table = torch.arange(pages, dtype=torch.int32).view(2, 40).cuda()

    def step(k, v, q, slots, n):
        mb.cache_write(cache, k, v, slots)
        return mb.cache_attention(q, cache, table, n)

    g = torch.Generator().manual_seed(6)
    ins, graphs = [], []
    for i in range(2):  # graph i owns places 500 + i of both sequences
        k, v = _kv(2, heads, dim, torch.float16, seed=i)
        q = torch.randn((2, heads * group, dim), generator=g).half().cuda()
        slots = torch.tensor([500 + i, 40 * page + 500 + i], device="cuda")
        n = torch.tensor([499, 300], dtype=torch.int32, device="cuda")
        ins.append((k, v, q, slots, n))
        step(*ins[-1])
    torch.cuda.synchronize()
    for a in ins:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = step(*a)
        graphs.append((gr, y))
    for rounds in range(3):
        for i, a in enumerate(ins):
            a[2].copy_(torch.randn(a[2].shape, generator=g).half())
            a[4].fill_(100 * rounds + 30 + i)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for a, (_, y) in zip(ins, graphs):
            assert torch.equal(y, mb.cache_attention(a[2], cache, table, a[4]))
            _check_attention(y, a[2], cache, table.cpu().numpy(), a[4].tolist(), 0.125)


@pytest.mark.parametrize("bits", [8, 4])
def test_offsets_past_32_bits(bits):
    """A cache whose codes take more than 4 GB: its last pages."""
    page, heads, dim = 256, 8, 256
    pages = (9 << 29) // (heads * page * dim * bits // 8) + 1  # 4.5 GB a side
    cache = mb.QuantizedCache.allocate(pages, page, heads, dim, bits=bits)
    assert cache.k_codes.nbytes > 1 << 32
    n = 300
    slots = torch.arange(pages * page - n, pages * page, device="cuda")
    slots[0] = 5
    k, v = _kv(n, heads, dim, torch.float16, seed=3)
    mb.cache_write(cache, k, v, slots)
    got = mb.cache_read(cache, slots, torch.float32)
    for x, y in zip((k, v), got):
        codes, scales = serving.encode(_np(x), bits)
        _check_values(y, serving.values(codes, scales, bits))
    q = torch.randn((1, heads, dim), generator=torch.Generator().manual_seed(1)).half().cuda()
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    last = mb.QuantizedCache(*(t[-1:].clone() for t in (cache.k_codes, cache.v_codes,
                                                        cache.k_scales, cache.v_scales)))
    m = torch.tensor([256], dtype=torch.int32, device="cuda")
    out = mb.cache_attention(q, cache, table, m)
    assert torch.equal(out, mb.cache_attention(q, last, table * 0, m))
    _check_attention(out, q, last, np.zeros((1, 1), np.int32), [256], 1 / 16)


@pytest.mark.parametrize("bits", [8, 4])
def test_every_way_into_a_cache_call_agrees(bits):
    """Strided keys, slots, tables, lengths and queries, subclasses and given
    outputs: what the cache holds and the attention are the same."""
    cache, other = (mb.QuantizedCache.allocate(5, 16, 2, 64, bits=bits) for _ in range(2))
    k, v = _kv(70, 2, 64, torch.float16, seed=3)
    slots = torch.randperm(80, generator=torch.Generator().manual_seed(1))[:70].cuda()
    mb.cache_write(cache, k, v, slots)
    mb.cache_write(other, torch.stack([k, v], -1)[..., 0], torch.nn.Parameter(v),
                   torch.stack([slots, slots], 1)[:, 0])
    for a, b in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales),
                    (other.k_codes, other.v_codes, other.k_scales, other.v_scales)):
        assert torch.equal(a, b)
    read = mb.cache_read(cache, slots)
    again = mb.cache_read(cache, torch.stack([slots, slots], 1)[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(read, again))
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(2)).half().cuda()
    table = torch.tensor([[0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [2, 2, 2, 2, 2]], dtype=torch.int32).cuda()
    lengths = torch.tensor([80, 33, 0], dtype=torch.int32).cuda()
    want = mb.cache_attention(q, cache, table, lengths)
    out = torch.empty_like(want)
    for args in ((q, cache, table, lengths, 0.125, out),
                 (torch.stack([q, q], -1)[..., 0], cache, table, lengths),
                 (torch.nn.Parameter(q), cache, table, lengths),
                 (q, cache, table.t().contiguous().t(), torch.stack([lengths, lengths], 1)[:, 0]),
                 (q, cache, table, lengths, torch.tensor(0.125).item()),
                 (torch.stack([q, q], 1)[:, 0], cache, table, lengths)):
        got = mb.cache_attention(*args)
        assert torch.equal(got, want) and not got.requires_grad
    assert torch.equal(mb.cache_attention(q, cache, table, lengths, 0),
                       mb.cache_attention(q, cache, table, lengths, 0.0))
