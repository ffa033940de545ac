"""cache_attention over batches whose sequences without tokens lie anywhere:
first, in the middle, next to each other, last.  A CTA that takes several
sequences in turn has to pass those without tokens and begin the next at its
first token."""
import math

import pytest
import torch

import memboost_b200 as mb
from test_gpu_cache import _check_attention, _filled

pytestmark = pytest.mark.gpu

# batch, longest, kv_heads, query heads a kv_head, head_dim: many units a CTA, an
# eighth of one, and tables short enough that a CTA takes a row
SHAPES = [(16, 2048, 32, 1, 128), (24, 3000, 8, 8, 64), (32, 1000, 8, 12, 64), (40, 700, 2, 1, 96),
          (300, 90, 2, 1, 32), (200, 200, 8, 1, 32)]


def _lengths(batch, longest, where):
    n = [1 + (longest - 1) * ((7 * i) % 11) // 10 for i in range(batch)]
    n[0] = longest
    for i, x in where(batch).items():
        n[i] = x
    return n


WHERE = {
    "first": lambda b: {0: 0},
    "middle": lambda b: {b // 3: 0, 2 * b // 3: 0},
    "pairs": lambda b: {i: 0 for i in (b // 4, b // 4 + 1, b // 2, b // 2 + 1, b // 2 + 2)},
    "negative": lambda b: {1: -1, b // 2: -2 ** 31, b - 2: -7},
    "last": lambda b: {b - 1: 0},
    "all but one": lambda b: {i: 0 for i in range(b) if i != b // 2},
    "all": lambda b: {i: 0 for i in range(b)},
}


@pytest.mark.parametrize("where", WHERE, ids=[w.replace(" ", "-") for w in WHERE])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("batch,longest,heads,group,dim", SHAPES)
def test_sequences_without_tokens(batch, longest, heads, group, dim, bits, where):
    page = 64
    lengths = _lengths(batch, longest, WHERE[where])
    pages = 40  # shared by the sequences
    cache = _filled(pages, page, heads, dim, bits, seed=batch + bits)
    width = -(-longest // page)
    g = torch.Generator().manual_seed(longest)
    table = torch.randint(0, pages, (batch, width), generator=g, dtype=torch.int32)
    q = torch.randn((batch, heads * group, dim), generator=g).half().cuda()
    n = torch.tensor(lengths, dtype=torch.int32)
    got = mb.cache_attention(q, cache, table.cuda(), n.cuda())
    _check_attention(got, q, cache, table.numpy(), lengths, 1 / math.sqrt(dim))
    assert all((got[b] == 0).all() for b in range(batch) if lengths[b] <= 0)


@pytest.mark.parametrize("bits", [8, 4])
def test_replayed_with_other_sequences_empty(bits):
    """A captured call takes the lengths as they are when it is replayed."""
    batch, longest, heads, dim, page = 16, 2048, 32, 64, 64
    cache = _filled(40, page, heads, dim, bits, seed=bits)
    g = torch.Generator().manual_seed(bits)
    table = torch.randint(0, 40, (batch, longest // page), generator=g, dtype=torch.int32)
    q = torch.randn((batch, heads, dim), generator=g).half().cuda()
    table_, n = table.cuda(), torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    mb.cache_attention(q, cache, table_, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mb.cache_attention(q, cache, table_, n)
    for where in WHERE.values():
        lengths = _lengths(batch, longest, where)
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(got, q, cache, table.numpy(), lengths, 1 / math.sqrt(dim))
