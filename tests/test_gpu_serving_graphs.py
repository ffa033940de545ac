"""The 8-bit and cache calls behind what is no kernel, and across streams: each
kernel is set up while the one before it in the stream ends, so its inputs
coming from a copy, a fill, another stream or another graph are looked at by
themselves."""
import pytest
import torch

import memboost_b200 as mb

pytestmark = pytest.mark.gpu


class _Step:
    """A layer's calls on buffers of their own: x quantised, multiplied, its
    product stored as keys and values, attended to and read back."""

    def __init__(self, seed, tokens=24, big=False):
        g = torch.Generator().manual_seed(seed)
        n = 4096 if big else 256
        self.w = mb.quantize_int8((torch.randn((2 * 2 * 64, n), generator=g) / 16).half().cuda())
        self.x = torch.zeros((tokens, n), dtype=torch.float16, device="cuda")
        self.slots = torch.zeros(tokens, dtype=torch.int64, device="cuda")
        self.table = torch.zeros((tokens, 40), dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        self.cache = mb.QuantizedCache.allocate(40, 16, 2, 64, bits=8)
        self.held = mb.QuantizedCache.allocate(40, 16, 2, 64, bits=4)

    def inputs(self, seed):
        g = torch.Generator().manual_seed(seed)
        t = self.x.shape[0]
        return (torch.randn(self.x.shape, generator=g).half().cuda(),
                torch.randperm(640, generator=g)[:t].cuda(),
                torch.randint(0, 40, self.table.shape, generator=g, dtype=torch.int32).cuda(),
                torch.randint(0, 641, (t,), generator=g, dtype=torch.int32).cuda())

    def buffers(self):
        return self.x, self.slots, self.table, self.lengths

    def run(self):
        kv = mb.int8_matmul(self.x, self.w).view(-1, 2, 2, 64)
        mb.cache_write(self.cache, kv[:, 0], kv[:, 1], self.slots)
        mb.cache_write(self.held, kv[:, 1], kv[:, 0], self.slots)
        out = [mb.cache_attention(kv[:, 0], c, self.table, self.lengths)
               for c in (self.cache, self.held)]
        read = mb.cache_read(self.cache, self.slots) + mb.cache_read(self.held, self.slots)
        codes = mb.quantize_int8(out[0].flatten(1))
        return [kv, *out, *read, codes.codes, codes.scales, mb.dequantize_int8(codes)]

    def expected(self, values):
        """Each call by itself, the GPU waited for between them."""
        self.cache.k_codes.zero_(), self.cache.v_codes.zero_()
        self.cache.k_scales.zero_(), self.cache.v_scales.zero_()
        for t in (self.held.k_codes, self.held.v_codes, self.held.k_scales, self.held.v_scales):
            t.zero_()
        for to, value in zip(self.buffers(), values):
            to.copy_(value)
        torch.cuda.synchronize()
        calls = {n: getattr(mb, n) for n in ("int8_matmul", "cache_write", "cache_attention",
                                             "cache_read", "quantize_int8", "dequantize_int8")}
        try:
            for name, fn in calls.items():
                def waited(*args, _fn=fn, **kwargs):
                    got = _fn(*args, **kwargs)
                    torch.cuda.synchronize()
                    return got
                setattr(mb, name, waited)
            return [t.clone() for t in self.run()]
        finally:
            for name, fn in calls.items():
                setattr(mb, name, fn)


def _equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("big", [False, True])
def test_captured_behind_copies_and_fills(big):
    step = _Step(1, big=big)
    first, second = step.inputs(2), step.inputs(3)
    staged = [t.clone() for t in first]
    want = [step.expected(v) for v in (first, second)]
    for t in (step.cache, step.held):
        for part in (t.k_codes, t.v_codes, t.k_scales, t.v_scales):
            part.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for to in step.buffers():
            to.zero_()
        step.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in (step.cache, step.held):
            for part in (c.k_codes, c.v_codes, c.k_scales, c.v_scales):
                part.zero_()
        for to, value in zip(step.buffers(), staged):
            to.copy_(value)
        got = step.run()
    for values, expected in ((first, want[0]), (second, want[1]), (first, want[0])):
        for to, value in zip(staged, values):
            to.copy_(value)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(got, expected)


def test_inputs_written_on_another_stream():
    step = _Step(4)
    values = [step.inputs(s) for s in (5, 6, 7)]
    want = [step.expected(v) for v in values]
    writer = torch.cuda.Stream()
    for _ in range(5):
        for v, expected in zip(values, want):
            writer.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(writer):
                for c in (step.cache, step.held):
                    for part in (c.k_codes, c.v_codes, c.k_scales, c.v_scales):
                        part.zero_()
                torch.mm(torch.ones((2048, 2048), device="cuda"), torch.ones((2048, 2048), device="cuda"))
                for to, value in zip(step.buffers(), v):
                    to.copy_(value)
            torch.cuda.current_stream().wait_stream(writer)
            assert _equal(step.run(), expected)


def test_calls_back_to_back_on_the_same_buffers():
    """Outputs of one call are inputs of the next, whose kernel is set up before
    they are written; weights too are made right before their product."""
    g = torch.Generator().manual_seed(8)
    w = (torch.randn((512, 512), generator=g) / 24).half().cuda()
    x = torch.randn((40, 512), generator=g).half().cuda()
    want = x
    for _ in range(20):
        a, b = mb.quantize_int8(want), mb.quantize_int8(w)
        torch.cuda.synchronize()
        want = mb.int8_matmul(a, b)
        torch.cuda.synchronize()
    for _ in range(5):
        y = x
        for _ in range(20):
            y = mb.int8_matmul(y, mb.quantize_int8(w))
        assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x
        for _ in range(20):
            y = mb.int8_matmul(mb.quantize_int8(y), mb.quantize_int8(w))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
