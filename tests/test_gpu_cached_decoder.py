"""The 8-bit projections and the quantised cache in the decoder that uses them:
prompts in chunks (with padding), then single tokens.  What each layer's cache
holds equals the oracle's encoding of the keys and values the layer computed,
and the attention of single tokens lies within its bound of the 64-bit one."""
import math

import numpy as np
import pytest
import torch

import memboost_b200 as mb
from memboost_b200 import llama
from oracle import serving
from test_gpu_cache import _check_attention, _check_fields

pytestmark = pytest.mark.gpu

CFG = llama.LlamaConfig(n_embd=256, n_layer=2, n_head=4, n_kv_heads=2, n_inner=512)


def _layers(cfg, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {f"layers.{i}.{name}": mb.quantize(
        (torch.randn(llama.projection_shape(cfg, name), generator=g) * 0.06).half().cuda())
        for i in range(cfg.n_layer) for name in llama.PROJECTIONS}


class _Capture(dict):
    """Keeps what block_forward hands over, and works out the layer's rotated
    query, key and value with the same operations."""

    def __init__(self, cfg, linear):
        super().__init__(attn=self.attn, o=self.o, mlp=lambda x: None, down=lambda x: None)
        self.cfg, self.linear = cfg, linear

    def attn(self, x):
        self.x = x

    def o(self, y):
        self.y = y

    def qkv(self, cos, sin, positions):
        B, T, _ = self.x.shape
        hd = self.cfg.n_embd // self.cfg.n_head
        out = []
        for name, heads in (("q", self.cfg.n_head), ("k", self.cfg.n_kv_heads),
                            ("v", self.cfg.n_kv_heads)):
            t = self.linear[f"self_attn.{name}_proj"](self.x).view(B, T, heads, hd)
            if name != "v":
                t = llama._rotate(t.transpose(1, 2), cos, sin, positions).transpose(1, 2)
            out.append(t)
        return out


@pytest.mark.parametrize("bits", [8, 4])
def test_prompt_chunks_and_tokens(bits):
    layers = _layers(CFG)
    B, hd = 3, CFG.n_embd // CFG.n_head
    dec = llama.CachedDecoder(CFG, layers, batch=B, max_tokens=150, page_size=48, bits=bits)
    assert dec.max_tokens == 192
    mirrors = [serving.Cache(c) for c in dec.caches]
    g = torch.Generator().manual_seed(1)
    lengths = np.zeros(B, np.int64)
    for T, counts in ((70, [70, 33, 1]), (20, [20, 20, 3])) + ((1, [1, 1, 1]),) * 4:
        x = torch.randn((B, T, CFG.n_embd), generator=g).half().cuda()
        caps = [_Capture(CFG, lin) for lin in dec.linears]
        tokens = None if T == 1 else torch.tensor(counts, dtype=torch.int32, device="cuda")
        y = dec(x, tokens, capture=caps)
        assert y.shape == x.shape and torch.isfinite(y).all()
        positions = torch.from_numpy(lengths[:, None] + np.arange(T)).cuda()
        for cap, cache, mirror in zip(caps, dec.caches, mirrors):
            q, k, v = cap.qkv(dec.cos, dec.sin, positions)
            for b in range(B):
                n = counts[b]
                at = positions[b, :n].cpu().numpy()
                slots = dec.page_table[b].cpu().numpy()[at // 48].astype(np.int64) * 48 + at % 48
                mirror.write(k[b, :n].double().cpu().numpy(), v[b, :n].double().cpu().numpy(),
                             slots)
            _check_fields(cache, mirror)
            if T == 1:
                _check_attention(cap.y.view(B, CFG.n_head, hd), q[:, 0], cache,
                                 dec.page_table.cpu().numpy(), lengths + 1, 1 / math.sqrt(hd))
        lengths += np.array(counts)
        assert dec.lengths.tolist() == lengths.tolist()


def test_chunk_behind_another_reads_the_cache():
    """A second chunk attends to what the cache holds: its attention equals a
    product with the oracle's values of all tokens, to the rounding of a
    16-bit attention (scores and sums in fp32, probabilities and output in
    16 bits: a few half steps of 2^-11 on sums of weights 1)."""
    layers = _layers(CFG, seed=3)
    dec = llama.CachedDecoder(CFG, layers, batch=1, max_tokens=64, page_size=16, n_layers=1)
    g = torch.Generator().manual_seed(2)
    dec(torch.randn((1, 21, CFG.n_embd), generator=g).half().cuda())
    cap = _Capture(CFG, dec.linears[0])
    dec(torch.randn((1, 10, CFG.n_embd), generator=g).half().cuda(), capture=[cap])
    positions = torch.arange(21, 31, device="cuda")[None]
    q, _, _ = cap.qkv(dec.cos, dec.sin, positions)
    mirror = serving.Cache(dec.caches[0])
    for t in range(10):
        want, weight, *_ = serving.attention(q[:, t].double().cpu().numpy(), mirror,
                                             dec.page_table.cpu().numpy(), [22 + t], 1 / 8)
        got = cap.y[0, t].view(1, CFG.n_head, 64).double().cpu().numpy()
        # keys, values, probabilities and the output in fp16; scores of a few
        assert np.all(np.abs(got - want) <= 16 * 2.0 ** -11 * weight + 2.0 ** -24)


def test_decoder_refusals():
    dec = llama.CachedDecoder(CFG, _layers(CFG), batch=2, max_tokens=32, page_size=16, n_layers=1)
    with pytest.raises(RuntimeError, match="x must be"):
        dec(torch.zeros((1, 4, 256), dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError, match="do not fit"):
        dec(torch.zeros((2, 33, 256), dtype=torch.float16, device="cuda"))
    dec(torch.zeros((2, 32, 256), dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError, match="do not fit"):
        dec(torch.zeros((2, 1, 256), dtype=torch.float16, device="cuda"))


def test_counts_of_tokens_outside_the_chunk():
    """Counts beyond the chunk count as the whole of it, negative ones as none,
    so a sequence's end stays within its pages; other types are refused."""
    dec = llama.CachedDecoder(CFG, _layers(CFG), batch=3, max_tokens=16, page_size=16, n_layers=1)
    for bad in (torch.tensor([1, 1, 1]).cuda(), torch.ones(2, dtype=torch.int32).cuda(),
                torch.ones(3, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="tokens must be int32"):
            dec(torch.zeros((3, 4, 256), dtype=torch.float16, device="cuda"), bad)
    x = torch.randn((3, 4, 256), generator=torch.Generator().manual_seed(0)).half().cuda()
    dec(x, torch.tensor([2, 4, 0], dtype=torch.int32).cuda())
    dec(x, torch.tensor([5, 2 ** 31 - 1, -3], dtype=torch.int32).cuda())
    assert dec.lengths.tolist() == [6, 8, 0]
    y = dec(x[:, :1])
    assert dec.lengths.tolist() == [7, 9, 1] and torch.isfinite(y).all()


@pytest.mark.parametrize("max_tokens", [48, 96])
def test_padded_chunks_fill_the_cache(max_tokens):
    """Chunks padded for different sequences: what fits by the sequences' own
    lengths is taken, also where the places with padding are more, and is
    stored as with more room; one token too many is refused."""
    layers = _layers(CFG, seed=5)
    dec = llama.CachedDecoder(CFG, layers, batch=2, max_tokens=max_tokens, page_size=16,
                              n_layers=1)
    mirror = serving.Cache(dec.caches[0])
    g = torch.Generator().manual_seed(7)
    lengths = np.zeros(2, np.int64)
    for T, counts in ((20, [20, 2]), (20, [0, 20]), (20, [20, 3]), (12, [1, 12]), (1, [1, 1]),
                      (30, [6, 0]), (9, [0, 9]), (1, [0, 1])):
        x = torch.randn((2, T, CFG.n_embd), generator=g).half().cuda()
        cap = _Capture(CFG, dec.linears[0])
        y = dec(x, torch.tensor(counts, dtype=torch.int32, device="cuda"), capture=[cap])
        assert torch.isfinite(y).all()
        positions = torch.from_numpy(lengths[:, None] + np.arange(T)).cuda()
        _, k, v = cap.qkv(dec.cos, dec.sin, positions.clamp(max=dec.max_tokens - 1))
        for b in range(2):
            n = counts[b]
            at = positions[b, :n].cpu().numpy()
            slots = dec.page_table[b].cpu().numpy()[at // 16].astype(np.int64) * 16 + at % 16
            mirror.write(k[b, :n].double().cpu().numpy(), v[b, :n].double().cpu().numpy(), slots)
        _check_fields(dec.caches[0], mirror)
        lengths += np.array(counts)
        assert dec.lengths.tolist() == lengths.tolist()
    assert lengths.tolist() == [48, 48]
    if max_tokens == 48:
        x = torch.zeros((2, 1, CFG.n_embd), dtype=torch.float16, device="cuda")
        with pytest.raises(RuntimeError, match="1 tokens do not fit behind 48 of 48"):
            dec(x, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
        y = dec(x, torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
        assert torch.isfinite(y).all() and dec.lengths.tolist() == [48, 48]
