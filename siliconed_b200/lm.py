"""A decoder in 8 bits on the operators of ``lm_abi``: paged key-value cache, block-scaled layers, decode steps.

Per layer and step: the residual addition, RMS norm and quantization (one call), the q / k / v product, QK-norm, rotation
and append to the paged cache, the attention over it, its quantization and output product, and the same around the
SwiGLU MLP.  The residual stream is fp32 and is only touched by the norms.  ``python -m siliconed_b200.lm`` runs a small
decoder with random weights: requests of different lengths join and leave one batch.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import dit_abi, lm_abi
from .lm_abi import BLOCK, LmError

E4M3_MAX = 448.0


def _device(device) -> torch.device:
    """The device with its index: a bare "cuda" is another one whenever the current device changes."""
    device = torch.device("cuda") if device is None else torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


@dataclass
class DecoderConfig:
    """The defaults are the widths of the text encoder whose int8 shapes the encoder prefill workload uses."""
    dim: int = 2560
    hidden: int = 9728
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    layers: int = 2
    vocab: int = 4096
    max_pos: int = 4096
    theta: float = 1e6
    eps: float = 1e-6
    pairs: str = "halves"


class BlockWeight:
    """An [n, k] weight as e4m3 codes with one fp32 scale per 128 x 128 values (the layout such weights are published in)."""

    def __init__(self, codes, scales, bias=None):
        self.codes, self.scales, self.bias = codes, scales, bias

    @classmethod
    def quantize(cls, w, bias=None) -> "BlockWeight":
        n, k = w.shape
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        padded = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
        scales = (padded.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(1e-30)
        codes = (padded / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        codes = codes.view(torch.uint8).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous().view(torch.float8_e4m3fn)
        return cls(codes, scales.contiguous(), bias)

    def dequantize(self):
        """fp32 [n, k]."""
        n, k = self.codes.shape
        return self.codes.float() * self.scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]

    def __call__(self, codes, scales, out=None):
        return lm_abi.linear_block_fp8(codes, scales, self.codes, self.scales, self.bias, out)


class PagedCache:
    """Keys and values of up to ``seqs`` sequences in pages of one pool, for every layer.

    ``e4m3`` keeps them in 8 bits with a scale per token and head.  Pages are handed out on the host (``extend``) and given
    back when a sequence leaves (``release``); the device sees the page table.
    """

    def __init__(self, cfg: DecoderConfig, seqs: int, pages: int, page_size: int = 16, e4m3: bool = False, device=None):
        device = _device(device)
        shape = (cfg.layers, pages, cfg.kv_heads, page_size, cfg.head_dim)
        kind = torch.float8_e4m3fn if e4m3 else torch.bfloat16
        self.k, self.v = (torch.zeros(shape, dtype=kind, device=device) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(shape[:4], device=device) for _ in range(2)) if e4m3 else (None, None)
        self.page_size = page_size
        self.max_pos = cfg.max_pos  # the rotation table's rows: fewer than the table's slots where pages do not divide it
        self.width = -(-cfg.max_pos // page_size)
        self.table = torch.zeros(seqs, self.width, dtype=torch.int32, device=device)
        self.lengths = [0] * seqs
        self._pages: list[list[int]] = [[] for _ in range(seqs)]
        self._free = list(range(pages - 1, -1, -1))
        self._unused = list(range(seqs - 1, -1, -1))
        self._live: set[int] = set()

    def admit(self) -> int:
        """A sequence number for a new request."""
        if not self._unused:
            raise LmError("PagedCache.admit: every sequence is in use")
        seq = self._unused.pop()
        self._live.add(seq)
        return seq

    def extend(self, seqs, count: int = 1) -> None:
        """Room for ``count`` more tokens of each sequence; the table's new entries go to the device in one copy."""
        if count < 0 or len(set(seqs)) != len(seqs) or not self._live.issuperset(seqs):
            raise LmError(f"PagedCache.extend: sequences in use, each once, and a count of 0 or more: got {seqs}, {count}")
        rows, columns, pages = [], [], []
        need = [-(-(self.lengths[s] + count) // self.page_size) - len(self._pages[s]) for s in seqs]
        if sum(need) > len(self._free):
            raise LmError(f"PagedCache.extend: {sum(need)} pages wanted, {len(self._free)} free")
        if any(self.lengths[s] + count > self.max_pos for s in seqs):
            raise LmError(f"PagedCache.extend: a sequence longer than {self.max_pos} positions")
        for s, n in zip(seqs, need):
            for _ in range(n):
                page = self._free.pop()
                rows.append(s)
                columns.append(len(self._pages[s]))
                pages.append(page)
                self._pages[s].append(page)
            self.lengths[s] += count
        if pages:
            where = torch.tensor([rows, columns, pages], dtype=torch.int64).to(self.table.device)
            self.table[where[0], where[1]] = where[2].to(torch.int32)

    def release(self, seq: int) -> None:
        """The sequence's pages are free for others."""
        if seq not in self._live:
            raise LmError(f"PagedCache.release: sequence {seq} is not in use")
        self._live.remove(seq)
        self._free.extend(reversed(self._pages[seq]))
        self._pages[seq] = []
        self.lengths[seq] = 0
        self._unused.append(seq)

    def layer(self, i: int):
        """(k, v, k_scale, v_scale) of one layer."""
        return (self.k[i], self.v[i], None if self.k_scale is None else self.k_scale[i],
                None if self.v_scale is None else self.v_scale[i])


def rotation_table(cfg: DecoderConfig, device):
    """fp32 [max_pos, head_dim / 2, 2]: (cos, sin) of every position and pair."""
    inv = cfg.theta ** (-torch.arange(0, cfg.head_dim, 2, device=device, dtype=torch.float64) / cfg.head_dim)
    angle = torch.arange(cfg.max_pos, device=device, dtype=torch.float64)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


class DecoderLayer:
    def __init__(self, cfg: DecoderConfig, g, device):
        def weight(n, k):
            return BlockWeight.quantize(torch.randn(n, k, generator=g, device=device) / math.sqrt(k))

        def norm(d):
            return 1 + 0.1 * torch.randn(d, generator=g, device=device)

        self.cfg = cfg
        self.norm1, self.norm2 = norm(cfg.dim), norm(cfg.dim)
        self.norm_q, self.norm_k = norm(cfg.head_dim), norm(cfg.head_dim)
        self.qkv = weight((cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim, cfg.dim)
        self.out = weight(cfg.dim, cfg.heads * cfg.head_dim)
        self.gate_up = weight(2 * cfg.hidden, cfg.dim)
        self.down = weight(cfg.dim, cfg.hidden)

    def forward(self, x, delta, freqs, positions, table, lengths, cache, workspace=None):
        """One new token per sequence: x fp32 [batch, dim] += delta in place; returns the layer's own addition (bf16).  The
        tensors' device is the current one (the activation runs on the current device's stream)."""
        cfg = self.cfg
        batch = x.shape[0]
        _, codes, scales = lm_abi.rms_norm_quantize(x, delta, self.norm1, cfg.eps)
        q = lm_abi.append_paged(self.qkv(codes, scales), cfg.heads, cfg.kv_heads, self.norm_q, self.norm_k, cfg.eps, freqs,
                                cfg.pairs, None, positions, table, *cache)
        o = lm_abi.paged_attention(q, *cache, table, lengths, 1 / math.sqrt(cfg.head_dim), workspace=workspace)
        _, codes, scales = lm_abi.rms_norm_quantize(o.view(batch, -1), norm=False)
        _, codes, scales = lm_abi.rms_norm_quantize(x, self.out(codes, scales), self.norm2, cfg.eps)
        h = self.gate_up(codes, scales)
        h = dit_abi.swiglu(h, cfg.hidden, torch.empty(batch, cfg.hidden, dtype=torch.bfloat16, device=x.device))
        _, codes, scales = lm_abi.rms_norm_quantize(h, norm=False)
        return self.down(codes, scales)


class Decoder:
    """Embedding, layers and logits with random weights of a seed; ``step`` decodes one token for each given sequence."""

    def __init__(self, cfg: DecoderConfig, seed: int = 0, device=None):
        device = _device(device)
        g = torch.Generator(device=device).manual_seed(seed)
        self.cfg, self.device = cfg, device
        self.embedding = torch.randn(cfg.vocab, cfg.dim, generator=g, device=device)
        self.layers = [DecoderLayer(cfg, g, device) for _ in range(cfg.layers)]
        self.norm = 1 + 0.1 * torch.randn(cfg.dim, generator=g, device=device)
        self.head = BlockWeight.quantize(torch.randn(cfg.vocab, cfg.dim, generator=g, device=device) / math.sqrt(cfg.dim))
        self.freqs = rotation_table(cfg, device)

    def forward(self, tokens, positions, table, lengths, cache: PagedCache, workspace=None):
        """Logits fp32 [batch, vocab] of tokens int64 [batch], each below vocab (not checked here: they are on the device), at
        positions int32 [batch]; table int32 [batch, width] and lengths int32 [batch] (the new tokens counted) are the
        sequences' rows."""
        with torch.cuda.device(self.device):
            x, delta = self.embedding[tokens], None
            for i, layer in enumerate(self.layers):
                delta = layer.forward(x, delta, self.freqs, positions, table, lengths, cache.layer(i), workspace)
            _, codes, scales = lm_abi.rms_norm_quantize(x, delta, self.norm, self.cfg.eps)
            return self.head(codes, scales, torch.empty(x.shape[0], self.cfg.vocab, device=x.device))

    def step(self, tokens: list[int], seqs: list[int], cache: PagedCache):
        """Appends one token to each sequence and returns its logits."""
        # an index past the embedding is a failed assertion on the device, which ends the process's CUDA context
        if len(tokens) != len(seqs) or not all(0 <= t < self.cfg.vocab for t in tokens):
            raise LmError(f"Decoder.step: a token below {self.cfg.vocab} for each sequence: got {tokens} for {seqs}")
        if not seqs:
            return torch.empty(0, self.cfg.vocab, device=self.device)
        cache.extend(seqs)
        lengths = torch.tensor([cache.lengths[s] for s in seqs], dtype=torch.int32).to(self.device)
        rows = torch.tensor(seqs).to(self.device)
        return self.forward(torch.tensor(tokens).to(self.device), lengths - 1, cache.table[rows], lengths, cache)


def main() -> None:
    """Three requests in one batch: one joins late, one leaves early and its pages serve another."""
    torch.manual_seed(0)
    cfg = DecoderConfig(layers=4)
    model = Decoder(cfg)
    for e4m3 in (False, True):
        cache = PagedCache(cfg, seqs=4, pages=64, e4m3=e4m3)
        live = {cache.admit(): 1, cache.admit(): 2}  # sequence -> its next token
        for t in range(40):
            if t == 10:
                live[cache.admit()] = 3
            if t == 25:
                gone = next(iter(live))
                del live[gone]
                cache.release(gone)
                live[cache.admit()] = 4
            logits = model.step(list(live.values()), list(live), cache)
            live = dict(zip(live, logits.argmax(-1).tolist()))
        batch = 16
        cache = PagedCache(cfg, seqs=batch, pages=batch * 64, e4m3=e4m3)
        seqs = [cache.admit() for _ in range(batch)]
        cache.extend(seqs, 1000)
        table = cache.table[torch.tensor(seqs).to(model.device)]
        lengths = torch.full((batch,), 1000, dtype=torch.int32, device=model.device)
        tokens = torch.zeros(batch, dtype=torch.int64, device=model.device)
        workspace = lm_abi.attention_workspace(cfg.heads, cfg.kv_heads, cfg.head_dim)
        run = lambda: model.forward(tokens, lengths - 1, table, lengths, cache, workspace)  # noqa: E731
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        graph.replay()
        start.record()
        for _ in range(50):
            graph.replay()
        stop.record()
        torch.cuda.synchronize()
        us = start.elapsed_time(stop) / 50 * 1e3
        print(f"{'e4m3' if e4m3 else 'bf16'} cache: tokens {list(live.values())}; {batch} sequences of 1000 tokens, "
              f"{cfg.layers} layers: {us:.0f} us a step ({batch / us * 1e6:.0f} tokens/s)")
        status = lm_abi.errors()
        if status != (lm_abi.OK, 0):
            raise LmError(f"device status {status}")


if __name__ == "__main__":
    main()
