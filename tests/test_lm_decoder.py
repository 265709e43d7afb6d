"""The decoder example (siliconed_b200.lm): the operators together.

Two decoders that quantize activations to e4m3 drift apart by that rounding's own noise as soon as one sum differs in its
last bit (a code moved by a step of 2^-3 moves others), so a long run is not compared end to end: every call of a run
with joining and leaving requests is checked against the 64-bit formula on the inputs it got, with test_lm's bars, and
what it got against what came before it.  A request's first token, whose attention has the one weight 1, is compared
with a plain decoder on the same weights within 5e-2 (a wrong layer order, weight or norm is an error of order one)."""
import math

import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")


def test_cache_hands_out_and_takes_back_pages():
    from siliconed_b200.lm import DecoderConfig, PagedCache
    from siliconed_b200.lm_abi import LmError
    cfg = DecoderConfig(dim=256, hidden=512, heads=2, kv_heads=1, layers=1, max_pos=64)
    cache = PagedCache(cfg, seqs=3, pages=6, page_size=16, device="cpu")
    a, b = cache.admit(), cache.admit()
    cache.extend([a, b], 17)
    assert cache.lengths[a] == 17 and len({*cache.table[a, :2].tolist(), *cache.table[b, :2].tolist()}) == 4
    cache.extend([a], 15)
    with pytest.raises(LmError):
        cache.extend([a], 33)       # past the table
    with pytest.raises(LmError):
        cache.extend([a, b], 32)    # four pages wanted, two free
    assert cache.lengths[a] == 32 and cache.lengths[b] == 17
    first = cache.table[a, :2].tolist()
    cache.release(a)
    c = cache.admit()
    cache.extend([c], 20)
    assert cache.table[c, :2].tolist() == first
    cache.admit()
    with pytest.raises(LmError):
        cache.admit()


def test_cache_refuses_positions_past_the_rotation_table():
    """Pages of 24 give 50 positions three pages, 72 slots: positions 50 .. have no row in the rotation table."""
    from siliconed_b200.lm import DecoderConfig, PagedCache
    from siliconed_b200.lm_abi import LmError
    cfg = DecoderConfig(dim=256, hidden=512, heads=2, kv_heads=1, layers=1, max_pos=50)
    cache = PagedCache(cfg, seqs=2, pages=8, page_size=24, device="cpu")
    a, b = cache.admit(), cache.admit()
    cache.extend([a, b], 49)
    cache.extend([a])
    with pytest.raises(LmError):
        cache.extend([a])
    with pytest.raises(LmError):
        cache.extend([b], 2)
    assert cache.lengths[a] == 50 and cache.lengths[b] == 49 and len(cache._free) == 2


def test_cache_takes_sequences_in_use_once_each():
    """A sequence named twice would get the pages of one extension for the length of two; one that is not in use, pages
    that the next request admitted under its number would inherit."""
    from siliconed_b200.lm import DecoderConfig, PagedCache
    from siliconed_b200.lm_abi import LmError
    cfg = DecoderConfig(dim=256, hidden=512, heads=2, kv_heads=1, layers=1, max_pos=64)
    cache = PagedCache(cfg, seqs=3, pages=8, page_size=16, device="cpu")
    a, b = cache.admit(), cache.admit()
    cache.extend([a, b], 16)
    unused = ({0, 1, 2} - {a, b}).pop()
    for seqs, count in (([a, a], 16), ([a, b, a], 1), ([unused], 1), ([3], 1), ([-1], 1), ([a], -1)):
        with pytest.raises(LmError):
            cache.extend(seqs, count)
    assert cache.lengths == [16 if s in (a, b) else 0 for s in range(3)] and len(cache._free) == 6
    cache.release(a)
    for seq in (a, unused, 3, -1):
        with pytest.raises(LmError):
            cache.release(seq)
    assert len(cache._free) == 7 and sorted(cache._unused) == sorted((a, unused))
    cache.extend([], 1)
    cache.extend([b], 0)
    assert cache.lengths[b] == 16


def test_step_refuses_tokens_that_the_embedding_does_not_have():
    """Refused on the host, before anything reaches the cache or the device (there an index out of range is an assertion)."""
    from siliconed_b200.lm import Decoder, DecoderConfig, PagedCache
    from siliconed_b200.lm_abi import LmError
    cfg = DecoderConfig(dim=256, hidden=512, heads=2, kv_heads=1, layers=1, vocab=300, max_pos=64)
    cache = PagedCache(cfg, seqs=2, pages=8, page_size=16, device="cpu")
    model = Decoder.__new__(Decoder)  # the configuration alone: nothing else may be looked at
    model.cfg = cfg
    a, b = cache.admit(), cache.admit()
    for tokens, seqs in (([300, 0], [a, b]), ([0, -1], [a, b]), ([0], [a, b]), ([0, 1], [a])):
        with pytest.raises(LmError):
            model.step(tokens, seqs, cache)
    assert cache.lengths == [0, 0] and len(cache._free) == 8


def test_forward_runs_on_the_models_device(monkeypatch):
    """The activation between the products goes to the current device's stream: it has to be the model's device."""
    import contextlib
    from siliconed_b200 import lm
    entered, seen = [], []

    @contextlib.contextmanager
    def guard(device):
        entered.append(device)
        yield
        entered.pop()

    class Layer:
        def forward(self, *args):
            seen.append(list(entered))

    monkeypatch.setattr(torch.cuda, "device", guard)
    monkeypatch.setattr(lm.lm_abi, "rms_norm_quantize", lambda *a: (seen.append(list(entered)), None, None))
    model = lm.Decoder.__new__(lm.Decoder)
    model.cfg = lm.DecoderConfig(dim=4, layers=2, vocab=3)
    model.device, model.layers, model.embedding = torch.device("cuda", 1), [Layer(), Layer()], torch.zeros(3, 4)
    model.freqs = model.norm = None
    model.head = lambda codes, scales, out: out
    cache = lm.PagedCache(lm.DecoderConfig(layers=2, max_pos=16, kv_heads=1), seqs=1, pages=1, device="cpu")
    out = model.forward(torch.tensor([1, 2]), None, None, None, cache)
    assert out.shape == (2, 3) and seen == [[model.device]] * 3 and not entered


def test_step_of_no_sequences():
    from siliconed_b200.lm import Decoder, DecoderConfig, PagedCache
    cfg = DecoderConfig(dim=256, hidden=512, heads=2, kv_heads=1, layers=1, vocab=300, max_pos=64)
    model = Decoder.__new__(Decoder)
    model.cfg, model.device = cfg, torch.device("cpu")
    logits = model.step([], [], PagedCache(cfg, seqs=2, pages=8, page_size=16, device="cpu"))
    assert logits.shape == (0, 300) and logits.dtype == torch.float32


def test_weight_quantization_on_the_host():
    from siliconed_b200.lm import BlockWeight
    g = torch.Generator().manual_seed(0)
    w = torch.randn(200, 300, generator=g)
    q = BlockWeight.quantize(w)
    assert q.scales.shape == (2, 3) and q.codes.shape == (200, 300)
    # half a step of a normal code, 2^-4 of the value; of a subnormal one 2^-10 of the scale
    room = torch.maximum(w.abs() * 2.0 ** -4, 2.0 ** -10 * q.scales.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300])
    assert bool(((q.dequantize() - w).abs() <= room * (1 + 1e-5)).all())


class Plain:
    """The decoder on plain tensors, one sequence, contexts kept as lists."""

    def __init__(self, model, e4m3):
        self.m, self.e4m3, self.kv = model, e4m3, [[] for _ in model.layers]

    @staticmethod
    def stored(x):
        return x.to(torch.bfloat16).float()

    def cached(self, h):
        """Key or value heads as the cache gives them back."""
        return torch.stack([self.quantized(row) for row in h]) if self.e4m3 else self.stored(h)

    @staticmethod
    def quantized(y):
        d = y.shape[-1]
        p = torch.nn.functional.pad(y, (0, -d % 128)).view(-1, 128)
        s = (p.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-30)
        return ((p / s).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s).view(-1)[:d]

    def norm(self, x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.m.cfg.eps) * w

    def product(self, y, w):
        return w.dequantize() @ self.quantized(y)

    def step(self, token, pos):
        cfg = self.m.cfg
        x = self.m.embedding[token].clone()
        cs = self.m.freqs[pos]
        half = cfg.head_dim // 2

        def turn(h):
            a, b = h[:, :half], h[:, half:]
            return torch.cat([a * cs[:, 0] - b * cs[:, 1], a * cs[:, 1] + b * cs[:, 0]], -1)

        for layer, kv in zip(self.m.layers, self.kv):
            h = self.stored(self.product(self.norm(x, layer.norm1), layer.qkv)).view(-1, cfg.head_dim)
            q, k, v = h.split([cfg.heads, cfg.kv_heads, cfg.kv_heads])
            kv.append((self.cached(turn(self.norm(k, layer.norm_k))), self.cached(v)))
            q = self.stored(turn(self.norm(q, layer.norm_q)))
            keys, values = (torch.stack([t[i] for t in kv], 1).repeat_interleave(cfg.heads // cfg.kv_heads, 0) for i in (0, 1))
            p = torch.softmax((keys @ q[:, :, None]).squeeze(-1) / math.sqrt(cfg.head_dim), -1)
            x = x + self.stored(self.product(self.stored((p[:, None] @ values).reshape(-1)), layer.out))
            g, u = self.stored(self.product(self.norm(x, layer.norm2), layer.gate_up)).split(cfg.hidden)
            x = x + self.stored(self.product(self.stored(g / (1 + torch.exp(-g)) * u), layer.down))
        return self.product(self.norm(x, self.m.norm), self.m.head)


@gpu
@needs_cuda
@pytest.mark.parametrize("e4m3", [False, True])
def test_first_token_matches_a_plain_decoder(e4m3):
    from siliconed_b200 import lm_abi
    from siliconed_b200.lm import Decoder, DecoderConfig, PagedCache
    cfg = DecoderConfig(dim=512, hidden=768, heads=8, kv_heads=2, layers=2, vocab=500, max_pos=128)
    model = Decoder(cfg, seed=3)
    cache = PagedCache(cfg, seqs=3, pages=12, page_size=16, e4m3=e4m3)
    seqs = [cache.admit() for _ in range(3)]
    for got, token in zip(model.step([7, 499, 0], seqs, cache), (7, 499, 0)):
        want = Plain(model, e4m3).step(token, 0)
        assert float((got - want).norm() / want.norm()) <= 5e-2
    assert lm_abi.errors() == (lm_abi.OK, 0)


@gpu
@needs_cuda
@pytest.mark.parametrize("e4m3", [False, True])
def test_every_call_of_a_run(e4m3, monkeypatch):
    import test_lm as ops
    from siliconed_b200 import lm, lm_abi
    cfg = lm.DecoderConfig(dim=512, hidden=768, heads=8, kv_heads=2, layers=2, vocab=500, max_pos=128)
    model = lm.Decoder(cfg, seed=3)
    cache = lm.PagedCache(cfg, seqs=3, pages=12, page_size=16, e4m3=e4m3)
    log = []
    real = {n: getattr(lm_abi, n) for n in ("rms_norm_quantize", "append_paged", "paged_attention", "linear_block_fp8")}

    def norm(x, delta=None, weight=None, eps=1e-6, **kw):
        z = x.double() if delta is None else x.double() + delta.double()
        y = z * weight.double() if weight is not None else z
        if kw.get("norm", True):
            y = y / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
        out = real["rms_norm_quantize"](x, delta, weight, eps, **kw)
        assert torch.equal(out[0], z.to(x.dtype)) or x.dtype == torch.float32  # fp32: one rounding of the sum
        assert float((out[0].double() - z).abs().max()) <= 2.0 ** -24 * float(z.abs().max())
        ops.check_codes(out[1], out[2], y)
        log.append(("norm", x, out[1], delta))
        return out

    def linear(codes, scales, weight, weight_scales, bias, out):
        y = real["linear_block_fp8"](codes, scales, weight, weight_scales, bias, out)
        ops.check_product(codes, scales, weight, weight_scales, bias, y)
        log.append(("linear", codes, y, weight))
        return y

    def append(qkv, heads, kv_heads, nq, nk, eps, freqs, pairs, seq, positions, table, k, v, ks, vs):
        assert log[-1][2] is qkv and seq is None
        q = real["append_paged"](qkv, heads, kv_heads, nq, nk, eps, freqs, pairs, seq, positions, table, k, v, ks, vs)
        x = qkv.double().view(len(qkv), -1, cfg.head_dim)
        want = ops.head_ref(x[:, :heads], nq, freqs[positions.long()], pairs, eps)
        assert float(((q.double() - want).abs() - ops.U * 1.01 * want.abs() - 2e-6 * want.abs().amax(-1, keepdim=True)).max()) <= 0
        if not e4m3:
            t = torch.arange(len(qkv), device="cuda")
            page = table[t, positions.long() // 16].long()
            assert torch.equal(v[page, :, positions.long() % 16], qkv.view(len(qkv), -1, cfg.head_dim)[:, heads + kv_heads:])
        log.append(("append", qkv, q, k))
        return q

    def attention(q, k, v, ks, vs, table, lengths, scale, workspace=None):
        assert log[-1][2] is q and log[-1][3] is k
        lse = torch.empty(q.shape[:2], device="cuda")
        out = real["paged_attention"](q, k, v, ks, vs, table, lengths, scale, None, lse, workspace)
        ops.check_attention(q, (k, ks), (v, vs), table, lengths.tolist(), scale, out, lse)
        log.append(("attention", q, out, None))
        return out

    for n, f in zip(real, (norm, append, attention, linear)):
        monkeypatch.setattr(lm_abi, n, f)
    g = torch.Generator().manual_seed(1)
    seqs, ages, first_pages = {}, {}, None
    for t in range(40):
        if t in (0, 5, 30):  # the third request gets the pages that the first one gave back
            if t == 30:
                first_pages = cache.table[seqs["r0"], :2].tolist()
                cache.release(seqs.pop("r0"))
            name = f"r{len(ages)}"
            seqs[name], ages[name] = cache.admit(), 0
        log.clear()
        logits = model.step(torch.randint(cfg.vocab, (len(seqs),), generator=g).tolist(), list(seqs.values()), cache)
        for name in seqs:
            ages[name] += 1
            assert cache.lengths[seqs[name]] == ages[name]
        per_layer = ["norm", "linear", "append", "attention", "norm", "linear", "norm", "linear", "norm", "linear"]
        assert [e[0] for e in log] == per_layer * cfg.layers + ["norm", "linear"]
        assert log[-1][2] is logits
        for i, e in enumerate(log):
            if e[0] == "linear":
                assert e[1] is log[i - 1][2]            # the codes of the quantization before it
        for i, layer in enumerate(model.layers):
            w = [e[3] for e in log[10 * i:10 * i + 10] if e[0] == "linear"]
            assert all(a is b.codes for a, b in zip(w, (layer.qkv, layer.out, layer.gate_up, layer.down)))
            assert log[10 * i + 6][1] is log[10 * i][1] and log[10 * i + 6][3] is log[10 * i + 5][2]  # the stream, the addition
            assert (log[10 * i][3] is None) == (i == 0) and log[10 * i + 10][3] is log[10 * i + 9][2]
    assert cache.table[seqs["r2"], :1].tolist() == first_pages[:1]
    assert lm_abi.errors() == (lm_abi.OK, 0)


@gpu
@needs_cuda
@pytest.mark.parametrize("head_dim", [64, 128])
def test_cache_rows_of_a_run_in_8_bits(head_dim, monkeypatch):
    """What every append of a run leaves in an e4m3 cache, codes and scales, against the 64-bit formula on what it got."""
    import test_lm as ops
    from siliconed_b200 import lm, lm_abi
    cfg = lm.DecoderConfig(dim=512, hidden=768, heads=8, kv_heads=2, head_dim=head_dim, layers=2, vocab=500, max_pos=48)
    model = lm.Decoder(cfg, seed=5)
    cache = lm.PagedCache(cfg, seqs=2, pages=8, page_size=16, e4m3=True)
    real, calls = lm_abi.append_paged, []

    def append(qkv, heads, kv_heads, nq, nk, eps, freqs, pairs, seq, positions, table, k, v, ks, vs):
        q = real(qkv, heads, kv_heads, nq, nk, eps, freqs, pairs, seq, positions, table, k, v, ks, vs)
        x = qkv.double().view(len(qkv), -1, head_dim)
        at = positions.long()
        page, slot = table[torch.arange(len(qkv), device="cuda"), at // 16].long(), at % 16
        for c, s, ref in ((k, ks, ops.head_ref(x[:, heads:heads + kv_heads], nk, freqs[at], pairs, eps)), (v, vs, x[:, heads + kv_heads:])):
            got = c.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn)
            ops.check_cache_rows(got.reshape(-1, head_dim), s[page, :, slot].reshape(-1), ref.reshape(-1, head_dim))
        calls.append(len(qkv))
        return q

    monkeypatch.setattr(lm_abi, "append_paged", append)
    seqs = [cache.admit(), cache.admit()]
    for t in range(18):
        model.step([t, 499 - t], seqs, cache)
    assert calls == [2] * 18 * cfg.layers
    assert lm_abi.errors() == (lm_abi.OK, 0)


@gpu
@needs_cuda
def test_decoder_step_in_a_graph():
    from siliconed_b200 import lm_abi
    from siliconed_b200.lm import Decoder, DecoderConfig, PagedCache
    cfg = DecoderConfig(dim=256, hidden=512, heads=4, kv_heads=2, layers=2, vocab=300, max_pos=64)
    model = Decoder(cfg)
    cache = PagedCache(cfg, seqs=2, pages=8)
    seqs = [cache.admit(), cache.admit()]
    cache.extend(seqs, 20)
    cache.k.normal_(), cache.v.normal_()
    table = cache.table[torch.tensor(seqs).cuda()]
    lengths = torch.tensor([20, 7], dtype=torch.int32, device="cuda")
    positions = lengths - 1
    tokens = torch.tensor([5, 6], device="cuda")
    workspace = lm_abi.attention_workspace(cfg.heads, cfg.kv_heads, cfg.head_dim)
    want = model.forward(tokens, positions, table, lengths, cache, workspace)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.forward(tokens, positions, table, lengths, cache, workspace)
    for _ in range(2):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)
    assert lm_abi.errors() == (lm_abi.OK, 0)
