"""The decoder operators (libsiliconed_lm) against plain 64-bit implementations.

Bars, from the formats' rounding: u = 2^-8 is the largest relative error of a rounding to bf16 (8 significant bits), 2^-4 of one to a
normal e4m3 code, 2^-10 (of the scale) of a subnormal one.  fp32 work adds the terms named at each check.
"""
import ctypes
import math
import subprocess

import pytest

torch = pytest.importorskip("torch")

from siliconed_b200 import lm_abi  # noqa: E402
from siliconed_b200.lm_abi import LmError  # noqa: E402

gpu = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
U = 2.0 ** -8
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def clean():
    assert lm_abi.errors() == (lm_abi.OK, 0)


# ------------------------------------------------------------------------------------------------ the library


def test_library_exports_exactly_the_header():
    lm_abi.load()
    names = lm_abi.header_functions()
    assert names == set(lm_abi.SIGNATURES), names ^ set(lm_abi.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", lm_abi.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if " T " in line} == names


def test_null_and_bad_arguments_are_refused():
    lib = lm_abi.load()
    p = ctypes.c_void_p(4096)  # never dereferenced: a later argument is refused first, or the device is missing
    bad = lm_abi.INVALID_ARG
    norm = lib.sl_rms_norm_quantize
    assert norm(None, 0, None, 0, None, 1e-6, 1, 2, 128, None, p, p, None) == bad
    assert norm(p, 7, None, 0, None, 1e-6, 1, 2, 128, None, p, p, None) == bad          # type
    assert norm(p, 0, None, 0, None, 1e-6, 1, 2, 120, None, p, p, None) == bad          # d
    assert norm(p, 0, None, 0, None, 1e-6, 1, 2, 16400, None, p, p, None) == bad
    assert norm(p, 0, None, 0, None, 1e-6, 1, -1, 128, None, p, p, None) == bad         # rows
    assert norm(p, 0, p, 0, None, 1e-6, 1, 2, 128, None, p, p, None) == bad             # delta without x_out
    assert norm(ctypes.c_void_p(4098), 0, None, 0, None, 1e-6, 1, 2, 128, None, p, p, None) == bad
    assert norm(None, 0, None, 0, None, 1e-6, 1, 0, 128, None, None, None, None) == lm_abi.OK
    app = lib.sl_append_paged
    args = [p, 2, 4, 2, 128, None, None, 1e-6, p, 16, 0, p, p, p, 2, 4, 8, 16, 0, p, p, None, None, p, None]
    for at, value in [(0, None), (1, -1), (2, 0), (3, 0), (4, 96), (8, None), (9, 0), (10, 2), (12, None), (13, None),
                      (14, 0), (15, 0), (16, 0), (17, 0), (18, 1), (18, 2), (19, None), (20, None), (21, p), (23, None)]:
        assert app(*[value if i == at else a for i, a in enumerate(args)]) == bad, at
    assert app(*[3 if i == 1 else None if i == 11 else a for i, a in enumerate(args)]) == bad  # 3 tokens, 2 sequences
    att = lib.sl_paged_attention
    args = [p, p, p, None, None, 0, p, p, 2, 4, 2, 128, 4, 8, 16, 0.1, p, None, p, 1 << 30, None]
    for at, value in [(0, None), (1, None), (2, None), (3, p), (5, 1), (5, 2), (6, None), (7, None), (8, -1), (9, 3), (10, 0),
                      (11, 100), (12, 0), (13, 0), (13, 1 << 40), (14, 0), (15, math.inf), (16, None), (18, None)]:
        assert att(*[value if i == at else a for i, a in enumerate(args)]) == bad, at
    lin = lib.sl_linear_block_fp8
    args = [p, p, p, p, None, 4, 128, 256, p, 0, None]
    for at, value in [(0, None), (1, None), (2, None), (3, None), (5, -1), (6, 0), (7, 0), (7, 100), (8, None), (9, 2)]:
        assert lin(*[value if i == at else a for i, a in enumerate(args)]) == bad, at
    assert lib.sl_paged_attention_workspace(4, 2, 128, None) == bad


def test_packed_arguments_are_the_headers_structs():
    """The packed calls' formats against the header: the same types in the same order, and no null struct taken."""
    lib = lm_abi.load()
    text = open(lm_abi.HEADER).read()
    for name, form in lm_abi._PACKED.items():
        body = text[:text.index("} " + name + "_args;")].rsplit("typedef struct {", 1)[1]
        codes = ""
        for member in body.strip().rstrip(";").split(";"):
            base = member.replace("const", "").split()[0]
            for field in member.split(","):
                codes += "P" if "*" in field else {"int": "i", "int64_t": "q", "float": "f", "size_t": "N"}[base]
        assert "@" + codes == form.format, name
        assert getattr(lib, name + "_with")(None) == lm_abi.INVALID_ARG
    assert lm_abi._PACKED["sl_rms_norm_quantize"].size % 8 == 0  # ends with the stream


def test_nothing_to_do_is_a_no_op():
    """Zero rows, tokens or sequences, the append's table of no sequences among them; pointers are not looked at."""
    lib = lm_abi.load()
    assert lib.sl_append_paged(None, 0, 4, 2, 128, None, None, 1e-6, None, 16, 0, None, None, None, 0, 4, 8, 16, 0, None, None,
                               None, None, None, None) == lm_abi.OK
    assert lib.sl_append_paged(None, 0, 4, 2, 128, None, None, 1e-6, None, 16, 0, None, None, None, -1, 4, 8, 16, 0, None, None,
                               None, None, None, None) == lm_abi.INVALID_ARG
    assert lib.sl_paged_attention(None, None, None, None, None, 0, None, None, 0, 4, 2, 128, 4, 8, 16, 0.1, None, None, None, 0,
                                  None) == lm_abi.OK
    assert lib.sl_linear_block_fp8(None, None, None, None, None, 0, 128, 256, None, 0, None) == lm_abi.OK


@gpu
@needs_cuda
def test_attention_refuses_a_workspace_that_does_not_fit():
    q = torch.zeros(2, 4, 128, dtype=BF, device="cuda")
    cache = torch.zeros(4, 2, 16, 128, dtype=BF, device="cuda")
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    good = lm_abi.attention_workspace(4, 2, 128)
    for bad in (1 << 24, good.cpu(), good.float(), good[:-16], good[::2]):
        with pytest.raises(LmError):
            lm_abi.paged_attention(q, cache, cache, None, None, table, lens, 0.1, workspace=bad)
    lm_abi.paged_attention(q, cache, cache, None, None, table, lens, 0.1, workspace=good)
    clean()


def test_few_workspaces_are_kept(monkeypatch):
    """One a stream and kind for streams in use, but not one for every stream that ever was."""
    stream = [0]
    monkeypatch.setattr(lm_abi, "_workspaces", {})
    monkeypatch.setattr(lm_abi, "attention_workspace", lambda *a: object())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: stream[0], raising=False)
    kinds = [(8, 1, 64), (8, 1, 128), (16, 1, 64), (16, 1, 128)]
    first = [lm_abi._stream_workspace(*kind, 0) for kind in kinds]
    assert len({id(w) for w in first}) == 4
    assert all(lm_abi._stream_workspace(*kind, 0) is w for kind, w in zip(kinds, first))
    for stream[0] in range(1, 100):
        one = lm_abi._stream_workspace(8, 1, 64, 0)
        assert lm_abi._stream_workspace(8, 1, 64, 0) is one
    assert len(lm_abi._workspaces) == lm_abi._MOST_WORKSPACES


@gpu
@needs_cuda
def test_wrappers_of_no_sequences():
    def table(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")

    kc, vc = (torch.zeros(4, 2, 16, 128, dtype=BF, device="cuda") for _ in range(2))
    qkv = torch.zeros(0, 8 * 128, dtype=BF, device="cuda")
    q = lm_abi.append_paged(qkv, 4, 2, None, None, 1e-6, rope_table(16, 128), "halves", None, table(0), table(0, 3), kc, vc)
    assert q.shape == (0, 4, 128)
    assert lm_abi.paged_attention(q, kc, vc, None, None, table(0, 3), table(0), 0.1).shape == (0, 4, 128)
    with pytest.raises(LmError):
        lm_abi.append_paged(torch.zeros(1, 8 * 128, dtype=BF, device="cuda"), 4, 2, None, None, 1e-6, rope_table(16, 128), "halves",
                            table(1), table(1), table(0, 3), kc, vc)
    clean()


def test_warps_come_together_before_a_cluster_barrier():
    """The aligned barrier instructions are undefined for a warp whose lanes are apart."""
    lines = [line.split("//")[0].strip() for line in open(lm_abi.HERE + "/csrc/lm/sl_linear.cu")]
    code = [line for line in lines if line]
    at = [i for i, line in enumerate(code) if "cluster_barrier()" in line]
    assert at and code.count("cluster_sync();") >= 4
    for i in at:  # a __syncwarp() with nothing after it that parts the lanes
        before = code[max(0, i - 3):i]
        assert "__syncwarp();" in before
        assert not set(before[before.index("__syncwarp();") + 1:]) - {"sc::tc_fence_before();", "if (parts > 1) {"}


def test_no_load_is_promised_to_be_constant():
    """The kernels start before the one ahead of them has written their inputs: a read-only load may be moved above the wait."""
    import glob
    import re
    for path in glob.glob(lm_abi.HERE + "/csrc/lm/*"):
        code = re.sub(r"//[^\n]*", "", open(path).read())
        for word in ("__restrict", "__ldg", "global.nc"):
            assert word not in code, (path, word)


def test_copies_in_flight_are_drained_after_a_wait_that_gave_up(tmp_path):
    """The order of a warp's copies (sl_ring.cuh) on the host, against a model of the slots' barriers: whenever a wait gives
    up, the drain waits for every copy still on its way, from the one that was waited for on, each with its phase's parity."""
    (tmp_path / "ring.cc").write_text(r"""
#include <cstdio>
#include <deque>
#include "sl_ring.cuh"
template <int kSlots>
bool run(unsigned seed, int ahead) {
  for (int stop = 0; stop < 60; ++stop) {
    sl::Ring<kSlots> order;
    unsigned used[kSlots] = {}, random = seed * 7919u + stop;
    std::deque<unsigned> flight;  // the slots of the copies on their way
    unsigned next = 0;
    for (int taken = 0;;) {
      random = random * 1664525u + 1013904223u;
      if (flight.size() < static_cast<size_t>(ahead) && (flight.empty() || random >> 31)) {
        if (order.fill != next) return false;
        flight.push_back(next);
        next = (next + 1) % kSlots;
        order.filled();
        continue;
      }
      if (order.take != flight.front() || order.parity() != (used[flight.front()] & 1)) return false;
      if (taken++ == stop) break;  // this wait gives up
      ++used[flight.front()];
      flight.pop_front();
      order.taken();
    }
    bool good = true;
    order.drain([&](uint32_t slot, uint32_t parity) {
      good = good && !flight.empty() && slot == flight.front() && parity == (used[slot]++ & 1);
      if (!flight.empty()) flight.pop_front();
    });
    if (!good || !flight.empty()) return false;
  }
  return true;
}
int main() {
  for (unsigned seed = 0; seed < 50; ++seed)
    for (int ahead = 1; ahead <= 8; ++ahead)
      if ((ahead <= 2 && !run<2>(seed, ahead)) || (ahead <= 3 && !run<3>(seed, ahead)) || (ahead <= 4 && !run<4>(seed, ahead)) ||
          !run<8>(seed, ahead))
        return 1;
  std::puts("ok");
}
""")
    source = lm_abi.HERE + "/csrc/lm"
    subprocess.run(["g++", "-std=c++17", "-I", source, "-x", "c++", str(tmp_path / "ring.cc"), "-o", str(tmp_path / "ring")], check=True)
    assert subprocess.run([str(tmp_path / "ring")], capture_output=True, text=True).stdout == "ok\n"
    # the attention keeps its copies in that order, and drains them where its waits give up
    text = open(source + "/sl_attention.cu").read()
    assert "Ring<kSlots> order" in text and "if (gave_up) order.drain(" in text and "phases ^=" not in text


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 128)
    with pytest.raises(LmError):
        lm_abi.rms_norm_quantize(x)
    with pytest.raises(LmError):
        lm_abi.linear_block_fp8(x.to(F8), x, x.to(F8), x)
    with pytest.raises(LmError):
        lm_abi.paged_attention(x, x, x, None, None, x, x, 1.0)
    with pytest.raises(LmError):
        lm_abi.append_paged(x, 1, 1, None, None, 1e-6, x, "halves", None, x, x, x, x)


@gpu
@needs_cuda
def test_wrappers_refuse_what_does_not_fit():
    x = torch.zeros(4, 256, device="cuda")
    with pytest.raises(LmError):
        lm_abi.rms_norm_quantize(x[:, :128])                              # strides
    with pytest.raises(LmError):
        lm_abi.rms_norm_quantize(x.half())
    with pytest.raises(LmError):
        lm_abi.rms_norm_quantize(x, x_out=torch.empty_like(x))           # x_out without delta
    with pytest.raises(LmError):
        lm_abi.rms_norm_quantize(x, delta=x[:2])
    c, s, w = x.to(F8), torch.ones(4, 2, device="cuda"), torch.zeros(130, 256, device="cuda").to(F8)
    with pytest.raises(LmError):
        lm_abi.linear_block_fp8(c, s, w, torch.ones(1, 2, device="cuda"))  # two blocks of rows
    q = torch.zeros(2, 6, 128, dtype=BF, device="cuda")
    cache = torch.zeros(4, 4, 16, 128, dtype=BF, device="cuda")
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(LmError):
        lm_abi.paged_attention(q, cache, cache, None, None, table, lens, 1.0)  # 4 does not divide 6
    with pytest.raises(LmError):
        lm_abi.paged_attention(q, cache[:, :2], cache[:, :2], None, None, table, lens, 1.0)
    with pytest.raises(LmError):
        lm_abi.paged_attention(q, cache[:, :2].contiguous().to(F8), cache[:, :2].contiguous().to(F8), None, None, table, lens, 1.0)
    with pytest.raises(LmError):
        lm_abi.paged_attention(q, cache[:, :2].contiguous(), cache[:, :2].contiguous(), None, None, table, lens.long(), 1.0)
    clean()


# ------------------------------------------------------------------------------------------------ norm + quantization


def scale_ref(y):
    return (y.abs().amax(-1) / 448.0).clamp_min(1e-30)


def check_codes(codes, scales, y):
    """Codes and scales of rows y (64-bit): scales within 3e-6, codes within half a step of y / s."""
    rows, d = y.shape
    for i in range(scales.shape[1]):
        part = y[:, 128 * i:128 * i + 128]
        s = scale_ref(part)
        # fp32: at most 80 additions deep in the sum of squares (halved by the root) and 8 further roundings
        assert float(((scales[:, i].double() - s).abs() / s).max()) <= 3e-6
        want = part / s[:, None]
        off = (codes[:, 128 * i:128 * i + 128].double() - want).abs()
        assert float((off / torch.clamp(want.abs() * 2.0 ** -4, min=2.0 ** -10)).max()) <= 1 + 2e-4


@gpu
@needs_cuda
@pytest.mark.parametrize("rows,d", [(1, 16), (3, 144), (5, 128), (7, 2560), (130, 3840), (2, 8208), (1, 16384), (600, 4096)])
@pytest.mark.parametrize("stream", [BF, torch.float32])
@pytest.mark.parametrize("delta", [None, BF, torch.float32])
def test_rms_norm_quantize(rows, d, stream, delta):
    g = gen(rows * d)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 3).to(stream)
    dx = None if delta is None else torch.randn(rows, d, generator=g, device="cuda").to(delta)
    w = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    keep = x.clone()
    out = None if delta is None else torch.empty_like(x)
    xo, codes, scales = lm_abi.rms_norm_quantize(x, dx, w, 1e-5, out)
    z = keep.double() + (0 if dx is None else dx.double())
    assert torch.equal(x, keep)
    assert torch.equal(xo, (keep.float() + (0 if dx is None else dx.float())).to(stream))
    y = z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * w.double()
    check_codes(codes, scales, y)
    again = lm_abi.rms_norm_quantize(x, dx, w, 1e-5)  # in place, the same codes
    assert torch.equal(again[1].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[2], scales)
    assert again[0] is x and torch.equal(x, xo)
    _, codes, scales = lm_abi.rms_norm_quantize(keep, norm=False)
    check_codes(codes, scales, keep.double())
    clean()


@gpu
@needs_cuda
def test_norm_of_zeros_and_of_non_finite_blocks():
    x = torch.zeros(4, 400, device="cuda")
    x[1, 5], x[1, 130] = math.nan, 3.0
    x[2, 300], x[2, 301] = -math.inf, 1.0
    x[3] = 1e-38
    _, codes, scales = lm_abi.rms_norm_quantize(x, norm=False)
    c = codes.float()
    assert torch.equal(scales[0], torch.full((4,), 1e-30, device="cuda")) and not c[0].any()
    assert math.isnan(float(scales[1, 0])) and float(scales[1, 1]) == pytest.approx(3 / 448) and float(c[1, 130]) == 448
    assert math.isinf(float(scales[2, 2])) and math.isnan(float(c[2, 300])) and float(c[2, 301]) == 0
    assert float(scales[2, 3]) == pytest.approx(1e-30)
    assert torch.equal(scales[3], torch.full((4,), 1e-30, device="cuda"))  # below the floor: codes of 1e-38 / 1e-30
    assert not c[3].any()
    _, codes, scales = lm_abi.rms_norm_quantize(x[:1], eps=1e-6)
    assert not codes.float().any() and torch.equal(scales[0], torch.full((4,), 1e-30, device="cuda"))
    empty = lm_abi.rms_norm_quantize(torch.empty(0, 256, device="cuda"))
    assert empty[1].shape == (0, 256)
    clean()


# ------------------------------------------------------------------------------------------------ the append


def rope_table(max_pos, dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    ang = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def paged(seqs, width, spare=2, seed=0):
    pages = seqs * width + spare
    perm = torch.randperm(pages, generator=gen(seed), device="cuda")[: seqs * width].to(torch.int32)
    return perm.view(seqs, width).contiguous(), pages


def head_ref(x, norm, cs, pairs, eps=1e-6):
    """x [tokens, heads, dim] in 64 bits, normalised and rotated."""
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    out = torch.empty_like(x)
    half = x.shape[-1] // 2
    first, second = (slice(0, None, 2), slice(1, None, 2)) if pairs == "adjacent" else (slice(0, half), slice(half, None))
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    return out


@gpu
@needs_cuda
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 3, 3), (128, 5, 1)])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_append_paged(dim, heads, kv_heads, pairs, e4m3, norm):
    g = gen(dim + heads)
    size, width, seqs = 24, 4, 3
    table, pages = paged(seqs, width)
    spans = [(0, 31), (90, 6), (24, 1)]  # page borders, the last slot, a single token
    seq = torch.tensor([i for i, (_, n) in enumerate(spans) for _ in range(n)] + [1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([p + j for p, n in spans for j in range(n)] + [-1], dtype=torch.int32, device="cuda")
    tokens = len(seq)
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g, device="cuda").to(BF)
    qkv[4] = 0
    freqs = rope_table(width * size, dim)
    nq = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda") if norm else None
    nk = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda") if norm else None
    kind = F8 if e4m3 else BF
    kc, vc = (torch.randn(pages, kv_heads, size, dim, generator=g, device="cuda").to(kind) for _ in range(2))
    ks, vs = (torch.rand(pages, kv_heads, size, generator=g, device="cuda") for _ in range(2)) if e4m3 else (None, None)
    raw = torch.uint8 if e4m3 else torch.int16
    before = [t if t is None else t.clone() for t in (kc, vc, ks, vs)]
    q = lm_abi.append_paged(qkv, heads, kv_heads, nq, nk, 1e-6, freqs, pairs, seq, pos, table, kc, vc, ks, vs)
    live = pos >= 0
    x = qkv.double().view(tokens, heads + 2 * kv_heads, dim)
    cs = freqs[pos.clamp_min(0).long()]
    qr, kr, vr = head_ref(x[:, :heads], nq, cs, pairs), head_ref(x[:, heads:heads + kv_heads], nk, cs, pairs), x[:, heads + kv_heads:]

    def near(got, ref):  # one bf16 rounding; fp32: about 20 roundings of values up to the head's largest
        room = U * 1.01 * ref.abs() + 2e-6 * ref.abs().amax(-1, keepdim=True) + 1e-30
        assert float(((got.double() - ref).abs() / room).max()) <= 1

    near(q[live], qr[live])
    assert not q[~live].any()
    touched = torch.zeros(pages, size, dtype=torch.bool, device="cuda")
    page, slot = table[seq.long(), pos.clamp_min(0).long() // size].long()[live], (pos.long() % size)[live]
    touched[page, slot] = True
    for cache, scale, old, old_scale, ref in ((kc, ks, before[0], before[2], kr), (vc, vs, before[1], before[3], vr)):
        same = (cache.view(raw) == old.view(raw)).all(-1)
        assert bool(same.transpose(1, 2)[~touched].all())
        got = cache.view(raw)[page, :, slot].view(kind)
        if e4m3:
            assert torch.equal(scale.transpose(1, 2)[~touched], old_scale.transpose(1, 2)[~touched])
            r = ref[live].reshape(-1, dim)
            check_codes(got.reshape(-1, dim).contiguous(), scale[page, :, slot].reshape(-1, 1), r) if dim == 128 else None
            s = scale_ref(r)
            assert float(((scale[page, :, slot].reshape(-1).double() - s).abs() / s).max()) <= 3e-6
        else:
            near(got, ref[live])
    if not e4m3:
        assert torch.equal(vc[page, :, slot], qkv.view(tokens, -1, dim)[live][:, heads + kv_heads:])
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_append_writes_zeros_for_padding(dim, pairs):
    """Whatever there is to be multiplied with: eps 0 (0 * rsqrt(0) is NaN), NaN in the padded rows, in the rotation table's
    first row, for padding and for positions past the table."""
    size = 16
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    qkv = torch.ones(3, 4 * dim, dtype=BF, device="cuda")
    qkv[1:] = math.nan
    freqs = rope_table(20, dim)
    freqs[0] = math.nan
    norm = torch.ones(dim, device="cuda")
    kc, vc = (torch.zeros(2, 1, size, dim, dtype=BF, device="cuda") for _ in range(2))
    seq = torch.zeros(3, dtype=torch.int32, device="cuda")
    pos = torch.tensor([5, -1, 20], dtype=torch.int32, device="cuda")
    q = lm_abi.append_paged(qkv, 2, 1, norm, norm, 0.0, freqs, pairs, seq, pos, table, kc, vc)
    assert lm_abi.errors()[0] == lm_abi.OUT_OF_RANGE  # position 20
    assert not q[1:].any() and bool(q[0].isfinite().all())
    assert int(vc.any(-1).sum()) == 1 and int(kc.any(-1).sum()) == 1
    clean()


def check_cache_rows(codes, scales, y):
    """Rows of an e4m3 cache against 64-bit heads y [rows, dim]: a head's fp32 work is within 2e-6 of its largest value, which
    is code 448, so a code is within half a step (2^-4 of a normal code, 2^-10 of a subnormal one) and 448 * 2e-6 < 1e-3."""
    s = scale_ref(y)
    assert float(((scales.double() - s).abs() / s).max()) <= 3e-6
    want = y / s[:, None]
    assert float(((codes.double() - want).abs() - torch.clamp(want.abs() * 2.0 ** -4, min=2.0 ** -10)).max()) <= 1e-3


@gpu
@needs_cuda
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("norm", [False, True])
def test_append_codes_of_an_8_bit_cache(dim, pairs, norm):
    """Every code of keys and values, heads of both sizes, channels of very different sizes."""
    g = gen(dim)
    heads, kv_heads, size, seqs, width = 6, 3, 16, 4, 3
    table, pages = paged(seqs, width, seed=dim)
    pos = torch.tensor([0, 15, 16, 47], dtype=torch.int32, device="cuda")
    qkv = torch.randn(seqs, heads + 2 * kv_heads, dim, generator=g, device="cuda")
    qkv = (qkv * 10.0 ** (3 * torch.rand(dim, generator=g, device="cuda") - 2)).to(BF).view(seqs, -1)
    freqs = rope_table(width * size, dim)
    nq, nk = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda") if norm else None for _ in range(2))
    kc, vc = (torch.zeros(pages, kv_heads, size, dim, device="cuda").to(F8) for _ in range(2))
    ks, vs = (torch.zeros(pages, kv_heads, size, device="cuda") for _ in range(2))
    lm_abi.append_paged(qkv, heads, kv_heads, nq, nk, 1e-6, freqs, pairs, None, pos, table, kc, vc, ks, vs)
    x = qkv.double().view(seqs, -1, dim)
    k, v = head_ref(x[:, heads:heads + kv_heads], nk, freqs[pos.long()], pairs), x[:, heads + kv_heads:]
    page, slot = table[torch.arange(seqs, device="cuda"), pos.long() // size].long(), pos.long() % size
    for cache, scale, ref in ((kc, ks, k), (vc, vs, v)):
        got = cache.view(torch.uint8)[page, :, slot].view(F8)
        check_cache_rows(got.reshape(-1, dim), scale[page, :, slot].reshape(-1), ref.reshape(-1, dim))
    clean()


@gpu
@needs_cuda
def test_append_reports_what_is_out_of_range():
    dim, size = 128, 16
    table = torch.tensor([[0, 1], [2, 9]], dtype=torch.int32, device="cuda")  # page 9 of 4
    qkv = torch.ones(4, 3 * dim, dtype=BF, device="cuda")
    kc = torch.zeros(4, 1, size, dim, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    freqs = rope_table(64, dim)

    def call(seq, pos):
        n = len(pos)
        lm_abi.append_paged(qkv[:n], 1, 1, None, None, 1e-6, freqs, "halves", torch.tensor(seq, dtype=torch.int32, device="cuda"),
                            torch.tensor(pos, dtype=torch.int32, device="cuda"), table, kc, vc)
        return lm_abi.errors()

    assert call([1], [16])[0] == lm_abi.OUT_OF_RANGE       # its page
    assert call([2], [3])[0] == lm_abi.OUT_OF_RANGE        # its sequence
    assert call([-1], [3])[0] == lm_abi.OUT_OF_RANGE
    assert call([0], [32])[0] == lm_abi.OUT_OF_RANGE       # past the table
    assert call([0], [64])[0] == lm_abi.OUT_OF_RANGE       # past the rotation table
    assert not kc.any() and not vc.any()
    assert call([0, 1], [31, 15]) == (lm_abi.OK, 0)
    assert bool(vc[1, 0, 15].any()) and bool(vc[2, 0, 15].any()) and int(vc.any(-1).sum()) == 2
    q = lm_abi.append_paged(qkv[:0], 1, 1, None, None, 1e-6, freqs, "halves", None, table.view(-1)[:0], table, kc, vc)
    assert q.shape == (0, 1, dim)
    clean()


# ------------------------------------------------------------------------------------------------ the attention


def make_cache(g, pages, kv_heads, size, dim, e4m3):
    out = []
    for _ in range(2):
        x = torch.randn(pages, kv_heads, size, dim, generator=g, device="cuda")
        if e4m3:
            s = scale_ref(x)
            out.append(((x / s[..., None]).clamp(-448, 448).to(F8), s.float()))
        else:
            out.append((x.to(BF), None))
    return out


def poison(cache, scale, table, lengths):
    """NaN wherever no token of a sequence lies."""
    pages, _, size, _ = cache.shape
    used = torch.zeros(pages, size, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        used[table[b].long()[t // size], t % size] = True
    if scale is None:
        cache.transpose(1, 2)[~used] = math.nan
    else:
        cache.view(torch.uint8).transpose(1, 2)[~used] = 0x7F
        scale.transpose(1, 2)[~used] = math.nan


def rows_of(cache, scale, table, b, n, head):
    t = torch.arange(n, device="cuda")
    size = cache.shape[2]
    page, slot = table[b].long()[t // size], t % size
    if scale is None:
        return cache[page, head, slot].double()
    return cache.view(torch.uint8)[page, head, slot].view(F8).double() * scale[page, head, slot].double()[:, None]


def check_attention(q, k, v, table, lengths, scale, out, lse):
    (kc, ks), (vc, vs) = k, v
    heads, kv_heads = q.shape[1], kc.shape[1]
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any() and bool((lse[b] == -math.inf).all())
            continue
        for h in range(kv_heads):
            of = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            kk, vv = rows_of(kc, ks, table, b, n, h), rows_of(vc, vs, table, b, n, h)
            s = q[b, of].double() @ kk.t() * scale
            p = torch.softmax(s, -1)
            ref, mass = p @ vv, p @ vv.abs()
            # p rounded to bf16 for the product and the output rounded to bf16; fp32 scores within 1e-5 of a weight
            room = U * 1.01 * (mass + ref.abs()) + 4e-5 * mass + 1e-30
            assert float(((out[b, of].double() - ref).abs() / room).max()) <= 1, (b, n, h)
            # fp32 accumulation of head_dim products, then exp2 and log2
            assert float((lse[b, of].double() - torch.logsumexp(s, -1)).abs().max()) <= 1e-4, (b, n, h)


@gpu
@needs_cuda
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads,size,lengths", [
    (128, 8, 2, 16, [1, 0, 15, 16, 17, 63, 64, 65, 128, 1000]),
    (128, 1, 1, 1, [37, 1]),
    (128, 5, 5, 24, [100, 4097, 3]),
    (128, 32, 2, 64, [700, 0, 0, 129]),          # 16 query heads a key-value head
    (128, 12, 1, 8, [333]),                       # 12: the second tile of 8 is half empty
    (128, 40, 1, 16, [257, 64]),                  # 40: three tiles of 16, the last half empty
    (64, 8, 1, 16, [1, 2, 100, 0, 2049]),
    (64, 14, 7, 24, [511, 31]),
    (64, 24, 2, 128, [60, 1025]),
    (128, 4, 4, 16, [20000, 5, 0, 3000]),
])
def test_paged_attention(e4m3, dim, heads, kv_heads, size, lengths):
    g = gen(dim * heads + size)
    width = max(1, -(-max(lengths) // size)) + 1
    table, pages = paged(len(lengths), width, seed=size)
    k, v = make_cache(g, pages, kv_heads, size, dim, e4m3)
    for c in (k, v):
        poison(*c, table, lengths)
    q = (torch.randn(len(lengths), heads, dim, generator=g, device="cuda") * 2).to(BF)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    lse = torch.empty(len(lengths), heads, device="cuda")
    scale = 1 / math.sqrt(dim)
    out = lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, scale, lse=lse)
    check_attention(q, k, v, table, lengths, scale, out, lse)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    for _ in range(3):  # the workspace is ready for the next call, and every call gives the same bits
        lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, scale, again, lse2)
        assert torch.equal(again.view(torch.int16), out.view(torch.int16)) and torch.equal(lse, lse2)
    assert torch.equal(lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, scale), out)  # without lse
    clean()


@gpu
@needs_cuda
def test_attention_of_many_sequences():
    """More sequences than one launch takes, most of them short, some empty; another stream than the inputs'."""
    g = gen(5)
    batch, heads, kv_heads, dim, size = 1500, 4, 2, 128, 16
    lengths = [(7 * i) % 50 for i in range(batch)]
    table, pages = paged(batch, 4)
    k, v = make_cache(g, pages, kv_heads, size, dim, False)
    q = torch.randn(batch, heads, dim, generator=g, device="cuda").to(BF)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    lse = torch.empty(batch, heads, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = lm_abi.paged_attention(q, k[0], v[0], None, None, table, lens, 0.1, lse=lse)
    torch.cuda.current_stream().wait_stream(side)
    some = list(range(0, 40)) + list(range(1000, 1060)) + [batch - 1]
    check_attention(q[some], k, v, table[some], [lengths[i] for i in some], 0.1, out[some], lse[some])
    assert lm_abi.paged_attention(q[:0], k[0], v[0], None, None, table[:0], lens[:0], 0.1).shape == (0, heads, dim)
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads", [(64, 8), (64, 7), (128, 8), (64, 16), (128, 16)])
@pytest.mark.parametrize("long,others", [(80000, 0), (131072, 50)])
def test_one_long_context_among_many_sequences(dim, heads, e4m3, long, others):
    """One key-value head and 64 sequences of which one holds nearly all the tokens: its context is cut over nearly every
    CTA of the launch, all of whose parts the last one to arrive adds."""
    g = gen(dim + heads + others)
    size, batch = 64, 64
    lengths = [others] * batch
    lengths[batch // 3] = long
    width = -(-long // size)
    pages = width + batch + 3
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(batch, width, dtype=torch.int32, device="cuda")
    table[:, 0] = perm[width:width + batch]
    table[batch // 3] = perm[:width]
    k, v = make_cache(g, pages, 1, size, dim, e4m3)
    q = (torch.randn(batch, heads, dim, generator=g, device="cuda") * 2).to(BF)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    lse, lse2 = torch.empty(batch, heads, device="cuda"), torch.empty(batch, heads, device="cuda")
    scale = 1 / math.sqrt(dim)
    out = lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, scale, lse=lse)
    check_attention(q, k, v, table, lengths, scale, out, lse)
    again = lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, scale, lse=lse2)
    assert torch.equal(again, out) and torch.equal(lse, lse2)
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("dim", [64, 128])
def test_e4m3_cache_decodes_every_code(dim):
    """A context of one token gives its value row: all finite codes, exactly, in v and (as a sum of one) in k."""
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8, device="cuda")
    n = -(-len(codes) // dim)
    rows = torch.zeros(n * dim, dtype=torch.uint8, device="cuda")
    rows[: len(codes)] = codes
    vc = rows.view(n, 1, 1, dim).view(F8)
    ones = torch.ones(n, 1, 1, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    lens = torch.ones(n, dtype=torch.int32, device="cuda")
    q = torch.zeros(n, 1, dim, dtype=BF, device="cuda")
    out = lm_abi.paged_attention(q, vc, vc, ones, ones, table, lens, 1.0)
    assert torch.equal(out.float().view(-1), vc.float().view(-1))
    for d in range(dim):  # k: q picks one dim, the score is the code
        q.zero_()
        q[:, :, d] = 1
        lse = torch.empty(n, 1, device="cuda")
        lm_abi.paged_attention(q, vc, vc, ones, ones, table, lens, 1.0, lse=lse)
        want = vc.float()[:, 0, 0, d]
        assert float((lse[:, 0] - want).abs().max()) <= 448 * 2.0 ** -22  # log2(e) there and ln 2 back
    clean()


@gpu
@needs_cuda
def test_attention_extremes():
    """Scores far apart, equal scores, infinities in v, a NaN in k; offsets past 2^32 bytes of the cache."""
    g = gen(9)
    dim, size = 128, 16
    table = torch.tensor([[3, 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    kc = torch.zeros(4, 1, size, dim, dtype=BF, device="cuda")
    vc = torch.randn(4, 1, size, dim, generator=g, device="cuda").to(BF)
    q = torch.ones(1, 1, dim, dtype=BF, device="cuda")
    lse = torch.empty(1, 1, device="cuda")
    v = rows_of(vc, None, table, 0, 20, 0)
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0, lse=lse)
    assert float((out[0, 0].double() - v.mean(0)).abs().max()) <= 2 * U * float(v.abs().max())
    assert float(lse) == pytest.approx(math.log(20), abs=1e-6)
    kc[1, 0, 3] = 300.0  # token 19: a score of 38400 against zeros
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0, lse=lse)
    assert torch.equal(out[0, 0], vc[1, 0, 3]) and float(lse) == 38400
    kc[1, 0, 3] = -300.0
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0, lse=lse)
    assert float(lse) == pytest.approx(math.log(19), abs=1e-6)
    vc[3, 0, 0, 5], vc[3, 0, 1, 6] = math.inf, math.nan
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0)
    assert float(out[0, 0, 5]) == math.inf and math.isnan(float(out[0, 0, 6])) and bool(out[0, 0, 7:].isfinite().all())
    kc[3, 0, 2, 0] = math.nan
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0, lse=lse)
    assert bool(out.isnan().all()) and math.isnan(float(lse))
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 8, 2), (128, 32, 2), (64, 32, 2)])
def test_attention_loses_no_more_than_its_output_rounding(dim, heads, kv_heads, e4m3):
    """p's own rounding on the way to the product with v: upper 8 bits and the rest rounded to 8 (2^-7 2^-8 of p at most) over a
    bf16 cache, f16 (2^-11, twice as much for the scale's product) over an e4m3 one.  Values that nearly cancel show it."""
    g = gen(dim + heads)
    lengths = [2, 3, 5, 40, 700]
    table, pages = paged(len(lengths), 45)
    k, v = make_cache(g, pages, kv_heads, 16, dim, e4m3)
    q = (torch.randn(len(lengths), heads, dim, generator=g, device="cuda") * 2).to(BF)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = lm_abi.paged_attention(q, k[0], v[0], k[1], v[1], table, lens, 1 / math.sqrt(dim))
    for b, n in enumerate(lengths):
        for h in range(kv_heads):
            of = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            kk, vv = rows_of(*k, table, b, n, h), rows_of(*v, table, b, n, h)
            p = torch.softmax(q[b, of].double() @ kk.t() / math.sqrt(dim), -1)
            ref, mass = p @ vv, p @ vv.abs()
            room = U * 1.01 * ref.abs() + (4e-5 + (2.0 ** -10 if e4m3 else 2.0 ** -15)) * mass
            assert float(((out[b, of].double() - ref).abs() / room).max()) <= 1, (b, n, h)
    clean()


@gpu
@needs_cuda
def test_infinite_values_stay_infinite():
    """Whatever p is: 1, a power of two, all of its bits set, tiny."""
    dim, size = 128, 16
    q = torch.zeros(1, 1, dim, dtype=BF, device="cuda")
    q[..., 0] = 1
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([4], dtype=torch.int32, device="cuda")
    for far in (0.0, -1.0, -0.3, -7.7, -60.0):  # the second token's score below the first one's
        kc, vc = (torch.zeros(1, 1, size, dim, dtype=BF, device="cuda") for _ in range(2))
        kc[0, 0, :, 0] = 3
        kc[0, 0, 1, 0] = 3 + far
        vc[0, 0, 1, 3], vc[0, 0, 1, 4], vc[0, 0, 2, 5], vc[0, 0, 3, 6] = math.inf, -math.inf, math.inf, -math.inf
        out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 1.0)[0, 0]
        assert [float(out[i]) for i in (3, 4, 5, 6)] == [math.inf, -math.inf, math.inf, -math.inf], far
        assert not out[:3].any() and not out[7:].any()
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("n", [1, 20, 3000, 40000])
def test_scores_that_are_all_minus_infinity(n):
    """Zeros and lse -inf, in one warp's step and over a context cut between CTAs."""
    dim, size = 128, 16
    width = -(-n // size)
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    kc, vc = (torch.randn(width, 1, size, dim, generator=gen(n), device="cuda").to(BF) for _ in range(2))
    kc[..., 7] = -math.inf
    q = torch.ones(1, 2, dim, dtype=BF, device="cuda")
    lse = torch.empty(1, 2, device="cuda")
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.05, lse=lse)
    assert not out.any() and bool((lse == -math.inf).all())
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("n", [1, 20, 3000, 40000])
def test_a_score_of_infinity(n):
    """+inf among finite scores: what the formula gives, lse +inf and inf / inf = NaN.  -inf for the other head: left out."""
    g = gen(n)
    dim, size = 128, 16
    width = -(-n // size)
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    kc, vc = (torch.randn(width, 1, size, dim, generator=g, device="cuda").to(BF) for _ in range(2))
    q = torch.randn(1, 2, dim, generator=g, device="cuda").to(BF)
    q[0, 0, 0], q[0, 1, 0] = 1, -1
    kc[(n // 2) // size, 0, (n // 2) % size, 0] = math.inf
    lse = torch.empty(1, 2, device="cuda")
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.05, lse=lse)
    assert bool(out[0, 0].isnan().all()) and float(lse[0, 0]) == math.inf
    keep = [i for i in range(n) if i != n // 2]
    if not keep:
        assert not out[0, 1].any() and float(lse[0, 1]) == -math.inf
    else:
        kk, vv = (rows_of(c, None, table, 0, n, 0)[keep] for c in (kc, vc))
        s = q[0, 1:].double() @ kk.t() * 0.05
        p = torch.softmax(s, -1)
        ref, mass = p @ vv, p @ vv.abs()
        assert float(((out[0, 1:].double() - ref).abs() / (U * 1.01 * (mass + ref.abs()) + 4e-5 * mass)).max()) <= 1
        assert float((lse[0, 1:].double() - torch.logsumexp(s, -1)).abs().max()) <= 1e-4
    clean()


@gpu
@needs_cuda
def test_cache_beyond_four_gigabytes():
    dim, size, kv_heads = 128, 64, 8
    pages = (5 << 30) // (size * kv_heads * dim * 2)
    kc = torch.zeros(pages, kv_heads, size, dim, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.tensor([[pages - 1, 0], [pages - 2, pages - 3]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([63, 64], dtype=torch.int32, device="cuda")
    g = gen(11)
    qkv = torch.randn(2, (16 + 16) * dim, generator=g, device="cuda").to(BF)
    q = lm_abi.append_paged(qkv, 16, 8, None, None, 1e-6, rope_table(128, dim), "halves", None, pos, table, kc, vc)
    assert torch.equal(vc[pages - 1, :, 63], qkv[0].view(-1, dim)[24:]) and torch.equal(vc[pages - 3, :, 0], qkv[1].view(-1, dim)[24:])
    lens = torch.tensor([64, 65], dtype=torch.int32, device="cuda")
    lse = torch.empty(2, 16, device="cuda")
    out = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.09, lse=lse)
    check_attention(q, (kc, None), (vc, None), table, [64, 65], 0.09, out, lse)
    clean()


@gpu
@needs_cuda
def test_attention_reports_what_is_out_of_range():
    g = gen(3)
    (kc, _), (vc, _) = make_cache(g, 4, 1, 16, 128, False)
    q = torch.randn(1, 2, 128, generator=g, device="cuda").to(BF)
    good = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([20], dtype=torch.int32, device="cuda")
    want = lm_abi.paged_attention(q, kc, vc, None, None, good, n * 0 + 16, 0.1)
    for bad in (-1, 4, 2 ** 31 - 1):
        out = lm_abi.paged_attention(q, kc, vc, None, None, torch.tensor([[0, bad]], dtype=torch.int32, device="cuda"), n, 0.1)
        assert lm_abi.errors()[0] == lm_abi.OUT_OF_RANGE
        assert float((out - want).abs().max()) <= 2 * U * float(vc.abs().max())  # the tokens of that page are left out
    lm_abi.paged_attention(q, kc, vc, None, None, good, n * 0 + 33, 0.1)  # past the table
    assert lm_abi.errors()[0] == lm_abi.OUT_OF_RANGE
    lm_abi.paged_attention(q, kc, vc, None, None, good, n * 0 - 1, 0.1)
    assert lm_abi.errors()[0] == lm_abi.OUT_OF_RANGE
    lm_abi.paged_attention(q, kc, vc, None, None, good, n, 0.1)
    clean()


@gpu
@needs_cuda
def test_attention_in_a_graph():
    """Captured without a warm-up: the graph zeroes a workspace of its own, and eager calls keep theirs."""
    g = gen(4)
    table, pages = paged(3, 30)
    (kc, _), (vc, _) = make_cache(g, pages, 2, 16, 128, False)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(BF)
    lens = torch.tensor([400, 30, 77], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    lm_abi.attention_workspace(8, 2, 128)  # loads the library before the capture
    lm_abi.errors()
    with torch.cuda.graph(graph):
        lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.1, out)
    want = lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.1)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    q.copy_(torch.randn(3, 8, 128, generator=g, device="cuda"))
    lens.copy_(torch.tensor([1, 480, 0]))
    graph.replay()
    assert torch.equal(out, lm_abi.paged_attention(q, kc, vc, None, None, table, lens, 0.1))
    clean()


# ------------------------------------------------------------------------------------------------ the product


def block_weight(g, n, k, scale=0.05):
    kb, nb = -(-k // 128), -(-n // 128)
    w = torch.randn(n, k, generator=g, device="cuda") * scale
    ws = torch.rand(nb, kb, generator=g, device="cuda") * 0.01 + 1e-3
    spread = ws.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return (w / spread).clamp(-448, 448).to(F8), ws


def check_product(codes, scales, w, ws, bias, y):
    (m, k), n = codes.shape, w.shape[0]
    a = codes.double() * scales.double().repeat_interleave(128, 1)[:, :k]
    b = w.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref, mass = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        ref = ref + bias.double()
        mass = mass + bias.double().abs()
    # fp32 sums of k products (an error of 1e-6 of the terms' sum), one rounding to the output's type
    room = 1e-6 * mass + (U * 1.01 * ref.abs() if y.dtype == BF else 0) + 1e-30
    assert float(((y.double() - ref).abs() / room).max()) <= 1


@gpu
@needs_cuda
@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 33, 64, 65, 127, 128, 129, 300, 1000])
@pytest.mark.parametrize("n,k", [(128, 128), (1, 16), (100, 48), (136, 144), (130, 1024), (384, 1040), (2560, 4096)])
def test_linear_block_fp8(m, n, k):
    g = gen(m * 7 + n)
    x = torch.randn(m, k, generator=g, device="cuda")
    _, codes, scales = lm_abi.rms_norm_quantize(x, norm=False)
    w, ws = block_weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda").to(BF)
    y = lm_abi.linear_block_fp8(codes, scales, w, ws, bias)
    check_product(codes, scales, w, ws, bias, y)
    out = torch.full((m, n), math.nan, device="cuda")
    lm_abi.linear_block_fp8(codes, scales, w, ws, None, out)
    check_product(codes, scales, w, ws, None, out)
    again = torch.empty_like(out)
    lm_abi.linear_block_fp8(codes, scales, w, ws, None, again)
    assert torch.equal(out, again)
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("m,n", [(150, 9727), (700, 5001), (700, 5002), (705, 5004), (700, 5008), (2001, 2567)])
def test_linear_rows_that_start_on_any_value(m, n):
    """Outputs whose rows start on 2, 4, 8 and 16 bytes, from both kernels, and nothing written past them."""
    g = gen(n)
    k = 1040
    _, codes, scales = lm_abi.rms_norm_quantize(torch.randn(m, k, generator=g, device="cuda"), norm=False)
    w, ws = block_weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda").to(BF)
    for dtype in (BF, torch.float32):
        room = torch.full((m * n + 4096,), -7.0, dtype=dtype, device="cuda")
        y = room[:m * n].view(m, n)
        lm_abi.linear_block_fp8(codes, scales, w, ws, bias, y)
        check_product(codes, scales, w, ws, bias, y)
        assert bool((room[m * n:] == -7.0).all())
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("m,n,k", [(500, 2567, 5040), (500, 2568, 5040), (300, 3882, 6160), (250, 2500, 9744), (250, 2496, 9744)])
def test_linear_with_k_shared_by_several_pairs(m, n, k):
    """Few tiles and a long K, shared unevenly by 2 to 4 pairs.  A part has no more blocks than the longest K above, and the
    parts add at most three roundings of 6e-8: the same bars."""
    g = gen(n + k)
    _, codes, scales = lm_abi.rms_norm_quantize(torch.randn(m, k, generator=g, device="cuda"), norm=False)
    w, ws = block_weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda").to(BF)
    for dtype in (BF, torch.float32):
        y, again = (torch.full((m, n), math.nan, dtype=dtype, device="cuda") for _ in range(2))
        lm_abi.linear_block_fp8(codes, scales, w, ws, bias, y)
        check_product(codes, scales, w, ws, bias, y)
        lm_abi.linear_block_fp8(codes, scales, w, ws, bias, again)
        assert torch.equal(y, again)
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("m", [3, 40, 500])
def test_linear_keeps_scales_apart_and_nan_in_its_row(m):
    """Scales of very different sizes (a block's partial product must not be rounded against another's), a NaN block."""
    g = gen(m)
    n, k = 300, 640
    codes = torch.randn(m, k, generator=g, device="cuda").to(F8)
    scales = 10.0 ** torch.randint(-6, 7, (m, 5), generator=g, device="cuda").float()
    w = torch.randn(n, k, generator=g, device="cuda").to(F8)
    ws = 10.0 ** torch.randint(-6, 7, (3, 5), generator=g, device="cuda").float()
    y = lm_abi.linear_block_fp8(codes, scales, w, ws, None, torch.empty(m, n, device="cuda"))
    check_product(codes, scales, w, ws, None, y)
    scales[1, 2] = math.nan
    y = lm_abi.linear_block_fp8(codes, scales, w, ws)
    assert bool(y[1].isnan().all()) and int(y.isnan().any(1).sum()) == 1
    assert lm_abi.linear_block_fp8(codes[:0], scales[:0], w, ws).shape == (0, n)
    clean()


@gpu
@needs_cuda
@pytest.mark.parametrize("m,n,k", [(1500, 2560, 1024), (1501, 2567, 1040), (500, 2560, 5040)])
def test_many_rows_keep_scales_apart_and_nan_in_its_row(m, n, k):
    """The same of the kernel of CTA pairs: whole tiles, rows that start on any value, K shared by several pairs."""
    g = gen(m + k)
    kb, nb = -(-k // 128), -(-n // 128)
    codes = torch.randn(m, k, generator=g, device="cuda").to(F8)
    scales = 10.0 ** torch.randint(-6, 7, (m, kb), generator=g, device="cuda").float()
    w = torch.randn(n, k, generator=g, device="cuda").to(F8)
    ws = 10.0 ** torch.randint(-6, 7, (nb, kb), generator=g, device="cuda").float()
    y = lm_abi.linear_block_fp8(codes, scales, w, ws, None, torch.empty(m, n, device="cuda"))
    check_product(codes, scales, w, ws, None, y)
    scales[257, kb - 1] = math.nan
    for dtype in (BF, torch.float32):
        y = lm_abi.linear_block_fp8(codes, scales, w, ws, None, torch.empty(m, n, dtype=dtype, device="cuda"))
        assert bool(y[257].isnan().all()) and int(y.isnan().any(1).sum()) == 1
    clean()
