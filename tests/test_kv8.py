"""8-bit KV cache: append and attention against plain implementations.

The quantiser is compared bit for bit with the same three fp32 operations in torch and, in 64 bits, with the definition
(half a code step); the attention with the 64-bit softmax over what the cache holds. Its error bound is worked out
from the data of each case: with S1 = max sum |q k| / sqrt(D), n keys and a 16-bit result,

    |o - o64| <= eps/2 |o64| + 2 max|v| (4 (D + 8) 2^-24 S1 + n 2^-24 + 2^-20)

The score of a key carries the split's remainder (2^-22 |q k|) and D + 8 roundings of fp32 sums; a weight's relative
error is that of the score on both sides of the quotient (twice, and twice for max - score), the exponential and the
split of the weight add less than 2^-20, the fp32 sum over n keys at most n 2^-24.

From 64 query rows of a kv head on, at a position known on the host, the weights are rounded to f16 once, 2^-12 of a
weight, and q where the result is bf16: 2^-12 of each of a score's terms, so 2^-12 S1 of a score, twice for the quotient.
The bound then has 2 max|v| (2^-12 + 2^-11 S1 for bf16) more.
"""

import math

import pytest
import torch

from tests._util import DTYPES, require_b200

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LIMIT = {"e4m3": 448.0, "int8": 127.0}


def quantise(x, code):
    """[..., 32, d] fp32 -> codes and scales with the documented operations."""
    a = x.abs().amax((-1, -2))
    fine = torch.isfinite(a)
    a = torch.where(fine, a, torch.ones_like(a)).clamp(min=2.0 ** -60)
    inv = a.reciprocal() * LIMIT[code]
    y = torch.where(fine[..., None, None], x * inv[..., None, None], torch.zeros_like(x))
    y = y.round().to(torch.int8) if code == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.where(fine, a / torch.full_like(a, LIMIT[code]), torch.full_like(a, math.nan))
    return y, scale


def rope(x, cos, sin, start):
    """Interleaved pairs of x [B, S, heads, d] rotated from position start[b] on."""
    at = start[:, None] + torch.arange(x.shape[1], device=x.device)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def make_cache(B, hkv, d, cap, starts, dtype, code, gen, garbage=True):
    """A cache whose sequences hold `starts` random tokens, with NaN patterns in everything that none of them holds,
    and the rows as the attention reads them, [B][2, hkv, start, d] fp64."""
    from tinker_b200.kernels import kv8_append, kv8_dequantize, kv8_empty
    kc, vc, sc, tail = kv8_empty(B, hkv, d, cap, dtype, CODES[code])
    if garbage:
        kc.view(torch.uint8).fill_(0x7f)
        vc.view(torch.uint8).fill_(0x7f)
        sc.fill_(math.nan)
        tail.fill_(math.nan)
    rows = []
    for b, n in enumerate(starts):
        part = kc[b:b + 1], vc[b:b + 1], sc[b:b + 1], tail[b:b + 1]
        if n:
            k = (torch.randn(1, n, hkv * d, device="cuda", generator=gen) * 1.5).to(dtype)
            v = torch.randn(1, n, hkv * d, device="cuda", generator=gen).to(dtype)
            kv8_append(k, v, *part, 0)
        rows.append(torch.cat([t.double() for t in kv8_dequantize(*part, n)]))
    return kc, vc, sc, tail, rows


def exact(q, k, v, cos, sin, rows, starts, hq, hkv, d, on_host=True):
    """64-bit rows of the attention and each element's bound."""
    B, S = q.shape[:2]
    once = on_host and hq // hkv * S >= 64
    dtype, g = q.dtype, hq // hkv
    st = torch.tensor(starts, device="cuda")
    q4, k4 = q.double().reshape(B, S, hq, d), k.float().reshape(B, S, hkv, d)
    if cos is not None:
        q4 = rope(q4, cos.double(), sin.double(), st)
        k4 = rope(k4, cos, sin, st)
    k4 = k4.to(dtype).double()
    v4 = v.double().reshape(B, S, hkv, d)
    out = torch.empty(B, S, hq, d, dtype=torch.float64, device="cuda")
    tol = torch.empty_like(out)
    for b in range(B):
        n = starts[b] + S
        for h in range(hq):
            K = torch.cat([rows[b][0, h // g], k4[b, :, h // g]])
            V = torch.cat([rows[b][1, h // g], v4[b, :, h // g]])
            s = q4[b, :, h] @ K.T / math.sqrt(d)
            s1 = (q4[b, :, h].abs() @ K.abs().T / math.sqrt(d)).max()
            future = torch.arange(n, device="cuda")[None] > starts[b] + torch.arange(S, device="cuda")[:, None]
            o = torch.softmax(s.masked_fill(future, -math.inf), -1) @ V
            out[b, :, h] = o
            tol[b, :, h] = torch.finfo(dtype).eps / 2 * o.abs() + 2 * V.abs().max() * (
                4 * (d + 8) * 2.0 ** -24 * s1 + n * 2.0 ** -24 + 2.0 ** -20 + once * (2.0 ** -12 + (dtype == torch.bfloat16) * 2.0 ** -11 * s1))
    return out.reshape(B, S, hq * d), tol.reshape(B, S, hq * d), k4.to(dtype), v4.to(dtype)


# ---------------------------------------------------------------------------- CPU


def _cpu_cache(B=1, hkv=2, d=64, nb=2, dtype=torch.float16, code=torch.int8):
    return (torch.zeros(B, hkv, nb, 32 * d, dtype=code), torch.zeros(B, hkv, nb, 32 * d, dtype=code),
            torch.zeros(B, hkv, nb, 2), torch.zeros(B, hkv, 2, 32, d, dtype=dtype))


def test_wrappers_refuse_cpu_tensors():
    from tinker_b200.kernels import kv8_append, kv8_attention
    q, kv = torch.zeros(1, 1, 4 * 64, dtype=torch.float16), torch.zeros(1, 1, 2 * 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kv8_append(kv, kv, *_cpu_cache(), 0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kv8_attention(q, kv, kv, None, None, *_cpu_cache(), 4, 2, 64)


def test_cache_checks():
    """What the wrappers refuse, on the checks alone."""
    from tinker_b200.kernels.kv_cache8 import _check_cache
    good = _cpu_cache()
    assert _check_cache("x", *good, 1, 2, 64, torch.float16) == (2, 1)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _check_cache("x", *good, 1, 2, 64, torch.float32)
    with pytest.raises(TypeError, match="both be float8"):
        _check_cache("x", good[0].view(torch.uint8), *good[1:], 1, 2, 64, torch.float16)
    with pytest.raises(TypeError, match="both be float8"):
        _check_cache("x", good[0], good[1].view(torch.float8_e4m3fn), *good[2:], 1, 2, 64, torch.float16)
    with pytest.raises(TypeError, match="tail"):
        _check_cache("x", *good, 1, 2, 64, torch.bfloat16)
    for B, h, d in ((2, 2, 64), (1, 1, 64), (1, 2, 128)):
        with pytest.raises(ValueError, match="does not match"):
            _check_cache("x", *good, B, h, d, torch.float16)
    with pytest.raises(ValueError, match="do not match"):
        _check_cache("x", good[0], good[1], good[2][:, :, :1], good[3], 1, 2, 64, torch.float16)
    with pytest.raises(ValueError, match="contiguous"):
        _check_cache("x", good[0].transpose(2, 3).contiguous().transpose(2, 3), *good[1:], 1, 2, 64, torch.float16)


def test_c_entry_refusals():
    import ctypes
    from tinker_b200 import _lib, build
    build.build()
    lib = _lib.lib()
    p = ctypes.c_void_p(4096)

    def append(fmt=0, seq=3, heads=2, d=64, start=0, dtype=0, stride=128, k=p, cache=p, nb=2, scales=p):
        return lib.tk_kv8_append(k, stride, p, stride, cache, p, scales, p, nb, fmt, 1, seq, heads, d, start, dtype, None)

    def attention(start=0, seq=1, hq=4, hkv=2, qs=256, cos=p, sin=p, rows=64, pos=None, step=0, out=p, nb=2):
        return lib.tk_kv8_attention(p, qs, p, 128, p, 128, p, p, p, p, nb, 0, cos, sin, rows, out, 256, 1, seq, hq,
                                    hkv, 64, start, pos, step, None, 0, 0, None)

    bad, unsup = _lib.TK_ERR_INVALID, _lib.TK_ERR_UNSUPPORTED
    assert append(fmt=2) == bad and append(dtype=2) == bad and append(start=62) == bad and append(start=-1) == bad
    assert append(d=96, stride=192) == unsup and append(stride=120) == bad and append(stride=132) == bad
    assert append(k=None) == bad and append(cache=None) == bad and append(k=ctypes.c_void_p(4098)) == bad
    assert append(scales=ctypes.c_void_p(4100)) == bad and append(seq=-1) == bad and append(nb=1 << 27) == bad
    assert append(seq=0) == _lib.TK_OK
    assert attention(start=64) == bad and attention(start=-1) == bad and attention(hq=3) == bad
    assert attention(sin=None) == bad and attention(rows=5, start=5) == bad and attention(qs=64) == bad
    assert attention(pos=p, step=2) == bad and attention(out=ctypes.c_void_p(4104)) == bad and attention(out=None) == bad
    assert attention(seq=0) == _lib.TK_OK


def test_unpack_is_the_documented_order():
    from tinker_b200.kernels.kv_cache8 import kv8_unpack
    for d in (64, 128):
        flat = torch.arange(32 * d, dtype=torch.int64)
        key = torch.empty(32, d, dtype=torch.int64)
        val = torch.empty(32, d, dtype=torch.int64)
        for j in range(4):
            for h in range(d // 64):
                for lane in range(32):
                    n, q = lane // 4, lane % 4
                    at = ((j * (d // 64) + h) * 32 + lane) * 16
                    key[8 * (n // 2) + 2 * j + n % 2, 64 * h + 16 * q:64 * h + 16 * q + 16] = flat[at:at + 16]
        for m in range(d // 16):
            for lane in range(32):
                r, q = lane // 4, lane % 4
                for e in range(2):
                    at = (m * 32 + lane) * 16 + 8 * e
                    val[8 * q:8 * q + 8, 16 * m + 8 * e + r] = flat[at:at + 8]
        for part in (0, 8):  # the numbers do not fit in a byte: a byte of them at a time
            codes = ((flat >> part) & 255).to(torch.uint8)
            assert torch.equal(kv8_unpack(codes, False, d).long(), (key >> part) & 255)
            assert torch.equal(kv8_unpack(codes, True, d).long(), (val >> part) & 255)


# ---------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("B, hkv, d, start, S", [(1, 1, 64, 0, 1), (2, 3, 64, 31, 1), (1, 2, 128, 5, 26), (3, 2, 64, 5, 27),
                                                 (2, 1, 128, 5, 28), (1, 4, 64, 0, 127), (2, 2, 128, 63, 33),
                                                 (1, 2, 64, 40, 300), (2, 2, 64, 64, 31)])
def test_append(dt, code, B, hkv, d, start, S):
    """Codes, scales and open rows bit for bit; nothing else is written; codes within half a step of the rows."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_blocks
    from tinker_b200.kernels.kv_cache8 import kv8_unpack
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(start * 1000 + S)
    nb = kv8_blocks(start + S) + 1
    kc, vc = (torch.randint(0, 100, (B, hkv, nb, 32 * d), device="cuda", generator=g, dtype=torch.uint8).view(CODES[code])
              for _ in range(2))
    sc = torch.randn(B, hkv, nb, 2, device="cuda", generator=g)
    tail = torch.randn(B, hkv, 2, 32, d, device="cuda", generator=g).to(dtype)
    w = (torch.randn(B, S, 3 * hkv * d, device="cuda", generator=g) * 3).to(dtype)  # k and v are slices of it
    k, v = w[..., :hkv * d], w[..., 2 * hkv * d:]
    was = [t.clone() for t in (kc, vc, sc, tail)]
    kv8_append(k, v, kc, vc, sc, tail, start)
    r, first = start % 32, start // 32
    whole, rest = (r + S) // 32, (r + S) % 32
    new = torch.stack([k.reshape(B, S, hkv, d), v.reshape(B, S, hkv, d)], 2).permute(0, 3, 2, 1, 4)  # [B, hkv, 2, S, d]
    rows = torch.cat([was[3][:, :, :, :r], new], 3)
    want_tail = was[3].clone()
    if whole:
        want_tail[:, :, :, :rest] = rows[:, :, :, whole * 32:]
        blocks = rows[:, :, :, :whole * 32].float().unflatten(3, (whole, 32))
        codes, scales = quantise(blocks, code)
        for i, t in enumerate((kc, vc)):
            got = kv8_unpack(t[:, :, first:first + whole], i == 1, d)
            assert torch.equal(got.view(torch.uint8), codes[:, :, i].view(torch.uint8))
            assert torch.equal(sc[:, :, first:first + whole, i], scales[:, :, i])
            x, s = blocks[:, :, i].double(), scales[:, :, i].double()[..., None, None]
            half = s / 2 if code == "int8" else torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10)
            # x (M (1 / a)) carries three roundings and a / M one: |x| 4 2^-24 beside the half step (5 for their products)
            assert ((got.double() * s - x).abs() <= half + 5 * 2.0 ** -24 * x.abs()).all()
    else:
        want_tail[:, :, :, r:r + S] = new
    assert torch.equal(tail, want_tail)
    for t, o in zip((kc, vc, sc), was):
        t, o = (t, o) if t.dtype == torch.float32 else (t.view(torch.uint8), o.view(torch.uint8))
        assert torch.equal(t[:, :, :first], o[:, :, :first]) and torch.equal(t[:, :, first + whole:], o[:, :, first + whole:])


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_append_extreme_blocks(dt, code):
    """Zeros, the smallest and largest magnitudes, values below the scale's floor, infinities and NaN, each in a head of
    its own; a block that is not finite reads as NaN, its neighbours are not touched by it."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_dequantize, kv8_empty
    dtype, d = DTYPES[dt], 64
    x = torch.randn(8, 32, d, device="cuda").to(dtype)
    x[0] = 0
    x[1] = torch.finfo(dtype).smallest_normal * x[1]
    x[2] = (x[2].float().clamp(-1, 1) * torch.finfo(dtype).max).to(dtype)
    x[3] = (x[3].float() * 2.0 ** (-70 if dt == "bf16" else -23)).to(dtype)
    x[4, 7, 9] = math.inf
    x[5, 31, 63] = math.nan
    x[6, 0, 0] = -math.inf
    x[7, :, 1:] = 0
    k = x.transpose(0, 1).reshape(1, 32, 8 * d).contiguous()
    v = x.flip(0).transpose(0, 1).reshape(1, 32, 8 * d).contiguous()
    cache = kv8_empty(1, 8, d, 32, dtype, CODES[code])
    kv8_append(k, v, *cache, 0)
    for got, rows in zip(kv8_dequantize(*cache, 32), (x, x.flip(0))):
        codes, scale = quantise(rows.float(), code)
        want = codes.float() * scale[:, None, None]
        assert torch.equal(torch.nan_to_num(got[0], nan=7.0), torch.nan_to_num(want, nan=7.0))
        assert torch.equal(torch.isnan(want).all((1, 2)), ~torch.isfinite(rows).all(2).all(1))


@pytest.mark.gpu
def test_contents_do_not_depend_on_the_split():
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_empty
    B, hkv, d, n = 2, 2, 64, 203
    k, v = (torch.randn(B, n, hkv * d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    whole = kv8_empty(B, hkv, d, n, torch.bfloat16, torch.int8)
    kv8_append(k, v, *whole, 0)
    parts = kv8_empty(B, hkv, d, n, torch.bfloat16, torch.int8)
    at = 0
    for m in (1, 30, 2, 31, 1, 64, 3, 65, 6):
        kv8_append(k[:, at:at + m], v[:, at:at + m], *parts, at)
        at += m
    assert at == n
    rest = n % 32
    for a, b in zip(whole[:3], parts[:3]):
        assert torch.equal(a, b)
    assert torch.equal(whole[3][:, :, :, :rest], parts[3][:, :, :, :rest])


ATTENTION = [  # dt, code, B, hq, hkv, d, starts, S
    ("fp16", "e4m3", 1, 16, 4, 64, [127], 1),
    ("bf16", "int8", 2, 14, 2, 64, [300, 300], 1),
    ("bf16", "e4m3", 1, 32, 8, 128, [31], 1),            # completes a block
    ("fp16", "int8", 2, 8, 2, 128, [63, 63], 1),         # the same, with a block before it
    ("fp16", "e4m3", 1, 4, 4, 64, [0], 1),               # the first token
    ("bf16", "int8", 1, 16, 1, 64, [1000], 1),           # two row blocks for one token
    ("fp16", "int8", 1, 16, 1, 128, [31], 1),            # the same, completing a block
    ("bf16", "e4m3", 1, 16, 16, 64, [32], 1),            # an empty open block
    ("fp16", "e4m3", 1, 14, 2, 64, [20011], 1),          # split over many chunks
    ("bf16", "int8", 5, 8, 4, 64, [0, 31, 32, 777, 4000], 1),   # each at its own position
    ("fp16", "e4m3", 3, 32, 8, 128, [1, 95, 2048], 1),
    ("bf16", "e4m3", 2, 8, 2, 64, [33, 33], 2),          # a chunk inside the open block
    ("fp16", "int8", 1, 8, 2, 128, [30], 5),             # across a block's end
    ("bf16", "int8", 1, 32, 8, 64, [0], 40),             # a prompt
    ("fp16", "e4m3", 2, 14, 2, 64, [517, 517], 67),
    ("bf16", "e4m3", 1, 4, 4, 128, [64], 64),
    ("fp16", "int8", 1, 16, 4, 64, [1025], 257),
    ("fp16", "e4m3", 3, 8, 2, 64, [0, 45, 400], 35),     # chunks at positions of their own
    # the tensor-core form: one query tile or two, an odd number of pairs, keys split or not, tiles that end anywhere
    ("bf16", "e4m3", 1, 32, 8, 128, [2000], 130),
    ("fp16", "int8", 2, 16, 4, 64, [128, 128], 96),
    ("bf16", "int8", 1, 14, 2, 64, [5000], 150),
    ("bf16", "e4m3", 5, 32, 8, 64, [63] * 5, 200),
    ("fp16", "e4m3", 1, 8, 4, 128, [0], 300),
    ("bf16", "int8", 1, 16, 1, 128, [127], 33),
    ("fp16", "e4m3", 2, 4, 4, 64, [1000, 1000], 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tables", [True, False])
@pytest.mark.parametrize("dt, code, B, hq, hkv, d, starts, S", ATTENTION)
def test_attention(dt, code, B, hq, hkv, d, starts, S, tables):
    """Rows within the bound of the 64-bit softmax, with NaN in all that no sequence holds; then the cache holds the new
    rows exactly as an append of the rotated keys leaves it."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, precompute_rope_tables
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(sum(starts) + S + d)
    cap = max(starts) + S
    kc, vc, sc, tail, rows = make_cache(B, hkv, d, cap, starts, dtype, code, g)
    w = torch.randn(B, S, (hq + 2 * hkv) * d, device="cuda", generator=g).to(dtype)
    q, k, v = w.split([hq * d, hkv * d, hkv * d], -1)
    cos = sin = None
    if tables:
        cos, sin = precompute_rope_tables(d, cap, 1e4, device="cuda")
    want, tol, k_new, v_new = exact(q, k, v, cos, sin, rows, starts, hq, hkv, d, on_host=len(set(starts)) == 1)
    after = [t.clone() for t in (kc, vc, sc, tail)]
    for b in range(B):
        kv8_append(k_new[b:b + 1].reshape(1, S, -1), v_new[b:b + 1].reshape(1, S, -1), *(t[b:b + 1] for t in after),
                   starts[b])
    pos = torch.tensor(starts, dtype=torch.int32, device="cuda") if len(set(starts)) > 1 else None
    out = kv8_attention(q, k, v, cos, sin, kc, vc, sc, tail, hq, hkv, d, start_pos=starts[0], position=pos)
    assert out.dtype == dtype and out.shape == (B, S, hq * d)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"error / bound {(err / tol).max().item()}"
    for got, exp in zip((kc, vc), after):
        assert torch.equal(got.view(torch.uint8), exp.view(torch.uint8))
    assert torch.equal(torch.nan_to_num(sc, nan=-1.0), torch.nan_to_num(after[2], nan=-1.0))
    assert torch.equal(torch.nan_to_num(tail, nan=-1.0), torch.nan_to_num(after[3], nan=-1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 20, 40])
def test_large_and_small_magnitudes(S):
    """bf16 rows far outside f16's range (and scales as far apart) give the 64-bit result."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_dequantize, kv8_empty
    B, hq, hkv, d, n = 1, 4, 2, 64, 130
    cache = kv8_empty(B, hkv, d, 256, torch.bfloat16)
    k = torch.randn(B, n, hkv * d, device="cuda") * 2.0 ** -40
    v = torch.randn(B, n, hkv * d, device="cuda") * 2.0 ** 60
    v[:, 64:96] *= 2.0 ** -90
    k, v = k.bfloat16(), v.bfloat16()
    kv8_append(k, v, *cache, 0)
    rows = [torch.cat([t.double() for t in kv8_dequantize(*cache, n)])]
    q = (torch.randn(B, S, hq * d, device="cuda") * 2.0 ** 40).bfloat16()
    kn = (torch.randn(B, S, hkv * d, device="cuda") * 2.0 ** -40).bfloat16()
    vn = (torch.randn(B, S, hkv * d, device="cuda") * 2.0 ** 60).bfloat16()
    want, tol, _, _ = exact(q, kn, vn, None, None, rows, [n], hq, hkv, d)
    out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d, start_pos=n)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_a_block_that_is_not_finite_shows_only_where_it_is_read():
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_empty
    cache = kv8_empty(2, 2, 64, 128, torch.float16)
    k, v = (torch.randn(2, 96, 128, device="cuda", dtype=torch.float16) for _ in range(2))
    k[1, 40, 3] = math.inf  # sequence 1, head 0
    kv8_append(k, v, *cache, 0)
    q, kn, vn = torch.randn(2, 1, 256, device="cuda").half(), *(torch.randn(2, 1, 128, device="cuda").half() for _ in range(2))
    out = kv8_attention(q, kn, vn, None, None, *cache, 4, 2, 64, start_pos=96).reshape(2, 4, 64)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, 2:]).all() and torch.isnan(out[1, :2]).all()


@pytest.mark.gpu
def test_position_tensor_graph_and_shared_workspace():
    """A captured step replayed over a block's end equals eager steps bit for bit, with one workspace that another shape
    used in between; the workspace's counters are zero afterwards."""
    require_b200()
    from tinker_b200.kernels import kv8_attention, kv8_attention_workspace, precompute_rope_tables
    B, hq, hkv, d, start, cap, steps = 2, 16, 4, 64, 1020, 1100, 40
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = make_cache(B, hkv, d, cap, [start] * B, torch.float16, "e4m3", g)[:4]
    twin = [t.clone() for t in cache]
    cos, sin = precompute_rope_tables(d, cap, 1e4, device="cuda")
    ws = torch.zeros(max(kv8_attention_workspace(B, hq, hkv, d, s, cap) for s in (1, 3)), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    w = torch.randn(steps, B, 1, (hq + 2 * hkv) * d, device="cuda", generator=g).half()
    static, pos = w[0].clone(), torch.full((1,), start, dtype=torch.int32, device="cuda")
    split = [hq * d, hkv * d, hkv * d]

    def step():
        return kv8_attention(*static.split(split, -1), cos, sin, *cache, hq, hkv, d, position=pos, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        pos.add_(1)
    for i in range(steps):
        static.copy_(w[i])
        graph.replay()
        if i % 7 == 0:  # another shape on the same workspace
            other = make_cache(1, hkv, d, 400, [390], torch.float16, "e4m3", g)[:4]
            kv8_attention(*w[:3].reshape(1, 3 * B, -1)[:, :3].split(split, -1), cos, sin, *other, hq, hkv, d,
                          start_pos=390, workspace=ws)
        want = kv8_attention(*w[i].split(split, -1), cos, sin, *twin, hq, hkv, d, start_pos=start + i, workspace=ws)
        # the eager plan may split otherwise, so the sums differ in their last bits only
        assert (out.float() - want.float()).abs().max() <= 2 * 2.0 ** -11 * want.float().abs().max()
    torch.cuda.synchronize()
    for a, b in zip(cache, twin):
        assert torch.equal(torch.nan_to_num(a.float(), nan=-1.0), torch.nan_to_num(b.float(), nan=-1.0))
    assert int(ws[:4 * 148 * 3 * 4].view(torch.int32).abs().sum()) == 0  # three counters for each CTA


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 3])
def test_positions_outside_the_cache(S):
    """A sequence whose position does not fit records device error 2 and keeps its cache; the others are served."""
    require_b200()
    from tinker_b200 import _lib
    from tinker_b200.kernels import kv8_attention, precompute_rope_tables
    B, hq, hkv, d, cap = 4, 8, 2, 64, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    kc, vc, sc, tail, rows = make_cache(B, hkv, d, cap, [10, 20, 30, 40], torch.float16, "int8", g)
    cos, sin = precompute_rope_tables(d, cap, 1e4, device="cuda")
    w = torch.randn(B, S, (hq + 2 * hkv) * d, device="cuda", generator=g).half()
    q, k, v = w.split([hq * d, hkv * d, hkv * d], -1)
    want, tol, _, _ = exact(q, k, v, cos, sin, rows, [10, 20, 30, 40], hq, hkv, d)
    was = [t.clone() for t in (kc, vc, sc, tail)]
    _lib.device_error(clear=True)
    pos = torch.tensor([10, cap - S + 1, -1, 40], dtype=torch.int32, device="cuda")
    out = kv8_attention(q, k, v, cos, sin, kc, vc, sc, tail, hq, hkv, d, position=pos)
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 2
    for b in (0, 3):
        assert ((out[b].double() - want[b]).abs() <= tol[b]).all()
    for b in (1, 2):
        for t, o in zip((kc, vc, sc, tail), was):
            assert torch.equal(torch.nan_to_num(t[b].float(), nan=-1.0), torch.nan_to_num(o[b].float(), nan=-1.0))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^31 bytes: the last sequence's rows lie beyond what 32 bits reach."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_dequantize, kv8_empty
    hq, hkv, d, cap, n, S = 16, 8, 128, 1100000, 200, 1
    cache = kv8_empty(2, hkv, d, cap, torch.bfloat16, torch.int8)
    assert cache[0].numel() > 2 ** 31
    last = [t[1:] for t in cache]
    k, v = (torch.randn(1, n, hkv * d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kv8_append(k, v, *last, 0)
    rows = [torch.zeros(2, hkv, 0, d, dtype=torch.float64, device="cuda"),
            torch.cat([t.double() for t in kv8_dequantize(*last, n)])]
    rows = [rows[0].reshape(2, hkv, 0, d), rows[1].reshape(2, hkv, n, d)]
    w = torch.randn(2, S, (hq + 2 * hkv) * d, device="cuda", dtype=torch.bfloat16)
    q, kn, vn = w.split([hq * d, hkv * d, hkv * d], -1)
    want, tol, _, _ = exact(q, kn, vn, None, None, rows, [0, n], hq, hkv, d)
    out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d,
                        position=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_other_stream_repeat_and_refusals():
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, precompute_rope_tables
    B, hq, hkv, d, n = 1, 14, 2, 64, 5000
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc, sc, tail, rows = make_cache(B, hkv, d, n + 40, [n], torch.bfloat16, "e4m3", g)
    cos, sin = precompute_rope_tables(d, n + 40, 1e4, device="cuda")
    w = torch.randn(B, 1, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16()
    q, k, v = w.split([hq * d, hkv * d, hkv * d], -1)
    want, tol, _, _ = exact(q, k, v, cos, sin, rows, [n], hq, hkv, d)
    outs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            outs.append(kv8_attention(q, k, v, cos, sin, kc, vc, sc, tail, hq, hkv, d, start_pos=n))
    side.synchronize()
    assert ((outs[0].double() - want).abs() <= tol).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    # an odd token stride and transposed inputs are copied, not refused
    odd = torch.randn(B, 1, hq * d + 3, device="cuda").bfloat16()[..., 3:]
    kv8_attention(odd, k, v, cos, sin, kc, vc, sc, tail, hq, hkv, d, start_pos=n)
    empty = kv8_attention(q[:, :0], k[:, :0], v[:, :0], cos, sin, kc, vc, sc, tail, hq, hkv, d, start_pos=n)
    assert empty.shape == (1, 0, hq * d)
    args = (kc, vc, sc, tail, hq, hkv, d)
    with pytest.raises(ValueError, match="capacity"):
        kv8_attention(q, k, v, cos, sin, *args, start_pos=kc.shape[2] * 32)
    with pytest.raises(ValueError, match="both RoPE tables"):
        kv8_attention(q, k, v, cos, None, *args, start_pos=3)
    with pytest.raises(TypeError, match="float32"):
        kv8_attention(q, k, v, cos.half(), sin.half(), *args, start_pos=3)
    with pytest.raises(RuntimeError, match="table"):
        kv8_attention(q, k, v, cos[:9], sin[:9], *args, start_pos=9)
    with pytest.raises(TypeError, match="position"):
        kv8_attention(q, k, v, cos, sin, *args, position=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="position"):
        kv8_attention(q, k, v, cos, sin, *args, position=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="workspace"):
        kv8_attention(q, k, v, cos, sin, *args, start_pos=n, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(TypeError, match="all"):
        kv8_attention(q, k.half(), v, cos, sin, *args, start_pos=n)
    with pytest.raises(ValueError, match="capacity"):
        kv8_append(k, v, kc, vc, sc, tail, kc.shape[2] * 32)


@pytest.mark.gpu
def test_chunk_of_more_sequences_than_are_laid_out_at_once():
    """Operands of all sequences would take more than the gigabyte that the call allows itself: it goes in groups."""
    require_b200()
    from tinker_b200.kernels import kv8_attention, kv8_attention_workspace
    B, hq, hkv, d, n, S = 16, 32, 8, 128, 20000, 16
    one = kv8_attention_workspace(1, hq, hkv, d, S, n + S) - kv8_attention_workspace(1, hq, hkv, d, 1, 1)
    assert B * one > 2 ** 30
    g = torch.Generator(device="cuda").manual_seed(4)
    kc, vc, sc, tail, rows = make_cache(B, hkv, d, n + S, [n] * B, torch.bfloat16, "e4m3", g, garbage=False)
    w = torch.randn(B, S, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16()
    q, k, v = w.split([hq * d, hkv * d, hkv * d], -1)
    out = kv8_attention(q, k, v, None, None, kc, vc, sc, tail, hq, hkv, d, start_pos=n)
    for b in (0, 7, 12, 13, 15):
        want, tol, _, _ = exact(q[b:b + 1], k[b:b + 1], v[b:b + 1], None, None, rows[b:b + 1], [n], hq, hkv, d)
        assert ((out[b:b + 1].double() - want).abs() <= tol).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("S", [9, 40])  # 18 and 80 query rows of a kv head: the one form and the other
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_tokens_that_are_not_finite_stay_behind_the_mask(S, dt, what, bad):
    """A NaN or an infinity in a later token of a chunk: the rows before it are what they are without it, in both forms;
    the rows that see a value that is not finite are NaN."""
    require_b200()
    from tinker_b200.kernels import kv8_attention
    dtype, hq, hkv, d, n, at = DTYPES[dt], 8, 4, 64, 130, 6
    g = torch.Generator(device="cuda").manual_seed(S)
    kc, vc, sc, tail, rows = make_cache(2, hkv, d, 256, [n, n], dtype, "e4m3", g, garbage=False)
    w = torch.randn(2, S, (hq + 2 * hkv) * d, device="cuda", generator=g).to(dtype)
    q, k, v = (t.contiguous() for t in w.split([hq * d, hkv * d, hkv * d], -1))
    want, tol, _, _ = exact(q, k, v, None, None, rows, [n, n], hq, hkv, d)
    (k if what == "k" else v)[0, at, d + 3] = bad  # sequence 0, kv head 1: heads 2 and 3
    out = kv8_attention(q, k, v, None, None, kc, vc, sc, tail, hq, hkv, d, start_pos=n).double()
    ok = torch.ones(2, S, hq * d, dtype=torch.bool, device="cuda")
    ok[0, at:, 2 * d:4 * d] = False
    assert torch.isfinite(out[ok]).all()
    assert ((out - want).abs() <= tol)[ok].all()
    if what == "v":
        assert torch.isnan(out[0, at:, 2 * d:4 * d]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("who, gap", [("own", 10.0), ("own", 14.0), ("first", 13.0)])
@pytest.mark.parametrize("S", [1, 9, 40])  # 40: 80 query rows of a kv head, the tensor-core form
@pytest.mark.parametrize("size", [0.05, 0.002])
@pytest.mark.parametrize("dt, code", [("fp16", "e4m3"), ("fp16", "int8"), ("bf16", "e4m3")])
def test_small_weights_beside_a_dominant_token(dt, code, size, S, who, gap):
    """One token's score lies far above thousands of others that make up a part of the result together: the weights of
    those keep their bits, whatever the values' scales. `own`: the query's own token, in 16 bits; `first`: the first one,
    whose block has a hundred times the others' scale. Values have a mean, so weights that the sum of values loses and the
    denominator keeps would show.

    A relative error e of the weights moves o by at most 2 e sum p |v|; e is that of the module's head. To it comes half of
    f16's smallest number, 2^-25, where the largest weight f is 2^11 (tensor cores) or 2^15: with a weight w and a code c
    for each key o is sum w c / (w_f / scale_f), c = v / scale, so it moves by at most 2^-36 (2^-40) r sum |v|, r the scale
    of the dominant token's block over the least (1 for `own`, whose tile has the smaller one; 200 for `first`)."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_dequantize, kv8_empty
    dtype, B, hq, hkv, d, n = DTYPES[dt], 20, 16, 8, 128, 7000
    g = torch.Generator(device="cuda").manual_seed(S)
    cache = kv8_empty(B, hkv, d, n + S, dtype, CODES[code])
    q = torch.randn(B, S, hq // hkv, hkv, d, device="cuda", generator=g)
    q[:, :, 1:] = q[:, :, :1] * (1 + 0.05 * torch.randn(B, S, hq // hkv - 1, hkv, 1, device="cuda", generator=g))
    q = q.transpose(2, 3)  # the heads of a kv head look the same way
    if who == "first":
        q[:] = q[:, :1]
    kn = q[:, :, :, 0] * (gap * math.sqrt(d) / q[:, :, :, 0].square().sum(-1, keepdim=True))
    k = torch.randn(B, n, hkv, d, device="cuda", generator=g) * 0.02
    v = size * (1 + 0.3 * torch.randn(B, n, hkv, d, device="cuda", generator=g))
    vn = size * (1 + 0.3 * torch.randn(B, S, hkv, d, device="cuda", generator=g))
    if who == "first":
        k[:, 0], kn = kn[:, 0], torch.randn(B, S, hkv, d, device="cuda", generator=g) * 0.02
        k[:, 1:32] = 0
        v[:, 1] *= 100
    q, kn, vn, k, v = (t.reshape(B, t.shape[1], -1).to(dtype) for t in (q, kn, vn, k, v))
    kv8_append(k, v, *cache, 0)
    rows = {b: torch.cat([t.double() for t in kv8_dequantize(*(t[b:b + 1] for t in cache), n)]) for b in (0, B - 1)}
    out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d, start_pos=n).double().reshape(B, S, hq, d)
    once = hq // hkv * S >= 64
    for b in rows:
        for h in range(hq):
            x, j = q[b, :, h * d:(h + 1) * d].double(), h // (hq // hkv)
            K = torch.cat([rows[b][0, j], kn[b, :, j * d:(j + 1) * d].double()])
            V = torch.cat([rows[b][1, j], vn[b, :, j * d:(j + 1) * d].double()])
            s = x @ K.T / math.sqrt(d)
            s1 = (x.abs() @ K.abs().T / math.sqrt(d)).max()
            future = torch.arange(n + S, device="cuda")[None] > n + torch.arange(S, device="cuda")[:, None]
            p = torch.softmax(s.masked_fill(future, -math.inf), -1)
            e = 4 * (d + 8) * 2.0 ** -24 * s1 + n * 2.0 ** -24 + 2.0 ** -20
            e += once * (2.0 ** -12 + (dtype == torch.bfloat16) * 2.0 ** -11 * s1)
            tol = torch.finfo(dtype).eps / 2 * (p @ V).abs() + 2 * e * (p @ V.abs())
            tol += torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2  # half a step of a result below the normal numbers
            tol += (2.0 ** -36 if once else 2.0 ** -40) * (200 if who == "first" else 1) * V.abs().sum(0)
            err = (out[b, :, h] - p @ V).abs()
            assert (err <= tol).all(), f"error / bound {(err / tol).max().item()}"


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 20, 40])  # 40: the tensor-core form
@pytest.mark.parametrize("power", [60, 70, 110])
@pytest.mark.parametrize("small", ["first", "middle", "open", "large first"])
def test_blocks_of_zeros_beside_large_values(small, power, S):
    """bf16 values of 2^60 and more beside blocks of zeros (whose scale is the least that there is): the weights of those
    count in the denominator, in whatever order the blocks come and however they are split and merged."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_dequantize, kv8_empty
    B, hq, hkv, d, n = 2, 4, 2, 64, 1000
    g = torch.Generator(device="cuda").manual_seed(S)
    cache = kv8_empty(B, hkv, d, 1088, torch.bfloat16)
    k = torch.randn(B, n, hkv * d, device="cuda", generator=g).bfloat16()
    v = torch.randn(B, n, hkv * d, device="cuda", generator=g) * 2.0 ** power
    vn = torch.randn(B, S, hkv * d, device="cuda", generator=g) * 2.0 ** power
    if small == "first":
        v[:, :640] = 0
    elif small == "middle":
        v[:, 320:352] = 0
        v[:, 608:800] = 0
    elif small == "open":
        v[:, 992:] = 0
        vn[:] = 0
    else:
        v[:, 32:] = 0
    v, vn = v.bfloat16(), vn.bfloat16()
    kv8_append(k, v, *cache, 0)
    rows = [torch.cat([t.double() for t in kv8_dequantize(*(t[b:b + 1] for t in cache), n)]) for b in range(B)]
    q = torch.randn(B, S, hq * d, device="cuda", generator=g).bfloat16()
    kn = torch.randn(B, S, hkv * d, device="cuda", generator=g).bfloat16()
    want, tol, _, _ = exact(q, kn, vn, None, None, rows, [n] * B, hq, hkv, d)
    out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d, start_pos=n)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"error / bound {(err / tol).max().item()}"


@pytest.mark.gpu
@pytest.mark.parametrize("S", [9, 40])  # 18 and 80 query rows of a kv head: the one form and the other
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("power", [-40, 20])
def test_a_token_that_is_not_finite_leaves_the_others_their_range(power, bad, what, S):
    """bf16 keys and values outside f16's range beside a token that is not finite, in the same 32 tokens: the rows before
    it are what they are without it."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_dequantize, kv8_empty
    B, hq, hkv, d, n, at = 2, 8, 4, 64, 130, 6
    g = torch.Generator(device="cuda").manual_seed(S)
    cache = kv8_empty(B, hkv, d, 256, torch.bfloat16)
    k, v = ((torch.randn(B, n, hkv * d, device="cuda", generator=g) * 2.0 ** power).bfloat16() for _ in range(2))
    kv8_append(k, v, *cache, 0)
    rows = [torch.cat([t.double() for t in kv8_dequantize(*(t[b:b + 1] for t in cache), n)]) for b in range(B)]
    q = (torch.randn(B, S, hq * d, device="cuda", generator=g) * 2.0 ** -power).bfloat16()
    kn, vn = ((torch.randn(B, S, hkv * d, device="cuda", generator=g) * 2.0 ** power).bfloat16() for _ in range(2))
    want, tol, _, _ = exact(q, kn, vn, None, None, rows, [n] * B, hq, hkv, d)
    (kn if what == "k" else vn)[0, at, d + 3] = bad  # sequence 0, kv head 1: heads 2 and 3
    out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d, start_pos=n).double()
    seen = torch.zeros(B, S, hq * d, dtype=torch.bool, device="cuda")
    seen[0, at:, 2 * d:4 * d] = True
    assert torch.isnan(out[seen]).all()
    assert ((out - want).abs() <= tol)[~seen].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("S, n", [(1, 70), (1, 95), (3, 70), (40, 70)])
def test_rows_that_see_a_token_that_is_not_finite_are_nan(S, n, bad, what, dt):
    """In every form, and as they are once the token's block is complete; other heads and sequences are not."""
    require_b200()
    from tinker_b200.kernels import kv8_append, kv8_attention, kv8_empty
    dtype, B, hq, hkv, d = DTYPES[dt], 2, 8, 4, 64
    g = torch.Generator(device="cuda").manual_seed(n)
    for where in ("open", "own"):
        cache = kv8_empty(B, hkv, d, 160, dtype)
        k, v = (torch.randn(B, n, hkv * d, device="cuda", generator=g).to(dtype) for _ in range(2))
        q, kn, vn = (torch.randn(B, S, h * d, device="cuda", generator=g).to(dtype) for h in (hq, hkv, hkv))
        if where == "open":
            (k if what == "k" else v)[0, n - 2, d + 3] = bad  # sequence 0, kv head 1: heads 2 and 3
        else:
            (kn if what == "k" else vn)[0, S - 1, d + 3] = bad
        kv8_append(k, v, *cache, 0)
        out = kv8_attention(q, kn, vn, None, None, *cache, hq, hkv, d, start_pos=n)
        seen = torch.zeros(B, S, hq * d, dtype=torch.bool, device="cuda")
        seen[0, 0 if where == "open" else S - 1:, 2 * d:4 * d] = True
        assert torch.isnan(out[seen]).all() and torch.isfinite(out[~seen]).all()
        nxt = kv8_attention(q[:, :1], k[:, :1], v[:, :1], None, None, *cache, hq, hkv, d, start_pos=n + S)
        assert torch.isnan(nxt[0, :, 2 * d:4 * d]).all() and torch.isfinite(nxt[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt, code, B, hq, hkv, d, n", [("fp16", "e4m3", 1, 64, 1, 64, 500), ("bf16", "int8", 3, 71, 1, 64, 63),
                                                        ("bf16", "e4m3", 2, 128, 2, 128, 130)])
def test_one_token_of_many_heads(dt, code, B, hq, hkv, d, n):
    """64 and more query heads for a kv head, one new token, the position on the host or on the device."""
    require_b200()
    from tinker_b200 import _lib
    from tinker_b200.kernels import kv8_attention, kv8_attention_workspace
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(n)
    kc, vc, sc, tail, rows = make_cache(B, hkv, d, n + 1, [n] * B, dtype, code, g)
    w = torch.randn(B, 1, (hq + 2 * hkv) * d, device="cuda", generator=g).to(dtype)
    q, k, v = w.split([hq * d, hkv * d, hkv * d], -1)
    want, tol, _, _ = exact(q, k, v, None, None, rows, [n] * B, hq, hkv, d, on_host=False)
    ws = torch.zeros(kv8_attention_workspace(B, hq, hkv, d, 1, n + 1), dtype=torch.uint8, device="cuda")
    for kw in (dict(start_pos=n), dict(start_pos=n, workspace=ws),
               dict(position=torch.tensor([n], dtype=torch.int32, device="cuda"))):
        cache = [t.clone() for t in (kc, vc, sc, tail)]
        n0 = _lib.launch_counter[0]
        out = kv8_attention(q, k, v, None, None, *cache, hq, hkv, d, **kw)
        assert _lib.launch_counter[0] - n0 == 1
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("ragged", [True, False])
def test_rows_of_a_position_outside_the_cache_are_nan(ragged, S, d):
    """They are what the call returns for that sequence, not whatever was in memory."""
    require_b200()
    from tinker_b200 import _lib
    from tinker_b200.kernels import kv8_attention
    B, hq, hkv, cap = 300, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    cache = make_cache(B, hkv, d, cap, [10] * B, torch.float16, "int8", g, garbage=False)[:4]
    q, k, v = (torch.randn(B, S, h * d, device="cuda", generator=g).half() for h in (hq, hkv, hkv))
    pos = torch.full((B,), 10, dtype=torch.int32, device="cuda")
    pos[[0, 7, 299]] = torch.tensor([-1, cap - S + 1, 1 << 30], dtype=torch.int32, device="cuda")
    if not ragged:
        pos = pos[7:8].clone()
    was = [t.clone() for t in cache]
    _lib.device_error(clear=True)
    torch.empty(B * S * hq * d, dtype=torch.float16, device="cuda").fill_(1.0)  # what the rows may be made of
    out = kv8_attention(q, k, v, None, None, *cache, hq, hkv, d, position=pos)
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 2
    bad = torch.zeros(B, dtype=torch.bool, device="cuda")
    bad[[0, 7, 299]] = True
    if not ragged:
        bad[:] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    for t, o in zip(cache, was):
        assert torch.equal(t[bad].view(torch.uint8), o[bad].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dt, B, hq, hkv, d, n, S", [("fp16", 1, 8, 2, 64, 100, 1), ("fp16", 1, 8, 2, 64, 100, 3),
                                                     ("bf16", 1, 32, 8, 128, 2000, 130), ("fp16", 1, 32, 8, 128, 2000, 130),
                                                     ("bf16", 8, 32, 8, 64, 40, 256), ("bf16", 16, 32, 8, 128, 20000, 16)])
def test_launches_are_counted(dt, B, hq, hkv, d, n, S):
    """The counter grows by the kernels that a capture of the call holds (a memset of the workspace is none of ours)."""
    require_b200()
    import ctypes
    from tinker_b200 import _lib
    from tinker_b200.kernels import kv8_attention, kv8_attention_workspace, kv8_empty
    dtype = DTYPES[dt]
    cache = kv8_empty(B, hkv, d, n + S, dtype)
    q, k, v = (torch.randn(B, S, h * d, device="cuda").to(dtype) for h in (hq, hkv, hkv))
    ws = torch.zeros(kv8_attention_workspace(B, hq, hkv, d, S, n + S), dtype=torch.uint8, device="cuda")

    def call():
        return kv8_attention(q, k, v, None, None, *cache, hq, hkv, d, start_pos=n, workspace=ws)
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    n0 = _lib.launch_counter[0]
    with torch.cuda.graph(graph):
        out = call()
    counted = _lib.launch_counter[0] - n0
    nodes = ctypes.c_size_t()
    cudart = ctypes.CDLL("libcudart.so.12")
    assert cudart.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    assert counted == nodes.value and out.shape == q.shape
