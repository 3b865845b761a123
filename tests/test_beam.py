"""Beam selection and cache reordering against plain implementations in 64 bits.

Scores: the chunks' fp32 sums carry at most 48 2^-24 from their additions, 2^-22 from the exponential and 2^-21 from its
argument, relative to the sum, so a logsumexp is off by less than 4e-6; the result is rounded once to fp32 (2^-24).
Selections have to be the same wherever two neighbours in the order are further apart than twice that, and exactly the
same where the order is exact: equal logits of one beam, equal rows, -inf.
"""

import math

import pytest
import torch

from tests._util import DTYPES, require_b200

NEAR = 4e-6


def plain(logits, scores, n, finished=None, eos=None):
    """(values fp64, flat places), best first, ties to the lower place."""
    B, K, V = logits.shape
    x = logits.double()
    top = torch.finfo(logits.dtype).max
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).clamp(max=top)
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    lp = (x - m) - (x - m).exp().sum(-1, keepdim=True).log()  # logits near the type's lowest do not swallow the logarithm
    lp = torch.where(torch.isinf(x), x, lp)
    s = torch.where(torch.isnan(scores), torch.full_like(scores, -math.inf), scores).double()[..., None]
    c = s + lp
    if finished is not None:
        only = torch.full_like(c, -math.inf)
        only[..., eos] = s[..., 0]
        c = torch.where(finished[..., None], only, c)
    val, at = c.reshape(B, K * V).sort(dim=-1, descending=True, stable=True)
    return val[:, :n + 1], at[:, :n + 1]


def check(logits, scores, n, finished=None, eos=None):
    from tinker_b200.kernels import beam_select
    got, beams, tokens = beam_select(logits, scores, n, finished=finished, eos_token_id=eos)
    V = logits.shape[2]
    val, at = plain(logits, scores, n, finished, eos)
    want = val[:, :n]
    assert got.shape == beams.shape == tokens.shape == want.shape
    assert beams.dtype == tokens.dtype == torch.int64 and got.dtype == torch.float32
    low = torch.isinf(want)
    assert torch.equal(torch.isinf(got), low)
    assert ((got.double() - want).abs() <= NEAR + 2.0 ** -24 * want.abs())[~low].all()
    gap = val[:, :-1] - val[:, 1:]
    gap = torch.where(torch.isnan(gap), torch.zeros_like(gap), gap)  # -inf - -inf: an exact tie
    if gap.shape[1] < n:
        gap = torch.cat([gap, gap.new_full((gap.shape[0], 1), math.inf)], 1)
    tight = (gap > 0) & (gap <= 2 * NEAR + 2.0 ** -40 * want.abs().clamp(max=1e30))
    loose = tight.clone()
    loose[:, 1:] |= tight[:, :-1]
    same = (beams * V + tokens) == at[:, :n]
    assert (same | loose).all(), (beams * V + tokens, at[:, :n], want)
    assert loose.float().mean() < 0.2
    return got, beams, tokens


# ---------------------------------------------------------------------------- CPU


def test_wrappers_refuse_cpu_tensors():
    from tinker_b200.kernels import beam_select, kv8_reorder, kv_reorder
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))
    c, p = torch.zeros(2, 1, 4, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kv_reorder(c, c, p, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kv8_reorder(c, c, c, c, p, 1)


def test_c_entry_refusals():
    import ctypes
    from tinker_b200 import _lib, build
    build.build()
    lib = _lib.lib()
    p = ctypes.c_void_p(4096)

    def select(row=100, batch=1, beams=2, vocab=100, n=2, ws=p, dtype=0, fin=None, eos=-1, logits=p):
        return lib.tk_beam_select(logits, row, p, fin, eos, p, p, p, batch, beams, vocab, n, ws, 0, dtype, None)

    def reorder(k=p, par=p, layers=1, groups=1, beams=2, heads=1, cap=8, d=64, length=4, dtype=0):
        return lib.tk_kv_reorder(k, p, par, layers, groups, beams, heads, cap, d, length, None, dtype, None)

    bad, unsup = _lib.TK_ERR_INVALID, _lib.TK_ERR_UNSUPPORTED
    assert select(dtype=9) == bad and select(row=99) == bad and select(n=0) == unsup and select(n=65) == unsup
    assert select(vocab=1, row=1, n=3) == bad and select(beams=0) == bad and select(vocab=0) == bad
    assert select(fin=p, eos=-1) == bad and select(fin=p, eos=100) == bad and select(logits=None) == bad
    assert select(beams=1025, row=100) == unsup and select(batch=40000) == bad and select(batch=0) == _lib.TK_OK
    assert reorder(dtype=2) == bad and reorder(length=9) == bad and reorder(length=-1) == bad and reorder(k=None) == bad
    assert reorder(beams=33) == unsup and reorder(d=60) == unsup and reorder(par=None) == bad
    assert reorder(k=ctypes.c_void_p(4104)) == bad and reorder(groups=70000) == bad and reorder(beams=0) == bad
    assert reorder(layers=0) == _lib.TK_OK and reorder(length=0) == _lib.TK_OK and reorder(beams=1) == _lib.TK_OK
    assert lib.tk_kv8_reorder(p, p, ctypes.c_void_p(4100), p, p, 1, 1, 2, 1, 1, 64, 4, None, None) == bad
    assert lib.tk_kv8_reorder(p, p, p, p, p, 1, 1, 2, 1, 1, 64, 33, None, None) == bad
    assert lib.tk_kv8_reorder(p, p, p, None, p, 1, 1, 2, 1, 1, 64, 4, None, None) == bad


def test_python_argument_checks():
    from tinker_b200.kernels.beam import _check_parents, _length_args
    with pytest.raises(ValueError, match="parents"):
        _check_parents("x", torch.zeros(2, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="parents"):
        _check_parents("x", torch.zeros(2, 3, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="length"):
        _length_args("x", 9, 8, torch.device("cpu"))
    with pytest.raises(TypeError, match="int32"):
        _length_args("x", torch.zeros(1, dtype=torch.int64), 8, torch.device("cpu"))


# ---------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("B, K, V, n", [(1, 1, 1, 1), (1, 4, 32000, 8), (2, 3, 5, 8), (3, 5, 2047, 10), (1, 2, 2048, 4),
                                        (2, 2, 2049, 64), (1, 16, 8193, 32), (4, 8, 50257, 16), (1, 1, 151936, 64),
                                        (60, 5, 1001, 5), (2, 40, 333, 40), (1, 700, 40, 3)])
def test_select(dt, B, K, V, n):
    require_b200()
    g = torch.Generator(device="cuda").manual_seed(V + n)
    logits = (torch.randn(B, K, V, device="cuda", generator=g) * 3).to(DTYPES[dt])
    scores = -torch.rand(B, K, device="cuda", generator=g) * 6
    check(logits, scores, n)
    if K >= 3 and V > 2:
        fin = torch.zeros(B, K, dtype=torch.bool, device="cuda")
        fin[:, 1] = True
        scores[:, 1] = -0.5
        scores[0, 2] = -math.inf
        got, beams, tokens = check(logits, scores, n, fin, 2)
        live = torch.isfinite(got)
        assert (tokens[live & (beams == 1)] == 2).all()  # a finished beam gives its end token and nothing else


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "fp32"])
def test_strided_and_misaligned_rows(dt):
    """Rows that start anywhere, and equal rows at different alignments: their ties go to the lower beam."""
    require_b200()
    from tinker_b200.kernels import beam_select
    base = (torch.randn(2, 3, 4099, device="cuda") * 2).to(DTYPES[dt])
    scores = torch.tensor([[-1.0, -2.0, -1.5], [0.0, -0.1, -0.2]], device="cuda")
    check(base[:, :, 1:], scores, 6)
    check(base[:, :, 3:4001], scores, 6)
    check(base.transpose(1, 2).contiguous().transpose(1, 2), scores, 6)
    check(base[:, :1], scores[:, :1].contiguous(), 6)
    same = base[:, :1].expand(2, 3, 4099).contiguous()  # odd length: the rows' alignments differ
    got, beams, tokens = beam_select(same, torch.zeros(2, 3, device="cuda"), 6)
    want = same[:, 0].float().sort(dim=-1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(beams, torch.tensor([[0, 1, 2] * 2] * 2, device="cuda"))
    assert torch.equal(tokens, want.repeat_interleave(3, 1))
    assert torch.equal(got[:, 0], got[:, 1]) and torch.equal(got[:, 0], got[:, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_ties_masks_and_special_values(dt):
    require_b200()
    dtype = DTYPES[dt]
    B, K, V = 2, 4, 20011
    zero = torch.zeros(B, K, device="cuda")
    steps = -torch.arange(K, device="cuda").float().repeat(B, 1)
    flat = torch.zeros(B, K, V, device="cuda", dtype=dtype)
    _, beams, tokens = check(flat, zero, 8)  # all equal: the lowest places
    assert (beams == 0).all() and torch.equal(tokens, torch.arange(8, device="cuda").expand(B, 8))
    check(flat, steps, 64)
    coarse = torch.randint(0, 3, (B, K, V), device="cuda").to(dtype)  # thousands of ties at the top
    check(coarse, steps, 33)
    signed = flat.clone()
    signed[:, :, ::2] = -0.0  # -0 and 0 are equal
    check(signed, steps, 8)
    for low in (-math.inf, torch.finfo(dtype).min):
        masked = torch.full((B, K, V), low, device="cuda", dtype=dtype)
        check(masked, steps, 8)  # nothing is left
        masked[:, 1, 17] = 0.5
        masked[1, 3, V - 1] = 2.0
        check(masked, steps, 8)
    odd = (torch.randn(B, K, V, device="cuda") * 2).to(dtype)
    odd[0, 0, 5] = math.nan
    odd[0, 1] = math.nan
    odd[1, 2, 100] = math.inf
    odd[1, 3, 7] = -math.inf
    check(odd, steps, 16)
    dead = torch.full((B, K), -math.inf, device="cuda")
    check(odd, dead, 8)
    first = dead.clone()
    first[:, 0] = 0  # the first step: one beam lives
    check(odd, first, 8)
    nan = steps.clone()
    nan[0, 0] = math.nan
    check(odd, nan, 8)
    fin = torch.ones(B, K, dtype=torch.bool, device="cuda")
    for eos in (0, 3, V - 1):
        _, beams, tokens = check(odd, steps, 4, fin, eos)
        assert (tokens == eos).all()
        check(odd, steps, 9, fin, eos)  # more than the finished beams have
        check(odd, dead, 9, fin, eos)


@pytest.mark.gpu
def test_select_captured_and_refusals():
    require_b200()
    from tinker_b200.kernels import beam_select
    logits = torch.randn(2, 4, 999, device="cuda").half()
    scores = torch.randn(2, 4, device="cuda")
    beam_select(logits, scores, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_select(logits, scores, 8)
    for seed in range(3):
        logits.copy_(torch.randn(2, 4, 999, device="cuda"))
        graph.replay()
        for a, b in zip(out, beam_select(logits, scores, 8)):
            assert torch.equal(a, b)
    assert beam_select(logits[:0], scores[:0], 3)[0].shape == (0, 3)
    assert beam_select(logits, scores)[0].shape == (2, 4)
    for bad in (lambda: beam_select(logits[0], scores), lambda: beam_select(logits, scores.half()),
                lambda: beam_select(logits, scores[:, :3]), lambda: beam_select(logits, scores, 0),
                lambda: beam_select(logits[:, :, :1], scores, 5),
                lambda: beam_select(logits, scores, finished=torch.zeros(2, 4, dtype=torch.bool, device="cuda")),
                lambda: beam_select(logits, scores, finished=torch.zeros(2, 4, device="cuda"), eos_token_id=1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="num_select"):
        beam_select(logits, scores, 65)


def _reordered(t, parents, fill):
    """Rows of t [layers, rows, ...] by parents, in the places that `fill` selects (a slice of dimension 3)."""
    G, K = parents.shape
    src = (parents + torch.arange(G, device="cuda")[:, None] * K).reshape(-1)
    t = t.clone()
    raw = t.view(torch.uint8) if t.element_size() == 1 else t
    raw[:, :, :, fill] = raw[:, src][:, :, :, fill]
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("G, K", [(1, 1), (1, 2), (3, 3), (2, 5), (2, 8), (1, 13), (2, 16), (1, 32)])
@pytest.mark.parametrize("length", [0, 1, 31, 32, 33, 90])
def test_reorder(G, K, length):
    """Random parents (cycles, repeats, rows that stay) in both caches; the positions behind the length stay."""
    require_b200()
    from tinker_b200.kernels import kv8_empty, kv8_reorder, kv_reorder
    L, H, d, cap = 2, 3, 64, 90
    g = torch.Generator(device="cuda").manual_seed(K * 100 + length)
    for parents in (torch.randint(0, K, (G, K), device="cuda", generator=g),
                    torch.arange(K, device="cuda").roll(1).repeat(G, 1), torch.arange(K, device="cuda").repeat(G, 1)):
        k, v = (torch.randn(L, G * K, H, cap, d, device="cuda", generator=g).bfloat16() for _ in range(2))
        want = [_reordered(t, parents, slice(0, length)) for t in (k, v)]
        kv_reorder(k, v, parents, length)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
        one = [t[0].clone() for t in (k, v)]
        want = [_reordered(t[None], parents, slice(0, length))[0] for t in one]
        kv_reorder(*one, parents, torch.tensor([length], dtype=torch.int32, device="cuda"))  # no layers, device length
        assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])
        c = kv8_empty(G * K, H, d, cap, torch.float16, torch.int8, layers=L)
        for t in c[:2]:
            t.copy_(torch.randint(-127, 128, t.shape, device="cuda", generator=g))
        c[2].normal_(generator=g)
        c[3].normal_(generator=g)
        nb, rest = length // 32, length % 32
        want = [_reordered(t, parents, slice(0, nb)) for t in c[:3]]
        tail = c[3].flatten(2, 3)
        want.append(_reordered(tail, parents, slice(0, rest)).reshape(c[3].shape))
        at = length if K % 2 else torch.tensor([length], dtype=torch.int32, device="cuda")
        kv8_reorder(*c, parents, at)
        for t, w in zip(c, want):
            assert torch.equal(t, w)


@pytest.mark.gpu
def test_reorder_odd_heads_errors_and_refusals():
    require_b200()
    from tinker_b200 import _lib
    from tinker_b200.kernels import kv8_empty, kv8_reorder, kv_reorder
    k, v = (torch.randn(6, 1, 50, 72, device="cuda").half() for _ in range(2))  # head_dim 72
    p = torch.tensor([[1, 0, 0], [2, 2, 1]], device="cuda")
    want = [_reordered(t[None], p, slice(0, 50))[0] for t in (k, v)]
    kv_reorder(k, v, p, 50)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    _lib.device_error(clear=True)
    bad = torch.tensor([[1, 0, 3], [0, 2, 1]], device="cuda")  # group 0 names a row outside it
    want = [torch.cat([t[:3], _reordered(t[None, 3:], bad[1:], slice(0, 50))[0]]) for t in (k, v)]
    kv_reorder(k, v, bad, 50)
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 4
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    kv_reorder(k, v, p, torch.tensor([51], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 2
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    for call in (lambda: kv_reorder(k, v[:3], p, 1), lambda: kv_reorder(k, v, p[:1], 1), lambda: kv_reorder(k, v, p, 51),
                 lambda: kv_reorder(k.transpose(2, 3), v.transpose(2, 3), p, 1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        kv_reorder(k.float(), v.float(), p, 1)
    c = kv8_empty(6, 1, 64, 64)
    with pytest.raises(ValueError, match="scales"):
        kv8_reorder(c[0], c[1], c[2][:, :, :1], c[3], p, 1)
    with pytest.raises(ValueError, match="tail"):
        kv8_reorder(*c[:3], c[3].float(), p, 1)
    with pytest.raises(RuntimeError, match="32 beams"):
        kv_reorder(torch.zeros(33, 1, 4, 8, device="cuda").half(), torch.zeros(33, 1, 4, 8, device="cuda").half(),
                   torch.zeros(1, 33, dtype=torch.int64, device="cuda"), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_long_rows_that_stream(dt):
    """Enough rows that a CTA's segment is longer than what it holds at once: masked beginnings, maxima anywhere, rising
    and falling logits, references that prove too low, ties across the segment, NaN and +inf."""
    require_b200()
    dtype = DTYPES[dt]
    B, K, V = 60, 10, 50021
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = (torch.randn(B, K, V, device="cuda", generator=g) * 2).to(dtype)
    scores = -torch.rand(B, K, device="cuda", generator=g) * 4
    check(logits, scores, 20)
    low = -math.inf if dt == "fp16" else torch.finfo(dtype).min
    logits[0, :, :40000] = low                   # a masked beginning
    logits[1] = low                              # nothing left
    logits[2] = low
    logits[2, 3, 49999] = 1.0                    # one token left, at the end
    logits[3, :, 30000:] += 200                  # the maximum far above the first elements
    logits[4, :, 30000:] -= 200
    logits[5] = torch.linspace(-20, 20, V, device="cuda").to(dtype)   # rising: every element is a new maximum
    logits[6] = torch.linspace(20, -20, V, device="cuda").to(dtype)
    logits[7] = 1.5                              # all equal
    logits[8, :, 9000:] = 3.0                    # thousands of equal ones behind the first elements
    logits[9, 0, 45000] = math.nan
    logits[10, 1, 45000] = math.inf
    logits[11] = -1500.0                         # far below zero throughout
    logits[12, :, :20000] = -600.0               # a plausible reference that is too low
    check(logits, scores, 20)
    check(logits[:, :, 1:], scores, 7)           # rows that start anywhere


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("V, n", [(2300, 64), (2049, 8), (4500, 40), (33000, 64), (9000, 64)])
def test_short_last_chunks_and_scattered_masks(V, n, dt):
    """Chunks that end after a few elements, and rows of which a few stretches are not masked, so that the threads'
    maxima say little about the n-th best."""
    require_b200()
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (torch.randn(2, 3, V, device="cuda", generator=g) * 3).to(dtype)
    scores = torch.tensor([[0.0, -0.5, -1.0], [-1.0, 0.0, -9.0]], device="cuda")
    check(logits, scores, n)
    low = -math.inf if dt != "bf16" else torch.finfo(dtype).min
    masked = torch.full_like(logits, low)
    for at in (0, 700, 1500, V - 30):
        masked[:, :, at:at + 300] = logits[:, :, at:at + 300]
    masked[0, 1] = low
    masked[0, 1, 100:103] = 1.0
    check(masked, scores, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("B, K, V", [(2, 4, 20011), (1, 3, 700), (60, 10, 50021)])  # the last one streams
def test_finite_logits_of_any_magnitude(B, K, V, dt):
    """One logit far above the others, up to the type's largest: its token at its beam's score, whatever the magnitude and
    wherever it lies; and whole rows far below zero."""
    require_b200()
    from tinker_b200.kernels import beam_select
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(V)
    top = torch.finfo(dtype).max
    for size in (1e6, 3e9, 1e10, 7e14, 1e30, 2.5e38, top):
        logits = (torch.randn(B, K, V, device="cuda", generator=g) * 2).to(dtype)
        at = torch.randint(0, V, (B, K), device="cuda", generator=g)
        at[:, 0] = 3  # among the first elements
        logits.scatter_(2, at[..., None], torch.full((B, K, 1), size, device="cuda", dtype=torch.float64).to(dtype))
        scores = -torch.rand(B, K, device="cuda", generator=g).cumsum(1)
        got, beams, tokens = beam_select(logits, scores, K)
        assert torch.equal(tokens, at)
        assert ((got.double() - scores.double()).abs() <= NEAR + 2.0 ** -24 * scores.double().abs()).all()  # log 1, as above
        assert torch.equal(beams, torch.arange(K, device="cuda").expand(B, K))
    low = (torch.randn(B, K, V, device="cuda", generator=g) * 2).to(dtype)
    low[:, 1] = -3e9
    low[:, 2] = -1e30
    check(low, torch.zeros(B, K, device="cuda"), 4)
