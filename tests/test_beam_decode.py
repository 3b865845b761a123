"""Cached decoding with an 8-bit cache, and beam search, at the model level: the operators as a run."""

import math

import pytest
import torch

from tests._util import DTYPES, require_b200
from tests.test_kv_cache import _decoder


@pytest.mark.gpu
@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("prompt_len", [100, 8])
def test_decoder_with_8bit_cache(prompt_len, dt, code):
    """Prefill and graph steps over several blocks against the same decoder with a 16-bit cache. A code is off by at most
    2^-4 of a value (e4m3) or 1/254 of a block's largest (int8); the logits of the random model (of the order of 1) may
    move by a few hundredths, and a wrong block, scale or row moves them by their own size."""
    require_b200()
    import tinker_b200
    from bench_model import make_tokens
    cfg, _, model = _decoder(3, DTYPES[dt])
    B, steps = 2, 70
    tokens = make_tokens(cfg, B, prompt_len + steps, seed=3).cuda()
    outs = []
    for kind in (None, code):
        for graph in (True, False):
            dec = tinker_b200.CachedDecoder(model, batch_size=B, capacity=200, cuda_graph=graph, cache_dtype=kind)
            with torch.inference_mode():
                got = [dec.prefill(tokens[:, :prompt_len]).float().clone()]
                got += [dec.decode(tokens[:, t]).float().clone() for t in range(prompt_len, prompt_len + steps)]
            outs.append(torch.stack(got))
            assert dec.length == prompt_len + steps
            dec.release()
    full, full_eager, eight, eight_eager = outs
    rms = full.square().mean().sqrt()
    assert (eight - eight_eager).square().mean().sqrt() <= 2e-2 * rms  # graph and eager split the keys otherwise
    assert (eight - full).square().mean().sqrt() <= 8e-2 * rms


@pytest.mark.gpu
def test_chunked_prefill_and_cache_contents():
    """A prompt in three pieces (the later ones read the cache) leaves the same 8-bit cache up to the rounding of the
    rows' own computation, and reset serves a second prompt."""
    require_b200()
    import tinker_b200
    from bench_model import make_tokens
    from tinker_b200.kernels import kv8_dequantize
    cfg, _, model = _decoder(2)
    tokens = make_tokens(cfg, 2, 150, seed=5).cuda()
    dec = tinker_b200.CachedDecoder(model, batch_size=2, capacity=160, cache_dtype=torch.int8)
    ref = tinker_b200.CachedDecoder(model, batch_size=2, capacity=160)
    with torch.inference_mode():
        dec.generate(tokens[:, 90:130], 3)
        dec.reset()
        for lo, hi in ((0, 50), (50, 53), (53, 150)):
            got = dec.prefill(tokens[:, lo:hi]).float().clone()
        want = ref.prefill(tokens).float()
    assert dec.length == 150
    assert (got - want).square().mean().sqrt() <= 8e-2 * want.square().mean().sqrt()
    k, v = kv8_dequantize(dec.cache.k[0], dec.cache.v[0], dec.cache.scales[0], dec.cache.tail[0], 150)
    for x, y in ((k, ref.cache.k[0]), (v, ref.cache.v[0])):  # layer 0 sees the same tokens: one code step apart at most
        y = y[:, :, :150].float()
        assert (x - y).abs().max() <= y.abs().max() / 254 * 1.2 + 2.0 ** -9 * y.abs().max()


@pytest.mark.gpu
def test_cache_dtype_refusals():
    require_b200()
    import tinker_b200
    _, _, model = _decoder(1)
    with pytest.raises(TypeError, match="cache_dtype"):
        tinker_b200.CachedDecoder(model, 1, 64, cache_dtype=torch.float32)
    with pytest.raises(ValueError, match="fused decode step"):
        tinker_b200.CachedDecoder(model, 1, 64, cache_dtype=torch.int8, fused_step=True)
    dec = tinker_b200.CachedDecoder(model, 4, 40, cache_dtype=torch.int8)
    assert dec.cache.capacity == 64
    prompt = torch.zeros(1, 41, dtype=torch.long)
    with pytest.raises(ValueError, match="capacity"):
        dec.prefill(prompt.repeat(4, 1))
    for bad in ((prompt, 3, 2), (prompt[0], 4, 2), (prompt.repeat(2, 1), 4, 2)):
        with pytest.raises(ValueError):
            dec.beam_search(*bad)


def _scored(model, prompt, seqs, eos):
    """The sum of log-probabilities of every beam's tokens (up to the end token) by the full forward, fp64."""
    P, K, n = seqs.shape
    S = prompt.shape[1]
    full = torch.cat([prompt.repeat_interleave(K, 0), seqs.reshape(P * K, n).to(prompt.device)], 1)
    with torch.inference_mode():
        lp = torch.log_softmax(model(full).double()[:, S - 1:-1], -1)
    lp = lp.gather(2, full[:, S:, None])[..., 0].reshape(P, K, n)
    if eos is not None:
        ended = (seqs == eos).int().cumsum(2) - (seqs == eos).int()
        lp = torch.where(ended.to(lp.device) > 0, 0.0, lp)
    return lp.sum(2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [None, torch.int8])
@pytest.mark.parametrize("P, K, n, eos", [(1, 4, 40, None), (3, 3, 20, 17), (2, 1, 9, None), (1, 8, 6, 5)])
def test_beam_search(P, K, n, eos, kind):
    """The returned scores are those of the full forward over the returned sequences (so every cache row followed its
    beam through every step), sorted, all beams different; one beam is the greedy path."""
    require_b200()
    import tinker_b200
    from bench_model import make_tokens
    cfg, _, model = _decoder(2)
    prompt = make_tokens(cfg, P, 30, seed=7).cuda()
    dec = tinker_b200.CachedDecoder(model, batch_size=P * K, capacity=128, cache_dtype=kind)
    seqs, scores = dec.beam_search(prompt, K, n, eos_token_id=eos)
    assert seqs.shape[:2] == (P, K) and seqs.shape[2] <= n and scores.shape == (P, K)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    want = _scored(model, prompt, seqs, eos)
    # logits agree to 2e-2 (the bar of the cached decoder), so a log-probability of a token to twice that
    assert (scores.double() - want).abs().max() <= 4e-2 * seqs.shape[2] * (1 if kind is None else 3)
    for p in range(P):
        assert len({tuple(r.tolist()) for r in seqs[p]}) == K
    if K == 1:
        one = tinker_b200.CachedDecoder(model, batch_size=P, capacity=128, cache_dtype=kind)
        assert torch.equal(seqs[:, 0], one.generate(prompt, n))


@pytest.mark.gpu
def test_beam_search_is_the_exhaustive_search_when_wide():
    """Beams enough for every prefix of a tiny vocabulary: the best sequences of all."""
    require_b200()
    import itertools
    import tinker_b200
    from bench_model import TINY, build_model
    cfg = TINY.with_(vocab_size=5)
    model = tinker_b200.optimize(build_model(cfg, seed=1).to("cuda"), dtype=torch.float16, cuda_graph=False)
    prompt = torch.tensor([[1, 4, 2], [0, 0, 3]], device="cuda")
    dec = tinker_b200.CachedDecoder(model, batch_size=2 * 25, capacity=32)
    seqs, scores = dec.beam_search(prompt, 25, 3)
    every = torch.tensor(list(itertools.product(range(5), repeat=3)))
    val = _scored(model, prompt, every[None].repeat(2, 1, 1), None)
    best = val.sort(dim=1, descending=True).values[:, :25]
    assert (scores.double() - best).abs().max() <= 0.12  # three tokens of 4e-2
    seqs, scores = dec.beam_search(prompt, 25, 3, eos_token_id=4, length_penalty=1.0)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    ended = (seqs == 4).int().cumsum(2)
    assert ((seqs == 4) | (ended == 0)).all()  # only the end token follows an end token
    assert torch.isfinite(scores).all() and not math.isnan(scores.sum().item())
    assert dec.beam_search(prompt, 25, 0)[0].shape == (2, 25, 0)


@pytest.mark.gpu
def test_beam_search_and_the_capacity():
    """A search that cannot fit is refused before it begins, and leaves the decoder as it was; one that may end early runs
    as far as the cache goes."""
    require_b200()
    import tinker_b200
    from bench_model import make_tokens
    cfg, _, model = _decoder(1)
    prompt = make_tokens(cfg, 1, 30, seed=7).cuda()
    dec = tinker_b200.CachedDecoder(model, batch_size=3, capacity=40)
    full, scores = dec.beam_search(prompt, 3, 11)  # 30 + 11 - 1 positions
    assert full.shape == (1, 3, 11) and dec.length == 40
    with pytest.raises(ValueError, match="capacity 40"):
        dec.beam_search(prompt, 3, 12)
    assert dec.length == 40  # nothing ran
    with pytest.raises(ValueError, match="capacity 40"):
        dec.beam_search(make_tokens(cfg, 1, 41, seed=7), 3, 1, eos_token_id=1)
    assert dec.beam_search(make_tokens(cfg, 1, 60, seed=7), 3, 0)[0].shape == (1, 3, 0)  # nothing to place
    ends = int(next(t for t in range(cfg.vocab_size) if not (full == t).any()))  # never chosen, so no beam ends
    seqs, got = dec.beam_search(prompt, 3, 50, eos_token_id=ends)
    assert torch.equal(seqs, full) and torch.equal(got, scores)
