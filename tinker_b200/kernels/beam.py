"""Beam search on the sm_100a kernel library: the selection over beams and vocabulary, and the KV
caches' rows following the beams.

The reference has neither a KV cache nor a decoding loop (eb1386/TinKer README.md:97-103). A step of
``CachedDecoder.beam_search`` is ``beam_select`` on the logits of the step, then ``kv_reorder`` (or
``kv8_reorder``) of the cache by the beams that the selected candidates extend.
"""

from __future__ import annotations

import functools

import torch

from tinker_b200 import _lib
from tinker_b200.kernels._common import launch


@functools.lru_cache(maxsize=256)
def _workspace_bytes(idx: int, batch: int, beams: int, vocab: int, num_select: int, dtype: int) -> int:
    with torch.cuda.device(idx):
        n = _lib.lib().tk_beam_select_workspace(batch, beams, vocab, num_select, dtype)
    if n < 0:
        raise RuntimeError(f"tk_beam_select_workspace: {_lib.last_error()}")
    return n


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num_select: int | None = None,
                finished: torch.Tensor | None = None, eos_token_id: int | None = None):
    """The best ``num_select`` (default: the number of beams) continuations of every sequence.

    logits [batch, beams, vocab] (float16, bfloat16 or float32), scores [batch, beams] float32, the
    beams' log-probabilities so far. A continuation of beam k by token v is worth
    ``scores[k] + logits[k, v] - logsumexp(logits[k])``; the best come first, ties go to the lower
    ``k * vocab + v``. ``finished`` [batch, beams] bool (needs ``eos_token_id``): a finished beam has one
    continuation, ``eos_token_id`` at its score unchanged. A beam with score -inf (or NaN) has none:
    all its tokens are worth -inf, like NaN and -inf logits; a +inf logit counts as the largest finite
    value. Returns ``(scores float32, beams int64, tokens int64)``, each [batch, num_select].
    """
    idx = _lib.cuda_index(logits, scores)
    if logits.dim() != 3:
        raise ValueError(f"beam_select: logits must be [batch, beams, vocab], got {tuple(logits.shape)}")
    B, K, V = logits.shape
    n = K if num_select is None else int(num_select)
    if scores.shape != (B, K) or scores.dtype is not torch.float32:
        raise ValueError(f"beam_select: scores must be float32 [{B}, {K}]")
    if K < 1 or V < 1 or not 1 <= n <= K * V:
        raise ValueError(f"beam_select: cannot select {n} of {K} x {V} continuations")
    fin_ptr, eos = None, -1
    if finished is not None:
        _lib.cuda_index(logits, finished)
        if finished.shape != (B, K) or finished.dtype is not torch.bool:
            raise ValueError(f"beam_select: finished must be bool [{B}, {K}]")
        if eos_token_id is None or not 0 <= int(eos_token_id) < V:
            raise ValueError("beam_select: finished beams need an eos_token_id inside the vocabulary")
        finished = finished.contiguous()
        fin_ptr, eos = finished.data_ptr(), int(eos_token_id)
    st = logits.stride()
    row = st[1] if K > 1 else st[0]
    if (V > 1 and st[2] != 1) or row < V or (B > 1 and K > 1 and st[0] != K * st[1]):
        logits = logits.contiguous()
        row = V
    scores = scores.contiguous()
    out = scores.new_empty((B, n))
    beams = torch.empty((B, n), dtype=torch.int64, device=out.device)
    tokens = torch.empty_like(beams)
    if B == 0:
        return out, beams, tokens
    dtype = _lib.dtype_code(logits.dtype)
    need = _workspace_bytes(idx, B, K, V, n, dtype)
    ws = torch.empty(need, dtype=torch.uint8, device=out.device)
    launch(idx, "tk_beam_select", 2, _lib.lib().tk_beam_select, logits.data_ptr(), row, scores.data_ptr(), fin_ptr, eos,
           out.data_ptr(), beams.data_ptr(), tokens.data_ptr(), B, K, V, n, ws.data_ptr(), need, dtype)
    return out, beams, tokens


def _check_parents(what: str, parents: torch.Tensor, rows: int) -> torch.Tensor:
    if parents.dim() != 2 or parents.dtype is not torch.int64 or parents.numel() != rows:
        raise ValueError(f"{what}: parents must be int64 [groups, beams] with groups * beams = {rows} rows, "
                         f"got {tuple(parents.shape)} {parents.dtype}")
    return parents.contiguous()


def _length_args(what: str, length, capacity: int, device) -> tuple[int, int | None]:
    if isinstance(length, torch.Tensor):
        if length.dtype is not torch.int32 or length.device != device or length.numel() != 1:
            raise TypeError(f"{what}: a length tensor must be one int32 on the cache's device")
        return 0, length.data_ptr()
    length = int(length)
    if not 0 <= length <= capacity:
        raise ValueError(f"{what}: length {length} outside the cache's {capacity} positions")
    return length, None


def kv_reorder(k_cache: torch.Tensor, v_cache: torch.Tensor, parents: torch.Tensor, length) -> None:
    """Reorder the rows of a KV cache in place: of each group of beams, row i becomes what row
    ``parents[g, i]`` was. Only positions below ``length`` (an int, or a one-element int32 CUDA tensor that
    is read when the kernel runs) are moved, and rows that are their own parent are not touched.

    k_cache, v_cache: [rows, num_kv_heads, capacity, head_dim], or the same with a leading layer
    dimension; parents: int64 [groups, beams], groups * beams = rows, at most 32 beams. A group with a
    parent outside its beams stays as it is and device error 4 is recorded.
    """
    idx = _lib.cuda_index(k_cache, v_cache, parents)
    if k_cache.dim() not in (4, 5) or k_cache.shape != v_cache.shape or k_cache.dtype is not v_cache.dtype:
        raise ValueError("kv_reorder: k_cache and v_cache must both be [(layers,) rows, heads, capacity, head_dim]")
    if k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"kv_reorder: the cache must be float16 or bfloat16, got {k_cache.dtype}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("kv_reorder: the caches must be contiguous")
    rows, heads, cap, d = k_cache.shape[-4:]
    layers = k_cache.shape[0] if k_cache.dim() == 5 else 1
    parents = _check_parents("kv_reorder", parents, rows)
    n, n_ptr = _length_args("kv_reorder", length, cap, k_cache.device)
    groups, beams = parents.shape
    if rows == 0 or layers == 0 or heads == 0 or d == 0:
        return
    launch(idx, "tk_kv_reorder", 1 if beams > 1 and (n or n_ptr) else 0, _lib.lib().tk_kv_reorder, k_cache.data_ptr(),
           v_cache.data_ptr(), parents.data_ptr(), layers, groups, beams, heads, cap, d, n, n_ptr,
           _lib.dtype_code(k_cache.dtype))


def kv8_reorder(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, tail: torch.Tensor,
                parents: torch.Tensor, length) -> None:
    """``kv_reorder`` of an 8-bit cache (``kernels/kv_cache8.py``): the blocks, scales and open rows
    that hold positions below ``length``. The tensors may have a leading layer dimension."""
    idx = _lib.cuda_index(k_cache, v_cache, scales, tail, parents)
    lead = k_cache.shape[:-3]
    if k_cache.dim() not in (4, 5) or k_cache.shape != v_cache.shape or k_cache.dtype is not v_cache.dtype:
        raise ValueError("kv8_reorder: k_cache and v_cache must both be [(layers,) rows, heads, blocks, 32 * head_dim]")
    if k_cache.dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError(f"kv8_reorder: the cache must be float8_e4m3fn or int8, got {k_cache.dtype}")
    rows, heads, nb = k_cache.shape[-4:-1]
    d = k_cache.shape[-1] // 32
    if scales.shape != (*lead, heads, nb, 2) or scales.dtype is not torch.float32:
        raise ValueError(f"kv8_reorder: scales {tuple(scales.shape)} {scales.dtype} do not match the cache")
    if tail.shape != (*lead, heads, 2, 32, d) or tail.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"kv8_reorder: tail {tuple(tail.shape)} {tail.dtype} does not match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and scales.is_contiguous() and tail.is_contiguous()):
        raise ValueError("kv8_reorder: the cache tensors must be contiguous")
    layers = k_cache.shape[0] if k_cache.dim() == 5 else 1
    parents = _check_parents("kv8_reorder", parents, rows)
    n, n_ptr = _length_args("kv8_reorder", length, nb * 32, k_cache.device)
    groups, beams = parents.shape
    if rows == 0 or layers == 0 or heads == 0 or d == 0:
        return
    launch(idx, "tk_kv8_reorder", 1 if beams > 1 and (n or n_ptr) else 0, _lib.lib().tk_kv8_reorder, k_cache.data_ptr(),
           v_cache.data_ptr(), scales.data_ptr(), tail.data_ptr(), parents.data_ptr(), layers, groups, beams, heads, nb,
           d, n, n_ptr)
