"""KV cache in 8 bits on the sm_100a kernel library: append, attention, and reading it back.

The reference has no KV cache (eb1386/TinKer README.md:102); ``kernels/kv_cache.py`` keeps one in the
model type, this one in half of that. Keys (after RoPE) and values are stored in blocks of
``KV8_BLOCK`` = 32 tokens, each block and kv head with one float32 scale for its keys and one for its
values; the rows of the block that is not complete yet stay in 16 bits:

    k_cache, v_cache  [batch, num_kv_heads, num_blocks, 32 * head_dim]  float8_e4m3fn or int8 codes
    scales            [batch, num_kv_heads, num_blocks, 2]              float32 (keys, values)
    tail              [batch, num_kv_heads, 2 (keys, values), 32, head_dim]  model type

With a the largest magnitude of a block, at least 2^-60, and M = 448 (e4m3) or 127 (int8):
``scale = a / M``, ``code = round(x * (M * (1 / a)))``, ties to even. A block that holds a NaN or an
infinity gets the scale NaN. A block is quantised once, when its last token arrives, so what the
cache holds does not depend on how the tokens were split into calls. Codes are stored in the order in
which the kernels read them; ``kv8_dequantize`` gives rows back.

Positions go up: the rows of the open block below the position must be the ones that earlier calls
left in the tail. A cache may start over at 0 or at any multiple of 32 that it holds.
"""

from __future__ import annotations

import functools

import torch

from tinker_b200 import _lib
from tinker_b200.kernels._common import launch

KV8_BLOCK = 32
KV8_FORMATS = {torch.float8_e4m3fn: 0, torch.int8: 1}


def kv8_blocks(positions: int) -> int:
    """Blocks that a cache of ``positions`` tokens needs."""
    return (positions + KV8_BLOCK - 1) // KV8_BLOCK


def kv8_empty(batch: int, num_kv_heads: int, head_dim: int, capacity: int, dtype: torch.dtype = torch.float16,
              code: torch.dtype = torch.float8_e4m3fn, device="cuda", layers: int | None = None):
    """Empty ``(k_cache, v_cache, scales, tail)`` for ``capacity`` positions (rounded up to whole
    blocks); with ``layers`` each gets a leading dimension."""
    if code not in KV8_FORMATS:
        raise TypeError(f"unsupported cache type {code}; expected float8_e4m3fn or int8")
    lead = (batch,) if layers is None else (layers, batch)
    nb = kv8_blocks(capacity)
    # zeros by bytes: torch fills float8 tensors through a slower path
    k, v = (torch.zeros(*lead, num_kv_heads, nb, KV8_BLOCK * head_dim, dtype=torch.uint8, device=device).view(code)
            for _ in range(2))
    scales = torch.zeros(*lead, num_kv_heads, nb, 2, dtype=torch.float32, device=device)
    tail = torch.zeros(*lead, num_kv_heads, 2, KV8_BLOCK, head_dim, dtype=dtype, device=device)
    return k, v, scales, tail


def kv8_attention_workspace(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, seq: int,
                            max_kv: int) -> int:
    """Bytes of zero-filled workspace ``kv8_attention`` needs for these sizes when at most ``max_kv``
    keys are attended (the cache's capacity when the position is a tensor)."""
    n = _lib.lib().tk_kv8_attention_workspace(batch, num_heads, num_kv_heads, head_dim, seq, max_kv)
    if n < 0:
        raise RuntimeError(f"tk_kv8_attention_workspace: {_lib.last_error()}")
    return int(n)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(idx: int, *sizes) -> int:
    """``kv8_attention_workspace`` on device ``idx``."""
    with torch.cuda.device(idx):
        return kv8_attention_workspace(*sizes)


@functools.lru_cache(maxsize=256)
def _launches(idx: int, *sizes) -> int:
    """Kernels that a call on device ``idx`` launches."""
    with torch.cuda.device(idx):
        return _lib.lib().tk_kv8_attention_launches(*sizes)


def _rows(t: torch.Tensor, B: int, S: int, width: int) -> tuple[torch.Tensor, int]:
    """(tensor, token stride) of [B, S, width] rows that start on 16 bytes and follow one another at one
    stride; anything else is copied."""
    if t.shape != (B, S, width):
        raise ValueError(f"expected shape ({B}, {S}, {width}), got {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    tok = s1 if S > 1 else (s0 if B > 1 else width)
    if s2 == 1 and tok >= width and tok % 8 == 0 and (B == 1 or S == 1 or s0 == S * s1) and t.data_ptr() % 16 == 0:
        return t, tok
    return t.clone(memory_format=torch.contiguous_format), width


def _check_cache(what: str, k_cache, v_cache, scales, tail, batch: int, heads: int, head_dim: int,
                 dtype: torch.dtype) -> tuple[int, int]:
    """(blocks, format code) of a cache that fits the call; raises otherwise."""
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"{what}: rows must be float16 or bfloat16, got {dtype}")
    code = KV8_FORMATS.get(k_cache.dtype)
    if code is None or v_cache.dtype is not k_cache.dtype:
        raise TypeError(f"{what}: k_cache and v_cache must both be float8_e4m3fn or both int8")
    if scales.dtype is not torch.float32 or tail.dtype is not dtype:
        raise TypeError(f"{what}: scales must be float32 and the tail of the rows' type")
    shape = k_cache.shape
    nb = shape[2] if len(shape) == 4 else 0
    if shape != (batch, heads, nb, KV8_BLOCK * head_dim) or v_cache.shape != shape:
        raise ValueError(f"{what}: cache shape {tuple(shape)} / {tuple(v_cache.shape)} does not match batch {batch}, "
                         f"{heads} kv heads, head_dim {head_dim}")
    if scales.shape != (batch, heads, nb, 2) or tail.shape != (batch, heads, 2, KV8_BLOCK, head_dim):
        raise ValueError(f"{what}: scales {tuple(scales.shape)} or tail {tuple(tail.shape)} do not match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and scales.is_contiguous() and tail.is_contiguous()):
        raise ValueError(f"{what}: the cache tensors must be contiguous")
    return nb, code


def kv8_attention(q, k, v, cos_table, sin_table, k_cache, v_cache, scales, tail, num_heads, num_kv_heads, head_dim,
                  start_pos: int = 0, position: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of S new tokens per sequence against an 8-bit cache, then their append.

    q: [B, S, num_heads * head_dim], k / v: [B, S, num_kv_heads * head_dim] (column slices of a fused
    projection are read in place); cos_table / sin_table: float32 [max_seq_len, head_dim // 2], or both
    None when q and k are rotated already. The new tokens sit at ``start_pos ..``, or from
    ``position`` on, an int32 CUDA tensor of one element or of one per sequence that is read when the
    kernel runs (one CUDA graph serves every step); a position outside the cache or the tables then
    records device error 2, leaves that sequence's cache untouched and gives rows of NaN for it. Keys of complete blocks
    are read as ``code * scale``, those of the open block and of this call in 16 bits. A row that sees a
    token whose key or value holds a NaN or an infinity is NaN throughout. q and the softmax's weights are
    products in two parts of 11 bits; from 64 query rows of a kv head on (S > 1, position on the host) on
    tensor-core tiles, where the weights are rounded to 11 bits, and q too for bfloat16. ``workspace``:
    zero-filled uint8 CUDA tensor of at least ``kv8_attention_workspace(...)`` bytes, left so that
    later calls of any shape can use it, but not calls that overlap in time (allocated per call when
    omitted). Returns [B, S, num_heads * head_dim] in q's dtype.
    """
    idx = _lib.cuda_index(q, k, v, k_cache, v_cache, scales, tail)
    dtype = q.dtype
    if q.dim() != 3 or k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("kv8_attention: q, k, v must be [batch, seq, heads * head_dim], all float16 or all bfloat16")
    B, S, width = q.shape
    nb, code = _check_cache("kv8_attention", k_cache, v_cache, scales, tail, B, num_kv_heads, head_dim, dtype)
    q, qs = _rows(q, B, S, num_heads * head_dim)
    k, ks = _rows(k, B, S, num_kv_heads * head_dim)
    v, vs = _rows(v, B, S, num_kv_heads * head_dim)
    cos_ptr = sin_ptr = None
    rows = 0
    if cos_table is not None or sin_table is not None:
        if cos_table is None or sin_table is None:
            raise ValueError("kv8_attention: give both RoPE tables or neither")
        _lib.cuda_index(q, cos_table, sin_table)
        if cos_table.dtype is not torch.float32 or sin_table.dtype is not torch.float32:
            raise TypeError("kv8_attention: the RoPE tables must be float32")
        if cos_table.dim() != 2 or cos_table.shape[1] != head_dim // 2 or sin_table.shape != cos_table.shape:
            raise ValueError(f"RoPE tables must be [max_seq_len, {head_dim // 2}], got {tuple(cos_table.shape)}")
        cos_table, sin_table = cos_table.contiguous(), sin_table.contiguous()
        cos_ptr, sin_ptr, rows = cos_table.data_ptr(), sin_table.data_ptr(), cos_table.shape[0]
    pos_ptr, step = None, 0
    if position is not None:
        n = position.numel()
        if position.dtype is not torch.int32 or position.get_device() != idx or n not in (1, B):
            raise TypeError("kv8_attention: position must be an int32 tensor on q's device with 1 or batch elements")
        if n > 1:
            position = position.contiguous()
            step = 1
        pos_ptr, start_pos = position.data_ptr(), 0
    else:
        start_pos = int(start_pos)
        if start_pos < 0 or start_pos + S > nb * KV8_BLOCK:
            raise ValueError(f"kv8_attention: positions {start_pos}..{start_pos + S - 1} exceed the cache capacity "
                             f"{nb * KV8_BLOCK}")
    out = q.new_empty((B, S, width))
    if B == 0 or S == 0:
        return out
    need = base = _workspace_bytes(idx, 1, num_heads, num_kv_heads, head_dim, 1, 1)  # independent of the other sizes
    if S > 1 and pos_ptr is None:
        need = _workspace_bytes(idx, B, num_heads, num_kv_heads, head_dim, S, start_pos + S)
    if workspace is None:  # only the form for few rows counts on zeros
        workspace = (torch.empty if need > base else torch.zeros)(need, dtype=torch.uint8, device=out.device)
    elif workspace.nbytes < need or workspace.get_device() != idx or not workspace.is_contiguous():
        raise ValueError(f"kv8_attention: workspace smaller than the {need} bytes needed, or not contiguous")
    kernels = 1 if S == 1 else 2
    if need > base:
        kernels = _launches(idx, B, num_heads, num_kv_heads, head_dim, S, start_pos, _lib.dtype_code(dtype))
    launch(idx, "tk_kv8_attention", kernels, _lib.lib().tk_kv8_attention, q.data_ptr(), qs, k.data_ptr(), ks,
           v.data_ptr(), vs, k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), tail.data_ptr(), nb, code,
           cos_ptr, sin_ptr, rows, out.data_ptr(), width, B, S, num_heads, num_kv_heads, head_dim, start_pos, pos_ptr,
           step, workspace.data_ptr(), need, _lib.dtype_code(dtype))
    return out


def kv8_append(k, v, k_cache, v_cache, scales, tail, start_pos: int = 0) -> None:
    """Append k (already rotated) and v, [B, S, num_kv_heads * head_dim], at ``start_pos``."""
    idx = _lib.cuda_index(k, v, k_cache, v_cache, scales, tail)
    if k.dim() != 3 or k_cache.dim() != 4 or v.dtype is not k.dtype:
        raise ValueError("kv8_append: k and v must be [batch, seq, heads * head_dim] of one type, the cache "
                         "[batch, heads, blocks, 32 * head_dim]")
    B, S, _ = k.shape
    _, hkv, _, block = k_cache.shape
    D = block // KV8_BLOCK
    nb, code = _check_cache("kv8_append", k_cache, v_cache, scales, tail, B, hkv, D, k.dtype)
    k, ks = _rows(k, B, S, hkv * D)
    v, vs = _rows(v, B, S, hkv * D)
    start_pos = int(start_pos)
    if start_pos < 0 or start_pos + S > nb * KV8_BLOCK:
        raise ValueError(f"kv8_append: positions {start_pos}..{start_pos + S - 1} exceed the cache capacity "
                         f"{nb * KV8_BLOCK}")
    launch(idx, "tk_kv8_append", 1 if B * S else 0, _lib.lib().tk_kv8_append, k.data_ptr(), ks, v.data_ptr(), vs,
           k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), tail.data_ptr(), nb, code, B, S, hkv, D, start_pos,
           _lib.dtype_code(k.dtype))


def kv8_unpack(codes: torch.Tensor, values: bool, head_dim: int) -> torch.Tensor:
    """Codes [..., 32 * head_dim] in the kernels' order -> [..., 32, head_dim] by token and column."""
    lead, n = codes.shape[:-1], codes.dim() - 1
    x = codes.view(torch.uint8)
    if values:  # [m][r][q][e][t]: token 8q + t, column 16m + 8e + r
        x = x.reshape(*lead, head_dim // 16, 8, 4, 2, 8)
        x = x.permute(*range(n), n + 2, n + 4, n, n + 3, n + 1)
    else:  # [j][h][a][e][q][i]: token 8a + 2j + e, column 64h + 16q + i
        x = x.reshape(*lead, 4, head_dim // 64, 4, 2, 4, 16)
        x = x.permute(*range(n), n + 2, n, n + 3, n + 1, n + 4, n + 5)
    return x.reshape(*lead, KV8_BLOCK, head_dim).view(codes.dtype)


def kv8_dequantize(k_cache, v_cache, scales, tail, length: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of positions ``0 .. length - 1`` as the attention reads them, float32
    [batch, num_kv_heads, length, head_dim] each (for inspection and tests: plain torch operations)."""
    head_dim = tail.shape[-1]
    nb, rest = length // KV8_BLOCK, length % KV8_BLOCK
    if length < 0 or nb + (rest > 0) > k_cache.shape[2]:
        raise ValueError(f"kv8_dequantize: length {length} exceeds the cache")
    out = []
    for i, codes in enumerate((k_cache, v_cache)):
        x = kv8_unpack(codes[:, :, :nb], i == 1, head_dim).float() * scales[:, :, :nb, i, None, None]
        out.append(torch.cat([x.flatten(2, 3), tail[:, :, i, :rest].float()], 2))
    return out[0], out[1]
