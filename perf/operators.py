"""Cases that measure the 8-bit KV cache (append, attention), beam selection and cache reordering.

``run`` computes each operator in plain elementary torch operations (``own`` false) or through
``tinker_b200.kernels`` (``own`` true). The 8-bit cache keeps, for every sequence and kv head, blocks of 32
tokens: codes (float8_e4m3fn or int8) and one float32 scale for the block's keys and one for its values; the rows
of the last, incomplete block stay in 16 bits in ``tail`` [B, heads, 2 (k, v), 32, D]. A block's codes are stored in
the order in which a warp's matrix instructions take them (``_pack_keys``, ``_pack_values``).
"""

import math

import numpy as np
import torch

own = False

BLOCK = 32
LIMIT = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
FLOOR = 2.0 ** -60  # the least magnitude that a block's scale follows
HEADS = [(16, 4, 64), (14, 2, 64), (32, 8, 64), (8, 4, 128), (32, 8, 128), (16, 1, 64), (16, 16, 64)]


# ---------------------------------------------------------------------------- the cases


def listed():
    def att(name, **kw):
        return {"name": name, "op": "attention", "ragged": False, "S": 1, **kw}
    return [
        # one decode step of one sequence after a short prompt: latency alone
        att("decode_b1_127", B=1, hq=16, hkv=4, d=64, start=127, type="fp16", code="e4m3"),
        # a full batch at the end of a 2048-token context; the step completes a block
        att("decode_b64_2047", B=64, hq=16, hkv=4, d=64, start=2047, type="fp16", code="e4m3"),
        # two long documents on a model with few kv heads: the key axis has to be split
        att("decode_b2_100003", B=2, hq=14, hkv=2, d=64, start=100003, type="bf16", code="int8"),
        # wide heads, long contexts, the largest decode step
        att("decode_b16_16001", B=16, hq=32, hkv=8, d=128, start=16001, type="bf16", code="e4m3"),
        # continuous batching: every sequence at its own position
        att("decode_ragged_b48", B=48, hq=32, hkv=8, d=64, start=8191, type="fp16", code="int8", ragged=True),
        # the next piece of a long prompt against what is cached
        att("chunk_512_at_7001", B=1, hq=32, hkv=8, d=128, start=7001, S=512, type="bf16", code="e4m3"),
        # a short prompt's keys and values go into the cache
        {"name": "append_127", "op": "append", "B": 1, "hkv": 4, "d": 64, "start": 0, "S": 127, "type": "fp16", "code": "int8"},
        # a batch of long prompts
        {"name": "append_b16_4001", "op": "append", "B": 16, "hkv": 8, "d": 128, "start": 0, "S": 4001, "type": "bf16", "code": "e4m3"},
        # one beam search step of one prompt
        {"name": "select_1x4_32000", "op": "select", "B": 1, "K": 4, "V": 32000, "n": 8, "type": "fp16", "done": False},
        # a batch of beam searches over a large vocabulary, some beams finished
        {"name": "select_32x8_151936", "op": "select", "B": 32, "K": 8, "V": 151936, "n": 16, "type": "bf16", "done": True},
        # the 16-bit cache of all layers follows the beams of one prompt
        {"name": "reorder_1x4_301", "op": "reorder", "L": 18, "B": 1, "K": 4, "s": 2, "hkv": 4, "d": 64, "length": 301, "type": "fp16", "code": "none"},
        # the 8-bit cache of all layers follows the beams of a batch
        {"name": "reorder8_8x8_2001", "op": "reorder", "L": 16, "B": 8, "K": 8, "s": 4, "hkv": 8, "d": 64, "length": 2001, "type": "bf16", "code": "e4m3"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "chunk", "append", "select", "select", "reorder"])
    ty, code = rng.choice(["fp16", "bf16"]), rng.choice(["e4m3", "int8"])
    hq, hkv, d = rng.choice(HEADS)
    if op == "decode":
        B = _spread(rng, 1, 64)
        start = _spread(rng, 1, min(131000, (500 << 20) // (B * hkv * d * 2))) - 1
        return {"op": "attention", "B": B, "hq": hq, "hkv": hkv, "d": d, "start": start, "S": 1, "type": ty, "code": code,
                "ragged": rng.random() < 0.3}
    if op == "chunk":
        B, S = _spread(rng, 1, 4), _spread(rng, 2, 512)
        start = _spread(rng, 1, min(32000, (110 << 20) // (B * hq * S))) - 1
        return {"op": "attention", "B": B, "hq": hq, "hkv": hkv, "d": d, "start": start, "S": S, "type": ty, "code": code, "ragged": False}
    if op == "append":
        B = _spread(rng, 1, 32)
        return {"op": "append", "B": B, "hkv": hkv, "d": d, "start": _spread(rng, 1, 2000) - 1,
                "S": _spread(rng, 1, min(16000, (120 << 20) // (B * hkv * d * 2))), "type": ty, "code": code}
    if op == "select":
        B, K = _spread(rng, 1, 48), _spread(rng, 1, 16)
        V = _spread(rng, 1000, min(152064, max(1000, (70 << 20) // (B * K * 4))))
        return {"op": "select", "B": B, "K": K, "V": V, "n": rng.choice([K, 2 * K]), "type": rng.choice(["fp16", "bf16", "fp32"]),
                "done": rng.random() < 0.5}
    L, B, K = rng.choice([2, 16, 18, 24]), _spread(rng, 1, 8), _spread(rng, 2, 12)
    top = (1 << 30) // (L * B * K * hkv * d * 4)
    return {"op": "reorder", "L": L, "B": B, "K": K, "s": max(1, K // 2), "hkv": hkv, "d": d, "length": _spread(rng, 1, min(8000, max(1, top))),
            "type": ty, "code": rng.choice(["e4m3", "int8", "none"])}


def _starts(c):
    """The position of each sequence of an attention case: the same for all, or spread over 0 .. start."""
    if not c["ragged"]:
        return [c["start"]] * c["B"]
    return [int((b * 0.6180339887498949) % 1.0 * (c["start"] + 1)) if b else c["start"] for b in range(c["B"])]


def _blocks(positions):
    return (positions + BLOCK - 1) // BLOCK


def work(c):
    if c["op"] == "attention":
        starts, d, S = _starts(c), c["d"], c["S"]
        codes = sum(2 * d * (s // BLOCK * BLOCK) + 8 * (s // BLOCK) for s in starts) * c["hkv"]
        open_rows = sum(s % BLOCK for s in starts) * c["hkv"] * 4 * d
        new = c["B"] * S * d * (c["hq"] * 4 + c["hkv"] * 4) + S * d * 4
        stored = c["B"] * S * c["hkv"] * d * (4 if S < BLOCK else 2)
        keys = sum(S * s + S * (S + 1) // 2 for s in starts)
        return {"bytes": codes + open_rows + new + stored, "flops": 4 * c["hq"] * d * keys}
    if c["op"] == "append":
        rows = c["B"] * c["hkv"] * c["d"]
        r = c["start"] % BLOCK
        whole = (r + c["S"]) // BLOCK
        return {"bytes": rows * (4 * c["S"] + (4 * r if whole else 0) + 2 * BLOCK * whole + 4 * ((r + c["S"]) % BLOCK)),
                "flops": 4 * rows * c["S"]}
    if c["op"] == "select":
        size = 4 if c["type"] == "fp32" else 2
        rows = c["B"] * c["K"] - (c["B"] * (c["K"] // 4) if c["done"] else 0)
        return {"bytes": rows * c["V"] * size + c["B"] * c["n"] * 20, "flops": 4 * rows * c["V"]}
    return {"bytes": c["B"] * (c["s"] + c["K"] - 1) * _row_bytes(c), "flops": 0}


def _row_bytes(c):
    """What one row of a reordered cache holds over all layers and heads."""
    n, each = c["length"], c["L"] * c["hkv"]
    if c["code"] == "none":
        return each * n * c["d"] * 4
    return each * (n // BLOCK * (2 * BLOCK * c["d"] + 8) + n % BLOCK * c["d"] * 4)


# ---------------------------------------------------------------------------- inputs


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _tables(d, rows):
    inv = 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def _new_cache(c, positions, batch):
    nb = _blocks(positions)
    code = CODE[c["code"]]
    return {"k_cache": torch.zeros(batch, c["hkv"], nb, BLOCK * c["d"], dtype=torch.uint8, device="cuda").view(code),
            "v_cache": torch.zeros(batch, c["hkv"], nb, BLOCK * c["d"], dtype=torch.uint8, device="cuda").view(code),
            "scales": torch.zeros(batch, c["hkv"], nb, 2, device="cuda"),
            "tail": torch.zeros(batch, c["hkv"], 2, BLOCK, c["d"], dtype=TYPE[c["type"]], device="cuda")}


def _parents(c, seed):
    """For every group of K beams a parent for each, s of them with children elsewhere, one beam that stays."""
    rng, out = np.random.RandomState(seed % (1 << 32)), []
    for _ in range(c["B"]):
        for _ in range(20000):
            p = rng.permutation(np.resize(rng.permutation(c["K"])[:c["s"]], c["K"]))
            moved = p != np.arange(c["K"])
            if moved.sum() == c["K"] - 1 and len(set(p[moved])) == c["s"]:
                break
        out.append(p)
    return torch.tensor(np.stack(out), dtype=torch.int64, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    ty = TYPE[c["type"]]
    if c["op"] == "attention":
        B, S, d, starts = c["B"], c["S"], c["d"], _starts(c)
        top = max(starts) + S
        st = _new_cache(c, top, B)
        # what earlier steps stored: keys with some strong channels, values without
        gain = 1 + 3 * (torch.rand(c["hkv"], 1, 1, d, generator=g, device="cuda") < 0.05).float()
        nb = st["scales"].shape[2]
        for b in range(B):  # a sequence at a time: the 32-bit rows of all would not fit beside the cache
            k = (_randn(g, c["hkv"], nb, BLOCK, d) * gain).to(ty).float()
            v = _randn(g, c["hkv"], nb, BLOCK, d).to(ty).float()
            kc, ks = _quantise(k, c["code"])
            vc, vs = _quantise(v, c["code"])
            st["k_cache"].view(torch.uint8)[b] = _pack_keys(kc)
            st["v_cache"].view(torch.uint8)[b] = _pack_values(vc)
            st["scales"][b] = torch.stack([ks, vs], -1)
        st["tail"].copy_(_randn(g, *st["tail"].shape))
        w = _randn(g, B, S, (c["hq"] + 2 * c["hkv"]) * d).to(ty)  # one projection: q, k and v are its columns
        st["qkv"] = w
        st["cos"], st["sin"] = _tables(d, top)
        st["position"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if c["ragged"] else None
    elif c["op"] == "append":
        st = _new_cache(c, c["start"] + c["S"], c["B"])
        st["tail"].copy_(_randn(g, *st["tail"].shape))
        w = _randn(g, c["B"], c["S"], 2 * c["hkv"] * c["d"]).to(ty)
        st["k"], st["v"] = w[..., :c["hkv"] * c["d"]], w[..., c["hkv"] * c["d"]:]
    elif c["op"] == "select":
        B, K, V = c["B"], c["K"], c["V"]
        st = {"logits": (_randn(g, B, K, V) * 2.5).to(ty)}
        st["scores"] = -torch.rand(B, K, generator=g, device="cuda").cumsum(1) * 4
        st["finished"], st["eos"] = None, None
        if c["done"]:
            order = torch.rand(B, K, generator=g, device="cuda").argsort(1)
            st["finished"], st["eos"] = order < K // 4, 2
    else:
        rows, nb = c["B"] * c["K"], _blocks(c["length"])
        if c["code"] == "none":
            shape = (c["L"], rows, c["hkv"], c["length"], c["d"])
            st = {"k": torch.empty(shape, dtype=ty, device="cuda"), "v": torch.empty(shape, dtype=ty, device="cuda")}
            st["k"].normal_(generator=g)
            st["v"].normal_(generator=g)
        else:
            shape = (c["L"], rows, c["hkv"], nb, BLOCK * c["d"])
            st = {n: torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8).view(CODE[c["code"]]) for n in ("k", "v")}
            st["scales"] = torch.rand(c["L"], rows, c["hkv"], nb, 2, generator=g, device="cuda") + 0.01
            st["tail"] = _randn(g, c["L"], rows, c["hkv"], 2, BLOCK, c["d"]).to(ty)
        st["parents"] = _parents(c, seed)
    st["case"] = c
    return st


# ---------------------------------------------------------------------------- plain forms


def _quantise(x, code):
    """Codes (as values, 32 bits) and scales of blocks x [..., 32, d]; a block that is not finite gets the scale NaN."""
    a = x.abs().amax((-1, -2))
    fine = torch.isfinite(a)
    a = torch.where(fine, a, 1.0).clamp(min=FLOOR)
    y = torch.where(fine[..., None, None], x * (LIMIT[code] / a)[..., None, None], 0.0)
    y = y.round().to(torch.int8) if code == "int8" else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return y, torch.where(fine, a / torch.tensor(LIMIT[code], device=x.device), float("nan"))


def _pack_keys(codes):
    """[..., 32 tokens, d] -> [..., 32 * d] bytes: token 8a + 2j + e, column 64h + 16q + i at (j, h, a, e, q, i)."""
    x = codes.view(torch.uint8)
    lead, d = x.shape[:-2], x.shape[-1]
    n = len(lead)
    x = x.reshape(*lead, 4, 4, 2, d // 64, 4, 16)
    return x.permute(*range(n), n + 1, n + 3, n, n + 2, n + 4, n + 5).reshape(*lead, BLOCK * d)


def _pack_values(codes):
    """[..., 32 tokens, d] -> [..., 32 * d] bytes: token 8q + t, column 16m + 8e + r at (m, r, q, e, t)."""
    x = codes.view(torch.uint8)
    lead, d = x.shape[:-2], x.shape[-1]
    n = len(lead)
    x = x.reshape(*lead, 4, 8, d // 16, 2, 8)
    return x.permute(*range(n), n + 2, n + 4, n, n + 3, n + 1).reshape(*lead, BLOCK * d)


def _unpack_keys(b, code, d):
    lead = b.shape[:-1]
    n = len(lead)
    x = b.view(torch.uint8).reshape(*lead, 4, d // 64, 4, 2, 4, 16)
    return x.permute(*range(n), n + 2, n, n + 3, n + 1, n + 4, n + 5).reshape(*lead, BLOCK, d).view(CODE[code]).float()


def _unpack_values(b, code, d):
    lead = b.shape[:-1]
    n = len(lead)
    x = b.view(torch.uint8).reshape(*lead, d // 16, 8, 4, 2, 8)
    return x.permute(*range(n), n + 2, n + 4, n, n + 3, n + 1).reshape(*lead, BLOCK, d).view(CODE[code]).float()


def _rotate(x, cos, sin):
    """Interleaved pairs of x [B, heads, S, d] by the angles cos, sin [B, 1, S, d / 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _store(st, k, v, start):
    """Append rows k, v [B, heads, S, d] (16 bits) at position `start`, the same for all sequences."""
    code, S = st["case"]["code"], k.shape[2]
    r, first = start % BLOCK, start // BLOCK
    whole, rest = (r + S) // BLOCK, (r + S) % BLOCK
    rows = torch.stack([k, v], 2)
    if not whole:
        st["tail"][:, :, :, r:r + S] = rows
        return
    rows = torch.cat([st["tail"][:, :, :, :r], rows], 3)
    blocks = rows[:, :, :, :whole * BLOCK].float().unflatten(3, (whole, BLOCK))
    codes, scales = _quantise(blocks, code)
    at = slice(first, first + whole)
    st["k_cache"].view(torch.uint8)[:, :, at] = _pack_keys(codes[:, :, 0])
    st["v_cache"].view(torch.uint8)[:, :, at] = _pack_values(codes[:, :, 1])
    st["scales"][:, :, at] = scales.permute(0, 1, 3, 2)
    st["tail"][:, :, :, :rest] = rows[:, :, :, whole * BLOCK:]


def _store_one(st, k, v, position):
    """Append one row for each sequence, each at its own position."""
    code, b = st["case"]["code"], torch.arange(k.shape[0], device="cuda")
    at = position.long()
    full = (at % BLOCK == BLOCK - 1)[:, None, None]
    rows = torch.stack([k[:, :, 0], v[:, :, 0]], 2)
    blocks = torch.cat([st["tail"][:, :, :, :-1], rows[:, :, :, None]], 3).float()
    codes, scales = _quantise(blocks, code)
    kc, vc = st["k_cache"].view(torch.uint8), st["v_cache"].view(torch.uint8)
    n = at // BLOCK
    kc[b, :, n] = torch.where(full, _pack_keys(codes[:, :, 0]), kc[b, :, n])
    vc[b, :, n] = torch.where(full, _pack_values(codes[:, :, 1]), vc[b, :, n])
    st["scales"][b, :, n] = torch.where(full, scales, st["scales"][b, :, n])
    st["tail"][b, :, :, at % BLOCK] = torch.where(full[..., None], st["tail"][b, :, :, at % BLOCK], rows)


def _plain_attention(st):
    c = st["case"]
    B, S, d, hq, hkv = c["B"], c["S"], c["d"], c["hq"], c["hkv"]
    start = st["position"].long() if c["ragged"] else torch.full((B,), c["start"], device="cuda")
    qkv = st["qkv"].unflatten(-1, (hq + 2 * hkv, d)).transpose(1, 2)
    at = start[:, None] + torch.arange(S, device="cuda")
    cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]
    q = _rotate(qkv[:, :hq].float(), cos, sin)
    k = _rotate(qkv[:, hq:hq + hkv].float(), cos, sin).to(qkv.dtype)
    v = qkv[:, hq + hkv:]
    # keys from the complete blocks, from the open block, from this call; where each of them sits
    sc = st["scales"][..., None, None, :]
    keys = torch.cat([(_unpack_keys(st["k_cache"], c["code"], d) * sc[..., 0]).flatten(2, 3), st["tail"][:, :, 0].float(), k.float()], 2)
    vals = torch.cat([(_unpack_values(st["v_cache"], c["code"], d) * sc[..., 1]).flatten(2, 3), st["tail"][:, :, 1].float(), v.float()], 2)
    n = keys.shape[2] - BLOCK - S
    base = start // BLOCK * BLOCK
    i = torch.arange(n, device="cuda")[None].expand(B, n)
    j = base[:, None] + torch.arange(BLOCK, device="cuda")
    where = torch.cat([torch.where(i < base[:, None], i, 1 << 40), torch.where(j < start[:, None], j, 1 << 40), at], 1)
    q = q.reshape(B, hkv, hq // hkv, S, d).flatten(2, 3)
    score = torch.matmul(q, keys.transpose(2, 3)) / math.sqrt(d)
    seen = (where[:, None, :] <= at[:, :, None]).repeat(1, hq // hkv, 1)[:, None]
    score = torch.where(seen, score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p, vals) / p.sum(-1, keepdim=True)
    o = o.reshape(B, hq, S, d).transpose(1, 2).reshape(B, S, hq * d).to(qkv.dtype)
    if c["ragged"]:
        _store_one(st, k, v, st["position"])
    else:
        _store(st, k, v, c["start"])
    return o


def _plain_select(st):
    c = st["case"]
    B, K, V = c["B"], c["K"], c["V"]
    x = st["logits"].float()
    x = torch.where(torch.isnan(x), float("-inf"), x).clamp(max=torch.finfo(st["logits"].dtype).max)
    top = x.amax(-1, keepdim=True)
    safe = torch.where(torch.isinf(top), 0.0, top)
    lse = safe.double() + torch.exp(x - safe).double().sum(-1, keepdim=True).log()
    cand = st["scores"].double()[..., None] + torch.where(torch.isinf(x), x.double(), x.double() - lse)
    if st["finished"] is not None:
        only = torch.where(torch.arange(V, device="cuda") == st["eos"], st["scores"].double()[..., None], float("-inf"))
        cand = torch.where(st["finished"][..., None], only, cand)
    val, idx = cand.reshape(B, K * V).sort(dim=-1, descending=True, stable=True)
    val, idx = val[:, :c["n"]], idx[:, :c["n"]]
    return val.float(), idx // V, idx % V


def _plain_reorder(st):
    c = st["case"]
    n, rows = c["length"], c["B"] * c["K"]
    src = (st["parents"] + torch.arange(c["B"], device="cuda")[:, None] * c["K"]).reshape(rows)
    if c["code"] == "none":
        for t in (st["k"], st["v"]):
            t[:, :, :, :n] = t[:, src, :, :n]
        return st["k"], st["v"]
    whole, rest = n // BLOCK, n % BLOCK
    for t in (st["k"].view(torch.uint8), st["v"].view(torch.uint8), st["scales"]):
        t[:, :, :, :whole] = t[:, src, :, :whole]
    st["tail"][:, :, :, :, :rest] = st["tail"][:, src, :, :, :rest]
    return st["k"], st["v"], st["scales"], st["tail"]


def run(state):
    st = state
    c = st["case"]
    if c["op"] == "attention":
        if own:
            from tinker_b200.kernels import kv8_attention, kv8_attention_workspace
            q, k, v = st["qkv"].split([c["hq"] * c["d"], c["hkv"] * c["d"], c["hkv"] * c["d"]], -1)
            if "workspace" not in st:  # zeroed scratch that a decoder keeps beside its cache
                need = kv8_attention_workspace(c["B"], c["hq"], c["hkv"], c["d"], c["S"], st["scales"].shape[2] * BLOCK)
                st["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
            out = kv8_attention(q, k, v, st["cos"], st["sin"], st["k_cache"], st["v_cache"], st["scales"], st["tail"], c["hq"],
                                c["hkv"], c["d"], start_pos=c["start"], position=st["position"], workspace=st["workspace"])
        else:
            out = _plain_attention(st)
        return out, st["k_cache"], st["v_cache"], st["scales"], st["tail"]
    if c["op"] == "append":
        if own:
            from tinker_b200.kernels import kv8_append
            kv8_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["scales"], st["tail"], c["start"])
        else:
            k, v = (st[n].unflatten(-1, (c["hkv"], c["d"])).transpose(1, 2) for n in ("k", "v"))
            _store(st, k, v, c["start"])
        return st["k_cache"], st["v_cache"], st["scales"], st["tail"]
    if c["op"] == "select":
        if own:
            from tinker_b200.kernels import beam_select
            return beam_select(st["logits"], st["scores"], c["n"], finished=st["finished"], eos_token_id=st["eos"])
        return _plain_select(st)
    if own:
        from tinker_b200.kernels import kv8_reorder, kv_reorder
        if c["code"] == "none":
            kv_reorder(st["k"], st["v"], st["parents"], c["length"])
            return st["k"], st["v"]
        kv8_reorder(st["k"], st["v"], st["scales"], st["tail"], st["parents"], c["length"])
        return st["k"], st["v"], st["scales"], st["tail"]
    return _plain_reorder(st)


# ---------------------------------------------------------------------------- in 64 bits


def _exact_code(x, code):
    """x [..., 32, d] in 64 bits -> (nearest codes as values, scale), ties to even."""
    a = x.abs().amax((-1, -2), keepdim=True).clamp(min=FLOOR)
    y = x * (LIMIT[code] / a)
    if code == "int8":
        step = torch.ones_like(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step, a[..., 0, 0] / LIMIT[code]


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] == "attention":
        starts, S, d, hq, hkv = _starts(c), c["S"], c["d"], c["hq"], c["hkv"]
        if c["B"] * hq * S * (max(starts) + S) > 300e6:
            return None
        x = st["qkv"].double().reshape(c["B"], S, hq + 2 * hkv, d)
        out = torch.empty(c["B"], S, hq, d, dtype=torch.float64, device="cuda")
        for b, p in enumerate(starts):
            ang = torch.complex(st["cos"][p:p + S].double(), st["sin"][p:p + S].double())[:, None]
            turned = torch.view_as_real(torch.view_as_complex(x[b, :, :hq + hkv].reshape(S, hq + hkv, d // 2, 2).contiguous()) * ang)
            turned = turned.reshape(S, hq + hkv, d)
            new = turned[:, hq:].to(st["qkv"].dtype).double()
            nb, r = p // BLOCK, p % BLOCK
            seen = torch.arange(p + S, device="cuda")[None] > p + torch.arange(S, device="cuda")[:, None]
            for h in range(hkv):
                kb = _unpack_keys(st["k_cache"][b, h, :nb], c["code"], d).double() * st["scales"][b, h, :nb, 0].double()[:, None, None]
                vb = _unpack_values(st["v_cache"][b, h, :nb], c["code"], d).double() * st["scales"][b, h, :nb, 1].double()[:, None, None]
                K = torch.cat([kb.reshape(-1, d), st["tail"][b, h, 0, :r].double(), new[:, h]])
                V = torch.cat([vb.reshape(-1, d), st["tail"][b, h, 1, :r].double(), x[b, :, hq + hkv + h]])
                for i in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    s = (turned[:, i] @ K.T / math.sqrt(d)).masked_fill(seen, float("-inf"))
                    out[b, :, i] = torch.softmax(s, -1) @ V
        return out.reshape(c["B"], S, hq * d), None, None, None, None
    if c["op"] == "append":
        d, S, start = c["d"], c["S"], c["start"]
        r, first, code = start % BLOCK, start // BLOCK, c["code"]
        whole = (r + S) // BLOCK
        rows = torch.stack([st[n].double().reshape(c["B"], S, c["hkv"], d).permute(0, 2, 1, 3) for n in ("k", "v")], 2)
        tail = st["tail"].double()
        if not whole:
            tail[:, :, :, r:r + S] = rows
            return None, None, st["scales"].double(), tail
        rows = torch.cat([tail[:, :, :, :r], rows], 3)
        tail[:, :, :, :rows.shape[3] - whole * BLOCK] = rows[:, :, :, whole * BLOCK:]
        codes, sc = _exact_code(rows[:, :, :, :whole * BLOCK].reshape(c["B"], c["hkv"], 2, whole, BLOCK, d), code)
        scales = st["scales"].double()
        scales[:, :, first:first + whole] = sc.permute(0, 1, 3, 2)
        if code == "int8":
            return None, None, scales, tail
        out = []
        for i, pack in ((0, _pack_keys), (1, _pack_values)):  # codes are whole sixteenths of a byte pattern: pack their patterns
            full = torch.zeros(c["B"], c["hkv"], _blocks(start + S), BLOCK * d, dtype=torch.float64, device="cuda")
            full[:, :, first:first + whole] = pack(codes[:, :, i].to(torch.float8_e4m3fn)).view(torch.float8_e4m3fn).double()
            out.append(full)
        return out[0], out[1], scales, tail
    if c["op"] == "select":
        B, K, V = c["B"], c["K"], c["V"]
        best = torch.empty(B, c["n"], dtype=torch.float64, device="cuda")
        for b in range(B):
            lp = torch.log_softmax(st["logits"][b].double(), -1) + st["scores"][b].double()[:, None]
            if st["finished"] is not None:
                done = st["finished"][b]
                lp[done] = float("-inf")
                lp[done, st["eos"]] = st["scores"][b].double()[done]
            best[b] = lp.reshape(-1).topk(c["n"]).values
        return best, None, None
    return None
