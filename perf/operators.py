"""The operators of the 4-bit KV cache: writing it (quantise), reading it back, attending over it.

A cached key or value row of one kv head is stored as GGUF Q4_0 blocks of 32
values: one binary16 scale d and 32 codes c in 0..15, standing for (c - 8) d.

  append   d = f16(m / -8) with m the block's value of largest magnitude (the
           lowest index on ties), c = clamp(rint(x / d), -8, 7) + 8, rint half
           to even, c = 8 where d = 0; the call returns the rows as the cache
           now holds them.
  read     (c - 8) d for a range of tokens of every layer, as fp32 or binary16.
  decode   one query token per sequence: softmax(q K^T / sqrt(head_dim)) V over
           the sequence's cached tokens (and the token appended by the call),
           grouped-query heads, zeros for a sequence that holds no token.

`own` false: elementary torch operations in fp32; `own` true: this package's
KV4Cache.  Queries and keys are used as given (already rotated).
"""
import math

import torch

own = False

_DEV = "cuda"


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # A decoder's per-layer call early in a chat, Qwen2.5-0.5B heads: the call's latency.
        dict(name="decode_65_tokens", op="decode", layers=1, seqs=1, tokens=65, ragged=False, kv_heads=2, group=7,
             head_dim=64, page_tokens=128, f16=False, append=False),
        # Every layer of a 3B decode step at a 4K context, the benchmark's headline shape.
        dict(name="decode_3b_4k", op="decode", layers=36, seqs=1, tokens=4097, ragged=False, kv_heads=2, group=8,
             head_dim=128, page_tokens=128, f16=False, append=False),
        # One layer of a serving batch: 64 sequences of 0 to 8192 tokens, 7B heads (an idle slot among them).
        dict(name="decode_7b_ragged64", op="decode", layers=1, seqs=64, tokens=8192, ragged=True, kv_heads=4, group=7,
             head_dim=128, page_tokens=128, f16=False, append=False),
        # Every layer of a 7B decode step over a long document.
        dict(name="decode_7b_32k", op="decode", layers=28, seqs=1, tokens=32768, ragged=False, kv_heads=4, group=7,
             head_dim=128, page_tokens=128, f16=False, append=False),
        # A whole step of the 0.5B model's cache: quantise the new token, attend, read the stored row back.
        dict(name="step_05b_1000", op="decode", layers=24, seqs=1, tokens=1000, ragged=False, kv_heads=2, group=7,
             head_dim=64, page_tokens=64, f16=False, append=True),
        # One key/value head per query head, binary16 queries, a few odd lengths.
        dict(name="decode_mha_f16_odd", op="decode", layers=4, seqs=3, tokens=777, ragged=True, kv_heads=8, group=1,
             head_dim=128, page_tokens=64, f16=True, append=False),
        # One token of every layer of the 0.5B model (a step whose attention runs elsewhere): latency.
        dict(name="append_1_token", op="append", layers=24, tokens=1, base=100, kv_heads=2, head_dim=64,
             page_tokens=128, f16=False),
        # A whole prompt of the 3B model, every layer.
        dict(name="append_3b_2k", op="append", layers=36, tokens=2048, base=0, kv_heads=2, head_dim=128,
             page_tokens=128, f16=True),
        # One layer of a prompt's later chunk: an odd count that starts inside a page.
        dict(name="append_chunk_777", op="append", layers=1, tokens=777, base=37, kv_heads=4, head_dim=128,
             page_tokens=128, f16=False),
        # A page of one layer, for a prefix that another sequence shares: latency.
        dict(name="read_1_page", op="read", layers=1, tokens=128, base=0, kv_heads=2, head_dim=64, page_tokens=128,
             f16=False),
        # The history of a 7B sequence, every layer, as the binary16 rows that a prompt pass attends.
        dict(name="read_7b_16k", op="read", layers=28, tokens=16384, base=0, kv_heads=4, head_dim=128,
             page_tokens=128, f16=True),
        # A few layers from an odd first token, fp32.
        dict(name="read_odd_f32", op="read", layers=3, tokens=4097, base=5, kv_heads=2, head_dim=128, page_tokens=192,
             f16=False),
    ]


_MOST = 28 * 32768 * 4 * 128  # values of K (or V) of the largest listed attention case
_MOST_BYTES = 1.2e9           # of the largest listed case's pass


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "append", "read"])
    hd = rng.choice([64, 128])
    kvh = rng.choice([1, 2, 4, 8])
    layers = _log_uniform(rng, 1, 36)
    page = rng.choice([64, 128, 192])
    f16 = rng.random() < 0.5
    if op == "decode":
        seqs = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 64)
        most = _MOST // (layers * seqs * kvh * hd)
        tokens = _log_uniform(rng, 1, max(1, min(32768, most)))
        return dict(op=op, layers=layers, seqs=seqs, tokens=tokens, ragged=seqs > 1, kv_heads=kvh,
                    group=rng.choice([1, 2, 4, 5, 6, 7, 8, 12, 16]), head_dim=hd, page_tokens=page, f16=f16,
                    append=seqs == 1 and rng.random() < 0.5)
    value = 2 * ((2 if op == "append" else 1) * (2 if f16 else 4) + 18 / 32)  # bytes that a key and its value move
    tokens = _log_uniform(rng, 1, max(1, min(32768, int(_MOST_BYTES / value) // (layers * kvh * hd))))
    return dict(op=op, layers=layers, tokens=tokens, base=rng.choice([0, 1, 5, 16, 37, 64, 129]), kv_heads=kvh,
                head_dim=hd, page_tokens=page, f16=f16)


def _lengths(case):
    """Cached tokens of each sequence: spread evenly over 0 .. tokens in a ragged batch."""
    s, t = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [t] * s
    return [t if i == s - 1 else int(t * ((i * 0.6180339887498949) % 1.0)) for i in range(s)]


def work(case):
    hd, kvh, layers = case["head_dim"], case["kv_heads"], case["layers"]
    row = kvh * (hd // 32) * 18  # bytes of one token's keys (or values) in the cache
    in_bytes = 2 if case["f16"] else 4
    if case["op"] == "decode":
        n = sum(_lengths(case))
        heads = kvh * case["group"]
        new = case["seqs"] if case["append"] else 0
        byt = 2 * n * row + case["seqs"] * heads * hd * (in_bytes + 4)
        byt += new * 2 * (kvh * hd * (in_bytes + 4) + row)  # new rows in, their blocks, and the rows read back
        return {"bytes": layers * byt, "flops": layers * 4 * heads * hd * (n + new)}
    n = layers * case["tokens"]
    if case["op"] == "append":  # rows in, blocks out, stored rows out
        return {"bytes": n * 2 * (2 * kvh * hd * in_bytes + row), "flops": n * 2 * kvh * hd * 5}
    return {"bytes": n * 2 * (row + kvh * hd * in_bytes), "flops": n * 2 * kvh * hd * 2}


# ---------------------------------------------------------------- inputs

def _rows(gen, shape, outliers):
    """Key or value rows: unit normal values; keys have a few strong channels, as trained models do."""
    x = torch.randn(shape, generator=gen, device=_DEV, dtype=torch.float32)
    if outliers:
        hd = shape[-1]
        gain = torch.ones(hd, device=_DEV)
        gain[torch.randint(0, hd, (max(1, hd // 16),), generator=gen, device=_DEV)] = 5.0
        x *= gain
    return x


def _blocks(x):
    """fp32 rows [..., head_dim] as raw Q4_0 blocks [..., head_dim / 32, 18] uint8: byte j of a block's 16
    holds value j (low nibble) and value j + 16 (high nibble)."""
    codes, d = _quantise(x)
    c = codes.to(torch.uint8)
    packed = c[..., :16] | (c[..., 16:] << 4)
    return torch.cat([d.view(torch.uint8), packed], dim=-1)


def _cached(gen, case, seqs, tokens):
    """Raw blocks of keys and values [layers, seqs, tokens, kv_heads, blocks, 18], made layer by layer."""
    hd, kvh = case["head_dim"], case["kv_heads"]
    shape = (seqs, tokens, kvh, hd)
    k = torch.empty((case["layers"], seqs, tokens, kvh, hd // 32, 18), dtype=torch.uint8, device=_DEV)
    v = torch.empty_like(k)
    for layer in range(case["layers"]):
        k[layer] = _blocks(_rows(gen, shape, True))
        v[layer] = _blocks(_rows(gen, shape, False))
    return k, v


def _inputs(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    hd, kvh, layers = case["head_dim"], case["kv_heads"], case["layers"]
    typ = torch.float16 if case["f16"] else torch.float32
    s = {"case": case}
    if case["op"] == "decode":
        heads = kvh * case["group"]
        s["k"], s["v"] = _cached(gen, case, case["seqs"], case["tokens"])
        s["q"] = (2.0 * torch.randn((layers, case["seqs"], heads, hd), generator=gen, device=_DEV)).to(typ)
        if case["append"]:
            s["k_new"] = _rows(gen, (layers, 1, kvh, hd), True).to(typ)
            s["v_new"] = _rows(gen, (layers, 1, kvh, hd), False).to(typ)
    elif case["op"] == "append":
        shape = (layers, case["tokens"], kvh, hd)
        s["k"] = _rows(gen, shape, True).to(typ)
        s["v"] = _rows(gen, shape, False).to(typ)
        s["v"][:, 0, 0] = 0.0  # a padding row: blocks of zeros
    else:
        s["k"], s["v"] = _cached(gen, case, 1, case["base"] + case["tokens"])
    return s


_engine = None


def _own_engine():
    global _engine
    if _engine is None:
        from tinymetalagent_b200 import AttnEngine
        _engine = AttnEngine(0)
    return _engine


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        eng = _own_engine()
        hd, kvh, layers = case["head_dim"], case["kv_heads"], case["layers"]
        decode = case["op"] == "decode"
        lens = _lengths(case) if decode else [case["base"] + (case["tokens"] if case["op"] == "read" else 0)]
        room = max(lens) + (1 if decode else case["tokens"])
        cache = eng.kv4_cache(layers=layers, max_seqs=len(lens), max_tokens_per_seq=room, kv_heads=kvh, head_dim=hd,
                              page_tokens=case["page_tokens"])
        torch.cuda.synchronize()
        if case["op"] != "append":
            # sequences that grow together take their pages in turn
            for t in range(case["page_tokens"], room + case["page_tokens"], case["page_tokens"]):
                for i, n in enumerate(lens):
                    if t - case["page_tokens"] < n:
                        cache.reserve(i, min(t, room))
            for i, n in enumerate(lens):
                if n:
                    k, v = s["k"][:, i, :n].contiguous(), s["v"][:, i, :n].contiguous()
                    torch.cuda.synchronize()
                    cache.write_q4_0(0, layers, i, 0, n, k, v)
                    eng.synchronize()
            del s["k"], s["v"]
        elif case["base"]:
            zero = torch.zeros((layers, case["base"], kvh, hd // 32, 18), dtype=torch.uint8, device=_DEV)
            torch.cuda.synchronize()
            cache.write_q4_0(0, layers, 0, 0, case["base"], zero, zero)
            eng.synchronize()
        s["cache"] = cache
        f32, typ = torch.float32, (torch.float16 if case["f16"] else torch.float32)
        if decode:
            s["seq_ids"] = list(range(case["seqs"]))
            s["out"] = torch.empty((layers, case["seqs"], kvh * case["group"], hd), dtype=f32, device=_DEV)
            rows = (layers, 1, kvh, hd)
        else:
            rows = (layers, case["tokens"], kvh, hd)
        s["k_rows"] = torch.empty(rows, dtype=typ, device=_DEV)
        s["v_rows"] = torch.empty(rows, dtype=typ, device=_DEV)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "decode":
        return _plain_decode(s, case)
    typ = torch.float16 if case["f16"] else torch.float32
    if case["op"] == "append":
        return {"k": _stand_for(*_quantise(s["k"].float())).to(typ), "v": _stand_for(*_quantise(s["v"].float())).to(typ)}
    begin = case["base"]
    return {"k": _values(s["k"][:, 0, begin:]).to(typ), "v": _values(s["v"][:, 0, begin:]).to(typ)}


def _run_own(s, case):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_NO_ROPE, TE_ATTN_OUTPUT_F16
    cache, layers = s["cache"], case["layers"]
    f16 = TE_ATTN_INPUT_F16 if case["f16"] else 0
    rows16 = TE_ATTN_OUTPUT_F16 if case["f16"] else 0
    if case["op"] == "append":
        cache.append(0, layers, 0, s["k"], s["v"], case["tokens"], k_stored=s["k_rows"], v_stored=s["v_rows"],
                     flags=TE_ATTN_NO_ROPE | f16 | rows16)
        return {"k": s["k_rows"], "v": s["v_rows"]}
    if case["op"] == "read":
        cache.read(0, layers, 0, case["base"], case["tokens"], s["k_rows"], s["v_rows"], flags=rows16)
        return {"k": s["k_rows"], "v": s["v_rows"]}
    heads = case["kv_heads"] * case["group"]
    if not case["append"]:
        cache.decode(0, layers, s["seq_ids"], s["q"], s["out"], heads, flags=TE_ATTN_NO_ROPE | f16)
        return {"out": s["out"]}
    cache.decode(0, layers, s["seq_ids"], s["q"], s["out"], heads, k_new=s["k_new"], v_new=s["v_new"],
                 flags=TE_ATTN_NO_ROPE | TE_ATTN_ADVANCE | f16)
    cache.read(0, layers, 0, case["tokens"], 1, s["k_rows"], s["v_rows"], flags=rows16)
    cache.truncate(0, case["tokens"])  # the next pass appends the same token again
    return {"out": s["out"], "k": s["k_rows"], "v": s["v_rows"]}


# ---------------------------------------------------------------- the plain form

def _quantise(x):
    """fp32 rows [..., head_dim] -> codes [..., head_dim / 32, 32] (0..15, fp32) and binary16 scales [..., 1]."""
    b = x.unflatten(-1, (-1, 32))
    m = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = (m * -0.125).clamp(-65504.0, 65504.0).to(torch.float16)
    df = d.float()
    t = torch.where(df == 0, torch.zeros_like(b), b / df)
    return t.round().clamp(-8.0, 7.0) + 8.0, d


def _stand_for(codes, d):
    return ((codes - 8.0) * d.float()).flatten(-2)


def _values(blocks):
    """Raw Q4_0 blocks [..., n, 18] uint8 -> fp32 values [..., 32 n]."""
    d = blocks[..., 0:2].contiguous().view(torch.float16)
    q = blocks[..., 2:]
    return _stand_for(torch.cat([q & 15, q >> 4], dim=-1).float(), d)


def _plain_decode(s, case):
    layers, seqs, kvh, hd = case["layers"], case["seqs"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    k, v = _values(s["k"]), _values(s["v"])  # [layers, seqs, tokens, kv_heads, hd]
    if case["append"]:
        k_row = _stand_for(*_quantise(s["k_new"].float()))
        v_row = _stand_for(*_quantise(s["v_new"].float()))
        k = torch.cat([k, k_row[:, :, None]], dim=2)
        v = torch.cat([v, v_row[:, :, None]], dim=2)
    n = torch.tensor([x + int(case["append"]) for x in lens], device=_DEV)
    q = s["q"].float().view(layers, seqs, kvh, case["group"], hd)
    sc = torch.matmul(q, k.permute(0, 1, 3, 4, 2)) / math.sqrt(hd)  # [layers, seqs, kv_heads, group, tokens]
    past = torch.arange(k.shape[2], device=_DEV) >= n[:, None]
    sc = sc.masked_fill(past[None, :, None, None, :], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 1, 3, 2, 4)) / total
    out = torch.where(total > 0, out, torch.zeros_like(out)).reshape(layers, seqs, kvh * case["group"], hd)
    if not case["append"]:
        return {"out": out}
    typ = torch.float16 if case["f16"] else torch.float32
    return {"out": out, "k": k_row.to(typ), "v": v_row.to(typ)}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_row(x):
    """What the blocks of these rows stand for, in fp64."""
    r = x.double().reshape(-1, 32)
    at = r.abs().argmax(1)
    top = r[torch.arange(r.shape[0], device=r.device), at]
    d = (top / -8.0).clamp(-65504.0, 65504.0).to(torch.float16).double()[:, None]
    steps = torch.where(d == 0.0, 0.0, r / torch.where(d == 0.0, 1.0, d))
    return (steps.round().clamp(-8.0, 7.0) * d).reshape(x.shape)


def _exact_read(raw):
    """The values of raw blocks [..., n, 18], in fp64."""
    lo, hi = raw[..., 0].to(torch.int32), raw[..., 1].to(torch.int32)
    d = (lo + 256 * hi).to(torch.int16).view(torch.float16).double()
    val = torch.empty(raw.shape[:-1] + (32,), dtype=torch.float64, device=raw.device)
    val[..., :16] = torch.remainder(raw[..., 2:], 16).double()
    val[..., 16:] = torch.div(raw[..., 2:], 16, rounding_mode="floor").double()
    return ((val - 8.0) * d[..., None]).reshape(raw.shape[:-2] + (-1,))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "append":
        return {"k": _exact_row(s["k"]), "v": _exact_row(s["v"])}
    if case["op"] == "read":
        out = {}
        for name in ("k", "v"):
            out[name] = torch.stack([_exact_read(layer[0, case["base"]:]) for layer in s[name]])
        return out
    layers, kvh, group, hd = case["layers"], case["kv_heads"], case["group"], case["head_dim"]
    out = torch.zeros((layers, case["seqs"], kvh * group, hd), dtype=torch.float64, device=_DEV)
    rows = {}
    if case["append"]:
        rows = {"k": _exact_row(s["k_new"]), "v": _exact_row(s["v_new"])}
    for layer in range(layers):
        for i, n in enumerate(_lengths(case)):
            if n == 0:
                continue  # only batches hold an idle slot, and they append nothing
            k, v = _exact_read(s["k"][layer, i, :n]), _exact_read(s["v"][layer, i, :n])
            if rows:
                k, v = torch.cat([k, rows["k"][layer]]), torch.cat([v, rows["v"][layer]])
            for h in range(kvh):
                q = s["q"][layer, i, h * group:(h + 1) * group].double()
                z = (k[:, h] @ q.T) * hd ** -0.5
                w = torch.exp(z - z.max(0).values)
                out[layer, i, h * group:(h + 1) * group] = (w.T @ v[:, h]) / w.sum(0)[:, None]
    return {"out": out, **rows}
