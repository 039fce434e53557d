"""The 4-bit KV cache on the GPU against a plain restatement: stored blocks bit for bit, attention against
fp64 over the values the blocks stand for.

The attention's tolerance follows from its arithmetic.  With B the largest sum |q_d k_d| / sqrt(hd) over
a head's tokens, a score is off by at most B (2^-22 [two-part query] + 12 2^-23 [fp32 sums, which the tensor
core may truncate] + 3 2^-23 [scaling and exponent]); weights move by that in relative terms, twice (weight
and sum).  The two-part weights add 2^-21, and each of the n / 16 accumulation steps of the second product
at most 2^-22.  All of it multiplies the largest |value|.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the plain restatement

def quantise(x):
    """fp32 rows [..., hd] -> raw Q4_0 blocks [..., hd / 32, 18] uint8."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    mag = np.abs(b)
    bad = ~np.isfinite(b).all(-1)
    at = np.argmax(np.where(np.isfinite(mag), mag, 0), -1)[..., None]
    m = np.take_along_axis(b, at, -1)
    with np.errstate(all="ignore"):
        d = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16)
        df = d.astype(np.float32)
        r = np.clip(np.rint(np.where(df == 0, np.float32(0), b / df)), -8, 7)
    c = np.where(bad[..., None], 8, np.nan_to_num(r) + 8).astype(np.uint8)
    bits = d.view(np.uint16)
    bits = np.where(bad[..., None], np.uint16(0x7FFF), bits).astype(np.uint16)
    return np.concatenate([bits.view(np.uint8), c[..., :16] | (c[..., 16:] << 4)], -1)


def values(blocks):
    """Raw blocks [..., n, 18] -> fp64 values [..., 32 n]."""
    d = np.ascontiguousarray(blocks[..., :2]).view(np.float16).astype(np.float64)
    q = blocks[..., 2:]
    c = np.concatenate([q & 15, q >> 4], -1).astype(np.float64)
    return ((c - 8) * d).reshape(*blocks.shape[:-2], -1)


def rotate(port, rows, positions, theta=1e6):
    """fp32 rows [n, heads, hd] rotated at their positions, by the oracle."""
    out = np.array(rows, np.float32)
    for i, pos in enumerate(positions):
        r = np.ascontiguousarray(out[i]).ravel()
        port.rope_f32(r, rows.shape[1], rows.shape[2], int(pos), theta)
        out[i] = r.reshape(rows.shape[1:])
    return out


def attend(q, k, v):
    """q [heads, hd], k and v [n, kv_heads, hd] fp64 -> out [heads, hd] and its tolerance [heads, 1]."""
    heads, hd = q.shape
    n, kvh = k.shape[:2]
    out, tol = np.zeros((heads, hd)), np.zeros((heads, 1))
    for h in range(heads if n else 0):
        kk, vv = k[:, h // (heads // kvh)], v[:, h // (heads // kvh)]
        s = kk @ q[h] / np.sqrt(hd)
        w = np.exp(s - s.max())
        out[h] = (w / w.sum()) @ vv
        big = (np.abs(kk) @ np.abs(q[h])).max() / np.sqrt(hd)
        ds = big * (2.0**-22 + 15 * 2.0**-23)
        tol[h] = np.abs(vv).max() * (2 * ds + 2.0**-21 + (n / 16 + 8) * 2.0**-22)
    return out, tol


def check(got, q, k, v):
    exp, tol = attend(np.asarray(q, np.float64), k, v)
    err = np.abs(np.asarray(got, np.float64) - exp)
    assert np.isfinite(got).all() and (err <= tol).all(), (err.max(), tol.min())


# ---------------------------------------------------------------- helpers

def dev(x, typ=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if typ is None else t.to(typ)).cuda()


def ready(engine):
    """Orders the engine's stream after torch's (the inputs' copies)."""
    import torch
    torch.cuda.synchronize()
    return engine


def blocks_of(cache, layers, seq, begin, n):
    import torch
    shape = (layers, n, cache.kv_heads, cache.head_dim // 32, 18)
    k = torch.zeros(shape, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    torch.cuda.synchronize()
    cache.read_q4_0(0, layers, seq, begin, n, k, v)
    cache.engine.synchronize()
    return k.cpu().numpy(), v.cpu().numpy()


def fill(cache, seq, k, v, begin=0):
    """Rows [layers, n, kv_heads, hd] into the cache as blocks made here; returns the values they stand for."""
    kb, vb = quantise(k), quantise(v)
    kd, vd = dev(kb), dev(vb)
    ready(cache.engine)
    cache.write_q4_0(0, k.shape[0], seq, begin, k.shape[1], kd, vd)
    cache.engine.synchronize()
    return values(kb), values(vb)


def run_decode(cache, seqs, q, heads, **kw):
    import torch
    from tinymetalagent_b200 import TE_ATTN_PARTIAL
    width = q.shape[-1] + (2 if kw.get("flags", 0) & TE_ATTN_PARTIAL else 0)
    out = torch.full((*q.shape[:-1], width), float("nan"), device="cuda")
    for name in ("k_new", "v_new"):
        if kw.get(name) is not None:
            kw[name] = dev(kw[name])
    qd = dev(q)
    ready(cache.engine)
    cache.decode(0, q.shape[0], seqs, qd, out, heads, **kw)
    cache.engine.synchronize()
    return out.cpu().numpy()


def rows(rng, *shape, gain=1.0):
    return (rng.standard_normal(shape) * gain).astype(np.float32)


# ---------------------------------------------------------------- writing

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,first,n,f16,rope,bias", [
    (2, 0, 1, False, True, False), (2, 37, 3, False, True, True), (1, 5, 43, True, True, False),
    (3, 64, 64, False, False, False), (4, 15, 130, True, False, True), (2, 128, 16, False, True, True)])
def test_append_blocks_bit_exact(port, engine, hd, kvh, first, n, f16, rope, bias):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_NO_ROPE, TE_ATTN_QKV_BIAS
    rng = np.random.default_rng(hd + first + n)
    layers, p0 = 2, 700
    typ = np.float16 if f16 else np.float32
    cache = engine.kv4_cache(layers=layers, max_seqs=2, max_tokens_per_seq=320, kv_heads=kvh, head_dim=hd,
                             page_tokens=64, max_position=p0 + 320)
    cache.reset(1, p0)
    old_k, old_v = rows(rng, layers, max(first, 1), kvh, hd), rows(rng, layers, max(first, 1), kvh, hd)
    if first:
        fill(cache, 1, old_k, old_v)
    k, v = rows(rng, layers, n, kvh, hd).astype(typ), rows(rng, layers, n, kvh, hd, gain=3).astype(typ)
    kb, vb = rows(rng, layers, kvh * hd), rows(rng, layers, kvh * hd)
    if bias:
        cache.set_qkv_bias(0, kvh, None, kb, vb)
    flags = TE_ATTN_ADVANCE | (TE_ATTN_INPUT_F16 if f16 else 0) | (0 if rope else TE_ATTN_NO_ROPE) | \
        (TE_ATTN_QKV_BIAS if bias else 0)
    kd, vd = dev(k), dev(v)
    ready(engine)
    cache.append(0, layers, 1, kd, vd, n, flags=flags)
    assert cache.length(1) == first + n
    got_k, got_v = blocks_of(cache, layers, 1, 0, first + n)
    for layer in range(layers):
        kk, vv = k[layer].astype(np.float32), v[layer].astype(np.float32)
        if bias:
            kk, vv = kk + kb[layer].reshape(kvh, hd), vv + vb[layer].reshape(kvh, hd)
        if rope:
            kk = rotate(port, kk, range(p0 + first, p0 + first + n))
        assert np.array_equal(got_k[layer, first:], quantise(kk))
        assert np.array_equal(got_v[layer, first:], quantise(vv))
        if first:  # the tokens that were there
            assert np.array_equal(got_k[layer, :first], quantise(old_k[layer]))
            assert np.array_equal(got_v[layer, :first], quantise(old_v[layer]))
    cache.close()


def edge_rows(hd):
    """Rows whose blocks lie at the quantiser's edges."""
    e = np.zeros((12, hd), np.float32)
    e[1] = 1.0                                 # all equal: the first is m, all at the range's far end
    e[2, ::2], e[2, 1::2] = 2.0, -2.0          # ties in magnitude with both signs
    e[3, 5], e[3, 9] = -4.0, 4.0               # the lower index wins
    e[4] = np.linspace(-8, 8, hd)              # quotients at halves
    e[5] = np.arange(hd) % 17 * 0.5 - 4.0
    e[6, 0] = 1e-7                             # d a binary16 subnormal
    e[7, 3] = 1e-9                             # d rounds to zero
    e[8, 1], e[8, 2] = 4e5, -3.0               # close to the largest scale
    e[9, 1] = 3e38                             # d saturates
    e[10, 0::3], e[10, 1::3] = 7.0, -6.999
    e[11] = 6e-8
    return e


@pytest.mark.parametrize("hd", [64, 128])
def test_append_edges_and_non_finite(engine, hd):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_NO_ROPE
    import torch
    e = edge_rows(hd)
    bad = np.stack([rows(np.random.default_rng(i), hd) for i in range(3)])
    bad[0, 3], bad[1, 40], bad[2, 33] = np.nan, np.inf, -np.inf
    x = np.concatenate([e, bad])[None, :, None, :]
    n = x.shape[1]
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=64, kv_heads=1, head_dim=hd)
    kd, vd = dev(x), dev(x[:, ::-1])
    ks, vs = torch.zeros_like(kd), torch.zeros_like(vd)
    ready(engine)
    cache.append(0, 1, 0, kd, vd, n, ks, vs, flags=TE_ATTN_ADVANCE | TE_ATTN_NO_ROPE)
    got_k, got_v = blocks_of(cache, 1, 0, 0, n)
    exp = quantise(x)
    assert np.array_equal(got_k, exp) and np.array_equal(got_v, exp[:, ::-1])
    stored = ks.cpu().numpy().astype(np.float64)
    want = values(exp)
    assert np.array_equal(np.isnan(stored), np.isnan(want))
    assert np.isnan(want).sum() == 3 * 32  # only the blocks that hold the bad values
    ok = ~np.isnan(want)
    assert np.array_equal(stored[ok], want[ok])
    assert np.array_equal(vs.cpu().numpy()[:, ::-1][ok], ks.cpu().numpy()[ok])
    cache.close()


@pytest.mark.parametrize("hd,f16", [(64, True), (128, False), (128, True)])
def test_append_returns_what_it_stored(engine, hd, f16):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_OUTPUT_F16
    import torch
    rng = np.random.default_rng(3)
    n, kvh, layers = 51, 2, 3
    cache = engine.kv4_cache(layers=layers, max_seqs=1, max_tokens_per_seq=128, kv_heads=kvh, head_dim=hd)
    typ = np.float16 if f16 else np.float32
    kd, vd = dev(rows(rng, layers, n, kvh, hd).astype(typ)), dev(rows(rng, layers, n, kvh, hd).astype(typ))
    out16 = TE_ATTN_OUTPUT_F16 if f16 else 0
    out = [torch.zeros_like(kd) for _ in range(4)]
    ready(engine)
    cache.append(0, layers, 0, kd, vd, n, out[0], out[1],
                 flags=TE_ATTN_ADVANCE | out16 | (TE_ATTN_INPUT_F16 if f16 else 0))
    cache.read(0, layers, 0, 0, n, out[2], out[3], flags=out16)
    engine.synchronize()
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])
    got_k, got_v = blocks_of(cache, layers, 0, 0, n)
    assert np.array_equal(out[2].cpu().numpy(), values(got_k).astype(np.float32).astype(typ))
    assert np.array_equal(out[3].cpu().numpy(), values(got_v).astype(np.float32).astype(typ))
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("f16,out16", [(False, True), (True, False), (False, False), (True, True)])
@pytest.mark.parametrize("first,n", [(0, 1), (5, 40), (13, 3), (16, 77)])
def test_append_returns_either_type_from_either(engine, hd, f16, out16, first, n):
    """Returned rows of the other type, single tokens and ranges that start inside a tile; what lies around the
    returned rows stays as it was."""
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_OUTPUT_F16
    import torch
    rng = np.random.default_rng(31)
    kvh, layers = 3, 2
    cache = engine.kv4_cache(layers=layers, max_seqs=1, max_tokens_per_seq=128, kv_heads=kvh, head_dim=hd)
    if first:
        fill(cache, 0, rows(rng, layers, first, kvh, hd), rows(rng, layers, first, kvh, hd))
    typ, out_type = np.float16 if f16 else np.float32, torch.float16 if out16 else torch.float32
    kd, vd = dev(rows(rng, layers, n, kvh, hd).astype(typ)), dev(rows(rng, layers, n, kvh, hd).astype(typ))
    count = layers * n * kvh * hd
    room = [torch.full((count + 64,), 7.0, device="cuda", dtype=out_type) for _ in range(2)]
    back = [torch.zeros(count, device="cuda", dtype=out_type) for _ in range(2)]
    ready(engine)
    flags = TE_ATTN_OUTPUT_F16 if out16 else 0
    cache.append(0, layers, 0, kd, vd, n, room[0][32:-32], room[1][32:-32],
                 flags=TE_ATTN_ADVANCE | flags | (TE_ATTN_INPUT_F16 if f16 else 0))
    cache.read(0, layers, 0, first, n, back[0], back[1], flags=flags)
    engine.synchronize()
    for r, b in zip(room, back):
        assert torch.equal(r[32:-32], b)
        assert (r[:32] == 7).all() and (r[-32:] == 7).all()
    cache.close()


@pytest.mark.parametrize("f16", [False, True])
def test_append_takes_columns_of_a_wider_output(engine, f16):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_NO_ROPE
    rng = np.random.default_rng(8)
    n, kvh, hd, h = 21, 2, 64, 6 * 64
    qkv = rows(rng, n, h + 2 * kvh * hd).astype(np.float16 if f16 else np.float32)
    t = dev(qkv)
    cache = engine.kv4_cache(layers=1, max_seqs=2, max_tokens_per_seq=64, kv_heads=kvh, head_dim=hd)
    flags = TE_ATTN_ADVANCE | TE_ATTN_NO_ROPE | (TE_ATTN_INPUT_F16 if f16 else 0)
    ready(engine)
    cache.append(0, 1, 0, t[:, h:h + kvh * hd], t[:, h + kvh * hd:], n, flags=flags)
    a = blocks_of(cache, 1, 0, 0, n)
    k, v = t[:, h:h + kvh * hd].contiguous(), t[:, h + kvh * hd:].contiguous()
    ready(engine)
    cache.append(0, 1, 1, k, v, n, flags=flags)
    b = blocks_of(cache, 1, 1, 0, n)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    assert np.array_equal(a[0][0], quantise(qkv[:, h:h + kvh * hd].astype(np.float32).reshape(n, kvh, hd)))
    with pytest.raises(ValueError):
        cache.append(0, 1, 0, t[:, h:h + kvh * hd], v, n, flags=flags)
    cache.close()


# ---------------------------------------------------------------- reading

@pytest.mark.parametrize("hd,page", [(64, 64), (128, 192)])
def test_read_ranges_and_pages_out_of_order(engine, hd, page):
    from tinymetalagent_b200 import TE_ATTN_OUTPUT_F16
    import torch
    rng = np.random.default_rng(page)
    layers, kvh, n = 2, 3, 2 * page + 17
    cache = engine.kv4_cache(layers=layers, max_seqs=2, max_tokens_per_seq=3 * page, kv_heads=kvh, head_dim=hd,
                             page_tokens=page)
    for t in range(page, 3 * page + 1, page):  # the two sequences take pages in turn
        cache.reserve(0, t)
        cache.reserve(1, t)
    fill(cache, 0, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    k, v = fill(cache, 1, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    for begin, m in [(0, 1), (0, n), (5, 11), (15, 2), (16, 16), (page - 1, 2), (page - 3, page + 9), (n - 1, 1)]:
        for typ, flag in ((torch.float32, 0), (torch.float16, TE_ATTN_OUTPUT_F16)):
            a = torch.full((layers, m, kvh, hd), 7.0, dtype=typ, device="cuda")
            b = torch.full_like(a, 7.0)
            ready(engine)
            cache.read(0, layers, 1, begin, m, a, b, flags=flag)
            engine.synchronize()
            np_typ = np.float16 if flag else np.float32
            assert np.array_equal(a.cpu().numpy(), k[:, begin:begin + m].astype(np.float32).astype(np_typ))
            assert np.array_equal(b.cpu().numpy(), v[:, begin:begin + m].astype(np.float32).astype(np_typ))
    cache.close()


def test_blocks_round_trip_one_layer_at_a_time(engine):
    import torch
    rng = np.random.default_rng(1)
    layers, kvh, hd, n = 3, 2, 128, 45
    kb, vb = quantise(rows(rng, layers, n, kvh, hd)), quantise(rows(rng, layers, n, kvh, hd))
    cache = engine.kv4_cache(layers=layers, max_seqs=1, max_tokens_per_seq=64, kv_heads=kvh, head_dim=hd)
    kd, vd = dev(kb), dev(vb)
    ready(engine)
    for layer in (2, 0, 1):
        cache.write_q4_0(layer, 1, 0, 0, n, kd[layer].contiguous(), vd[layer].contiguous())
        engine.synchronize()
    a, b = blocks_of(cache, layers, 0, 0, n)
    assert np.array_equal(a, kb) and np.array_equal(b, vb)
    one = torch.zeros((1, 7, kvh, hd // 32, 18), dtype=torch.uint8, device="cuda")
    two = torch.zeros_like(one)
    ready(engine)
    cache.read_q4_0(1, 1, 0, 9, 7, one, two)
    engine.synchronize()
    assert np.array_equal(one.cpu().numpy()[0], kb[1, 9:16]) and np.array_equal(two.cpu().numpy()[0], vb[1, 9:16])
    cache.close()


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 64, 65, 127, 129, 777, 3001])
def test_decode_lengths(engine, hd, n):
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(n)
    layers, kvh, heads = 2, 2, 14
    cache = engine.kv4_cache(layers=layers, max_seqs=1, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
    k, v = fill(cache, 0, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    q = rows(rng, layers, 1, heads, hd, gain=2)
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)
    for layer in range(layers):
        check(out[layer, 0], q[layer, 0], k[layer], v[layer])
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 5, 8, 9, 16, 20])
def test_decode_groups_ragged_batch(engine, hd, group):
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(group)
    kvh, lens, layers = 2, [200, 0, 1, 333, 64], 2
    heads = kvh * group
    cache = engine.kv4_cache(layers=layers, max_seqs=6, max_tokens_per_seq=384, kv_heads=kvh, head_dim=hd,
                             page_tokens=64)
    order = [4, 1, 3, 0, 5]
    for t in range(64, 385, 64):
        for s in order:
            cache.reserve(s, t)
    kv = [fill(cache, s, rows(rng, layers, m, kvh, hd), rows(rng, layers, m, kvh, hd)) if m else None
          for s, m in zip(order, lens)]
    q = rows(rng, layers, len(lens), heads, hd)
    out = run_decode(cache, order, q, heads, flags=TE_ATTN_NO_ROPE)
    for layer in range(layers):
        for i, m in enumerate(lens):
            if m == 0:
                assert (out[layer, i] == 0).all()
            else:
                check(out[layer, i], q[layer, i], kv[i][0][layer], kv[i][1][layer])
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,group,f16,bias", [(0, 7, False, False), (1, 8, True, False), (15, 3, False, True),
                                              (16, 12, False, False), (64, 7, True, True), (500, 7, False, True)])
def test_decode_appends_rotates_and_attends_as_stored(port, engine, hd, n, group, f16, bias):
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_INPUT_F16, TE_ATTN_QKV_BIAS
    rng = np.random.default_rng(n + hd)
    layers, kvh, p0 = 2, 2, 40
    heads = kvh * group
    typ = np.float16 if f16 else np.float32
    cache = engine.kv4_cache(layers=layers, max_seqs=2, max_tokens_per_seq=n + 2, kv_heads=kvh, head_dim=hd,
                             page_tokens=64, max_position=p0 + n + 2)
    cache.reset(1, p0)
    if n:
        fill(cache, 1, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    qb, kb, vb = rows(rng, layers, heads * hd), rows(rng, layers, kvh * hd), rows(rng, layers, kvh * hd)
    if bias:
        cache.set_qkv_bias(0, heads, qb, kb, vb)
    flags = TE_ATTN_ADVANCE | (TE_ATTN_INPUT_F16 if f16 else 0) | (TE_ATTN_QKV_BIAS if bias else 0)
    for step in range(2):
        q = rows(rng, layers, 1, heads, hd).astype(typ)
        kn, vn = rows(rng, layers, 1, kvh, hd).astype(typ), rows(rng, layers, 1, kvh, hd).astype(typ)
        out = run_decode(cache, [1], q, heads, k_new=kn, v_new=vn, flags=flags)
        assert cache.length(1) == n + step + 1
        ck, cv = blocks_of(cache, layers, 1, 0, n + step + 1)
        for layer in range(layers):
            qq, kk, vv = (a[layer].astype(np.float32) for a in (q, kn, vn))
            if bias:
                qq = qq + qb[layer].reshape(heads, hd)
                kk, vv = kk + kb[layer].reshape(kvh, hd), vv + vb[layer].reshape(kvh, hd)
            pos = [p0 + n + step]
            assert np.array_equal(ck[layer, -1:], quantise(rotate(port, kk, pos)))
            assert np.array_equal(cv[layer, -1:], quantise(vv))
            check(out[layer, 0], rotate(port, qq, pos)[0], values(ck[layer]), values(cv[layer]))
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["keys_grow", "keys_shrink", "values_grow", "values_shrink", "values_tiny",
                                  "values_huge", "one_token_wins", "queries_tiny", "queries_huge"])
def test_decode_extreme_scales(engine, hd, kind):
    """Scores and values whose size changes along the sequence: the reference exponent, the value scale's
    exponent and the query's power of two all move."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(17)
    n, kvh, heads = 1000, 1, 7
    ramp = np.linspace(0, 1, n)[None, :, None, None]
    k, v, q = rows(rng, 1, n, kvh, hd), rows(rng, 1, n, kvh, hd), rows(rng, 1, 1, heads, hd)
    if kind == "keys_grow":
        k = k * (16.0 ** ramp)
    elif kind == "keys_shrink":
        k = k * (16.0 ** (1 - ramp))
    elif kind == "values_grow":
        v = v * (2.0 ** (30 * ramp - 15))
    elif kind == "values_shrink":
        v = v * (2.0 ** (15 - 30 * ramp))
    elif kind == "values_tiny":
        v = v * 2.0 ** -18
    elif kind == "values_huge":
        v = v * 2.0 ** 15
    elif kind == "one_token_wins":
        k[0, 613] = 4.0 * q[0, 0, 0] / np.abs(q[0, 0, 0]).max()
        q = q * 12
    elif kind == "queries_tiny":
        q, k = q * 1e-30, k * 1e4
    else:
        q, k = q * 1e25, k * 1e-5
        k[:] *= 1e-20  # scales far below binary16: every key reads as zero
    k, v, q = (np.asarray(a, np.float32) for a in (k, v, q))
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
    kk, vv = fill(cache, 0, k, v)
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)
    check(out[0, 0], q[0, 0], kk[0], vv[0])
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("small", [2.0 ** -6, 2.0 ** -12])
@pytest.mark.parametrize("at", [0, 300, 998])
def test_decode_beside_a_token_of_huge_values(engine, hd, small, at):
    """A token whose values are 2^17 and more times the others', and whose weight is nothing for the even heads and
    everything for the odd ones: the even heads' outputs are as exact as without it."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(23)
    n, heads = 1000, 7
    k, v, q = rows(rng, 1, n, 1, hd), rows(rng, 1, n, 1, hd, gain=small), rows(rng, 1, 1, heads, hd)
    k[..., 0] = 0
    k[0, at] = 0
    k[0, at, 0, 0] = -400
    v[0, at] = np.where(rng.random((1, hd)) < 0.5, 1, -1) * 2.0 ** 17
    q[..., 0::2, 0] = 8
    q[..., 1::2, 0] = -8
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=1, head_dim=hd)
    kk, vv = fill(cache, 0, k, v)
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0]
    others = np.arange(n) != at
    check(out[1::2], q[0, 0, 1::2], kk[0], vv[0])
    check(out[0::2], q[0, 0, 0::2], kk[0, others], vv[0, others])
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [3, 16, 130])
def test_decode_ignores_what_lies_past_the_length(engine, hd, n):
    """Blocks past the end of the sequence (here NaN and infinite scales, left by a truncation) have no part."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(n)
    kvh, heads, room = 2, 8, 192
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=room, kv_heads=kvh, head_dim=hd)
    k, v = fill(cache, 0, rows(rng, 1, n, kvh, hd), rows(rng, 1, n, kvh, hd))
    q = rows(rng, 1, 1, heads, hd)
    want = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)
    check(want[0, 0], q[0, 0], k[0], v[0])
    junk = np.full((1, room - n, kvh, hd // 32, 18), 0xFF, np.uint8)  # NaN scales
    junk[..., 0::2, 0], junk[..., 0::2, 1] = 0x00, 0x7C               # infinite scales
    jd = dev(junk)
    ready(engine)
    cache.write_q4_0(0, 1, 0, n, room - n, jd, jd)
    engine.synchronize()
    cache.truncate(0, n)
    assert np.array_equal(run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE), want)
    cache.close()


def test_decode_non_finite_inputs_stay_where_they_belong(engine):
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(4)
    n, kvh, heads, hd = 100, 2, 8, 64
    cache = engine.kv4_cache(layers=1, max_seqs=2, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
    kr, vr = rows(rng, 1, n, kvh, hd), rows(rng, 1, n, kvh, hd)
    k, v = fill(cache, 0, kr, vr)
    q = rows(rng, 1, 1, heads, hd)
    q[0, 0, 5, 7], q[0, 0, 2, 0] = np.nan, np.inf
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0]
    assert np.isnan(out[[2, 5]]).all()
    rest = [0, 1, 3, 4, 6, 7]
    exp, tol = attend(np.nan_to_num(q[0, 0], posinf=0.0).astype(np.float64), k[0], v[0])
    assert (np.abs(out[rest] - exp[rest]) <= tol[rest]).all()
    # a NaN value row of kv head 1: that block of the output of its heads
    vr[0, 50, 1, 33] = np.nan
    k, v = fill(cache, 1, kr, vr)
    q = rows(rng, 1, 1, heads, hd)
    out = run_decode(cache, [1], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0]
    assert np.isnan(out[4:, 32:]).all() and np.isfinite(out[4:, :32]).all() and np.isfinite(out[:4]).all()
    cache.close()


def test_decode_is_reproducible_and_capturable(engine):
    import torch
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE, AttnEngine
    rng = np.random.default_rng(9)
    layers, n, kvh, heads, hd = 3, 2500, 2, 14, 128
    eng = AttnEngine(0, stream=torch.cuda.Stream().cuda_stream)
    cache = eng.kv4_cache(layers=layers, max_seqs=1, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
    k, v = fill(cache, 0, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    q = rows(rng, layers, 1, heads, hd)
    first = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)
    for _ in range(5):
        assert np.array_equal(run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE), first)
    qd, out = dev(q), torch.zeros(q.shape, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.ExternalStream(eng.stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.decode(0, layers, [0], qd, out, heads, flags=TE_ATTN_NO_ROPE)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        eng.synchronize()
        assert np.array_equal(out.cpu().numpy(), first)
    del graph
    cache.close()
    eng.close()


def test_decode_more_sequences_than_one_launch_takes(engine):
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(6)
    S, kvh, heads, hd = 70, 1, 4, 64
    cache = engine.kv4_cache(layers=1, max_seqs=S, max_tokens_per_seq=64, kv_heads=kvh, head_dim=hd)
    lens = [(7 * i) % 64 + 1 for i in range(S)]
    kv = [fill(cache, s, rows(rng, 1, m, kvh, hd), rows(rng, 1, m, kvh, hd)) for s, m in enumerate(lens)]
    q = rows(rng, 1, S, heads, hd)
    out = run_decode(cache, list(range(S)), q, heads, flags=TE_ATTN_NO_ROPE)
    for s in range(S):
        check(out[0, s], q[0, s], kv[s][0][0], kv[s][1][0])
    cache.close()


@pytest.mark.parametrize("hd,group,append", [(64, 3, False), (64, 9, True), (128, 2, True), (128, 8, False)])
def test_decode_more_groups_than_resident_ctas(engine, hd, group, append):
    """More (layer, kv head, sequence) groups than the GPU holds CTAs: ranges that begin and end inside groups, CTAs
    with several groups, empty and one-token sequences between long ones; two launches share the scratch."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(hd + group)
    layers, kvh, S = 3, 8, 14
    lens = [1500, 0, 1, 37, 513, 1030, 0, 64, 700, 255, 256, 257, 1200, 5]
    heads = kvh * group
    cache = engine.kv4_cache(layers=layers, max_seqs=S, max_tokens_per_seq=1504, kv_heads=kvh, head_dim=hd,
                             page_tokens=64)
    kv = [fill(cache, s, rows(rng, layers, m, kvh, hd), rows(rng, layers, m, kvh, hd)) if m else
          (np.zeros((layers, 0, kvh, hd)),) * 2 for s, m in enumerate(lens)]
    kw = {}
    if append:
        kn, vn = rows(rng, layers, S, kvh, hd), rows(rng, layers, S, kvh, hd)
        kw = dict(k_new=kn, v_new=vn)
        kv = [(np.concatenate([k, values(quantise(kn[:, i:i + 1]))], 1),
               np.concatenate([v, values(quantise(vn[:, i:i + 1]))], 1)) for i, (k, v) in enumerate(kv)]
    for _ in range(2):
        q = rows(rng, layers, S, heads, hd)
        out = run_decode(cache, list(range(S)), q, heads, flags=TE_ATTN_NO_ROPE, **dict(kw))
        for layer in range(layers):
            for i in range(S):
                if kv[i][0].shape[1] == 0:
                    assert (out[layer, i] == 0).all()
                else:
                    check(out[layer, i], q[layer, i], kv[i][0][layer], kv[i][1][layer])
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layers,kvh,lens", [
    (9, 8, [60, 0, 1, 33, 17]),            # 360 groups of one unit: every cut falls on or just inside a group
    (5, 8, [300, 2, 0, 40, 700, 9, 64, 1, 255]),
    (1, 1, [12000] + [3] * 63),            # one long sequence before many short ones
    (1, 2, [3] * 40 + [20000] + [0] * 20)])
def test_decode_short_sequences_between_cuts(engine, hd, layers, kvh, lens):
    """Groups that are not worth splitting: a CTA's range begins with a group or has tokens of the one before."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(hd + layers)
    S, group = len(lens), 2
    cache = engine.kv4_cache(layers=layers, max_seqs=S, max_tokens_per_seq=max(lens), kv_heads=kvh, head_dim=hd,
                             page_tokens=64, total_pages=sum(-(-m // 64) for m in lens))
    kv = [fill(cache, s, rows(rng, layers, m, kvh, hd), rows(rng, layers, m, kvh, hd)) if m else None
          for s, m in enumerate(lens)]
    q = rows(rng, layers, S, kvh * group, hd)
    first = run_decode(cache, list(range(S)), q, kvh * group, flags=TE_ATTN_NO_ROPE)
    out = run_decode(cache, list(range(S)), q, kvh * group, flags=TE_ATTN_NO_ROPE)
    assert np.array_equal(first, out)
    for layer in range(layers):
        for i, m in enumerate(lens):
            if m == 0:
                assert (out[layer, i] == 0).all()
            else:
                check(out[layer, i], q[layer, i], kv[i][0][layer], kv[i][1][layer])
    cache.close()


@pytest.mark.parametrize("cut", [0, 37, 64, 299])
def test_partial_records_merge_to_the_whole(port, engine, cut):
    """A sequence split over two caches (the second a shard at a position offset): partial records, merged."""
    import torch
    from tinymetalagent_b200 import TE_ATTN_PARTIAL
    rng = np.random.default_rng(cut)
    n, kvh, heads, hd = 300, 2, 14, 128
    kr, vr = rows(rng, 1, n, kvh, hd), rows(rng, 1, n, kvh, hd)
    q = rows(rng, 1, 1, heads, hd)
    parts = []
    for begin, end in ((0, cut), (cut, n)):
        cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
        cache.reset(0, begin)
        if end > begin:
            fill(cache, 0, kr[:, begin:end], vr[:, begin:end])
        parts.append(run_decode(cache, [0], q, heads, q_positions=[n - 1], flags=TE_ATTN_PARTIAL))
        cache.close()
    if cut == 0:
        assert np.array_equal(parts[0][..., :hd], np.zeros((1, 1, heads, hd))) and (parts[0][..., hd + 1] == 0).all()
        assert np.isneginf(parts[0][..., hd]).all()
    rec, out = dev(np.stack(parts)), torch.zeros((heads, hd), device="cuda")
    ready(engine)
    engine.merge_partials(rec, 2, heads, hd, out)
    engine.synchronize()
    check(out.cpu().numpy(), rotate(port, q[0], [n - 1])[0], values(quantise(kr[0])), values(quantise(vr[0])))


def test_pages_return_and_a_full_pool_leaves_the_cache_usable(engine):
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE, TinyEngineError
    rng = np.random.default_rng(2)
    kvh, heads, hd = 1, 4, 64
    cache = engine.kv4_cache(layers=1, max_seqs=2, max_tokens_per_seq=256, kv_heads=kvh, head_dim=hd, page_tokens=64,
                             total_pages=4)
    fill(cache, 0, rows(rng, 1, 100, kvh, hd), rows(rng, 1, 100, kvh, hd))
    with pytest.raises(TinyEngineError) as e:
        cache.reserve(1, 200)  # four pages wanted, two free
    assert e.value.status == 4
    k, v = fill(cache, 1, rows(rng, 1, 128, kvh, hd), rows(rng, 1, 128, kvh, hd))
    cache.reset(0)
    k2, v2 = fill(cache, 0, rows(rng, 1, 70, kvh, hd), rows(rng, 1, 70, kvh, hd))
    q = rows(rng, 1, 2, heads, hd)
    out = run_decode(cache, [1, 0], q, heads, flags=TE_ATTN_NO_ROPE)
    check(out[0, 0], q[0, 0], k[0], v[0])
    check(out[0, 1], q[0, 1], k2[0], v2[0])
    cache.close()


# ---------------------------------------------------------------- refusals

def test_refusals(engine):
    import torch
    import tinymetalagent_b200 as T
    from tinymetalagent_b200 import runtime as R
    bad = R.TE_STATUS_INVALID_ARGUMENT
    kvh, hd, heads = 2, 64, 4
    cache = engine.kv4_cache(layers=2, max_seqs=2, max_tokens_per_seq=64, kv_heads=kvh, head_dim=hd)
    f = torch.zeros(4096, device="cuda")
    torch.cuda.synchronize()
    a = f.data_ptr()
    lib, h = cache.lib, cache.handle
    u32 = ctypes.c_uint32

    def dec(layer=0, layers=1, ids=(0,), n=None, q=a, k=None, v=None, heads=heads, out=a, flags=0, qp=None):
        arr = (u32 * len(ids))(*ids)
        pos = (ctypes.c_int64 * len(qp))(*qp) if qp else None
        return lib.te_kv4_attention_decode(h, layer, layers, arr, len(ids) if n is None else n, pos, q, k, v, heads,
                                           out, flags)

    assert dec() == 0  # an empty sequence: zeros
    for kw in (dict(q=None), dict(out=None), dict(layers=0), dict(layer=2), dict(layer=1, layers=2**64 - 1),
               dict(ids=(2,)), dict(ids=(0, 0)), dict(n=0), dict(heads=3), dict(heads=0), dict(k=a), dict(v=a),
               dict(q=a + 4), dict(out=a + 8), dict(flags=T.TE_ATTN_HOST_BUFFERS), dict(qp=(64,)), dict(qp=(-1,)),
               dict(flags=T.TE_ATTN_QKV_BIAS), dict(ids=(0, 1, 1))):
        assert dec(**kw) == bad, kw

    def app(layer=0, layers=1, seq=0, k=a, v=a, n=1, stride=0, ks=None, vs=None, flags=0):
        return lib.te_kv4_append(h, layer, layers, seq, k, v, n, stride, ks, vs, flags)

    for kw in (dict(k=None), dict(v=None), dict(n=0), dict(n=65), dict(n=2**64 - 1), dict(seq=2), dict(layers=3),
               dict(layer=2**64 - 1), dict(k=a + 4), dict(ks=a), dict(vs=a), dict(ks=a + 4, vs=a), dict(stride=64),
               dict(stride=129), dict(flags=T.TE_ATTN_PARTIAL), dict(flags=T.TE_ATTN_QKV_BIAS)):
        assert app(**kw) == bad, kw
    assert cache.length(0) == 0

    def rd(begin=0, n=1, k=a, v=a, flags=0, layer=0, layers=1):
        return lib.te_kv4_cache_read(h, layer, layers, 0, begin, n, k, v, flags)

    assert rd() == bad  # nothing cached yet
    assert app(n=4, flags=T.TE_ATTN_ADVANCE) == 0 and rd(n=4) == 0
    for kw in (dict(n=5), dict(begin=4), dict(begin=2**64 - 1, n=2), dict(begin=1, n=2**64 - 1), dict(k=None),
               dict(v=a + 4), dict(flags=1), dict(layers=3), dict(n=0)):
        assert rd(**kw) == bad, kw
    assert lib.te_kv4_cache_write_q4_0(h, 0, 1, 0, 5, 1, a, a) == bad      # past the length
    assert lib.te_kv4_cache_write_q4_0(h, 0, 1, 0, 4, 61, a, a) == bad     # past max_tokens_per_seq
    assert lib.te_kv4_cache_write_q4_0(h, 0, 1, 0, 0, 1, a + 1, a) == bad  # alignment
    assert lib.te_kv4_cache_read_q4_0(h, 0, 1, 0, 4, 1, a, a) == bad
    assert lib.te_kv4_cache_seq_truncate(h, 0, 5) == bad
    assert cache.length(0) == 4
    # the sequence is full: the token does not fit, and nothing changes
    cache.append(0, 1, 0, torch.zeros((1, 60, kvh, hd), device="cuda"), torch.zeros((1, 60, kvh, hd), device="cuda"), 60,
                 flags=T.TE_ATTN_ADVANCE)
    assert dec(k=a, v=a, flags=T.TE_ATTN_ADVANCE) == bad and cache.length(0) == 64
    engine.synchronize()

    # the binding's own checks
    q = torch.zeros((1, 1, heads, hd), device="cuda")
    with pytest.raises(ValueError):
        cache.decode(0, 1, [0], q.half(), q, heads)
    with pytest.raises(ValueError):
        cache.decode(0, 1, [0], q.cpu(), q, heads)
    with pytest.raises(ValueError):
        cache.decode(0, 1, [0], q.transpose(2, 3), q, heads)
    with pytest.raises(ValueError):
        cache.decode(0, 1, [0, 1], q, q, heads)
    with pytest.raises(ValueError):
        cache.read(0, 1, 0, 0, 3, q, q)
    with pytest.raises(ValueError):
        cache.decode(0, 1, [0], q, q, heads, q_positions=[1, 2])
    cache.close()
    for kw in (dict(head_dim=96), dict(page_tokens=32), dict(layers=0), dict(rope_theta=0.0), dict(kv_heads=0)):
        args = dict(layers=1, max_seqs=1, max_tokens_per_seq=64, kv_heads=1, head_dim=64)
        with pytest.raises(T.TinyEngineError):
            engine.kv4_cache(**{**args, **kw})


def test_offsets_past_32_bits(engine):
    """A pool of more than 4 GiB: the last pages of the last layer are the right ones."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(12)
    layers, kvh, hd, room = 24, 8, 128, 196608  # 24 * 8 * 12288 tiles * 2304 B = 5.4 GB
    cache = engine.kv4_cache(layers=layers, max_seqs=2, max_tokens_per_seq=room // 2, kv_heads=kvh, head_dim=hd,
                             page_tokens=128, max_position=256)
    cache.reserve(0, room // 2)
    n = 200
    k, v = fill(cache, 1, rows(rng, layers, n, kvh, hd), rows(rng, layers, n, kvh, hd))
    q = rows(rng, layers, 1, kvh, hd)
    out = run_decode(cache, [1], q, kvh, flags=TE_ATTN_NO_ROPE)
    for layer in (0, layers - 1):
        check(out[layer, 0], q[layer, 0], k[layer], v[layer])
    a, b = blocks_of(cache, layers, 1, 0, n)
    assert np.array_equal(values(a), k) and np.array_equal(values(b), v)
    cache.close()
