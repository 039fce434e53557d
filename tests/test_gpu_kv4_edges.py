"""The 4-bit cache where a call meets what other calls left: recorded graphs and scratch that grows, pools that run
out; and the attention's arithmetic at the ends of its inputs' ranges."""
import numpy as np
import pytest

from test_gpu_kv4 import blocks_of, check, dev, fill, quantise, ready, rows, run_decode, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["kv4", "f16"])
def test_recorded_decode_survives_larger_scratch(kind):
    """A recorded decode writes its partial records where the scratch was when it was recorded.  A later, larger call
    of the same engine takes larger scratch: the recorded one's has to stay its own."""
    import torch
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE, AttnEngine
    rng = np.random.default_rng(41)
    n, kvh, heads, hd = 1500, 2, 16, 128
    eng = AttnEngine(0, stream=torch.cuda.Stream().cuda_stream)
    make = eng.kv4_cache if kind == "kv4" else eng.kv_cache
    cache = make(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=kvh, head_dim=hd)
    if kind == "kv4":
        fill(cache, 0, rows(rng, 1, n, kvh, hd), rows(rng, 1, n, kvh, hd))
    else:
        k, v = (dev(rows(rng, n, kvh, hd), torch.float16) for _ in range(2))
        ready(eng)
        cache.write_f16(0, 0, 0, k, v)
    q, out = dev(rows(rng, 1, 1, heads, hd)), torch.zeros((1, 1, heads, hd), device="cuda")
    ready(eng)
    cache.decode(0, 1, [0], q, out, heads, flags=TE_ATTN_NO_ROPE)
    eng.synchronize()
    want = out.cpu().numpy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(eng.stream)):
        cache.decode(0, 1, [0], q, out, heads, flags=TE_ATTN_NO_ROPE)
    # more than 200 CTAs' records: over 1.7 MB, where the first call's scratch is 1 MB
    big = eng.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=80000, kv_heads=kvh, head_dim=hd)
    kb = torch.zeros((1, 80000, kvh, hd // 32, 18), dtype=torch.uint8, device="cuda")
    big_out = torch.full((1, 1, heads, hd), 7.0, device="cuda")
    ready(eng)
    big.write_q4_0(0, 1, 0, 0, 80000, kb, kb)
    big.decode(0, 1, [0], q, big_out, heads, flags=TE_ATTN_NO_ROPE)
    eng.synchronize()
    assert (big_out == 0).all()
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.ExternalStream(eng.stream)):
            graph.replay()
        eng.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
        big.decode(0, 1, [0], q, big_out, heads, flags=TE_ATTN_NO_ROPE)
    eng.synchronize()
    del graph
    big.close()
    cache.close()
    eng.close()


def test_a_batch_that_runs_out_of_pages_takes_none():
    """Two sequences at the end of their pages, one page free: the step is refused, and the page is still free."""
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, TE_ATTN_NO_ROPE, AttnEngine, TinyEngineError
    rng = np.random.default_rng(43)
    kvh, heads, hd = 1, 4, 64
    eng = AttnEngine(0)
    cache = eng.kv4_cache(layers=1, max_seqs=3, max_tokens_per_seq=256, kv_heads=kvh, head_dim=hd, page_tokens=64,
                          total_pages=3)
    kv = [fill(cache, s, rows(rng, 1, 64, kvh, hd), rows(rng, 1, 64, kvh, hd)) for s in range(2)]
    q, kn, vn = rows(rng, 1, 2, heads, hd), rows(rng, 1, 2, kvh, hd), rows(rng, 1, 2, kvh, hd)
    with pytest.raises(TinyEngineError) as e:
        run_decode(cache, [0, 1], q, heads, k_new=kn, v_new=vn, flags=TE_ATTN_ADVANCE | TE_ATTN_NO_ROPE)
    assert e.value.status == 4
    assert cache.length(0) == cache.length(1) == 64
    cache.reserve(2, 64)  # the free page
    cache.reset(2)
    out = run_decode(cache, [1], q[:, 1:], heads, k_new=kn[:, 1:], v_new=vn[:, 1:],
                     flags=TE_ATTN_ADVANCE | TE_ATTN_NO_ROPE)
    k, v = (np.concatenate([old[0], values(quantise(new[0, 1:]))]) for old, new in zip(kv[1], (kn, vn)))
    check(out[0, 0], q[0, 1], k, v)
    cache.close()
    eng.close()


def one_token_wins(engine, hd, size, rest=0.0, gain=1.0):
    """70 tokens whose keys stand for `rest` but for one, whose keys are at the smallest scale there is, under queries
    of about `size`: that token has all of the weight.  Its values come back, off by what two binary16 parts of a
    weight leave (2^-22 of it) and the division (2^-23)."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(47)
    n, heads, at = 70, 3, 13
    k, v = np.full((1, n, 1, hd), rest, np.float32), rows(rng, 1, n, 1, hd, gain=gain)
    k[0, at] = 2.0**-21
    q = (size * (0.5 + 0.5 * rng.random((1, 1, heads, hd)))).astype(np.float32)
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=1, head_dim=hd)
    kk, vv = fill(cache, 0, k, v)
    assert (kk[0, at] == 2.0**-21).all() and (kk[0, at + 1:] == rest).all()
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0].astype(np.float64)
    assert (np.abs(out - vv[0, at, 0]) <= 2.0**-21 * np.abs(vv[0, at, 0])).all(), np.abs(out - vv[0, at, 0]).max()
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0**40, 2.0**50, 2.0**70, 2.0**100])
def test_decode_large_scores(engine, hd, size):
    """Scores so large (2^23 and more) that their own rounding is larger than the exponents of the weights."""
    one_token_wins(engine, hd, size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gain", [2.0**-16, 2.0**-12, 2.0**6, 2.0**15])
@pytest.mark.parametrize("size,rest", [(2.0**50, 0.0), (2.0**100, 0.0), (2.0**114, -(2.0**17))])
def test_decode_large_scores_beside_small_and_large_values(engine, hd, size, rest, gain):
    one_token_wins(engine, hd, size, rest, gain)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0**117, 2.0**127])
def test_decode_queries_up_to_the_end_of_fp32(engine, hd, size):
    one_token_wins(engine, hd, size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0**114, 2.0**127])
def test_decode_scores_below_fp32(engine, hd, size):
    """Scores that overflow to minus infinity beside finite ones have no weight, also where a warp sees no others."""
    one_token_wins(engine, hd, size, rest=-(2.0**17))


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_only_scores_below_fp32(engine, hd):
    """Every score minus infinity: nothing is attended, as over no token."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(53)
    n, heads = 300, 2
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=1, head_dim=hd)
    fill(cache, 0, np.full((1, n, 1, hd), -(2.0**17), np.float32), rows(rng, 1, n, 1, hd))
    out = run_decode(cache, [0], np.full((1, 1, heads, hd), 2.0**120, np.float32), heads, flags=TE_ATTN_NO_ROPE)
    assert (out == 0).all()
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,at", [(40, 0), (128, 0), (128, 127), (1000, 500)])
@pytest.mark.parametrize("sigma", [1.0, 0.1, 0.02, 2.0**-13])
def test_decode_beside_a_token_without_values(engine, hd, n, at, sigma):
    """A token whose values are zero takes nearly all of the weight (as first tokens of trained models do), by 0 to 18
    nats: what is left of the others is as exact as without it.

    The bound counts what they contribute, A = sum(w max|v|) / sum(w), not the largest value.  A score has one term
    here: it is off by its factor's roundings (3 2^-24 of it), the offset's (2^-21 of a weight) and the exponential's
    (2^-22), which count in a weight and in the sum; two-part weights and products leave 2^-21 and 2^-23, and each of
    n / 16 + 8 additions 2^-22."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(59)
    gaps = np.array([0.0, 4, 8, 10, 12, 14, 18])
    heads = len(gaps)
    k, v = np.zeros((1, n, 1, hd), np.float32), rows(rng, 1, n, 1, hd, gain=sigma)
    k[0, at, 0, 0], v[0, at] = np.sqrt(hd), 0
    q = np.zeros((1, 1, heads, hd), np.float32)
    q[0, 0, :, 0] = gaps
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=1, head_dim=hd)
    kk, vv = (a[0, :, 0] for a in fill(cache, 0, k, v))
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0].astype(np.float64)
    for h in range(heads):
        s = kk @ q[0, 0, h].astype(np.float64) / np.sqrt(hd)
        w = np.exp(s)
        ds = 3 * 2.0**-24 * np.abs(s).max() + 2.0**-21 + 2.0**-22
        mass = (w @ np.abs(vv).max(1)) / w.sum()
        tol = mass * (2 * ds + 2.0**-21 + 2.0**-23 + (n / 16 + 8) * 2.0**-22)
        err = np.abs(out[h] - (w @ vv) / w.sum()).max()
        assert err <= tol, (gaps[h], err / mass, tol / mass)
    cache.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 4, 70])
@pytest.mark.parametrize("small", [2.0**-9, 2.0**-13, 2.0**-17])
def test_decode_blocks_of_small_values_beside_ordinary_ones(engine, hd, n, small):
    """Blocks of 32 values far below the row's others (scales of small / 4 or so, down to binary16 subnormals): their
    outputs are exact against their own values.  All tokens have the same score, so that a weight's error cancels; it
    is above 2^13, and beside it a product's two parts are off by 2^-24 (on the grid of binary16's subnormals) next to
    the terms of the bound above."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(61)
    heads = 7
    k, v, q = np.zeros((1, n, 1, hd), np.float32), rows(rng, 1, n, 1, hd), np.zeros((1, 1, heads, hd), np.float32)
    k[..., 0] = 1
    q[0, 0, :, 0] = np.linspace(0.3, 2.9, heads)
    v[..., 32:] *= small
    cache = engine.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=n, kv_heads=1, head_dim=hd)
    fill(cache, 0, k, v)
    raw = quantise(v)[0, :, 0]
    vv, d = values(raw), np.abs(np.ascontiguousarray(raw[..., :2]).view(np.float16)[..., 0].astype(np.float64))
    out = run_decode(cache, [0], q, heads, flags=TE_ATTN_NO_ROPE)[0, 0].astype(np.float64)
    for b in range(hd // 32):
        cols = slice(32 * b, 32 * b + 32)
        mass = np.abs(vv[:, cols]).max(1).mean()
        tol = mass * (2.0**-21 + 2.0**-23 + (n / 16 + 8) * 2.0**-22 + 2.0**-24 / (2.0**13 * d[:, b].mean()))
        err = np.abs(out[:, cols] - vv[:, cols].mean(0)).max()
        assert err <= tol, (b, err / mass, tol / mass)
    cache.close()


def test_profile_line_of_an_engine_without_a_4_bit_cache():
    """The line has the eight kinds that it had before there was a 4-bit cache; its kinds join as they run."""
    import torch
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, AttnEngine
    eng = AttnEngine(0)
    eng.profile(True)

    def kinds():
        return [f.split("=")[0] for f in eng.profile_report().split(": ", 1)[1].split()][1:]

    old = ["decode", "append", "merge", "prefill_prep", "prefill_attn", "matvec", "exchange", "step"]
    assert kinds() == old
    cache = eng.kv4_cache(layers=1, max_seqs=1, max_tokens_per_seq=64, kv_heads=1, head_dim=64)
    x = torch.zeros((1, 2, 1, 64), device="cuda")
    torch.cuda.synchronize()
    cache.append(0, 1, 0, x, x, 2, flags=TE_ATTN_ADVANCE)
    assert kinds() == old + ["kv4_append"]
    cache.read(0, 1, 0, 0, 2, x, x)
    assert kinds() == old + ["kv4_append", "kv4_read"]
    cache.close()
    eng.close()


def test_a_refused_allocation_does_not_fail_later_calls():
    """A cache larger than the GPU is refused; the launches after it, of either cache, report their own outcome."""
    import torch
    from tinymetalagent_b200 import TE_ATTN_ADVANCE, AttnEngine, TinyEngineError
    rng = np.random.default_rng(67)
    eng = AttnEngine(0)
    small = dict(layers=1, max_seqs=1, max_tokens_per_seq=64, kv_heads=1, head_dim=64)
    caches = eng.kv4_cache(**small), eng.kv_cache(**small)
    x, kb = dev(rows(rng, 1, 3, 1, 64)), dev(quantise(rows(rng, 1, 3, 1, 64)))
    for call in (lambda: caches[0].write_q4_0(0, 1, 0, 0, 3, kb, kb),
                 lambda: caches[1].append_rope(0, 1, 0, x, x, 3, TE_ATTN_ADVANCE),
                 lambda: caches[0].append(0, 1, 0, x, x, 3, flags=TE_ATTN_ADVANCE)):
        ready(eng)
        with pytest.raises(TinyEngineError) as e:  # 600 GB
            eng.kv4_cache(layers=64, max_seqs=1, max_tokens_per_seq=1 << 20, kv_heads=64, head_dim=128, max_position=64)
        assert e.value.status == 4
        call()
    eng.synchronize()
    assert caches[0].length(0) == 6 and caches[1].length(0) == 3
    torch.cuda.synchronize()
    eng.close()
