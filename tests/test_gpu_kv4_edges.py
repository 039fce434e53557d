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


def one_token_wins(engine, hd, size, rest=0.0):
    """70 tokens whose keys stand for `rest` but for one, whose keys are at the smallest scale there is, under queries
    of about `size`: that token has all of the weight.  Its values come back, off by what two binary16 parts of a
    weight leave (2^-22 of it) and the division (2^-23)."""
    from tinymetalagent_b200 import TE_ATTN_NO_ROPE
    rng = np.random.default_rng(47)
    n, heads, at = 70, 3, 13
    k, v = np.full((1, n, 1, hd), rest, np.float32), rows(rng, 1, n, 1, hd)
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
