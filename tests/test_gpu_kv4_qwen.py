"""The qwen2 decoder over the 4-bit cache (QwenDecoder(kv_bits=4)) against a plain fp64 forward pass of the same
synthetic model that stores what the cache stores: Q4_0 blocks of the rotated keys and the values; a prompt's own rows
in binary16 while it is attended.

The bar is the layer-step tests': |h - ref| <= 2e-2 + 2e-2 |ref| for hidden states, 5e-2 + 2e-2 |ref| for logits.  A
key or value that lies at a rounding boundary may take the neighbouring code in one of the two passes; one code of
one value moves a hidden state by far less than the bar.
"""
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent))
sys.path.insert(0, str(Path(__file__).resolve().parent / "golden"))
from gguf_synth import GGML_Q4_0, GGML_Q8_0, write_qwen2  # noqa: E402
from test_gpu_kv4 import quantise, rotate, values  # noqa: E402

MODELS = {
    "hd64": dict(layers=2, hidden=256, heads=4, kv_heads=2, ffn=512, vocab=512, quant_attn=GGML_Q8_0,
                 quant_ffn=GGML_Q4_0, seed=11),
    "hd128": dict(layers=3, hidden=512, heads=4, kv_heads=1, ffn=1024, vocab=640, quant_attn=GGML_Q4_0,
                  quant_ffn=GGML_Q8_0, seed=12),
    "group7": dict(layers=2, hidden=448, heads=7, kv_heads=1, ffn=640, vocab=384, quant_attn=GGML_Q8_0,
                   quant_ffn=GGML_Q4_0, seed=13, tied=True),
}


class Plain:
    """The forward pass in fp64, token rows [T, hidden]."""

    def __init__(self, path, port):
        from tinymetalagent_b200.gguf import GGUFFile
        self.f, self.port = GGUFFile(path), port
        self.d = self.f.qwen2_dims()
        d = self.d
        self.k = [np.zeros((0, d["kv_heads"], d["head_dim"])) for _ in range(d["layers"])]
        self.v = [a.copy() for a in self.k]

    def w(self, name):
        t = self.f.tensors[name]
        raw = np.array(t.data)
        if t.ggml_type == 0:
            return raw.view(np.float32).astype(np.float64)
        width = 18 if t.ggml_type == GGML_Q4_0 else 34
        b = raw.reshape(t.rows, t.cols // 32, width)
        if t.ggml_type == GGML_Q4_0:
            return values(b)
        scale = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
        return (b[..., 2:].view(np.int8).astype(np.float64) * scale).reshape(t.rows, t.cols)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.d["eps"]) * w

    def run(self, tokens, prompt):
        """Hidden states after `tokens`; prompt: attended in binary16, else (one token) as stored."""
        d = self.d
        H, heads, kvh, hd = d["hidden"], d["heads"], d["kv_heads"], d["head_dim"]
        x = self.w("token_embd.weight")[tokens]
        for layer in range(d["layers"]):
            p = f"blk.{layer}."
            n = len(self.k[layer])
            a = self.norm(x, self.w(p + "attn_norm.weight"))
            q, k, v = ((a @ self.w(p + f"attn_{s}.weight").T + self.w(p + f"attn_{s}.bias")).astype(np.float32)
                       for s in "qkv")
            pos = range(n, n + len(tokens))
            q = rotate(self.port, q.reshape(-1, heads, hd), pos, d["rope_base"]).astype(np.float64)
            k = rotate(self.port, k.reshape(-1, kvh, hd), pos, d["rope_base"])
            v = v.reshape(-1, kvh, hd)
            ks, vs = values(quantise(k)), values(quantise(v))
            if prompt:
                half = lambda z: z.astype(np.float16).astype(np.float64)  # noqa: E731
                ka, va = np.concatenate([half(self.k[layer]), half(k)]), np.concatenate([half(self.v[layer]), half(v)])
            else:
                ka, va = np.concatenate([self.k[layer], ks]), np.concatenate([self.v[layer], vs])
            o = np.zeros((len(tokens), heads, hd))
            for t in range(len(tokens)):
                for h in range(heads):
                    kk, vv = ka[:n + t + 1, h // (heads // kvh)], va[:n + t + 1, h // (heads // kvh)]
                    s = kk @ q[t, h] / np.sqrt(hd)
                    e = np.exp(s - s.max())
                    o[t, h] = e @ vv / e.sum()
            self.k[layer] = np.concatenate([self.k[layer], ks])
            self.v[layer] = np.concatenate([self.v[layer], vs])
            x = x + o.reshape(-1, H) @ self.w(p + "attn_output.weight").T
            a = self.norm(x, self.w(p + "ffn_norm.weight"))
            g, u = a @ self.w(p + "ffn_gate.weight").T, a @ self.w(p + "ffn_up.weight").T
            x = x + (g / (1 + np.exp(-g)) * u) @ self.w(p + "ffn_down.weight").T
        self.x = x[-1]
        return self.x

    def logits(self):
        head = "output.weight" if "output.weight" in self.f.tensors else "token_embd.weight"
        return self.norm(self.x, self.w("output_norm.weight")) @ self.w(head).T


def close(got, ref, atol, rtol, what):
    err = np.abs(got - ref) - (atol + rtol * np.abs(ref))
    assert err.max() <= 0, f"{what}: max excess {err.max():.3e}, max abs diff {np.abs(got - ref).max():.3e}"


@pytest.mark.parametrize("name", list(MODELS))
def test_prompts_and_steps_over_the_4_bit_cache(tmp_path, port, engine, name):
    from tinymetalagent_b200.qwen import QwenDecoder
    path = tmp_path / "m.gguf"
    write_qwen2(path, **MODELS[name])
    ref = Plain(path, port)
    dec = QwenDecoder(engine, path, 64, kv_bits=4)
    assert not dec.fused_step and dec.kv_bits == 4
    rng = np.random.default_rng(7)
    toks = rng.integers(0, MODELS[name]["vocab"], 40).tolist()

    def both(n, got):
        close(dec.x.cpu().numpy() if got is None else got.cpu().numpy(), ref.x, 2e-2, 2e-2, f"{name} after {n}")
        nxt = dec.project_next()
        lref = ref.logits()
        close(dec.logits.cpu().numpy(), lref, 5e-2, 2e-2, f"{name} logits after {n}")
        top = np.sort(lref)[-2:]
        assert top[1] - top[0] < 0.1 or nxt == int(np.argmax(lref))

    dec.prefill_prompt(toks[:21])          # a first prompt
    ref.run(toks[:21], True)
    both(21, None)
    for i in range(21, 25):                # single tokens
        got = dec.forward_token(toks[i], i)
        ref.run([toks[i]], False)
        both(i + 1, got)
    dec.prefill_prompt(toks[25:34], 25)    # a later prompt over the stored history
    ref.run(toks[25:34], True)
    both(34, None)
    got = dec.forward_token(toks[34], 34)
    ref.run([toks[34]], False)
    both(35, got)
    assert dec.cache.length(0) == 35
    dec.close()


def test_recorded_greedy_steps_over_the_4_bit_cache(tmp_path, engine):
    import torch
    from tinymetalagent_b200 import AttnEngine
    from tinymetalagent_b200.qwen import QwenDecoder
    path = tmp_path / "m.gguf"
    write_qwen2(path, **MODELS["hd64"])
    prompt, steps = [3, 99, 250, 7, 42], 12
    eng = AttnEngine(0)
    out = []
    for recorded in (False, True):
        dec = QwenDecoder(eng, path, 64, kv_bits=4)
        dec.prefill_prompt(prompt)
        tok = dec.project_next()
        if recorded:
            dec.capture_greedy(len(prompt), steps)
            seq = dec.replay_greedy(tok)
            torch.cuda.synchronize()
            out.append(seq.cpu().tolist())
        else:
            seq = [tok]
            for i in range(steps):
                dec.forward_token(seq[-1], len(prompt) + i)
                seq.append(dec.project_next())
            out.append(seq)
        dec.close()
    eng.close()
    assert out[0] == out[1]


def test_kv_bits_is_checked(engine):
    from tinymetalagent_b200.qwen import QwenDecoder
    with pytest.raises(ValueError):
        QwenDecoder(engine, "nowhere.gguf", 8, kv_bits=8)
