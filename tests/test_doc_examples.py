"""The integration examples of the 4-bit cache and of the decoder say what the code takes: the C example compiles
against the installed header, the Python calls bind to the signatures."""
import ast
import inspect
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
DOCS = sorted(p for p in ROOT.glob("*.md") if "te_kv4_cache_create" in p.read_text())


def test_c_example_of_the_4_bit_cache_compiles(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    blocks = [b for p in DOCS for b in re.findall(r"```c\n(.*?)```", p.read_text(), re.S) if "te_kv4_cache_create" in b]
    assert blocks
    for block in blocks:
        src = tmp_path / "example.c"
        src.write_text('#include <stddef.h>\n#include <stdint.h>\n#include "tinyengine_attn.h"\n'
                       "void example(te_attn_engine *eng, size_t L, size_t heads, uint32_t seq, size_t other, size_t n_tokens,\n"
                       "             const float *k, const float *v, const float *q, const float *k_new, const float *v_new,\n"
                       "             float *k_stored, float *v_stored, float *out, uint16_t *k_rows, uint16_t *v_rows,\n"
                       "             unsigned char *k_blocks, unsigned char *v_blocks);\n"
                       "void example(te_attn_engine *eng, size_t L, size_t heads, uint32_t seq, size_t other, size_t n_tokens,\n"
                       "             const float *k, const float *v, const float *q, const float *k_new, const float *v_new,\n"
                       "             float *k_stored, float *v_stored, float *out, uint16_t *k_rows, uint16_t *v_rows,\n"
                       "             unsigned char *k_blocks, unsigned char *v_blocks) {\n" + block + "}\n")
        r = subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", str(ROOT / "include"),
                            str(src)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr


def test_decoder_calls_bind_to_its_signature():
    from tinymetalagent_b200.qwen import QwenDecoder
    sig = inspect.signature(QwenDecoder)
    seen = 0
    for p in DOCS:
        for call in re.findall(r"QwenDecoder\([^()`]*\)", p.read_text()):
            node = ast.parse(call, mode="eval").body
            if any(isinstance(a, ast.Constant) and a.value is ... for a in node.args):
                continue  # "...": the other arguments are as elsewhere
            sig.bind(*node.args, **{k.arg: k.value for k in node.keywords})
            seen += 1
    assert seen > 0
