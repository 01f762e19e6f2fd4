"""CPU-side checks of the language-model operators' boundary (no kernel runs):
the header's symbols are exactly what liboperatorlib_lm.so exports, the headers
compile on their own, every refusal of lm_c.h happens before any HIP call, the
predicates hold at their boundaries under ASan + UBSan, and the torch schema is
the documented one."""

from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest

import operatorlib

REPO = Path(__file__).resolve().parents[1]
INCLUDE = REPO / "include"
CSRC = REPO / "orin-cuda-operator-library_amd" / "csrc"
HEADER = INCLUDE / "operatorlib" / "lm_c.h"
CPP_HEADER = INCLUDE / "operatorlib" / "lm_operators.h"
INVALID = operatorlib.HIP_ERROR_INVALID_VALUE
FAKE = 0x100000  # 16- and 256-byte aligned; never dereferenced
SIZE = {"f16": 2, "f32": 4}


@pytest.fixture(scope="module")
def lib():
    return operatorlib.lm_clib()


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return re.findall(r"\b(operatorlib_\w+)\s*\(", text)


def test_symbols(lib):
    assert sorted(declared()) == sorted(operatorlib.LM_C_SYMBOLS)
    nm = shutil.which("nm")
    if nm:
        out = subprocess.run([nm, "-D", "--defined-only", str(operatorlib.LM_LIBRARY_PATH)],
                             capture_output=True, text=True, check=True).stdout
        exported = {x.split()[-1] for x in out.splitlines() if x.split()[-1].startswith("operatorlib_")}
        assert exported == set(declared())
    assert lib.operatorlib_lm_abi_version() == 1


def test_headers_stand_alone(tmp_path):
    src = tmp_path / "abi.c"
    src.write_text("#include <operatorlib/lm_c.h>\n"
                   "int main(void) { operatorlib_strides_t s = {0, 0, 0}; return (int)s.batch; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", str(INCLUDE), "-c",
                    str(src), "-o", str(tmp_path / "abi.o")], check=True)


def test_cpp_api_covers_the_c_abi():
    names = re.findall(r"inline\s+hipError_t\s+(\w+)\s*\(", CPP_HEADER.read_text())
    launchers = [n for n in declared() if n[-4:] in ("_f16", "_f32")]
    assert sorted("operatorlib_" + n for n in names) == sorted(launchers)


class Call:
    """Arguments of a good call by name; `call(x=...)` changes some."""

    def __init__(self, fn, args):
        self.fn, self.args = fn, args

    def __call__(self, **kw):
        assert set(kw) <= set(self.args), kw
        return self.fn(*{**self.args, **kw}.values())


def rope(lib, t):
    return Call(getattr(lib, f"operatorlib_rope_append_{t}"), dict(
        q=FAKE, qs=512, k=FAKE, ks=256, v=FAKE, vs=256, positions=FAKE, rows=1, axes=None,
        frequencies=FAKE, slots=FAKE, q_out=FAKE, k_out=None, key_cache=FAKE, value_cache=2 * FAKE,
        tokens=3, q_heads=4, kv_heads=2, head_dim=128, rotary_dim=128, interleaved=0, pages=5,
        page_size=16, stream=None))


ROPE_BAD = [dict([(n, None)]) for n in ("q", "k", "v", "positions", "frequencies", "slots", "q_out",
                                        "key_cache", "value_cache")]
ROPE_BAD += [{n: x} for n in ("tokens", "q_heads", "kv_heads", "head_dim", "pages", "page_size") for x in (0, -1)]
ROPE_BAD += [dict(rows=0), dict(rotary_dim=-2), dict(rotary_dim=127), dict(rotary_dim=130), dict(qs=511),
             dict(ks=255), dict(vs=255), dict(value_cache=FAKE), dict(value_cache=FAKE + 16 * 2 * 128),
             dict(value_cache=FAKE - 16), dict(tokens=2 ** 24 - 7), dict(pages=2 ** 27),
             dict(q_heads=2 ** 31 - 2 ** 20 - 4, head_dim=1, rotary_dim=0, qs=2 ** 31),
             dict(pages=2 ** 31 - 1, page_size=2 ** 31 - 1), dict(q_heads=2 ** 24, qs=2 ** 31),
             dict(q_heads=2 ** 31 - 1, kv_heads=2 ** 31 - 1, qs=2 ** 60, ks=2 ** 60, vs=2 ** 60),
             dict(tokens=2 ** 31 - 1, q_heads=2 ** 31 - 1, qs=2 ** 40)]


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("bad", ROPE_BAD, ids=str)
def test_rope_append_rejects(lib, t, bad):
    assert rope(lib, t)(**bad) == INVALID


def paged(lib, t, ws=False):
    args = dict(q=FAKE, q_stride=512, key_cache=FAKE, value_cache=FAKE, page_table=FAKE, table_stride=9,
                lengths=FAKE, slopes=None, output=FAKE, batch=3, q_heads=4, kv_heads=2, head_dim=128,
                pages=30, page_size=16, max_pages=9, scale=0.1, window=0, softcap=0.0)
    if ws:
        args |= dict(workspace=FAKE, workspace_bytes=1 << 40)
    args |= dict(stream=None)
    return Call(getattr(lib, f"operatorlib_paged_attention_{t}{'_ws' if ws else ''}"), args)


RULES_BAD = [dict(scale=x) for x in (0.0, -1.0, math.inf, math.nan, 2.0 ** -101, 2.0 ** 101)]
RULES_BAD += [dict(softcap=x) for x in (-1.0, math.inf, math.nan, 2.0 ** -101, 2.0 ** 101)] + [dict(window=-1)]
RULES_BAD += [dict(scale=2.0 ** 60, softcap=2.0 ** -60), dict(scale=2.0 ** -60, softcap=2.0 ** 60)]
PAGED_BAD = [{n: None} for n in ("q", "key_cache", "value_cache", "page_table", "lengths", "output")]
PAGED_BAD += [{n: x} for n in ("batch", "q_heads", "kv_heads", "head_dim", "pages", "page_size", "max_pages")
              for x in (0, -1)]
PAGED_BAD += [{n: FAKE + 8} for n in ("q", "key_cache", "value_cache", "output")] + RULES_BAD
PAGED_BAD += [dict(kv_heads=3), dict(head_dim=136, q_stride=1024), dict(head_dim=126), dict(q_stride=511),
              dict(q_stride=514), dict(table_stride=8), dict(pages=2 ** 31 - 1),
              dict(pages=2 ** 31 - 1, page_size=2 ** 31 - 1),
              dict(max_pages=2 ** 28, table_stride=2 ** 28),
              dict(batch=2 ** 20, max_pages=2 ** 16, table_stride=2 ** 16),
              dict(batch=2 ** 30, q_heads=4)]


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("bad", PAGED_BAD, ids=str)
def test_paged_attention_rejects(lib, t, ws, bad):
    assert paged(lib, t, ws)(**bad) == INVALID


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_paged_attention_workspace(lib, t):
    size = getattr(lib, f"operatorlib_paged_attention_{t}_workspace_size")
    need = size(3, 4, 2, 128, 16, 9)
    assert need > 0
    call = paged(lib, t, True)
    for bad in (dict(workspace_bytes=need - 1), dict(workspace=None), dict(workspace=FAKE + 16)):
        assert call(**bad) == INVALID
    assert size(3, 4, 2, 128, 16, 1) == 0               # one step covers every key
    assert size(0, 4, 2, 128, 16, 9) == 0 and size(3, 4, 3, 128, 16, 9) == 0  # refused sizes
    # bounded whatever the batch: two partial results per workgroup, and 8 bytes a row
    assert size(64, 32, 8, 128, 16, 8192) <= 512 * 2 * 32 * 132 * 4 + 64 * 8 * 8


def masked(lib, t):
    s = operatorlib.Strides
    args = dict(q=FAKE, qs=s(4 * 80 * 64, 80 * 64, 64), k=FAKE, ks=s(2 * 80 * 64, 80 * 64, 64), v=FAKE,
                vs=s(2 * 80 * 64, 80 * 64, 64), slopes=None, documents=None, prefixes=None, output=FAKE,
                os=s(4 * 80 * 64, 80 * 64, 64), batch=2, q_heads=4, kv_heads=2, sequence=80, head_dim=64,
                scale=0.1, causal=1, window=0, softcap=0.0, stream=None)
    return Call(getattr(lib, f"operatorlib_masked_attention_{t}"), args)


MASKED_BAD = [{n: None} for n in ("q", "k", "v", "output")] + [{n: FAKE + 8} for n in ("q", "k", "v", "output")]
MASKED_BAD += [{n: x} for n in ("batch", "q_heads", "kv_heads", "sequence", "head_dim") for x in (0, -1)] + RULES_BAD
MASKED_BAD += [dict(kv_heads=3), dict(head_dim=136), dict(head_dim=62), dict(sequence=2 ** 20 + 1),
               dict(batch=2 ** 30), dict(batch=2 ** 20, q_heads=2 ** 10)]
MASKED_BAD += [{n: operatorlib.Strides(*x)} for n in ("qs", "ks", "vs", "os")
               for x in ((0, 0, 63), (0, 0, 56), (-64, 0, 64), (0, -64, 64), (0, 0, -64), (2, 0, 64), (0, 2, 64),
                         (0, 0, 66), (0, 0, 2 ** 24), (0, 0, 2 ** 62))]


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("bad", MASKED_BAD, ids=lambda b: next(iter(b)))
def test_masked_attention_rejects(lib, t, bad):
    assert masked(lib, t)(**bad) == INVALID


def test_masked_attention_one_token_with_a_wide_stride(lib):
    """A tile of 64 rows is addressed even of one token: its stride is bounded too."""
    s = operatorlib.Strides(0, 0, 2 ** 25)
    assert masked(lib, "f16")(sequence=1, ks=s) == INVALID


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_predicates_under_asan_ubsan(tmp_path):
    exe = tmp_path / "lm_validate_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", f"-I{CSRC}",
                    str(REPO / "tests" / "host" / "lm_validate_check.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, text=True, timeout=300)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert proc.returncode == 0 and "failures=0" in proc.stdout, proc.stdout + proc.stderr


SCHEMA = [
    "rope_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor frequencies, Tensor slots, "
    "Tensor(a!) key_cache, Tensor(b!) value_cache, *, Tensor? axes=None, bool interleaved=False, "
    "bool return_keys=False) -> (Tensor, Tensor)",
    "paged_attention(Tensor q, Tensor key_cache, Tensor value_cache, Tensor page_table, Tensor lengths, *, "
    "float? scale=None, int window=0, float softcap=0.0, Tensor? slopes=None) -> Tensor",
    "masked_attention(Tensor q, Tensor k, Tensor v, *, bool causal=False, int window=0, float softcap=0.0, "
    "Tensor? slopes=None, Tensor? documents=None, Tensor? prefixes=None, float? scale=None) -> Tensor",
]


@pytest.mark.parametrize("text", SCHEMA, ids=lambda s: s.split("(")[0])
def test_torch_schema(text):
    import torch
    operatorlib.load_operatorlib()
    got = getattr(torch.ops.operatorlib, text.split("(")[0]).default._schema
    assert got == torch._C.parse_schema("operatorlib::" + text)
    with pytest.raises((NotImplementedError, RuntimeError)):  # no CPU kernel
        t = torch.ones(1, 1, 1, 8)
        torch.ops.operatorlib.masked_attention(t, t, t)
