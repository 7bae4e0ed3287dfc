"""Argument checks of the paged cache: every call here is refused on the host
(or has nothing to do), so no GPU is needed."""
import ctypes
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from attnprofile_b200 import cache  # noqa: E402

P = 4096  # an address that is aligned and never read
R = 8192  # another


def call(engine, name, pack, good, **change):
    assert set(change) <= set(good)
    a = {**good, **change}
    return getattr(engine.lib(), name)(pack(*[0 if v is None else v for v in a.values()]), None)


TABLES = dict(lens=P, new_lens=P, tables=P, free=P, free_count=P, kv_lens=P, starts=P, slots=P,
              free_left=P, status=P, table_stride=8, batch=4, width=8, num_blocks=64,
              block_size=16, tokens=9)


@pytest.mark.parametrize("change,code", [
    ({"block_size": 8}, "UNSUPPORTED"), ({"block_size": 48}, "UNSUPPORTED"),
    ({"batch": 16385}, "UNSUPPORTED"), ({"batch": -1}, "INVALID_ARG"),
    ({"width": -1}, "INVALID_ARG"), ({"table_stride": 7}, "INVALID_ARG"),
    ({"num_blocks": 0}, "INVALID_ARG"), ({"num_blocks": 2 ** 27}, "INVALID_ARG"),
    ({"tokens": -1}, "INVALID_ARG"), ({"slots": P + 1}, "MISALIGNED"),
    *[({k: None}, "INVALID_ARG") for k in ("lens", "new_lens", "tables", "free", "free_count",
                                           "kv_lens", "starts", "slots", "free_left", "status")],
])
def test_block_tables_refusals(engine, change, code):
    assert call(engine, "attn_block_tables", cache._TABLES, TABLES, **change) == engine.ERR[code]


TRIM = dict(lens=P, keep=P, tables=P, free=P, free_count=P, lens_left=P, free_left=P, status=P,
            table_stride=8, batch=4, width=8, num_blocks=64, block_size=16)


@pytest.mark.parametrize("change,code", [
    ({"block_size": 24}, "UNSUPPORTED"), ({"batch": 16385}, "UNSUPPORTED"),
    ({"batch": -2}, "INVALID_ARG"), ({"table_stride": 3}, "INVALID_ARG"),
    ({"num_blocks": -1}, "INVALID_ARG"), ({"keep": P + 3}, "MISALIGNED"),
    *[({k: None}, "INVALID_ARG") for k in ("lens", "keep", "tables", "free", "free_count",
                                           "lens_left", "free_left", "status")],
])
def test_block_trim_refusals(engine, change, code):
    assert call(engine, "attn_block_trim", cache._TRIM, TRIM, **change) == engine.ERR[code]


APPEND = dict(k=P, v=P, slots=P, k_codes=P, v_codes=P, k_scale=P, v_scale=P, k_token=256,
              k_head=128, v_token=256, v_head=128, tokens=5, kv_heads=2, D=128, dtype=0, code=0,
              num_blocks=64, block_size=16)


@pytest.mark.parametrize("change,code", [
    ({"D": 96}, "UNSUPPORTED"), ({"dtype": 2}, "UNSUPPORTED"), ({"code": 2}, "UNSUPPORTED"),
    ({"block_size": 256}, "UNSUPPORTED"), ({"tokens": -1}, "INVALID_ARG"),
    ({"kv_heads": 0}, "INVALID_ARG"), ({"kv_heads": 65536}, "INVALID_ARG"),
    ({"num_blocks": 2 ** 27}, "INVALID_ARG"), ({"k": P + 8}, "MISALIGNED"),
    ({"v": P + 2}, "MISALIGNED"), ({"slots": P + 2}, "MISALIGNED"), ({"k_codes": P + 8}, "MISALIGNED"),
    ({"k_token": 260}, "MISALIGNED"), ({"v_head": 4}, "MISALIGNED"),
    *[({k: None}, "INVALID_ARG") for k in ("k", "v", "slots", "k_codes", "v_codes", "k_scale",
                                           "v_scale")],
])
def test_cache_append_refusals(engine, change, code):
    assert call(engine, "attn_cache_append", cache._APPEND, APPEND, **change) == engine.ERR[code]


def test_cache_append_of_nothing(engine):
    assert call(engine, "attn_cache_append", cache._APPEND, APPEND, tokens=0, k=None) == 0


ATTN = dict(q=P, out=R, k_codes=P, v_codes=P, k_scale=P, v_scale=P, tables=P, kv_lens=P, starts=P,
            workspace=P, workspace_bytes=1 << 30, q_token=512, q_head=128, o_token=512, o_head=128,
            table_stride=8, tokens=3, heads=4, kv_heads=2, D=128, dtype=1, code=1, num_blocks=64,
            block_size=32, width=8, batch=3, max_new=1, causal=1, scale=0.0)


@pytest.mark.parametrize("change,code", [
    ({"D": 256}, "UNSUPPORTED"), ({"dtype": -1}, "UNSUPPORTED"), ({"code": 7}, "UNSUPPORTED"),
    ({"block_size": 0}, "UNSUPPORTED"), ({"heads": 5}, "INVALID_ARG"),
    ({"heads": 0}, "INVALID_ARG"), ({"kv_heads": -2}, "INVALID_ARG"),
    ({"tokens": -1}, "INVALID_ARG"), ({"batch": -1}, "INVALID_ARG"),
    ({"max_new": -1}, "INVALID_ARG"), ({"max_new": 2 ** 31 - 1}, "INVALID_ARG"),
    ({"table_stride": 7}, "INVALID_ARG"), ({"scale": -1.0}, "INVALID_ARG"),
    ({"scale": float("nan")}, "INVALID_ARG"), ({"scale": float("inf")}, "INVALID_ARG"),
    ({"out": P}, "INVALID_ARG"), ({"o_token": 0}, "INVALID_ARG"), ({"o_head": 0}, "INVALID_ARG"),
    ({"starts": P + 2}, "MISALIGNED"), ({"v_scale": P + 1}, "MISALIGNED"),
    ({"q": P + 8}, "MISALIGNED"), ({"out": P + 2}, "MISALIGNED"), ({"q_token": 516}, "MISALIGNED"),
    ({"o_head": 132}, "MISALIGNED"), ({"workspace": P + 4}, "MISALIGNED"),
    *[({k: None}, "INVALID_ARG") for k in ("q", "out", "k_codes", "v_codes", "k_scale", "v_scale",
                                           "tables", "kv_lens", "starts")],
])
def test_attn_cached_refusals(engine, change, code):
    assert call(engine, "attn_cached", cache._CACHED, ATTN, **change) == engine.ERR[code]


@pytest.mark.parametrize("change", [{"tokens": 0}, {"batch": 0}, {"max_new": 0}])
def test_attn_cached_of_nothing(engine, change):
    assert call(engine, "attn_cached", cache._CACHED, ATTN, q=None, **change) == 0


@pytest.mark.parametrize("args,code", [
    ((4, 3, 64, 1, 16, 9), "INVALID_ARG"), ((4, 0, 64, 1, 16, 9), "INVALID_ARG"),
    ((4, 2, 80, 1, 16, 9), "UNSUPPORTED"), ((4, 2, 64, -1, 16, 9), "INVALID_ARG"),
    ((4, 2, 64, 1, 24, 9), "UNSUPPORTED"), ((4, 2, 64, 1, 16, -1), "INVALID_ARG"),
])
def test_workspace_refusals(engine, args, code):
    out = ctypes.c_ulonglong()
    assert engine.lib().attn_cached_workspace(*args, ctypes.byref(out)) == engine.ERR[code]
    assert engine.lib().attn_cached_workspace(4, 2, 64, 1, 16, 9, None) == engine.ERR["INVALID_ARG"]


def test_short_requests_need_no_workspace(engine):
    out = ctypes.c_ulonglong(7)
    assert engine.lib().attn_cached_workspace(4, 2, 64, 1, 16, 32, ctypes.byref(out)) == 0
    assert out.value == 0


def test_no_arguments_at_all(engine):
    for name in ("attn_block_tables", "attn_block_trim", "attn_cache_append", "attn_cached"):
        assert getattr(engine.lib(), name)(None, None) == engine.ERR["INVALID_ARG"]


def test_python_face_refuses_cpu_tensors_and_shapes(engine):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.ones(4, 2)
    with pytest.raises(ValueError, match="CUDA"):
        engine.PagedCache(k, k, s, s)
    with pytest.raises(TypeError):
        engine.PagedCache(k.half(), k.half(), s, s)
    with pytest.raises(ValueError):
        engine.PagedCache(k[:, :, :8], k[:, :, :8], s, s)
    with pytest.raises(ValueError):
        engine.PagedCache(k, k[:2], s, s)
    with pytest.raises(ValueError, match="CUDA"):
        engine.BlockPool(torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 16)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_argument_structs_are_as_long_as_the_header_s(tmp_path):
    """The C side may copy a struct whole, its padding too."""
    packs = {"attn_block_tables_args": (cache._TABLES, TABLES),
             "attn_block_trim_args": (cache._TRIM, TRIM),
             "attn_cache_append_args": (cache._APPEND, APPEND),
             "attn_cached_args": (cache._CACHED, ATTN)}
    source, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text('#include <stdio.h>\n#include "attnprof.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu\\n", sizeof({name}));\n' for name in packs) + "  return 0;\n}\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-std=c99", "-I", str(include), str(source), "-o", str(exe)], check=True)
    sizes = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    for size, (name, (pack, good)) in zip(sizes, packs.items()):
        assert len(pack(*good.values())) == int(size), name


@pytest.mark.parametrize("torch_there", [True, False])
def test_names_that_a_star_import_brings(torch_there):
    """Without torch the dense engine's names come, with it the cache's too."""
    root = Path(__file__).resolve().parent.parent
    code = ("import sys\n" + ("" if torch_there else "sys.modules['torch'] = None\n") +
            f"sys.path.insert(0, {str(root)!r})\nfrom attnprofile_b200 import *\n"
            "print('attn' in globals(), 'attn_cached' in globals())\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-800:]
    assert r.stdout.split() == ["True", str(torch_there)]
