"""Paged-cache entry points refuse bad arguments before any CUDA call (no GPU needed)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from cutilegpt_b200 import _lib as L

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gpt_b200.h")
S3 = L.strides3(64, 64, 64)
ONE = 256   # any non-null address: nothing is read before the checks


def cache(**changes):
    s = L.PagedKvStruct(k_pages=ONE, v_pages=ONE, n_pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=2048,
                        head_stride=1024, slot_stride=64, page_table=ONE, ld_page_table=4, max_pages=4, seq_lens=ONE,
                        batch=4, prefix_table=ONE, ld_prefix_table=4, max_prefix_pages=4, prefix_lens=ONE, n_groups=2)
    for k, v in changes.items():
        setattr(s, k, v)
    return s


def attend(kv, q=ONE, T=1, H=4, scale=0.125, ws=None, nbytes=0, dtype=L.GPT_BF16, strides=S3):
    return L.lib().gpt_attention_shared_prefix(q, strides, ONE, strides, T, H, kv and ctypes.byref(kv), scale, ws, nbytes,
                                               dtype, None)


def append(kv, k=ONE, T=1, H=4, cos_sin=ONE, n_pos=8, rot=64, dtype=L.GPT_BF16, q=ONE):
    return L.lib().gpt_paged_kv_append(q, S3, k, S3, ONE, S3, ONE, S3, T, H, kv and ctypes.byref(kv), cos_sin, n_pos, rot, 0,
                                       dtype, None)


BAD_CACHES = [({"n_pages": 0}, L.GPT_ERR_SHAPE), ({"n_pages": 1 << 31}, L.GPT_ERR_SHAPE), ({"page_size": 0}, L.GPT_ERR_SHAPE),
              ({"head_dim": 0}, L.GPT_ERR_SHAPE), ({"head_dim": 257}, L.GPT_ERR_SHAPE), ({"kv_heads": 0}, L.GPT_ERR_SHAPE),
              ({"batch": -1}, L.GPT_ERR_SHAPE), ({"max_pages": 0}, L.GPT_ERR_SHAPE), ({"ld_page_table": 3}, L.GPT_ERR_SHAPE),
              ({"max_pages": 1 << 40, "ld_page_table": 1 << 40}, L.GPT_ERR_SHAPE), ({"n_groups": 3}, L.GPT_ERR_SHAPE),
              ({"max_prefix_pages": 0}, L.GPT_ERR_SHAPE), ({"ld_prefix_table": 1}, L.GPT_ERR_SHAPE),
              ({"slot_stride": -64}, L.GPT_ERR_SHAPE), ({"k_pages": None}, L.GPT_ERR_ARG), ({"seq_lens": None}, L.GPT_ERR_ARG),
              ({"prefix_lens": None}, L.GPT_ERR_ARG), ({"page_table": None}, L.GPT_ERR_ARG)]


@pytest.mark.parametrize("changes,status", BAD_CACHES, ids=lambda x: str(x)[:40])
def test_bad_caches_are_refused(changes, status):
    assert attend(cache(**changes)) == status
    assert append(cache(**changes)) == status
    assert L.lib().gpt_last_error_string()


def test_bad_arguments_are_refused():
    assert attend(None) == L.GPT_ERR_ARG and append(None) == L.GPT_ERR_ARG
    assert attend(cache(), dtype=7) == L.GPT_ERR_DTYPE and append(cache(), dtype=7) == L.GPT_ERR_DTYPE
    assert attend(cache(), H=3) == L.GPT_ERR_SHAPE and attend(cache(), H=0) == L.GPT_ERR_SHAPE
    assert attend(cache(), T=-1) == L.GPT_ERR_SHAPE and attend(cache(), T=1 << 29) == L.GPT_ERR_SHAPE
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(cache(), scale=scale) == L.GPT_ERR_ARG
    assert attend(cache(), q=None) == L.GPT_ERR_ARG and append(cache(), k=None) == L.GPT_ERR_ARG
    for rot, status in ((3, L.GPT_ERR_SHAPE), (66, L.GPT_ERR_SHAPE), (-2, L.GPT_ERR_SHAPE)):
        assert append(cache(), rot=rot) == status
    assert append(cache(), n_pos=0) == L.GPT_ERR_SHAPE
    assert append(cache(), cos_sin=None) == L.GPT_ERR_ARG and append(cache(), q=None) == L.GPT_ERR_ARG
    assert append(cache(), H=0) == L.GPT_ERR_SHAPE and append(cache(), T=-1) == L.GPT_ERR_SHAPE
    # nothing to do is no error
    assert attend(cache(batch=0)) == L.GPT_OK and append(cache(), T=0) == L.GPT_OK and attend(cache(), T=0) == L.GPT_OK


def test_workspace_is_required_and_checked():
    size = L.lib().gpt_attention_shared_prefix_workspace_size
    kv = cache(max_prefix_pages=4096, ld_prefix_table=4096)
    need = size(1, 4, ctypes.byref(kv), L.GPT_BF16)
    assert need > 0
    assert attend(kv) == L.GPT_ERR_ARG and attend(kv, ws=ONE, nbytes=need - 1) == L.GPT_ERR_ARG
    assert attend(kv, ws=ONE + 4, nbytes=need) == L.GPT_ERR_ALIGN
    assert size(1, 3, ctypes.byref(kv), L.GPT_BF16) == 0 and size(0, 4, ctypes.byref(kv), L.GPT_BF16) == 0
    assert size(1, 4, None, L.GPT_BF16) == 0 and size(1, 4, ctypes.byref(cache(n_pages=0)), L.GPT_BF16) == 0


def test_struct_layout_matches_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    fields = [f[0] for f in L.PagedKvStruct._fields_]
    body = "".join(f'  printf("{f} %zu\\n", offsetof(gpt_paged_kv, {f}));\n' for f in fields)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n{body}'
                   f'  printf("sizeof %zu\\n", sizeof(gpt_paged_kv));\n  return 0;\n}}\n')
    subprocess.run([gcc, "-o", str(exe), str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for f in fields:
        assert int(got[f]) == getattr(L.PagedKvStruct, f).offset, f
    assert int(got["sizeof"]) == ctypes.sizeof(L.PagedKvStruct)
