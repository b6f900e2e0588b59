"""CPU tests of the prompt cache's argument checks: they raise before anything touches a GPU."""
import ctypes

import pytest
import torch

from conftest import HAS_GPU


@pytest.fixture(scope="module")
def pc():
    import abstracts_search_amd._native as nat
    nat.build("encoder")
    import abstracts_search_amd.prompt_cache as m
    return m


@pytest.mark.parametrize("change", [dict(dtype=torch.float32), dict(head_dim=96), dict(n_layers=0), dict(n_kv_heads=0), dict(n_pages=0),
                                    dict(max_entries=0), dict(max_tokens=0)])
def test_bad_configurations(pc, change):
    a = dict(n_layers=2, n_kv_heads=2, head_dim=64, n_pages=4)
    a.update(change)
    with pytest.raises(ValueError):
        pc.PromptCache(**a)


@pytest.mark.skipif(HAS_GPU, reason="checks the no-GPU failure mode")
def test_no_cpu_fallback(pc):
    with pytest.raises(RuntimeError, match="no HIP device"):
        pc.PromptCache(2, 2, 64, 4)


def test_c_entries_refuse_null_and_bad_arguments(pc):
    lib = pc._Lib.get()
    h, n = ctypes.c_void_p(), ctypes.c_int32()
    assert lib.mi_prompt_cache_create(None, 0, None, ctypes.byref(h)) != 0
    for bad in ((0, 2, 64, 1, 4, 1, 0), (2, 2, 96, 1, 4, 1, 0), (2, 2, 64, 0, 4, 1, 0), (2, 2, 64, 1, 0, 1, 0), (2, 2, 64, 1, 1 << 30, 1, 0),
                (2, 2, 64, 1, 4, 0, 0), (2, 2, 64, 1, 4, 1, -1)):
        assert lib.mi_prompt_cache_create(ctypes.byref(pc._Cfg(*bad)), 0, None, ctypes.byref(h)) != 0
        assert b"prompt cache" in lib.mi_enc_last_error()
    assert lib.mi_prompt_cache_new(None, None, ctypes.byref(n)) != 0
    assert lib.mi_prompt_cache_reserve(None, 0, 1, None) != 0
    assert lib.mi_prompt_cache_fork(None, 0, 1, ctypes.byref(n), None, None) != 0
    assert lib.mi_prompt_cache_free(None, 0, None, None) != 0
    assert lib.mi_prompt_cache_compact(None, None, None) != 0
    assert lib.mi_prompt_cache_resize(None, None, 1, None) != 0
    assert lib.mi_prompt_attention(None, None, None) != 0
    assert b"null argument" in lib.mi_enc_last_error()
    assert lib.mi_prompt_cache_destroy(None) == 0


def test_the_argument_block_is_the_headers_struct(pc):
    """the packed form of mi_prompt_attn has the C layout (every field at its natural alignment, in the header's order)"""
    import re
    from conftest import ROOT
    txt = open(f"{ROOT}/include/mi_encoder.h").read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct mi_prompt_attn \{(.*?)\}", txt, re.S).group(1), flags=re.S)
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    fields = []
    for line in body.split(";"):
        line = " ".join(line.split())
        if not line:
            continue
        base, names = re.match(r"(?:const )?(\w+) (.*)", line).groups()
        for name in names.split(","):
            name = name.strip()
            fields.append((name.lstrip("*"), ctypes.c_void_p if name.startswith("*") else kinds[base]))
    S = type("S", (ctypes.Structure,), {"_fields_": fields})
    assert ctypes.sizeof(S) == pc._ATTN.size
    vals = list(range(1, len(fields) + 1))
    s = S.from_buffer_copy(pc._ATTN.pack(*vals))
    assert [int(getattr(s, f)) for f, _ in fields] == vals


@pytest.mark.parametrize("change", [dict(n_layers=2 ** 32 + 1), dict(n_kv_heads=2 ** 32 + 2), dict(n_pages=2 ** 32 + 4), dict(max_entries=2 ** 32 + 1),
                                    dict(max_tokens=2 ** 32 + 1), dict(max_tokens=-1)])
def test_configurations_beyond_32_bits(pc, change):
    """ctypes would cut them to numbers that look right"""
    with pytest.raises(ValueError, match="int32"):
        pc.PromptCache(**{**dict(n_layers=2, n_kv_heads=2, head_dim=64, n_pages=4), **change})
