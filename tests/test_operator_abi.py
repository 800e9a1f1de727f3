"""Host side of the norm, the key/value cache and attention: struct layouts and the argument
checks that run before any CUDA call (no device needed)."""
import ctypes
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structs_match_header_layout(pkg, tmp_path):
    L = pkg._lib
    structs = {"gs_rms_norm_args": L.GsRmsNormArgs, "gs_kv_cache_desc": L.GsKvCacheDesc, "gs_kv_rows": L.GsKvRows,
               "gs_attention_args": L.GsAttentionArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gsampler.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));')
    for name in ("GS_DTYPE_E4M3", "GS_DTYPE_INT8", "GS_KV_ERR_SLOT", "GS_KV_ERR_PAGE", "GS_KV_ERR_LENGTH", "GS_KV_ERR_TIMEOUT"):
        lines.append(f'printf("{name} %d\\n", (int){name});')
    lines.append("return 0; }")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"
    for name in ("GS_DTYPE_E4M3", "GS_DTYPE_INT8"):
        assert int(got[name]) == getattr(L, name)
    for name in ("SLOT", "PAGE", "LENGTH", "TIMEOUT"):
        assert int(got["GS_KV_ERR_" + name]) == getattr(L, "KV_ERR_" + name)


def test_null_handles_and_arguments_are_refused(pkg):
    L = pkg._lib
    lib = L.lib()
    h = ctypes.c_void_p()
    assert lib.gs_rms_norm(None, ctypes.byref(L.GsRmsNormArgs()), None) == L.GS_EINVAL
    assert lib.gs_kv_cache_create(None, ctypes.byref(L.GsKvCacheDesc()), ctypes.byref(h)) == L.GS_EINVAL
    assert lib.gs_kv_cache_create(None, None, None) == L.GS_EINVAL
    assert lib.gs_kv_write(None, ctypes.byref(L.GsKvRows()), None) == L.GS_EINVAL
    assert lib.gs_kv_read(None, ctypes.byref(L.GsKvRows()), None) == L.GS_EINVAL
    assert lib.gs_attention(None, ctypes.byref(L.GsAttentionArgs()), None) == L.GS_EINVAL
    assert lib.gs_kv_cache_check(None, None) == L.GS_EINVAL
    assert lib.gs_kv_cache_destroy(None) == L.GS_OK
    assert lib.gs_kv_cache_last_error(None) == b""


def test_packed_arguments_have_the_structs_layout(pkg):
    """norm.py and kv_cache.py pack the argument structures with struct formats."""
    import importlib
    norm = importlib.import_module("gemma-webgpu-engine_b200.norm")
    kv = importlib.import_module("gemma-webgpu-engine_b200.kv_cache")
    L = pkg._lib
    for packer, cls in ((norm._RMS_NORM_ARGS, L.GsRmsNormArgs), (kv._KV_ROWS, L.GsKvRows), (kv._ATTENTION_ARGS, L.GsAttentionArgs)):
        assert packer.size == ctypes.sizeof(cls), cls
        values = [i + 1 for i in range(len(cls._fields_))]
        got = cls.from_buffer_copy(packer.pack(*values))
        assert [int(getattr(got, f)) for f, _ in cls._fields_] == values
