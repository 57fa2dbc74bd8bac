"""The structs of the token-at-a-time operators, as ctypes mirrors and as a C compiler lays the header's out."""
import ctypes
import shutil
import pytest
import test_abi_cpu
from thunderworld_b200 import _lib


@pytest.mark.skipif(shutil.which('gcc') is None, reason='gcc not available')
def test_ctypes_mirrors_have_the_header_layout(tmp_path, monkeypatch):
    mirrors = {'TwMatvecArgs': _lib.MatvecArgs, 'TwPagedAttentionArgs': _lib.PagedAttentionArgs, 'TwCache': _lib.Cache, 'TwAppendArgs': _lib.AppendArgs}
    assert all(issubclass(m, ctypes.Structure) for m in mirrors.values())
    monkeypatch.setattr(test_abi_cpu, 'STRUCTS', mirrors)
    test_abi_cpu.test_ctypes_mirrors_have_the_header_layout(tmp_path)
