"""Rules on the text of the native sources: checked without a compiler or a GPU."""
import re
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
SUFFIXES = {".hip", ".h", ".hpp", ".cpp", ".cu", ".s", ".inc", ".patch", ".py", ".sh"}

# Scalar stores, scalar atomics and the scalar data cache's write-back / discard, as instructions or as builtins
# (`..._s_<op>`); put together here so that this file does not itself hold one.
SCALAR_CACHE_WRITE = re.compile(r"(?<![A-Za-z0-9])" + "s_" + r"(?:(?:buffer_|scratch_)?(?:store|atomic)_\w+|dcache_(?:wb|discard)\w*)")


def sources(folder):
    return sorted(p for p in (REPO / folder).rglob("*") if p.is_file() and (p.suffix in SUFFIXES or p.name == "Makefile"))


@pytest.mark.parametrize("op", ["store_dwordx2 s[0:1], s[2:3], 0x0", "buffer_store_dword s0, s[4:7], 0x0",
                                "scratch_store_dword s0, s1, 0x0", "atomic_add s0, s[2:3], 0x0",
                                "buffer_atomic_add s0, s[4:7], 0x0", "dcache_wb", "dcache_wb_vol", "dcache_discard s[0:1], 0x0"])
def test_pattern_sees_every_form(op):
    assert SCALAR_CACHE_WRITE.search("\t" + "s_" + op)
    assert SCALAR_CACHE_WRITE.search("__builtin_amdgcn_" + "s_" + op)


@pytest.mark.parametrize("text", ["s_load_dwordx2 s[0:1], s[2:3], 0x0", "global_store_dwordx2 v0, v[2:3], s[0:1]",
                                  "buffer_store_dword v0, off, s[0:3], 0", "scratch_store_dword off, v0, off",
                                  "ds_store_b64 v0, v[2:3]", "s_memtime s[0:1]"])
def test_pattern_leaves_the_rest(text):
    assert not SCALAR_CACHE_WRITE.search(text)


@pytest.mark.parametrize("folder", ["hydra_pspec_amd", "include", "tools"])
def test_no_source_writes_through_the_scalar_data_cache(folder):
    """Debugging branches and comments included: data goes to memory through vector stores only."""
    files = sources(folder)
    assert files
    found = [f"{p.relative_to(REPO)}:{no}: {m.group(0)}" for p in files
             for no, line in enumerate(p.read_text(errors="replace").splitlines(), 1)
             for m in SCALAR_CACHE_WRITE.finditer(line)]
    assert not found, "\n".join(found)
