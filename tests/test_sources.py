"""What the tree's sources, scripts and build files must not hold, whether or not a target builds them (no GPU)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIRS = ("harkdb_amd", "include", "oracle", "tests", "tools")
SUFFIXES = (".hip", ".h", ".hpp", ".c", ".cc", ".cpp", ".inc", ".s", ".S", ".py", ".sh", ".mk", ".cmake")


def sources():
    for name in sorted(os.listdir(ROOT)):
        if name.endswith(SUFFIXES) or name == "Makefile":
            yield name
    for top in DIRS:
        for path, dirs, names in os.walk(os.path.join(ROOT, top)):
            dirs[:] = sorted(d for d in dirs if d not in ("build", "__pycache__"))
            for name in sorted(names):
                if name.endswith(SUFFIXES) or name == "Makefile":
                    yield os.path.relpath(os.path.join(path, name), ROOT)


def scalar_cache_writes(text):
    """(line, word) of every scalar memory instruction or builtin that writes: a store, an atomic, a write-back or a discard of the
    scalar data cache.  The scalar loads and that cache's invalidation are not meant."""
    found = []
    for number, line in enumerate(text.splitlines(), 1):
        for word in re.findall(r"(?<![a-z0-9])s_[a-z0-9_]+", line):
            parts = word.split("_")[1:]
            if "store" in parts or "atomic" in parts or ("dcache" in parts and "inv" not in parts):
                found.append((number, word))
    return found


def test_the_walk_reaches_the_kernels():
    seen = set(sources())
    assert {"bench.py", "harkdb_amd/csrc/k_fgb.hip", "harkdb_amd/csrc/Makefile", "tools/ubench.hip", "tests/test_sources.py"} <= seen


@pytest.mark.parametrize("writes", [("store", "dword"), ("scratch", "store", "dword"), ("buffer", "atomic", "add"), ("dcache", "wb")])
def test_a_write_is_seen(writes):
    word = "_".join(("s",) + writes)
    assert scalar_cache_writes("nop\n  " + word + " s0, s[2:3], 0x0") == [(2, word)]
    assert scalar_cache_writes("// __builtin_amdgcn_" + word + "()") == [(1, word)]


@pytest.mark.parametrize("line", ["s_load_dwordx4 s[0:3], s[4:5], 0x0", "s_dcache_inv", "global_atomic_add v0, v1, s[2:3]",
                                  "ds_add_u32 v0, v1", "keys_store(a)", "buffer_store_dword v0, v1, s[0:3], 0"])
def test_a_vector_store_or_a_scalar_load_is_not(line):
    assert scalar_cache_writes(line) == []


def test_no_source_writes_through_the_scalar_data_cache():
    """Comments included.  All of the engine's device data is written by vector stores and vector / LDS atomics; a source that
    writes through the scalar data cache keeps the whole tree from being run where such code is not accepted."""
    found = []
    for name in sources():
        with open(os.path.join(ROOT, name), encoding="utf-8", errors="replace") as f:
            found += ["%s:%d %s" % (name, number, word) for number, word in scalar_cache_writes(f.read())]
    assert not found, "\n".join(found)


NO_PACKED_F32 = "-Xclang -target-feature -Xclang -packed-fp32-ops"


@pytest.mark.parametrize("where", ["harkdb_amd/csrc", "tools"])
def test_every_unit_is_compiled_without_packed_f32(where):
    """Some forms of the packed f32 add, multiply and fma have given wrong results now and then, and the compiler makes them by
    itself out of ordinary float code: no unit may be compiled with them on, whether or not its present code would get any."""
    r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, where)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    compiles = [line for line in r.stdout.splitlines() if "hipcc" in line and ".hip" in line and "check_hidden_loads" not in line]
    units = [n for n in os.listdir(os.path.join(ROOT, where)) if n.endswith(".hip")]
    assert len(compiles) == len(units)
    assert [line for line in compiles if NO_PACKED_F32 not in line] == []


@pytest.mark.parametrize("script", ["tools/check_hidden_loads.py", "tools/ab_build.sh"])
def test_the_scripts_compile_as_the_makefile_does(script):
    with open(os.path.join(ROOT, script)) as f:
        text = f.read()
    assert NO_PACKED_F32 in re.sub(r"[\",\s]+", " ", text)
