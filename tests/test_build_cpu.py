"""How the library is built."""
import importlib.util
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _build():
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "aiter_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_no_flag_trades_the_kernels_code_for_build_time():
    """--split-compile optimises the functions of a module apart from one another: registers and spills of every kernel change (the
    blockscale pair kernel spilled 92 bytes instead of 8, 8192 x 4096 x 4096 222 us instead of 138).  The same goes for lower
    optimisation levels, register caps over all kernels and approximate arithmetic."""
    flags = _build().NVCC_FLAGS
    assert "-O3" in flags
    for flag in flags:
        name = flag.lstrip("-").split("=")[0]
        assert name not in ("split-compile", "split-compile-extended", "Ofast-compile", "maxrregcount", "use_fast_math", "G", "device-debug"), flag


def test_the_extension_takes_the_librarys_function_types_from_its_header():
    """A pointer type written out by hand can differ from the function behind it (three long long for three int) without a word from the
    compiler, since the addresses arrive as integers."""
    import re

    with open(os.path.join(ROOT, "aiter_b200", "csrc", "host.cpp")) as f:
        source = f.read()
    assert not re.findall(r"using\s+\w+\s*=\s*[^;]*\(\*\)\s*\(", source), "a hand-written function pointer type"
    header = open(os.path.join(ROOT, "include", "aiter_b200.h")).read()
    names = re.findall(r"ENTRY\((aiter_b200_\w+)\)", source)
    assert len(names) >= 6 and all(re.search(rf"\b{n}\(", header) for n in names)
