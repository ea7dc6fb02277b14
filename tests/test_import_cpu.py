"""The package imports without the extension in front of the library, and with a library from before the operators that use it
(AITER_B200_LIBRARY compares builds); those operators then fail by name."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "aiter_b200")

OLD_LIBRARY = """
const char* aiter_get_last_error(void) { return ""; }
const char* aiter_b200_kernel_list(void) { return "an old build"; }
const char* aiter_b200_heuristic_name(void) { return ""; }
unsigned long long aiter_b200_launch_count(void) { return 7; }
int aiter_ctypes_abi_version(void) { return 2; }
"""


def _run(program, cwd, **env):
    return subprocess.run([sys.executable, "-c", program], cwd=cwd, env={**os.environ, **env}, capture_output=True, text=True, timeout=300)


USE = """
import torch, aiter_b200 as ab
print(ab.kernel_list()[:12])
for call in (lambda: ab.act_and_mul(torch.zeros(2, 64)), lambda: ab.gated_residual_norm(torch.zeros(2, 64)), lambda: ab.gemm_a16w16_fused(torch.zeros(2, 64), torch.zeros(8, 64))):
    try:
        call()
    except ImportError as e:
        print("refused:", e)
"""


def test_a_library_from_before_the_fused_operators(tmp_path):
    (tmp_path / "old.c").write_text(OLD_LIBRARY)
    old = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(old), str(tmp_path / "old.c")], check=True)
    p = _run(USE, ROOT, AITER_B200_LIBRARY=str(old))
    assert p.returncode == 0, p.stderr[-2000:]
    assert "an old build" in p.stdout and p.stdout.count("was built before this operator") == 3, p.stdout


def test_without_the_extension(tmp_path):
    shutil.copytree(PACKAGE, tmp_path / "aiter_b200", ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    os.symlink(os.path.join(PACKAGE, "csrc", "libaiter_b200.so"), tmp_path / "aiter_b200" / "csrc" / "libaiter_b200.so")
    p = _run(USE, tmp_path, PYTHONPATH=str(tmp_path), AITER_B200_LIBRARY="")
    assert p.returncode == 0, p.stderr[-2000:]
    assert "kernelName" in p.stdout and p.stdout.count("is missing: build it with") == 3, p.stdout
