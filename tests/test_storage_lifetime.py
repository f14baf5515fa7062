"""The C++ host API's storage objects against the order in which a program lets go of them."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "tenstorrent-wh-blockspmm_b200")


def test_storage_outlives_its_device(tmp_path):
    """Buffers and uploaded matrices destroyed after CloseDevice release
    through a handle that is still open (the C entries are recorders)."""
    exe = str(tmp_path / "storage")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{ROOT}/include",
                    os.path.join(ROOT, "tests", "cpp", "test_storage_lifetime.cpp"), "-pthread", f"-L{PKG}", "-lbsp",
                    f"-Wl,-rpath,{PKG}", "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
