"""The host barriers between the shards of a context that lists a device more than once, without a
device: tests/native/peer_group.cpp, built against the library's headers and run."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_barriers(tmp_path):
    lib = os.path.join(ROOT, "mymedialite_amd", "lib")
    exe = str(tmp_path / "peer_group")
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__",
                    "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "mymedialite_amd", "csrc"), "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "native", "peer_group.cpp"), "-o", exe, "-L" + lib,
                    "-lmml_hip", "-L/opt/rocm/lib", "-lamdhip64", "-lrccl", "-pthread",
                    "-Wl,-rpath," + lib + ":/opt/rocm/lib"], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr
    assert p.stdout.count("ok:") == 7
