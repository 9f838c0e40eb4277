"""AdamW without memory for the staging of one of its tensors, on the CPU: the library's host code on a HIP runtime that only counts
(tests/host/adamw_refused.cpp)."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"
CLANG = "/opt/rocm/lib/llvm/bin/clang++"


def test_a_refused_tensor_leaves_the_others(tmp_path):
    inc = ["-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "pulp-trainlib_amd", "csrc")]
    objs = []
    for src in ("pulp-trainlib_amd/csrc/ptl_adamw.hip", "pulp-trainlib_amd/csrc/ptl_runtime.hip", "tests/host/adamw_refused.cpp"):
        objs.append(str(tmp_path / (os.path.basename(src) + ".o")))
        subprocess.check_call([HIPCC, "--offload-arch=gfx950", "--offload-host-only"] + inc + ["-c", os.path.join(ROOT, src), "-o", objs[-1]])
    # (the device's code, which is not there)
    gone = set(re.findall(r"\bU (__hip_fatbin\w*)", subprocess.check_output(["nm"] + objs, text=True)))
    exe = str(tmp_path / "adamw_refused")
    subprocess.check_call([CLANG, "-pthread"] + objs + ["-Wl,--defsym=%s=0" % s for s in sorted(gone)] + ["-o", exe])
    res = subprocess.run([exe], stdout=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, res.stdout
