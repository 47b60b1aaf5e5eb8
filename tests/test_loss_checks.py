"""What the losses over logit rows refuse, and how a call is cut into workgroups: compiled for the host
(tests/native/loss_checks.cpp). And the exports of their header, and calls without a sampler."""
import ctypes as C
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_checks_and_plans(tmp_path):
    exe = str(tmp_path / "loss_checks")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-o", exe,
                    os.path.join(ROOT, "tests", "native", "loss_checks.cpp")], check=True)
    p = subprocess.run([exe], capture_output=True, text=True)
    assert p.returncode == 0, p.stdout + p.stderr
    assert "runtime error" not in p.stderr, p.stderr


def test_the_header_is_exported_and_refuses_a_null_sampler():
    text = open(os.path.join(ROOT, "include", "geist_loss_hip.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(geist_hip_\w+)\s*\(", text)))
    lib = C.CDLL(os.path.join(ROOT, "geistlib_amd", "lib", "libgeist_sampler_hip.so"))
    assert names == ["geist_hip_distill_rows", "geist_hip_loss_workspace_bytes",
                     "geist_hip_policy_loss_rows", "geist_hip_preference_loss"]
    for name in names:
        assert hasattr(lib, name)
    assert lib.geist_hip_distill_rows(None, None, None, None, None, C.c_size_t(0)) == 2
    assert lib.geist_hip_policy_loss_rows(None, None, None, None, None, None, None, C.c_size_t(0)) == 2
    assert lib.geist_hip_preference_loss(None, None, None, None, None, None, None, C.c_size_t(0)) == 2


def test_the_header_is_plain_c(tmp_path):
    src = tmp_path / "plain.c"
    src.write_text('#include "geist_loss_hip.h"\nint main(void) { struct geist_hip_loss_rows r = {0}; '
                   "return (int) r.rows; }\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o",
                    str(tmp_path / "plain"), str(src)], check=True)
