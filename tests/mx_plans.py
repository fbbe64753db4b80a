"""The plans of MXFP4 calls (acfun_amd/csrc/mx_plan.hpp), asked of a small program built
with g++."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CUS = 256


def build(folder):
    """The program, in `folder`."""
    exe = os.path.join(str(folder), "mx_plan_print")
    src = os.path.join(HERE, "mx_plan", "mx_plan_print.cpp")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                        "-o", exe, src], capture_output=True, text=True)
    assert r.returncode == 0, "mx_plan_print did not build:\n" + r.stderr
    return exe


def ask(exe, lines):
    """One answer for each line."""
    r = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout.split("\n")[:len(lines)]


def gemm(M, N, K, cus=CUS):
    return f"gemm {M} {N} {K} {cus}"


def fc(M, N, K, elem=2, cus=CUS):
    return f"fc {M} {N} {K} {elem} {cus}"
