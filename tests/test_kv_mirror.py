"""Runs the C++ host mirror's key/value cache and attention (tests/host_cpp/test_kv_mirror.cpp), and checks that the V
binding declares what the header does."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "host_cpp", "test_kv_mirror")


def _run(*args):
    return subprocess.run([BIN, *args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)


def test_refusals_without_device():
    if not os.path.exists(BIN):   # built by __graft_entry__.build(); this is the CPU-side fallback
        subprocess.run(["make", "-C", os.path.join(HERE, "host_cpp"), "test_kv_mirror"], check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    res = _run("--no-device")
    assert res.returncode == 0 and "kv mirror (no device): ok" in res.stdout, res.stdout


@pytest.mark.gpu
def test_on_device(hip):
    assert os.path.exists(BIN), "tests/host_cpp/test_kv_mirror is not built"
    res = _run()
    assert res.returncode == 0 and "kv mirror: ok" in res.stdout, res.stdout


def test_v_declarations_have_the_arguments_of_the_header():
    root = os.path.dirname(HERE)
    header = open(os.path.join(root, "include", "vtl_hip.h")).read()
    binding = open(os.path.join(root, "vtl_amd", "vbind", "kv_cache_hip_d_hip.v")).read()
    v_of = {"int": "int", "float": "f32", "size_t": "usize", "int64_t": "i64"}
    found = 0
    for name, args in re.findall(r"^fn C\.(vtl_hip_\w+)\((.*)\)", binding, re.M):
        declared = re.search(r"^(?:int|size_t) " + name + r"\(([^)]*)\)", header, re.M).group(1)
        wanted = []
        for arg in " ".join(declared.split()).split(", "):
            arg = arg.replace("const ", "")
            kind, what = re.fullmatch(r"(\w+) (\**)\w+", arg).group(1, 2)
            wanted.append("&C." + kind if kind.startswith("vtl_hip_") else "&voidptr" if what == "**" else "voidptr" if what else v_of[kind])
        assert [a.split()[1] for a in args.split(", ")] == wanted, name
        found += 1
    assert found == 8
    for struct in ("vtl_hip_kv_cache", "vtl_hip_kv_batch"):
        body = re.search(r"typedef struct \{([^}]*)\} " + struct + ";", header).group(1)
        body = re.sub(r"/\*.*?\*/", "", body)
        fields = [f.strip(" *") for line in body.split(";") if line.strip() for f in re.sub(r"^\s*(const )?\w+ ", "", line).split(",")]
        declared = re.search(r"struct C\." + struct + r" \{([^}]*)\}", binding).group(1)
        assert [line.split()[0] for line in declared.strip().splitlines()] == fields
