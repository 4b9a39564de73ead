"""What the calls on the int8 key/value cache enqueue, without a GPU: on a HIP runtime that keeps count and runs no kernel
(tests/host_runtime/fake_runtime.cpp)."""
import ctypes as C
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest

from vtl_amd import attention_i8_workspace, capi

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

_PRELUDE = r"""
import ctypes as C, re, sys
fake = C.CDLL(sys.argv[2], mode=C.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[1])
from vtl_amd import capi
fake.fake_set(1, 0, 0, 0)
ONE = 1 << 20                  # an address that nothing here reads

def launches():
    buf = C.create_string_buffer(1 << 20)
    n = fake.fake_log(buf, C.c_size_t(len(buf)))
    lines = [l.split() for l in buf.raw[:n].decode().splitlines()]
    return [(l[4], int(l[3])) for l in lines if l[0] == "launch"]

def attention(kv_heads, heads, dim, batch, rows, starts=ONE, most_rows=0, most_length=0, max_pages=4, page=16):
    cache = capi.KVCache(ONE, 4, page, kv_heads, dim)
    b = capi.KVBatch(batch, max_pages, ONE, ONE, starts, rows, most_rows, most_length)
    launches()
    st = capi.status("vtl_hip_attention_i8_f32", C.byref(cache), C.byref(b), 1 << 30, heads * dim, heads, 0.125, 1, 1 << 50, heads * dim, ONE, 1 << 40)
    return st, launches()
"""


@pytest.fixture(scope="module")
def fake_runtime(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("runtime") / "libfake_runtime.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "host_runtime", "fake_runtime.cpp"), "-o", out], check=True)
    return out


def _run(fake, program):
    res = subprocess.run([sys.executable, "-c", _PRELUDE + program, ROOT, fake], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip().endswith("done"), res.stdout[-3000:]


def test_grids_of_very_many_sequences(fake_runtime):
    """A grid has less than 2^32 threads in a row, whatever number of waves a workgroup would have."""
    _run(fake_runtime, r"""
for batch in (1 << 19, (1 << 20) - 1, 1 << 20, (1 << 21) - 1):
    st, log = attention(8, 8, 64, batch, batch)
    assert st == capi.OK and len(log) >= 1, (batch, st)
    name, blocks = log[0]
    waves = int(re.search(r"attention_many_kernelILi64ELi(\d)E", name).group(1))
    assert blocks % (8 * batch) == 0 and 8 * batch * 64 * waves < 1 << 32, (batch, waves)
    assert waves == (8 if batch < 1 << 20 else 4), (batch, waves)
assert attention(8, 8, 64, 1 << 21, 1 << 21)[0] == capi.ERR_UNSUPPORTED
print("done")
""")


def test_variants_for_few_rows(fake_runtime):
    """Which of them a call takes, and that its parts are added up by a launch of their own while a graph is recorded and on streams without
    counters, and within the launch on others."""
    _run(fake_runtime, r"""
sys.path.insert(0, sys.argv[1] + "/tests")
from kv_cases import SHARED
for variant, (lengths, counts, heads, kv_heads, dim) in SHARED.items():
    rows = len(lengths) if counts is None else sum(counts)
    def names(stream):
        capi.call("vtl_hip_set_stream", stream)
        st, log = attention(kv_heads, heads, dim, len(lengths), rows, ONE if counts else None, max(counts or [1]), max(lengths), 1 + max(lengths) // 16)
        assert st == capi.OK
        return [re.sub(r"Li(\d+)E", r"\1 ", re.search(r"attention_(\w+?_kernelI(?:Li\d+E)+)", n).group(1)) for n, _ in log]
    few, join = ("%s_kernelI%d %d %d " % (what, *variant) for what in ("few", "few_join"))
    assert names(None) == [few], (variant, names(None))
    for stream in range(2, 17):       # the null stream is the first
        assert names(stream) == [few]
    assert names(17) == [few, join], (variant, names(17))
    fake.fake_set(1, 1, 0, 0)
    assert names(2) == [few, join]
    fake.fake_set(1, 0, 0, 0)
print("done")
""")


def test_workspace_of_the_python_mirror():
    one = 1 << 20
    cache = SimpleNamespace(handle=capi.KVCache(one, 400, 64, 8, 128))
    some = SimpleNamespace(handle=capi.KVBatch(2, 150, one, one, None, 2, 1, 9000))
    none = SimpleNamespace(handle=capi.KVBatch(2, 1, one, one, None, 2, 1, 60))
    need = attention_i8_workspace(cache, some, 32)
    assert need == capi.lib().vtl_hip_attention_i8_workspace(C.byref(cache.handle), C.byref(some.handle), 32) and need > 1 << 16
    assert attention_i8_workspace(cache, none, 32) < need and attention_i8_workspace(cache, none, 31) == 0


def test_workspace_of_the_cpp_mirror(fake_runtime, tmp_path):
    """What the mirror says is enough for the call, and one byte less is refused."""
    (tmp_path / "ws.cpp").write_text(r"""
#include "vtl_hip.hpp"
extern "C" int check()
{
    vtl::HipKVCache cache(400, 64, 8, 128);
    vtl::HipTensor<int32_t> table({2, 150}), lengths({2});
    vtl::HipKVBatch batch(table, lengths, nullptr, 0, 1, 9000);
    vtl::HipTensor<float> q({2, 32 * 128});
    const size_t need = vtl::attention_i8_workspace(cache, batch, 32);
    vtl::HipStorage<uint8_t> enough(need), less(need - 1);
    vtl::attention_i8_hip(cache, batch, q, 32, 0.1f, true, &enough);
    try {
        vtl::attention_i8_hip(cache, batch, q, 32, 0.1f, true, &less);
    } catch (const vtl::HipError &) {
        return need > 1 << 16;
    }
    return 0;
}
""")
    lib, program = os.path.join(ROOT, "vtl_amd"), str(tmp_path / "ws.so")
    subprocess.run(["g++", "-std=c++17", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(lib, "host"), str(tmp_path / "ws.cpp"),
                    "-o", program, "-L", lib, "-lvtlhip", "-Wl,-rpath," + lib], check=True)
    _run(fake_runtime, f"assert C.CDLL({program!r}).check() == 1\nprint('done')\n")
