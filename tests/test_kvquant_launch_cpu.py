"""How the kernels of the 8-bit KV cache are launched, and what the library remembers of it: kvquant*.cu over a stand-in for the CUDA runtime that
launches nothing and writes down what it was asked for."""
import ctypes as C
import os
import re
import subprocess

import pytest

from denograd_b200 import build as B
from denograd_b200 import ffi
from tests.test_kvquant_cpu import CALLS, HOOKS, LAUNCHES, desc
from tests.util import ROOT

MORE_HOOKS = """
extern "C" __attribute__((visibility("default"))) void fake_give_up(jg_dev* dev, int code) { *dev->err_word = code; }
extern "C" __attribute__((visibility("default"))) int fake_is_fresh(jg_dev* dev, uint64_t p) { return jg_is_fresh(dev, (const void*)p); }
"""
ATTRIBUTES = """
#include <cuda_runtime_api.h>
extern "C" {
__attribute__((visibility("default"))) int fake_cooperative = 0, fake_early = 0, fake_grid = 0;  // of the last launch
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void*, void**) {
  fake_launches++;
  fake_cooperative = fake_early = 0;
  fake_grid = (int)(c->gridDim.x * c->gridDim.y * c->gridDim.z);
  for (unsigned i = 0; i < c->numAttrs; i++) {
    if (c->attrs[i].id == cudaLaunchAttributeCooperative) fake_cooperative = c->attrs[i].val.cooperative;
    if (c->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) fake_early = c->attrs[i].val.programmaticStreamSerializationAllowed;
  }
  return cudaSuccess;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    (d / "hooks.cu").write_text(HOOKS + MORE_HOOKS)
    plain = "cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { fake_launches++; return cudaSuccess; }\n"
    head, rest = LAUNCHES.split(plain)
    counter = head.split('extern "C" {\n')[1]
    (d / "launches.cpp").write_text(ATTRIBUTES.replace('extern "C" {\n', 'extern "C" {\n' + counter) + rest)
    so = str(d / "libfake.so")
    kvq = sorted(f for f in os.listdir(B.CSRC) if f.startswith("kvquant") and f.endswith(".cu"))
    subprocess.run([B.nvcc(), *B.ARCH, *B.FLAGS, "-I", B.CSRC, "-cudart", "none", "-shared", "-o", so, str(d / "hooks.cu"), str(d / "launches.cpp"),
                    os.path.join(ROOT, "tests", "fake_cudart.cpp"), os.path.join(B.CSRC, "device.cu"), *[os.path.join(B.CSRC, f) for f in kvq]], check=True)
    lib = C.CDLL(so)
    for name, args in ffi.SIGNATURES.items():
        if name.startswith(("jg_kvq_", "jg_device_", "jg_graph_")):
            getattr(lib, name).argtypes = args
    lib.jg_last_error.restype = C.c_char_p
    lib.fake_is_fresh.argtypes = [C.c_void_p, C.c_uint64]
    lib.fake_give_up.argtypes = [C.c_void_p, C.c_int]
    return lib


@pytest.fixture
def dev(lib):
    h = C.c_void_p()
    assert lib.jg_device_open(0, C.byref(h)) == 0
    return h


@pytest.fixture
def kv(lib, dev):
    h = C.c_void_p()
    assert lib.jg_kvq_create(dev, C.byref(desc()), ffi.KVQ_INT8, C.byref(h)) == 0
    yield h
    assert lib.jg_kvq_destroy(h) == 0


def last(lib, what):
    return C.c_int.in_dll(lib, "fake_" + what).value


@pytest.mark.parametrize("fmt", [ffi.KVQ_INT8, ffi.KVQ_E4M3])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_ctas_that_wait_for_one_another_run_at_once(lib, dev, fmt, head_dim):
    """The pieces of a long item are added up by all its CTAs, each of which waits for the others': without a cooperative launch two handles' launches
    on one GPU could each have half of the SMs and wait for the other half."""
    h = C.c_void_p()
    assert lib.jg_kvq_create(dev, C.byref(desc(head_dim=head_dim)), fmt, C.byref(h)) == 0
    width = 8 * head_dim
    many = dict(CALLS["attn"][0], max_count=60, ldo=width, ldq=width)
    assert lib.jg_kvq_attn(dev, h, *many.values()) == 0
    assert last(lib, "cooperative") == 1 and last(lib, "early") == 0
    few = dict(many, max_count=1)
    assert lib.jg_kvq_attn(dev, h, *few.values()) == 0
    assert last(lib, "cooperative") == 0 and last(lib, "early") == 1  # nobody waits there
    assert lib.jg_kvq_destroy(h) == 0


# a call, its arguments in place of the usual ones, and what it writes: (argument, bytes)
@pytest.mark.parametrize("name,args,written", [
    ("write", dict(q_out=1 << 20, ldq=520, R=5), [("q_out", 5 * 520 * 2)]), ("write", dict(q_out=0, ldq=0), []), ("decode", dict(out=1 << 20, ldo=520, B=5), [("out", 5 * 520 * 2)]),
    ("attn", dict(out=1 << 20, ldo=512, R=20), [("out", 20 * 512 * 2)]), ("attn", dict(out=1 << 20, ldo=512, R=200, max_count=60), [("out", 200 * 512 * 2)]),
    ("read", dict(k=1 << 20, v=1 << 24, ld=136, R=20), [("k", 20 * 136 * 2), ("v", 20 * 136 * 2)])])
def test_what_is_written_is_no_weight_to_read_early(lib, dev, kv, name, args, written):
    """Projections ask for their weights ahead of their dependency, but not for a matrix that the launches in front of them write: K and V as they are read
    back, say, whose product with queries is the next call."""
    args = dict(CALLS[name][0], **args)
    assert getattr(lib, f"jg_kvq_{name}")(dev, kv, *args.values()) == 0, lib.jg_last_error()
    for what, n in written:
        at = args[what]
        assert [lib.fake_is_fresh(dev, p) for p in (at - 2, at, at + n // 2, at + n - 2, at + n)] == [0, 1, 1, 1, 0]
    assert not lib.fake_is_fresh(dev, 1 << 28) and not lib.fake_is_fresh(dev, CALLS[name][0]["pos"])
    assert lib.jg_device_sync(dev) == 0
    assert not any(lib.fake_is_fresh(dev, args[what]) for what, _ in written)


def test_a_wait_that_gave_up_is_named(lib, dev, kv):
    """Its own codes for the kernel of chunks, in the message as they are in the kernel."""
    with open(os.path.join(B.CSRC, "kvquant_chunk.cu")) as f:
        used = set(re.findall(r"atomicCAS\(a\.err, 0, (\w+)\)", f.read()))
    names = ["JG_WAIT_KVQ_PLAN", "JG_WAIT_KVQ_CODES", "JG_WAIT_KVQ_PRODUCTS", "JG_WAIT_KVQ_SOFTMAX", "JG_WAIT_KVQ_PIECES"]
    assert used == set(names)
    for code, what in zip(range(6, 11), ("plan", "codes", "products", "softmax", "pieces of other CTAs")):
        assert lib.jg_kvq_attn(dev, kv, *dict(CALLS["attn"][0], max_count=60).values()) == 0
        lib.fake_give_up(dev, code)
        assert lib.jg_device_sync(dev) == ffi.JG_ETIMEDOUT
        message = lib.jg_last_error().decode()
        assert f"code {code}:" in message and f"{code} = {what}" in message and "8-bit KV cache" in message
        assert lib.jg_device_sync(dev) == 0


def test_bytes_are_those_of_codes_scales_and_table(lib, kv):
    n = C.c_uint64()
    assert lib.jg_kvq_bytes(kv, C.byref(n)) == 0
    assert n.value == 2 * 12 * 16 * 2 * (2 * 64 + 4) + 3 * 4 * 4  # layers, pages, positions, kv heads; without the workspace
