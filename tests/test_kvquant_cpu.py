"""The 8-bit KV cache without a GPU: what the calls refuse (kvquant*.cu over a stand-in for the CUDA runtime that launches nothing), what the
Python class refuses, the codes against known answers, and which calls a model with such a cache makes."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from denograd_b200 import build as B
from denograd_b200 import ffi
from tests import kvquant_ref as R
from tests.fake_ffi import Recorder
from tests.golden.gen_golden import TINY
from tests.util import ROOT

HOOKS = """
#include "common.cuh"
void jg_pair_reset(jg_dev*) {}
int jg_peer_error(jg_dev*, int* code) { *code = 0; return JG_OK; }
int jg_peer_run_boundary(jg_dev*) { return JG_OK; }
"""
LAUNCHES = """
#include <cuda_runtime_api.h>
extern "C" {
__attribute__((visibility("default"))) int fake_launches = 0;
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { fake_launches++; return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) { a->numRegs = 128; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, CUstream_st*) { return 0; }
cudaError_t __cudaGetKernel(cudaKernel_t* k, const void* f) { *k = (cudaKernel_t)f; return cudaSuccess; }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    (d / "hooks.cu").write_text(HOOKS)
    (d / "launches.cpp").write_text(LAUNCHES)
    so = str(d / "libfake.so")
    kvq = sorted(f for f in os.listdir(B.CSRC) if f.startswith("kvquant") and f.endswith(".cu"))
    subprocess.run([B.nvcc(), *B.ARCH, *B.FLAGS, "-I", B.CSRC, "-cudart", "none", "-shared", "-o", so, str(d / "hooks.cu"), str(d / "launches.cpp"),
                    os.path.join(ROOT, "tests", "fake_cudart.cpp"), os.path.join(B.CSRC, "device.cu"), *[os.path.join(B.CSRC, f) for f in kvq]], check=True)
    lib = C.CDLL(so)
    for name, args in ffi.SIGNATURES.items():
        if name.startswith(("jg_kvq_", "jg_device_", "jg_graph_")):
            getattr(lib, name).argtypes = args
    lib.jg_last_error.restype = C.c_char_p
    return lib


@pytest.fixture
def dev(lib):
    h = C.c_void_p()
    assert lib.jg_device_open(0, C.byref(h)) == 0
    return h


def desc(**kw):
    d = dict(n_layers=2, n_kv_heads=2, head_dim=64, page_size=16, n_pages=12, max_batch=3, max_pages_per_seq=4, n_heads=8, n_split=0)
    return ffi.KvDesc(**dict(d, **kw))


@pytest.fixture
def kv(lib, dev):
    h = C.c_void_p()
    assert lib.jg_kvq_create(dev, C.byref(desc()), ffi.KVQ_INT8, C.byref(h)) == 0
    yield h
    assert lib.jg_kvq_destroy(h) == 0


@pytest.mark.parametrize("kw,fmt", [({"head_dim": 96}, 0), ({"page_size": 48}, 0), ({"n_heads": 7}, 0), ({"n_heads": 18}, 0), ({"n_layers": 0}, 0), ({"n_pages": 0}, 1),
                                    ({"max_batch": 1 << 20, "max_pages_per_seq": 1 << 12}, 0), ({"max_pages_per_seq": 1 << 28, "max_batch": 1}, 0), ({}, 2), ({}, -1),
                                    ({"max_pages_per_seq": (1 << 20) + 1, "max_batch": 1}, 0), ({"n_pages": 1 << 30, "n_kv_heads": 8}, 0)])
def test_create_refuses(lib, dev, kw, fmt):
    h = C.c_void_p()
    assert lib.jg_kvq_create(dev, C.byref(desc(**kw)), fmt, C.byref(h)) == ffi.JG_EINVAL
    assert not h.value and lib.jg_last_error().startswith(b"kvq_create")


def test_null_handles(lib, dev):
    h = C.c_void_p()
    assert lib.jg_kvq_create(None, C.byref(desc()), 0, C.byref(h)) == ffi.JG_EINVAL
    assert lib.jg_kvq_create(dev, None, 0, C.byref(h)) == ffi.JG_EINVAL
    assert lib.jg_kvq_destroy(None) == 0
    assert lib.jg_kvq_bytes(None, C.byref(C.c_uint64())) == ffi.JG_EINVAL
    assert lib.jg_kvq_set_block_table(None, None) == ffi.JG_EINVAL


def test_bytes(lib, kv):
    n = C.c_uint64()
    assert lib.jg_kvq_bytes(kv, C.byref(n)) == 0
    assert 2 * 12 * 16 * 2 * (2 * 64 + 4) <= n.value <= 2 * 12 * 16 * 2 * (2 * 64 + 4) + 3 * 4 * 4 + (200 << 20)  # codes, scales, table, a workspace


def test_bad_pages(lib, kv):
    t = np.arange(12, dtype=np.int32)
    assert lib.jg_kvq_set_block_table(kv, t.ctypes.data) == 0
    for bad in (-1, 12, 2 ** 31 - 1):
        t[7] = bad
        assert lib.jg_kvq_set_block_table(kv, t.ctypes.data) == ffi.JG_EINVAL
        assert b"outside the pool" in lib.jg_last_error()


# the arguments behind (dev, kv), all valid; then by place what they may not be
P = 0x1000
CALLS = {
    "write": (dict(layer=1, q_out=P, ldq=512, qkv=P, ldx=768, table=P, table_rows=9, pos=P, seq=P, R=5, H=8),
              dict(layer=[-1, 2], q_out=[P + 2], ldq=[504, 513, -512], qkv=[0, P + 8], ldx=[760, 772, -768], table=[P + 4], table_rows=[0, -1], pos=[0, P + 1], seq=[P + 2], R=[0, -1, 2 ** 31 - 1], H=[4, 0])),
    "decode": (dict(layer=1, out=P, ldo=512, qkv=P, ldx=768, table=P, table_rows=9, pos=P, seq=P, B=5, H=8),
               dict(layer=[-1, 2], out=[0, P + 2], ldo=[504, 513], qkv=[0, P + 8], ldx=[760, 772], table=[P + 4], table_rows=[0, -1], pos=[0, P + 1], seq=[P + 2], B=[0, -1, 65536], H=[4, 0])),
    "attn": (dict(layer=1, out=P, ldo=512, q=P, ldq=512, R=20, pos=P, count=P, first=P, seq=P, B=5, max_count=4, step=1, H=8),
             dict(layer=[-1, 2], out=[0, P + 2], ldo=[504, 513], q=[0, P + 8], ldq=[504, 515], R=[0, -1], pos=[0, P + 1], count=[P + 1], first=[P + 2], seq=[P + 3], B=[0, -1, 65536], max_count=[0, -4, 65], step=[0, -1], H=[4, 0])),
    "read": (dict(layer=1, k=P, v=P, ld=128, R=20, pos=P, count=P, first=P, seq=P, B=5, max_count=4, step=1),
             dict(layer=[-1, 2], k=[0, P + 2], v=[0, P + 8], ld=[120, 129], R=[0, -1], pos=[0, P + 1], count=[P + 1], first=[P + 2], seq=[P + 3], B=[0, -1, 65536], max_count=[0, -4, 65, 2 ** 31 - 1], step=[0, -1])),
}


def launches(lib):
    return C.c_int.in_dll(lib, "fake_launches").value


@pytest.mark.parametrize("name", CALLS)
def test_calls_refuse(lib, dev, kv, name):
    good, bad = CALLS[name]
    fn = getattr(lib, f"jg_kvq_{name}")
    n = launches(lib)
    for arg, values in bad.items():
        for x in values:
            assert fn(dev, kv, *dict(good, **{arg: x}).values()) == ffi.JG_EINVAL, (arg, x)
            assert lib.jg_last_error().startswith(b"kvq_")
    few = {"write": {"R": 4}, "decode": {"B": 4}}.get(name, {"B": 4})  # rows are slots: there are three
    assert fn(dev, kv, *dict(good, seq=0, **few).values()) == ffi.JG_EINVAL
    assert fn(None, kv, *good.values()) == ffi.JG_EINVAL
    assert fn(dev, None, *good.values()) == ffi.JG_EINVAL
    other = C.c_void_p()
    assert lib.jg_device_open(0, C.byref(other)) == 0
    assert fn(other, kv, *good.values()) == ffi.JG_EINVAL  # another device's cache
    assert launches(lib) == n
    for also in ({}, {"seq": 0, **{k: 3 for k in few}}, *([{"q_out": 0, "ldq": 0}, {"table": 0, "table_rows": 0}] if name == "write" else []),
                 *([{"count": 0, "first": 0}] if "count" in good else [])):
        assert fn(dev, kv, *dict(good, **also).values()) == 0, lib.jg_last_error()
    assert launches(lib) > n


def test_nothing_is_made_or_moved_inside_a_capture(lib, dev, kv):
    h, g = C.c_void_p(), C.c_void_p()
    assert lib.jg_graph_begin(dev) == 0
    assert lib.jg_kvq_create(dev, C.byref(desc()), 0, C.byref(h)) == ffi.JG_EINVAL
    assert lib.jg_kvq_set_block_table(kv, np.zeros(12, np.int32).ctypes.data) == ffi.JG_EINVAL
    for name, (good, _) in CALLS.items():
        assert getattr(lib, f"jg_kvq_{name}")(dev, kv, *good.values()) == 0, lib.jg_last_error()
    assert lib.jg_graph_end(dev, C.byref(g)) == 0


# ------------------------------------------------------------------------------------------------ the Python class
class KvqRecorder(Recorder):
    def call(self, name, *args):
        if name == "jg_kvq_create":
            args[-1]._obj.value = self._handle()
        super().call(name, *args)


@pytest.fixture
def rec(monkeypatch):
    from tests import fake_ffi
    monkeypatch.setattr(fake_ffi, "Recorder", KvqRecorder)
    with fake_ffi.recording() as r:
        yield r


def test_class_refuses(rec):
    from denograd_b200.device import Device, Tensor
    from denograd_b200.kvquant import QuantKVCache
    dev = Device["CUDA"]
    with pytest.raises(ValueError, match="dtype"):
        QuantKVCache(dev, 1, 8, 2, 64, 100, 3, dtype="int4")
    kv = QuantKVCache(dev, 1, 8, 2, 64, 100, 3, page_size=16)
    half, ints = (lambda *s: Tensor.empty(s, "float16")), (lambda n: Tensor.empty((n,), "int32"))
    with pytest.raises(ValueError, match="block table"):
        kv.set_block_table(np.zeros((3, 6), np.int32))
    kv.set_block_table(np.zeros((3, 7), np.int32))
    for make in (lambda: kv.write(0, half(3, 760), ints(3)), lambda: kv.write(0, half(3, 768), ints(2)), lambda: kv.write(0, half(3, 768), ints(3), seq=ints(2)),
                 lambda: kv.write(0, half(3, 768), ints(3), q_out=half(2, 512)), lambda: kv.write(0, half(3, 768), ints(3), q_out=half(3, 504)),
                 lambda: kv.write(0, half(3, 768), ints(3), freqs_cis=half(9, 64, 2)), lambda: kv.decode(0, half(3, 768), ints(2)),
                 lambda: kv.decode(0, half(3, 768), ints(3), out=half(2, 512)), lambda: kv.attend(0, half(7, 512), ints(2)),
                 lambda: kv.attend(0, half(8, 512), ints(2), count=ints(2)), lambda: kv.attend(0, half(8, 512), ints(2), count=ints(1), max_count=4),
                 lambda: kv.attend(0, half(8, 512), ints(2), out=half(7, 512)), lambda: kv.read(0, ints(2)), lambda: kv.read(0, ints(2), k=half(4, 128)),
                 lambda: kv.read(0, ints(2), k=half(4, 128), v=half(3, 128)), lambda: kv.read(0, ints(2), k=half(4, 128), v=half(4, 136))):
        with pytest.raises(ValueError):
            make()
    for make in (lambda: kv.write(0, Tensor.empty((3, 768), "float32"), ints(3)), lambda: kv.write(0, half(3, 768), Tensor.empty((3,), "float32")),
                 lambda: kv.attend(0, half(8, 512), ints(2), seq=half(2))):
        with pytest.raises(TypeError):
            make()
    assert not [c for c in rec.calls if c[0].startswith("jg_kvq_") and c[0] not in ("jg_kvq_create", "jg_kvq_set_block_table")]
    q = half(8, 520)
    kv.attend(0, q, ints(2))
    assert rec.calls[-1][0] == "jg_kvq_attn" and rec.calls[-1][5:9] == (512, q.ptr, 520, 8) and rec.calls[-1][-4:] == (2, 4, 2, 8)


def test_class_refuses_tensors_of_another_device(rec):
    from denograd_b200.device import CUDA, Device, Tensor
    from denograd_b200.kvquant import QuantKVCache
    dev, other = Device["CUDA"], CUDA("CUDA:1")
    kv = QuantKVCache(dev, 1, 8, 2, 64, 100, 3, page_size=16)
    t = lambda where, *s: Tensor.empty(s, "float16", where)  # noqa: E731
    i = lambda where, n: Tensor.empty((n,), "int32", where)  # noqa: E731
    n = len(rec.calls)
    for make in (lambda: kv.write(0, t(other, 3, 768), i(dev, 3)), lambda: kv.write(0, t(dev, 3, 768), i(other, 3)), lambda: kv.decode(0, t(dev, 3, 768), i(dev, 3), out=t(other, 3, 512)),
                 lambda: kv.decode(0, t(dev, 3, 768), i(dev, 3), freqs_cis=t(other, 9, 32, 2)), lambda: kv.attend(0, t(dev, 6, 512), i(dev, 3), seq=i(other, 3)),
                 lambda: kv.read(0, i(dev, 2), max_count=2, k=t(other, 4, 128), v=t(dev, 4, 128))):
        with pytest.raises(ValueError, match="CUDA:1"):
            make()
    assert not [c for c in rec.calls[n:] if c[0].startswith("jg_kvq_")]


@pytest.mark.parametrize("fused", [True, False])
def test_a_model_uses_it(rec, fused, monkeypatch):
    from denograd_b200.llama3 import Llama3
    with pytest.raises(ValueError, match="kv_dtype"):
        Llama3(size="1B", args=TINY, kv_dtype="int4")
    llm = Llama3(size="1B", args=TINY, kv_dtype="fp8", max_context=64, max_batch=2, tied_output=False, temperature=0, fused=fused)
    m = llm.model
    L = len(m.layers)
    assert not [c for c in rec.calls if c[0] == "jg_kvcache_create"]
    n = len(rec.calls)
    m._step(m._workspace(2))
    names = [c[0] for c in rec.calls[n:]]
    assert names.count("jg_kvq_decode") == L and not [x for x in names if x.startswith(("jg_attn", "jg_rope", "jg_step"))]
    if fused:
        n = len(rec.calls)
        m._forward_rows(np.zeros((2, 12), np.int32), 3, last=True)
        names = [c[0] for c in rec.calls[n:]]
        assert names.count("jg_kvq_write") == names.count("jg_kvq_attn") == L and not [x for x in names if x.startswith(("jg_attn", "jg_rope"))]
    m.new_cache()
    assert [c[0] for c in rec.calls].count("jg_kvq_create") == 2 and [c[0] for c in rec.calls].count("jg_kvq_destroy") == 1
    del llm, m


def test_other_models_refuse_it():
    from denograd_b200 import registry
    with pytest.raises(registry.UnsupportedDtype, match="kv_dtype"):
        registry._hybrid({"architecture": "Matulorn"}, "", None, 8, 1, kv_dtype="int8")


# ------------------------------------------------------------------------------------------------ the reference of the GPU tests
def test_known_codes():
    x = np.array([[127, -63.5, 0.5, 1.5, 0, 126.5, -0.25, 2.5]], np.float16)
    c, s = R.codes(x, "int8")
    assert s[0, 0] == 1 and c[0].tolist() == [127, -64, 0, 2, 0, 126, 0, 2]
    c, s = R.codes(x * np.float16(1.0078125), "int8")  # 128 / 127 is rounded up to 9/8
    assert s[0, 0] == 1.125 and c[0, 0] == 114
    assert R.codes(np.float16([[2.0 ** -24, 0]]), "int8")[1][0, 0] == 2.0 ** -24
    assert R.codes(np.float16([[65504, 1]]), "int8")[1][0, 0] == 576 and R.codes(np.float16([[65504, 1]]), "int8")[0][0, 0] == 113
    c, s = R.codes(np.float16([[448, 17, 19, 0.001953125, 0.0009765625, -300]]), "fp8")
    assert s[0, 0] == 1 and c[0].tolist() == [448, 16, 20, 0.001953125, 0, -288]
    assert R.codes(np.float16([[449, 0]]), "fp8")[1][0, 0] == 2 and R.codes(np.float16([[1e-3, 0]]), "fp8")[1][0, 0] == 2.0 ** -15
    assert (R.codes(np.float16([[65504, -63000]]), "fp8")[0] * 256).tolist() == [[61440, -61440]]
    k, v = R.stored(np.float16([[1, 2], [3, np.inf]]), np.float16([[5, 6], [7, 8]]), "int8")
    assert np.isnan(k[1]).all() and np.isnan(v[1]).all() and v[0, 1] == 5.9921875  # 118 x 13/256
