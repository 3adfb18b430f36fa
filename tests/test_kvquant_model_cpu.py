"""Llama models with an 8-bit KV cache under tensor parallelism, without a GPU: which calls each rank makes.  And what `write` refuses of its output."""
import ctypes as C

import numpy as np
import pytest

from denograd_b200 import ffi
from tests.golden.gen_golden import TINY
from tests.test_kvquant_cpu import KvqRecorder


class Descs(KvqRecorder):
    descs: list = []

    def call(self, name, *args):
        if name == "jg_kvq_create":
            d = args[1]._obj
            Descs.descs.append({f: getattr(d, f) for f, _ in ffi.KvDesc._fields_})
        super().call(name, *args)


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8"])
@pytest.mark.parametrize("rank", [0, 1])
def test_a_rank_of_two(monkeypatch, kv_dtype, rank):
    """Each rank has the cache of its own heads; everything else is what the fp16 cache's model calls."""
    from tests import fake_ffi
    monkeypatch.setattr(fake_ffi, "Recorder", Descs)
    monkeypatch.setattr(Descs, "descs", [])
    with fake_ffi.recording() as rec:
        from denograd_b200.device import Device
        from denograd_b200.llama3 import Llama3
        from denograd_b200.multi import TensorParallel
        tp = TensorParallel.__new__(TensorParallel)
        tp.dev, tp.rank, tp.world, tp.handle = Device["CUDA"], rank, 2, C.c_void_p(0x77)
        tp.peer_capacity = tp.twoshot_capacity = tp._partial_ptr = 0
        made = {}
        for kv in ("float16", kv_dtype):
            llm = Llama3(size="1B", args=TINY, kv_dtype=kv, max_context=64, max_batch=3, tied_output=True, temperature=0, tp=tp)
            n = len(rec.calls)
            llm.model._step(llm.model._workspace(3))
            llm.model._forward_rows(np.zeros((2, 12), np.int32), 3, last=True)
            made[kv] = rec.kernels(n)
            llm.model.new_cache()
        d = Descs.descs[0]
        assert len(Descs.descs) == 2 and (d["n_heads"], d["n_kv_heads"], d["head_dim"], d["n_layers"], d["max_batch"]) == (2, 1, 64, 2, 3)
        decode, write, attend = ([c for c in made[kv_dtype] if c[0] == "jg_kvq_" + x] for x in ("decode", "write", "attn"))
        assert len(decode) == len(write) == len(attend) == TINY["n_layers"]
        assert all(c[-1] == 2 for c in decode + write + attend)  # this rank's query heads
        assert all(c[-2] == 3 for c in decode) and all(c[-2] == 24 for c in write) and all(c[-4:-1] == (2, 12, 2) for c in attend)
        attention = ("jg_kvq_", "jg_attn", "jg_rope")
        assert [c[0] for c in made[kv_dtype] if not c[0].startswith(attention)] == [c[0] for c in made["float16"] if not c[0].startswith(attention)]
        del llm, tp


def test_rotated_queries_in_place_have_the_same_rows(monkeypatch):
    from tests import fake_ffi
    monkeypatch.setattr(fake_ffi, "Recorder", KvqRecorder)
    with fake_ffi.recording() as rec:
        from denograd_b200.device import Device, Tensor
        from denograd_b200.kvquant import QuantKVCache
        kv = QuantKVCache(Device["CUDA"], 1, 8, 2, 64, 100, 3, page_size=16)
        x, pos = Tensor.empty((3, 768), "float16"), Tensor.empty((3,), "int32")
        kv.write(0, x, pos, q_out=x)
        n = len(rec.calls)
        with pytest.raises(ValueError, match="rows of 512 and not 768"):  # row 1 of the result would lie in row 0's K
            kv.write(0, x, pos, q_out=Tensor(x.buf, shape=(4, 512)))
        assert len(rec.calls) == n
        one = x.view_rows(0, 1)
        kv.write(0, one, pos, q_out=Tensor(one.buf, shape=(1, 512)))  # a row by itself has no other
        del kv
