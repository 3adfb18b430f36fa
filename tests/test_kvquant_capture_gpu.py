"""Calls of the 8-bit KV cache that are captured before any of them has run on a handle, and replayed."""
import numpy as np
import pytest

from denograd_b200.device import CUDA, CUDAGraph, Tensor
from denograd_b200.kvquant import QuantKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,hd", [("int8", 64), ("fp8", 64), ("int8", 128), ("fp8", 128)])
def test_first_calls_are_captured(fmt, hd):
    H, G, n, B = 8, 2, 300, 2
    rng = np.random.default_rng(51)
    rows, new = rng.standard_normal((B * n, (H + 2 * G) * hd)).astype(np.float16), rng.standard_normal((B, (H + 2 * G) * hd)).astype(np.float16)

    def run(captured: bool) -> list[np.ndarray]:
        own = CUDA("CUDA").init()
        kv = QuantKVCache(own, 1, H, G, hd, n + 1, B, page_size=32, dtype=fmt)
        ints = lambda x: Tensor(np.asarray(x, np.int32), device=own)  # noqa: E731
        half = lambda *s: Tensor.zeros(s, "float16", own)  # noqa: E731
        x, y = Tensor(rows, device=own), Tensor(new, device=own)
        at, slot, zero, last, first = ints(np.tile(np.arange(n), B)), ints(np.repeat(np.arange(B), n)), ints([0, 0]), ints([n, n]), ints([0, n])
        near = ints([n - 2, n - 2])
        many, few, one, k, v = half(B * n, H * hd), half(2 * B, H * hd), half(B, H * hd), half(B * n, G * hd), half(B * n, G * hd)

        def calls():
            kv.write(0, x, at, seq=slot)
            kv.attend(0, x, zero, first=first, max_count=n, out=many)
            kv.attend(0, x.view_rows(0, 2 * B), near, out=few)
            kv.decode(0, y, last, out=one)
            kv.read(0, zero, first=first, max_count=n, k=k, v=v)

        own.synchronize()
        if captured:
            g = CUDAGraph(own)
            with g:
                calls()
            own.synchronize()
            assert not many.numpy().any()
            for _ in range(3):
                g.launch()
        else:
            calls()
        own.synchronize()
        got = [t.numpy().copy() for t in (many, few, one, k, v)]
        kv.close()
        return got

    a, b = run(True), run(False)
    for p, q in zip(a, b):
        assert p.any() and np.isfinite(p).all()
        np.testing.assert_array_equal(p.view(np.uint16), q.view(np.uint16))
