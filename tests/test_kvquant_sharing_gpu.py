"""Sums of the 8-bit cache's attention that many CTAs share, on the GPU: contexts whose items lie so that one CTA has the last piece of an item, a group by
itself, and the first piece of the next one (tests/kvquant_line_walk.cpp lists them).  Every call gives the same bits, whatever ran before it.
And rows that are read back and then taken as weights."""
import numpy as np
import pytest

from denograd_b200.device import Tensor
from tests.test_kvquant_gpu import Cache, ints

pytestmark = pytest.mark.gpu


# (query heads, kv heads, head dim, contexts, new positions of each): new = 1 is a decode, more are columns of short chunks
@pytest.mark.parametrize("H,G,hd,ahead,new,fmt", [(8, 8, 64, [20724, 7137, 3324, 4400], 1, "int8"), (16, 8, 128, [16527, 12298], 1, "fp8"), (5, 5, 64, [131000], 1, "int8"),
                                                  (32, 4, 64, [8000] * 7, 1, "int8"), (16, 8, 64, [20000, 15000], 1, "fp8"), (32, 8, 64, [59054 - 3, 7135 - 3], 3, "int8")])
def test_neighbouring_items_of_many_pieces(dev, H, G, hd, ahead, new, fmt):
    rng = np.random.default_rng(31)
    B = len(ahead)
    c = Cache(dev, H, G, hd, fmt, 64, max(ahead) + new, B, rng)
    other = Cache(dev, 8, 2, 64, "int8", 16, 1500, 2, rng)
    c.fill(ahead)
    other.fill([1400, 300])
    pos = np.array(ahead)
    pt, po = ints(dev, pos), ints(dev, [1400, 300])
    xo, qo, out_o = Tensor(other.rows(2), device=dev), Tensor(other.rows(80), device=dev), Tensor.zeros((80, 8 * 64), "float16", dev)
    x = c.rows(B * new)
    xt = Tensor(x, device=dev)
    rows_pos, rows_seq = (pos[None] + np.arange(new)[:, None]).reshape(-1), np.tile(np.arange(B), new)
    q = c.note(x, rows_pos, rows_seq)
    if new > 1:
        c.kv.write(0, xt, ints(dev, rows_pos), seq=ints(dev, rows_seq))
    poison = np.full((B * new, H * hd), 7, np.float16)
    outs = [Tensor(poison, device=dev) for _ in range(8)]
    first = None
    for turn in range(25):
        for i, out in enumerate(outs):
            if new == 1:
                c.kv.decode(0, xt, pt, out=out)
            else:
                c.kv.attend(0, xt, pt, out=out)
            if i % 2:  # another cache's calls in between, of either kernel
                other.kv.decode(0, xo, po)
            if i % 4 == 3:
                other.kv.attend(0, qo, ints(dev, [0, 100]), out=out_o)
        for out in outs:
            got = out.numpy()
            if first is None:
                first = got.copy()
                c.check(first, q, rows_pos, rows_seq)
            np.testing.assert_array_equal(got.view(np.uint16), first.view(np.uint16))
            out.assign(poison)
    c.check_stored()
    c.close()
    other.close()


@pytest.mark.parametrize("M", [1, 4, 16, 200])
def test_rows_read_back_are_the_next_projection(dev, M):
    """q.K^T as a projection whose weights are the K rows of the call in front of it: those of this turn, not of the last one."""
    rng = np.random.default_rng(33)
    hd, n = 128, 4096
    c = Cache(dev, 1, 1, hd, "int8", 64, n, 2, rng)
    c.fill([n, n])
    q = rng.standard_normal((M, hd)).astype(np.float16)
    qt, zero = Tensor(q, device=dev), ints(dev, [0])
    k, v = (Tensor.zeros((n, hd), "float16", dev) for _ in range(2))
    slots = [ints(dev, [0]), ints(dev, [1])]
    outs = [Tensor.empty((M, n), "float16", dev) for _ in range(8)]
    dev.synchronize()
    for i, out in enumerate(outs):
        c.kv.read(0, zero, seq=slots[i & 1], max_count=n, k=k, v=v)
        dev.call("jg_linear", out.ptr, qt.ptr, k.ptr, 0, 0, M, n, hd)
    for i, out in enumerate(outs):
        held = c.k[i & 1, :, 0].astype(np.float64)
        want, size = q.astype(np.float64) @ held.T, np.abs(q.astype(np.float64)) @ np.abs(held).T
        # rounded to fp16 once, behind a sum of 128 exact products in 32 bits
        assert (np.abs(out.numpy() - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + hd * 2.0 ** -23 * size).all(), i
    c.close()
