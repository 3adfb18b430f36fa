"""Attention over the 8-bit KV cache on the GPU at contexts of 2^24 positions, where the line of work that is cut over the CTAs has more units than 32-bit
products hold.  A few pages stand for whole stretches of the context."""
import numpy as np
import pytest

from denograd_b200.device import Tensor
from denograd_b200.kvquant import QuantKVCache
from tests import kvquant_ref as R
from tests.test_kvquant_gpu import ints

pytestmark = pytest.mark.gpu
G, HD, PAGE, PARTS, CONTEXT = 8, 64, 64, 64, 1 << 24


class Stretches:
    """Page p of 64 stands for the p-th 64th of a slot's context.  Keys are the same in each page, values of page p are 1 in column p and 0 elsewhere: column
    p of a result is the share of the context that page p stands for, so a stretch that is lost or counted twice shows in its columns."""

    def __init__(self, dev, H, seed):
        rng = np.random.default_rng(seed)
        self.dev, self.H = dev, H
        self.kv = QuantKVCache(dev, 1, H, G, HD, CONTEXT, 1, page_size=PAGE, dtype="int8", n_pages=PARTS)
        n = self.kv.max_pages_per_seq
        self.of = (np.arange(n) * PARTS // n).astype(np.int32)
        self.keys = rng.standard_normal((PAGE, G, HD)).astype(np.float16)
        x = np.zeros((PARTS, PAGE, H + 2 * G, HD), np.float16)
        x[:, :, H:H + G] = self.keys
        for p in range(PARTS):
            x[p, :, H + G:, p] = 1
        self.x = x
        self.kv.set_block_table((np.arange(n, dtype=np.int32) % PARTS)[None])  # positions 0 .. are the pages themselves, while they are filled
        m = PARTS * PAGE
        self.kv.write(0, Tensor(x.reshape(m, -1), device=dev), ints(dev, np.arange(m)), seq=ints(dev, np.zeros(m)))
        dev.synchronize()
        self.kv.set_block_table(self.of[None])
        k, v = R.stored(self.keys, x[0, :, H + G:], "int8")
        self.k, self.one = k.astype(np.float64), float(v[0, 0, 0])

    def check(self, got, q, last, tol):
        """A row [H, hd] of results of queries q over positions 0 .. last."""
        w = np.exp(np.einsum("grd,tgd->grt", q.astype(np.float64).reshape(G, -1, HD), self.k) / np.sqrt(HD)).reshape(self.H, PAGE)
        full, rest = (last + 1) // PAGE, (last + 1) % PAGE
        want = np.bincount(self.of[:full], minlength=PARTS)[None] * w.sum(-1, keepdims=True)
        if rest:
            want[:, self.of[full]] += w[:, :rest].sum(-1)
        want *= self.one / want.sum(-1, keepdims=True)
        off = np.abs(got.astype(np.float64) - want)
        assert (off <= tol * want).all(), f"off by {(off / (tol * want)).max():.2f} of what is allowed"


# How far a column may be off, relative to it: its rounding to fp16 and that of its weights (2^-11 each), what the weights' errors leave of the sum they are
# divided by (2^-11 in all), and the roundings of the 32-bit sums.  A column grows within its own 64th of the context only, by products of 16 positions: 16
# roundings of 2^-23 at most for each, and a lane's sum of weights by a few terms a tile, 2^-24 each.
#   few queries: a warp sees a quarter of 2^18 positions of a 64th, 4096 tiles; sums of two weights a tile, 2^18 * 8 units over 296 CTAs at least: 7085 tiles
#   chunks: 2^18 positions, 16384 products; sums of 32 weights a tile in each of four parts, 2^23 / 148 = 56 700 tiles
FEW = 3 * 2.0 ** -11 + 4096 * 16 * 2.0 ** -23 + 7085 * 2 * 2.0 ** -24
CHUNK = 3 * 2.0 ** -11 + 16384 * 16 * 2.0 ** -23 + 56700 * 32 * 2.0 ** -24


def test_decode(dev):
    c = Stretches(dev, 16, 41)
    rng = np.random.default_rng(42)
    for pos in (CONTEXT - 6, CONTEXT - 1, (1 << 23) + 777):
        x = c.x[c.of[pos // PAGE], pos % PAGE].copy()[None]  # the new token is what its row of the page holds already
        x[:, :c.H] = rng.standard_normal((1, c.H, HD))
        out = Tensor(np.full((1, c.H * HD), 7, np.float16), device=dev)
        c.kv.decode(0, Tensor(x.reshape(1, -1), device=dev), ints(dev, [pos]), out=out)
        c.check(out.numpy().reshape(c.H, HD), x[0, :c.H], pos, FEW)
    c.kv.close()


# columns of a short chunk: 16; rows of a long one: eight items of 256 of each kv head, looked at by one warp (up to 32 items) or by all threads
@pytest.mark.parametrize("H,new,most,tol", [(64, 2, 2, FEW), (64, 256, 256, CHUNK), (64, 256, 1200, CHUNK)])
def test_attend(dev, H, new, most, tol):
    c = Stretches(dev, H, 43)
    q = np.random.default_rng(44).standard_normal((new, H, HD)).astype(np.float16)
    out = Tensor(np.full((new, H * HD), 7, np.float16), device=dev)
    ahead = CONTEXT - new
    c.kv.attend(0, Tensor(q.reshape(new, -1), device=dev), ints(dev, [ahead]), count=ints(dev, [new]), first=ints(dev, [0]), max_count=most, out=out)
    got = out.numpy().reshape(new, H, HD)
    for i in sorted({0, 1, new // 3, new // 2, new - 2, new - 1}):
        c.check(got[i], q[i], ahead + i, tol)
    c.kv.close()
