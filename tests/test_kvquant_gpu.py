"""The 8-bit KV cache on the GPU against kvquant_ref.py: storing, reading back, attention of single tokens and of chunks, and a run of them
together.  What is stored is compared to the bit; attention with the errors that its roundings allow."""
import numpy as np
import pytest

from denograd_b200 import CUDAGraph
from denograd_b200.device import Tensor
from denograd_b200.kvquant import QuantKVCache
from tests import kvquant_ref as R

pytestmark = pytest.mark.gpu
SHAPES = [(8, 8, 64), (8, 4, 128), (6, 2, 64), (16, 4, 128), (10, 2, 64), (6, 1, 128), (7, 1, 64), (16, 2, 128), (8, 1, 64)]


def ints(dev, x):
    return Tensor(np.asarray(x, np.int32), device=dev)


def table(n, hd):
    angle = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    return np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float16)


class Cache:
    """A QuantKVCache beside what it should hold: k, v [slot, position, G, hd]."""

    def __init__(self, dev, H, G, hd, fmt, page, max_ctx, slots, rng, layers=1):
        self.dev, self.H, self.G, self.hd, self.fmt, self.rng = dev, H, G, hd, fmt, rng
        self.kv = QuantKVCache(dev, layers, H, G, hd, max_ctx, slots, page_size=page, dtype=fmt)
        self.kv.set_block_table(rng.permutation(self.kv.n_pages).astype(np.int32).reshape(slots, -1))
        self.n = self.kv.max_pages_per_seq * page
        self.k, self.v = (np.zeros((slots, self.n, G, hd), np.float16) for _ in range(2))

    def split(self, x):
        x = x.reshape(len(x), -1)[:, :(self.H + 2 * self.G) * self.hd].reshape(len(x), self.H + 2 * self.G, self.hd)
        return x[:, :self.H], x[:, self.H:self.H + self.G], x[:, self.H + self.G:]

    def rows(self, n, scale=1.0):
        x = self.rng.standard_normal((n, self.H + 2 * self.G, self.hd)) * scale
        x[:, self.H:self.H + self.G] *= 1 + 4 * (self.rng.random((1, self.G, self.hd)) < 0.05)  # keys with channels that stand out
        return x.astype(np.float16).reshape(n, -1)

    def note(self, x, pos, seq, cs=None):
        """Remembers rows as stored; their rotated queries."""
        q, k, v = self.split(x)
        if cs is not None:
            q, k = R.rotate(q, cs, pos), R.rotate(k, cs, pos)
        self.k[seq, pos], self.v[seq, pos] = R.stored(k, v, self.fmt)
        return q

    def fill(self, lens):
        """Positions 0 .. lens[s] - 1 of every slot, as they are (no rotation)."""
        pos = np.concatenate([np.arange(n) for n in lens])
        seq = np.repeat(np.arange(len(lens)), lens)
        if len(pos):
            x = self.rows(len(pos))
            self.kv.write(0, Tensor(x, device=self.dev), ints(self.dev, pos), seq=ints(self.dev, seq))
            self.note(x, pos, seq)

    def check_stored(self):
        slots = len(self.k)
        k, v = self.kv.read(0, ints(self.dev, np.zeros(slots)), max_count=self.n, first=ints(self.dev, np.arange(slots) * self.n), rows=slots * self.n)
        same(k.numpy().reshape(self.k.shape), self.k, "K")
        same(v.numpy().reshape(self.v.shape), self.v, "V")

    def check(self, got, q, pos, seq, what=""):
        """Rows of attention `got` [n, H * hd] of queries q at positions pos of slots seq."""
        for i, (t, s) in enumerate(zip(pos, seq)):
            want, tol = R.attention(q[i], self.k[s], self.v[s], int(t))
            off = np.abs(got[i].astype(np.float64) - want)
            assert (off <= tol).all(), f"{what} row {i} (position {t} of slot {s}): off by {(off / tol).max():.2f} of what is allowed"

    def close(self):
        self.kv.close()


def same(got, want, what):
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} differ, first at {np.argwhere(bad)[0]}: {got[bad][0]!r}, not {want[bad][0]!r}"


# ------------------------------------------------------------------------------------------------ storing and reading back
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd", SHAPES)
def test_store(dev, H, G, hd, fmt):
    rng = np.random.default_rng(H * hd + G)
    for page, n in ((16, 1), (32, 7), (64, 130)):
        c = Cache(dev, H, G, hd, fmt, page, 200, 3, rng, layers=2)
        cs = table(c.n, hd)
        at = rng.permutation(3 * c.n)[:n]
        pos, seq = at % c.n, at // c.n
        pad = 24  # columns behind a row, and rows of q_out that are longer than Q
        x = np.concatenate([c.rows(n), rng.standard_normal((n, pad)).astype(np.float16)], 1)
        xt, q_out = Tensor(x, device=dev), Tensor(np.full((n + 1, H * hd + 8), 7, np.float16), device=dev)
        c.kv.write(0, xt, ints(dev, pos), seq=ints(dev, seq), freqs_cis=Tensor(cs, device=dev), q_out=q_out)
        q = c.note(x, pos, seq, cs)
        got = q_out.numpy()
        same(got[:n, :H * hd], q.reshape(n, -1), "Q")
        assert (got[:n, H * hd:] == 7).all() and (got[n:] == 7).all()
        same(xt.numpy(), x, "the input")
        c.check_stored()
        k, v = c.kv.read(1, ints(dev, [0, 0, 0]), max_count=c.n, rows=3 * c.n)
        assert not k.numpy().any() and not v.numpy().any()  # the other layer
        # in place, without an angle, without Q
        c.kv.write(0, xt, ints(dev, pos), seq=ints(dev, seq), freqs_cis=Tensor(cs, device=dev), q_out=xt)
        x[:, :H * hd] = q.reshape(n, -1)
        same(xt.numpy(), x, "Q in place")
        c.kv.write(0, xt, ints(dev, pos), seq=ints(dev, seq))
        c.note(x, pos, seq)
        c.check_stored()
        c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_store_values_of_every_size(dev, fmt):
    """Rows around every border of the scales: powers of two, multiples of 127 and 448, the smallest numbers, the largest, ties, zeros."""
    rng = np.random.default_rng(5)
    tops = np.array([int(b) for b in range(1, 0x7C00, 37)] + [1, 2, 3, 0x3FF, 0x400, 0x7BFF, 0x7BFE, 0x7BF0], np.uint16).view(np.float16)
    exact = np.array([m * 127 * 2.0 ** e for m in range(8, 16) for e in range(-28, 6)] + [448 * 2.0 ** e for e in range(-30, 8)])
    tops = np.concatenate([tops, exact[exact == exact.astype(np.float16)].astype(np.float16)])
    n = len(tops)
    c = Cache(dev, 1, 1, 64, fmt, 64, n, 1, rng)
    x = np.zeros((n, 3, 64), np.float16)
    share = rng.choice([0, 0.5 / 127, 1 / 127, 1.5 / 127, 63.5 / 127, 0.5, 0.25, 1e-3, 1e-5, 17 / 16 / 2, 1], (n, 2, 64)) * rng.choice([-1, 1], (n, 2, 64))
    x[:, 1:] = (share * tops[:, None, None].astype(np.float64)).astype(np.float16)
    x[:, 1:, 0] = tops[:, None]
    x[5, 1:] = 0
    x[6, 1:] = -0.0
    x = x.reshape(n, -1)
    c.kv.write(0, Tensor(x, device=dev), ints(dev, np.arange(n)), seq=ints(dev, np.zeros(n)))
    c.note(x, np.arange(n), np.zeros(n, int))
    assert np.isfinite(c.k).all()
    c.check_stored()
    c.close()


def test_store_skips_what_is_outside(dev):
    rng = np.random.default_rng(6)
    c = Cache(dev, 4, 2, 64, "int8", 16, 48, 2, rng)
    pos, seq = np.array([-1, 48, 40, 3, 0, 2 ** 31 - 1, 41]), np.array([0, 0, 0, 2, -1, 1, 1])
    x = c.rows(7)
    q_out = Tensor(np.full((7, 4 * 64), 7, np.float16), device=dev)
    c.kv.write(0, Tensor(x, device=dev), ints(dev, pos), seq=ints(dev, seq), freqs_cis=Tensor(table(41, 64), device=dev), q_out=q_out)
    q = c.note(x[2:3], pos[2:3], seq[2:3], table(48, 64))  # the only row inside the cache and the table
    c.check_stored()
    got = q_out.numpy()
    same(got[2], q.reshape(-1), "Q")
    assert (np.delete(got, 2, 0) == 7).all()
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_read(dev, fmt):
    rng = np.random.default_rng(7)
    c = Cache(dev, 4, 2, 128, fmt, 32, 100, 4, rng)
    c.fill([100, 0, 57, 1])
    pos, count, seq, first = [90, 0, -2, 55, 0], [20, 0, 5, 400, 3], [0, 1, 2, 2, 9], [3, 0, 40, 60, 30]
    k, v = (Tensor(np.full((70, 2 * 128 + 8), 7, np.float16), device=dev) for _ in range(2))
    c.kv.read(0, ints(dev, pos), count=ints(dev, count), first=ints(dev, first), seq=ints(dev, seq), max_count=21, k=k, v=v)
    for got, held in ((k, c.k), (v, c.v)):
        want = np.full((70, 2 * 128 + 8), 7, np.float16)
        for p, n, s, f in zip(pos, count, seq, first):
            for i in range(min(n, 21)):
                if f + i < 70:
                    inside = s < 4 and 0 <= p + i < c.n
                    want[f + i, :256] = held[s, p + i].reshape(-1) if inside else 0
        same(got.numpy(), want, "rows")
    c.close()


# ------------------------------------------------------------------------------------------------ one new token a row
def test_read_many_stretches(dev):
    """More stretches than a launch has CTAs for at their full length: each goes over its rows in turns."""
    rng = np.random.default_rng(26)
    c = Cache(dev, 4, 2, 64, "int8", 16, 1400, 3, rng)
    c.fill([1400, 900, 50])
    B, most = 300, 1300
    pos, seq, count = rng.integers(0, 60, B), rng.integers(0, 3, B), np.where(rng.random(B) < 0.2, most, rng.integers(0, 40, B))
    first = np.concatenate([[0], np.cumsum(count)[:-1]])
    k, v = c.kv.read(0, ints(dev, pos), count=ints(dev, count), first=ints(dev, first), seq=ints(dev, seq), max_count=most, rows=int(count.sum()) + 1)
    k, v = k.numpy().reshape(-1, 2, 64), v.numpy().reshape(-1, 2, 64)
    for b in range(B):
        at = slice(first[b], first[b] + count[b])
        same(k[at], c.k[seq[b], pos[b]:pos[b] + count[b]], f"K of {b}")
        same(v[at], c.v[seq[b], pos[b]:pos[b] + count[b]], f"V of {b}")
    assert not k[-1].any() and not v[-1].any()
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd", SHAPES)
def test_decode(dev, H, G, hd, fmt):
    rng = np.random.default_rng(H + G + hd)
    for page, lens in ((64, [547]), (16, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 500]), (32, [1021, 3]), (64, [0])):
        B = len(lens)
        c = Cache(dev, H, G, hd, fmt, page, max(lens) + 1, B + 1, rng)
        cs = table(c.n, hd)
        seq = rng.permutation(B + 1)[:B]
        held = np.zeros(B + 1, int)
        held[seq] = lens
        c.fill(held)
        x = c.rows(B)
        xt, out = Tensor(x, device=dev), Tensor(np.full((B + 1, H * hd + 8), 7, np.float16), device=dev)
        for _ in range(2):  # again: the same token at the same place
            c.kv.decode(0, xt, ints(dev, lens), freqs_cis=Tensor(cs, device=dev), seq=ints(dev, seq), out=out)
            got = out.numpy()
        q = c.note(x, np.array(lens), seq, cs)
        c.check(got[:, :H * hd], q, lens, seq, f"page {page}")
        assert (got[:B, H * hd:] == 7).all() and (got[B] == 7).all()
        same(xt.numpy(), x, "the input")
        c.check_stored()
        c.close()


@pytest.mark.parametrize("H,G,hd,B,fmt", [(32, 8, 128, 3, "int8"), (8, 1, 64, 40, "fp8"), (16, 8, 64, 70, "int8"), (4, 1, 128, 1, "fp8")])
def test_decode_long_and_many(dev, H, G, hd, B, fmt):
    rng = np.random.default_rng(B)
    lens = np.minimum((np.exp(rng.uniform(0, np.log(6000), B))).astype(int), 200000 // (B * G))
    lens[0] = 30011 // (G if G < 8 else 4)
    c = Cache(dev, H, G, hd, fmt, 64, int(lens.max()) + 1, B, rng)
    c.fill(lens)
    x = c.rows(B)
    out = c.kv.decode(0, Tensor(x, device=dev), ints(dev, lens))  # row b is slot b, nothing is rotated
    q = c.note(x, lens, np.arange(B))
    c.check(out.numpy(), q, lens, np.arange(B))
    c.check_stored()
    c.close()


def test_decode_rows_outside(dev):
    rng = np.random.default_rng(8)
    c = Cache(dev, 8, 2, 64, "int8", 16, 64, 4, rng)
    c.fill([20, 50, 30, 7])
    pos, seq = np.array([-1, 64, 50, 5, 2, 45]), np.array([0, 1, 1, 4, -1, 2])
    x = c.rows(6)
    out = Tensor(np.full((6, 8 * 64), 7, np.float16), device=dev)
    cs = table(45, 64)
    c.kv.decode(0, Tensor(x, device=dev), ints(dev, pos), freqs_cis=Tensor(cs, device=dev), seq=ints(dev, seq), out=out)
    assert not out.numpy().any()  # 50 and 45 lie behind the table
    c.check_stored()
    c.kv.decode(0, Tensor(x, device=dev), ints(dev, pos), freqs_cis=Tensor(table(64, 64), device=dev), seq=ints(dev, seq), out=out)
    live = [2, 5]
    q = c.note(x[live], pos[live], seq[live], table(64, 64))
    got = out.numpy()
    c.check(got[live], q, pos[live], seq[live])
    assert not np.delete(got, live, 0).any()
    c.check_stored()
    c.close()


# ------------------------------------------------------------------------------------------------ chunks
def attend(c, ahead, new, regular, seed, extra=3, slots=None):
    rng = np.random.default_rng(seed)
    B = len(ahead)
    seq = rng.permutation(slots or B + 1)[:B]
    held = np.zeros(slots or B + 1, int)
    held[seq] = np.array(ahead) + np.array(new)
    c.fill(held)
    if regular:
        step, first, rows = B, np.arange(B), B * new[0]
    else:
        step, first, rows = 1, np.concatenate([[0], np.cumsum(new)[:-1]]), sum(new)
    q = rng.standard_normal((rows + extra, c.H * c.hd + 8)).astype(np.float16)
    out = Tensor(np.full((rows + extra, c.H * c.hd + 16), 7, np.float16), device=c.dev)
    kw = {} if regular else {"count": ints(c.dev, new), "first": ints(c.dev, first)}
    c.kv.attend(0, Tensor(q, device=c.dev), ints(c.dev, ahead), seq=ints(c.dev, seq), max_count=max(new), step=step, out=out, **kw)
    got = out.numpy()
    assert (got[rows:] == 7).all() and (got[:, c.H * c.hd:] == 7).all()
    for b in range(B):
        at = first[b] + np.arange(new[b]) * step
        some = np.unique(np.concatenate([np.arange(min(new[b], 3)), rng.integers(0, max(new[b], 1), min(new[b], 12)), np.arange(max(0, new[b] - 3), new[b])]).astype(int))
        c.check(got[at[some], :c.H * c.hd], q[at[some], :c.H * c.hd].reshape(-1, c.H, c.hd), ahead[b] + some, [seq[b]] * len(some), f"sequence {b}")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd", SHAPES)
def test_attend(dev, H, G, hd, fmt):
    rng = np.random.default_rng(H * G + hd)
    cases = [(64, [0], [1], True), (16, [0, 5], [2, 2], True), (32, [300, 0, 17], [5, 5, 5], True), (64, [0], [200], True), (16, [130, 64], [129, 129], True),
             (64, [0, 127, 128, 500, 3, 0, 90, 1], [1, 0, 64, 33, 128, 65, 300, 2], False), (32, [1000, 0], [1, 257], False)]
    for i, (page, ahead, new, regular) in enumerate(cases):
        c = Cache(dev, H, G, hd, fmt, page, max(a + n for a, n in zip(ahead, new)), len(ahead) + 1, rng)
        attend(c, ahead, new, regular, seed=i)
        c.close()


@pytest.mark.parametrize("H,G,hd,ahead,new,fmt", [(32, 8, 128, [2500], [700], "int8"), (16, 8, 64, [0] * 40, [97] * 40, "fp8"), (8, 1, 128, [9000, 100], [40, 40], "int8"),
                                                  (8, 1, 64, [20011], [7], "fp8"), (12, 4, 64, [3000, 0, 10, 700], [1, 900, 64, 4], "int8"), (4, 4, 128, [4100], [16], "fp8")])
def test_attend_long_and_many(dev, H, G, hd, ahead, new, fmt):
    c = Cache(dev, H, G, hd, fmt, 64, max(a + n for a, n in zip(ahead, new)), len(ahead) + 1, np.random.default_rng(9))
    attend(c, ahead, new, len(set(new)) == 1, seed=3)
    c.close()


# Queries of a kv head on either side of 8, 16, 24 and 32, where the kernel for few of them takes more columns, and beyond it; long caches, so that
# (sequence, kv head)s are shared
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd,new", [(8, 1, 128, [2]), (8, 1, 128, [3, 3]), (8, 1, 64, [3]), (8, 1, 128, [4]), (12, 4, 64, [8, 7, 8]), (12, 4, 128, [6, 8]), (12, 4, 128, [9, 8]),
                                        (2, 2, 64, [24]), (2, 2, 128, [25, 17]), (2, 1, 128, [9, 12]), (8, 1, 64, [4, 4]), (12, 4, 64, [10]), (12, 4, 64, [11, 9, 3]),
                                        (2, 2, 64, [25, 32]), (2, 2, 64, [33, 30])])
def test_attend_few_queries(dev, H, G, hd, new, fmt):
    ahead = [2907, 66, 0][:len(new)]
    c = Cache(dev, H, G, hd, fmt, 32, max(a + n for a, n in zip(ahead, new)), len(new) + 1, np.random.default_rng(21))
    attend(c, ahead, new, False, seed=13)
    c.close()


# Prompts that the tensor cores' form cuts into items of 128 rows where they leave half of the SMs idle, and into 256 where they do not: sequences and
# rows on either side of the choice
@pytest.mark.parametrize("H,G,hd,new,ahead", [(32, 8, 128, [300], 0), (32, 8, 64, [576], 0), (32, 8, 128, [577], 100), (32, 8, 64, [640], 0), (8, 1, 64, [129], 900), (4, 1, 64, [33] * 16, 0),
                                              (4, 1, 64, [33] * 17, 0), (4, 4, 128, [128, 129, 256, 257], 40), (8, 1, 128, [700, 40], 200), (16, 8, 64, [64, 0, 65, 1, 200], 700), (4, 1, 64, [45], 1100), (8, 2, 128, [45], 1900),
                                              (32, 8, 64, [45] * 20, 1000), (4, 1, 128, [900], 600)])
def test_attend_prompts(dev, H, G, hd, new, ahead):
    c = Cache(dev, H, G, hd, "int8", 64, ahead + max(new), len(new) + 1, np.random.default_rng(22))
    attend(c, [ahead] * len(new), new, False, seed=14)
    c.close()


# Few rows behind long contexts: an item is cut into 2, 3 and many pieces, with rows left over, empty sequences among them, several on a CTA
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd,new,ahead", [(4, 1, 64, [9], 1900), (4, 1, 128, [45], 6000), (8, 1, 64, [45, 0, 33], 3100), (12, 4, 128, [50, 1], 2500), (3, 1, 64, [77], 12345),
                                              (16, 2, 128, [31, 40, 32], 4000)])
def test_attend_pieces(dev, H, G, hd, new, ahead, fmt):
    c = Cache(dev, H, G, hd, fmt, 32, ahead + max(new), len(new) + 1, np.random.default_rng(27))
    attend(c, [ahead - 611 * b for b in range(len(new))], new, False, seed=16)
    c.close()


@pytest.mark.parametrize("most", [3, 40])  # short chunks and long ones have kernels of their own
def test_attend_rows_outside(dev, most):
    rng = np.random.default_rng(10)
    c = Cache(dev, 4, 2, 64, "int8", 16, 96, 3, rng)
    c.fill([96, 60, 30])
    R_ = 4 * most
    q = rng.standard_normal((R_, 4 * 64)).astype(np.float16)
    out = Tensor(np.full((R_, 4 * 64), 7, np.float16), device=dev)
    pos, count, first, seq = [94, -1, 5, 0, 20], [most, most, most + 5, most - 1, 2], [0, most, 2 * most, 3 * most, R_ - 1], [0, 1, 2, 3, 1]
    c.kv.attend(0, Tensor(q, device=dev), ints(dev, pos), count=ints(dev, count), first=ints(dev, first), seq=ints(dev, seq), max_count=most, out=out)
    got = out.numpy()
    want = {}
    for p, n, f, s in zip(pos, count, first, seq):
        for i in range(min(n, most)):
            if f + i < R_:
                want[f + i] = (p + i, s) if s < 3 and 0 <= p + i < 96 else None
    for r in range(R_):
        if want.get(r) is None:
            assert not got[r].any(), r
        else:
            c.check(got[r:r + 1], q[r:r + 1].reshape(1, 4, 64), [want[r][0]], [want[r][1]], f"row {r}")
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_position_that_is_not_finite(dev, fmt, what, bad):
    """It is seen by the rows behind it, as NaN, and by nobody else: not by rows ahead of it, nor by other heads or sequences."""
    rng = np.random.default_rng(11)
    H, G, hd, n, at = 4, 2, 64, 150, 70
    c = Cache(dev, H, G, hd, fmt, 32, 256, 2, rng)
    x = c.rows(2 * n)
    pos, seq = np.tile(np.arange(n), 2), np.repeat([0, 1], n)
    x[at, (H + (1 if what == "k" else G + 1)) * hd + 5] = bad  # kv head 1 of position 70 of slot 0
    c.kv.write(0, Tensor(x, device=dev), ints(dev, pos), seq=ints(dev, seq))
    c.note(x, pos, seq)
    c.check_stored()
    assert np.isnan(c.k[0, at, 1]).all() and np.isnan(c.v[0, at, 1]).all() and np.isnan(c.k).sum() == hd
    q = rng.standard_normal((2 * n, H * hd)).astype(np.float16)

    def check(got, p, s):
        got = got.reshape(-1, G, H // G * hd)
        hit = np.zeros(got.shape[:2], bool)
        hit[:, 1] = (np.asarray(p) >= at) & (np.asarray(s) == 0)
        assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()

    out = c.kv.attend(0, Tensor(q, device=dev), ints(dev, [0, 0]), first=ints(dev, [0, n]), max_count=n, seq=ints(dev, [0, 1])).numpy()
    check(out, pos, seq)
    some = [at - 3, at - 2, at - 1, at, at + 1, n - 1]
    out = c.kv.attend(0, Tensor(q[:6], device=dev), ints(dev, some), max_count=1, seq=ints(dev, [0] * 6)).numpy()  # short chunks
    check(out, some, [0] * 6)
    y = c.rows(2)
    check(c.kv.decode(0, Tensor(y, device=dev), ints(dev, [n, n])).numpy(), [n, n], [0, 1])
    y = c.rows(2)
    check(c.kv.decode(0, Tensor(y, device=dev), ints(dev, [at - 1, at - 1])).numpy(), [at - 1, at - 1], [0, 1])  # what lies behind is hidden
    y = c.rows(2)
    y[0, (H + (1 if what == "k" else G + 1)) * hd + 9] = bad  # the new token itself
    check(c.kv.decode(0, Tensor(y, device=dev), ints(dev, [at, at])).numpy(), [at, at], [0, 1])
    c.close()


def test_scores_far_apart(dev):
    """One key above all others by far, the first or the last of the context or in its middle; scores of thousands; values of any size."""
    rng = np.random.default_rng(12)
    H, G, hd, n = 4, 1, 64, 700
    for k_scale, v_scale, spike in ((1, 1, 0), (1, 1, 699), (1, 1, 350), (60, 1, None), (1e-4, 1e-4, None), (1, 3e4, 3), (1e-7, 1e-7, None)):
        c = Cache(dev, H, G, hd, "int8", 64, n + 1, 1, rng)
        x = c.rows(n)
        x = x.reshape(n, H + 2, hd).astype(np.float64) * np.array([1] * H + [k_scale, v_scale])[:, None]
        x = np.clip(x, -65504, 65504).astype(np.float16)
        q = rng.standard_normal((40, H * hd)).astype(np.float16)
        if spike is not None:
            x[spike, H] = (q[0].reshape(H, hd)[0] * 8).astype(np.float16)
        x = x.reshape(n, -1)
        c.kv.write(0, Tensor(x, device=dev), ints(dev, np.arange(n)), seq=ints(dev, np.zeros(n)))
        c.note(x, np.arange(n), np.zeros(n, int))
        for m in (1, 40):
            out = c.kv.attend(0, Tensor(q[:m], device=dev), ints(dev, [n - m])).numpy()
            c.check(out, q[:m].reshape(m, H, hd), n - m + np.arange(m), [0] * m, f"{k_scale} {v_scale} {spike}")
        c.close()


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_a_conversation(dev, fmt):
    """Prompts of different lengths, then single tokens, then drafted ones, in slots that are used again, replayed from a graph."""
    rng = np.random.default_rng(13)
    H, G, hd = 8, 2, 128
    c = Cache(dev, H, G, hd, fmt, 16, 400, 4, rng)
    cs = table(c.n, hd)
    ct = Tensor(cs, device=dev)
    for seqs in ([2, 0, 3], [1, 2, 0]):
        new = np.array([150, 1, 77])
        first = np.concatenate([[0], np.cumsum(new)[:-1]])
        pos, seq = np.concatenate([np.arange(n) for n in new]), np.repeat(seqs, new)
        x = c.rows(len(pos))
        xt = Tensor(x, device=dev)
        c.kv.write(0, xt, ints(dev, pos), seq=ints(dev, seq), freqs_cis=ct, q_out=xt)
        out = c.kv.attend(0, xt, ints(dev, [0, 0, 0]), count=ints(dev, new), first=ints(dev, first), seq=ints(dev, seqs), max_count=150)
        c.check(out.numpy(), c.note(x, pos, seq, cs), pos, seq, "prompt")
        lens = new.copy()
        xt, pt, st = Tensor(c.rows(3), device=dev), ints(dev, lens), ints(dev, seqs)
        out = c.kv.decode(0, xt, pt, freqs_cis=ct, seq=st)
        c.note(xt.numpy(), lens, seqs, cs)
        with CUDAGraph(dev) as g:
            c.kv.decode(0, xt, pt, freqs_cis=ct, seq=st, out=out)
            dev.call("jg_pos_advance", pt.ptr, 3)
        for _ in range(20):
            x = c.rows(3)
            xt.assign(x)
            g.launch()
            q = c.note(x, lens, seqs, cs)
            c.check(out.numpy(), q, lens, seqs, "token")
            lens = lens + 1
        x = c.rows(15)  # five drafted tokens each, position-major
        pos, seq = (lens[None] + np.arange(5)[:, None]).reshape(-1), np.tile(seqs, 5)
        xt = Tensor(x, device=dev)
        c.kv.write(0, xt, ints(dev, pos), seq=ints(dev, seq), freqs_cis=ct, q_out=xt)
        out = c.kv.attend(0, xt, ints(dev, lens), seq=ints(dev, seqs))
        c.check(out.numpy(), c.note(x, pos, seq, cs), pos, seq, "draft")
        c.check_stored()
    c.close()


def test_graphs_share_a_workspace(dev):
    """Captured calls of two caches whose (sequence, kv head)s are shared by many CTAs, replayed in turn and among eager ones: the same bits every time."""
    rng = np.random.default_rng(23)
    a, b = Cache(dev, 8, 2, 128, "int8", 64, 3200, 2, rng), Cache(dev, 4, 2, 64, "fp8", 16, 2100, 3, rng)
    a.fill([2900, 3000])
    b.fill([1900, 40, 1000])
    xa, pa = Tensor(a.rows(200), device=dev), ints(dev, [2900, 3000])
    xb, pb = Tensor(b.rows(3), device=dev), ints(dev, [1900, 40, 1000])
    rows, seq = ints(dev, np.concatenate([2900 + np.arange(100), 3000 + np.arange(100)])), ints(dev, np.repeat([0, 1], 100))
    first = ints(dev, [0, 100])
    outs = [Tensor.zeros((200, 8 * 128), "float16", dev), Tensor.zeros((200, 8 * 128), "float16", dev), Tensor.zeros((3, 4 * 64), "float16", dev)]
    ka, va = (Tensor.zeros((200, 2 * 128), "float16", dev) for _ in range(2))

    def many():
        a.kv.write(0, xa, rows, seq=seq)
        a.kv.attend(0, xa, pa, first=first, max_count=100, out=outs[0])
        a.kv.read(0, pa, first=first, max_count=100, k=ka, v=va)

    def few():
        b.kv.decode(0, xb, pb, out=outs[2])
        a.kv.attend(0, xa, pa, first=first, max_count=3, out=outs[1])

    many()
    few()
    want = [t.numpy().copy() for t in (*outs, ka, va)]
    q = a.note(xa.numpy(), np.concatenate([2900 + np.arange(100), 3000 + np.arange(100)]), np.repeat([0, 1], 100))
    some = [0, 50, 99, 100, 199]
    a.check(want[0][some], q[some], [2900, 2950, 2999, 3000, 3099], [0, 0, 0, 1, 1])
    b.check(want[2], b.note(xb.numpy(), np.array([1900, 40, 1000]), np.arange(3)), [1900, 40, 1000], [0, 1, 2])
    with CUDAGraph(dev) as g1:
        many()
    with CUDAGraph(dev) as g2:
        few()
    for turn in ((g1.launch, g2.launch), (g2.launch, few, g1.launch), (many, g2.launch, g1.launch, g2.launch), (g1.launch, g1.launch, few)):
        for t in (*outs, ka, va):
            t.assign(np.zeros(t.shape, np.float16))
        for call in turn:
            call()
        for got, w in zip((*outs, ka, va), want):
            np.testing.assert_array_equal(got.numpy().view(np.uint16), w.view(np.uint16))
    a.close()
    b.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_pages_beyond_4_gib(dev, fmt):
    """Pages at the end of pools of more than 2^32 codes."""
    rng = np.random.default_rng(24)
    H, G, hd, page, n_pages = 8, 8, 128, 64, 66000
    c = Cache.__new__(Cache)
    c.dev, c.H, c.G, c.hd, c.fmt, c.rng = dev, H, G, hd, fmt, rng
    c.kv = QuantKVCache(dev, 1, H, G, hd, 512, 2, page_size=page, dtype=fmt, n_pages=n_pages)
    c.kv.set_block_table(np.stack([n_pages - 1 - np.arange(8), 65536 - 4 + np.arange(8)]).astype(np.int32))
    c.n = 512
    c.k, c.v = (np.zeros((2, c.n, G, hd), np.float16) for _ in range(2))
    attend(c, [250, 3], [140, 400], False, seed=15, slots=2)
    c.check_stored()
    pos = np.array([390, 403])
    x = c.rows(2)
    out = c.kv.decode(0, Tensor(x, device=dev), ints(dev, pos))
    c.check(out.numpy(), c.note(x, pos, np.arange(2)), pos, np.arange(2))
    c.check_stored()
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_a_slot_used_again(dev, fmt):
    """Behind a conversation's end lie rows of an earlier one, of the largest scales and of none."""
    rng = np.random.default_rng(25)
    c = Cache(dev, 8, 2, 128, fmt, 16, 160, 2, rng)
    x = c.rows(320)
    old = c.split(x)
    old[1][:] = np.where(rng.random(old[1].shape) < 0.5, 65504, -65504)
    old[2][:] = np.where(rng.random(old[2].shape) < 0.5, 65504, -65504)
    old[1][::3] = np.nan
    c.kv.write(0, Tensor(x, device=dev), ints(dev, np.tile(np.arange(160), 2)), seq=ints(dev, np.repeat([0, 1], 160)))
    c.fill([37, 90])
    for i in range(20):
        pos = np.array([37, 90]) + i
        y = c.rows(2)
        out = c.kv.decode(0, Tensor(y, device=dev), ints(dev, pos))
        c.check(out.numpy(), c.note(y, pos, np.arange(2)), pos, np.arange(2), f"token {i}")
    for most in (2, 9):  # few queries and many, over a tile with rows of both
        q = rng.standard_normal((2 * most, 8 * 128)).astype(np.float16)
        pos = np.array([57, 110]) - most
        out = c.kv.attend(0, Tensor(q, device=dev), ints(dev, pos), first=ints(dev, [0, most]), max_count=most)
        c.check(out.numpy(), q.reshape(-1, 8, 128), np.concatenate([pos[0] + np.arange(most), pos[1] + np.arange(most)]), np.repeat([0, 1], most), "chunk")
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("fused", [True, False])
def test_a_model(dev, fmt, fused):
    """A Llama with an 8-bit cache: prompt in one call, tokens through the captured step.  The attention of its last layer is that of the
    rows its own projections made, over what they leave in the cache."""
    from denograd_b200 import synth
    from denograd_b200.llama3 import Llama3
    from tests.golden.gen_golden import TINY
    B, S, n = 2, 20, 5
    llm = Llama3(size="1B", args=TINY, kv_dtype=fmt, max_context=64, max_batch=B, tied_output=True, temperature=0, fused=fused).load_synthetic()
    m = llm.model
    H, G, hd, last = m.n_heads, m.n_kv_heads, m.head_dim, len(m.layers) - 1
    cs = m.freqs_cis.numpy()
    k, v = (np.zeros((B, 64, G, hd), np.float16) for _ in range(2))

    def check(ws, pos, seq, rotated):
        x = ws.qkv.numpy().reshape(len(pos), H + 2 * G, hd)
        q = x[:, :H] if rotated else R.rotate(x[:, :H], cs, pos)
        k[seq, pos], v[seq, pos] = R.stored(R.rotate(x[:, H:H + G], cs, pos), x[:, H + G:], fmt)
        got = ws.attn.numpy()
        for i, (t, s) in enumerate(zip(pos, seq)):
            want, tol = R.attention(q[i], k[s], v[s], int(t))
            assert (np.abs(got[i] - want) <= tol).all(), (t, s)

    toks = synth.prompt_tokens(S, TINY["vocab_size"], batch=B, seed=3)
    if fused:
        tok = m.forward(toks, 0)
        check(m._workspace(B * S, rows=True), np.repeat(np.arange(S), B), np.tile(np.arange(B), S), True)
    else:  # a position at a time: what each leaves is read from the cache
        tok = m.forward(toks, 0)
        got = m._kv.read(last, ints(dev, [0] * B), max_count=S, step=B, rows=B * S)
        k[:, :S], v[:, :S] = (t.numpy().reshape(S, B, G, hd).swapaxes(0, 1) for t in got)
    for i in range(n):
        ws = m._workspace(B)
        tok = m.call(tok.numpy().reshape(B, 1), S + i)
        if fused:
            check(ws, np.full(B, S + i), np.arange(B), False)
    got = m._kv.read(last, ints(dev, [0] * B), max_count=64, step=B, rows=B * 64)
    if fused:
        for t, held in zip(got, (k, v)):
            same(t.numpy().reshape(64, B, G, hd).swapaxes(0, 1), held, "the cache")
    ids = llm.generate(toks, 8)
    assert ids.shape == (B, 8)
    # the device loop takes the same steps
    llm.reset()
    first = llm._prefill(toks).numpy()
    again = np.concatenate([first[:, None], m.decode_loop(first, S, 7)], 1)
    assert (again == ids).all()
