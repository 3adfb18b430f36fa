"""Queries that are not finite over the 8-bit KV cache, on the GPU."""
import numpy as np
import pytest

from denograd_b200.device import Tensor
from tests import kvquant_ref as R
from tests.test_kvquant_gpu import Cache, ints

pytestmark = pytest.mark.gpu


def signed(c, x):
    """Keys that are positive in channel 5 and negative in channel 6."""
    k = c.split(x)[1]
    k[..., 5], k[..., 6] = 1 + np.abs(k[..., 5]) / 8, -1 - np.abs(k[..., 6]) / 8


# (new positions, context ahead): short chunks within a CTA and shared, long ones of one tile, of one item, of two pieces and of many
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,hd,new,ahead", [(4, 2, 64, 1, 40), (4, 2, 64, 3, 900), (4, 1, 128, 2, 9000), (8, 2, 64, 40, 0), (4, 2, 64, 200, 300), (4, 1, 128, 45, 1500), (4, 1, 64, 40, 12000)])
def test_a_query_that_is_not_finite(dev, H, G, hd, new, ahead, fmt):
    """A softmax over scores of which all are -inf, or one inf, is NaN: that query's row, in that head, and no other."""
    rng = np.random.default_rng(35)
    n = ahead + new
    c = Cache(dev, H, G, hd, fmt, 64, n, 1, rng)
    x = c.rows(n)
    signed(c, x)
    c.kv.write(0, Tensor(x, device=dev), ints(dev, np.arange(n)), seq=ints(dev, np.zeros(n)))
    c.note(x, np.arange(n), np.zeros(n, int))
    q = rng.standard_normal((new + 2, H, hd)).astype(np.float16)
    bad = np.zeros((new + 2, H), bool)
    for i, (channel, value) in enumerate([(5, -np.inf), (6, np.inf), (5, np.inf), (6, -np.inf), (9, np.inf), (3, np.nan)]):
        row, head = (i * 7) % new, i % H
        if not bad[row, head]:
            q[row, head, channel], bad[row, head] = value, True
    q[new:, 0, 5] = -np.inf  # the last two lie behind the cache: zeros
    q[new:, 1, 6] = -np.inf
    pos = ints(dev, [ahead, c.n])
    out = Tensor(np.full((new + 2, H * hd), 7, np.float16), device=dev)
    c.kv.attend(0, Tensor(q.reshape(new + 2, -1), device=dev), pos, count=ints(dev, [new, 2]), first=ints(dev, [0, new]), seq=ints(dev, [0, 0]), max_count=max(new, 2), out=out)
    got = out.numpy().reshape(new + 2, H, hd)
    assert not got[new:].any()
    assert np.isnan(got[:new][bad[:new]]).all()
    clean = np.where(bad[:new, :, None], np.float16(0), q[:new])
    kept = np.where(bad[:new, :, None], np.float16(0), got[:new])
    some = np.unique(np.concatenate([np.flatnonzero(bad[:new].any(1)), [0, new - 1]]))
    for r in some:
        want, tol = R.attention(clean[r], c.k[0], c.v[0], ahead + int(r))
        off = np.abs(kept[r].astype(np.float64).reshape(-1) - want)
        assert (off <= tol)[~np.repeat(bad[r], hd)].all(), r
    c.close()


@pytest.mark.parametrize("n", [0, 1, 70, 9000])
def test_a_new_query_that_is_not_finite(dev, n):
    rng = np.random.default_rng(36)
    H, G, hd = 4, 2, 64
    c = Cache(dev, H, G, hd, "int8", 32, n + 1, 3, rng)
    x = c.rows(3 * n + 3)
    signed(c, x)
    pos, seq = np.tile(np.arange(n), 3), np.repeat(np.arange(3), n)
    if n:
        c.kv.write(0, Tensor(x[:3 * n], device=dev), ints(dev, pos), seq=ints(dev, seq))
        c.note(x[:3 * n], pos, seq)
    y = x[3 * n:]
    q = c.split(y)[0]
    q[0, 1, 5], q[1, 3, 6], q[2, 0, 5] = -np.inf, np.inf, np.inf
    out = Tensor(np.full((3, H * hd), 7, np.float16), device=dev)
    c.kv.decode(0, Tensor(y, device=dev), ints(dev, [n] * 3), out=out)
    got = out.numpy().reshape(3, H, hd)
    hit = np.zeros((3, H), bool)
    hit[0, 1] = hit[1, 3] = hit[2, 0] = True
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
    c.kv.decode(0, Tensor(y, device=dev), ints(dev, [c.n, -1, 2 ** 31 - 1]), out=out)
    assert not out.numpy().any()  # outside the cache
    c.close()


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8"])
def test_a_rank_by_itself(dev, kv_dtype):
    """A model under tensor parallelism, of one rank: the cache holds what the plain model's does, to the bit, behind the same tokens."""
    from denograd_b200 import synth
    from denograd_b200.llama3 import Llama3
    from denograd_b200.multi import TensorParallel
    from tests.golden.gen_golden import TINY
    toks = synth.prompt_tokens(20, TINY["vocab_size"], batch=2, seed=3)
    tp = TensorParallel(dev, 0, 1, TensorParallel.unique_id())
    ids, held = [], []
    for rank in (None, tp):
        llm = Llama3(size="1B", args=TINY, kv_dtype=kv_dtype, max_context=64, max_batch=2, tied_output=True, temperature=0, tp=rank).load_synthetic()
        m = llm.model
        ids.append(llm.generate(toks, 8, batched=True))
        held.append(m._kv.read(0, ints(dev, [0, 0]), max_count=20, step=2, rows=40)[0].numpy())  # the first layer's: no sum between ranks is in it yet
        dev.synchronize()
        m._forward_jit.clear()
        m._loop_graph.clear()
        del llm, m
    dev.synchronize()
    tp.close()
    assert (ids[0] == ids[1]).all() and held[0].any()
    np.testing.assert_array_equal(held[0].view(np.uint16), held[1].view(np.uint16))
