"""The operators of the 8-bit KV cache, through the calls that a program makes, and in a plain form.

A cache holds K and V of each (position, kv head) as 8-bit codes and a scale, in pages that a block table names:

  store    new rows of wq|wk|wv: Q and K are rotated, K and V go into the cache; what was stored is read back as fp16
  decode   one new token a row: stored as above, and its attention over all positions up to its own; the new K and V are read back
  attend   a chunk of new positions for each of several sequences, already stored, over the cache up to their own position
  read     stretches of the cache as fp16 rows

Formats: "int8", code = rint(x / scale) with scale = max |x| / 127 rounded up to 4 significant bits; "fp8", e4m3 codes with a power
of two.  In both, code x scale is an fp16 number.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    def case(name, op, fmt, heads, kv_heads, dim, page, batch, context, new=1, ragged=False):
        return {"name": name, "op": op, "format": fmt, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch,
                "context": context, "new": new, "ragged": ragged, "mix": 1}

    return [
        # one user chatting with the smallest model: one token behind a prompt of the benchmark's length
        case("decode 1B chat", "decode", "int8", 32, 8, 64, 64, 1, 547),
        # the benchmark's batch: 32 conversations of the 8B, 4100 positions each
        case("decode 8B 32 x 4100", "decode", "int8", 32, 8, 128, 64, 32, 4100),
        # a server's batch: conversations of 1 to 9001 positions, small pages
        case("decode 8B ragged", "decode", "fp8", 32, 8, 128, 16, 61, 9001, ragged=True),
        # one row of the 70B behind a whole book
        case("decode 70B book", "decode", "int8", 64, 8, 128, 64, 1, 131001),
        # drafted tokens of eight conversations, checked at once
        case("attend 8B drafts", "attend", "int8", 32, 8, 128, 32, 8, 3001, 5),
        # the benchmark's prompt
        case("attend 8B prompt 512", "attend", "int8", 32, 8, 128, 64, 1, 0, 512),
        # one portion of a long document (largest call)
        case("attend 8B document", "attend", "fp8", 32, 8, 128, 64, 1, 6001, 2048),
        # portions of 1 to 700 positions, conversations of any length, smallest model, small pages
        case("attend 1B mixed", "attend", "int8", 32, 8, 64, 16, 24, 4000, 700, ragged=True),
        # a single token is stored (smallest call)
        case("store 1B token", "store", "fp8", 32, 8, 64, 16, 1, 66, 1),
        # two prompts of the benchmark's length for long documents
        case("store 8B 2 x 1900", "store", "int8", 32, 8, 128, 64, 2, 0, 1900),
        # the start of a conversation, copied out for a new one
        case("read 1B 45", "read", "fp8", 32, 8, 64, 16, 1, 0, 45),
        # eight conversations that leave the cache
        case("read 8B ragged", "read", "int8", 32, 8, 128, 64, 8, 0, 4096, ragged=True),
    ]


def draw(rng) -> dict:
    """One more case of the same ranges: 1 to 64 sequences, contexts of 0 to 131072 positions, chunks of 1 to 4096, one to eight
    query heads to a kv head."""
    def spread(lo: int, hi: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(["decode", "decode", "attend", "attend", "store", "read"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads, dim = kv_heads * rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128])
    case = {"op": op, "format": rng.choice(["int8", "fp8"]), "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64]),
            "ragged": rng.random() < 0.5, "mix": rng.randint(2, 1 << 20)}
    batch = spread(1, 64)
    most = 131000 * 8 * 128 // (kv_heads * dim * batch)  # positions of a sequence
    if op == "decode":
        return dict(case, batch=batch, context=spread(1, min(131000, most)), new=1)
    if op == "attend":
        new = spread(1, min(2048, int((6e10 / (heads * dim * batch)) ** 0.5)))
        pairs = (1 << 33) // (heads * dim * new * batch)  # queries times keys, and the plain form's scores
        return dict(case, batch=batch, context=rng.choice([0, spread(1, max(2, min(20000, most, pairs, (1 << 28) // (heads * new * batch))))]), new=new)
    new = spread(1, min(4096, 8192 // batch if op == "store" else most, 32768 // batch))
    return dict(case, batch=batch, context=rng.choice([0, rng.randint(1, 900)]), new=new)


def lengths(case: dict) -> tuple[list[int], list[int]]:
    """(positions in the cache ahead of the new ones, number of new ones) of every sequence.  Ragged ones spread over their
    logarithm, a few have nothing new; the first is the longest."""
    r = random.Random(case["mix"])
    n = case["batch"]
    ahead, new = [case["context"]] * n, [case["new"]] * n
    if case["ragged"]:
        ahead = [ahead[0]] + [int(math.exp(r.uniform(0, math.log(ahead[0] + 1)))) for _ in range(n - 1)]
        if case["new"] > 1:
            new = [new[0]] + [0 if r.random() < 0.06 else int(math.exp(r.uniform(0, math.log(new[0] + 0.99)))) for _ in range(n - 1)]
    if case["op"] == "decode":
        ahead = [max(0, a - 1) for a in ahead]  # the new token is the last position of the context
    return ahead, new


# ------------------------------------------------------------------------------------------------ what a program has in hand
def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    H, G, D, page, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    ahead, new = lengths(case)
    slots = B + 1
    pages_per = -(-max(a + n for a, n in zip(ahead, new)) // page) + 1
    order = np.random.default_rng(seed)
    table = order.permutation(slots * pages_per).astype(np.int32).reshape(slots, pages_per)
    seq = order.permutation(slots)[:B].astype(np.int32)
    regular = not case["ragged"]
    first = np.arange(B) if regular else np.concatenate([[0], np.cumsum(new)[:-1]])
    step = B if regular else 1
    rows = sum(new)

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    # keys have channels that stand out, values have tokens that do
    loud = 1 + 5 * (torch.rand(1, G, 1, D, device=dev, generator=gen) < 0.04)
    k = (rand(slots * pages_per, G, page, D) * 0.9 * loud).half()
    v = (rand(slots * pages_per, G, page, D) * torch.exp(0.5 * rand(slots * pages_per, G, page, 1))).half()
    qkv = rand(rows, (H + 2 * G) * D).half()
    t = torch.arange(pages_per * page, device=dev, dtype=torch.float64)[:, None]
    angle = t * 500000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    cs = torch.stack([angle.cos(), angle.sin()], -1).half()

    def ints(x):
        return torch.as_tensor(np.asarray(x, np.int32), device=dev)

    lens = torch.tensor(new)
    if regular:
        row_pos = [ahead[b] + i for i in range(case["new"]) for b in range(B)]
        row_seq = list(seq) * case["new"]
    else:
        row_pos = [ahead[b] + i for b in range(B) for i in range(new[b])]
        row_seq = np.repeat(seq, lens)
    s = {"op": case["op"], "format": case["format"], "heads": H, "kv_heads": G, "dim": D, "page": page, "batch": B, "rows": rows, "most": max(new),
         "step": step, "qkv": qkv, "cs": cs, "pos": ints(ahead), "count": ints(new), "first": ints(first), "seq": ints(seq),
         "row_pos": ints(row_pos), "row_seq": ints(row_seq), "table": ints(table)}
    if own:
        return prepare_own(s, table, k, v)
    s["k"], s["k_scale"] = quantise(k, s["format"])
    s["v"], s["v_scale"] = quantise(v, s["format"])
    return s


def prepare_own(s: dict, table: np.ndarray, k: torch.Tensor, v: torch.Tensor) -> dict:
    """The framework's cache with the same contents, and its tensors over the inputs."""
    from denograd_b200.device import Buffer, Device, Tensor
    from denograd_b200.kvquant import QuantKVCache
    dev = Device["CUDA"]
    H, G, D, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    slots, pages_per = table.shape
    kinds = {torch.float16: "float16", torch.int32: "int32"}

    def wrap(t):
        return Tensor(Buffer.external(dev, t.data_ptr(), t.numel(), kinds[t.dtype]), shape=tuple(t.shape))

    cache = QuantKVCache(dev, 1, H, G, D, pages_per * page, slots, page_size=page, dtype=s["format"])
    cache.set_block_table(table)
    at = torch.arange(pages_per * page, dtype=torch.int32, device="cuda")
    for slot in range(slots):
        ids = s["table"][slot].long()
        for lo in range(0, pages_per, 16384 // page):  # rows of one call
            some = ids[lo:lo + 16384 // page]
            n = len(some) * page
            x = torch.zeros(n, H + 2 * G, D, dtype=torch.float16, device="cuda")
            x[:, H:H + G] = k[some].transpose(1, 2).reshape(n, G, D)
            x[:, H + G:] = v[some].transpose(1, 2).reshape(n, G, D)
            pos, seq = at[lo * page:lo * page + n].clone(), torch.full((n,), slot, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            cache.write(0, wrap(x.view(n, -1)), wrap(pos), seq=wrap(seq))
            dev.synchronize()
    half = lambda n, w: torch.zeros(n, w, dtype=torch.float16, device="cuda")  # noqa: E731
    s["cache"] = cache
    s["out"], s["k_out"], s["v_out"] = half(s["rows"], H * D), half(s["rows"], G * D), half(s["rows"], G * D)
    s["t"] = {n: wrap(s[n]) for n in ("qkv", "cs", "pos", "count", "first", "seq", "row_pos", "row_seq", "out", "k_out", "v_out")}
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s: dict):
    if own:
        return run_own(s)
    op, H, G, D = s["op"], s["heads"], s["kv_heads"], s["dim"]
    rows, B, n = s["rows"], s["batch"], s["most"]
    if op == "read":
        k, v = gather(s, s["row_pos"], s["row_seq"])
        return {"k": k.half().view(rows, G * D), "v": v.half().view(rows, G * D)}
    x = s["qkv"].view(rows, H + 2 * G, D)
    if op in ("store", "decode"):
        q, k = (rotate(part, s["cs"], s["row_pos"]).half() for part in (x[:, :H], x[:, H:H + G]))
        new = store(s, k, x[:, H + G:])
        if op == "store":
            return dict(new, q=q.reshape(rows, H * D))
        x = q
    # the rows as [sequence, position], those that a sequence lacks as zeros
    i = torch.arange(n, device=x.device)
    there = i < s["count"][:, None]
    at = torch.where(there, s["first"][:, None] + i * s["step"], 0).long()
    q = x[:, :H].float()[at].view(B, n, G, H // G, D)
    last = s["pos"][:, None] + i  # what a row sees: positions 0 .. last
    context = s["table"].shape[1] * s["page"]
    t = torch.arange(context, device=x.device)
    k, v = (part.view(B, context, G, D) for part in gather(s, t.repeat(B), s["seq"].repeat_interleave(context)))
    scores = torch.einsum("bngrd,btgd->bgrnt", q, k) * (1.0 / math.sqrt(D))
    scores = torch.where(t <= last[:, :, None], scores.permute(1, 2, 0, 3, 4), -math.inf).permute(2, 0, 1, 3, 4)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.einsum("bgrnt,btgd->bngrd", e / e.sum(-1, keepdim=True), v)
    out = torch.zeros(rows, H * D, dtype=torch.float16, device=x.device)
    out[at[there]] = o[there].reshape(-1, H * D).half()
    return dict(new, out=out) if op == "decode" else {"out": out}


def run_own(s: dict):
    t, cache, op = s["t"], s["cache"], s["op"]
    if op == "attend":
        cache.attend(0, t["qkv"], t["pos"], count=t["count"], first=t["first"], seq=t["seq"], max_count=s["most"], step=s["step"], out=t["out"])
        return {"out": s["out"]}
    if op == "store":
        cache.write(0, t["qkv"], t["row_pos"], seq=t["row_seq"], freqs_cis=t["cs"], q_out=t["out"])
    elif op == "decode":
        cache.decode(0, t["qkv"], t["pos"], freqs_cis=t["cs"], seq=t["seq"], out=t["out"])
    cache.read(0, t["pos"], count=t["count"], first=t["first"], seq=t["seq"], max_count=s["most"], step=s["step"], k=t["k_out"], v=t["v_out"])
    got = {"k": s["k_out"], "v": s["v_out"]}
    if op != "read":
        got["q" if op == "store" else "out"] = s["out"]
    return got


def rotate(x: torch.Tensor, cs: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """Pairs of neighbouring values of [rows, heads, dim] turned by their row's angles, in 32 bits."""
    c, s = cs[pos.long()].float()[:, None].unbind(-1)
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def quantise(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of the last axis."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        share = top / 127
        grain = torch.exp2((torch.frexp(share).exponent - 4).clamp(min=-24).float())
        scale = torch.ceil(share / grain) * grain
        code = torch.where(scale > 0, torch.round(x / scale), 0.0)
        most = torch.floor(65504 / scale).clamp(max=127)
        return torch.minimum(torch.maximum(code, -most), most).to(torch.int8), scale.half()
    share = torch.frexp(top / 448)
    e = (share.exponent - (share.mantissa == 0.5).int()).clamp(min=-15).float()
    scale = torch.where(top > 0, torch.exp2(e), 0.0)
    most = torch.where(scale < 256, 448.0, 240.0)
    code = torch.where(scale > 0, x / scale, 0.0)
    return torch.minimum(torch.maximum(code, -most), most).to(torch.float8_e4m3fn), scale.half()


def store(s: dict, k: torch.Tensor, v: torch.Tensor) -> dict:
    """Puts rows [rows, kv heads, dim] into the cache; what they are from then on."""
    t = s["row_pos"].long()
    page, slot = s["table"][s["row_seq"].long(), t // s["page"]].long(), t % s["page"]
    got = {}
    for name, x in (("k", k), ("v", v)):
        code, scale = quantise(x, s["format"])
        byte, into = (c.view(torch.uint8) for c in (code, s[name]))  # an 8-bit float is moved as its byte
        into[page, :, slot] = byte
        s[name + "_scale"][page, :, slot] = scale
        got[name] = (code.float() * scale.float()).half().reshape(len(t), -1)
    return got


def gather(s: dict, t: torch.Tensor, seq: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of positions t of sequences seq, as 32-bit rows [., kv heads, dim]."""
    page, slot = s["table"][seq.long(), t.long() // s["page"]].long(), t.long() % s["page"]
    return tuple(s[n].view(torch.uint8)[page, :, slot].view(s[n].dtype).float() * s[n + "_scale"][page, :, slot].float() for n in ("k", "v"))


# ------------------------------------------------------------------------------------------------ what a pass has to do
def work(case: dict) -> dict:
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    ahead, new = lengths(case)
    rows = sum(new)
    cached = G * (2 * D + 4)  # codes and scales of a position
    x, q, kv = (H + 2 * G) * D * 2, H * D * 2, G * D * 2
    if case["op"] == "read":
        return {"bytes": rows * (cached + 2 * kv), "flops": 0}
    if case["op"] == "store":
        return {"bytes": rows * (x + D * 2 + q + cached + 2 * kv), "flops": 0}
    seen = sum(a * n + n * (n + 1) // 2 for a, n in zip(ahead, new))
    flops = 4.0 * H * D * seen
    if case["op"] == "decode":
        return {"bytes": sum(ahead) * cached + rows * (x + D * 2 + q + cached + 2 * kv), "flops": flops}
    return {"bytes": sum(a + n for a, n in zip(ahead, new) if n) * cached + rows * 2 * q, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    """The same results from the definitions, a sequence at a time."""
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    H, G, D, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    table = s["table"].cpu().numpy()
    ahead, new = lengths(case)
    seqs, firsts = s["seq"].tolist(), s["first"].tolist()
    values = {n: s[n].double() * s[n + "_scale"].double() for n in ("k", "v")}
    qkv = s["qkv"].double().view(s["rows"], H + 2 * G, D)
    empty = lambda heads: torch.zeros(s["rows"], heads * D, dtype=torch.float64, device="cuda")  # noqa: E731
    got = {"k": empty(G), "v": empty(G), "q": empty(H), "out": empty(H)}
    for b, (a, n) in enumerate(zip(ahead, new)):
        if n == 0:
            continue
        at = firsts[b] + torch.arange(n, device="cuda") * s["step"]
        ids = torch.as_tensor(table[seqs[b]].astype(np.int64), device="cuda")
        k, v = (values[name][ids].permute(0, 2, 1, 3).reshape(-1, G, D)[:a + n].clone() for name in ("k", "v"))
        q = qkv[at, :H]
        if case["op"] in ("store", "decode"):
            angles = torch.complex(*s["cs"][a:a + n].double().unbind(-1))[:, None]
            turn = lambda x: torch.view_as_real(torch.view_as_complex(x.reshape(n, -1, D // 2, 2).contiguous()) * angles).reshape(n, -1, D)  # noqa: B023, E731
            q = turn(q).half().double()
            k[a:] = nearest(turn(qkv[at, H:H + G]).half().double(), case["format"])
            v[a:] = nearest(qkv[at, H + G:], case["format"])
        got["k"][at], got["v"][at], got["q"][at] = (x.reshape(n, -1) for x in (k[a:], v[a:], q))
        if case["op"] in ("decode", "attend"):
            hide = torch.arange(a + n, device="cuda") > a + torch.arange(n, device="cuda")[:, None]
            for g in range(G):
                score = q[:, g * (H // G):(g + 1) * (H // G)].transpose(0, 1) @ k[:, g].T / D ** 0.5
                weight = torch.softmax(score.masked_fill(hide, -math.inf), -1)
                got["out"][at, g * (H // G) * D:(g + 1) * (H // G) * D] = (weight @ v[:, g]).transpose(0, 1).reshape(n, -1)
    keep = {"store": ("k", "v", "q"), "decode": ("k", "v", "out"), "attend": ("out",), "read": ("k", "v")}[case["op"]]
    return {name: got[name] for name in keep}


def nearest(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The values that stand for x in 8 bits."""
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        low = torch.floor(torch.log2((top / 127).clamp(min=2.0 ** -40)) + 1e-13)
        unit = torch.exp2((low - 3).clamp(min=-24))
        scale = torch.ceil(top / (127 * unit) - 1e-13) * unit
        n = torch.round(x / scale.clamp(min=2.0 ** -24))
        n = torch.where(n.abs() * scale > 65504, n - n.sign(), n)
        return n.clamp(-127, 127) * scale
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -40) / 448) - 1e-13).clamp(min=-15))
    y = x / scale
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20)) + 1e-13).clamp(min=-6) - 3)
    n = torch.round(y / unit) * unit
    return torch.where(n.abs() * scale > 65504, n.sign() * 240, n) * scale
