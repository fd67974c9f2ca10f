"""The operators that verify drafted tokens over a quantized cache, as cases that can be timed and checked.

Five operators, each with a plain form in elementary torch operations and the framework's own call:

  rope       rotary positions of (tokens, heads, head) rows from a table of cosines and sines
  append     one layer's new tokens: queries rotated, keys rotated and quantized with the values into the paged
             cache (one scale for each token and head), then the written rows read back
  read       a batch's cached keys and values back as floating point rows
  attention  the queries of a batch's drafted tokens over their cached context and, by a bit mask, each other
  logprobs   log probabilities of given tokens, the entropy, and the most probable alternatives of each row

Layouts (the ones a user's program keeps):

  pages      kq, vq: (pages, kv_heads, page, head) int8, or (pages, kv_heads, page, head / 2) uint8 holding two's
             complement nibbles, element 2i in the low half of byte i; ks, vs: (pages, kv_heads, page) float32. The
             value is the integer times its row's scale.
  table      (batch, most pages) int32 page numbers; position p of sequence b is slot p % page of page
             table[b, p // page]
  cu, lens   rows cu[b] .. cu[b + 1] - 1 are sequence b's, at positions lens[b] and on
  rope table (positions, rot) float32: cos of the rot / 2 angles, then sin
  tree       (rows, words) int64: bit j of a row's words allows the sequence's j-th new token
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
DEV = "cuda"


def listed():
    return [
        # one token of the 0.5B configuration (14 + 2 heads of 64): a decode step's smallest call
        dict(name="rope_token", op="rope", tokens=1, heads=16, head=64, rot=64, layout="half", dtype="float32",
             theta=1e6, scaling="none", start=700),
        # a long document's prompt: half of each head rotated in neighbouring pairs, positions scaled for 128k
        dict(name="rope_prompt", op="rope", tokens=8192, heads=40, head=128, rot=64, layout="pairs",
             dtype="bfloat16", theta=1e6, scaling="yarn", start=120000),
        # a batch's decode step, one token each, whose rows go into an int8 cache
        dict(name="append_step", op="append", batch=32, drafts=1, ctx=2047, heads=14, kv_heads=2, head=64, rot=64,
             layout="half", dtype="float32", bits=8, page=16),
        # ragged prompts of up to 2,000 tokens into an int4 cache
        dict(name="append_prompts", op="append", batch=8, drafts=2000, ctx=333, heads=32, kv_heads=8, head=128,
             rot=128, layout="half", dtype="bfloat16", bits=4, page=64),
        # stories15M's context (6 heads of 48) back as floats, for a check or a move to another cache
        dict(name="read_short", op="read", batch=4, ctx=255, kv_heads=6, head=48, dtype="float32", bits=8, page=16),
        # a batch of long contexts handed to code that wants bf16
        dict(name="read_long", op="read", batch=8, ctx=16383, kv_heads=8, head=128, dtype="bfloat16", bits=8,
             page=64),
        # single token decode of the 0.5B configuration: latency
        dict(name="attn_token", op="attention", batch=1, drafts=1, ctx=1000, heads=14, kv_heads=2, head=64,
             dtype="float32", bits=8, page=16, tree=False),
        # a serving batch, one token a sequence, ragged contexts: memory bound
        dict(name="attn_serving", op="attention", batch=64, drafts=1, ctx=8000, heads=32, kv_heads=8, head=128,
             dtype="bfloat16", bits=8, page=64, tree=False),
        # one very long context in int4, a short draft of five tokens
        dict(name="attn_long", op="attention", batch=1, drafts=5, ctx=131001, heads=32, kv_heads=8, head=128,
             dtype="float16", bits=4, page=128, tree=True),
        # trees of up to 64 drafted tokens over long contexts: the largest
        dict(name="attn_trees", op="attention", batch=16, drafts=64, ctx=16000, heads=32, kv_heads=8, head=128,
             dtype="bfloat16", bits=8, page=32, tree=True),
        # one row of the 0.5B configuration's vocabulary: the token sampled, five alternatives
        dict(name="logprobs_token", op="logprobs", rows=1, vocab=151936, ids=1, top=5, dtype="float32"),
        # a batch of trees or prompts scored over the same vocabulary
        dict(name="logprobs_batch", op="logprobs", rows=2000, vocab=151936, ids=4, top=20, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attention", "attention", "logprobs"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    heads, kv_heads, head = rng.choice([(14, 2, 64), (6, 6, 48), (12, 12, 64), (32, 8, 128), (10, 5, 80), (9, 1, 96)])
    bits, page = rng.choice([8, 8, 4]), rng.choice([16, 32, 64, 128, 256])
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 6000), heads=rng.randint(1, 40), head=head,
                    rot=rng.choice([head, head, 32, head - 16]), layout=rng.choice(["half", "pairs"]), dtype=dtype,
                    theta=rng.choice([1e4, 1e6]), scaling=rng.choice(["none", "linear", "yarn"]),
                    start=_log(rng, 1, 120000))
    if op == "append":
        batch = _log(rng, 1, 32)
        return dict(op=op, batch=batch, drafts=_log(rng, 1, 8000 // batch), ctx=_log(rng, 1, 8000), heads=heads,
                    kv_heads=kv_heads, head=head, rot=rng.choice([head, head, 32]),
                    layout=rng.choice(["half", "pairs"]), dtype=dtype, bits=bits, page=page)
    if op == "read":
        batch = _log(rng, 1, 32)
        return dict(op=op, batch=batch, ctx=_log(rng, 1, 100000 // batch), kv_heads=kv_heads, head=head, dtype=dtype,
                    bits=bits, page=page)
    if op == "attention":
        drafts = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 200)])
        batch = _log(rng, 1, 64)
        most = min(131000, 500000 // batch, 16 * 64 * 16000 // (batch * drafts))
        return dict(op=op, batch=batch, drafts=drafts, ctx=_log(rng, 1, most), heads=heads, kv_heads=kv_heads,
                    head=head, dtype=dtype, bits=bits, page=page, tree=rng.choice([True, False]))
    vocab = rng.choice([32000, 65536, 151936, _log(rng, 2, 200000)])
    return dict(op=op, rows=_log(rng, 1, 80000000 // max(vocab, 40000)), vocab=vocab, ids=rng.randint(1, 4),
                top=rng.randint(0, min(32, vocab)), dtype=dtype)


def _lens(c):
    """(cached tokens, new tokens) of each sequence: a spread that the case alone decides."""
    b = c["batch"]
    drafts = c.get("drafts", 0)
    lens = [c["ctx"] - c["ctx"] * i * 7 // (8 * b) for i in range(b)]
    new = [max(1, drafts - drafts * (i * 5 % 7) // 16) for i in range(b)]
    if b >= 4:
        lens[1] = 0  # a sequence that begins here
        if c["op"] != "read" and drafts > 1:
            new[2] = 0  # one that waits
    return lens, new


def _frequencies(c):
    """The rot / 2 frequencies in 64 bits, scaled for long contexts, and the factor of the cosines and sines."""
    half = c["rot"] // 2
    f = c["theta"] ** (-np.arange(half) / half)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "yarn":  # stretched by 4 from 32768 positions: slow pairs interpolated, fast ones kept
        turn = lambda n: half * math.log(32768 / (n * 2 * math.pi)) / math.log(c["theta"])  # noqa: E731
        lo, hi = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), half - 1)
        keep = 1 - np.clip((np.arange(half) - lo) / max(hi - lo, 1e-3), 0, 1)
        return f / 4.0 * (1 - keep) + f * keep, 0.1 * math.log(4.0) + 1
    return f, 1.0


def _rope_table(c, most):
    f, factor = _frequencies(c)
    a = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * torch.from_numpy(f).to(DEV)
    return torch.cat([a.cos() * factor, a.sin() * factor], 1).float()


def _pages(c, lens, new, g):
    """The batch's page table, in an order that use has mixed, and how many pages there are."""
    need = [-(-(n + m) // c["page"]) for n, m in zip(lens, new)]
    total = sum(need) + 3
    order = torch.randperm(total, device=DEV, generator=g).int()
    table = torch.full((c["batch"], max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def _cache(c, total, g):
    """Pages of quantized values of unit size: (integers, scales)."""
    shape = (total, c["kv_heads"], c["page"], c["head"])
    most, size = (127, 40.0) if c["bits"] == 8 else (7, 2.5)
    q = torch.empty(shape, dtype=torch.int8, device=DEV)
    for i in range(0, total, 4096):
        r = torch.randn(q[i:i + 4096].shape, device=DEV, generator=g)
        q[i:i + 4096] = (r * size).round().clamp(-most, most).to(torch.int8)
    s = (0.5 + torch.rand(shape[:3], device=DEV, generator=g)) / size
    if c["bits"] == 4:
        u = (q & 15).to(torch.uint8)
        q = u[..., 0::2] | (u[..., 1::2] << 4)
    return q, s


def _trees(c, lens, new, g):
    """A random tree of the new tokens of each sequence: the ancestors' bits and the depths."""
    rng = np.random.default_rng(int(torch.randint(1 << 30, (1,), device=DEV, generator=g)))
    n, words = max(new), -(-max(new) // 64)
    bits = np.zeros((c["batch"], n, n), bool)
    for j in range(n):
        bits[:, j, j] = True
        if j and c.get("tree", False):
            parent = np.maximum(rng.integers(-1, j, c["batch"]), j - 8)
            on = np.nonzero(parent >= 0)[0]
            bits[on, j] |= bits[on, parent[on]]
        elif j:
            bits[:, j] |= bits[:, j - 1]
    if c["batch"] >= 4 and c["op"] == "attention":
        bits[1, 0] = False  # no context and nothing allowed: an empty row
    word = np.zeros((c["batch"], n, words * 64), np.uint64)
    word[:, :, :n] = bits
    word = (word.reshape(c["batch"], n, words, 64) << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64)
    rows = [(b, i) for b, m in enumerate(new) for i in range(m)]
    b, i = np.array(rows).reshape(-1, 2).T
    depth = np.array(lens)[b] + np.maximum(bits.sum(-1)[b, i] - 1, 0)
    return torch.from_numpy(word[b, i].view(np.int64)).to(DEV), torch.from_numpy(depth.astype(np.int32)).to(DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"c": c}
    if c["op"] == "rope":
        s["x"] = torch.randn(c["tokens"], c["heads"], c["head"], device=DEV, generator=g).to(dt)
        s["pos"] = torch.arange(c["start"], c["start"] + c["tokens"], device=DEV, dtype=torch.int32)
        s["rope"] = _rope_table(c, c["start"] + c["tokens"])
        s["out"] = torch.empty_like(s["x"])
        return s
    if c["op"] == "logprobs":
        s["x"] = torch.empty(c["rows"], c["vocab"], device=DEV, dtype=dt)
        for i in range(0, c["rows"], 512):
            s["x"][i:i + 512] = torch.randn(s["x"][i:i + 512].shape, device=DEV, generator=g) * 2.5
        s["ids"] = torch.randint(c["vocab"], (c["rows"], c["ids"]), device=DEV, generator=g, dtype=torch.int32)
        return s
    lens, new = _lens(c)
    read = c["op"] == "read"
    if read:
        lens, new = [0] * c["batch"], lens
    s["most"], s["most_len"] = max(new), max(n + m for n, m in zip(lens, new))
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device=DEV)
    s["table"], total = _pages(c, lens, new, g)
    (s["kq"], s["ks"]), (s["vq"], s["vs"]) = _cache(c, total, g), _cache(c, total, g)
    rows, head, kvh = sum(new), c["head"], c["kv_heads"]
    if read:
        s["k"], s["v"] = (torch.empty(rows, kvh, head, device=DEV, dtype=dt) for _ in "kv")
        return s
    if c["op"] == "append":
        # one row of queries, keys and values a token, as the projection leaves them
        qkv = torch.randn(rows, c["heads"] + 2 * kvh, head, device=DEV, generator=g).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([c["heads"], kvh, kvh], 1)
        _, s["pos"] = _trees(c, lens, new, g) if c["drafts"] < 200 else (None, torch.cat(
            [torch.arange(n, n + m, device=DEV, dtype=torch.int32) for n, m in zip(lens, new)]))
        s["rope"] = _rope_table(dict(c, theta=1e6, scaling="none"), s["most_len"])
        s["q_out"] = torch.empty(rows, c["heads"], head, device=DEV, dtype=dt)
        s["k_out"], s["v_out"] = (torch.empty(rows, kvh, head, device=DEV) for _ in "kv")
        return s
    s["q"] = (torch.randn(rows, c["heads"], head, device=DEV, generator=g) * 2).to(dt)
    tree, _ = _trees(c, lens, new, g)
    s["tree"] = tree if c["tree"] or c["batch"] >= 4 else None  # none: each new token sees those before it
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(rows, c["heads"], device=DEV)
    return s


def _mvb():
    """The package (its folder's name has dashes) as the module mvb."""
    if "mvb" not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "local-llama-pynq-z2_b200")
        spec = importlib.util.spec_from_file_location("mvb", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules["mvb"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["mvb"])
    return sys.modules["mvb"]


def run(s):
    c = s["c"]
    return (_own if own else _plain)[c["op"]](s, c)


# ---- the framework's calls ----

def _own_rope(s, c):
    _mvb().rope(s["x"], s["pos"], s["rope"], s["out"], layout=c["layout"])
    return s["out"]


def _own_append(s, c):
    mvb = _mvb()
    cache = mvb.KvCache(s["kq"], s["ks"], s["vq"], s["vs"])
    mvb.kv_append(cache, s["k"], s["v"], s["table"], s["cu"], s["lens"], positions=s["pos"], rope=s["rope"],
                  layout=c["layout"], q=s["q"], q_out=s["q_out"])
    mvb.kv_read(cache, s["table"], s["cu"], s["lens"], s["k_out"], s["v_out"])
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _own_read(s, c):
    mvb = _mvb()
    mvb.kv_read(mvb.KvCache(s["kq"], s["ks"], s["vq"], s["vs"]), s["table"], s["cu"], s["lens"], s["k"], s["v"])
    return {"k": s["k"], "v": s["v"]}


def _own_attention(s, c):
    mvb = _mvb()
    mvb.tree_attention(s["q"], mvb.KvCache(s["kq"], s["ks"], s["vq"], s["vs"]), s["table"], s["cu"], s["lens"],
                       s["out"], tree=s["tree"], max_new=s["most"], max_len=s["most_len"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_logprobs(s, c):
    r = _mvb().logprobs(s["x"], s["ids"], top=c["top"])
    return {"logp": r.logp, "entropy": r.entropy, "top_ids": r.top_ids, "top_logp": r.top_logp}


_own = {"rope": _own_rope, "append": _own_append, "read": _own_read, "attention": _own_attention,
        "logprobs": _own_logprobs}


# ---- the plain forms ----

def _rotate(x, pos, table, layout):
    """x (rows, heads, head) with its first rot elements rotated, in x's type."""
    rot = table.shape[1]
    t = table[pos.long()].to(x.dtype)
    cos, sin = t[:, None, :rot // 2], t[:, None, rot // 2:]
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    y = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rope(s, c):
    s["out"].copy_(_rotate(s["x"].float(), s["pos"], s["rope"], c["layout"]))
    return s["out"]


def _slots(s, c):
    """(page, slot) of each new row."""
    row = torch.arange(int(s["q" if "q" in s else "k"].shape[0]), device=DEV)
    b = torch.searchsorted(s["cu"][1:].contiguous(), row.int(), right=True)
    p = s["lens"].long()[b] + row - s["cu"].long()[b]
    return s["table"].long()[b, p // c["page"]], p % c["page"]


def _quantize(x, bits):
    """x in 64 bits -> integers and the scale of each row, in 32 bits: the largest magnitude over 127 or 7."""
    most = 127 if bits == 8 else 7
    scale = (x.abs().amax(-1) / most).float()
    r = (x / scale.double()[..., None]).round().clamp(-most, most)
    q = torch.where(scale[..., None] > 0, r, 0).to(torch.int8)
    if bits == 4:
        u = (q & 15).to(torch.uint8)
        q = u[..., 0::2] | (u[..., 1::2] << 4)
    return q, scale


def _values(q, scale, bits):
    if bits == 4:
        lo, hi = (q & 15).to(torch.int8), (q >> 4).to(torch.int8)
        q = torch.stack([lo, hi], -1).flatten(-2)
        q = torch.where(q > 7, q - 16, q)
    return q.float() * scale[..., None]


def _plain_append(s, c):
    s["q_out"].copy_(_rotate(s["q"].float(), s["pos"], s["rope"], c["layout"]))
    page, slot = _slots(s, c)
    # values next to the border between two integers want 64 bits
    k = _rotate(s["k"].double(), s["pos"], s["rope"], c["layout"])
    s["kq"][page, :, slot], s["ks"][page, :, slot] = _quantize(k, c["bits"])
    s["vq"][page, :, slot], s["vs"][page, :, slot] = _quantize(s["v"].double(), c["bits"])
    s["k_out"].copy_(_values(s["kq"][page, :, slot], s["ks"][page, :, slot], c["bits"]))
    s["v_out"].copy_(_values(s["vq"][page, :, slot], s["vs"][page, :, slot], c["bits"]))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _plain_read(s, c):
    page, slot = _slots(s, c)
    s["k"].copy_(_values(s["kq"][page, :, slot], s["ks"][page, :, slot], c["bits"]))
    s["v"].copy_(_values(s["vq"][page, :, slot], s["vs"][page, :, slot], c["bits"]))
    return {"k": s["k"], "v": s["v"]}


def _allowed(s, n, length):
    """(batch, n, length): whether new token i may see position t."""
    t = torch.arange(length, device=DEV)
    i = torch.arange(n, device=DEV)
    cu, lens = s["cu"].long(), s["lens"].long()[:, None, None]
    new = (cu[1:] - cu[:-1])[:, None, None]
    j = t - lens  # (batch, 1, length)
    if s["tree"] is None:
        seen = j <= i[:, None]
    else:
        row = (cu[:-1, None] + i).clamp(max=s["tree"].shape[0] - 1)
        at = j.clamp(0, n - 1)
        word = s["tree"][row].gather(2, (at >> 6).expand(-1, n, -1))
        seen = ((word >> (at & 63)) & 1) > 0
    return (j < 0) | ((j < new) & seen)


def _padded(s, c, n, length):
    """The batch with every sequence at the largest size: queries, keys and values in 32 bits."""
    cu = s["cu"].long()
    row = (cu[:-1, None] + torch.arange(n, device=DEV)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row]
    t = torch.arange(length, device=DEV)
    page = s["table"].long()[:, t // c["page"]].clamp(min=0)
    k = _values(s["kq"][page, :, t % c["page"]], s["ks"][page, :, t % c["page"]], c["bits"])
    v = _values(s["vq"][page, :, t % c["page"]], s["vs"][page, :, t % c["page"]], c["bits"])
    return q, k, v


def _plain_attention(s, c):
    n, length, group = s["most"], s["most_len"], c["heads"] // c["kv_heads"]
    q, k, v = _padded(s, c, n, length)  # (b, n, heads, d), (b, t, kv, d)
    q = q.unflatten(2, (c["kv_heads"], group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # (b, kv, group * n, d)
    x = q @ k.permute(0, 2, 3, 1) * (1 / math.sqrt(c["head"]))
    seen = _allowed(s, n, length)[:, None].repeat(1, 1, group, 1)
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0, m)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    y = (e @ v.transpose(1, 2)) / torch.where(z > 0, z, 1)
    lse = (m + z.log())[..., 0]
    back = lambda a: a.unflatten(2, (group, n)).transpose(1, 3).transpose(2, 3)  # noqa: E731  (b, n, kv, group, ...)
    cu = s["cu"].long()
    keep = torch.arange(n, device=DEV) < (cu[1:] - cu[:-1])[:, None]
    s["out"].copy_(back(y)[keep].flatten(1, 2))
    s["lse"].copy_(back(lse)[keep].flatten(1, 2))
    return {"out": s["out"], "lse": s["lse"]}


def _order(x):
    """Integers in the order of float32 values, -0 and +0 alike."""
    i = (x + 0.0).view(torch.int32).long()
    return torch.where(i < 0, -(i & 0x7FFFFFFF), i)


def _plain_logprobs(s, c):
    x = s["x"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    logp = x.gather(1, s["ids"].long()) - lse
    entropy = (lse - (e * x).sum(-1, keepdim=True) / z)[:, 0]
    del e
    # the largest values, the lowest index first among equal ones
    key = (_order(x) << 20) | (0xFFFFF - torch.arange(c["vocab"], device=DEV))
    at = 0xFFFFF - (key.topk(c["top"], -1).values & 0xFFFFF)
    return {"logp": logp, "entropy": entropy, "top_ids": at.int(), "top_logp": x.gather(1, at) - lse}


_plain = {"rope": _plain_rope, "append": _plain_append, "read": _plain_read, "attention": _plain_attention,
          "logprobs": _plain_logprobs}


def work(case):
    c = case
    size = {"float32": 4}.get(c["dtype"], 2)
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"] * c["head"]
        return {"bytes": 2 * n * size + c["tokens"] * (4 + c["rot"] * 4), "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * (8 * c["ids"] + 4 + 8 * c["top"]), "flops": 5 * n}
    lens, new = _lens(c)
    row = c["kv_heads"] * (c["head"] * c["bits"] // 8 + 4)  # one cached token's keys (or values)
    if c["op"] == "read":
        n = sum(lens)
        return {"bytes": 2 * n * (row + c["kv_heads"] * c["head"] * size), "flops": 2 * n * c["kv_heads"] * c["head"]}
    if c["op"] == "append":
        n, q, kv = sum(new), c["heads"] * c["head"], c["kv_heads"] * c["head"]
        # read the projection's row and the table's, write the queries, write the cache and read it back, write that
        return {"bytes": n * (size * (2 * q + 2 * kv) + 4 + 4 * c["rot"] + 4 * row + 2 * kv * 4),
                "flops": n * (3 * (c["heads"] + c["kv_heads"]) * c["rot"] + 8 * kv)}
    seen = sum((n + m) for n, m in zip(lens, new) if m)
    pairs = sum((n + (m + 1) / 2) * m for n, m in zip(lens, new))
    rows = sum(new)
    return {"bytes": int(2 * seen * row + rows * c["heads"] * (2 * c["head"] * size + 4)),
            "flops": int(4 * pairs * c["heads"] * c["head"])}


# ---- the definitions in 64 bits ----

def _turned(x, pos, table, layout):
    """Rotation as a product of complex numbers."""
    rot = table.shape[1]
    w = torch.complex(*table[pos.long()].double().unsqueeze(1).chunk(2, -1))
    x = x.double()
    y = x.clone()
    if layout == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot].contiguous()) * w
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * w
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def _nibbles(q):
    """Integers of packed bytes, by arithmetic."""
    q = q.long()
    lo, hi = q % 16, q // 16
    return torch.stack([(lo + 8) % 16 - 8, (hi + 8) % 16 - 8], -1).reshape(*q.shape[:-1], -1)


def _held(x, bits):
    """What a row stands for after it was quantized."""
    top = 2 ** (bits - 1) - 1
    scale = (x.abs().max(-1, keepdim=True)[0] / top).float().double()
    return torch.nan_to_num(torch.round(x / scale)).clamp(-top, top) * scale


def _cached(s, c, b, n):
    """Keys and values of sequence b's first n positions."""
    got = []
    for q, scale in ((s["kq"], s["ks"]), (s["vq"], s["vs"])):
        at = s["table"][b, :-(-n // c["page"])].long()
        x = (_nibbles(q[at]) if c["bits"] == 4 else q[at]).double() * scale[at].double().unsqueeze(-1)
        got.append(x.transpose(1, 2).reshape(-1, c["kv_heads"], c["head"])[:n])
    return got


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "rope":
        return _turned(s["x"], s["pos"], s["rope"], c["layout"])
    if c["op"] == "append":
        return {"q": _turned(s["q"], s["pos"], s["rope"], c["layout"]),
                "k": _held(_turned(s["k"], s["pos"], s["rope"], c["layout"]), c["bits"]),
                "v": _held(s["v"].double(), c["bits"])}
    if c["op"] == "logprobs":
        logp, entropy, top = [], [], []
        for i in range(0, c["rows"], 128):
            y = torch.log_softmax(s["x"][i:i + 128].double(), -1)
            logp.append(y.gather(1, s["ids"][i:i + 128].long()))
            entropy.append(-(y.exp() * y).sum(-1))
            top.append(y.topk(c["top"], -1).values)  # equal values are alike here
        return {"logp": torch.cat(logp), "entropy": torch.cat(entropy), "top_ids": None, "top_logp": torch.cat(top)}
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    if c["op"] == "read":
        both = [_cached(s, c, b, cu[b + 1] - cu[b]) for b in range(c["batch"])]
        return {"k": torch.cat([k for k, _ in both]), "v": torch.cat([v for _, v in both])}
    out, lse = [], []
    for b in range(c["batch"]):
        n, new = lens[b], cu[b + 1] - cu[b]
        if not new:
            continue
        k, v = _cached(s, c, b, n + new)
        see = torch.ones(new, n + new, dtype=torch.bool, device=DEV)
        if s["tree"] is None:
            see[:, n:] = torch.ones(new, new, device=DEV).tril() > 0
        else:
            w = s["tree"][cu[b]:cu[b + 1]].cpu().numpy().view(np.uint8)
            see[:, n:] = torch.from_numpy(np.unpackbits(w, axis=1, bitorder="little")[:, :new]).to(DEV) > 0
        group = c["heads"] // c["kv_heads"]
        q = s["q"][cu[b]:cu[b + 1]].double()
        y, z = torch.zeros_like(q), torch.full((new, c["heads"]), -math.inf, device=DEV, dtype=torch.float64)
        for h in range(c["heads"]):
            x = torch.where(see, q[:, h] @ k[:, h // group].T / math.sqrt(c["head"]), -math.inf)
            z[:, h] = torch.logsumexp(x, -1)
            y[:, h] = torch.where(see.any(-1, keepdim=True), torch.softmax(x, -1), 0.0) @ v[:, h // group]
        out.append(y)
        lse.append(z)
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
