"""Serving operators on CUDA tensors: what stands between the quantized matmuls when a batch of sequences verifies one, a
chain or a tree of new tokens each over a paged cache held in 8 or 4 bits.

    cache = mvb.KvCache.empty(pages=4096, kv_heads=2, page=32, head=64, bits=8)     # one a layer
    freq, factor = mvb.rope_frequencies(64, 1e6)                                    # once
    table = mvb.rope_table(freq, positions=32768, factor=factor)                    # once
    # every layer of a step: rows of the batch's new tokens, sequence after sequence
    mvb.kv_append(cache, k, v, pages, cu, lens, positions=pos, rope=table, q=q, q_out=q)
    mvb.tree_attention(q, cache, pages, cu, lens, out, tree=mask, max_new=8, max_len=5000)
    # after the head: which drafts the model would have taken
    r = mvb.logprobs(logits, drafted, top=5)

A batch: rows cu[b] .. cu[b + 1] - 1 are sequence b's new tokens (cu: batch + 1 int32), which stand at its positions
lens[b], lens[b] + 1, .. (lens: batch int32, the tokens cached before this call); pages (batch, columns) int32 names the
page of each run of positions. Sequences may have no new token and no cached one; rows behind cu[batch] are left as they
are. All of it is read on the device: a call may be captured in a CUDA graph and replayed with other contents.

Checks: types, shapes, strides and devices are checked here (ValueError) and in the library (MatvecError). What only the
device can see (a page number, position or length out of range) is skipped there, never followed, and reported by
serve_status(). Calls are asynchronous on `stream` (default: the current stream of the tensors' device) and may run on any
device; they keep no state and use no workspace, so calls on several streams do not meet.
"""
import ctypes as C
import math
from collections import namedtuple

_TYPES = {}


def _torch():
    import torch
    if not _TYPES:
        _TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    return torch


def _mvb():
    import sys
    return sys.modules[__package__]


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _call(name, device, stream, *args):
    """One library call on `device` (made current for it) and `stream`."""
    torch = _torch()
    m = _mvb()
    f = getattr(m.lib(), name)
    handle = (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = f(*args, handle)
    else:
        with torch.cuda.device(device):
            rc = f(*args, handle)
    if rc != 0:
        m.check(rc, name)


def _on(device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}: one device is needed")
    _need(device.type == "cuda", f"CUDA tensors are needed, not {device.type}")


def _rows(name, t, heads, head):
    """Checks a (rows, heads, head) tensor whose heads lie next to one another; its row stride."""
    _need(t.dim() == 3 and (heads is None or t.shape[1] == heads) and (head is None or t.shape[2] == head),
          f"{name} is {tuple(t.shape)}: (rows, {heads or 'heads'}, {head or 'head'}) is needed")
    st = t.stride()
    _need(st[2] == 1 and (st[1] == t.shape[2] or t.shape[1] == 1), f"{name}: the heads of a row must be contiguous")
    _need(t.dtype in _TYPES, f"{name} is {t.dtype}: float32, bfloat16 or float16 is needed")
    return st[0] if t.shape[0] > 1 else t.shape[1] * t.shape[2]  # a single row's stride says nothing


def _int32(name, t, shape):
    torch = _torch()
    _need(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name} is {t.dtype} {tuple(t.shape)}: contiguous int32 {shape} is needed")


class KvCache:
    """A layer's paged cache: kq, vq (pages, kv_heads, page, head) int8 or (.., head / 2) uint8 of nibbles (element 2i
    low, two's complement), ks, vs (pages, kv_heads, page) float32. value = integer * scale. Only views are kept."""

    __slots__ = ("kq", "ks", "vq", "vs", "pages", "kv_heads", "page", "head", "bits", "device", "args")

    def __init__(self, kq, ks, vq, vs):
        torch = _torch()
        _need(kq.dim() == 4 and kq.dtype in (torch.int8, torch.uint8),
              "kq: (pages, kv_heads, page, head) int8, or uint8 with two elements a byte, is needed")
        self.pages, self.kv_heads, self.page, width = kq.shape
        self.bits = 8 if kq.dtype == torch.int8 else 4
        self.head = width * 8 // self.bits
        _need(vq.shape == kq.shape and vq.dtype == kq.dtype, "vq must be like kq")
        for name, t in (("ks", ks), ("vs", vs)):
            _need(t.shape == kq.shape[:3] and t.dtype == torch.float32, f"{name} must be float32 {tuple(kq.shape[:3])}")
        for t in (kq, ks, vq, vs):
            _need(t.is_contiguous(), "the cache's tensors must be contiguous")
        self.device = kq.device
        _on(self.device, ks, vq, vs)
        self.kq, self.ks, self.vq, self.vs = kq, ks, vq, vs
        self.args = (kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), self.pages, self.page, self.kv_heads,
                     self.head, self.bits)

    @classmethod
    def empty(cls, pages, kv_heads, page, head, bits=8, device="cuda"):
        """A cache of `pages` pages of `page` tokens (a power of two from 16), uninitialised."""
        torch = _torch()
        _need(bits in (4, 8), f"bits={bits}: 4 or 8 is needed")
        _need(head % 2 == 0, f"head={head}: an even size is needed")
        dt, width = (torch.int8, head) if bits == 8 else (torch.uint8, head // 2)
        q = [torch.empty(pages, kv_heads, page, width, dtype=dt, device=device) for _ in "kv"]
        s = [torch.empty(pages, kv_heads, page, device=device) for _ in "kv"]
        return cls(q[0], s[0], q[1], s[1])


def _batch(cache, pages, cu, lens):
    _need(pages.dim() == 2 and cu.dim() == 1 and lens.dim() == 1, "pages (batch, columns), cu and lens (vectors) are needed")
    b = pages.shape[0]
    _int32("pages", pages, (b, pages.shape[1]))
    _int32("cu", cu, (b + 1,))
    _int32("lens", lens, (b,))
    _on(cache.device, pages, cu, lens)
    return (pages.data_ptr(), pages.shape[1], cu.data_ptr(), lens.data_ptr(), b)


_LAYOUTS = {"half": 0, "pairs": 1}


def _layout(layout):
    _need(layout in _LAYOUTS, f"layout={layout!r}: 'half' or 'pairs' is needed")
    return _LAYOUTS[layout]


def rope_frequencies(rot, theta, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """The rot / 2 rotary frequencies theta^(-2i / rot) in 64 bits (numpy), scaled for contexts `factor` times longer, and
    the factor that the table's cosines and sines take. scaling: None; "linear" (positions divided by factor); "ntk" (the
    base raised to theta * factor^(rot / (rot - 2))); "yarn" (pairs that turn fewer than `slow` times in `original`
    positions are divided by factor, those that turn more than `fast` times kept, a ramp between; the factor is
    0.1 ln(factor) + 1)."""
    import numpy as np
    _need(rot > 0 and rot % 2 == 0 and theta > 0, f"rot={rot} theta={theta}: an even rot and a positive base are needed")
    _need(factor >= 1.0, f"factor={factor}: at least 1 is needed")
    half = rot // 2
    if scaling == "ntk":
        _need(rot > 2, "ntk needs rot > 2")
        theta = theta * factor ** (rot / (rot - 2))
    f = float(theta) ** (-np.arange(half) / half)
    if scaling in (None, "ntk"):
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    _need(scaling == "yarn", f"scaling={scaling!r}: None, 'linear', 'ntk' or 'yarn' is needed")
    _need(original is not None and original > 0 and theta > 1, "yarn needs original positions and a base above 1")
    turn = lambda n: half * math.log(original / (n * 2 * math.pi)) / math.log(theta)  # noqa: E731
    lo, hi = max(math.floor(turn(fast)), 0), min(math.ceil(turn(slow)), half - 1)
    keep = 1 - np.clip((np.arange(half) - lo) / max(hi - lo, 1e-3), 0, 1)
    return f / factor * (1 - keep) + f * keep, (0.1 * math.log(factor) + 1 if factor > 1 else 1.0)


def rope_table(frequencies, positions, out=None, start=0, factor=1.0, device="cuda", stream=None):
    """(positions, rot) float32: row p holds factor * cos of the rot / 2 angles (start + p) * frequencies, then factor *
    sin, angles and functions in 64 bits. frequencies: float64, numpy or a CUDA tensor."""
    torch = _torch()
    if not torch.is_tensor(frequencies):
        frequencies = torch.as_tensor(frequencies, dtype=torch.float64, device=out.device if out is not None else device)
    _need(frequencies.dtype == torch.float64 and frequencies.dim() == 1 and frequencies.is_contiguous(),
          "frequencies: a float64 vector is needed")
    half = frequencies.numel()
    if out is None:
        out = torch.empty(positions, 2 * half, device=frequencies.device)
    _need(out.dtype == torch.float32 and tuple(out.shape) == (positions, 2 * half) and out.is_contiguous(),
          f"out: contiguous float32 {(positions, 2 * half)} is needed")
    _on(out.device, frequencies)
    if stream is not None:
        for t in (out, frequencies):
            t.record_stream(stream)
    _call("mvb_rope_table", out.device, stream, frequencies.data_ptr(), out.data_ptr(), half, positions, start,
          float(factor))
    return out


def _table(table):
    torch = _torch()
    _need(table.dtype == torch.float32 and table.dim() == 2 and table.is_contiguous(),
          "rope table: contiguous float32 (positions, rot) is needed")


def rope(x, positions, table, out=None, layout="half", stream=None):
    """x (tokens, heads, head) with the first rot elements of each head turned by the table's row of the token's position;
    the other elements as they are. layout "half": pairs (i, i + rot / 2); "pairs": (2i, 2i + 1). out: x's shape and
    type, x itself for in place (the default); it must not overlap x otherwise."""
    torch = _torch()
    out = x if out is None else out
    xs = _rows("x", x, None, None)
    _, heads, head = x.shape
    os_ = _rows("out", out, heads, head)
    _need(out.dtype == x.dtype and out.shape[0] == x.shape[0], "out must be like x")
    _need(positions.dtype == torch.int32, "positions: int32 is needed")
    _int32("positions", positions, (x.shape[0],))
    _table(table)
    _on(x.device, out, positions, table)
    _call("mvb_rope", x.device, stream, x.data_ptr(), positions.data_ptr(), table.data_ptr(), out.data_ptr(),
          _TYPES[x.dtype], x.shape[0], heads, head, table.shape[1], table.shape[0], _layout(layout), xs, os_)
    return out


def kv_append(cache, k, v, pages, cu, lens, positions=None, rope=None, layout="half", q=None, q_out=None, stream=None):
    """The batch's new keys and values (rows, kv_heads, head) quantized into the cache at their sequences' positions
    lens[b] and on: scale = max |x| / 127 (or / 7), integers rounded to nearest even. With a rope table the keys are
    turned first (and q into q_out, rows of queries, in the same launch; q_out may be q) by the rows' `positions`
    (int32; default the position in the cache; a tree's are those of its depth). A row with an infinity or a NaN is held
    with the scale NaN. Sequences must not share a page that the call writes."""
    torch = _torch()
    _TYPES  # filled by _torch()
    ks, vs = _rows("k", k, cache.kv_heads, cache.head), _rows("v", v, cache.kv_heads, cache.head)
    n = k.shape[0]
    _need(v.shape[0] == n and v.dtype == k.dtype, "v must be like k")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, k, v, positions, rope, q, q_out)
    if positions is not None:
        _int32("positions", positions, (n,))
        _need(rope is not None, "positions without a rope table")
    if rope is not None:
        _table(rope)
    qs = qos = heads = 0
    if q is not None:
        _need(rope is not None and q_out is not None, "queries need a rope table and q_out")
        qs, qos = _rows("q", q, None, cache.head), _rows("q_out", q_out, None, cache.head)
        heads = q.shape[1]
        _need(q.shape[0] == n and q_out.shape == q.shape and q.dtype == k.dtype and q_out.dtype == k.dtype,
              "q and q_out must have k's rows and type")
    _call("mvb_kv_append", cache.device, stream, *cache.args, *b, n, k.data_ptr(), ks, v.data_ptr(), vs, _TYPES[k.dtype],
          None if rope is None else rope.data_ptr(), None if positions is None else positions.data_ptr(),
          0 if rope is None else rope.shape[1], 0 if rope is None else rope.shape[0], _layout(layout),
          None if q is None else q.data_ptr(), qs, None if q is None else q_out.data_ptr(), qos, heads)


def kv_read(cache, pages, cu, lens, k_out, v_out, stream=None):
    """Cached keys and values back: rows cu[b] .. cu[b + 1] - 1 of k_out and v_out (rows, kv_heads, head; float32,
    bfloat16 or float16) become sequence b's positions lens[b] and on (lens of zeros and cu of running lengths: whole
    contexts). integer * scale, rounded to the output's type."""
    _torch()
    ks, vs = _rows("k_out", k_out, cache.kv_heads, cache.head), _rows("v_out", v_out, cache.kv_heads, cache.head)
    n = k_out.shape[0]
    _need(v_out.shape[0] == n and v_out.dtype == k_out.dtype, "v_out must be like k_out")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, k_out, v_out)
    _call("mvb_kv_read", cache.device, stream, *cache.args, *b, n, k_out.data_ptr(), ks, v_out.data_ptr(), vs,
          _TYPES[k_out.dtype])


def tree_mask(parents):
    """The mask bits of trees of new tokens: parents[i] is the row (within its sequence, below i) of token i's parent, or
    -1 for a child of the cached context. One sequence: a vector; several of the same size: (batch, n). Returns int64
    (.., n, words) on the parents' device: bit j of row i is set where j is i or one of its ancestors."""
    import numpy as np
    torch = _torch()
    p = np.asarray(parents.cpu() if torch.is_tensor(parents) else parents, dtype=np.int64)
    n = p.shape[-1]
    flat = p.reshape(math.prod(p.shape[:-1]), n)
    _need(bool(((flat < np.arange(n)) & (flat >= -1)).all()), "a parent is -1 or a row before its child")
    bits = np.zeros((flat.shape[0], n, max(1, (n + 63) // 64) * 64), bool)
    for i in range(n):
        has = np.nonzero(flat[:, i] >= 0)[0]
        bits[has, i] = bits[has, flat[has, i]]
        bits[:, i, i] = True
    words = np.packbits(bits, axis=-1, bitorder="little").view("<i8")
    words = torch.from_numpy(words.reshape(*p.shape, -1).copy())
    return words.to(parents.device) if torch.is_tensor(parents) else words


def tree_attention(q, cache, pages, cu, lens, out, tree=None, scale=None, max_new=None, max_len=None, lse=None, stream=None):
    """Attention of the batch's new tokens over their sequences' cached positions and, of the new ones (appended already,
    token i at position lens[b] + i), over those their mask allows. q, out (rows, heads, head), heads a multiple of the
    cache's kv_heads. tree (rows, words) int64: bit j of a row allows its sequence's j-th new token; None: each sees those
    before it and itself, so that one new token a sequence is a decode step and many are a prompt. scale: default
    1 / sqrt(head). max_new: at least the most new tokens of a sequence (default: all rows); sequences with more are
    skipped and reported. max_len: about the longest lens[b] + new tokens (default: the page table's reach), which only
    decides how finely the work is split. lse (rows, heads) float32: the log of the sum of exponentials. A row that may
    see nothing gives zeros and lse -inf."""
    torch = _torch()
    qs, os_ = _rows("q", q, None, cache.head), _rows("out", out, None, cache.head)
    n, heads, head = q.shape
    _need(out.shape == q.shape and out.dtype == q.dtype, "out must be like q")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, q, out, tree, lse)
    words = 0
    if tree is not None:
        _need(tree.dtype == torch.int64 and tree.dim() == 2 and tree.shape[0] == n and tree.is_contiguous(),
              f"tree: contiguous int64 ({n}, words) is needed")
        words = tree.shape[1]
    if lse is not None:
        _need(lse.dtype == torch.float32 and tuple(lse.shape) == (n, heads) and lse.is_contiguous(),
              f"lse: contiguous float32 {(n, heads)} is needed")
    reach = pages.shape[1] * cache.page
    _call("mvb_tree_attention", cache.device, stream, q.data_ptr(), qs, *cache.args, *b, n, heads, _TYPES[q.dtype],
          None if tree is None else tree.data_ptr(), words, 1.0 / math.sqrt(head) if scale is None else float(scale),
          n if max_new is None else max_new, reach if max_len is None else max_len, out.data_ptr(), os_,
          None if lse is None else lse.data_ptr())
    return out


LogProbs = namedtuple("LogProbs", "logp entropy top_ids top_logp")


def logprobs(logits, ids=None, top=0, entropy=True, stream=None):
    """Log probabilities under softmax(logits) of each row (rows, vocab; any row stride): of the given tokens `ids`
    (rows, n) int32 (-1: no token, 0.0), the entropy in nats, and the `top` (at most 64) most probable tokens, equal
    logits by the lowest id. Returns LogProbs(logp (rows, n), entropy (rows), top_ids (rows, top) int32, top_logp (rows,
    top)); what was not asked for is None or has no columns. A row that holds a NaN or +inf, or no finite logit, is all
    NaN (its top ids still order the logits, NaN last)."""
    torch = _torch()
    _need(logits.dim() == 2 and logits.dtype in _TYPES, "logits: (rows, vocab) float32, bfloat16 or float16 is needed")
    n, vocab = logits.shape
    _need(logits.stride(1) == 1 or vocab == 1, "logits: the elements of a row must be contiguous")
    dev = logits.device
    nids = 0
    if ids is not None:
        _need(ids.dim() == 2 and ids.shape[0] == n, f"ids: ({n}, count) is needed")
        _int32("ids", ids, tuple(ids.shape))
        nids = ids.shape[1]
    _on(dev, ids)
    with torch.cuda.stream(stream) if stream is not None else _NOTHING:
        logp = torch.empty(n, nids, device=dev) if ids is not None else None
        ent = torch.empty(n, device=dev) if entropy else None
        top_ids = torch.empty(n, top, dtype=torch.int32, device=dev)
        top_logp = torch.empty(n, top, device=dev)
    _call("mvb_logprobs", dev, stream, logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], n, vocab,
          ids.data_ptr() if nids else None, nids, logp.data_ptr() if nids else None,
          None if ent is None else ent.data_ptr(), top, top_ids.data_ptr() if top else None,
          top_logp.data_ptr() if top else None)
    return LogProbs(logp, ent, top_ids, top_logp)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_NOTHING = _Nothing()

#: what serve_status() returns
STATUS = {0: "ok", 1: "a page number out of range", 2: "a length or a row range out of range",
          3: "a rotary position outside its table", 4: "a token id outside the vocabulary"}


def serve_status(stream=None, device=None):
    """Synchronizes `stream` and returns the first thing that the serving operators found out of range on the device since
    the last call (a key of STATUS; 0: nothing), clearing it. Outputs of a call that reported are not to be used."""
    torch = _torch()
    m = _mvb()
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        rc = m.lib().mvb_serve_status(C.c_void_p((torch.cuda.current_stream() if stream is None else stream).cuda_stream))
    if rc < 0:
        m.check(rc, "mvb_serve_status")
    return rc
