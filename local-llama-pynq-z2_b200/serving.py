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
device; they keep no state, and memory that a call needs is its own, so calls on several streams do not meet, but for the
device's one serve_status().
"""
import ctypes as C
import math
import sys
from collections import namedtuple

_TYPES = {}     # torch element types -> the library's codes; filled with _T, the torch module, by _torch()
_T = None
_raw_stream = None


def _torch():
    """torch, imported at the first use (the package itself does not need it)."""
    global _T, _raw_stream
    if _T is None:
        import torch
        _TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _T = torch
    return _T


def _mvb():
    return sys.modules[__package__]


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _call(name, device, stream, *args):
    """One library call on `device` (made current for it) and `stream`. These calls take a few microseconds on the device
    for a single token, so the host side is kept short: no formatted text before a check has failed, no stream object."""
    m = _mvb()
    f = getattr(m.lib(), name)
    index = device.index
    handle = _raw_stream(index) if stream is None else stream.cuda_stream
    if _T.cuda.current_device() == index:
        rc = f(*args, handle)
    else:
        with _T.cuda.device(device):
            rc = f(*args, handle)
    if rc != 0:
        m.check(rc, name)


def _on(device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}: one device is needed")
    if device.type != "cuda":
        raise ValueError(f"CUDA tensors are needed, not {device.type}")


def _rows(name, t, heads, head):
    """Checks a (rows, heads, head) tensor whose heads lie next to one another; its row stride."""
    shape = t.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or (head is not None and shape[2] != head):
        raise ValueError(f"{name} is {tuple(shape)}: (rows, {heads or 'heads'}, {head or 'head'}) is needed")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and shape[2] != 1) or (s1 != shape[2] and shape[1] != 1):
        raise ValueError(f"{name}: the heads of a row must be contiguous")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} is {t.dtype}: float32, bfloat16 or float16 is needed")
    return s0 if shape[0] > 1 else shape[1] * shape[2]  # a single row's stride says nothing


def _out_rows(name, t, heads, head):
    """_rows of a tensor that is written: its rows must not share memory (an expanded one's do)."""
    stride = _rows(name, t, heads, head)
    if stride < t.shape[1] * t.shape[2]:
        raise ValueError(f"{name}: rows {stride} elements apart overlap")
    return stride


def _int32(name, t, *shape):
    if t.dtype is not _T.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)}: contiguous int32 {shape} is needed")


class KvCache:
    """A layer's paged cache: kq, vq (pages, kv_heads, page, head) int8 or (.., head / 2) uint8 of nibbles (element 2i
    low, two's complement), ks, vs (pages, kv_heads, page) float32. value = integer * scale. Only views are kept."""

    __slots__ = ("kq", "ks", "vq", "vs", "pages", "kv_heads", "page", "head", "bits", "device", "args")

    def __init__(self, kq, ks, vq, vs):
        torch = _T or _torch()
        shape = kq.shape
        self.bits = bits = {torch.int8: 8, torch.uint8: 4}.get(kq.dtype, 0)
        if len(shape) != 4 or not bits:
            raise ValueError("kq: (pages, kv_heads, page, head) int8, or uint8 with two elements a byte, is needed")
        if vq.shape != shape or vq.dtype is not kq.dtype:
            raise ValueError("vq must be like kq")
        for t in (ks, vs):
            if t.shape != shape[:3] or t.dtype is not torch.float32:
                raise ValueError(f"ks and vs must be float32 {tuple(shape[:3])}")
        if not (kq.is_contiguous() and vq.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
            raise ValueError("the cache's tensors must be contiguous")
        self.device = device = kq.device
        _on(device, ks, vq, vs)
        self.kq, self.ks, self.vq, self.vs = kq, ks, vq, vs
        self.pages, self.kv_heads, self.page, width = shape
        self.head = width if bits == 8 else 2 * width
        self.args = (kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), self.pages, self.page, self.kv_heads,
                     self.head, bits)

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
    shape = pages.shape
    if len(shape) != 2:
        raise ValueError("pages: (batch, columns) is needed")
    b, cols = shape
    _int32("pages", pages, b, cols)
    _int32("cu", cu, b + 1)
    _int32("lens", lens, b)
    return pages.data_ptr(), cols, cu.data_ptr(), lens.data_ptr(), b


_LAYOUTS = {"half": 0, "pairs": 1}


def _layout(layout):
    if layout not in _LAYOUTS:
        raise ValueError(f"layout={layout!r}: 'half' or 'pairs' is needed")
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
    lo, hi = max(math.floor(turn(fast)), 0), min(math.ceil(turn(slow)), rot - 1)  # hi may lie behind the last pair
    keep = 1 - np.clip((np.arange(half) - lo) / max(hi - lo, 1e-3), 0, 1)
    return f / factor * (1 - keep) + f * keep, (0.1 * math.log(factor) + 1 if factor > 1 else 1.0)


def rope_table(frequencies, positions, out=None, start=0, factor=1.0, device="cuda", stream=None):
    """(positions, rot) float32: row p holds factor * cos of the rot / 2 angles (start + p) * frequencies, then factor *
    sin, angles and functions in 64 bits. frequencies: float64, numpy or a CUDA tensor."""
    torch = _torch()
    if stream is not None:  # what is made here belongs to the stream that uses it
        with torch.cuda.stream(stream):
            return rope_table(frequencies, positions, out, start, factor, device)
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
    _call("mvb_rope_table", out.device, None, frequencies.data_ptr(), out.data_ptr(), half, positions, start,
          float(factor))
    return out


def _table(table):
    if table.dtype is not _T.float32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("rope table: contiguous float32 (positions, rot) is needed")
    return table.shape


def rope(x, positions, table, out=None, layout="half", stream=None):
    """x (tokens, heads, head) with the first rot elements of each head turned by the table's row of the token's position;
    the other elements as they are. layout "half": pairs (i, i + rot / 2); "pairs": (2i, 2i + 1). out: x's shape and
    type, x itself for in place (the default); it must not overlap x otherwise."""
    _T or _torch()
    out = x if out is None else out
    xs = _rows("x", x, None, None)
    n, heads, head = x.shape
    os_ = _out_rows("out", out, heads, head)
    if out.dtype is not x.dtype or out.shape[0] != n:
        raise ValueError("out must be like x")
    _int32("positions", positions, n)
    reach, rot = _table(table)
    device = x.device
    _on(device, out, positions, table)
    _call("mvb_rope", device, stream, x.data_ptr(), positions.data_ptr(), table.data_ptr(), out.data_ptr(),
          _TYPES[x.dtype], n, heads, head, rot, reach, _layout(layout), xs, os_)
    return out


def kv_append(cache, k, v, pages, cu, lens, positions=None, rope=None, layout="half", q=None, q_out=None, stream=None):
    """The batch's new keys and values (rows, kv_heads, head) quantized into the cache at their sequences' positions
    lens[b] and on: scale = max |x| / 127 (or / 7), integers rounded to nearest even. With a rope table the keys are
    turned first (and q into q_out, rows of queries, in the same launch; q_out may be q) by the rows' `positions`
    (int32; default the position in the cache; a tree's are those of its depth). A row with an infinity or a NaN is held
    with the scale NaN. Sequences must not share a page that the call writes."""
    _T or _torch()
    ks, vs = _rows("k", k, cache.kv_heads, cache.head), _rows("v", v, cache.kv_heads, cache.head)
    n, dtype = k.shape[0], k.dtype
    if v.shape[0] != n or v.dtype is not dtype:
        raise ValueError("v must be like k")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, k, v, pages, cu, lens, positions, rope, q, q_out)
    pos = table = qp = qop = None
    reach = rot = qs = qos = heads = 0
    if rope is not None:
        reach, rot = _table(rope)
        table = rope.data_ptr()
    if positions is not None:
        if rope is None:
            raise ValueError("positions without a rope table")
        _int32("positions", positions, n)
        pos = positions.data_ptr()
    if q is not None:
        if rope is None or q_out is None:
            raise ValueError("queries need a rope table and q_out")
        qs, heads = _rows("q", q, None, cache.head), q.shape[1]
        qos = _out_rows("q_out", q_out, heads, cache.head)
        if q.shape[0] != n or q_out.shape[0] != n or q.dtype is not dtype or q_out.dtype is not dtype:
            raise ValueError("q and q_out must have k's rows and type")
        qp, qop = q.data_ptr(), q_out.data_ptr()
    _call("mvb_kv_append", cache.device, stream, *cache.args, *b, n, k.data_ptr(), ks, v.data_ptr(), vs, _TYPES[dtype],
          table, pos, rot, reach, _layout(layout), qp, qs, qop, qos, heads)


def kv_read(cache, pages, cu, lens, k_out, v_out, stream=None):
    """Cached keys and values back: rows cu[b] .. cu[b + 1] - 1 of k_out and v_out (rows, kv_heads, head; float32,
    bfloat16 or float16) become sequence b's positions lens[b] and on (lens of zeros and cu of running lengths: whole
    contexts). integer * scale, rounded to the output's type."""
    _T or _torch()
    ks, vs = (_out_rows(name, t, cache.kv_heads, cache.head) for name, t in (("k_out", k_out), ("v_out", v_out)))
    n = k_out.shape[0]
    if v_out.shape[0] != n or v_out.dtype is not k_out.dtype:
        raise ValueError("v_out must be like k_out")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, k_out, v_out, pages, cu, lens)
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
    words = torch.from_numpy(words.reshape(*p.shape, bits.shape[-1] // 64).copy())
    return words.to(parents.device) if torch.is_tensor(parents) else words


def tree_attention(q, cache, pages, cu, lens, out, tree=None, scale=None, max_new=None, max_len=None, lse=None, stream=None):
    """Attention of the batch's new tokens over their sequences' cached positions and, of the new ones (appended already,
    token i at position lens[b] + i), over those their mask allows. q, out (rows, heads, head; out may be q), heads a multiple
    of the cache's kv_heads. tree (rows, words) int64: bit j of a row allows its sequence's j-th new token; None: each sees those
    before it and itself, so that one new token a sequence is a decode step and many are a prompt. scale: default
    1 / sqrt(head). max_new: at least the most new tokens of a sequence (default: all rows, or the page table's reach where
    that is less; ceil(max_new * heads / kv_heads / 128) * kv_heads <= 65535); sequences with more are skipped and reported. max_len: about the longest lens[b] + new tokens (default: the page table's reach), which only
    decides how finely the work is split. lse (rows, heads) float32: the log of the sum of exponentials. A row that may
    see nothing gives zeros and lse -inf."""
    _T or _torch()
    qs, os_ = _rows("q", q, None, cache.head), _out_rows("out", out, None, cache.head)
    n, heads, head = shape = q.shape
    dtype = q.dtype
    if out.shape != shape or out.dtype is not dtype:
        raise ValueError("out must be like q")
    b = _batch(cache, pages, cu, lens)
    _on(cache.device, q, out, pages, cu, lens, tree, lse)
    words, tp, lp = 0, None, None
    if tree is not None:
        if tree.dtype is not _T.int64 or tree.dim() != 2 or tree.shape[0] != n or not tree.is_contiguous():
            raise ValueError(f"tree: contiguous int64 ({n}, words) is needed")
        words, tp = tree.shape[1], tree.data_ptr()
    if lse is not None:
        if lse.dtype is not _T.float32 or lse.shape != (n, heads) or not lse.is_contiguous():
            raise ValueError(f"lse: contiguous float32 {(n, heads)} is needed")
        lp = lse.data_ptr()
    max_new = min(n, b[1] * cache.page) if max_new is None else max_new
    max_len = b[1] * cache.page if max_len is None else max_len
    work, wp, wn = None, None, 0
    if b[4] * cache.kv_heads <= 18 and max_len >= 16384:  # few jobs, long contexts: a workspace may help
        wn = _mvb().lib().mvb_tree_attention_work(n, heads, cache.kv_heads, head, b[4], max_new, max_len)
        if wn:
            if stream is None:
                work = _T.empty(wn, dtype=_T.uint8, device=cache.device)
            else:  # memory of the stream that uses it
                with _T.cuda.stream(stream):
                    work = _T.empty(wn, dtype=_T.uint8, device=cache.device)
            wp = work.data_ptr()
    _call("mvb_tree_attention", cache.device, stream, q.data_ptr(), qs, *cache.args, *b, n, heads, _TYPES[dtype], tp, words,
          head ** -0.5 if scale is None else float(scale), max_new, max_len, out.data_ptr(), os_, lp, wp, wn)
    return out


LogProbs = namedtuple("LogProbs", "logp entropy top_ids top_logp")


def logprobs(logits, ids=None, top=0, entropy=True, stream=None):
    """Log probabilities under softmax(logits) of each row (rows, vocab; any row stride): of the given tokens `ids`
    (rows, n) int32 (-1: no token, 0.0), the entropy in nats, and the `top` (at most 64) most probable tokens, equal
    logits by the lowest id. Returns LogProbs(logp (rows, n), entropy (rows), top_ids (rows, top) int32, top_logp (rows,
    top)); what was not asked for is None or has no columns. A row that holds a NaN or +inf, or no finite logit, is all
    NaN (its top ids still order the logits, NaN last)."""
    torch = _T or _torch()
    if logits.dim() != 2 or logits.dtype not in _TYPES:
        raise ValueError("logits: (rows, vocab) float32, bfloat16 or float16 is needed")
    n, vocab = logits.shape
    stride, one = logits.stride()
    if one != 1 and vocab != 1:
        raise ValueError("logits: the elements of a row must be contiguous")
    dev = logits.device
    _on(dev, ids)
    nids, ip = 0, None
    if ids is not None:
        if ids.dim() != 2:
            raise ValueError(f"ids: ({n}, count) is needed")
        nids = ids.shape[1]
        _int32("ids", ids, n, nids)
        ip = ids.data_ptr() if nids else None
    if stream is None:
        out = _results(torch, dev, n, nids, top, ids is not None, entropy)
    else:  # memory of the stream that writes it
        with torch.cuda.stream(stream):
            out = _results(torch, dev, n, nids, top, ids is not None, entropy)
    logp, ent, top_ids, top_logp = out
    _call("mvb_logprobs", dev, stream, logits.data_ptr(), stride, _TYPES[logits.dtype], n, vocab, ip, nids,
          logp.data_ptr() if nids else None, ent.data_ptr() if entropy else None, top,
          top_ids.data_ptr() if top else None, top_logp.data_ptr() if top else None)
    return out


def _results(torch, dev, n, nids, top, has_ids, entropy):
    f32 = torch.float32
    return LogProbs(torch.empty((n, nids), dtype=f32, device=dev) if has_ids else None,
                    torch.empty((n,), dtype=f32, device=dev) if entropy else None,
                    torch.empty((n, top), dtype=torch.int32, device=dev),
                    torch.empty((n, top), dtype=f32, device=dev))


#: what serve_status() returns
STATUS = {0: "ok", 1: "a page number out of range", 2: "a length or a row range out of range",
          3: "a rotary position outside its table", 4: "a token id outside the vocabulary",
          5: "a wait inside a kernel that gave up (a fault of the library or the device)"}


def serve_status(stream=None, device=None):
    """Synchronizes `stream` and returns what the serving operators found out of range on the device since the last call (a
    key of STATUS; 0: nothing), clearing it. Outputs of a call that reported are not to be used. The report is the device's, not
    the stream's: ask in one place, after the streams whose calls it answers for."""
    torch = _torch()
    m = _mvb()
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        rc = m.lib().mvb_serve_status(C.c_void_p((torch.cuda.current_stream() if stream is None else stream).cuda_stream))
    if rc < 0:
        m.check(rc, "mvb_serve_status")
    return rc
