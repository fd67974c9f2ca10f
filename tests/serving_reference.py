"""Plain forms of the serving operators in 64 bits (numpy), and batches to run them on."""
import numpy as np


def f64(t):
    return t.detach().cpu().double().numpy()


def rope(x, pos, table, layout):
    """x (rows, heads, head) float64; table (positions, rot) float64."""
    rot = table.shape[1]
    y = x.copy()
    c, s = table[pos][:, None, :rot // 2], table[pos][:, None, rot // 2:]
    if layout == "half":
        i0, i1 = np.arange(rot // 2), np.arange(rot // 2) + rot // 2
    else:
        i0, i1 = np.arange(0, rot, 2), np.arange(1, rot, 2)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def quantize(x, bits):
    """Rows of float64 -> integers and fp32 scales (as float64)."""
    most = 127 if bits == 8 else 7
    scale = (np.abs(x).max(-1) / most).astype(np.float32).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(scale[..., None] > 0, np.rint(x / scale[..., None]), 0)
    return np.clip(q, -most, most), scale


def unpack(q, bits):
    """Cache integers (numpy int8, or uint8 nibbles) -> float64."""
    if bits == 8:
        return q.astype(np.float64)
    u = np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1).astype(np.int64)
    return np.where(u > 7, u - 16, u).astype(np.float64)


def slots(pages, cu, lens, page):
    """(page, slot) of every row below cu[-1]."""
    out = []
    for b in range(len(lens)):
        for i in range(cu[b + 1] - cu[b]):
            p = lens[b] + i
            out.append((pages[b, p // page], p % page))
    return np.array(out, dtype=np.int64).reshape(-1, 2)


def attention(q, k, v, allowed, scale):
    """One sequence: q (n, heads, d), k, v (t, kv, d), allowed (n, t) -> out, lse."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out, lse = np.zeros_like(q), np.full((n, heads), -np.inf)
    for h in range(heads):
        with np.errstate(invalid="ignore"):
            x = np.where(allowed, (q[:, h] @ k[:, h // group].T) * scale, -np.inf)
        m = x.max(-1, keepdims=True) if x.shape[1] else np.full((n, 1), -np.inf)
        m0 = np.where(np.isinf(m), 0, m)
        e = np.where(allowed, np.exp(x - m0), 0)
        z = e.sum(-1, keepdims=True)
        with np.errstate(divide="ignore"):
            lse[:, h] = (m0 + np.log(z))[:, 0]
        out[:, h] = e @ v[:, h // group] / np.where(z > 0, z, 1)
    return out, lse


class Case:
    """A batch with its cache on the GPU: sequences of given cached and new lengths, pages in random order, slots behind
    the lengths filled with NaN scales."""

    def __init__(self, torch, mvb, lens, new, kv_heads, head, bits, page, seed=0, spare=3, pad_rows=0):
        self.torch, self.mvb, self.bits, self.page = torch, mvb, bits, page
        self.lens, self.new = np.array(lens, np.int32), np.array(new, np.int32)
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + pad_rows
        self.kv_heads, self.head = kv_heads, head
        rng = self.rng = np.random.default_rng(seed)
        need = [-(-(int(a) + int(b)) // page) for a, b in zip(lens, new)]
        total = sum(need) + spare
        order = rng.permutation(total).astype(np.int32)
        self.pages = np.full((len(lens), max(max(need), 1) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.pages[b, :n] = order[at:at + n]
            at += n
        most, size = (127, 40.0) if bits == 8 else (7, 2.5)
        shape = (total, kv_heads, page, head)
        self.q_np, self.s_np = [], []
        for _ in "kv":
            q = np.clip(np.rint(rng.standard_normal(shape) * size), -most, most).astype(np.int8)
            s = (rng.uniform(0.5, 1.5, shape[:3]) / size).astype(np.float32)
            keep = np.zeros(shape[:1] + shape[2:3], bool)
            for b in range(len(lens)):
                p = np.arange(int(lens[b]) + int(new[b]))
                keep[self.pages[b, p // page], p % page] = True
            s = np.where(keep[:, None, :], s, np.float32(np.nan))
            if bits == 4:
                u = (q & 15).astype(np.uint8)
                q = u[..., 0::2] | (u[..., 1::2] << 4)
            self.q_np.append(q)
            self.s_np.append(s)
        cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.cu_, self.lens_, self.pages_ = cu(self.cu), cu(self.lens), cu(self.pages)
        self.cache = mvb.KvCache(cu(self.q_np[0]), cu(self.s_np[0]), cu(self.q_np[1]), cu(self.s_np[1]))

    def batch(self):
        return self.pages_, self.cu_, self.lens_

    def values(self, b, n, which):
        """The first n positions of sequence b: (n, kv_heads, head) float64, from the cache as it is now."""
        q = (self.cache.kq, self.cache.vq)[which].cpu().numpy()
        s = (self.cache.ks, self.cache.vs)[which].cpu().numpy()
        p = np.arange(n)
        pg, sl = self.pages[b, p // self.page], p % self.page
        return unpack(q[pg, :, sl], self.bits) * s[pg, :, sl].astype(np.float64)[..., None]
