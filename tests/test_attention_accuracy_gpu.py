"""How accurate mvb_tree_attention is where weights and value scales spread over many magnitudes: value scales that the mask
hides, outliers of no weight, a key that stands far above a long context, and long contexts in fp32. Against 64 bits, with
a bound for each row from that row's own weights (`bound`)."""
import numpy as np
import pytest

from serving_reference import Case, f64

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "a CUDA device is required"
    t.cuda.set_device(0)
    return t


@pytest.fixture(autouse=True)
def clean_status(request):
    yield
    assert request.getfixturevalue("mvb").serve_status() == 0


def bound(torch, dt, q, k, v, vscale, allowed, scale, together, margin):
    """(outputs, lse, tolerance of the outputs, tolerance of lse) of one sequence and one kv head: q (n, group, d), k, v (t, d),
    vscale (t).

    S, in units of the natural log:
      q in fp16 after a power of two: the row's largest element is at least 2^8 there, a rounding of what is below 2^-14 at
      most 2^-25: 2^-33 max|q| an element; an fp32 q in two parts besides 2^-11 * 2^-11 of each element.
      Exact products, summed by the tensor core in steps of 16, each cut at 2^-23 of the running sum: at most
      (d / 16) * parts * 2^-23 of sum |q k|.
      Four roundings of products (scale * log2 e, times the key's, times S; the argument of exp2): 2^-24 each of S, and of the
      argument, which is |S - max| and up to 12 bits (8.4) that the running maximum may be behind.
    A weight p: exp2's 2 ulp (2^-22) besides; its error moves the output by p * error * (|v| + |out|).
    P' = p * vs in fp16: two roundings of products, then 2^-11 (one part: bf16) or 2^-22 (two parts) of itself, and at most 2^-25
    in units where the largest P' of the accumulator lies at or above 2^(14 - margin): 2^(margin - 39) of that, `together` keys
    sharing an accumulator. The worst that any split makes of it: the largest weights in accumulators of their own.
    Sums: O is cut at 2^-23 of its running sum for every 16 keys and part; a running sum is a difference of two values of the
    cumulative sum. The sum of weights: one rounding a term, in chains of at most together / 8, of signs that do not
    conspire (4 sqrt). Sixteen further roundings where parts are joined.
    The output's rounding: half a step, which below the smallest normal number is that number's (fp16: 2^-14 * 2^-11)."""
    info = torch.finfo(dt)
    n, group, d = q.shape
    t = k.shape[0]
    f32 = dt == torch.float32
    qp, pp = (2 if f32 else 1), (1 if dt == torch.bfloat16 else 2)
    steps = (64 if d <= 64 else 128) // 16
    out, lse = np.zeros_like(q), np.full((n, group), -np.inf)
    tol, lse_tol = np.zeros_like(q), np.zeros((n, group))
    va = np.abs(v)
    ints = np.where(vscale[:, None] > 0, va / np.where(vscale > 0, vscale, 1)[:, None], 0)
    for h in range(group):
        s = np.where(allowed, (q[:, h] @ k.T) * scale, -np.inf)
        top = s.max(-1, keepdims=True)
        ds = (np.abs(q[:, h]) @ np.abs(k).T) * abs(scale) * ((2.0 ** -22 if f32 else 0) + steps * qp * 2.0 ** -23)
        ds += 2.0 ** -33 * np.abs(q[:, h]).max(-1, keepdims=True) * np.abs(k).sum(-1) * abs(scale)
        with np.errstate(invalid="ignore"):
            e = np.where(allowed, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
            rel = np.where(allowed, ds + 4 * 2.0 ** -24 * np.abs(s) + 2.0 ** -24 * (np.abs(s - top) + 9) + 2.0 ** -22, 0)
        z = e.sum(-1, keepdims=True)
        p = e / np.where(z > 0, z, 1)
        out[:, h] = p @ v
        with np.errstate(divide="ignore"):
            lse[:, h] = (np.where(np.isfinite(top), top, 0) + np.log(z))[:, 0]
        sums = 4 * np.sqrt(together / 8 + 64) * 2.0 ** -24 + 16 * 2.0 ** -24
        moved = (p * rel).sum(-1, keepdims=True)
        err = (p * rel) @ va + np.abs(out[:, h]) * (moved + sums) + (2.0 ** -23 + (2.0 ** -11, 2.0 ** -22)[pp - 1]) * (p @ va)
        w = np.sort(p * vscale, -1)[:, ::-1][:, :-(-t // together)]  # the largest weight of each accumulator, at worst
        err += 2.0 ** (margin - 39) * min(together, t) * w.sum(-1, keepdims=True) * ints.max(0)
        pad = -t % 16
        c = np.matmul(np.pad(p, ((0, 0), (0, pad))).reshape(n, -1, 1, 16), np.pad(v, ((0, pad), (0, 0))).reshape(-1, 16, d))
        c = np.cumsum(c[:, :, 0], 1)
        run = np.maximum(c.max(1), 0) - np.minimum(c.min(1), 0)
        err += (together / 16 + 16) * pp * 2.0 ** -23 * run
        tol[:, h] = err + np.maximum(info.eps / 2 * np.abs(out[:, h]), info.smallest_normal * info.eps / 2)
        lse_tol[:, h] = moved[:, 0] + sums + 2.0 ** -22 * np.abs(np.where(np.isfinite(lse[:, h]), lse[:, h], 0)) + 2.0 ** -22
    return out, lse, tol, lse_tol


def check(torch, mvb, c, q, tree_bits=None, scale=None, together=4096, margin=8, **kw):
    """One call against 64 bits; tree_bits (rows, most new) or a causal chain. Returns the worst error in units of its bound."""
    dt, heads = q.dtype, q.shape[1]
    group, sc = heads // c.kv_heads, scale if scale is not None else c.head ** -0.5
    out, lse = torch.full_like(q, 9.0), torch.full((c.rows, heads), 9.0, device="cuda")
    words = None
    if tree_bits is not None:
        wide = np.zeros((c.rows, -(-tree_bits.shape[1] // 64) * 64), bool)
        wide[:, :tree_bits.shape[1]] = tree_bits
        words = torch.from_numpy(np.packbits(wide, axis=1, bitorder="little").view("<i8").copy()).cuda()
    mvb.tree_attention(q, c.cache, *c.batch(), out, tree=words, scale=scale, lse=lse, max_new=int(c.new.max()), **kw)
    worst = 0.0
    vs = c.cache.vs.cpu().numpy().astype(np.float64)
    for b in range(len(c.lens)):
        ctx, n, r0 = int(c.lens[b]), int(c.new[b]), int(c.cu[b])
        if not n:
            continue
        allowed = np.ones((n, ctx + n), bool)
        allowed[:, ctx:] = np.tril(np.ones((n, n), bool)) if tree_bits is None else tree_bits[r0:r0 + n, :n]
        k, v = c.values(b, ctx + n, 0), c.values(b, ctx + n, 1)
        p = np.arange(ctx + n)
        for h in range(c.kv_heads):
            at = slice(h * group, (h + 1) * group)
            want, want_lse, tol, lse_tol = bound(
                torch, dt, f64(q)[r0:r0 + n, at], k[:, h], v[:, h], vs[c.pages[b, p // c.page], h, p % c.page], allowed, sc,
                together, margin if dt != torch.bfloat16 else 12)
            off = np.abs(f64(out)[r0:r0 + n, at] - want)
            with np.errstate(invalid="ignore", divide="ignore"):
                worst = max(worst, np.nan_to_num(off / tol, nan=0.0, posinf=1e9).max())
            assert np.all(off <= tol), (b, h, worst, off.max(), np.abs(want).max())
            seen = allowed.any(1)
            assert np.all(np.abs(f64(lse)[r0:r0 + n, at] - want_lse)[seen] <= lse_tol[seen])
    return worst, out


KINDS = [(2, 64, 3), (2, 128, 3), (7, 64, 3), (7, 128, 3), (7, 64, 9), (7, 64, 40), (7, 128, 40), (7, 64, 60), (7, 128, 60)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,head,tokens", KINDS)
def test_hidden_value_scales(torch, mvb, dtype, bits, heads, head, tokens):
    """A new token whose value scale is finite but large is nothing to the rows that its mask hides it from: the same bits; and
    the row that sees it is right."""
    c = Case(torch, mvb, [2000], [tokens], 1, head, bits, 16, seed=heads)
    torch.manual_seed(tokens)
    q = (torch.randn(tokens, heads, head, device="cuda") * 2).to(getattr(torch, dtype))
    see = np.eye(tokens, dtype=bool)
    _, clean = check(torch, mvb, c, q, see)
    slot = (int(c.pages[0, 2001 // 16]), slice(None), 2001 % 16)
    others = [i for i in range(tokens) if i != 1]
    most = 1e30 if dtype != "float16" else 0.0
    for bad in (1e3, 1e6, 1e30):
        c.cache.vs[slot] = bad
        if bad <= most:
            _, out = check(torch, mvb, c, q, see)
        else:  # the row that sees it leaves fp16's range
            out = torch.empty_like(q)
            words = torch.from_numpy(np.packbits(np.pad(see, ((0, 0), (0, 64 - tokens))), axis=1,
                                                 bitorder="little").view("<i8").copy()).cuda()
            mvb.tree_attention(q, c.cache, *c.batch(), out, tree=words, max_new=tokens)
        assert torch.equal(out[others], clean[others])


def dominant(torch, c, rows, heads, dtype, nats, value, at=0, above=0.0):
    """Queries near one direction and a cache in which position `at` scores about `nats` above keys of `above` +- 0.3; its value
    row has `value` times the others' scale. Returns the queries."""
    g = np.random.default_rng(int(abs(nats) * 10) + rows)
    d = c.head
    u = g.standard_normal(d)
    u /= np.abs(u).max()
    q = np.broadcast_to(u, (rows, heads, d)) * (1 + 0.02 * g.standard_normal((rows, heads, 1)))
    q = q + 0.01 * g.standard_normal((rows, heads, d))
    most = 127 if c.bits == 8 else 7
    rounded = np.rint(u * most) * np.sign(nats)
    per = float(rounded @ u) * d ** -0.5  # a score for each unit of that key's scale
    s = c.s_np[0].copy()
    # other keys: scores of +- 0.3
    size = np.nanmean(s) * (40 if c.bits == 8 else 2.5) * np.linalg.norm(u) * d ** -0.5
    s *= 0.3 / size
    pg, sl = int(c.pages[0, at // c.page]), at % c.page
    kq = c.q_np[0].copy()
    packed = rounded.astype(np.int8)
    if c.bits == 4:
        x = (packed & 15).astype(np.uint8)
        packed = x[0::2] | (x[1::2] << 4)
    kq[pg, :, sl] = packed
    s[pg, :, sl] = nats / per
    v = c.s_np[1].copy()
    v[pg, :, sl] *= value
    for t, a in ((c.cache.kq, kq), (c.cache.ks, s.astype(np.float32)), (c.cache.vs, v.astype(np.float32))):
        t.copy_(torch.from_numpy(a))
    return torch.from_numpy(q).cuda().to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,head,tokens", [(4, 64, 1), (4, 128, 2), (6, 128, 3), (4, 128, 12), (3, 64, 50)])
@pytest.mark.parametrize("value", [0.0, 1e-3, 1.0])
@pytest.mark.parametrize("nats", [4.0, 8.0, 12.0, 16.0])
def test_dominant_key(torch, mvb, dtype, heads, head, tokens, value, nats):
    """The first token of a trained decoder's context: far above the other keys, its value near zero or not."""
    c = Case(torch, mvb, [16000], [tokens], 1, head, 8, 64, seed=head)
    q = dominant(torch, c, tokens, heads, dtype, nats, value)
    check(torch, mvb, c, q, max_len=16000 + tokens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,tokens", [(4, 1), (4, 5), (4, 12), (4, 50)])
@pytest.mark.parametrize("at", [9000, 15990])
def test_late_dominant_key(torch, mvb, dtype, heads, tokens, at):
    """The same inside and at the end of a context: what was summed before it keeps its share."""
    c = Case(torch, mvb, [16000], [tokens], 1, 128, 4, 32, seed=at)
    q = dominant(torch, c, tokens, heads, dtype, 14.0, 1e-4, at=at)
    check(torch, mvb, c, q, max_len=16000 + tokens)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("heads,head,tokens", [(4, 64, 1), (4, 128, 3), (4, 128, 6), (4, 64, 12), (4, 128, 20)])
@pytest.mark.parametrize("nats", [12.0, 16.0, 18.0])
def test_dominant_key_above_equal_ones(torch, mvb, dtype, heads, head, tokens, nats):
    """The other keys weigh alike, so that what a weight is off by does not average out, in one CTA; the dominant value is zero
    in half of its elements, where the others are all there is."""
    c = Case(torch, mvb, [4000], [tokens], 1, head, 8, 64, seed=head)
    q = dominant(torch, c, tokens, heads, dtype, nats, 1.0)
    pg = int(c.pages[0, 0])
    top = c.cache.kq[pg, :, 0].clone()
    c.cache.kq.zero_()
    c.cache.kq[pg, :, 0] = top
    c.cache.vq.copy_(c.cache.vq.abs().clamp(min=20))
    c.cache.vq[pg, :, 0, ::2] = 0
    c.cache.vs.copy_(torch.where(c.cache.vs.isnan(), c.cache.vs, torch.full_like(c.cache.vs, 0.5)))
    check(torch, mvb, c, q, together=4000, max_len=16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,head,tokens", [(4, 64, 1), (4, 128, 5), (4, 128, 12), (3, 64, 50), (3, 128, 100)])
def test_value_outliers(torch, mvb, dtype, heads, head, tokens):
    """Value scales over 2^24 of range, and a huge one on a key of no weight."""
    c = Case(torch, mvb, [3000], [tokens], 1, head, 8, 16, seed=3)
    torch.manual_seed(0)
    q = torch.randn(tokens, heads, head, device="cuda").to(getattr(torch, dtype))
    c.cache.vs.mul_(torch.exp2(torch.randint(-12, 1, c.cache.vs.shape, device="cuda").float()))
    check(torch, mvb, c, q)
    c = Case(torch, mvb, [3000], [tokens], 1, head, 8, 16, seed=4)
    q = dominant(torch, c, tokens, heads, dtype, -40.0, 2.0 ** 24, at=700)
    check(torch, mvb, c, q)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("ctx,heads,kv_heads,head,tokens", [
    (20000, 4, 1, 128, 1), (20000, 4, 2, 64, 12), (20000, 4, 2, 128, 30), (20000, 2, 1, 64, 40), (130000, 2, 1, 128, 2),
    (130000, 1, 1, 128, 30)])
def test_long_fp32(torch, mvb, bits, ctx, heads, kv_heads, head, tokens):
    """fp32 callers over long contexts: no whole tile, and no second part of q or of P, can be missing."""
    c = Case(torch, mvb, [ctx], [tokens], kv_heads, head, bits, 64, seed=tokens)
    torch.manual_seed(1)
    q = torch.randn(tokens, heads, head, device="cuda") * 2
    check(torch, mvb, c, q, together=4096, max_len=ctx + tokens)


@pytest.mark.parametrize("dtype,ctx,span", [("float32", 60000, 16), ("float16", 60000, 128), ("bfloat16", 60000, 128)])
@pytest.mark.parametrize("heads,head,tokens", [(1, 64, 30), (1, 128, 40), (3, 64, 60), (3, 128, 60)])
@pytest.mark.parametrize("max_len", [16, 60100])
def test_sums_do_not_drift(torch, mvb, dtype, ctx, span, heads, head, tokens, max_len):
    """Values of one sign, whose sums the tensor core cuts in one direction: what is lost stays that of one span of keys, however
    many a CTA has, so that max_len decides the split alone. (The sums of the spans, 60 at most, are rounded to nearest: within
    the bound's roundings of a join.)"""
    c = Case(torch, mvb, [ctx], [tokens], 1, head, 8, 64, seed=tokens)
    torch.manual_seed(2)
    c.cache.vq.copy_(c.cache.vq.abs().clamp(min=30))
    q = (torch.randn(tokens, heads, head, device="cuda")).to(getattr(torch, dtype))
    check(torch, mvb, c, q, together=64 * span, max_len=max_len)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,head,tokens", [(4, 64, 1), (4, 128, 5), (3, 64, 50), (3, 128, 100)])
@pytest.mark.parametrize("nats", [1e4, 3e6, 4e7, 1e9, 1e12, -1e9])
def test_huge_scores(torch, mvb, dtype, heads, head, tokens, nats):
    """One key far above all others, by more than fp32 can tell a score from the next (or all others far above one, and alike
    but for their values): the row is that key's value."""
    c = Case(torch, mvb, [900], [tokens], 1, head, 8, 64, seed=head)
    q = dominant(torch, c, tokens, heads, dtype, nats, 1.0, at=500)
    out, lse = torch.empty_like(q), torch.empty(tokens, heads, device="cuda")
    mvb.tree_attention(q, c.cache, *c.batch(), out, max_new=tokens, lse=lse)
    if nats < 0:
        keep = c.cache.ks[int(c.pages[0, 7]), :, 500 % 64].clone()
        assert float(keep.max()) > 0
        check(torch, mvb, c, q)
        return
    v = c.values(0, 501, 1)[500, 0]
    half = torch.finfo(q.dtype).eps / 2
    # P's parts; a score above 2^24 leaves its unit no whole number next to it but itself, so that P' is the value scale, held in
    # steps of at most 2^-24
    vs = float(c.cache.vs[int(c.pages[0, 500 // 64]), 0, 500 % 64])
    p = max(2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -22, 2.0 ** -25 / vs if nats > 2 ** 23 else 0.0)
    assert np.all(np.abs(f64(out) - v) <= (half + p + 2.0 ** -21) * np.abs(v))
    k = c.values(0, 501, 0)[500, 0]
    want = f64(q) @ k * head ** -0.5
    # q's parts, the cut sums of at most 128 products, the scale's four roundings: all relative to sum |q k|, here the score
    assert np.all(np.abs(f64(lse) - want) <= 2.0 ** -18 * np.abs(want))
