"""GPU tests of the 4-bit key / value cache: kv4_append, kv4_read and kv4_attention against plain forms in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Case:
    """A pool filled with stale contents (codes at random, params NaN where `dirty`), a scattered table, and the call's tokens."""

    def __init__(self, lens, new, heads, dim, group, page, seed=0, dirty=True, spare=3, pad_tokens=0):
        from oxicuda_b200 import ops
        self.lens_l, self.new_l, self.heads, self.dim, self.group, self.page = list(lens), list(new), heads, dim, group, page
        g = self.g = _gen(seed)
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g, device="cuda").cpu().tolist()
        wide = max(need + [1]) + 1
        table = torch.full((len(lens), wide), -7, dtype=torch.int32)          # entries that no token needs name no page
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table = table.cuda()
        self.lens = torch.tensor(self.lens_l, dtype=torch.int32, device="cuda")
        self.cu_l = [0]
        for n in self.new_l:
            self.cu_l.append(self.cu_l[-1] + n)
        self.cu = torch.tensor(self.cu_l, dtype=torch.int32, device="cuda")
        self.tokens = self.cu_l[-1] + pad_tokens
        shape = (self.pages, heads, page)
        mk = lambda: torch.randint(0, 256, shape + (dim // 2,), dtype=torch.uint8, device="cuda", generator=g)  # noqa: E731
        par = lambda: torch.full(shape + (dim // group, 2), float("nan") if dirty else 0.5, dtype=torch.float16, device="cuda")  # noqa: E731
        self.cache = ops.Kv4Cache(mk(), par(), mk(), par())

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=self.g).to(dtype)

    def place(self, b, pos):
        """(pages, slots) of positions `pos` of sequence b."""
        return self.table[b].long()[pos // self.page], pos % self.page

    def fill(self):
        """Every token of every sequence gets a value, through the plain quantizer; returns nothing."""
        for b, n in enumerate(self.lens_l):
            if n <= 0:
                continue
            pg, sl = self.place(b, torch.arange(n, device="cuda"))
            for keys in (True, False):
                x = self.normal(n, self.heads, self.dim) * (2.0 if keys else 0.7) + 0.3
                x[:, :, 3] *= 6.0
                codes, params = quantize(x, self.group)
                c, p = (self.cache.k_codes, self.cache.k_params) if keys else (self.cache.v_codes, self.cache.v_params)
                c[pg, :, sl] = pack(codes, keys)
                p[pg, :, sl] = params

    def rows(self, b, keys):
        """All tokens of sequence b as f64 [len, heads, dim], straight from the definition of the layout."""
        n = max(self.lens_l[b], 0)
        pg, sl = self.place(b, torch.arange(n, device="cuda"))
        c, p = (self.cache.k_codes, self.cache.k_params) if keys else (self.cache.v_codes, self.cache.v_params)
        return decode(c[pg, :, sl], p[pg, :, sl], keys)


def quantize(x, group):
    """The definition in f32: x [..., dim] -> codes int64, params f16 [..., dim / group, 2]."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504, 65504)
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, m = ((hi - lo) / torch.full_like(hi, 15)).half(), lo.half()      # a true division: by a Python number it is a product with 1 / 15
    c = torch.where(s > 0, torch.round((g - m.float()) / s.float()).clamp(0, 15), torch.zeros_like(g))
    return c.flatten(-2).long(), torch.cat([s, m], -1)


def order(dim, keys):
    """order[p] = the natural word at place p of a row."""
    if keys:
        return [4 * i + c for c in range(4) for i in range(dim // 32)]
    return [8 * i + r for r in range(8) for i in range(dim // 64)]


def pack(codes, keys):
    w = codes.unflatten(-1, (-1, 8))[..., order(codes.shape[-1], keys), :].flatten(-2)
    return (w[..., 0::2] | (w[..., 1::2] << 4)).to(torch.uint8)


def decode(packed, params, keys):
    """bytes and params -> f64 values."""
    dim = packed.shape[-1] * 2
    nib = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))
    nat = torch.empty_like(nib)
    nat[..., order(dim, keys), :] = nib
    g = nat.flatten(-2).double().unflatten(-1, (params.shape[-2], -1))
    return (g * params[..., :1].double() + params[..., 1:].double()).flatten(-2)


DIMS = [(64, 64), (128, 64), (128, 128)]


# ------------------------------------------------------------------------------------------- append, read

@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,page,lens,new,pad", [
    (1, 16, [1], [1], 0), (3, 32, [5, 0, 33, 17], [5, 0, 1, 17], 0), (8, 64, [64, 65, 200], [2, 65, 3], 5),
    (2, 16, [2, 40], [5, 7], 1),                       # more tokens than positions: the first three have no place
    (5, 128, [300] * 40, [9] * 40, 0)])
def test_append_then_read(dim, group, dtype, heads, page, lens, new, pad):
    """Codes and params equal the f32 definition bit for bit, nothing else in the pool changes, and reading gives c * s + m rounded once."""
    from oxicuda_b200 import ops
    c = Case(lens, new, heads, dim, group, page, seed=len(lens), pad_tokens=pad)
    x = c.normal(c.tokens, 2 * heads + 3, dim) * 3
    x[:, :, 1] = 0.25                                   # a constant element, and in one row a constant group
    x[0, :, :] = 1.5
    x = x.to(DT[dtype])
    k, v = x[:, 3:3 + heads], x[:, 3 + heads:]          # columns of a wider product
    want = [t.clone() for t in (c.cache.k_codes, c.cache.k_params, c.cache.v_codes, c.cache.v_params)]
    for b, n in enumerate(new):
        pos = torch.arange(lens[b] - n, lens[b], device="cuda")
        ok = pos >= 0
        pg, sl = c.place(b, pos[ok])
        for i, src in ((0, k), (2, v)):
            codes, params = quantize(src[c.cu_l[b]:c.cu_l[b + 1]][ok], group)
            want[i][pg, :, sl] = pack(codes, i == 0)
            want[i + 1][pg, :, sl] = params
    ops.kv4_append(c.cache, k, v, c.table, c.lens, c.cu)
    for got, w in zip((c.cache.k_codes, c.cache.k_params, c.cache.v_codes, c.cache.v_params), want):
        assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
    for out in ("bf16", "f16", "f32"):
        ko, vo = (torch.full((c.tokens, heads, dim), 7.0, dtype=DT[out], device="cuda") for _ in range(2))
        ops.kv4_read(c.cache, c.table, c.lens, c.cu, c.tokens, dtype=DT[out], k_out=ko, v_out=vo)
        for got, keys in ((ko, True), (vo, False)):
            for b, n in enumerate(new):
                mine = got[c.cu_l[b]:c.cu_l[b + 1]]
                first = max(n - lens[b], 0)
                full = c.rows(b, keys)[max(lens[b] - n, 0):]
                assert torch.equal(mine[first:], full.float().to(DT[out]))
                assert (mine[:first] == 0).all()        # tokens before position 0
            assert (got[c.cu_l[-1]:] == 7.0).all()      # rows behind the last sequence are left as they were


def test_append_of_values_that_f16_cannot_hold():
    """NaN is stored as zero, infinities and larger values as the largest f16; neighbours keep the codes the definition gives them."""
    from oxicuda_b200 import ops
    c = Case([6], [6], 2, 128, 64, 16, dirty=False)
    x = c.normal(6, 4, 128)
    x[0, 0, 5], x[1, 1, 64], x[2, 2, 0], x[3, 3, 127] = float("nan"), float("inf"), float("-inf"), 1e30
    x[4] = 1e-9
    x[5, :, ::2] = 1e-7
    ops.kv4_append(c.cache, x[:, :2], x[:, 2:], c.table, c.lens, c.cu)
    pg, sl = c.place(0, torch.arange(6, device="cuda"))
    for cc, pp, src, keys in ((c.cache.k_codes, c.cache.k_params, x[:, :2], True), (c.cache.v_codes, c.cache.v_params, x[:, 2:], False)):
        codes, params = quantize(src, 64)
        assert torch.equal(cc[pg, :, sl], pack(codes, keys)) and torch.equal(pp[pg, :, sl], params)
        assert torch.isfinite(decode(cc[pg, :, sl], pp[pg, :, sl], keys)).all()


@pytest.mark.parametrize("shift", [1, 4])
def test_append_from_rows_that_are_not_aligned(shift):
    from oxicuda_b200 import ops
    c = Case([40, 3], [40, 3], 3, 128, 128, 16)
    flat = c.normal(43 * 3 * 131 + 64, dtype=torch.bfloat16)
    k = torch.as_strided(flat, (43, 3, 128), (3 * 131, 131, 1), shift)
    ops.kv4_append(c.cache, k, k, c.table, c.lens, c.cu)
    got, _ = ops.kv4_read(c.cache, c.table, c.lens, c.cu, 43, dtype=torch.float32)
    codes, params = quantize(k, 128)
    want = codes.double() * params[..., 0].double().repeat_interleave(128, -1) + params[..., 1].double().repeat_interleave(128, -1)
    assert torch.equal(got, want.float())


def test_error_of_the_stored_values():
    """|x - x^| is at most half a step and the rounding of the step and offset to f16: s (1/2 + 15 * 2^-11 + 2^-11 |m| / s ...)."""
    from oxicuda_b200 import ops
    c = Case([500], [500], 4, 128, 64, 64)
    x = c.normal(500, 8, 128)
    k, v = x[:, :4], x[:, 4:]
    ops.kv4_append(c.cache, k, v, c.table, c.lens, c.cu)
    got = torch.cat(ops.kv4_read(c.cache, c.table, c.lens, c.cu, 500, dtype=torch.float32), 1)
    g, o = x.unflatten(-1, (2, 64)), got.unflatten(-1, (2, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = (hi - lo) / 15
    # inside the rounded range half a step; at its ends the range moved by the rounding of m and of 15 s
    bound = s * (1 + 2.0 ** -11) / 2 + lo.abs() * 2.0 ** -11 + 15 * s * 2.0 ** -11
    assert ((g - o).abs() <= bound).all()


# ------------------------------------------------------------------------------------------- attention

def reference(c, q, scale, causal, window, drop=None):
    """Per query row: o and lse in f64, and what the bound needs: A = sum of p (15 s + |m|), X = the largest sum of |q| (15 s + |m|), N."""
    t, hq, dim = q.shape
    per = hq // c.heads
    o = torch.zeros(t, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device="cuda")
    big = torch.zeros(t, hq, 1, dtype=torch.float64, device="cuda")
    step = torch.zeros(t, hq, 1, dtype=torch.float64, device="cuda")
    err = torch.zeros(t, hq, 1, dtype=torch.float64, device="cuda")
    for b, n in enumerate(c.new_l):
        length = max(c.lens_l[b], 0)
        if n == 0 or length == 0:
            continue
        k, v = c.rows(b, True), c.rows(b, False)
        pg, sl = c.place(b, torch.arange(length, device="cuda"))
        size = lambda p: (15 * p[pg, :, sl][..., 0].double() + p[pg, :, sl][..., 1].double().abs()).amax(-1)  # noqa: E731  [len, heads]
        ks, vs = size(c.cache.k_params), size(c.cache.v_params)
        vstep = c.cache.v_params[pg, :, sl][..., 0].double().amax(-1)
        pos = length - n + torch.arange(n, device="cuda")
        at = torch.arange(length, device="cuda")
        see = at[None] <= pos[:, None] if causal else torch.ones(n, length, dtype=torch.bool, device="cuda")
        if window:
            see = see & (at[None] > pos[:, None] - window)
        if drop is not None:
            see = see & ~drop[b][None, :length]
        rows = slice(c.cu_l[b], c.cu_l[b + 1])
        for h in range(hq):
            kv = h // per
            qq = q[rows, h].double()
            kk, vv = k[:, kv].clone(), v[:, kv].clone()
            if drop is not None:
                kk[drop[b][:length]], vv[drop[b][:length]] = 0, 0
            x = (qq @ kk.T) * scale
            x[~see] = -math.inf
            any_ = see.any(1)
            lse[rows, h] = torch.logsumexp(x, 1)
            p = torch.softmax(x, 1)
            p[~any_] = 0
            o[rows, h] = p @ vv
            fin = torch.nan_to_num(vs[:, kv]) if drop is not None else vs[:, kv]
            kfin = torch.nan_to_num(ks[:, kv]) if drop is not None else ks[:, kv]
            big[rows, h, 0] = p @ fin
            step[rows, h, 0] = torch.nan_to_num(vstep[:, kv]).max()
            err[rows, h, 0] = abs(scale) * qq.abs().sum(1) * kfin.max()
    return o, lse, big, step, err


def check(c, q, out, lse, scale, causal, window, drop=None):
    """The bound, per element.  x: the tensor core adds D / 16 partial sums, each short of at most 2^-22 of the largest sum (truncation), and there
    are a few f32 operations: |dx| <= 16 * 2^-22 * X with X the sum of |q| |k^|'s terms; a wrong x moves p and the sum by twice that.  w is rounded
    to f16 (2^-11; twice that fine, 2^-21, for f16 outputs, which use two terms), at worst by 2^-25 of the largest in the subnormal range, times
    codes up to 15; f32 sums of N terms in 128 lanes.  The output is rounded once: eps / 2 of its type."""
    o, ref_lse, big, step, err = reference(c, q, scale, causal, window, drop)
    n = max(c.lens_l + [1])
    dx = 16 * 2.0 ** -22 * err
    rounding = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -21
    if many_rows(c, q):                                  # keys, values and p are f16 operands of the tensor core there
        rounding, dx = 3 * 2.0 ** -11, dx + 2.0 ** -11 * err
    tol = torch.finfo(q.dtype).eps / 2 * o.abs() + (rounding + 2 * dx + (n / 128 + 16) * 2.0 ** -24) * big + n * 2.0 ** -25 * 15 * step + 1e-30
    live = slice(0, c.cu_l[-1])
    diff = (out[live].double() - o[live]).abs()
    assert torch.isfinite(out[live]).all()
    worst = (diff / tol[live].expand_as(diff)).max().item() if diff.numel() else 0.0
    assert worst <= 1, f"off by {worst:.3f} of the bound"
    if lse is not None:
        seen = torch.isfinite(ref_lse[live])
        assert torch.equal(seen, torch.isfinite(lse[live])) and (lse[live][~seen] == -math.inf).all()
        d = (lse[live].double() - ref_lse[live]).abs()[seen]
        t = (2 * dx[live][..., 0] + ref_lse[live].abs() * 2.0 ** -22 + (n / 128 + 16) * 2.0 ** -24 + 2.0 ** -21)[seen]
        assert (d <= t).all(), (d / t).max().item()
    return worst


def many_rows(c, q):
    """Whether some sequence may have gone to the kernel for many query rows."""
    return c.tokens * (q.shape[1] // c.heads) > 64


def attend(c, q, scale=None, causal=True, window=0, max_tokens=None, **kw):
    from oxicuda_b200 import ops
    return ops.kv4_attention(q, c.cache, c.table, c.lens, c.cu, max_tokens=max(c.new_l + [0]) if max_tokens is None else max_tokens, scale=scale, causal=causal,
                             window=window, want_lse=True, **kw)


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per", [1, 4, 7])
def test_one_token_at_many_lengths(dim, group, dtype, per):
    lens = [0, 1, 2, 15, 16, 17, 31, 127, 128, 129, 255, 300, 1000, 1]
    c = Case(lens, [1] * len(lens), 3, dim, group, 16, seed=per)
    c.fill()
    q = c.normal(c.tokens, 3 * per, dim, dtype=DT[dtype])
    out, lse = attend(c, q)
    check(c, q, out, lse, dim ** -0.5, True, 0)
    assert (out[0] == 0).all()                          # a sequence without keys


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 40), (True, 129), (False, 0)])
def test_runs_of_tokens(dim, group, dtype, causal, window):
    """Runs that end inside row blocks and tiles, a prompt from nothing, more tokens than positions, a sequence without tokens."""
    lens, new = [70, 5, 40, 3, 200, 131, 64], [7, 5, 0, 6, 1, 131, 33]
    c = Case(lens, new, 2, dim, group, 32, seed=window, pad_tokens=3)
    c.fill()
    q = c.normal(c.tokens, 6, dim, dtype=DT[dtype])
    keep = torch.full((c.tokens, 6, dim), 3.0, dtype=q.dtype, device="cuda")
    keep_lse = torch.full((c.tokens, 6), 3.0, device="cuda")
    out, lse = attend(c, q, causal=causal, window=window, out=keep, lse=keep_lse)
    check(c, q, out, lse, dim ** -0.5, causal, window)
    assert (out[c.cu_l[-1]:] == 3.0).all() and (lse[c.cu_l[-1]:] == 3.0).all()
    # a caller who does not know the longest run, or says it too small, gets the same rows within the same bound
    for said in (0, 1):
        out2, lse2 = attend(c, q, causal=causal, window=window, max_tokens=said)
        check(c, q, out2, lse2, dim ** -0.5, causal, window)


@pytest.mark.parametrize("per,new", [(1, 1), (8, 1), (16, 1), (5, 3), (8, 8), (64, 1), (33, 2)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_groups_of_query_heads(per, new, page):
    c = Case([400, 77], [new, new], 2, 128, 64, page, seed=per)
    c.fill()
    q = c.normal(c.tokens, 2 * per, 128, dtype=torch.bfloat16)
    out, lse = attend(c, q, scale=0.2)
    check(c, q, out, lse, 0.2, True, 0)


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per,page,lens,new,causal,window", [
    (1, 16, [300], [300], True, 0), (4, 64, [129], [128], True, 0), (4, 32, [1000, 70], [257, 70], True, 0), (3, 16, [500, 64, 333], [87, 64, 130], True, 0),
    (4, 64, [700], [300], True, 1), (4, 64, [700], [300], True, 130), (8, 128, [400], [33], False, 0), (2, 64, [40], [100], True, 0),
    (5, 64, [0, 200], [30, 40], True, 0), (16, 64, [260], [260], True, 300)])
def test_prompts(dim, group, dtype, per, page, lens, new, causal, window):
    """Many rows a kv head: blocks and tiles that end inside, windows, rows that see nothing, a sequence without keys."""
    c = Case(lens, new, 2, dim, group, page, seed=per + page, pad_tokens=2)
    c.fill()
    q = c.normal(c.tokens, 2 * per, dim, dtype=DT[dtype])
    out, lse = attend(c, q, causal=causal, window=window, out=torch.full_like(q, 3.0))
    check(c, q, out, lse, dim ** -0.5, causal, window)
    assert (out[c.cu_l[-1]:] == 3.0).all()
    again, _ = attend(c, q, causal=causal, window=window, out=torch.full_like(q, 3.0))
    assert torch.equal(out, again)


@pytest.mark.parametrize("scale", [0.3, -0.1, 0.0])
@pytest.mark.parametrize("rows", [3, 90])
def test_scales_of_either_sign(scale, rows):
    c = Case([200], [rows], 1, 128, 64, 16)
    c.fill()
    q = c.normal(rows, 1, 128, dtype=torch.bfloat16)
    out, lse = attend(c, q, scale=scale)
    check(c, q, out, lse, scale, True, 0)


def test_a_mixed_batch():
    """Single tokens, short runs and prompts together: each sequence goes to the kernel for its number of rows."""
    new = [1, 200, 0, 3, 16, 17, 1, 90]
    lens = [900, 200, 50, 3, 1000, 400, 1, 2000]
    c = Case(lens, new, 2, 128, 64, 32)
    c.fill()
    for dt in ("bf16", "f16"):
        q = c.normal(c.tokens, 8, 128, dtype=DT[dt])
        out, lse = attend(c, q)
        check(c, q, out, lse, 128 ** -0.5, True, 0)


def test_a_batch_that_looks_alike():
    """As many tokens as sequences times the longest run: all go to one kernel, whatever the offsets then say."""
    for new in ([40, 40, 40], [118, 1, 1], [0, 119, 1]):
        c = Case([300, 119, 77], new, 2, 128, 64, 32)
        c.fill()
        q = c.normal(c.tokens, 8, 128, dtype=torch.bfloat16)
        out, lse = attend(c, q, max_tokens=40)
        check(c, q, out, lse, 128 ** -0.5, True, 0)


@pytest.mark.parametrize("heads,per,lens,new", [(1, 4, [9000], [20]), (2, 4, [5000, 3000], [80, 40]), (1, 1, [20000], [100])])
@pytest.mark.parametrize("dim,group", DIMS)
def test_few_blocks_share_their_keys(heads, per, lens, new, dim, group):
    c = Case(lens, new, heads, dim, group, 64)
    c.fill()
    q = c.normal(c.tokens, heads * per, dim, dtype=torch.bfloat16)
    for causal in (True, False):
        out, lse = attend(c, q, causal=causal)
        check(c, q, out, lse, dim ** -0.5, causal, 0)


def test_large_scores_in_prompts():
    """The reference moves in the middle of a tile and between tiles, by more than f16 could hold."""
    c = Case([700], [150], 2, 128, 64, 16, seed=9)
    c.fill()
    c.cache.k_params.mul_(6)
    c.cache.v_params.mul_(torch.exp2(torch.randint(-6, 7, c.cache.v_params.shape[:3], device="cuda", generator=c.g).float()).half()[..., None, None])
    q = (c.normal(c.tokens, 4, 128) * 4).bfloat16()
    out, lse = attend(c, q)
    check(c, q, out, lse, 128 ** -0.5, True, 0)


def test_the_largest_values_in_prompts():
    """Values at the ends of f16's range do not overflow on their way into the products."""
    from oxicuda_b200 import ops
    c = Case([200], [200], 1, 128, 64, 16)
    x = torch.where(c.normal(200, 2, 128) > 0, 65504.0, -65504.0)
    ops.kv4_append(c.cache, x[:, :1], x[:, 1:], c.table, c.lens, c.cu)
    q = c.normal(200, 1, 128, dtype=torch.bfloat16) * 1e-4
    out, lse = attend(c, q)
    check(c, q, out, lse, 128 ** -0.5, True, 0)


def test_rows_with_nan_or_infinite_queries_spoil_themselves_only():
    for new in (3, 100):
        c = Case([300], [new], 1, 128, 64, 16)
        c.fill()
        q = c.normal(new, 4, 128, dtype=torch.bfloat16)
        good, _ = attend(c, q)
        good = good.clone()
        q[1, 2, 7], q[2, 0, 100] = float("nan"), float("inf")
        out, _ = attend(c, q)
        keep = torch.ones(new, 4, dtype=torch.bool, device="cuda")
        keep[1, 2], keep[2, 0] = False, False
        assert torch.equal(out[keep], good[keep]) and out[1, 2].isnan().all() and out[2, 0].isnan().all()


def test_pages_that_the_table_does_not_give_in_prompts():
    from oxicuda_b200 import ops
    c = Case([400, 100], [150, 100], 2, 128, 64, 16)
    c.fill()
    drop = [torch.zeros(500, dtype=torch.bool, device="cuda") for _ in range(2)]
    good = c.table.clone()
    c.table[0, 2], c.table[0, 20], c.table[1, 0] = c.pages, -1, 1 << 30
    drop[0][32:48], drop[0][320:336], drop[1][0:16] = True, True, True
    q = c.normal(c.tokens, 4, 128, dtype=torch.bfloat16)
    out, lse = attend(c, q)
    assert ops.handle().device_status() == 15
    c.table = good
    check(c, q, out, lse, 128 ** -0.5, True, 0, drop)


@pytest.mark.parametrize("heads,lens", [(1, [70001]), (2, [30000, 1, 9, 20011]), (8, [4097] * 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_contexts_are_split_and_joined(heads, lens, dtype):
    c = Case(lens, [1] * len(lens), heads, 128, 64, 64, seed=heads)
    c.fill()
    q = c.normal(c.tokens, heads * 4, 128, dtype=DT[dtype])
    out, lse = attend(c, q)
    check(c, q, out, lse, 128 ** -0.5, True, 0)
    again, _ = attend(c, q)
    assert torch.equal(out, again)                      # results do not depend on timing


def test_many_sequences():
    lens = [(7 * i) % 90 for i in range(700)]
    new = [1 if i % 5 else 0 for i in range(700)]
    c = Case(lens, new, 1, 64, 64, 16, seed=1)
    c.fill()
    q = c.normal(c.tokens, 2, 64, dtype=torch.bfloat16)
    out, lse = attend(c, q)
    check(c, q, out, lse, 64 ** -0.5, True, 0)


def test_large_scores_and_uneven_values():
    """Scores far apart (the reference moves many times), value rows whose steps differ by 2^20, zero rows."""
    c = Case([600], [4], 2, 128, 64, 16, seed=9)
    c.fill()
    c.cache.k_params.mul_(4)
    scale_by = torch.exp2(torch.randint(-14, 7, c.cache.v_params.shape[:3], device="cuda", generator=c.g).float()).half()
    c.cache.v_params.mul_(scale_by[..., None, None])
    c.cache.v_params[..., 0][scale_by > 32] = 0         # constant groups: step 0
    for dt in (torch.bfloat16, torch.float16):
        q = (c.normal(c.tokens, 8, 128) * 5).to(dt)
        out, lse = attend(c, q)
        check(c, q, out, lse, 128 ** -0.5, True, 0)


def test_strided_queries_and_outputs():
    c = Case([100, 30], [3, 2], 2, 128, 128, 16)
    c.fill()
    wide = c.normal(c.tokens, 20, 128, dtype=torch.bfloat16)
    q = wide[:, 1:9]
    home = torch.full((c.tokens, 8, 160), 5.0, dtype=torch.bfloat16, device="cuda")
    out, lse = attend(c, q, out=home[:, :, 16:144])
    check(c, q, out, lse, 128 ** -0.5, True, 0)
    assert (home[:, :, :16] == 5).all() and (home[:, :, 144:] == 5).all()
    flat = c.normal(c.tokens * 8 * 130 + 8, dtype=torch.bfloat16)
    q = torch.as_strided(flat, (c.tokens, 8, 128), (8 * 130, 130, 1), 1)      # rows at odd elements
    out, lse = attend(c, q)
    check(c, q, out, lse, 128 ** -0.5, True, 0)


@pytest.mark.parametrize("dim,group", DIMS)
def test_log_sum_exp_of_few_keys(dim, group):
    """The products are cut, not rounded, where the tensor core lines them up; what that costs stays below two f32 roundings of the terms' sum
    X = sum of |scale q| (15 s + |m|), each 2^-24 X / sqrt(12) in the root mean square at most: together below 2^-25 X."""
    c = Case([1 + i % 5 for i in range(60)], [1] * 60, 8, dim, group, 16)
    c.fill()
    q = c.normal(c.tokens, 24, dim, dtype=torch.float16)
    _, lse = attend(c, q)
    _, ref, _, _, x = reference(c, q, dim ** -0.5, True, 0)
    rms = lambda t: t.double().square().mean().sqrt()  # noqa: E731
    assert rms(lse.double() - ref) <= 2.0 ** -25 * rms(x)


@pytest.mark.parametrize("dim,group", DIMS)
def test_f16_outputs_are_off_by_their_own_rounding(dim, group):
    """Scores of standard deviation 2.5: most weights are far below the largest.  w is good to 2^-21 and the rest is f32, so the error is that of
    the final rounding to f16 (a tenth is left for all else)."""
    c = Case([3000, 700], [4, 4], 3, dim, group, 16)
    c.fill()
    q = (c.normal(c.tokens, 6, dim) * 2.5).to(torch.float16)
    out, _ = attend(c, q)
    ref = reference(c, q, dim ** -0.5, True, 0)[0]
    rms = lambda t: t.double().square().mean().sqrt()  # noqa: E731
    assert rms(out.double() - ref) <= 1.1 * rms(ref.to(torch.float16).double() - ref)


def test_one_token_whose_stride_means_nothing():
    c = Case([100], [1], 2, 128, 128, 16)
    c.fill()
    q = torch.as_strided(c.normal(8 * 128, dtype=torch.bfloat16), (1, 8, 128), (1, 128, 1))
    home = torch.zeros(8 * 128, dtype=torch.bfloat16, device="cuda")
    out, lse = attend(c, q, out=torch.as_strided(home, (1, 8, 128), (3, 128, 1)))
    check(c, q, out, lse, 128 ** -0.5, True, 0)


@pytest.mark.parametrize("shape,strides", [((4, 8, 128), (0, 128, 1)), ((4, 8, 128), (1024, 0, 1)), ((4, 8, 128), (1022, 128, 1)), ((4, 8, 128), (128, 510, 1))])
def test_outputs_whose_rows_overlap_are_refused(shape, strides):
    from oxicuda_b200.errors import BlasError
    c = Case([100], [4], 2, 128, 128, 16)
    c.fill()
    home = torch.zeros(8 * 1024, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(BlasError, match="overlap"):
        attend(c, c.normal(*shape, dtype=torch.bfloat16), out=torch.as_strided(home, shape, strides))
    assert (home == 0).all()


def test_places_that_the_table_does_not_give():
    """A page number outside the pool and a position behind the table are left out, never followed, and reported once."""
    from oxicuda_b200 import ops
    c = Case([100, 100], [2, 2], 2, 128, 64, 16)
    c.fill()
    h = ops.handle()
    assert h.device_status() == 0
    drop = [torch.zeros(200, dtype=torch.bool, device="cuda") for _ in range(2)]
    good = c.table.clone()
    c.table[0, 2], c.table[1, 0] = c.pages, -1
    drop[0][32:48], drop[1][0:16] = True, True
    bad = c.table.clone()
    q = c.normal(c.tokens, 8, 128, dtype=torch.bfloat16)
    out, lse = attend(c, q)
    assert h.device_status() == 15 and h.device_status() == 0
    c.table = good
    check(c, q, out, lse, 128 ** -0.5, True, 0, drop)
    # append skips such a token, read gives zeros
    before = [t.clone() for t in (c.cache.k_codes, c.cache.k_params)]
    bad[:, 98 // 16] = 1 << 30
    k = c.normal(c.tokens, 2, 128, dtype=torch.bfloat16)
    ops.kv4_append(c.cache, k, k, bad, c.lens, c.cu)
    assert h.device_status() == 15
    assert torch.equal(c.cache.k_codes, before[0]) and torch.equal(c.cache.k_params.view(torch.int16), before[1].view(torch.int16))
    ko, vo = ops.kv4_read(c.cache, bad, c.lens, c.cu, c.tokens)
    assert h.device_status() == 15 and (ko == 0).all() and (vo == 0).all()
    # a table that is too short for the lengths
    short = good[:, :3].contiguous()
    out, _ = ops.kv4_attention(q, c.cache, short, c.lens, c.cu, want_lse=True, causal=False)
    keep = [torch.arange(200, device="cuda") >= 48 for _ in range(2)]
    o, _, _, _, _ = reference(c, q, 128 ** -0.5, False, 0, keep)
    assert (out.double() - o).abs().max() <= 0.02 * o.abs().max()
    h.device_status()


@pytest.mark.parametrize("new", [2, 40])
def test_a_table_shorter_than_the_lengths(new):
    """Keys behind the table are left out; the queries keep the positions that the lengths give them, with window and without."""
    from oxicuda_b200 import ops
    for window in (0, 30):
        c = Case([100, 60], [new, new], 2, 128, 64, 16)
        c.fill()
        q = c.normal(c.tokens, 8, 128, dtype=torch.bfloat16)
        short = c.table[:, :5].contiguous()             # 80 positions
        out, lse = ops.kv4_attention(q, c.cache, short, c.lens, c.cu, window=window, want_lse=True)
        assert ops.handle().device_status() == 15
        drop = [torch.arange(200, device="cuda") >= 80 for _ in range(2)]
        check(c, q, out, lse, 128 ** -0.5, True, window, drop)


def test_workspace_and_threads():
    """A given workspace of the stated size serves; a smaller one is refused; threads with streams of their own share the library's handle."""
    import threading
    from oxicuda_b200 import ops
    from oxicuda_b200.errors import BlasError
    c = Case([5000, 33], [1, 1], 2, 128, 64, 16)
    c.fill()
    qs = [c.normal(2, 8, 128, dtype=torch.bfloat16) for _ in range(4)]
    want = [attend(c, q)[0] for q in qs]
    n = ops.kv4_attention_workspace_bytes(c.cache, c.table, c.lens, c.cu, 2, 8, 1)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert torch.equal(attend(c, qs[0], workspace=ws)[0], want[0])
    with pytest.raises(BlasError) as e:
        attend(c, qs[0], workspace=ws[:-16])
    assert e.value.variant == "BufferTooSmall"
    torch.cuda.synchronize()
    got = [[] for _ in qs]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                got[i].append(attend(c, qs[i])[0])
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, outs in zip(want, got):
        assert len(outs) == 30 and all(torch.equal(o, w) for o in outs)


def test_nothing_to_do():
    from oxicuda_b200 import ops
    c = Case([5], [0], 2, 64, 64, 16)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    out, lse = attend(c, q)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    k = torch.empty(0, 2, 64, device="cuda")
    ops.kv4_append(c.cache, k, k, c.table, c.lens, c.cu)
    ko, _ = ops.kv4_read(c.cache, c.table, c.lens, c.cu, 0)
    assert ko.shape == (0, 2, 64)
    # tokens of the call that belong to no sequence
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    home = torch.full((3, 4, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    attend(c, q, out=home)
    assert (home == 2).all()
    ops.kv4_attention(q, c.cache, c.table[:0], c.lens[:0], torch.zeros(1, dtype=torch.int32, device="cuda"), out=home)
    assert (home == 2).all()


def test_offsets_behind_two_gigabytes():
    """A pool whose last pages lie more than 2^31 bytes (and 2^31 codes) from its start."""
    from oxicuda_b200 import ops
    pages, page, heads, dim = 40000, 128, 8, 128        # 2.6 GB of codes each
    cache = ops.Kv4Cache.empty(pages, page, heads, dim, 64)
    c = Case([200, 130], [200, 130], heads, dim, 64, page)
    c.cache, c.pages = cache, pages
    c.table = torch.tensor([[pages - 1, pages - 3], [pages - 2, 17]], dtype=torch.int32, device="cuda")
    x = c.normal(c.tokens, 2 * heads, dim, dtype=torch.bfloat16)
    ops.kv4_append(cache, x[:, :heads], x[:, heads:], c.table, c.lens, c.cu)
    ko, vo = ops.kv4_read(cache, c.table, c.lens, c.cu, c.tokens, dtype=torch.float32)
    for got, src in ((ko, x[:, :heads]), (vo, x[:, heads:])):
        codes, params = quantize(src, 64)
        want = codes.double() * params[..., 0].double().repeat_interleave(64, -1) + params[..., 1].double().repeat_interleave(64, -1)
        assert torch.equal(got, want.float())
    q = c.normal(c.tokens, heads, dim, dtype=torch.bfloat16)
    out, lse = attend(c, q)
    check(c, q, out, lse, dim ** -0.5, True, 0)


def test_streams_and_graphs():
    """The call on a side stream; a captured step replayed after its inputs changed; two graphs replayed at once."""
    from oxicuda_b200 import ops
    c = Case([3000, 50, 700], [1, 1, 1], 4, 128, 64, 64)
    c.fill()
    qs = [c.normal(3, 16, 128, dtype=torch.bfloat16) for _ in range(3)]
    want = [attend(c, q)[0].clone() for q in qs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = attend(c, qs[0])[0]
    side.synchronize()
    assert torch.equal(got, want[0])
    q_in = [qs[0].clone(), qs[1].clone()]
    graphs, outs = [], []
    for i in range(2):
        with torch.cuda.stream(side):
            attend(c, q_in[i])
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(attend(c, q_in[i])[0])
        graphs.append(g)
    q_in[1].copy_(qs[2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[2])
    assert ops.handle().device_status() == 0


def test_steps_of_a_layer():
    """A prompt and then single tokens through the layer's pieces as they are used: norm + E4M3, the fused QKV product, append, attention,
    E4M3 and the O product, the seam to the next block; each piece against its own plain form on the inputs it got."""
    from oxicuda_b200 import ops
    torch.manual_seed(0)
    hidden, hq, hkv, dim, page = 1024, 8, 2, 128, 16
    w_qkv = torch.randn((hq + 2 * hkv) * dim, hidden, device="cuda", dtype=torch.bfloat16) * 0.03
    w_o = torch.randn(hidden, hq * dim, device="cuda", dtype=torch.bfloat16) * 0.03
    wq, sq = ops.fp8_quant_dynamic(w_qkv)
    wo, so = ops.fp8_quant_dynamic(w_o)
    norm1, norm2 = (1 + 0.1 * torch.randn(hidden, device="cuda") for _ in range(2))
    sx = torch.tensor([0.02], device="cuda")
    c = Case([37, 20, 5], [32, 18, 1], hkv, dim, 64, page)       # the lengths after the last step
    c.lens_l = [32, 18, 1]
    steps = [[32, 18, 1]] + [[1, 1, 1]] * 2
    for i, new in enumerate(steps):
        if i:
            c.lens_l = [a + b for a, b in zip(c.lens_l, new)]
        c.new_l = new
        c.cu_l = [0] + list(np.cumsum(new))
        c.cu = torch.tensor(c.cu_l, dtype=torch.int32, device="cuda")
        c.lens = torch.tensor(c.lens_l, dtype=torch.int32, device="cuda")
        c.tokens = c.cu_l[-1]
        x = torch.randn(c.tokens, hidden, device="cuda", dtype=torch.bfloat16)
        h8 = ops.rmsnorm_fp8_quant_rows(x, norm1, sx)
        qkv = ops.gemm_fp8(h8, wq, sx, sq[1:]).view(c.tokens, hq + 2 * hkv, dim)
        ops.kv4_append(c.cache, qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], c.table, c.lens, c.cu)
        o, lse = attend(c, qkv[:, :hq])
        check(c, qkv[:, :hq], o, lse, dim ** -0.5, True, 0)
        for b, n in enumerate(new):                              # what this step wrote is what the definition says
            codes, params = quantize(qkv[c.cu_l[b]:c.cu_l[b + 1], hq:hq + hkv], 64)
            pg, sl = c.place(b, torch.arange(c.lens_l[b] - n, c.lens_l[b], device="cuda"))
            assert torch.equal(c.cache.k_codes[pg, :, sl], pack(codes, True)) and torch.equal(c.cache.k_params[pg, :, sl], params)
        o8, s8 = ops.fp8_quant_dynamic(o.view(c.tokens, hq * dim))
        y = ops.gemm_fp8(o8, wo, s8[1:], so[1:])
        r, n8 = ops.residual_rmsnorm_fp8(y, x, norm2, sx)
        rr = x.double() + y.double()
        hh = rr / torch.sqrt((rr * rr).mean(-1, keepdim=True) + 1e-5) * norm2.double() / 0.02
        assert ((r.double() - rr).abs() <= 2.0 ** -8 * rr.abs() + 1e-6).all()
        got = n8.view(torch.float8_e4m3fn).double()
        assert ((got - hh.clamp(-448, 448)).abs() <= 2.0 ** -4 * hh.abs() * 1.0001 + 2.0 ** -10 + 1e-6).all()
    assert ops.handle().device_status() == 0
