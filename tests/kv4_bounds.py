"""What attention over the 4-bit cache may be off by, from the roundings that the kernels make; on any device, in 64 bits.

u = 2^-11 / sqrt(3) is the most that the rounding of a number to f16 is off by in the root mean square, relative to the number (half a step, evenly
spread).  Sequences of more than 64 query rows per kv head (many rows): keys, values and p are f16 numbers, so
    o is off by  sum p v (d_p + d_v) + sum p dx (v - o),   dx = scale * sum q k d_k,   each d independent of the others,
and the log of the sum by sum p dx.  Others (few rows): keys and values are exact, and for bf16 outputs w = p s is one f16 number: sum p s c d_w.
A row of an output is held to four standard deviations of this and half a step of its own rounding; all rows together to a tenth more than what
this and the rounding of the reference itself come to.  What f32 does besides is small and bounded: a score is cut 2^-22 of the sum of its terms' sizes
short -- q k for many rows, q c s and q m, which may cancel, for few -- and the sums of N keys lose 2^-24 at each of N / 16 steps."""
import math

import torch

U = 2.0 ** -11 / math.sqrt(3)


def goes_to_many_rows(new, per, max_tokens, tokens=None):
    """Per sequence: whether the kernel for many query rows takes it, in a call of `tokens` rows (those behind the last sequence among them)."""
    tokens = tokens or sum(new)
    tiles = min(max_tokens or tokens, tokens) * per > 64
    alike = len(new) == 1 or (max_tokens > 0 and tokens // max_tokens >= len(new))
    return [tiles and (alike or n * per > 64) for n in new]


class Expected:
    """o, lse and what they may be off by, per query row [tokens, q_heads, ...].  rows[b] = (k, v, s c of v, |s c| + |m| of k) of sequence b,
    [len, heads, dim] in f64."""

    def __init__(self, rows, new, q, scale, causal=True, window=0, max_tokens=None, see=None):
        t, hq, dim = q.shape
        dev = q.device
        heads = rows[0][0].shape[1]
        per = hq // heads
        z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
        self.dtype, self.live = q.dtype, sum(new)
        self.o, self.lse = z(t, hq, dim), torch.full((t, hq), -math.inf, dtype=torch.float64, device=dev)
        self.var, self.cut = z(t, hq, dim), z(t, hq, dim)               # variance in units of u^2; what f32 may add
        self.lse_var, self.lse_cut = z(t, hq), z(t, hq)
        many = goes_to_many_rows(new, per, max(new) if max_tokens is None else max_tokens, t)
        at0 = 0
        for b, n in enumerate(new):
            length = rows[b][0].shape[0]
            at, pos = torch.arange(length, device=dev), length - n + torch.arange(n, device=dev)
            if see is not None:
                sees = see[b]
            else:
                sees = at[None] <= pos[:, None] if causal else torch.ones(n, length, dtype=torch.bool, device=dev)
                if window:
                    sees = sees & (at[None] > pos[:, None] - window)
            mine = slice(at0, at0 + n)
            at0 += n
            if n == 0 or length == 0:
                continue
            any_ = sees.any(1)
            for h in range(hq):
                k, v, sc, size = (r[:, h // per] for r in rows[b])
                qq = q[mine, h].double()
                x = qq @ k.T * scale
                x[~sees] = -math.inf
                self.lse[mine, h] = torch.logsumexp(x, 1)
                p = torch.softmax(x, 1)
                p[~any_] = 0
                o = p @ v
                self.o[mine, h] = o
                p2 = p * p
                terms = abs(scale) * (qq.abs() @ (k.abs() if many[b] else size).T)
                if many[b]:
                    w2 = p2 * (scale * scale) * (qq.square() @ k.square().T)
                    self.var[mine, h] = 2 * (p2 @ v.square()) + (w2 @ v.square() - 2 * o * (w2 @ v) + o * o * w2.sum(1, keepdim=True)).clamp(min=0)
                    self.lse_var[mine, h] = w2.sum(1)
                elif q.dtype == torch.bfloat16:
                    self.var[mine, h] = p2 @ sc.square()
                pt = p * terms
                self.cut[mine, h] = 2.0 ** -22 * (pt @ v.abs() + o.abs() * pt.sum(1, keepdim=True)) + (length / 16 + 32) * 2.0 ** -24 * (p @ v.abs())
                self.lse_cut[mine, h] = 2.0 ** -22 * pt.sum(1) + self.lse[mine, h].abs().nan_to_num(posinf=0.0) * 2.0 ** -22 + (math.sqrt(length) + 16) * 2.0 ** -24

    def worst(self, out, lse=None, dims=slice(None)):
        """The largest of error / bound over the rows of `out` (of its elements `dims`), all of it, and the rows of lse."""
        rms = lambda x, d=None: x.square().mean() ** 0.5 if d is None else x.square().mean(d).sqrt()  # noqa: E731
        live = slice(0, self.live)
        o, var, cut = (x[live, :, dims] for x in (self.o, self.var, self.cut))
        e = out[live, :, dims].double() - o
        if not torch.isfinite(e).all():
            return math.inf
        info = torch.finfo(self.dtype)
        half = torch.maximum(info.eps / 2 * o.abs(), torch.full_like(o, info.smallest_normal * info.eps / 2))      # of a step
        row = rms(e, -1) / (rms(half, -1) + 4 * U * rms(var.sqrt(), -1) + rms(cut, -1))
        own = o.to(self.dtype).double() - o
        whole = rms(e) / (1.1 * (rms(own).square() + U * U * var.mean()).sqrt() + rms(cut) + info.smallest_normal * info.eps)
        w = max(row.max().item(), whole.item())
        if lse is not None:
            d, ref = lse[live].double(), self.lse[live]
            seen = torch.isfinite(ref)
            if not torch.equal(seen, torch.isfinite(d)) or not (d[~seen] == -math.inf).all():
                return math.inf
            off = (d - ref).abs()[seen] / (4 * U * self.lse_var[live].sqrt() + self.lse_cut[live])[seen]
            w = max(w, off.max().item() if off.numel() else 0.0)
        return w


def rows_of(c):
    """rows of a Case's sequences, from what its pool holds."""
    out = []
    for b, n in enumerate(c.lens_l):
        k, v = c.rows(b, True), c.rows(b, False)
        pg, sl = c.place(b, torch.arange(max(n, 0), device=c.table.device))
        km, vm = (p[pg, :, sl][..., 1].double().repeat_interleave(c.group, -1) for p in (c.cache.k_params, c.cache.v_params))
        out.append((k, v, v - vm, (k - km).abs() + km.abs()))
    return out
