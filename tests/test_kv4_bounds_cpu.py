"""CPU tests of the bounds that the GPU tests hold attention over the 4-bit cache to: what the kernels' roundings give is let through, and outputs
that are wrong -- nothing computed, a tile of keys left out, a mask or a window off by one, rows in the wrong place -- are not."""
import math

import pytest
import torch

from kv4_bounds import Expected, goes_to_many_rows
from test_gpu_kv4 import quantize

# per, lens, new, causal, window: the shapes of the prompt tests, of the ones whose blocks share their keys, and of runs and single tokens
SHAPES = [(1, [300], [300], True, 0), (4, [129], [128], True, 0), (4, [1000, 70], [257, 70], True, 0), (3, [500, 64, 333], [87, 64, 130], True, 0),
          (4, [700], [300], True, 1), (4, [700], [300], True, 130), (8, [400], [33], False, 0), (16, [260], [260], True, 300),
          (4, [9000], [20], True, 0), (4, [9000], [20], False, 0), (4, [5000, 3000], [80, 40], True, 0), (1, [20000], [100], True, 0), (8, [400, 77], [8, 8], True, 0),
          (4, [900, 300], [1, 1], True, 0), (4, [200, 131, 5], [7, 33, 5], True, 40)]


def make(per, lens, new, dim=64, group=64, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for n in lens:
        kv = []
        for keys in (True, False):
            x = torch.randn(n, 1, dim, generator=g) * (2.0 if keys else 0.7) + 0.3
            x[:, :, 3] *= 6.0
            c, p = quantize(x, group)
            s, m = (p[..., i].double().repeat_interleave(group, -1) for i in (0, 1))
            kv += [c * s + m, c * s, m]
        rows.append((kv[0], kv[3], kv[4], kv[1].abs() + kv[2].abs()))
    return rows, torch.randn(sum(new), per, dim, generator=g)


def seen(lens, new, causal, window, shift=0, wider=0):
    out = []
    for length, n in zip(lens, new):
        at, pos = torch.arange(length)[None], (length - n + torch.arange(n))[:, None]
        s = at <= pos + shift if causal else torch.ones(n, length, dtype=torch.bool)
        out.append(s & (at > pos + shift - window - wider) if window else s)
    return out


def as_the_kernels_round(rows, new, q, scale, see, many, dtype, g):
    """The formula with keys, values and p (many rows) or p s (few rows, bf16 outputs) in f16, and the output in its own type."""
    o = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64)
    f16 = lambda x: x.half().double()  # noqa: E731
    at = 0
    for b, n in enumerate(new):
        k, v, sc, _ = (r[:, 0] for r in rows[b])
        if many[b]:
            k, v = f16(k), f16(v)
        for h in range(q.shape[1]):
            x = (q[at:at + n, h].double() @ k.T * scale).masked_fill(~see[b], -math.inf)
            top = x.amax(1, keepdim=True).clamp(min=-1e30)
            p = (x - top).exp()
            z = p.sum(1, keepdim=True)
            lse[at:at + n, h] = (top + z.log())[:, 0]
            y = f16(p) @ v if many[b] else f16(p * 0.37) / 0.37 @ sc + p @ (v - sc) if dtype == torch.bfloat16 else p @ v
            o[at:at + n, h] = y / z
        at += n
    return o.to(dtype), lse.float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per,lens,new,causal,window", SHAPES)
def test_right_outputs_pass_and_wrong_ones_do_not(dtype, per, lens, new, causal, window):
    rows, q = make(per, lens, new, seed=len(lens) + per)
    q, scale = q.to(dtype), 0.125
    e = Expected(rows, new, q, scale, causal, window)
    see = seen(lens, new, causal, window)
    many = goes_to_many_rows(new, per, max(new))
    out, lse = as_the_kernels_round(rows, new, q, scale, see, many, dtype, None)
    assert e.worst(out, lse) <= 1
    # the output alone
    for wrong in (torch.zeros_like(out), out.roll(1, 0), out.flip(-1), out * 1.01):
        assert e.worst(wrong) > 1
    assert e.worst(out, lse + 0.01) > 1
    # output and lse of a wrong set of keys
    sets = []
    for first in {0, (max(lens) // 2) // 128 * 128}:
        sets.append([s & ~((torch.arange(s.shape[1]) >= first) & (torch.arange(s.shape[1]) < first + 128))[None] for s in see])
    if causal:
        sets += [seen(lens, new, causal, window, shift=d) for d in (-1, 1)]
    if window:
        sets += [seen(lens, new, causal, window, wider=d) for d in (-1, 1)]
    for other in sets:
        if all(torch.equal(a, b) for a, b in zip(other, see)):
            continue
        assert e.worst(*as_the_kernels_round(rows, new, q, scale, other, many, dtype, None)) > 1


def test_which_kernel_takes_a_sequence():
    assert goes_to_many_rows([8, 8], 8, 8) == [False, False]
    assert goes_to_many_rows([1, 200, 17], 4, 200) == [False, True, True]
    assert goes_to_many_rows([1, 200, 16], 4, 200) == [False, True, False]
    assert goes_to_many_rows([118, 1, 1], 4, 40) == [True, True, True]
    assert goes_to_many_rows([10], 4, 0) == [False] and goes_to_many_rows([10, 10], 4, 0) == [False, False]
