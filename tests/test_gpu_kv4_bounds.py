"""GPU tests of attention over the 4-bit cache against what its roundings may be off by, row by row and all rows together."""
import pytest
import torch

from kv4_bounds import Expected, rows_of
from test_gpu_kv4 import DIMS, DT, Case, attend
from test_kv4_bounds_cpu import SHAPES

pytestmark = pytest.mark.gpu


def held(c, q, scale, causal, window, max_tokens=None):
    out, lse = attend(c, q, scale=scale, causal=causal, window=window, max_tokens=max_tokens)
    worst = Expected(rows_of(c), c.new_l, q, scale, causal, window, max_tokens=max_tokens).worst(out, lse)
    assert worst <= 1, f"{worst:.3f} of the bound"


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per,lens,new,causal,window", SHAPES)
def test_rows_are_off_by_their_roundings(dim, group, dtype, per, lens, new, causal, window):
    c = Case(lens, new, 2, dim, group, 32, seed=per + len(lens))
    c.fill()
    q = c.normal(c.tokens, 2 * per, dim, dtype=DT[dtype])
    held(c, q, dim ** -0.5, causal, window)


@pytest.mark.parametrize("max_tokens", [0, 1, 40, 200])
def test_mixed_batches_are_off_by_their_roundings(max_tokens):
    new = [1, 200, 0, 3, 16, 17, 1, 90]
    c = Case([900, 200, 50, 3, 1000, 400, 1, 2000], new, 2, 128, 64, 32)
    c.fill()
    held(c, c.normal(c.tokens, 8, 128, dtype=torch.bfloat16), 128 ** -0.5, True, 0, max_tokens)


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per,lens,new,window", [(1, [300, 77], [5, 1], 0), (4, [300, 77], [5, 2], 50), (4, [500], [300], 0), (4, [500, 130], [300, 20], 129), (2, [900], [128], 128)])
def test_the_edges_of_the_mask(dim, group, dtype, per, lens, new, window):
    """Scores that rise by 8 from key to key: a row's output is the last value that it sees, and a row that saw one key more or less would give
    another one.  Falling ones: the first value that it sees, which is the window's edge."""
    for falling in (False, True):
        c = Case(lens, new, 2, dim, group, 16, seed=dim)
        c.fill()
        for b, n in enumerate(lens):
            at = torch.arange(n, device="cuda")
            pg, sl = c.place(b, at)
            c.cache.k_params[pg, :, sl] = torch.stack([torch.zeros_like(at), -at if falling else at], -1).half()[:, None, None]
        q = torch.ones(c.tokens, 2 * per, dim, dtype=DT[dtype], device="cuda")
        held(c, q, 8 / dim, True, window)


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,new", [([500], [300]), ([5000], [40]), ([500, 70], [5, 2])])
def test_small_keys_and_values(dim, group, dtype, lens, new):
    """Steps and offsets below f16's normal range, down to a step of 2^-24, are held as they are: what comes out is as good as for large ones."""
    from oxicuda_b200 import ops
    for kf, vf in ((1.0, 2.0 ** -10), (2.0 ** -12, 2.0 ** -14), (2.0 ** -16, 2.0 ** -16), (2.0 ** -18, 2.0 ** -18), (1.0, 2.0 ** -21), (2.0 ** -21, 1.0)):
        c = Case(lens, new, 2, dim, group, 32, seed=dim, dirty=False)
        k, v = c.normal(sum(lens), 2, dim) * 2 * kf, c.normal(sum(lens), 2, dim) * vf
        all_ = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")
        ops.kv4_append(c.cache, k, v, c.table, c.lens, all_)
        q = c.normal(c.tokens, 8, dim, dtype=DT[dtype])
        held(c, q, dim ** -0.5 / kf, True, 0)
        held(c, q, dim ** -0.5 / kf, True, 60)


def test_values_at_the_end_of_f16():
    """A group that spans f16's whole range: the largest value, which the rounding of the step lifts to 65536, counts as at least 65504."""
    from oxicuda_b200 import ops
    for new in (1, 200):
        c = Case([200], [new], 1, 128, 64, 16, dirty=False)
        x = torch.full((200, 2, 128), 65504.0, device="cuda")
        x[:, :, ::2] = -65504.0
        x[:, 0] *= 1e-4
        ops.kv4_append(c.cache, x[:, :1], x[:, 1:], c.table, c.lens, torch.tensor([0, 200], dtype=torch.int32, device="cuda"))
        out, _ = attend(c, c.normal(new, 1, 128, dtype=torch.bfloat16))
        assert (out[..., ::2] == -65536.0).all() and (out[..., 1::2] == 65536.0).all()       # to the nearest bf16


@pytest.mark.parametrize("dtype,ratio", [("bf16", 19), ("f16", 15)])
@pytest.mark.parametrize("lens,new", [([500], [1]), ([900, 70], [4, 2]), ([3000], [16]), ([400], [60])])
def test_groups_whose_steps_are_far_apart(dtype, ratio, lens, new):
    """The second group of every value row is 2^-ratio of the first, and is held to its own outputs' roundings.  p is taken 2^10 above the reference,
    so the second group's largest w is 2^(10 - ratio) and off by 2^-25 at worst: 2^(ratio - 35) of itself, below the 2^-11 of its rounding (bf16) and
    a quarter of a step of the output (f16, 2^-13)."""
    c = Case(lens, new, 2, 128, 64, 32, seed=ratio)
    c.fill()
    first = 2.0 ** 6 if dtype == "bf16" else 2.0 ** 9
    c.cache.v_params[..., 0, :].mul_(first)
    c.cache.v_params[..., 1, :].mul_(first * 2.0 ** -ratio)
    q = c.normal(c.tokens, 8, 128, dtype=DT[dtype])
    out, lse = attend(c, q)
    e = Expected(rows_of(c), new, q, 128 ** -0.5)
    for dims in (slice(0, 64), slice(64, 128)):
        worst = e.worst(out, lse, dims)
        assert worst <= 1, f"{worst:.3f} of the bound for elements from {dims.start} on"


@pytest.mark.parametrize("per,lens,new", [(1, [300], [350]), (4, [300, 40], [350, 3]), (1, [5, 60], [9, 61]), (2, [20], [30])])
@pytest.mark.parametrize("window", [2 ** 31 - 2 ** 6, 2 ** 31 - 5, 2 ** 31 - 1, 2 ** 40])
def test_the_widest_windows_with_queries_before_the_first_position(per, lens, new, window):
    """A call may have more tokens than positions; a window that holds everything hides nothing, whatever its width."""
    c = Case(lens, new, 2, 128, 64, 16, seed=per)
    c.fill()
    q = c.normal(c.tokens, 2 * per, 128, dtype=torch.bfloat16)
    held(c, q, 128 ** -0.5, True, window)
    assert torch.equal(attend(c, q, window=window)[0], attend(c, q)[0])


@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("power", [-110, -60, 60, 110, 118])
def test_queries_of_any_size(new, power):
    """Queries and scale by a power of two up and down: the same scores, so the same bits."""
    c = Case([300], [new], 1, 128, 64, 16)
    c.fill()
    q = c.normal(new, 4, 128, dtype=torch.bfloat16)
    q[:, 1, :64] *= 2.0 ** -12
    scaled = q * 2.0 ** power
    # 2^-110 takes elements of 2^-16 and less below bf16's normal range, 2^-126, where the product above loses bits of them; the way back up loses none
    q = (scaled.float() * 2.0 ** -power).bfloat16()
    want, want_lse = attend(c, q, scale=0.1)
    out, lse = attend(c, scaled, scale=0.1 * 2.0 ** -power)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
