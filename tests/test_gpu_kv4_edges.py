"""GPU tests of the 4-bit cache at the edges of what its calls allow."""
import pytest
import torch

from test_gpu_kv4 import DIMS, DT, Case, attend, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [16, 17, 63, 64, 500])
@pytest.mark.parametrize("max_tokens", [0, 1, 64])
def test_a_call_without_sequences(tokens, max_tokens):
    """Nothing is written, whatever number of query rows there is."""
    from oxicuda_b200 import ops
    c = Case([5], [0], 2, 64, 64, 16)
    q = torch.ones(tokens, 8, 64, dtype=torch.bfloat16, device="cuda")
    home, lse = torch.full_like(q, 2.0), torch.full((tokens, 8), 2.0, device="cuda")
    nobody = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.kv4_attention_workspace_bytes(c.cache, c.table[:0], c.lens[:0], nobody, tokens, 8, max_tokens) == 0
    ops.kv4_attention(q, c.cache, c.table[:0], c.lens[:0], nobody, max_tokens=max_tokens, out=home, lse=lse)
    assert (home == 2).all() and (lse == 2).all()


@pytest.mark.parametrize("dim,group", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per,page,lens,new,window", [
    (4, 16, [700, 300], [3, 1], 130), (4, 64, [700, 300], [16, 16], 200), (4, 64, [700], [300], 130), (2, 16, [1000, 333], [100, 47], 77), (4, 256, [900, 40], [90, 40], 301),
    (1, 64, [6000], [150], 3333), (4, 32, [900, 700, 400], [1, 100, 2], 99), (8, 4096, [5000], [20], 500)])
def test_nothing_in_front_of_a_window_is_looked_at(dim, group, dtype, per, page, lens, new, window):
    """Pages whose positions no query of the call sees may have been given back: entries that name no page are no error, entries that name a page
    nobody has written (params NaN) and unwritten places of the first page change no bit of the result."""
    from oxicuda_b200 import ops
    c = Case(lens, new, 2, dim, group, page, seed=window)
    c.fill()
    q = c.normal(c.tokens, 2 * per, dim, dtype=DT[dtype])
    h = ops.handle()
    h.device_status()
    want, want_lse = attend(c, q, window=window)
    check(c, q, want, want_lse, dim ** -0.5, True, window)
    first = [max(length - n + 1 - window, 0) for length, n in zip(lens, new)]                # the first position that a query sees
    assert any(f // page for f in first) or any(f % 128 for f in first)
    good = c.table.clone()
    blank = (set(range(c.pages)) - set(good[good >= 0].tolist())).pop()                      # a page of the pool that no sequence holds
    for params in (c.cache.k_params, c.cache.v_params):
        assert params[blank].isnan().all()
    for entry in (-1, c.pages, blank):
        c.table = good.clone()
        for b, f in enumerate(first):
            c.table[b, :f // page] = entry
            pg, sl = good[b].long()[f // page], torch.arange(f % page, device="cuda")
            for params in (c.cache.k_params, c.cache.v_params):
                params[pg, :, sl] = float("nan")
        out, lse = attend(c, q, window=window)
        assert h.device_status() == 0
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
