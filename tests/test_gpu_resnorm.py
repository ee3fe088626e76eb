"""GPU tests of the fused residual / norm / quantize seam against its formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def plain(y, residual, weight, eps, post, gate, alpha):
    t = y.double()
    if post is not None:
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        t = t * gate.double()
    r = residual.double() + alpha * t
    return t, r, r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * weight.double()


def make(rows, cols, dtype, rdtype, post, gate, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return {"y": rnd(rows, cols).to(DT[dtype]), "residual": (2 * rnd(rows, cols)).to(DT[rdtype]), "weight": 1 + 0.2 * rnd(cols),
            "post_weight": 1 + 0.2 * rnd(cols) if post else None,
            "gate": None if gate == "none" else rnd(cols).to(DT[dtype]) if gate == "row" else rnd(rows, cols).to(DT[dtype])}


def bounds(t, r, h, alpha):
    """f32 arithmetic: t carries a few roundings and its norm's (a sum of at most 16384 squares in chains of 32 and a tree: below 64 * 2^-24 of it,
    halved by the root), r one more of the sum; h the same again, relative to what r is made of."""
    dt = 48 * 2.0 ** -24 * abs(alpha) * t.abs() + 2.0 ** -24 * r.abs()
    rms = torch.sqrt((r * r).mean(-1, keepdim=True)) + 1e-20
    rel = torch.sqrt((dt * dt).mean(-1, keepdim=True)) / rms + 48 * 2.0 ** -24
    dh = h.abs() * rel + h.abs() * dt / r.abs().clamp(min=1e-30) + 1e-30
    return dt, dh


CASES = [(1, 8), (1, 8192), (3, 1024), (5, 1032), (7, 4104), (2, 16384), (300, 64), (301, 4096), (299, 8200), (297, 1000), (400, 16384)]


@pytest.mark.parametrize("rows,cols", CASES)
@pytest.mark.parametrize("dtype,rdtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "full"), (True, "row"), (False, "full")])
def test_residual_rmsnorm(rows, cols, dtype, rdtype, post, gate):
    from oxicuda_b200 import ops
    a = make(rows, cols, dtype, rdtype, post, gate, rows + cols)
    t, r, h = plain(a["y"], a["residual"], a["weight"], 1e-5, a["post_weight"], a["gate"], 0.7)
    dt, dh = bounds(t, r, h, 0.7)
    got_r, got_h = ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], eps=1e-5, post_weight=a["post_weight"], gate=a["gate"], alpha=0.7)
    assert got_r.dtype == a["residual"].dtype and got_h.dtype == a["y"].dtype
    assert ((got_r.double() - r).abs() <= torch.finfo(got_r.dtype).eps / 2 * r.abs() + 1.001 * dt + 1e-7).all()
    assert ((got_h.double() - h).abs() <= torch.finfo(got_h.dtype).eps / 2 * h.abs() + 1.001 * dh + 1e-7).all()


@pytest.mark.parametrize("rows,cols", [(1, 8), (33, 8192), (310, 1032), (300, 16384)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantised_outputs(rows, cols, dtype):
    """E4M3: the rounded h is within half a step of h / scale (saturating at 448); INT8 per row: the scale is absmax / 127 and every code within
    half a step of h / scale.  Both to the f32 error of h."""
    from oxicuda_b200 import ops
    a = make(rows, cols, dtype, dtype, True, "full", 5)
    t, r, h = plain(a["y"], a["residual"], a["weight"], 1e-6, a["post_weight"], a["gate"], 1.5)
    _, dh = bounds(t, r, h, 1.5)
    more = dict(eps=1e-6, post_weight=a["post_weight"], gate=a["gate"], alpha=1.5)
    for s in (0.003, 0.02):                             # the smaller one saturates
        scale = torch.tensor([s], device="cuda")
        r1, q = ops.residual_rmsnorm_fp8(a["y"], a["residual"], a["weight"], scale, **more)
        want = (h / scale.double()).clamp(-448, 448)
        got = q.view(torch.float8_e4m3fn).double()
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 + 1.1 * dh / scale.double()).all()
    r2, q8, sc = ops.residual_rmsnorm_int8_rows(a["y"], a["residual"], a["weight"], **more)
    assert torch.equal(r1, r2)
    top = h.abs().amax(1)
    assert ((sc.double() - top / 127).abs() <= (top / 127) * 2.0 ** -22 + dh.amax(1) / 127).all()
    assert ((q8.double() * sc.double()[:, None] - h).abs() <= sc.double()[:, None] * 0.5001 + dh).all() and q8.min() >= -127


def test_in_place_strided_and_isolated_rows():
    from oxicuda_b200 import ops
    a = make(50, 1024, "bf16", "bf16", False, "none")
    wide = torch.zeros(50, 1536, dtype=torch.bfloat16, device="cuda")
    y, res = wide[:, 512:], torch.randn(50, 2048, device="cuda").bfloat16()
    y.copy_(a["y"])
    gate = torch.randn(50, 1040, device="cuda").bfloat16()[:, :1024]
    want_r, want_h = ops.residual_rmsnorm(a["y"], res[:, :1024].contiguous(), a["weight"], gate=gate.contiguous())
    right = res[:, 1024:].clone()
    got_r, got_h = ops.residual_rmsnorm(y, res[:, :1024], a["weight"], gate=gate, residual_out=res[:, :1024])
    assert got_r.data_ptr() == res.data_ptr() and torch.equal(got_r, want_r) and torch.equal(got_h, want_h) and torch.equal(res[:, 1024:], right)
    # a row with a NaN or an infinity spoils itself only
    a = make(300, 1032, "bf16", "bf16", True, "row")
    r0, h0 = ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], post_weight=a["post_weight"], gate=a["gate"])
    a["y"][3, 5], a["residual"][290, 7] = float("nan"), float("inf")
    r1, h1 = ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], post_weight=a["post_weight"], gate=a["gate"])
    keep = [i for i in range(300) if i not in (3, 290)]
    assert torch.equal(r0[keep], r1[keep]) and torch.equal(h0[keep], h1[keep]) and h1[3].isnan().all() and h1[290].isnan().any()


def test_zero_rows_and_graph():
    from oxicuda_b200 import ops
    z = torch.zeros(4, 512, dtype=torch.float16, device="cuda")
    w = torch.ones(512, device="cuda")
    r, h = ops.residual_rmsnorm(z, z, w, post_weight=w, gate=z)
    assert (r == 0).all() and (h == 0).all()
    _, q, s = ops.residual_rmsnorm_int8_rows(z, z, w)
    assert (q == 0).all() and torch.isfinite(s).all()
    a = make(64, 8192, "bf16", "f32", True, "full")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], post_weight=a["post_weight"], gate=a["gate"])
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        r, h = ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], post_weight=a["post_weight"], gate=a["gate"])
    a["y"].mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    r2, h2 = ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], post_weight=a["post_weight"], gate=a["gate"])
    assert torch.equal(r, r2) and torch.equal(h, h2)


def test_refusals():
    from oxicuda_b200 import ops
    from oxicuda_b200.errors import BlasError, QuantError
    a = make(4, 64, "bf16", "bf16", False, "none")
    y, r, w = a["y"], a["residual"], a["weight"]
    with pytest.raises(QuantError):
        ops.residual_rmsnorm(y, r[:3], w)
    with pytest.raises(QuantError):
        ops.residual_rmsnorm(y, r, w[:32])
    with pytest.raises(QuantError):
        ops.residual_rmsnorm(y, r, w, gate=y[:2])
    with pytest.raises(QuantError) as e:
        ops.residual_rmsnorm(y[:0], r[:0], w)
    assert e.value.variant == "EmptyInput"
    with pytest.raises(TypeError):
        ops.residual_rmsnorm(y, r.half(), w)
    with pytest.raises(TypeError):
        ops.residual_rmsnorm(y.t(), r.t(), w[:4])
    with pytest.raises(BlasError) as e:
        ops.residual_rmsnorm(y[:, :60], r[:, :60], w[:60])
    assert e.value.variant == "InvalidDimension"
    with pytest.raises(BlasError) as e:
        ops.residual_rmsnorm(y[:, 4:60], r[:, 4:60], w[:56].clone())
    assert e.value.variant == "InvalidArgument"
