"""GPU tests of the fused residual norm on rows that hold a NaN or an infinity."""
import pytest
import torch

from test_gpu_resnorm import make

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("rows,cols", [(9, 64), (300, 64), (300, 1032), (9, 1024), (299, 8200), (9, 16384)])
@pytest.mark.parametrize("dtype,rdtype", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "full")])
def test_bad_rows_show_and_spoil_themselves_only(rows, cols, dtype, rdtype, post, gate):
    """Whatever the row goes out as, it is seen to be bad: NaN elements, NaN codes of E4M3, a NaN scale of INT8.  The other rows keep their bits."""
    from oxicuda_b200 import ops
    a = make(rows, cols, dtype, rdtype, post, gate, rows)
    more = dict(post_weight=a["post_weight"], gate=a["gate"], alpha=0.7)
    scale = torch.tensor([0.02], device="cuda")
    run = lambda: (ops.residual_rmsnorm(a["y"], a["residual"], a["weight"], **more), ops.residual_rmsnorm_fp8(a["y"], a["residual"], a["weight"], scale, **more),  # noqa: E731
                   ops.residual_rmsnorm_int8_rows(a["y"], a["residual"], a["weight"], **more))
    good = run()
    bad = {1: ("y", NAN, 0), 2: ("residual", NAN, cols - 1), 4: ("residual", INF, cols // 2), 5: ("y", INF, 3), rows - 1: ("residual", -INF, 7)}
    for r, (name, value, at) in bad.items():
        a[name][r, at] = value
    (r1, h), (r2, q), (r3, q8, sc) = run()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[list(bad)] = False
    bits = lambda x: x.contiguous().view(torch.uint8)  # noqa: E731
    for got, want in ((r1, good[0][0]), (h, good[0][1]), (r2, good[1][0]), (q, good[1][1]), (r3, good[2][0]), (q8, good[2][1]), (sc, good[2][2])):
        assert torch.equal(bits(got[keep]), bits(want[keep]))
    e4m3 = q.view(torch.float8_e4m3fn).float()
    for r in bad:
        assert h[r].isnan().any() and e4m3[r].isnan().any() and sc[r].isnan()
    assert torch.isfinite(sc[keep]).all() and not e4m3[keep].isnan().any()


def test_a_bad_row_shows_behind_the_int8_product():
    from oxicuda_b200 import ops
    a = make(64, 512, "bf16", "bf16", False, "none")
    a["residual"][7, 100], a["residual"][9, 3] = INF, NAN
    w, ws = ops.int8_quant_rows(torch.randn(256, 512, device="cuda"))
    _, q8, sc = ops.residual_rmsnorm_int8_rows(a["y"], a["residual"], a["weight"])
    y = ops.gemm_w8a8(q8, w, sc, ws)
    assert y[7].isnan().all() and y[9].isnan().all()
    y[7], y[9] = 0, 0
    assert torch.isfinite(y).all()
