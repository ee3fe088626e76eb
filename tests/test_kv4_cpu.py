"""CPU tests of the checks in front of the 4-bit cache and the fused residual norm: what is refused, with which error, before anything is launched.
A handle is faked as zeroed memory: its compute capability is 0.0, so a call whose arguments are all right ends at UnsupportedOperation."""
import ctypes as C

import pytest
import torch

OK_BUT_NO_DEVICE = 13


@pytest.fixture(scope="module")
def lib():
    from oxicuda_b200 import _build, _ffi
    _build.build()
    return _ffi.load()


@pytest.fixture()
def fake():
    return C.create_string_buffer(4096)


def _descs(**kw):
    from oxicuda_b200 import _ffi
    c = dict(k_codes=0x1000, k_params=0x2000, v_codes=0x3000, v_params=0x4000, pages=8, page_size=16, heads=2, dim=128, group=64)
    b = dict(block_table=0x5000, table_width=4, seq_lens=0x6000, cu_tokens=0x7000, seqs=2, tokens=3)
    a = dict(q=0x8000, q_token_stride=1024, q_head_stride=128, out=0x9000, out_token_stride=1024, out_head_stride=128, lse=None, q_heads=8, max_tokens=0,
             window=0, scale=0.1, causal=1, dtype=1)
    for k, v in kw.items():
        for d in (c, b, a):
            if k in d:
                d[k] = v
    return tuple(pack(*[0 if v is None else v for v in d.values()]) for pack, d in ((_ffi.kv4_cache, c), (_ffi.kv4_batch, b), (_ffi.kv4_attention_args, a)))


def _append(lib, h, c, b, k=0xA000, v=0xB000, strides=(256, 128, 256, 128), dtype=1):
    return lib.oxq_kv4_append(h, c, b, k, strides[0], strides[1], v, strides[2], strides[3], dtype)


POOL = [("dim", 96, 13), ("dim", 256, 13), ("group", 32, 2), ("group", 0, 2), ("page_size", 8, 15), ("page_size", 48, 15), ("page_size", 8192, 15), ("pages", 0, 10),
        ("heads", 0, 10), ("k_codes", None, 15), ("v_params", 0x4008, 15), ("seqs", -1, 10), ("tokens", -1, 10), ("table_width", -1, 10), ("seq_lens", None, 15),
        ("cu_tokens", None, 15), ("block_table", None, 15), ("tokens", 1 << 31, 10), ("table_width", 1 << 27, 10), ("table_width", (1 << 26) + 1, 10)]


@pytest.mark.parametrize("key,value,status", POOL)
def test_pool_and_batch(lib, fake, key, value, status):
    c, b, a = _descs(**{key: value})
    assert _append(lib, fake, c, b) == status
    assert lib.oxq_kv4_read(fake, c, b, 0xA000, 0xB000, 1) == status
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10000, 1 << 30) == status
    assert lib.oxq_last_error_string(fake)


def test_group_of_128_needs_a_head_of_128(lib, fake):
    c, b, _ = _descs(dim=64, group=128)
    assert _append(lib, fake, c, b) == 2
    c, b, _ = _descs(dim=64, group=64)
    assert _append(lib, fake, c, b) == OK_BUT_NO_DEVICE


def test_append_and_read(lib, fake):
    c, b, _ = _descs()
    assert _append(lib, fake, c, b) == OK_BUT_NO_DEVICE
    assert _append(lib, fake, c, b, dtype=7) == 15
    assert _append(lib, fake, c, b, k=None) == 15 and _append(lib, fake, c, b, v=None) == 15
    assert _append(lib, fake, c, b, strides=(-256, 128, 256, 128)) == 15
    assert _append(lib, None, c, b) == 15
    assert lib.oxq_kv4_append(fake, None, b, 0xA000, 1, 1, 0xB000, 1, 1, 1) == 15
    read = lambda k, v, dt=1: lib.oxq_kv4_read(fake, c, b, k, v, dt)  # noqa: E731
    assert read(0xA000, 0xB000) == OK_BUT_NO_DEVICE
    assert read(0xA008, 0xB000) == 15 and read(0xA000, None) == 15 and read(0xA000, 0xB000, 9) == 15
    for kw in ({"tokens": 0}, {"seqs": 0}):              # nothing to do is not an error
        c, b, a = _descs(**kw)
        assert _append(lib, fake, c, b, k=None, v=None) == 0
        assert lib.oxq_kv4_read(fake, c, b, None, None, 1) == 0
        assert lib.oxq_kv4_attention(fake, c, b, a, None, 0) == 0


@pytest.mark.parametrize("key,value,status", [
    ("dtype", 0, 15), ("q_heads", 7, 12), ("q_heads", 0, 12), ("window", -1, 15), ("scale", float("nan"), 15), ("scale", float("inf"), 15), ("max_tokens", -1, 10), ("q", None, 15),
    ("out", None, 15), ("out", 0x9002, 15), ("out_token_stride", 1023, 15), ("q_token_stride", -1, 15), ("q_token_stride", 1023, OK_BUT_NO_DEVICE), ("dtype", 2, OK_BUT_NO_DEVICE),
    ("lse", 0xC000, OK_BUT_NO_DEVICE), ("window", 1 << 40, OK_BUT_NO_DEVICE), ("causal", 0, OK_BUT_NO_DEVICE)])
def test_attention(lib, fake, key, value, status):
    c, b, a = _descs(**{key: value})
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10000, 1 << 30) == status


@pytest.mark.parametrize("tokens,heads,strides,status", [
    (3, 8, (1024, 128), 13), (3, 8, (128, 384), 13), (3, 8, (1152, 132), 13),     # rows apart, in either order
    (3, 8, (0, 128), 15), (3, 8, (1024, 0), 15), (3, 8, (1024, 64), 15), (3, 8, (1022, 128), 15), (3, 8, (128, 382), 15), (3, 8, (128, 128), 15),
    (1, 8, (1, 128), 13), (1, 8, (0, 128), 13), (1, 8, (1024, 64), 15), (3, 2, (256, 128), 13), (3, 2, (254, 128), 15), (3, 2, ((1 << 62), 128), 13),
    (3, 2, (128, 1 << 62), 13), (1, 2, (0, 126), 15)])
def test_output_rows_that_overlap(lib, fake, tokens, heads, strides, status):
    c, b, a = _descs(tokens=tokens, q_heads=heads, out_token_stride=strides[0], out_head_stride=strides[1])
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10000, 1 << 30) == status


def test_the_strides_of_one_token_and_one_head_are_not_looked_at(lib, fake):
    c, b, a = _descs(tokens=1, heads=1, q_heads=1, q_token_stride=7, q_head_stride=5, out_token_stride=3, out_head_stride=1)
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10000, 1 << 30) == OK_BUT_NO_DEVICE


def test_attention_window_and_workspace(lib, fake):
    c, b, a = _descs(window=4, causal=0)
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10000, 1 << 30) == 15
    c, b, a = _descs()
    assert lib.oxq_kv4_attention(fake, c, b, a, None, 0) == OK_BUT_NO_DEVICE      # a machine of no SMs needs no workspace
    assert lib.oxq_kv4_attention(fake, c, b, a, 0x10008, 1 << 30) == 11
    assert lib.oxq_kv4_attention(fake, c, b, None, 0x10000, 1 << 30) == 15
    n = C.c_size_t(0)
    size = lambda c, b, heads, most, out=C.byref(n): lib.oxq_kv4_attention_workspace_bytes(fake, c, b, heads, most, out)  # noqa: E731
    assert size(c, b, 7, 0) == 12 and size(c, b, 8, -1) == 10 and size(c, b, 8, 0, None) == 15
    assert size(_descs(dim=96)[0], b, 8, 0) == 13
    assert size(c, b, 8, 0) == 0


def test_residual_norm(lib, fake):
    from oxicuda_b200 import _ffi

    def call(rows=4, cols=64, out=0x9000, scale=0xA000, fn="oxq_residual_rmsnorm_fp8", **kw):
        a = dict(y=0x1000, y_ld=64, dtype=1, residual=0x2000, residual_ld=64, residual_dtype=1, gate=0x3000, gate_ld=0, post_weight=0x4000, weight=0x5000, alpha=1.0,
                 eps=1e-5, residual_out=0x6000, residual_out_ld=64)
        a.update(kw)
        s = _ffi.residual_norm(*[0 if v is None else v for v in a.values()])
        if fn == "oxq_residual_rmsnorm":
            return lib.oxq_residual_rmsnorm(fake, s, rows, cols, out)
        if fn == "oxq_residual_rmsnorm_int8_rows":
            return lib.oxq_residual_rmsnorm_int8_rows(fake, s, rows, cols, out, scale)
        return lib.oxq_residual_rmsnorm_fp8(fake, s, rows, cols, scale, out)

    for fn in ("oxq_residual_rmsnorm", "oxq_residual_rmsnorm_fp8", "oxq_residual_rmsnorm_int8_rows"):
        assert call(fn=fn) == OK_BUT_NO_DEVICE
        assert call(fn=fn, rows=0) == 1 and call(fn=fn, cols=0) == 1
        assert call(fn=fn, cols=60) == 10 and call(fn=fn, cols=16392, y_ld=16392) == 10
        for key in ("y", "residual", "weight", "residual_out"):
            assert call(fn=fn, **{key: None}) == 15
        for key in ("y", "residual", "weight", "residual_out", "gate", "post_weight"):
            assert call(fn=fn, **{key: 0x1008}) == 15
        assert call(fn=fn, out=None) == 15 and call(fn=fn, out=0x9004) == 15
        for key in ("y_ld", "residual_ld", "residual_out_ld", "gate_ld"):
            assert call(fn=fn, **{key: 56}) == 15 and call(fn=fn, **{key: 68}) == 15
        assert call(fn=fn, dtype=5) == 15 and call(fn=fn, residual_dtype=2) == 13 and call(fn=fn, residual_dtype=0) == OK_BUT_NO_DEVICE
        assert call(fn=fn, gate=None, gate_ld=3, post_weight=None) == OK_BUT_NO_DEVICE
    assert call(scale=None) == 15 and call(fn="oxq_residual_rmsnorm_int8_rows", scale=None) == 15


def test_the_python_layer_takes_device_tensors_only():
    from oxicuda_b200 import ops
    x = torch.zeros(4, 64)
    with pytest.raises(TypeError):
        ops.residual_rmsnorm(x, x, torch.ones(64))
    codes, params = torch.zeros(2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 1, 16, 1, 2, dtype=torch.float16)
    with pytest.raises(TypeError):
        ops.Kv4Cache(codes, params, codes, params)


def test_the_layout_of_rows():
    """The places that the header states, walked element by element against a second statement of them."""
    for dim in (64, 128):
        for keys in (True, False):
            lanes = 4 if keys else 8
            seen = set()
            for d in range(dim):
                word = d // 8
                i, c = word // lanes, word % lanes
                place = c * (dim // (8 * lanes)) + i
                assert 0 <= place < dim // 8
                seen.add((place, d % 8))
                if keys:                                 # a quad's lane c holds words c, 4 + c, ... side by side: one load per row
                    assert place // (dim // 32) == c
                else:
                    assert place // (dim // 64) == c
            assert len(seen) == dim
