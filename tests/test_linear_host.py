"""CPU: what the products with their epilogues and the plan of the ragged ones refuse, before
anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture
def pc():
    import pulsar_cuda

    return pulsar_cuda


def _refuses(pc, fn, base, cases):
    """Types and shapes are refused with a message before the device is looked at, which refuses
    the base call itself here: its tensors are on the CPU."""
    for msg, over in cases:
        args = dict(base, **over)
        with pytest.raises(RuntimeError, match=msg):
            getattr(pc, fn)(**args)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        getattr(pc, fn)(**base)


def test_group_rows_refusals(pc):
    idx = torch.zeros(3, 2, dtype=torch.int64)
    _refuses(pc, "moe_group_rows", dict(topk_idx=idx, num_experts=4), [
        ("topk_idx must be int64", dict(topk_idx=idx.int())),
        (r"topk_idx must be \[N, K\]", dict(topk_idx=idx.view(-1))),
        (r"topk_idx must be \[N, K\]", dict(topk_idx=idx[:, :0])),
        ("1 <= E <= 1024, got 0", dict(num_experts=0)),
        ("1 <= E <= 1024, got 1025", dict(num_experts=1025)),
    ])


def test_fused_linear_refusals(pc):
    bf = torch.bfloat16
    x, w = torch.zeros(5, 8, dtype=bf), torch.zeros(6, 8, dtype=bf)
    base = dict(x=x, weight=w)
    common = [
        ("x must be bfloat16 or float32", dict(x=x.double(), weight=w.double())),
        ("x must be bfloat16 or float32", dict(x=x.half(), weight=w.half())),
        ("weight must have the dtype of x", dict(weight=w.float())),
        (r"weight must be \[d_out, d_in\]", dict(weight=w[None])),
        (r"x must be \[\.\.\., d_in\]", dict(x=x[:, :7])),
        ("weight must not be empty", dict(x=x[:, :0], weight=w[:, :0])),
        ("weight must not be empty", dict(weight=w[:0])),
        ("activation must be one of", dict(activation="tanh")),
        ("even number of output columns, got 5", dict(weight=w[:5], activation="swiglu")),
    ]
    _refuses(pc, "fused_linear_forward", base, common + [
        ("bias must have the dtype", dict(bias=torch.zeros(6, dtype=torch.float64))),
        (r"bias must be \[6\]", dict(bias=torch.zeros(8, dtype=bf))),
        (r"residual must be \[5, 6\]", dict(residual=torch.zeros(5, 8, dtype=bf))),
        (r"residual must be \[5, 3\]", dict(residual=torch.zeros(5, 6, dtype=bf),
                                                 activation="swiglu")),
        ("residual must have the dtype", dict(residual=torch.zeros(5, 6))),
    ])
    dy = torch.zeros(5, 6, dtype=bf)
    _refuses(pc, "fused_linear_backward", dict(base, dy=dy), common + [
        (r"dy must be \[5, 6\]", dict(dy=dy[:4])),
        (r"dy must be \[5, 3\]", dict(activation="swiglu", pre=dy)),
        ("dy must have the dtype", dict(dy=dy.float())),
        ("pre is needed for every activation but none", dict(activation="gelu")),
        (r"pre must be \[5, 6\]", dict(activation="gelu", pre=dy[:, :3])),
    ])


def test_grouped_linear_refusals(pc):
    bf = torch.bfloat16
    x, w = torch.zeros(5, 8, dtype=bf), torch.zeros(2, 8, 6, dtype=bf)
    off = torch.tensor([0, 2, 5], dtype=torch.int32)
    base = dict(x=x, weight=w, offsets=off)
    common = [
        ("weight must have the dtype of x", dict(weight=w.float())),
        (r"weight must be \[E, d_in, d_out\]", dict(weight=w[0])),
        (r"x must be \[R, d_in\]", dict(x=x[None])),
        (r"x must be \[R, d_in\]", dict(x=x[:, :6])),
        ("offsets must be 1-dimensional int32", dict(offsets=off.long())),
        (r"offsets must have E \+ 1 elements", dict(offsets=off[:2])),
        ("rows must be 1-dimensional int32", dict(rows=off.long())),
        ("weight must not be empty", dict(weight=w[:0], offsets=off[:1])),
        ("activation must be one of", dict(activation="SiLU")),
    ]
    _refuses(pc, "grouped_linear_forward", base, common + [
        (r"bias must be \[2, 6\]", dict(bias=torch.zeros(6, dtype=bf))),
    ])
    dy = torch.zeros(5, 6, dtype=bf)
    _refuses(pc, "grouped_linear_backward", dict(base, dy=dy), common + [
        (r"dy must be \[5, 6\]", dict(dy=dy[:4])),
        (r"dy must be \[3, 6\]", dict(rows=off)),
    ])


def test_strides_are_refused_by_the_native_half():
    """Checked before any launch, so CPU tensors show it."""
    import pulsar_cuda as pc

    x, w = torch.zeros(5, 8), torch.zeros(6, 8)
    off = torch.tensor([0, 2, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="weight must have a unit stride"):
        pc._OPS.fused_linear_forward(x, torch.zeros(6, 16)[:, ::2], None, None, 0, 0)
    with pytest.raises(RuntimeError, match="x must be contiguous, or 2-dimensional"):
        pc._OPS.fused_linear_forward(torch.zeros(5, 16)[:, ::2], w, None, None, 0, 0)
    with pytest.raises(RuntimeError, match="x must be contiguous, or 2-dimensional"):
        pc._OPS.fused_linear_forward(torch.zeros(2, 8, 5).transpose(1, 2), w, None, None, 0, 0)
    with pytest.raises(RuntimeError, match="residual must be contiguous"):
        pc._OPS.fused_linear_forward(x, w, None, torch.zeros(6, 5).t(), 0, 0)
    with pytest.raises(RuntimeError, match="x must be contiguous, or 2-dimensional"):
        pc._OPS.grouped_linear_forward(torch.zeros(8, 5).t(), torch.zeros(2, 8, 6), off, None, None,
                                       0, 0)


def test_c_entries_refuse_before_any_launch():
    from pulsar_cuda import _lib

    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)
    bf = _lib.PULSAR_BF16

    def refused(rc, msg):
        assert rc != 0 and msg in lib.pulsar_last_error(), lib.pulsar_last_error()

    assert lib.pulsar_moe_group_rows_workspace_bytes(16, 4, 16) == 0
    assert lib.pulsar_moe_group_rows_workspace_bytes(16384, 4, 16) == 64 * 16 * 4
    for bad in ((-1, 4, 16), (4, 0, 16), (4, 4, 0), (4, 4, 1025), (2 ** 30, 4, 16)):
        assert lib.pulsar_moe_group_rows_workspace_bytes(*bad) == -1
    refused(lib.pulsar_moe_group_rows(p, p, p, p, 4, 4, 2000, None, None), b"bad shape")
    refused(lib.pulsar_moe_group_rows(None, p, p, p, 4, 4, 16, None, None), b"null pointer")
    refused(lib.pulsar_moe_group_rows(p, p, p, p, 16384, 4, 16, None, None), b"workspace")

    def fwd(x=p, x_rs=8, w=p, w_out=8, w_in=1, y=p, rows=4, d_in=8, d_out=6, act=0, dt=bf, bias=None,
            bdt=0, ws=None):
        return lib.pulsar_fused_linear_forward(x, x_rs, w, w_out, w_in, bias, bdt, None, 0, y, None,
                                               rows, d_in, d_out, act, dt, ws, None)

    for kw, msg in ((dict(x=None), b"null"), (dict(w=None), b"null"), (dict(y=None), b"null"),
                    (dict(dt=5), b"dtype"), (dict(act=7), b"activation"), (dict(act=-1), b"activation"),
                    (dict(act=6, d_out=5), b"even"), (dict(w_in=2, w_out=16), b"strides"),
                    (dict(w_out=7), b"overlap"), (dict(w_out=0), b"overlap"), (dict(x_rs=7), b"overlap"),
                    (dict(rows=-1), b"shape"), (dict(d_in=0), b"shape"), (dict(d_out=0), b"shape"),
                    (dict(rows=2 ** 31), b"shape"), (dict(bias=p, bdt=9), b"bias dtype"),
                    (dict(x_rs=9), b"workspace"), (dict(d_in=7), b"workspace"),
                    (dict(x_rs=9, ws=p.value + 8), b"workspace")):
        refused(fwd(**kw), msg)
    assert fwd(rows=0, x=None) == 0
    odd = p.value + 2

    def fwd_bytes(x=p, x_rs=8, w=p, w_out=8, w_in=1, rows=4, d_in=8, d_out=6, act=0):
        return lib.pulsar_fused_linear_forward_workspace_bytes(x, x_rs, w, w_out, w_in, rows, d_in,
                                                               d_out, act, bf)

    # whole aligned rows need none; a copy is padded to chunks of 8 elements and 256 bytes
    assert fwd_bytes() == 0 and fwd_bytes(rows=0, x=odd) == 0
    assert fwd_bytes(x=odd) == 256 and fwd_bytes(x_rs=9) == 256 and fwd_bytes(w=odd) == 256
    assert fwd_bytes(d_in=7, rows=100) == 100 * 16 + 192 + 256
    assert fwd_bytes(w_out=1, w_in=8) == 256 and fwd_bytes(w_out=1, w_in=8, d_out=8) == 0
    assert fwd_bytes(w_out=1, w_in=8, d_out=8, act=6) == 256
    assert fwd_bytes(d_out=0) == -1 and fwd_bytes(act=9) == -1
    n = lib.pulsar_fused_linear_backward_workspace_bytes(p, p, 8, p, 8, 1, 4, 8, 6, 2, bf)
    assert n == 256
    refused(lib.pulsar_fused_linear_backward(p, p, 8, p, 8, 1, p, p, p, None, 4, 8, 6, 2, bf, None,
                                             None), b"workspace")
    refused(lib.pulsar_fused_linear_backward(p, p, 8, p, 8, 1, None, p, p, None, 4, 8, 6, 2, bf, p,
                                             None), b"null")
    refused(lib.pulsar_grouped_linear_forward(p, 8, 4, None, None, p, 48, 6, 1, None, 0, p, None, 4,
                                              2, 8, 6, 0, bf, None, None), b"null")
    refused(lib.pulsar_grouped_linear_forward(p, 8, 4, None, p, p, 48, 6, 1, None, 0, p, None, 4,
                                              0, 8, 6, 0, bf, None, None), b"shape")
    refused(lib.pulsar_grouped_linear_forward(p, 8, 4, None, p, p, 48, 6, 1, None, 0, p, None, 4,
                                              2, 8, 6, 0, bf, None, None), b"workspace")
    refused(lib.pulsar_grouped_linear_backward(p, p, 8, 4, None, None, p, 48, 6, 1, None, p, p, None,
                                               4, 2, 8, 6, 0, bf, None, None), b"null")


def test_rows_of_x_without_an_index():
    """Row i is then x's row i: fewer rows of x than rows of y would be read past their end."""
    from pulsar_cuda import _lib

    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)
    for x_rows in (0, 3, 5):
        assert lib.pulsar_grouped_linear_forward(p, 8, x_rows, None, p, p, 64, 8, 1, None, 0, p, None, 4, 2,
                                                 8, 8, 0, _lib.PULSAR_BF16, None, None) != 0
        assert b"without an index" in lib.pulsar_last_error()
        assert lib.pulsar_grouped_linear_backward(p, p, 8, x_rows, None, p, p, 64, 8, 1, None, p, p, None,
                                                  4, 2, 8, 8, 0, _lib.PULSAR_BF16, None, None) != 0
        assert b"without an index" in lib.pulsar_last_error()
