"""What the student operators (embedding, gated pair, distillation loss) refuse, answered on the host before any device is
touched, and their workspace sizes.  No GPU needed."""
import ctypes as C

import pytest

A = 1 << 20  # an address that looks like device memory; no call here gets as far as using it


def view(capi, data=A, offset=0, stride=(8, 1)):
    v = capi.View2()
    v.data, v.offset = data, offset
    v.stride[0], v.stride[1] = stride
    return C.byref(v)


def embed(tt, dtype=None, index_dtype=None, count=4, vocab=10, dim=8, index=A, table=2 * A, rs=8, cs=1, out=3 * A):
    capi = tt._capi
    return capi.lib.ttamd_embedding_forward(0, capi.F32 if dtype is None else dtype, capi.I32 if index_dtype is None else index_dtype, count,
                                            vocab, dim, index, table, rs, cs, 1.0, out, None)


def test_embedding_refusals(tt):
    capi = tt._capi
    assert embed(tt, dtype=capi.I32) == capi.ERR_UNSUPPORTED_DTYPE
    assert embed(tt, dtype=42) == capi.ERR_UNSUPPORTED_DTYPE
    for bad in (capi.F32, capi.U8, capi.BOOL, 42):
        assert embed(tt, index_dtype=bad) == capi.ERR_UNSUPPORTED_DTYPE
    for kw in (dict(count=-1), dict(vocab=0), dict(dim=0), dict(count=1 << 31), dict(vocab=(1 << 28) + 1), dict(dim=(1 << 21) + 1),
               dict(rs=-1), dict(cs=-1), dict(index=None), dict(table=None), dict(out=None), dict(table=A + 2), dict(out=A + 1),
               dict(index=A + 2)):
        assert embed(tt, **kw) == capi.ERR_INVALID_ARGUMENT, kw
        assert b"embedding" in capi.lib.ttamd_last_error_string()


def test_embedding_backward_refusals(tt):
    capi, lib = tt._capi, tt._capi.lib
    n = C.c_size_t()
    query = lib.ttamd_embedding_backward_workspace
    assert query(capi.I32, 4, 10, 8, C.byref(n)) == capi.ERR_UNSUPPORTED_DTYPE
    assert query(capi.F32, 4, 0, 8, C.byref(n)) == capi.ERR_INVALID_ARGUMENT
    assert query(capi.F32, 4, 10, 8, None) == capi.ERR_INVALID_ARGUMENT
    # a long list of positions of a huge table, which would keep the device busy for minutes
    assert query(capi.F32, 1 << 30, 1 << 28, 1, C.byref(n)) == capi.ERR_INVALID_ARGUMENT
    assert query(capi.F32, (1 << 20) + 1, 1 << 28, 1, C.byref(n)) == capi.ERR_INVALID_ARGUMENT
    assert query(capi.F32, 1 << 20, 1 << 28, 1, C.byref(n)) == capi.OK
    assert query(capi.F32, (1 << 31) - 1, 1 << 17, 1, C.byref(n)) == capi.OK
    assert query(capi.F32, 4, 10, 8, C.byref(n)) == capi.OK and n.value == 0  # few positions need none
    assert query(capi.F32, 400, 10, 8, C.byref(n)) == capi.OK and n.value > 0
    need = n.value

    def call(index_dtype=capi.I32, count=400, dy=A, index=2 * A, grad=3 * A, ws=4 * A, size=need):
        return lib.ttamd_embedding_backward(0, capi.F32, index_dtype, count, 10, 8, dy, index, 1.0, 0, grad, ws, size, None)

    assert call(index_dtype=capi.F32) == capi.ERR_UNSUPPORTED_DTYPE
    for kw in (dict(count=-1), dict(dy=None), dict(index=None), dict(grad=None), dict(ws=None), dict(size=need - 1), dict(dy=A + 1),
               dict(grad=A + 2), dict(ws=A + 4), dict(index=A + 1)):
        assert call(**kw) == capi.ERR_INVALID_ARGUMENT, kw


def test_gated_linear_refusals(tt):
    capi, lib = tt._capi, tt._capi.lib
    n = C.c_size_t()
    assert lib.ttamd_gated_linear_workspace(capi.I64, 3, 8, 8, 0, C.byref(n)) == capi.ERR_UNSUPPORTED_DTYPE
    assert lib.ttamd_gated_linear_workspace(capi.F32, 3, 0, 8, 0, C.byref(n)) == capi.ERR_INVALID_ARGUMENT
    assert lib.ttamd_gated_linear_workspace(capi.F32, 3, 8, 8, 0, None) == capi.ERR_INVALID_ARGUMENT
    for big in (((1 << 26) + 1, 1, 1), (1, (1 << 26) + 1, 1), (1, 1, (1 << 26) + 1), (1 << 26, 1 << 15, 1), (1, 1 << 26, 1 << 15)):
        assert lib.ttamd_gated_linear_workspace(capi.F32, *big, 1, C.byref(n)) == capi.ERR_INVALID_ARGUMENT, big
    for large in ((1 << 26, 1, 1), (1, 1 << 26, 1), (1, 1, 1 << 26)):
        assert lib.ttamd_gated_linear_workspace(capi.F32, *large, 1, C.byref(n)) == capi.OK, large
    assert lib.ttamd_gated_linear_workspace(capi.F32, 3, 8, 8, 1, C.byref(n)) == capi.OK

    def forward(dtype=capi.F32, act=0, rows=3, x=view(capi), wg=view(capi), wu=view(capi), out=2 * A, gate=None, up=None, ws=3 * A, size=1 << 30):
        return lib.ttamd_gated_linear_forward(0, dtype, act, rows, 8, 8, x, wg, wu, None, None, out, gate, up, ws, size, None)

    assert forward(dtype=capi.I32) == capi.ERR_UNSUPPORTED_DTYPE
    for kw in (dict(act=4), dict(act=-1), dict(rows=-1), dict(x=None), dict(wg=view(capi, data=None)), dict(wu=view(capi, offset=-1)),
               dict(wu=view(capi, stride=(8, -1))), dict(x=view(capi, stride=((1 << 32) + 1, 1))), dict(x=view(capi, data=A + 2)), dict(out=None), dict(out=A + 1), dict(gate=4 * A),
               dict(up=4 * A), dict(ws=3 * A + 4)):
        assert forward(**kw) == capi.ERR_INVALID_ARGUMENT, kw

    def backward(act=0, dh=A, gate=A, up=A, dx=2 * A, dwg=3 * A, dwu=4 * A, ws=5 * A, size=1 << 30, x=view(capi)):
        return lib.ttamd_gated_linear_backward(0, capi.F32, act, 3, 8, 8, dh, x, view(capi), view(capi), gate, up, dx, dwg, dwu, None, None, ws, size, None)

    for kw in (dict(act=9), dict(dh=None), dict(gate=None), dict(up=None), dict(dx=None), dict(dwg=None), dict(dwu=None), dict(ws=None),
               dict(size=8), dict(dh=A + 2), dict(dwu=A + 3), dict(x=None)):
        assert backward(**kw) == capi.ERR_INVALID_ARGUMENT, kw


def test_distill_loss_refusals(tt):
    capi, lib = tt._capi, tt._capi.lib
    n = C.c_size_t()
    query = lib.ttamd_distill_loss_workspace
    assert query(capi.BOOL, 3, 8, 2, C.byref(n)) == capi.ERR_UNSUPPORTED_DTYPE
    for rows, cols, top in ((-1, 8, 2), (3, 0, 2), (3, 8, 0), (3, 8, 1025), (3, 1 << 30, 2)):
        assert query(capi.F32, rows, cols, top, C.byref(n)) == capi.ERR_INVALID_ARGUMENT
    assert query(capi.F32, 3, 8, 2, C.byref(n)) == capi.OK
    need = n.value

    def call(index_dtype=capi.I64, z=A, stride=8, index=2 * A, logit=3 * A, weight=None, t=1.0, loss=4 * A, grad=5 * A, ws=6 * A, size=need):
        return lib.ttamd_distill_loss(0, capi.F32, index_dtype, 3, 8, 2, z, stride, index, logit, weight, t, loss, grad, ws, size, None)

    for bad in (capi.U8, capi.F32):
        assert call(index_dtype=bad) == capi.ERR_UNSUPPORTED_DTYPE
    for kw in (dict(stride=7), dict(t=0.0), dict(t=-1.0), dict(t=float("nan")), dict(t=float("inf")), dict(z=None), dict(index=None),
               dict(logit=None), dict(loss=None), dict(grad=None), dict(ws=None), dict(size=need - 1), dict(z=A + 2), dict(index=A + 4),
               dict(weight=A + 1), dict(ws=A + 4), dict(grad=A), dict(grad=A + 4 * 16)):
        assert call(**kw) == capi.ERR_INVALID_ARGUMENT, kw
    call(grad=A)
    assert b"the gradient shares memory with the logits" in lib.ttamd_last_error_string()


def test_shared_memory_is_refused(tt):
    """A result over an operand or another result; what only lies between an operand's rows, or next to it, is left alone."""
    capi, lib = tt._capi, tt._capi.lib

    def shared(status):
        return status == capi.ERR_INVALID_ARGUMENT and b"shares memory with" in lib.ttamd_last_error_string()

    # table: rows of 32 bytes, 64 apart (10 of them); out: 128 bytes
    assert shared(embed(tt, rs=16, out=2 * A + 9 * 64 + 28)) and not shared(embed(tt, rs=16, out=2 * A + 9 * 64 + 32))
    assert shared(embed(tt, rs=16, out=2 * A - 124)) and not shared(embed(tt, rs=16, out=2 * A - 128))
    assert shared(embed(tt, count=1, rs=16, out=2 * A + 28)) and not shared(embed(tt, count=1, rs=16, out=2 * A + 32))
    assert shared(embed(tt, count=1, rs=16, out=2 * A + 36))
    assert shared(embed(tt, out=A + 12)) and not shared(embed(tt, out=A + 16))                  # over the indices, behind them
    # columns 64 bytes apart, rows neighbours (a transposed view): 10 x 4 bytes in each
    assert shared(embed(tt, count=1, dim=2, rs=1, cs=16, out=2 * A + 36)) and not shared(embed(tt, count=1, dim=2, rs=1, cs=16, out=2 * A + 40))
    assert shared(embed(tt, count=1, dim=2, rs=1, cs=16, out=2 * A + 100)) and not shared(embed(tt, count=1, dim=2, rs=1, cs=16, out=2 * A + 104))
    assert shared(embed(tt, rs=0, cs=0, out=2 * A)) and not shared(embed(tt, rs=0, cs=0, out=2 * A + 4))
    assert shared(embed(tt, vocab=1 << 28, rs=1 << 32, out=2 * A + (9 << 34)))                  # (a reach of 2^62 bytes)

    def scatter(dy=A, index=2 * A, grad=3 * A, ws=4 * A):
        return lib.ttamd_embedding_backward(0, capi.F32, capi.I32, 400, 10, 8, dy, index, 1.0, 0, grad, ws, A, None)

    assert not shared(scatter())
    for kw in (dict(grad=A), dict(grad=2 * A), dict(ws=A), dict(ws=2 * A), dict(ws=3 * A), dict(grad=A + 399 * 32)):
        assert shared(scatter(**kw)), kw

    def forward(out=2 * A, gate=3 * A, up=4 * A, ws=5 * A, bg=6 * A, bu=None):
        return lib.ttamd_gated_linear_forward(0, capi.F32, 0, 3, 8, 8, view(capi), view(capi, 7 * A), view(capi, 8 * A, 1), bg, bu, out, gate, up, ws, A, None)

    assert not shared(forward())
    for kw in (dict(out=A), dict(out=7 * A), dict(out=8 * A + 4), dict(out=3 * A), dict(gate=4 * A), dict(up=A), dict(ws=A), dict(ws=2 * A), dict(out=6 * A),
               dict(bu=2 * A)):
        assert shared(forward(**kw)), kw

    def backward(dx=2 * A, dwg=3 * A, dwu=4 * A, dbg=9 * A, dbu=10 * A, ws=5 * A):
        return lib.ttamd_gated_linear_backward(0, capi.F32, 0, 3, 8, 8, 6 * A, view(capi), view(capi, 7 * A), view(capi, 8 * A), 11 * A, 12 * A, dx, dwg, dwu, dbg,
                                               dbu, ws, A, None)

    assert not shared(backward())
    for kw in (dict(dx=A), dict(dx=6 * A), dict(dx=11 * A), dict(dx=12 * A), dict(dwg=7 * A), dict(dwu=8 * A), dict(dwg=4 * A), dict(dbg=10 * A), dict(dbu=A),
               dict(ws=9 * A), dict(ws=A)):
        assert shared(backward(**kw)), kw

    def distill(z=A, stride=16, index=2 * A, logit=3 * A, weight=None, loss=4 * A, grad=5 * A, ws=6 * A):
        return lib.ttamd_distill_loss(0, capi.F32, capi.I64, 3, 8, 2, z, stride, index, logit, weight, 1.0, loss, grad, ws, A, None)

    assert not shared(distill()) and not shared(distill(loss=A + 32))                           # (between two rows of logits)
    for kw in (dict(loss=A + 64), dict(grad=2 * A), dict(grad=3 * A), dict(loss=5 * A), dict(ws=A), dict(ws=5 * A), dict(weight=4 * A)):
        assert shared(distill(**kw)), kw


class _Memory:
    """A storage without a device behind it."""

    def __init__(self, device):
        self.ptr, self.nbytes, self.device = A, 1 << 20, device


def test_python_argument_checks(tt):
    capi, Dev = tt._capi, tt.Device("amd", 1)

    def t(shape, dtype=capi.F32, device=tt.kAMD, stride=None):
        return tt.Tensor(_Memory(device), dtype, shape, stride)

    ids, table = t((2, 3), capi.I64), t((10, 8))
    for call in (
        lambda: tt.embedding(ids, t((10, 8, 1))),
        lambda: tt.embedding(t((2, 3)), table),
        lambda: tt.embedding(t((2, 3), capi.BOOL), table),
        lambda: tt.embedding(ids, t((10, 8), capi.I32)),
        lambda: tt.embedding(t((2, 3), capi.I64, Dev), table),
        lambda: tt.embedding(ids, table, out=t((2, 8))),
        lambda: tt.embedding(ids, table, out=t((2, 3, 8), capi.F64)),
        lambda: tt.embedding(ids, table, out=t((2, 3, 8), stride=(48, 16, 2))),
        lambda: tt.embedding_backward(t((2, 4, 8)), ids, 10),
        lambda: tt.embedding_backward(t((2, 3, 8)), ids, 10, accumulate=True),
        lambda: tt.embedding_backward(t((2, 3, 8)), ids, 10, out=t((9, 8))),
        lambda: tt.gated_linear(t((4, 8)), t((8, 6)), t((8, 5))),
        lambda: tt.gated_linear(t((4, 7)), t((8, 6)), t((8, 6))),
        lambda: tt.gated_linear(t((4, 8)), t((8, 6)), t((8, 6), capi.F64)),
        lambda: tt.gated_linear(t((4, 8)), t((8, 6)), t((8, 6)), activation="tanh"),
        lambda: tt.gated_linear(t((4, 8)), t((8, 6)), t((8, 6)), b_gate=t((5,))),
        lambda: tt.gated_linear(t((4, 8)), t((8, 6)), t((8, 6)), out=t((4, 5))),
        lambda: tt.gated_linear_backward(t((4, 6)), t((4, 8)), t((8, 6)), t((8, 6)), t((4, 6)), t((4, 5))),
        lambda: tt.gated_linear_backward(t((4, 6)), t((2, 2, 8)), t((8, 6)), t((8, 6)), t((4, 6)), t((4, 6))),
        lambda: tt.gated_linear_backward(t((4, 6)), t((4, 8)), t((8, 6)), t((8, 6)), t((4, 6)), t((4, 6)), out=(None,) * 3),
        lambda: tt.distill_loss(t((4, 8)), t((4, 2), capi.I64), t((4, 3))),
        lambda: tt.distill_loss(t((4, 8)), t((5, 2), capi.I64), t((5, 2))),
        lambda: tt.distill_loss(t((4, 8)), t((4, 2)), t((4, 2))),
        lambda: tt.distill_loss(t((4, 8)), t((4, 2), capi.I32), t((4, 2), capi.F64)),
        lambda: tt.distill_loss(t((4, 8)), t((4, 2), capi.I32), t((4, 2)), row_weight=t((3,))),
        lambda: tt.distill_loss(t((4, 8)), t((4, 2), capi.I32), t((4, 2)), out=(t((1,)), t((4, 9)))),
    ):
        with pytest.raises(tt.TTException):
            call()


def test_gated_variant_names(tt):
    """The kernels by size and view, without a device."""
    capi = tt._capi

    def name(rows, inner, hidden, backward=0, code=capi.F32, order=(1, 1, 1), address=256):
        views = []
        for cols, lines, col in zip((inner, hidden, hidden), (rows, inner, inner), order):
            v = capi.View2()
            v.data, v.stride[0], v.stride[1] = address, cols if col == 1 else 1, 1 if col == 1 else lines
            views.append(v)
        return capi.lib.ttamd_gated_linear_variant(code, rows, inner, hidden, *(C.byref(v) for v in views), backward).decode()

    assert [name(n, 1024, 4096) for n in (1, 2, 3, 4)] == ["gated_f32_rows%d" % n for n in (1, 2, 4, 4)]
    assert name(16, 1024, 4096) == "gated_f32_few16" and name(32, 2048, 8192) == "gated_f32_few32"
    assert name(1024, 784, 1024) == "gated_f32_64x128_halves" and name(4096, 1024, 4096) == "gated_f32_256x128"
    assert name(777, 500, 1001, code=capi.F64) == "gated_f64_64x64"
    assert name(16, 1024, 4096, order=(1, 0, 1)) == "gated_f32_products"
    assert name(4096, 1024, 4096, 1).startswith("gated_backward_f32_128x128") and name(64, 64, 64, 1) == "gated_backward_f32_64x64"
    assert name(300, 4, 1 << 20, 1, capi.F64) == "gated_backward_f64_products"
    assert name(0, 4, 4) == "empty" and name(0, 4, 4, 1) == "empty"
    assert name(1, 0, 4) == "invalid" and name(1, 4, 4, code=capi.I32) == "invalid" and name(1, 4, 4, address=257) == "invalid"
    assert capi.lib.ttamd_gated_linear_variant(capi.F32, 1, 4, 4, None, None, None, 0) == b"invalid"
