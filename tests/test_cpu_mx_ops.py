"""Microscaled operators without a GPU: the oracle against torch's own number types, and everything the entry points refuse."""
import numpy as np
import pytest
import torch

from clip_assisted_data_labeling_amd import _lib, mx_ops as mx
from oracle import mx_oracle as ora


def test_the_oracle_rounds_like_the_types():
    f = np.float32
    v = np.concatenate([np.linspace(0, 460, 20001), ora.grid("e4m3"), (ora.grid("e4m3")[1:] + ora.grid("e4m3")[:-1]) / 2]).astype(f)
    want = torch.from_numpy(v).clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ora.nearest_code(v.astype(np.float64), "e4m3"), want)
    half = {0.25: 0, 0.75: 2, 1.25: 2, 1.75: 4, 2.5: 4, 3.5: 6, 5.0: 6, 7.0: 7, 0.26: 1, 0.74: 1, 5.01: 7, 4.99: 6}
    assert ora.nearest_code(np.array(list(half)), "e2m1").tolist() == list(half.values())
    codes, scale = ora.quantize(np.array([[7.9] + [0.0] * 31, [8.0] + [0.0] * 31]), "e2m1")
    assert codes[:, 0].tolist() == [7, 6] and scale[:, 0].tolist() == [127, 128]
    assert ora.values(codes, scale, "e2m1", 1).ravel().tolist() == [6.0, 8.0]


def test_quantising_twice_changes_nothing():
    x = np.random.RandomState(0).randn(5, 200) * 3
    for fmt in ("e2m1", "e4m3"):
        c, s = ora.quantize(x, fmt)
        v = ora.values(c, s, fmt, 200)
        c2, s2 = ora.quantize(v, fmt)
        assert np.array_equal(ora.values(c2, s2, fmt, 200), v)
        assert np.array_equal(ora.unpack(ora.pack(c, fmt), fmt), c)


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(2, 64)
    q = mx.MXTensor(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), "e2m1", 64)
    for call in (lambda: mx.quantize(x), lambda: mx.norm_quantize(x, torch.ones(64)), lambda: mx.dequantize(q), lambda: mx.linear(q, q)):
        with pytest.raises(_lib.ClipencError, match="no CPU path"):
            call()


P = 4096      # an address that is never read: every call below is refused before anything is launched


def _refused(name, *args, match):
    lib = _lib.load()
    assert getattr(lib, name)(*args) != 0
    assert match in lib.clipenc_last_error().decode(), lib.clipenc_last_error()


@pytest.mark.parametrize("args,match", [
    ((None, 0, 2, 64, 64, 0, P, P, None), "NULL"), ((P, 0, 2, 64, 64, 0, None, P, None), "NULL"), ((P, 0, 2, 64, 64, 0, P, None, None), "NULL"),
    ((P, 3, 2, 64, 64, 0, P, P, None), "in_dtype"), ((P, 0, -1, 64, 64, 0, P, P, None), "rows"), ((P, 0, 2, 0, 64, 0, P, P, None), "columns"),
    ((P, 0, 2, (1 << 20) + 1, 1 << 21, 0, P, P, None), "columns"), ((P, 0, 2, 64, 63, 0, P, P, None), "apart"), ((P, 0, 2, 64, 64, 2, P, P, None), "fmt"),
    ((P + 1, 0, 2, 64, 64, 0, P, P, None), "aligned"), ((P, 0, 2, 64, 64, 0, P + 8, P, None), "aligned"), ((P, 0, 2, 64, 64, 0, P, P + 2, None), "aligned")])
def test_quant_refuses(args, match):
    _refused("clipenc_op_quant_mx", *args, match=match)


@pytest.mark.parametrize("args,match", [
    ((None, P, 0, 2, 64, P, 0, None), "NULL"), ((P, P, 3, 2, 64, P, 0, None), "fmt"), ((P, P, 0, 2, 64, P, 4, None), "out_dtype"),
    ((P, P, 0, 2, 0, P, 0, None), "columns"), ((P, P, 0, 2, 64, None, 0, None), "NULL"), ((P, P, 0, 2, 64, P + 2, 2, None), "aligned")])
def test_dequant_refuses(args, match):
    _refused("clipenc_op_dequant_mx", *args, match=match)


def _norm(**k):
    a = dict(x=P, dt=0, rows=2, k=64, ld=64, r=P, ldr=64, norm=0, g=P, b=None, eps=1e-6, fmt=1, h=P + 65536, q=P, s=P, st=None)
    a.update(k)
    return tuple(a.values())


@pytest.mark.parametrize("change,match", [
    (dict(x=None), "NULL"), (dict(g=None), "gamma"), (dict(g=P + 2), "4-byte"), (dict(b=P + 1), "4-byte"), (dict(q=None), "NULL"), (dict(s=None), "NULL"), (dict(h=None), "together"),
    (dict(r=None), "together"), (dict(k=16385, ld=16385, ldr=16385), "at most"), (dict(norm=2), "norm"), (dict(fmt=3), "fmt"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(ldr=63), "apart"), (dict(dt=7), "in_dtype"), (dict(h=P, ld=70), "only where"), (dict(h=P + 65537), "aligned"), (dict(rows=-3), "rows")])
def test_norm_refuses(change, match):
    _refused("clipenc_op_norm_quant_mx", *_norm(**change), match=match)


def _gemm(**k):
    a = dict(a=P, sa=P, fmt=1, w=P, sw=P, m=4, n=8, k=64, bias=None, act=-1, res=None, out=P, dt=0, st=None)
    a.update(k)
    return tuple(a.values())


@pytest.mark.parametrize("change,match", [
    (dict(a=None), "NULL"), (dict(sa=None), "NULL"), (dict(w=None), "NULL"), (dict(sw=None), "NULL"), (dict(out=None), "NULL"), (dict(fmt=2), "a_fmt"), (dict(m=-1), "shape"),
    (dict(n=-1), "shape"), (dict(k=0), "shape"), (dict(k=1 << 21), "shape"), (dict(act=2), "act"), (dict(act=0, res=P), "exclusive"), (dict(dt=5), "out_dtype"),
    (dict(a=P + 8), "aligned"), (dict(w=P + 1), "aligned"), (dict(sw=P + 1), "aligned"), (dict(bias=P + 2), "aligned"), (dict(out=P + 1), "aligned"), (dict(res=P + 1), "aligned")])
def test_gemm_refuses(change, match):
    _refused("clipenc_op_gemm_mx", *_gemm(**change), match=match)


def _linear(**k):
    a = dict(x=P, dt=0, ld=64, fmt=1, w=P, sw=P, m=400, n=8, k=64, bias=None, act=-1, res=None, out=P, odt=0, ws=P, wsb=1 << 20, st=None)
    a.update(k)
    return tuple(a.values())


@pytest.mark.parametrize("change,match", [
    (dict(x=None), "NULL"), (dict(ld=63), "apart"), (dict(dt=3), "in_dtype"), (dict(fmt=2), "x_fmt"), (dict(ws=None), "scratch"), (dict(wsb=100), "scratch"), (dict(ws=P + 8), "scratch"),
    (dict(w=None), "NULL"), (dict(act=9), "act"), (dict(out=None), "NULL"), (dict(k=0, ld=64), "shape")])
def test_linear_refuses(change, match):
    _refused("clipenc_op_linear_mx", *_linear(**change), match=match)


def test_zero_rows_launch_nothing():
    lib = _lib.load()
    assert lib.clipenc_op_quant_mx(None, 0, 0, 64, 64, 0, None, None, None) == 0
    assert lib.clipenc_op_dequant_mx(None, None, 0, 0, 64, None, 0, None) == 0
    assert lib.clipenc_op_norm_quant_mx(None, 0, 0, 64, 64, None, 0, 0, None, None, 1e-6, 1, None, None, None, None) == 0
    assert lib.clipenc_op_gemm_mx(None, None, 1, None, None, 0, 8, 64, None, -1, None, None, 0, None) == 0
    assert lib.clipenc_op_linear_mx(None, 0, 64, 1, None, None, 0, 8, 64, None, -1, None, None, 0, None, 0, None) == 0
    assert lib.clipenc_op_linear_mx_ws_bytes(0, 8, 64, 1) == 0 and lib.clipenc_op_linear_mx_ws_bytes(400, 8, 64, 1) >= 400 * (64 + 2)


@pytest.mark.parametrize("change", [dict(m=(1 << 30) + 1), dict(n=(1 << 30) + 1)])
def test_linear_refuses_more_rows_than_its_indices_hold(change):
    _refused("clipenc_op_linear_mx", *_linear(**change), match="at most")


@pytest.mark.parametrize("rows,out", [((1 << 30) + 1, 4), (3, (1 << 32) + 3)])
def test_the_wrapper_refuses_more_rows_than_an_int_holds(monkeypatch, rows, out):
    checked = iter([(0, 0, out, 64), (1, 0, rows, 64)])
    monkeypatch.setattr(mx, "_check_quantised", lambda *a: next(checked))
    q = mx.MXTensor(None, None, "e4m3", 64)
    with pytest.raises(ValueError, match="at most"):
        mx.linear(q, q)


class _Wide:
    """A tensor on a GPU of more columns than 32 bits hold, as far as the checks look at it."""
    is_cuda, dtype, shape, requires_grad = True, torch.bfloat16, (1, (1 << 32) + 64), False

    def stride(self):
        return (1 << 32) + 64, 1

    def get_device(self):
        return 0


def test_the_wrapper_refuses_more_columns_than_an_int_holds():
    x = _Wide()
    for call in (lambda: mx.quantize(x), lambda: mx.norm_quantize(x, torch.ones(64)), lambda: mx.linear(x, _coded(64))):
        with pytest.raises(ValueError, match="columns"):
            call()
    for cols in ((1 << 32) + 64, (1 << 20) + 1, 0, -64):
        for call in (lambda: mx.dequantize(_coded(cols)), lambda: mx.linear(_coded(cols), _coded(64)), lambda: mx.linear(_coded(64), _coded(cols))):
            with pytest.raises(ValueError, match="columns"):
                call()


def _coded(cols):
    """Says that it has `cols` columns, on what would be a GPU."""
    class Data:
        is_cuda, dtype, shape, device = True, torch.uint8, (1, max(cols, 0) + 127 >> 7 << 6), "cuda:0"
        is_contiguous, get_device = (lambda self: True), (lambda self: 0)

    class Scale(Data):
        requires_grad = False
        shape = (1, max(cols, 0) + 127 >> 7 << 2)
    return mx.MXTensor(Data(), Scale(), "e2m1", cols)


def test_tensors_that_require_a_gradient_are_refused():
    """Their gradient would be lost without a word; under no_grad they get as far as any CPU tensor."""
    x, r, v, p = torch.zeros(2, 64), torch.zeros(2, 64), torch.ones(64), lambda t: torch.nn.Parameter(t.clone())
    q = mx.MXTensor(torch.zeros(64, 64, dtype=torch.uint8), torch.zeros(64, 4, dtype=torch.uint8), "e2m1", 64)
    row = mx.MXTensor(torch.zeros(2, 128, dtype=torch.uint8), p(v[:2]), "e4m3_row", 64)
    calls = [lambda: mx.dequantize(row), lambda: mx.quantize(p(x)), lambda: mx.norm_quantize(p(x), v), lambda: mx.norm_quantize(x, p(v)), lambda: mx.norm_quantize(x, v, bias=p(v)),
             lambda: mx.norm_quantize(x, v, residual=p(r)), lambda: mx.linear(p(x), q), lambda: mx.linear(x, q, bias=p(v)), lambda: mx.linear(q, q, bias=p(v)),
             lambda: mx.linear(x, q, residual=p(r)), lambda: mx.linear(x * p(x), q)]
    for call in calls:
        with pytest.raises(ValueError, match="no backward"):
            call()
    with torch.no_grad():
        for call in calls:
            with pytest.raises(_lib.ClipencError, match="no CPU path"):
                call()
