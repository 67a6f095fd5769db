"""The device operators' host side (include/azb200.h, "device operators"),
without a GPU: sizes, and every argument check, which comes before the device
is touched. Pointers here are made-up addresses that no call may follow."""
import ctypes as C

import pytest

import azb200 as E

P = 1 << 20   # an aligned address


def test_workspace():
    w = E.lib().azb_mx4_linear_workspace
    assert w(1, 4096, 4096) == 0 and w(2000, 3000, 8) == 2000 * 16 + 16 * 512
    assert w(8192, 8192, 8192) == 8192 * 4096 + 64 * 64 * 512
    assert w(2000, 0, 8) == w(2000, 3000, 0) == w(2000, (1 << 22) + 1, 8) == 0


def call(fn, *args):
    e = C.create_string_buffer(1024)
    rc = getattr(E.lib(), fn)(*args, e, 1024)
    return rc, e.value.decode()


def sizes(rows, cols):
    a, b = C.c_size_t(), C.c_size_t()
    rc, msg = call("azb_mx4_sizes", rows, cols, C.byref(a), C.byref(b))
    return (a.value, b.value) if rc == 0 else msg


@pytest.mark.parametrize("rows,cols,codes,scales", [
    (1, 1, 16, 512), (1, 32, 16, 512), (1, 33, 32, 512), (128, 128, 128 * 64, 512), (129, 129, 129 * 80, 4 * 512),
    (0, 64, 0, 0), (362, 722, 362 * 23 * 16, 3 * 6 * 512),
])
def test_sizes(rows, cols, codes, scales):
    assert sizes(rows, cols) == (codes, scales)


@pytest.mark.parametrize("rows,cols", [(-1, 4), (4, 0), (4, -3), ((1 << 22) + 1, 4), (4, (1 << 26) + 1)])
def test_sizes_refused(rows, cols):
    assert "azb_mx4_sizes: a matrix of" in sizes(rows, cols)
    assert E.lib().azb_mx4_linear_workspace(rows, 4, cols) == 0


def quantise(x=P, type=0, rows=2, cols=8, ld=8, codes=P, scales=P):
    return call("azb_mx4_quantise", 0, x, type, rows, cols, ld, codes, scales, None)


def product(xc=P, xs=P, m=2, wc=P, ws=P, n=3, k=8, bias=None, out=P, type=0, ld=3):
    return call("azb_mx4_product", 0, xc, xs, m, wc, ws, n, k, bias, 0, out, type, ld, None)


def linear(x=P, xt=0, m=2000, k=8, xld=8, wc=P, ws=P, n=3000, out=P, type=0, ld=3000, work=P, bytes=None):
    need = E.lib().azb_mx4_linear_workspace(m, n, k) if bytes is None else bytes
    return call("azb_mx4_linear", 0, x, xt, m, k, xld, wc, ws, n, None, 0, out, type, ld, work, need, None)


@pytest.mark.parametrize("fn,kw,text", [
    (quantise, dict(x=None), "null x"), (quantise, dict(type=2), "unknown element type 2"),
    (quantise, dict(cols=0), "a matrix of 2 x 0"), (quantise, dict(ld=-1), "negative row stride"),
    (quantise, dict(codes=None), "null codes or scales"), (quantise, dict(codes=P + 8), "aligned to 16"),
    (quantise, dict(x=P + 2), "aligned to 4"), (quantise, dict(x=P + 1, type=1), "aligned to 2"),
    (product, dict(xs=None), "null x"), (product, dict(wc=None), "null w"), (product, dict(out=None), "null out"),
    (product, dict(ld=2), "rows overlap"), (product, dict(m=-1), "a matrix of -1 x 8"),
    (product, dict(type=7), "unknown element type"), (product, dict(k=0), "a matrix of 2 x 0"),
    (product, dict(ws=P + 4), "aligned to 16"),
    (linear, dict(work=None), "the workspace holds"), (linear, dict(bytes=16), "the workspace holds 16 bytes of"),
    (linear, dict(work=P + 64), "aligned to 256"), (linear, dict(x=None), "null x or out"),
    (linear, dict(xld=-8), "negative row stride"), (linear, dict(xt=-1), "unknown element type -1"),
])
def test_mx4_refusals(fn, kw, text):
    rc, msg = fn(**kw)
    assert rc == -1 and text in msg, msg


def test_nothing_to_do_needs_no_gpu():
    assert quantise(rows=0, x=None, codes=None, scales=None)[0] == 0
    assert product(m=0, xc=None, xs=None, out=None)[0] == 0
    assert product(n=0, wc=None, ws=None, ld=0)[0] == 0
    assert sample(rows=0, logits=None, moves=None)[0] == 0


def sample(**kw):
    a = E.SampleArgs()
    a.logits, a.noise, a.moves = P, P, P
    a.rows, a.cols, a.ld, a.noise_ld = 2, 8, 8, 8
    a.temperature, a.top_p = 1.0, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return call("azb_sample_moves", 0, C.byref(a), None)


@pytest.mark.parametrize("kw,text", [
    (dict(logits=None), "null logits or moves"), (dict(moves=None), "null logits or moves"),
    (dict(noise=None), "null noise"), (dict(cols=0), "2 rows of 0"), (dict(rows=-1), "-1 rows of 8"),
    (dict(ld=-1), "negative row stride"), (dict(type=3), "unknown element type"),
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=1.5), "top_p"),
    (dict(top_p=float("nan")), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=2.0), "min_p"),
    (dict(moves=P + 4), "moves must be aligned to 8"), (dict(logits=P + 2), "aligned to 4"),
])
def test_sample_refusals(kw, text):
    rc, msg = sample(**kw)
    assert rc == -1 and text in msg, msg


def test_null_arguments():
    assert call("azb_sample_moves", 0, None, None) == (-1, "azb_sample_moves: null argument")
    assert E.lib().azb_infer_device_logits(None) is None


def test_python_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    import azb_ops as A

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        A.mx4_quantise(x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        A.mx4_quantise([1.0])
    with pytest.raises(ValueError, match="CUDA tensor"):
        A.sample_moves(x, x)
    with pytest.raises(ValueError, match="an Mx4 is needed"):
        A.mx4_product(x, x)
    with pytest.raises(ValueError, match="bytes of codes"):
        A.Mx4(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(4, dtype=torch.uint8), 2, 8)


@pytest.mark.parametrize("call_", [
    lambda at: product(bias=at),
    lambda at: call("azb_mx4_linear", 0, P, 0, 2, 8, 8, P, P, 3, at, 0, P, 0, 3, P, 1 << 20, None),
    lambda at: call("azb_mx4_linear", 0, P, 0, 2000, 8, 8, P, P, 3000, at, 0, P, 0, 3000, P, 1 << 20, None),
    lambda at: sample(temperature_rows=at), lambda at: sample(top_p_rows=at), lambda at: sample(min_p_rows=at),
    lambda at: sample(top_k_rows=at),
])
def test_misaligned_numbers_are_refused(call_):
    """The kernels read the bias and the per-row settings as whole 4-byte numbers."""
    for off in (1, 2, 3):
        rc, msg = call_(P + off)
        assert rc == -1 and "must be aligned to 4 bytes" in msg, msg
