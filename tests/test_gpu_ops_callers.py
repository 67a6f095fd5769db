"""Callers of the device operators (include/azb200.h, "device operators")
beside the plain one: several host threads, several users of one device's error
word, and torch's ways of following a computation, which these calls cannot
take part in and therefore refuse."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(engine):
    import azb_ops

    return azb_ops


def test_a_lost_gradient_is_refused(ops):
    """Forward-mode tangents and the noise's gradient as any other gradient."""
    import torch
    import torch.autograd.forward_ad as fw

    x, b = torch.ones(4, 64, device="cuda"), torch.ones(4, device="cuda")
    w = ops.mx4_quantise(x)
    noise = torch.rand(4, 64, device="cuda")
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.mx4_quantise(d), lambda: ops.mx4_product(d, w), lambda: ops.mx4_product(d[0], w),
                     lambda: ops.mx4_product(x, w, bias=fw.make_dual(b, b)), lambda: ops.sample_moves(d, noise),
                     lambda: ops.sample_moves(x, noise, temperature=fw.make_dual(b, b)),
                     lambda: ops.sample_moves(x, fw.make_dual(noise, noise))):
            with pytest.raises(ValueError, match="no backward pass"):
                call()
        ops.mx4_product(fw.unpack_dual(d).primal, w)
        with fw._set_fwd_grad_enabled(False):
            ops.mx4_quantise(d)
    with pytest.raises(ValueError, match="noise requires a gradient"):
        ops.sample_moves(x, noise.clone().requires_grad_())
    with torch.no_grad():
        ops.sample_moves(x, noise.clone().requires_grad_())


def test_a_negated_view_is_refused(ops):
    """A view whose values are its memory's, negated."""
    import torch

    x = torch.ones(4, 64, device="cuda")
    n = torch._neg_view(x)
    w = ops.mx4_quantise(x)
    for call in (lambda: ops.mx4_quantise(n), lambda: ops.mx4_product(n, w), lambda: ops.mx4_product(n[0], w),
                 lambda: ops.mx4_product(x, w, bias=torch._neg_view(x[0, :4])), lambda: ops.sample_moves(n, x),
                 lambda: ops.sample_moves(x, n), lambda: ops.sample_moves(x, x, temperature=torch._neg_view(x[:, 0].clone()))):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    assert bool((ops.mx4_values(ops.mx4_quantise(n.resolve_neg())) == -1).all())


def test_traces_and_wrapped_tensors_are_refused(ops):
    """The calls run below torch's dispatcher: a trace would hold their results
    as constants, and a tensor that stands for others has no memory to read."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    x = torch.ones(4, 64, device="cuda")
    w = ops.mx4_quantise(x)
    calls = (lambda x: ops.mx4_values(ops.mx4_quantise(x)), lambda x: ops.mx4_product(x, w), lambda x: ops.sample_moves(x, x)[0])
    for call in calls:
        with pytest.raises(ValueError, match="trac"):
            make_fx(call)(x)
        with pytest.raises(ValueError, match="trac"):
            torch.jit.trace(call, x)
        with pytest.raises(ValueError):
            torch.func.vmap(call)(x[None])
        with pytest.raises(ValueError):
            torch.func.grad(lambda x: call(x).sum())(x)
        with FakeTensorMode() as mode, pytest.raises(ValueError):
            call(mode.from_tensor(x))

    class Wrapped(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError("not reached")

    with pytest.raises(ValueError, match="subclass"):
        ops.mx4_quantise(torch.Tensor._make_subclass(Wrapped, x))

    class Counting(TorchDispatchMode):   # looks on, and is no trace
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Counting():
        assert torch.equal(ops.mx4_product(x, w), torch.full((4, 4), 64.0, device="cuda"))
    assert torch.equal(ops.mx4_product(torch.nn.Parameter(x, requires_grad=False), w), torch.full((4, 4), 64.0, device="cuda"))


@pytest.mark.parametrize("m,n,k", [(1, 100, 300), (40, 100, 300), (2000, 2000, 64)])
def test_a_host_threads_first_call_may_be_a_product(ops, m, n, k):
    """No call of that thread has touched the device before."""
    import torch

    x, w = ops.mx4_quantise(torch.ones(m, k, device="cuda")), ops.mx4_quantise(torch.ones(n, k, device="cuda"))
    plain = torch.ones(m, k, device="cuda")
    out = torch.zeros(m, n, device="cuda")
    torch.cuda.synchronize()
    got = {}

    def through_c():
        e = C.create_string_buffer(1024)
        rc = ops.azb200.lib().azb_mx4_product(0, *x.pointers(), m, *w.pointers(), n, k, None, 0, out.data_ptr(), 0, n, None, e, 1024)
        got["c"] = (rc, e.value)

    def through_python(name, x):
        try:
            got[name] = ops.mx4_product(x, w, dtype=torch.float32)
        except Exception as e:
            got[name] = e

    for target, args in ((through_c, ()), (through_python, ("mx4", x)), (through_python, ("plain", plain))):
        t = threading.Thread(target=target, args=args)
        t.start()
        t.join()
    torch.cuda.synchronize()
    ref = torch.full((m, n), float(k), device="cuda")
    assert got["c"] == (0, b"") and torch.equal(out, ref)
    for name in ("mx4", "plain"):
        assert isinstance(got[name], torch.Tensor) and torch.equal(got[name], ref), got[name]


def child(text):
    """Runs Python code in a process of its own, whose first calls are its."""
    env = dict(os.environ, PYTHONPATH=os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero-go_b200"))
    r = subprocess.run([sys.executable, "-c", text], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    return r.stdout


FIRST_CALLS = """
import ctypes as C, threading
import torch, azb200 as E
L = E.lib()
logits = torch.zeros(1, 1 << 17, device="cuda")
noise = torch.full((1, 1 << 17), 0.5, device="cuda")
moves = torch.zeros(64, dtype=torch.int64, device="cuda")
data = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
out = torch.zeros(1 << 14, device="cuda")
torch.cuda.synchronize()

def sample(cols, type):
    a = E.SampleArgs(logits=logits.data_ptr(), type=type, rows=1, cols=cols, ld=cols, noise=noise.data_ptr(), noise_ld=cols,
                     temperature=1.0, top_p=1.0, moves=moves.data_ptr())
    e = C.create_string_buffer(1024)
    return L.azb_sample_moves(0, C.byref(a), None, e, 1024), cols, type, e.value

def product(k, m):
    p = data.data_ptr()
    e = C.create_string_buffer(1024)
    return L.azb_mx4_product(0, p, p, m, p, p, 100, k, None, 0, out.data_ptr(), 0, 100, None, e, 1024), k, m, e.value

sets = [[(sample, c, t) for c in sizes] for t in (0, 1)
        for sizes in ([1100, 8192, 2000, 5000, 3000, 7000, 4000, 6000], [8200, 16384, 9000, 12000, 10000, 15000, 11000, 13000],
                      [16400, 32768, 40000, 65536, 20000, 60000, 50000, 30000])]
sets += [[(product, k, m) for k in (768, 512, 256, 600) for m in (1, 128)]]
failed = []
for calls in sets:
    ready = threading.Barrier(len(calls))
    def one(f, *args):
        ready.wait()
        r = f(*args)
        if r[0]: failed.append(r)
    threads = [threading.Thread(target=one, args=c) for c in calls]
    [t.start() for t in threads]
    [t.join() for t in threads]
    failed += [r for r in (c[0](*c[1:]) for c in calls) if r[0]]
torch.cuda.synchronize()
assert not failed, failed
"""


def test_first_calls_from_several_threads():
    """Every call of a kernel's first ones, of different sizes at once, and
    each of those sizes afterwards."""
    for _ in range(2):
        child(FIRST_CALLS)


def test_every_user_learns_of_a_wait_that_ran_out():
    """Whoever asks first, and after other products that went well."""
    out = child("""
import torch, azb200 as E, azb_ops as A
w = A.mx4_quantise(torch.ones(4, 64, device="cuda"))
A.check(0)
E.cuda_probe.ops_wait(1000000)
for user in ("first", "second"):
    try:
        A.check(0)
        print(user, "no error")
    except E.CudaError as e:
        print(user, e)
    assert bool((A.mx4_product(torch.ones(3, 64, device="cuda"), w) == 64).all())
""")
    assert [line.split(" ", 1) for line in out.splitlines()] == [[u, "cuda: bounded wait ran out"] for u in ("first", "second")]
