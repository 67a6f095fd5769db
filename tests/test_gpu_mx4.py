"""4-bit microscaled matrices on the GPU against the form's definition in 64
bits (numpy, from the element's bits; include/azb200.h states it).

Quantised values are exact, so they are compared for equality. A product's
tolerance is that of an fp32 sum of K exact terms in any order, each addition
off by at most one unit in the last place of a partial sum (the tensor core
may truncate), which no partial sum's magnitude sum |x||w| exceeds:
K * 2^-23 * sum |x||w|, and one more rounding for the bias and one for the
float32 output. A bfloat16 output is the float32 one rounded to nearest even,
bit for bit.
"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TABLE = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@pytest.fixture(scope="module")
def ops(engine):
    import azb_ops

    return azb_ops


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def quantised(x):
    """The values x's 4-bit form holds, in 64 bits."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32), np.float32)
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(v).max(-1)
    field = (top.view(np.int32) >> 23) & 255
    e = np.maximum(field - 129, -127)
    scale = np.ldexp(1.0, e)[..., None]
    bad = ~np.isfinite(v).all(-1)
    y = np.where(bad[..., None], 0, v).astype(np.float64) / scale
    d = np.abs(np.abs(y)[..., None] - TABLE)
    best = d.min(-1)
    code = np.where((d[..., ::2] == best[..., None]).any(-1), d[..., ::2].argmin(-1) * 2, d.argmin(-1))
    out = np.copysign(TABLE[code], y) * scale
    out[bad] = np.nan
    return out.reshape(rows, -1)[:, :cols]


def same(a, b):
    return np.array_equal(np.asarray(a, np.float64), b, equal_nan=True)


def gpu(torch, x, dtype):
    return torch.as_tensor(x, device="cuda").to(getattr(torch, dtype))


def host(t):
    return t.double().cpu().numpy()


def normals(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (2, 8), (1, 31), (3, 32), (5, 33), (128, 128), (129, 127),
                                       (1, 722), (362, 722), (77, 1031), (300, 2048), (1, 70001)])
def test_values(ops, torch, rows, cols, dtype):
    x = gpu(torch, normals(rows * 1000 + cols, rows, cols) * np.exp(normals(cols, cols)), dtype)
    q = ops.mx4_quantise(x)
    ref = quantised(x.float().cpu().numpy())
    for out in (torch.float32, torch.bfloat16):
        assert same(host(ops.mx4_values(q, out)), ref)


def test_rounding_edges_and_special_blocks(ops, torch):
    edges = np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -5, 7.9, -7.99, 0.2499999, 0.2500001, -0.0])
    rows = []
    for exponent in (-149 + 23, -126, -124, -20, 0, 60, 125):
        rows.append(np.pad(edges * 2.0 ** exponent, (0, 16)))
    with np.errstate(over="ignore"):
        x = np.stack(rows).astype(np.float32)
    x[0, 20:24] = [1e-45, -1e-45, 1e-40, -3e-39]
    special = np.zeros((8, 32), np.float32)
    special[1, 5] = np.inf
    special[2, 31] = -np.inf
    special[3, 0] = np.nan
    special[4, :] = 1e-45
    special[5, :] = np.finfo(np.float32).max
    special[6, 3] = -np.finfo(np.float32).max
    special[7, :] = np.finfo(np.float32).tiny
    x = np.concatenate([x, special])
    x = np.concatenate([x, x[::-1]], 1)          # a bad block next to a good one
    q = ops.mx4_quantise(gpu(torch, x, "float32"))
    assert same(host(ops.mx4_values(q, torch.float32)), quantised(x))
    assert same(host(ops.mx4_values(q, torch.bfloat16)), quantised(x))


def test_layout_is_the_documented_one(ops, torch):
    rows, cols = 150, 300
    x = normals(3, rows, cols)
    q = ops.mx4_quantise(gpu(torch, x, "float32"))
    codes, scales = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    blocks = 10
    assert codes.shape == (rows, 160) and scales.size == 2 * 3 * 512
    nibble = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    at = ((r // 128) * 3 + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    scale = np.ldexp(1.0, scales[at].astype(int) - 127)
    values = np.where(nibble & 8, -1, 1) * TABLE[nibble & 7] * np.repeat(scale, 32, 1)
    assert np.array_equal(values[:, :cols], quantised(x)) and not nibble[:, cols:].any()
    rest = np.ones(scales.size, bool)
    rest[at] = False
    assert not scales[rest].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("offset,stride,cols", [(0, 80, 64), (1, 81, 64), (3, 99, 45), (8, 72, 72), (5, 0, 64)])
def test_strided_sources(ops, torch, dtype, offset, stride, cols):
    base = gpu(torch, normals(9, 40 * 100), dtype)
    x = torch.as_strided(base, (40, cols), (stride, 1), offset)
    q = ops.mx4_quantise(x)
    assert same(host(ops.mx4_values(q, x.dtype)), quantised(x.float().cpu().numpy()))


def test_source_offsets_pass_32_bits(ops, torch):
    ld = (1 << 30) + 11
    base = torch.empty(4 * ld + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(base, (5, 64), (ld, 1), 0)
    x.copy_(gpu(torch, normals(4, 5, 64), "bfloat16"))
    assert same(host(ops.mx4_values(ops.mx4_quantise(x), torch.float32)), quantised(x.float().cpu().numpy()))


def raw(ops, fn, *args):
    e = C.create_string_buffer(1024)
    assert getattr(ops.azb200.lib(), fn)(*args, e, 1024) == 0, e.value


@pytest.mark.parametrize("cols", [(1 << 26) - 5, 1 << 26])
def test_longest_rows(ops, torch, cols):
    """A row of 2^26 columns is the blocks of 2^16 rows of 1024."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1 << 16, 1024, generator=g, device="cuda", dtype=torch.bfloat16)
    x.view(-1)[cols:] = 0
    a, b = ops.mx4_quantise(x.view(1, -1)[:, :cols]), ops.mx4_quantise(x)
    assert torch.equal(a.codes.flatten(), b.codes.flatten())
    assert torch.equal(ops.mx4_values(a, torch.bfloat16)[0], ops.mx4_values(b, torch.bfloat16).flatten()[:cols])


def test_strided_outputs_leave_the_rest_alone(ops, torch):
    x, w = gpu(torch, normals(5, 9, 70), "float32"), gpu(torch, normals(6, 37, 70), "float32")
    qx, qw = ops.mx4_quantise(x), ops.mx4_quantise(w)
    out = torch.full((9, 101), -7.0, device="cuda")
    raw(ops, "azb_mx4_values", 0, *qx.pointers(), 9, 70, out.data_ptr(), 0, 101, None)
    assert same(host(out[:, :70]), quantised(x.cpu().numpy())) and bool((out[:, 70:] == -7).all())
    out.fill_(-7.0)
    raw(ops, "azb_mx4_product", 0, *qx.pointers(), 9, *qw.pointers(), 37, 70, None, 0, out.data_ptr(), 0, 101, None)
    assert torch.equal(out[:, :37], ops.mx4_product(qx, qw)) and bool((out[:, 37:] == -7).all())


# ---------------------------------------------------------------- product

SHAPES = [(1, 1, 1), (1, 128, 256), (1, 362, 722), (1, 1000, 4096), (3, 5, 33), (15, 129, 65), (16, 64, 64),
          (17, 300, 511), (33, 127, 2000), (64, 256, 1025), (65, 31, 300), (100, 640, 96), (128, 128, 128),
          (129, 130, 257), (192, 4000, 64), (300, 362, 722), (1000, 1100, 320), (2100, 2500, 31), (1, 3, 9000),
          (2049, 2311, 513), (1793, 1936, 1000), (9000, 130, 70), (130, 20000, 65)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ops, torch, m, n, k, dtype):
    x, w = gpu(torch, normals(m + k, m, k), dtype), gpu(torch, normals(n + k, n, k), dtype)
    bias = gpu(torch, normals(n, n), "float32")
    qw = ops.mx4_quantise(w)
    a, b = quantised(x.float().cpu().numpy()), quantised(w.float().cpu().numpy())
    ref, size = a @ b.T, np.abs(a) @ np.abs(b).T
    for bb, relu in ((None, False), (bias, True)):
        y = ref if bb is None else ref + host(bb)
        s = size if bb is None else size + np.abs(host(bb))
        out = ops.mx4_product(x, qw, bias=bb, relu=relu, dtype=torch.float32)
        got = host(out)
        tol = (k + 1) * 2.0 ** -23 * s + 2.0 ** -24 * np.abs(y) + 2.0 ** -149
        assert (np.abs(got - (np.maximum(y, 0) if relu else y)) <= tol).all()
        assert torch.equal(ops.mx4_product(x, qw, bias=bb, relu=relu, dtype=torch.bfloat16), out.bfloat16())
    # quantised beforehand or on the way: the same bits
    assert torch.equal(ops.mx4_product(ops.mx4_quantise(x), qw, dtype=x.dtype), ops.mx4_product(x, qw))
    ops.check(0)


@pytest.mark.parametrize("m,n,k", [(1, 130, 1500), (20, 70, 513), (130, 400, 260), (300, 140, 1000)])
def test_product_exact_on_small_integers(ops, torch, m, n, k):
    """Integers whose sums stay below 2^24 leave no room for rounding."""
    r = np.random.default_rng(m)
    values = np.array([-6, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6], np.float32)
    x, w = r.choice(values, (m, k)), r.choice(values, (n, k))
    x[:, ::32], w[:, ::32] = 4, -4   # every block's scale is 1
    got = host(ops.mx4_product(gpu(torch, x, "float32"), ops.mx4_quantise(gpu(torch, w, "float32"))))
    assert np.array_equal(got, x.astype(np.float64) @ w.astype(np.float64).T)


def test_product_scales_reach_every_block(ops, torch):
    """One block at a time differs from zero, at scales far apart."""
    k, n = 32 * 19, 200
    x = np.zeros((19, k), np.float32)
    w = np.zeros((n, k), np.float32)
    for b in range(19):
        x[b, b * 32 + b] = 3.0 * 2.0 ** (b - 9)
        w[:, b * 32 + b] = 1.5 * 2.0 ** ((np.arange(n) + b) % 40 - 20)
    got = host(ops.mx4_product(gpu(torch, x, "float32"), ops.mx4_quantise(gpu(torch, w, "float32"))))
    assert np.array_equal(got, x.astype(np.float64) @ w.astype(np.float64).T)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_nan_stays_in_its_row(ops, torch, m):
    x, w = normals(1, m, 100), normals(2, 150, 100)
    x[m // 2, 3] = np.inf
    w[149, 99] = np.nan
    y = host(ops.mx4_product(gpu(torch, x, "float32"), ops.mx4_quantise(gpu(torch, w, "float32")), relu=True))
    bad = np.isnan(y)
    assert bad[m // 2].all() and bad[:, 149].all()
    bad[m // 2], bad[:, 149] = False, False
    assert not bad.any()


def test_product_is_repeatable_and_takes_vectors(ops, torch):
    x, w = gpu(torch, normals(1, 5, 4000), "bfloat16"), ops.mx4_quantise(gpu(torch, normals(2, 300, 4000), "bfloat16"))
    y = ops.mx4_product(x, w)
    for _ in range(5):
        assert torch.equal(ops.mx4_product(x, w), y)
    v = ops.mx4_product(x[0], w, dtype=torch.float32)
    assert v.shape == (300,) and v.dtype == torch.float32
    assert torch.equal(v, ops.mx4_product(x[:1], w, dtype=torch.float32)[0])


def test_mx4_from_its_parts(ops, torch):
    q = ops.mx4_quantise(gpu(torch, normals(3, 45, 100), "float32"))
    again = ops.Mx4(q.codes.clone(), q.scales.clone(), 45, 100)
    assert torch.equal(ops.mx4_values(again), ops.mx4_values(q)) and again.nbytes() == q.nbytes()


def test_empty_sides(ops, torch):
    w = ops.mx4_quantise(gpu(torch, normals(2, 30, 40), "float32"))
    assert ops.mx4_product(torch.empty(0, 40, device="cuda"), w).shape == (0, 30)
    none = ops.mx4_quantise(torch.empty(0, 40, device="cuda"))
    assert ops.mx4_product(torch.ones(3, 40, device="cuda"), none).shape == (3, 0)
    assert ops.mx4_values(none).shape == (0, 40)


def test_other_stream_and_graph(ops, torch):
    x, w = gpu(torch, normals(1, 70, 500), "float32"), ops.mx4_quantise(gpu(torch, normals(2, 90, 500), "float32"))
    ref = ops.mx4_product(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.mx4_product(x, w) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref) for y in again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.mx4_product(x, w)
        v = ops.mx4_values(ops.mx4_quantise(y))
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, 2 * ref) and same(host(v), quantised(y.cpu().numpy()))


def test_refusals(ops, torch):
    x = torch.ones(4, 64, device="cuda")
    w = ops.mx4_quantise(x)
    for call, text in [
        (lambda: ops.mx4_quantise(x.half()), "float32 or bfloat16"),
        (lambda: ops.mx4_quantise(x.t()), "columns must be adjacent"),
        (lambda: ops.mx4_quantise(x[0]), "a matrix is needed"),
        (lambda: ops.mx4_quantise(x[:, :0]), "at least one column"),
        (lambda: ops.mx4_quantise(x.clone().requires_grad_()), "no backward pass"),
        (lambda: ops.mx4_product(x, w, bias=x[0, :4].clone().requires_grad_()), "bias requires a gradient"),
        (lambda: ops.mx4_values(w, torch.float16), "float32 or bfloat16"),
        (lambda: ops.mx4_product(x[:, :32], w), "x has 32 columns, w 64"),
        (lambda: ops.mx4_product(x, x), "an Mx4 is needed"),
        (lambda: ops.mx4_product(x, w, bias=torch.ones(3, device="cuda")), "bias: 4 adjacent"),
        (lambda: ops.mx4_product(x, w, bias=torch.ones(4)), "bias on cpu"),
        (lambda: ops.mx4_product(x.cpu(), w), "CUDA tensor"),
        (lambda: ops.mx4_product(w, ops.mx4_quantise(x[:, :32])), "x has 64 columns, w 32"),
        (lambda: ops.Mx4(w.codes, w.scales[:-1], 4, 64), "bytes of codes and scales"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    ops.check(0)


def test_products_that_fill_the_accumulators_follow_at_once(ops, torch):
    """A small product of plain x lets the next launch in early; the next here
    takes the whole of the tensor core's memory on every SM."""
    m, n, k = 40000, 100, 256
    x, w = ops.mx4_quantise(gpu(torch, normals(1, m, k), "bfloat16")), ops.mx4_quantise(gpu(torch, normals(2, n, k), "bfloat16"))
    one, v = gpu(torch, normals(3, 1, k), "float32"), ops.mx4_quantise(gpu(torch, normals(4, 3000, k), "float32"))
    ref, small = ops.mx4_product(x, w), ops.mx4_product(one, v)
    torch.cuda.synchronize()
    got = [(ops.mx4_product(one, v), ops.mx4_product(x, w)) for _ in range(50)]
    assert all(torch.equal(a, small) and torch.equal(b, ref) for a, b in got)
    ops.check(0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,ld", [(15400, 257, 257), (15400, 257, 301), (257, 15401, 15401), (15401, 264, 264), (15401, 264, 304),
                                    (300, 15400, 15416)])
def test_large_products_with_tails_and_strides(ops, torch, m, n, ld, dtype):
    """Several tiles of 256 x 256 a pair of CTAs, the last ones with a few rows
    or columns, output rows at multiples of 16 bytes and elsewhere, and rows
    and columns that are NaN. Integers leave no room for rounding."""
    r = np.random.default_rng(m + n)
    values = np.array([-6, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6], np.float32)
    k = 70
    x, w, bias = r.choice(values, (m, k)), r.choice(values, (n, k)), r.integers(-9, 10, n).astype(np.float32)
    x[:, ::32], w[:, ::32] = 4, -4   # every block's scale is 1
    ref = x.astype(np.float64) @ w.astype(np.float64).T + bias
    bad_rows, bad_cols = [0, 255, 256, m - 1], [3, n - 1]
    x[bad_rows, [1, 33, 66, 69]] = [np.inf, np.nan, -np.inf, np.nan]
    w[bad_cols, [5, 68]] = [np.nan, np.inf]
    ref[bad_rows], ref[:, bad_cols] = np.nan, np.nan
    qx, qw = ops.mx4_quantise(gpu(torch, x, "float32")), ops.mx4_quantise(gpu(torch, w, "float32"))
    b = gpu(torch, bias, "float32")
    for relu in (0, 1):
        out = gpu(torch, np.full((m, ld), -7.0), dtype)
        raw(ops, "azb_mx4_product", 0, *qx.pointers(), m, *qw.pointers(), n, k, b.data_ptr(), relu, out.data_ptr(),
            int(dtype == "bfloat16"), ld, None)
        want = torch.as_tensor(np.maximum(ref, 0) if relu else ref, device="cuda").to(out.dtype)
        assert torch.equal(out[:, :n].isnan(), want.isnan()) and torch.equal(out[:, :n].nan_to_num(0.5), want.nan_to_num(0.5))
        assert bool((out[:, n:] == -7).all())
    ops.check(0)


def test_rounding_edges_and_special_blocks_of_bfloat16(ops, torch):
    """As of float32, whose sources have code of their own: ties, the numbers
    next to them, subnormals, the largest number, infinities and NaN."""
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    edges = np.concatenate([[6.0, -0.0, 7.96875, -7.96875], ties, -ties, ties * (1 - 2.0 ** -8), ties * (1 + 2.0 ** -7)])
    rows = [np.pad(edges * 2.0 ** e, (0, 32 - edges.size)) for e in (-130, -126, -124, -60, 0, 60, 124)]
    special = np.zeros((9, 32))
    special[1, 5] = np.inf
    special[2, 31] = -np.inf
    special[3, 0] = np.nan
    special[4, :] = 2.0 ** -133                      # the least subnormal
    special[5, :] = float(torch.finfo(torch.bfloat16).max)
    special[6, 3] = -float(torch.finfo(torch.bfloat16).max)
    special[7, :] = 2.0 ** -126
    special[8, :] = np.where(np.arange(32) % 2, 2.0 ** -133 * 100, -(2.0 ** -126))
    x = np.concatenate([np.stack(rows), special])
    x = np.concatenate([x, x[::-1]], 1)              # a bad block next to a good one
    x = torch.as_tensor(x, device="cuda").to(torch.bfloat16)
    w = np.eye(64, dtype=np.float32)
    for cols, pad in ((64, 0), (64, 1), (64, 4), (61, 3)):
        v = torch.nn.functional.pad(x, (pad, 9))[:, pad:pad + cols]
        ref = quantised(v.float().cpu().numpy())
        q = ops.mx4_quantise(v)
        assert same(host(ops.mx4_values(q, torch.float32)), ref) and same(host(ops.mx4_values(q, torch.bfloat16)), ref)
        for m in (1, 16):                            # quantised by the product's own CTAs: a row of the identity each
            y = host(ops.mx4_product(v[:m], ops.mx4_quantise(gpu(torch, w[:, :cols], "float32")), dtype=torch.float32))
            bad = np.isnan(ref[:m]).any(1)
            assert np.isnan(y[bad]).all() and np.array_equal(y[~bad][:, :cols], ref[:m][~bad])


def test_two_streams_at_once(ops, torch):
    """Products of every kind on two streams, with nothing between them."""
    shapes = [(1, 4096, 4096), (16, 1000, 2000), (40, 3000, 700), (333, 1111, 2501), (3000, 2000, 300), (3001, 2001, 300)]
    x = [gpu(torch, normals(m, m, k), "bfloat16") for m, n, k in shapes]
    w = [ops.mx4_quantise(gpu(torch, normals(n, n, k), "bfloat16")) for m, n, k in shapes]
    ref = [ops.mx4_product(a, b) for a, b in zip(x, w)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    order = np.random.default_rng(5)
    for _ in range(300):
        i, s = int(order.integers(len(shapes))), streams[int(order.integers(2))]
        with torch.cuda.stream(s):
            got.append((i, ops.mx4_product(x[i], w[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref[i]) for i, y in got)
    ops.check(0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [4097, 4098, 4099, 4100, 4103, 4104])
def test_large_products_write_no_further_than_their_rows(ops, torch, n, dtype):
    """Output rows that start at multiples of 16 bytes and end elsewhere."""
    m, k, ld = 800, 64, 4112
    x, w = ops.mx4_quantise(gpu(torch, normals(1, m, k), "float32")), ops.mx4_quantise(gpu(torch, normals(2, n, k), "float32"))
    out = gpu(torch, np.full((m, ld), -7.0), dtype)
    raw(ops, "azb_mx4_product", 0, *x.pointers(), m, *w.pointers(), n, k, None, 0, out.data_ptr(), int(dtype == "bfloat16"), ld, None)
    assert torch.equal(out[:, :n], ops.mx4_product(x, w, dtype=out.dtype)) and bool((out[:, n:] == -7).all())
