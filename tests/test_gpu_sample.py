"""The move sampler on the GPU against its definition in 64 bits (numpy).

Moves are whole numbers and compared for equality, except where the 64-bit
result itself hangs on less than fp32 can resolve: the race's two best keys
closer than 1e-4, or a top-p or min-p cut within 1e-5 of a column's share.
Such rows may give any of the columns in question, and must be rare. logprob:
|x| carries three roundings of 2^-24 and the sum at most cols / 1024 + 16 of
them per thread and tree, so 3e-7 |x| + 1e-5 for up to 2^17 columns.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOW, HIGH = 2.0 ** -25, 1 - 2.0 ** -24


@pytest.fixture(scope="module")
def ops(engine):
    import azb_ops

    return azb_ops


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def reference(logits, noise, legal, t, k, p, mp):
    """(moves a row may give, logprob of each column) by the definition; the
    first move is the 64-bit one."""
    l = logits.astype(np.float64)
    ok = ~np.isnan(l) & (l > -np.inf)
    if legal is not None:
        ok &= legal != 0
    ids = np.flatnonzero(ok)
    if ids.size == 0:
        return [-1], None
    ids = ids[np.argsort(-l[ids], kind="stable")]
    ls = l[ids]
    if not t > 0:
        return [int(ids[0])], np.zeros(l.size)
    t = np.float64(np.float32(t))
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(ls == ls[0], 0.0, (ls - ls[0]) / t)
    w = np.exp(x)
    logprob = np.full(l.size, -np.inf)
    logprob[ids] = x - np.log(w.sum())
    n = min(k, ids.size) if k > 0 else ids.size
    sets = []
    for slack in (0.0, -1e-5, 1e-5):
        keep = np.ones(n, bool)
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]]) / w[:n].sum()
            keep &= before < np.float64(np.float32(p)) + slack
        if mp > 0:
            keep &= w[:n] >= np.float64(np.float32(mp)) - slack
        keep[0] = True
        u = np.clip(np.nan_to_num(noise[ids[:n]].astype(np.float64), nan=0.0), LOW, HIGH)
        key = np.where(keep, x[:n] - np.log(-np.log(u)), -np.inf)
        sets.append((ids[:n], key))
    idn, key = sets[0]
    first = int(idn[key == key.max()].min())
    near = {int(i) for i_, kk in sets for i in i_[kk >= kk.max() - 1e-4]}
    exact_ties = {int(i) for i in idn[key == key.max()]}
    return [first] + sorted(near - exact_ties), logprob


def run(ops, torch, logits, noise, legal=None, dtype="float32", **kw):
    to = lambda a, d: None if a is None else torch.as_tensor(a, device="cuda").to(d)
    for name, d in (("temperature", torch.float32), ("top_p", torch.float32), ("min_p", torch.float32), ("top_k", torch.int32)):
        if isinstance(kw.get(name), np.ndarray):
            kw[name] = to(kw[name], d)
    m, lp = ops.sample_moves(to(logits, getattr(torch, dtype)), to(noise, torch.float32),
                             legal=to(legal, torch.bool), **kw)
    return m.cpu().numpy(), lp.double().cpu().numpy()


def check(ops, torch, logits, noise, legal=None, dtype="float32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    if dtype == "bfloat16":
        logits = torch.as_tensor(logits).to(torch.bfloat16).float().numpy()
    m, lp = run(ops, torch, logits, noise, legal, dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    unsure = 0
    for r in range(logits.shape[0]):
        at = lambda v: v[r] if isinstance(v, np.ndarray) else v
        moves, ref = reference(logits[r], noise[r], None if legal is None else legal[r], at(temperature), at(top_k),
                               at(top_p), at(min_p))
        unsure += len(moves) > 1
        assert m[r] in (moves if len(moves) > 1 else moves[:1]), (r, m[r], moves)
        if m[r] < 0:
            assert lp[r] == -np.inf
            continue
        want = ref[m[r]]
        assert abs(lp[r] - want) <= 1e-5 + 3e-7 * abs(want) if np.isfinite(want) else lp[r] == want, (r, lp[r], want)
    assert unsure <= max(1, logits.shape[0] // 50)
    return m, lp


def data(seed, rows, cols, spread=3.0):
    r = np.random.default_rng(seed)
    return (r.standard_normal((rows, cols)) * spread).astype(np.float32), r.random((rows, cols), np.float32), r


COLS = [1, 2, 26, 31, 32, 33, 82, 128, 129, 362, 384, 385, 1000, 1024, 1025, 4097, 9001, 50001]
FILTERS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
           dict(top_k=50, top_p=0.95, min_p=0.01, temperature=0.7), dict(top_p=0.3, temperature=1.7)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("filters", FILTERS, ids=str)
@pytest.mark.parametrize("cols", COLS)
def test_sizes_and_filters(ops, torch, cols, filters, dtype):
    logits, noise, r = data(cols, 9, cols)
    legal = r.random((9, cols)) < 0.6
    check(ops, torch, logits, noise, None, dtype, **filters)
    check(ops, torch, logits, noise, legal, dtype, **filters)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [70001, 131072, 450001])
def test_wide_rows(ops, torch, cols, dtype):
    """Rows beyond what shared memory holds."""
    logits, noise, r = data(cols, 3, cols)
    legal = r.random((3, cols)) < 0.6
    logits[1, ::7] = np.nan
    logits[2, 5::3] = -np.inf
    for f in FILTERS:
        check(ops, torch, logits, noise, None, dtype, **f)
    check(ops, torch, logits, noise, legal, dtype, top_k=50, top_p=0.9)
    check(ops, torch, logits, noise, legal, dtype, min_p=0.1)
    check(ops, torch, logits, noise, legal, dtype, temperature=0.0)
    check(ops, torch, logits, noise, legal, dtype, top_k=3000, top_p=0.999)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [16385, 32768, 50001, 65536])
def test_many_wide_rows(ops, torch, cols, dtype):
    """More rows than run at once: fewer CTAs a row."""
    logits, noise, r = data(cols, 110, cols)
    legal = r.random((110, cols)) < 0.6
    legal[3], legal[7, 1:] = False, False
    check(ops, torch, logits, noise, legal, dtype)
    check(ops, torch, logits, noise, None, dtype, top_p=0.9)
    check(ops, torch, logits, noise, legal, dtype, top_k=16, top_p=0.95, min_p=0.01, temperature=0.7)
    check(ops, torch, logits, noise, None, dtype, top_k=40)


@pytest.mark.parametrize("cols", [600001, 900001])
def test_widest_rows_bfloat16(ops, torch, cols):
    """Slices beyond 16-bit places, and beyond shared memory, in the shorter type."""
    logits, noise, r = data(cols, 2, cols)
    for f in FILTERS:
        check(ops, torch, logits, noise, None, "bfloat16", **f)


def test_top_k_beyond_32_bits_is_off(ops, torch):
    logits, noise, r = data(4, 6, 300)
    for k in (300, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        m, lp = run(ops, torch, logits, noise, top_k=k)
        assert (m == run(ops, torch, logits, noise)[0]).all()


@pytest.mark.parametrize("cols", [20000, 100001])
def test_wide_rows_with_ties_and_infinities(ops, torch, cols):
    logits, noise, r = data(8, 4, cols, 1.0)
    for f in FILTERS:
        check(ops, torch, np.round(logits), noise, **f)
    check(ops, torch, np.zeros_like(logits), noise, top_k=777)
    check(ops, torch, np.zeros_like(logits), noise, top_p=0.25)
    logits[0, [5, 77, cols - 1]] = np.inf
    logits[1, cols - 1] = np.inf
    logits[2] = -np.inf
    logits[3] = np.nan
    logits[3, cols // 2] = -3e38
    for f in FILTERS:
        m, lp = check(ops, torch, logits, noise, **f)
        assert m[1] == cols - 1 and m[2] == -1 and m[3] == cols // 2 and lp[3] == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_wide_rows_with_strides(ops, torch, dtype):
    """Rows of odd length and offset, of logits, legality and noise alike."""
    cols = 70003
    logits, noise, r = data(12, 5, cols + 9)
    legal = r.random((5, cols + 9)) < 0.5
    if dtype == "bfloat16":
        logits = torch.as_tensor(logits).to(torch.bfloat16).float().numpy()
    L, N = torch.as_tensor(logits, device="cuda").to(getattr(torch, dtype)), torch.as_tensor(noise, device="cuda")
    A = torch.as_tensor(legal, device="cuda")
    for off in (0, 1, 3, 8):
        cut = slice(off, off + cols)
        m, lp = ops.sample_moves(L[:, cut], N[:, cut], legal=A[:, cut], top_p=0.9)
        for row in range(5):
            moves, ref = reference(logits[row, cut], noise[row, cut], legal[row, cut], 1.0, 0, 0.9, 0.0)
            assert int(m[row]) in moves
            assert abs(float(lp[row]) - ref[int(m[row])]) <= 1e-5 + 3e-7 * abs(ref[int(m[row])])


@pytest.mark.parametrize("cols", [362, 3000])
def test_many_ties(ops, torch, cols):
    """Logits on a coarse grid: every cut falls inside a group of equal ones."""
    logits, noise, r = data(5, 64, cols, 1.0)
    logits = np.round(logits)
    for f in FILTERS:
        check(ops, torch, logits, noise, **f)
    check(ops, torch, np.zeros_like(logits), noise, top_k=7)
    check(ops, torch, np.zeros_like(logits), noise, top_p=0.25)


@pytest.mark.parametrize("cols", [100, 1000, 2000])
def test_tied_cut_keeps_the_lowest_columns(ops, torch, cols):
    logits = np.zeros((3, cols), np.float32)
    logits[:, 50] = 1.0
    noise = np.tile(np.linspace(0.01, 0.99, cols, dtype=np.float32), (3, 1))   # the last kept column wins
    noise[:, 50] = 1e-6
    for k in (2, 30, 52, 90):
        m, _ = run(ops, torch, logits, noise, top_k=k)
        assert (m == (k - 2 if k <= 51 else k - 1)).all(), (k, m)


@pytest.mark.parametrize("cols", [82, 362, 1024, 5000])
def test_per_row_settings(ops, torch, cols):
    rows = 40
    logits, noise, r = data(11, rows, cols)
    t = r.choice([0.0, 0.3, 1.0, 2.0, -1.0, np.nan], rows).astype(np.float32)
    k = r.choice([0, -3, 1, 5, cols, cols + 5], rows).astype(np.int32)
    p = r.choice([1.0, 0.5, 0.9, 0.0, np.nan, 1.5], rows).astype(np.float32)
    mp = r.choice([0.0, 0.1, -1.0, np.nan, 1.0], rows).astype(np.float32)
    legal = r.random((rows, cols)) < 0.5
    off = lambda v, o: np.where(np.isnan(v), o, v)
    m, lp = run(ops, torch, logits, noise, legal, temperature=t, top_k=k, top_p=p, min_p=mp)
    for i in range(rows):
        pi, ki = off(p, 1.0)[i], int(k[i])
        if pi <= 0:
            pi, ki = 1.0, 1
        moves, _ = reference(logits[i], noise[i], legal[i], off(t, 0.0)[i], ki, pi, off(mp, 0.0)[i])
        assert m[i] in moves, i


@pytest.mark.parametrize("cols", [7, 362, 4000])
def test_rows_with_nothing_and_with_one(ops, torch, cols):
    logits, noise, _ = data(2, 6, cols)
    legal = np.ones((6, cols), bool)
    legal[0] = False
    logits[1] = -np.inf
    logits[2] = np.nan
    legal[3] = False
    legal[3, cols - 1] = True
    logits[4, :-1] = -np.inf
    for f in (dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.2), dict(temperature=0.0)):
        m, lp = check(ops, torch, logits, noise, legal, **f)
        assert (m[:3] == -1).all() and (lp[:3] == -np.inf).all() and m[3] == m[4] == cols - 1
        assert lp[3] == lp[4] == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [40, 362, 3000])
def test_extreme_logits(ops, torch, cols, dtype):
    logits, noise, r = data(3, 8, cols)
    low = float(torch.finfo(getattr(torch, dtype)).min)
    logits[0, r.random(cols) < 0.7] = low             # masked by the lowest number
    logits[1] = low                                   # all of them: a uniform row
    logits[2, [3, 17]] = np.inf                       # the infinite ones share everything
    logits[3, 5] = np.nan
    logits[4, 2] = -low                               # the largest number
    logits[5] = np.where(r.random(cols) < 0.5, -np.inf, logits[5])
    logits[6] = 0.0
    logits[6, ::2] = -0.0                             # both zeros are one logit
    logits[7] *= 1e30
    for f in (dict(), dict(top_k=4), dict(top_p=0.7), dict(min_p=0.1), dict(temperature=0.01), dict(temperature=0.0)):
        m, _ = check(ops, torch, logits, noise, None, dtype, **f)
        assert m[2] in (3, 17) and m[4] == 2 and m[3] != 5


@pytest.mark.parametrize("cols", [362, 2000])
def test_noise_at_its_ends(ops, torch, cols):
    logits, noise, _ = data(8, 4, cols)
    noise[0] = 0.0
    noise[1] = 1.0
    noise[2] = np.nan
    noise[3, :] = 0.5
    m, _ = check(ops, torch, logits, noise)
    assert (m == logits.argmax(1)).all()              # equal noise everywhere: the largest logit


@pytest.mark.parametrize("cols", [362, 1024, 6000])
def test_greedy_takes_the_first_largest(ops, torch, cols):
    logits, _, _ = data(4, 50, cols)
    logits = np.round(logits)
    t = torch.as_tensor(logits, device="cuda")
    m, lp = ops.sample_moves(t, None, temperature=0.0)
    assert np.array_equal(m.cpu().numpy(), logits.argmax(1)) and bool((lp == 0).all())


@pytest.mark.parametrize("cols", [82, 362, 700, 3001, 20000])
def test_rows_do_not_depend_on_the_batch(ops, torch, cols):
    logits, noise, _ = data(6, 37, cols)
    f = dict(temperature=0.9, top_k=30, top_p=0.9)
    m, lp = run(ops, torch, logits, noise, **f)
    for r in (0, 1, 20, 36):
        m1, lp1 = run(ops, torch, logits[r:r + 1], noise[r:r + 1], **f)
        assert m1[0] == m[r] and lp1[0] == lp[r]
    again, lp2 = run(ops, torch, logits, noise, **f)
    assert np.array_equal(again, m) and np.array_equal(lp2, lp)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [45, 362, 1500, 9999])
def test_strides_and_offsets(ops, torch, cols, dtype):
    logits, noise, r = data(7, 5, cols)
    legal = r.random((5, cols)) < 0.7
    ref, _ = run(ops, torch, logits, noise, legal, dtype, top_k=20, top_p=0.9)
    d = getattr(torch, dtype)
    for pad in (1, 3, 8):
        wide = lambda a, t: torch.zeros(5, cols + 2 * pad, dtype=t, device="cuda").copy_(
            torch.nn.functional.pad(torch.as_tensor(a, device="cuda").to(t), (pad, pad)))[:, pad:pad + cols]
        m, _ = ops.sample_moves(wide(logits, d), wide(noise, torch.float32), legal=wide(legal, torch.uint8).mul(3),
                                top_k=20, top_p=0.9)
        assert np.array_equal(m.cpu().numpy(), ref)
    one = torch.as_tensor(logits[:1], device="cuda").to(d).expand(5, cols)      # a broadcast row
    m, _ = ops.sample_moves(one, torch.as_tensor(noise, device="cuda"))
    m2, _ = ops.sample_moves(one.contiguous(), torch.as_tensor(noise, device="cuda"))
    assert torch.equal(m, m2)


def test_offsets_pass_32_bits(ops, torch):
    ld, cols = (1 << 30) + 5, 1200
    base = torch.empty(4 * ld + cols, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(base, (5, cols), (ld, 1), 0)
    logits, noise, _ = data(1, 5, cols)
    view.copy_(torch.as_tensor(logits, device="cuda"))
    n = torch.as_tensor(noise, device="cuda")
    assert torch.equal(ops.sample_moves(view, n, top_p=0.9)[0], ops.sample_moves(view.contiguous(), n, top_p=0.9)[0])


@pytest.mark.parametrize("cols", [5, 1500])
def test_frequencies(ops, torch, cols):
    """Drawn frequencies of a kept set: within 6 standard deviations."""
    rows = 40000
    g = torch.Generator(device="cuda").manual_seed(1)
    row = torch.full((cols,), -9.0, device="cuda")
    row[:5] = torch.tensor([1.0, 0.5, 0.0, -0.5, -1.0], device="cuda")
    m, _ = ops.sample_moves(row.expand(rows, cols), torch.rand(rows, cols, generator=g, device="cuda"), temperature=0.8,
                            top_k=4)
    p = np.exp(np.array([1.0, 0.5, 0.0, -0.5]) / np.float32(0.8))
    p /= p.sum()
    got = np.bincount(m.cpu().numpy(), minlength=5)
    assert got[4:].sum() == 0
    assert (np.abs(got[:4] - rows * p) <= 6 * np.sqrt(rows * p * (1 - p))).all(), got


def test_other_stream_and_graph(ops, torch):
    logits, noise, _ = data(7, 300, 362)
    l, n = torch.as_tensor(logits, device="cuda"), torch.as_tensor(noise, device="cuda")
    ref = ops.sample_moves(l, n, top_k=9)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.sample_moves(l, n, top_k=9)[0]
    torch.cuda.synchronize()
    assert torch.equal(again, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, _ = ops.sample_moves(l, n, top_k=9)
    l.copy_(l.flip(0))
    n.copy_(n.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(m, ref.flip(0))


def test_refusals_and_empty(ops, torch):
    l, n = torch.zeros(3, 40, device="cuda"), torch.rand(3, 40, device="cuda")
    for call, text in [
        (lambda: ops.sample_moves(l.half(), n), "float32 or bfloat16"),
        (lambda: ops.sample_moves(l, n, temperature=torch.ones(3, device="cuda").requires_grad_()), "no backward pass"),
        (lambda: ops.sample_moves(l.t(), n.t()), "columns must be adjacent"),
        (lambda: ops.sample_moves(l, n.double()), "noise: float32"),
        (lambda: ops.sample_moves(l, n[:, :39]), "noise: float32"),
        (lambda: ops.sample_moves(l, None), "null noise"),
        (lambda: ops.sample_moves(l, n.cpu()), "it is on cpu"),
        (lambda: ops.sample_moves(l, n, legal=torch.ones(3, 40, device="cuda")), "legal: bool or uint8"),
        (lambda: ops.sample_moves(l, n, temperature=-1.0), "temperature"),
        (lambda: ops.sample_moves(l, n, top_p=1.2), "top_p"),
        (lambda: ops.sample_moves(l, n, top_k=torch.ones(3, device="cuda")), "top_k: a number, or 3"),
        (lambda: ops.sample_moves(l, n, min_p=torch.ones(2, device="cuda")), "min_p: a number, or 3"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    m, lp = ops.sample_moves(l[:0], n[:0])
    assert m.shape == lp.shape == (0,)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [362, 1024, 5000, 16384, 50001, 450001])
def test_noise_out_of_range_is_clamped(ops, torch, cols, dtype):
    """Numbers outside (0, 1) are read as its ends, wherever they stand and
    whatever stands beside them."""
    logits, noise, r = data(cols + 1, 6, cols)
    kind = r.random((6, cols))
    for i, odd in enumerate((np.nan, -0.5, -20.0, -1e9, -np.inf)):
        noise[(kind >= 0.15 * i) & (kind < 0.15 * i + 0.15)] = odd
    at = r.integers(0, cols, 6)
    noise[np.arange(6), at] = [1.0, 2.0, 1e9, np.inf, 0.0, 1.0]
    logits[0], noise[0] = 0.0, -100.0                 # the same number everywhere: the largest logit
    logits[0, cols - 3] = 1.0
    logits[1, :] = -9.0                               # the largest logit's is the lowest, another's ordinary
    noise[1, :] = np.nan
    logits[1, [2, cols - 5]] = [0.0, -2.0]
    noise[1, cols - 5] = 0.5
    for f in (dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=50, top_p=0.95, temperature=0.7)):
        m, _ = check(ops, torch, logits, noise, None, dtype, **f)
        assert m[0] == cols - 3
        if f.get("top_p", 1.0) == 1.0:
            assert m[1] == cols - 5


@pytest.mark.parametrize("cols", [1, 5, 362, 1024, 1025, 5000, 50001])
def test_per_row_top_p_below_zero_keeps_the_first(ops, torch, cols):
    logits, noise, _ = data(cols, 10, cols)
    legal = np.ones((10, cols), bool)
    legal[:5] = False
    legal[np.arange(5), [0, cols - 1, cols // 2, 0, cols - 1]] = True
    p = np.tile(np.array([-0.5, -5.0, -1e30, -np.inf, 0.0], np.float32), 2)
    for k in (0, 1, 7):
        m, lp = run(ops, torch, logits, noise, legal, top_p=p, top_k=k)
        assert np.array_equal(m, np.where(legal, logits, -np.inf).argmax(1)), (k, m)
        assert (lp[:5] == 0).all()


@pytest.mark.parametrize("cols", [40, 362, 3000, 20000])
def test_extreme_temperatures(ops, torch, cols):
    """Temperatures near the type's ends, with logits as far apart."""
    r = np.random.default_rng(cols)
    noise = r.random((6, cols), np.float32)
    unit = r.standard_normal((6, cols)).astype(np.float32)
    unit = np.clip(unit, -3, 3) / 3
    for t, scale in ((3.4e38, 1.6e38), (2e38, 1.6e38), (1.5e38, 1e38), (1e37, 1e37), (1e-30, 1e-30), (2e-37, 1e-36)):
        for f in (dict(), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.5)):
            check(ops, torch, unit * np.float32(scale), noise, temperature=t, **f)
    inf = np.array([np.inf, 1.0, np.inf, 1.0, np.inf, np.inf], np.float32)   # per row: every logit the same
    logits = np.where(r.random((6, cols)) < 0.5, np.float32(-np.inf), unit)
    m, lp = run(ops, torch, logits, noise, temperature=inf)
    for i in np.flatnonzero(np.isinf(inf)):
        n = np.isfinite(logits[i]).sum()
        assert np.isfinite(logits[i, m[i]]) and abs(lp[i] + np.log(n)) <= 1e-5
        assert m[i] == np.where(np.isfinite(logits[i]), noise[i], -1).argmax()


def test_two_streams_at_once(ops, torch):
    """Rows of every kernel on two streams, with nothing between them."""
    cases = []
    for rows, cols in ((300, 362), (40, 5000), (64, 16384), (9, 50001), (200, 50001), (2, 131072)):
        logits, noise, _ = data(cols, rows, cols)
        cases.append((torch.as_tensor(logits, device="cuda"), torch.as_tensor(noise, device="cuda"),
                      dict(top_k=50, top_p=0.9) if rows % 2 else dict(top_p=0.8)))
    ref = [ops.sample_moves(l, n, **f) for l, n, f in cases]
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    order = np.random.default_rng(6)
    for _ in range(300):
        i, s = int(order.integers(len(cases))), streams[int(order.integers(2))]
        with torch.cuda.stream(s):
            got.append((i, ops.sample_moves(cases[i][0], cases[i][1], **cases[i][2])))
    torch.cuda.synchronize()
    assert all(torch.equal(m, ref[i][0]) and torch.equal(lp, ref[i][1]) for i, (m, lp) in got)
