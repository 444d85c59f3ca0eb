"""The token-sequence operators against plain implementations in 64 bits.

Tolerances, with u(t) half the spacing of type t at 1 (2^-8 bf16, 2^-11 fp16, 2^-24 fp32)
and s(t) half its smallest subnormal:

* a looked-up value is one product in 32 bits and one rounding: u(fp32) |w| + u(out) |w|
  (1 + u(fp32)) + s(out), w the product with the scale as rounded to 32 bits;
* a gradient is a sum of m terms in 32 bits in some order, one product and one rounding: at
  most (m - 1) u(fp32) / (1 - m u(fp32)) sum |x| for the sum, then as above, and one more
  u(fp32) of the result where it is added to a row.

Index operators are compared exactly."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _gen(*seed):
    return np.random.default_rng(list(seed))


def _values(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)


def _close(got, want, tol):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


# ------------------------------------------------------------------------- lookup

def _check_lookup(eb, table, tokens, *, scale=1.0, first=0, out=None, dtype=None):
    got = eb.embedding(table, tokens, scale=scale, first=first, out=out, dtype=dtype)
    if out is not None:
        assert got is out
    assert got.dtype == (dtype or (out.dtype if out is not None else table.dtype))
    ids = tokens.cpu().long() - first
    known = (ids >= 0) & (ids < table.shape[0]) & (tokens.cpu() >= first)
    padded = torch.cat((table.cpu().double(), torch.zeros(1, table.shape[1], dtype=torch.float64)))
    want = padded[torch.where(known, ids, table.shape[0])] * float(np.float32(scale))
    u32 = half_step(torch.float32)
    _close(got, want, want.abs() * (u32 + half_step(got.dtype) * (1 + u32)) + least(got.dtype))
    return got


@pytest.mark.parametrize("dim", (1, 2, 8, 33, 64, 255, 256, 257, 777, 1024, 4100, 20003))
@pytest.mark.parametrize("n", (1, 31, 1000))
def test_lookup_sizes(eb, n, dim):
    rng = _gen(1, n, dim)
    table = _values(rng, (513, dim), torch.bfloat16).cuda()
    ids = torch.from_numpy(rng.integers(-2, 516, n)).cuda()
    _check_lookup(eb, table, ids, scale=dim ** 0.5)


@pytest.mark.parametrize("source", FLOATS)
@pytest.mark.parametrize("target", FLOATS)
@pytest.mark.parametrize("ids_type", (torch.int32, torch.int64))
def test_lookup_types(eb, source, target, ids_type):
    rng = _gen(2)
    table = _values(rng, (300, 264), source)
    table[7, :5] = torch.tensor([0.0, -0.0, 1e-7, 3e4, 6e-8]).to(source)  # subnormal halves among them
    ids = torch.from_numpy(rng.integers(0, 300, (3, 50))).to(ids_type)
    ids[1, 3] = 7
    _check_lookup(eb, table.cuda(), ids.cuda(), scale=0.37, dtype=target)


def test_lookup_is_exact_without_a_scale(eb):
    for dtype in FLOATS:
        table = _values(_gen(3), (100, 40), dtype).cuda()
        table[3, 0], table[3, 1], table[3, 2] = float("inf"), float("-inf"), float("nan")
        ids = torch.arange(99, -1, -1).cuda()
        got = eb.embedding(table, ids)
        assert torch.equal(got.nan_to_num(5.0), table[ids].nan_to_num(5.0)) and got[96, 2].isnan()


def test_lookup_strides(eb):
    rng = _gen(4)
    wide = _values(rng, (200, 96), torch.float16).cuda()
    ids = torch.from_numpy(rng.integers(-1, 200, (12, 34))).cuda()
    for table in (wide[:, 8:72], wide[:, 3:70], wide[::2], wide[50:51], wide[:, 5:6]):
        for tokens in (ids, ids.t(), ids[:, ::3], ids[3], ids[0, 0], ids[:0], ids.view(3, 4, 34),
                       ids[0].expand(5, 34), ids[:, :1].expand(12, 7)):
            _check_lookup(eb, table, tokens.remainder(table.shape[0] + 1) - 1 if tokens.numel() else tokens)
            _check_lookup(eb, table, tokens)
    # an output inside a larger one, both token axes strided
    room = torch.full((12, 40, 80), 7.0, dtype=torch.float16, device="cuda")
    out = room[:, 2:36, 8:72]
    _check_lookup(eb, wide[:, 8:72], ids, out=out)
    room[:, 2:36, 8:72] = 7.0
    assert bool((room == 7.0).all())
    # wider outputs at every 4 bytes of a 32-byte word
    for shift in range(8):
        room = torch.full((12, 34, 272), 7.0, device="cuda")
        _check_lookup(eb, _values(_gen(4, shift), (200, 264), torch.float16).cuda(), ids,
                      out=room[..., shift:shift + 264])
        assert bool((room[..., :shift] == 7.0).all()) and bool((room[..., shift + 264:] == 7.0).all())
    # the token axes the other way round
    swapped = torch.empty(34, 12, 64, dtype=torch.float16, device="cuda").transpose(0, 1)
    _check_lookup(eb, wide[:, 8:72], ids, out=swapped)
    # three axes that do not join
    with pytest.raises(ValueError, match="join"):
        eb.embedding(wide, ids.view(3, 4, 34).transpose(0, 2))


def test_lookup_of_a_shard(eb):
    rng = _gen(5)
    table = _values(rng, (1000, 128), torch.float32).cuda()
    ids = torch.from_numpy(rng.integers(0, 1000, 777)).cuda()
    parts = [eb.embedding(table[a:b], ids, first=a, scale=3.0) for a, b in ((0, 300), (300, 301), (301, 1000))]
    assert torch.equal(parts[0] + parts[1] + parts[2], eb.embedding(table, ids, scale=3.0))
    far = torch.tensor([2**62, -2**62, 2**63 - 1, -2**63, 5, 2**31 + 3], device="cuda")
    got = _check_lookup(eb, table, far, first=2**31)
    assert torch.equal(got[5], table[3]) and int((got != 0).any(1).sum()) == 1
    assert not _check_lookup(eb, table, far, first=2**62 + 1).any()
    assert not eb.embedding(table[:0], ids).any()


def test_lookup_past_32_bits(eb):
    """A table and an output of more than 2^31 elements each."""
    rows, dim = 1_100_000, 2048
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    last = torch.arange(rows - 64, rows, device="cuda")
    table[last] = torch.randn(64, dim, device="cuda").to(torch.bfloat16)
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    ids[-64:] = last.flip(0).int()
    got = eb.embedding(table, ids)
    assert torch.equal(got[-64:], table[last.flip(0)]) and not got[:-64].any()


# ------------------------------------------------------------------------- gradient

def _check_gradient(eb, grad, tokens, rows, *, scale=1.0, first=0, out=None, dtype=None, accumulate=False):
    before = out.double().cpu() if accumulate else None
    got = eb.embedding_grad(grad, tokens, rows, scale=scale, first=first, out=out, dtype=dtype,
                            accumulate=accumulate)
    dim = grad.shape[-1]
    ids = tokens.cpu().long().reshape(-1) - first
    known = (ids >= 0) & (ids < rows) & (tokens.cpu().reshape(-1) >= first)
    x = grad.cpu().double().reshape(-1, dim)
    ids, x = ids[known], x[known]
    total = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids, x)
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids, x.abs())
    m = torch.bincount(ids, minlength=rows).double()[:, None]
    s, u32 = float(np.float32(scale)), half_step(torch.float32)
    summed = (m - 1).clamp(min=0) * u32 / (1 - m * u32) * size
    want = total * s
    tol = summed * abs(s) + u32 * (want.abs() + summed * abs(s))
    if accumulate:
        want = want + before
        tol = tol * (1 + u32) + u32 * want.abs()
    tol = tol + half_step(got.dtype) * (want.abs() + tol) + least(got.dtype)
    _close(got, want, tol)
    if accumulate:
        untouched = torch.ones(rows, dtype=torch.bool)
        untouched[ids] = False
        assert torch.equal(got.cpu()[untouched].double(), before[untouched])
    return got


def _ids(rng, kind, n, rows):
    if kind == "uniform":
        return rng.integers(0, rows, n)
    if kind == "skewed":  # the r-th most frequent about 1/r as often as the first, some padding
        rank = np.minimum(np.exp(rng.random(n) * np.log(rows)).astype(np.int64) - 1, rows - 1).clip(0)
        ids = rng.permutation(rows)[rank]
        return np.where(rng.random(n) < 0.1, -1, ids)
    if kind == "one":
        return np.full(n, rows - 1)
    if kind == "none":
        return np.where(np.arange(n) % 2 == 0, -1, rows)
    return np.arange(n)[::-1] % rows  # falling


@pytest.mark.parametrize("kind", ("uniform", "skewed", "one", "none", "falling"))
@pytest.mark.parametrize("n,rows,dim", [(0, 5, 8), (1, 1, 1), (1, 300, 64), (7, 3, 24), (65, 2, 520), (301, 8209, 40),
                                        (4096, 511, 72), (4096, 512, 33), (4097, 513, 64), (9000, 40009, 777),
                                        (20000, 1000, 128), (5000, 300000, 16), (60, 9, 20000), (60, 9, 20003),
                                        (3000, 40, 2052)])
def test_gradient_sizes(eb, n, rows, dim, kind):
    rng = _gen(6, n, rows, dim)
    grad = _values(rng, (n, dim), torch.bfloat16).cuda()
    _check_gradient(eb, grad, torch.from_numpy(_ids(rng, kind, n, rows)).cuda(), rows, dtype=torch.float32)


@pytest.mark.parametrize("kind", ("uniform", "skewed", "one"))
@pytest.mark.parametrize("n,rows", [(512, 70000), (513, 300), (1024, 511), (1025, 262143), (8192, 300),
                                    (8193, 70000), (65536, 300000), (65537, 5000), (131072, 262144),
                                    (131073, 700), (131073, 300000), (530000, 70000)])
def test_gradient_sorts(eb, n, rows, kind):
    """Every size at which the sort changes its form, of one to three passes."""
    rng = _gen(19, n, rows)
    grad = _values(rng, (n, 8), torch.float32).cuda()
    ids = torch.from_numpy(_ids(rng, kind, n, rows)).cuda()
    got = _check_gradient(eb, grad, ids, rows)
    # the runs' order is that of the tokens: a sum of whole numbers of one run's positions is exact
    place = (torch.arange(n, device="cuda") % 64).float()[:, None].expand(n, 8)
    want = torch.zeros(rows + 1, dtype=torch.float64, device="cuda")
    want.index_add_(0, torch.where(ids < 0, rows, ids), place[:, 0].double())
    if float(want[:rows].max()) < 2**24:
        assert torch.equal(eb.embedding_grad(place, ids, rows)[:, 3].double(), want[:rows])
    assert torch.equal(eb.embedding_grad(grad, ids, rows), got)


@pytest.mark.parametrize("dim", (4, 60, 520, 521))
@pytest.mark.parametrize("longest", (3, 40, 130, 2600))
def test_gradient_runs(eb, dim, longest):
    """Runs of every length around the chunks', beginning and ending everywhere in them; whole numbers, so that
    any order of the sums is exact and a row lost, doubled or split shows."""
    for seed in range(6):
        rng = _gen(21, dim, longest, seed)
        lengths = rng.integers(0, longest + 1, 40) if seed % 2 else \
            rng.choice([n for n in (0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 256, 257, 2048,
                                    2111) if n <= longest], 60)
        rows = len(lengths)
        ids = np.repeat(np.arange(rows), lengths)
        ids = np.concatenate((ids, np.full(rng.integers(0, 30), rows)))  # and some without a row
        ids = torch.from_numpy(rng.permutation(ids)).cuda()
        grad = torch.from_numpy(rng.integers(-8, 9, (ids.numel(), dim)).astype(np.float32)).cuda()
        want = torch.zeros(rows + 1, dim, dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double())[:rows]
        assert torch.equal(eb.embedding_grad(grad, ids, rows).double(), want)
        assert torch.equal(eb.embedding_grad(grad.bfloat16(), ids, rows, dtype=torch.float32).double(), want)
        out = torch.ones(rows, dim, device="cuda")
        eb.embedding_grad(grad.half(), ids, rows, scale=2.0, out=out, accumulate=True)
        assert torch.equal(out.double(), 1 + 2 * want)


@pytest.mark.parametrize("source", FLOATS)
@pytest.mark.parametrize("target", FLOATS)
@pytest.mark.parametrize("accumulate", (False, True))
@pytest.mark.parametrize("n,dim", [(700, 64), (700, 37), (9000, 136)])
def test_gradient_types(eb, source, target, accumulate, n, dim):
    rng = _gen(7, n)
    rows = 350
    grad = _values(rng, (n, dim), source).cuda()
    ids = torch.from_numpy(_ids(rng, "skewed", n, rows)).int().cuda()
    out = _values(rng, (rows, dim), target).cuda()
    _check_gradient(eb, grad, ids, rows, scale=0.3, out=out, accumulate=accumulate)


@pytest.mark.parametrize("n", (600, 6000))
def test_gradient_strides(eb, n):
    rng = _gen(8, n)
    rows, dim = 97, 64
    ids = torch.from_numpy(rng.integers(-1, rows, (6, n // 6))).cuda()
    base = _values(rng, (n // 6, 6, 72), torch.float16).cuda()
    for grad in (base[..., 8:72].transpose(0, 1), base[..., 3:67].transpose(0, 1),
                 torch.ones((), dtype=torch.float16, device="cuda").expand(6, n // 6, dim),  # a sum's gradient
                 base[:, 0, :64].unsqueeze(0).expand(6, n // 6, dim),
                 base[0, :, :64].unsqueeze(1).expand(6, n // 6, dim),
                 base[..., :1].transpose(0, 1).expand(6, n // 6, dim),
                 torch.as_strided(base, (6, n // 6, dim), (1, 6, n))):
        _check_gradient(eb, grad, ids, rows, dtype=torch.float32)
    grad = base[..., 8:72].transpose(0, 1)
    _check_gradient(eb, grad, ids.t().contiguous().t(), rows)
    _check_gradient(eb, grad.reshape(2, 3, n // 6, dim), ids.view(2, 3, n // 6), rows)
    # a table's gradient inside a larger plane; what lies around it stays
    for columns in (slice(8, 72), slice(3, 67), slice(4, 68)):
        room = torch.full((rows + 2, 80), 5.0, device="cuda")
        _check_gradient(eb, grad, ids, rows, out=room[1:-1, columns])
        room[1:-1, columns] = 5.0
        assert bool((room == 5.0).all())


def test_gradient_of_a_shard(eb):
    rng = _gen(9)
    grad = _values(rng, (6000, 48), torch.bfloat16).cuda()
    ids = torch.from_numpy(rng.integers(0, 1000, 6000)).cuda()
    whole = eb.embedding_grad(grad, ids, 1000, dtype=torch.float32)
    for first, rows in ((0, 400), (400, 600), (999, 1), (5000, 30)):
        part = _check_gradient(eb, grad, ids, rows, first=first, dtype=torch.float32)
        if first < 1000:
            assert torch.allclose(part, whole[first:first + rows], rtol=1e-5, atol=1e-4)
    assert eb.embedding_grad(grad, ids, 0).shape == (0, 48)
    assert eb.embedding_grad(grad[:, :0], ids, 7).shape == (7, 0)


def test_gradient_ignores_what_padding_holds(eb):
    for n in (500, 5000):
        grad = torch.ones(n, 40, dtype=torch.bfloat16, device="cuda")
        ids = torch.arange(n, device="cuda") % 7
        ids[::3] = -1
        grad[::3] = float("nan")
        assert torch.equal(eb.embedding_grad(grad, ids, 9)[:, 0].float().cpu(),
                           torch.bincount(ids[ids >= 0], minlength=9).float().bfloat16().float().cpu())
        grad[4], ids[4] = float("inf"), 8
        got = eb.embedding_grad(grad, ids, 9)
        assert bool(got[8].isinf().all()) and bool(got[:8].isfinite().all())


@pytest.mark.parametrize("n,dim", [(4000, 256), (30000, 264), (30000, 71)])
def test_gradient_bits_do_not_depend_on_the_run(eb, n, dim):
    """The same bits from a repeated call, a graph, misaligned memory and beside other work."""
    rng = _gen(10, n)
    rows = 5000
    grad = _values(rng, (n, dim), torch.float32).cuda()
    ids = torch.from_numpy(_ids(rng, "skewed", n, rows)).cuda()
    want = eb.embedding_grad(grad, ids, rows).clone()
    shifted = torch.empty(n, dim + 1, device="cuda")[:, 1:]
    shifted.copy_(grad)
    assert torch.equal(eb.embedding_grad(shifted, ids, rows), want)
    # rows on words, off them, and values apart from one another: the same sums, added the same way
    base = _values(rng, (rows, dim), torch.float32).cuda()
    strided = torch.empty(dim, n, device="cuda").t()
    strided.copy_(grad)
    added = [eb.embedding_grad(g, ids, rows, out=o, scale=0.3, accumulate=True)
             for g in (grad, shifted, strided) for o in (base.clone(), torch.cat((base[:, :1], base), 1)[:, 1:])]
    assert all(torch.equal(added[0], other) for other in added[1:])
    assert torch.equal(eb.embedding_grad(strided, ids, rows), want)
    call = eb.EmbeddingGrad(grad, ids, rows)
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(5):
        with torch.cuda.stream(side):
            busy @ busy
        assert torch.equal(call(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    call.out.fill_(-1.0)
    graph.replay()
    assert torch.equal(call.out, want)
    ids.copy_(ids.flip(0))
    grad.copy_(grad.flip(0))
    graph.replay()
    _check_gradient(eb, grad, ids, rows)
    assert torch.equal(call.out, eb.embedding_grad(grad, ids, rows))


def test_gradient_is_that_of_the_lookup(eb):
    """Central differences of sum(y * c) in 32 bits; the function is linear, so they carry only roundings."""
    rng = _gen(11)
    table = _values(rng, (30, 16), torch.float32).cuda()
    ids = torch.from_numpy(rng.integers(-1, 30, (4, 25))).cuda()
    c = _values(rng, (4, 25, 16), torch.float32).cuda()
    got = eb.embedding_grad(c, ids, 30, scale=1.5).double().cpu()

    def value(t):
        return float((eb.embedding(t, ids, scale=1.5).double() * c.double()).sum())

    for v, k in ((0, 0), (3, 7), (29, 15), (11, 2)):
        up, down = table.clone(), table.clone()
        up[v, k] += 0.5
        down[v, k] -= 0.5
        step = float(up[v, k].double() - down[v, k].double())
        # every looked-up value carries at most 2^-24 |1.5 w|, |w| < 6, times |c| < 6, in at most 100 terms
        tol = 2 * 100 * 2**-24 * 9 * 6 / step + 1e-4
        assert abs((value(up) - value(down)) / step - got[v, k]) <= tol


def test_gradient_past_32_bits(eb):
    n, dim, rows = 1_100_000, 2048, 3
    grad = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda").expand(n, dim)
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    ids[-1000:] = 2
    full = grad.contiguous()
    full[-1000:] = 3.0
    for g, last in ((grad, 1000.0), (full, 3000.0)):
        got = eb.embedding_grad(g, ids, rows, dtype=torch.float32)
        assert bool((got[0] == n - 1000).all()) and not got[1].any() and bool((got[2] == last).all())
    wide = eb.embedding_grad(full[-2:], ids[-2:] * (n // 2), n + 1, dtype=torch.bfloat16)
    assert bool((wide[n] == 6.0).all()) and not wide[:n].any()


# ------------------------------------------------------------------------- block tables

def _want_tables(lengths, held, table, pool, count, block, used, terminated):
    """One request after the other, in whole numbers."""
    table, used = table.copy(), None if used is None else used.copy()
    width, asked, taken, short = table.shape[1], 0, 0, 0
    count = count if 0 <= count <= len(pool) else 0
    blocks = []
    for r in range(len(lengths)):
        have = min(max(int(held[r]), 0), width)
        if terminated is not None and terminated[r]:
            if used is not None:
                for b in table[r, :have]:
                    if 0 <= b < len(used):
                        used[b] = 0
            blocks.append(0)
            continue
        need = -(-max(int(lengths[r]), 0) // block)
        more = max(0, need - have) if need <= width else 0
        asked += more
        if need > width or (more and asked > count):
            short += 1
            blocks.append(have)
            continue
        for j in range(more):
            table[r, have + j] = pool[asked - more + j]
            if used is not None and 0 <= pool[asked - more + j] < len(used):
                used[pool[asked - more + j]] = 1
        taken = asked if more else taken
        blocks.append(max(need, have))
    return table, used, np.array(blocks, np.int32), np.array([taken, short], np.int32)


def _check_tables(eb, lengths, held, table, pool, count, block, used=None, terminated=None):
    want = _want_tables(lengths, held, table, pool, count, block, used, terminated)
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (lengths, held, table, pool)]
    used_ = None if used is None else torch.from_numpy(used).cuda()
    term = None if terminated is None else torch.from_numpy(terminated).cuda()
    cell = torch.tensor([count], dtype=torch.int32, device="cuda")
    call = eb.BlockTables(*dev, cell, block=block, used=used_, terminated=term)
    for _ in range(2):  # a repeated call gives the same
        blocks, cells = call()
        assert np.array_equal(dev[2].cpu().numpy(), want[0])
        assert used is None or np.array_equal(used_.cpu().numpy(), want[1])
        assert np.array_equal(blocks.cpu().numpy(), want[2]) and np.array_equal(cells.cpu().numpy(), want[3])
    return want


@pytest.mark.parametrize("requests", (0, 1, 2, 33, 513, 2048, 2049, 8192, 8193, 20000))
@pytest.mark.parametrize("block", (1, 16, 24))
@pytest.mark.parametrize("dtype", (np.int32, np.int64))
def test_tables(eb, requests, block, dtype):
    rng = _gen(12, requests, block)
    width = 20
    for share, done in ((2.0, 0.0), (0.6, 0.2), (0.0, 1.0)):
        held = rng.integers(0, width + 1, requests).astype(np.int32)
        lengths = (held.astype(np.int64) * block + rng.integers(-2 * block, 3 * block, requests)).astype(dtype)
        blocks = max(1, requests * width)
        owner = rng.permutation(2 * blocks).astype(np.int32)
        table = np.full((requests, width), -1, np.int32)
        table[np.arange(width) < held[:, None]] = owner[:int(held.sum())]
        used = np.zeros(2 * blocks, np.uint8)
        used[owner[:int(held.sum())]] = 1
        pool = np.flatnonzero(used == 0).astype(np.int32)
        count = min(len(pool), int(requests * share))
        _check_tables(eb, lengths, held, table, pool, count, block, used, rng.random(requests) < done)


def test_tables_at_the_edges(eb):
    i32 = np.int32
    pool = np.arange(10, 20, dtype=i32)
    table = np.full((4, 3), -7, i32)
    zeros = np.zeros(4, i32)
    for lengths, held, count in (
            ([0, 0, 0, 0], [0, 0, 0, 0], 10), ([48, 49, 48, 0], [0, 0, 0, 3], 10),  # 49: past the row
            ([48, 48, 48, 48], [0, 0, 0, 0], 10), ([48, 48, 48, 1], [0, 0, 0, 0], 9), ([16, 16, 16, 16], [1] * 4, 0),
            ([-5, 2**31 - 1, 1, 1], [0, 0, 0, 0], 2), ([1, 1, 1, 1], [-3, 9, 3, 0], 4), ([48] * 4, [0] * 4, -1),
            ([48] * 4, [0] * 4, 11), ([1] * 4, [0] * 4, 3)):
        _check_tables(eb, np.array(lengths, i32), np.array(held, i32), table, pool, count, 16)
    # ids outside the mask are handed out, and nothing is written for them
    odd = np.array([5, -1, 100, 2**31 - 1, 0, 1], i32)
    _check_tables(eb, np.array([48, 48, 0, 0], i32), zeros, table, odd, 6, 16, np.zeros(8, np.uint8))
    # neither may a terminated request's row name what the mask does not have
    rows = np.array([[3, -1, 2**31 - 1], [1, 2, 9], [0, 0, 0], [4, 4, 4]], i32)
    _check_tables(eb, np.full(4, 40, np.int64), np.array([3, 2, 0, 99], i32), rows, pool[:0], 0, 16,
                  np.ones(6, np.uint8), np.array([True, True, True, True]))
    # width 0, and lengths in 64 bits past every row
    _check_tables(eb, np.array([0, 1, 0, 2**62]), zeros, table[:, :0], pool, 10, 16)
    _check_tables(eb, np.array([2**62, -2**62, 2**63 - 1, 5]), zeros, table, pool, 10, 16)


def test_tables_in_a_wider_plane(eb):
    plane = torch.full((5, 16), -1, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([3, 70, 0, 33, 16], device="cuda")
    held = torch.zeros(5, dtype=torch.int32, device="cuda")
    pool = torch.arange(100, 150, dtype=torch.int32, device="cuda")
    count = torch.tensor([50], dtype=torch.int32, device="cuda")
    blocks, cells = eb.block_tables(lengths, held, plane[:, 3:9], pool, count, block=16)
    assert blocks.tolist() == [1, 5, 0, 3, 1] and cells.tolist() == [10, 0]
    assert plane[:, :3].eq(-1).all() and plane[:, 9:].eq(-1).all()
    assert plane[1, 3:9].tolist() == [101, 102, 103, 104, 105, -1] and plane[3, 3:6].tolist() == [106, 107, 108]


# ------------------------------------------------------------------------- slots

def _want_slots(table, start, fresh, capacity, block, terminated, bits=64):
    slots, positions, requests = np.full(capacity, -1, np.int64), np.zeros(capacity, np.int64), \
        np.full(capacity, -1, np.int32)
    offsets, q = [0], 0
    for r in range(len(start)):
        n = 0 if terminated is not None and terminated[r] else max(int(fresh[r]), 0)
        inside = max(0, min(n, capacity - q))
        p = max(int(start[r]), 0) + np.arange(inside, dtype=object)
        for i, at in enumerate(p):
            b = at // block
            if b < table.shape[1] and table[r, b] >= 0 and int(table[r, b]) * block + at % block < 2 ** (bits - 1):
                slots[q + i] = int(table[r, b]) * block + at % block
        wrap = 2 ** (8 * start.dtype.itemsize)  # a position past its type wraps
        positions[q:q + inside] = [(int(at) + wrap // 2) % wrap - wrap // 2 for at in p]
        requests[q:q + inside] = r
        q += n
        offsets.append(min(q, 2**31 - 1))
    return slots, positions, requests, np.array(offsets, np.int64)


def _check_slots(eb, table, start, fresh, capacity, block, terminated=None, dtype=torch.int64):
    want = _want_slots(table, start, fresh, capacity, block, terminated, 64 if dtype == torch.int64 else 32)
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, start, fresh)]
    term = None if terminated is None else torch.from_numpy(terminated).cuda()
    got = eb.slot_map(*dev, capacity, block=block, terminated=term, dtype=dtype)
    assert got[0].dtype == dtype and got[1].dtype == dev[1].dtype
    for g, w, name in zip(got, want, ("slots", "positions", "requests", "offsets")):
        assert np.array_equal(g.cpu().numpy().astype(np.int64), w), name


@pytest.mark.parametrize("requests", (0, 1, 5, 513, 2048, 2049, 8192, 8193))
@pytest.mark.parametrize("block", (1, 16, 24))
@pytest.mark.parametrize("dtype,slot", [(np.int32, torch.int64), (np.int64, torch.int32)])
def test_slots(eb, requests, block, dtype, slot):
    rng = _gen(13, requests, block)
    width = 12
    table = rng.integers(-1, 1000, (requests, width)).astype(np.int32)
    start = rng.integers(-2, width * block, requests).astype(dtype)
    for kind, done in (("one", 0.1), ("ragged", 0.3), ("none", 0.0), ("ragged", 1.0)):
        fresh = {"one": np.ones(requests), "none": np.zeros(requests),
                 "ragged": rng.integers(-1, 9, requests) * (rng.random(requests) < 0.3)}[kind].astype(dtype)
        total = int(fresh.clip(0).sum())
        for capacity in {0, 1, total, max(0, total - 3), total + 5}:
            _check_slots(eb, table, start, fresh, capacity, block, rng.random(requests) < done, slot)


def test_slots_at_the_edges(eb):
    table = np.array([[0, 7, 2**31 - 1], [-1, 5, 6], [2**30, 1, 1]], np.int32)
    start = np.array([0, 3, 30])
    fresh = np.array([60, 40, 2])
    for slot in (torch.int32, torch.int64):  # slots past 2^31 fit one of the two
        _check_slots(eb, table, start, fresh, 103, 16, None, slot)
    for s in (2**62, 2**63 - 1, 2**31, -2**63):
        _check_slots(eb, table, np.array([s if s < 2**63 - 8 else s - 40, 0, s if s < 2**62 else 3]), fresh, 103, 16)
    # more tokens than an int32 counts: offsets stop there
    _check_slots(eb, table, start, np.array([2**31, 5, 2**62]), 50, 16)
    _check_slots(eb, table, start.astype(np.int32), np.array([2**31 - 1] * 3, np.int32), 50, 16)
    # width 0
    _check_slots(eb, table[:, :0], start, fresh, 20, 16)
    # one long request between thousands without tokens
    fresh = np.zeros(8000, np.int64)
    fresh[[0, 4000, 7999]] = 3, 5000, 2
    _check_slots(eb, np.arange(8000 * 4, dtype=np.int32).reshape(8000, 4), np.zeros(8000, np.int64), fresh, 5100, 2048)


# ------------------------------------------------------------------------- refusals

def test_refusals(eb):
    dev = dict(device="cuda")
    table = torch.zeros(10, 16, **dev)
    ids = torch.zeros(4, dtype=torch.int64, **dev)
    with pytest.raises(TypeError):
        eb.embedding(table.double(), ids)
    with pytest.raises(TypeError):
        eb.embedding(table, ids.short())
    with pytest.raises(TypeError):
        eb.embedding(table, ids, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        eb.embedding(table, ids.cpu())
    for bad in (table.t(), table[0], table[:1].expand(10, 16)):
        with pytest.raises(ValueError):
            eb.embedding(bad, ids)
    with pytest.raises(ValueError, match="first"):
        eb.embedding(table, ids, first=-1)
    with pytest.raises(ValueError, match="autograd"):
        eb.embedding(table.clone().requires_grad_(), ids)
    with torch.no_grad():
        eb.embedding(table.clone().requires_grad_(), ids)
    for out in (torch.zeros(4, 15, **dev), torch.zeros(16, 4, **dev).t(), torch.zeros(1, 16, **dev).expand(4, 16)):
        with pytest.raises(ValueError):
            eb.embedding(table, ids, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        eb.embedding(table, ids, out=table[:4])
    grad = torch.zeros(4, 16, **dev)
    with pytest.raises(ValueError, match="shape"):
        eb.embedding_grad(grad[:3], ids, 10)
    with pytest.raises(ValueError, match="rows"):
        eb.embedding_grad(grad, ids, -1)
    with pytest.raises(ValueError, match="accumulate"):
        eb.embedding_grad(grad, ids, 10, accumulate=True)
    with pytest.raises(ValueError, match="overlaps"):
        eb.embedding_grad(grad, ids, 4, out=grad)
    with pytest.raises(ValueError, match="shape"):
        eb.embedding_grad(grad, ids, 10, out=table[:9])
    with pytest.raises(ValueError, match="autograd"):
        eb.embedding_grad(grad.clone().requires_grad_(), ids, 10)
    tables = torch.zeros(3, 4, dtype=torch.int32, **dev)
    lengths = torch.zeros(3, dtype=torch.int32, **dev)
    pool, count = torch.zeros(8, dtype=torch.int32, **dev), torch.zeros(1, dtype=torch.int32, **dev)
    good = dict(lengths=lengths, held=lengths, table=tables, pool=pool, count=count, block=16)
    eb.block_tables(**good)
    for change, error in ((dict(lengths=lengths.float()), TypeError), (dict(held=lengths.long()), TypeError),
                          (dict(lengths=lengths[:2]), ValueError), (dict(table=tables.t()), ValueError),
                          (dict(table=tables.long()), TypeError), (dict(pool=pool[::2]), ValueError),
                          (dict(count=pool), ValueError), (dict(block=0), ValueError),
                          (dict(pool=tables[0]), ValueError), (dict(used=pool), TypeError),
                          (dict(used=torch.zeros(3, 2, dtype=torch.bool, **dev)), ValueError),
                          (dict(terminated=torch.zeros(2, dtype=torch.bool, **dev)), ValueError),
                          (dict(block=2**31), ValueError), (dict(pool=pool.cpu()), ValueError)):
        with pytest.raises(error):
            eb.block_tables(**{**good, **change})
    good = dict(table=tables, start=lengths, fresh=lengths, capacity=5, block=16)
    eb.slot_map(**good)
    for change, error in ((dict(fresh=lengths.long()), TypeError), (dict(capacity=-1), ValueError),
                          (dict(capacity=2**31 - 1), ValueError), (dict(dtype=torch.int16), TypeError),
                          (dict(block=-1), ValueError), (dict(terminated=lengths), TypeError),
                          (dict(start=lengths[:2]), ValueError)):
        with pytest.raises(error):
            eb.slot_map(**{**good, **change})


# ------------------------------------------------------------------------- streams, and all of them together

def test_other_streams(eb):
    rng = _gen(14)
    table = _values(rng, (500, 64), torch.bfloat16).cuda()
    ids = torch.from_numpy(rng.integers(0, 500, 6000)).cuda()
    grad = _values(rng, (6000, 64), torch.bfloat16).cuda()
    want = eb.embedding(table, ids), eb.embedding_grad(grad, ids, 500)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    late = torch.zeros_like(ids)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        late.copy_(ids)
    got = eb.embedding(table, late, stream=side), eb.embedding_grad(grad, late, 500, stream=side)
    call = eb.EmbeddingGrad(grad, late, 500)
    again = call(side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(again, want[1])


def test_a_decode_loop_in_one_graph(eb):
    """Free list, tables, slots and rows of a pass as one captured graph, replayed until every sequence has
    ended: each token's cache slot is its own, and what a sequence wrote reads back through its table."""
    rng = _gen(15)
    requests, width, block, blocks, dim, rows = 40, 8, 4, 200, 64, 100
    stop = torch.from_numpy(rng.integers(0, width * block + 1, requests)).int().cuda()
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    one = torch.ones(requests, dtype=torch.int32, device="cuda")
    wanted = torch.empty_like(lengths)
    held = torch.zeros(requests, dtype=torch.int32, device="cuda")
    tables = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    used = torch.zeros(blocks, dtype=torch.bool, device="cuda")
    terminated = stop == 0
    weights = _values(rng, (rows, dim), torch.bfloat16).cuda()
    cache = torch.zeros(blocks * block + 1, dim, dtype=torch.bfloat16, device="cuda")
    tokens = torch.empty(48, dtype=torch.int32, device="cuda")
    free = eb.Compactor(used)
    grow = eb.BlockTables(wanted, held, tables, free.index_map, free.count, block=block, used=used,
                          terminated=terminated)
    spot = eb.SlotMap(tables, lengths, one, 48, block=block, terminated=terminated)
    look = eb.Embedding(weights, tokens)

    def step():
        torch.add(lengths, 1, out=wanted)
        free()
        grow()
        held.copy_(grow.blocks)
        slots, positions, owner, _ = spot()
        tokens.copy_(torch.where(owner < 0, -1, (owner * 7 + positions) % rows))
        cache[torch.where(slots < 0, blocks * block, slots)] = look()
        lengths.add_((~terminated).int())
        terminated.logical_or_(lengths >= stop)

    state = [x.clone() for x in (lengths, held, tables, used, terminated)]
    step()  # warm up, then back to the start
    for x, was in zip((lengths, held, tables, used, terminated), state):
        x.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    done_at = {}
    for n in range(width * block + 1):
        before = terminated.cpu().numpy().copy()
        graph.replay()
        assert grow.cells[1].item() == 0
        live = np.flatnonzero(~before)
        slots = spot.slots.cpu().numpy()
        assert len(set(slots[:len(live)])) == len(live) and (slots[len(live):] == -1).all()
        assert (spot.requests.cpu().numpy()[:len(live)] == live).all()
        rows_ = tables.cpu().numpy()
        have = held.cpu().numpy()
        names = [int(b) for r in live for b in rows_[r, :have[r]]]
        assert len(set(names)) == len(names)  # no block has two owners
        assert int(used.sum()) == len(names)
        for r in np.flatnonzero(terminated.cpu().numpy() & ~before):
            length = int(lengths[r])
            assert length == int(stop[r])
            at = [int(rows_[r, p // block]) * block + p % block for p in range(length)]
            want = weights[(r * 7 + torch.arange(length, device="cuda")) % rows]
            assert torch.equal(cache[at], want)
            done_at[r] = n
    graph.replay()
    assert bool(terminated.all()) and not used.any() and not held.any()
    assert len(done_at) == int((stop > 0).sum()) and not cache[-1].any()


def test_a_training_step(eb):
    """Rows looked up, a gradient through a plain layer, and the table's gradient accumulated over two batches:
    what torch's own differentiation of the same formulas gives in 64 bits."""
    rng = _gen(16)
    rows, dim, scale = 700, 96, 96 ** 0.5
    table = _values(rng, (rows, dim), torch.bfloat16).cuda()
    total = torch.zeros(rows, dim, device="cuda")
    exact = torch.zeros(rows, dim, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(exact)
    m = 0
    for seed in (0, 1):
        ids = torch.from_numpy(_ids(_gen(17, seed), "skewed", 4 * 1500, rows)).view(4, 1500).cuda()
        c = _values(_gen(18, seed), (4, 1500, dim), torch.bfloat16).cuda()
        y = eb.embedding(table, ids, scale=scale)
        dy = (c * torch.where(y > 0, 1.0, 0.0)).to(torch.bfloat16)  # of sum(c * relu(y)), exact
        eb.embedding_grad(dy, ids, rows, scale=scale, out=total, accumulate=True)
        leaf = table.double().requires_grad_()
        known = (ids >= 0)[..., None]
        out = torch.where(known, leaf[ids.clamp(min=0)] * float(np.float32(scale)), 0.0)
        (out.relu() * c.double()).sum().backward()
        exact += leaf.grad
        size.index_add_(0, ids.clamp(min=0).flatten(), (dy.double() * known).abs().flatten(0, 1))
        m += 6000
    u = half_step(torch.float32)
    tol = (m + 6) * u / (1 - m * u) * size * float(np.float32(scale))
    assert bool(((total.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("n", (500, 9000, 140000))
def test_in_the_body_of_a_device_loop(eb, n):
    """Captured into a WHILE node's body, as the until-done loop runs: three passes, each adding the gradient of
    one batch, looking up the rows of the next and taking one more block for every request; calls right before
    the loop, as the first and last of its body, and right after a loop and a memset."""
    import ctypes

    from eagle_b200 import _abi
    from eagle_b200.graphs import CaptureConditional, Graph, StreamCapturer

    rng = _gen(20, n)
    rows, dim, requests, passes = 500, 64, 3000, 3
    table = _values(rng, (rows, dim), torch.float32).cuda()
    ids = torch.from_numpy(_ids(rng, "skewed", n, rows)).cuda()
    grad = _values(rng, (n, dim), torch.float32).cuda()
    total = torch.zeros(rows, dim, device="cuda")
    cells = torch.tensor([0, passes, 0, 0], dtype=torch.int32, device="cuda")
    lengths = torch.full((requests,), 5, dtype=torch.int32, device="cuda")
    held = torch.ones(requests, dtype=torch.int32, device="cuda")
    tables = torch.zeros(requests, 4, dtype=torch.int32, device="cuda")
    pool = torch.arange(requests, dtype=torch.int32, device="cuda")
    count = torch.tensor([requests], dtype=torch.int32, device="cuda")
    grow = eb.BlockTables(lengths, held, tables, pool, count, block=4)
    spot = eb.SlotMap(tables, held, held, requests + 7, block=4)
    look = eb.Embedding(table, ids, scale=2.0)
    add = eb.EmbeddingGrad(grad, ids, rows, out=total, accumulate=True)
    want = eb.embedding_grad(grad, ids, rows)
    first, after, last = eb.Embedding(table, ids), eb.EmbeddingGrad(total, ids[:rows], rows), eb.Embedding(table, ids)
    origin = torch.cuda.Stream()
    s = origin.cuda_stream
    torch.cuda.synchronize()
    at = cells.data_ptr()
    loop = CaptureConditional(s, count_ptr=at, baseline_ptr=at + 4, loop_cap=10, counter_ptr=at + 8)
    cap = StreamCapturer(s)
    cap.begin()
    first(origin)
    body = loop.begin()
    on = torch.cuda.ExternalStream(body)
    for call in (grow, spot, look):
        call(on)
    d = _abi.new(_abi.CellOpDesc, op=_abi.CELL_BUMP, device=-1, stream=int(body))
    d.p[0] = at
    _abi.check(_abi.lib().eagle_backend_cell_op(ctypes.byref(d)))
    add(on)
    loop.end()
    after(origin)
    _abi.check(_abi.lib().eagle_backend_memset_device(at + 12, 4, s))
    last(origin)
    launcher = Graph.from_captured(cap.end()).launcher()
    launcher.stream(s)
    launcher.launch()
    launcher.synchronize()
    assert cells.tolist()[:2] == [passes, passes]
    assert torch.equal(total, want + want + want)
    assert torch.equal(look.out, eb.embedding(table, ids, scale=2.0))
    assert torch.equal(first.out, eb.embedding(table, ids)) and torch.equal(last.out, first.out)
    assert torch.equal(after.out, eb.embedding_grad(total, ids[:rows], rows))
    assert grow.cells.tolist() == [requests, 0] and torch.equal(tables[:, 1], pool)
    assert spot.offsets[-1].item() == requests
    # position 1 lies in the first block, whose id is 0
    assert bool((spot.slots[:requests] == 1).all()) and bool((spot.slots[requests:] == -1).all())


# ------------------------------------------------------------------------- waits that run out

@pytest.mark.parametrize("dim", (1024, 1023))
@pytest.mark.parametrize("asked", (0, 1, 2, 5))
@pytest.mark.parametrize("lengths", ([3, 2, 3, 2], [2, 5, 4, 1], [40, 3, 1], [1, 39, 2, 2], [8, 8, 8]))
def test_gradient_wait_gives_up(eb, dim, asked, lengths):
    """Some rows of the first chunk (8 sorted positions here) are never asked for: the runs whose rows had all come
    are right, those that needed the others NaN and no others, and the call can tell; the same workspace then
    serves a whole gradient. Every wait ends: 1024 polls."""
    import ctypes

    from eagle_b200 import _abi

    chunk, group = 8, 4
    ids = np.repeat(np.arange(len(lengths) + 20), lengths + [2] * 20)
    rows, n = int(ids[-1]) + 2, len(ids)
    grad = _values(_gen(22, dim), (n, dim), torch.bfloat16).cuda()
    out = torch.full((rows, dim), 5.0, device="cuda")
    call = eb.EmbeddingGrad(grad, torch.from_numpy(ids).cuda(), rows, out=out)
    want = call().clone()
    call.check()
    d = _abi.new(_abi.EmbeddingDesc)
    ctypes.memmove(ctypes.byref(d), ctypes.byref(call._desc), ctypes.sizeof(d))
    d.stream = torch.cuda.current_stream().cuda_stream
    _abi.check(_abi.lib().eagle_backend_x_b200_embedding_grad_wait_check(ctypes.byref(d), 1024, asked))
    torch.cuda.synchronize()
    # the first chunk sums its own 8 positions, and those of a run that goes on over one boundary only
    starts = np.cumsum([0] + lengths)
    last = int(np.searchsorted(starts, chunk - 1, side="right")) - 1
    whole = starts[last] > 0 and starts[last + 1] <= 2 * chunk and starts[last + 1] > chunk
    summed = starts[last + 1] if whole else chunk
    lost = set(ids[min(group * asked, summed):summed].tolist())
    for r in range(rows):
        if r in lost:
            assert bool(out[r].isnan().all()), r
        else:
            assert torch.equal(out[r], want[r]), r
    if lost:
        with pytest.raises(eb.BackendError, match="wait"):
            call.check()
    else:
        call.check()
    assert torch.equal(call(), want)
    call.check()


# ------------------------------------------------------------------------- rows that serve one request after the other

@pytest.mark.parametrize("requests", (0, 1, 5, 513, 2048, 2049, 8192, 8193))
@pytest.mark.parametrize("dtype,slot", [(np.int32, torch.int64), (np.int64, torch.int32)])
def test_slots_of_held_blocks(eb, requests, dtype, slot):
    """Entries past what a request holds are as good as absent."""
    rng = _gen(23, requests)
    width, block = 12, 16
    table = rng.integers(-1, 1000, (requests, width)).astype(np.int32)
    held = rng.integers(-2, width + 4, requests).astype(np.int32)
    start = rng.integers(-2, width * block, requests).astype(dtype)
    fresh = rng.integers(0, 40, requests).astype(dtype)
    own = np.where(np.arange(width) < held[:, None], table, -1)
    total = int(fresh.sum())
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, start, fresh, held)]
    for capacity in {0, max(0, total - 3), total + 5}:
        want = _want_slots(own, start, fresh, capacity, block, None, 64 if slot == torch.int64 else 32)
        got = eb.slot_map(*dev[:3], capacity, block=block, held=dev[3], dtype=slot)
        for g, w, name in zip(got, want, ("slots", "positions", "requests", "offsets")):
            assert np.array_equal(g.cpu().numpy().astype(np.int64), w), name


def test_a_reused_row_left_short(eb):
    """The loop of a paged cache, its rows reused: a request that comes into a finished one's row while others took
    the blocks it gave back has no slot among theirs, in a replayed graph."""
    dev = dict(dtype=torch.int32, device="cuda")
    block, width, blocks = 4, 3, 6
    lengths = torch.tensor([12, 4, 0], **dev)
    held, start, fresh = (torch.zeros(3, **dev) for _ in range(3))
    tables = torch.full((3, width), -1, **dev)
    used = torch.zeros(blocks, dtype=torch.bool, device="cuda")
    terminated = torch.zeros(3, dtype=torch.bool, device="cuda")
    free = eb.Compactor(used)
    grow = eb.BlockTables(lengths, held, tables, free.index_map, free.count, block=block, used=used,
                          terminated=terminated)
    spot = eb.SlotMap(tables, start, fresh, 16, block=block, held=held, terminated=terminated)

    def step():
        free()
        grow()
        held.copy_(grow.blocks)
        spot()

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    assert held.tolist() == [3, 1, 0] and tables[0].tolist() == [0, 1, 2]
    terminated[0] = True  # request 0 ends
    graph.replay()
    assert held.tolist() == [0, 1, 0] and int(used.sum()) == 1
    lengths.copy_(torch.tensor([0, 12, 12], **dev))  # the others take all but one of the blocks
    graph.replay()
    assert held.tolist() == [0, 3, 3] and int(used.sum()) == 6
    terminated[0] = False  # and the next request comes into its row
    lengths[0] = 9
    start.copy_(torch.tensor([0, 4, 0], **dev))
    fresh.copy_(torch.tensor([9, 2, 3], **dev))
    graph.replay()
    assert grow.cells.tolist() == [0, 1] and held.tolist() == [0, 3, 3]
    assert tables[0].tolist() == [0, 1, 2]  # what the one before left
    assert spot.offsets.tolist() == [0, 9, 11, 14]
    assert spot.slots[:9].eq(-1).all() and spot.requests[:9].eq(0).all() and spot.positions[:9].tolist() == list(range(9))
    rows = tables.cpu().numpy()
    assert spot.slots[9:14].tolist() == [rows[1, 1] * 4, rows[1, 1] * 4 + 1] + [rows[2, 0] * 4 + i for i in range(3)]


# ------------------------------------------------------------------------- calls that were refused

def test_axes_that_join_behind_the_first(eb):
    """Tokens of three axes whose last two join, and whose first two do not, are looked up and summed."""
    rng = _gen(24)
    table = _values(rng, (50, 24), torch.bfloat16).cuda()
    ids = torch.from_numpy(rng.integers(-1, 50, (40, 3))).cuda().t().view(3, 8, 5)
    _check_lookup(eb, table, ids)
    _check_gradient(eb, _values(rng, (3, 8, 5, 24), torch.float32).cuda(), ids, 50)
    _check_gradient(eb, _values(rng, (3, 40, 30), torch.float32).cuda()[..., 3:27].unflatten(1, (8, 5)), ids, 50)


def test_columns_of_one_plane(eb):
    """The table and its output, or a gradient and the table's, in columns of one plane: what lies around stays."""
    rng = _gen(25)
    for cut, dtype in ((64, torch.bfloat16), (61, torch.bfloat16), (700, torch.float32), (1023, torch.float16)):
        plane = _values(rng, (300, 2 * cut + 3), dtype).cuda()
        was = plane.clone()
        ids = torch.from_numpy(rng.integers(-1, 300, 300)).cuda()
        left, right = plane[:, :cut], plane[:, cut + 2:2 * cut + 2]
        _check_lookup(eb, left, ids, out=right)
        assert torch.equal(left, was[:, :cut]) and torch.equal(plane[:, cut:cut + 2], was[:, cut:cut + 2])
        _check_gradient(eb, right, ids, 300, out=left)
        assert torch.equal(plane[:, cut:cut + 2], was[:, cut:cut + 2]) and torch.equal(plane[:, -1], was[:, -1])


# ------------------------------------------------------------------------- tensors that are not what their memory holds

def test_dual_tensors_are_refused(eb):
    from torch.autograd import forward_ad

    table, ids = torch.zeros(10, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        with pytest.raises(ValueError, match="tangent"):
            eb.embedding(dual, ids)
        with pytest.raises(ValueError, match="tangent"):
            eb.embedding_grad(dual[:4], ids, 10)
        assert torch.equal(eb.embedding(forward_ad.unpack_dual(dual).tangent, ids), torch.ones(4, 16, device="cuda"))


def test_negated_views_are_refused(eb):
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    view = torch.randn(4, 16, dtype=torch.complex64, device="cuda").conj().imag
    with pytest.raises(ValueError, match="negates"):
        eb.embedding_grad(view, ids, 10)
    with pytest.raises(ValueError, match="negates"):
        eb.embedding(view[:, :1], ids)
    _check_gradient(eb, view.resolve_neg(), ids, 10)


@pytest.mark.parametrize("value", (2**64 + 16, 16.5))
def test_numbers_that_a_desc_would_cut_are_refused(eb, value):
    dev = dict(device="cuda")
    ids, cells = torch.zeros(4, dtype=torch.int64, **dev), torch.zeros(3, dtype=torch.int32, **dev)
    tables = torch.zeros(3, 4, dtype=torch.int32, **dev)
    for call in (lambda: eb.embedding(torch.zeros(10, 16, **dev), ids, first=value),
                 lambda: eb.embedding_grad(torch.zeros(4, 16, **dev), ids, 10, first=value),
                 lambda: eb.embedding_grad(torch.zeros(4, 16, **dev), ids, value),
                 lambda: eb.block_tables(cells, cells, tables, cells, cells[:1], block=value),
                 lambda: eb.slot_map(tables, cells, cells, 8, block=value),
                 lambda: eb.slot_map(tables, cells, cells, value, block=16)):
        with pytest.raises(ValueError, match="whole"):
            call()


# ------------------------------------------------------------------------- memory that another stream still reads

@pytest.mark.parametrize("form", ("function", "object"))
def test_inputs_stay_until_the_stream_is_past_them(eb, form):
    """Tensors dropped right after a call on another stream: their memory is not given to others while that stream,
    kept busy here, has yet to read it."""
    n, rows, dim = 5000, 300, 64
    rng = _gen(26)
    table, grad = _values(rng, (rows, dim), torch.float32), _values(rng, (n, dim), torch.float32)
    ids = torch.from_numpy(rng.integers(0, rows, n))
    lengths = torch.from_numpy(rng.integers(0, 60, n)).int()
    plane, pool = torch.zeros(n, 4, dtype=torch.int32), torch.arange(n * 4, dtype=torch.int32)
    none, count = torch.zeros(n, dtype=torch.int32), torch.tensor([n * 4], dtype=torch.int32)
    cases = [("embedding", eb.Embedding, (table, ids), (), {}),
             ("embedding_grad", eb.EmbeddingGrad, (grad, ids), (rows,), {}),
             ("block_tables", eb.BlockTables, (lengths, none, plane, pool, count), (), dict(block=16)),
             ("slot_map", eb.SlotMap, (plane, none, lengths), (n * 60,), dict(block=16))]
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    for name, kind, inputs, rest, keys in cases:
        def first(out):
            return out[0] if isinstance(out, tuple) else out

        want = first(getattr(eb, name)(*(x.cuda() for x in inputs), *rest, **keys)).clone()
        mine = [x.cuda() for x in inputs]
        places = {x.data_ptr() for x in mine}
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy @ busy
        if form == "function":
            got = first(getattr(eb, name)(*mine, *rest, **keys, stream=side))
        else:
            got = first(kind(*mine, *rest, **keys)(side))
        sizes = [(x.numel(), x.dtype) for x in mine]
        mine.clear()
        again = [torch.empty(size, dtype=dtype, device="cuda") for size, dtype in sizes * 3]
        assert not side.query()
        assert not places & {x.data_ptr() for x in again}, name
        side.synchronize()
        assert torch.equal(got, want), name


# ------------------------------------------------------------------------- the order of the sums

def _in_order(grad, ids, rows):
    """The sums of float32 rows as documented, in float32: the tokens sorted by id, equal ones in token order, the
    sorted order cut into chunks of 8 to 64 by the sizes; a run in which two chunks or more begin is added up chunk by
    chunk, any other at once; of up to 32 parts one after the other, of more in equal shares whose sums are added."""
    n, dim = grad.shape
    chunk = 8
    while chunk < 64 and n * ((dim + 7) // 8) // 32 // (2 * chunk) >= (4096 if dim >= 512 else 2048):
        chunk *= 2
    lanes = 4
    while lanes < 32 and lanes * 4 < dim:
        lanes *= 2

    def added(rows_):
        return np.cumsum(rows_, axis=0, dtype=np.float32)[-1]

    want = np.zeros((rows, dim), np.float32)
    order = np.argsort(ids, kind="stable")
    order = order[(ids[order] >= 0) & (ids[order] < rows)]
    keys = ids[order]
    starts = np.flatnonzero(np.r_[True, keys[1:] != keys[:-1]]) if keys.size else []
    for b, e in zip(starts, np.r_[starts[1:], keys.size]):
        x = grad[order[b:e]]
        cuts = np.arange(-(-b // chunk) * chunk, e, chunk)
        if len(cuts) < 2:
            want[keys[b]] = added(x)
            continue
        parts = np.array([added(p) for p in np.split(x, cuts[cuts > b] - b)])
        if len(parts) > 32:
            each = -(-len(parts) // (256 // lanes))
            parts = np.array([added(parts[i:i + each]) for i in range(0, len(parts), each)])
        want[keys[b]] = added(parts)
    return want


@pytest.mark.parametrize("kind", ("uniform", "skewed", "one"))
@pytest.mark.parametrize("n,rows,dim", [(900, 300, 8), (3000, 50, 520), (3000, 700, 513), (8000, 1500, 33), (8000, 300, 264),
                                        (60000, 4000, 24), (100000, 9000, 8), (100000, 300, 72), (140000, 2000, 8),
                                        (140000, 70000, 40), (600000, 5000, 4)])
def test_gradient_order(eb, n, rows, dim, kind):
    """The bits of each row, in every form of the sort and of the sums: equal ids in token order, chunk by chunk."""
    rng = _gen(27, n, dim)
    ids = _ids(rng, kind, n, rows)
    grad = rng.standard_normal((n, dim)).astype(np.float32)
    want = _in_order(grad, ids, rows)
    if kind == "one" or n > 4 * rows:  # another order of equal ids, or other cuts, would show
        back = _in_order(grad[::-1].copy(), ids[::-1].copy(), rows)
        assert not np.array_equal(back, want)
    dev, dev_ids = torch.from_numpy(grad).cuda(), torch.from_numpy(ids).cuda()
    got = eb.embedding_grad(dev, dev_ids, rows)
    assert np.array_equal(got.cpu().numpy(), want)
    # in another memory order, and added to what is there
    strided = torch.empty(dim, n, device="cuda").t()
    strided.copy_(dev)
    out = torch.from_numpy(rng.standard_normal((rows, dim)).astype(np.float32)).cuda()
    before = out.cpu().numpy().copy()
    eb.embedding_grad(strided, dev_ids.int(), rows, out=out, accumulate=True)
    named = np.bincount(ids[ids >= 0], minlength=rows)[:, None] > 0
    assert np.array_equal(out.cpu().numpy(), np.where(named, before + want, before))


@pytest.mark.parametrize("n", (100, 50000, 140000))
def test_gradient_of_many_rows(eb, n):
    """A table of more than 2^27 rows, whose ids take four passes; whole numbers, so that the sums are exact."""
    rows, dim = 2**27 + 5, 2
    rng = _gen(28, n)
    ids = torch.from_numpy(np.r_[rng.integers(0, rows, n - 50), np.full(25, rows - 1), np.arange(25)]).cuda()
    grad = torch.from_numpy(rng.integers(1, 9, (n, dim)).astype(np.float32)).half().cuda()
    got = eb.embedding_grad(grad, ids, rows)
    named, place = torch.unique(ids, return_inverse=True)
    want = torch.zeros(named.numel(), dim, device="cuda").index_add_(0, place, grad.float())
    assert torch.equal(got[named].float(), want)
    assert int(got.count_nonzero()) == named.numel() * dim


# ------------------------------------------------------------------------- the largest sizes

def test_a_million_requests(eb):
    """As many requests as are taken: 2^20, a third of them ended, in closed form."""
    requests, block, width = 2**20, 8, 3
    r = torch.arange(requests, device="cuda")
    ended = r % 3 == 1
    held = torch.where(r % 2 == 0, 1, 0).int()
    tables = torch.where(torch.arange(width, device="cuda") < held[:, None], r[:, None], -1).int()
    need = (r % 3 == 0).long() * 2 + (r % 3 == 2).long() * (r % 4)  # three blocks at most, four where the row is too narrow
    need = torch.where(r % 300 == 2, width + 1, need)
    lengths = torch.where(need > 0, need * block - r % block, 0).int()
    fresh = torch.where(ended | (need > width), 0, (need - held).clamp(min=0))
    upto = torch.cumsum(fresh, 0)
    available = int(upto[-1]) - 7
    pool = (torch.randperm(2 * requests, device="cuda") + requests).int()
    used = torch.zeros(3 * requests, dtype=torch.uint8, device="cuda")
    used[r[held > 0]] = 1
    fits = ended | (need <= held) | ((need <= width) & (upto <= available))
    want = tables.clone()
    now = fits & (fresh > 0)
    for j in range(width):
        row = now & (j < fresh)
        want[row, (held[row] + j).long()] = pool[(upto - fresh + j)[row]]
    want_used = used.clone()
    want_used[r[ended & (held > 0)]] = 0
    want_used[pool[:int(upto[now].max())].long()] = 1
    count = torch.tensor([available], dtype=torch.int32, device="cuda")
    blocks, cells = eb.block_tables(lengths, held, tables, pool, count, block=block, used=used, terminated=ended)
    assert torch.equal(tables, want) and torch.equal(used, want_used)
    assert torch.equal(blocks.long(), torch.where(ended, 0, torch.where(fits, torch.maximum(need, held), held)))
    assert cells.tolist() == [int(upto[now].max()), int((~fits).sum())] and cells[1] > 0

    new = torch.where(ended, 0, r % 5)
    total, capacity = int(new.sum()), int(new.sum()) + 9
    got = eb.slot_map(tables, blocks, (r % 5).int(), capacity, block=block, held=blocks, terminated=ended)
    owner = torch.repeat_interleave(r, new)
    offsets = torch.cat((new.new_zeros(1), torch.cumsum(new, 0)))
    position = blocks[owner] + torch.arange(total, device="cuda") - offsets[owner]
    column = position // block
    entry = torch.where(column < blocks[owner], tables[owner, column.clamp(max=width - 1)].long(), -1)
    assert torch.equal(got[0][:total], torch.where(entry < 0, -1, entry * block + position % block))
    assert torch.equal(got[1][:total].long(), position) and torch.equal(got[2][:total].long(), owner)
    assert got[0][total:].eq(-1).all() and got[1][total:].eq(0).all() and got[2][total:].eq(-1).all()
    assert torch.equal(got[3].long(), offsets)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_the_widest_rows(eb, dtype):
    """2^24 values a row, and one less, which lies on no words; whole numbers, so that every sum is exact."""
    for dim in (2**24, 2**24 - 1):
        table = torch.randint(-4, 5, (2, dim), device="cuda").to(dtype)
        ids = torch.tensor([1, -1, 0], device="cuda")
        got = eb.embedding(table, ids, scale=2.0)
        assert torch.equal(got[0], 2 * table[1]) and torch.equal(got[2], 2 * table[0]) and not got[1].any()
        ids = torch.tensor([0] * 3 + [1] * 30 + [2] * 2 + [0] * 165, device="cuda")
        got = eb.embedding_grad(table[1].expand(200, dim), ids, 3, dtype=torch.float32)
        for row, n in enumerate((168, 30, 2)):
            assert torch.equal(got[row], n * table[1].float())


def test_gradient_wait_gives_up_past_one_cluster(eb):
    """The same where the sort takes several kernels and the call zeroes its workspace by a memset: chunks of 64."""
    import ctypes

    from eagle_b200 import _abi

    n, dim = 140001, 512
    ids = torch.arange(n, device="cuda") // 3
    rows = int(ids[-1]) + 1
    grad = torch.ones(n, dim, dtype=torch.bfloat16, device="cuda")
    call = eb.EmbeddingGrad(grad, ids, rows)
    d = _abi.new(_abi.EmbeddingDesc)
    ctypes.memmove(ctypes.byref(d), ctypes.byref(call._desc), ctypes.sizeof(d))
    d.stream = torch.cuda.current_stream().cuda_stream
    _abi.check(_abi.lib().eagle_backend_x_b200_embedding_grad_wait_check(ctypes.byref(d), 1024, 1))
    torch.cuda.synchronize()
    lost = torch.zeros(rows, dtype=torch.bool, device="cuda")
    lost[1:22] = True  # positions 4 to 65: the run that starts at 63 is summed where it starts
    assert torch.equal(call.out.isnan().all(1), lost) and bool((call.out[~lost] == 3.0).all())
    with pytest.raises(eb.BackendError, match="wait"):
        call.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    call.check(side)
    assert bool((call.out == 3.0).all())
