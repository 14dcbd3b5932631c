"""The paged cache where its calls meet one another's state and incomplete books: shared pages, lists
that name what is not there, tables with holes, values that are not finite, weights of many small
parts, streams. Tolerances of outputs are those of test_gpu_pages.py, derived there."""

import math

import pytest

from aero_b200 import native_cuda as nc
from test_gpu_pages import close, join, open_cache, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda").reshape(-1)


# ------------------------------------------------------------------ books
@pytest.mark.parametrize("D,shift", [(64, 0), (64, 1), (128, 0)])
def test_append_leaves_shared_pages_alone(D, shift):
    """Rows for a full page that a fork shares are skipped, with a code; rows for the sequences' own
    pages, in the same call, are written; when the last but one holder is gone, so is the refusal."""
    from aero_b200.pages import PagedCache
    c = PagedCache(2, 12, 8, 2, D, 3, 4, dtype=F16)
    c.k().normal_()
    c.v().normal_()
    c.extend(i32([0]), i32([19]))  # two full pages and three rows of a third
    c.fork(i32([0]), i32([1]))
    c.extend(i32([0, 1]), i32([1, 1]))
    c.check()
    table = c.tables()[0].tolist()
    assert table[0][:2] == table[1][:2] and table[0][2] != table[1][2]
    k, v = (torch.randn((4, 2, D + shift), device="cuda").to(F16)[..., shift:] for _ in range(2))
    seqs, pos = [0, 1, 0, 1], [3, 15, 19, 19]
    want = c.k().clone(), c.v().clone()
    for t in (2, 3):
        for w, x in zip(want, (k, v)):
            w[1, table[seqs[t]][2], :, 3] = x[t]
    c.append(1, k, v, i32(seqs), i32(pos))
    assert c.status() == 8
    assert torch.equal(c.k(), want[0]) and torch.equal(c.v(), want[1])
    c.free(i32([1]))
    c.append(1, k[:1], v[:1], i32([0]), i32([3]))
    c.check()
    assert torch.equal(c.k(1)[table[0][0], :, 3], k[0]) and torch.equal(c.v(1)[table[0][0], :, 3], v[0])


@pytest.mark.parametrize("n", [3, 256, 257, 1200])
def test_free_of_a_bad_list_changes_nothing(n):
    """Lists with a number outside the cache, or one twice, on both sides of the length that takes a
    check of its own."""
    from aero_b200.pages import PagedCache
    c = PagedCache(1, 2 * n, 8, 1, 64, n, 3, dtype=F16)
    c.extend(i32(range(n)), i32([1 + s % 16 for s in range(n)]))
    before = [t.clone() for t in c.tables()]
    for bad in ([n] + list(range(1, n)), list(range(n - 1)) + [-1], list(range(n - 1)) + [0], [1, 1], [n]):
        c.free(i32(bad))
        assert c.status() == 1, bad[:3]
        assert all(torch.equal(x, y) for x, y in zip(before, c.tables()))
    c.free(i32(range(n - 1, -1, -1)))
    c.check()
    table, length, refs = c.tables()
    assert (table == -1).all() and not length.any() and not refs.any()


# ------------------------------------------------------------------ values that are not finite
def poke(c, which, j, value, columns=slice(None), seq=0):
    """Position j of a sequence: `columns` of its row in every kv head set to a value."""
    P = c.page_size
    which[int(c.tables()[0][seq, j // P]), :, j % P, columns] = value


def test_value_that_all_later_rows_see_costs_no_more():
    """A long prompt whose first V row is not finite in three columns: those columns of every row are
    not finite either, the others come out to the bit, in about the same time."""
    T, H, HK, D = 4096, 32, 4, 128
    c, _, _ = open_cache([T], 64, HK, D, F16)
    q = (2 * torch.randn((T, H, D), device="cuda")).half()
    out = torch.empty_like(q)

    def timed():
        best = math.inf
        for _ in range(4):
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            c.attend(0, q, i32([0]), start, out=out)
            e1.record()
            torch.cuda.synchronize()
            best = min(best, e0.elapsed_time(e1))
        return best, out.clone()

    start = i32([0, T])
    clean, want = timed()
    poke(c, c.v(0), 0, math.nan, slice(5, 8))
    took, got = timed()
    c.check()
    assert torch.isnan(got[..., 5:8]).all()
    assert torch.equal(got[..., :5], want[..., :5]) and torch.equal(got[..., 8:], want[..., 8:])
    assert took < 3 * clean, (took, clean)


@pytest.mark.parametrize("n,T,P,HK,G,D,dtype,window,sinks,bad", [
    (500, 300, 16, 2, 3, 64, F16, 0, 0, [0, 250, 333, 499]),
    (500, 300, 64, 1, 8, 128, BF16, 0, 0, [201, 202, 203, 320, 450]),
    (900, 400, 16, 2, 4, 128, F16, 130, 5, [2, 4, 5, 480, 600, 633, 764]),
    (900, 300, 8, 1, 2, 192, BF16, 100, 129, [128, 129, 501, 700, 801, 802]),
    (700, 200, 32, 1, 5, 256, F16, 0, 0, [499, 500, 620, 699]),
    (4000, 40, 64, 1, 4, 64, BF16, 0, 0, [100, 3970, 3999]),    # split over CTAs and joined
    (3000, 260, 16, 1, 1, 256, F16, 700, 40, [39, 40, 2050, 2100, 2800, 2999])])
def test_rows_beside_values_that_are_not_finite(n, T, P, HK, G, D, dtype, window, sinks, bad):
    """V rows not finite in some columns, seen by some rows of a tile and not by others: a row that
    does not see them comes out as without them, one that does has no finite value there alone."""
    c, K, V = open_cache([n], P, HK, D, dtype)
    q = (2 * torch.randn((T, HK * G, D), device="cuda")).to(dtype)
    columns = [d for d in range(D) if d % 7 == 3]
    for i, j in enumerate(bad):
        poke(c, c.v(0), j, (math.inf, math.nan, -math.inf)[i % 3], columns)
    got = c.attend(0, q, i32([0]), i32([0, T]), window=window, sinks=sinks)
    c.check()
    pos = [n - T + t for t in range(T)]
    sees = [any(j <= p and (not window or j > p - window or j < sinks) for j in bad) for p in pos]
    pick = sorted({t for j in bad for t in range(j - n + T - 3, j - n + T + 4)} |
                  {t for j in bad for t in range(j - n + T + window - 3, j - n + T + window + 4)} | set(range(0, T, 41)))
    pick = [t for t in pick if 0 <= t < T]
    ref = reference(q[pick], K[0], V[0], [pos[t] for t in pick], window, sinks, 1 / math.sqrt(D))
    some = torch.tensor([sees[t] for t in pick], device="cuda")
    fine = torch.ones(D, dtype=torch.bool, device="cuda")
    fine[columns] = False
    mine = got[pick]
    assert not torch.isfinite(mine[some][..., ~fine]).any()
    close(mine[..., fine], tuple(x[..., fine] for x in ref), dtype)
    if not all(sees[t] for t in pick):
        close(mine[~some], tuple(x[~some] for x in ref), dtype)
    assert torch.equal(got.nan_to_num(0, 1, -1), c.attend(0, q, i32([0]), i32([0, T]), window=window, sinks=sinks).nan_to_num(0, 1, -1))


@pytest.mark.parametrize("window,sinks", [(100, 2**31 - 1), (2**31 - 1, 3), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1)])
def test_largest_windows_and_sinks_beside_bad_values(window, sinks):
    """As many first tokens or as wide a window as 32 bits hold: plain causal attention, also where rows
    are computed again."""
    c, K, V = open_cache([500], 16, 1, 64, F16)
    q = torch.randn((300, 4, 64), device="cuda").half()
    poke(c, c.v(0), 333, math.inf)
    want = c.attend(0, q, i32([0]), i32([0, 300]))
    got = c.attend(0, q, i32([0]), i32([0, 300]), window=window, sinks=sinks)
    c.check()
    pick = [0, 5, 130, 131, 132]
    close(got[pick], reference(q[pick], K[0], V[0], [200 + t for t in pick], 0, 0, 0.125), F16)
    assert not torch.isfinite(got[133:]).any() and not torch.isfinite(want[133:]).any()
    one = c.attend(0, q[:1], i32([0]), window=window, sinks=sinks)
    assert not torch.isfinite(one).any()


# ------------------------------------------------------------------ tables with holes
def holes(c, pages, seq=0):
    """The books with these places of a sequence's row empty, as a keeper of books elsewhere may have them."""
    table, length, refs = (t.clone() for t in c.tables())
    for i in pages:
        refs[int(table[seq, i])] -= 1
        table[seq, i] = -1
    c.set_tables(table, length, refs)


@pytest.mark.parametrize("P,T,window,sinks", [(16, 60, 100, 5), (8, 40, 33, 0), (64, 100, 70, 64), (128, 300, 200, 0), (16, 20, 100, 5)])
@pytest.mark.parametrize("D", [64, 192])
def test_pages_before_the_window_need_not_be_there(P, T, window, sinks, D):
    """A sequence that gave up the pages that its new tokens no longer see: no code, the same bits."""
    n = 900
    c, K, V = open_cache([n], P, 1, D, F16)
    q = torch.randn((T, 4, D), device="cuda").half()
    ask = [(q, i32([0]), i32([0, T])), (q[-1:], i32([0]))]
    want = [c.attend(0, *x, window=window, sinks=sinks) for x in ask]
    first = (n - T - window + 1) // P  # the first page that a token's window reaches
    holes(c, range(-(-sinks // P), first))
    got = [c.attend(0, *x, window=window, sinks=sinks) for x in ask]
    c.check()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("P,D,dtype,window", [(8, 64, F16, 0), (16, 128, BF16, 0), (64, 128, F16, 300), (128, 192, F16, 0), (256, 256, BF16, 0)])
def test_visible_positions_without_a_page_count_as_zeros(P, D, dtype, window):
    """In both forms, beside other sequences and after calls that left other rows in the CTAs' memory:
    the result with zeros there, and the code."""
    n, T, HK = 700, 120, 2
    c, K, V = open_cache([n, 300], P, HK, D, dtype)
    q = (2 * torch.randn((T, 2 * HK, D), device="cuda")).to(dtype)
    gone = [0, 1, (n - 1) // P] if P < 128 else [1, (n - 1) // P]
    holes(c, gone)
    K, V = K[0].clone(), V[0].clone()
    for i in gone:
        K[i * P:(i + 1) * P] = 0
        V[i * P:(i + 1) * P] = 0
    c.status()
    many = c.attend(0, q, i32([0, 1]), i32([0, T, T]), window=window)
    assert c.status() == 5
    one = c.attend(0, q[:2], i32([0, 1]), window=window)
    assert c.status() == 5
    pick = [0, 1, 31, 60, T - 2, T - 1]
    sc = 1 / math.sqrt(D)
    close(many[pick], reference(q[pick], K, V, [n - T + t for t in pick], window, 0, sc), dtype)
    close(one[:1], reference(q[:1], K, V, [n - 1], window, 0, sc), dtype)
    # and where a value that is not finite lies beside them
    j = n - 40 if (n - 40) // P not in gone else (n - 1) // P * P - 10
    poke(c, c.v(0), j, math.inf)
    many = c.attend(0, q, i32([0, 1]), i32([0, T, T]), window=window)
    pick = [t for t in (0, 5, j - n + T - 2, j - n + T - 1) if 0 <= t < j - n + T]
    if pick:
        close(many[pick], reference(q[pick], K, V, [n - T + t for t in pick], window, 0, sc), dtype)


# ------------------------------------------------------------------ many small weights
@pytest.mark.parametrize("form", ["one", "many", "tiles", "beside"])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, F16), (256, F16), (64, BF16)])
def test_many_small_weights_are_not_lost(form, D, dtype):
    """65535 positions, each of 2^-25.2 of the weight of one: together 0.17 % of all. All V rows are 1
    but that one's, which is 0, so the output is their share. Tolerance: the weights' rounding in the
    cache's type u = 2^-11 (f16) or 2^-8 (bf16), the same for the output, and 2^-14 for f32 scores,
    exponentials and sums, all relative to the output."""
    from aero_b200.pages import PagedCache
    n, P, T = 65536, 256, {"one": 1, "many": 5, "tiles": 64, "beside": 64}[form]
    c = PagedCache(1, n // P, P, 1, D, 1, n // P, dtype=dtype)
    c.extend(i32([0]), i32([n]))
    c.v().fill_(1.0)
    score = torch.tensor(25.2 * math.log(2), dtype=dtype, device="cuda")
    page = int(c.tables()[0][0, 11])  # the heavy one somewhere in the first tiles
    c.k(0)[page, 0, 77, 0] = score
    c.v(0)[page, 0, 77] = 0.0
    q = torch.zeros((T, 2, D), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    if form == "beside":  # rows beside a value that is not finite, computed again
        poke(c, c.v(0), n - 1, math.inf)
    out = c.attend(0, q, i32([0]), None if form == "one" else i32([0, T]), scale=1.0)
    c.check()
    if form == "beside":
        out = out[:-1]
    seen = torch.arange(n - T, n, device="cuda", dtype=torch.float64)[:out.shape[0]]  # light ones that a row sees
    want = (seen / (seen + torch.exp(score.double())))[:, None, None].expand(out.shape)
    assert 0.001 < float(want.min()) < 0.002
    u = 2.0**-11 if dtype == F16 else 2.0**-8
    assert ((out.double() - want).abs() <= (2 * u + 2.0**-14) * want).all(), float((out.double() / want - 1).abs().max())


@pytest.mark.parametrize("G", [1, 8, 16])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, F16), (192, F16), (256, BF16)])
def test_single_tokens_are_as_exact_as_their_type(D, dtype, G):
    """Token by token, weights lose nothing that the output's type could show. Tolerance: the output's own
    rounding u|o| (u = 2^-11 in f16, 2^-8 in bf16), the weights' two values u^2 sum w|v|, and 2^-14 sum w|v|
    for f32 scores, exponentials and sums."""
    lens = [3000, 200, 64, 1]
    c, K, V = open_cache(lens, 32, 2, D, dtype)
    q = torch.randn((len(lens), 2 * G, D), device="cuda").to(dtype)
    u = 2.0**-11 if dtype == F16 else 2.0**-8
    few = c.attend(0, q[:3], i32([0, 1]), i32([0, 2, 3]))
    for got, refs in (
            (c.attend(0, q, i32(range(4))), [reference(q[s:s + 1], K[s], V[s], [lens[s] - 1], 0, 0, 1 / math.sqrt(D)) for s in range(4)]),
            (few, [reference(q[:2], K[0], V[0], [2998, 2999], 0, 0, 1 / math.sqrt(D)),
                   reference(q[2:3], K[1], V[1], [199], 0, 0, 1 / math.sqrt(D))])):
        out, mag, _ = join(refs)
        tol = u * out.abs() + (u * u + 2.0**-14) * mag + 2.0**-25
        err = (got.double() - out).abs()
        assert (err <= tol).all(), f"worst {float((err / tol).max()):.3f} of the tolerance"
    c.check()


# ------------------------------------------------------------------ streams
def test_capture_on_a_blocking_stream_after_the_default_one():
    """A stream of cudaStreamCreate, which waits for the default stream and the other way round, captured
    when the cache last ran on the default stream; then calls there again."""
    import ctypes
    raw = ctypes.c_void_p()
    assert int(torch.cuda.cudart().cudaStreamCreate(ctypes.addressof(raw))) == 0
    s = torch.cuda.ExternalStream(raw.value)
    c, K, V = open_cache([100, 40], 16, 2, 64, F16)
    q, seqs = torch.randn((2, 4, 64), device="cuda").half(), i32([0, 1])
    want = c.attend(0, q, seqs)
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.attend(0, q, seqs, out=out)
    g.replay()
    assert torch.equal(out, want) and torch.equal(c.attend(0, q, seqs), want)
    c.check()
    torch.cuda.synchronize()


def test_explicit_stream_and_back():
    """set_stream with a torch stream and with a raw one: calls run there whatever torch's current stream
    is, behind what the cache did before; None follows torch's again."""
    c, K, V = open_cache([100, 40], 16, 2, 64, F16)
    q, seqs = torch.randn((2, 4, 64), device="cuda").half(), i32([0, 1])
    k, v = (torch.randn((2, 2, 64), device="cuda").half() for _ in range(2))
    one, pos = i32([1, 1]), i32([100, 40])
    out = torch.empty_like(q)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(int(4e8))  # the cache's calls below wait for this one's stream
        c.extend(seqs, one)
    c.set_stream(b)
    c.append(0, k, v, seqs, pos)
    busy = not b.query()
    c.set_stream(a.cuda_stream)
    c.attend(0, q, seqs, out=out)
    a.synchronize()
    assert busy
    want = join([reference(q[i:i + 1], torch.cat([K[i], k[i:i + 1]]), torch.cat([V[i], v[i:i + 1]]), [n], 0, 0, 0.125)
                 for i, n in enumerate((100, 40))])
    close(out, want, F16)
    c.set_stream(None)
    assert torch.equal(c.attend(0, q, seqs), out)
    c.check()


def test_every_call_in_a_capture():
    """One graph of all calls (which a call that allocated or synchronised would end), the split form of
    attend among them, replayed on new data; eager calls on a twin give the same books, pages and outputs."""
    from aero_b200.logits import adjust
    from aero_b200.pages import PagedCache

    def setup(seed):
        c = PagedCache(1, 80, 16, 1, 128, 6, 40, dtype=F16)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        c.k().normal_(generator=g)
        c.v().normal_(generator=g)
        c.extend(i32([0, 1]), i32([600, 37]))
        return c

    q = torch.randn((40, 8, 128), device="cuda").half()
    k = torch.randn((3, 1, 128), device="cuda").half()
    x = torch.randn((2, 1000), device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)] + [torch.zeros_like(q[:3]), torch.zeros_like(x)]
    ids = {n: i32(v) for n, v in dict(s=[0, 1], n=[1, 1], rs=[0, 1, 0], rp=[600, 37, 599], par=[0, 1], kid=[2, 3], gone=[1, 3],
                                       start=[0, 36, 40], src=[0], dst=[79], three=[0, 2, 0]).items()}
    hist, hn = i32(range(20)).reshape(2, 10), i32([10, 4])

    def step(c, outs):
        c.extend(ids["s"], ids["n"])
        c.append(0, k, k, ids["rs"], ids["rp"])
        c.attend(0, q, ids["s"], ids["start"], out=outs[0])
        c.fork(ids["par"], ids["kid"])
        c.attend(0, q, ids["s"], ids["start"], window=100, sinks=3, out=outs[1])
        c.free(ids["gone"])
        c.copy(ids["src"], ids["dst"])
        c.compact()
        c.attend(0, q[:3], ids["three"], out=outs[2])
        adjust(x, history=hist, n_history=hn, repetition=rep, out=outs[3])

    rep = torch.full((2,), 1.5, device="cuda")
    step(setup(0), [o.clone() for o in outs])  # kernels loaded
    c, twin = setup(1), setup(1)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(c, outs)
    q.normal_()
    k.normal_()
    x.normal_()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    mine = [o.clone() for o in outs]
    step(twin, outs)
    assert all(torch.equal(a, b) for a, b in zip(mine, outs)) and mine[0].abs().max() > 0
    assert all(torch.equal(a, b) for a, b in zip(c.tables(), twin.tables()))
    assert torch.equal(c.k(), twin.k()) and torch.equal(c.v(), twin.v())
    c.check()
    twin.check()
