"""The 8-bit key/value cache where it meets the unusual: blocks of zeros, scattered NaN values, lengths beyond the block table, ragged
batches with sums, long sums, malformed calls. Against float64 forms, with the tolerances that ``test_kv8`` derives."""
import math

import pytest
import torch

from legion_b200 import ops
from test_kv8 import NAN, WHERE, attend, cum, filled, gen, gpu, i32, near, on, randn, status, tables


def call(device, q, cache, table, lens, new, scale, **more):
    more = {k: v.to(device) if isinstance(v, torch.Tensor) and k == "sink" else v for k, v in more.items()}
    return ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), scale, **more)


def holding(k, v, page, device, seed=0):
    """A cache with one sequence of these rows, its table."""
    n, heads = k.shape[:2]
    table, blocks = tables([n], page, seed)
    cache = ops.Kv8Cache.empty(blocks, page, heads, k.shape[2], v.shape[2])
    ops.kv8_append(cache, k.bfloat16(), v.bfloat16(), i32(table), i32([n]), i32([0, n]), n)
    return on(cache, device), table


# ----------------------------------------------------------------------------------------------- value blocks of zeros
def near_sums(got, start, weight, off):
    want, tol = weight.sum(2), off.sum(2)
    assert bool(((got.cpu().double() - start.double() - want).abs() <= tol + 2.0 ** -23 * (start.double() + want)).all())


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size", [0, -13, -20, -24, -50])
@pytest.mark.parametrize("form", ["plain", "sink"])
def test_zero_values_beside_small_ones(device, new, size, form):
    """A block whose values are all zero has the scale 0. It adds to the denominator and takes nothing from the bits of the others,
    however small they are."""
    n, heads, kv, D = 256, 8, 2, 64
    v = randn(n, kv, D, seed=2) * 2.0 ** size
    v[32:48] = 0
    cache, table = holding(randn(n, kv, D, seed=1), v, 16, device)
    assert not bool(cache.v_scale[table[0][2]].any())
    q, more = randn(new, heads, D, seed=3).bfloat16(), {"sink": randn(heads, seed=4)} if form == "sink" else {}
    want, tol, weight, off = attend(q, cache, table, [n], [new], 0.125, **more)
    start = torch.rand(1, kv, n, generator=gen(5))
    w = start.clone().to(device)
    near(call(device, q, cache, table, [n], [new], 0.125, weights=w, **more), want, tol)
    near_sums(w[0], start[0], weight[0], off[0])
    assert status(device) == 0


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sink", [False, True])
def test_nothing_but_zero_values(device, new, sink):
    n, heads, kv, D = 300, 4, 2, 32
    cache, table = holding(randn(n, kv, D, seed=1), torch.zeros(n, kv, D), 32, device)
    q, more = randn(new, heads, D, seed=3).bfloat16(), {"sink": randn(heads, seed=4)} if sink else {}
    _, _, weight, off = attend(q, cache, table, [n], [new], 0.2, **more)
    w = torch.zeros(1, kv, n, device=device)
    assert not bool(call(device, q, cache, table, [n], [new], 0.2, weights=w, **more).any())
    near_sums(w[0], torch.zeros(kv, n), weight[0], off[0])
    assert status(device) == 0


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("sharp", [1.0, 30.0])
def test_prompt_far_apart_scales(device, sharp):
    """Rows of a prompt over blocks whose values differ by 2^40."""
    n, new = 300, 50
    v = randn(n, 1, 64, seed=2) * torch.exp2(torch.linspace(-30, 10, n).round())[torch.randperm(n, generator=gen(3))].view(n, 1, 1)
    cache, table = holding(randn(n, 1, 64, seed=1), v, 16, device)
    q = randn(new, 8, 64, seed=5).mul(sharp).bfloat16()
    want, tol, _, _ = attend(q, cache, table, [n], [new], 0.125)
    near(call(device, q, cache, table, [n], [new], 0.125), want, tol)


# ---------------------------------------------------------------------------------------------------- NaN values in prompts
NANS = [  # page, heads, kv heads, dk, dv, length, new, window, {(position, column)}
    (64, 8, 1, 128, 128, 600, 600, 0, [(10, 0), (481, 7), (500, 5), (505, 0)]),
    (64, 8, 1, 128, 128, 600, 600, 100, [(385, 3), (500, 3), (500, 5), (20, 9)]),
    (16, 16, 2, 256, 256, 400, 90, 0, [(5, 255), (330, 0), (399, 200)]),
    (16, 16, 2, 256, 256, 400, 90, 40, [(290, 17), (350, 17), (330, 255), (371, 255)]),
    (8, 6, 2, 64, 176, 300, 300, 33, [(t, (7 * t) % 176) for t in range(0, 300, 9)]),
    (32, 10, 1, 80, 48, 260, 260, 7, [(t, 3) for t in range(0, 260, 20)] + [(100, c) for c in range(48)]),
    (64, 8, 2, 64, 64, 3000, 20, 0, [(3, 1), (1500, 1), (2990, 2), (2999, 63)]),
    (64, 8, 2, 64, 64, 3000, 20, 1100, [(1882, 1), (1890, 33), (2400, 2), (2990, 33)]),
    (64, 4, 2, 192, 64, 200, 30, 1, [(171, 4), (180, 5), (199, 6)]),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,kv,dk,dv,n,new,window,nans", NANS)
def test_prompt_nan_values_reach_the_rows_that_see_them(device, page, heads, kv, dk, dv, n, new, window, nans):
    """Several NaN values: a row is NaN in the columns of those it sees, and in no others."""
    cache, table = filled([n], page, kv, dk, dv, seed=6, device=device)
    for t, c in nans:
        cache.v.view(torch.uint8)[table[0][t // page], kv - 1, t % page, c] = NAN
    q = randn(new, heads, dk, seed=7).bfloat16()
    want, tol, _, _ = attend(q, cache, table, [n], [new], dk ** -0.5, window=window)
    assert bool(want.isnan().any()) and not bool(want.isnan().all())
    near(call(device, q, cache, table, [n], [new], dk ** -0.5, window=window), want, tol)
    assert status(device) == 0


# ---------------------------------------------------------------------------------------------- lengths beyond the block table
@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("held,new,cells", [(0, 20, 16), (15, 5, 16), (16, 3, 16), (30, 20, 32), (40, 2, 32)])
def test_append_beyond_the_table_writes_rows_where_they_belong(device, held, new, cells):
    """Rows whose positions lie behind the table's last block are left out; the others go to their own cells."""
    page, D, blocks = 16, 32, cells // 16
    table = [list(range(1, blocks + 1))]
    caches = [ops.Kv8Cache.empty(5, page, 1, D, D, device) for _ in range(2)]
    x = randn(held + new, 1, D, seed=1).bfloat16().to(device)
    inside = min(held, cells)
    for c in caches:
        ops.kv8_append(c, x[:inside], x[:inside], i32(table, device), i32([inside], device), i32([0, inside], device), inside)
    ops.kv8_append(caches[0], x[held:], x[held:], i32(table, device), i32([held + new], device), i32([0, new], device), new)
    fit = max(0, min(held + new, cells) - held)
    if fit:
        ops.kv8_append(caches[1], x[held:held + fit], x[held:held + fit], i32(table, device), i32([held + fit], device), i32([0, fit], device), fit)
    for name in caches[0].__slots__:
        assert torch.equal(*(getattr(c, name).view(torch.uint8) for c in caches))
    assert status(device) == 0


@gpu
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("new", [[1, 1, 1], [10, 3, 30]])
def test_attention_beyond_the_table_is_recorded(window, new):
    """A sequence with more tokens than its table has blocks for is left out; the others of the call are not touched by it. (On the
    CPU the call is refused.)"""
    device, heads, D, lens = "cuda:0", 4, 64, [30, 65, 50]
    cache, table = filled(lens, 16, 2, D, D, seed=8, device=device)
    q = randn(sum(new), heads, D, seed=9).bfloat16()
    want, tol, weight, off = attend(q, cache, table, lens, new, 0.125, window=window)
    w, out = torch.full((3, 2, 70), 0.5, device=device), torch.full((sum(new), heads, D), 7.0, dtype=torch.bfloat16, device=device)
    short = i32([row[:4] for row in table], device)          # 64 cells
    ops.kv8_attention(q.to(device), cache, short, i32(lens, device), i32(cum(new), device), max(new), 0.125, window=window, weights=w, out=out)
    assert status(device) != 0
    mine = torch.ones(sum(new), dtype=torch.bool)
    mine[new[0]:new[0] + new[1]] = False
    near(out[mine.to(device)], want[mine], tol[mine])
    assert bool((out[~mine.to(device)] == 7.0).all()) and bool((w[1] == 0.5).all())
    for i in (0, 2):
        got = w[i, :, :lens[i]].cpu().double() - 0.5
        assert bool(((got - weight[i].sum(2)).abs() <= off[i].sum(2) + 2.0 ** -23 * (0.5 + weight[i].sum(2))).all())


def test_attention_and_eviction_beyond_the_table_are_refused_on_the_cpu():
    cache, table = filled([35], 16, 2, 32, 32)
    short, q, w = i32([table[0][:2]]), randn(1, 4, 32).bfloat16(), torch.zeros(1, 2, 40)
    with pytest.raises(ValueError, match="table"):
        ops.kv8_attention(q, cache, short, i32([35]), i32([0, 1]), 1, 0.2)
    with pytest.raises(ValueError, match="table"):
        ops.kv8_evict(cache, short, i32([35]), w, 16, i32([[0]]))
    with pytest.raises(ValueError, match="sums"):
        ops.kv8_evict(cache, i32(table), i32([35]), w[..., :30], 16, i32([[0]]))
    with pytest.raises(ValueError, match="sums"):
        ops.kv8_attention(q, cache, i32(table), i32([35]), i32([0, 1]), 1, 0.2, weights=w[..., :30])


# --------------------------------------------------------------------------------------------------------------- long sums
@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("n,heads", [(2600, 8), (1900, 16)])
def test_sums_of_many_equal_weights(device, n, heads):
    """A key that gets the same 0.88 from each of 20800 to 30400 rows and heads: additions that all round one way must not add up.
    Products of the scores are exact here; a weight is off by its exponent's rounding (scores of 12 and log-sum-exps in 32 bits,
    a step of 2^-20 each) and by the exponential's, together below 2^-18; 2^-17 is asked for."""
    D = 16
    k = torch.full((n, 1, D), -8.0)
    k[0], k[1] = 1.0, 0.75
    cache, table = holding(k, torch.ones(n, 1, D), 64, device)
    q = torch.ones(n, heads, D, dtype=torch.bfloat16)
    w = torch.zeros(1, 1, n, device=device)
    call(device, q, cache, table, [n], [n], 0.5, weights=w)
    # position 0 sees key 0 alone
    big = heads * (1 + (n - 1) / (1 + math.exp(-2)))
    small = heads * (n - 1) / (1 + math.exp(2))
    got = w[0, 0].cpu().double()
    assert abs(float(got[0]) / big - 1) <= 2.0 ** -17 and abs(float(got[1]) / small - 1) <= 2.0 ** -17
    assert status(device) == 0


# ------------------------------------------------------------------------------------------------- sums of ragged batches
RAGGED = [  # page, heads, kv heads, D, lengths, new tokens, observed rows
    (16, 8, 2, 64, [500] + [1] * 20, [500] + [1] * 20, 0),
    (64, 40, 8, 64, [30, 400, 3, 0, 77], [30, 130, 3, 0, 5], 0),
    (64, 40, 8, 64, [30, 400, 3, 0, 77], [30, 130, 3, 0, 5], 100),
    (32, 6, 2, 96, [1, 300, 1], [1, 300, 1], 7),
    (16, 5, 1, 160, [9] * 30 + [333], [9] * 30 + [260], 0),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,kv,D,lens,new,observe", RAGGED)
def test_sums_of_ragged_batches(device, page, heads, kv, D, lens, new, observe):
    cache, table = filled(lens, page, kv, D, D, seed=31, device=device)
    q = randn(sum(new), heads, D, seed=32).bfloat16()
    want_o, tol_o, weight, off = attend(q, cache, table, lens, new, D ** -0.5, window=200)
    start = torch.rand(len(lens), kv, max(lens), generator=gen(1))
    w = start.clone().to(device)
    near(call(device, q, cache, table, lens, new, D ** -0.5, window=200, weights=w, observe=observe), want_o, tol_o)
    assert status(device) == 0
    for i, (n, m) in enumerate(zip(lens, new)):
        rows = torch.arange(weight[i].shape[2]) % max(m, 1) >= (m - observe if observe else 0)
        want, tol = weight[i][:, :, rows].sum(2), off[i][:, :, rows].sum(2)
        got = w[i].cpu().double() - start[i].double()
        assert bool(((got[:, :n] - want).abs() <= tol + 2.0 ** -23 * (start[i, :, :n] + want)).all())
        assert not bool(got[:, n:].any())


@gpu
@pytest.mark.parametrize("observe", [0, 64])
def test_sums_of_a_ragged_batch_take_scratch_by_its_rows(observe):
    """One long prompt beside 63 single tokens: 8255 rows of 8 heads a kv head, 17 KB for every 64 of them, not 64 times the longest."""
    device, lens = "cuda:0", [8192] + [1] * 63
    cache, table = filled(lens, 64, 4, 64, 64, seed=3, device=device)
    q = randn(sum(lens), 32, 64, seed=4).bfloat16().to(device)
    w = torch.zeros(64, 4, 8192, device=device)
    args = (q, cache, i32(table, device), i32(lens, device), i32(cum(lens), device), 8192, 0.125)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.kv8_attention(*args, weights=w, observe=observe)
    # records of both codings of the rows (256 bytes a row and head of 128 columns, 16 for its scale, log-sum-exp and position), the
    # output, log-sum-exps, and one record of 64 rows more for every sequence and head
    rows = (sum(lens) if observe == 0 else min(sum(lens), 64 * observe)) * 32
    assert torch.cuda.max_memory_allocated() - before <= 2 * (rows * 272 + 64 * 4 * 64 * 272) + q.numel() * 2 + sum(lens) * 32 * 4 + (1 << 22)
    # softmax weights: every row and head gives 1
    total = float(w.double().sum())
    rows = [min(n, observe) if observe else n for n in lens]
    assert abs(total - 32 * sum(rows)) <= 2.0 ** -16 * 32 * sum(rows) and status(device) == 0


# --------------------------------------------------------------------------------------------------------- malformed calls
BAD = {  # what: change of the call's arguments
    "queries of two dimensions": lambda a: a.update(q=a["q"][0]),
    "keys of three dimensions": lambda a: setattr(a["cache"], "k", a["cache"].k[0]),
    "values of three dimensions": lambda a: setattr(a["cache"], "v", a["cache"].v[0]),
    "a cache without heads": lambda a: [setattr(a["cache"], n, getattr(a["cache"], n)[:, :0]) for n in a["cache"].__slots__],
    "a table of one dimension": lambda a: a.update(table=a["table"][0]),
    "no query heads": lambda a: a.update(q=a["q"][:, :0]),
    "head size": lambda a: a.update(q=a["q"][..., :16]),
}


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("what", list(BAD))
def test_malformed_calls_are_value_errors(device, new, what):
    cache, table = filled([20], 16, 2, 32, 32, device=device)
    a = dict(cache=cache, q=randn(new, 4, 32).bfloat16().to(device), table=i32(table, device))
    BAD[what](a)
    with pytest.raises(ValueError, match="kv8_attention"):
        ops.kv8_attention(a["q"], a["cache"], a["table"], i32([20], device), i32([0, new], device), new, 0.2)
    if "quer" not in what and what != "head size":
        with pytest.raises(ValueError, match="kv8_evict"):
            ops.kv8_evict(a["cache"], a["table"], i32([20], device), torch.zeros(1, 2, 20, device=device), 16, i32([[1]], device))


@gpu
def test_a_cache_and_rows_on_different_devices():
    device = "cuda:0"
    cache, table = filled([20], 16, 2, 32, 32, device=device)
    q, k, where = randn(1, 4, 32).bfloat16(), randn(1, 2, 32).bfloat16(), (i32(table), i32([20]), i32([0, 1]))
    with pytest.raises(ValueError, match="devices"):
        ops.kv8_attention(q, cache, *where, 1, 0.2)
    with pytest.raises(ValueError, match="devices"):
        ops.kv8_append(cache, k, k, *where, 1)
    with pytest.raises(ValueError, match="devices"):
        ops.kv8_evict(cache, *where[:2], torch.zeros(1, 2, 20), 16, i32([[1]]))


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("budget", [0, -1, 17, 1 << 45])
def test_budgets_are_checked_before_results_are_allocated(device, budget):
    cache, table = filled([20], 16, 2, 32, 32, device=device)
    with pytest.raises(ValueError, match="kv8_evict"):
        ops.kv8_evict(cache, i32(table, device), i32([20], device), torch.zeros(1, 2, 20, device=device), budget, i32([[1]], device))


# ---------------------------------------------------------------------------------------------------------------- launches
@gpu
@pytest.mark.parametrize("lens,new,sums", [([1000], [1], False), ([1000], [1], True), ([10], [1], True), ([3000], [5], False), ([3000], [5], True),
                                           ([200] * 60, [200] * 60, True)])
def test_launches_are_counted(lens, new, sums):
    """The launch counter against the kernels of the captured call."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    device = "cuda:0"
    cache, table = filled(lens, 64, 1, 64, 64, device=device)
    q = randn(sum(new), 4, 64).bfloat16().to(device)
    args = (q, cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), 0.125)
    w = torch.zeros(len(lens), 1, max(lens), device=device) if sums else None
    before = ops.sm100.LAUNCHES["n"]
    ops.kv8_attention(*args, weights=w)
    counted = ops.sm100.LAUNCHES["n"] - before
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        ops.kv8_attention(*args, weights=w)
    err, _, n = runtime.cudaGraphGetNodes(g.raw_cuda_graph())
    assert int(err) == 0 and n == counted


# ------------------------------------------------------------------------------------------------------------------- outputs
def test_output_rows_that_overlap_are_refused():
    if not ops.sm100.have_ext():
        pytest.skip("extension not built")
    cache, table = filled([20], 16, 2, 32, 32)
    C, st = ops.sm100.ext(), torch.zeros(4, dtype=torch.int32)
    q = randn(3, 4, 32).bfloat16()
    for out in (torch.zeros(1, 4, 32, dtype=torch.bfloat16).expand(3, 4, 32), torch.zeros(300, dtype=torch.bfloat16).as_strided((3, 4, 32), (64, 32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            C.kv8_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, i32(table), i32([20]), i32([0, 3]), 3, 0.1, 0, 0.0, None, 1,
                            out, st, None, 0, 1)


@gpu
@pytest.mark.parametrize("fault", ["length", "rows"])
def test_rows_that_are_left_out_stay_as_they_were(fault):
    """Where the keys of a prompt call are split, the join leaves the rows of a sequence that was left out alone, too."""
    device, heads, D, lens, new = "cuda:0", 4, 64, [1500, 1700, 0, 1200], [5, 9, 0, 2]
    cache, table = filled(lens, 16, 2, D, D, seed=8, device=device)
    q = randn(sum(new), heads, D, seed=9).bfloat16()
    want, tol, _, _ = attend(q, cache, table, lens, new, 0.125)
    most = 9 if fault == "length" else 8                     # (a sequence with more rows than the call allows)
    width = 100 if fault == "length" else len(table[0])      # (1600 cells)
    assert ops.kv8._prompt_splits(4, 2, most * 2, 256, 13) > 1
    out = torch.full((sum(new), heads, D), 7.0, dtype=torch.bfloat16, device=device)
    ops.kv8_attention(q.to(device), cache, i32([row[:width] for row in table], device), i32(lens, device), i32(cum(new), device), most, 0.125,
                      max_ctx=1700, out=out)
    assert status(device) != 0
    mine = torch.ones(sum(new), dtype=torch.bool)
    mine[5:14] = False
    near(out[mine.to(device)], want[mine], tol[mine])
    assert bool((out[~mine.to(device)] == 7.0).all())


@gpu
def test_captured_prompts_replayed_with_other_lengths():
    """Prompt rows with sums in a graph; lengths, rows and row bounds change between replays."""
    device, heads, kv, D = "cuda:0", 8, 2, 64
    plans = [([900, 400, 30], [20, 7, 30]), ([1000, 33, 64], [1, 33, 23]), ([57, 640, 1], [57, 0, 0])]
    cache, table = filled([1000, 640, 64], 16, kv, D, D, seed=5, device=device)
    T = 57
    q, cu, ctx = torch.zeros(T, heads, D, dtype=torch.bfloat16, device=device), i32([0, 0, 0, 0], device), i32([0, 0, 0], device)
    w, tab = torch.zeros(3, kv, 1000, device=device), i32(table, device)

    def body():
        return ops.kv8_attention(q, cache, tab, ctx, cu, T, 0.125, weights=w, observe=9, window=500)
    body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = body()
    for j, (lens, new) in enumerate(plans):
        rows = randn(T, heads, D, seed=50 + j).bfloat16()
        q.copy_(rows)
        cu.copy_(i32(cum(new)))
        ctx.copy_(i32(lens))
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        want, tol, weight, off = attend(rows[:sum(new)], cache, table, lens, new, 0.125, window=500)
        near(out[:sum(new)], want, tol)
        for i, (n, m) in enumerate(zip(lens, new)):
            last = torch.arange(weight[i].shape[2]) % max(m, 1) >= m - 9
            assert bool(((w[i, :, :n].cpu().double() - weight[i][:, :, last].sum(2)).abs() <= off[i][:, :, last].sum(2) + 2.0 ** -23 * weight[i].sum(2)).all())
    assert status(device) == 0


@gpu
def test_blocks_behind_4_gigabytes():
    """Offsets that pass 32 bits: everything in the last blocks of a cache of 4.6 GB of keys and as much of values, bit for bit as in a
    small one."""
    device, page, kv, heads, D, lens = "cuda:0", 64, 4, 8, 256, [300, 70]
    results = []
    for blocks in (30, 70000):
        cache = ops.Kv8Cache.empty(blocks, page, kv, D, device=device)
        top = blocks - 1
        table = i32([[top - 2 * j - i for j in range(5)] for i in range(2)], device)
        dst = i32([[top - 10 - 2 * j - i for j in range(2)] for i in range(2)], device)
        x = randn(sum(lens), kv, D, seed=1).bfloat16().to(device)
        ops.kv8_append(cache, x, x, table, i32(lens, device), i32(cum(lens), device), 300)
        got = []
        for new in ([1, 1], [40, 3]):
            q = randn(sum(new), heads, D, seed=2).bfloat16().to(device)
            w = torch.zeros(2, kv, 300, device=device)
            got += [ops.kv8_attention(q, cache, table, i32(lens, device), i32(cum(new), device), max(new), 0.06, weights=w), w]
        got += list(ops.kv8_evict(cache, table, i32(lens, device), w, 100, dst, 2, 30))
        ids = torch.cat([table.flatten(), dst.flatten()]).long()
        got += [t[ids] for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
        results.append(got)
        del cache
    assert status(device) == 0 and bool(results[0][0].float().abs().amax() > 0)
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [1, 40])
def test_zero_values_that_take_nearly_all_of_the_weight(device, new):
    """Keys with zero values 44 above the others in score: what is left of the others' weight, 2^-60, keeps its bits."""
    n, heads, D = 200, 8, 16
    k, v = randn(n, 1, D, seed=1) * 0.1, randn(n, 1, D, seed=2) * 2.0 ** -10
    k[32:48], v[32:48] = 5.5, 0
    cache, table = holding(k, v, 16, device)
    q = torch.ones(new, heads, D, dtype=torch.bfloat16)
    want, tol, _, _ = attend(q, cache, table, [n], [new], 0.5)
    assert 2.0 ** -90 < float(want.abs().max()) < 2.0 ** -60
    near(call(device, q, cache, table, [n], [new], 0.5), want, tol)
    assert status(device) == 0


@pytest.mark.parametrize("device", WHERE)
def test_lengths_below_zero_hold_nothing(device):
    cache, table = filled([20, 20], 16, 2, 32, 32, device=device)
    before, lens, x = on(cache, "cpu"), i32([-3, 20], device), randn(2, 2, 32).bfloat16().to(device)
    tab, cu = i32(table, device), i32([0, 1, 1], device)
    ops.kv8_append(cache, x, x, tab, lens, cu, 1)
    w = torch.rand(2, 2, 20, generator=gen(1)).to(device)
    kept = ops.kv8_evict(cache, tab, lens, w, 8, i32([[5], [6]], device))
    assert kept[0].tolist() == [0, 8] and bool((kept[1][0] == -1).all()) and not bool(kept[2][0].any())
    sums = w.clone()
    assert not bool(ops.kv8_attention(x[:1].repeat(1, 2, 1), cache, tab[:1], lens[:1], cu[:2], 1, 0.2, weights=w[:1]).any())
    assert torch.equal(w, sums) and status(device) == 0
    for n in cache.__slots__:
        assert torch.equal(getattr(before, n)[:6].view(torch.uint8), getattr(cache, n)[:6].cpu().view(torch.uint8))


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("n", [100, 1000])
def test_a_sink_that_takes_nearly_all_of_the_weight(device, new, n):
    """A sink 44 above every score, values of zero beside others: keys keep their 2^-60 of a weight."""
    heads, D = 8, 16
    k, v = torch.full((n, 1, D), -5.5), randn(n, 1, D, seed=2)
    v[32:48] = 0
    cache, table = holding(k, v, 16, device)
    q, sink = torch.ones(new, heads, D, dtype=torch.bfloat16), torch.zeros(heads)
    for lens, window in (([n], 0), ([n], 45), ([47], 5), ([47], 0)):      # (the last rows of 47 see zero values alone through a window of 5)
        want, tol, weight, off = attend(q, cache, table, lens, [new], 0.5, window=window, sink=sink)
        sums = torch.zeros(1, 1, n, device=device)
        near(call(device, q, cache, table, lens, [new], 0.5, window=window, sink=sink, weights=sums), want, tol)
        got, full, err = sums[0, 0, :lens[0]].cpu().double(), weight[0][0].sum(1), off[0][0].sum(1)
        assert float(full.max()) < 2.0 ** -50 and bool(((got - full).abs() <= err + 2.0 ** -23 * full).all())
    assert status(device) == 0
