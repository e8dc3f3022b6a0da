"""The 8-bit key/value cache: appending, attention, eviction, against float64 forms written from their definitions. On CPU the
reference ops, on a GPU the kernels.

Tolerances of the attention, fixed beforehand: an output of bf16 is off by 2^-8 of itself (its rounding) and by the error of the
probabilities times sum p |v|. A probability is off by 2^-9 (three e5m2 terms, or one half) and by the error of its score, twice
(numerator and denominator): queries split into 8-bit terms keep 2^-21 of the largest query value (prompts: 2^-17 of the row's), sums of D products in 32 bits
D 2^-23 of the sum of magnitudes, the soft cap 2^-19 of the cap. A key's weight, its probability times the scale of its values, is
also off by up to 2^-28 of the largest weight of its row: e5m2 ends at a step of 2^-16, half of it is lost at most, and the largest
weight lies at 2^11 or above."""
import math

import pytest
import torch

from legion_b200 import ops

gpu = pytest.mark.gpu
WHERE = [pytest.param("cpu", id="cpu"), pytest.param("cuda:0", id="gpu", marks=gpu)]
E4 = torch.float8_e4m3fn
NAN = 0x7F


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


def i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def cum(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def status(device):
    """The kernels' status word, cleared."""
    if device == "cpu":
        return 0
    torch.cuda.synchronize()
    return ops.sm100.Workspace.get(device).check()


def tables(lens, page, seed=0, spare=2):
    """Block table with blocks in random order (block 0 is nobody's) and the number of blocks."""
    per = [-(-n // page) for n in lens]
    order = (torch.randperm(sum(per), generator=gen(seed)) + 1).tolist()
    rows, at = [], 0
    for k in per:
        rows.append(order[at:at + k] + [0] * (max(per) - k + 1))
        at += k
    return rows, sum(per) + 1 + spare


def code_values():
    """Value of every e4m3 code, from the format: sign, 4 bits of exponent, 3 of mantissa, 0x7f and 0xff NaN."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(math.nan if (c & 127) == 127 else (-v if c & 128 else v))
    return torch.tensor(out, dtype=torch.float64)


CODES = code_values()


def decode(codes, scale):
    return CODES[codes.cpu().view(torch.uint8).long()] * scale.cpu().double()[:, :, None, None]


def encode(x):
    """float64 to the nearest code's value, ties to the even mantissa."""
    pos = CODES[:127]
    m = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(pos, m).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = m - pos[lo], pos[hi] - m
    idx = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(x.isnan(), x, torch.copysign(pos[idx], x))


def power(amax):
    if amax == 0:
        return 0.0
    return 2.0 ** max(math.frexp(amax)[1] - 1 - 7, -60)


class Oracle:
    """A cache in float64: code values and scales."""

    def __init__(self, n_blocks, heads, page, dk, dv):
        self.c = [torch.zeros(n_blocks, heads, page, d, dtype=torch.float64) for d in (dk, dv)]
        self.s = [torch.zeros(n_blocks, heads, dtype=torch.float64) for _ in range(2)]
        self.page = page

    def append(self, k, v, table, lens, new):
        cu, most = cum(new), torch.finfo(torch.bfloat16).max
        for x, c, s in zip((k, v), self.c, self.s):
            x = x.double().clamp(-most, most)
            for i, (n, m) in enumerate(zip(lens, new)):
                for b in range(max(0, n - m) // self.page, -(-n // self.page)):
                    lo, hi = max(n - m, b * self.page), min(n, (b + 1) * self.page)
                    if lo >= hi:
                        continue
                    blk = table[i][b]
                    for h in range(c.shape[1]):
                        rows = x[cu[i] + lo - (n - m):cu[i] + hi - (n - m), h]
                        if lo % self.page == 0:
                            c[blk, h], s[blk, h] = 0, 0
                        fin = rows[~rows.isnan()]
                        old = float(s[blk, h])
                        now = max(old, power(float(fin.abs().max()) if fin.numel() else 0.0))
                        if now != old or now == 0:
                            c[blk, h] = encode(c[blk, h] * (old / now if now else 0.0))
                        c[blk, h, lo % self.page:lo % self.page + hi - lo] = encode(rows / now if now else rows * 0.0)
                        s[blk, h] = now

    def same(self, cache):
        for c, s, codes, scale in zip(self.c, self.s, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            assert torch.equal(scale.cpu().double(), s)
            got = CODES[codes.cpu().view(torch.uint8).long()]
            assert torch.equal(got.nan_to_num(nan=1e9), c.nan_to_num(nan=1e9))


def attend(q, cache, table, lens, new, scale, window=0, softcap=0.0, sink=None):
    """(out, tolerance, weights [kv heads, keys, rows of the heads that share one] of every sequence, their tolerance) in float64."""
    k_all, v_all = decode(cache.k, cache.k_scale), decode(cache.v, cache.v_scale)
    page, kv = cache.k.shape[2], cache.k.shape[1]
    T, H, D = q.shape
    out, tol = torch.zeros(T, H, v_all.shape[3], dtype=torch.float64), torch.zeros(T, H, v_all.shape[3], dtype=torch.float64)
    off_w = [torch.zeros(kv, n, H // kv * m, dtype=torch.float64) for n, m in zip(lens, new)]
    weight = [torch.zeros(kv, n, H // kv * m, dtype=torch.float64) for n, m in zip(lens, new)]
    cu = cum(new)
    for i, (n, m) in enumerate(zip(lens, new)):
        if n == 0 or m == 0:
            continue
        blocks = table[i][:-(-n // page)]
        pos = torch.arange(n - m, n)[:, None]
        seen = torch.arange(n) <= pos
        if window:
            seen &= torch.arange(n) > pos - window
        for h in range(H):
            g = h // (H // kv)
            k, v = k_all[blocks, g].flatten(0, 1)[:n], v_all[blocks, g].flatten(0, 1)[:n]
            vs = cache.v_scale.cpu().double()[blocks, g].repeat_interleave(page)[:n]
            qh = q[cu[i]:cu[i + 1], h].double().cpu()
            s = qh @ k.T * scale
            most = (qh.abs().nan_to_num(0, 0, 0) @ k.abs().nan_to_num().T * scale)
            off = float(most.max()) * D * 2.0 ** -23 + 2.0 ** (-21 if max(new) == 1 else -17) * float(q[cu[i]:cu[i + 1]].abs().float().nan_to_num(0, 0, 0).max()) * float(k.abs().nan_to_num().sum(1).max()) * abs(scale)
            if softcap:
                s, off = softcap * torch.tanh(s / softcap), off + softcap * 2.0 ** -19
            s = s.masked_fill(~seen, -math.inf)
            if sink is not None:
                s = torch.cat([s, sink[h].double().cpu().expand(m, 1)], 1)
            p = torch.softmax(s, 1)[:, :n]
            p = torch.where(seen.any(1, keepdim=True), torch.where(seen, p, torch.zeros_like(p)), torch.zeros_like(p))
            for r in range(m):                      # NaN values only where they are seen
                at = seen[r]
                out[cu[i] + r, h] = p[r, at] @ v[at]
                least = 2.0 ** -28 * (p[r] * vs).nan_to_num(0, 0, 0).max() * (v / vs[:, None].clamp_min(1e-300))[at].abs().sum(0)
                tol[cu[i] + r, h] = out[cu[i] + r, h].abs() * 2.0 ** -8 + (2.0 ** -9 + 2 * off) * (p[r, at] @ v[at].abs()) + least
            weight[i][g, :, (h % (H // kv)) * m:(h % (H // kv) + 1) * m] = p.T
            off_w[i][g, :, (h % (H // kv)) * m:(h % (H // kv) + 1) * m] = (2 * off + 2.0 ** -20) * p.T
    return out, tol + 1e-30, weight, off_w


def near(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    bad = ((got - want).abs() > tol) & ~want.isnan()
    worst = ((got - want).abs() / tol).nan_to_num().max() if got.numel() else 0
    assert not bool(bad.any()), f"{int(bad.sum())} of {got.numel()} outside, worst {float(worst):.2f} of the tolerance"


def filled(lens, page, heads, dk, dv, seed=0, device="cpu", k=1.0):
    """A cache with sequences of these lengths (through the reference, on the CPU), its table and a float64 view of it."""
    table, n_blocks = tables(lens, page, seed)
    cache = ops.Kv8Cache.empty(n_blocks, page, heads, dk, dv)
    T = sum(lens)
    grow = torch.exp2(randn(T, heads, 1, seed=seed + 5))
    ops.kv8_append(cache, (randn(T, heads, dk, seed=seed + 1) * grow * k).bfloat16(), (randn(T, heads, dv, seed=seed + 2) * grow).bfloat16(),
                   i32(table), i32(lens), i32(cum(lens)), max(lens + [1]))
    return on(cache, device), table


def on(cache, device):
    return ops.Kv8Cache(*(getattr(cache, n).clone().to(device) for n in cache.__slots__))


# ----------------------------------------------------------------------------------------------------------- append
APPEND = [  # page, heads, dk, dv, steps of [(tokens of each sequence)]
    (16, 2, 64, 64, [[5, 0, 17], [1, 1, 1], [1, 0, 1], [40, 3, 16], [1, 29, 1]]),
    (64, 1, 128, 128, [[63], [1], [1], [200]]),
    (8, 3, 16, 48, [[1, 8], [7, 8], [1, 1]]),
    (64, 2, 256, 256, [[130, 1], [1, 1], [62, 63], [1, 1]]),
    (32, 4, 80, 192, [[33, 95, 2], [1, 1, 1]]),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,dk,dv,steps", APPEND)
def test_append(device, page, heads, dk, dv, steps):
    total = [sum(s) for s in zip(*steps)]
    table, n_blocks = tables(total, page, 3)
    cache, want = ops.Kv8Cache.empty(n_blocks, page, heads, dk, dv, device), Oracle(n_blocks, heads, page, dk, dv)
    lens = [0] * len(total)
    for j, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        T = sum(new)
        # magnitudes that grow from step to step and differ from token to token: scales move in blocks that hold tokens
        size = torch.exp2(randn(T, 1, 1, seed=j) * 2 + j)
        wide = (randn(T, heads * (dk + dv) + 8, seed=10 + j)).bfloat16().to(device)
        k, v = wide[:, :heads * dk].view(T, heads, dk), wide[:, heads * dk:heads * (dk + dv)].view(T, heads, dv)
        k, v = (k * size.to(device)).bfloat16(), (v * size.to(device)).bfloat16()
        if j % 2:           # rows apart, and not on 16 bytes
            wide = torch.zeros(T, heads * (dk + dv) + 9, dtype=torch.bfloat16, device=device)
            wide[:, 1:1 + heads * dk], wide[:, 1 + heads * dk:-8] = k.reshape(T, -1), v.reshape(T, -1)
            k, v = wide[:, 1:1 + heads * dk].view(T, heads, dk), wide[:, 1 + heads * dk:-8].view(T, heads, dv)
        ops.kv8_append(cache, k, v, i32(table, device), i32(lens, device), i32(cum(new), device), max(new))
        want.append(k.cpu(), v.cpu(), table, lens, new)
        assert status(device) == 0
        want.same(cache)


@pytest.mark.parametrize("device", WHERE)
def test_append_values_at_the_edges(device):
    """Zeros, the smallest and largest values, infinities, NaN; a block that was somebody else's."""
    page, D = 16, 32
    x = torch.zeros(48, 1, D)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, 1.0, 3e38])
    x[16, 0, :3] = torch.tensor([1e-30, -1e-38, 2e-25])
    x[20, 0, 5] = math.nan
    x[32, 0, :8] = torch.tensor([1.0, 255.0 / 256, 2.0 ** -14, 3 * 2.0 ** -15, 2.0 ** -17, 2.0 ** -18, -2.0 ** -16, 0.0])
    x = x.bfloat16()
    cache, want = ops.Kv8Cache.empty(5, page, 1, D, D, device), Oracle(5, 1, page, D, D)
    cache.k.view(torch.uint8).fill_(NAN)                      # blocks hold what was there before
    cache.k_scale.fill_(4.0)
    want.c[0].fill_(math.nan)
    want.s[0].fill_(4.0)
    args = ([[3, 1, 2]], [40], [40])
    ops.kv8_append(cache, x[:40].to(device), x[:40].to(device), *(i32(a, device) for a in (args[0], args[1], [0, 40])), 40)
    want.append(x[:40], x[:40], *args)
    want.same(cache)
    ops.kv8_append(cache, x[32:33].to(device) * 4, x[:1].to(device), i32(args[0], device), i32([41], device), i32([0, 1], device), 1)
    want.append(x[32:33] * 4, x[:1], args[0], [41], [1])
    want.same(cache)
    assert status(device) == 0


@pytest.mark.parametrize("device", WHERE)
def test_append_leaves_the_rest_alone(device):
    """Blocks of nobody and of sequences without new tokens, rows of no sequence."""
    lens = [30, 20, 0]
    cache, table = filled(lens, 16, 2, 32, 32, seed=4, device=device)
    before = on(cache, "cpu")
    k = randn(3, 2, 32).bfloat16().to(device)
    ops.kv8_append(cache, k, k, i32(table, device), i32([31, 20, 0], device), i32([0, 1, 1, 1], device), 1)
    mine = table[0][1]
    for n in cache.__slots__:
        a, b = getattr(before, n), getattr(cache, n).cpu()
        other = [i for i in range(a.shape[0]) if i != mine]
        a, b = (a.view(torch.uint8), b.view(torch.uint8)) if a.dtype == E4 else (a, b)
        assert torch.equal(a[other], b[other])
        assert not torch.equal(a[mine], b[mine]) or n.endswith("scale")
    assert status(device) == 0


@gpu
def test_append_bad_tables_are_recorded_and_not_followed():
    device = "cuda:0"
    cache = ops.Kv8Cache.empty(4, 16, 1, 32, 32, device)
    k = randn(20, 1, 32).bfloat16().to(device)
    for table, ctx, cu in (([[1, 4]], [20], [0, 20]), ([[1, -1]], [20], [0, 20]), ([[1, 2]], [20], [5, 25])):
        ops.kv8_append(cache, k, k, i32(table, device), i32(ctx, device), i32(cu, device), 20)
        assert status(device) != 0
        assert not bool(cache.k.view(torch.uint8)[[0, 2, 3]].any())
    # a length beyond the table: its cells end there
    ops.kv8_append(cache, k, k, i32([[2]], device), i32([20], device), i32([0, 20], device), 20)
    assert status(device) == 0 and bool(cache.k.view(torch.uint8)[2].any()) and not bool(cache.k.view(torch.uint8)[3].any())


# -------------------------------------------------------------------------------------------------------- attention
DECODE = [  # page, heads, kv heads, dk, dv, lengths
    (64, 8, 1, 128, 128, [1, 2, 127, 128, 129, 1000]),
    (16, 32, 4, 128, 128, [700, 1, 33]),
    (64, 16, 2, 256, 256, [300, 1000]),
    (8, 5, 5, 64, 64, [40, 9]),
    (32, 24, 2, 96, 160, [257, 64]),
    (64, 40, 1, 64, 256, [513]),
    (16, 6, 2, 192, 16, [130, 0, 5]),
    (64, 4, 2, 64, 64, [5000]),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,kv,dk,dv,lens", DECODE)
@pytest.mark.parametrize("form", ["plain", "window", "cap", "sink", "all"])
def test_decode(device, page, heads, kv, dk, dv, lens, form):
    cache, table = filled(lens, page, kv, dk, dv, seed=7, device=device)
    q = (randn(len(lens), heads, dk, seed=8) * 1.5).bfloat16()
    more = {"plain": {}, "window": {"window": 100}, "cap": {"softcap": 5.0}, "sink": {"sink": randn(heads, seed=9) * 2},
            "all": {"window": 33, "softcap": 20.0, "sink": randn(heads, seed=9)}}[form]
    new = [1] * len(lens)
    want, tol, _, _ = attend(q, cache, table, lens, new, dk ** -0.5, **more)
    if "sink" in more:
        more["sink"] = more["sink"].to(device)
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), 1, dk ** -0.5, **more)
    assert status(device) == 0
    near(got, want, tol)


PROMPT = [  # page, heads, kv heads, dk, dv, lengths, new tokens
    (64, 8, 1, 128, 128, [700], [700]),
    (64, 32, 4, 128, 128, [300, 1, 17, 640], [300, 1, 17, 5]),
    (16, 4, 4, 64, 64, [200, 129, 1000], [200, 64, 2]),
    (64, 16, 2, 256, 256, [260, 30], [260, 30]),
    (8, 10, 2, 80, 112, [131, 64], [100, 64]),
    (32, 24, 2, 96, 160, [257, 64, 0], [7, 64, 0]),
    (64, 6, 2, 192, 128, [400], [33]),
    (64, 40, 1, 64, 256, [513], [4]),
    (16, 5, 1, 16, 16, [90, 300], [90, 150]),
    (64, 8, 2, 128, 128, [6000], [3]),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,kv,dk,dv,lens,new", PROMPT)
@pytest.mark.parametrize("form", ["plain", "window", "cap", "sink", "all"])
def test_prompt(device, page, heads, kv, dk, dv, lens, new, form):
    cache, table = filled(lens, page, kv, dk, dv, seed=17, device=device)
    q = (randn(sum(new), heads, dk, seed=18) * 1.5).bfloat16()
    more = {"plain": {}, "window": {"window": 100}, "cap": {"softcap": 5.0}, "sink": {"sink": randn(heads, seed=9) * 2},
            "all": {"window": 33, "softcap": 20.0, "sink": randn(heads, seed=9)}}[form]
    want, tol, _, _ = attend(q, cache, table, lens, new, dk ** -0.5, **more)
    if "sink" in more:
        more["sink"] = more["sink"].to(device)
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), dk ** -0.5, **more)
    assert status(device) == 0
    near(got, want, tol)


@pytest.mark.parametrize("device", WHERE)
def test_prompt_rows_apart(device):
    lens, new, heads, kv, D = [200, 77, 300], [20, 0, 150], 8, 2, 64
    cache, table = filled(lens, 32, kv, D, D, seed=1, device=device)
    for shift in (0, 1):
        wide = randn(170, heads * D + 100 + shift, seed=2).bfloat16().to(device)
        q = wide[:, shift:shift + heads * D].view(170, heads, D)
        out = torch.full((172, heads * D + 24 + shift), 7.0, dtype=torch.bfloat16, device=device)
        mine = out[1:171, 8:8 + heads * D].unflatten(1, (heads, D))
        ops.kv8_attention(q, cache, i32(table, device), i32(lens, device), i32(cum(new), device), 150, 0.125, max_ctx=300, out=mine)
        want, tol, _, _ = attend(q.cpu(), cache, table, lens, new, 0.125)
        near(mine, want, tol)
        mine.fill_(7.0)
        assert bool((out == 7.0).all()) and status(device) == 0


@pytest.mark.parametrize("device", WHERE)
def test_prompt_propagates_nan_to_rows_that_see_it(device):
    lens, new = [300, 140], [300, 100]
    cache, table = filled(lens, 16, 1, 64, 64, seed=3, device=device)
    cache.v.view(torch.uint8)[table[0][9], 0, 5, 9] = NAN          # position 149
    cache.k.view(torch.uint8)[table[1][6], 0, 7, 0] = NAN          # position 103
    q = randn(400, 4, 64, seed=4).bfloat16()
    q[350, 1, 3] = math.nan
    want, tol, _, _ = attend(q, cache, table, lens, new, 0.125)
    assert bool(want[149:300, :, 9].isnan().all()) and not bool(want[:149].isnan().any())
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), 300, 0.125)
    near(got, want, tol)


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("heads,kv,D,lens", [(8, 2, 64, [(37 * i) % 300 for i in range(150)]), (4, 4, 32, [1] * 300),
                                             (34, 2, 64, [128, 129, 0, 640, 1, 1, 2000, 5])])
def test_decode_batches(device, heads, kv, D, lens):
    """Batches whose lengths are spread over the CTAs: more sequences than are kept at hand, groups inside and across CTAs, short
    ones in a row, lengths of zero, rows that not every sequence has."""
    cache, table = filled(lens, 16, kv, D, D, seed=11, device=device)
    new = [0 if i % 13 == 5 else 1 for i in range(len(lens))]
    q = randn(sum(new), heads, D, seed=12).bfloat16()
    want, tol, _, _ = attend(q, cache, table, lens, new, 0.2)
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), 1, 0.2)
    assert status(device) == 0
    near(got, want, tol)


@pytest.mark.parametrize("device", WHERE)
def test_decode_rows_apart(device):
    """Queries cut out of a projection, an output with rows of its own pitch, sequences without a row, max_ctx."""
    lens, heads, kv, D = [200, 77, 300], 8, 2, 64
    cache, table = filled(lens, 32, kv, D, D, seed=1, device=device)
    new = [1, 0, 1]
    for shift in (0, 1):
        wide = randn(2, heads * D + 100 + shift, seed=2).bfloat16().to(device)
        q = wide[:, shift:shift + heads * D].view(2, heads, D)
        out = torch.full((4, heads * D + 24), 7.0, dtype=torch.bfloat16, device=device)
        ops.kv8_attention(q, cache, i32(table, device), i32(lens, device), i32(cum(new), device), 1, 0.125, max_ctx=300,
                          out=out[1:3, 8:8 + heads * D].unflatten(1, (heads, D)))
        want, tol, _, _ = attend(q.cpu(), cache, table, lens, new, 0.125)
        near(out[1:3, 8:8 + heads * D].unflatten(1, (heads, D)), want, tol)
        out[1:3, 8:8 + heads * D] = 7.0
        assert bool((out == 7.0).all()) and status(device) == 0


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 1, 30]])
def test_attention_does_not_see_masked_garbage(device, new):
    """NaN codes and odd scales behind a sequence and in front of its window."""
    lens, window = [150, 70, 400], 40
    cache, table = filled(lens, 16, 2, 64, 64, seed=3, device=device)
    q = randn(sum(new), 4, 64, seed=4).bfloat16()
    want, tol, _, _ = attend(q, cache, table, lens, new, 0.125, window=window)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        raw = codes.view(torch.uint8)
        raw[0], scale[0] = NAN, math.nan
        for i, n in enumerate(lens):
            raw[table[i][n // 16], :, n % 16:] = NAN
            first = n - new[i] - window + 1
            raw[table[i][first // 16], :, :first % 16] = NAN
            raw[table[i][: first // 16]] = NAN
            scale[table[i][: first // 16]] = math.inf
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), 0.125, window=window)
    assert status(device) == 0
    near(got, want, tol)


@pytest.mark.parametrize("device", WHERE)
def test_decode_propagates_nan(device):
    lens = [150, 70, 300]
    cache, table = filled(lens, 16, 1, 64, 64, seed=3, device=device)
    cache.v.view(torch.uint8)[table[0][3], 0, 5, 9] = NAN
    cache.k.view(torch.uint8)[table[1][0], 0, 0, 0] = NAN
    q = randn(3, 4, 64, seed=4).bfloat16()
    q[2, 1, 3], q[2, 2, 0] = math.nan, math.inf
    want, tol, _, _ = attend(q, cache, table, lens, [1] * 3, 0.125)
    want[2, 2] = math.nan                              # an infinite query value: infinity times zero among its products
    got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32([0, 1, 2, 3], device), 1, 0.125)
    near(got, want, tol)


@pytest.mark.parametrize("device", WHERE)
def test_decode_far_apart_scales(device):
    """Blocks whose values differ by 2^40: what the large ones leave of the small ones' weight must not overflow or vanish."""
    n, page = 300, 16
    table, blocks = tables([n], page)
    cache = ops.Kv8Cache.empty(blocks, page, 1, 64, 64)
    k, v = randn(n, 1, 64, seed=1).bfloat16(), randn(n, 1, 64, seed=2)
    v = (v * torch.exp2(torch.linspace(-30, 10, n).round())[torch.randperm(n, generator=gen(3))].view(n, 1, 1)).bfloat16()
    ops.kv8_append(cache, k, v, i32(table), i32([n]), i32([0, n]), n)
    cache = on(cache, device)
    for sharp in (1.0, 30.0):
        q = randn(1, 8, 64, seed=5).mul(sharp).bfloat16()
        want, tol, _, _ = attend(q, cache, table, [n], [1], 0.125)
        got = ops.kv8_attention(q.to(device), cache, i32(table, device), i32([n], device), i32([0, 1], device), 1, 0.125)
        near(got, want, tol)


# ---------------------------------------------------------------------------------------- sums of weights, eviction
WEIGHTS = [  # page, heads, kv heads, dk, dv, lengths, new tokens, observed rows
    (64, 8, 1, 128, 128, [300, 1, 700], [1, 1, 1], 0),
    (64, 40, 8, 128, 128, [129, 500], [1, 1], 0),
    (16, 32, 2, 64, 64, [257, 0, 130], [1, 1, 1], 0),
    (64, 24, 1, 256, 64, [400], [1], 0),
    (64, 8, 2, 128, 128, [300, 150], [300, 40], 0),
    (32, 6, 2, 64, 96, [300, 150, 90], [130, 0, 90], 32),
    (64, 5, 1, 256, 256, [600], [200], 64),
    (8, 3, 3, 48, 48, [140], [7], 1),
    (64, 4, 2, 64, 64, [5000], [3], 2),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,heads,kv,dk,dv,lens,new,observe", WEIGHTS)
@pytest.mark.parametrize("form", ["plain", "all"])
def test_sums_of_weights(device, page, heads, kv, dk, dv, lens, new, observe, form):
    cache, table = filled(lens, page, kv, dk, dv, seed=27, device=device)
    q = (randn(sum(new), heads, dk, seed=28) * 1.5).bfloat16()
    more = {"plain": {}, "all": {"window": 50, "softcap": 20.0, "sink": randn(heads, seed=9)}}[form]
    _, _, weight, off = attend(q, cache, table, lens, new, dk ** -0.5, **more)
    if "sink" in more:
        more["sink"] = more["sink"].to(device)
    L = max(lens) + 3
    start = torch.rand(len(lens), kv, L, generator=gen(1))
    big = torch.full((len(lens), kv + 1, L + 5), -3.0, device=device)
    w = big[:, 1:, 2:2 + L]
    w.copy_(start)
    ops.kv8_attention(q.to(device), cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), dk ** -0.5, weights=w,
                      observe=observe, **more)
    assert status(device) == 0
    for i, (n, m) in enumerate(zip(lens, new)):
        rows = torch.arange(weight[i].shape[2]) % max(m, 1) >= (m - observe if observe else 0)
        want, tol = weight[i][:, :, rows].sum(2), off[i][:, :, rows].sum(2)
        got = (w[i].cpu().double() - start[i].double())
        assert bool(((got[:, :n] - want).abs() <= tol + 2.0 ** -23 * (start[i, :, :n] + want)).all())
        assert not bool(got[:, n:].any())
    w.fill_(-3.0)
    assert bool((big == -3.0).all())


def evict(cache, table, lens, w, budget, dst, first, last):
    """The rules of eviction on code values, in float64: (kept, sums, keys and values by block, scales)."""
    page = cache.k.shape[2]
    kept, sums, blocks = [], [], {}
    for i, n in enumerate(lens):
        for h in range(w.shape[1]):
            order = sorted(range(n), key=lambda t: (not (t < first or t >= n - last), -float(w[i, h, t]), t))
            stay = sorted(order[:budget])
            kept.append(stay + [-1] * (budget - len(stay)))
            sums.append([float(w[i, h, t]) for t in stay] + [0.0] * (budget - len(stay)))
            for j in range(0, len(stay), page):
                for name in ("k", "v"):
                    codes, scale = CODES[getattr(cache, name).view(torch.uint8).long()], getattr(cache, name + "_scale").double()
                    part = stay[j:j + page]
                    src = [table[i][t // page] for t in part]
                    now = max(float(scale[s, h]) for s in src)
                    rows = torch.zeros(page, codes.shape[3], dtype=torch.float64)
                    for r, (t, s) in enumerate(zip(part, src)):
                        rows[r] = encode(codes[s, h, t % page] * (float(scale[s, h]) / now if now else 0.0))
                    blocks[name, dst[i][j // page], h] = rows, now
    return kept, sums, blocks


EVICT = [  # page, kv heads, dk, dv, lengths, budget, first, last
    (16, 2, 64, 64, [100, 40, 41, 0, 7], 40, 4, 8),
    (64, 1, 128, 32, [700], 130, 0, 0),
    (8, 3, 16, 48, [90, 33], 33, 33, 0),
    (64, 1, 32, 32, [1500], 1, 0, 1),
    (16, 1, 32, 16, [3000], 1000, 1, 100),
]


@pytest.mark.parametrize("device", WHERE)
@pytest.mark.parametrize("page,kv,dk,dv,lens,budget,first,last", EVICT)
@pytest.mark.parametrize("weights", ["spread", "equal", "ties", "signed"])
def test_evict(device, page, kv, dk, dv, lens, budget, first, last, weights):
    cache, table = filled(lens, page, kv, dk, dv, seed=5)
    w = torch.exp2(randn(len(lens), kv, max(lens) + 2, seed=6) * 4)
    if weights == "equal":
        w = torch.full_like(w, 0.25)
    elif weights == "ties":
        w = torch.round(w).clamp(max=3)
    elif weights == "signed":
        w = torch.round(randn(*w.shape, seed=8) * 4) / 4
        w[..., ::7] *= -0.0
    # block 0 and those behind the sequences' are free
    n_old, per = cache.k.shape[0], -(-budget // page)
    dst = (torch.randperm(len(lens) * per, generator=gen(2)) + n_old).view(len(lens), per).tolist()
    more = ops.Kv8Cache.empty(n_old + len(lens) * per, page, kv, dk, dv)
    for name in cache.__slots__:
        getattr(more, name).view(torch.uint8)[:] = 0x7F if name in "kv" else 0
        a, b = getattr(more, name), getattr(cache, name)
        (a.view(torch.uint8) if name in "kv" else a)[:n_old] = b.view(torch.uint8) if name in "kv" else b
    kept, sums, blocks = evict(more, table, lens, w, budget, dst, first, last)
    got = on(more, device)
    lens_out, kept_out, sums_out = ops.kv8_evict(got, i32(table, device), i32(lens, device), w.to(device), budget, i32(dst, device), first, last)
    assert status(device) == 0
    assert lens_out.tolist() == [min(n, budget) for n in lens]
    assert kept_out.flatten(0, 1).tolist() == kept
    assert sums_out.flatten(0, 1).tolist() == sums
    for name in ("k", "v"):
        codes = getattr(got, name).cpu().view(torch.uint8)
        before = getattr(more, name).view(torch.uint8)
        for blk in range(codes.shape[0]):
            for h in range(kv):
                if (name, blk, h) in blocks:
                    rows, now = blocks[name, blk, h]
                    assert torch.equal(CODES[codes[blk, h].long()], rows) and float(getattr(got, name + "_scale")[blk, h]) == now
                else:
                    assert torch.equal(codes[blk, h], before[blk, h])


@pytest.mark.parametrize("device", WHERE)
def test_a_chat_whose_cache_is_pruned(device):
    """Append, attend with sums, evict, go on in the new blocks: attention over what stayed equals the float64 form over the kept
    tokens, and a second eviction counts on."""
    page, kv, heads, D, budget = 16, 2, 8, 64, 48
    cache = ops.Kv8Cache.empty(40, page, kv, D, D, device)
    table = [[1, 2, 3, 4, 5, 6, 7, 8, 0, 0], [11, 12, 13, 14, 15, 16, 17, 18, 0, 0]]
    sums = torch.zeros(2, kv, 160, device=device)
    lens, step = [0, 0], 0
    spare = [[20, 21, 22, 23, 24, 25], [30, 31, 32, 33, 34, 35]]

    def forward(new):
        nonlocal lens, step
        lens, step = [a + b for a, b in zip(lens, new)], step + 1
        T = sum(new)
        k, v, q = (randn(T, h, D, seed=100 * step + j).bfloat16().to(device) for j, h in enumerate((kv, kv, heads)))
        args = (i32(table, device), i32(lens, device), i32(cum(new), device), max(new))
        ops.kv8_append(cache, k, v, *args)
        before = sums.cpu().double()
        out = ops.kv8_attention(q, cache, *args, 0.3, weights=sums)
        want, tol, weight, off = attend(q.cpu(), on(cache, "cpu"), table, lens, new, 0.3)
        near(out, want, tol)
        for i, n in enumerate(lens):
            got = sums[i, :, :n].cpu().double() - before[i, :, :n]
            assert bool(((got - weight[i].sum(2)).abs() <= off[i].sum(2) + 2.0 ** -22 * (1 + before[i, :, :n])).all())

    forward([100, 70])
    for _ in range(3):
        forward([1, 1])
    for again in range(2):
        dst = [s[:3] for s in spare]
        n, kept, w = ops.kv8_evict(cache, i32(table, device), i32(lens, device), sums, budget, i32(dst, device), 2, 10)
        lens = n.tolist()
        assert lens == [budget, budget] and kept.shape == (2, kv, budget)
        old = table
        table = [d + s[3:] + [0] * 4 for d, s in zip(dst, spare)]
        spare = [[b for b in o if b][:6] for o in old]
        sums.zero_()
        sums[..., :budget] = w
        forward([1, 1])
        forward([20, 3])
        forward([1, 1])
    assert status(device) == 0


# ------------------------------------------------------------------------------------- streams, graphs, many launches
@gpu
def test_two_streams_at_once():
    """Calls on two streams share no scratch: each gives what it gives alone."""
    device, cases = "cuda:0", []
    for j, (lens, new) in enumerate((([3000, 500, 77], [1, 1, 1]), ([900, 1500, 60], [300, 5, 60]))):
        cache, table = filled(lens, 16, 2, 64, 64, seed=j, device=device)
        q = randn(sum(new), 8, 64, seed=j + 9).bfloat16().to(device)
        args = (q, cache, i32(table, device), i32(lens, device), i32(cum(new), device), max(new), 0.125)
        w = torch.zeros(3, 2, max(lens), device=device)
        cases.append((args, ops.kv8_attention(*args, weights=w).clone(), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for j in (0, 1):
            with torch.cuda.stream(streams[j]):
                w = torch.zeros_like(cases[j][2])
                got[j].append((ops.kv8_attention(*cases[j][0], weights=w), w))
    torch.cuda.synchronize()
    for j in (0, 1):
        for o, w in got[j]:
            assert torch.equal(o, cases[j][1]) and torch.equal(w, cases[j][2])
    assert status(device) == 0


@gpu
def test_captured_and_replayed_with_new_data():
    """Append, attention with sums and eviction in two graphs that are replayed in turn, lengths and rows changed between replays."""
    device, page, kv, heads, D = "cuda:0", 16, 2, 8, 64
    graphs = []
    for j in range(2):
        cache = ops.Kv8Cache.empty(40, page, kv, D, D, device)
        table, dst = i32([list(range(1, 9)), list(range(9, 17))], device), i32([[20, 21], [22, 23]], device)
        ctx, cu = i32([40, 20], device), i32([0, 1, 2], device)
        k, v, q = (torch.zeros(2, h, D, dtype=torch.bfloat16, device=device) for h in (kv, kv, heads))
        sums = torch.zeros(2, kv, 128, device=device)

        def body():
            ops.kv8_append(cache, k, v, table, ctx, cu, 1)
            o = ops.kv8_attention(q, cache, table, ctx, cu, 1, 0.2, weights=sums)
            return (o,) + ops.kv8_evict(cache, table, ctx, sums, 24, dst, keep_first=2, keep_last=4)
        fill = randn(60, kv, D, seed=j).bfloat16().to(device)
        ops.kv8_append(cache, fill, fill, table, i32([39, 19], device), i32([0, 39, 58], device), 39)
        body()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = body()
        graphs.append((g, out, cache, (k, v, q), ctx, sums, table, (cu, dst)))      # (a graph keeps no tensor alive)
    for step in range(3):
        for j, (g, out, cache, rows, ctx, sums, table, _) in enumerate(graphs):
            for t, h in zip(rows, (kv, kv, heads)):
                t.copy_(randn(2, h, D, seed=100 * step + 10 * j + h))
            lens = [41 + step, 21 + step]
            ctx.copy_(i32(lens))
            sums.zero_()
            before = on(cache, "cpu")
            g.replay()
            torch.cuda.synchronize()
            ops.kv8_append(before, rows[0].cpu(), rows[1].cpu(), table.cpu(), i32(lens), i32([0, 1, 2]), 1)
            want, tol, weight, off = attend(rows[2].cpu(), before, table.tolist(), lens, [1, 1], 0.2)
            near(out[0], want, tol)
            assert out[1].tolist() == [24, min(24, lens[1])]
            for i, n in enumerate(lens):
                assert bool(((sums[i, :, :n].cpu().double() - weight[i].sum(2)).abs() <= off[i].sum(2) + 2.0 ** -22).all())
                kept = out[2][i, 0, :min(24, n)].tolist()
                assert kept == sorted(kept) and kept[:2] == [0, 1] and kept[-4:] == list(range(n - 4, n))
    assert status(device) == 0


@gpu
def test_the_same_call_gives_the_same_bits():
    device = "cuda:0"
    lens, new = [2000, 300, 1, 129], [1, 1, 1, 1]
    cache, table = filled(lens, 64, 2, 128, 128, seed=1, device=device)
    q = randn(4, 16, 128, seed=2).bfloat16().to(device)
    first = None
    for _ in range(10):
        w = torch.zeros(4, 2, 2000, device=device)
        o = ops.kv8_attention(q, cache, i32(table, device), i32(lens, device), i32(cum(new), device), 1, 0.1, weights=w)
        first = first or (o, w)
        assert torch.equal(o, first[0]) and torch.equal(w, first[1])


@gpu
def test_empty_calls():
    device = "cuda:0"
    cache, table = filled([20], 16, 2, 32, 32, device=device)
    none = torch.empty(0, 4, 32, dtype=torch.bfloat16, device=device)
    o = ops.kv8_attention(none, cache, i32(table, device), i32([20], device), i32([0, 0], device), 0, 1.0)
    assert o.shape == (0, 4, 32)
    ops.kv8_append(cache, none[:, :2], none[:, :2], i32(table, device), i32([20], device), i32([0, 0], device), 0)
    no_seqs = torch.empty(0, 3, dtype=torch.int32, device=device)
    o = ops.kv8_attention(none, cache, no_seqs, i32([], device), i32([0], device), 0, 1.0)
    lens, kept, sums = ops.kv8_evict(cache, no_seqs, i32([], device), torch.empty(0, 2, 5, device=device), 4, no_seqs)
    assert lens.shape == (0,) and kept.shape == (0, 2, 4) and status(device) == 0


# -------------------------------------------------------------------------------------------------------- refusals
def _refusals():
    def base():
        cache, table = filled([20], 16, 2, 32, 32)
        return dict(cache=cache, q=randn(1, 4, 32).bfloat16(), k=randn(1, 2, 32).bfloat16(), table=i32(table), ctx=i32([20]), cu=i32([0, 1]))
    return base


@pytest.mark.parametrize("what", ["float queries", "head size", "heads", "scale type", "int64 lengths", "bounds", "page", "code type",
                                  "odd head size", "window", "softcap", "devices"])
def test_refusals_need_no_gpu(what):
    """The extension's own checks of shapes and types, on CPU tensors."""
    if not ops.sm100.have_ext():
        pytest.skip("extension not built")
    a = _refusals()()
    c, kw = a["cache"], dict(window=0, softcap=0.0)
    if what == "float queries":
        a["q"] = a["q"].float()
    elif what == "head size":
        a["q"] = a["q"][..., :16]
    elif what == "heads":
        a["q"] = randn(1, 3, 32).bfloat16()
    elif what == "scale type":
        c.k_scale = c.k_scale.double()
    elif what == "int64 lengths":
        a["ctx"] = a["ctx"].long()
    elif what == "bounds":
        a["cu"] = i32([0])
    elif what == "page":
        a["cache"] = c = ops.Kv8Cache.empty(3, 24, 2, 32)
    elif what == "code type":
        c.v = c.v.view(torch.uint8)
    elif what == "odd head size":
        a["cache"], a["q"] = ops.Kv8Cache.empty(3, 16, 2, 40), randn(1, 4, 40).bfloat16()
        c = a["cache"]
    elif what == "window":
        kw["window"] = -1
    elif what == "softcap":
        kw["softcap"] = -2.0
    C, st = ops.sm100.ext(), torch.zeros(4, dtype=torch.int32)
    out = torch.zeros(1, a["q"].shape[1], c.v.shape[3], dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="kv8_attention"):
        C.kv8_attention(a["q"], c.k, c.v, c.k_scale, c.v_scale, a["table"], a["ctx"], a["cu"], 1, 0.1, kw["window"], kw["softcap"], None, 1,
                        out, st, None, 0, 1)
    if what in ("scale type", "int64 lengths", "bounds", "page", "code type", "devices"):
        with pytest.raises(ValueError, match="kv8_append"):
            C.kv8_append(c.k, c.v, c.k_scale, c.v_scale, a["k"], a["k"], a["table"], a["ctx"], a["cu"], 1, st)


@pytest.mark.parametrize("what", ["sums type", "sums shape", "rows overlap", "observe", "budget", "first and last", "blocks", "no budget"])
def test_refusals_of_sums_and_eviction_need_no_gpu(what):
    if not ops.sm100.have_ext():
        pytest.skip("extension not built")
    a = _refusals()()
    c, C, st = a["cache"], ops.sm100.ext(), torch.zeros(4, dtype=torch.int32)
    w, observe, budget, first, last, dst = torch.zeros(1, 2, 20), 0, 16, 0, 0, i32([[1, 2]])
    if what == "sums type":
        w = w.double()
    elif what == "sums shape":
        w = w[:, :1]
    elif what == "rows overlap":
        w = torch.zeros(1, 1, 20).expand(1, 2, 20)
    elif what == "observe":
        observe = -1
    elif what == "budget":
        budget = 40
    elif what == "first and last":
        first, last = 10, 7
    elif what == "blocks":
        dst = i32([[1, 2], [3, 4]])
    elif what == "no budget":
        budget = 0
    if what in ("sums type", "sums shape", "rows overlap", "observe"):
        with pytest.raises(ValueError, match="kv8_attention"):
            C.kv8_attention(a["q"], c.k, c.v, c.k_scale, c.v_scale, a["table"], a["ctx"], a["cu"], 1, 0.1, 0, 0.0, None, 1,
                            torch.zeros(1, 4, 32, dtype=torch.bfloat16), st, w, observe, 1)
    if what != "observe":
        with pytest.raises(ValueError, match="kv8_evict"):
            C.kv8_evict(c.k, c.v, c.k_scale, c.v_scale, a["table"], a["ctx"], w, budget, first, last, dst, i32([0]),
                        torch.zeros(1, 2, budget, dtype=torch.int32), torch.zeros(1, 2, budget), st)
        with pytest.raises(ValueError):
            ops.kv8_evict(c, a["table"], a["ctx"], w if what != "rows overlap" else w[:, :1], budget, dst, first, last)


def test_cpu_refusals():
    a = _refusals()()
    c = a["cache"]
    with pytest.raises(ValueError):
        ops.kv8_append(c, a["k"][:, :1], a["k"][:, :1], a["table"], a["ctx"], a["cu"], 1)
    with pytest.raises(ValueError):
        ops.kv8_attention(a["q"][..., :16], c, a["table"], a["ctx"], a["cu"], 1, 1.0)
    with pytest.raises(ValueError):
        ops.kv8_attention(a["q"], c, a["table"], a["ctx"], a["cu"], 1, 1.0, window=-1)
    with pytest.raises(ValueError):
        ops.kv8_attention(a["q"], ops.Kv8Cache(c.k, c.v, c.k_scale.double(), c.v_scale), a["table"], a["ctx"], a["cu"], 1, 1.0)
