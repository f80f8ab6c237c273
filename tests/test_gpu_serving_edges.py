"""The 8-bit projections and the paged cache where ordinary values do not reach:
scores far apart, infinities and NaN in the cache, batches whose work crosses
sequences, ties, and the ends of the floats' range.  The bounds are those of
test_gpu_serving_ops.py, whose helpers are used."""
import ctypes as C
import math

import pytest

import test_gpu_serving_ops as T
import xl_capi as X

pytestmark = pytest.mark.gpu

U = T.U
CACHES = pytest.mark.parametrize("cache", [0, 1, 2], ids=["fp32", "bf16", "fp16"])


@pytest.fixture(scope="module")
def torch(built):
    import torch

    torch.cuda.init()
    return torch


# ---- attention -----------------------------------------------------------------------------------------------------

class Pool:
    """A shuffled pool for many sequences, filled on the device; positions past each sequence's rows hold NaN."""

    def __init__(self, torch, dtype, lens, kv, d, page, seed):
        self.page, self.kv, self.d = page, kv, d
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = torch.tensor([(n + page - 1) // page for n in lens])
        total, wide = int(need.sum()) + 2, max(1, int(need.max()))
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
        column = torch.arange(wide)
        index = (need.cumsum(0) - need)[:, None] + column
        self.table = torch.where(column < need[:, None], order[index.clamp(max=total - 1)], 1 << 30).int()
        self.dt = self.table.cuda()
        t = T.types(torch)[dtype]
        self.k, self.v = (torch.empty((total, kv, page, d), dtype=t, device="cuda").normal_(generator=g) for _ in range(2))
        for b, n in enumerate(lens):
            if n % page:
                last = int(self.table[b, n // page])
                self.k[last, :, n % page:] = math.nan
                self.v[last, :, n % page:] = math.inf
        self.c = X.PagedKV(self.k.data_ptr(), self.v.data_ptr(), self.dt.data_ptr(), dtype, len(lens), kv, d, page, wide, total)

    def rows(self, b, n):
        """Positions 0 .. n - 1 of sequence b as views: [kv][n][d] copies in 64 bits."""
        pages = self.dt[b, :(n + self.page - 1) // self.page].long()
        return tuple(x[pages].permute(1, 0, 2, 3).reshape(self.kv, -1, self.d)[:, :n].double() for x in (self.k, self.v))

    def put(self, which, b, pos, value):
        """value (a row of d, or what broadcasts to it) at position pos of sequence b, in all heads."""
        (self.k if which == "k" else self.v)[int(self.table[b, pos // self.page]), :, pos % self.page] = value


def check(torch, pool, qkv, rope, b, n, out, heads):
    """Sequence b's output against 64 bits over what the cache holds, the kinds of its values (finite, an infinity, NaN)
    among them."""
    d, kv, group = pool.d, pool.kv, heads // pool.kv
    row = qkv[b].double().view(heads + 2 * kv, d)
    q = row[:heads]
    keys, values = pool.rows(b, n + 1)
    big = q.abs() + q.abs().roll(d // 2, -1) if rope is not None else q.abs()
    if rope is not None:
        q = T.rotate(torch, q, rope[n])
    q, big = q.view(kv, group, d), big.view(kv, group, d)
    s = torch.einsum("kgd,knd->kgn", q, keys) / math.sqrt(d)
    w = torch.softmax(s, -1)
    want = torch.empty((kv, group, d), dtype=torch.float64, device="cuda")
    reach = torch.empty_like(want)
    finite = torch.where(values.isfinite(), values, 0.0).abs()
    for h in range(kv):  # products and a sum, so that 0 x inf shows as it does in the definition
        for i in range(group):
            want[h, i] = (w[h, i][:, None] * values[h]).sum(0)
            reach[h, i] = (w[h, i][:, None] * finite[h]).sum(0)
    size = torch.where(keys.isfinite(), keys, 0.0).abs()
    ds = ((d + 8) * 2 * U + 8 * U + 2.0 ** -21) * torch.einsum("kgd,knd->kgn", big, size).amax(-1, keepdim=True) / math.sqrt(d)
    tol = (2 * ds + 2.0 ** -16 + (n + 17) * 2 * U + 2.0 ** -20) * reach
    got = out[b].double().view(kv, group, d)
    assert torch.equal(got.isnan(), want.isnan()), (b, int(got.isnan().sum()), int(want.isnan().sum()))
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf]), b
    ok = want.isfinite()
    off = (got - want).abs() - tol - T.half_step(torch, out.dtype) * (want.abs() + tol) - torch.finfo(out.dtype).tiny
    assert (off[ok] <= 0).all(), (b, float(off[ok].max()), float(tol[ok].max()))


@CACHES
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (10, 1, 128)])
@pytest.mark.parametrize("gap", [12, 16, 18, 21, 25])
def test_attend_small_weights(torch, cache, heads, kv, d, gap):
    """One position stands `gap` above the others and holds a value of zero, so the small weights are all of the output."""
    n = 1500
    p = Pool(torch, cache, [n + 1] * 3, kv, d, 16, seed=gap)
    for b, spot in enumerate((0, 700, n)):
        p.k[p.table[b].long().cuda(), :, :, 0] = 0.0
        p.put("k", b, spot, torch.eye(1, d, device="cuda")[0] * gap)
        p.put("v", b, spot, 0.0)
    qkv = torch.randn((3, (heads + 2 * kv) * d), generator=T.gen(torch, 2))
    rows = qkv.view(3, heads + 2 * kv, d)
    rows[:, :heads] *= 0.01
    rows[:, :heads, 0] = math.sqrt(d)
    rows[:, heads:, 0] = 0.0
    rows[2, heads:heads + kv] = torch.eye(1, d)[0] * gap
    rows[2, heads + kv:] = 0.0
    dq, out = qkv.cuda(), torch.empty((3, heads * d), device="cuda")
    pos = torch.full((3,), n, dtype=torch.int32, device="cuda")
    T.attend(torch, p, 0, dq, None, pos, out, heads, T.workspace(torch, p.c, heads))
    for b in range(3):
        check(torch, p, dq, None, b, n, out, heads)


def test_attend_queries_of_uneven_size(torch):
    """Query elements far below the row's largest count in full where the keys are small at the large ones."""
    heads, kv, d, n = 4, 2, 64, 400
    p = Pool(torch, 2, [n + 1], kv, d, 16, seed=4)
    p.k[..., 0] = 0.0
    p.k[..., 1:] *= 100
    qkv = torch.randn((1, (heads + 2 * kv) * d), generator=T.gen(torch, 3))
    rows = qkv.view(1, heads + 2 * kv, d)
    rows[:, :heads] *= 2e-3
    rows[:, :heads, 0] = 3e4
    rows[:, heads:heads + kv, 0] = 0.0
    dq, out = qkv.cuda(), torch.empty((1, heads * d), device="cuda")
    pos = torch.tensor([n], dtype=torch.int32, device="cuda")
    T.attend(torch, p, 0, dq, None, pos, out, heads, T.workspace(torch, p.c, heads))
    check(torch, p, dq, None, 0, n, out, heads)


@CACHES
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (8, 1, 128), (12, 1, 64), (32, 2, 128)])
def test_attend_fp32_rows_keep_their_bits(torch, cache, heads, kv, d):
    """Two positions, one element of the query that counts: out = 1 / (1 + e^-s) of a 24-bit s.  Nothing is summed but
    the query's parts (4 steps of 2u), the scale takes 4u more and the split 2^-21 at most; the rest as in the other
    bound."""
    batch = 64
    p = Pool(torch, cache, [2] * batch, kv, d, 4, seed=3)
    p.k.zero_()
    p.v.zero_()
    g = T.gen(torch, heads + d)
    qkv = torch.zeros((batch, heads + 2 * kv, d))
    qkv[:, :heads, 0] = (torch.rand((batch, heads), generator=g) * 40 - 20) * math.sqrt(d)
    qkv[:, heads:heads + kv, 0], qkv[:, heads + kv:] = 1.0, 1.0
    dq, out = qkv.view(batch, -1).cuda(), torch.empty((batch, heads * d), device="cuda")
    pos = torch.ones(batch, dtype=torch.int32, device="cuda")
    T.attend(torch, p, 0, dq, None, pos, out, heads, T.workspace(torch, p.c, heads))
    s = qkv[:, :heads, 0].double() / math.sqrt(d)
    want = torch.sigmoid(s)
    tol = (2 * (12 * U + 2.0 ** -21) * s.abs() + 2.0 ** -21 + 18 * 2 * U + 2.0 ** -20) * want
    off = (out.view(batch, heads, d).cpu().double() - want[..., None]).abs() - (tol + U * want)[..., None]
    assert (off <= 0).all(), float((off / want[..., None]).max())


def special(torch, p, rows, b, n, what, heads):
    """Makes sequence b (last position n) hold `what`; element 0 of every query is -1, element 1 is 4 sqrt(d)."""
    kv, d, mid = p.kv, p.d, n // 2
    unit = torch.zeros(d, device="cuda")
    if what == "key_out":  # a score of minus infinity: weight 0
        unit[0] = math.inf
        p.put("k", b, mid, unit)
    elif what == "keys_out":  # the first chunk of 64 positions and part of the second
        unit[0] = math.inf
        for t in range(min(80, n)):
            p.put("k", b, t, unit)
    elif what == "all_out":  # nothing is left: 0 / 0
        unit[0] = math.inf
        for t in range(n):
            p.put("k", b, t, unit)
        rows[b, heads:heads + kv, 0] = math.inf
    elif what == "key_in":  # a score of infinity: inf - inf in the softmax
        unit[0] = -math.inf
        p.put("k", b, mid, unit)
    elif what == "key_nan":
        unit[3] = math.nan
        p.put("k", b, mid, unit)
    elif what == "value":
        unit[3], unit[5], unit[7] = math.inf, -math.inf, math.inf
        p.put("v", b, mid, unit)
        unit[3], unit[5], unit[7] = 0.0, 0.0, -math.inf
        p.put("v", b, 0, unit)
    elif what == "value_far":  # at a weight of e^-60, e^-95 and, in the last position, e^-130
        for t, (down, column) in {0: (60, 2), mid: (95, 3), n: (130, 4)}.items():
            key = unit.clone()
            key[1], value = -down / 4.0, unit.clone()
            value[column] = math.inf
            if t == n:
                rows[b, heads:heads + kv] = key.cpu()
                rows[b, heads + kv:] = value.cpu()
            else:
                p.put("k", b, t, key)
                p.put("v", b, t, value)
    elif what == "value_out":  # 0 x inf
        unit[0] = math.inf
        p.put("k", b, mid, unit)
        unit[0], unit[9] = 0.0, math.inf
        p.put("v", b, mid, unit)
    elif what == "value_nan":
        unit[6] = math.nan
        p.put("v", b, n - 1 if n else 0, unit)
    elif what == "overflow":  # finite rows that a 16-bit cache stores as infinity
        rows[b, heads + kv:, 8] = 1e5
    else:
        assert what == "plain"


SPECIALS = ["plain", "key_out", "keys_out", "all_out", "key_in", "key_nan", "value", "value_far", "value_out", "value_nan",
            "overflow"]


@CACHES
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (8, 1, 128), (12, 1, 64), (32, 2, 128)])
@pytest.mark.parametrize("n,copies", [(1, 1), (90, 1), (700, 1), (90, 60)])
def test_attend_infinities_and_nan(torch, cache, heads, kv, d, n, copies):
    """Infinities and NaN in the cache, in sequences that one CTA takes, that several share, and (many of them) that
    follow one another in one CTA."""
    whats = SPECIALS * copies
    p = Pool(torch, cache, [n + 1] * len(whats), kv, d, 16, seed=n)
    p.k[..., 1] = 0.0
    qkv = torch.randn((len(whats), (heads + 2 * kv) * d), generator=T.gen(torch, n))
    rows = qkv.view(len(whats), heads + 2 * kv, d)
    rows[:, :heads, 0], rows[:, :heads, 1], rows[:, heads:heads + kv, 1] = -1.0, 4 * math.sqrt(d), 0.0
    for b, what in enumerate(whats):
        special(torch, p, rows, b, n, what, heads)
    dq = qkv.cuda()
    pos = torch.full((len(whats),), n, dtype=torch.int32, device="cuda")
    ws, outs = T.workspace(torch, p.c, heads), []
    for _ in range(2):
        out = torch.empty((len(whats), heads * d), device="cuda")
        T.attend(torch, p, 0, dq, None, pos, out, heads, ws)
        outs.append(out)
    torch.cuda.synchronize()
    for b in list(range(len(SPECIALS))) + list(range(len(whats) - len(SPECIALS), len(whats))) * (copies > 1):
        check(torch, p, dq, None, b, n, out, heads)
    assert torch.equal(outs[0].view(torch.int32), outs[1].view(torch.int32))


def test_attend_infinite_query(torch):
    """A query that is not finite makes its heads NaN and no other."""
    heads, kv, d, n = 8, 2, 64, 130
    for cache in (0, 1, 2):
        p = Pool(torch, cache, [n + 1] * 2, kv, d, 16, seed=1)
        qkv = torch.randn((2, (heads + 2 * kv) * d), generator=T.gen(torch, 6))
        rows = qkv.view(2, heads + 2 * kv, d)
        rows[0, 1, 5], rows[1, 6, 9] = math.inf, math.nan
        dq, out = qkv.cuda(), torch.empty((2, heads * d), device="cuda")
        pos = torch.full((2,), n, dtype=torch.int32, device="cuda")
        T.attend(torch, p, 0, dq, None, pos, out, heads, T.workspace(torch, p.c, heads))
        bad = out.view(2, heads, d).isnan()
        want = torch.zeros_like(bad)
        want[0, 1] = want[1, 6] = True
        assert torch.equal(bad, want)
        for b in range(2):
            check(torch, p, dq, None, b, n, out, heads)


def chunks(pos):
    return [n // 64 + 1 if n >= 0 else 1 for n in pos]


LONG = [
    # dtype, cache, batch, heads, kv, d, page, longest
    (1, 1, 70, 32, 8, 128, 64, 4000),
    (0, 2, 70, 32, 8, 64, 24, 3000),
    (2, 2, 66, 64, 4, 128, 32, 5000),
    (0, 0, 70, 26, 2, 64, 100, 6000),
    (0, 0, 45, 20, 4, 128, 16, 3000),
    (0, 1, 130, 64, 4, 64, 16, 2500),
]


@pytest.mark.parametrize("dtype,cache,batch,heads,kv,d,page,longest", LONG)
def test_attend_many_long_sequences(torch, dtype, cache, batch, heads, kv, d, page, longest):
    """More than eight chunks a CTA: stretches cross heads and sequences, and each warp's loop runs long.  Slots without
    a sequence and positions out of range lie among them."""
    t = T.types(torch)[dtype]
    g = T.gen(torch, batch + d)
    pos = [max(0, int(longest * (i + 1) / batch) - 1) for i in torch.randperm(batch, generator=g).tolist()]
    pos[3], pos[40] = -1, -1
    blocks = (heads // kv + 15) // 16 if heads // kv > 8 else 1
    grid = torch.cuda.get_device_properties(0).multi_processor_count * 3
    assert sum(chunks(pos)) * kv * blocks > 8 * grid
    p = Pool(torch, cache, [n + 1 for n in pos], kv, d, page, seed=batch)
    rope = T.rope_table(torch, longest + 1, d).cuda()
    given = list(pos)
    given[7], given[35] = -9, longest + 100  # no position of this cache
    d_pos = torch.tensor(given, dtype=torch.int32, device="cuda")
    ws, outs = T.workspace(torch, p.c, heads), []
    qkv = torch.randn((batch, (heads + 2 * kv) * d), generator=g).to(t).cuda()
    for _ in range(2):
        out = torch.full((batch + 1, heads * d), 5.0, dtype=t, device="cuda")
        T.attend(torch, p, dtype, qkv, rope, d_pos, out, heads, ws)
        outs.append(out)
    assert (out[batch] == 5).all() and (out[[3, 40]] == 0).all() and out[[7, 35]].isnan().all()
    as_int = torch.int32 if t == torch.float32 else torch.int16
    assert torch.equal(outs[0].view(as_int), outs[1].view(as_int))
    for b in sorted(set(range(0, batch, 5)) | {0, 1, 31, 32, 33, batch - 1}):
        if b not in (3, 7, 35, 40):
            check(torch, p, qkv, rope, b, pos[b], out, heads)


@CACHES
@pytest.mark.parametrize("batch,heads,kv,d", [(60, 16, 8, 64), (33, 64, 16, 128), (200, 24, 4, 64)])
def test_attend_more_pairs_than_ctas(torch, cache, batch, heads, kv, d):
    """More pairs than CTAs but few chunks: single chunks are cut across pairs and sequences."""
    g = T.gen(torch, batch)
    pos = [int(x) for x in torch.randint(0, 64, (batch,), generator=g)]
    pos[1], pos[batch - 2], pos[batch // 2] = 700, 300, -1
    grid = torch.cuda.get_device_properties(0).multi_processor_count * 3
    assert grid < sum(chunks(pos)) * kv < 8 * grid and batch * kv > grid
    p = Pool(torch, cache, [n + 1 for n in pos], kv, d, 16, seed=batch)
    rope = T.rope_table(torch, 701, d).cuda()
    d_pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    qkv = torch.randn((batch, (heads + 2 * kv) * d), generator=g).cuda()
    ws, outs = T.workspace(torch, p.c, heads), []
    for _ in range(2):
        out = torch.empty((batch, heads * d), device="cuda")
        T.attend(torch, p, 0, qkv, rope, d_pos, out, heads, ws)
        outs.append(out)
    assert torch.equal(*outs)
    for b, n in enumerate(pos):
        if n < 0:
            assert (out[b] == 0).all()
        else:
            check(torch, p, qkv, rope, b, n, out, heads)


def test_attend_on_two_streams_at_once(torch):
    """Two captured calls, each with a workspace of its own, replayed together many times: each holds to its 64-bit form,
    and every replay gives the same bits."""
    sides = []
    for i, (cache, batch, heads, kv, d, n) in enumerate([(1, 40, 32, 8, 128, 900), (2, 70, 12, 4, 64, 300)]):
        pos = [max(0, n * (b + 1) // batch - 1) for b in range(batch)]
        p = Pool(torch, cache, [x + 1 for x in pos], kv, d, 16, seed=i)
        if i:
            p.put("v", 5, 0, math.inf)
        qkv = torch.randn((batch, (heads + 2 * kv) * d), generator=T.gen(torch, i)).cuda()
        out, dp = torch.empty((batch, heads * d), device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")
        ws, stream, graph = T.workspace(torch, p.c, heads), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(5):
                T.attend(torch, p, 0, qkv, None, dp, out, heads, ws, stream=stream)
        sides.append((p, qkv, pos, out, heads, ws, stream, graph, dp))
    first = None
    for _ in range(10):
        for side in sides:
            with torch.cuda.stream(side[6]):
                side[7].replay()
        torch.cuda.synchronize()
        now = [side[3].view(torch.int32).clone() for side in sides]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))
    for p, qkv, pos, out, heads, *_ in sides:
        for b, n in enumerate(pos):
            check(torch, p, qkv, None, b, n, out, heads)


# ---- the product -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m,k", [(9, 130, 129), (12, 514, 2050), (16, 1000, 1536), (16, 20010, 300), (5, 40002, 272),
                                   (10, 256, 4096), (1, 80002, 130), (15, 600, 513)])
def test_linear_up_to_16_tokens(torch, dtype, n, m, k):
    """Features on the TMEM lanes with 16 token columns: K whole and split over 2, 4 and 8 CTAs, partial tiles."""
    T.test_linear(torch, dtype, n, m, k)


def test_linear_on_several_streams_against_64_bits(torch):
    """Calls of different shapes under way together, each held to its 64-bit form."""
    cases = []
    for i, (n, m, k) in enumerate([(8, 4608, 1536), (16, 1536, 4096), (32, 4608, 1536), (64, 1536, 4096), (100, 1536, 1536),
                                   (300, 4608, 1536), (12, 512, 2048)]):
        g = T.gen(torch, i + 50)
        (dx, x), (dw, w) = T.random_fp8(torch, n, k, g), T.random_fp8(torch, m, k, g)
        xs, ws = torch.rand((n, k // 128), generator=g), torch.rand((m // 128, k // 128), generator=g) * 1e-3
        cases.append((n, m, k, dx, dw, xs.cuda(), ws.cuda(), torch.empty((n, m), device="cuda"), torch.cuda.Stream(), x, w))
    torch.cuda.synchronize()
    for _ in range(20):
        for n, m, k, dx, dw, xs, ws, y, stream, _, _ in cases:
            X.check(X.lib().xl_op_linear_fp8(0, 0, X.ptr(dx), dx.stride(0), X.ptr(xs), X.ptr(dw), dw.stride(0), X.ptr(ws), None,
                                             X.ptr(y), n, m, k, C.c_void_p(stream.cuda_stream)))
    torch.cuda.synchronize()
    for n, m, k, dx, dw, xs, ws, y, stream, x, w in cases:
        want, bound = T.linear_reference(torch, 0, x, xs.cpu(), w, ws.cpu(), None, None)
        assert ((y.cpu().double() - want).abs() <= bound + U * want.abs()).all(), (n, m, k)


@pytest.mark.parametrize("n", [3, 12, 20, 100, 1100])
def test_linear_swiglu_of_large_negative_gates(torch, n):
    """silu(v) is v e^v to the end of the floats' range: gates of -60 to -91.5, where e^-v passes it, times 2^60."""
    m, k = 2602, 130
    g = T.gen(torch, n)
    dx, dw = (torch.zeros((r, T.pitch(k)), dtype=torch.uint8, device="cuda") for r in (n, m))
    xs, ws = torch.zeros((n, 2), device="cuda"), torch.zeros(((m + 127) // 128, 2), device="cuda")
    bias = torch.empty(m)
    bias[0::2] = -(60 + 31.5 * torch.rand(m // 2, generator=g))
    bias[1::2] = 2.0 ** 60
    y = torch.empty((n, m // 2), device="cuda")
    db = bias.cuda()
    X.check(X.lib().xl_op_linear_fp8(1, 0, X.ptr(dx), dx.stride(0), X.ptr(xs), X.ptr(dw), dw.stride(0), X.ptr(ws), X.ptr(db),
                                     X.ptr(y), n, m, k, X.stream()))
    v = bias[0::2].double()
    want = (v * torch.sigmoid(v) * bias[1::2].double()).expand(n, -1)
    off = (y.cpu().double() - want).abs() / want.abs()
    assert float(off.max()) <= 16 * U, float(off.max())


# ---- the norm --------------------------------------------------------------------------------------------------------

def near_ties(torch, groups, t, seed):
    """r, gamma of one row whose groups each hold two largest products that round to one fp32 number and differ: the
    larger comes second, a few lanes on, in the same lane, or at the group's end."""
    g = T.gen(torch, seed)
    r = (torch.randn(groups * 128, generator=g) * 0.05).to(t)
    gamma = torch.rand(groups * 128, generator=g) * 0.5 + 0.5
    for i in range(groups):
        first, second = i * 128 + 8 * (i % 13) + 1, i * 128 + [8 * (i % 13) + 5, 8 * (i % 13) + 20, 127][i % 3]
        while True:
            a, b = ((torch.rand(2, generator=g) + 1) * 2).to(t)
            wa = torch.rand((), generator=g) + 1
            product = (a.double() * wa.double())
            wb = (product / b.double()).float()
            for _ in range(2):
                exact = b.double() * wb.double()
                if exact > product and exact.float() == product.float():
                    break
                wb = torch.nextafter(wb, torch.tensor(math.inf))
            else:
                continue
            break
        r[first], gamma[first], r[second], gamma[second] = a, wa, b, wb
    return r, gamma


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("groups,n", [(8, 1), (64, 3), (64, 400), (250, 2)])
def test_norm_scale_of_tied_products(torch, dtype, groups, n):
    """The scale is made of the largest exact product, also where another one rounds to the same fp32 number."""
    t, k = T.types(torch)[dtype], groups * 128
    r, gamma = near_ties(torch, groups, t, groups + dtype)
    res = (r.float() * 2.0 ** torch.arange(n).remainder(5)[:, None]).to(t)  # powers of two keep the ties
    d_res, d_gamma = res.cuda(), gamma.cuda()
    q, s = torch.empty((n, k), dtype=torch.uint8, device="cuda"), torch.empty((n, groups), device="cuda")
    X.check(X.lib().xl_op_add_rmsnorm_fp8(dtype, None, X.ptr(d_res), None, X.ptr(d_gamma), X.ptr(q), k, X.ptr(s), n, k,
                                          X.stream()))
    some = list(range(min(n, 5)))
    _, (want_q, want_s) = T.norm_reference(torch, None, res[some], gamma)
    T.same(torch, s[some], want_s)
    T.same(torch, q[some].view(torch.float8_e4m3fn), want_q)
