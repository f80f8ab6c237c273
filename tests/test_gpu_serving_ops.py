"""The 8-bit projections and the paged cache (xl_op_quantize_fp8,
xl_op_add_rmsnorm_fp8, xl_op_linear_fp8, xl_op_kv_append_paged,
xl_op_attn_decode_paged) against plain 64-bit forms.

Tolerances.  u = 2^-24 is half a step of fp32.
* Bytes and scales are compared for equality: the bytes are defined as the
  nearest e4m3 value to the exact quotient by the stored scale.
* Sums of fp32 terms: a sum of N terms in any order is off by at most
  N 2u sum|terms| (2u a step also covers an accumulator that truncates).
* A result stored as type t adds half a step of t.
* Attention: a score is off by ds <= (D + 8) 2u (sum |q||k|) / sqrt(D) plus the
  rotation's 4u of the same magnitude and the operands' split (2^-21 of it); a
  weight is off by the factor exp(2 ds), its split by 2^-16, the sums over N
  positions by N 2u.  So the output is off by at most
  (2 ds + 2^-16 + (N + 16) 2u + 2^-20) sum_t w_t |v_t|.
"""
import ctypes as C
import math

import pytest

import xl_capi as X

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch(built):
    import torch

    torch.cuda.init()
    return torch


def types(torch):
    return {X.XL_F32: torch.float32, X.XL_BF16: torch.bfloat16, X.XL_F16: torch.float16}


def half_step(torch, t):
    return torch.finfo(t).eps / 2


def gen(torch, seed):
    return torch.Generator().manual_seed(seed)


def pitch(k):
    return (k + 15) // 16 * 16


GUARD = 0x5A


def fp8_out(torch, n, k):
    """Rows of pitch(k) bytes between guard bytes, so that a write outside shows."""
    return torch.full((n + 2, pitch(k)), GUARD, dtype=torch.uint8, device="cuda")


def e4m3_values(torch):
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return v[~v.isnan()].unique()


def nearest_e4m3(torch, x):
    """float64 -> the nearest e4m3 value (ties to an even last bit), by looking at both neighbours."""
    v = e4m3_values(torch)
    x = x.clamp(-448, 448).contiguous()
    hi = torch.searchsorted(v, x).clamp(1, len(v) - 1)
    a, b = v[hi - 1], v[hi]
    code = {float(t): i for i, t in enumerate(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double())
            if not math.isnan(float(t))}
    even = torch.tensor([code[float(t)] % 2 == 0 for t in v])
    up = (b - x < x - a) | ((b - x == x - a) & even[hi])
    return torch.where(up, b, a)


def quantise(torch, y, rows):
    """y float64 [n][k] -> (q values, scales), scale NaN where a group is not finite."""
    n, k = y.shape
    q = torch.empty_like(y)
    s = torch.empty(((n + rows - 1) // rows, (k + 127) // 128), dtype=torch.float64)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            part = y[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128]
            top = part.abs().max()
            sc = (top / 448).float().double() if torch.isfinite(part).all() else torch.tensor(math.nan, dtype=torch.float64)
            s[i, j] = sc
            if math.isnan(float(sc)):
                r = torch.full_like(part, math.nan)
            elif float(sc) == 0:
                r = torch.zeros_like(part)
            else:
                r = nearest_e4m3(torch, part / sc)
            q[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128] = r
    return q, s


def same(torch, got, want):
    """Equal, with NaN equal to NaN and the two zeros alike."""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    ok = (got == want) | (got.isnan() & want.isnan())
    assert ok.all(), (int((~ok).sum()), got[~ok][:4], want[~ok][:4])


def fp8_rows(torch, buf, n, k):
    """The values of rows 1 .. n of a guarded buffer, whose other bytes have to be untouched."""
    assert (buf[0] == GUARD).all() and (buf[n + 1] == GUARD).all() and (buf[:, k:] == GUARD).all()
    return buf[1:n + 1, :k].contiguous().view(torch.float8_e4m3fn).cpu().double()


def hard_values(torch, n, k, g, t):
    """Normal values with the places where rounding goes wrong among them: borders between e4m3 values (exact and
    next to exact), zeros, tiny and huge values, a group of zeros, groups that are not finite."""
    x = torch.randn((n, k), generator=g) * 0.05
    x[torch.rand((n, k), generator=g) < 0.05] = 0
    if n * k > 300:
        v = e4m3_values(torch)
        mid = ((v[1:] + v[:-1]) / 2).float()
        at = torch.randperm(min(n * k, 4096), generator=g)[:len(mid)]
        flat = x.view(-1)
        flat[at] = mid[:len(at)] * 2.0 ** -7  # the largest of these sets a scale near 2^-7
        flat[at[0]] = 448 * 2.0 ** -7
    if n > 2:
        x[1, :min(k, 128)] = 0
        x[2, :min(k, 128)] *= 1e-30 if t == torch.float32 else 1e-4
    if n > 4 and k > 256:
        x[3, 200] = math.inf
        x[4, 10] = math.nan
        x[4, 130:256] *= 3e4
    return x.to(t)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,k,rows,skew", [(1, 1, 1, 0), (3, 127, 1, 0), (5, 128, 1, 0), (8, 1536, 1, 0), (7, 4097, 1, 0),
                                           (33, 1000, 1, 24), (6, 520, 1, 1), (1, 1, 128, 0), (127, 129, 128, 0),
                                           (128, 128, 128, 0), (300, 1000, 128, 8), (257, 130, 128, 3)])
def test_quantize(torch, dtype, n, k, rows, skew):
    t = types(torch)[dtype]
    ldx = k + skew
    x = torch.zeros(n * ldx + skew, dtype=t)
    x = x[skew:].view(n, ldx)
    x[:, :k] = hard_values(torch, n, k, gen(torch, n * 1000 + k + dtype), t)
    x[:, k:] = 1e4  # between the rows: not part of them
    store = torch.zeros(n * ldx + skew, dtype=t, device="cuda")
    dx = store[skew:]  # an odd element offset where skew is odd
    dx.copy_(x.reshape(-1))
    q = fp8_out(torch, n, k)
    s = torch.full(((n + rows - 1) // rows * ((k + 127) // 128) + 2,), 7.0, device="cuda")
    X.check(X.lib().xl_op_quantize_fp8(dtype, X.ptr(dx), ldx, X.ptr(q[1]), q.stride(0), X.ptr(s[1:]), n, k, rows, X.stream()))
    torch.cuda.synchronize()
    want_q, want_s = quantise(torch, x[:, :k].double(), rows)
    assert s[0] == 7 and s[-1] == 7
    same(torch, s[1:-1].view(want_s.shape), want_s)
    same(torch, fp8_rows(torch, q, n, k), want_q)


@pytest.mark.parametrize("exponent", [-140, -126, -100, 60, 110])
def test_quantize_far_scales(torch, exponent):
    """Scales at both ends of fp32: their reciprocals or the values themselves leave the range of normal floats."""
    x = (torch.randn((4, 256), generator=gen(torch, 5)).double() * 2.0 ** exponent).float()
    q, s = fp8_out(torch, 4, 256), torch.empty((4, 2), device="cuda")
    dx = x.cuda()
    X.check(X.lib().xl_op_quantize_fp8(0, X.ptr(dx), 256, X.ptr(q[1]), q.stride(0), X.ptr(s), 4, 256, 1, X.stream()))
    torch.cuda.synchronize()
    want_q, want_s = quantise(torch, x.double(), 1)
    same(torch, s, want_s)
    same(torch, fp8_rows(torch, q, 4, 256), want_q)


def norm_reference(torch, delta, residual, gamma):
    r = residual if delta is None else (residual.float() + delta.float()).to(residual.dtype)
    y = r.double()
    y = y / (y.square().mean(1, keepdim=True) + 1e-6).sqrt() * gamma.double()
    return r, quantise(torch, y, 1)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,k,how", [(1, 1, "out"), (3, 64, "alias"), (2, 127, "none"), (8, 1536, "out"), (5, 2047, "alias"),
                                     (3, 2056, "none"), (3, 8192, "out"), (2, 9001, "out"), (1, 32768, "alias")])
def test_add_rmsnorm(torch, dtype, n, k, how):
    t = types(torch)[dtype]
    g = gen(torch, n + k + dtype)
    res = (torch.randn((n, k), generator=g) * 2).to(t)
    delta = None if how == "none" else (torch.randn((n, k), generator=g) * 0.5).to(t)
    gamma = torch.rand(k, generator=g) + 0.5
    gamma[torch.rand(k, generator=g) < 0.02] = 0
    if n > 2:
        res[1] = 0
        if delta is not None:
            delta[1] = 0  # a row of zeros: the norm's eps carries it
        res[2, k // 2] = math.inf if dtype else math.nan
    d_res, d_gamma = torch.cat([res, res[:1]]).cuda(), gamma.cuda()
    d_delta = None if delta is None else delta.cuda()
    out = None if how == "none" else d_res if how == "alias" else torch.full((n + 1, k), 3.0, dtype=t, device="cuda")
    q = fp8_out(torch, n, k)
    s = torch.full((n * ((k + 127) // 128) + 2,), 7.0, device="cuda")
    X.check(X.lib().xl_op_add_rmsnorm_fp8(dtype, X.ptr(d_delta), X.ptr(d_res), X.ptr(out), X.ptr(d_gamma), X.ptr(q[1]),
                                          q.stride(0), X.ptr(s[1:]), n, k, X.stream()))
    torch.cuda.synchronize()
    r, (want_q, want_s) = norm_reference(torch, delta, res, gamma)
    if out is not None:
        same(torch, out[:n], r)
        assert torch.equal(out[n].cpu(), res[0] if how == "alias" else torch.full((k,), 3.0, dtype=t))
    if how != "alias":
        same(torch, d_res[:n], res)
    assert s[0] == 7 and s[-1] == 7
    same(torch, s[1:-1].view(want_s.shape), want_s)
    same(torch, fp8_rows(torch, q, n, k), want_q)


def random_fp8(torch, n, k, g):
    """Device bytes [n][pitch] whose padding is NaN, the values in 64 bits, the scales."""
    v = (torch.randn((n, k), generator=g) * 120).clamp(-448, 448).to(torch.float8_e4m3fn)
    buf = torch.full((n, pitch(k)), 0x7F, dtype=torch.uint8)
    buf[:, :k] = v.view(torch.uint8)
    return buf.cuda(), v.double()


def spread(torch, s, size, dim):
    return s.repeat_interleave(128, dim).narrow(dim, 0, size)


def linear_reference(torch, mode, x, xs, w, ws, bias, y0):
    """(y, its bound without the output's own rounding) in 64 bits."""
    n, k = x.shape
    m = w.shape[0]
    xd = x * spread(torch, xs.double(), k, 1)
    wd = w * spread(torch, spread(torch, ws.double(), k, 1), m, 0)
    b = torch.zeros(m, dtype=torch.float64) if bias is None else bias.double()
    y = xd @ wd.T + b
    blocks = xs.shape[1]
    err = (min(k, 128) + blocks + 6) * 2 * U * (xd.abs() @ wd.abs().T + b.abs())
    if mode == 1:
        a, c, ea, ec = y[:, 0::2], y[:, 1::2], err[:, 0::2], err[:, 1::2]
        h = a * torch.sigmoid(a) * c
        # |silu'| <= 1.1; expf, the division and the products: 8 steps
        return h, 1.1 * ea * (c.abs() + ec) + (a * torch.sigmoid(a)).abs() * ec + 16 * U * h.abs()
    if mode == 2:
        return y + y0.double(), err + 2 * U * (y + y0.double()).abs()
    return y, err


LINEAR_SHAPES = [(1, 2, 1), (1, 130, 16), (2, 128, 128), (8, 576, 192), (17, 200, 300), (33, 384, 1536), (64, 256, 513),
                 (65, 1000, 257), (130, 258, 129), (300, 514, 1000), (257, 512, 2048), (1, 1030, 4096), (700, 1290, 640),
                 (3, 20010, 130), (1100, 2602, 200), (2100, 2706, 257), (1090, 2608, 640), (1500, 2336, 1050),
                 (100, 1000, 513), (128, 770, 256)]


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m,k", LINEAR_SHAPES)
def test_linear(torch, dtype, n, m, k):
    t = types(torch)[dtype]
    g = gen(torch, n + 3 * m + 7 * k + dtype)
    (dx, x), (dw, w) = random_fp8(torch, n, k, g), random_fp8(torch, m, k, g)
    blocks = (k + 127) // 128
    xs = torch.rand((n, blocks), generator=g) * 2.0 ** -6 + 1e-4
    ws = torch.rand(((m + 127) // 128, blocks), generator=g) * 2.0 ** -10 + 1e-6
    if n > 2:
        xs[1] *= 1000
        xs[2] = 0
    bias = torch.randn(m, generator=g) * 0.1
    dxs, dws, db = xs.cuda(), ws.cuda(), bias.cuda()
    for mode in (0, 1, 2):
        wide = m // 2 if mode == 1 else m
        y0 = torch.randn((n, wide), generator=g).to(t)
        # what lies before and behind y (16-byte aligned) has to stay
        lead = (wide * t.itemsize + 15) // 16 * 16 // t.itemsize
        flat = torch.full((lead + n * wide + lead,), 9.0, dtype=t, device="cuda")
        out = flat[lead:lead + n * wide].view(n, wide)
        out.copy_(y0)
        use = mode != 0 or n % 2 == 1
        X.check(X.lib().xl_op_linear_fp8(mode, dtype, X.ptr(dx), dx.stride(0), X.ptr(dxs), X.ptr(dw), dw.stride(0),
                                         X.ptr(dws), X.ptr(db) if use else None, X.ptr(out), n, m, k, X.stream()))
        torch.cuda.synchronize()
        want, bound = linear_reference(torch, mode, x, xs, w, ws, bias if use else None, y0)
        got = out.cpu().double()
        # a value past the type's largest (fp16: silu(a) c of row 1, scaled by 1000, passes 65504) is stored as infinity:
        # round-to-nearest overflows from max (1 + half a step) on, so there the sign is what is left to compare
        most = torch.finfo(t).max
        over = got.isinf() & (want.abs() + bound > most)
        assert (torch.sign(got) == torch.sign(want))[over].all()
        off = (got - want).abs() - bound - half_step(torch, t) * (want.abs() + bound) - torch.finfo(t).tiny * 2 ** -3
        off[over] = 0
        assert (off <= 0).all(), (mode, float(off.max()), torch.nonzero(off > 0)[:4])
        assert (flat[:lead] == 9).all() and (flat[lead + n * wide:] == 9).all()


def test_linear_infinite_and_nan_scales_stay_in_their_rows(torch):
    """A row whose scale is NaN (a group that was not finite) is NaN, and only that row."""
    g = gen(torch, 4)
    (dx, x), (dw, w) = random_fp8(torch, 140, 256, g), random_fp8(torch, 192, 256, g)
    xs, ws = torch.full((140, 2), 0.01), torch.full((2, 2), 0.01)
    xs[133, 1] = math.nan
    dxs, dws = xs.cuda(), ws.cuda()
    y = torch.empty((140, 192), device="cuda")
    X.check(X.lib().xl_op_linear_fp8(0, 0, X.ptr(dx), dx.stride(0), X.ptr(dxs), X.ptr(dw), dw.stride(0), X.ptr(dws), None,
                                     X.ptr(y), 140, 192, 256, X.stream()))
    torch.cuda.synchronize()
    bad = y.isnan().cpu()
    assert bad[133].all() and not bad[:133].any() and not bad[134:].any()


@pytest.mark.parametrize("n,m,k", [(3, 520, 384), (20, 520, 384), (100, 520, 384), (1100, 2600, 256)])
def test_linear_nan_operands(torch, n, m, k):
    """An e4m3 NaN makes its token's row, or its weight row's column, NaN, and nothing else."""
    g = gen(torch, n)
    (dx, x), (dw, w) = random_fp8(torch, n, k, g), random_fp8(torch, m, k, g)
    dx[n - 1, 130], dw[m - 3, 7] = 0x7F, 0xFF
    xs, ws = torch.full((n, k // 128), 0.01, device="cuda"), torch.full(((m + 127) // 128, k // 128), 0.01, device="cuda")
    y = torch.empty((n, m), device="cuda")
    X.check(X.lib().xl_op_linear_fp8(0, 0, X.ptr(dx), dx.stride(0), X.ptr(xs), X.ptr(dw), dw.stride(0), X.ptr(ws), None,
                                     X.ptr(y), n, m, k, X.stream()))
    torch.cuda.synchronize()
    want = torch.zeros((n, m), dtype=torch.bool)
    want[n - 1] = True
    want[:, m - 3] = True
    assert torch.equal(y.isnan().cpu(), want)


# ---- the paged cache ------------------------------------------------------------------------------------------------

class Paged:
    """A pool whose pages are handed out in a shuffled order; what no position holds is NaN (or the type's largest)."""

    def __init__(self, torch, dtype, lens, kv, d, page, seed, room=1, spare=2):
        self.torch, self.page, self.kv, self.d = torch, page, kv, d
        t = types(torch)[dtype]
        g = gen(torch, seed)
        need = [max(0, (n + page - 1) // page) for n in lens]
        self.max_pages = max(need + [1]) + room
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.table = torch.full((len(lens), self.max_pages), 1 << 30, dtype=torch.int32)  # past the need: never read
        at = 0
        for b, c in enumerate(need):
            self.table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
        self.k = torch.full((total, kv, page, d), math.nan, dtype=t)
        self.v = torch.full((total, kv, page, d), math.nan, dtype=t)
        self.v[..., ::2] = math.inf
        for b, n in enumerate(lens):
            for p in range(n):
                pg = int(self.table[b, p // page])
                self.k[pg, :, p % page] = torch.randn((kv, d), generator=g).to(t)
                self.v[pg, :, p % page] = torch.randn((kv, d), generator=g).to(t)
        self.dk, self.dv, self.dt = self.k.cuda(), self.v.cuda(), self.table.cuda()
        self.c = X.PagedKV(self.dk.data_ptr(), self.dv.data_ptr(), self.dt.data_ptr(), dtype, len(lens), kv, d, page,
                           self.max_pages, total)

    def rows(self, b, n):
        """Positions 0 .. n - 1 of sequence b as the device holds them now, [kv][n][d] in 64 bits."""
        pages = self.table[b, :(n + self.page - 1) // self.page].long()
        return tuple(x.cpu()[pages].permute(1, 0, 2, 3).reshape(self.kv, -1, self.d)[:, :n].double() for x in (self.dk, self.dv))


def rope_table(torch, length, d):
    a = torch.arange(length, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * torch.arange(d // 2, dtype=torch.float64) / d)
    return torch.stack([a.cos(), a.sin()], -1).float()


def rotate(torch, x, cs):
    a, b = x.double().chunk(2, -1)
    c, s = cs[..., 0].double(), cs[..., 1].double()
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def workspace(torch, cache, heads):
    n = X.lib().xl_op_attn_decode_paged_workspace_bytes(C.byref(cache), heads)
    assert n > 0
    return torch.zeros(n, dtype=torch.uint8, device="cuda")


def attend(torch, p, dtype, qkv, rope, pos, out, heads, ws, stream=None):
    X.check(X.lib().xl_op_attn_decode_paged(C.byref(p.c), dtype, X.ptr(qkv), X.ptr(rope), 0 if rope is None else rope.shape[0],
                                            X.ptr(pos), X.ptr(out), heads, X.ptr(ws), ws.numel(),
                                            X.stream() if stream is None else C.c_void_p(stream.cuda_stream)))


def check_attention(torch, p, qkv, rope, pos, out, heads):
    """out [batch][heads * d] against 64 bits over what the cache holds; the new rows themselves too."""
    t, store, d, kv = qkv.dtype, p.k.dtype, p.d, p.kv
    group = heads // kv
    rows = qkv.view(len(pos), heads + 2 * kv, d)
    for b, n in enumerate(pos):
        got = out[b].double().cpu().view(heads, d)
        if n < 0:
            assert (got == 0).all()
            continue
        q, k_new, v_new = rows[b, :heads], rows[b, heads:heads + kv], rows[b, heads + kv:]
        size = lambda x: x.double().abs()  # noqa: E731
        qr, kr = q.double(), k_new.double()
        err_k = torch.zeros_like(kr)
        if rope is not None:
            qr, kr = rotate(torch, q, rope[n]), rotate(torch, k_new, rope[n])
            pair = size(k_new)
            err_k = 4 * U * (pair + pair.roll(d // 2, -1))
        kk, vv = p.rows(b, n + 1)
        off = (kk[:, n] - kr).abs() - err_k - half_step(torch, store) * (kr.abs() + err_k) - torch.finfo(store).tiny
        assert (off <= 0).all(), (b, float(off.max()))
        assert torch.equal(vv[:, n], v_new.to(store).double())
        for h in range(heads):
            keys, values = kk[h // group], vv[h // group]
            s = keys @ qr[h] / math.sqrt(d)
            w = torch.softmax(s, 0)
            want = w @ values
            big = size(q[h]) + size(q[h]).roll(d // 2)
            ds = ((d + 8) * 2 * U + 8 * U + 2.0 ** -21) * float((keys.abs() @ big).max()) / math.sqrt(d)
            tol = (2 * ds + 2.0 ** -16 + (n + 17) * 2 * U + 2.0 ** -20) * (w @ values.abs())
            off = (got[h] - want).abs() - tol - half_step(torch, t) * (want.abs() + tol) - torch.finfo(t).tiny
            assert (off <= 0).all(), (b, h, float(off.max()), float(tol.max()))


ATTEND = [
    # dtype, cache, heads, kv, d, page, positions of the new tokens
    (0, 0, 24, 24, 64, 16, [0, 1, 15, 16, 17, 767, -1, 200]),
    (0, 0, 4, 1, 128, 32, [0, 31, 32, 333]),
    (1, 1, 32, 8, 128, 64, [500, -1, 0, 63, 64, 1023]),
    (2, 2, 6, 2, 64, 24, [47, 48, 49, 5]),
    (0, 1, 16, 2, 64, 100, [99, 100, 250]),
    (1, 0, 5, 5, 128, 1, [0, 7, 40]),
    (2, 1, 40, 2, 64, 8, [130, 7, 8]),
    (0, 2, 17, 1, 128, 13, [12, 13, 77]),
    (1, 2, 64, 1, 64, 128, [127, 128, 300]),
    (1, 1, 3, 3, 64, 7, [0]),
    (0, 0, 1, 1, 64, 256, [2047]),
    (1, 1, 8, 1, 128, 16, [3000]),
    (2, 2, 2, 1, 128, 48, [-1, -1]),
    (0, 0, 12, 1, 128, 8, [0, 300, 64]),
    (0, 0, 26, 2, 64, 16, [90, 1]),
    (1, 2, 10, 1, 128, 32, [65, 400]),
]


@pytest.mark.parametrize("dtype,cache,heads,kv,d,page,pos", ATTEND)
def test_attend(torch, dtype, cache, heads, kv, d, page, pos):
    t = types(torch)[dtype]
    p = Paged(torch, cache, [n + 1 for n in pos], kv, d, page, seed=heads + d + page)
    g = gen(torch, 77 + heads)
    rope = rope_table(torch, max(pos + [0]) + 1, d) if heads != 5 else None
    d_rope = None if rope is None else rope.cuda()
    d_pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    ws = workspace(torch, p.c, heads)
    for _ in range(2):  # the workspace comes back ready
        qkv = torch.randn((len(pos), (heads + 2 * kv) * d), generator=g).to(t)
        d_qkv = qkv.cuda()
        out = torch.full((len(pos) + 1, heads * d), 5.0, dtype=t, device="cuda")
        before = (p.dk.clone(), p.dv.clone())
        attend(torch, p, dtype, d_qkv, d_rope, d_pos, out, heads, ws)
        torch.cuda.synchronize()
        assert (out[len(pos)] == 5).all()
        check_attention(torch, p, qkv, rope, pos, out, heads)
        # everything but the new rows is as it was
        for now, then in zip((p.dk, p.dv), before):
            now, then = now.cpu(), then.cpu()
            for b, n in enumerate(pos):
                if n >= 0:
                    now[int(p.table[b, n // page]), :, n % page] = then[int(p.table[b, n // page]), :, n % page]
            assert torch.equal(now.view(torch.int16 if now.element_size() == 2 else torch.int32),
                               then.view(torch.int16 if now.element_size() == 2 else torch.int32))


@pytest.mark.parametrize("cache", [0, 1], ids=["fp32", "bf16"])
def test_attend_scores_of_any_size(torch, cache):
    """One position takes all the weight, wherever it lies; equal scores share it; scores of +-1e4 do not overflow."""
    heads, kv, d, n = 4, 2, 64, 300
    p = Paged(torch, cache, [n + 1] * 3, kv, d, 16, seed=3)
    qkv = torch.zeros((3, (heads + 2 * kv) * d))
    qkv[:, :heads * d] = 8.0
    for b, spot in enumerate((0, 150, n)):
        for t in range(n + 1):
            page, slot = int(p.table[b, t // 16]), t % 16
            p.k[page, :, slot] = 100.0 if t == spot else -100.0 if b == 1 else 0.0
    qkv[2, heads * d:(heads + kv) * d] = 100.0
    p.dk.copy_(p.k)
    out = torch.empty((3, heads * d), device="cuda")
    pos = torch.full((3,), n, dtype=torch.int32, device="cuda")
    dq = qkv.cuda()
    attend(torch, p, 0, dq, None, pos, out, heads, workspace(torch, p.c, heads))
    torch.cuda.synchronize()
    check_attention(torch, p, qkv, None, [n] * 3, out, heads)


def test_attend_out_of_range_positions_and_pages(torch):
    """A position that the table or the rope table cannot hold, and a page id outside the pool: NaN for that
    sequence alone; the cache is changed only where a good page takes a new row."""
    heads, kv, d, page = 4, 2, 64, 16
    lens = [20, 20, 20, 20, 20, 20]
    p = Paged(torch, 1, lens, kv, d, page, seed=9, room=0)
    p.table[2, 0] = -1                 # a bad page before the new row's
    p.table[3, 1] = p.k.shape[0]       # the new row's own page
    p.dt.copy_(p.table)
    pos = [19, 2 * page, 19, 19, -5, 19]
    qkv = torch.randn((6, (heads + 2 * kv) * d), generator=gen(torch, 1))
    rope = rope_table(torch, 2 * page, d)
    out = torch.empty((6, heads * d), device="cuda")
    before = p.dk.clone()
    dq, dr, dp = qkv.cuda(), rope.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda")
    ws = workspace(torch, p.c, heads)
    attend(torch, p, 0, dq, dr, dp, out, heads, ws)
    torch.cuda.synchronize()
    for b in (1, 2, 3, 4):
        assert out[b].isnan().all(), b
    changed = (p.dk.view(torch.int16) != before.view(torch.int16)).any(-1).any(1)  # [page][slot]
    allowed = torch.zeros_like(changed)
    for b in (0, 2, 5):
        allowed[int(p.table[b, 1]), 3] = True
    assert not (changed & ~allowed).any() and changed[int(p.table[0, 1]), 3]
    p.table[2:5] = 0
    for b in (0, 5):
        one = type(p).__new__(type(p))
        one.__dict__.update(p.__dict__)
        one.table = p.table[b:b + 1]
        check_attention(torch, one, qkv[b:b + 1], rope, [19], out[b:b + 1], heads)
    # the rope table is shorter than the position
    short = dr[:10].contiguous()
    attend(torch, p, 0, dq, short, dp, out, heads, ws)
    torch.cuda.synchronize()
    assert out.isnan().all()


def test_attend_shared_prefix_pages(torch):
    """Two sequences whose first pages are the same pages."""
    heads, kv, d, page = 8, 2, 128, 16
    p = Paged(torch, 2, [70, 70], kv, d, page, seed=2)
    p.table[1, :3] = p.table[0, :3]
    p.dt.copy_(p.table)
    pos = [66, 69]
    qkv = torch.randn((2, (heads + 2 * kv) * d), generator=gen(torch, 8)).half()
    rope = rope_table(torch, 70, d)
    out = torch.empty((2, heads * d), dtype=torch.float16, device="cuda")
    dq, dr, dp = qkv.cuda(), rope.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda")
    attend(torch, p, 2, dq, dr, dp, out, heads, workspace(torch, p.c, heads))
    torch.cuda.synchronize()
    check_attention(torch, p, qkv, rope, pos, out, heads)


def test_attend_one_workspace_for_calls_of_unlike_shapes(torch):
    """Calls in a row on one stream share a workspace, whatever their batch and heads; each repeats bit for bit."""
    big = Paged(torch, 1, [900, 30, 513], 2, 64, 16, seed=5)
    small = Paged(torch, 1, [400] * 7, 4, 64, 32, seed=6)
    ws = workspace(torch, big.c, 16)
    need = X.lib().xl_op_attn_decode_paged_workspace_bytes(C.byref(small.c), 4)
    if need > ws.numel():
        ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    rope = rope_table(torch, 1000, 64).cuda()
    runs = []
    for p, heads, pos in ((big, 16, [899, 29, 512]), (small, 4, [399] * 7)) * 2:
        qkv = torch.randn((len(pos), (heads + 2 * p.kv) * 64), generator=gen(torch, heads)).bfloat16().cuda()
        out = torch.empty((len(pos), heads * 64), dtype=torch.bfloat16, device="cuda")
        dp = torch.tensor(pos, dtype=torch.int32, device="cuda")
        attend(torch, p, 1, qkv, rope, dp, out, heads, ws)
        runs.append((p, qkv, pos, out, heads))
    torch.cuda.synchronize()
    for p, qkv, pos, out, heads in runs:
        check_attention(torch, p, qkv.cpu(), rope.cpu(), pos, out, heads)
    assert torch.equal(runs[0][3], runs[2][3]) and torch.equal(runs[1][3], runs[3][3])


def test_attend_captured_and_on_another_stream(torch):
    """A captured call replays with new inputs and positions in place, on a stream of its own."""
    heads, kv, d, page = 24, 24, 64, 16
    p = Paged(torch, 0, [100, 40], kv, d, page, seed=12)
    rope = rope_table(torch, 128, d)
    dr = rope.cuda()
    qkv = torch.zeros((2, (heads + 2 * kv) * d), device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros((2, heads * d), device="cuda")
    ws = workspace(torch, p.c, heads)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        attend(torch, p, 0, qkv, dr, pos, out, heads, ws, stream=side)
    for step in ([97, 37], [98, 38], [99, -1]):
        host = torch.randn(tuple(qkv.shape), generator=gen(torch, step[0]))
        qkv.copy_(host)
        pos.copy_(torch.tensor(step, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(torch, p, host, rope, step, out, heads)


@pytest.mark.parametrize("dtype,cache,heads,kv,d,page", [(0, 0, 24, 24, 64, 16), (1, 1, 32, 8, 128, 32), (2, 0, 4, 4, 64, 7),
                                                         (0, 2, 6, 3, 128, 100), (1, 2, 2, 1, 64, 1)])
@pytest.mark.parametrize("with_rope", [True, False], ids=["rope", "asis"])
def test_append(torch, dtype, cache, heads, kv, d, page, with_rope):
    """Ragged prompts behind what is held already; rows out of range are skipped, everything else stays."""
    t, store = types(torch)[dtype], types(torch)[cache]
    lens = [37, 5, 130]
    p = Paged(torch, cache, lens, kv, d, page, seed=d + page, room=0)
    p.table[p.table == 1 << 30] = -1
    p.dt.copy_(p.table)
    seq = [0] * 20 + [2] * 129 + [1] + [0, 3, -1, 1, 0, 2]
    pos = list(range(17, 37)) + list(range(1, 130)) + [4] + [p.max_pages * page, 0, 0, -1, 1 << 30, -7]
    live = 20 + 129 + 1
    rows = len(seq)
    qkv = torch.randn((rows, (heads + 2 * kv) * d), generator=gen(torch, 3)).to(t)
    rope = rope_table(torch, p.max_pages * page + 1, d) if with_rope else None
    dr = None if rope is None else rope.cuda()
    dq, ds, dp = qkv.cuda(), torch.tensor(seq, dtype=torch.int32, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")
    before = p.dk.clone(), p.dv.clone()
    X.check(X.lib().xl_op_kv_append_paged(C.byref(p.c), dtype, X.ptr(dq), X.ptr(dr), 0 if rope is None else rope.shape[0],
                                          X.ptr(ds), X.ptr(dp), rows, heads, X.stream()))
    torch.cuda.synchronize()
    now, then = [x.cpu() for x in (p.dk, p.dv)], [x.cpu() for x in before]
    split = qkv.view(rows, heads + 2 * kv, d)
    for i in range(live):
        pg, slot = int(p.table[seq[i], pos[i] // page]), pos[i] % page
        k = split[i, heads:heads + kv]
        want = k.double() if rope is None else rotate(torch, k, rope[pos[i]])
        size = k.double().abs()
        err = 0 * size if rope is None else 4 * U * (size + size.roll(d // 2, -1))
        off = (now[0][pg, :, slot].double() - want).abs() - err - half_step(torch, store) * (want.abs() + err) - \
            torch.finfo(store).tiny
        assert (off <= 0).all()
        assert torch.equal(now[1][pg, :, slot], split[i, heads + kv:].to(store))
        for x, y in zip(now, then):
            x[pg, :, slot] = y[pg, :, slot]
    for x, y in zip(now, then):
        as_int = torch.int16 if x.element_size() == 2 else torch.int32
        assert torch.equal(x.view(as_int), y.view(as_int))


# ---- a layer's serving step ------------------------------------------------------------------------------------------

def test_layer_step(torch):
    """A prompt appended, then decode steps of three sequences through one layer with 8-bit weights, every operator
    called as a serving loop calls it, captured into a graph and replayed.  Each operator's output is held to its own
    64-bit form on the inputs that it got, and the last hidden rows to a 64-bit layer over the same e4m3 weights."""
    hidden, heads, kv, d, ffn, page, batch = 256, 4, 2, 64, 512, 16, 3
    g = gen(torch, 21)
    lib, st = X.lib(), X.stream
    dev = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731

    def weight(m, k):
        w = (torch.randn((m, k), generator=g) * k ** -0.5).cuda()
        q, s = dev(m, pitch(k), dt=torch.uint8), dev((m + 127) // 128, (k + 127) // 128)
        X.check(lib.xl_op_quantize_fp8(0, X.ptr(w), k, X.ptr(q), pitch(k), X.ptr(s), m, k, 128, st()))
        torch.cuda.synchronize()
        return q, s

    qkv_m = (heads + 2 * kv) * d
    weights = {n: weight(m, k) for n, m, k in (("qkv", qkv_m, hidden), ("o", hidden, heads * d), ("w13", 2 * ffn, hidden),
                                               ("w2", hidden, ffn))}
    bias = {n: (torch.randn(q.shape[0], generator=g) * 0.02).cuda() for n, (q, s) in weights.items()}
    g1, g2 = (torch.rand(hidden, generator=g) + 0.5).cuda(), (torch.rand(hidden, generator=g) + 0.5).cuda()
    lens = [5, 33, 0]
    p = Paged(torch, 1, [n + 4 for n in lens], kv, d, page, seed=1)
    p.table[p.table == 1 << 30] = 0
    rope = rope_table(torch, 64, d)
    dr = rope.cuda()
    prompt = torch.randn((sum(lens), qkv_m), generator=g).cuda()
    seq = torch.tensor([0] * 5 + [1] * 33, dtype=torch.int32, device="cuda")
    at = torch.tensor(list(range(5)) + list(range(33)), dtype=torch.int32, device="cuda")
    X.check(lib.xl_op_kv_append_paged(C.byref(p.c), 0, X.ptr(prompt), X.ptr(dr), 64, X.ptr(seq), X.ptr(at), sum(lens), heads,
                                      st()))
    x, delta = dev(batch, hidden), dev(batch, hidden)
    x8, xs = dev(batch, hidden, dt=torch.uint8), dev(batch, hidden // 128)
    a8, as_ = dev(batch, heads * d, dt=torch.uint8), dev(batch, heads * d // 128)
    f8, fs = dev(batch, ffn, dt=torch.uint8), dev(batch, ffn // 128)
    h8, hs = dev(batch, hidden, dt=torch.uint8), dev(batch, hidden // 128)
    qkv, att, mid, x2 = dev(batch, qkv_m), dev(batch, heads * d), dev(batch, ffn), dev(batch, hidden)
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = workspace(torch, p.c, heads)

    def linear(mode, name, q, s, y, m, k):
        w, wsc = weights[name]
        X.check(lib.xl_op_linear_fp8(mode, 0, X.ptr(q), q.stride(0), X.ptr(s), X.ptr(w), w.stride(0), X.ptr(wsc),
                                     X.ptr(bias[name]), X.ptr(y), batch, m, k, st()))

    def step():
        X.check(lib.xl_op_add_rmsnorm_fp8(0, None, X.ptr(x), None, X.ptr(g1), X.ptr(x8), hidden, X.ptr(xs), batch, hidden, st()))
        linear(0, "qkv", x8, xs, qkv, qkv_m, hidden)
        X.check(lib.xl_op_attn_decode_paged(C.byref(p.c), 0, X.ptr(qkv), X.ptr(dr), 64, X.ptr(pos), X.ptr(att), heads,
                                            X.ptr(ws), ws.numel(), st()))
        X.check(lib.xl_op_quantize_fp8(0, X.ptr(att), heads * d, X.ptr(a8), heads * d, X.ptr(as_), batch, heads * d, 1, st()))
        linear(0, "o", a8, as_, delta, hidden, heads * d)
        X.check(lib.xl_op_add_rmsnorm_fp8(0, X.ptr(delta), X.ptr(x), X.ptr(x2), X.ptr(g2), X.ptr(h8), hidden, X.ptr(hs), batch,
                                          hidden, st()))
        linear(1, "w13", h8, hs, mid, 2 * ffn, hidden)
        X.check(lib.xl_op_quantize_fp8(0, X.ptr(mid), ffn, X.ptr(f8), ffn, X.ptr(fs), batch, ffn, 1, st()))
        linear(2, "w2", f8, fs, x2, hidden, ffn)

    # warm up once on the same positions: a second pass over them stores the same rows
    x.copy_(torch.randn((batch, hidden), generator=g))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    def values(q, s, k):
        return q[:, :k].contiguous().view(torch.float8_e4m3fn).cpu().double() * spread(torch, s.cpu().double(), k, 1)

    def plain(name, q, s, k):
        w, wsc = weights[name]
        m = w.shape[0]
        wd = w[:, :k].contiguous().view(torch.float8_e4m3fn).cpu().double()
        return linear_reference(torch, 0, q[:, :k].contiguous().view(torch.float8_e4m3fn).cpu().double(), s.cpu(), wd,
                                wsc.cpu(), bias[name].cpu(), None)

    for i in range(3):
        before = torch.randn((batch, hidden), generator=g)
        x.copy_(before)
        now = [n + i for n in lens]
        pos.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _, (wq, wsc) = norm_reference(torch, None, before, g1.cpu())
        same(torch, values(x8, xs, hidden), wq * spread(torch, wsc, hidden, 1))
        y, tol = plain("qkv", x8, xs, hidden)
        assert ((qkv.cpu().double() - y).abs() <= tol + U * y.abs()).all()
        check_attention(torch, p, qkv.cpu(), rope, now, att, heads)
        wq, wsc = quantise(torch, att.cpu().double(), 1)
        same(torch, values(a8, as_, heads * d), wq * spread(torch, wsc, heads * d, 1))
        y, tol = plain("o", a8, as_, heads * d)
        assert ((delta.cpu().double() - y).abs() <= tol + U * y.abs()).all()
        r, (wq, wsc) = norm_reference(torch, delta.cpu(), before, g2.cpu())
        same(torch, values(h8, hs, hidden), wq * spread(torch, wsc, hidden, 1))
        wq, wsc = quantise(torch, mid.cpu().double(), 1)
        same(torch, values(f8, fs, ffn), wq * spread(torch, wsc, ffn, 1))
        y, tol = plain("w2", f8, fs, ffn)
        want = r.double() + y
        assert ((x2.cpu().double() - want).abs() <= tol + 4 * U * (want.abs() + tol)).all()


# ---- far offsets, refusals that need a device, streams -----------------------------------------------------------------

def test_quantize_and_linear_past_2g(torch):
    """Matrices of more than 2^31 bytes and elements: their last rows."""
    m, k = 140001, 16384
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn((300, k), generator=gen(torch, 1)).bfloat16()
    x.zero_()
    x[-300:] = tail.cuda()
    q, s = torch.empty((m, k), dtype=torch.uint8, device="cuda"), torch.empty(((m + 127) // 128, k // 128), device="cuda")
    X.check(X.lib().xl_op_quantize_fp8(1, X.ptr(x), k, X.ptr(q), k, X.ptr(s), m, k, 128, X.stream()))
    torch.cuda.synchronize()
    first = (m - 300 + 127) // 128 * 128  # the first whole block of rows in the tail
    want_q, want_s = quantise(torch, tail[first - (m - 300):].double(), 128)
    same(torch, s[first // 128:], want_s)
    same(torch, q[first:].view(torch.float8_e4m3fn), want_q)
    rows = torch.empty_like(q)
    per_row = torch.empty((m, k // 128), device="cuda")
    X.check(X.lib().xl_op_quantize_fp8(1, X.ptr(x), k, X.ptr(rows), k, X.ptr(per_row), m, k, 1, X.stream()))
    torch.cuda.synchronize()
    want_rq, want_rs = quantise(torch, tail[-3:].double(), 1)
    same(torch, per_row[-3:], want_rs)
    same(torch, rows[-3:].view(torch.float8_e4m3fn), want_rq)
    for n in (2, 70):
        (dx, xv) = random_fp8(torch, n, k, gen(torch, n))
        xs = torch.rand((n, k // 128), generator=gen(torch, 9)) * 0.01
        dxs = xs.cuda()
        y = torch.empty((n, m), device="cuda")
        X.check(X.lib().xl_op_linear_fp8(0, 0, X.ptr(dx), k, X.ptr(dxs), X.ptr(q), k, X.ptr(s), None, X.ptr(y), n, m, k,
                                         X.stream()))
        torch.cuda.synchronize()
        want, bound = linear_reference(torch, 0, xv, xs, want_q, want_s.float(), None, None)
        off = (y[:, first:].cpu().double() - want).abs() - bound - U * want.abs()
        assert (off <= 0).all(), float(off.max())


def test_attend_and_append_past_2g(torch):
    """A pool of more than 2^31 elements: the pages at its end."""
    kv, d, page, heads = 2, 128, 64, 8
    pages = (1 << 31) // (kv * d * page) + 40
    c = X.PagedKV()
    k, v = (torch.empty((pages, kv, page, d), dtype=torch.float16, device="cuda") for _ in range(2))
    ids = [pages - 1, pages - 30, pages - 7, pages - 2]
    table = torch.tensor([ids], dtype=torch.int32)
    dt = table.cuda()
    c = X.PagedKV(k.data_ptr(), v.data_ptr(), dt.data_ptr(), 2, 1, kv, d, page, 4, pages)
    n = 3 * page + 17
    rope = rope_table(torch, n + 1, d)
    dr = rope.cuda()
    prompt = torch.randn((n, (heads + 2 * kv) * d), generator=gen(torch, 2))
    dp, seq, at = prompt.cuda(), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    X.check(X.lib().xl_op_kv_append_paged(C.byref(c), 0, X.ptr(dp), X.ptr(dr), n + 1, X.ptr(seq), X.ptr(at), n, heads, X.stream()))
    p = Paged.__new__(Paged)
    p.torch, p.page, p.kv, p.d, p.c, p.table = torch, page, kv, d, c, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    qkv = torch.randn((1, (heads + 2 * kv) * d), generator=gen(torch, 3))
    dq, pos, out = qkv.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), torch.empty((1, heads * d), device="cuda")
    attend(torch, p, 0, dq, dr, pos, out, heads, workspace(torch, c, heads))
    torch.cuda.synchronize()
    p.dk, p.dv = k[ids].contiguous(), v[ids].contiguous()  # the same pages under the numbers 0 .. 3
    p.k = p.dk
    split = prompt.view(n, heads + 2 * kv, d)
    keys, values = p.rows(0, n)
    assert torch.equal(values, split[:, heads + kv:].transpose(0, 1).half().double())
    want = rotate(torch, split[:, heads:heads + kv], rope[:n, None]).transpose(0, 1)
    assert ((keys - want).abs() <= half_step(torch, torch.float16) * want.abs() + 8 * U * 8).all()
    check_attention(torch, p, qkv, rope, [n], out, heads)


def test_host_memory_is_refused(torch):
    """A pointer to pageable host memory ends in a status before anything is launched."""
    host = torch.zeros(1 << 12)
    q, s = torch.empty((4, 256), dtype=torch.uint8, device="cuda"), torch.empty((4, 2), device="cuda")
    assert X.lib().xl_op_quantize_fp8(0, X.ptr(host) + -X.ptr(host) % 16, 256, X.ptr(q), 256, X.ptr(s), 4, 256, 1, X.stream()) == 1
    assert b"current device" in X.lib().xl_last_error()


def test_products_on_several_streams_at_once(torch):
    """Calls of different shapes under way together (clusters that share SMs) give what each gives alone."""
    cases = []
    for i, (n, m, k) in enumerate([(8, 4608, 1536), (16, 1536, 4096), (32, 4608, 1536), (64, 1536, 4096), (100, 1536, 1536),
                                   (300, 4608, 1536), (12, 512, 2048)]):
        g = gen(torch, i)
        (dx, x), (dw, w) = random_fp8(torch, n, k, g), random_fp8(torch, m, k, g)
        xs, ws = torch.rand((n, k // 128), generator=g).cuda(), (torch.rand((m // 128, k // 128), generator=g) * 1e-3).cuda()
        cases.append((n, m, k, dx, dw, xs, ws, torch.empty((n, m), device="cuda"), torch.cuda.Stream()))

    def call(c, y, stream):
        n, m, k, dx, dw, xs, ws = c[:7]
        X.check(X.lib().xl_op_linear_fp8(0, 0, X.ptr(dx), dx.stride(0), X.ptr(xs), X.ptr(dw), dw.stride(0), X.ptr(ws), None,
                                         X.ptr(y), n, m, k, C.c_void_p(stream.cuda_stream)))

    torch.cuda.synchronize()
    alone = []
    for c in cases:
        y = torch.empty_like(c[7])
        call(c, y, torch.cuda.current_stream())
        torch.cuda.synchronize()
        alone.append(y)
    for _ in range(20):
        for c in cases:
            call(c, c[7], c[8])
    torch.cuda.synchronize()
    for c, y in zip(cases, alone):
        assert torch.equal(c[7], y), c[:3]


def test_first_calls_inside_a_capture(torch):
    """Each operator's first call of a process may be the captured one (kernels are loaded, limits raised on the way)."""
    import os
    import subprocess
    import sys

    code = r'''
import ctypes as C, sys
sys.path[:0] = ["tests", "xingling-cpp_b200"]
import torch, xl_capi as X
z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")
side = torch.cuda.Stream(); st = C.c_void_p(side.cuda_stream)
x, q, s = z(600, 512) + 1, z(600, 512, dt=torch.uint8), z(600, 4)
w, ws = z(4096, 512, dt=torch.uint8) + 0x38, z(32, 4) + 1  # 0x38 is 1.0
g, y = z(512) + 1, z(600, 4096)
table, pos, seq = z(2, 4, dt=torch.int32), z(2, dt=torch.int32), z(2, dt=torch.int32)
table[1] = 1
k, v = z(2, 2, 16, 64), z(2, 2, 16, 64)
qkv, out = z(2, (4 + 4) * 64) + 1, z(2, 256)
c = X.PagedKV(k.data_ptr(), v.data_ptr(), table.data_ptr(), 0, 2, 2, 64, 16, 4, 2)
wk = z(X.lib().xl_op_attn_decode_paged_workspace_bytes(C.byref(c), 4), dt=torch.uint8)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
L, P = X.lib(), X.ptr
with torch.cuda.graph(graph, stream=side):
    X.check(L.xl_op_quantize_fp8(0, P(x), 512, P(q), 512, P(s), 600, 512, 1, st))
    X.check(L.xl_op_add_rmsnorm_fp8(0, None, P(x), None, P(g), P(q), 512, P(s), 600, 512, st))
    for n in (8, 16, 64, 100, 600):
        X.check(L.xl_op_linear_fp8(0, 0, P(q), 512, P(s), P(w), 512, P(ws), None, P(y), n, 4096, 512, st))
    X.check(L.xl_op_kv_append_paged(C.byref(c), 0, P(qkv), None, 0, P(seq), P(pos), 2, 4, st))
    X.check(L.xl_op_attn_decode_paged(C.byref(c), 0, P(qkv), None, 0, P(pos), P(out), 4, P(wk), wk.numel(), st))
graph.replay()
torch.cuda.synchronize()
assert (y - 512).abs().max() < 1e-2, y
assert (out == 1).all()
print("captured")
'''
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
