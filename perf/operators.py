"""The operators of a decoder layer's serving step with 8-bit weights over a paged key/value cache, as cases to time.

Five entry points of libxl_engine.so (include/xl_engine.h) are measured, each against its plain form in elementary
torch operations:

  quantize   xl_op_quantize_fp8       fp32 / bf16 / fp16 to e4m3 with a scale per 128 columns (of one row or of 128 rows)
  norm       xl_op_add_rmsnorm_fp8    residual addition, RMSNorm, output in e4m3 with scales
  linear     xl_op_linear_fp8         e4m3 x e4m3 product with a scale per block of 128, fused epilogues
  attend     xl_op_attn_decode_paged  RoPE, append and attention of one new token a sequence over a paged cache
  append     xl_op_kv_append_paged    RoPE and append of prompt rows to a paged cache

`own` selects which side run() takes: False the plain forms (they need nothing of this repository), True the calls
that a user makes of the library through its C ABI.
"""
import ctypes
import math
import os

import torch

own = False

F8 = torch.float8_e4m3fn
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"fp32": 0, "bf16": 1, "fp16": 2}  # XL_F32, XL_BF16, XL_F16
GROUP = 128
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the attention output of 8 sequences that decode together, before the out-projection (smallest: latency)
        dict(name="quantize_rows_8x1536", op="quantize", dtype="fp32", n=8, k=1536, rows=1),
        # the tied embedding table as LM-head weights, in 128 x 128 blocks (largest; a row count that 128 does not divide)
        dict(name="quantize_table_151669x1536", op="quantize", dtype="fp32", n=151669, k=1536, rows=128),
        # between two sublayers of a decode step of 8 sequences
        dict(name="norm_8x1536", op="norm", dtype="fp32", n=8, k=1536, delta=True),
        # a prompt batch of a wide model, an odd number of rows
        dict(name="norm_4095x8192_bf16", op="norm", dtype="bf16", n=4095, k=8192, delta=True),
        # the QKV projection of a decode step of 8 sequences
        dict(name="linear_8x4608x1536", op="linear", dtype="fp32", mode=0, bias=True, n=8, m=4608, k=1536),
        # the LM head for one new token: a stream of weights
        dict(name="linear_1x151669x1536", op="linear", dtype="fp32", mode=0, bias=False, n=1, m=151669, k=1536),
        # the gated half of the FFN for a prompt of 512 tokens
        dict(name="linear_512x8192x1536_swiglu", op="linear", dtype="fp32", mode=1, bias=True, n=512, m=8192, k=1536),
        # a projection of a wide model for a large prompt batch: bound by the tensor cores
        dict(name="linear_4096x8192x8192_bf16", op="linear", dtype="bf16", mode=0, bias=True, n=4096, m=8192, k=8192),
        # 8 sequences of this engine's own shape, lengths up to its context
        dict(name="attend_8x768_fp32", op="attend", dtype="fp32", cache="fp32", batch=8, heads=24, kv=24, d=64, page=16,
             longest=768),
        # a serving batch of ragged lengths with shared key/value heads (largest)
        dict(name="attend_64x8192_bf16", op="attend", dtype="bf16", cache="bf16", batch=64, heads=32, kv=8, d=128, page=64,
             longest=8192),
        # a prompt of 512 tokens of this engine's shape
        dict(name="append_512_fp32", op="append", dtype="fp32", cache="fp32", batch=1, rows=512, heads=24, kv=24, d=64,
             page=16),
        # a prefill batch of sixteen prompts
        dict(name="append_16384_bf16", op="append", dtype="bf16", cache="bf16", batch=16, rows=16384, heads=32, kv=8, d=128,
             page=32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear", "linear", "attend", "attend", "append"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "quantize":
        rows = rng.choice([1, 128])
        k = _log_int(rng, 64, 16384)
        return dict(op=op, dtype=dtype, n=_log_int(rng, 1, min(151669, (1 << 27) // k)), k=k, rows=rows)
    if op == "norm":
        k = _log_int(rng, 64, 16384)
        return dict(op=op, dtype=dtype, n=_log_int(rng, 1, min(16384, (1 << 25) // k)), k=k, delta=rng.random() < 0.8)
    if op == "linear":
        n, k = _log_int(rng, 1, 4096), _log_int(rng, 64, 8192)
        m = _log_int(rng, 64, min(151669, (1 << 38) // (n * k), (1 << 30) // max(n, k))) // 2 * 2
        return dict(op=op, dtype=dtype, mode=rng.choice([0, 0, 1, 2]), bias=rng.random() < 0.7, n=n, m=m, k=k)
    heads, kv = rng.choice([(24, 24), (32, 8), (16, 2), (12, 1), (40, 8), (64, 4)])
    d, page, cache = rng.choice([64, 128]), rng.choice([8, 16, 24, 32, 64, 100, 128]), rng.choice(["fp32", "bf16", "fp16"])
    if op == "attend":
        batch = _log_int(rng, 1, 128)
        most = min(131072, (1 << 30) // (batch * kv * d * 2 * DTYPES[cache].itemsize))
        return dict(op=op, dtype=dtype, cache=cache, batch=batch, heads=heads, kv=kv, d=d, page=page,
                    longest=_log_int(rng, 1, most))
    batch = _log_int(rng, 1, 32)
    return dict(op=op, dtype=dtype, cache=cache, batch=batch, rows=_log_int(rng, batch, 16384), heads=heads, kv=kv, d=d,
                page=page)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pitch(k):
    """Bytes between the rows of an e4m3 matrix: the library's matrix product wants a multiple of 16."""
    return (k + 15) // 16 * 16


def _fp8_rows(n, k):
    return torch.empty((n, _pitch(k)), dtype=torch.uint8, device="cuda").view(F8)[:, :k]


def _rope_table(length, d):
    """[length][d/2][2] cos and sin of pos * 10000^(-2j/d), the angles formed in 64 bits."""
    j = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2 * j / d)
    return torch.stack([a.cos(), a.sin()], -1).float()


def _ragged(case):
    """Rows that each sequence holds before and after the call, before they are shuffled by the seed. Attention: the new
    token's position and one more, spread evenly up to the longest, one in a batch over 4 a slot that no sequence holds
    (-1). Append: prompts from one row up behind a few rows held."""
    i, batch = torch.arange(case["batch"], device="cuda"), case["batch"]
    if case["op"] == "attend":
        before = (i + 1) * case["longest"] // batch - 1
        if batch > 4:
            before[0] = -1
        return before, before + 1
    end = 1 + i + (case["rows"] - batch) * (i + 1) * (i + 2) // (batch * (batch + 1))
    before = i * 97 % 300
    return before, before + torch.diff(end, prepend=end.new_zeros(1))


def _pages(held, page, g):
    """A page table that hands out a shuffled pool to sequences that hold so many rows (-1 past each), and the pool's size."""
    need = (held + page - 1) // page
    wide, total = max(1, int(need.max())), int(need.sum())
    pool = total + 3
    order = torch.randperm(pool, generator=g, device="cuda")
    column = torch.arange(wide, device="cuda")
    index = (need.cumsum(0) - need)[:, None] + column
    table = torch.where(column < need[:, None], order[index.clamp(max=pool - 1)], -1)
    return table.int(), pool


class _PagedKV(ctypes.Structure):
    """xl_paged_kv: what a program that owns a paged cache keeps of it."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "page_table")] + \
               [(n, ctypes.c_int) for n in ("dtype", "batch", "kv_heads", "head_dim", "page_size", "max_pages", "num_pages")]


def prepare(case, seed):
    g = _generator(seed)
    t = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "quantize":
        n, k, rows = case["n"], case["k"], case["rows"]
        # weights are normal; activations have a few columns that stand out
        x = torch.randn((n, k), generator=g, device="cuda") * 0.02
        if rows == 1:
            x *= torch.randn(k, generator=g, device="cuda").mul_(0.5).exp_() * 20
        s["x"] = x.to(t)
        s["q"] = _fp8_rows(n, k)
        s["scale"] = torch.empty(((n + rows - 1) // rows, (k + GROUP - 1) // GROUP), device="cuda")
    elif case["op"] == "norm":
        n, k = case["n"], case["k"]
        s["residual"] = (torch.randn((n, k), generator=g, device="cuda") * 1.5).to(t)
        s["delta"] = (torch.randn((n, k), generator=g, device="cuda") * 0.3).to(t) if case["delta"] else None
        s["gamma"] = torch.rand(k, generator=g, device="cuda") + 0.5
        s["sum"] = torch.empty((n, k), dtype=t, device="cuda") if case["delta"] else None
        s["q"] = _fp8_rows(n, k)
        s["scale"] = torch.empty((n, (k + GROUP - 1) // GROUP), device="cuda")
    elif case["op"] == "linear":
        n, m, k = case["n"], case["m"], case["k"]
        blocks = (k + GROUP - 1) // GROUP
        for name, rows in (("xq", n), ("wq", m)):
            s[name] = _fp8_rows(rows, k)
            s[name].copy_((torch.randn((rows, k), generator=g, device="cuda") * 130).clamp_(-448, 448).to(F8))
        s["xs"] = (torch.rand((n, blocks), generator=g, device="cuda") + 0.5) * (3.5 / 448)
        s["ws"] = (torch.rand(((m + GROUP - 1) // GROUP, blocks), generator=g, device="cuda") + 0.5) * (0.08 / 448)
        s["bias"] = torch.randn(m, generator=g, device="cuda") * 0.02 if case["bias"] else None
        s["y"] = torch.randn((n, m // 2 if case["mode"] == 1 else m), generator=g, device="cuda").to(t)
    else:
        shuffle = torch.randperm(case["batch"], generator=g, device="cuda")
        before, held = (x[shuffle] for x in _ragged(case))
        rows = case["batch"] if case["op"] == "attend" else case["rows"]
        if case["op"] == "attend":
            s["pos"] = before.int()
            s["live"] = (before >= 0).nonzero()[:, 0]
            s["out"] = torch.empty((rows, case["heads"] * case["d"]), dtype=t, device="cuda")
        else:
            length = held - before
            seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), length)
            s["seq"] = seq.int()
            s["pos"] = (torch.arange(rows, device="cuda") - (length.cumsum(0) - length)[seq] + before[seq]).int()
        s["table"], pool = _pages(held, case["page"], g)
        width = (case["heads"] + 2 * case["kv"]) * case["d"]
        s["qkv"] = torch.randn((rows, width), generator=g, device="cuda").to(t)
        s["rope"] = _rope_table(int(held.max()), case["d"])
        shape = (pool, case["kv"], case["page"], case["d"])
        for name in ("k", "v"):
            s[name] = torch.empty(shape, dtype=DTYPES[case["cache"]], device="cuda")
            s[name].normal_(generator=g)
        s["cache"] = _PagedKV(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), CODES[case["cache"]], case["batch"],
                              case["kv"], case["d"], case["page"], s["table"].shape[1], pool)
        s["ws"] = torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")  # a serving program's workspace, zeroed once
    return s


# ---- the library's calls -------------------------------------------------------------------------------------------

_LIB = None


def _lib():
    global _LIB
    if _LIB is None:
        p, i, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        _LIB = ctypes.CDLL(os.path.join(root, "xingling-cpp_b200", "libxl_engine.so"))
        _LIB.xl_last_error.restype = ctypes.c_char_p
        _LIB.xl_op_quantize_fp8.argtypes = [i, p, z, p, z, p, i, i, i, p]
        _LIB.xl_op_add_rmsnorm_fp8.argtypes = [i, p, p, p, p, p, z, p, i, i, p]
        _LIB.xl_op_linear_fp8.argtypes = [i, i, p, z, p, p, z, p, p, p, i, i, i, p]
        _LIB.xl_op_attn_decode_paged.argtypes = [p, i, p, p, i, p, p, i, p, z, p]
        _LIB.xl_op_kv_append_paged.argtypes = [p, i, p, p, i, p, p, i, i, p]
    return _LIB


def _check(status):
    if status != 0:
        raise RuntimeError("xl status %d: %s" % (status, _lib().xl_last_error().decode()))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    c, lib = s["case"], _lib()
    code, stream = CODES[c["dtype"]], torch.cuda.current_stream().cuda_stream
    if c["op"] == "quantize":
        _check(lib.xl_op_quantize_fp8(code, _ptr(s["x"]), c["k"], _ptr(s["q"]), s["q"].stride(0), _ptr(s["scale"]), c["n"],
                                      c["k"], c["rows"], stream))
        return dict(q=s["q"], scale=s["scale"])
    if c["op"] == "norm":
        _check(lib.xl_op_add_rmsnorm_fp8(code, _ptr(s["delta"]), _ptr(s["residual"]), _ptr(s["sum"]), _ptr(s["gamma"]),
                                         _ptr(s["q"]), s["q"].stride(0), _ptr(s["scale"]), c["n"], c["k"], stream))
        return dict(q=s["q"], scale=s["scale"], sum=s["sum"])
    if c["op"] == "linear":
        _check(lib.xl_op_linear_fp8(c["mode"], code, _ptr(s["xq"]), s["xq"].stride(0), _ptr(s["xs"]), _ptr(s["wq"]),
                                    s["wq"].stride(0), _ptr(s["ws"]), _ptr(s["bias"]), _ptr(s["y"]), c["n"], c["m"], c["k"],
                                    stream))
        return s["y"]
    cache = ctypes.byref(s["cache"])
    if c["op"] == "attend":
        _check(lib.xl_op_attn_decode_paged(cache, code, _ptr(s["qkv"]), _ptr(s["rope"]), s["rope"].shape[0],
                                           _ptr(s["pos"]), _ptr(s["out"]), c["heads"], _ptr(s["ws"]), s["ws"].numel(), stream))
        return dict(out=s["out"], k=s["k"], v=s["v"])
    _check(lib.xl_op_kv_append_paged(cache, code, _ptr(s["qkv"]), _ptr(s["rope"]), s["rope"].shape[0], _ptr(s["seq"]),
                                     _ptr(s["pos"]), c["rows"], c["heads"], stream))
    return dict(k=s["k"], v=s["v"])


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _e4m3(v):
    """The e4m3 value next to each of v (float64), ties to even: 3 bits after the leading one, steps of 2^-9 at least.
    In 64 bits, since a cast through 32 would round twice next to a border."""
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    return ((v / step).round() * step).clamp(-448, 448).to(F8)


def _quotients(y, scale):
    return torch.where(scale > 0, y / scale, torch.zeros_like(y))


def _plain_quantize(x, rows):
    n, k = x.shape
    y = torch.nn.functional.pad(x.double(), (0, -k % GROUP, 0, -n % rows))
    y = y.view(y.shape[0] // rows, rows, -1, GROUP)
    scale = (y.abs().amax((1, 3)) / 448).float()
    q = _e4m3(_quotients(y, scale.double()[:, None, :, None]))
    return q.view(y.shape[0] * rows, -1)[:n, :k], scale


def _plain_norm(delta, residual, gamma):
    r = residual if delta is None else (residual.float() + delta.float()).to(residual.dtype)
    y = r.double()
    y = y / (y.square().mean(1, keepdim=True) + EPS).sqrt() * gamma.double()
    q, scale = _plain_quantize(y, 1)
    return dict(q=q, scale=scale, sum=None if delta is None else r)


def _blocks(scale, dim, size):
    return scale.repeat_interleave(GROUP, dim).narrow(dim, 0, size)


def _plain_linear(s):
    c = s["case"]
    x = s["xq"].float() * _blocks(s["xs"], 1, c["k"])
    w = s["wq"].float() * _blocks(_blocks(s["ws"], 1, c["k"]), 0, c["m"])
    y = x @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["mode"] == 1:
        y = y[:, 0::2] / (1 + torch.exp(-y[:, 0::2])) * y[:, 1::2]
    if c["mode"] == 2:
        y = y + s["y"].float()
    s["y"].copy_(y)
    return s["y"]


def _rotate(x, cs):
    """Pairs (j, j + d/2) of x [rows][heads][d] turned by the angles of cs [rows][d/2][2]."""
    a, b = x.chunk(2, -1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def _split(s):
    c = s["case"]
    rows = s["qkv"].view(-1, c["heads"] + 2 * c["kv"], c["d"]).float()
    return rows.split([c["heads"], c["kv"], c["kv"]], 1)


def _store(s, k, v, seq, pos):
    """Rows k, v [rows][kv][d] into the pages of their sequences."""
    page = s["case"]["page"]
    at = s["table"][seq.long(), pos.long() // page].long()
    s["k"][at, :, pos.long() % page] = k.to(s["k"].dtype)
    s["v"][at, :, pos.long() % page] = v.to(s["v"].dtype)


def _plain_attend(s):
    c, live = s["case"], s["live"]
    q, k, v = _split(s)
    cs = s["rope"][s["pos"].clamp(min=0).long()]
    q, k = _rotate(q, cs), _rotate(k, cs)
    _store(s, k[live], v[live], live, s["pos"][live])
    batch, kv, d = c["batch"], c["kv"], c["d"]
    table = s["table"].clamp(min=0).long()
    keys, values = (s[name][table].transpose(1, 2).reshape(batch, kv, -1, d).float() for name in ("k", "v"))
    score = q.view(batch, kv, -1, d) @ keys.transpose(2, 3) / math.sqrt(d)
    score = score.masked_fill((torch.arange(keys.shape[2], device="cuda") > s["pos"][:, None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    o = (p @ values) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return dict(out=o.reshape(batch, -1).to(s["qkv"].dtype), k=s["k"], v=s["v"])


def _plain_append(s):
    _, k, v = _split(s)
    _store(s, _rotate(k, s["rope"][s["pos"].long()]), v, s["seq"], s["pos"])
    return dict(k=s["k"], v=s["v"])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "quantize":
        q, scale = _plain_quantize(state["x"], state["case"]["rows"])
        return dict(q=q, scale=scale)
    if op == "norm":
        return _plain_norm(state["delta"], state["residual"], state["gamma"])
    return {"linear": _plain_linear, "attend": _plain_attend, "append": _plain_append}[op](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "quantize":
        n, k = case["n"], case["k"]
        return dict(bytes=n * k * (size + 1) + 4 * -(-n // case["rows"]) * -(-k // GROUP), flops=3 * n * k)
    if case["op"] == "norm":
        n, k = case["n"], case["k"]
        return dict(bytes=n * k * (size * (3 if case["delta"] else 1) + 1) + 4 * k + 4 * n * -(-k // GROUP), flops=7 * n * k)
    if case["op"] == "linear":
        n, m, k = case["n"], case["m"], case["k"]
        blocks, wide = -(-k // GROUP), m // 2 if case["mode"] == 1 else m
        moved = (n + m) * k + 4 * blocks * (n + -(-m // GROUP)) + (4 * m if case["bias"] else 0)
        return dict(bytes=moved + n * wide * size * (2 if case["mode"] == 2 else 1), flops=2 * n * m * k)
    heads, kv, d, store = case["heads"], case["kv"], case["d"], DTYPES[case["cache"]].itemsize
    if case["op"] == "attend":
        batch = case["batch"]
        seen = sum((i + 1) * case["longest"] // batch for i in range(1 if batch > 4 else 0, batch))
        moved = seen * 2 * kv * d * store + batch * ((2 * heads + 2 * kv) * d * size + 2 * kv * d * store)
        return dict(bytes=moved, flops=4 * heads * d * seen)
    return dict(bytes=case["rows"] * (2 * kv * d * (size + store) + 4 * d + 8), flops=3 * case["rows"] * kv * d)


# ---- the definitions in 64 bits, apart from the plain forms ------------------------------------------------------------

def _exact_fp8(y, rows):
    """Every group of y (float64) divided by its stored 32-bit scale, as the nearest of the 256 e4m3 values."""
    n, k = y.shape
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(F8).double()
    values = codes[~codes.isnan()].unique()  # sorted; the two zeros are one
    middle = (values[1:] + values[:-1]) / 2
    # ties go to the even mantissa: the values with a last bit of 0 (value / its own step is even)
    step = torch.exp2(torch.floor(torch.log2(values.abs().clamp(min=2.0 ** -6))) - 3)
    even = (values / step) % 2 == 0
    q, scale = torch.empty((n, k), device="cuda"), torch.empty((-(-n // rows), -(-k // GROUP)), dtype=torch.float64, device="cuda")
    many = max(rows, (1 << 22) // k // rows * rows)
    for r0 in range(0, n, many):
        block = y[r0:r0 + many]
        for c0 in range(0, k, GROUP):
            part = block[:, c0:c0 + GROUP]
            top = part.abs().amax(1)
            if rows > 1:
                top = torch.stack([piece.max() for piece in top.split(rows)])
            sc = (top / 448).float().double()
            scale[r0 // rows:r0 // rows + len(sc), c0 // GROUP] = sc
            each = sc.repeat_interleave(rows)[:len(part), None]
            v = torch.where(each > 0, part / each, 0.0).contiguous()
            low = torch.searchsorted(middle, v, right=False).clamp(max=len(values) - 1)
            tie = (low < len(middle)) & (middle[low.clamp(max=len(middle) - 1)] == v) & ~even[low]
            q[r0:r0 + many, c0:c0 + GROUP] = values[low + tie.long()].float()
    return q.double(), scale


def _exact_rows(s, x):
    c = s["case"]
    half = c["d"] // 2
    cs = s["rope"].double()[s["pos"].long().clamp(min=0)]
    z = torch.view_as_complex(torch.stack([x[..., :half], x[..., half:]], -1).contiguous())
    z = z * torch.complex(cs[..., 0], -cs[..., 1])[:, None]
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        q, scale = _exact_fp8(s["x"].double(), case["rows"])
        return dict(q=q, scale=scale)
    if case["op"] == "norm":
        r = s["residual"].double()
        if s["delta"] is not None:
            r = r + s["delta"].double()
        stored = r.float().to(s["residual"].dtype).double()
        q, scale = _exact_fp8(stored * torch.rsqrt((stored * stored).sum(1, keepdim=True) / case["k"] + EPS) * s["gamma"], 1)
        return dict(q=q, scale=scale, sum=None if s["delta"] is None else r)
    if case["op"] == "linear":
        y = s["y"].double() if case["mode"] == 2 else torch.zeros((case["n"], case["m"]), dtype=torch.float64, device="cuda")
        for b in range(s["xs"].shape[1]):
            part = slice(b * GROUP, min(case["k"], (b + 1) * GROUP))
            sw = s["ws"][:, b].double().repeat_interleave(GROUP)[:case["m"]]
            y += torch.einsum("nc,mc->nm", s["xq"][:, part].double(), s["wq"][:, part].double()) * s["xs"][:, b, None].double() * sw
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["mode"] == 1:
            y = y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
        return y
    heads, kv, d, page = case["heads"], case["kv"], case["d"], case["page"]
    qkv = s["qkv"].double().view(-1, heads + 2 * kv, d)
    new_k, new_v = _exact_rows(s, qkv[:, heads:heads + kv]), qkv[:, heads + kv:]
    pos = s["pos"].long()
    seq = s["live"] if case["op"] == "attend" else s["seq"].long()
    rows = s["live"] if case["op"] == "attend" else torch.arange(case["rows"], device="cuda")
    at = s["table"].long()[seq, torch.div(pos[rows], page, rounding_mode="floor")]
    k, v = s["k"].double(), s["v"].double()
    k[at, :, pos[rows] % page], v[at, :, pos[rows] % page] = new_k[rows], new_v[rows]
    if case["op"] == "append":
        return dict(k=k, v=v)
    out = torch.zeros((case["batch"], heads, d), dtype=torch.float64, device="cuda")
    q, store = _exact_rows(s, qkv[:, :heads]), s["k"].dtype
    for b in s["live"].tolist():
        n = int(pos[b]) + 1
        pages = s["table"].long()[b, :-(-n // page)]
        kb, vb = (p[pages].permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :n].to(store).double() for p in (k, v))
        w = torch.softmax(torch.einsum("hgd,htd->hgt", q[b].view(kv, -1, d), kb) * d ** -0.5, -1)
        out[b] = torch.einsum("hgt,htd->hgd", w, vb).reshape(heads, d)
    return dict(out=out.reshape(case["batch"], -1), k=k, v=v)
