"""The operators of a served model at 8 bits, as cases to measure: matrices
and KV caches of e4m3 values, each block's scale a power of two.

Kinds of case:

- ``norm``: a block's output added to the residual stream, its RMSNorm, and
  that in 8 bits with a scale for each 128 elements (``fp8.AddNorm``), the
  values read back (``fp8.Dequantize``).
- ``linear``: 8-bit rows times 8-bit weights, both with a scale for each 128
  elements (``fp8.Gemm``).
- ``store``: a step's q, k and v rows turned by RoPE, k and v into 8-bit paged
  pools with a scale for each block and head (``paged8.PagedStore8``).
- ``load``: cached positions read back as 16- or 32-bit rows
  (``paged8.PagedLoad8``).
- ``attend``: attention of one new token a request over 8-bit pages
  (``paged8.PagedAttend8``).

An 8-bit value is e4m3 (448 the largest, no infinity) times its block's
scale, the smallest power of two, from 2^-126 on, that keeps the block's
largest magnitude within 448.

The plain forms are elementary torch operations in 32 bits, rounded once at
the end.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

NONE = -1            # 0xFFFFFFFF, as the int32 tensors hold it
EPS = 1e-5
LARGEST = 448.0      # e4m3's

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_E4M3 = torch.float8_e4m3fn


# The cases ------------------------------------------------------------------------


def listed():
    return [
        # A decode step's eight rows of the 1B model's residual stream, f32 as it keeps it.
        {"name": "norm-8x2048", "kind": "norm", "rows": 8, "k": 2048, "type": "f32", "residual": True},
        # A long prompt through a model of a width that is no multiple of 128.
        {"name": "norm-8191x5000-bf16", "kind": "norm", "rows": 8191, "k": 5000, "type": "bf16", "residual": True},
        # A decode step of eight rows through the 1B model's gate projection: the weights' stream.
        {"name": "linear-8x8192x2048", "kind": "linear", "m": 8, "n": 8192, "k": 2048, "out": "f32"},
        # A short prompt through a layer of ragged sizes.
        {"name": "linear-100x5000x3080", "kind": "linear", "m": 100, "n": 5000, "k": 3080, "out": "bf16"},
        # The 1B prefill's rows (4 x 2048) through its gate projection.
        {"name": "linear-8192x8192x2048", "kind": "linear", "m": 8192, "n": 8192, "k": 2048, "out": "f16"},
        # A decode step of a few conversations, a token each somewhere in its page: the smallest call.
        {"name": "store-8", "kind": "store", "requests": 8, "chunk": 1, "spare": 0, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "block": 64, "type": "f32", "q_type": "f16", "rotated": 32},
        # Chunks of several prompts, pages begun and not filled among them, the step padded.
        {"name": "store-33x248-bf16", "kind": "store", "requests": 33, "chunk": 248, "spare": 7, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 16, "type": "bf16", "q_type": "bf16", "rotated": 32},
        # A short prefix for a chunk's prefill, of the 1B model's heads.
        {"name": "load-100", "kind": "load", "tokens": 100, "kv_heads": 8, "head_dim": 64, "block": 64, "type": "f16"},
        # A long document's positions, an odd number of them.
        {"name": "load-32767-bf16", "kind": "load", "tokens": 32767, "kv_heads": 8, "head_dim": 128, "block": 16,
         "type": "bf16"},
        # Many short conversations, an odd group of query heads.
        {"name": "attend-41x700", "kind": "attend", "requests": 41, "longest": 700, "heads": 28, "kv_heads": 4,
         "head_dim": 64, "block": 16, "q_type": "f16", "window": 0},
        # One very long document: only a split over its length fills the card.
        {"name": "attend-1x131072", "kind": "attend", "requests": 1, "longest": 131072, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "block": 64, "q_type": "f16", "window": 0},
        # A large ragged batch, long and short together.
        {"name": "attend-64x16384-bf16", "kind": "attend", "requests": 64, "longest": 16384, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 16, "q_type": "bf16", "window": 0},
    ]


def _log(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "store", "load", "attend", "attend"])
    if kind == "norm":
        k = _log(rng, 8, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(32768, 8191 * 5000 // k)), "k": k,
                "type": rng.choice(["f32", "f16", "bf16"]), "residual": rng.choice([True, True, False])}
    if kind == "linear":
        m, n = _log(rng, 1, 8192), _log(rng, 16, 16384)
        k = _log(rng, 32, min(16384, max(32, 8192 * 8192 * 2048 // (m * n))))
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "f16", "bf16"])}
    d = rng.choice([64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8])
    block = rng.choice([8, 16, 16, 24, 64, 128])
    if kind == "store":
        n = _log(rng, 1, 256)
        most = max(1, 8184 * 8 * 128 // (n * kv * d))
        return {"kind": kind, "requests": n, "chunk": rng.choice([1, _log(rng, 1, min(4096, most))]),
                "spare": rng.choice([0, _log(rng, 1, 100)]), "heads": kv * rng.randint(1, 4), "kv_heads": kv,
                "head_dim": d, "block": block, "type": rng.choice(["f32", "f16", "bf16"]),
                "q_type": rng.choice(["f16", "bf16"]), "rotated": rng.choice([0, d // 4, d // 2])}
    if kind == "load":
        return {"kind": kind, "tokens": _log(rng, 1, 32767 * 8 * 128 // (2 * kv * d)), "kv_heads": kv, "head_dim": d,
                "block": block, "type": rng.choice(["f32", "f16", "bf16"])}
    n = _log(rng, 1, 200)
    longest = _log(rng, 16, min(131072, 64 * 16384 * 8 * 128 // (n * kv * d)))
    return {"kind": kind, "requests": n, "longest": longest, "heads": kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]),
            "kv_heads": kv, "head_dim": d, "block": block, "q_type": rng.choice(["f16", "bf16"]),
            "window": rng.choice([0, 0, 0, _log(rng, 8, 4096)])}


# What a program has in hand --------------------------------------------------------


class _Framework:
    """The device, opened once a process."""

    device = None


def _device():
    if _Framework.device is None:
        from furykernel_amd import runtime
        torch.cuda.init()
        _Framework.device = runtime.Device(0)
    return _Framework.device


class _Owner:
    """Gives back what a state holds, once neither the state nor any view of
    its buffers is left."""

    def __init__(self):
        self.held = []

    def __del__(self):
        if self.held:
            torch.cuda.synchronize()
        for b in self.held:
            b.free()


class _Span:
    """Device memory as torch takes it; a tensor over it keeps its owner."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False),
                                         "strides": None, "version": 2}


_VIEWS = {torch.float32: ("<f4", None), torch.float16: ("<f2", None), torch.bfloat16: ("<i2", torch.bfloat16),
          torch.int32: ("<i4", None), torch.uint8: ("|u1", None), _E4M3: ("|u1", _E4M3)}


class _Memory:
    """Buffers of the framework's, each with a tensor over the same memory."""

    def __init__(self):
        self.owner = _Owner()

    def empty(self, shape, dtype):
        typestr, as_type = _VIEWS[dtype]
        size = math.prod(shape) * dtype.itemsize
        buf = _device().alloc(max(size, 16))
        self.owner.held.append(buf)
        t = torch.as_tensor(_Span(self.owner, buf.ptr, shape, typestr), device="cuda")
        return buf, (t if as_type is None else t.view(as_type))

    def put(self, tensor):
        buf, view = self.empty(tuple(tensor.shape), tensor.dtype)
        view.copy_(tensor)
        return buf, view


class _State:
    """A pass (`go`) and what it needs; it returns its outputs."""

    def __init__(self, go):
        self.go = go


def prepare(case, seed):
    made = _INPUTS[case["kind"]](case, int(seed))
    go = (_OWN if own else _PLAIN)[case["kind"]](case, made)
    torch.cuda.synchronize()
    return _State(go)


def run(state):
    return state.go()


def exact(case, seed):
    """What `run` returns, from the definitions in binary64, on the same inputs."""
    return _EXACT[case["kind"]](case, _INPUTS[case["kind"]](case, int(seed)))


def work(case):
    return _WORK[case["kind"]](case)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _rng(seed):
    return np.random.default_rng(int(seed) * 2 + 1)


def _normal(gen, dims, dtype, std=1.0):
    return (torch.randn(dims, generator=gen, device="cuda") * std).to(dtype)


def _matrix(gen, rows, k, dtype):
    """Normals with some columns far larger, as activations and weights have."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    gain = torch.where(torch.rand((k,), generator=gen, device="cuda") < 0.02, 20.0, 1.0)
    return (x * gain).to(dtype)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _lengths(rng, n, longest):
    """Lengths spread over the logarithm up to the longest, the longest
    among them."""
    low = max(1.0, longest / 16)
    x = np.exp(rng.uniform(math.log(low), math.log(longest), n)) if longest > 1 else np.ones(n)
    x = np.clip(np.rint(x), 1, longest).astype(np.int64)
    x[rng.integers(n)] = longest
    return x


def _wide(name):
    return 4 if name == "f32" else 2


# 8-bit values ---------------------------------------------------------------------------


def _scale_of(big):
    """The scale of blocks whose largest magnitude is `big`, in 32 bits."""
    m, e = torch.frexp(big)              # big = m 2^e, m in [1/2, 1); 448 = 0.875 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(big > 0, e, -126).clamp(min=-126)
    return torch.ldexp(torch.ones_like(big), e)


def _blocks_of(x):
    """Rows by blocks of 128, zeros behind the last."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 128)).unflatten(1, (-1, 128))


def _plain_codes(x):
    """f32 rows' codes [rows, blocks, 128] and scales [rows, blocks, 1]."""
    x = _blocks_of(x)
    scale = _scale_of(x.abs().amax(-1, keepdim=True))
    return (x / scale).to(_E4M3), scale


def _exact_scale(big):
    """From the definition, in 64 bits."""
    e = torch.ceil(torch.log2(torch.where(big > 0, big, 1.0) / LARGEST)).clamp(min=-126)
    # (log2 is rounded: the power below it where that holds the value, the one above where this does not)
    e = torch.where(LARGEST * torch.exp2(e - 1) >= big, e - 1, torch.where(LARGEST * torch.exp2(e) < big, e + 1, e))
    return torch.exp2(torch.where(big > 0, e, -126.0).clamp(min=-126))


def _exact_code(y):
    """To the nearest e4m3, halfway cases to the even code: steps of 2^-3 of
    the power of two below, at least 2^-9."""
    exp = torch.frexp(y)[1].double() - 1
    step = torch.exp2(exp.clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_values(x):
    """Rows of binary64 as the 8-bit values they become, flat."""
    k = x.shape[1]
    x = _blocks_of(x)
    scale = _exact_scale(x.abs().amax(-1, keepdim=True))
    return (_exact_code(x / scale) * scale).flatten(1)[:, :k]


# norm: the residual's addition, RMSNorm, 8 bits -----------------------------------------------


def _norm_inputs(case, seed):
    gen, t, k = _generator(seed), _TYPES[case["type"]], case["k"]
    s = {"x": _matrix(gen, case["rows"], k, t), "gamma": _normal(gen, (k,), torch.float32, 0.1) + 1.0}
    if case["residual"]:
        s["residual"] = _matrix(gen, case["rows"], k, t)
    return s


def _norm_plain(case, s):
    k, t = case["k"], _TYPES[case["type"]]

    def go():
        h = s["x"]
        out = {}
        if case["residual"]:
            h = out["sum"] = (h.float() + s["residual"].float()).to(t)
        h = h.float()
        y = h * (1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)) * s["gamma"]
        codes, scale = _plain_codes(y)
        out["values"] = (codes.float() * scale).flatten(1)[:, :k].to(torch.bfloat16)
        return out

    return go


def _norm_own(case, s):
    from furykernel_amd import fp8
    mem, dev = _Memory(), _device()
    rows, k, t = case["rows"], case["k"], case["type"]
    held = fp8.Fp8Matrix(dev, rows, k)
    mem.owner.held.append(held)
    more, out = {}, {}
    if case["residual"]:
        more["residual"] = mem.put(s["residual"])[0]
        more["sum"], out["sum"] = mem.empty((rows, k), _TYPES[t])
    norm = fp8.AddNorm(dev, mem.put(s["x"])[0], held, eps=EPS, gamma=mem.put(s["gamma"])[0], x_type=t, **more)
    y, out["values"] = mem.empty((rows, k), torch.bfloat16)
    back = fp8.Dequantize(dev, held, y, y_type="bf16")

    def go():
        norm.enqueue()
        back.enqueue()
        return out

    return go


def _norm_exact(case, s):
    sums, values = [], []
    for i in range(0, case["rows"], 1024):
        h = s["x"][i:i + 1024].double()
        if case["residual"]:
            h = h + s["residual"][i:i + 1024].double()
            sums.append(h)
            h = h.to(_TYPES[case["type"]]).double()      # the norm is of what is stored
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * s["gamma"].double()
        values.append(_exact_values(y))
    return {"values": torch.cat(values), **({"sum": torch.cat(sums)} if sums else {})}


def _norm_work(case):
    rows, k = case["rows"], case["k"]
    n, wide = rows * k, _wide(case["type"])
    # x, the residual and the sum; codes and scales written and read; the values written
    return {"bytes": n * wide * (3 if case["residual"] else 1) + 4 * k + 2 * (n + rows * -(-k // 128)) + 2 * n,
            "flops": 8 * n}


# linear: 8-bit rows times 8-bit weights -----------------------------------------------------


def _linear_inputs(case, seed):
    gen = _generator(seed)
    return {"x": _matrix(gen, case["m"], case["k"], torch.bfloat16),
            "w": _normal(gen, (case["n"], case["k"]), torch.bfloat16, case["k"] ** -0.5)}


def _linear_plain(case, s):
    out = _TYPES[case["out"]]
    (xc, xs), (wc, ws) = (_plain_codes(s[i].float()) for i in "xw")     # as a program keeps them

    def go():
        x, w = ((c.float() * sc).flatten(1) for c, sc in ((xc, xs), (wc, ws)))
        return torch.matmul(x, w.t()).to(out)

    return go


def _linear_own(case, s):
    from furykernel_amd import fp8
    mem, dev, held = _Memory(), _device(), []
    for i, rows in (("x", case["m"]), ("w", case["n"])):
        held.append(fp8.Fp8Matrix(dev, rows, case["k"]))
        buf = mem.put(s[i])[0]
        torch.cuda.synchronize()
        fp8.Quantize(dev, buf, held[-1], x_type="bf16").enqueue()
    mem.owner.held += held
    y, view = mem.empty((case["m"], case["n"]), _TYPES[case["out"]])
    product = fp8.Gemm(dev, held[0], held[1], y, c_type=case["out"])

    def go():
        product.enqueue()
        return view

    return go


def _linear_exact(case, s):
    w = _exact_values(s["w"].double()).t()
    return torch.cat([_exact_values(x.double()) @ w for x in s["x"].split(1024)])


def _linear_work(case):
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": (m + n) * (k + -(-k // 128)) + m * n * _wide(case["out"]), "flops": 2 * m * n * k}


# store: rows into 8-bit pools --------------------------------------------------------------


def _pools(gen, blocks, kv, block, d, amplitude=1.0):
    """Pools that hold normals: codes of k and v, and scales [blocks][kv heads][k, v]."""
    codes, scales = [], []
    for _ in "kv":
        x = torch.randn((blocks, kv, block, d), generator=gen, device="cuda") * amplitude
        scale = _scale_of(x.abs().amax((2, 3)))
        codes.append((x / scale[..., None, None]).to(_E4M3))
        scales.append(scale)
    return {"k": codes[0], "v": codes[1], "scales": torch.stack(scales, -1)}


def _store_sizes(case):
    """New tokens of each request, the step's tokens and the pool's blocks, the
    same for every seed."""
    n, chunk, block = case["requests"], case["chunk"], case["block"]
    fresh = np.random.default_rng(n * 7 + chunk).integers((chunk + 1) // 2, chunk + 1, n)
    fresh[0] = chunk
    return fresh, int(fresh.sum()) + case["spare"], int((-(-(fresh + block - 1) // block)).sum()) + 4


def _store_inputs(case, seed):
    gen, rng = _generator(seed), _rng(seed)
    n, h, kv, d, block = (case[i] for i in ("requests", "heads", "kv_heads", "head_dim", "block"))
    fresh, tokens, blocks = _store_sizes(case)
    fresh = rng.permutation(fresh)
    order = rng.permutation(blocks)
    begun = np.where(rng.random(n) < 0.8, rng.integers(0, block, n), 0)    # positions of the first page held before
    slots, at, used = np.full(tokens, NONE), 0, 0
    for r in range(n):
        place = begun[r] + np.arange(fresh[r])
        if rng.random() >= 0.02:                                            # else one that did not fit
            slots[at:at + fresh[r]] = order[used + place // block] * block + place % block
        at += fresh[r]
        used += place[-1] // block + 1
    rotated, rows = case["rotated"], 4096
    freq = 10000.0 ** (-2.0 * np.arange(rotated) / d)
    angle = (np.arange(rows)[:, None] * freq.astype(np.float32)).astype(np.float32).astype(np.float64)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    loud = torch.exp2(torch.rand((tokens, 1), generator=gen, device="cuda") * 4 - 2)
    return {"qkv": (torch.randn((tokens, (h + 2 * kv) * d), generator=gen, device="cuda") * loud).to(_TYPES[case["type"]]),
            "slots": _cuda(slots.astype(np.int32)), "positions": _cuda(rng.integers(0, rows, tokens).astype(np.int32)),
            "rope": _cuda(rope), "qr": _normal(gen, (tokens, h, d), _TYPES[case["q_type"]]),
            **_pools(gen, blocks, kv, block, d)}


def _store_rows(case, s, dtype):
    """q, k, v as [tokens, heads, d], q and k turned, in `dtype`."""
    h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["rotated"]
    x = s["qkv"].to(dtype)
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([h * d, kv * d, kv * d], 1))
    c, sn = (t[:, None] for t in s["rope"][s["positions"].long()].to(dtype).unbind(-1))

    def turn(t):
        half = d // 2
        a, b = t[..., :n], t[..., half:half + n]
        return torch.cat([a * c - b * sn, t[..., n:half], b * c + a * sn, t[..., half + n:]], -1)

    return turn(q), turn(k), v


def _store_plain(case, s):
    block, kv, blocks = case["block"], case["kv_heads"], s["k"].shape[0]
    heads = torch.arange(kv, device="cuda")[None]
    places = torch.arange(block, device="cuda")[None]
    qr, scales = s["qr"].clone(), s["scales"].clone()
    # rows without a slot go to a block past the pool's, which is no output
    pools = [torch.cat([s[i], s[i][:1]]) for i in "kv"]

    def go():
        q, k, v = _store_rows(case, s, torch.float32)
        slot = s["slots"].long()
        live = slot >= 0
        qr.copy_(torch.where(live[:, None, None], q.to(qr.dtype), qr))
        at = torch.where(live, slot // block, blocks)
        place = torch.where(live, slot % block, 0)
        first = torch.full((blocks + 1,), block, device="cuda").scatter_reduce(0, at, place, "amin")[:blocks]
        for i, (pool, x) in enumerate(zip(pools, (k, v))):
            # the new rows' scale, and the block's own before them where it holds some already
            big = torch.zeros((blocks + 1, kv), device="cuda")
            big = big.scatter_reduce(0, at[:, None].expand(-1, kv), x.abs().amax(-1), "amax")[:blocks]
            before = scales[..., i]
            begins = (first == 0)[:, None]
            new = torch.where(begins, _scale_of(big), torch.maximum(before, _scale_of(big)))
            new = torch.where((first < block)[:, None], new, before)
            # rows stored before a scale that grew
            grown = ((places < first[:, None])[:, None] & (new != before)[..., None])[..., None]
            old = (pool[:blocks].float() * (before / new)[..., None, None]).to(_E4M3)
            pool[:blocks] = torch.where(grown, old.view(torch.uint8), pool[:blocks].view(torch.uint8)).view(_E4M3)
            over = torch.cat([new, new[:1]])[at]
            pool.view(torch.uint8)[at[:, None], heads, place[:, None]] = (x / over[..., None]).to(_E4M3).view(torch.uint8)
            scales[..., i] = new
        return {"qr": qr, "k": pools[0][:blocks], "v": pools[1][:blocks], "scales": scales}

    return go


def _store_own(case, s):
    from furykernel_amd import paged8
    mem = _Memory()
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    b = {i: mem.put(s[i]) for i in ("qkv", "slots", "positions", "qr", "k", "v", "scales")}
    rope = mem.put(s["rope"])[0] if case["rotated"] else None
    row = (h + 2 * kv) * d
    op = paged8.PagedStore8(_device(), q=b["qkv"][0], k=b["qkv"][0], v=b["qkv"][0], k_offset=h * d,
                            v_offset=(h + kv) * d, q_stride=row, k_stride=row, v_stride=row, slots=b["slots"][0],
                            positions=b["positions"][0], rope=rope, rope_rows=s["rope"].shape[0],
                            rotated=case["rotated"], qr=b["qr"][0], kpool=b["k"][0], vpool=b["v"][0],
                            scales=b["scales"][0], tokens=s["slots"].numel(), heads=h, kv_heads=kv, head_dim=d,
                            block_size=case["block"], blocks=s["k"].shape[0], rows_type=case["type"],
                            q_type=case["q_type"])
    views = {i: b[i][1] for i in ("qr", "k", "v", "scales")}

    def go():
        op.enqueue()
        return views

    return go


def _store_exact(case, s):
    """The definition, a block that tokens go into at a time."""
    block = case["block"]
    q, k, v = _store_rows(case, s, torch.float64)
    out = {"qr": s["qr"].double(), "k": s["k"].double(), "v": s["v"].double(), "scales": s["scales"].double()}
    slot = s["slots"].cpu().numpy()
    live = np.flatnonzero(slot >= 0)
    out["qr"][_cuda(live)] = q[_cuda(live)]
    if live.size == 0:
        return out
    for run in np.split(live, np.flatnonzero(np.diff(slot[live] // block)) + 1):
        b, place = int(slot[run[0]]) // block, int(slot[run[0]]) % block
        rows = slice(int(run[0]), int(run[-1]) + 1)
        for i, (name, x) in enumerate((("k", k), ("v", v))):
            x = x[rows].transpose(0, 1)                       # [kv heads, tokens, d]
            scale = _exact_scale(x.abs().amax((1, 2)))
            if place:
                before = out["scales"][b, :, i]
                scale = torch.maximum(scale, before)
                held = out[name][b, :, :place]
                held.copy_(_exact_code(held * (before / scale)[:, None, None]))
            out[name][b, :, place:place + len(run)] = _exact_code(x / scale[:, None, None])
            out["scales"][b, :, i] = scale
    return out


def _store_work(case):
    tokens, d, kv = int(_store_sizes(case)[0].sum()), case["head_dim"], case["kv_heads"]
    e = (case["heads"] + 2 * kv) * d
    # rows read, q written in 16 bits and k and v in 8, a block's scales for each page begun; slots, positions, angles
    return {"bytes": tokens * (e * _wide(case["type"]) + 2 * case["heads"] * d + 2 * kv * d + 8 + 8 * case["rotated"])
            + 8 * kv * _store_sizes(case)[2], "flops": tokens * (6 * case["rotated"] * (case["heads"] + kv) + 4 * kv * d)}


# load: cached positions as rows ---------------------------------------------------------------


def _load_inputs(case, seed):
    gen, rng = _generator(seed), _rng(seed)
    T, kv, d, block = case["tokens"], case["kv_heads"], case["head_dim"], case["block"]
    blocks = -(-T // block) + 4
    # positions in order, their pages anywhere; some rows of a padded step
    slots = (rng.permutation(blocks)[:, None] * block + np.arange(block)).reshape(-1)[:T]
    slots[rng.random(T) < 0.02] = NONE
    t = _TYPES[case["type"]]
    return {"slots": _cuda(slots.astype(np.int32)), **_pools(gen, blocks, kv, block, d),
            **{f"{i}_rows": _normal(gen, (T, kv, d), t) for i in "kv"}}


def _load_plain(case, s):
    block = case["block"]
    outs = [s[f"{i}_rows"].clone() for i in "kv"]

    def go():
        slot = s["slots"].long()
        live = (slot >= 0)[:, None, None]
        at, place = slot.clamp(min=0) // block, slot.clamp(min=0) % block
        scales = s["scales"][at]
        for i, (name, out) in enumerate(zip("kv", outs)):
            x = s[name].view(torch.uint8)[at, :, place].view(_E4M3).float() * scales[..., i, None]
            out.copy_(torch.where(live, x.to(out.dtype), out))
        return {"k": outs[0], "v": outs[1]}

    return go


def _load_own(case, s):
    from furykernel_amd import paged8
    mem = _Memory()
    b = {i: mem.put(s[i]) for i in ("slots", "k", "v", "scales", "k_rows", "v_rows")}
    op = paged8.PagedLoad8(_device(), slots=b["slots"][0], kpool=b["k"][0], vpool=b["v"][0], scales=b["scales"][0],
                           k=b["k_rows"][0], v=b["v_rows"][0], tokens=case["tokens"], kv_heads=case["kv_heads"],
                           head_dim=case["head_dim"], block_size=case["block"], blocks=s["k"].shape[0],
                           rows_type=case["type"])
    views = {"k": b["k_rows"][1], "v": b["v_rows"][1]}

    def go():
        op.enqueue()
        return views

    return go


def _load_exact(case, s):
    block = case["block"]
    slot = s["slots"].cpu().numpy()
    live = np.flatnonzero(slot >= 0)
    at, place, live = (_cuda(a.astype(np.int64)) for a in (slot[live] // block, slot[live] % block, live))
    out = {}
    for i, name in enumerate("kv"):
        out[name] = s[f"{name}_rows"].double()
        held = s[name].double() * s["scales"][..., i].double()[..., None, None]
        out[name][live] = held.transpose(1, 2)[at, place]
    return out


def _load_work(case):
    T, e = case["tokens"], case["kv_heads"] * case["head_dim"]
    return {"bytes": T * (2 * e * (1 + _wide(case["type"])) + 4) + 8 * case["kv_heads"] * -(-T // case["block"]),
            "flops": 2 * T * e}


# attend: one new token a request over 8-bit pages ------------------------------------------------


def _attend_lengths(case):
    rng = np.random.default_rng(case["requests"] * 31 + case["longest"])
    return _lengths(rng, case["requests"], case["longest"])


def _attend_inputs(case, seed):
    gen, rng = _generator(seed), _rng(seed)
    n, h, kv, d, block = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim", "block"))
    lengths = rng.permutation(_attend_lengths(case))
    pages = -(-lengths // block)
    blocks = int(pages.sum()) + 3
    order = rng.permutation(blocks)
    table = np.zeros((n, -(-case["longest"] // block)), np.int32)
    at = 0
    for r in range(n):
        table[r, :pages[r]] = order[at:at + pages[r]]
        at += pages[r]
    # blocks of different loudness, so of different scales
    loud = torch.exp2(torch.rand((blocks, kv, 1, 1), generator=gen, device="cuda") * 3 - 2)
    return {"q": _normal(gen, (n, h, d), _TYPES[case["q_type"]]), **_pools(gen, blocks, kv, block, d, loud),
            "table": _cuda(table), "lengths": _cuda(lengths.astype(np.int32))}


def _softmax_scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def _attend_plain(case, s):
    n, h, kv, d, block = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim", "block"))
    pages = s["table"].shape[1]
    keys = torch.arange(pages * block, device="cuda")[None]
    step = max(1, int((1 << 28) // (pages * block * kv * d)))   # requests at once: 1 GB of keys in 32 bits

    def go():
        out = []
        for r0 in range(0, n, step):
            rows = slice(r0, min(n, r0 + step))
            at = s["table"][rows].long()
            length = s["lengths"][rows].long()[:, None]

            def gather(i, name):   # [requests, kv heads, keys, d]
                x = s[name].view(torch.uint8)[at].view(_E4M3).float() * s["scales"][at][..., i, None, None]
                return x.transpose(1, 2).flatten(2, 3)

            q = s["q"][rows].float().unflatten(1, (kv, h // kv))
            score = torch.matmul(q, gather(0, "k").transpose(2, 3).contiguous()) * _softmax_scale(case)
            live = keys < length
            if case["window"]:
                live &= keys >= length - case["window"]
            score = score.masked_fill(~live[:, None, None], -math.inf)
            e = (score - score.amax(-1, keepdim=True)).exp()
            v = gather(1, "v").masked_fill(~live[:, None, :, None], 0.0)
            o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
            out.append(o.flatten(1, 2).to(s["q"].dtype))
        return out[0] if len(out) == 1 else torch.cat(out)

    return go


def _attend_own(case, s):
    from furykernel_amd import paged8
    mem = _Memory()
    b = {k: mem.put(s[k])[0] for k in ("q", "k", "v", "scales", "table", "lengths")}
    out, view = mem.empty(tuple(s["q"].shape), s["q"].dtype)
    sizes = dict(requests=case["requests"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                 block_size=case["block"], blocks=s["k"].shape[0], table_len=s["table"].shape[1],
                 window=case["window"])
    workspace, _ = mem.empty((paged8.attend8_workspace(**sizes),), torch.uint8)
    op = paged8.PagedAttend8(_device(), q=b["q"], kpool=b["k"], vpool=b["v"], scales=b["scales"], table=b["table"],
                             lengths=b["lengths"], out=out, workspace=workspace, scale=_softmax_scale(case),
                             q_type=case["q_type"], **sizes)

    def go():
        op.enqueue()
        return view

    return go


def _attend_exact(case, s):
    kv, block = case["kv_heads"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, length in enumerate(s["lengths"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        at = torch.arange(first, length, device="cuda")
        page, within = s["table"][r].long()[at // block], at % block
        for g in range(kv):
            k, v = (s[name].view(torch.uint8)[page, g, within].view(_E4M3).double()
                    * s["scales"][page, g, i].double()[:, None] for i, name in enumerate("kv"))
            heads = slice(g * case["heads"] // kv, (g + 1) * case["heads"] // kv)
            p = torch.softmax(s["q"][r, heads].double() @ k.t() * _softmax_scale(case), -1)
            out[r, heads] = p @ v
    return out


def _attend_work(case):
    keys = _attend_lengths(case)
    if case["window"]:
        keys = np.minimum(keys, case["window"])
    keys = int(keys.sum())
    n, h, kv, d = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim"))
    return {"bytes": 2 * keys * kv * d + 4 * n * h * d + 4 * n + (4 + 8 * kv) * (keys // case["block"]),
            "flops": 4 * keys * h * d}


_INPUTS = {"norm": _norm_inputs, "linear": _linear_inputs, "store": _store_inputs, "load": _load_inputs,
           "attend": _attend_inputs}
_PLAIN = {"norm": _norm_plain, "linear": _linear_plain, "store": _store_plain, "load": _load_plain,
          "attend": _attend_plain}
_OWN = {"norm": _norm_own, "linear": _linear_own, "store": _store_own, "load": _load_own, "attend": _attend_own}
_EXACT = {"norm": _norm_exact, "linear": _linear_exact, "store": _store_exact, "load": _load_exact,
          "attend": _attend_exact}
_WORK = {"norm": _norm_work, "linear": _linear_work, "store": _store_work, "load": _load_work,
         "attend": _attend_work}
